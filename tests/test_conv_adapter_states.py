"""The causal_conv1d adapter's checks of carried states, on the CPU: what does
not fit is refused rather than dropped or broadcast."""
import pytest
import torch

from test_conv_adapter import _adapter


def _args():
    return torch.zeros(2, 64, 5, dtype=torch.bfloat16), torch.zeros(64, 4, dtype=torch.bfloat16)


def test_final_states_out_without_final_states():
    with pytest.raises(ValueError, match="return_final_states"):
        _adapter().causal_conv1d_fn(*_args(), final_states_out=torch.zeros(2, 64, 3, dtype=torch.bfloat16))


@pytest.mark.parametrize("shape", [(2, 64, 4), (1, 64, 3), (2, 64, 1), (3, 2, 64, 3), (2, 3, 64)])
def test_states_of_another_shape(shape):
    """Among them shapes that a copy would broadcast to, or from."""
    m, st = _adapter(), torch.zeros(*shape, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="final_states_out must be"):
        m.causal_conv1d_fn(*_args(), return_final_states=True, final_states_out=st)
    with pytest.raises(ValueError, match="initial_states must be"):
        m.causal_conv1d_fn(*_args(), initial_states=st)


def test_states_that_fit_reach_the_device_check():
    st = torch.zeros(2, 64, 3, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        _adapter().causal_conv1d_fn(*_args(), initial_states=st, return_final_states=True, final_states_out=st)
