"""The causal_conv1d adapter's carried states and state pools, on the GPU,
against the 64-bit oracle and the op itself."""
import importlib
import sys
from pathlib import Path

import pytest
import torch

import ssm_cases as sc
from oracle import ssm_oracle as orc

pytestmark = pytest.mark.gpu

HF_DIR = Path(__file__).resolve().parent.parent / "qwen-drive-edge-orin_amd" / "hf"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def adapter():
    """Imported, then dropped from sys.modules again: transformers, imported
    later in this process, must not find it."""
    before = set(sys.modules)
    sys.path.insert(0, str(HF_DIR))
    try:
        return importlib.import_module("causal_conv1d")
    finally:
        sys.path.remove(str(HF_DIR))
        for name in set(sys.modules) - before:
            if name.split(".")[0] == "causal_conv1d":
                del sys.modules[name]


def test_states(adapter, dev):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 33, 64, generator=g).to(BF).transpose(1, 2)
    w = torch.randn(64, 4, generator=g).to(BF)
    s0 = torch.randn(2, 64, 3, generator=g).to(BF)
    ref, st, mag = orc.conv_prefill(x, w, None, s0, True)
    xd, wd, sd = x.to(dev), w.to(dev), s0.to(dev)
    y, fin = adapter.causal_conv1d_fn(xd, wd[:, None], None, initial_states=sd,
                                      return_final_states=True, activation="silu")
    torch.cuda.synchronize()
    # one rounding and an fp32 sum of four terms (SiLU's slope is at most 1.1)
    sc.close(y, ref, 2.0 ** -8 * ref.abs() + 2.0 ** -19 * mag + 1e-30, "adapter states y")
    assert torch.equal(fin.double().cpu(), st)
    out = torch.empty_like(fin)
    y2, fin2 = adapter.causal_conv1d_fn(xd, wd, None, initial_states=sd, return_final_states=True,
                                        final_states_out=out, activation="silu")
    only = adapter.causal_conv1d_fn(xd, wd, None, initial_states=sd, activation="silu")
    torch.cuda.synchronize()
    assert fin2 is out and torch.equal(out, fin) and torch.equal(y2, y) and torch.equal(only, y)


def test_pool(adapter, dev):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 64, generator=g).to(BF).to(dev)
    w = torch.randn(64, 4, generator=g).to(BF).to(dev)
    pool = torch.randn(5, 64, 4, generator=g).to(BF).to(dev)
    st = pool[[4, 1]].clone()
    y = adapter.causal_conv1d_update(x, pool, w, None, "silu",
                                     conv_state_indices=torch.tensor([4, -1, 1], device=dev))
    ref = adapter.causal_conv1d_update(x[[0, 2]], st, w, None, "silu")
    torch.cuda.synchronize()
    assert torch.equal(y[[0, 2]], ref) and (y[1] == 0).all() and torch.equal(pool[[4, 1]], st)
