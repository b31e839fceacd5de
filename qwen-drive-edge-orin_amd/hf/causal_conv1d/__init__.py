"""``causal_conv1d_fn`` / ``causal_conv1d_update`` with the calling
convention transformers uses for the causal-conv1d package
(models/qwen3_5/modeling_qwen3_5.py:199-240 for the torch fallbacks,
457-476 for the calls), backed by the gfx950 conv ops of ``gdn_hip``.

transformers imports ``causal_conv1d`` and takes these two functions when the
import succeeds, so putting the directory that holds this package on
``sys.path`` routes the Qwen3.5 gated-delta layers' convolutions here.

x is ``[B, D, T]`` (the update also takes ``[B, D]``), weight ``[D, K]`` or
``[D, 1, K]`` with K in 2..4, bias ``[D]`` or None, conv_state ``[B, D, L]``
with L in K-1..8 (updated in place).  x must be bf16 or fp16 and weight/bias
of x's dtype or fp32.  Outputs match the torch fallbacks' dtype steps: the
convolution in the weight dtype with an fp32 sum, SiLU in fp32, rounded to
x's dtype.  With initial states or asked for final ones, ``causal_conv1d_fn``
runs the form that carries them (one rounding, at the end; states ``[B, D,
K - 1]``), and ``conv_state_indices`` ``[B]`` makes conv_state a pool (an index
outside it is a row without a request: zeros, no state changes).  Features the
kernels do not implement (``seq_idx``, ``cache_seqlens``, activations other
than SiLU) raise; there is no silent fallback.
"""
from __future__ import annotations

import sys
from pathlib import Path

_PKG_DIR = Path(__file__).resolve().parents[2]   # .../qwen-drive-edge-orin_amd
if str(_PKG_DIR) not in sys.path:
    sys.path.insert(0, str(_PKG_DIR))

import gdn_hip  # noqa: E402

__all__ = ["causal_conv1d_fn", "causal_conv1d_update"]


def _silu(activation) -> bool:
    if activation is None:
        return False
    if activation in ("silu", "swish"):
        return True
    raise NotImplementedError(f"activation {activation!r} (only None, 'silu', 'swish')")


def _weight(weight):
    if weight.dim() == 3 and weight.shape[1] == 1:
        weight = weight.squeeze(1)
    if weight.dim() != 2:
        raise ValueError("weight must be [D, K] or [D, 1, K]")
    return weight


def _on_device(**tensors):
    for name, t in tensors.items():
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{name} must be on the HIP device (the ops have no CPU path)")


def causal_conv1d_fn(x, weight, bias=None, seq_idx=None, initial_states=None,
                     return_final_states=False, final_states_out=None, activation=None):
    """Causal depthwise conv1d over x [B, D, T]; returns [B, D, T] in x's
    dtype (a transposed view of a contiguous [B, T, D] buffer), and with
    return_final_states the pair of it and the last K - 1 tokens [B, D, K - 1]
    (in final_states_out where that is given)."""
    if seq_idx is not None:
        raise NotImplementedError("seq_idx is not supported")
    silu = _silu(activation)
    if final_states_out is not None and not return_final_states:
        raise ValueError("final_states_out goes with return_final_states=True")
    if x.dim() != 3:
        raise ValueError("x must be [B, D, T]")
    weight = _weight(weight)
    states = (x.shape[0], x.shape[1], weight.shape[1] - 1)
    for name, t in (("initial_states", initial_states), ("final_states_out", final_states_out)):
        if t is not None and tuple(t.shape) != states:
            raise ValueError(f"{name} must be [B, D, K - 1], here {list(states)}")
    _on_device(x=x, weight=weight, bias=bias, initial_states=initial_states,
               final_states_out=final_states_out)
    if initial_states is None and not return_final_states:
        return gdn_hip.causal_conv1d_fwd(x, weight, bias, silu)
    y, final = gdn_hip.causal_conv1d_prefill(x, weight, bias, initial_states, silu=silu,
                                             state_len=weight.shape[1] - 1)
    if not return_final_states:
        return y
    if final_states_out is not None:
        final = final_states_out.copy_(final)
    return y, final


def causal_conv1d_update(x, conv_state, weight, bias=None, activation=None, cache_seqlens=None,
                         conv_state_indices=None):
    """Decode step: x [B, D, T] or [B, D] is appended to conv_state (updated
    in place); returns the outputs for x's tokens in x's shape and dtype."""
    if cache_seqlens is not None:
        raise NotImplementedError("cache_seqlens is not supported")
    silu = _silu(activation)
    _on_device(x=x, conv_state=conv_state, weight=weight, bias=bias)
    squeeze = x.dim() == 2
    if squeeze:
        x = x.unsqueeze(-1)
    if x.dim() != 3:
        raise ValueError("x must be [B, D, T] or [B, D]")
    if conv_state_indices is None:
        y = gdn_hip.causal_conv1d_update(x, conv_state, _weight(weight), bias, silu)
    else:
        y = gdn_hip.causal_conv1d_update(x, conv_state, _weight(weight), bias, silu,
                                         slots=conv_state_indices)
    return y.squeeze(-1) if squeeze else y
