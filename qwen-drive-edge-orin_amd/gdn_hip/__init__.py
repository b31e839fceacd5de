"""gdn_hip: MI355X (gfx950) gated-delta-rule ops.

The compiled pieces live next to this file:
  libgdn_hip.so            C ABI (include/gdn_hip.h)
  deltanet_chunk_hip*.so   torch extension over it, the drop-in for the
                           reference's deltanet_chunk_cuda / _tco modules
                           (kernels/torch_binding.cpp:113-131)

``load()`` returns the extension module, whose ops are

  chunk_prefill(q, k, v, g, beta, s0=None, *, cu_seqlens=None, qk_l2norm=False,
                checked=False)                         -> [o, final_state]
  chunk_prefill_debug(...)  -> [o, final_state, T, A, cumsum_g, T_post_leaf, M, S_chunk]
  recurrent_step(q, k, v, g, beta, state, *, qk_l2norm=False) -> o
                                                        (state updated in place)
  recurrent_step_new(q, k, v, g, beta, state0=None, *, qk_l2norm=False) -> [o, state]
  chunk_prefill_norm(q, k, v, g, beta, z, weight, s0=None, *, eps=1e-6, checked=False,
                     fused=False)
                          -> [gated_rmsnorm(o, z, weight), final_state]
  chunk_prefill_fused(q, k, v, a, b, A_log, dt_bias, state) -> o
                          raw q/k/v and gate inputs     (state updated in place)
  gated_rmsnorm(x, z, weight, eps=1e-6) -> y
  causal_conv1d_fwd(x, weight, bias=None, silu=False) -> y      x, y [B, D, T]
  causal_conv1d_update(x, conv_state, weight, bias=None, silu=False, *, slots=None) -> y
                                                  (conv_state updated in place)

State-space layers (x, z [B, T, H, P], dt [B, T, H], B, C [B, T, G, N], states
fp32 [B, H, N, P]; A_log, D, dt_bias fp32 [H]):

  ssm_scan(x, dt, A_log, B, C, D=None, z=None, dt_bias=None, s0=None, *,
           cu_seqlens=None, blocks=None, block=0, dt_min=0, dt_max=inf) -> [y, final_state]
  ssm_step(x, dt, A_log, B, C, state, D=None, z=None, dt_bias=None, *, slots=None,
           dt_min=0, dt_max=inf) -> y             (state updated in place)
  causal_conv1d_prefill(x, weight, bias=None, state0=None, *, silu=False,
                        cu_seqlens=None, state_len=0) -> [y [B, D, T], state [N, D, L]]
  request_blocks(lengths, total_tokens, *, block=64, slots=None)
                          -> [cu_seqlens, blocks, token_slots, token_pos]
  ssm_scan_block(tokens, batch, heads, head_dim, groups, state_dim, num_seqs) -> block
                          for request_blocks, whose table several scans may share
  gated_groupnorm(x, z, weight, groups, eps=1e-6, *, gate_first=True) -> y

slots [B]: the states are a pool and row b uses state slots[b]; a slot outside
the pool is a row without a request (zeros, no state changes).

``checked=True`` synchronises after the call and raises when one of the
scan's bounded waits gave up (o and the state would then be incomplete);
the default leaves the call asynchronous.

There is no fallback: if the extension is not built, ``load()`` raises.
Build with ``python qwen-drive-edge-orin_amd/build.py``.
"""
from __future__ import annotations

import importlib
import math
from pathlib import Path

HERE = Path(__file__).resolve().parent
LIB_PATH = HERE / "libgdn_hip.so"
EXT_NAME = "deltanet_chunk_hip"

_mod = None


def ext_path() -> Path | None:
    hits = sorted(HERE.glob(f"{EXT_NAME}.cpython*.so"))
    return hits[0] if hits else None


def load():
    """Import the in-tree torch extension (raises ImportError when missing)."""
    global _mod
    if _mod is None:
        if not LIB_PATH.exists() or ext_path() is None:
            raise ImportError(
                f"gdn_hip native code is not built under {HERE}; run "
                "`python qwen-drive-edge-orin_amd/build.py`")
        import torch  # noqa: F401  (loads libc10/libtorch the extension links)
        _mod = importlib.import_module(f"{__name__}.{EXT_NAME}")
    return _mod


def chunk_prefill(q, k, v, g, beta, s0=None, *, cu_seqlens=None, qk_l2norm=False,
                  checked=False):
    return load().chunk_prefill(q, k, v, g, beta, s0, cu_seqlens=cu_seqlens, qk_l2norm=qk_l2norm,
                                checked=checked)


def chunk_prefill_debug(q, k, v, g, beta, s0=None, *, cu_seqlens=None):
    return load().chunk_prefill_debug(q, k, v, g, beta, s0, cu_seqlens=cu_seqlens)


def chunk_prefill_norm(q, k, v, g, beta, z, weight, s0=None, *, eps=1e-6, checked=False,
                       fused=False):
    return load().chunk_prefill_norm(q, k, v, g, beta, z, weight, s0, eps=eps, checked=checked,
                                     fused=fused)


def chunk_prefill_fused(q, k, v, a, b, A_log, dt_bias, state):
    return load().chunk_prefill_fused(q, k, v, a, b, A_log, dt_bias, state)


def recurrent_step(q, k, v, g, beta, state, *, qk_l2norm=False):
    return load().recurrent_step(q, k, v, g, beta, state, qk_l2norm=qk_l2norm)


def recurrent_step_new(q, k, v, g, beta, state0=None, *, qk_l2norm=False):
    return load().recurrent_step_new(q, k, v, g, beta, state0, qk_l2norm=qk_l2norm)


def gated_rmsnorm(x, z, weight, eps=1e-6):
    return load().gated_rmsnorm(x, z, weight, eps)


def causal_conv1d_fwd(x, weight, bias=None, silu=False):
    return load().causal_conv1d_fwd(x, weight, bias, silu)


def causal_conv1d_update(x, conv_state, weight, bias=None, silu=False, *, slots=None):
    if slots is None:
        return load().causal_conv1d_update(x, conv_state, weight, bias, silu)
    return load().causal_conv1d_update_slots(x, conv_state, weight, bias, silu, slots)


def ssm_scan(x, dt, A_log, B, C, D=None, z=None, dt_bias=None, s0=None, *, cu_seqlens=None,
             blocks=None, block=0, dt_min=0.0, dt_max=math.inf):
    return load().ssm_scan(x, dt, A_log, B, C, D, z, dt_bias, s0, cu_seqlens=cu_seqlens,
                           blocks=blocks, block=block, dt_min=dt_min, dt_max=dt_max)


def ssm_scan_block(tokens, batch, heads, head_dim, groups, state_dim, num_seqs):
    return load().ssm_scan_block(tokens, batch, heads, head_dim, groups, state_dim, num_seqs)


def ssm_step(x, dt, A_log, B, C, state, D=None, z=None, dt_bias=None, *, slots=None, dt_min=0.0,
             dt_max=math.inf):
    return load().ssm_step(x, dt, A_log, B, C, state, D, z, dt_bias, slots=slots, dt_min=dt_min,
                           dt_max=dt_max)


def causal_conv1d_prefill(x, weight, bias=None, state0=None, *, silu=False, cu_seqlens=None,
                          state_len=0):
    return load().causal_conv1d_prefill(x, weight, bias, state0, silu=silu, cu_seqlens=cu_seqlens,
                                        state_len=state_len)


def request_blocks(lengths, total_tokens, *, block=64, slots=None):
    return load().request_blocks(lengths, total_tokens, block=block, slots=slots)


def gated_groupnorm(x, z, weight, groups, eps=1e-6, *, gate_first=True):
    return load().gated_groupnorm(x, z, weight, groups, eps, gate_first=gate_first)
