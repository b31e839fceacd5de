"""64-bit CPU oracle of the state-space operators: the token recurrence of the
selective scan, the causal conv that carries a state, the tables of a packed
batch and the grouped gated norm.  Written from the formulas, token by token;
"parity unpinned": no reference file holds outputs for these operators.

The scan also returns, next to y and the state, the same recurrences over
absolute values: what a rounding error of the arithmetic is measured against.
"""
from __future__ import annotations

import torch


def _silu(x):
    return x / (1 + torch.exp(-x))


def softplus(x):
    return torch.where(x > 30, x, torch.log1p(torch.exp(torch.clamp(x, max=30.0))))


def ssm(x, dt, A_log, B, C, D=None, z=None, dt_bias=None, s0=None, dt_min=0.0,
        dt_max=float("inf")):
    """One batch: x, z [B, T, H, P], dt [B, T, H], B, C [B, T, G, N], s0 [B, H, N, P].
    Returns (y, S, y_abs, S_abs) in float64."""
    x, dt, A_log, B, C = (t.double().cpu() for t in (x, dt, A_log, B, C))
    nb, T, H, P = x.shape
    rep, N = H // B.shape[2], B.shape[3]
    B, C = B.repeat_interleave(rep, 2), C.repeat_interleave(rep, 2)
    bias = torch.zeros(H) if dt_bias is None else dt_bias.cpu()
    d = softplus(dt + bias.double()).clamp(dt_min, dt_max)
    a = torch.exp(-torch.exp(A_log) * d)
    S = torch.zeros(nb, H, N, P, dtype=torch.float64) if s0 is None else s0.double().cpu().clone()
    Sa = S.abs()
    Dv = torch.zeros(H, dtype=torch.float64) if D is None else D.double().cpu()
    y, ya = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        u = B[:, t, :, :, None] * (d[:, t, :, None] * x[:, t])[:, :, None, :]
        S = a[:, t, :, None, None] * S + u
        Sa = a[:, t, :, None, None] * Sa + u.abs()
        y[:, t] = (C[:, t, :, :, None] * S).sum(2) + Dv[:, None] * x[:, t]
        ya[:, t] = (C[:, t, :, :, None].abs() * Sa).sum(2) + (Dv[:, None] * x[:, t]).abs()
    if z is not None:
        g = _silu(z.double().cpu())
        y, ya = y * g, ya * g.abs()
    return y, S, ya, Sa


def ssm_packed(lengths, x, dt, A_log, B, C, D=None, z=None, dt_bias=None, s0=None, **kw):
    """The same over the packed sequences of one row; rows behind the last are zeros."""
    outs = [torch.zeros(x.shape, dtype=torch.float64), [], torch.zeros(x.shape, dtype=torch.float64), []]
    lo = 0
    for i, n in enumerate(lengths):
        cut = [None if t is None else t[:, lo:lo + n] for t in (x, dt, B, C, z)]
        r = ssm(cut[0], cut[1], A_log, cut[2], cut[3], D, cut[4], dt_bias,
                torch.zeros(1, x.shape[2], B.shape[3], x.shape[3]) if s0 is None else s0[i:i + 1], **kw)
        outs[0][:, lo:lo + n], outs[2][:, lo:lo + n] = r[0], r[2]
        outs[1].append(r[1])
        outs[3].append(r[3])
        lo += n
    return outs[0], torch.cat(outs[1]), outs[2], torch.cat(outs[3])


def conv_prefill(x, w, bias, state0, silu, lengths=None, state_len=0):
    """x [B, D, T], state0 [N, D, L] or None.  Returns (y, state, y_abs) in
    float64, y_abs the sum of absolute terms in front of the activation."""
    L = state0.shape[2] if state0 is not None else (state_len or w.shape[1])
    K = w.shape[1]
    x, w = x.double().cpu(), w.double().cpu()
    rows = [x[b] for b in range(x.shape[0])] if lengths is None else \
        list(torch.split(x[0][:, :sum(lengths)], lengths, dim=1))
    y, ya, states = [], [], []
    for i, r in enumerate(rows):
        old = torch.zeros(x.shape[1], L, dtype=torch.float64) if state0 is None else state0[i].double().cpu()
        line = torch.cat([old, r], dim=1)
        n = r.shape[1]
        acc = torch.zeros(x.shape[1], n, dtype=torch.float64)
        mag = torch.zeros_like(acc)
        if bias is not None:
            acc += bias.double().cpu()[:, None]
            mag += bias.double().cpu().abs()[:, None]
        for j in range(K):
            term = w[:, j:j + 1] * line[:, L - K + 1 + j:L - K + 1 + j + n]
            acc, mag = acc + term, mag + term.abs()
        y.append(_silu(acc) if silu else acc)
        ya.append(mag)
        states.append(line[:, line.shape[1] - L:])
    if lengths is None:
        return torch.stack(y), torch.stack(states), torch.stack(ya)
    return torch.cat(y, 1)[None], torch.stack(states), torch.cat(ya, 1)[None]


def request_blocks(lengths, total, block, slots=None):
    """Lists: cu_seqlens, blocks, token_slots, token_pos."""
    cu, table, slot, pos = [0], [], [], []
    for n, want in enumerate(lengths):
        lo = cu[-1]
        hi = min(lo + max(want, 0), total)
        cu.append(hi)
        starts = list(range(lo, hi, block)) or [lo]
        table += [[n, t, min(hi - t, block), i] for i, t in enumerate(starts)]
        slot += [n if slots is None else slots[n]] * (hi - lo)
        pos += list(range(hi - lo))
    table += [[-1, 0, 0, 0]] * (total // block + len(lengths) - len(table))
    slot += [-1] * (total - cu[-1])
    pos += [0] * (total - cu[-1])
    return cu, table, slot, pos


def gated_groupnorm(x, z, w, groups, eps, gate_first=True):
    x, g, w = x.double().cpu(), _silu(z.double().cpu()), w.double().cpu()
    u = x * g if gate_first else x
    v = u.reshape(*u.shape[:-1], groups, -1)
    u = (v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)).reshape(u.shape) * w
    return u if gate_first else u * g
