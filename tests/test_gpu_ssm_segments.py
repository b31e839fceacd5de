"""Split sequences whose segments are several 64-token chunks long: the first
pass's loop over chunks, its records, and their join, against the 64-bit
recurrence.  Decays are slow enough (0.05 to 0.99 over a segment) that what a
segment hands on is most of the next one's state."""
import pytest
import torch

import gdn_hip
import ssm_cases as sc
from oracle import ssm_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
ARGS = ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")


def _slow(*a, **kw):
    d = sc.inputs(*a, **kw)
    d["dt_bias"] = d["dt_bias"] - 3
    return d


def _s0(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _heads(d, heads, rep):
    """The inputs of some heads, each with its group."""
    out = dict(d)
    for k in ("x", "z", "dt"):
        out[k] = None if d[k] is None else d[k][:, :, heads]
    for k in ("A_log", "D", "dt_bias"):
        out[k] = d[k][heads]
    for k in "BC":
        out[k] = d[k][:, :, [h // rep for h in heads]]
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N", [64, 128, 256])
@pytest.mark.parametrize("block", [128, 192, 256])
def test_packed(dev, block, N, dtype):
    """A table of blocks of 2, 3 and 4 chunks; partial last segments, whole ones,
    sequences of one segment and of none between them."""
    lengths = [3 * block + 70, 0, 4 * block, 5, 2 * block + 1, block, 0, 5 * block - 1]
    T, n = sum(lengths), len(lengths)
    d = _slow(block + N, 1, T, 4, 64, 2, N, dtype)
    s0 = _s0(N, n, 4, N, 64)
    y, S, ya, Sa = orc.ssm_packed(lengths, **{k: d[k] for k in ARGS}, s0=s0)
    g = sc.to(d, dev)
    cu, table, _, _ = gdn_hip.request_blocks(torch.tensor(lengths, device=dev), T, block=block)
    print(f"packed segments of {block}, N={N} {dtype}", flush=True)
    oy, oS = gdn_hip.ssm_scan(*(g[k] for k in ARGS), s0.to(dev), cu_seqlens=cu, blocks=table, block=block)
    torch.cuda.synchronize()
    by, bS = sc.bounds(d, max(lengths), y, ya, Sa, dtype)
    sc.close(oy, y, by, "segments y")
    sc.close(oS, S, bS, "segments state")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,H,G,N,heads,few", [
    (1500, 64, 1, 64, [0, 31, 63], True),      # segments of 256, joined by the main pass
    (1141, 64, 8, 128, [0, 13, 63], True),     # of 192
    (1141, 32, 1, 256, [5, 31], False),        # of 128 with a state of 256
    (4096, 32, 2, 64, [0, 30], False),         # of 256, joined by a launch
    (3000, 64, 8, 128, [0, 40], False)])       # of 192
def test_fixed_length(dev, T, H, G, N, heads, few, dtype):
    """The segments that the scan chooses by itself, few and many."""
    block = gdn_hip.ssm_scan_block(T, 1, H, 64, G, N, 1)
    segs = -(-T // block)
    assert block >= 128 and (2 <= segs <= 6 if few else segs > 6)
    d = _slow(T + N, 1, T, H, 64, G, N, dtype)
    s0 = _s0(T, 1, H, N, 64)
    part = _heads(d, heads, H // G)
    y, S, ya, Sa = orc.ssm(**part, s0=s0[:, heads])
    g = sc.to(d, dev)
    print(f"{segs} segments of {block}, T={T} N={N} {dtype}", flush=True)
    oy, oS = gdn_hip.ssm_scan(*(g[k] for k in ARGS), s0.to(dev))
    torch.cuda.synchronize()
    by, bS = sc.bounds(part, T, y, ya, Sa, dtype)
    sc.close(oy[:, :, heads], y, by, "segments y")
    sc.close(oS[:, heads], S, bS, "segments state")
