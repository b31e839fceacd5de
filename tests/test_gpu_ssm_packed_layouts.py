"""Packed scans: every state width, odd head widths, mixed batches of prompts
and single tokens, thousands of sequences, and cu_seqlens out of order."""
import ctypes as ct

import pytest
import torch

import gdn_hip
import ssm_cases as sc
from gdn_hip import capi
from oracle import ssm_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
ARGS = ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")


def _s0(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _cu(lengths, first=0):
    return torch.tensor([first + sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)


def _c_scan(dev, g, cu, s0, seqs, block, table=None):
    """The C entry on contiguous tensors, with guards behind what it may write:
    (y, sf, whether the guards are as they were)."""
    _, T, H, P = g["x"].shape
    G, N = g["B"].shape[2:]
    dt = 0 if g["x"].dtype == BF else 1
    a = capi.SsmInputs(**{{"B": "b", "C": "c"}.get(k, k): g[k].data_ptr() for k in ARGS if g[k] is not None},
                       x_token=H * P, dt_token=H, b_token=G * N, c_token=G * N, z_token=H * P, batch=1,
                       tokens=T, heads=H, head_dim=P, groups=G, state_dim=N, io_dtype=dt, dt_dtype=dt,
                       dt_min=0.0, dt_max=1e30)
    lib = capi.lib()
    need = lib.gdn_ssm_scan_workspace_size(ct.byref(a), seqs, block, 1)
    assert need > 0
    ws = torch.full((need + 65536,), 0x5A, dtype=torch.uint8, device=dev)
    y = torch.full((T + 64, H, P), 7.0, dtype=g["x"].dtype, device=dev)
    sf = torch.full((seqs + 1, H, N, P), 7.0, device=dev)
    assert lib.gdn_ssm_scan(ct.byref(a), y.data_ptr(), s0.data_ptr(), sf.data_ptr(), cu.data_ptr(),
                            None if table is None else table.data_ptr(), seqs, block, ws.data_ptr(), need,
                            torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    whole = bool((ws[need:] == 0x5A).all() and (y[T:] == 7).all() and (sf[seqs] == 7).all())
    return y[:T][None], sf[:seqs], whole


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H,P,G,N", [(3, 16, 1, 16), (4, 48, 2, 16), (2, 32, 2, 32), (6, 48, 2, 64),
                                     (4, 80, 1, 128), (3, 96, 3, 256), (9, 64, 1, 256), (2, 256, 2, 64),
                                     (2, 128, 1, 128), (5, 112, 1, 32)])
@pytest.mark.parametrize("block", [64, 128])
def test_layouts(dev, block, H, P, G, N, dtype):
    lengths = [130, 0, 63, 256, 1, 64, 129]
    T, n = sum(lengths), len(lengths)
    d = sc.inputs(H * P + N, 1, T, H, P, G, N, dtype, z=H % 2 == 0)
    d["dt_bias"] = d["dt_bias"] - 2
    s0 = _s0(n, n, H, N, P)
    y, S, ya, Sa = orc.ssm_packed(lengths, **{k: d[k] for k in ARGS}, s0=s0)
    g = {k: None if v is None else v.contiguous().to(dev) for k, v in d.items()}
    print(f"packed H={H} P={P} G={G} N={N} {dtype}, blocks of {block}", flush=True)
    oy, oS, whole = _c_scan(dev, g, _cu(lengths).to(dev), s0.to(dev), n, block)
    assert whole
    by, bS = sc.bounds(d, max(lengths), y, ya, Sa, dtype)
    sc.close(oy, y, by, "packed y")
    sc.close(oS, S, bS, "packed state")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N", [16, 64])
def test_mixed_batch(dev, N, dtype):
    """Mostly single tokens, some prompts that are split, in tables of
    request_blocks; a batch this wide has a record for few of its sequences."""
    lengths = [1 if i % 13 else 150 + i for i in range(120)]
    lengths[7] = lengths[60] = 0
    T, n = sum(lengths), len(lengths)
    d = sc.inputs(N, 1, T, 4, 32, 2, N, dtype)
    d["dt_bias"] = d["dt_bias"] - 2
    s0 = _s0(n, n, 4, N, 32)
    y, S, ya, Sa = orc.ssm_packed(lengths, **{k: d[k] for k in ARGS}, s0=s0)
    g = sc.to(d, dev)
    by, bS = sc.bounds(d, max(lengths), y, ya, Sa, dtype)
    for block in (64, 192, 4096):
        cu, table, _, _ = gdn_hip.request_blocks(torch.tensor(lengths, device=dev), T, block=block)
        print(f"mixed batch, blocks of {block}, N={N} {dtype}", flush=True)
        oy, oS = gdn_hip.ssm_scan(*(g[k] for k in ARGS), s0.to(dev), cu_seqlens=cu, blocks=table, block=block)
        torch.cuda.synchronize()
        sc.close(oy, y, by, "mixed y")
        sc.close(oS, S, bS, "mixed state")


def test_thousands_of_sequences(dev):
    """4100 sequences of 0 to 3 tokens and two long ones, against the recurrence."""
    lengths = [i % 4 for i in range(4100)]
    lengths[100], lengths[4000] = 200, 300
    T, n = sum(lengths), len(lengths)
    d = sc.inputs(3, 1, T, 1, 16, 1, 64, z=False)
    s0 = _s0(1, n, 1, 64, 16)
    # sequences of one length are one batch of the oracle
    y, ya = torch.zeros(T, 1, 16, dtype=torch.float64), torch.zeros(T, 1, 16, dtype=torch.float64)
    S, Sa = torch.zeros(n, 1, 64, 16, dtype=torch.float64), torch.zeros(n, 1, 64, 16, dtype=torch.float64)
    cuts = _cu(lengths)
    for m in set(lengths):
        ids = [i for i, v in enumerate(lengths) if v == m]
        rows = torch.stack([torch.arange(int(cuts[i]), int(cuts[i]) + m) for i in ids])
        part = {k: (v[0][rows] if v is not None and v.dim() > 1 else v) for k, v in d.items()}
        r = orc.ssm(**part, s0=s0[ids])
        y[rows], S[ids], ya[rows], Sa[ids] = r
    g = sc.to(d, dev)
    print(f"{n} sequences", flush=True)
    oy, oS = gdn_hip.ssm_scan(*(g[k] for k in ARGS), s0.to(dev), cu_seqlens=cuts.to(dev))
    torch.cuda.synchronize()
    by, bS = sc.bounds(d, 300, y, ya, Sa, BF)
    sc.close(oy[0], y, by, "thousands y")
    sc.close(oS, S, bS, "thousands state")


@pytest.mark.parametrize("N", [16, 64])
@pytest.mark.parametrize("block", [64, 256])
@pytest.mark.parametrize("cu", [[40, -5, 700, 130, 2000], [600, 300, 0, 500, 10], [-3, -2, -1, 0, 0],
                                [0, 500, 0, 500, 0], [90, 90, 1 << 30, -(1 << 31), 600]])
def test_unordered_stays_in_bounds(dev, cu, block, N):
    """cu_seqlens out of order or out of range: undefined values, nothing outside."""
    d = sc.inputs(1, 1, 600, 2, 32, 1, N)
    g = {k: None if v is None else v.contiguous().to(dev) for k, v in d.items()}
    print(f"cu_seqlens {cu}, blocks of {block}, N={N}", flush=True)
    assert _c_scan(dev, g, torch.tensor(cu, dtype=torch.int32, device=dev),
                   _s0(1, 4, 2, N, 32).to(dev), 4, block)[2]


def test_a_table_of_other_lengths_stays_in_bounds(dev):
    """A table of another batch of the same size: that batch's results, or
    undefined ones, and nothing outside."""
    T, n = 600, 4
    d = sc.inputs(2, 1, T, 2, 32, 1, 64)
    g = {k: None if v is None else v.contiguous().to(dev) for k, v in d.items()}
    s0 = _s0(1, n, 2, 64, 32).to(dev)
    lengths = [300, 10, 200, 90]
    table = gdn_hip.request_blocks(torch.tensor([70, 400, 0, 130], device=dev), T, block=64)[1]
    print("a table of other lengths", flush=True)
    assert _c_scan(dev, g, _cu(lengths).to(dev), s0, n, 64, table)[2]
    table = table.flip(0).contiguous()
    table[:, 1] += 37
    table[:, 2] *= 1000
    print("a table upside down", flush=True)
    assert _c_scan(dev, g, _cu(lengths).to(dev), s0, n, 64, table)[2]
