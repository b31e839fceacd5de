"""GPU parity of the state-space scan and step against the 64-bit recurrence
(oracle/ssm_oracle.py), elementwise, at bounds derived in ssm_cases.bounds."""
import pytest
import torch

import gdn_hip
import ssm_cases as sc
from oracle import ssm_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _cu(lengths, dev):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32,
                        device=dev)


def _s0(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _check_scan(dev, d, s0, dtype, tag, **kw):
    T = d["x"].shape[1]
    y, S, ya, Sa = orc.ssm(d["x"], d["dt"], d["A_log"], d["B"], d["C"], d["D"], d["z"],
                           d["dt_bias"], s0, **kw)
    g = sc.to(d, dev)
    print(tag, flush=True)
    oy, oS = gdn_hip.ssm_scan(g["x"], g["dt"], g["A_log"], g["B"], g["C"], g["D"], g["z"],
                              g["dt_bias"], None if s0 is None else s0.to(dev), **kw)
    torch.cuda.synchronize()
    assert oy.dtype == dtype and oS.dtype == torch.float32
    by, bS = sc.bounds(d, T, y, ya, Sa, dtype)
    sc.close(oy, y, by, tag + " y")
    sc.close(oS, S, bS, tag + " state")
    return oy, oS


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300])
def test_scan_lengths(dev, T):
    d = sc.inputs(T, 2, T, 4, 64, 2, 128)
    _check_scan(dev, d, _s0(T, 2, 4, 128, 64), BF, f"scan T={T}")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H,P,G,N", [(3, 16, 1, 16), (2, 32, 2, 32), (6, 48, 2, 64), (8, 64, 1, 64),
                                     (5, 64, 5, 128), (4, 80, 1, 128), (2, 128, 1, 128),
                                     (3, 96, 3, 256), (9, 64, 1, 256), (2, 256, 2, 64)])
def test_scan_layouts(dev, H, P, G, N, dtype):
    d = sc.inputs(H * P + N, 1, 150, H, P, G, N, dtype, z=H % 2 == 0)
    _check_scan(dev, d, _s0(3, 1, H, N, P) if P != 80 else None, dtype,
                f"scan H={H} P={P} G={G} N={N} {dtype}")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scan_fast_decay_and_limits(dev, dtype):
    """Decays down to e^-100 a token, dt in fp32, dt limits."""
    d = sc.inputs(7, 1, 200, 4, 64, 2, 128, dtype, dt_dtype=torch.float32, slow=False)
    d["dt"] = d["dt"] * 4
    _check_scan(dev, d, _s0(8, 1, 4, 128, 64), dtype, f"scan fast {dtype}")
    _check_scan(dev, d, None, dtype, f"scan limits {dtype}", dt_min=0.02, dt_max=0.6)


def test_scan_reset_token(dev):
    """One token's decay wipes the state (log decay -1e5): what follows it in its
    chunk is as exact as without."""
    d = sc.inputs(9, 1, 128, 2, 64, 1, 128, dt_dtype=torch.float32)
    d["dt"][:, 70] = 1e5
    d["x"] = d["x"].clone()
    d["x"][:, 70] = 0
    _check_scan(dev, d, _s0(9, 1, 2, 128, 64), BF, "scan reset")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scan_resets_and_weak_decays(dev, dtype):
    """Every other token or so wipes the state, the others hardly decay it.

    The weight of one of 16 tokens for another of them is a difference of two
    sums of base-2 log decays, each held at -150 or above: sums of 2, 4, 8 and
    16 tokens below 512, 1024, 2048 and 4096 in magnitude are off by up to
    2^-16, 2^-15, 2^-14 and 2^-13, so the difference by 2 (15/8) 2^-13 and the
    weight by that times ln 2, relative: below 2^-11.5.  Sums of whole 16s keep
    the sign, and count only where they are no reset."""
    d = sc.inputs(21, 1, 330, 3, 64, 1, 128, dtype, dt_dtype=torch.float32)
    wipe = torch.rand(330, generator=torch.Generator().manual_seed(5)) < 0.5
    d["dt"] = torch.where(wipe[None, :, None], torch.tensor(1e4), d["dt"] - 2)
    d["x"] = torch.where(wipe[None, :, None, None], torch.zeros((), dtype=dtype), d["x"])
    s0 = _s0(4, 1, 3, 128, 64)
    y, S, ya, Sa = orc.ssm(d["x"], d["dt"], d["A_log"], d["B"], d["C"], d["D"], d["z"], d["dt_bias"], s0)
    g = sc.to(d, dev)
    oy, oS = gdn_hip.ssm_scan(g["x"], g["dt"], g["A_log"], g["B"], g["C"], g["D"], g["z"], g["dt_bias"], s0.to(dev))
    torch.cuda.synchronize()
    by, bS = sc.bounds(d, 330, y, ya, Sa, dtype)
    sc.close(oy, y, by + 2.0 ** -11.5 * ya, f"resets {dtype} y")
    sc.close(oS, S, bS, f"resets {dtype} state")


def test_scan_large_and_small_values(dev):
    """bf16 values far outside 16-bit floats of five exponent bits."""
    for f in (1e10, 1e-10):
        d = sc.inputs(11, 1, 130, 2, 64, 1, 64)
        d = {k: (v * f if k in "xBC" else v) for k, v in d.items()}
        _check_scan(dev, d, None, BF, f"scan values x {f}")


@pytest.mark.parametrize("lengths", [[5], [0, 64, 0, 1], [130, 0, 63, 200, 64, 1, 0], [1] * 40, [0, 0]])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_scan_packed(dev, lengths, dtype):
    T = sum(lengths)
    n = len(lengths)
    d = sc.inputs(T + n, 1, T, 4, 64, 2, 128, dtype)
    s0 = _s0(n, n, 4, 128, 64)
    y, S, ya, Sa = orc.ssm_packed(lengths, **{k: d[k] for k in ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")}, s0=s0)
    g = sc.to(d, dev)
    print(f"packed {lengths} {dtype}", flush=True)
    oy, oS = gdn_hip.ssm_scan(g["x"], g["dt"], g["A_log"], g["B"], g["C"], g["D"], g["z"],
                              g["dt_bias"], s0.to(dev), cu_seqlens=_cu(lengths, dev))
    torch.cuda.synchronize()
    if T:
        by, bS = sc.bounds(d, max(lengths), y, ya, Sa, dtype)
        sc.close(oy, y, by, f"packed {lengths} y")
        sc.close(oS, S, bS, f"packed {lengths} state")
    else:
        assert torch.equal(oS.cpu(), s0)


def test_scan_packed_with_a_table(dev):
    """The table of request_blocks gives what the scan's own gives, for the block it chose."""
    lengths = [700, 0, 65, 1, 300]
    d = sc.to(sc.inputs(1, 1, sum(lengths), 8, 64, 2, 128), dev)
    args = [d[k] for k in ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")]
    lens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    block = gdn_hip.ssm_scan_block(sum(lengths), 1, 8, 64, 2, 128, len(lengths))
    cu, table, slot, pos = gdn_hip.request_blocks(lens, sum(lengths), block=block)
    y0, s0 = gdn_hip.ssm_scan(*args, cu_seqlens=cu)
    y1, s1 = gdn_hip.ssm_scan(*args, cu_seqlens=cu, blocks=table, block=block)
    torch.cuda.synchronize()
    assert torch.equal(y0, y1) and torch.equal(s0, s1)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,H,N", [(1250, 2, 64), (1250, 1, 256)])
def test_scan_many_segments(dev, T, H, N, dtype):
    """More segments than the main pass joins by itself."""
    assert gdn_hip.ssm_scan_block(T, 1, H, 64, 1, N, 1) * 6 < T
    d = sc.inputs(T, 1, T, H, 64, 1, N, dtype)
    d["dt_bias"] = d["dt_bias"] - 3
    _check_scan(dev, d, _s0(T, 1, H, N, 64), dtype, f"scan T={T} N={N} {dtype}")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scan_many_segments_packed(dev, dtype):
    """Sequences of up to 9 segments in a table of 64-token blocks, enough
    records that the join takes 16 bytes a thread."""
    lengths = [520, 0, 410, 64, 65, 129]
    T, n = sum(lengths), len(lengths)
    d = sc.inputs(T, 1, T, 16, 64, 2, 128, dtype)
    d["dt_bias"] = d["dt_bias"] - 3
    s0 = _s0(n, n, 16, 128, 64)
    y, S, ya, Sa = orc.ssm_packed(lengths, **{k: d[k] for k in ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")}, s0=s0)
    g = sc.to(d, dev)
    cu, table, _, _ = gdn_hip.request_blocks(torch.tensor(lengths, device=dev), T)
    print(f"packed segments {dtype}", flush=True)
    oy, oS = gdn_hip.ssm_scan(g["x"], g["dt"], g["A_log"], g["B"], g["C"], g["D"], g["z"],
                              g["dt_bias"], s0.to(dev), cu_seqlens=cu, blocks=table, block=64)
    torch.cuda.synchronize()
    by, bS = sc.bounds(d, max(lengths), y, ya, Sa, dtype)
    sc.close(oy, y, by, "packed segments y")
    sc.close(oS, S, bS, "packed segments state")


def test_scan_more_sequences_than_one_group_sums(dev):
    """Past 4096 sequences the table takes two launches."""
    lengths = [1 + (i % 3) for i in range(4100)]
    T = sum(lengths)
    d = sc.to(sc.inputs(3, 1, T, 1, 16, 1, 64, z=False), dev)
    args = [d[k] for k in ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")]
    y, s = gdn_hip.ssm_scan(*args, cu_seqlens=_cu(lengths, dev))
    torch.cuda.synchronize()
    # sequences of one length as a batch
    cuts = torch.tensor([0] + lengths).cumsum(0)
    for n in (1, 2, 3):
        ids = [i for i, m in enumerate(lengths) if m == n]
        rows = torch.stack([torch.arange(int(cuts[i]), int(cuts[i]) + n) for i in ids]).to(dev)
        part = [a[0][rows] if a is not None and a.dim() > 1 else a for a in args]
        yb, sb = gdn_hip.ssm_scan(*part)
        torch.cuda.synchronize()
        assert torch.equal(y[0][rows], yb) and torch.equal(s[ids], sb)


def test_infinite_and_nan_steps(dev):
    """dt of -infinity or the type's lowest value is a step of 0 (the token
    changes nothing); NaN shows in the outputs from its token on."""
    for dtype in (BF, HF):
        d = sc.inputs(21, 1, 70, 2, 64, 1, 64, dtype)
        d["dt"] = d["dt"].clone()
        d["dt"][:, 20] = -float("inf")
        d["dt"][:, 40] = torch.finfo(dtype).min
        _check_scan(dev, d, _s0(2, 1, 2, 64, 64), dtype, f"masked steps {dtype}")
        g = sc.to(d, dev)
        st, fin = _s0(2, 1, 2, 64, 64).to(dev), None
        args = [g[k][:, 20:21] for k in ("x", "dt")] + [g["A_log"]] + [g[k][:, 20:21] for k in ("B", "C")]
        before = st.clone()
        gdn_hip.ssm_step(*args, st, dt_bias=g["dt_bias"])
        assert torch.equal(st, before)
        g["dt"][:, 66] = float("nan")
        y, fin = gdn_hip.ssm_scan(g["x"], g["dt"], g["A_log"], g["B"], g["C"], g["D"], g["z"], g["dt_bias"])
        torch.cuda.synchronize()
        assert torch.isfinite(y[:, :66]).all() and torch.isnan(y[:, 66:]).all() and torch.isnan(fin).all()


def test_fp16_extreme_scales(dev):
    """fp16 inputs at both ends of the type, steps up to 1e4: the scales in
    front of the products keep every part in range."""
    for fx, fb, fc, lift in ((2000.0, 100.0, 5e-6, 0.0), (1e-4, 1e-3, 1e3, -8.0), (1e-3, 1.0, 1.0, 9.2)):
        d = sc.inputs(31, 1, 140, 2, 64, 1, 64, HF, dt_dtype=torch.float32)
        d["x"], d["B"], d["C"] = d["x"] * fx, d["B"] * fb, d["C"] * fc
        assert all(torch.isfinite(d[k]).all() for k in "xBC")
        d["dt_bias"] = d["dt_bias"] + lift if lift < 9 else d["dt_bias"] + 10.0 ** 4
        d["D"] = d["D"] / fx
        _check_scan(dev, d, None, HF, f"fp16 scales x {fx} B {fb} step {lift}")


def test_scan_rows_behind_the_last_sequence(dev):
    """C entry: y rows behind the last packed sequence are left as they were."""
    import ctypes as ct

    from gdn_hip import capi
    lengths, T = [70, 9], 100
    d = sc.to(sc.inputs(2, 1, T, 4, 64, 1, 64), dev)
    x, dt, b, c = (d[k].contiguous() for k in ("x", "dt", "B", "C"))
    cu = _cu(lengths, dev)
    a = capi.SsmInputs(x=x.data_ptr(), dt=dt.data_ptr(), b=b.data_ptr(), c=c.data_ptr(),
                       A_log=d["A_log"].data_ptr(), x_token=256, dt_token=4, b_token=64, c_token=64,
                       batch=1, tokens=T, heads=4, head_dim=64, groups=1, state_dim=64, io_dtype=0,
                       dt_dtype=0, dt_min=0.0, dt_max=1e30)
    lib = capi.lib()
    block = lib.gdn_ssm_scan_block(ct.byref(a), 2)
    need = lib.gdn_ssm_scan_workspace_size(ct.byref(a), 2, block, 1)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    y = torch.full((T, 4, 64), 7.0, dtype=BF, device=dev)
    sf = torch.empty(2, 4, 64, 64, device=dev)
    assert lib.gdn_ssm_scan(ct.byref(a), y.data_ptr(), None, sf.data_ptr(), cu.data_ptr(), None, 2,
                            block, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert (y[79:] == 7.0).all() and not (y[:79] == 7.0).all(dim=-1).any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,T,H,P,G,N,z", [(1, 1, 4, 64, 1, 128, True), (3, 1, 5, 64, 5, 128, False),
                                           (2, 4, 6, 80, 2, 64, True), (2, 2, 3, 16, 1, 16, True),
                                           (1, 3, 2, 256, 1, 32, True), (2, 1, 3, 48, 3, 256, True),
                                           (70, 1, 8, 128, 2, 64, True)])
def test_step(dev, B, T, H, P, G, N, z, dtype):
    d = sc.inputs(B + T + N, B, T, H, P, G, N, dtype, z=z)
    s0 = _s0(4, B, H, N, P)
    y, S, ya, Sa = orc.ssm(**d, s0=s0)
    g = sc.to(d, dev)
    st = s0.to(dev)
    print(f"step B={B} T={T} H={H} P={P} G={G} N={N} {dtype}", flush=True)
    oy = gdn_hip.ssm_step(g["x"], g["dt"], g["A_log"], g["B"], g["C"], st, g["D"], g["z"], g["dt_bias"])
    torch.cuda.synchronize()
    by, bS = sc.bounds(d, T, y, ya, Sa, dtype)
    sc.close(oy, y, by, "step y")
    sc.close(st, S, bS, "step state")


def test_step_slots(dev):
    """A pool: rows without a request give zeros and touch nothing."""
    d = sc.to(sc.inputs(5, 5, 2, 4, 64, 2, 128), dev)
    args = [d[k] for k in ("x", "dt", "A_log", "B", "C")]
    rest = [d[k] for k in ("D", "z", "dt_bias")]
    pool = _s0(6, 9, 4, 128, 64).to(dev)
    before = pool.clone()
    for dt, past in ((torch.int32, 9), (torch.int64, 9), (torch.int64, 2 ** 32 + 1)):
        slots = [7, -1, 0, past, 3]
        pool.copy_(before)
        y = gdn_hip.ssm_step(*args, pool, *rest, slots=torch.tensor(slots, dtype=dt, device=dev))
        live = [0, 2, 4]
        st = before[[7, 0, 3]].contiguous()
        ref = gdn_hip.ssm_step(*[a[live] if a.dim() > 1 else a for a in args], st,
                               rest[0], rest[1][live], rest[2])
        torch.cuda.synchronize()
        assert torch.equal(y[live], ref) and (y[[1, 3]] == 0).all()
        assert torch.equal(pool[[7, 0, 3]], st)
        keep = [i for i in range(9) if i not in (7, 0, 3)]
        assert torch.equal(pool[keep], before[keep])


def test_scan_offsets_past_32_bits(dev):
    """2.2e9 elements of x: the last tokens against the recurrence from some way
    in front (a token decays by e^-0.7 on average, 100 of them to nothing)."""
    T, H = 540_700, 64
    x = torch.randn(1, T, H, 64, device=dev, dtype=BF)
    b, c = (torch.randn(1, T, 1, 64, device=dev, dtype=BF) for _ in range(2))
    dt = torch.randn(1, T, H, device=dev, dtype=BF)
    d = dict(x=x, dt=dt, A_log=torch.zeros(H, device=dev), B=b, C=c, D=None, z=x,
             dt_bias=torch.zeros(H, device=dev))
    n = 160
    cut = {k: (v if k in ("A_log", "dt_bias") else None if v is None else v[:, -n:]) for k, v in d.items()}
    cut = {k: None if v is None else v.cpu() for k, v in cut.items()}
    y, S, ya, Sa = orc.ssm(**cut)
    by, bS = sc.bounds(cut, n, y, ya, Sa, BF)
    for cu in (None, torch.tensor([0, T - n, T], dtype=torch.int32, device=dev)):
        print(f"scan over {T} tokens, packed {cu is not None}", flush=True)
        oy, oS = gdn_hip.ssm_scan(**d, cu_seqlens=cu)
        torch.cuda.synchronize()
        lo = 0 if cu is not None else 120
        sc.close(oy[:, T - n + lo:], y[:, lo:], by[:, lo:], "scan tail y")
        sc.close(oS[-1:], S, bS, "scan tail state")


def test_step_pool_past_32_bits(dev):
    """A pool of 4200 states of 2 MB: 2.2e9 elements."""
    pool = torch.zeros(4200, 64, 128, 64, device=dev)
    d = sc.inputs(3, 2, 1, 64, 64, 1, 128)
    y, S, ya, Sa = orc.ssm(**d)
    g = sc.to(d, dev)
    print("step, slots 4199 and 4100", flush=True)
    oy = gdn_hip.ssm_step(g["x"], g["dt"], g["A_log"], g["B"], g["C"], pool, g["D"], g["z"], g["dt_bias"],
                          slots=torch.tensor([4199, 4100], dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    by, bS = sc.bounds(d, 1, y, ya, Sa, BF)
    sc.close(oy, y, by, "step y")
    sc.close(pool[[4199, 4100]], S, bS, "step states")
    pool[[4199, 4100]] = 0
    assert not pool.any()


def test_no_tokens(dev):
    d = sc.to(sc.inputs(1, 2, 0, 4, 64, 2, 128), dev)
    args = [d[k] for k in ("x", "dt", "A_log", "B", "C")]
    s0 = _s0(1, 2, 4, 128, 64).to(dev)
    y, s = gdn_hip.ssm_scan(*args, d["D"], d["z"], d["dt_bias"], s0)
    assert y.shape == (2, 0, 4, 64) and torch.equal(s, s0)
    y, s = gdn_hip.ssm_scan(*args)
    assert (s == 0).all()
    st = s0.clone()
    assert gdn_hip.ssm_step(*args, st).shape == (2, 0, 4, 64) and torch.equal(st, s0)


def test_scan_continues_and_steps(dev):
    """A prompt in one call, in two, and its last tokens by steps agree to the bounds."""
    d = sc.inputs(12, 1, 200, 4, 64, 2, 128)
    y, S, ya, Sa = orc.ssm(**d)
    by, bS = sc.bounds(d, 200, y, ya, Sa, BF)
    g = sc.to(d, dev)
    seq = ("x", "dt", "B", "C", "z")

    def part(lo, hi):
        c = {k: (v[:, lo:hi] if k in seq else v) for k, v in g.items()}
        return [c[k] for k in ("x", "dt", "A_log", "B", "C")], [c[k] for k in ("D", "z", "dt_bias")]

    a, r = part(0, 130)
    y0, s = gdn_hip.ssm_scan(*a, *r)
    a, r = part(130, 190)
    y1, s = gdn_hip.ssm_scan(*a, *r, s)
    ys = [y0, y1]
    for lo, hi in ((190, 191), (191, 197), (197, 200)):
        a, r = part(lo, hi)
        ys.append(gdn_hip.ssm_step(*a, s, *r))
    torch.cuda.synchronize()
    sc.close(torch.cat(ys, 1), y, by, "pieces y")
    sc.close(s, S, bS, "pieces state")


def test_copied_layouts(dev):
    """Heads apart, odd offsets: copied in front of the kernels, the same bits."""
    d = sc.to(sc.inputs(13, 2, 70, 4, 64, 2, 128), dev)
    args = [d[k] for k in ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")]
    ref = gdn_hip.ssm_scan(*args)
    odd = list(args)
    odd[0] = args[0].transpose(1, 2).contiguous().transpose(1, 2)
    odd[1] = args[1].transpose(1, 2).contiguous().transpose(1, 2)
    buf = torch.empty(args[3].numel() + 3, dtype=BF, device=dev)[3:].view(args[3].shape)
    buf.copy_(args[3])
    odd[3] = buf
    got = gdn_hip.ssm_scan(*odd)
    torch.cuda.synchronize()
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
