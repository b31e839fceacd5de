"""GPU parity of the operators around the state-space scan: the conv that
carries its state, the tables of a packed batch, the grouped gated norm, conv
states in a pool, and a layer that runs them together."""
import random

import pytest
import torch
import torch.nn.functional as F

import gdn_hip
import ssm_cases as sc
from oracle import ssm_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _conv_inputs(seed, B, T, D, K, L, io, wd, seqs):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, D, generator=g).to(io).transpose(1, 2)
    w = (0.5 * torch.randn(D, K, generator=g)).to(wd)
    bias = (0.1 * torch.randn(D, generator=g)).to(wd)
    return x, w, bias, torch.randn(seqs, D, L, generator=g).to(io)


def _conv_bound(y, mag, io, silu):
    """fp32 sums of at most 5 terms (5 x 2^-24 of the absolute sum, SiLU's slope
    is at most 1.1 and its own error 2^-21), then half a step of the type."""
    half = torch.finfo(io).eps / 2
    return half * y.abs() + (8 * 2.0 ** -24 * mag * 1.1 + 2.0 ** -20 * y.abs()) * 1.01 + \
        torch.finfo(io).smallest_normal * half


def _check_conv(dev, x, w, bias, s0, silu, lengths, tag, state_len=0):
    y, st, mag = orc.conv_prefill(x, w, bias, s0, silu, lengths, state_len)
    cu = None if lengths is None else torch.tensor(
        [sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=dev)
    print(tag, flush=True)
    oy, os_ = gdn_hip.causal_conv1d_prefill(
        x.to(dev), w.to(dev), None if bias is None else bias.to(dev),
        None if s0 is None else s0.to(dev), silu=silu, cu_seqlens=cu, state_len=state_len)
    torch.cuda.synchronize()
    n = y.shape[2]
    sc.close(oy[:, :, :n], y, _conv_bound(y, mag, x.dtype, silu), tag)
    assert os_.dtype == x.dtype and torch.equal(os_.double().cpu(), st), tag + " state"


@pytest.mark.parametrize("T", [0, 1, 2, 3, 4, 5, 7, 8, 9, 31, 200])
def test_conv_lengths(dev, T):
    x, w, bias, s0 = _conv_inputs(T, 2, T, 264, 4, 4, BF, BF, 2)
    _check_conv(dev, x, w, bias, s0, True, None, f"conv T={T}")
    _check_conv(dev, x, w, None, None, False, None, f"conv T={T} zeros")


@pytest.mark.parametrize("io,wd", [(BF, BF), (HF, HF), (BF, F32), (HF, F32)])
@pytest.mark.parametrize("K,L", [(2, 1), (2, 8), (3, 2), (3, 3), (4, 3), (4, 4), (4, 7)])
def test_conv_types_taps_states(dev, io, wd, K, L):
    x, w, bias, s0 = _conv_inputs(K + L, 2, 21, 72, K, L, io, wd, 2)
    for silu in (False, True):
        _check_conv(dev, x, w, bias, s0, silu, None, f"conv K={K} L={L} {io} {wd} {silu}")
    _check_conv(dev, x, w, bias, None, True, None, f"conv K={K} L={L} no state", state_len=L)


@pytest.mark.parametrize("lengths", [[9], [0, 3, 0, 0, 1, 2, 40, 0], [1] * 30, [8, 8, 7, 9, 64, 5]])
@pytest.mark.parametrize("state", [True, False])
def test_conv_packed(dev, lengths, state):
    x, w, bias, s0 = _conv_inputs(len(lengths), 1, sum(lengths), 2056, 4, 4, BF, BF, len(lengths))
    _check_conv(dev, x, w, bias, s0 if state else None, True, lengths, f"conv packed {lengths} {state}")


def test_conv_packed_behind_and_unordered(dev):
    """Tokens behind the last sequence do not enter a state; an unordered
    cu_seqlens stays in bounds."""
    lengths = [20, 13]
    x, w, bias, s0 = _conv_inputs(5, 1, 50, 64, 4, 4, BF, BF, 2)
    _check_conv(dev, x, w, bias, s0, True, lengths, "conv behind")
    cu = torch.tensor([40, -5, 70], dtype=torch.int32, device=dev)
    gdn_hip.causal_conv1d_prefill(x.to(dev), w.to(dev), bias.to(dev), s0.to(dev), cu_seqlens=cu)
    torch.cuda.synchronize()


def test_conv_strided_and_then_update(dev):
    """A channel slice of a wider buffer in place; the state goes on into the update."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 60, 200, generator=g).to(BF)
    x = wide[:, :, 8:136].transpose(1, 2)
    w, bias = (0.5 * torch.randn(128, 4, generator=g)).to(BF), torch.randn(128, generator=g).to(BF)
    full, st, mag = orc.conv_prefill(x, w, bias, None, True)
    xd = wide.to(dev)[:, :, 8:136].transpose(1, 2)
    y0, s = gdn_hip.causal_conv1d_prefill(xd[:, :, :50], w.to(dev), bias.to(dev), silu=True)
    y1, s = gdn_hip.causal_conv1d_prefill(xd[:, :, 50:57], w.to(dev), bias.to(dev), s, silu=True)
    y2 = gdn_hip.causal_conv1d_update(xd[:, :, 57:], s, w.to(dev), bias.to(dev), True)
    torch.cuda.synchronize()
    # the update rounds the sum to bf16 in front of the activation too
    bound = _conv_bound(full, mag, BF, True)
    bound[:, :, 57:] += 1.1 * 2.0 ** -8 * mag[:, :, 57:]
    sc.close(torch.cat([y0, y1, y2], 2), full, bound, "conv pieces")
    assert torch.equal(s.double().cpu(), st)


@pytest.mark.parametrize("L,D", [(4, 256), (3, 257), (4, 6)])
def test_conv_update_slots(dev, L, D):
    g = torch.Generator().manual_seed(D)
    x = torch.randn(5, D, 2, generator=g).to(BF).to(dev)
    w = torch.randn(D, 4, generator=g).to(BF).to(dev)
    pool = torch.randn(8, D, L, generator=g).to(BF).to(dev)
    before = pool.clone()
    slots = torch.tensor([6, 8, 1, -3, 2], dtype=torch.int32, device=dev)
    y = gdn_hip.causal_conv1d_update(x, pool, w, None, True, slots=slots)
    st = before[[6, 1, 2]].contiguous()
    ref = gdn_hip.causal_conv1d_update(x[[0, 2, 4]].contiguous(), st, w, None, True)
    torch.cuda.synchronize()
    assert torch.equal(y[[0, 2, 4]], ref) and (y[[1, 3]] == 0).all()
    assert torch.equal(pool[[6, 1, 2]], st)
    keep = [0, 3, 4, 5, 7]
    assert torch.equal(pool[keep], before[keep])


@pytest.mark.parametrize("lengths,total,block,slots", [
    ([5], 5, 64, None), ([0], 0, 64, None), ([0, 0, 3], 3, 64, [4, 5, 6]), ([64, 65, 0, 127], 300, 64, None),
    ([1000, 1, 0, 500], 1200, 128, [3, 1, 2, 0]),     # cut at the capacity
    ([-5, 10, -1, 7], 20, 64, None), ([2 ** 31 - 1, 2 ** 31 - 1, 5], 1000, 256, None),
    ([1] * 600, 700, 64, None), ([0] * 300 + [9] + [0] * 300, 9, 64, None)])
def test_request_blocks(dev, lengths, total, block, slots):
    want = orc.request_blocks(lengths, total, block, slots)
    print(f"request_blocks {len(lengths)} requests, {total} tokens", flush=True)
    for dt in (torch.int32, torch.int64):
        got = gdn_hip.request_blocks(
            torch.tensor(lengths, dtype=dt, device=dev), total, block=block,
            slots=None if slots is None else torch.tensor(slots, dtype=dt, device=dev))
        torch.cuda.synchronize()
        for g, r in zip(got, want):
            assert g.dtype == torch.int32 and g.tolist() == r


@pytest.mark.parametrize("n", [255, 256, 257, 1023, 4096, 4097, 9000])
def test_request_blocks_many(dev, n):
    """Both launch forms (up to 4096 requests in one, more in two), random lengths."""
    rng = random.Random(n)
    lengths = [rng.choice([0, 1, 1, 1, rng.randrange(300)]) for _ in range(n)]
    total = sum(lengths) + rng.choice([0, 77])
    slots = list(range(n))
    rng.shuffle(slots)
    want = orc.request_blocks(lengths, total, 64, slots)
    got = gdn_hip.request_blocks(torch.tensor(lengths, dtype=torch.int32, device=dev), total,
                                 slots=torch.tensor(slots, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    for g, r in zip(got, want):
        assert g.tolist() == r


def test_request_blocks_64_bit_lengths(dev):
    got = gdn_hip.request_blocks(torch.tensor([3, 2 ** 40, 7], device=dev), 50)
    assert got[0].tolist() == [0, 3, 50, 50]


@pytest.mark.parametrize("io,wd", [(BF, BF), (HF, HF), (BF, F32), (HF, F32)])
@pytest.mark.parametrize("C,groups", [(8, 1), (16, 2), (128, 1), (136, 1), (512, 1), (520, 1), (1024, 1),
                                      (1032, 1), (2048, 1), (2056, 1), (4104, 1), (8192, 1), (8200, 1),
                                      (16384, 1), (4096, 8), (1536, 4)])
@pytest.mark.parametrize("gate_first", [True, False])
def test_groupnorm(dev, C, groups, io, wd, gate_first):
    g = torch.Generator().manual_seed(C)
    x, z = (torch.randn(5, C, generator=g).to(io) for _ in range(2))
    x[3] = 0
    w = (1 + 0.1 * torch.randn(C, generator=g)).to(wd)
    ref = orc.gated_groupnorm(x, z, w, groups, 1e-6, gate_first)
    y = gdn_hip.gated_groupnorm(x.to(dev), z.to(dev), w.to(dev), groups, 1e-6, gate_first=gate_first)
    torch.cuda.synchronize()
    half = torch.finfo(io).eps / 2
    # each factor within 2^-20 (SiLU 2^-21, the mean's sum log2(C) + 16 roundings of squares)
    sc.close(y, ref, (half + 2.0 ** -18) * ref.abs() + torch.finfo(io).smallest_normal * half,
             f"norm C={C}/{groups} {io} {wd}")


def test_groupnorm_rows_in_place(dev):
    """Slices of a projection, leading dimensions, an empty batch, a transposed view."""
    wide = torch.randn(2, 9, 600, generator=torch.Generator().manual_seed(1)).to(BF).to(dev)
    w = torch.ones(256, device=dev)
    x, z = wide[..., :256], wide[..., 264:520]
    ref = gdn_hip.gated_groupnorm(x.contiguous(), z.contiguous(), w, 2)
    assert torch.equal(gdn_hip.gated_groupnorm(x, z, w, 2), ref)
    assert torch.equal(gdn_hip.gated_groupnorm(x.transpose(0, 1), z.transpose(0, 1), w, 2),
                       ref.transpose(0, 1))
    assert gdn_hip.gated_groupnorm(x[:0], z[:0], w, 2).shape == (0, 9, 256)
    assert torch.equal(gdn_hip.gated_groupnorm(x[:, :1].expand(2, 9, 256), z, w, 2)[:, 0], ref[:, 0])
    torch.cuda.synchronize()


class _Layer:
    """conv -> scan -> norm over one layer's projections, as a serving program runs it."""

    def __init__(self, dev, H=4, P=64, G=2, N=128, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.H, self.P, self.G, self.N, self.dev = H, P, G, N, dev
        self.C = H * P + 2 * G * N
        rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.w, self.bias = (0.5 * rn(self.C, 4)).to(BF).to(dev), (0.1 * rn(self.C)).to(BF).to(dev)
        self.A_log, self.D = torch.log(0.1 + torch.rand(H, generator=g)).to(dev), rn(H).to(dev)
        self.dt_bias, self.nw = (-2 + rn(H)).to(dev), (1 + 0.1 * rn(H * P)).to(dev)

    def _split(self, conv):   # [B, C, T] -> x, B, C
        H, P, G, N = self.H, self.P, self.G, self.N
        x, b, c = torch.split(conv.transpose(1, 2), [H * P, G * N, G * N], dim=-1)
        return x.unflatten(-1, (H, P)), b.unflatten(-1, (G, N)), c.unflatten(-1, (G, N))

    def _out(self, y, z):
        return gdn_hip.gated_groupnorm(y.flatten(2), z, self.nw, self.G)

    def prompts(self, xbc, z, dt, conv_state, state, **packed):
        conv, conv_state = gdn_hip.causal_conv1d_prefill(
            xbc.transpose(1, 2), self.w, self.bias, conv_state, silu=True,
            cu_seqlens=packed.get("cu_seqlens"))
        x, b, c = self._split(conv)
        y, state = gdn_hip.ssm_scan(x, dt, self.A_log, b, c, self.D, None, self.dt_bias, state,
                                    **packed)
        return self._out(y, z), conv_state, state

    def tokens(self, xbc, z, dt, conv_pool, pool, slots):
        conv = gdn_hip.causal_conv1d_update(xbc.transpose(1, 2), conv_pool, self.w, self.bias,
                                            True, slots=slots)
        x, b, c = self._split(conv)
        y = gdn_hip.ssm_step(x, dt, self.A_log, b, c, pool, self.D, None, self.dt_bias, slots=slots)
        return self._out(y, z)


def _layer_inputs(layer, lengths, seed):
    g = torch.Generator().manual_seed(seed)
    T = sum(lengths)
    return [torch.randn(1, T, n, generator=g).to(BF).to(layer.dev) for n in
            (layer.C, layer.H * layer.P, layer.H)]


def _layer_oracle(layer, xbc, z, dt):
    """One sequence in 64 bits from the same bf16 projections."""
    conv, _, _ = orc.conv_prefill(xbc.transpose(1, 2), layer.w, layer.bias, None, True)
    x, b, c = layer._split(conv)
    y, S, _, _ = orc.ssm(x, dt, layer.A_log, b, c, layer.D, None, layer.dt_bias)
    return orc.gated_groupnorm(y.flatten(2), z, layer.nw, layer.G, 1e-6), S


def _rel(a, b):
    return ((a.double().cpu() - b).norm() / b.norm()).item()


def test_layer_serving(dev):
    """Requests packed by their lengths, then continued by steps out of a pool,
    against the 64-bit layer on each request's whole text.  Roundings to bf16 on
    the way to y: the conv's output (x, B and C: 3), the scan's y and the norm's
    output, each at most 2^-8 and independent: 5 x 2^-8 bounds the relative error."""
    layer = _Layer(dev)
    prompt, more = [70, 1, 130, 0, 64], 6
    seqs = [_layer_inputs(layer, [n + more], 40 + i) for i, n in enumerate(prompt)]
    lens = torch.tensor(prompt, dtype=torch.int32, device=dev)
    T = sum(prompt)
    block = gdn_hip.ssm_scan_block(T, 1, layer.H, layer.P, layer.G, layer.N, len(prompt))
    cu, table, tslot, tpos = gdn_hip.request_blocks(lens, T, block=block)
    packed = [torch.cat([s[k][:, :n] for s, n in zip(seqs, prompt)], 1) for k in range(3)]
    y, cs, st = layer.prompts(*packed, None, None, cu_seqlens=cu, blocks=table, block=block)
    order = torch.tensor([4, 0, 7, 2, 5], device=dev)
    conv_pool = torch.zeros(9, layer.C, 4, dtype=BF, device=dev)
    pool = torch.zeros(9, layer.H, layer.N, layer.P, device=dev)
    conv_pool[order], pool[order] = cs, st
    # a padded batch: two rows without a request
    slots = F.pad(order, (0, 2), value=-1).int()
    outs = []
    for lo, hi in ((0, 1), (1, 4), (4, 6)):
        rows = [torch.cat([s[k][:, n + lo:n + hi] for s, n in zip(seqs, prompt)]) for k in range(3)]
        rows = [torch.cat([r, torch.zeros_like(r[:2])]) for r in rows]
        outs.append(layer.tokens(*rows, conv_pool, pool, slots)[:5])
    torch.cuda.synchronize()
    outs = torch.cat(outs, 1)
    cuts = cu.tolist()
    for i, n in enumerate(prompt):
        ref, S = _layer_oracle(layer, *seqs[i])
        got = torch.cat([y[:, cuts[i]:cuts[i + 1]], outs[i:i + 1]], 1)
        e, es = _rel(got, ref), _rel(pool[order[i]][None], S)
        print(f"request {i}: y {e:.2e} state {es:.2e}", flush=True)
        assert e <= 5 * 2.0 ** -8 and es <= 3 * 2.0 ** -8
    unused = [1, 3, 6, 8]
    assert (pool[unused] == 0).all() and (conv_pool[unused] == 0).all()


def test_layer_captured(dev):
    """The serving step captured into a graph and replayed with eager work in
    between: the eager results each time.  The packed prompt call too, with its
    lengths changed on the device between replays."""
    layer = _Layer(dev)
    B = 4
    g = torch.Generator().manual_seed(1)
    new = [[torch.randn(B, 1, n, generator=g).to(BF).to(dev) for n in (layer.C, layer.H * layer.P, layer.H)]
           for _ in range(4)]
    slots = torch.tensor([3, 1, -1, 0], dtype=torch.int32, device=dev)
    conv0, pool0 = torch.randn(5, layer.C, 4, generator=g).to(BF).to(dev), torch.randn(5, layer.H, layer.N, layer.P, generator=g).to(dev)
    static = [t.clone() for t in new[0]]
    conv_pool, pool = conv0.clone(), pool0.clone()
    prompt = _layer_inputs(layer, [300], 9)
    lens = torch.tensor([100, 60, 140], dtype=torch.int32, device=dev)

    def packed():
        cu = gdn_hip.request_blocks(lens, 300)[0]
        return layer.prompts(*prompt, None, None, cu_seqlens=cu)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.tokens(*static, conv_pool, pool, slots)
        packed()
    torch.cuda.current_stream().wait_stream(side)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.tokens(*static, conv_pool, pool, slots)
    with torch.cuda.graph(graph2):
        pout = packed()
    conv_pool.copy_(conv0)
    pool.copy_(pool0)
    ec, ep = conv0.clone(), pool0.clone()
    for i, rows in enumerate(new):
        for s, r in zip(static, rows):
            s.copy_(r)
        lens.copy_(torch.tensor([[100, 60, 140], [0, 300, 0], [1, 2, 297], [64, 64, 172]][i], dtype=torch.int32))
        graph.replay()
        graph2.replay()
        ref = layer.tokens(*rows, ec, ep, slots)
        pref = packed()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(pool, ep) and torch.equal(conv_pool, ec)
        for a, b in zip(pout, pref):
            assert torch.equal(a, b)


def test_other_stream(dev):
    """Calls on a stream of the caller's own, ordered by it alone."""
    layer = _Layer(dev)
    ins = _layer_inputs(layer, [500], 3)
    ref = layer.prompts(*ins, None, None)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = layer.prompts(*[t.clone() for t in ins], None, None)
    s.synchronize()
    for a, b in zip(ref, got):
        assert torch.equal(a, b)


def test_request_blocks_largest(dev):
    """2^30 tokens, and lengths that pass them twice over."""
    total, block = 1 << 30, 1 << 20
    for lengths in ([2 ** 31 - 1, 2 ** 31 - 1, 5], [0, 2 ** 30, 2 ** 30]):
        print(f"request_blocks {lengths} in {total}", flush=True)
        cu, table, slot, pos = gdn_hip.request_blocks(
            torch.tensor(lengths, dtype=torch.int32, device=dev), total, block=block)
        torch.cuda.synchronize()
        full = lengths.index(max(lengths))
        assert cu.tolist() == [0] * (full + 1) + [total] * (3 - full)
        rows = [[n, 0, 0, 0] for n in range(full)] + \
            [[full, i * block, block, i] for i in range(total // block)] + \
            [[n, total, 0, 0] for n in range(full + 1, 3)]
        assert table.tolist() == rows + [[-1, 0, 0, 0]] * (table.shape[0] - len(rows))
        assert (slot == full).all() and torch.equal(pos, torch.arange(total, dtype=torch.int32, device=dev))


def test_conv_and_norm_offsets_past_32_bits(dev):
    T, D = 540_700, 4096   # 2.2e9 elements
    x = torch.randn(1, T, D, device=dev, dtype=BF)
    w = (0.5 * torch.randn(D, 4, generator=torch.Generator().manual_seed(1))).to(BF)
    tail = x[:, -40:].cpu().transpose(1, 2)
    for cu in (None, torch.tensor([0, T - 9, T], dtype=torch.int32, device=dev)):
        print(f"conv over {T} x {D}, packed {cu is not None}", flush=True)
        y, st = gdn_hip.causal_conv1d_prefill(x.transpose(1, 2), w.to(dev), silu=True, cu_seqlens=cu)
        torch.cuda.synchronize()
        ref, rst, mag = orc.conv_prefill(tail, w, None, None, True, None if cu is None else [31, 9])
        sc.close(y[:, :, -36:], ref[:, :, 4:], _conv_bound(ref, mag, BF, True)[:, :, 4:], "conv tail")
        assert torch.equal(st[-1:].double().cpu(), rst[-1:])
    print(f"norm of {T} x {D}", flush=True)
    y = gdn_hip.gated_groupnorm(x[0], x[0], w[:, 0].contiguous().to(dev), 2)
    torch.cuda.synchronize()
    last = x[0, -5:].cpu()
    ref = orc.gated_groupnorm(last, last, w[:, 0], 2, 1e-6)
    half = 2.0 ** -8
    sc.close(y[-5:], ref, (half + 2.0 ** -18) * ref.abs() + torch.finfo(BF).smallest_normal * half, "norm tail")


def test_conv_rows_behind_the_last_sequence(dev):
    """C entry: y rows behind the last packed sequence are left as they were."""
    from gdn_hip import capi
    x, w, _, s0 = _conv_inputs(8, 1, 100, 64, 4, 4, BF, BF, 3)
    xd, wd, sd = x.transpose(1, 2).contiguous().to(dev), w.to(dev), s0.to(dev)
    y = torch.full((1, 100, 64), 7.0, dtype=BF, device=dev)
    st = torch.empty_like(sd)
    cu = torch.tensor([0, 30, 30, 71], dtype=torch.int32, device=dev)
    assert capi.lib().gdn_causal_conv1d_prefill(
        xd.data_ptr(), wd.data_ptr(), None, sd.data_ptr(), y.data_ptr(), st.data_ptr(), 1, 100, 64, 4, 4,
        6400, 64, 6400, 64, cu.data_ptr(), 3, 0, 0, 1, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    ref, rst, mag = orc.conv_prefill(x, w, None, s0, True, [30, 0, 41])
    sc.close(y[:, :71].transpose(1, 2), ref, _conv_bound(ref, mag, BF, True), "conv in front")
    assert (y[:, 71:] == 7).all() and torch.equal(st.double().cpu(), rst)


def test_two_streams_at_once(dev):
    """Two prompts batches on two streams, neither waiting for the other."""
    layer = _Layer(dev)
    ins = [_layer_inputs(layer, lengths, seed) for lengths, seed in (([700, 3], 4), ([300, 400], 5))]
    refs = [layer.prompts(*i, None, None) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(layer.prompts(*ins[k], None, None))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            for a, b in zip(refs[k], out):
                assert torch.equal(a, b)
