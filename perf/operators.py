"""Workloads of the state-space operators: the selective scan over prompts and
over single tokens, the short causal convolution that carries its state, the
tables of a packed batch built from request lengths, and the grouped gated
norm behind the scan.

A layer has H heads of P channels with a state of N x P each, G groups of B
and C vectors, and a conv over H P + 2 G N channels of 4 taps.  Widths are the
4096 value channels of the gated-delta layer (32 heads of 128), its shards and
doubles.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

own = False

TAPS = 4
EPS = 1e-6
# 8 packed prompts of 512 .. 4096 tokens, 19,861 in all
VARLEN_8 = "1427 3804 2613 3898 660 2279 4069 1111"
MOST_TOKEN_HEADS = 19861 * 64      # tokens x heads of the longest listed scan
# (heads, channels a head, state, groups)
LAYERS = ((64, 64, 128, 8), (64, 64, 128, 1), (32, 128, 128, 8), (32, 128, 64, 2), (16, 64, 128, 2),
          (128, 64, 64, 8), (8, 64, 128, 1), (32, 64, 256, 1), (24, 64, 128, 1))


def listed():
    return [
        # a short turn added to a cached conversation, fp16: launches count
        dict(name="scan_T77_fp16", op="scan", B=1, T=77, H=32, P=128, N=64, G=2, z=True,
             dtype="float16"),
        # one prompt of ordinary length
        dict(name="scan_T1141", op="scan", B=1, T=1141, H=64, P=64, N=128, G=8, z=True,
             dtype="bfloat16"),
        # one long document on a shard with few heads, gate left to the norm
        dict(name="scan_T16384", op="scan", B=1, T=16384, H=16, P=64, N=128, G=2, z=False,
             dtype="bfloat16"),
        # a serving batch of packed prompts of uneven lengths
        dict(name="scan_packed_8", op="scan", lengths=VARLEN_8, H=64, P=64, N=128, G=8, z=True,
             dtype="bfloat16"),
        # one user's decode step: the smallest call
        dict(name="step_B1", op="step", B=1, T=1, H=64, P=64, N=128, G=8, z=True, slots=0,
             dtype="bfloat16"),
        # a continuous batch: 48 live requests in a pool of 64 states
        dict(name="step_B48_of_64", op="step", B=48, T=1, H=64, P=64, N=128, G=8, z=True, slots=64,
             dtype="bfloat16"),
        # the conv of a prompt that continues a cached one
        dict(name="conv_T1141", op="conv", B=1, T=1141, C=6144, state=True, dtype="bfloat16"),
        # the conv of the packed batch, fp16
        dict(name="conv_packed_8", op="conv", lengths=VARLEN_8, C=4352, state=True,
             dtype="float16"),
        # tables of the packed batch of 8 prompts
        dict(name="blocks_8", op="blocks", lengths=VARLEN_8, block=64, spare=0, slots=False),
        # tables of a large mixed batch: mostly single tokens, some prompts, padded capacity
        dict(name="blocks_1500", op="blocks", requests=1500, most=900, block=256, spare=1000,
             slots=True),
        # the norm of a decode batch: one row a request
        dict(name="norm_48", op="norm", rows=48, C=4096, groups=8, gate_first=True,
             dtype="bfloat16"),
        # the norm over the packed batch's tokens
        dict(name="norm_19861", op="norm", rows=19861, C=4096, groups=1, gate_first=True,
             dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(("scan", "scan", "scan", "step", "step", "conv", "blocks", "norm"))
    dt = rng.choice(("bfloat16", "bfloat16", "float16"))
    H, P, N, G = rng.choice(LAYERS)
    # lengths are bounded by the work of a head: P N relative to 64 x 128
    most = MOST_TOKEN_HEADS * 64 * 128 // (H * P * N)
    if op == "scan" and rng.random() < 0.4:
        n = _log_int(rng, 2, 24)
        ls = [_log_int(rng, 1, min(4096, most // n)) for _ in range(n)]
        if rng.random() < 0.3:
            ls[rng.randrange(n)] = 0
        return dict(op=op, lengths=" ".join(map(str, ls)), H=H, P=P, N=N, G=G,
                    z=rng.random() < 0.7, dtype=dt)
    if op == "scan":
        B = rng.choice((1, 1, 1, 2, 3, 5))
        return dict(op=op, B=B, T=_log_int(rng, 1, min(20000, most // B)), H=H, P=P, N=N, G=G,
                    z=rng.random() < 0.7, dtype=dt)
    if op == "step":
        B = _log_int(rng, 1, 48)
        # up to 6 tokens a call: the check of drafted tokens
        return dict(op=op, B=B, T=rng.choice((1, 1, 1, 2, 4, 6)), H=H, P=P, N=N, G=G,
                    z=rng.random() < 0.7, slots=rng.choice((0, B + rng.randint(0, 16))), dtype=dt)
    if op == "conv":
        C = H * P + 2 * G * N
        if rng.random() < 0.5:
            n = _log_int(rng, 2, 64)
            ls = [_log_int(rng, 1, min(4096, 19000 * 4096 // (C * n))) for _ in range(n)]
            return dict(op=op, lengths=" ".join(map(str, ls)), C=C, state=rng.random() < 0.7, dtype=dt)
        B = rng.choice((1, 1, 2, 4))
        return dict(op=op, B=B, T=_log_int(rng, 1, min(8192, 19000 * 4096 // (C * B))), C=C,
                    state=rng.random() < 0.7, dtype=dt)
    if op == "blocks":
        return dict(op=op, requests=_log_int(rng, 1, 6000), most=_log_int(rng, 2, 2000),
                    block=rng.choice((64, 128, 256, 512)), spare=rng.choice((0, 1, 500)),
                    slots=rng.random() < 0.5)
    C = rng.choice((1024, 2048, 4096, 4096, 8192))
    return dict(op=op, rows=_log_int(rng, 1, 19000 * 4096 // C), C=C, groups=rng.choice((1, 2, 4, 8, 8)),
                gate_first=rng.random() < 0.7, dtype=dt)


# ---------------------------------------------------------------- inputs
class _Rand:
    """Seeded draws on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def n(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def u(self, *shape):
        return torch.rand(*shape, generator=self.gen, device="cuda")

    def perm(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _lengths(case):
    return [int(x) for x in case["lengths"].split()]


def _packed(case, s):
    """(batch rows, tokens a row, sequences) of a case; packed ones get cu."""
    if "lengths" not in case:
        return case["B"], case["T"], case["B"]
    ls = torch.tensor(_lengths(case), device="cuda")
    s["cu"] = F.pad(ls.cumsum(0), (1, 0)).int()
    return 1, sum(_lengths(case)), len(_lengths(case))


def prepare(case, seed):
    r = _Rand(seed)
    s = dict(case)
    op = case["op"]
    if op == "blocks":
        if "lengths" in case:
            ls = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
            # the same requests in another order: another batch
            s["lens"] = ls[r.perm(len(ls))].contiguous()
        else:
            n = case["requests"]
            # three in four requests decode (one token), some are empty slots of the batch
            long = torch.exp(r.u(n) * math.log(case["most"])).int()
            kind = r.u(n)
            s["lens"] = torch.where(kind < 0.72, 1, torch.where(kind < 0.76, 0, long)).int()
        n = s["lens"].numel()
        # the capacity of the packed row: what the captured step was built for
        most = sum(_lengths(case)) if "lengths" in case else n * 2 + n * case["most"] // 5
        s["total"] = most + case["spare"]
        s["slot"] = r.perm(n + 7)[:n].int() if case["slots"] else None
        return s
    dt = getattr(torch, case["dtype"])
    if op == "norm":
        s.update(x=r.n(case["rows"], case["C"]).to(dt), gate=r.n(case["rows"], case["C"]).to(dt),
                 w=1 + 0.1 * r.n(case["C"]))
        return s
    B, T, seqs = _packed(case, s)
    if op == "conv":
        C = case["C"]
        s.update(x=r.n(B, T, C).to(dt).transpose(1, 2), w=(0.5 * r.n(C, TAPS)).to(dt),
                 bias=(0.1 * r.n(C)).to(dt),
                 state0=r.n(seqs, C, TAPS).to(dt) if case["state"] else None)
        return s
    H, P, N, G = (case[k] for k in "HPNG")
    # x, B and C are slices of the conv's output, dt and z of the layer's input projection
    conv = r.n(B, T, H * P + 2 * G * N)
    conv = (conv * torch.sigmoid(conv)).to(dt)
    x, b, c = torch.split(conv, [H * P, G * N, G * N], dim=-1)
    proj = torch.cat([r.n(B, T, H * P), 0.5 * r.n(B, T, H)], dim=-1).to(dt)
    # steps of 0.001 .. 0.1 (log-uniform over heads) at a zero projection, decays -1 .. -16
    step = torch.exp(math.log(1e-3) + math.log(100.0) * r.u(H))
    s.update(x=x.view(B, T, H, P), b=b.view(B, T, G, N), c=c.view(B, T, G, N),
             gate=proj[..., :H * P].view(B, T, H, P) if case["z"] else None,
             dt=proj[..., H * P:], A_log=torch.log(1 + 15 * r.u(H)),
             dt_bias=step + torch.log(-torch.expm1(-step)), D=1 + 0.1 * r.n(H))
    if op == "scan":
        s["state"] = 0.1 * r.n(seqs, H, N, P)
    else:
        s["state"] = 0.1 * r.n(case["slots"] or B, H, N, P)
        s["slot"] = r.perm(case["slots"])[:B].int() if case["slots"] else None
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    return {"scan": _plain_scan, "step": _plain_step, "conv": _plain_conv, "blocks": _plain_blocks,
            "norm": _plain_norm}[s["op"]](s)


def _own(s):
    ops = _library()
    op = s["op"]
    if op == "scan":
        return ops.ssm_scan(s["x"], s["dt"], s["A_log"], s["b"], s["c"], s["D"], s["gate"],
                            s["dt_bias"], s["state"], cu_seqlens=s.get("cu"))
    if op == "step":
        y = ops.ssm_step(s["x"], s["dt"], s["A_log"], s["b"], s["c"], s["state"], s["D"], s["gate"],
                         s["dt_bias"], slots=s["slot"])
        return y, s["state"]
    if op == "conv":
        return ops.causal_conv1d_prefill(s["x"], s["w"], s["bias"], s["state0"], silu=True,
                                         cu_seqlens=s.get("cu"))
    if op == "blocks":
        return ops.request_blocks(s["lens"], s["total"], block=s["block"], slots=s["slot"])
    return ops.gated_groupnorm(s["x"], s["gate"], s["w"], s["groups"], EPS,
                               gate_first=s["gate_first"])


def _library():
    pkg = str(Path(__file__).resolve().parents[1] / "qwen-drive-edge-orin_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gdn_hip

    return gdn_hip


def _silu(x):
    return x * torch.sigmoid(x)


def _rows_of(s, T):
    """For packed rows: the longest length, and for each token its sequence and position."""
    cu = s["cu"].long()
    t = torch.arange(T, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return max(_lengths(s)), seq, t - cu[:-1][seq]


def _plain_scan(s):
    """The scan by chunks of 64 tokens: products within a chunk under its decay
    matrix, the chunks' states joined by the decay matrix between chunks.  Sums
    of logarithms are in 64 bits (differences of long sums), the rest in 32."""
    x, b, c = (s[k].float() for k in "xbc")
    d = F.softplus(s["dt"].float() + s["dt_bias"])
    T0, H, P, N = x.shape[1], x.shape[2], x.shape[3], b.shape[3]
    where = None
    if "cu" in s:
        longest, seq, pos = _rows_of(s, T0)
        where = (seq, pos)

        def spread(v):
            out = v.new_zeros(s["cu"].numel() - 1, longest, *v.shape[2:])
            out[where] = v[0]
            return out

        x, b, c, d = spread(x), spread(b), spread(c), spread(d)
    S0, Q, T = s["state"], 64, x.shape[1]
    nc = max(1, -(-T // Q))
    x, b, c, d = (F.pad(v, (0, 0) * (v.dim() - 2) + (0, nc * Q - T)) for v in (x, b, c, d))
    B, rep = x.shape[0], H // b.shape[2]
    # [B, H, chunk, Q, ..]
    x, d = (v.reshape(B, nc, Q, H, -1).permute(0, 3, 1, 2, 4) for v in (x, d))
    b, c = (v.view(B, nc, Q, -1, N).permute(0, 3, 1, 2, 4).repeat_interleave(rep, dim=1) for v in (b, c))
    la = (-torch.exp(s["A_log"]).view(1, H, 1, 1) * d[..., 0]).double()
    cum = la.cumsum(-1)
    low = torch.ones(Q, Q, dtype=torch.bool, device=x.device).tril()
    decay = torch.exp((cum[..., :, None] - cum[..., None, :]).masked_fill(~low, -math.inf)).float()
    xd = x * d
    inside = (torch.matmul(c, b.transpose(-1, -2)) * decay) @ xd
    left = torch.exp(cum[..., -1:] - cum).float()
    local = torch.matmul((b * left[..., None]).transpose(-1, -2), xd)        # [B, H, nc, N, P]
    # the state in front of chunk i: S0 and the chunks before it, decayed
    tot = F.pad(cum[..., -1].cumsum(-1), (1, 0))
    before = torch.ones(nc + 1, nc + 1, dtype=torch.bool, device=x.device).tril()
    between = torch.exp((tot[..., :, None] - tot[..., None, :]).masked_fill(~before, -math.inf)).float()
    parts = torch.cat([S0[:, :, None], local], dim=2).flatten(3)
    states = (between @ parts).view(B, H, nc + 1, N, P)
    y = inside + torch.matmul(c * torch.exp(cum).float()[..., None], states[:, :, :nc])
    y = y + s["D"].view(1, H, 1, 1, 1) * x
    y = y.permute(0, 2, 3, 1, 4).reshape(B, nc * Q, H, P)
    y = y[where][None] if where is not None else y[:, :T0]
    if s["gate"] is not None:
        y = y * _silu(s["gate"].float())
    return [y.to(s["x"].dtype).contiguous(), states[:, :, nc].contiguous()]


def _plain_step(s):
    """Up to a few tokens: each from the state and the tokens before it."""
    x, b, c = (s[k].float() for k in "xbc")
    B, T, H, P = x.shape
    rep = H // b.shape[2]
    b, c = (v.repeat_interleave(rep, dim=2) for v in (b, c))
    d = F.softplus(s["dt"].float() + s["dt_bias"])
    cum = (-torch.exp(s["A_log"]) * d).cumsum(1)                             # [B, T, H]
    S0 = s["state"] if s["slot"] is None else s["state"][s["slot"].long()]
    low = torch.ones(T, T, dtype=torch.bool, device=x.device).tril()
    decay = torch.exp((cum[:, :, None] - cum[:, None]).masked_fill(~low[None, :, :, None], -math.inf))
    score = (c[:, :, None] * b[:, None]).sum(-1) * decay * d[:, None]        # [B, t, s, H]
    y = (score[..., None] * x[:, None]).sum(2)
    y = y + ((c * torch.exp(cum)[..., None])[..., None] * S0[:, None]).sum(3)
    y = y + s["D"].view(1, 1, H, 1) * x
    if s["gate"] is not None:
        y = y * _silu(s["gate"].float())
    w = torch.exp(cum[:, -1:] - cum) * d
    S = torch.exp(cum[:, -1])[..., None, None] * S0
    S = S + ((b * w[..., None])[..., None] * x[..., None, :]).sum(1)
    if s["slot"] is None:
        s["state"].copy_(S)
    else:
        s["state"][s["slot"].long()] = S
    return y.to(s["x"].dtype), s["state"]


def _plain_conv(s):
    x, w = s["x"], s["w"].float()
    B, C, T = x.shape
    xt = x.transpose(1, 2)                                                   # [B, T, C]
    if "cu" in s:
        longest, seq, pos = _rows_of(s, T)
        rows = xt.new_zeros(s["cu"].numel() - 1, longest, C)
        rows[seq, pos] = xt[0]
        n = (s["cu"][1:] - s["cu"][:-1]).long()
    else:
        rows, n = xt, torch.full((B,), T, device=x.device)
    st = s["state0"].transpose(1, 2) if s["state0"] is not None else rows.new_zeros(rows.shape[0], TAPS, C)
    window = torch.cat([st, rows], dim=1)                                    # [B, L + T, C]
    taps = window.float()[:, 1:].unfold(1, TAPS, 1)
    y = _silu((taps * w).sum(-1) + s["bias"].float()).to(x.dtype)
    last = n[:, None] + torch.arange(TAPS, device=x.device)
    state = torch.gather(window, 1, last[..., None].expand(-1, -1, C)).transpose(1, 2).contiguous()
    return [(y[seq, pos][None] if "cu" in s else y).transpose(1, 2), state]


def _plain_blocks(s):
    lens, total, block = s["lens"].long(), s["total"], s["block"]
    n, dev = lens.numel(), lens.device
    cu = F.pad(lens.cumsum(0), (1, 0)).clamp(max=total)
    lens = cu[1:] - cu[:-1]
    count = torch.clamp((lens + block - 1) // block, min=1)                  # a row for empty ones too
    end = count.cumsum(0)
    row = torch.arange(total // block + n, device=dev)
    req = torch.searchsorted(end, row, right=True)
    live = req < n
    q = req.clamp(max=n - 1)
    idx = row - (end - count)[q]
    rows = torch.minimum(lens[q] - idx * block, torch.full_like(idx, block))
    table = torch.stack([q, cu[:-1][q] + idx * block, rows, idx], dim=1)
    none = torch.tensor([-1, 0, 0, 0], device=dev)
    table = torch.where(live[:, None], table, none)
    t = torch.arange(total, device=dev)
    tr = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    on = tr < n
    tq = tr.clamp(max=n - 1)
    slot = tq if s["slot"] is None else s["slot"].long()[tq]
    return [cu.int(), table.int(), torch.where(on, slot, -1).int(),
            torch.where(on, t - cu[:-1][tq], 0).int()]


def _plain_norm(s):
    x, g = s["x"].float(), _silu(s["gate"].float())
    u = x * g if s["gate_first"] else x
    v = u.view(u.shape[0], s["groups"], -1)
    u = (v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)).view(u.shape) * s["w"]
    return (u if s["gate_first"] else u * g).to(s["x"].dtype)


# ---------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["C"]
        return {"bytes": 6 * n + 4 * case["C"], "flops": 12 * n}
    if op == "blocks":
        n = len(_lengths(case)) if "lengths" in case else case["requests"]
        total = sum(_lengths(case)) if "lengths" in case else n * 2 + n * case["most"] // 5
        total += case["spare"]
        return {"bytes": 4 * n * (2 if case["slots"] else 1) + 4 * (n + 1)
                + 16 * (total // case["block"] + n) + 8 * total, "flops": 4 * total}
    seqs = len(_lengths(case)) if "lengths" in case else case["B"]
    tokens = sum(_lengths(case)) if "lengths" in case else seqs * case["T"]
    if op == "conv":
        C = case["C"]
        return {"bytes": 4 * tokens * C + 2 * TAPS * C * seqs * (2 if case["state"] else 1)
                + 2 * (TAPS + 1) * C, "flops": (2 * TAPS + 5) * tokens * C}
    H, P, N, G = (case[k] for k in "HPNG")
    return {"bytes": tokens * (2 * H * P * (3 if case["z"] else 2) + 4 * G * N + 2 * H)
            + 8 * seqs * H * N * P + 12 * H, "flops": tokens * H * (5 * N * P + 8 * P)}


# ---------------------------------------------------------------- 64-bit results
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "blocks":
        return None
    if op == "norm":
        x, g, w = s["x"].double(), s["gate"].double(), s["w"].double()
        gate = g / (1 + torch.exp(-g))
        if case["gate_first"]:
            x = x * gate
        size = case["C"] // case["groups"]
        out = torch.empty_like(x)
        for k in range(case["groups"]):
            part = x[:, k * size:(k + 1) * size]
            ms = part.square().sum(1, keepdim=True) / size
            out[:, k * size:(k + 1) * size] = part / torch.sqrt(ms + EPS)
        out = out * w
        return out if case["gate_first"] else out * gate
    cuts = [0]
    for n in (_lengths(case) if "lengths" in case else [case["T"]] * case["B"]):
        cuts.append(cuts[-1] + n)
    if op == "conv":
        flat = s["x"].transpose(1, 2).reshape(-1, case["C"]).double()
        w, bias, ys, states = s["w"].double(), s["bias"].double(), [], []
        for i, (lo, hi) in enumerate(zip(cuts, cuts[1:])):
            old = s["state0"][i].t().double() if case["state"] else flat.new_zeros(TAPS, case["C"])
            line = torch.cat([old, flat[lo:hi]])
            acc = bias.expand(hi - lo, -1)
            for j in range(TAPS):
                acc = acc + line[1 + j:1 + j + hi - lo] * w[:, j]
            ys.append(acc / (1 + torch.exp(-acc)))
            states.append(line[line.shape[0] - TAPS:].t())
        y = torch.cat(ys).view(s["x"].shape[0], -1, case["C"]).transpose(1, 2)
        return [y, torch.stack(states)]
    # the recurrence itself, token by token over all sequences at once
    H, P, N, G = (case[k] for k in "HPNG")
    lens = torch.tensor([b - a for a, b in zip(cuts, cuts[1:])], device="cuda")
    first = torch.tensor(cuts[:-1], device="cuda")
    flat = {k: s[k].reshape(-1, *s[k].shape[2:]) for k in ("x", "b", "c", "dt")}
    S = s["state"].double()
    slot = s.get("slot")
    if slot is not None:
        pool, S = S, S[slot.long()]
    A, bias = -torch.exp(s["A_log"].double()), s["dt_bias"].double()
    y = torch.zeros(flat["x"].shape, dtype=torch.float64, device="cuda")
    longest = max(b - a for a, b in zip(cuts, cuts[1:]))
    for t in range(longest):
        live = (lens > t).nonzero()[:, 0] if "lengths" in case else slice(None)
        at = (first + t)[live]
        d = torch.log1p(torch.exp(flat["dt"][at].double() + bias))
        xt = flat["x"][at].double()
        bt = flat["b"][at].double().repeat_interleave(H // G, dim=1)
        ct = flat["c"][at].double().repeat_interleave(H // G, dim=1)
        new = torch.exp(A * d)[..., None, None] * S[live] + bt[..., None] * (d[..., None] * xt)[:, :, None]
        S[live] = new
        y[at] = torch.matmul(ct[:, :, None], new)[:, :, 0] + s["D"].double()[:, None] * xt
    y = y.view(s["x"].shape)
    if s["gate"] is not None:
        z = s["gate"].double()
        y = y * z / (1 + torch.exp(-z))
    if slot is not None:
        pool[slot.long()] = S
        S = pool
    return [y, S] if op == "scan" else (y, S)
