"""The scan where values or decays of very different size meet: resets among
weak decays, channels of mixed magnitude, states far from 1, and inputs that
are not finite."""
import pytest
import torch

import gdn_hip
import ssm_cases as sc
from oracle import ssm_oracle as orc

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
ARGS = ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")


def _scan(d, dev, s0=None, **kw):
    g = sc.to(d, dev)
    out = gdn_hip.ssm_scan(*(g[k] for k in ARGS), None if s0 is None else s0.to(dev), **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
def test_resets_cost_no_precision(dev, dtype):
    """The weight of one token for another behind the same reset is as exact as
    without any reset.

    A term of y whose decay is e^-L has a relative error of (16 + L) 2^-22: each
    token's logarithm within 2^-22 of itself, their sums within 2^-24 a step.
    Here L is below 8, that is 2^-17.4; M enters the product in two parts, of
    bf16 2^-18 off, and then y is rounded."""
    T = 640
    d = sc.inputs(50, 1, T, 3, 64, 1, 64, dtype, dt_dtype=torch.float32, z=False)
    # 13 resets and 3 weak decays in every 16 tokens: x enters at the first weak
    # one, the y of the next two is one weight each, and no term cancels another
    at = torch.arange(T) % 16
    d["dt"] = torch.where((at < 13)[None, :, None], torch.tensor(1e4), d["dt"] - 1)
    d["x"] = torch.where((at == 13)[None, :, None, None], d["x"].abs(), torch.zeros((), dtype=dtype))
    d["B"], d["C"] = d["B"].abs(), d["C"].abs()
    y, S, ya, Sa = orc.ssm(**d)
    print(f"resets {dtype}", flush=True)
    oy, oS = _scan(d, dev)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half
    sc.close(oy, y, half * y.abs() + 2.0 ** -16.5 * (1 + half) * ya + tiny, f"resets {dtype} y")


def test_fp16_large_steps_of_zeros(dev):
    """Steps of 1e4 whose x is 0 leave the state of the other tokens exact."""
    T = 640
    d = sc.inputs(51, 1, T, 3, 64, 1, 64, HF, dt_dtype=torch.float32, z=False)
    wipe = torch.rand(T, generator=torch.Generator().manual_seed(0)) < 0.5
    d["dt"] = torch.where(wipe[None, :, None], torch.tensor(1e4), d["dt"] - 2)
    d["x"] = torch.where(wipe[None, :, None, None], torch.zeros((), dtype=HF), d["x"])
    for n in range(T - 6, T):   # the last token a reset, and not
        e = {k: (v[:, :n] if k in ("x", "dt", "B", "C") else v) for k, v in d.items()}
        y, S, ya, Sa = orc.ssm(**e)
        print(f"large steps, {n} tokens", flush=True)
        oy, oS = _scan(e, dev)
        # (16 + L) 2^-22 of a term of decay e^-L, as above
        sc.close(oS, S, 2.0 ** -17 * Sa + 1e-30, "large steps state")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_d_x_is_rounded_once(dev, dtype):
    """With C = 0, y is D x: rounded to the type as the 64-bit product is, wherever
    that lies further from a border than what three bf16 parts of D (2^-24) and
    two sums in fp32 are off, or two fp16 parts (2^-22): 2^-21 and 2^-20 of it."""
    d = sc.inputs(5, 1, 300, 512, 16, 1, 32, dtype, z=False)   # many values of D
    d["C"] = torch.zeros_like(d["C"])
    print(f"D x {dtype}", flush=True)
    oy, _ = _scan(d, dev)
    y = d["D"].double()[:, None] * d["x"].double()
    away = 2.0 ** (-21 if dtype == BF else -20) * y.abs()
    clear = (y - away).to(dtype) == (y + away).to(dtype)
    clear &= y.abs() > torch.finfo(dtype).smallest_normal   # (below, fp16 is in steps of 2^-24)
    assert clear.double().mean() > 0.99
    assert torch.equal(oy.cpu()[clear], y.to(dtype)[clear])


@pytest.mark.parametrize("N", [32, 64, 128, 256])
@pytest.mark.parametrize("T", [20, 64, 150])
def test_fp16_channels_of_mixed_magnitude(dev, T, N):
    """Small channels next to an outlier keep every bit of their states: bounds
    are elementwise, so each channel is held to its own size."""
    d = sc.inputs(T, 1, T, 2, 96, 1, N, HF, z=False)
    size = 10.0 ** (-3 + 3 * torch.rand(96, generator=torch.Generator().manual_seed(N)))
    size[::13] = 1.5e4
    d["x"] = (d["x"].float().clamp(-4, 4) * size).to(HF)
    d["C"] = (d["C"].float() * 1e-3).to(HF)
    d["D"] = d["D"] * 0
    s0 = torch.randn(1, 2, N, 96, generator=torch.Generator().manual_seed(T)) * size
    y, S, ya, Sa = orc.ssm(**d, s0=s0)
    assert y.abs().max() < 6e4
    print(f"mixed channels T={T} N={N}", flush=True)
    oy, oS = _scan(d, dev, s0)
    by, bS = sc.bounds(d, T, y, ya, Sa, HF)
    sc.close(oS, S, bS, "mixed state")
    sc.close(oy, y, by, "mixed y")


def test_fp16_state_far_above_what_is_read(dev):
    """A state of 2^50 that C never reads, and steps of 0: y is 0, not NaN."""
    d = sc.inputs(3, 1, 70, 2, 64, 1, 64, HF, z=False)
    d["dt"] = torch.full_like(d["dt"], -float("inf"))
    d["C"] = torch.zeros_like(d["C"])
    d["D"] = torch.zeros_like(d["D"])
    s0 = 2.0 ** 50 * torch.randn(1, 2, 64, 64, generator=torch.Generator().manual_seed(1))
    oy, oS = _scan(d, dev, s0)
    assert (oy == 0).all() and torch.allclose(oS.cpu(), s0, rtol=2e-7)


BAD = [float("inf"), -float("inf"), float("nan")]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("N", [32, 128, 256])
@pytest.mark.parametrize("bad", BAD)
def test_x_not_finite(dev, bad, N, dtype):
    """A value of x that is not finite shows in its channel from its token on,
    and in nothing else: every other value is that of the call without it."""
    for T, t, p in ((200, 41, 3), (200, 0, 63), (64, 63, 40), (500, 130, 17), (17, 16, 1)):
        d = sc.inputs(T + t, 1, T, 2, 64, 1, N, dtype)
        d["dt_bias"] = d["dt_bias"] - 3
        d["x"] = d["x"].clone()
        d["x"][0, t, 1, p] = 0
        ry, rS = _scan(d, dev)
        d["x"][0, t, 1, p] = bad
        print(f"x {bad} at token {t} of {T}, N={N} {dtype}", flush=True)
        oy, oS = _scan(d, dev)
        assert not torch.isfinite(oy[0, t:, 1, p]).any() and not torch.isfinite(oS[0, 1, :, p]).any()
        oy[0, t:, 1, p], oS[0, 1, :, p] = ry[0, t:, 1, p], rS[0, 1, :, p]
        assert torch.equal(oy, ry) and torch.equal(oS, rS)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bad", BAD)
def test_others_not_finite(dev, bad, dtype):
    """C and z: their token's y alone.  B and dt: y from its token on.  s0: its
    channel's y.  Nothing in front, and no other channel."""
    T, t = 150, 75
    d = sc.inputs(6, 1, T, 2, 64, 1, 64, dtype)
    d["dt_bias"] = d["dt_bias"] - 3
    s0 = torch.randn(1, 2, 64, 64, generator=torch.Generator().manual_seed(1))
    ry, rS = _scan(d, dev, s0)
    step = torch.finfo(dtype).eps   # fp16: another scale of M, a rounding border away

    def near(a, b):
        assert torch.isfinite(a).all() and ((a.float() - b.float()).abs() <= step * (1 + b.float().abs())).all()

    for k in ("C", "z", "B", "dt"):
        e = dict(d)
        e[k] = d[k].clone()
        e[k][(0, t, 0, 5)[:d[k].dim()] if k != "dt" else (0, t, 1)] = bad
        print(f"{k} {bad} {dtype}", flush=True)
        if k == "dt" and bad == -float("inf"):
            continue   # a step of 0
        oy, oS = _scan(e, dev, s0)
        if k == "C":
            assert not torch.isfinite(oy[0, t]).any()
            oy[0, t] = ry[0, t]
        elif k == "z":
            assert not torch.isfinite(oy[0, t, 0, 5])
            oy[0, t, 0, 5] = ry[0, t, 0, 5]
        elif k == "B":
            assert not torch.isfinite(oy[0, t:]).any() and not torch.isfinite(oS[0, :, 5]).any()
            oy[0, t:], oS = ry[0, t:], rS
        else:
            assert not torch.isfinite(oy[0, t:, 1]).any() and not torch.isfinite(oS[0, 1]).any()
            oy[0, t:, 1], oS[0, 1] = ry[0, t:, 1], rS[0, 1]
        near(oy, ry)
        assert torch.allclose(oS, rS, rtol=1e-5, atol=1e-5)
    s = s0.clone()
    s[0, 1, 7, 9] = bad
    oy, oS = _scan(d, dev, s)
    assert not torch.isfinite(oy[0, :, 1, 9]).any() and not torch.isfinite(oS[0, 1, 7, 9])
    oy[0, :, 1, 9], oS[0, 1, 7, 9] = ry[0, :, 1, 9], rS[0, 1, 7, 9]
    assert torch.equal(oy, ry) and torch.equal(oS, rS)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_x_not_finite_in_a_split_sequence(dev, dtype):
    """Through the first pass, its records and their join."""
    T, t = 1250, 300
    assert gdn_hip.ssm_scan_block(T, 1, 2, 64, 1, 64, 1) == 64
    d = sc.inputs(8, 1, T, 2, 64, 1, 64, dtype)
    d["dt_bias"] = d["dt_bias"] - 3
    d["x"] = d["x"].clone()
    d["x"][0, t, 1, 7] = 0
    ry, rS = _scan(d, dev)
    d["x"][0, t, 1, 7] = float("inf")
    oy, oS = _scan(d, dev)
    assert not torch.isfinite(oy[0, t:, 1, 7]).any() and not torch.isfinite(oS[0, 1, :, 7]).any()
    oy[0, t:, 1, 7], oS[0, 1, :, 7] = ry[0, t:, 1, 7], rS[0, 1, :, 7]
    assert torch.equal(oy, ry) and torch.equal(oS, rS)
