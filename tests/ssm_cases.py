"""Seeded inputs and error bounds shared by the state-space tests."""
import torch

from oracle import ssm_oracle as orc


def inputs(seed, B, T, H, P, G, N, dtype=torch.bfloat16, z=True, dt_dtype=None, slow=True):
    """CPU tensors of a layer: x, B, C slices of one conv output, z and dt of one projection."""
    g = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=g)

    conv = rn(B, T, H * P + 2 * G * N).to(dtype)
    x, b, c = torch.split(conv, [H * P, G * N, G * N], dim=-1)
    proj = torch.cat([rn(B, T, H * P), rn(B, T, H)], dim=-1).to(dtype)
    dt = proj[..., H * P:]
    if dt_dtype is not None:
        dt = dt.to(dt_dtype)
    return dict(x=x.unflatten(-1, (H, P)), dt=dt,
                A_log=torch.log(0.05 + (1 if slow else 15) * torch.rand(H, generator=g)),
                B=b.unflatten(-1, (G, N)), C=c.unflatten(-1, (G, N)), D=rn(H),
                z=proj[..., :H * P].unflatten(-1, (H, P)) if z else None,
                dt_bias=-2 + rn(H))


def to(d, dev):
    # a slice moves as a slice: strides are kept by moving its base
    out = {}
    for k, v in d.items():
        out[k] = None if v is None else v.to(dev) if v.is_contiguous() or v.dim() < 3 else \
            v._base.to(dev).as_strided(v.size(), v.stride(), v.storage_offset())
    return out


def bounds(d, T, y, ya, Sa, dtype):
    """Elementwise bounds of (y, state).  Arithmetic: a state is a sum over at
    most T tokens whose decays are products of up to T factors, each factor's
    logarithm A d with a relative error of 2^-22 and the sums of logarithms
    with one of 2^-24 per token, all against the recurrence of absolute values;
    y adds operands split into two 8-bit parts (2^-16 relative, two products).
    Then y's own rounding, half a step of its type."""
    la = (torch.exp(d["A_log"].double()) * orc.softplus(d["dt"].double() + d["dt_bias"].double())).max().item()
    arith = (16 + 4 * T * (1 + min(la, 8.0))) * 2.0 ** -24
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half
    return half * y.abs() + (arith + 2.0 ** -15) * (1 + half) * ya + tiny, arith * Sa + 1e-30


def close(got, ref, bound, tag):
    got = got.double().cpu()
    assert got.shape == ref.shape, tag
    assert torch.isfinite(got).all(), f"{tag}: not finite"
    worst = ((got - ref).abs() / bound).max().item() if got.numel() else 0.0
    print(f"{tag}: {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, f"{tag}: {worst:.3f} of the bound"
