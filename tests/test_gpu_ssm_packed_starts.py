"""Packed rows whose first sequence does not start at token 0."""
import pytest
import torch

import gdn_hip
import ssm_cases as sc
from gdn_hip import capi
from oracle import ssm_oracle as orc

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("T,D", [(60, 64), (3080, 4096)], ids=["short runs", "long runs"])
@pytest.mark.parametrize("K", [2, 4])
@pytest.mark.parametrize("first", [1, 2, 5, 8])
def test_conv(dev, first, K, T, D):
    """Every row from cu_seqlens[0] on is its sequence's alone (the taps in front
    of it are state0's), and the rows before it are left as they were; 3080
    tokens of 4096 channels take the instance with the longer runs.

    Bound: at most 5 terms in fp32 (5 x 2^-24 of the absolute sum, SiLU's slope
    at most 1.1), SiLU's own 2^-20, half a step of bf16."""
    g = torch.Generator().manual_seed(10 * first + K)
    lengths = [3, 0, 21, T - first - 24 - 5]
    x = torch.randn(1, T, D, generator=g).to(BF)
    w = (0.5 * torch.randn(D, K, generator=g)).to(BF)
    s0 = torch.randn(4, D, 4, generator=g).to(BF)
    cu = torch.tensor([first + sum(lengths[:i]) for i in range(5)], dtype=torch.int32, device=dev)
    xd, wd, sd = x.to(dev), w.to(dev), s0.to(dev)
    y = torch.full((T, D), 7.0, dtype=BF, device=dev)
    st = torch.empty_like(sd)
    print(f"conv from token {first}, K={K}, {T} x {D}", flush=True)
    assert capi.lib().gdn_causal_conv1d_prefill(
        xd.data_ptr(), wd.data_ptr(), None, sd.data_ptr(), y.data_ptr(), st.data_ptr(), 1, T, D, K, 4,
        T * D, D, T * D, D, cu.data_ptr(), 4, 0, 0, 1, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    ref, rst, mag = orc.conv_prefill(x[:, first:].transpose(1, 2), w, None, s0, True, lengths)
    bound = 2.0 ** -8 * ref.abs() + (8 * 2.0 ** -24 * mag * 1.1 + 2.0 ** -20 * ref.abs()) * 1.01 + 2.0 ** -134
    sc.close(y[first:T - 5].t()[None], ref, bound, "conv y")
    assert (y[:first] == 7).all() and (y[T - 5:] == 7).all()
    assert torch.equal(st.double().cpu(), rst)


@pytest.mark.parametrize("first", [1, 63, 64, 100])
def test_scan(dev, first):
    """The same of the scan."""
    lengths = [70, 0, 130, 9]
    T = first + sum(lengths) + 3
    d = sc.inputs(first, 1, T, 4, 64, 2, 128)
    seq = ("x", "dt", "B", "C", "z")
    y, S, ya, Sa = orc.ssm_packed(lengths, **{k: (v[:, first:-3] if k in seq else v) for k, v in d.items()})
    g = sc.to(d, dev)
    cu = torch.tensor([first + sum(lengths[:i]) for i in range(5)], dtype=torch.int32, device=dev)
    print(f"scan from token {first}", flush=True)
    oy, oS = gdn_hip.ssm_scan(*(g[k] for k in ("x", "dt", "A_log", "B", "C", "D", "z", "dt_bias")), cu_seqlens=cu)
    torch.cuda.synchronize()
    by, bS = sc.bounds(d, 130, y, ya, Sa, BF)
    sc.close(oy[:, first:-3], y, by, "scan y")
    sc.close(oS, S, bS, "scan state")
