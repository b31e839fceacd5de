"""The scan where decays of very different size meet."""
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
