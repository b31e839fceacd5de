"""Host checks of the state-space entries, all before any launch (no GPU), and
the 64-bit oracle against its own closed forms."""
import ctypes as ct

import pytest
import torch

import gdn_hip
from gdn_hip import capi
from oracle import ssm_oracle as orc

INVALID = capi.HIP_ERROR_INVALID_VALUE
P = 1 << 20   # an aligned non-null address, never read


def _inputs(**over):
    a = dict(x=P, dt=P, b=P, c=P, z=P, A_log=P, D=P, dt_bias=P, x_batch=512, x_token=256,
             dt_batch=8, dt_token=4, b_batch=512, b_token=256, c_batch=512, c_token=256,
             z_batch=512, z_token=256, batch=2, tokens=2, heads=4, head_dim=64, groups=2,
             state_dim=128, io_dtype=0, dt_dtype=0, dt_min=0.0, dt_max=1e30)
    a.update(over)
    return capi.SsmInputs(**a)


BAD = [dict(x=None), dict(dt=None), dict(b=None), dict(c=None), dict(A_log=None), dict(x=P + 8),
       dict(z=P + 2), dict(b=P + 4), dict(x_token=12), dict(c_token=-8), dict(b_token=1 << 24),
       dict(x_token=1 << 24), dict(heads=1 << 18, groups=2),
       dict(dt_token=-1), dict(z_batch=4), dict(batch=0), dict(tokens=-1), dict(heads=0),
       dict(groups=3), dict(groups=0), dict(head_dim=8), dict(head_dim=72), dict(head_dim=272),
       dict(state_dim=48), dict(state_dim=512), dict(io_dtype=2), dict(dt_dtype=1),
       dict(dt_min=-1.0), dict(dt_min=2.0, dt_max=1.0), dict(dt_max=float("nan"))]


@pytest.mark.parametrize("bad", BAD, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_ssm_refuses(bad):
    lib, a = capi.lib(), _inputs(**bad)
    assert lib.gdn_ssm_step(ct.byref(a), P, P, None, 0, None) == INVALID
    assert lib.gdn_ssm_scan(ct.byref(a), P, P, 2 * P, None, None, a.batch, 64, P, 1 << 40, None) == INVALID


def test_ssm_refuses_outputs_and_tables():
    lib, a, r = capi.lib(), _inputs(), ct.byref(_inputs())
    assert lib.gdn_ssm_step(r, None, P, None, 0, None) == INVALID
    assert lib.gdn_ssm_step(r, P, None, None, 0, None) == INVALID
    assert lib.gdn_ssm_step(r, P, P + 2, None, 0, None) == INVALID
    assert lib.gdn_ssm_step(r, P, P, P, 0, None) == INVALID           # an empty pool
    assert lib.gdn_ssm_step(None, P, P, None, 0, None) == INVALID
    need = lib.gdn_ssm_scan_workspace_size(r, 2, 64, 0)
    assert need > 0
    ok = [r, P, P, 2 * P, None, None, 2, 64, P, need, None]
    assert lib.gdn_ssm_scan(r, P, P, P, None, None, 2, 64, P, need, None) == INVALID   # sf is s0

    def scan(**over):
        args = list(ok)
        for k, v in over.items():
            args[int(k[1:])] = v
        return lib.gdn_ssm_scan(*args)

    assert scan(_1=None) == INVALID and scan(_3=None) == INVALID
    assert scan(_8=None) == INVALID and scan(_9=need - 1) == INVALID and scan(_8=P + 16) == INVALID
    assert scan(_6=3) == INVALID                                      # not the batch
    assert scan(_4=P) == INVALID                                      # packed with batch 2
    assert scan(_5=P) == INVALID                                      # a table without cu_seqlens
    for block in (0, 32, 96, 1 << 21):
        assert scan(_7=block) == INVALID
    assert lib.gdn_ssm_scan_workspace_size(r, 2, 96, 0) == 0
    assert lib.gdn_ssm_scan_workspace_size(r, 5, 64, 1) == 0          # batch 2 is not packed
    assert lib.gdn_ssm_scan_block(r, 0) == 0
    assert lib.gdn_ssm_scan_block(r, 2) % 64 == 0 and lib.gdn_ssm_scan_block(r, 2) >= 64


def test_scan_without_tokens_still_needs_a_log():
    """States pass through such a call, and its kernels read A_log."""
    lib = capi.lib()
    for state_dim in (16, 128):
        a = _inputs(tokens=0, A_log=None, state_dim=state_dim)
        assert lib.gdn_ssm_scan(ct.byref(a), P, P, 2 * P, None, None, 2, 64, P, 1 << 40, None) == INVALID


@pytest.mark.parametrize("tokens", [0, 1, 1000, 1 << 17, 1 << 30])
def test_block_is_one_the_scan_takes(tokens):
    """Blocks and workspaces for one sequence, many, and more than fill the chip."""
    lib = capi.lib()
    for seqs in (1, 2, 40, 3000):
        for heads, state_dim in ((2, 32), (64, 128), (64, 256)):
            a = _inputs(batch=1, tokens=tokens, heads=heads, state_dim=state_dim)
            block = lib.gdn_ssm_scan_block(ct.byref(a), seqs)
            assert 64 <= block <= 1 << 20 and block % 64 == 0
            assert lib.gdn_ssm_scan_workspace_size(ct.byref(a), seqs, block, 1) > 0


def test_workspace_covers_every_split():
    """The packed bound holds for any lengths, empty sequences too."""
    lib = capi.lib()
    for tokens, seqs, block in ((0, 1, 64), (1000, 7, 64), (1 << 20, 3, 512), (130, 200, 128)):
        a = _inputs(batch=1, tokens=tokens)
        assert lib.gdn_ssm_scan_workspace_size(ct.byref(a), seqs, block, 1) > 0


def test_request_blocks_refuses():
    lib = capi.lib()
    assert lib.gdn_request_block_rows(1000, 3, 64) == 1000 // 64 + 3
    for bad in ((-1, 3, 64), ((1 << 30) + 1, 3, 64), (10, 0, 64), (10, 3, 32), (10, 3, 100), (10, 3, 0),
                (10, (1 << 24) + 1, 64)):
        assert lib.gdn_request_block_rows(*bad) == 0
    ok = [P, None, 3, 100, 64, P, P, P, P, P, None]
    for i, v in ((0, None), (2, 0), (3, -1), (4, 63), (5, None), (6, None), (7, None), (8, None),
                 (9, None), (7, P + 4), (8, P + 8), (9, P + 4)):
        args = list(ok)
        args[i] = v
        assert lib.gdn_request_blocks(*args) == INVALID


def test_conv_prefill_refuses():
    lib = capi.lib()
    ok = [P, P, None, P, P, 2 * P, 2, 5, 64, 4, 4, 320, 64, 320, 64, None, 2, 0, 0, 1, None]
    for i, v in ((0, None), (1, None), (4, None), (5, None), (5, P), (0, P + 2), (3, P + 8), (6, 0),
                 (7, -1), (8, 12), (8, 0), (9, 1), (9, 5), (10, 2), (10, 9), (11, 4), (12, -8),
                 (14, 7), (16, 3), (16, 0), (15, P), (17, 2), (18, 1), (19, 2)):
        args = list(ok)
        args[i] = v
        assert lib.gdn_causal_conv1d_prefill(*args) == INVALID, (i, v)


def test_update_slots_refuses():
    lib = capi.lib()
    ok = [P, P, P, None, P, P, 4, 2, 1, 64, 4, 4, 64, 64, 1, 256, 4, 64, 64, 1, 0, 0, 1, None]
    for i, v in ((0, None), (1, None), (5, None), (6, 0), (6, -1), (10, 5), (11, 2), (11, 9), (20, 2)):
        args = list(ok)
        args[i] = v
        assert lib.gdn_causal_conv1d_update_slots(*args) == INVALID, (i, v)


def test_groupnorm_refuses():
    lib = capi.lib()
    ok = [P, 512, P, 512, P, P, 10, 512, 2, 1e-6, 1, 0, 0, None]
    for i, v in ((0, None), (2, None), (4, None), (5, None), (0, P + 2), (1, 4), (3, -8), (6, -1),
                 (7, 4), (8, 3), (8, 0), (8, 128), (9, -1.0), (9, float("nan")), (10, 2), (11, 2),
                 (12, 1)):
        args = list(ok)
        args[i] = v
        assert lib.gdn_gated_groupnorm_forward(*args) == INVALID, (i, v)
    assert lib.gdn_gated_groupnorm_forward(*(ok[:7] + [16392, 1] + ok[9:])) == INVALID
    assert lib.gdn_gated_groupnorm_forward(*(ok[:6] + [0] + ok[7:])) == 0      # no rows


def _cpu_args():
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    bc = torch.zeros(1, 2, 2, 128, dtype=torch.bfloat16)
    return [x, torch.zeros(1, 2, 4), torch.zeros(4), bc, bc]


def test_ops_refuse_host_tensors():
    a = _cpu_args()
    with pytest.raises(RuntimeError, match="HIP device"):
        gdn_hip.ssm_scan(*a)
    with pytest.raises(RuntimeError, match="HIP device"):
        gdn_hip.ssm_step(*a, torch.zeros(1, 4, 128, 64))
    x = torch.zeros(1, 64, 5, dtype=torch.bfloat16)
    w = torch.zeros(64, 4, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        gdn_hip.causal_conv1d_prefill(x, w)
    with pytest.raises(RuntimeError, match="HIP device"):
        gdn_hip.request_blocks(torch.zeros(3, dtype=torch.int32), 10)
    with pytest.raises(RuntimeError, match="HIP device"):
        gdn_hip.gated_groupnorm(x, x, torch.ones(5), 1)
    with pytest.raises(RuntimeError):
        gdn_hip.causal_conv1d_update(x, torch.zeros(3, 64, 4, dtype=torch.bfloat16), w,
                                     slots=torch.zeros(1, dtype=torch.int32))


def test_oracle_scan_closed_form():
    """y_t = sum_s (C_t . B_s) e^{c_t - c_s} d_s x_s against the recurrence."""
    g = torch.Generator().manual_seed(1)
    T, N, Pd = 9, 16, 8
    x, b, c = (torch.randn(1, T, 1, n, generator=g, dtype=torch.float64) for n in (Pd, N, N))
    dt, A_log = torch.randn(1, T, 1, generator=g, dtype=torch.float64), torch.tensor([0.3]).double()
    y, S, _, _ = orc.ssm(x, dt, A_log, b, c)
    d = torch.nn.functional.softplus(dt[0, :, 0])
    cum = (-A_log.exp() * d).cumsum(0)
    L = torch.exp(cum[:, None] - cum).tril()
    M = (c[0, :, 0] @ b[0, :, 0].t()) * L * d
    assert torch.allclose(y[0, :, 0], M @ x[0, :, 0], atol=1e-12)
    w = torch.exp(cum[-1] - cum) * d
    assert torch.allclose(S[0, 0], (b[0, :, 0] * w[:, None]).t() @ x[0, :, 0], atol=1e-12)


def test_oracle_tables():
    cu, table, slot, pos = orc.request_blocks([70, 0, 3], 80, 64, [5, 6, 7])
    assert cu == [0, 70, 70, 73]
    assert table == [[0, 0, 64, 0], [0, 64, 6, 1], [1, 70, 0, 0], [2, 70, 3, 0]]
    assert slot == [5] * 70 + [7] * 3 + [-1] * 7 and pos == list(range(70)) + [0, 1, 2] + [0] * 7
