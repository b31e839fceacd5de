"""How many rows, records and bytes a split scan takes, on the CPU."""
import ctypes as ct
import random

import pytest

from gdn_hip import capi

P = 1 << 20   # an aligned non-null address, never read


def _inputs(tokens, heads=64, head_dim=64, groups=8, state_dim=128, batch=1):
    n, g = heads * head_dim, groups * state_dim
    return capi.SsmInputs(x=P, dt=P, b=P, c=P, A_log=P, x_token=n, dt_token=heads, b_token=g, c_token=g,
                          batch=batch, tokens=tokens, heads=heads, head_dim=head_dim, groups=groups,
                          state_dim=state_dim, io_dtype=0, dt_dtype=0, dt_min=0.0, dt_max=1e30)


def _splits():
    rng = random.Random(1)
    yield [0] * 50
    yield [64] * 40
    yield [65] * 40
    yield [63] * 40
    yield [1] * 300 + [5000]
    yield [129, 0, 1, 128, 127, 4096, 0, 0, 255, 256, 257]
    for _ in range(200):
        n = rng.randrange(1, 60)
        yield [rng.choice((0, 1, 63, 64, 65, rng.randrange(2000))) for _ in range(n)]


@pytest.mark.parametrize("block", [64, 128, 192, 1024])
def test_rows_and_records_of_any_split(block):
    """Rows stay within the bound that is allocated without the lengths, and the
    records of segments with another behind them, at first token / block, are
    distinct and within (tokens - 1) / block, wherever the first sequence starts."""
    lib = capi.lib()
    for lengths in _splits():
        for lead in (0, 1, 40):
            total = lead + sum(lengths)
            rows = sum(max(1, -(-n // block)) for n in lengths)
            assert rows <= lib.gdn_request_block_rows(total, len(lengths), block)
            recs, lo = [], lead
            for n in lengths:
                recs += [t // block for t in range(lo, lo + n - block, block)]
                lo += n
            assert len(set(recs)) == len(recs)
            assert all(0 <= r < max(total - 1, 0) // block for r in recs)
    assert lib.gdn_request_block_rows(0, 7, block) == 7   # one row an empty sequence


@pytest.mark.parametrize("block", [64, 256, 1 << 20])
@pytest.mark.parametrize("seqs,tokens", [(1500, 1500), (1500, 12000), (1, 4096), (4000, 0)])
def test_workspace_holds_no_more_records_than_can_be(seqs, tokens, block):
    """A batch of single tokens takes megabytes, not a state for each request."""
    a = _inputs(tokens)
    need = capi.lib().gdn_ssm_scan_workspace_size(ct.byref(a), seqs, block, 1)
    state = a.heads * a.head_dim * a.state_dim * 4
    records = max(tokens - 1, 0) // block
    rows = tokens // block + seqs
    assert records * state < need <= records * (state + 4 * 2 * a.heads) + 40 * rows + 4096


def test_workspace_of_fixed_lengths():
    """The last segment of a sequence has no record; a state of 16 rows has none at all."""
    a = _inputs(1000, batch=3)
    state = a.heads * a.head_dim * a.state_dim * 4
    need = capi.lib().gdn_ssm_scan_workspace_size(ct.byref(a), 3, 256, 0)
    assert 9 * state < need < 10 * state
    assert capi.lib().gdn_ssm_scan_workspace_size(ct.byref(a), 3, 1024, 0) < 4096
    a = _inputs(4096, state_dim=16)
    assert 0 < capi.lib().gdn_ssm_scan_workspace_size(ct.byref(a), 5, 64, 1) < 4096
