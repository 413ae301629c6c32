"""Prompt attention with score modifications when q_start is not well formed:
which rows are computed, which are left as they were, and what is reported."""
import numpy as np
import pytest

from oracle import attention_mod as orc
from tests.test_gpu_attention_mod import Case, i32, torch_cuda  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

T = 60


@pytest.mark.parametrize("q_start,bad", [
    ([0, 30, 20, 60], True),    # decreases: the middle sequence has no rows, the others share ten
    ([0, 40, 50, 90], True),    # leaves the rows at the end
    ([-4, 10, 20, 60], True),   # and at the start
    ([0, 10, 5, 5], True),      # decreases, most rows uncovered
    ([0, 25, 70, 80], True),    # the last sequence lies behind the rows
    ([5, 20, 20, 41], False),   # well formed, with rows before the first and behind the last sequence
    ([0, 0, 0, 0], False),      # no rows at all
    ([60, 60, 60, 60], False),
])
@pytest.mark.parametrize("ctx", [[0, 0, 0], [40, 7, 1500]])
def test_rows_of_each_sequence(torch_cuda, q_start, bad, ctx):  # noqa: F811
    torch = torch_cuda
    from python.kinetic_rt import _lib
    c = Case(torch, ctx, q_lens=[20, 20, 20], seed=18)
    wide = torch.zeros(3, 110, dtype=torch.int32, device="cuda")  # room for any sequence's tokens
    full = np.random.Generator(np.random.PCG64(19)).integers(0, c.blocks, (3, 110)).astype(np.int32)
    wide.copy_(torch.from_numpy(full))
    c.table_d, c.table = wide, full
    a = c.args(max_len=110 * 16)
    start = i32(torch, q_start)
    a.q_start = start.data_ptr()
    for _ in range(2):
        c.out.fill_(9.0)
        c.lse.fill_(7.0)
        c.launch(a)
        rc, bits = _lib.read_status(c.ws)
        assert bits == (8 if bad else 0)
        c.ws[:4] = 0
        covers, rows = np.zeros(T, int), [None] * T
        for s in range(3):
            first, end = max(q_start[s], 0), min(q_start[s + 1], T)
            whole = 0 <= q_start[s] <= q_start[s + 1] <= T
            for t in range(first, end):
                covers[t] += 1
                if whole:
                    rows[t] = (s, ctx[s] + t - first, ctx[s] + end - first, 0, 0)
        rows = [r if n == 1 else None for r, n in zip(rows, covers)]
        ref, lse, tol, tol_lse = orc.paged_attention_mod(c.q, c.pool, c.table, rows, c.H, c.K, c.tpb)
        got, got_lse = c.result()
        keep = np.array([r is not None for r in rows])
        assert (np.abs(got - ref) <= tol)[keep].all()
        assert (np.abs(got_lse - lse)[keep] <= tol_lse[keep]).all()
        assert (got[covers == 0] == 9.0).all() and (got_lse[covers == 0] == 7.0).all()
        assert np.isfinite(got[covers > 0]).all() and (got_lse[covers > 0] != 7.0).all()
