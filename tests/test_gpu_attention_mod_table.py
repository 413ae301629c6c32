"""Sequences that reach beyond their block table, and block tables that are
column slices of wider ones, against oracle/attention_mod.py in 64 bits."""
import numpy as np
import pytest

from oracle import attention_mod as orc
from tests.test_gpu_attention_mod import Case, i32, torch_cuda  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def hold(c, rows, softcap=0.0, window=0):
    ref, lse, tol, tol_lse = orc.paged_attention_mod(c.q, c.pool, c.table, rows, c.H, c.K, c.tpb, softcap, window)
    got, got_lse = c.result()
    assert (np.abs(got - ref) <= tol).all()
    dead = np.isneginf(lse)
    assert (np.isneginf(got_lse) == dead).all()
    assert (np.abs(np.where(dead, 0, got_lse) - np.where(dead, 0, lse)) <= tol_lse).all()


@pytest.mark.parametrize("softcap,window", [(0.0, 0), (30.0, 0), (0.0, 40), (20.0, 90)])
@pytest.mark.parametrize("pos0", [300, 380, 5000, 2 ** 30])
def test_prompt_beyond_its_table(torch_cuda, pos0, softcap, window):  # noqa: F811
    """Keys end with the table: rows near its end see what their window leaves of it, far ones with a window nothing."""
    torch = torch_cuda
    from python.kinetic_rt import _lib
    c = Case(torch, [310, 100], q_lens=[74, 20], seed=90)  # tables of 384 positions
    cap = c.table.shape[1] * c.tpb
    a = c.args(softcap=softcap, window=window)
    start = i32(torch, [pos0, 100])
    a.q_pos0 = start.data_ptr()
    c.launch(a)
    rc, bits = _lib.read_status(c.ws)
    assert bits == (0 if pos0 + 74 <= cap else 8)
    rows = [(0, pos0 + i, min(pos0 + 74, cap), 0, 0) for i in range(74)] + [(1, 100 + i, 120, 0, 0) for i in range(20)]
    hold(c, rows, softcap, window)


def test_prompt_beyond_its_table_with_prefix_and_starts(torch_cuda):  # noqa: F811
    torch = torch_cuda
    from python.kinetic_rt import _lib
    c = Case(torch, [0], q_lens=[40], seed=91)  # 48 positions
    first = [0, 47, 48, 1 << 30, 20] * 8
    a = c.args(kv_start=first, prefix=[10 ** 6])
    start = i32(torch, [2 ** 20])
    a.q_pos0 = start.data_ptr()
    c.launch(a)
    assert _lib.read_status(c.ws)[1] == 8
    hold(c, [(0, 2 ** 20 + i, 48, first[i], 10 ** 6) for i in range(40)])
