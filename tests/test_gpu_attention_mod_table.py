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


# ------------------------------------------------------------ column slices
def sliced(torch, table, columns, last):
    """The table as columns of a wider one whose other entries name no block (last: the slice ends with the memory)."""
    S, n = table.shape
    wide = torch.full((S, 3 * n), 2 ** 30, dtype=torch.int32, device="cuda")
    at = 2 * n if last else n
    wide[:, at:at + n] = torch.from_numpy(table).cuda()
    return wide[:, at:at + columns]


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("q_lens", [None, [70, 30, 64]])
def test_attention_on_a_slice_of_a_table(torch_cuda, q_lens, last):  # noqa: F811
    torch = torch_cuda
    c = Case(torch, [300, 17, 128], q_lens=q_lens, seed=92)
    c.table_d = sliced(torch, c.table, c.table.shape[1], last)
    c.check(softcap=30.0)


@pytest.mark.parametrize("last", [False, True])
def test_prompt_beyond_a_slice(torch_cuda, last):  # noqa: F811
    """Keys end with the slice, though its row goes on."""
    torch = torch_cuda
    from python.kinetic_rt import _lib
    c = Case(torch, [310, 100], q_lens=[74, 20], seed=93)
    c.table_d = sliced(torch, c.table, 20, last)  # 320 of 384 positions
    c.launch(c.args(max_len=320))
    assert _lib.read_status(c.ws)[1] == 8
    hold(c, [(0, 310 + i, 320, 0, 0) for i in range(74)] + [(1, 100 + i, 120, 0, 0) for i in range(20)])


@pytest.mark.parametrize("q_lens", [None, [70, 30]])
def test_bound_beyond_a_slice_is_refused(torch_cuda, q_lens):  # noqa: F811
    torch = torch_cuda
    c = Case(torch, [300, 100], q_lens=q_lens, seed=94)
    c.table_d = sliced(torch, c.table, 10, False)
    with pytest.raises(ValueError, match="cannot hold"):
        c.launch(c.args())


@pytest.mark.parametrize("last", [False, True])
def test_append_to_a_slice(torch_cuda, last):  # noqa: F811
    """Tokens within the slice go to their slots; one behind it is reported and left out, its q is rotated all the same."""
    torch = torch_cuda
    from python.kinetic_rt import _lib
    H, K, tpb = 4, 2, 16
    table = np.array([[3, 0, 5], [1, 4, 2]], np.int32)
    x = torch.randn(4, (H + 2 * K) * 128, device="cuda").to(torch.bfloat16)
    pool = torch.full((6, tpb, 2, K, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    q_out = torch.zeros(4, H * 128, dtype=torch.bfloat16, device="cuda")
    ws = torch.zeros(_lib.rope_append_workspace_bytes(), dtype=torch.uint8, device="cuda")
    index, seq = [0, 33, 47, 31], [0, 0, 1, 1]  # columns 0, 2 (beyond the slice), 2 (beyond), 1
    f = 0.5 ** torch.arange(64, dtype=torch.float64, device="cuda")
    cut = sliced(torch, table, 2, last)
    _lib.rope_append(_lib.rope_append_args(x[:, :H * 128], x[:, H * 128:(H + K) * 128], x[:, (H + K) * 128:], f,
                                           i32(torch, [0] * 4), i32(torch, seq), cut, pool, q_out, H, K, 6, tpb, ws,
                                           cache_index=i32(torch, index)))
    assert _lib.read_status(ws)[1] == 8
    assert torch.equal(q_out, x[:, :H * 128])  # position 0: not turned
    want = torch.full_like(pool, 7.0)
    for t, (b, o) in ((0, (3, 0)), (3, (4, 15))):
        want[b, o] = x[t, H * 128:].view(2, K, 128)
    assert torch.equal(pool, want)


# ------------------------------------------------------------- single rows
def turned(t):
    """A tensor of one row whose row stride is 1, as a transposed column has it."""
    assert t.shape[0] == 1
    u = t.reshape(-1, 1).clone().T
    assert u.stride(0) == 1 and u.shape == t.shape
    return u


@pytest.mark.parametrize("q_lens", [None, [1]])
def test_attention_of_one_row_of_any_stride(torch_cuda, q_lens):  # noqa: F811
    torch = torch_cuda
    c = Case(torch, [300], q_lens=q_lens, seed=95)
    c.q_d, c.out, c.lse, c.table_d = (turned(t) for t in (c.q_d, c.out, c.lse, c.table_d))
    c.check(softcap=30.0)


def test_append_of_one_row_of_any_stride(torch_cuda):  # noqa: F811
    torch = torch_cuda
    from python.kinetic_rt import _lib
    H, K = 4, 2
    q, k, v = (turned(torch.randn(1, n * 128, device="cuda").to(torch.bfloat16)) for n in (H, K, K))
    pool = torch.zeros(2, 16, 2, K, 128, dtype=torch.bfloat16, device="cuda")
    q_out = turned(torch.zeros(1, H * 128, dtype=torch.bfloat16, device="cuda"))
    ws = torch.zeros(_lib.rope_append_workspace_bytes(), dtype=torch.uint8, device="cuda")
    f = 0.5 ** torch.arange(64, dtype=torch.float64, device="cuda")
    _lib.rope_append(_lib.rope_append_args(q, k, v, f, i32(torch, [0]), i32(torch, [0]), turned(i32(torch, [[1, 0]])), pool,
                                           q_out, H, K, 2, 16, ws, cache_index=i32(torch, [19])))
    assert _lib.read_status(ws) == (0, 0)
    assert torch.equal(q_out, q) and torch.equal(pool[0, 3, 0].reshape(1, -1), k) and torch.equal(pool[0, 3, 1].reshape(1, -1), v)
