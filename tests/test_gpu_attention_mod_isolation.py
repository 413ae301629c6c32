"""What a row of the attentions with score modifications may depend on, bit for
bit: its own sequence's visible keys and queries, and nothing that lies beside
them (other rows of the tile, cache slots behind the last token, what earlier
kernels left in shared memory)."""
import numpy as np
import pytest

from tests.test_gpu_attention_mod import Case, i32, slopes_of, torch_cuda  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

MODS = [dict(softcap=20.0), dict(softcap=50.0), dict(softcap=30.0, slopes=slopes_of(10)), dict()]


def outputs(c, a, torch, rows=None):
    c.out.fill_(9.0)
    c.lse.fill_(7.0)
    c.launch(a)
    torch.cuda.synchronize()
    return c.out[:rows].clone(), c.lse[:rows].clone()


def same(a, b):
    return all((x == y).all() for x, y in zip(a, b))


@pytest.mark.parametrize("kw", MODS)
@pytest.mark.parametrize("fill", [1000.0, float("nan")])
def test_prefill_rows_that_do_not_exist(torch_cuda, kw, fill):  # noqa: F811
    """A group of 5 heads leaves 3 of a tile's 128 rows without queries.  Another call leaves large values or NaN where
    theirs would lie."""
    torch = torch_cuda
    c = Case(torch, [0, 300], q_lens=[180, 130], n_heads=10, n_kv_heads=2, seed=70)
    other = Case(torch, [0] * 80, q_lens=[256] * 80, n_heads=2, n_kv_heads=2, seed=71)
    quiet = Case(torch, [0] * 80, q_lens=[256] * 80, n_heads=2, n_kv_heads=2, seed=71, amp=0.0)
    other.q_d.fill_(fill)
    a, b, z = c.args(**kw), other.args(), quiet.args()
    got = []
    for before in (z, b, z):
        other.launch(before)
        got.append(outputs(c, a, torch))
    assert same(got[0], got[1]) and same(got[0], got[2])


@pytest.mark.parametrize("kw", MODS)
@pytest.mark.parametrize("fill", [1000.0, float("nan")])
def test_prefill_rows_of_the_next_sequence(torch_cuda, kw, fill):  # noqa: F811
    """The last tile of a sequence holds queries of the next one."""
    torch = torch_cuda
    c = Case(torch, [0, 40, 0], q_lens=[70, 33, 90], n_heads=10, n_kv_heads=5, seed=72)
    a = c.args(**kw)
    want = outputs(c, a, torch, 103)
    c.q_d[103:].fill_(fill)
    assert same(outputs(c, a, torch, 103), want)


@pytest.mark.parametrize("kw", MODS)
@pytest.mark.parametrize("ctx", [0, 700])
@pytest.mark.parametrize("fill", [1000.0, float("nan"), float("inf")])
def test_slots_behind_the_last_token(torch_cuda, kw, ctx, fill):  # noqa: F811
    """Prompts and single tokens: what a block's unwritten slots hold, and slots before the window."""
    torch = torch_cuda
    kw = dict(kw, window=200)
    for q_lens in ([69, 20], None):
        c = Case(torch, [ctx + 1, 5 + ctx], q_lens=q_lens, n_heads=10, n_kv_heads=2, seed=73)
        a = c.args(**kw)
        want = outputs(c, a, torch)
        seen = []
        for s in range(2):
            first = c.ctx[s] if q_lens else c.ctx[s] - 1  # position of the first query
            seen += [(c.table[s, j // 16], j % 16) for j in range(max(0, first - 199), c.total[s])]
        blocks, slots = (torch.tensor(np.array(v), device="cuda") for v in zip(*seen))
        kept = c.pool_d[blocks, slots].clone()
        c.pool_d.fill_(fill)
        c.pool_d[blocks, slots] = kept
        assert same(outputs(c, a, torch), want)


def test_prefill_one_row_live(torch_cuda):  # noqa: F811
    """Rows whose mask leaves nothing do not touch the live ones beside them."""
    torch = torch_cuda
    c = Case(torch, [0], q_lens=[64], n_heads=4, n_kv_heads=1, seed=74)
    start = [1 << 30] * 64
    start[13] = 0
    a = c.args(softcap=20.0, kv_start=start)
    want = outputs(c, a, torch)
    dead = [t for t in range(64) if t != 13]
    c.q_d[dead] = float("nan")
    assert same(outputs(c, a, torch), want)


@pytest.mark.parametrize("q_lens,ctx,window", [([61], [0], 0), ([100] * 30, [0] * 30, 0), ([203, 90], [1001, 30], 300)])
def test_unwritten_slots_cost_nothing(torch_cuda, q_lens, ctx, window):  # noqa: F811
    """A fresh cache may hold NaN behind the last token; the same call on zeros there takes as long (a scan for values to
    add back made it 50 times as long, the bound is 5)."""
    torch = torch_cuda
    c = Case(torch, ctx, q_lens=q_lens, n_heads=32, n_kv_heads=8, seed=75)
    a = c.args(window=window)
    unseen = torch.ones(c.blocks, c.tpb, dtype=torch.bool, device="cuda")
    for s in range(c.S):
        for j in range(c.total[s]):
            unseen[c.table[s, j // 16], j % 16] = False
    took = {}
    for fill in (0.0, float("nan")):
        c.pool_d[unseen] = fill
        c.launch(a)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        times = []
        for _ in range(5):
            start.record()
            for _ in range(10):
                c.launch(a)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        took[fill == 0.0] = min(times)
    assert torch.isfinite(c.out).all()
    assert took[False] < 5 * took[True], took
