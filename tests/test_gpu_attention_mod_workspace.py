"""One workspace for calls of the attentions with score modifications that
follow one another: of both kinds, of any sizes, heads and windows, and with
different parts of the buffer given to them."""
import numpy as np
import pytest

from oracle import attention_mod as orc
from tests.test_gpu_attention_mod import Case, i32, slopes_of, torch_cuda  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def checked(c, a, ws, size, only=None, **mods):
    from python.kinetic_rt import _lib
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    rows = c.rows()
    if only is not None:
        rows = [r if t in only else None for t, r in enumerate(rows)]
    ref, lse, tol, tol_lse = orc.paged_attention_mod(c.q, c.pool, c.table, rows, c.H, c.K, c.tpb,
                                                     mods.get("softcap", 0.0), mods.get("window", 0))
    c.out.fill_(9.0)
    c.lse.fill_(7.0)
    c.launch(a)
    assert _lib.read_status(ws) == (0, 0)
    got, got_lse = c.result()
    keep = [t for t, r in enumerate(rows) if r is not None]
    assert (np.abs(got - ref) <= tol)[keep].all()
    dead = np.isneginf(lse)
    assert (np.isneginf(got_lse) == dead)[keep].all()
    assert (np.abs(np.where(dead, 0, got_lse) - np.where(dead, 0, lse)) <= tol_lse)[keep].all()


def test_prompts_and_single_tokens(torch_cuda):  # noqa: F811
    """A split prompt whose parts fill the buffer to its end, then single tokens whose splits merge through it."""
    torch = torch_cuda
    prompt = Case(torch, [9000], q_lens=[65], seed=80)
    one = Case(torch, [20011, 33, 0, 5000], n_heads=16, n_kv_heads=2, seed=81)
    few = Case(torch, [3000, 700], seed=82)
    args = [c.args() for c in (prompt, one, few)]
    size = max(a.workspace_bytes for a in args)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    for c, a in zip((prompt, one, few, prompt, few, one, one), [args[i] for i in (0, 1, 2, 0, 2, 1, 1)]):
        checked(c, a, ws, size)


def test_windows_heads_and_sizes(torch_cuda):  # noqa: F811
    """Few long sequences, many short ones, other heads, a window: in turn."""
    torch = torch_cuda
    kinds = [(Case(torch, [30000], n_heads=8, n_kv_heads=1, seed=83), {}),
             (Case(torch, [40] * 8 + [8300, 5000], n_heads=8, n_kv_heads=8, seed=84), dict(softcap=30.0)),
             (Case(torch, [20000, 19000, 20011], n_heads=32, n_kv_heads=2, seed=85), {}),
             (Case(torch, [30000], n_heads=8, n_kv_heads=1, seed=83), dict(window=4000))]
    args = [c.args(**kw) for c, kw in kinds]
    size = max(a.workspace_bytes for a in args)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    for i in (0, 1, 2, 1, 3, 2, 0, 1, 3, 0):
        checked(kinds[i][0], args[i], ws, size, **kinds[i][1])


def test_part_of_the_buffer(torch_cuda):  # noqa: F811
    """A large call is given the whole buffer, a smaller one as much as it needs."""
    torch = torch_cuda
    large = Case(torch, [20000, 19000, 20011], n_heads=32, n_kv_heads=2, seed=85)
    small = Case(torch, [20011], n_heads=16, n_kv_heads=2, seed=86)
    args = [large.args(), small.args()]
    need = [a.workspace_bytes for a in args]
    ws = torch.zeros(max(need) + 5000, dtype=torch.uint8, device="cuda")
    for i, size in ((0, ws.numel()), (1, need[1]), (1, ws.numel()), (0, need[0]), (1, need[1] + 4)):
        checked((large, small)[i], args[i], ws, size)


def test_more_pairs_than_counters(torch_cuda):  # noqa: F811
    """2100 sequences of 8 KV heads under a bound that splits them; a buffer that other calls have written to."""
    torch = torch_cuda
    from python.kinetic_rt import _lib
    S, H, K, tpb, blocks, bound = 2100, 8, 8, 64, 200, 8256
    rng = np.random.Generator(np.random.PCG64(87))
    lens = rng.integers(0, 40, S)
    lens[[0, 700, 2099]] = 8256, 8200, 8193  # two pieces
    c = Case(torch, [12800], n_heads=H, n_kv_heads=K, tpb=tpb, seed=88, spare=0)  # its pool is shared by all
    assert c.blocks == blocks
    table = rng.integers(0, blocks, (S, bound // tpb)).astype(np.int32)
    q = torch.randn(S, H * 128, device="cuda").to(torch.bfloat16)
    out = torch.zeros(S, H * 128, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(S, H, dtype=torch.float32, device="cuda")
    ws = torch.full((_lib.attention_mod_workspace_bytes(S, H, K, bound),), 77, dtype=torch.uint8, device="cuda")
    ws[:8192 + 65536] = 0
    a = _lib.attention_mod_args(q, c.pool_d, torch.from_numpy(table).cuda(), i32(torch, lens), out, H, K, blocks, tpb, bound,
                                ws, lse=lse)
    rows = [(s, int(n) - 1, int(n), 0, 0) if s in (0, 1, 2, 700, 1500, 2098, 2099) else None for s, n in enumerate(lens)]
    ref, ref_lse, tol, tol_lse = orc.paged_attention_mod(q.float().cpu().numpy().reshape(S, H, 128), c.pool, table, rows, H,
                                                         K, tpb)
    keep = [t for t, r in enumerate(rows) if r is not None and lens[t] > 0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _lib.paged_attention_decode_mod(a)
    for call in (lambda: _lib.paged_attention_decode_mod(a), graph.replay, graph.replay):
        out.fill_(9.0)
        call()
        assert _lib.read_status(ws) == (0, 0)
        got = out.float().cpu().numpy().reshape(S, H, 128)
        assert (np.abs(got - ref) <= tol)[keep].all()
        assert (np.abs(lse.cpu().numpy() - ref_lse)[keep] <= tol_lse[keep]).all()
        assert (got[lens == 0] == 0).all()
