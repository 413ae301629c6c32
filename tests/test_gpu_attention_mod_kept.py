"""One prompt call, made for the largest batch and captured once, on batches of
different shapes: the tensors are rewritten before each replay."""
import numpy as np
import pytest

from oracle import attention_mod as orc
from tests.test_gpu_attention_mod import Case, torch_cuda  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

ROWS, SEQS, CAP = 300, 6, 4096


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kw", [dict(), dict(softcap=20.0, window=700)])
def test_one_struct_for_every_batch(torch_cuda, kw, captured):  # noqa: F811
    torch = torch_cuda
    from python.kinetic_rt import _lib
    c = Case(torch, [CAP], n_heads=8, n_kv_heads=2, seed=110)  # a pool; its sequences are laid out anew for each batch
    rng = np.random.Generator(np.random.PCG64(111))
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.zeros(ROWS, 1024, dtype=torch.bfloat16, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(ROWS, 8, dtype=torch.float32, device="cuda")
    table, q_start, q_pos0 = z(SEQS, CAP // 16), z(SEQS + 1), z(SEQS)
    ws = torch.zeros(_lib.prefill_attention_mod_workspace_bytes(ROWS, SEQS, 8, 2, CAP), dtype=torch.uint8, device="cuda")
    a = _lib.prefill_attention_mod_args(q, c.pool_d, table, q_start, q_pos0, out, 8, 2, c.blocks, 16, CAP, ws, lse=lse,
                                        **kw)
    run = lambda: _lib.paged_attention_prefill_mod(a)  # noqa: E731
    if captured:
        run()  # (no rows yet)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        run = graph.replay
    for ctx, n in (([0], [300]), ([4000, 0, 17], [9, 1, 200]), ([0] * 6, [50] * 6), ([2000, 1000], [1, 0]), ([], []),
                   ([0, 4090], [5, 6])):
        starts = np.concatenate([[0], np.cumsum(n)]).astype(int)
        rows = starts[-1]
        blocks = rng.integers(0, c.blocks, (SEQS, CAP // 16)).astype(np.int32)
        table.copy_(torch.from_numpy(blocks))
        q_start.copy_(torch.tensor([*starts] + [rows] * (SEQS - len(n)), dtype=torch.int32))
        q_pos0.copy_(torch.tensor(ctx + [0] * (SEQS - len(n)), dtype=torch.int32))
        x = torch.randn(ROWS, 1024, device="cuda").to(torch.bfloat16)
        q.copy_(x)
        out.fill_(9.0)
        lse.fill_(7.0)
        run()
        assert _lib.read_status(ws) == (0, 0)
        told = [(s, ctx[s] + i, ctx[s] + n[s], 0, 0) if i % 7 in (0, 6) or i + 1 == n[s] else None for s in range(len(n))
                for i in range(n[s])]
        got, got_lse = out.float().cpu().numpy().reshape(ROWS, 8, 128), lse.cpu().numpy()
        if rows:
            ref, ref_lse, tol, tol_lse = orc.paged_attention_mod(x.float().cpu().numpy().reshape(ROWS, 8, 128)[:rows],
                                                                 c.pool, blocks, told, 8, 2, 16, kw.get("softcap", 0.0),
                                                                 kw.get("window", 0))
            keep = np.array([r is not None for r in told])
            assert (np.abs(got[:rows] - ref) <= tol)[keep].all()
            assert (np.abs(got_lse[:rows] - ref_lse)[keep] <= tol_lse[keep]).all()
        assert (got[rows:] == 9.0).all() and (got_lse[rows:] == 7.0).all()
