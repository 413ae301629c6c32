"""GPU tests of paged attention with score modifications (decode and prompts)
against oracle/attention_mod.py in 64 bits.

Tolerances are per element and come from the arithmetic: every weight is
rounded to bf16 once (2^-8 relative) for the product with V, the output once
(2^-8), scores and sums carry fp32 errors; the oracle adds these up
(paged_attention_mod's tol_out and tol_lse).
"""
import numpy as np
import pytest

from oracle import attention_mod as orc
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def to_dev(torch, bits):
    return torch.from_numpy(np.ascontiguousarray(bits).view(np.int16)).view(torch.bfloat16).cuda()


def i32(torch, v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


class Case:
    """Random cache, queries and tables.  q_lens None: decode (one row a
    sequence, ctx tokens cached, its own among them)."""

    def __init__(self, torch, ctx, q_lens=None, n_heads=8, n_kv_heads=2, tpb=16, seed=0, q_pad=0, rows_pad=0, amp=3.0,
                 spare=3, edit_pool=None):
        rng = np.random.Generator(np.random.PCG64(seed))
        self.torch, self.ctx, self.q_lens = torch, list(ctx), q_lens
        self.H, self.K, self.tpb = n_heads, n_kv_heads, tpb
        self.S = len(ctx)
        self.total = [c + (q_lens[s] if q_lens else 0) for s, c in enumerate(ctx)]
        self.max_len = max(max(self.total), 1)
        bps = -(-self.max_len // tpb)
        self.blocks = self.S * bps + spare
        self.table = rng.permutation(self.blocks).astype(np.int32)[:self.S * bps].reshape(self.S, bps)
        pool = rng.standard_normal((self.blocks, tpb, 2, n_kv_heads, 128), dtype=np.float32)
        if edit_pool:
            edit_pool(pool, self)
        bits = f32_to_bf16_bits(pool)
        self.pool = bf16_bits_to_f32(bits)
        self.T = sum(q_lens) if q_lens else self.S
        qb = f32_to_bf16_bits(amp * rng.standard_normal((self.T, n_heads, 128), dtype=np.float32))
        self.q = bf16_bits_to_f32(qb)
        W = n_heads * 128
        self.pool_d = to_dev(torch, bits)
        self.q_d = torch.zeros(self.T + rows_pad, W + q_pad, dtype=torch.bfloat16, device="cuda")
        self.q_d[:self.T, :W] = to_dev(torch, qb.reshape(self.T, W))
        self.out = torch.full((self.T + rows_pad, W + q_pad), 9.0, dtype=torch.bfloat16, device="cuda")
        self.lse = torch.full((self.T + rows_pad, n_heads + 1), 7.0, dtype=torch.float32, device="cuda")
        self.table_d = torch.from_numpy(self.table).cuda()

    def slot(self, s, j):
        return self.table[s, j // self.tpb], j % self.tpb

    def args(self, kv_start=None, prefix=None, slopes=None, softcap=0.0, window=0, scale=0.0, max_len=None):
        from python.kinetic_rt import _lib
        torch = self.torch
        z = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")  # noqa: E731
        kw = dict(softcap=softcap, window=window, scale=scale, lse=self.lse,
                  alibi_slopes=None if slopes is None else torch.tensor(np.asarray(slopes), dtype=torch.float32,
                                                                       device="cuda"),
                  kv_start=None if kv_start is None else i32(torch, kv_start))
        max_len = max_len or self.max_len
        if self.q_lens is None:
            self.ws = z(_lib.attention_mod_workspace_bytes(self.S, self.H, self.K, max_len, window))
            return _lib.attention_mod_args(self.q_d, self.pool_d, self.table_d, i32(torch, self.ctx), self.out, self.H,
                                           self.K, self.blocks, self.tpb, max_len, self.ws, **kw)
        starts = np.concatenate([[0], np.cumsum(self.q_lens)])
        self.ws = z(_lib.prefill_attention_mod_workspace_bytes(self.q_d.shape[0], self.S, self.H, self.K, max_len))
        if kv_start is not None and len(kv_start) < self.q_d.shape[0]:
            kw["kv_start"] = i32(torch, list(kv_start) + [0] * (self.q_d.shape[0] - len(kv_start)))
        return _lib.prefill_attention_mod_args(self.q_d, self.pool_d, self.table_d, i32(torch, starts),
                                               i32(torch, self.ctx), self.out, self.H, self.K, self.blocks, self.tpb,
                                               max_len, self.ws,
                                               prefix_lens=None if prefix is None else i32(torch, prefix), **kw)

    def launch(self, a):
        from python.kinetic_rt import _lib
        (_lib.paged_attention_decode_mod if self.q_lens is None else _lib.paged_attention_prefill_mod)(a)

    def rows(self, kv_start=None, prefix=None):
        if self.q_lens is None:
            return [(s, c - 1, max(c, 0), 0 if kv_start is None else kv_start[s], 0) for s, c in enumerate(self.ctx)]
        rows = []
        for s, n in enumerate(self.q_lens):
            for i in range(n):
                rows.append((s, self.ctx[s] + i, self.total[s], 0 if kv_start is None else kv_start[len(rows)],
                             0 if prefix is None else prefix[s]))
        return rows

    def result(self):
        W = self.H * 128
        return (self.out[:self.T, :W].float().cpu().numpy().reshape(self.T, self.H, 128).astype(np.float64),
                self.lse[:self.T, :self.H].cpu().numpy().astype(np.float64))

    def check(self, kv_start=None, prefix=None, slopes=None, softcap=0.0, window=0, scale=0.0, only=None, calls=2):
        from python.kinetic_rt import _lib
        a = self.args(kv_start, prefix, slopes, softcap, window, scale)
        rows = self.rows(kv_start, prefix)
        if only is not None:
            rows = [r if t in only else None for t, r in enumerate(rows)]
        ref, lse, tol, tol_lse = orc.paged_attention_mod(self.q, self.pool, self.table, rows, self.H, self.K, self.tpb,
                                                         softcap, window,
                                                         None if slopes is None else np.float32(slopes),
                                                         scale or None)
        keep = [t for t, r in enumerate(rows) if r is not None]
        for _ in range(calls):  # a second call finds the workspace as the first one left it
            self.out.fill_(9.0)
            self.lse.fill_(7.0)
            self.launch(a)
            rc, bits = _lib.read_status(self.ws)
            assert rc == 0 and bits == 0, f"status {bits:#x}"
            got, got_lse = self.result()
            bad = ~(np.abs(got - ref) <= tol)[keep]
            assert not bad.any(), (f"{bad.sum()} of {bad.size} out of bounds, rows {np.unique(np.nonzero(bad)[0])[:8]}, "
                                   f"worst {np.abs(got - ref)[keep].max()}")
            dead = np.isneginf(lse)
            assert (np.isneginf(got_lse) == dead)[keep].all()
            off = np.abs(np.where(dead, 0, got_lse) - np.where(dead, 0, lse))
            assert (off <= tol_lse)[keep].all(), off[keep].max()
            # what lies beside the results stays as it was
            W = self.H * 128
            assert (self.out[:, W:] == 9.0).all() and (self.out[self.T:] == 9.0).all()
            assert (self.lse[:, self.H:] == 7.0).all() and (self.lse[self.T:] == 7.0).all()
        return got, got_lse


def slopes_of(H):
    return [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]


# ----------------------------------------------------------------- decode
@pytest.mark.parametrize("softcap,bias,window", [(0.0, False, 0), (20.0, False, 0), (0.0, True, 0), (50.0, True, 100),
                                                 (0.0, False, 1), (0.0, False, 17)])
@pytest.mark.parametrize("H,K", [(8, 2), (3, 1), (16, 1), (5, 5)])
def test_decode_lengths(torch_cuda, H, K, softcap, bias, window):
    """Lengths around the 16-token chunks, one empty sequence, an odd group."""
    c = Case(torch_cuda, [1, 15, 16, 17, 100, 257, 0, 1030], n_heads=H, n_kv_heads=K, seed=H + K, q_pad=64)
    c.check(softcap=softcap, slopes=slopes_of(H) if bias else None, window=window)


def test_decode_kv_start(torch_cuda):
    """First visible positions inside, at the end of and behind the sequence; negative counts as 0."""
    c = Case(torch_cuda, [100, 100, 100, 100, 64, 1], seed=2, tpb=32)
    c.check(kv_start=[0, 50, 99, 100, -5, 7], softcap=30.0)


def test_decode_long_split(torch_cuda):
    """One long sequence beside short ones: many splits, one split, none."""
    c = Case(torch_cuda, [20011, 33, 0, 5000], n_heads=16, n_kv_heads=2, seed=5)
    c.check(slopes=slopes_of(16))
    c.check(window=4097, softcap=50.0)


def test_decode_scale(torch_cuda):
    Case(torch_cuda, [77, 300], seed=6).check(scale=0.25, softcap=5.0)


def poison(pool, c, where):
    """NaN and infinities in K and V at (sequence, position)."""
    for i, (s, j) in enumerate(where):
        b, o = c.slot(s, j)
        pool[b, o, 0] = np.nan
        pool[b, o, 1] = [np.nan, np.inf, -np.inf][i % 3]


def test_decode_ignores_what_is_not_visible(torch_cuda):
    """Cache slots behind the last token and before the window hold NaN and infinities."""
    ctx = [37, 200, 129]

    def edit(pool, c):
        poison(pool, c, [(0, 37), (0, 47), (1, 0), (1, 130), (1, 200), (1, 207), (2, 60), (2, 129)])

    c = Case(torch_cuda, ctx, seed=7, edit_pool=edit, spare=3)
    got, lse = c.check(window=66, softcap=30.0)
    assert np.isfinite(got).all() and np.isfinite(lse).all()


def test_decode_visible_nan_shows(torch_cuda):
    """A NaN that is visible makes its heads' results NaN, and no other's."""

    def edit(pool, c):
        b, o = c.slot(1, 20)
        pool[b, o, 1, 0, 5] = np.nan  # V of KV head 0, dim 5

    c = Case(torch_cuda, [40, 40], seed=8, edit_pool=edit)
    c.launch(c.args())
    got, lse = c.result()
    want = np.zeros((2, 8, 128), bool)
    want[1, :4, 5] = True
    assert (np.isnan(got) == want).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("prompt", [False, True])
def test_bad_block_is_masked_and_reported(torch_cuda, prompt):
    torch = torch_cuda
    from python.kinetic_rt import _lib
    c = Case(torch, [20, 40] if not prompt else [0, 0], q_lens=[20, 40] if prompt else None, seed=9)
    c.table_d[1, 1] = c.blocks + 70  # positions 16 .. 31 of sequence 1
    c.launch(c.args())
    rc, bits = _lib.read_status(c.ws)
    assert bits & 8
    got, _ = c.result()
    rows = c.rows()
    for t, (s, pos, length, _, _) in enumerate(rows):
        k, v = orc.gather_kv(c.pool, c.table[s], pos + 1, 16)
        keep = np.array([j for j in range(pos + 1) if not (s == 1 and 16 <= j < 32)])
        for h in range(c.H):
            o, _, a, fuzz = orc.attention_row(c.q[t, h].astype(float), k[keep, h // 4].astype(float),
                                              v[keep, h // 4].astype(float), pos, 0, len(keep), 128 ** -0.5)
            assert (np.abs(got[t, h] - o) <= (2.0 ** -8 + 2 * fuzz + 1e-5) * a + 2.0 ** -8 * np.abs(o) + 1e-30).all()
    c.launch(c.args())  # counters are consistent: the next call reports the same again
    assert _lib.read_status(c.ws)[1] & 8


def test_decode_length_beyond_max_is_cut(torch_cuda):
    torch = torch_cuda
    from python.kinetic_rt import _lib
    c = Case(torch, [100, 300, 7], seed=10)
    c.launch(c.args(max_len=250))
    assert _lib.read_status(c.ws)[1] & 8
    got, _ = c.result()
    ref, _, tol, _ = orc.paged_attention_mod(c.q, c.pool, c.table, [(0, 99, 100, 0, 0), (1, 249, 250, 0, 0),
                                                                    (2, 6, 7, 0, 0)], c.H, c.K, 16)
    assert (np.abs(got - ref) <= tol).all()


# ---------------------------------------------------------------- prompts
@pytest.mark.parametrize("softcap,bias,window", [(0.0, False, 0), (20.0, False, 0), (0.0, True, 0), (50.0, True, 70),
                                                 (0.0, False, 1)])
@pytest.mark.parametrize("H,K", [(8, 2), (3, 1), (5, 1), (16, 1), (2, 2)])
def test_prefill_ragged(torch_cuda, H, K, softcap, bias, window):
    """Lengths around tiles and blocks, an empty sequence, cached prefixes, padded rows and strides."""
    c = Case(torch_cuda, [0, 0, 5, 128, 300, 0], q_lens=[1, 70, 33, 0, 129, 16], n_heads=H, n_kv_heads=K, seed=H * K,
             q_pad=8, rows_pad=37)
    c.check(softcap=softcap, slopes=slopes_of(H) if bias else None, window=window)


@pytest.mark.parametrize("tpb", [16, 48])
def test_prefill_prefix(torch_cuda, tpb):
    """Prefixes that end inside the cached part, inside the prompt, behind it, and none; with a window too."""
    c = Case(torch_cuda, [200, 10, 0, 0], q_lens=[40, 150, 90, 60], seed=12, tpb=tpb)
    prefix = [100, 77, 1000, 0]
    c.check(prefix=prefix)
    c.check(prefix=prefix, window=50, slopes=slopes_of(8), softcap=30.0)


def test_prefill_documents(torch_cuda):
    """Documents packed into one sequence, and rows that see nothing."""
    L = 400
    bounds = [0, 7, 130, 131, 256, 300]
    start = [max(b for b in bounds if b <= t) for t in range(L)]
    for t in range(0, L, 13):
        start[t] = 1 << 30
    c = Case(torch_cuda, [0, 3], q_lens=[L, 50], n_heads=4, n_kv_heads=2, seed=13)
    c.check(kv_start=start + [0] * 49 + [2 ** 31 - 1], slopes=slopes_of(4))


def test_prefill_nothing_visible(torch_cuda):
    c = Case(torch_cuda, [0, 0], q_lens=[5, 200], seed=14)
    c.check(kv_start=[1 << 30] * 205)


def test_prefill_long(torch_cuda):
    """A long prompt, some rows checked: many key blocks, the lazy rescaling."""
    n = 3001
    c = Case(torch_cuda, [1040], q_lens=[n], n_heads=4, n_kv_heads=1, seed=15, amp=8.0)
    c.check(only=set(range(0, n, 97)) | {n - 1})
    c.check(only=set(range(0, n, 97)) | {n - 1}, window=1500, softcap=30.0)


def test_prefill_growing_scores(torch_cuda):
    """Row maxima that rise from block to block by far more than 2^8, and rows that stay below."""

    def edit(pool, c):
        for j in range(c.total[0]):
            b, o = c.slot(0, j)
            pool[b, o, 0] = (j // 100) * 2.0 - 3.0
            pool[b, o, 0, :, 1::2] *= 0.5

    c = Case(torch_cuda, [0], q_lens=[700], n_heads=2, n_kv_heads=1, seed=16, edit_pool=edit)
    c.check()


def test_prefill_ignores_what_is_not_visible(torch_cuda):
    """NaN and infinities behind the sequence, at later positions, before the
    window and in other documents reach no row that does not see them."""
    n = 300

    def edit(pool, c):
        # (1, 40 ..): behind the sequence's last token; (0, 250): seen by rows 250 .. 289
        poison(pool, c, [(1, j) for j in range(40, 64)])
        b, o = c.slot(0, 250)
        pool[b, o, 1, 0, 3] = np.nan
        pool[b, o, 1, 0, 4] = np.inf
        pool[b, o, 1, 1, 5] = -np.inf

    c = Case(torch_cuda, [0, 0], q_lens=[n, 40], seed=17, edit_pool=edit)
    c.launch(c.args(window=40))
    got, lse = c.result()
    want = np.zeros(got.shape, bool)
    want[250:290, :4, 3:5] = True
    want[250:290, 4:, 5] = True
    assert (~np.isfinite(got) == want).all()
    assert np.isnan(got[250:290, :4, 3]).all() and np.isposinf(got[250:290, :4, 4]).all()
    assert np.isneginf(got[250:290, 4:, 5]).all() and np.isfinite(lse).all()
    clean = np.where(np.isfinite(c.pool), c.pool, 0)
    ref, _, tol, _ = orc.paged_attention_mod(c.q, clean, c.table, c.rows(), c.H, c.K, 16, 0.0, 40)
    assert (np.abs(np.where(want, 0, got) - np.where(want, 0, ref)) <= tol).all()


@pytest.mark.parametrize("q_start", [[0, 30, 20, 60], [0, 40, 50, 90], [-4, 10, 20, 60]])
def test_prefill_bad_q_start_is_reported(torch_cuda, q_start):
    """Starts that decrease or leave the rows set status bit 8; good sequences are computed."""
    torch = torch_cuda
    from python.kinetic_rt import _lib
    c = Case(torch, [0, 0, 0], q_lens=[20, 20, 20], seed=18)
    a = c.args()
    bad = i32(torch, q_start)
    a.q_start = bad.data_ptr()
    c.launch(a)
    assert _lib.read_status(c.ws)[1] & 8
    assert torch.isfinite(c.out.float()).all()


# ------------------------------------------------ streams, graphs, together
@pytest.mark.parametrize("prompt", [False, True])
def test_side_stream_and_graph(torch_cuda, prompt):
    """The same call eagerly, on a side stream, and captured and replayed on changed inputs."""
    torch = torch_cuda
    c = Case(torch, [4000, 17], q_lens=[90, 33] if prompt else None, seed=19)
    a = c.args(softcap=30.0, window=3000)
    c.launch(a)
    want = c.out.clone(), c.lse.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.out.zero_()
        c.launch(a)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c.out, want[0]) and torch.equal(c.lse, want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.launch(a)
    q0 = c.q_d.clone()
    c.q_d.mul_(-0.5)
    g.replay()
    half = c.out.clone()
    c.launch(a)
    assert torch.equal(c.out, half)
    c.q_d.copy_(q0)
    c.out.zero_()
    for _ in range(3):
        g.replay()
    assert torch.equal(c.out, want[0]) and torch.equal(c.lse, want[1])


def test_decode_is_the_prompts_last_row(torch_cuda):
    """Prompt rows and single tokens agree: every row of a prompt against decode at its length."""
    torch = torch_cuda
    L = 150
    p = Case(torch, [0], q_lens=[L], seed=20)
    kw = dict(softcap=25.0, window=60, slopes=slopes_of(8))
    p.launch(p.args(**kw))
    got, lse = p.result()
    d = Case(torch, list(range(1, L + 1)), seed=20)
    d.pool_d, d.blocks = p.pool_d, p.blocks
    d.table_d = p.table_d.repeat(L, 1)
    d.q_d.copy_(p.q_d)
    d.launch(d.args(**kw))
    one, lse1 = d.result()
    _, _, tol, tol_lse = orc.paged_attention_mod(p.q, p.pool, p.table, p.rows(), 8, 2, 16, 25.0, 60,
                                                 np.float32(slopes_of(8)))
    assert (np.abs(got - one) <= 2 * tol).all() and (np.abs(lse - lse1) <= 2 * tol_lse).all()


@pytest.mark.parametrize("seqs,ctx,H,K", [(1, 700, 4, 1), (2, 1024, 8, 2), (5, 3000, 4, 2), (160, 40, 1, 1),
                                          (310, 33, 2, 1)])
def test_decode_sizes_share_a_workspace(torch_cuda, seqs, ctx, H, K):
    """One workspace, made for a larger batch of other heads' shape, serves calls with many and with no splits."""
    from python.kinetic_rt import _lib
    ws = torch_cuda.zeros(_lib.attention_mod_workspace_bytes(512, 8, 2, 4096), dtype=torch_cuda.uint8, device="cuda")
    rng = np.random.Generator(np.random.PCG64(77))
    lens = rng.integers(0, ctx + 1, seqs)
    lens[0] = ctx
    for n, L, h, k in ((seqs, lens, H, K), (3, [2000, 1, 900], 8, 2), (seqs, lens, H, K)):
        case = Case(torch_cuda, list(map(int, L)), n_heads=h, n_kv_heads=k)
        a = case.args()
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        case.launch(a)
        rc, bits = _lib.read_status(ws)
        assert rc == 0 and bits == 0
        got, got_lse = case.result()
        ref, lse, tol, tol_lse = orc.paged_attention_mod(case.q, case.pool, case.table, case.rows(), h, k, case.tpb)
        assert (np.abs(got - ref) <= tol).all()
        seen = ~np.isneginf(lse)
        assert (np.isneginf(got_lse) == ~seen).all()
        assert (np.abs(got_lse[seen] - lse[seen]) <= np.broadcast_to(tol_lse, lse.shape)[seen]).all()


# Few rows behind a long cache: the keys of an item are split over CTAs and joined.
@pytest.mark.parametrize("softcap,bias,window", [(0.0, False, 0), (30.0, False, 0), (0.0, True, 0), (50.0, True, 1500)])
@pytest.mark.parametrize("H,K", [(8, 2), (5, 1), (16, 1)])
def test_prefill_few_rows_long_cache(torch_cuda, H, K, softcap, bias, window):
    """Sequences of many pieces, of two, of one, and of none."""
    c = Case(torch_cuda, [9000, 1, 1100, 0, 513], q_lens=[7, 30, 1, 0, 70], n_heads=H, n_kv_heads=K, seed=31 + H,
             q_pad=8, rows_pad=5)
    c.check(softcap=softcap, slopes=slopes_of(H) if bias else None, window=window)


def test_prefill_few_rows_prefix_and_starts(torch_cuda):
    """Rows whose keys lie in some of the pieces only, rows that see nothing, and a prefix beyond the rows' positions."""
    c = Case(torch_cuda, [5000, 2500], q_lens=[40, 3], seed=32)
    start = [0, 4990, 1 << 30, 3000, 5001] * 8 + [0, 2400, 2 ** 31 - 1]
    c.check(kv_start=start, prefix=[0, 2503])
    c.check(kv_start=start, softcap=20.0)
    c.check(kv_start=[1 << 30] * 43)


def test_prefill_few_rows_not_finite(torch_cuda):
    """V values that are not finite, in blocks that only some rows see, reach the rows that see them across pieces."""

    def edit(pool, c):
        for j, d, v in ((700, 3, np.nan), (2900, 4, np.inf), (4003, 5, -np.inf), (4010, 6, np.nan)):
            b, o = c.slot(0, j)
            pool[b, o, 1, 0, d] = v

    c = Case(torch_cuda, [4000], q_lens=[12], seed=33, edit_pool=edit)
    start = [0, 701, 2901, 4004] * 3
    c.launch(c.args(kv_start=start))
    got, lse = c.result()
    want = np.zeros(got.shape, bool)
    for r in range(12):
        for j, d in ((700, 3), (2900, 4), (4003, 5), (4010, 6)):
            want[r, :4, d] = start[r] <= j <= 4000 + r
    assert (~np.isfinite(got) == want).all()
    assert (np.isfinite(lse).all(axis=1) == [start[r] <= 4000 + r for r in range(12)]).all()  # row 3 sees nothing
    clean = np.where(np.isfinite(c.pool), c.pool, 0)
    ref, _, tol, _ = orc.paged_attention_mod(c.q, clean, c.table, c.rows(start), c.H, c.K, 16)
    assert (np.abs(np.where(want, 0, got) - np.where(want, 0, ref)) <= tol).all()


def test_prefill_sizes_share_a_workspace(torch_cuda):
    """One workspace, made for the largest call, serves split and whole items in turn."""
    from python.kinetic_rt import _lib
    ws = torch_cuda.zeros(_lib.prefill_attention_mod_workspace_bytes(4096, 16, 8, 2, 8192), dtype=torch_cuda.uint8,
                          device="cuda")
    for ctx, q_lens in (([4000, 0], [9, 2]), ([0] * 9, [600] * 9), ([8000], [3]), ([4000, 0], [9, 2])):
        case = Case(torch_cuda, ctx, q_lens=q_lens, seed=34)
        a = case.args()
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        case.launch(a)
        rc, bits = _lib.read_status(ws)
        assert rc == 0 and bits == 0
        rows = [r if t % 61 == 0 else None for t, r in enumerate(case.rows())]
        ref, lse, tol, tol_lse = orc.paged_attention_mod(case.q, case.pool, case.table, rows, 8, 2, 16)
        got, got_lse = case.result()
        assert (np.abs(got - ref) <= tol)[::61].all()
        assert (np.abs(got_lse - lse) <= tol_lse)[::61].all()


def test_prefill_many_sequences(torch_cuda):
    """More sequences than the search for the work takes in one pass, empty ones among them."""
    rng = np.random.Generator(np.random.PCG64(40))
    q_lens = [int(n) for n in rng.choice([0, 1, 1, 2, 40], 300)]
    c = Case(torch_cuda, [int(n) for n in rng.integers(0, 60, 300)], q_lens=q_lens, n_heads=4, n_kv_heads=2, seed=41,
             rows_pad=3)
    c.check(softcap=30.0)


def test_calls_at_once(torch_cuda):
    """Prompt, split prompt and decode calls on three streams at the same time, each with its own workspace."""
    torch = torch_cuda
    cases = [Case(torch, [0, 0], q_lens=[900, 700], seed=42), Case(torch, [6000], q_lens=[9], seed=43),
             Case(torch, [3000, 20, 900], seed=44)]
    args = [c.args(softcap=30.0) for c in cases]
    alone = []
    for c, a in zip(cases, args):
        c.launch(a)
        torch.cuda.synchronize()
        alone.append((c.out.clone(), c.lse.clone()))
        c.out.fill_(9.0)
        c.lse.fill_(7.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for c, a, s in zip(cases, args, streams):
            with torch.cuda.stream(s):
                c.launch(a)
    torch.cuda.synchronize()
    for c, (out, lse) in zip(cases, alone):
        assert torch.equal(c.out, out) and torch.equal(c.lse, lse)


@pytest.mark.parametrize("prompt", [False, True])
def test_blocks_far_into_a_large_pool(torch_cuda, prompt):
    """Blocks more than 2^32 bytes into the pool give what the same blocks give at its start."""
    torch = torch_cuda
    near = Case(torch, [700, 90], q_lens=[70, 5] if prompt else None, n_heads=8, n_kv_heads=8, seed=45)
    a = near.args(softcap=30.0)
    near.launch(a)
    torch.cuda.synchronize()
    want = near.out.clone(), near.lse.clone()
    far = (9 << 29) // (near.tpb * 2 * 8 * 256)  # 4.5 GiB of blocks before them
    pool = torch.empty((far + near.blocks,) + tuple(near.pool_d.shape[1:]), dtype=torch.bfloat16, device="cuda")
    pool[far:].copy_(near.pool_d)
    near.pool_d, near.blocks = pool, far + near.blocks
    near.table_d += far
    near.out.fill_(9.0)
    near.lse.fill_(7.0)
    near.launch(near.args(softcap=30.0))
    torch.cuda.synchronize()
    assert torch.equal(near.out, want[0]) and torch.equal(near.lse, want[1])


def test_prefill_long_causal_items_are_split(torch_cuda):
    """A long prompt of one KV head: its last items are in pieces, its first whole; ascending and (bias) descending."""
    n = 4100
    c = Case(torch_cuda, [0], q_lens=[n], n_heads=8, n_kv_heads=1, seed=46)
    only = set(range(5, n, 211)) | {0, n - 1}
    c.check(only=only)
    c.check(only=only, slopes=slopes_of(8))
    c.check(only=only, slopes=slopes_of(8), softcap=30.0, prefix=[2000])


@pytest.mark.parametrize("seqs,ctx,H,K", [(60, 40, 8, 8), (320, 17, 5, 1), (45, 900, 16, 8), (170, 300, 2, 2)])
def test_decode_many_short_sequences(torch_cuda, seqs, ctx, H, K):
    """More CTAs than two per SM, with few chunks each; empty sequences and single tokens among them."""
    rng = np.random.Generator(np.random.PCG64(seqs))
    lens = [int(n) for n in rng.integers(0, ctx + 1, seqs)]
    lens[:3] = [ctx, 1, 0]
    c = Case(torch_cuda, lens, n_heads=H, n_kv_heads=K, seed=47)
    c.check(softcap=20.0, slopes=slopes_of(H), only=set(range(0, seqs, 7)) | {1, 2})


def test_prefill_short_keys_under_a_large_bound(torch_cuda):
    """max_kv_len far above the lengths: the split follows the real ones."""
    c = Case(torch_cuda, [1500, 40], q_lens=[6, 20], seed=48)
    rows = c.rows()
    ref, lse, tol, tol_lse = orc.paged_attention_mod(c.q, c.pool, c.table, rows, 8, 2, 16)
    c.table_d = torch_cuda.cat([c.table_d, torch_cuda.zeros(2, 8192, dtype=torch_cuda.int32, device="cuda")], dim=1)
    c.launch(c.args(max_len=131072))
    got, got_lse = c.result()
    assert (np.abs(got - ref) <= tol).all() and (np.abs(got_lse - lse) <= tol_lse).all()
