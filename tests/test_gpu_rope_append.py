"""GPU tests of krt_rope_append against oracle/attention_mod.rope in 64 bits.

Tolerance per element: one bf16 rounding of the result (2^-8 relative) plus
the fp32 errors of a rotation, 2^-21 of the pair's magnitude (cos and sin off
by about 2^-22: the fraction of a turn is rounded to fp32, 2 pi 2^-25, and the
sine itself; two products and a sum, 2^-24 each).
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


def run(torch, T, H, K, R, interleaved, fp32=False, tpb=16, factor=1.0, far=0, seed=0, pad=0, skip=(), lost=()):
    """skip: padding tokens; lost: tokens whose block lies outside the pool."""
    from python.kinetic_rt import _lib
    rng = np.random.Generator(np.random.PCG64(seed))
    seqs = 3
    index = np.array([t // seqs + 5 for t in range(T)], np.int32)
    token_seq = np.array([t % seqs for t in range(T)], np.int32)
    positions = index + far
    bps = -(-(int(index.max()) + 1) // tpb)
    blocks = seqs * bps + 2
    table = rng.permutation(blocks).astype(np.int32)[:seqs * bps].reshape(seqs, bps)
    for t in skip:
        token_seq[t] = -1
    for t in lost:
        token_seq[t] = seqs + 4
    W = (H + 2 * K) * 128
    x = rng.standard_normal((T, W + pad), dtype=np.float32)
    if not fp32:
        x = bf16_bits_to_f32(f32_to_bf16_bits(x))
    f = 10000.0 ** (-np.arange(R // 2) / (R // 2)) * 1.1
    xd = torch.from_numpy(x).cuda()
    xd = xd if fp32 else xd.to(torch.bfloat16)
    pool0 = rng.standard_normal((blocks, tpb, 2, K, 128), dtype=np.float32)
    pool = torch.from_numpy(pool0).cuda().to(torch.bfloat16)
    pool0 = pool.float().cpu().numpy()
    q_out = torch.full((T, H * 128 + 8), 9.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.zeros(_lib.rope_append_workspace_bytes(), dtype=torch.uint8, device="cuda")
    i32 = lambda v: torch.from_numpy(np.asarray(v, np.int32)).cuda()  # noqa: E731
    a = _lib.rope_append_args(xd[:, :H * 128], xd[:, H * 128:(H + K) * 128], xd[:, (H + K) * 128:W],
                              torch.from_numpy(f).cuda(), i32(positions), i32(token_seq), i32(table), pool, q_out, H, K,
                              blocks, tpb, ws, interleaved=interleaved, factor=factor, cache_index=i32(index))
    _lib.rope_append(a)
    _, bits = _lib.read_status(ws)
    assert bool(bits & 8) == bool(len(lost)) and bits & ~8 == 0
    heads = x[:, :W].reshape(T, H + 2 * K, 128).astype(np.float64)
    ref = heads.copy()
    ref[:, :H + K] = orc.rope(heads[:, :H + K], positions, f, R, interleaved, factor)
    tol = 2.0 ** -8 * np.abs(ref) + 2.0 ** -21 * factor * 2 * np.abs(heads).max()
    got = q_out.float().cpu().numpy()
    assert (got[:, H * 128:] == 9.0).all()
    got = got[:, :H * 128].reshape(T, H, 128)
    want_pool, tol_pool = pool0.astype(np.float64), np.zeros(pool0.shape)
    for t in range(T):
        if t in skip:
            assert (got[t] == 9.0).all()
            continue
        assert (np.abs(got[t] - ref[t, :H]) <= tol[t, :H]).all(), t
        if t in lost:
            continue
        b, o = table[token_seq[t], index[t] // tpb], index[t] % tpb
        want_pool[b, o, 0], want_pool[b, o, 1] = ref[t, H:H + K], ref[t, H + K:]
        tol_pool[b, o, 0] = tol[t, H:H + K]
        tol_pool[b, o, 1] = 2.0 ** -8 * np.abs(ref[t, H + K:]) if fp32 else 0.0  # bf16 v is copied
    # written slots within the tolerance, every other slot as it was
    assert (np.abs(pool.float().cpu().numpy() - want_pool) <= tol_pool).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R", [2, 10, 16, 48, 64, 96, 112, 126, 128])
def test_rotary_dims(torch_cuda, R, interleaved):
    run(torch_cuda, 7, 4, 2, R, interleaved, seed=R, pad=8, factor=1.2)
    run(torch_cuda, 7, 3, 1, R, interleaved, seed=R, fp32=True, tpb=5)


@pytest.mark.parametrize("far", [0, 131000, 2 ** 30, -100])
def test_far_positions(torch_cuda, far):
    run(torch_cuda, 9, 2, 1, 128, False, far=far, seed=3)


@pytest.mark.parametrize("T", [1, 1183, 1184, 1189])
def test_token_counts(torch_cuda, T):
    """One token per CTA, and several with a ragged end."""
    run(torch_cuda, T, 5, 1, 64, True, seed=T)


def test_padding_and_lost_tokens(torch_cuda):
    run(torch_cuda, 12, 2, 2, 128, False, seed=6, skip=(0, 5), lost=(3, 11))


def test_matches_the_fused_kernels_rotation(torch_cuda):
    """The rotation of the whole head in halves, as the fused QKV kernels apply
    it from their table (rope_cache): the same cache and queries follow."""
    torch = torch_cuda
    from python.kinetic_rt import _lib
    from python.kinetic_rt.decoder import rope_cache, rope_inv_freq
    T, H, K = 6, 4, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, (H + 2 * K) * 128, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.tensor([0, 3, 50, 51, 1000, 2047], dtype=torch.int32, device="cuda")
    cos, sin = rope_cache(torch, 2048, 128, 5e5)
    f, factor = rope_inv_freq(torch, 128, 5e5)
    pool = torch.zeros(T * 128, 16, 2, K, 128, dtype=torch.bfloat16, device="cuda")
    table = torch.arange(T * 128, dtype=torch.int32, device="cuda").view(T, 128)
    q_out = torch.empty(T, H * 128, dtype=torch.bfloat16, device="cuda")
    ws = torch.zeros(_lib.rope_append_workspace_bytes(), dtype=torch.uint8, device="cuda")
    seq = torch.arange(T, dtype=torch.int32, device="cuda")
    _lib.rope_append(_lib.rope_append_args(x[:, :H * 128], x[:, H * 128:(H + K) * 128], x[:, (H + K) * 128:], f, pos, seq,
                                           table, pool, q_out, H, K, T * 128, 16, ws, factor=factor))
    assert _lib.read_status(ws)[0] == 0
    h = x.view(T, H + 2 * K, 128).double()
    c, s = cos[pos.long()].double()[:, None], sin[pos.long()].double()[:, None]
    ref = h * c + torch.cat([-h[..., 64:], h[..., :64]], -1) * s
    tol = 2.0 ** -8 * ref.abs() + 2.0 ** -20 * h.abs().max()
    assert ((q_out.view(T, H, 128).double() - ref[:, :H]).abs() <= tol[:, :H]).all()
    for t in range(T):
        p = int(pos[t])
        kv = pool[t * 128 + p // 16, p % 16]
        assert ((kv[0].double() - ref[t, H:H + K]).abs() <= tol[t, H:H + K]).all()
        assert torch.equal(kv[1], x.view(T, H + 2 * K, 128)[t, H + K:])


def test_side_stream_and_graph(torch_cuda):
    torch = torch_cuda
    from python.kinetic_rt import _lib
    T, H, K = 40, 4, 2
    x = torch.randn(T, (H + 2 * K) * 128, device="cuda").to(torch.bfloat16)
    pool = torch.zeros(3, 16, 2, K, 128, dtype=torch.bfloat16, device="cuda")
    q_out = torch.zeros(T, H * 128, dtype=torch.bfloat16, device="cuda")
    ws = torch.zeros(_lib.rope_append_workspace_bytes(), dtype=torch.uint8, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    f = 0.5 ** torch.arange(32, dtype=torch.float64, device="cuda")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    a = _lib.rope_append_args(x[:, :512], x[:, 512:768], x[:, 768:], f, pos, torch.zeros_like(pos), table, pool, q_out, H,
                              K, 3, 16, ws, interleaved=True)
    _lib.rope_append(a)
    want = q_out.clone(), pool.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _lib.rope_append(a)
    q_out.zero_(), pool.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q_out, want[0]) and torch.equal(pool, want[1])


def test_blocks_far_into_a_large_pool(torch_cuda):
    """A slot more than 2^32 bytes into the pool; the slots around it stay as they were."""
    torch = torch_cuda
    from python.kinetic_rt import _lib
    H, K, tpb = 4, 8, 16
    far = (9 << 29) // (tpb * 2 * K * 256)  # 4.5 GiB of blocks before the used ones
    pool = torch.empty(far + 2, tpb, 2, K, 128, dtype=torch.bfloat16, device="cuda")
    pool[far:] = 7.0
    x = torch.randn(3, (H + 2 * K) * 128, device="cuda").to(torch.bfloat16)
    q_out = torch.zeros(3, H * 128, dtype=torch.bfloat16, device="cuda")
    ws = torch.zeros(_lib.rope_append_workspace_bytes(), dtype=torch.uint8, device="cuda")
    pos = torch.tensor([0, 17, 31], dtype=torch.int32, device="cuda")
    table = torch.tensor([[far + 1, far]], dtype=torch.int32, device="cuda")
    f = 0.5 ** torch.arange(64, dtype=torch.float64, device="cuda")
    _lib.rope_append(_lib.rope_append_args(x[:, :H * 128], x[:, H * 128:(H + K) * 128], x[:, (H + K) * 128:], f, pos,
                                           torch.zeros_like(pos), table, pool, q_out, H, K, far + 2, tpb, ws))
    assert _lib.read_status(ws) == (0, 0)
    got = pool[far:, :, 1]
    want = torch.full_like(got, 7.0)
    for t, (b, o) in enumerate(((1, 0), (0, 1), (0, 15))):
        want[b, o] = x[t, (H + K) * 128:].view(K, 128)
    assert torch.equal(got, want)


@pytest.mark.parametrize("T,H,K,R,interleaved,fp32", [(700, 4, 1, 90, False, False), (700, 30, 2, 128, False, True),
                                                      (2500, 2, 1, 10, True, False), (2499, 1, 1, 66, False, True)])
def test_many_tokens(torch_cuda, T, H, K, R, interleaved, fp32):
    """Two warps and one warp per token, CTAs of several tokens, the last one not full."""
    run(torch_cuda, T, H, K, R, interleaved, fp32=fp32, seed=T + R, skip=(3, T - 1), lost=(8, 640))
