"""The rotary append and both attentions with score modifications run together,
as a model uses them: two layers of different kinds over one block table, a
ragged batch of prompts in two chunks, then decode steps from one CUDA graph.

The append is held to oracle/attention_mod.rope (one bf16 rounding, 2^-8, and
2^-21 of the pair for the fp32 rotation), the attention to the 64-bit oracle
on the rotated queries and the cache that the append left."""
import numpy as np
import pytest

from oracle import attention_mod as orc
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu

H, K, TPB, R, S, MAX_LEN = 8, 2, 16, 96, 3, 160
W = (H + 2 * K) * 128
FACTOR = 1.0625
LAYERS = [dict(softcap=30.0), dict(window=40, slopes=[2.0 ** -(h + 1) for h in range(H)])]


@pytest.fixture(scope="module")
def torch_cuda():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


class Layer:
    def __init__(self, torch, mods, table, seed):
        from python.kinetic_rt import _lib
        self.torch, self.mods, self.table = torch, mods, table
        self.rng = np.random.Generator(np.random.PCG64(seed))
        self.blocks = int(table.max()) + 2
        self.table_d = torch.from_numpy(table).cuda()
        self.pool = torch.zeros(self.blocks, TPB, 2, K, 128, dtype=torch.bfloat16, device="cuda")
        self.freq = 10000.0 ** (-np.arange(R // 2) / (R // 2))
        self.freq_d = torch.from_numpy(self.freq).cuda()
        z = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")  # noqa: E731
        self.ws = [z(_lib.rope_append_workspace_bytes()),
                   z(_lib.prefill_attention_mod_workspace_bytes(512, S, H, K, MAX_LEN)),
                   z(_lib.attention_mod_workspace_bytes(S, H, K, MAX_LEN, mods.get("window", 0)))]
        slopes = mods.get("slopes")
        self.kw = dict(softcap=mods.get("softcap", 0.0), window=mods.get("window", 0),
                       alibi_slopes=None if slopes is None else torch.tensor(slopes, device="cuda"))

    def projections(self, n):
        """q, k, v of n tokens, side by side, as a QKV projection leaves them."""
        bits = f32_to_bf16_bits(2.0 * self.rng.standard_normal((n, W), dtype=np.float32))
        return self.torch.from_numpy(bits.view(np.int16)).view(self.torch.bfloat16), bf16_bits_to_f32(bits)

    def append(self, x, positions, token_seq, q):
        from python.kinetic_rt import _lib
        return _lib.rope_append_args(x[:, :H * 128], x[:, H * 128:(H + K) * 128], x[:, (H + K) * 128:], self.freq_d,
                                     positions, token_seq, self.table_d, self.pool, q, H, K, self.blocks, TPB,
                                     self.ws[0], interleaved=True, factor=FACTOR)

    def check(self, x, rows, q, out, lse, before):
        """rows: (sequence, position, length) of each token; before: the cache before the step."""
        from python.kinetic_rt import _lib
        for ws in self.ws:
            assert _lib.read_status(ws) == (0, 0)
        pos = np.array([r[1] for r in rows])
        heads = x.reshape(len(rows), H + 2 * K, 128).astype(np.float64)
        ref = heads.copy()
        ref[:, :H + K] = orc.rope(heads[:, :H + K], pos, self.freq, R, True, FACTOR)
        pair = np.repeat(np.hypot(heads[..., 0::2], heads[..., 1::2]), 2, axis=-1) * FACTOR
        tol = 2.0 ** -8 * np.abs(ref) + 2.0 ** -21 * pair + 2.0 ** -133
        got_q = q.float().cpu().numpy().reshape(len(rows), H, 128)
        pool = self.pool.float().cpu().numpy()
        assert (np.abs(got_q - ref[:, :H]) <= tol[:, :H]).all()
        want = before.copy()
        for t, (s, p, _) in enumerate(rows):
            slot = pool[self.table[s, p // TPB], p % TPB]
            assert (np.abs(slot - ref[t, H:].reshape(2, K, 128)) <= tol[t, H:].reshape(2, K, 128)).all()
            want[self.table[s, p // TPB], p % TPB] = slot
        assert (pool == want).all()  # nothing else was written
        slopes = self.mods.get("slopes")
        ref, ref_lse, tol, tol_lse = orc.paged_attention_mod(
            got_q, pool, self.table, [(s, p, n, 0, 0) for s, p, n in rows], H, K, TPB, self.mods.get("softcap", 0.0),
            self.mods.get("window", 0), None if slopes is None else np.float32(slopes))
        assert (np.abs(out.float().cpu().numpy().reshape(-1, H, 128) - ref) <= tol).all()
        assert (np.abs(lse.cpu().numpy() - ref_lse) <= tol_lse).all()


def test_prompt_chunks_then_decode(torch_cuda):
    torch = torch_cuda
    from python.kinetic_rt import _lib
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
    rng = np.random.Generator(np.random.PCG64(50))
    bps = MAX_LEN // TPB
    table = rng.permutation(S * bps).astype(np.int32).reshape(S, bps)
    layers = [Layer(torch, m, table, 60 + i) for i, m in enumerate(LAYERS)]
    lens = np.zeros(S, int)

    # prompts, in two chunks
    for chunk in ([70, 33, 1], [5, 0, 64]):
        T = sum(chunk)
        rows = [(s, lens[s] + i, lens[s] + n) for s, n in enumerate(chunk) for i in range(n)]
        for layer in layers:
            xh, x = layer.projections(T)
            xd = xh.cuda()
            q = torch.empty(T, H * 128, dtype=torch.bfloat16, device="cuda")
            out, lse = torch.empty_like(q), torch.empty(T, H, dtype=torch.float32, device="cuda")
            before = layer.pool.float().cpu().numpy()
            _lib.rope_append(layer.append(xd, i32([r[1] for r in rows]), i32([r[0] for r in rows]), q))
            starts = np.concatenate([[0], np.cumsum(chunk)])
            _lib.paged_attention_prefill_mod(_lib.prefill_attention_mod_args(
                q, layer.pool, layer.table_d, i32(starts), i32(lens), out, H, K, layer.blocks, TPB, MAX_LEN,
                layer.ws[1], lse=lse, **layer.kw))
            layer.check(x, rows, q, out, lse, before)
        lens += chunk

    # decode: both layers in one graph; its inputs, positions and lengths are rewritten before each replay
    positions, seq_lens, token_seq = i32([0] * S), i32([0] * S), i32(range(S))
    state = []
    for layer in layers:
        x = torch.zeros(S, W, dtype=torch.bfloat16, device="cuda")
        q = torch.zeros(S, H * 128, dtype=torch.bfloat16, device="cuda")
        out, lse = torch.zeros_like(q), torch.zeros(S, H, dtype=torch.float32, device="cuda")
        state.append((x, q, out, lse, layer.append(x, positions, token_seq, q), _lib.attention_mod_args(
            q, layer.pool, layer.table_d, seq_lens, out, H, K, layer.blocks, TPB, MAX_LEN, layer.ws[2], lse=lse,
            **layer.kw)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for x, q, out, lse, append, attend in state:
            _lib.rope_append(append)
            _lib.paged_attention_decode_mod(attend)
    for _ in range(4):
        lens += 1
        positions.copy_(i32(lens - 1))
        seq_lens.copy_(i32(lens))
        rows = [(s, lens[s] - 1, lens[s]) for s in range(S)]
        inputs = []
        for layer, st in zip(layers, state):
            xh, x = layer.projections(S)
            st[0].copy_(xh.cuda())
            inputs.append((x, layer.pool.float().cpu().numpy()))
        graph.replay()
        torch.cuda.synchronize()
        for layer, st, (x, before) in zip(layers, state, inputs):
            layer.check(x, rows, st[1], st[2], st[3], before)
