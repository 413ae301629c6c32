"""CPU checks of oracle/attention_mod.py: against torch's attention with an
explicit mask and bias, and against the half-split rotation of the fused layer."""
import numpy as np
import pytest
import torch

from oracle import attention_mod as orc
from oracle.torch_ref import rotate_half


@pytest.mark.parametrize("softcap,window,kv_start,prefix,bias", [
    (0.0, 0, 0, 0, False), (0.0, 7, 0, 0, False), (0.0, 0, 9, 0, True), (0.0, 5, 3, 30, True), (3.0, 0, 0, 20, False)])
def test_attention_mod_matches_torch(softcap, window, kv_start, prefix, bias):
    rng = np.random.Generator(np.random.PCG64(3))
    B, L, H, K = 16, 40, 4, 2
    pool = rng.standard_normal((4, B, 2, K, 128))
    table = np.array([[2, 0, 3]])
    q = rng.standard_normal((L, H, 128))
    slopes = 2.0 ** -np.arange(1, H + 1) if bias else None
    rows = [(0, i, L, kv_start, prefix) for i in range(L)]
    out, lse, _, _ = orc.paged_attention_mod(q, pool, table, rows, H, K, B, softcap, window, slopes)
    kv = torch.from_numpy(np.concatenate([pool[b] for b in table[0]])[:L])
    k, v = (kv[:, i].permute(1, 0, 2).repeat_interleave(H // K, 0) for i in (0, 1))
    pos = torch.arange(L)
    ok = (pos[None] <= pos[:, None]) | (pos[None] < prefix)
    ok &= pos[None] >= kv_start
    if window:
        ok &= pos[:, None] - pos[None] < window
    x = torch.from_numpy(q).permute(1, 0, 2) @ k.transpose(1, 2) / np.sqrt(128)
    if softcap:
        x = softcap * torch.tanh(x / softcap)
    if bias:
        x = x - torch.from_numpy(slopes)[:, None, None] * (pos[:, None] - pos[None]).abs()
    x = x.masked_fill(~ok, -np.inf)
    seen = ok.any(-1)
    ref = (torch.softmax(x, -1) @ v).permute(1, 0, 2)[seen]
    np.testing.assert_allclose(out[seen.numpy()], ref.numpy(), atol=1e-12)
    np.testing.assert_allclose(lse[seen.numpy()], torch.logsumexp(x, -1).T[seen].numpy(), atol=1e-12)
    assert (out[~seen.numpy()] == 0).all() and np.isneginf(lse[~seen.numpy()]).all()


def test_rope_matches_the_half_split_reference():
    rng = np.random.Generator(np.random.PCG64(4))
    x = rng.standard_normal((5, 3, 128))
    pos, f = np.array([0, 1, 77, 4095, 100000]), 10000.0 ** (-np.arange(0, 128, 2) / 128)
    emb = torch.from_numpy(np.concatenate([np.outer(pos, f)] * 2, -1))[:, None]
    xt = torch.from_numpy(x)
    ref = xt * emb.cos() + rotate_half(xt) * emb.sin()
    np.testing.assert_allclose(orc.rope(x, pos, f, 128, False), ref.numpy(), atol=1e-12)


def test_rope_interleaved_is_a_permutation_of_halves():
    rng = np.random.Generator(np.random.PCG64(5))
    x, R = rng.standard_normal((4, 2, 128)), 24
    pos, f = np.array([3, 9, 27, 81]), rng.random(R // 2)
    perm = np.concatenate([np.arange(0, R, 2), np.arange(1, R, 2), np.arange(R, 128)])
    got = orc.rope(x, pos, f, R, True, 1.25)
    np.testing.assert_allclose(got[..., perm], orc.rope(x[..., perm], pos, f, R, False, 1.25), atol=1e-12)
    assert (got[..., R:] == x[..., R:]).all()
