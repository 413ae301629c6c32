"""Score caps over the whole range that the calls take, single tokens and
prompts, against oracle/attention_mod.py in 64 bits.

Tolerance of a score x (natural units): the dot product as in the oracle, and
of the cap 2^-19 of |x| (the polynomials' relative error is 1.5e-6 < 2^-19.3,
its coefficients, powers and the product round about six times, 2^-24 each),
or, for scores beyond the polynomials' range, the exponent form's 4 roundings
of the cap, 2^-22 c, there less than 2^-17 of |x| >= 0.05 c."""
import numpy as np
import pytest

from oracle import attention_mod as orc
from tests.test_gpu_attention_mod import Case, torch_cuda  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def row(q, k, v, scale, cap):
    s = (k @ q) * scale
    x = cap * np.tanh(s / cap)
    top = x.max()
    e = np.exp(x - top)
    w = e / e.sum()
    fuzz = 2.0 ** -24 * 130 * scale * (np.abs(k) @ np.abs(q)).max() + (2.0 ** -19 + 2.0 ** -17) * np.abs(x).max()
    return w @ v, top + np.log(e.sum()), w @ np.abs(v), fuzz


@pytest.mark.parametrize("scale", [0.0, 1.0, 1e-3])
@pytest.mark.parametrize("cap", [1e-30, 1e-6, 0.02, 1.0, 30.0, 700.0, 900.0, 1e4, 1e5, 1e6, 1e8, 1e12, 1e20, 1e30, 3e38])
@pytest.mark.parametrize("q_lens", [None, [40, 3]])
def test_caps(torch_cuda, q_lens, cap, scale):  # noqa: F811
    c = Case(torch_cuda, [150, 61] if q_lens is None else [100, 0], q_lens=q_lens, n_heads=4, n_kv_heads=2, seed=100)
    cap, scale_used = float(np.float32(cap)), float(np.float32(scale)) or 128 ** -0.5
    c.launch(c.args(softcap=cap, scale=scale))
    got, got_lse = c.result()
    for t, (s, pos, length, _, _) in list(enumerate(c.rows()))[::7]:
        k, v = orc.gather_kv(c.pool, c.table[s], pos + 1, c.tpb)
        for h in range(c.H):
            o, lse, a, fuzz = row(c.q[t, h].astype(float), k[:, h // 2].astype(float), v[:, h // 2].astype(float),
                                  scale_used, cap)
            rel = 2.0 ** -8 + 2 * (fuzz + 2.0 ** -20 + (pos + 1) * 2.0 ** -24)
            assert (np.abs(got[t, h] - o) <= rel * a + 2.0 ** -8 * np.abs(o) + 1e-30).all()
            assert abs(got_lse[t, h] - lse) <= fuzz + 2.0 ** -20 + (pos + 1) * 2.0 ** -24 + 2.0 ** -22 * abs(lse)


@pytest.mark.parametrize("cap", [30.0, 1e3, 1e5])
def test_scores_from_far_below_to_far_above_the_cap(torch_cuda, cap):  # noqa: F811
    """One call with scores on both sides of the polynomials' range."""
    def edit(pool, c):
        pool[..., 0, :, :] *= np.exp2(np.arange(c.blocks) % 9 - 4)[:, None, None, None] * cap / 60

    for q_lens in (None, [90]):
        c = Case(torch_cuda, [300], q_lens=q_lens, n_heads=4, n_kv_heads=2, seed=101, edit_pool=edit)
        c.launch(c.args(softcap=cap))
        got, got_lse = c.result()
        for t, (s, pos, length, _, _) in list(enumerate(c.rows()))[::13]:
            k, v = orc.gather_kv(c.pool, c.table[s], pos + 1, c.tpb)
            for h in range(c.H):
                o, lse, a, fuzz = row(c.q[t, h].astype(float), k[:, h // 2].astype(float), v[:, h // 2].astype(float),
                                      128 ** -0.5, cap)
                rel = 2.0 ** -8 + 2 * (fuzz + 2.0 ** -20 + (pos + 1) * 2.0 ** -24)
                assert (np.abs(got[t, h] - o) <= rel * a + 2.0 ** -8 * np.abs(o) + 1e-30).all()
                assert abs(got_lse[t, h] - lse) <= fuzz + 2.0 ** -20 + (pos + 1) * 2.0 ** -24 + 2.0 ** -22 * abs(lse)
