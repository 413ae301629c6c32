"""krt_rope_append with q_out in columns of the tensor that holds q, k and v."""
import pytest

from tests.test_gpu_rope_append import torch_cuda  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("front", [False, True])
@pytest.mark.parametrize("T", [1, 2, 70])
def test_queries_beside_their_projection(torch_cuda, T, front, fp32):  # noqa: F811
    """Rows of [q | k | v] and q_out, in either order: they alternate in memory and do not overlap."""
    torch = torch_cuda
    from python.kinetic_rt import _lib
    H, K, tpb = 4, 2, 16
    W, Q, e = (H + 2 * K) * 128, H * 128, 2 if fp32 else 1
    wide = torch.zeros(T, e * W + Q, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(T, W, device="cuda")
    x = x if fp32 else x.to(torch.bfloat16)
    inside, q_out = (wide[:, Q:], wide[:, :Q]) if front else (wide[:, :e * W], wide[:, e * W:])
    if fp32:
        inside = inside.view(torch.float32)
    inside.copy_(x)
    ws = torch.zeros(_lib.rope_append_workspace_bytes(), dtype=torch.uint8, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    table = torch.arange(5, dtype=torch.int32, device="cuda").view(1, 5)
    f = 0.5 ** torch.arange(64, dtype=torch.float64, device="cuda")
    got = []
    for src, q in ((x, torch.zeros(T, Q, dtype=torch.bfloat16, device="cuda")), (inside, q_out)):
        pool = torch.zeros(5, tpb, 2, K, 128, dtype=torch.bfloat16, device="cuda")
        _lib.rope_append(_lib.rope_append_args(src[:, :Q], src[:, Q:Q + K * 128], src[:, Q + K * 128:], f, pos,
                                               torch.zeros_like(pos), table, pool, q, H, K, 5, tpb, ws))
        assert _lib.read_status(ws) == (0, 0)
        got.append((q.clone(), pool))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert torch.equal(inside, x)
