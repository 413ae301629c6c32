"""Limits of the attention calls with score modifications, on the CPU: what the
size functions answer for shapes that the calls refuse, and for the largest."""
import os

import pytest

from python.kinetic_rt import _lib
from tests.test_capi_mod_validation import FAKE, call, decode, prefill, rope

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libkrt.so not built")

BIG = 2 ** 31 - 1


@pytest.mark.parametrize("group", [17, 32, 128, 129, 256, 4096])
def test_no_workspace_for_groups_that_are_refused(group):
    """More query heads per KV head than the kernels take: 0, as for other shapes that a call refuses."""
    assert _lib.prefill_attention_mod_workspace_bytes(64, 1, group, 1, 4096) == 0
    assert _lib.attention_mod_workspace_bytes(4, group, 1, 4096) == 0
    assert _lib.prefill_attention_mod_workspace_bytes(64, 1, 16, 1, 4096) > 0
    assert _lib.attention_mod_workspace_bytes(4, 16, 1, 4096) > 0


def test_sizes_of_the_largest_shapes():
    """No overflow: sizes grow with every argument up to its end."""
    few = _lib.prefill_attention_mod_workspace_bytes(1, 1, 1, 1, BIG)
    for args in ((BIG, 1, 1, 1, BIG), (BIG, BIG, 16, 1, BIG), (BIG, BIG, 16 * 65535, 65535, BIG)):
        assert few <= _lib.prefill_attention_mod_workspace_bytes(*args) < 1 << 28
    assert _lib.attention_mod_workspace_bytes(BIG, 16, 1, BIG) > _lib.attention_mod_workspace_bytes(1 << 20, 16, 1, BIG)


@pytest.mark.parametrize("fn,args", [("krt_paged_attention_decode_mod", decode), ("krt_paged_attention_prefill_mod", prefill)])
@pytest.mark.parametrize("heads", [1 << 25, 16 * 65536])
def test_more_heads_than_a_stride_can_tell(fn, args, heads):
    """n_heads * 128 beyond 32 bits would let any row stride pass."""
    rc, msg = call(fn, args(n_heads=heads, n_kv_heads=heads // 16, lse=FAKE, lse_stride=heads))
    assert rc == _lib.KRT_ERR_UNSUPPORTED and "n_kv_heads" in msg, (rc, msg)


@pytest.mark.parametrize("over,text", [(dict(block_table_columns=62), "cannot hold"), (dict(block_table_columns=-1), "columns"),
                                       (dict(block_table_columns=65), "columns")])
@pytest.mark.parametrize("fn,args", [("krt_paged_attention_decode_mod", decode), ("krt_paged_attention_prefill_mod", prefill)])
def test_block_table_columns(fn, args, over, text):
    """The columns of a row, not its stride, have to hold the longest sequence (1000 tokens take 63 blocks of 16)."""
    rc, msg = call(fn, args(**over))
    assert rc == _lib.KRT_ERR_INVALID and text in msg, (rc, msg)


@pytest.mark.parametrize("columns", [-1, 5])
def test_rope_append_block_table_columns(columns):
    rc, msg = call("krt_rope_append", rope(block_table_columns=columns))
    assert rc == _lib.KRT_ERR_INVALID and "columns" in msg, (rc, msg)


def test_row_stride_of_one_row():
    torch = pytest.importorskip("torch")
    assert _lib._row_stride(torch.empty(512, 1).T, 512) == 512
    assert _lib._row_stride(torch.empty(1, 520)[:, :512], 512) == 512
    assert _lib._row_stride(torch.empty(2, 520)[:, :512], 512) == 520


@pytest.mark.parametrize("at", [0, 16, 2032, 2048, 2304, 2544, 6160, -16, 2064 + 5 * 8192])
def test_rope_append_rows_that_share_columns(at):
    """Ten rows of 8192 bytes with q in [0, 2048), k in [2048, 2304) and v in [2304, 2560).  q_out's rows (2048 bytes, of
    the same pitch) overlap one of them unless they start in 2560 .. 6144."""
    q = FAKE + (1 << 20)
    over = dict(n_kv_heads=1, q=q, k=q + 2048, v=q + 2304, q_out=q + at, q_stride=4096, k_stride=4096, v_stride=4096,
                q_out_stride=4096)
    rc, msg = call("krt_rope_append", rope(**over))
    assert rc == _lib.KRT_ERR_INVALID and "overlaps" in msg, (rc, msg)
