"""Argument checks of the attention calls with score modifications and of the
rotary append, on the CPU: every case is rejected before any CUDA call, so the
pointers are fake, aligned and never dereferenced."""
import ctypes
import os

import pytest

from python.kinetic_rt import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libkrt.so not built")

FAKE = 0x10000
NAN, INF = float("nan"), float("inf")


def call(fn, a):
    h = _lib.lib()
    rc = getattr(h, fn)(ctypes.byref(a) if a is not None else None, None)
    return rc, h.krt_last_error().decode()


def decode(**over):
    a = _lib.PagedAttentionModArgs()
    for name in ("q", "kv_pool", "block_table", "seq_lens", "out", "workspace"):
        setattr(a, name, FAKE)
    a.num_seqs, a.n_heads, a.n_kv_heads, a.head_dim = 4, 32, 8, 128
    a.q_stride = a.out_stride = 4096
    a.block_table_stride, a.num_blocks, a.tokens_per_block = 64, 512, 16
    a.max_seq_len, a.workspace_bytes = 1000, 1 << 30
    for k, v in over.items():
        setattr(a, k, v)
    return a


def prefill(**over):
    a = _lib.PagedPrefillAttentionModArgs()
    for name in ("q", "kv_pool", "block_table", "q_start", "q_pos0", "out", "workspace"):
        setattr(a, name, FAKE)
    a.num_tokens, a.num_seqs, a.n_heads, a.n_kv_heads, a.head_dim = 100, 4, 32, 8, 128
    a.q_stride = a.out_stride = 4096
    a.block_table_stride, a.num_blocks, a.tokens_per_block = 64, 512, 16
    a.max_kv_len, a.workspace_bytes = 1000, 1 << 30
    for k, v in over.items():
        setattr(a, k, v)
    return a


COMMON = [
    (dict(q=None), _lib.KRT_ERR_INVALID, "NULL"),
    (dict(workspace=None), _lib.KRT_ERR_INVALID, "NULL"),
    (dict(num_seqs=0), _lib.KRT_ERR_INVALID, "positive"),
    (dict(n_kv_heads=0), _lib.KRT_ERR_INVALID, "positive"),
    (dict(head_dim=64), _lib.KRT_ERR_UNSUPPORTED, "head_dim"),
    (dict(n_heads=30), _lib.KRT_ERR_UNSUPPORTED, "n_kv_heads"),
    (dict(n_heads=34, n_kv_heads=2, q_stride=8192, out_stride=8192), _lib.KRT_ERR_UNSUPPORTED, "16 per KV head"),
    (dict(tokens_per_block=24), _lib.KRT_ERR_UNSUPPORTED, "multiple of 16"),
    (dict(num_blocks=0), _lib.KRT_ERR_INVALID, "geometry"),
    (dict(num_blocks=1 << 27), _lib.KRT_ERR_UNSUPPORTED, "2^31"),
    (dict(block_table_stride=10), _lib.KRT_ERR_INVALID, "block table"),
    (dict(q_stride=4092), _lib.KRT_ERR_INVALID, "strides"),
    (dict(out_stride=4100), _lib.KRT_ERR_INVALID, "strides"),
    (dict(lse=FAKE, lse_stride=31), _lib.KRT_ERR_INVALID, "lse_stride"),
    (dict(scale=-1.0), _lib.KRT_ERR_INVALID, "scale"),
    (dict(scale=NAN), _lib.KRT_ERR_INVALID, "scale"),
    (dict(softcap=-30.0), _lib.KRT_ERR_INVALID, "softcap"),
    (dict(softcap=INF), _lib.KRT_ERR_INVALID, "softcap"),
    (dict(softcap=NAN), _lib.KRT_ERR_INVALID, "softcap"),
    (dict(window=-1), _lib.KRT_ERR_INVALID, "window"),
    (dict(out=FAKE + 8), _lib.KRT_ERR_INVALID, "aligned"),
    (dict(workspace_bytes=64), _lib.KRT_ERR_WORKSPACE, "needed"),
]


@pytest.mark.parametrize("over,code,text", COMMON + [(dict(max_seq_len=0), _lib.KRT_ERR_INVALID, "positive")])
def test_decode_mod_rejects(over, code, text):
    rc, msg = call("krt_paged_attention_decode_mod", decode(**over))
    assert rc == code and text in msg and msg.startswith("krt_paged_attention_decode_mod"), (rc, msg)


@pytest.mark.parametrize("over,code,text", COMMON + [(dict(max_kv_len=0), _lib.KRT_ERR_INVALID, "positive"),
                                                     (dict(num_tokens=0), _lib.KRT_ERR_INVALID, "positive")])
def test_prefill_mod_rejects(over, code, text):
    rc, msg = call("krt_paged_attention_prefill_mod", prefill(**over))
    assert rc == code and text in msg and msg.startswith("krt_paged_attention_prefill_mod"), (rc, msg)


def rope(**over):
    a = _lib.RopeAppendArgs()
    for i, name in enumerate(("q", "k", "v", "inv_freq", "positions", "token_seq", "block_table", "kv_pool", "q_out",
                              "workspace")):
        setattr(a, name, FAKE + (i << 32))
    a.num_tokens, a.n_heads, a.n_kv_heads, a.head_dim, a.rotary_dim = 10, 8, 2, 128, 64
    a.q_stride, a.k_stride, a.v_stride, a.q_out_stride = 1536, 1536, 1536, 1024
    a.num_seqs, a.block_table_stride, a.num_blocks, a.tokens_per_block = 2, 4, 8, 16
    a.workspace_bytes = 8192
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code,text", [
    (dict(k=None), _lib.KRT_ERR_INVALID, "NULL"),
    (dict(num_tokens=0), _lib.KRT_ERR_INVALID, "positive"),
    (dict(head_dim=96), _lib.KRT_ERR_UNSUPPORTED, "head_dim"),
    (dict(rotary_dim=0), _lib.KRT_ERR_INVALID, "rotary_dim"),
    (dict(rotary_dim=63), _lib.KRT_ERR_INVALID, "rotary_dim"),
    (dict(rotary_dim=130), _lib.KRT_ERR_INVALID, "rotary_dim"),
    (dict(dtype=7), _lib.KRT_ERR_UNSUPPORTED, "float32"),
    (dict(q_stride=1000), _lib.KRT_ERR_INVALID, "strides"),
    (dict(v_stride=1540), _lib.KRT_ERR_INVALID, "strides"),
    (dict(dtype=_lib.KRT_DTYPE_FLOAT32, v_stride=1538), _lib.KRT_ERR_INVALID, "strides"),
    (dict(k=FAKE + 8), _lib.KRT_ERR_INVALID, "aligned"),
    (dict(tokens_per_block=0), _lib.KRT_ERR_INVALID, "geometry"),
    (dict(factor=NAN), _lib.KRT_ERR_INVALID, "factor"),
    (dict(workspace_bytes=4), _lib.KRT_ERR_WORKSPACE, "needed"),
    (dict(q_out=FAKE), _lib.KRT_ERR_INVALID, "overlaps"),
    (dict(q_out=FAKE + (1 << 32) + 1024), _lib.KRT_ERR_INVALID, "overlaps"),
])
def test_rope_append_rejects(over, code, text):
    rc, msg = call("krt_rope_append", rope(**over))
    assert rc == code and text in msg and msg.startswith("krt_rope_append"), (rc, msg)


@pytest.mark.parametrize("fn", ["krt_paged_attention_decode_mod", "krt_paged_attention_prefill_mod", "krt_rope_append"])
def test_null_args(fn):
    rc, msg = call(fn, None)
    assert rc == _lib.KRT_ERR_INVALID and "NULL" in msg


def test_workspace_sizes():
    assert _lib.attention_mod_workspace_bytes(4, 32, 8, 65536) > _lib.attention_mod_workspace_bytes(4, 32, 8, 65536, 64)
    assert _lib.attention_mod_workspace_bytes(4, 30, 8, 100) == 0
    assert _lib.attention_mod_workspace_bytes(4, 32, 8, 100, -1) == 0
    assert _lib.prefill_attention_mod_workspace_bytes(100, 4, 32, 8, 1000) >= 8192
    assert _lib.prefill_attention_mod_workspace_bytes(0, 4, 32, 8, 1000) == 0
    assert _lib.rope_append_workspace_bytes() > 0


def test_python_arguments_must_be_cuda_tensors():
    torch = pytest.importorskip("torch")
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    ws = torch.zeros(8192, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA device"):
        _lib.attention_mod_args(bf(2, 512), bf(4, 16, 2, 1, 128), i32(2, 2), i32(2), bf(2, 512), 4, 1, 4, 16, 32, ws)
    with pytest.raises(ValueError, match="CUDA device"):
        _lib.prefill_attention_mod_args(bf(2, 512), bf(4, 16, 2, 1, 128), i32(1, 2), i32(2), i32(1), bf(2, 512), 4, 1, 4,
                                        16, 32, ws)
    with pytest.raises(ValueError, match="CUDA device"):
        _lib.rope_append_args(bf(2, 512), bf(2, 128), bf(2, 128), torch.zeros(64, dtype=torch.float64), i32(2), i32(2),
                              i32(1, 2), bf(4, 16, 2, 1, 128), bf(2, 512), 4, 1, 4, 16, ws)


@pytest.mark.parametrize("stream", [None, 0, 77])
@pytest.mark.parametrize("call", [_lib.paged_attention_decode_mod, _lib.paged_attention_prefill_mod, _lib.rope_append])
def test_another_current_device_is_refused(monkeypatch, call, stream):
    """A launch would run on the current device: with tensors of another one it does not start."""
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    args = _lib.RopeAppendArgs()
    args._index = 0
    args._ref = None
    with pytest.raises(ValueError, match="current device is cuda:1"):
        call(args, stream)
