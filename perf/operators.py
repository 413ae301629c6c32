"""Measured cases of the paged-cache operators with score modifications.

Three operators that work on one paged KV cache (pool [block][token][K|V]
[kv_head][128] bf16, int32 block tables):

  rope    rotary positions (half or interleaved pairs, part of the head,
          frequencies scaled for long contexts) of q and k, with k and v
          appended to the cache
  prefill attention of prompt tokens whose scores are capped by a tanh, get a
          bias that falls with distance, and are masked by a window, by the
          start of a document or by a prefix that is visible to all
  decode  the same for one new token per sequence

`run` computes them in plain torch (own = False) or calls the framework's
kernels (own = True); `exact` is their definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

HEAD_DIM = 128


# ------------------------------------------------------------------ cases
def _prefill(name, **kw):
    c = dict(op="prefill", seqs=1, q_len=64, ctx=0, ragged=False, n_heads=32, n_kv_heads=8, tpb=16, cap=0.0,
             window=0, alibi=False, prefix=0, doc=0, empty=0)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _decode(name, **kw):
    c = dict(op="decode", seqs=1, ctx=4224, ragged=False, n_heads=32, n_kv_heads=8, tpb=16, cap=0.0, window=0,
             alibi=False, doc=0)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _rope(name, **kw):
    c = dict(op="rope", seqs=64, q_len=1, ctx=2048, ragged=False, offset=0, n_heads=32, n_kv_heads=8, tpb=16,
             rotary=128, interleaved=False, stretch=1.0, fp32=False)
    c.update(kw)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # a short first prompt of a chat, alone on the GPU: the call's latency
        _prefill("prefill_1x64_cap", cap=50.0),
        # a batch of equal prompts through a model with capped scores
        _prefill("prefill_8x2048_cap", seqs=8, q_len=2048, cap=50.0),
        # long prompts, one rank's heads of a large model under tensor parallelism, a sliding-window layer
        _prefill("prefill_4x8192_window", seqs=4, q_len=8192, n_heads=8, n_kv_heads=1, window=4096, cap=30.0),
        # several documents packed into one row, distance bias, padding rows among them
        _prefill("prefill_docs_alibi", q_len=8192, alibi=True, doc=1531, empty=61),
        # later chunks of ragged prompts behind a cached part, instructions as a prefix visible to all
        _prefill("prefill_chunks_prefix", seqs=6, q_len=517, ctx=3700, ragged=True, n_heads=64, prefix=4000, tpb=32),
        # one user's decode step
        _decode("decode_1_alibi", alibi=True),
        # a full decode batch at a long context, capped scores
        _decode("decode_128_cap", seqs=128, cap=50.0),
        # a decode batch on one rank's heads, a sliding-window layer
        _decode("decode_256_window", seqs=256, ctx=2112, n_heads=8, n_kv_heads=1, window=1024, cap=30.0),
        # few sequences at long ragged contexts: the length has to be split
        _decode("decode_3_long", seqs=3, ctx=65536, ragged=True, n_heads=64, alibi=True, tpb=32),
        # one decode step's new tokens, far positions
        _rope("rope_64", ctx=4096, offset=100000, stretch=8.0),
        # prompts, interleaved pairs in half of the head
        _rope("rope_8x2048_interleaved", seqs=8, q_len=2048, ctx=0, rotary=64, interleaved=True),
        # long ragged prompts from a projection that leaves 32-bit results, scaled frequencies
        _rope("rope_4x8192_fp32", seqs=4, q_len=8192, ctx=0, ragged=True, n_heads=8, n_kv_heads=1, stretch=8.0,
              fp32=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "decode", "decode", "rope"])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    heads = kv * group
    if heads > 64:
        kv, heads = max(1, 64 // group), max(1, 64 // group) * group
    tpb = rng.choice([16, 16, 32, 48, 64])
    mods = dict(cap=rng.choice([0.0, 0.0, 20.0, 30.0, 50.0]), alibi=rng.random() < 0.4)
    if op == "prefill":
        q_len, ctx = _log(rng, 1, 8192), rng.choice([0, 0, _log(rng, 1, 8192)])
        # no more score values than the largest listed case computes plainly
        most = 4 * 8192 * 8192 * 8 / (q_len * (q_len + ctx) * heads)
        if most < 1:
            q_len = max(1, int(q_len * most * 0.9))
            most = 4 * 8192 * 8192 * 8 / (q_len * (q_len + ctx) * heads)
        seqs = _log(rng, 1, max(1, min(64, int(most))))
        return _prefill(None, seqs=seqs, q_len=q_len, ctx=ctx, ragged=rng.random() < 0.6, n_heads=heads, n_kv_heads=kv,
                        tpb=tpb, window=rng.choice([0, 0, _log(rng, 1, 8192)]),
                        prefix=rng.choice([0, 0, _log(rng, 1, q_len + ctx)]),
                        doc=rng.choice([0, 0, _log(rng, 16, 8192)]), empty=rng.choice([0, 0, rng.randint(2, 97)]), **mods)
    if op == "decode":
        ctx = _log(rng, 1, 65536)
        seqs = _log(rng, 1, max(1, min(256, 128 * 4224 * 8 // (ctx * kv))))
        return _decode(None, seqs=seqs, ctx=ctx, ragged=rng.random() < 0.6, n_heads=heads, n_kv_heads=kv, tpb=tpb,
                       window=rng.choice([0, 0, _log(rng, 1, 65536)]), doc=rng.choice([0, 0, _log(rng, 16, 8192)]), **mods)
    q_len = rng.choice([1, _log(rng, 1, 8192)])
    seqs = _log(rng, 1, max(1, min(256, 16384 * 48 // (q_len * (heads + 2 * kv)))))
    return _rope(None, seqs=seqs, q_len=q_len, ctx=rng.choice([0, _log(rng, 1, 4096)]), ragged=rng.random() < 0.5,
                 offset=rng.choice([0, 0, _log(rng, 1, 1000000)]), n_heads=heads, n_kv_heads=kv, tpb=tpb,
                 rotary=2 * rng.randint(1, 64) if rng.random() < 0.5 else rng.choice([32, 64, 96, 128]),
                 interleaved=rng.random() < 0.5, stretch=rng.choice([1.0, 2.0, 8.0, 32.0]), fp32=rng.random() < 0.3)


def _lens(c):
    """(tokens before the new ones, new tokens) of each sequence."""
    got = []
    for s in range(c["seqs"]):
        n, ctx = c.get("q_len", 1), c["ctx"]
        if c["ragged"]:
            n -= (s * 53) % max(1, n // 2)
            ctx -= (s * 1031) % (ctx // 2 + 1)
        got.append((ctx, n))
    return got


def _slopes(c):
    return [2.0 ** (-8.0 * (h + 1) / c["n_heads"]) for h in range(c["n_heads"])]


def _bounds(c, s_ctx, s_n, row, pos):
    """Half-open range of visible positions of one query row."""
    if c.get("empty") and row % c["empty"] == 1:
        return 0, 0
    lo = (pos // c["doc"]) * c["doc"] if c["doc"] else 0
    if c["window"]:
        lo = max(lo, pos - c["window"] + 1)
    return lo, max(lo, min(s_ctx + s_n, max(pos + 1, c.get("prefix", 0))))


def work(case):
    """Visible (query, key) pairs times 4 * 128 operations a head; q, the visible cache and the results once."""
    c, kv_bytes = case, 2 * case["n_kv_heads"] * HEAD_DIM * 2
    if c["op"] == "rope":
        tokens = sum(n for _, n in _lens(c))
        values = tokens * (c["n_heads"] + 2 * c["n_kv_heads"]) * HEAD_DIM
        rotated = tokens * (c["n_heads"] + c["n_kv_heads"]) * c["rotary"]
        return {"bytes": values * ((4 if c["fp32"] else 2) + 2) + tokens * 12, "flops": 3 * rotated}
    pairs = rows = seen = 0
    for ctx, n in _lens(c):
        if c["op"] == "decode":
            ctx, n = ctx - 1, 1  # the new token is the last of the `ctx` cached ones
        first, last = 1 << 60, 0
        for i in range(n):
            lo, hi = _bounds(c, ctx, n, rows + i, ctx + i)
            if hi > lo:
                pairs += hi - lo
                first, last = min(first, lo), max(last, hi)
        rows += n
        seen += max(0, last - first)
    q = rows * c["n_heads"] * HEAD_DIM * 2
    return {"bytes": 2 * q + 4 * rows * c["n_heads"] + seen * kv_bytes, "flops": 4 * HEAD_DIM * c["n_heads"] * pairs}


# ----------------------------------------------------------------- inputs
def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    lens = _lens(c)
    total = [ctx + (n if c["op"] != "decode" else 0) for ctx, n in lens]
    per_seq = -(-max(total) // c["tpb"])
    blocks = c["seqs"] * per_seq + 3
    st = dict(case=c, blocks=blocks, max_len=max(total))
    st["table"] = torch.randperm(blocks, generator=g, device=dev)[:c["seqs"] * per_seq].to(torch.int32).view(c["seqs"], per_seq)
    st["pool"] = torch.randn(blocks, c["tpb"], 2, c["n_kv_heads"], HEAD_DIM, generator=g, device=dev, dtype=torch.bfloat16)
    rows = sum(n for _, n in lens)
    if c["op"] == "rope":
        heads = c["n_heads"] + 2 * c["n_kv_heads"]
        st["qkv"] = torch.randn(rows, heads * HEAD_DIM, generator=g, device=dev,
                                dtype=torch.float32 if c["fp32"] else torch.bfloat16)
        index = torch.cat([torch.arange(ctx, ctx + n, dtype=torch.int32) for ctx, n in lens])
        st["index"] = index.to(dev)
        st["positions"] = (index + c["offset"]).to(dev)
        st["token_seq"] = torch.cat([torch.full((n,), s, dtype=torch.int32) for s, (_, n) in enumerate(lens)]).to(dev)
        st["inv_freq"], st["factor"] = _inv_freq(c)
        st["inv_freq"] = st["inv_freq"].to(dev)
        st["q_out"] = torch.empty(rows, c["n_heads"] * HEAD_DIM, device=dev, dtype=torch.bfloat16)
        return st
    # capped models reach the cap with a few scores: queries of a few times unit size
    st["q"] = 3 * torch.randn(rows, c["n_heads"] * HEAD_DIM, generator=g, device=dev, dtype=torch.bfloat16)
    st["out"] = torch.empty(rows, c["n_heads"] * HEAD_DIM, device=dev, dtype=torch.bfloat16)
    st["lse"] = torch.empty(rows, c["n_heads"], device=dev, dtype=torch.float32)
    st["slopes"] = torch.tensor(_slopes(c), dtype=torch.float32, device=dev) if c["alibi"] else None
    if c["op"] == "decode":
        st["seq_lens"] = _int32([ctx for ctx, _ in lens], dev)
        st["kv_start"] = _int32([(ctx - 1) // c["doc"] * c["doc"] for ctx, _ in lens], dev) if c["doc"] else None
        return st
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    st["q_start"], st["q_pos0"] = _int32(starts, dev), _int32([ctx for ctx, _ in lens], dev)
    st["kv_start"] = st["prefix_lens"] = None
    if c["doc"] or c["empty"]:
        pos = torch.cat([torch.arange(ctx, ctx + n) for ctx, n in lens])
        first = pos // c["doc"] * c["doc"] if c["doc"] else torch.zeros_like(pos)
        if c["empty"]:  # a row that starts behind every cached token sees nothing
            first = torch.where(torch.arange(rows) % c["empty"] == 1, torch.full_like(first, 1 << 30), first)
        st["kv_start"] = first.to(torch.int32).to(dev)
    if c["prefix"]:
        st["prefix_lens"] = _int32([c["prefix"]] * c["seqs"], dev)
    return st


def _inv_freq(c):
    """Rotary frequencies, fp64: wavelengths beyond the trained context of 8192 are stretched, short ones
    kept, those between blended; and the factor on cos and sin that goes with it."""
    f = 5e5 ** (-torch.arange(0, c["rotary"], 2, dtype=torch.float64) / c["rotary"])
    turns = 8192 * f / (2 * math.pi)
    keep = ((turns - 1) / 3).clamp(0, 1)
    return f * keep + f / c["stretch"] * (1 - keep), 0.1 * math.log(c["stretch"]) + 1


# -------------------------------------------------------------- the passes
def run(state):
    if own:
        return _run_own(state)
    return _plain_rope(state) if state["case"]["op"] == "rope" else _plain_attention(state)


def _plain_rope(st):
    c = st["case"]
    H, K, R, T = c["n_heads"], c["n_kv_heads"], c["rotary"], st["qkv"].shape[0]
    x = st["qkv"].view(T, H + 2 * K, HEAD_DIM)
    qk = x[:, :H + K].float()
    angle = st["positions"].double()[:, None] * st["inv_freq"][None, :]
    cos, sin = (angle.cos() * st["factor"]).float()[:, None], (angle.sin() * st["factor"]).float()[:, None]
    if c["interleaved"]:
        a, b = qk[..., 0:R:2], qk[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = qk[..., :R // 2], qk[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    qk = torch.cat([turned, qk[..., R:]], -1).to(torch.bfloat16)
    st["q_out"].view(T, H, HEAD_DIM).copy_(qk[:, :H])
    at = st["index"].long()
    block = st["table"][st["token_seq"].long(), at // c["tpb"]].long()
    st["pool"][block, at % c["tpb"], 0] = qk[:, H:]
    st["pool"][block, at % c["tpb"], 1] = x[:, H + K:].to(torch.bfloat16)
    return {"q": st["q_out"], "pool": st["pool"]}


def _plain_attention(st):
    c = st["case"]
    H, K, S, N = c["n_heads"], c["n_kv_heads"], c["seqs"], st["max_len"]
    G = H // K
    rows = st["q"].shape[0]
    keys = torch.arange(N, device="cuda")
    if c["op"] == "decode":
        L, length = 1, st["seq_lens"].long()
        row = torch.arange(S, device="cuda")[:, None]
        pos = (length - 1)[:, None]
        there = torch.ones(S, 1, dtype=torch.bool, device="cuda")
        ahead = pos + 1
    else:
        L = c["q_len"]
        first, n = st["q_start"][:-1].long(), (st["q_start"][1:] - st["q_start"][:-1]).long()
        off = torch.arange(L, device="cuda")
        there = off[None, :] < n[:, None]
        row = torch.where(there, first[:, None] + off[None, :], first[:, None])
        pos = st["q_pos0"].long()[:, None] + off[None, :]
        length = st["q_pos0"].long() + n
        ahead = pos + 1 if st["prefix_lens"] is None else torch.maximum(pos + 1, st["prefix_lens"].long()[:, None])
    low = torch.zeros_like(pos) if st["kv_start"] is None else st["kv_start"].long()[row]
    if c["window"]:
        low = torch.maximum(low, pos - c["window"] + 1)
    high = torch.minimum(ahead, length[:, None])
    seen = (keys >= low[..., None]) & (keys < high[..., None])  # [S, L, N]
    slot = st["table"].long()[:, keys // c["tpb"]]
    k = st["pool"][slot, keys % c["tpb"], 0].permute(0, 2, 3, 1).float()  # [S, K, 128, N]
    q = st["q"].view(rows, K, G, HEAD_DIM)[row].permute(0, 2, 3, 1, 4).reshape(S, K, G * L, HEAD_DIM).float()
    x = torch.matmul(q, k).mul_(1 / math.sqrt(HEAD_DIM)).view(S, K, G, L, N)
    del k
    if c["cap"]:
        x.div_(c["cap"]).tanh_().mul_(c["cap"])
    if c["alibi"]:
        away = (keys[None, None, :] - pos[..., None]).abs().float()
        x.sub_(st["slopes"].view(1, K, G, 1, 1) * away[:, None, None])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    v = st["pool"][slot, keys % c["tpb"], 1].permute(0, 2, 1, 3).float()  # [S, K, N, 128]
    y = torch.matmul(x.view(S, K, G * L, N), v).view(S, K, G, L, HEAD_DIM)
    y = torch.where(total > 0, y / total, torch.zeros_like(y))
    lse = (top + total.log())[..., 0]  # log 0 = -inf where nothing is seen
    y = y.permute(0, 3, 1, 2, 4).reshape(S, L, H * HEAD_DIM)
    lse = lse.permute(0, 3, 1, 2).reshape(S, L, H)
    st["out"].copy_(y[there])
    st["lse"].copy_(lse[there])
    return {"out": st["out"], "lse": st["lse"]}


def _krt():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kinetic-rt_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from python.kinetic_rt import _lib
    return _lib


def _run_own(st):
    """The framework's calls; the argument structs and workspaces are made once per state, as its decoder keeps them."""
    c, krt = st["case"], _krt()
    H, K = c["n_heads"], c["n_kv_heads"]
    zeros = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")  # noqa: E731
    if c["op"] == "rope":
        if "plan" not in st:
            x = st["qkv"]
            st["plan"] = krt.rope_append_args(
                x[:, :H * HEAD_DIM], x[:, H * HEAD_DIM:(H + K) * HEAD_DIM], x[:, (H + K) * HEAD_DIM:], st["inv_freq"],
                st["positions"], st["token_seq"], st["table"], st["pool"], st["q_out"], H, K, st["blocks"], c["tpb"],
                zeros(krt.rope_append_workspace_bytes()), interleaved=c["interleaved"], factor=st["factor"],
                cache_index=st["index"])
        krt.rope_append(st["plan"])
        return {"q": st["q_out"], "pool": st["pool"]}
    mods = dict(softcap=c["cap"], window=c["window"], alibi_slopes=st["slopes"], kv_start=st["kv_start"], lse=st["lse"])
    if c["op"] == "decode":
        if "plan" not in st:
            ws = zeros(krt.attention_mod_workspace_bytes(c["seqs"], H, K, st["max_len"], c["window"]))
            st["plan"] = krt.attention_mod_args(st["q"], st["pool"], st["table"], st["seq_lens"], st["out"], H, K,
                                                st["blocks"], c["tpb"], st["max_len"], ws, **mods)
        krt.paged_attention_decode_mod(st["plan"])
    else:
        if "plan" not in st:
            ws = zeros(krt.prefill_attention_mod_workspace_bytes(st["q"].shape[0], c["seqs"], H, K, st["max_len"]))
            st["plan"] = krt.prefill_attention_mod_args(st["q"], st["pool"], st["table"], st["q_start"], st["q_pos0"],
                                                        st["out"], H, K, st["blocks"], c["tpb"], st["max_len"], ws,
                                                        prefix_lens=st["prefix_lens"], **mods)
        krt.paged_attention_prefill_mod(st["plan"])
    return {"out": st["out"], "lse": st["lse"]}


# --------------------------------------------------------------- 64 bits
def exact(case, seed):
    c, st = case, prepare(case, seed)
    H, K, B = c["n_heads"], c["n_kv_heads"], c["tpb"]
    table = st["table"].long()
    if c["op"] == "rope":
        T, R = st["qkv"].shape[0], c["rotary"]
        x = st["qkv"].double().view(T, H + 2 * K, HEAD_DIM)
        turn = torch.polar(torch.full((T, R // 2), st["factor"], dtype=torch.float64, device="cuda"),
                           torch.outer(st["positions"].double(), st["inv_freq"]))
        pair = [slice(0, R, 2), slice(1, R, 2)] if c["interleaved"] else [slice(0, R // 2), slice(R // 2, R)]
        z = torch.complex(x[:, :H + K, pair[0]].contiguous(), x[:, :H + K, pair[1]].contiguous()) * turn[:, None]
        x[:, :H + K, pair[0]], x[:, :H + K, pair[1]] = z.real, z.imag
        pool = st["pool"].double().view(-1, 2, K, HEAD_DIM)
        at = st["index"].long()
        slot = table[st["token_seq"].long(), at // B] * B + at % B
        pool[slot, 0], pool[slot, 1] = x[:, H:H + K], x[:, H + K:]
        return {"q": x[:, :H].reshape(T, -1), "pool": pool.view(st["pool"].shape)}
    out = torch.zeros(st["q"].shape[0], K, H // K, HEAD_DIM, dtype=torch.float64, device="cuda")
    lse = torch.full((st["q"].shape[0], K, H // K), -math.inf, dtype=torch.float64, device="cuda")
    slopes = torch.tensor(_slopes(c), dtype=torch.float32, device="cuda").double().view(K, H // K)
    row = 0
    for s, (ctx, n) in enumerate(_lens(c)):
        if c["op"] == "decode":
            ctx, n = ctx - 1, 1
        keys = torch.arange(ctx + n, device="cuda")
        kv = st["pool"].view(-1, 2, K, HEAD_DIM)[table[s, keys // B] * B + keys % B].double()
        for i in range(0, n, 512):
            m = min(512, n - i)
            pos = torch.arange(ctx + i, ctx + i + m, device="cuda")[:, None]
            ok = (keys <= pos) | (keys < c.get("prefix", 0))
            if c["window"]:
                ok &= pos - keys < c["window"]
            if c["doc"]:
                ok &= torch.div(pos, c["doc"], rounding_mode="floor") * c["doc"] <= keys
            if c.get("empty"):
                ok &= (torch.arange(row + i, row + i + m, device="cuda")[:, None] % c["empty"]) != 1
            q = st["q"][row + i:row + i + m].double().view(m, K, H // K, HEAD_DIM)
            w = torch.einsum("mkgd,nkd->kgmn", q, kv[:, 0]) / math.sqrt(HEAD_DIM)
            if c["cap"]:
                w = c["cap"] * torch.tanh(w / c["cap"])
            if c["alibi"]:
                w = w - slopes[:, :, None, None] * (keys - pos).abs().double()
            w = torch.where(ok, w, -math.inf)
            z = torch.logsumexp(w, -1)
            w = torch.where(ok, torch.exp(w - z[..., None]), 0.0)
            out[row + i:row + i + m] = torch.einsum("kgmn,nkd->mkgd", w, kv[:, 1])
            lse[row + i:row + i + m] = z.permute(2, 0, 1)
        row += n
    return {"out": out.reshape(st["q"].shape), "lse": lse.reshape(st["lse"].shape)}
