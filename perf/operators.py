"""What a decoder layer does between its matrix products, as measurable cases: the residual stream with its norms, the paged
8-bit key/value cache, and the attention that reads it.

A case is a dict of plain values; `op` says which operator it is:

  norm       h' = h + s * g * rms(b; w_post), n = rms(h'; w_pre), with rms(x; w) = x / sqrt(mean(x^2) + eps) * (offset + w)
  append     new queries, keys and values of a batch of sequences: an optional rms norm per head, the rotation by position, keys and
             values into the pages of the cache
  attention  the sequences' new queries against their pages, causal, with optional window, softcap and sinks

The cache: pages of `page` tokens; key codes [pages, kv_heads, page, head_dim], value codes [pages, kv_heads, head_dim, page], both
e4m3 bytes, and a power-of-two scale for each page and head.  The scale of a page is the smallest power of two 2^e, -40 <= e <= 60,
with max |x| <= 448 * 2^e over the tokens that were written to it; while a page fills it only grows, and the codes that are there
already are rounded again for the larger scale.

A sequence's length counts the new tokens; the new tokens are its last ones.  Where `own` is false the operators are computed with
elementary torch operations in 32 bits (angles in 64), otherwise by the framework's kernels."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOG2_E = 1.4426950408889634


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # A decode token's residual between two blocks of a 2560-wide model, all in f32 as the matvecs leave it.
        {"op": "norm", "name": "norm_1_row", "rows": 1, "hidden": 2560, "block": "f32", "stream": "f32", "normed": "f32", "gate": "none",
         "post": True},
        # A short ragged prompt in half precision with a gate for every row and channel.
        {"op": "norm", "name": "norm_77_rows_gated", "rows": 77, "hidden": 2880, "block": "f16", "stream": "f16", "normed": "f16", "gate": "rows",
         "post": True},
        # A prefill chunk: f32 products and residual stream, the next product's bf16 activations.
        {"op": "norm", "name": "norm_4096_rows", "rows": 4096, "hidden": 3840, "block": "f32", "stream": "f32", "normed": "bf16",
         "gate": "channels", "post": True},
        # One token of one conversation, queries and keys normed per head.
        {"op": "append", "name": "append_1_token", "sequences": 1, "new_lo": 1, "new_hi": 1, "len_lo": 1000, "len_hi": 1000, "page": 64,
         "q_heads": 8, "kv_heads": 4, "head_dim": 256, "rot": 256, "type": "f32", "norm": True, "interleaved": False, "base": 1e6, "far": 0},
        # A decode step of 64 conversations.
        {"op": "append", "name": "append_64_sequences", "sequences": 64, "new_lo": 1, "new_hi": 1, "len_lo": 1, "len_hi": 2048, "page": 64,
         "q_heads": 64, "kv_heads": 8, "head_dim": 64, "rot": 64, "type": "bf16", "norm": False, "interleaved": False, "base": 150000.0, "far": 0},
        # Ragged prompts, none of them ending with a page.
        {"op": "append", "name": "append_prompts", "sequences": 5, "new_lo": 777, "new_hi": 3001, "len_lo": 777, "len_hi": 3501, "page": 64,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "rot": 128, "type": "f32", "norm": True, "interleaved": True, "base": 10000.0, "far": 0},
        # Attention of one token over a short context.
        {"op": "attention", "name": "attention_1_token_1000", "sequences": 1, "new_lo": 1, "new_hi": 1, "len_lo": 1000, "len_hi": 1000, "page": 64,
         "q_heads": 8, "kv_heads": 4, "head_dim": 256, "type": "f32", "out": "f32", "window": 0, "softcap": 0.0, "sinks": False},
        # ... and over a very long one.
        {"op": "attention", "name": "attention_1_token_131072", "sequences": 1, "new_lo": 1, "new_hi": 1, "len_lo": 131072, "len_hi": 131072,
         "page": 64, "q_heads": 16, "kv_heads": 8, "head_dim": 256, "type": "f32", "out": "f32", "window": 0, "softcap": 0.0, "sinks": False},
        # A decode step of 64 conversations of very different lengths, with a sink for each head.
        {"op": "attention", "name": "attention_64_sequences", "sequences": 64, "new_lo": 1, "new_hi": 1, "len_lo": 100, "len_hi": 8192, "page": 64,
         "q_heads": 64, "kv_heads": 8, "head_dim": 64, "type": "bf16", "out": "bf16", "window": 0, "softcap": 0.0, "sinks": True},
        # A prompt through a layer with a sliding window, f32 in and out.
        {"op": "attention", "name": "attention_prompt_2048_window", "sequences": 1, "new_lo": 2048, "new_hi": 2048, "len_lo": 2048, "len_hi": 2048,
         "page": 64, "q_heads": 8, "kv_heads": 4, "head_dim": 256, "type": "f32", "out": "f32", "window": 1024, "softcap": 0.0, "sinks": False},
        # A long prompt through a full layer.
        {"op": "attention", "name": "attention_prompt_8192", "sequences": 1, "new_lo": 8192, "new_hi": 8192, "len_lo": 8192, "len_hi": 8192,
         "page": 64, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "type": "bf16", "out": "bf16", "window": 0, "softcap": 0.0, "sinks": False},
        # Single tokens and prompt chunks together, small pages, capped scores.
        {"op": "attention", "name": "attention_mixed", "sequences": 12, "new_lo": 1, "new_hi": 301, "len_lo": 400, "len_hi": 16001, "page": 16,
         "q_heads": 16, "kv_heads": 8, "head_dim": 128, "type": "f16", "out": "f16", "window": 0, "softcap": 50.0, "sinks": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _one(rng):
    op = rng.choice(["norm", "append", "attention", "attention"])
    if op == "norm":
        hidden = _log_int(rng, 64, 16384)
        block = rng.choice(["f32", "bf16", "f16"])
        return {"op": op, "rows": _log_int(rng, 1, 8192), "hidden": hidden if rng.random() < 0.25 else max(64, hidden // 64 * 64), "block": block,
                "stream": rng.choice(["f32", block]), "normed": rng.choice(["f32", "bf16", block]), "gate": rng.choice(["none", "channels", "rows"]),
                "post": rng.random() < 0.7}
    kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 96, 128, 128, 192, 256])
    decode = rng.random() < 0.5
    new_hi = 1 if decode else _log_int(rng, 2, 8192)
    new_lo = 1 if decode else max(1, int(new_hi * rng.choice([0.0, 0.1, 0.5, 1.0])))
    len_hi = max(new_hi, _log_int(rng, 1, 131072 if op == "attention" else 8192))
    c = {"op": op, "sequences": _log_int(rng, 1, 128), "new_lo": new_lo, "new_hi": new_hi,
         "len_lo": max(new_lo, int(len_hi * rng.choice([0.01, 0.3, 1.0]))), "len_hi": len_hi, "page": rng.choice([16, 32, 64, 64, 128]),
         "q_heads": kv_heads * rng.choice([1, 2, 4, 5, 8]), "kv_heads": kv_heads, "head_dim": head_dim, "type": rng.choice(["f32", "bf16", "f16"])}
    if op == "append":
        return {**c, "rot": rng.choice([head_dim, head_dim, head_dim // 2]), "norm": rng.random() < 0.5, "interleaved": rng.random() < 0.3,
                "base": rng.choice([10000.0, 150000.0, 1e6]), "far": rng.choice([0, 0, 1])}
    return {**c, "out": rng.choice([c["type"], c["type"], "bf16"]), "window": rng.choice([0, 0, 128, 1024]), "softcap": rng.choice([0.0, 0.0, 50.0]),
            "sinks": rng.random() < 0.3}


def draw(rng):
    every = listed()
    big = {op: {k: max(work(c)[k] for c in every if c["op"] == op) for k in ("bytes", "flops")} for op in ("norm", "append", "attention")}
    while True:
        c = _one(rng)
        w = work(c)
        if w["bytes"] > big[c["op"]]["bytes"] or w["flops"] > big[c["op"]]["flops"]:
            continue
        if c["op"] != "norm":
            padded = c["sequences"] * c["len_hi"]  # what a batch in one rectangle holds
            if padded * c["kv_heads"] * c["head_dim"] > 5e8 or (c["op"] == "attention" and padded * c["new_hi"] * c["q_heads"] > 2.2e9):
                continue
        return c


# ---- sizes of a batch -----------------------------------------------------------------------------------------------

def _sizes(c):
    """(new tokens, length) of each sequence: spread between the case's bounds, the longest first of all."""
    n = c["sequences"]
    spread = [(i * 0.6180339887498949) % 1.0 for i in range(n)]
    new = [max(c["new_lo"], int(round(c["new_hi"] * (c["new_lo"] / c["new_hi"]) ** f))) for f in spread]
    far = [(i * 0.7548776662466927) % 1.0 for i in range(n)]
    return [(t, max(t, int(round(c["len_hi"] * (c["len_lo"] / c["len_hi"]) ** f)))) for t, f in zip(new, far)]


def _width(c):
    return max(-(-t // c["page"]) for _, t in _sizes(c))


_ITEM = {"f32": 4, "bf16": 2, "f16": 2}


def _pairs(new, length, window):
    """Visible (query, key) pairs of a sequence's new tokens, and the keys that at least one of them sees."""
    if not window:
        return new * length - new * (new - 1) // 2, length
    first = length - new  # position of the first new token: it sees min(first + 1, window) keys
    short = max(0, min(new, window - 1 - first))  # tokens that see fewer than `window`
    pairs = short * (first + 1) + short * (short - 1) // 2 + (new - short) * window
    return pairs, min(length, window + new - 1)


def work(case):
    c = case
    if c["op"] == "norm":
        n = c["rows"] * c["hidden"]
        moved = n * (_ITEM[c["block"]] + 2 * _ITEM[c["stream"]] + _ITEM[c["normed"]]) + 4 * c["hidden"] * (1 + c["post"])
        moved += {"none": 0, "channels": 4 * c["hidden"], "rows": 4 * n}[c["gate"]]
        return {"bytes": moved, "flops": 8 * n}
    d, item = c["head_dim"], _ITEM[c["type"]]
    sizes = _sizes(c)
    tokens = sum(t for t, _ in sizes)
    tables = 4 * sum(-(-t // c["page"]) for _, t in sizes) + 8 * c["sequences"]
    if c["op"] == "append":
        pages = sum(-(-length // c["page"]) - (length - new) // c["page"] for new, length in sizes)
        return {"bytes": tokens * d * (2 * c["q_heads"] * item + 2 * c["kv_heads"] * (item + 1)) + 16 * pages * c["kv_heads"] + tables,
                "flops": tokens * d * 6 * (c["q_heads"] + c["kv_heads"])}
    seen = [_pairs(new, length, c["window"]) for new, length in sizes]
    keys = sum(k for _, k in seen)
    return {"bytes": tokens * c["q_heads"] * d * (item + _ITEM[c["out"]]) + keys * c["kv_heads"] * (2 * d + 8 / c["page"]) + tables,
            "flops": 4 * d * c["q_heads"] * sum(p for p, _ in seen)}


# ---- inputs ---------------------------------------------------------------------------------------------------------

class _State:
    pass


def _encode(x, dims):
    """e4m3 codes of x and the power-of-two scales over `dims`."""
    amax = x.abs().amax(dims, keepdim=True)
    e = torch.ceil(torch.log2((amax.double() / 448).clamp(min=2.0 ** -40)))
    scale = torch.exp2(e).float()
    return (x / scale).to(torch.float8_e4m3fn).view(torch.uint8), scale.flatten(1)


def _values(gen, shape, sigma=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * sigma


def _cache(s, c, gen):
    sizes = _sizes(c)
    need = sum(-(-t // c["page"]) for _, t in sizes)
    s.pages = need + 3
    h, d, p = c["kv_heads"], c["head_dim"], c["page"]
    # a few channels of the keys are much larger than the rest, and so are a few tokens of the values
    loud = 1 + 6 * (torch.rand((h, 1, d), generator=gen, device="cuda") < 0.03)
    s.k_codes, s.k_scales = _encode(_values(gen, (s.pages, h, p, d)) * loud, (2, 3))
    tall = 1 + 3 * (torch.rand((s.pages, h, 1, p), generator=gen, device="cuda") < 0.02)
    s.v_codes, s.v_scales = _encode(_values(gen, (s.pages, h, d, p)) * tall, (2, 3))
    order = torch.randperm(s.pages, generator=gen, device="cuda")[:need].int().cpu()
    s.width = _width(c)
    table, at = torch.full((len(sizes), s.width), -1, dtype=torch.int32), 0
    for b, (_, length) in enumerate(sizes):
        n = -(-length // p)
        table[b, :n] = order[at: at + n]
        at += n
    s.table = table.cuda()
    s.kv_len = torch.tensor([t for _, t in sizes], dtype=torch.int32, device="cuda")
    s.q_start = torch.tensor([0] + [t for t, _ in sizes], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    s.tokens = sum(t for t, _ in sizes)
    s.new_max = max(t for t, _ in sizes)


def prepare(case, seed):
    c, s = case, _State()
    s.c = c
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "norm":
        n = (c["rows"], c["hidden"])
        s.h = _values(gen, n, 4.0).to(TYPES[c["stream"]])
        s.b = _values(gen, n, 0.7).to(TYPES[c["block"]])
        s.gate = {"none": None, "channels": lambda: 1 + _values(gen, n[1:], 0.2), "rows": lambda: _values(gen, n)}[c["gate"]]
        s.gate = s.gate and s.gate()
        s.post = _values(gen, n[1:], 0.1) if c["post"] else None
        s.pre = _values(gen, n[1:], 0.1)
        s.scale, s.offset, s.eps = 0.75, 1.0, 1e-6
        s.h_out, s.normed = torch.empty_like(s.h), torch.empty(n, dtype=TYPES[c["normed"]], device="cuda")
        return s
    _cache(s, c, gen)
    hq, h, d, t = c["q_heads"], c["kv_heads"], c["head_dim"], TYPES[c["type"]]
    if c["op"] == "append":
        # queries, keys and values as one product leaves them, a row for each token
        s.qkv = _values(gen, (s.tokens, (hq + 2 * h) * d)).to(t)
        s.q_out = torch.empty((s.tokens, hq, d), dtype=t, device="cuda")
        s.inv_freq = (c["base"] ** (-torch.arange(c["rot"] // 2, dtype=torch.float64) * 2 / c["rot"])).float().cuda()
        if c["far"]:  # positions that no cache holds from the start: the frequencies are what such a context's are multiplied to
            s.inv_freq = s.inv_freq * 64
        s.q_norm = 1 + _values(gen, (d,), 0.1) if c["norm"] else None
        s.k_norm = 1 + _values(gen, (d,), 0.1) if c["norm"] else None
        return s
    s.q = _values(gen, (s.tokens, hq, d), 1.5).to(t)
    s.out = torch.empty((s.tokens, hq, d), dtype=TYPES[c["out"]], device="cuda")
    s.sinks = _values(gen, (hq,)) if c["sinks"] else None
    s.scale = d ** -0.5
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------

_backend = []


def _hip():
    import larql_amd
    if not _backend:
        _backend.append(larql_amd.HipBackend())
    return larql_amd, _backend[0]


def _at(t):
    return None if t is None else t.data_ptr()


def _kv(s, hip):
    c = s.c
    return (hip.KvCache(k_codes=_at(s.k_codes), v_codes=_at(s.v_codes), k_scales=_at(s.k_scales), v_scales=_at(s.v_scales), num_pages=s.pages,
                        kv_heads=c["kv_heads"], head_dim=c["head_dim"], page_tokens=c["page"]),
            hip.KvBatch(kv_len=_at(s.kv_len), block_table=_at(s.table), q_start=_at(s.q_start), sequences=c["sequences"], table_width=s.width,
                        tokens=s.tokens, max_new_tokens=s.new_max))


def _own_norm(s):
    hip, be = _hip()
    if not hasattr(s, "args"):
        c, fmt = s.c, {"f32": hip.FMT_F32, "bf16": hip.FMT_BF16, "f16": hip.FMT_F16}
        s.args = hip.ResidualNorm(rows=c["rows"], hidden=c["hidden"], block=_at(s.b), block_stride=c["hidden"], block_format=fmt[c["block"]],
                                  residual=_at(s.h), residual_stride=c["hidden"], residual_out=_at(s.h_out), residual_out_stride=c["hidden"],
                                  residual_format=fmt[c["stream"]], normed=_at(s.normed), normed_stride=c["hidden"],
                                  normed_format=fmt[c["normed"]], gate=_at(s.gate), gate_stride=c["hidden"] if c["gate"] == "rows" else 0,
                                  post_weight=_at(s.post), pre_weight=_at(s.pre), residual_scale=s.scale, norm_offset=s.offset, eps=s.eps)
    assert be.dev_residual_norm(s.args), be.last_error()
    return s.h_out, s.normed


def _own_append(s):
    hip, be = _hip()
    c = s.c
    if not hasattr(s, "args"):
        fmt = {"f32": hip.FMT_F32, "bf16": hip.FMT_BF16, "f16": hip.FMT_F16}
        s.cache, s.batch = _kv(s, hip)
        hq, h, d = c["q_heads"], c["kv_heads"], c["head_dim"]
        row, item = s.qkv.shape[1], s.qkv.element_size()
        s.args = hip.KvAppend(format=fmt[c["type"]], q_heads=hq, q=_at(s.qkv), q_stride=row, q_out=_at(s.q_out), q_out_stride=hq * d,
                              k=_at(s.qkv) + hq * d * item, k_stride=row, v=_at(s.qkv) + (hq + h) * d * item, v_stride=row,
                              inv_freq=_at(s.inv_freq), rot_dim=c["rot"], interleaved=int(c["interleaved"]), rope_scale=1.0, q_norm=_at(s.q_norm),
                              k_norm=_at(s.k_norm), norm_offset=0.0, norm_eps=1e-6)
    assert be.dev_kv_append(s.cache, s.batch, s.args), be.last_error()
    return {"q": s.q_out, "k": s.k_codes.view(torch.float8_e4m3fn), "v": s.v_codes.view(torch.float8_e4m3fn), "k_scales": s.k_scales,
            "v_scales": s.v_scales}


def _own_attention(s):
    hip, be = _hip()
    c = s.c
    if not hasattr(s, "args"):
        fmt = {"f32": hip.FMT_F32, "bf16": hip.FMT_BF16, "f16": hip.FMT_F16}
        s.cache, s.batch = _kv(s, hip)
        row = c["q_heads"] * c["head_dim"]
        s.args = hip.Attention(q=_at(s.q), q_stride=row, q_format=fmt[c["type"]], out=_at(s.out), out_stride=row, out_format=fmt[c["out"]],
                               q_heads=c["q_heads"], causal=1, window=c["window"], scale=s.scale, softcap=c["softcap"], sinks=_at(s.sinks))
        s.workspace = torch.empty(be.attention_workspace_bytes(s.cache, s.batch, s.args), dtype=torch.uint8, device="cuda")
    assert be.dev_attention(s.cache, s.batch, s.args, _at(s.workspace), s.workspace.numel()), be.last_error()
    return s.out


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _rms(x, w, offset, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * (offset + w)


def _plain_norm(s):
    b = s.b.float()
    if s.post is not None:
        b = _rms(b, s.post, s.offset, s.eps)
    if s.gate is not None:
        b = b * s.gate
    h = s.h.float() + s.scale * b
    return h.to(s.h_out.dtype), _rms(h, s.pre, s.offset, s.eps).to(s.normed.dtype)


def _new_tokens(s):
    """(sequence, position) of every new token."""
    token = torch.arange(s.tokens, device="cuda")
    b = torch.bucketize(token, s.q_start[1:].long(), right=True)
    return b, s.kv_len.long()[b] - s.q_start.long()[b + 1] + token


def _turn(x, angle, interleaved):
    """x [tokens, heads, d] with the first 2 * angle.shape[1] channels rotated."""
    half = angle.shape[1]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turned, rest = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _stored(s, codes, scales, x, b, pos, tokens_last):
    """x [tokens, heads, d] into codes / scales (in place).  tokens_last: the codes of a page are [d, page] instead of [page, d]."""
    p, w = s.c["page"], s.width
    rows, heads = s.table.shape[0] * w, x.shape[1]
    old = (s.kv_len - (s.q_start[1:] - s.q_start[:-1])).long()  # tokens that were there before
    page_at = torch.arange(w, device="cuda") * p
    kept = (old[:, None] - page_at).clamp(0, p).reshape(-1)  # of each entry of the table
    key = b * w + pos // p
    amax = torch.zeros((rows, heads), device="cuda").index_reduce_(0, key, x.abs().amax(-1), "amax")
    touched = torch.zeros(rows, dtype=torch.bool, device="cuda").index_fill_(0, key, True)
    page = s.table.long().reshape(-1)[touched]
    kept = kept[touched][:, None]
    new = torch.exp2(torch.ceil(torch.log2((amax[touched].double() / 448).clamp(min=2.0 ** -40)))).float()
    before = scales[page]
    after = torch.where(kept > 0, torch.maximum(before, new), new)
    values = codes[page].view(torch.float8_e4m3fn).float()
    slot = torch.arange(p, device="cuda")
    there = (slot < kept)[:, None, None, :] if tokens_last else (slot < kept)[:, None, :, None]
    again = (values * (before / after)[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[page] = torch.where(there, again, codes[page])
    scales[page] = after
    at = s.table.long()[b, pos // p]
    code = (x / scales[at][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    if tokens_last:
        codes.transpose(2, 3)[at, :, pos % p] = code
    else:
        codes[at, :, pos % p] = code


def _plain_append(s):
    c = s.c
    hq, h, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    x = s.qkv.float().view(s.tokens, hq + 2 * h, d)
    q, k, v = x[:, :hq], x[:, hq: hq + h], x[:, hq + h:]
    if c["norm"]:
        q, k = _rms(q, s.q_norm, 0.0, 1e-6), _rms(k, s.k_norm, 0.0, 1e-6)
    b, pos = _new_tokens(s)
    angle = pos.double()[:, None] * s.inv_freq.double()
    q, k = _turn(q, angle, c["interleaved"]), _turn(k, angle, c["interleaved"])
    _stored(s, s.k_codes, s.k_scales, k, b, pos, False)
    _stored(s, s.v_codes, s.v_scales, v, b, pos, True)
    return {"q": q.to(s.q_out.dtype), "k": s.k_codes.view(torch.float8_e4m3fn), "v": s.v_codes.view(torch.float8_e4m3fn), "k_scales": s.k_scales,
            "v_scales": s.v_scales}


def _rectangle(s, dtype):
    """Keys [b, h, d, length] and values [b, h, length, d] of the whole batch, and the padded new tokens' rows and positions."""
    c = s.c
    h, d, p, w = c["kv_heads"], c["head_dim"], c["page"], s.width
    n = c["sequences"]
    page = s.table.long().clamp(min=0)
    k = (s.k_codes[page].view(torch.float8_e4m3fn).to(dtype) * s.k_scales[page].to(dtype)[..., None, None]).permute(0, 2, 4, 1, 3).reshape(n, h, d, w * p)
    v = (s.v_codes[page].view(torch.float8_e4m3fn).to(dtype) * s.v_scales[page].to(dtype)[..., None, None]).permute(0, 2, 1, 4, 3).reshape(n, h, w * p, d)
    v = v * (torch.arange(w * p, device="cuda") < s.kv_len[:, None])[:, None, :, None]
    new = (s.q_start[1:] - s.q_start[:-1]).long()[:, None]
    t = torch.arange(s.new_max, device="cuda")[None]
    live = t < new
    row = torch.where(live, s.q_start[:-1].long()[:, None] + t, 0)
    pos = s.kv_len.long()[:, None] - new + t
    return k, v, row, pos, live


def _plain_attention(s):
    c = s.c
    hq, h, d, n = c["q_heads"], c["kv_heads"], c["head_dim"], c["sequences"]
    g = hq // h
    k, v, row, pos, live = _rectangle(s, torch.float32)
    q = s.q.float()[row].view(n, s.new_max, h, g, d).permute(0, 2, 3, 1, 4).reshape(n, h, g * s.new_max, d)
    x = torch.matmul(q * s.scale, k)
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    key = torch.arange(k.shape[-1], device="cuda")
    seen = (key <= pos[..., None]) & live[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    x = x.view(n, h, g, s.new_max, -1).masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True)
    if s.sinks is not None:
        total = total + torch.exp(s.sinks.view(1, h, g, 1, 1) - m)
    o = torch.matmul(x.view(n, h, g * s.new_max, -1), v).view(n, h, g, s.new_max, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s.new_max, hq, d)
    return o[live].to(s.out.dtype)


def run(state):
    op = state.c["op"]
    if own:
        return {"norm": _own_norm, "append": _own_append, "attention": _own_attention}[op](state)
    return {"norm": _plain_norm, "append": _plain_append, "attention": _plain_attention}[op](state)


# ---- the definitions, in 64 bits ------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attention": _exact_attention}[case["op"]](s)


def _exact_norm(s):
    def rms(x, w):
        return x / ((x ** 2).sum(1, keepdim=True) / x.shape[1] + s.eps).sqrt() * (w.double() + s.offset)

    b = s.b.double()
    b = b if s.post is None else rms(b, s.post)
    b = b if s.gate is None else b * s.gate.double()
    h = s.h.double() + s.scale * b
    return h, rms(h, s.pre)


def _exact_append(s):
    """Codes as the numbers that they round: value / scale."""
    c = s.c
    hq, h, d, p = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    x = s.qkv.double().reshape(s.tokens, hq + 2 * h, d)
    pos = torch.cat([torch.arange(length - new, length) for new, length in _sizes(c)]).cuda()
    half = c["rot"] // 2
    angle = torch.outer(pos.double(), s.inv_freq.double())
    z = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(y, w):
        if w is not None:
            y = y / ((y ** 2).sum(2, keepdim=True) / d + 1e-6).sqrt() * w.double()
        y = y.clone()
        lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if c["interleaved"] else (slice(0, half), slice(half, 2 * half))
        r = torch.complex(y[..., lo], y[..., hi]) * z
        y[..., lo], y[..., hi] = r.real, r.imag
        return y

    got = {"q": turned(x[:, :hq], s.q_norm)}
    table, at = s.table.cpu().tolist(), 0
    parts = {"k": (s.k_codes, s.k_scales, turned(x[:, hq: hq + h], s.k_norm)), "v": (s.v_codes, s.v_scales, x[:, hq + h:])}
    for name, (codes, scales, values) in parts.items():
        codes, scales, at = codes.view(torch.float8_e4m3fn).double(), scales.double(), 0
        codes = codes.transpose(2, 3).contiguous() if name == "v" else codes
        for b, (new, length) in enumerate(_sizes(c)):
            first = length - new
            for j in range(first // p, -(-length // p)):
                lo, hi = max(first, j * p), min(length, j * p + p)
                y, page = values[at + lo - first: at + hi - first].transpose(0, 1), table[b][j]  # [heads, tokens, d]
                e = torch.ceil(torch.log2(y.abs().amax((1, 2)) / 448).clamp(min=-40.0))
                scale = torch.exp2(e)
                if lo > j * p:
                    scale = torch.maximum(scale, scales[page])
                    codes[page, :, : lo - j * p] *= (scales[page] / scale)[:, None, None]
                codes[page, :, lo - j * p: hi - j * p] = y / scale[:, None, None]
                scales[page] = scale
            at += new
        got[name], got[name + "_scales"] = codes.transpose(2, 3) if name == "v" else codes, scales
    return got


def _exact_attention(s):
    c = s.c
    hq, h, d, p = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    g, at = hq // h, 0
    out = torch.zeros((s.tokens, hq, d), dtype=torch.float64, device="cuda")
    k_all, v_all = s.k_codes.view(torch.float8_e4m3fn), s.v_codes.view(torch.float8_e4m3fn)
    for b, (new, length) in enumerate(_sizes(c)):
        page = s.table[b, : -(-length // p)].long()
        pos = torch.arange(length - new, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None]
        hidden = key > pos
        if c["window"]:
            hidden = hidden | (key <= pos - c["window"])
        for i in range(h):
            k = (k_all[page, i].double() * s.k_scales[page, i].double()[:, None, None]).reshape(-1, d)[:length].t().contiguous()
            v = (v_all[page, i].double() * s.v_scales[page, i].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:length]
            for j in range(i * g, i * g + g):
                x = s.q[at: at + new, j].double() @ k * s.scale
                if c["softcap"]:
                    x = torch.tanh(x / c["softcap"]) * c["softcap"]
                x = x.masked_fill(hidden, -math.inf)
                if s.sinks is not None:
                    x = torch.cat((x, s.sinks[j].double().expand(new, 1)), 1)
                x = torch.softmax(x, 1)[:, :length]
                out[at: at + new, j] = x @ v
        at += new
    return out
