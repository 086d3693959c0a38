"""Residual and norms, the paged 8-bit cache and its attention (larql_hip_dev_residual_norm, _kv_append, _attention) against
plain implementations in 64 bits.

Bounds count roundings.  u = 2^-24 is half a step of f32; a result type rounds by HALF[type] of the value at most."""
import ctypes
import math

import numpy as np
import pytest
import torch

import larql_amd as hip
from larql_amd import _lib as L

gpu = pytest.mark.gpu
U = 2.0 ** -24
FMT = {"f32": hip.FMT_F32, "bf16": hip.FMT_BF16, "f16": hip.FMT_F16}
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {t: torch.finfo(TYPE[t]).eps / 2 for t in TYPE}
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}  # below a type's smallest normal number half a step is absolute
ITEM = {"f32": 4, "bf16": 2, "f16": 2}


def raw(x, t):
    """x as the bytes of type t (numpy), and the values that those stand for in 64 bits."""
    y = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(TYPE[t])
    b = y.view(torch.int32 if t == "f32" else torch.int16).numpy()
    return b, y.double().numpy()


def values(b, t):
    return torch.from_numpy(np.ascontiguousarray(b)).view(TYPE[t]).double().numpy()


def e4m3(b):
    return torch.from_numpy(np.ascontiguousarray(b)).view(torch.float8_e4m3fn).double().numpy()


def close(got, want, bound, what=""):
    bad = ~(np.abs(got - want) <= bound) & ~(np.isnan(got) & np.isnan(want))
    assert not bad.any(), (what, int(bad.sum()), bad.size, got[bad][:4], want[bad][:4], np.broadcast_to(bound, bad.shape)[bad][:4])


class Dev:
    """Device buffers of one test."""

    def __init__(self, be):
        self.be = be

    def put(self, a):
        return self.be.to_device(np.ascontiguousarray(a))

    def get(self, p, like):
        return self.be.d2h(p, like.shape, like.dtype)


# ---- residual and norms --------------------------------------------------------------------------------------------

def ref_rms(x, w, offset, eps):
    return x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * (offset + w if w is not None else 1.0)


def norm_case(be, rows, hidden, block="f32", stream="f32", normed="f32", gate="none", post=True, pre=True, pad=0, shift=0, with_block=True,
              want_h=True, want_n=True, in_place=False, scale=0.75, offset=1.0, eps=1e-6, spoil=None):
    rng = np.random.default_rng(rows * 7 + hidden)
    d = Dev(be)
    wide = hidden + pad

    def strided(sigma, t):
        x = (rng.standard_normal((rows, wide)) * sigma).astype(np.float32)
        if spoil is not None and sigma == 4.0:
            x[spoil] = np.nan
        bits, v = raw(x, t)
        flat = np.concatenate([np.zeros(shift, bits.dtype), bits.reshape(-1)])
        return flat, d.put(flat) + shift * ITEM[t], v[:, :hidden]

    bits_b, p_b, b = strided(0.7, block)
    bits_h, p_h, h = strided(4.0, stream)
    g = rng.standard_normal((rows, wide) if gate == "rows" else wide).astype(np.float32)
    w_post, w_pre = (rng.standard_normal(hidden).astype(np.float32) * 0.1 for _ in range(2))
    mark = {"f32": np.int32(0x40490FDB), "bf16": np.int16(0x4049), "f16": np.int16(0x4248)}
    out_h = np.full(rows * wide + shift, mark[stream])
    out_n = np.full(rows * wide + shift, mark[normed])
    p_oh = p_h if in_place else d.put(out_h) + shift * ITEM[stream]
    p_on = d.put(out_n) + shift * ITEM[normed]
    args = hip.ResidualNorm(rows=rows, hidden=hidden, block=p_b if with_block else None, block_stride=wide, block_format=FMT[block],
                            residual_format=FMT[stream], residual=p_h, residual_stride=wide, residual_out=p_oh if want_h else None,
                            residual_out_stride=wide, normed=p_on if want_n else None, normed_stride=wide, normed_format=FMT[normed],
                            residual_scale=scale, gate=d.put(g) if gate != "none" else None, gate_stride=wide if gate == "rows" else 0,
                            post_weight=d.put(w_post) if post else None, pre_weight=d.put(w_pre) if pre else None, norm_offset=offset, eps=eps)
    assert be.dev_residual_norm(args), be.last_error()
    be.synchronize()
    add = np.zeros_like(h)
    if with_block:
        add = ref_rms(b, w_post.astype(np.float64), offset, eps) if post else b
        add = scale * add * (1.0 if gate == "none" else g[..., :hidden].astype(np.float64))
    want = h + add
    # products of 32-bit numbers, a sum of squares (chains of at most 32 and a tree of 16: positive terms), root and quotient
    err_h = 64 * U * (np.abs(h) + np.abs(add))
    rows_bad = [] if spoil is None else [spoil]
    if want_h:
        bits = be.d2h(p_oh - shift * ITEM[stream], out_h.shape, out_h.dtype)
        got = values(bits[shift:], stream).reshape(rows, wide)
        close(got[:, :hidden], want, err_h + HALF[stream] * np.abs(want) + TINY[stream], "h")
        if pad and not in_place:
            assert (bits[shift:].reshape(rows, wide)[:, hidden:] == mark[stream]).all() and (bits[:shift] == mark[stream]).all()
    if want_n:
        n = ref_rms(want, w_pre.astype(np.float64) if pre else None, offset, eps)
        r = np.abs(n) / np.maximum(np.abs(want), 1e-30)
        bits = be.d2h(p_on - shift * ITEM[normed], out_n.shape, out_n.dtype)
        got = values(bits[shift:], normed).reshape(rows, wide)
        close(got[:, :hidden], n, r * err_h + 64 * U * np.abs(n) + HALF[normed] * np.abs(n) + TINY[normed], "n")
        for i in rows_bad:
            assert np.isnan(got[i, :hidden]).all()
        if pad:
            assert (bits[shift:].reshape(rows, wide)[:, hidden:] == mark[normed]).all()


@gpu
@pytest.mark.parametrize("hidden", [1, 7, 8, 63, 64, 65, 511, 512, 520, 1023, 1024, 2048, 2560, 2880, 4097, 8192, 10240, 16384, 32760, 32768])
@pytest.mark.parametrize("rows", [1, 5])
def test_norm_sizes(be, rows, hidden):
    norm_case(be, rows, hidden)


@gpu
@pytest.mark.parametrize("block,stream,normed", [("f32", "f32", "bf16"), ("bf16", "bf16", "bf16"), ("f16", "f32", "f16"), ("f32", "bf16", "f32"),
                                                 ("bf16", "f16", "f32")])
@pytest.mark.parametrize("gate", ["none", "channels", "rows"])
@pytest.mark.parametrize("hidden", [200, 333, 2880])
def test_norm_types_and_gates(be, block, stream, normed, gate, hidden):
    norm_case(be, 9, hidden, block, stream, normed, gate)


@gpu
@pytest.mark.parametrize("how", [{"with_block": False}, {"post": False}, {"pre": False}, {"want_h": False}, {"want_n": False}, {"in_place": True},
                                 {"post": False, "gate": "rows", "scale": -1.5}, {"offset": 0.0, "eps": 1e-2}, {"pad": 8}, {"pad": 3},
                                 {"shift": 1}, {"pad": 5, "shift": 3, "gate": "rows"}, {"in_place": True, "pad": 8, "gate": "channels"}])
@pytest.mark.parametrize("stream", ["f32", "bf16"])
def test_norm_parts_strides_and_alignment(be, how, stream):
    norm_case(be, 6, 640, "f32", stream, "bf16", **how)


@gpu
def test_norm_keeps_a_bad_row_to_itself(be):
    norm_case(be, 9, 448, spoil=4)
    norm_case(be, 9, 4480, spoil=0)


@gpu
def test_norm_of_zero_rows_and_many_rows(be):
    assert be.dev_residual_norm(hip.ResidualNorm(rows=0, hidden=64))
    assert be.dev_residual_norm(hip.ResidualNorm(rows=64, hidden=0))
    norm_case(be, 3000, 129)
    norm_case(be, 2049, 1032, "bf16", "f32", "bf16")


# ---- the cache -----------------------------------------------------------------------------------------------------

class Cache:
    """A cache in host memory in the documented layout, with random codes everywhere, and its sequences' pages in random order."""

    def __init__(self, rng, seqs, kv_heads, head_dim, page, width_more=1, spare=2, sigma=1.0):
        self.h, self.d, self.p, self.seqs = kv_heads, head_dim, page, seqs
        need = [-(-n // page) for n in (max(length, 0) for _, length in seqs)]
        self.pages = sum(need) + spare
        self.width = max(need + [1]) + width_more
        self.k, self.ks = self.encoded(rng, (self.pages, kv_heads, page, head_dim), sigma)
        self.v, self.vs = self.encoded(rng, (self.pages, kv_heads, head_dim, page), sigma)
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(seqs), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at: at + n]
            at += n
        self.kv_len = np.array([length for _, length in seqs], np.int32)
        self.q_start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.tokens = int(self.q_start[-1])
        self.max_new = max([n for n, _ in seqs] + [0])

    @staticmethod
    def encoded(rng, shape, sigma):
        x = (rng.standard_normal(shape) * sigma * np.exp2(rng.integers(-2, 3, shape[:2]))[..., None, None]).astype(np.float32)
        e = exponent(np.abs(x).max((2, 3)))
        codes = torch.from_numpy((x / np.exp2(e)[..., None, None]).astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        return codes.copy(), np.exp2(e).astype(np.float32)

    def upload(self, be):
        d = Dev(be)
        self.dev = {n: d.put(getattr(self, n)) for n in ("k", "v", "ks", "vs", "table", "kv_len", "q_start")}
        cache = hip.KvCache(k_codes=self.dev["k"], v_codes=self.dev["v"], k_scales=self.dev["ks"], v_scales=self.dev["vs"], num_pages=self.pages,
                            kv_heads=self.h, head_dim=self.d, page_tokens=self.p)
        batch = hip.KvBatch(kv_len=self.dev["kv_len"], block_table=self.dev["table"], q_start=self.dev["q_start"], sequences=len(self.seqs),
                            table_width=self.width, tokens=self.tokens, max_new_tokens=self.max_new)
        return cache, batch

    def download(self, be):
        return {n: be.d2h(self.dev[n], getattr(self, n).shape, getattr(self, n).dtype) for n in ("k", "v", "ks", "vs")}

    def keys_values(self, s, length):
        """[kv_heads, length, d] of each in 64 bits; holes as zeros, and which keys are there."""
        k, v = np.zeros((2, self.h, length, self.d))
        there = np.zeros(length, bool)
        for j in range(-(-length // self.p)):
            page, n = (self.table[s, j] if j < self.width else -1), min(self.p, length - j * self.p)
            if 0 <= page < self.pages:
                at = slice(j * self.p, j * self.p + n)
                with np.errstate(invalid="ignore"):
                    k[:, at] = e4m3(self.k[page][:, :n]) * self.ks[page].astype(np.float64)[:, None, None]
                    v[:, at] = e4m3(self.v[page][:, :, :n]).transpose(0, 2, 1) * self.vs[page].astype(np.float64)[:, None, None]
                there[at] = True
        return k, v, there


def exponent(amax):
    """The smallest e with amax <= 448 * 2^e, within the format's range."""
    with np.errstate(divide="ignore"):
        e = np.ceil(np.log2(np.asarray(amax, np.float64) / 448))
    return np.maximum(e, -40)


def ref_rotate(x, pos, inv_freq, rot, interleaved, rope_scale):
    """x [tokens, heads, d]; also |a| + |b| of each element's pair."""
    half = rot // 2
    ang = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    c, s = rope_scale * np.cos(ang)[:, None], rope_scale * np.sin(ang)[:, None]
    y, size = x.copy(), np.abs(x)
    i, j = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(half), np.arange(half, rot))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    both = np.abs(x[..., i]) + np.abs(x[..., j])
    size[..., i] = size[..., j] = both * abs(rope_scale)
    return y, size


def append_case(be, seqs, kv_heads=2, group=2, head_dim=64, page=16, t="f32", rot=None, interleaved=False, norm=False, fused=True, base=10000.0,
                with_q=True, rope_scale=1.0, loud=None, holes=(), seed=0, cache=None, far=1.0, in_place=False):
    rng = np.random.default_rng(seed + 13 * head_dim + page)
    rot = head_dim if rot is None else rot
    c = cache or Cache(rng, seqs, kv_heads, head_dim, page)
    for s, j in holes:
        c.table[s, j] = [-1, c.pages, 0x7FFFFFFF][(s + j) % 3]
    hq = kv_heads * group
    width = (hq + 2 * kv_heads) * head_dim if fused else hq * head_dim
    rows = c.tokens + 3  # rows behind the last sequence
    x = rng.standard_normal((rows, (hq + 2 * kv_heads) * head_dim)).astype(np.float32)
    if loud is not None:
        x *= np.asarray(loud, np.float32)[np.arange(rows) % len(loud)][:, None]
    bits, x = raw(x, t)
    d = Dev(be)
    kv = kv_heads * head_dim
    if fused:
        p_q = d.put(bits)
        p_k, p_v = p_q + hq * head_dim * ITEM[t], p_q + (hq * head_dim + kv) * ITEM[t]
        strides = (width, width, width)
    else:
        p_q, p_k, p_v = (d.put(np.ascontiguousarray(bits[:, a: a + n])) for a, n in ((0, hq * head_dim), (hq * head_dim, kv), (hq * head_dim + kv, kv)))
        strides = (hq * head_dim, kv, kv)
    q_mark = np.full((rows, hq * head_dim), 0x3C00, bits.dtype)
    p_out = p_q if in_place else d.put(q_mark)
    out_stride = strides[0] if in_place else hq * head_dim
    inv_freq = (far * base ** (-np.arange(rot // 2) * 2.0 / max(rot, 1))).astype(np.float32)
    qn, kn = (1 + 0.1 * rng.standard_normal(head_dim).astype(np.float32) for _ in range(2))
    cache_args, batch = c.upload(be)
    args = hip.KvAppend(format=FMT[t], interleaved=int(interleaved), q_heads=hq if with_q else 0, q=p_q if with_q else None, q_stride=strides[0],
                        q_out=p_out, q_out_stride=out_stride, k=p_k, k_stride=strides[1], v=p_v, v_stride=strides[2], inv_freq=d.put(inv_freq),
                        rot_dim=rot, rope_scale=rope_scale, q_norm=d.put(qn) if norm else None, k_norm=d.put(kn) if norm else None,
                        norm_offset=0.25, norm_eps=1e-6)
    assert be.dev_kv_append(cache_args, batch, args), be.last_error()
    be.synchronize()
    # the definition
    x = x.reshape(rows, hq + 2 * kv_heads, head_dim)
    q, k, v = x[:, :hq], x[:, hq: hq + kv_heads], x[:, hq + kv_heads:]
    if norm:
        q, k = ref_rms(q, qn.astype(np.float64), 0.25, 1e-6), ref_rms(k, kn.astype(np.float64), 0.25, 1e-6)
    pos = np.full(rows, -1, np.int64)
    live = np.zeros(rows, bool)
    for s, (new, length) in enumerate(seqs):
        at = slice(c.q_start[s], c.q_start[s] + new)
        pos[at], live[at] = np.arange(length - new, length), True
    q, q_size = ref_rotate(q, pos, inv_freq, rot, interleaved, rope_scale)
    k, k_size = ref_rotate(k, pos, inv_freq, rot, interleaved, rope_scale)
    # an angle of at most half a turn in 32 bits (2 pi U / 2 off), its sine and cosine, two products and a sum; the norm as above
    err = (16 + 48 * norm) * U
    if with_q:
        got = be.d2h(p_out, (rows, out_stride), bits.dtype)[:, : hq * head_dim]
        g = values(got, t).reshape(rows, hq, head_dim)
        close(g[live], q[live], err * q_size[live] + HALF[t] * np.abs(q[live]) + TINY[t], "q")
        if not in_place:
            assert (got[~live] == q_mark[~live]).all()
    after = c.download(be)
    for codes, scales, new_x, size, name in (("k", "ks", k, k_size, "k"), ("v", "vs", v, np.abs(v), "v")):
        want_s = getattr(c, scales).copy()
        touched = np.zeros(getattr(c, codes).shape, bool)
        got = e4m3(after[codes])
        assert np.isfinite(got[np.isfinite(e4m3(getattr(c, codes)))]).all()
        for s, (new, length) in enumerate(seqs):
            first = length - new
            for j in range(max(first, 0) // page, -(-length // page) if new and length > 0 else 0):
                pg = c.table[s, j] if j < c.width else -1
                if not 0 <= pg < c.pages:
                    continue
                lo, hi = max(first, j * page), min(length, j * page + page)
                a, b = lo - j * page, hi - j * page
                for h in range(kv_heads):
                    y = new_x[c.q_start[s] + lo - first: c.q_start[s] + hi - first, h]
                    e = exponent(np.abs(y).max())
                    if a:
                        e = max(e, math.log2(getattr(c, scales)[pg, h]))
                    want_s[pg, h] = 2.0 ** e
                    page_codes = (lambda z: z[pg, h].T if name == "v" else z[pg, h])
                    step = 2.0 ** e * 2.0 ** -9
                    slack = err * size[c.q_start[s] + lo - first: c.q_start[s] + hi - first, h]
                    close(page_codes(got)[a:b] * 2.0 ** e, y, np.maximum(2.0 ** -4 * (np.abs(y) + slack), step / 2) + slack, name)
                    if a:  # older codes: exact, or half a step of the smallest codes where they became subnormal
                        was = page_codes(e4m3(getattr(c, codes)))[:a] * float(getattr(c, scales)[pg, h])
                        close(page_codes(got)[:a] * 2.0 ** e, was, step / 2 if 2.0 ** e > getattr(c, scales)[pg, h] else 0.0, name + " older")
                    page_codes(touched)[:b] = True
        assert (after[scales] == want_s).all(), name
        assert (after[codes][~touched] == getattr(c, codes)[~touched]).all(), name
    return c, cache_args, batch, args, after


SEQS = [(1, 1), (1, 17), (5, 5), (3, 33), (16, 32), (17, 40), (0, 9), (40, 40), (1, 48), (2, 17)]


@gpu
@pytest.mark.parametrize("head_dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_append_sizes(be, head_dim, page):
    append_case(be, SEQS, head_dim=head_dim, page=page, norm=head_dim % 64 == 0)


@gpu
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [0, 8, 64, 128])
def test_append_types_and_rotations(be, t, interleaved, rot):
    append_case(be, SEQS, kv_heads=3, group=1, head_dim=128, page=32, t=t, rot=rot, interleaved=interleaved, norm=t == "bf16", fused=rot != 64,
                rope_scale=1.25)


@gpu
@pytest.mark.parametrize("how", [{"with_q": False}, {"in_place": True}, {"far": 3000.0}, {"group": 8, "kv_heads": 1}, {"group": 5},
                                 {"holes": [(3, 2), (5, 1), (7, 0)]}, {"loud": [1e-3, 1.0, 1e4, 3e-8]}, {"loud": [0.0]}, {"loud": [1e-14]},
                                 {"loud": [1e17]}])
def test_append_ways(be, how):
    append_case(be, SEQS, **how)


@gpu
def test_append_one_token_each(be):
    append_case(be, [(1, n) for n in (1, 2, 16, 17, 64, 65, 100, 129)] * 9, head_dim=128, page=64, t="bf16")
    append_case(be, [(1, 5), (0, 3), (1, 16), (0, 0)], page=16)


@gpu
def test_append_many_sequences_and_a_long_prompt(be):
    append_case(be, [(i % 4, 5 + i % 50) for i in range(200)], kv_heads=1, head_dim=32, page=16)
    append_case(be, [(700, 1000), (0, 0), (1, 1), (333, 333)], kv_heads=1, group=1, head_dim=128, page=64, t="bf16")


@gpu
def test_a_page_filled_token_by_token_keeps_its_codes_within_half_a_step_of_its_scale(be):
    rng = np.random.default_rng(3)
    h, d, p, n = 2, 64, 32, 32
    c = Cache(rng, [(1, n)], h, d, p)
    x = (rng.standard_normal((n, 2 * h * d)) * np.exp2(rng.integers(-6, 7, n))[:, None]).astype(np.float32)
    cache, batch = c.upload(be)
    dv = Dev(be)
    for i in range(n):
        row = dv.put(x[i])
        be.h2d(c.dev["kv_len"], np.array([i + 1], np.int32))
        args = hip.KvAppend(format=FMT["f32"], k=row, k_stride=2 * h * d, v=row + 4 * h * d, v_stride=2 * h * d, rot_dim=0)
        for _ in range(1 + i % 2):  # the same token again changes nothing
            assert be.dev_kv_append(cache, batch, args)
        be.synchronize()
    after = c.download(be)
    pg = c.table[0, 0]
    x = x.reshape(n, 2, h, d).astype(np.float64)
    for name, scales, y in (("k", "ks", x[:, 0]), ("v", "vs", x[:, 1])):
        for i in range(h):
            e = float(exponent(np.abs(y[:, i]).max()))
            assert after[scales][pg, i] == 2.0 ** e
            got = e4m3(after[name])[pg, i]
            got = (got.T if name == "v" else got) * 2.0 ** e
            # one rounding to the code's own step, and one of at most half the smallest step each time that the scale grew: those
            # halves shrink with the scale, a geometric sum below one step of the last
            close(got, y[:, i], np.maximum(2.0 ** -4 * np.abs(y[:, i]), 0.0) + 2.0 ** e * 2.0 ** -9, name)


@gpu
def test_a_block_with_a_number_that_is_none_says_so_and_stays_finite(be):
    rng = np.random.default_rng(5)
    h, d, p = 2, 64, 16
    for bad in (np.nan, np.inf, -np.inf, 1e30):
        c = Cache(rng, [(20, 36), (1, 4)], h, d, p)
        x = rng.standard_normal((21, 2 * h * d)).astype(np.float32)
        x[3, 5] = bad            # key head 0, position 19: page 1
        x[18, h * d + d + 7] = bad  # value head 1, position 34: page 2
        cache, batch = c.upload(be)
        row = Dev(be).put(x)
        assert be.dev_kv_append(cache, batch, hip.KvAppend(format=FMT["f32"], k=row, k_stride=2 * h * d, v=row + 4 * h * d, v_stride=2 * h * d))
        be.synchronize()
        after = c.download(be)
        nan_k, nan_v = np.isnan(after["ks"]), np.isnan(after["vs"])
        assert nan_k.sum() == 1 and nan_k[c.table[0, 1], 0] and nan_v.sum() == 1 and nan_v[c.table[0, 2], 1]
        assert np.isfinite(e4m3(after["k"])).all() and np.isfinite(e4m3(after["v"])).all()
        # a later token does not make such a block a number again
        be.h2d(c.dev["q_start"], np.array([0, 1, 2], np.int32))
        be.h2d(c.dev["kv_len"], np.array([37, 5], np.int32))
        assert be.dev_kv_append(cache, batch, hip.KvAppend(format=FMT["f32"], k=row, k_stride=2 * h * d, v=row + 4 * h * d, v_stride=2 * h * d))
        be.synchronize()
        assert np.isnan(c.download(be)["vs"][c.table[0, 2], 1])


@gpu
def test_append_leaves_sequences_out_whose_rows_do_not_fit(be):
    rng = np.random.default_rng(6)
    h, d, p = 1, 32, 16
    c = Cache(rng, [(2, 20), (3, 18), (2, 5)], h, d, p)
    x = rng.standard_normal((7, 2 * h * d)).astype(np.float32)
    cache, batch = c.upload(be)
    row = Dev(be).put(x)
    args = hip.KvAppend(format=FMT["f32"], k=row, k_stride=2 * h * d, v=row + 4 * h * d, v_stride=2 * h * d)
    for starts in ([0, 2, 1, 8], [-2, 0, 0, 9], [0, 7, 7, 7]):  # falling / below 0 / beyond the rows / more than max_new_tokens
        be.h2d(c.dev["q_start"], np.array(starts, np.int32))
        fits = [0 <= a <= b <= 7 and b - a <= 3 for a, b in zip(starts, starts[1:])]
        if any(f and b > a for f, a, b in zip(fits, starts, starts[1:])):
            continue
        assert be.dev_kv_append(cache, batch, args)
        be.synchronize()
        after = c.download(be)
        for n in after:
            assert (after[n] == getattr(c, n)).all()
    # more new tokens than the sequence is long: those before its first position are left out
    be.h2d(c.dev["q_start"], np.array([0, 3, 3, 3], np.int32))
    be.h2d(c.dev["kv_len"], np.array([1, 0, -5], np.int32))
    assert be.dev_kv_append(cache, batch, args)
    be.synchronize()
    got = e4m3(c.download(be)["k"])[c.table[0, 0], 0, 0]
    y = x[2, :d].astype(np.float64)
    s = 2.0 ** float(exponent(np.abs(y).max()))
    close(got * s, y, np.maximum(2.0 ** -4 * np.abs(y), s * 2.0 ** -10))


# ---- attention -----------------------------------------------------------------------------------------------------

def ref_attention(c, q, scale, causal, window, softcap, sinks):
    """[tokens, heads, d]; sums of |weight * value|, and the largest |x| and sum of |q k| of each row."""
    out = np.zeros(q.shape)
    size, xmax, qk = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    group = q.shape[1] // c.h
    for s, (new, length) in enumerate(c.seqs):
        keys, vals, there = c.keys_values(s, max(min(length, c.width * c.p), 0))
        j = np.arange(keys.shape[1])
        pos = np.arange(length - new, length)
        for i in range(q.shape[1]):
            k, v = keys[i // group], vals[i // group]
            for n in range(new):
                row = c.q_start[s] + n
                seen = there.copy()
                if causal:
                    seen &= j <= pos[n]
                if window:
                    seen &= j > pos[n] - window
                if not seen.any():
                    continue
                x = k[seen] @ q[row, i] * scale
                if softcap:
                    x = softcap * np.tanh(x / softcap)
                m = x.max()
                p = np.exp(x - m)
                total = p.sum() + (np.exp(float(sinks[i]) - m) if sinks is not None else 0.0)
                out[row, i] = p @ v[seen] / total
                size[row, i] = p @ np.abs(v[seen]) / total
                xmax[row, i] = np.abs(x).max()
                qk[row, i] = (np.abs(k[seen]) @ np.abs(q[row, i])).max()
    return out, size, xmax, qk


def attention_case(be, seqs, kv_heads=2, group=2, head_dim=64, page=16, t="f32", out="f32", causal=True, window=0, softcap=0.0, sinks=None, scale=None,
                   holes=(), seed=0, sigma=1.0, q_sigma=1.0, pad=0, cache=None, spoil_tail=False, rows_more=3):
    rng = np.random.default_rng(seed + 31 * head_dim + page)
    c = cache or Cache(rng, seqs, kv_heads, head_dim, page, sigma=sigma)
    for s, j in holes:
        c.table[s, j] = [-1, c.pages, 0x7FFFFFFF][(s + j) % 3]
    if spoil_tail:  # what lies behind a sequence's last key and in pages of no sequence may be anything
        used = set()
        for s, (_, length) in enumerate(seqs):
            for j in range(-(-length // page)):
                pg, n = c.table[s, j], min(page, length - j * page)
                if not 0 <= pg < c.pages:
                    continue
                used.add(int(pg))
                c.k[pg][:, n:], c.v[pg][:, :, n:] = 0x7F, 0xFF
        for pg in set(range(c.pages)) - used:
            c.k[pg], c.v[pg], c.ks[pg], c.vs[pg] = 0x7F, 0x7F, np.nan, np.inf
    hq = kv_heads * group
    rows, width = c.tokens + rows_more, hq * head_dim + pad
    bits, q = raw(rng.standard_normal((rows, width)) * q_sigma, t)
    q = q[:, : hq * head_dim].reshape(rows, hq, head_dim)
    mark = np.full((rows, width), 0x3C00, np.int32 if out == "f32" else np.int16)
    d = Dev(be)
    p_out = d.put(mark)
    cache_args, batch = c.upload(be)
    scale = head_dim ** -0.5 if scale is None else scale
    sink_values = None if sinks is None else np.asarray(sinks, np.float32)[np.arange(hq) % len(sinks)]
    args = hip.Attention(q=d.put(bits), q_stride=width, q_format=FMT[t], out=p_out, out_stride=width, out_format=FMT[out], q_heads=hq,
                         causal=int(causal), window=window, scale=scale, softcap=softcap, sinks=None if sinks is None else d.put(sink_values))
    n = be.attention_workspace_bytes(cache_args, batch, args)
    guard = np.full(64, 0xA5, np.uint8)
    ws = be.malloc(n + 64)
    be.h2d(ws + n, guard)
    assert be.dev_attention(cache_args, batch, args, ws, n), be.last_error()
    be.synchronize()
    got_bits = be.d2h(p_out, mark.shape, mark.dtype)
    assert (be.d2h(ws + n, (64,), np.uint8) == guard).all()
    got = values(got_bits, out)[:, : hq * head_dim].reshape(rows, hq, head_dim)
    want, size, xmax, qk = ref_attention(c, q, scale, causal, window, softcap, sink_values)
    # Scores: sums of products with f16 pairs (2^-22 each, 2^-38 of the row's largest element) or, into 16 bits, one f16 of an f32
    # query (2^-11), and f32 sums; exponent and sums of weights in f32 (an exponent x ln 2 of at most xmax + 60: its rounding, and
    # that of the cap, which is as small as the scores where it is far above them); weights as f16 pairs or one f16 (2^-11).  A relative error e of the weights moves the result by 2 e size.
    one = out != "f32"
    e = 2.0 ** -20 * abs(scale) * qk + (2.0 ** -11 * abs(scale) * qk if one and t == "f32" else 0.0)
    e = e + 32 * U * (60 + xmax + 2 * np.minimum(softcap, 4 * xmax)) + (2.0 ** -11 if one else 2.0 ** -21)
    bound = (2 * e[..., None] * np.exp(np.minimum(e, 1))[..., None]) * size + HALF[out] * np.abs(want) + TINY[out]
    close(got[: c.tokens], want[: c.tokens], bound[: c.tokens])
    assert (got_bits[c.tokens:] == mark[c.tokens:]).all()
    if pad:
        assert (got_bits[:, hq * head_dim:] == mark[:, hq * head_dim:]).all()
    return c, got, want


RAGGED = [(1, 1), (1, 64), (1, 65), (3, 3), (1, 300), (5, 129), (0, 7), (20, 20), (17, 100)]


@gpu
@pytest.mark.parametrize("head_dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("t,out", [("f32", "f32"), ("bf16", "bf16")])
def test_attention_sizes(be, head_dim, page, t, out):
    attention_case(be, RAGGED, head_dim=head_dim, page=page, t=t, out=out)


@gpu
@pytest.mark.parametrize("t,out", [("f32", "bf16"), ("f32", "f16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (1, 16), (2, 3), (3, 8), (1, 40), (4, 1)])
def test_attention_types_and_heads(be, t, out, kv_heads, group):
    attention_case(be, RAGGED, kv_heads, group, t=t, out=out)


@gpu
@pytest.mark.parametrize("how", [{"window": 1}, {"window": 16}, {"window": 100}, {"causal": False}, {"causal": False, "window": 50},
                                 {"softcap": 5.0, "q_sigma": 6.0}, {"softcap": 30.0, "window": 33}, {"softcap": 1e5}, {"sinks": [0.0, 3.0, -2.0, 60.0]},
                                 {"sinks": [-np.inf, -200.0]}, {"sinks": [1.0], "window": 20}, {"scale": -0.3}, {"scale": 0.0}, {"pad": 8},
                                 {"spoil_tail": True}, {"spoil_tail": True, "window": 40}, {"spoil_tail": True, "causal": False},
                                 {"holes": [(1, 0), (4, 3), (5, 8), (7, 1), (8, 6)]}, {"holes": [(4, j) for j in range(19)]},
                                 {"holes": [(4, 18), (3, 0)], "spoil_tail": False, "sinks": [0.5]}, {"sigma": 1e-9}, {"sigma": 1e12, "scale": 1e-13},
                                 {"q_sigma": 1e-20}, {"q_sigma": 1e15, "scale": 1e-16}, {"q_sigma": 25.0}])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_attention_ways(be, how, out):
    attention_case(be, RAGGED, out=out, **how)


@gpu
@pytest.mark.parametrize("t,out", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("seqs", [[(1, 20000)], [(2, 9001), (1, 3), (1, 4097)], [(33, 5000)], [(1, 1 + 97 * i) for i in range(70)]])
def test_attention_long_rows_in_pieces(be, t, out, seqs):
    attention_case(be, seqs, kv_heads=1, group=4, head_dim=64, page=64, t=t, out=out, spoil_tail=True)


@gpu
@pytest.mark.parametrize("t,out", [("f32", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("how", [{}, {"window": 900}, {"causal": False, "window": 2000}, {"softcap": 20.0}, {"sinks": [1.0, -1.0]},
                                 {"holes": [(0, 3), (0, 40), (1, 0), (2, 17)]}])
@pytest.mark.parametrize("head_dim", [64, 192])
def test_attention_of_rows_in_pieces_beside_whole_ones(be, t, out, how, head_dim):
    """Few and many rows, long and short, in one batch: both kernels, and the joining of both."""
    attention_case(be, [(40, 3000), (1, 2500), (130, 1500), (2, 64), (20, 20), (5, 4100)], kv_heads=1, group=3, head_dim=head_dim, page=64, t=t,
                   out=out, spoil_tail=True, **how)


@gpu
@pytest.mark.parametrize("t,out", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("how", [{}, {"window": 77}, {"causal": False}, {"softcap": 20.0}, {"sinks": [1.0]}])
def test_attention_prompts(be, t, out, how):
    attention_case(be, [(150, 150), (1, 90), (64, 64), (130, 400), (257, 257)], kv_heads=1, group=2, head_dim=128, page=32, t=t, out=out,
                   spoil_tail=True, **how)
    attention_case(be, [(200, 333), (65, 65)], kv_heads=2, group=3, head_dim=64, page=16, t=t, out=out, **how)


@gpu
@pytest.mark.parametrize("head_dim", [32, 96, 192, 256])
@pytest.mark.parametrize("t,out", [("f32", "f32"), ("f16", "f16")])
def test_attention_prompts_of_every_head_dim(be, head_dim, t, out):
    attention_case(be, [(140, 200), (100, 100), (3, 70)], kv_heads=1, group=2, head_dim=head_dim, page=64, t=t, out=out, spoil_tail=True)


@gpu
@pytest.mark.parametrize("head_dim", [64, 256])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("seqs", [[(1, 200), (4, 130)], [(70, 200), (64, 64)]])
def test_attention_weighs_blocks_of_very_different_scales(be, seqs, out, head_dim):
    rng = np.random.default_rng(9)
    t = "f32" if out == "f32" else "f16"
    if out != "f16":  # value blocks 2^-40 .. 2^60 apart from each other in one row, the large ones on keys that weigh little
        c = Cache(rng, seqs, 2, head_dim, 16)
        c.vs[:] = np.exp2(rng.integers(-40, 61, c.vs.shape)).astype(np.float32)
        attention_case(be, seqs, cache=c, head_dim=head_dim, t=t, out=out)
    c = Cache(rng, seqs, 2, head_dim, 16)
    c.vs[:] = np.exp2(rng.integers(-12, 4, c.vs.shape)).astype(np.float32)
    attention_case(be, seqs, cache=c, head_dim=head_dim, t=t, out=out, q_sigma=6.0)
    # and those of one row that its weights all but leave out
    c.vs[:] = 2.0 ** -20
    c.vs[::3] = 1.0
    attention_case(be, seqs, cache=c, head_dim=head_dim, t=t, out=out, q_sigma=3.0)


@gpu
@pytest.mark.parametrize("new", [1, 70])
def test_a_block_that_is_no_number_spoils_the_rows_that_see_it_only(be, new):
    rng = np.random.default_rng(10)
    seqs = [(new, 100), (new, 100), (new, 100)]
    c = Cache(rng, seqs, 2, 64, 16)
    c.ks[c.table[0, 3], 1] = np.nan   # keys 48 .. 63, key/value head 1
    c.vs[c.table[1, 5], 0] = np.nan   # keys 80 .. 95, key/value head 0
    c.vs[c.table[2, 6], 1] = np.nan   # keys 96 .. 111
    _, got, _ = attention_case(be, seqs, cache=c)
    bad = np.isnan(got[: c.tokens]).any(-1)
    assert (bad == np.isnan(got[: c.tokens]).all(-1)).all()
    for s, (key, heads) in enumerate([(48, [2, 3]), (80, [0, 1]), (96, [2, 3])]):
        pos = np.arange(100 - new, 100)
        want = np.zeros((new, 4), bool)
        want[:, heads] = (pos >= key)[:, None]
        assert (bad[c.q_start[s]: c.q_start[s + 1]] == want).all()


@gpu
def test_a_query_that_is_no_number_spoils_its_row_only(be):
    rng = np.random.default_rng(11)
    c = Cache(rng, [(6, 40)], 1, 64, 16)
    cache, batch = c.upload(be)
    d = Dev(be)
    for bad in (np.nan, np.inf):
        q = rng.standard_normal((6, 2, 64)).astype(np.float32)
        q[2, 1, 5] = bad
        out = d.put(np.zeros((6, 2, 64), np.float32))
        args = hip.Attention(q=d.put(q), q_stride=128, q_format=FMT["f32"], out=out, out_stride=128, out_format=FMT["f32"], q_heads=2, causal=1,
                             scale=0.125)
        n = be.attention_workspace_bytes(cache, batch, args)
        assert be.dev_attention(cache, batch, args, be.malloc(n), n)
        be.synchronize()
        got = be.d2h(out, q.shape, np.float32)
        spoilt = np.isnan(got).all(-1)
        assert spoilt[2, 1] and spoilt.sum() == 1 and np.isnan(got).sum() == 64


@gpu
def test_attention_of_lengths_zero_and_rows_that_do_not_fit(be):
    # no keys, more new tokens than keys (rows before the first position see nothing): zeros; a sequence left out: rows as they were
    c, got, want = attention_case(be, [(2, 0), (3, 1), (5, 2), (0, 0), (1, 1)], kv_heads=1, page=16)
    assert (got[:2] == 0).all() and (got[2:4] == 0).all() and (got[4] != 0).any() and (got[5:8] == 0).all()
    rng = np.random.default_rng(12)
    c = Cache(rng, [(2, 20), (2, 20)], 1, 32, 16)
    cache, batch = c.upload(be)
    d = Dev(be)
    for starts in ([0, 3, 2], [2, 1, 5], [-1, 0, 5]):
        be.h2d(c.dev["q_start"], np.array(starts, np.int32))
        out = d.put(np.full((4, 32), 7, np.float32))
        args = hip.Attention(q=d.put(np.ones((4, 32), np.float32)), q_stride=32, q_format=FMT["f32"], out=out, out_stride=32,
                             out_format=FMT["f32"], q_heads=1, causal=1, scale=1.0)
        n = be.attention_workspace_bytes(cache, batch, args)
        assert be.dev_attention(cache, batch, args, be.malloc(n), n)
        be.synchronize()
        assert (be.d2h(out, (4, 32), np.float32) == 7).all()


@gpu
def test_a_table_shorter_than_its_sequence_masks_what_it_does_not_list(be):
    rng = np.random.default_rng(13)
    c = Cache(rng, [(1, 90), (70, 90)], 1, 64, 16)
    full, c.width = c.table, 4
    c.table = np.ascontiguousarray(full[:, :4])
    attention_case(be, c.seqs, kv_heads=1, cache=c)


@gpu
def test_offsets_beyond_32_bits(be):
    """A cache of more than 2^32 bytes: pages at its end."""
    h, d, p, pages = 8, 256, 128, 17000  # 4.4 GB of codes each
    rng = np.random.default_rng(14)
    near = Cache(rng, [(2, 200), (130, 150)], h, d, p, spare=0)
    kb, vb = (be.malloc(pages * h * d * p) for _ in range(2))
    ks, vs = (be.malloc(pages * h * 4) for _ in range(2))
    moved = (near.table + (pages - near.pages) * (near.table >= 0)).astype(np.int32)
    for base, a, item in ((kb, near.k, h * d * p), (vb, near.v, h * d * p), (ks, near.ks, 4 * h), (vs, near.vs, 4 * h)):
        be.h2d(base + (pages - near.pages) * item, a)
    dv = Dev(be)
    near.dev = {"kv_len": dv.put(near.kv_len), "q_start": dv.put(near.q_start)}
    cache = hip.KvCache(k_codes=kb, v_codes=vb, k_scales=ks, v_scales=vs, num_pages=pages, kv_heads=h, head_dim=d, page_tokens=p)
    batch = hip.KvBatch(kv_len=near.dev["kv_len"], block_table=dv.put(moved), q_start=near.dev["q_start"], sequences=2, table_width=near.width,
                        tokens=near.tokens, max_new_tokens=near.max_new)
    x = rng.standard_normal((near.tokens, 3, h, d)).astype(np.float32)
    row = dv.put(x)
    out = dv.put(np.zeros((near.tokens, h, d), np.float32))
    app = hip.KvAppend(format=FMT["f32"], k=row + 4 * h * d, k_stride=3 * h * d, v=row + 8 * h * d, v_stride=3 * h * d)
    att = hip.Attention(q=row, q_stride=3 * h * d, q_format=FMT["f32"], out=out, out_stride=h * d, out_format=FMT["f32"], q_heads=h, causal=1,
                        scale=d ** -0.5)
    n = be.attention_workspace_bytes(cache, batch, att)
    assert be.dev_kv_append(cache, batch, app) and be.dev_attention(cache, batch, att, be.malloc(n), n)
    be.synchronize()
    got = be.d2h(out, (near.tokens, h, d), np.float32)
    for name, base, item in (("k", kb, h * d * p), ("v", vb, h * d * p), ("ks", ks, 4 * h), ("vs", vs, 4 * h)):
        a = getattr(near, name)
        setattr(near, name, be.d2h(base + (pages - near.pages) * item, a.shape, a.dtype))
    k, v, _ = near.keys_values(0, 200)
    close(k[:, 198:], x[:2, 1].transpose(1, 0, 2).astype(np.float64), 2.0 ** -4 * np.abs(x[:2, 1].transpose(1, 0, 2)) + 2.0 ** -10 * near.ks.max())
    want, size, xmax, qk = ref_attention(near, x[:, 0].astype(np.float64), d ** -0.5, True, 0, 0.0, None)
    e = 2.0 ** -20 * d ** -0.5 * qk + 32 * U * (60 + xmax) + 2.0 ** -21
    close(got, want, 2 * e[..., None] * size + U * np.abs(want))


# ---- together ------------------------------------------------------------------------------------------------------

class Layer:
    """Norm, append and attention of one layer for a batch of decoding sequences, in device memory."""

    def __init__(self, be, rng, seqs, h=2, group=2, d=64, p=16):
        self.be, self.h, self.d, self.hq, self.hidden = be, h, d, h * group, h * group * d
        self.c = Cache(rng, seqs, h, d, p, width_more=6, spare=4 + 6 * len(seqs))
        free = [i for i in range(self.c.pages) if i not in set(self.c.table.reshape(-1).tolist())]
        for s in range(len(seqs)):
            for j in range(self.c.width):
                if self.c.table[s, j] < 0 and free:
                    self.c.table[s, j] = free.pop()
        n, dv = self.c.tokens, Dev(be)
        self.cache, self.batch = self.c.upload(be)
        self.x = dv.put(rng.standard_normal((n, self.hidden)).astype(np.float32))
        self.qkv = dv.put(rng.standard_normal((n, (self.hq + 2 * h) * d)).astype(np.float32))
        self.q, self.o, self.h_out, self.n_out = (dv.put(np.zeros((n, self.hidden), np.float32)) for _ in range(4))
        freq = dv.put((10000.0 ** (-np.arange(d // 2) * 2.0 / d)).astype(np.float32))
        row = (self.hq + 2 * h) * d
        self.app = hip.KvAppend(format=FMT["f32"], q_heads=self.hq, q=self.qkv, q_stride=row, q_out=self.q, q_out_stride=self.hidden,
                                k=self.qkv + 4 * self.hidden, k_stride=row, v=self.qkv + 4 * (self.hidden + h * d), v_stride=row, inv_freq=freq,
                                rot_dim=d, rope_scale=1.0)
        self.att = hip.Attention(q=self.q, q_stride=self.hidden, q_format=FMT["f32"], out=self.o, out_stride=self.hidden, out_format=FMT["f32"],
                                 q_heads=self.hq, causal=1, scale=d ** -0.5)
        self.ws_bytes = be.attention_workspace_bytes(self.cache, self.batch, self.att)
        self.ws = be.malloc(self.ws_bytes)
        w = dv.put(rng.standard_normal(self.hidden).astype(np.float32))
        self.norm = hip.ResidualNorm(rows=n, hidden=self.hidden, block=self.o, block_stride=self.hidden, block_format=FMT["f32"],
                                     residual_format=FMT["f32"], residual=self.x, residual_stride=self.hidden, residual_out=self.h_out,
                                     residual_out_stride=self.hidden, normed=self.n_out, normed_stride=self.hidden, normed_format=FMT["f32"],
                                     residual_scale=1.0, post_weight=w, pre_weight=w, norm_offset=1.0, eps=1e-6)

    def eager(self):
        assert self.be.dev_kv_append(self.cache, self.batch, self.app) and self.be.dev_attention(self.cache, self.batch, self.att, self.ws, self.ws_bytes)
        assert self.be.dev_residual_norm(self.norm)

    def plans(self):
        return [self.be.plan_create_kv_append(self.cache, self.batch, self.app),
                self.be.plan_create_attention(self.cache, self.batch, self.att, self.ws, self.ws_bytes), self.be.plan_create_residual_norm(self.norm)]

    def results(self):
        self.be.synchronize()
        n = self.c.tokens
        return [self.be.d2h(p, (n, self.hidden), np.float32) for p in (self.q, self.o, self.h_out, self.n_out)] + list(self.c.download(self.be).values())


@gpu
def test_a_layers_step_recorded_as_one_sequence_follows_growing_lengths(be):
    """The recorded step and the eager one, each on a cache of its own, for several tokens with other work between."""
    seqs = [(1, 3), (1, 31), (1, 32), (1, 90), (1, 1)]
    a, b = (Layer(be, np.random.default_rng(20), seqs) for _ in range(2))
    plans = a.plans()
    assert all(plans)
    seq = be.sequence_create(plans)
    assert seq and be.sequence_launch_count(seq) == sum(be.plan_launch_count(p) for p in plans)
    rng = np.random.default_rng(21)
    for step in range(5):
        lens = np.array([n + step for _, n in seqs], np.int32)
        x = rng.standard_normal((5, (a.hq + 2 * a.h) * a.d)).astype(np.float32)
        for layer in (a, b):
            be.h2d(layer.c.dev["kv_len"], lens)
            be.h2d(layer.qkv, x)
        assert be.sequence_run(seq)
        b.eager()
        for got, want in zip(a.results(), b.results()):
            assert (got.view(np.uint8) == want.view(np.uint8)).all(), step
        # the eager result against the definition
        layer = b
        for n, v in b.c.download(be).items():
            setattr(layer.c, n, v)
        layer.c.seqs = [(1, int(n)) for n in lens]
        q = b.results()[0].reshape(5, b.hq, b.d).astype(np.float64)
        want, size, xmax, qk = ref_attention(b.c, q, b.d ** -0.5, True, 0, 0.0, None)
        e = 2.0 ** -20 * b.d ** -0.5 * qk + 32 * U * (60 + xmax) + 2.0 ** -21
        close(b.results()[1].reshape(want.shape), want, 2 * e[..., None] * size + U * np.abs(want))
    be.sequence_destroy(seq)
    for p in plans:
        be.plan_destroy(p)


@gpu
def test_two_contexts_and_calls_in_a_row_give_the_same(be):
    other = hip.HipBackend()
    try:
        seqs = [(1, 40), (7, 50), (1, 700)]
        a, b = Layer(be, np.random.default_rng(22), seqs), Layer(other, np.random.default_rng(22), seqs)
        for _ in range(3):
            a.eager()
            b.eager()
        for got, want in zip(a.results(), b.results()):
            assert (got.view(np.uint8) == want.view(np.uint8)).all()
    finally:
        other.close()


@gpu
def test_results_repeat_bit_for_bit(be):
    layer = Layer(be, np.random.default_rng(23), [(3, 2000), (1, 17), (40, 60)])
    layer.eager()
    first = layer.results()
    for _ in range(3):
        layer.eager()
        for got, want in zip(layer.results(), first):
            assert (got.view(np.uint8) == want.view(np.uint8)).all()


# ---- refusals (no kernel runs; without a context a call that would be served is LARQL_E_ARG) ------------------------

def _sound():
    cache = hip.KvCache(k_codes=4096, v_codes=8192, k_scales=64, v_scales=128, num_pages=4, kv_heads=2, head_dim=64, page_tokens=16)
    batch = hip.KvBatch(kv_len=64, block_table=64, q_start=64, sequences=1, table_width=4, tokens=3, max_new_tokens=3)
    app = hip.KvAppend(format=FMT["f32"], q_heads=4, q=4096, q_stride=256, q_out=8192, q_out_stride=256, k=4096, k_stride=128, v=4096, v_stride=128,
                       inv_freq=64, rot_dim=64, rope_scale=1.0)
    att = hip.Attention(q=4096, q_stride=256, q_format=FMT["f32"], out=8192, out_stride=256, out_format=FMT["bf16"], q_heads=4, causal=1, scale=0.1)
    norm = hip.ResidualNorm(rows=2, hidden=64, block=4096, block_stride=64, block_format=FMT["f32"], residual_format=FMT["f32"], residual=4096,
                            residual_stride=64, residual_out=8192, residual_out_stride=64, normed=16384, normed_stride=64, normed_format=FMT["bf16"],
                            residual_scale=1.0, eps=1e-6)
    return {"cache": cache, "batch": batch, "app": app, "att": att, "norm": norm}


def _call(op, s):
    ref = ctypes.byref
    if op == "app":
        return L.lib.larql_hip_dev_kv_append(None, ref(s["cache"]), ref(s["batch"]), ref(s["app"]))
    if op == "att":
        n = max(L.lib.larql_hip_attention_workspace_bytes(ref(s["cache"]), ref(s["batch"]), ref(s["att"])), s.get("ws_bytes", 1 << 40))
        return L.lib.larql_hip_dev_attention(None, ref(s["cache"]), ref(s["batch"]), ref(s["att"]), s.get("ws", 4096), n if "ws_bytes" not in s else s["ws_bytes"])
    return L.lib.larql_hip_dev_residual_norm(None, ref(s["norm"]))


@pytest.mark.parametrize("op", ["app", "att", "norm"])
def test_a_sound_call_passes_the_checks(op):
    assert _call(op, _sound()) == L.E_ARG  # (no context)


_KV = [("cache", "head_dim", 0, L.REFUSED_SHAPE), ("cache", "head_dim", 48, L.REFUSED_SHAPE), ("cache", "head_dim", 288, L.REFUSED_SHAPE),
       ("cache", "page_tokens", 0, L.REFUSED_SHAPE), ("cache", "page_tokens", 24, L.REFUSED_SHAPE), ("cache", "page_tokens", 256, L.REFUSED_SHAPE),
       ("cache", "kv_heads", 0, L.REFUSED_SHAPE), ("cache", "kv_heads", 5000, L.REFUSED_SHAPE), ("cache", "num_pages", 0, L.REFUSED_SHAPE),
       ("cache", "num_pages", 1 << 31, L.UNSUPPORTED), ("cache", "k_codes", 4104, L.REFUSED_SHAPE), ("cache", "v_codes", None, L.E_ARG),
       ("cache", "k_scales", 66, L.REFUSED_SHAPE), ("batch", "table_width", 0, L.REFUSED_SHAPE), ("batch", "table_width", (1 << 26) + 1, L.UNSUPPORTED), ("batch", "sequences", (1 << 16) + 1, L.UNSUPPORTED),
       ("batch", "tokens", 1 << 25, L.UNSUPPORTED), ("batch", "q_start", None, L.E_ARG), ("batch", "block_table", 66, L.REFUSED_SHAPE),
       ("batch", "kv_len", None, L.E_ARG)]
_APP = [("app", "format", hip.FMT_Q4_K, L.UNSUPPORTED), ("app", "rot_dim", 72, L.REFUSED_SHAPE), ("app", "rot_dim", 12, L.REFUSED_SHAPE),
        ("app", "inv_freq", None, L.E_ARG), ("app", "inv_freq", 66, L.REFUSED_SHAPE), ("app", "k", None, L.E_ARG), ("app", "v", None, L.E_ARG), ("app", "q_out", None, L.E_ARG),
        ("app", "k_stride", 127, L.REFUSED_SHAPE), ("app", "k_stride", 64, L.REFUSED_SHAPE), ("app", "v", 4104, L.REFUSED_SHAPE),
        ("app", "q_stride", 200, L.REFUSED_SHAPE), ("app", "q_out", 8200, L.REFUSED_SHAPE), ("app", "k_norm", 72, L.REFUSED_SHAPE),
        ("app", "q_heads", 5, L.REFUSED_SHAPE), ("app", "v_stride", 1 << 23, L.UNSUPPORTED), ("app", "q_out_stride", 1 << 23, L.UNSUPPORTED)]
_ATT = [("att", "q_format", hip.FMT_Q8_0, L.UNSUPPORTED), ("att", "out_format", -1, L.UNSUPPORTED), ("att", "q_heads", 0, L.REFUSED_SHAPE),
        ("att", "q_heads", 3, L.REFUSED_SHAPE), ("att", "q", None, L.E_ARG), ("att", "out", None, L.E_ARG), ("att", "out_stride", 252, L.REFUSED_SHAPE),
        ("att", "q_stride", 258, L.REFUSED_SHAPE), ("att", "out", 8200, L.REFUSED_SHAPE), ("att", "softcap", -1.0, L.REFUSED_SHAPE),
        ("att", "softcap", math.nan, L.REFUSED_SHAPE), ("att", "softcap", 1e-7, L.REFUSED_SHAPE), ("att", "scale", math.inf, L.REFUSED_SHAPE), ("att", "window", 1 << 31, L.UNSUPPORTED),
        ("att", "sinks", 66, L.REFUSED_SHAPE)]
_NORM = [("norm", "hidden", 32769, L.UNSUPPORTED), ("norm", "block_format", hip.FMT_MXFP4, L.UNSUPPORTED), ("norm", "residual", None, L.E_ARG),
         ("norm", "residual_stride", 63, L.REFUSED_SHAPE), ("norm", "normed_stride", 1, L.REFUSED_SHAPE), ("norm", "residual", 4098, L.REFUSED_SHAPE),
         ("norm", "normed", 16385, L.REFUSED_SHAPE), ("norm", "normed_format", 77, L.UNSUPPORTED)]


@pytest.mark.parametrize("op,which,field,value,code",
                         [("app", *c) for c in _KV + _APP] + [("att", *c) for c in _KV + _ATT] + [("norm", *c) for c in _NORM])
def test_refusals(op, which, field, value, code):
    s = _sound()
    setattr(s[which], field, value)
    assert _call(op, s) == code
    if op == "att":
        assert L.lib.larql_hip_attention_workspace_bytes(ctypes.byref(s["cache"]), ctypes.byref(s["batch"]), ctypes.byref(s["att"])) == 0


# A result in place of its operand: the same rows, or another row's elements are overwritten before they are read.
@pytest.mark.parametrize("how,code", [({"normed": 4096, "normed_format": FMT["f32"]}, L.E_ARG), ({"normed": 4096}, L.REFUSED_SHAPE),
                                      ({"normed": 4096, "normed_format": FMT["f32"], "normed_stride": 128}, L.REFUSED_SHAPE),
                                      ({"normed": 4096, "normed_format": FMT["f32"], "normed_stride": 128, "rows": 1}, L.E_ARG),
                                      ({"normed": 4096, "rows": 1}, L.REFUSED_SHAPE), ({"residual_out": 4096 + 4096, "residual": 8192}, L.E_ARG),
                                      ({"residual": 8192, "residual_out_stride": 128}, L.REFUSED_SHAPE)])
def test_a_norms_result_in_place_has_the_operands_rows(how, code):
    s = _sound()
    for field, value in how.items():
        setattr(s["norm"], field, value)
    assert _call("norm", s) == code


@pytest.mark.parametrize("stride,tokens,code", [(256, 3, L.E_ARG), (512, 3, L.REFUSED_SHAPE), (512, 1, L.E_ARG)])
def test_queries_rotated_in_place_have_the_same_rows(stride, tokens, code):
    s = _sound()
    s["app"].q_out, s["app"].q_out_stride, s["batch"].tokens = s["app"].q, stride, tokens
    assert _call("app", s) == code


def test_refusals_of_the_workspace_and_of_null_arguments():
    s = _sound()
    n = L.lib.larql_hip_attention_workspace_bytes(ctypes.byref(s["cache"]), ctypes.byref(s["batch"]), ctypes.byref(s["att"]))
    assert n > 0
    assert _call("att", {**s, "ws_bytes": n - 1}) == L.REFUSED_SHAPE
    assert _call("att", {**s, "ws_bytes": n, "ws": 4100}) == L.REFUSED_SHAPE
    assert _call("att", {**s, "ws_bytes": n, "ws": None}) == L.E_ARG
    assert L.lib.larql_hip_dev_kv_append(None, None, None, None) == L.E_ARG
    assert L.lib.larql_hip_dev_attention(None, None, None, None, None, 0) == L.E_ARG
    assert L.lib.larql_hip_dev_residual_norm(None, None) == L.E_ARG
    out = ctypes.c_void_p(1)
    assert L.lib.larql_hip_plan_create_attention(None, None, None, None, None, 0, ctypes.byref(out)) == L.E_ARG


@pytest.mark.parametrize("field", ["sequences", "tokens", "max_new_tokens"])
def test_an_empty_batch_needs_no_workspace(field):
    s = _sound()
    setattr(s["batch"], field, 0)
    assert L.lib.larql_hip_attention_workspace_bytes(ctypes.byref(s["cache"]), ctypes.byref(s["batch"]), ctypes.byref(s["att"])) == 0


@gpu
def test_refused_calls_answer_false_with_a_reason_and_empty_ones_do_nothing(be):
    layer = Layer(be, np.random.default_rng(30), [(1, 40), (2, 700)])  # (every pointer is one of a buffer, should a call be served after all)
    cache, batch, ws, n = layer.cache, layer.batch, layer.ws, layer.ws_bytes
    cache.head_dim = 48
    assert not be.dev_kv_append(cache, batch, layer.app) and "head_dim" in be.last_error()
    assert be.plan_create_attention(cache, batch, layer.att, ws, n) is None
    cache.head_dim = layer.d
    assert not be.dev_attention(cache, batch, layer.att, ws, n - 1) and "workspace" in be.last_error()
    before = layer.results()
    batch.tokens = 0
    assert be.dev_kv_append(cache, batch, layer.app) and be.dev_attention(cache, batch, layer.att, 0, 0)
    plan = be.plan_create_attention(cache, batch, layer.att, 0, 0)
    assert plan and be.plan_launch_count(plan) == 0 and be.plan_run(plan)
    be.plan_destroy(plan)
    for got, want in zip(layer.results(), before):
        assert (got.view(np.uint8) == want.view(np.uint8)).all()
