"""The layer operators at the ends of what their documentation allows: precision where the plain bounds of test_layer_ops.py are
wide, batches whose rows do not fit, launches of more workgroups than one grid dimension takes, recording."""
import ctypes

import numpy as np
import pytest

import larql_amd as hip
from larql_amd import _lib as L
from test_layer_ops import (FMT, HALF, TINY, U, Cache, Dev, Layer, _call, _sound, append_case, attention_case, close, e4m3, raw,
                            ref_attention, values)

gpu = pytest.mark.gpu


def attention(be, c, q, t, out, scale, causal=True, window=0, softcap=0.0):
    """The results of queries q [tokens, heads, d] (values of type t) over the cache c."""
    d = Dev(be)
    rows, width = q.shape[0], q.shape[1] * q.shape[2]
    cache, batch = c.upload(be)
    p_out = d.put(np.zeros((rows, width), np.int32 if out == "f32" else np.int16))
    args = hip.Attention(q=d.put(raw(q.reshape(rows, width), t)[0]), q_stride=width, q_format=FMT[t], out=p_out, out_stride=width, out_format=FMT[out],
                         q_heads=q.shape[1], causal=int(causal), window=window, scale=scale, softcap=softcap)
    n = be.attention_workspace_bytes(cache, batch, args)
    assert be.dev_attention(cache, batch, args, be.malloc(n), n), be.last_error()
    be.synchronize()
    return values(be.d2h(p_out, (rows, width), np.int32 if out == "f32" else np.int16), out).reshape(q.shape)


# ---- attention: precision ------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("head_dim", [64, 96, 256])
@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("out", ["bf16", "f16"])
def test_f32_queries_keep_their_bits_whatever_the_result(be, new, out, head_dim):
    """Queries whose products with the keys are large and cancel: what is lost of a query's elements is large beside the scores."""
    rng = np.random.default_rng(head_dim + new)
    c = Cache(rng, [(new, 24)], 1, head_dim, 16, sigma=1.0)
    keys, _, _ = c.keys_values(0, 24)
    basis = np.linalg.qr(keys[0].T)[0]
    q = rng.standard_normal((new, 1, head_dim)) * 50
    q = (q - q @ basis @ basis.T + rng.standard_normal((new, 1, head_dim)) * 0.2).astype(np.float32)
    got = attention(be, c, q, "f32", out, 1.0, causal=False)
    want, size, xmax, qk = ref_attention(c, q.astype(np.float64), 1.0, False, 0, 0.0, None)
    # queries as f16 pairs: 2^-22 of an element; f32 sums of at most 256 products: their roundings, 8 of them at a time and the parts, 2^-20 of the
    # sum of |q k|; exponents of at most 60 + |x|; one f16 of a weight: 2^-11
    e = 2.0 ** -20 * qk + 32 * U * (60 + xmax) + 2.0 ** -11
    close(got, want, 2 * e[..., None] * size + HALF[out] * np.abs(want) + TINY[out])


def two_keys(be, many, t, out, xmax, softcap=0.0, head_dim=32):
    """Every query sees two keys, with one channel in the product and values +1 and -1: a result is the difference of its two weights, so
    what the weights are off by is not lost among larger errors.  Results, the definition's."""
    rng = np.random.default_rng(7)
    seqs = [(200, 200)] if many else [(1, 2 + 5 * i) for i in range(60)]
    c = Cache(rng, seqs, 2, head_dim, 16)
    for a in (c.k, c.v):
        a[:] = 0
    c.k[..., 0] = rng.integers(0x30, 0x38, c.k.shape[:-1]) | 0x80 * rng.integers(0, 2, c.k.shape[:-1])  # 0.5 .. 0.94, either sign
    c.v[..., 0::2], c.v[..., 1::2] = 0x38, 0xB8  # 1, -1
    c.ks[:], c.vs[:] = 1.0, 1.0
    q = np.zeros((c.tokens, 4, head_dim))
    q[..., 0] = rng.uniform(-xmax, xmax, q.shape[:2])
    q = raw(q, t)[1]
    want, _, _, _ = ref_attention(c, q, 1.0, True, 2, softcap, None)
    return attention(be, c, q, t, out, 1.0, window=2, softcap=softcap), want


@gpu
@pytest.mark.parametrize("head_dim", [32, 128, 192])
@pytest.mark.parametrize("t,out", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16")])
def test_few_rows_into_16_bits_lose_nothing_but_the_results_rounding(be, t, out, head_dim):
    got, want = two_keys(be, False, t, out, 0.004, head_dim=head_dim)
    # logarithms of |x| < 0.01 (a few u), + 12 rounded at their size (16 u log2, half: 5.5 u), an exponential's last place (2 u), pairs (2 u): 12 u a
    # weight at most, half the difference of two of them, a few u of sum, quotient and product
    close(got, want, 32 * U + HALF[out] * np.abs(want) + TINY[out])


@gpu
@pytest.mark.parametrize("cap", [1.0, 2.0, 30.0, 64.0, 65.0, 1e4])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("head_dim", [32, 128, 256])
def test_a_cap_costs_f32_results_nothing(be, many, cap, head_dim):
    got, want = two_keys(be, many, "f32", "f32", 0.5, cap, head_dim)
    # logarithms of |x| <= 0.5: a dozen roundings of them at most (6 u); + 7 rounded at its size (half of 8 u log2: 2.8 u); an exponential's last
    # place (2 u), pairs (2 u): 13 u a weight, half the difference of two of them, a few u of sum, quotient and product
    close(got, want, 24 * U + 8 * U * np.abs(want))


# ---- batches in which some sequences' rows do not fit ---------------------------------------------------------------

# q_start, rows, max_new_tokens, and (new tokens, length) of the sequences, no new tokens for those that are left out
UNEVEN = [([4, 6, 0, 2], 6, 2, [(2, 20), (0, 18), (2, 5)]),            # the second falls
          ([0, 2, 1, 8], 7, 3, [(2, 20), (0, 18), (0, 5)]),            # ... and the third has more than max_new_tokens
          ([0, 2, 1, 1], 7, 3, [(2, 20), (0, 18), (0, 5)]),
          ([5, 7, 4, 5, 0, 4], 7, 4, [(2, 33), (0, 9), (1, 17), (0, 40), (4, 4)]),
          ([-2, 0, 3, 9], 7, 3, [(0, 20), (3, 18), (0, 5)]),           # below 0, beyond the rows
          ([3, 4, 0, 1, 3], 4, 1, [(1, 20), (0, 18), (1, 5), (0, 16)])]  # one token each: the kernel for that


@gpu
@pytest.mark.parametrize("starts,rows,most,seqs", UNEVEN)
@pytest.mark.parametrize("page", [16, 64])
def test_append_serves_the_sequences_whose_rows_fit(be, starts, rows, most, seqs, page):
    c = Cache(np.random.default_rng(page), seqs, 2, 64, page)
    c.q_start, c.tokens, c.max_new = np.array(starts, np.int32), rows, most
    append_case(be, seqs, cache=c, page=page, norm=True)


@gpu
@pytest.mark.parametrize("many", [False, True])
def test_attention_serves_the_sequences_whose_rows_fit(be, many):
    n = 70 if many else 2
    seqs = [(n, 100), (0, 18), (n, 90)]
    c = Cache(np.random.default_rng(1), seqs, 2, 64, 16)
    c.q_start, c.tokens, c.max_new = np.array([n, 2 * n, 0, n], np.int32), 2 * n, n
    attention_case(be, seqs, cache=c)


@gpu
def test_queries_find_their_sequence_among_many(be):
    seqs = [(0 if i % 5 == 2 else 1 + i % 3, 9 + i) for i in range(300)]
    c = Cache(np.random.default_rng(2), seqs, 1, 32, 16)
    at = np.cumsum([0] + [n for n, _ in seqs[::-1]]).astype(np.int32)  # the rows of later sequences first: every other start falls
    starts, served = [], []
    for (n, length), a in zip(seqs, at[:-1][::-1]):
        starts += [a, a + n]  # a sequence, and one between its end and the next one's start that falls or is empty
        served += [(n, length), (0, 7)]
    c = Cache(np.random.default_rng(2), served[:-1], 1, 32, 16)
    c.q_start, c.tokens, c.max_new = np.array(starts, np.int32), int(at[-1]), 3
    append_case(be, served[:-1], cache=c, kv_heads=1, head_dim=32)


# ---- more workgroups than one dimension of a grid takes (2^32 threads) ----------------------------------------------

@gpu
def test_norm_of_more_rows_than_a_grid_dimension_takes(be):
    rows = (1 << 26) + 5  # four rows a workgroup of 256 threads
    rng = np.random.default_rng(3)
    bits, h = raw(rng.standard_normal(rows, dtype=np.float32) * 2, "bf16")
    d = Dev(be)
    p = d.put(bits)
    args = hip.ResidualNorm(rows=rows, hidden=1, residual=p, residual_stride=1, residual_format=FMT["bf16"], normed=p, normed_stride=1,
                            normed_format=FMT["bf16"], norm_offset=0.0, eps=0.5)
    n = be.malloc(2 * rows)
    args.normed = n
    assert be.dev_residual_norm(args), be.last_error()
    be.synchronize()
    want = h / np.sqrt(h * h + 0.5)
    close(values(be.d2h(n, (rows,), np.int16), "bf16"), want, (16 * U + HALF["bf16"]) * np.abs(want) + TINY["bf16"])
    be.free(p)
    be.free(n)


@gpu
@pytest.mark.parametrize("kernel", ["one", "several"])
def test_append_of_more_workgroups_than_a_grid_dimension_takes(be, kernel):
    """The new tokens of the last sequence, or the last rows, through a launch of more than 2^24 workgroups of 256 threads."""
    rng = np.random.default_rng(4)
    d = Dev(be)
    h, dim, n, sequences, rows = (1024, 256, 1, 1 << 16, 1) if kernel == "one" else (1, 32, 5, 1, 1 << 24)
    c = Cache(rng, [(n, 9)], h, dim, 16, width_more=0)
    cache, batch = c.upload(be)
    table, kv_len = np.full((sequences, 1), -1, np.int32), np.full(sequences, 3, np.int32)
    q_start = np.zeros(sequences + 1, np.int32)
    table[-1], kv_len[-1], q_start[-2:] = c.table[0, 0], 9, (rows - n, rows)
    batch.block_table, batch.kv_len, batch.q_start = d.put(table), d.put(kv_len), d.put(q_start)
    batch.sequences, batch.tokens, batch.max_new_tokens = sequences, rows, n
    x = rng.standard_normal((n, h, dim)).astype(np.float32)
    bits, x = raw(x.reshape(n, -1), "bf16")
    width = h * dim
    p = be.malloc(2 * rows * width)
    q_out = be.malloc(2 * rows * width)
    be.h2d(p + 2 * (rows - n) * width, bits)
    args = hip.KvAppend(format=FMT["bf16"], q_heads=h, q=p, q_stride=width, q_out=q_out, q_out_stride=width, k=p, k_stride=width, v=p, v_stride=width)
    assert be.dev_kv_append(cache, batch, args), be.last_error()
    be.synchronize()
    assert (be.d2h(q_out + 2 * (rows - n) * width, bits.shape, np.int16) == bits).all()
    after = c.download(be)
    page = c.table[0, 0]
    for name, scales in (("k", "ks"), ("v", "vs")):
        codes = e4m3(after[name])[page]
        got = (codes if name == "k" else codes.transpose(0, 2, 1))[:, 9 - n: 9] * after[scales][page].astype(np.float64)[:, None, None]
        y = x.reshape(n, h, dim).transpose(1, 0, 2)
        close(got, y, np.maximum(2.0 ** -4 * np.abs(y), after[scales][page].astype(np.float64)[:, None, None] * 2.0 ** -10), name)
        others = [i for i in range(c.pages) if i != page]
        assert (after[name][others] == getattr(c, name)[others]).all()
    be.free(p)
    be.free(q_out)


@gpu
def test_attention_of_more_workgroups_than_a_grid_dimension_takes(be):
    rng = np.random.default_rng(5)
    d = Dev(be)
    h, dim, n, sequences = 1024, 32, 40, 8300  # a workgroup of 512 threads for each sequence and head at least
    c = Cache(rng, [(n, n)], h, dim, 64, width_more=0)
    cache, batch = c.upload(be)
    table, kv_len = np.full((sequences, 1), -1, np.int32), np.full(sequences, 3, np.int32)
    q_start = np.zeros(sequences + 1, np.int32)
    table[-1], kv_len[-1], q_start[-1] = c.table[0, 0], n, n
    batch.block_table, batch.kv_len, batch.q_start, batch.sequences = d.put(table), d.put(kv_len), d.put(q_start), sequences
    bits, q = raw(rng.standard_normal((n, h * dim)), "f32")
    out = d.put(np.zeros((n, h * dim), np.float32))
    args = hip.Attention(q=d.put(bits), q_stride=h * dim, q_format=FMT["f32"], out=out, out_stride=h * dim, out_format=FMT["f32"], q_heads=h, causal=1,
                         scale=dim ** -0.5)
    ws = be.attention_workspace_bytes(cache, batch, args)
    assert be.dev_attention(cache, batch, args, be.malloc(ws), ws), be.last_error()
    be.synchronize()
    q = q.reshape(n, h, dim)
    want, size, xmax, qk = ref_attention(c, q, dim ** -0.5, True, 0, 0.0, None)
    e = 2.0 ** -20 * dim ** -0.5 * qk + 32 * U * (60 + xmax) + 2.0 ** -21
    close(be.d2h(out, (n, h * dim), np.float32).reshape(n, h, dim), want, 2 * e[..., None] * size + U * np.abs(want))


@pytest.mark.parametrize("op,batch,cache,other,code",
                         [("app", {"tokens": 1 << 24, "max_new_tokens": 9}, {"kv_heads": 512}, {"k_stride": 1 << 15, "v_stride": 1 << 15}, L.E_ARG),
                          ("app", {"tokens": 1 << 24, "max_new_tokens": 9}, {"kv_heads": 1024}, {"k_stride": 1 << 16, "v_stride": 1 << 16}, L.UNSUPPORTED),
                          ("app", {"sequences": 1 << 16, "max_new_tokens": 1}, {"kv_heads": 1024}, {"k_stride": 1 << 16, "v_stride": 1 << 16}, L.E_ARG),
                          ("att", {"tokens": 1 << 24}, {"kv_heads": 512}, {"q_heads": 8192, "q_stride": 1 << 19, "out_stride": 1 << 19}, L.E_ARG),
                          ("att", {"tokens": 1 << 24, "max_new_tokens": 1 << 24}, {"kv_heads": 1024},
                           {"q_heads": 16384, "q_stride": 1 << 20, "out_stride": 1 << 20}, L.UNSUPPORTED),
                          ("norm", {}, {}, {"rows": 1 << 31}, L.UNSUPPORTED), ("norm", {}, {}, {"rows": (1 << 31) - 1}, L.E_ARG)])
def test_calls_of_more_workgroups_than_a_launch_takes_are_refused(op, batch, cache, other, code):
    s = _sound()
    for which, fields in (("batch", batch), ("cache", cache), (op, other)):
        for field, value in fields.items():
            setattr(s[which], field, value)
    assert _call(op, s) == code


# ---- recording -------------------------------------------------------------------------------------------------------

@gpu
def test_recording_a_layers_step_changes_nothing_that_it_works_on(be):
    """What lies in the buffers then is no step's: a residual in place would be added to, a page's scale would grow for good."""
    seqs = [(1, 3), (1, 31), (2, 40), (1, 90), (1, 1)]
    a, b = (Layer(be, np.random.default_rng(24), seqs, d=224) for _ in range(2))
    for layer in (a, b):
        layer.norm.residual_out, layer.norm.normed = layer.x, layer.o  # in place
    x = be.d2h(a.qkv, (a.c.tokens, (a.hq + 2 * a.h) * a.d), np.float32)
    be.h2d(a.qkv, np.full_like(x, np.nan))  # not written yet

    def state(layer):
        return layer.results() + [be.d2h(layer.x, (layer.c.tokens, layer.hidden), np.float32)]

    before = state(a)
    plans = a.plans()
    seq = be.sequence_create(plans)
    assert seq
    for got, want in zip(state(a), before):
        assert (got.view(np.uint8) == want.view(np.uint8)).all()
    be.h2d(a.qkv, x)
    for _ in range(3):
        assert be.sequence_run(seq)
        b.eager()
        for got, want in zip(state(a), state(b)):
            assert (got.view(np.uint8) == want.view(np.uint8)).all()
    be.sequence_destroy(seq)
    for p in plans:
        be.plan_destroy(p)


# ---- attention: long rows in pieces ----------------------------------------------------------------------------------

def _workspace(**fields):
    s = _sound()
    s["batch"].table_width = 4096
    for field, value in fields.items():
        setattr(s["batch"] if field in ("tokens", "max_new_tokens") else s["att"], field, value)
    return L.lib.larql_hip_attention_workspace_bytes(ctypes.byref(s["cache"]), ctypes.byref(s["batch"]), ctypes.byref(s["att"]))


def test_the_keys_that_a_window_without_causal_lets_a_row_see():
    """Those behind its start up to the sequence's end: with many new tokens far more than the window, so the row is split."""
    for tokens in (3, 300):
        sizes = {"tokens": tokens, "max_new_tokens": tokens, "window": 64}
        assert _workspace(**sizes) == _workspace(causal=0, **sizes) < _workspace(tokens=tokens, max_new_tokens=tokens)
    sizes = {"tokens": 5000, "max_new_tokens": 5000, "q_heads": 2}
    assert _workspace(window=64, **sizes) < _workspace(window=64, causal=0, **sizes) == _workspace(**sizes)


@gpu
@pytest.mark.parametrize("new", [1, 40, 1500])
@pytest.mark.parametrize("window", [1, 100, 5000])
def test_attention_in_a_window_that_is_open_to_later_keys(be, new, window):
    attention_case(be, [(new, 6000), (1, 2000), (min(new, 40), 40)], kv_heads=1, group=2, head_dim=64, page=64, causal=False, window=window, spoil_tail=True)


@gpu
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("t,out", [("f32", "f32"), ("f16", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_small_weights_are_held_to_their_floor(be, many, t, out):
    """A row of two keys with values in channels of their own: what is lost of a small weight shows where nothing else is added."""
    rng = np.random.default_rng(8)
    seqs = [(200, 200)] if many else [(1, 2 + 5 * i) for i in range(60)]
    c = Cache(rng, seqs, 1, 64, 16)
    for a in (c.k, c.v):
        a[:] = 0
    c.k[:, :, 0::2, 0], c.k[:, :, 1::2, 0] = 0x38, 0xB8              # keys 1, -1
    c.v[:, :, 0::2, 0::2], c.v[:, :, 1::2, 1::2] = 0x38, 0x38        # the one's value in even channels, the other's in odd ones
    c.ks[:], c.vs[:] = 1.0, 1.0
    q = np.zeros((c.tokens, 4, 64))
    q[..., 0] = rng.uniform(-13, 13, q.shape[:2])                    # weights down to 2^-37 of each other
    q = raw(q, t)[1]
    want, _, _, _ = ref_attention(c, q, 1.0, True, 2, 0.0, None)
    got = attention(be, c, q, t, out, 1.0, window=2)
    # scores of at most 13 with a few roundings of them, exponents of at most 64: 128 u of a weight; its floor, the larger one's being 1 at most
    floor = 2.0 ** -31 if out == "f32" else 2.0 ** -36
    weight = 2.0 ** -10 if many and out != "f32" else 128 * U
    close(got, want, weight * np.abs(want) + floor + HALF[out] * np.abs(want))
    assert (want[..., :2].min(-1) < floor / 2).any()
