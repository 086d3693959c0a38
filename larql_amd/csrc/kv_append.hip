// kv_append.hip — new queries, keys and values of a step's sequences: rms norm per head, rotation by position, and keys and values
// as e4m3 codes into the pages of the cache, a power-of-two scale for each page and head.
//
// A workgroup owns one head of one page that gets new tokens, so the page's scale is decided and its codes are written in one
// place, with no atomics: the new elements stay in registers between the largest |x| and the codes.  Where the scale of a page with
// older tokens grows, their codes are rounded again for it (a power of two: exact unless a code becomes subnormal).
//
// Prompts in f32 are bound by memory: 7747 tokens of 32/8 heads of 128, normed and rotated, 78-84 us for 388 MB (a large copy of that: 77).  Loads
// have no condition and offsets of 32 bits (with conditions 209 us, in 64 bits 139).  16-bit elements are converted by their type where they are
// loaded, so that a thread waits for one load before the next: the same tokens in bf16 59 us for 203 MB (a copy: 40).
// A token of each sequence is bound by its chain of waits: lengths, the two halves of the activations, norm weights, the table, the page's scale.
// 3.6 us for one of 8/4 heads of 256, 4.3 for 64 of 64/8 heads of 64 (9.8 and 20 us through the kernel for several).  Every workgroup of several
// tokens searches the sequences: two tokens each of 1024 take 59 us, of 4096 550.
#include "kernels.h"
#include "layer.h"

namespace larql {

constexpr uint32_t kAppendThreads = 256;

// 8 channels of one head and token, as four pairs (lo[i], hi[i]) that turn together
struct Quad {
    f32x4_t lo, hi;
};

// Channels of the pairs 4g .. 4g+3: (p, p + rot/2) inside the rotated part of a halved layout, else (2p, 2p + 1).
__device__ __forceinline__ bool halved(const KvAppendArgs &A, uint32_t g) { return !A.interleaved && 8 * g < A.rot_dim; }
__device__ __forceinline__ Quad load_quad(const KvAppendArgs &A, const void *row, int type, uint32_t at, uint32_t g) {
    const bool h = halved(A, g);
    const uint32_t a = at + (h ? 4 * g : 8 * g), b = at + (h ? 4 * g + A.rot_dim / 2 : 8 * g + 4);
    const f32x4_t u = load4(row, type, a), v = load4(row, type, b);
    if (h) return {u, v};
    return {f32x4_t{u[0], u[2], v[0], v[2]}, f32x4_t{u[1], u[3], v[1], v[3]}};
}
__device__ __forceinline__ void store_quad(const KvAppendArgs &A, void *row, int type, uint32_t at, uint32_t g, const Quad &q) {
    if (halved(A, g)) {
        store4(row, type, at + 4 * g, q.lo);
        store4(row, type, at + 4 * g + A.rot_dim / 2, q.hi);
    } else {
        store8(row, type, at + 8 * g, {f32x4_t{q.lo[0], q.hi[0], q.lo[1], q.hi[1]}, f32x4_t{q.lo[2], q.hi[2], q.lo[3], q.hi[3]}});
    }
}

// cos and sin of position * inv_freq[4g + i], times rope_scale.  Far positions lose the angle in 32 bits: whole turns leave in 64, then
// quarter turns; what is left, at most an eighth, goes through the Taylor series (next terms below 2e-9 and 2e-10).
struct Turn {
    f32x4_t c, s;
};
__device__ __forceinline__ void turn_of(const KvAppendArgs &A, int32_t pos, f32x4_t freq, Turn &t) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const double turns = (double)pos * (double)freq[i] * 0.15915494309189533577;
        const float r = (float)(turns - rint(turns)), quarters = rintf(4.f * r);
        const float x = fmaf(quarters, -0.25f, r) * 6.283185307179586f, x2 = x * x;
        const float sn = x * fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), 1.f);
        const float cs = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
        const int q = (int)quarters;
        const float a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;  // |cos|, |sin| of the whole angle; cos < 0 in quarters 1, 2, sin < 0 in 2, 3
        t.c[i] = ((q + 1) & 2 ? -a : a) * A.rope_scale;
        t.s[i] = (q & 2 ? -b : b) * A.rope_scale;
    }
}
__device__ __forceinline__ f32x4_t load_freq(const KvAppendArgs &A, uint32_t g) {  // (4-byte aligned)
    return f32x4_t{A.inv_freq[4 * g], A.inv_freq[4 * g + 1], A.inv_freq[4 * g + 2], A.inv_freq[4 * g + 3]};
}
__device__ __forceinline__ void rotate(Quad &q, const Turn &t) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = q.lo[i], b = q.hi[i];
        q.lo[i] = a * t.c[i] - b * t.s[i];
        q.hi[i] = b * t.c[i] + a * t.s[i];
    }
}
// rms norm over the LPH lanes of a head (lanes beyond head_dim hold zeros)
template <uint32_t LPH>
__device__ __forceinline__ void norm_quad(const KvAppendArgs &A, Quad &q, const Quad &w) {
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) sq = fmaf(q.lo[i], q.lo[i], fmaf(q.hi[i], q.hi[i], sq));
#pragma unroll
    for (uint32_t m = 1; m < LPH; m *= 2) sq += __shfl_xor(sq, (int)m, 64);
    const float r = 1.f / sqrtf(sq / (float)A.kv.head_dim + A.norm_eps);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        q.lo[i] *= r * (A.norm_offset + w.lo[i]);
        q.hi[i] *= r * (A.norm_offset + w.hi[i]);
    }
}

__device__ __forceinline__ uint32_t pack_fp8(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
__device__ __forceinline__ uint32_t rescale_fp8(uint32_t v, float ratio) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
    return pack_fp8(a[0] * ratio, a[1] * ratio, b[0] * ratio, b[1] * ratio);
}
__device__ __forceinline__ float pow2f(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// The page (sequence s, place j in its table) that is the item-th of all pages with new tokens; false beyond the last.
__device__ __forceinline__ bool find_page(const KvArgs &kv, uint32_t item, uint32_t &s, uint32_t &j) {
    const uint32_t lane = threadIdx.x % 64;
    for (uint32_t base = 0; base < kv.sequences; base += 64) {
        uint32_t pages = 0, first = 0;
        if (base + lane < kv.sequences) {
            const NewTokens t = new_tokens(kv, base + lane);
            if (t.n && t.len) {
                first = (uint32_t)max(t.len - (int32_t)t.n, 0) >> kv.page_shift;
                pages = ((uint32_t)(t.len - 1) >> kv.page_shift) - first + 1;
            }
        }
        const uint32_t upto = wave_inclusive_sum(pages), all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        if (item < all) {
            const uint32_t at = (uint32_t)__builtin_ctzll(__ballot(upto > item));
            s = base + at;
            j = (uint32_t)__builtin_amdgcn_readlane((int)(first + item - (upto - pages)), (int)at);
            return true;
        }
        item -= all;
    }
    return false;
}

// The sequence that row `token` belongs to: whichever holds it (row starts may fall between sequences: the one between is left out).
__device__ __forceinline__ bool find_token(const KvArgs &kv, uint32_t token, NewTokens &t) {
    const uint32_t lane = threadIdx.x % 64;
    for (uint32_t base = 0; base < kv.sequences; base += 64) {
        NewTokens of = {};
        if (base + lane < kv.sequences) of = new_tokens(kv, base + lane);
        const uint64_t holds = __ballot(token - of.row < of.n);  // (a row before the first wraps round)
        if (holds) {
            const int at = (int)__builtin_ctzll(holds);
            t.row = (uint32_t)__builtin_amdgcn_readlane((int)of.row, at);
            t.n = (uint32_t)__builtin_amdgcn_readlane((int)of.n, at);
            t.len = __builtin_amdgcn_readlane(of.len, at);
            return true;
        }
    }
    return false;
}

// A page's scale with its new elements: the exponent, and whether it is a number.  amax: the largest new |x| as bits (a NaN or an
// infinity above every number), older: tokens that the page held before.
struct Scale {
    int e, old_e;
    bool finite;
};
__device__ __forceinline__ Scale scale_of(uint32_t amax, bool older, float old_scale) {
    // 448 = 1.75 * 2^8: the smallest e with |x| <= 448 * 2^e
    Scale s;
    s.e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    s.finite = amax < 0x7F800000u && s.e <= kScaleMaxExp;
    s.e = max(s.e, kScaleMinExp);
    const uint32_t old_bits = __builtin_bit_cast(uint32_t, old_scale) & 0x7FFFFFFFu;
    s.old_e = (int)(old_bits >> 23) - 127;
    if (older) {
        s.finite = s.finite && old_bits < 0x7F800000u;
        s.e = max(s.e, s.old_e);
    }
    return s;
}
__device__ __forceinline__ float scale_value(const Scale &s) { return s.finite ? pow2f(s.e) : __builtin_nanf(""); }
__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t quad_amax(const Quad &q) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) m = max(m, max(abs_bits(q.lo[i]), abs_bits(q.hi[i])));
    return m;
}

// The codes of a page's older tokens, for a larger scale, by `threads` threads.
__device__ __forceinline__ void rescale_keys(uint8_t *codes, uint32_t head_dim, uint32_t older, float ratio, uint32_t thread, uint32_t threads) {
    for (uint32_t i = thread; i < older * head_dim / 4; i += threads) {
        uint32_t *at = (uint32_t *)codes + i;
        *at = rescale_fp8(*at, ratio);
    }
}
__device__ __forceinline__ void rescale_values(uint8_t *codes, uint32_t head_dim, uint32_t page_shift, uint32_t older, float ratio, uint32_t thread,
                                               uint32_t threads) {
    const uint32_t words = (older + 3) / 4;
    for (uint32_t i = thread; i < head_dim * words; i += threads) {
        const uint32_t c = i % words;
        uint32_t *at = (uint32_t *)(codes + ((size_t)(i / words) << page_shift)) + c;
        const uint32_t v = *at, keep = older - 4 * c >= 4 ? 0u : ~0u << (8 * (older - 4 * c));
        *at = (rescale_fp8(v & ~keep, ratio) & ~keep) | (v & keep);
    }
}

// The codes of a key's 8 channels.
__device__ __forceinline__ void store_key(const KvAppendArgs &A, uint8_t *row, uint32_t g, const Quad &q, float inv, bool finite) {
    uint32_t a = 0, b = 0;
    if (finite) {
        a = pack_fp8(q.lo[0] * inv, q.lo[1] * inv, q.lo[2] * inv, q.lo[3] * inv);
        b = pack_fp8(q.hi[0] * inv, q.hi[1] * inv, q.hi[2] * inv, q.hi[3] * inv);
    }
    if (halved(A, g)) {
        *(uint32_t *)(row + 4 * g) = a;
        *(uint32_t *)(row + 4 * g + A.rot_dim / 2) = b;
    } else {  // lo and hi alternate
        *(u32x2_t *)(row + 8 * g) = u32x2_t{__builtin_amdgcn_perm(b, a, 0x05010400u), __builtin_amdgcn_perm(b, a, 0x07030602u)};
    }
}

// One new token a sequence: LPH lanes (8 channels each) serve a head of it, keys, values and queries alike, with nothing to wait for but
// the loads (lengths and rows; the activations and the table; the page's scale).
template <uint32_t LPH>
__global__ void __launch_bounds__(kAppendThreads) kv_append_one_kernel(KvAppendArgs A, uint32_t blocks) {
    const KvArgs &kv = A.kv;
    const uint32_t s = block_number() / blocks, g = threadIdx.x % LPH;
    if (s >= kv.sequences) return;
    const uint32_t head = (block_number() % blocks) * (kAppendThreads / LPH) + threadIdx.x / LPH;  // keys, values, queries
    const bool is_k = head < kv.kv_heads, is_v = !is_k && head < 2 * kv.kv_heads, is_q = !is_k && !is_v && A.q && head < 2 * kv.kv_heads + A.q_heads;
    const bool in_head = 8 * g < kv.head_dim && (is_k || is_v || is_q), turns = 8 * g < A.rot_dim && !is_v;
    const NewTokens t = new_tokens(kv, s);
    if (t.n != 1) return;
    const uint32_t h = is_k ? head : is_v ? head - kv.kv_heads : head - 2 * kv.kv_heads;
    const float *norm = is_k ? A.k_norm : is_q ? A.q_norm : nullptr;
    Quad x = {}, w = {};
    f32x4_t freq = {0.f, 0.f, 0.f, 0.f};
    if (in_head) {
        const void *src = (const char *)(is_k ? A.k : is_v ? A.v : A.q) + t.row * (is_k ? A.k_stride : is_v ? A.v_stride : A.q_stride) * elem_bytes(A.type);
        const uint32_t at = h * kv.head_dim;
        if (is_v) {
            const Eight v = load8(src, A.type, at + 8 * g);
            x = {v.a, v.b};
        } else {
            x = load_quad(A, src, A.type, at, g);
            if (norm) w = load_quad(A, norm, ELEM_F32, 0, g);
            if (turns) freq = load_freq(A, g);
        }
    }
    const uint32_t slot = (uint32_t)max(t.len - 1, 0) & ((1u << kv.page_shift) - 1);
    const uint32_t page = is_q || t.len == 0 ? ~0u : kv_page(kv, kv.block_table + (size_t)s * kv.table_width, (uint32_t)(t.len - 1));
    const bool stored = (is_k || is_v) && page != ~0u;
    const size_t of_page = stored ? (size_t)page * kv.kv_heads + h : 0;
    float *scale_at = (is_v ? kv.v_scales : kv.k_scales) + of_page;
    const float old_scale = stored && slot ? *scale_at : 1.f;
    Quad y = x;
    if (A.q_norm || A.k_norm) norm_quad<LPH>(A, y, w);  // (whole wavefronts)
    if (norm) x = y;
    if (turns) {
        Turn turn;
        turn_of(A, t.len - 1, freq, turn);
        rotate(x, turn);
    }
    uint32_t amax = quad_amax(x);
#pragma unroll
    for (uint32_t m = 1; m < LPH; m *= 2) amax = max(amax, (uint32_t)__shfl_xor((int)amax, (int)m, 64));
    if (is_q && in_head) store_quad(A, (char *)A.q_out + t.row * A.q_out_stride * elem_bytes(A.type), A.type, h * kv.head_dim, g, x);
    if (!stored) return;
    const Scale sc = scale_of(amax, slot != 0, old_scale);
    uint8_t *codes = (is_v ? kv.v_codes : kv.k_codes) + of_page * ((size_t)kv.head_dim << kv.page_shift);
    if (sc.finite && slot && sc.e > sc.old_e) {
        const float ratio = pow2f(max(sc.old_e - sc.e, -126));
        if (is_v) rescale_values(codes, kv.head_dim, kv.page_shift, slot, ratio, g, LPH);
        else rescale_keys(codes, kv.head_dim, slot, ratio, g, LPH);
    }
    // (a word of a value row can hold older tokens and the new one: its bytes are written by the wavefront that rescaled the word,
    // after it, and to the same place in memory order)
    if (is_v) __threadfence_block();
    if (g == 0) *scale_at = scale_value(sc);
    if (!in_head) return;
    const float inv = sc.finite ? pow2f(-sc.e) : 0.f;
    if (is_k) {
        store_key(A, codes + (size_t)slot * kv.head_dim, g, x, inv, sc.finite);
    } else {
        uint32_t a = 0, b = 0;
        if (sc.finite) {
            a = pack_fp8(x.lo[0] * inv, x.lo[1] * inv, x.lo[2] * inv, x.lo[3] * inv);
            b = pack_fp8(x.hi[0] * inv, x.hi[1] * inv, x.hi[2] * inv, x.hi[3] * inv);
        }
        uint8_t *col = codes + ((size_t)(8 * g) << kv.page_shift) + slot;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            col[(size_t)i << kv.page_shift] = (uint8_t)(a >> (8 * i));
            col[(size_t)(4 + i) << kv.page_shift] = (uint8_t)(b >> (8 * i));
        }
    }
}

// Several new tokens a sequence.  A workgroup serves one head of one page, keys or values, or the queries of one token.  Keys and queries: LPH
// lanes (8 channels each) a head, kAppendThreads / LPH tokens or heads at once, NP times a page.  Values: a thread takes two channels of 16 keys,
// so that it stores the 16 bytes that lie together.
template <uint32_t LPH, int NP>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(KvAppendArgs A, uint32_t page_blocks) {
    constexpr uint32_t kTokens = kAppendThreads / LPH;
    constexpr int NV = (NP + 3) / 4;
    __shared__ uint32_t part[kAppendThreads / 64];
    const KvArgs &kv = A.kv;
    const uint32_t g0 = threadIdx.x % LPH, g = 8 * g0 < kv.head_dim ? g0 : 0;  // (lanes beyond head_dim load what another does)
    const bool in_head = 8 * g0 < kv.head_dim, turns = 8 * g < A.rot_dim;
    Quad w = {};
    f32x4_t freq = {0.f, 0.f, 0.f, 0.f};
    const uint32_t block = block_number();
    if (block >= page_blocks) {  // the queries of one token
        const uint32_t token = block - page_blocks, first = threadIdx.x / LPH;
        if (!A.q || token >= kv.tokens) return;
        const char *src = (const char *)A.q + token * A.q_stride * elem_bytes(A.type);
        char *dst = (char *)A.q_out + token * A.q_out_stride * elem_bytes(A.type);
        const auto load = [&](uint32_t head) { return load_quad(A, src, A.type, min(head, A.q_heads - 1) * kv.head_dim, g); };
        Quad q[2];  // (loads that nothing before them decides: they leave first, and the next heads' before these are done)
#pragma unroll
        for (uint32_t i = 0; i < 2; i++) q[i] = load(first + i * kTokens);
        if (turns) freq = load_freq(A, g);
        if (A.q_norm) w = load_quad(A, A.q_norm, ELEM_F32, 0, g);
        NewTokens t;
        if (!find_token(kv, token, t)) return;
        Turn turn;
        if (turns) turn_of(A, t.len - (int32_t)t.n + (int32_t)(token - t.row), freq, turn);
        for (uint32_t head0 = 0; head0 < A.q_heads; head0 += 2 * kTokens) {
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) {
                const uint32_t head = head0 + first + i * kTokens;
                Quad y = q[i];
                if (head0 + 2 * kTokens < A.q_heads) q[i] = load(head + 2 * kTokens);
                if (!in_head) y = {};
                if (A.q_norm) norm_quad<LPH>(A, y, w);
                if (turns) rotate(y, turn);
                if (in_head && head < A.q_heads) store_quad(A, dst, A.type, head * kv.head_dim, g, y);
            }
        }
        return;
    }
    const uint32_t part_of = block % (2 * kv.kv_heads), head = part_of % kv.kv_heads;
    const bool is_v = part_of >= kv.kv_heads;
    uint32_t s, j;
    if (!find_page(kv, block / (2 * kv.kv_heads), s, j)) return;
    const uint32_t page = kv_page(kv, kv.block_table + (size_t)s * kv.table_width, j << kv.page_shift);
    if (page == ~0u) return;
    const NewTokens t = new_tokens(kv, s);
    const uint32_t P = 1u << kv.page_shift, base = j << kv.page_shift;
    const int32_t first = t.len - (int32_t)t.n;             // position of the sequence's first new token
    const uint32_t lo = (uint32_t)max(first, (int32_t)base) - base, hi = min((uint32_t)t.len - base, P);  // new slots of this page
    float *scale_at = (is_v ? kv.v_scales : kv.k_scales) + (size_t)page * kv.kv_heads + head;
    const float old_scale = lo ? *scale_at : 1.f;
    uint8_t *codes = (is_v ? kv.v_codes : kv.k_codes) + ((size_t)page * kv.kv_heads + head) * ((size_t)kv.head_dim << kv.page_shift);
    // this head's elements of the page's first new token, and how far a slot's are from there (the nearest new slot's: loads need no condition)
    const char *src = (const char *)(is_v ? A.v : A.k) +
                      ((t.row + (size_t)((int32_t)(base + lo) - first)) * (is_v ? A.v_stride : A.k_stride) + (size_t)head * kv.head_dim) * elem_bytes(A.type);
    const uint32_t stride = (uint32_t)(is_v ? A.v_stride : A.k_stride);  // (at most kMaxRowStride: 128 rows within 32 bits)
    const auto off_of = [&](uint32_t slot) { return (min(max(slot, lo), hi - 1) - lo) * stride; };
    const auto page_scale = [&](uint32_t amax) {
        amax = wave_max_u32(amax);
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = amax;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kAppendThreads / 64; i++) amax = max(amax, part[i]);
        const Scale sc = scale_of(amax, lo != 0, old_scale);
        if (threadIdx.x == 0) *scale_at = scale_value(sc);
        return sc;
    };
    uint32_t amax = 0;
    if (!is_v) {
        Quad x[NP];
#pragma unroll
        for (int p = 0; p < NP; p++)
            x[p] = load_quad(A, src, A.type, off_of((uint32_t)p * kTokens + threadIdx.x / LPH), g);
        if (turns) freq = load_freq(A, g);
        if (A.k_norm) w = load_quad(A, A.k_norm, ELEM_F32, 0, g);
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const uint32_t slot = (uint32_t)p * kTokens + threadIdx.x / LPH;
            if (!in_head) x[p] = {};
            if (A.k_norm) norm_quad<LPH>(A, x[p], w);
            if (turns) {
                Turn turn;
                turn_of(A, (int32_t)(base + slot), freq, turn);
                rotate(x[p], turn);
            }
            if (in_head && slot >= lo && slot < hi) amax = max(amax, quad_amax(x[p]));
        }
        const Scale sc = page_scale(amax);
        if (sc.finite && lo && sc.e > sc.old_e) rescale_keys(codes, kv.head_dim, lo, pow2f(max(sc.old_e - sc.e, -126)), threadIdx.x, kAppendThreads);
        const float inv = sc.finite ? pow2f(-sc.e) : 0.f;
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const uint32_t slot = (uint32_t)p * kTokens + threadIdx.x / LPH;
            if (in_head && slot >= lo && slot < hi) store_key(A, codes + (size_t)slot * kv.head_dim, g, x[p], inv, sc.finite);
        }
        return;
    }
    const uint32_t pairs = kv.head_dim / 2, units = pairs * (P / 16);  // (16 keys, two channels) each
    f32x2_t x[NV][16];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const uint32_t u = min(threadIdx.x + (uint32_t)v * kAppendThreads, units - 1), d = u % pairs * 2, slot0 = u / pairs * 16;
#pragma unroll
        for (int i = 0; i < 16; i++) x[v][i] = load2(src, A.type, off_of(slot0 + (uint32_t)i) + d);
    }
#pragma unroll
    for (int v = 0; v < NV; v++)  // (other threads' units and other slots' rows: elements of this page's new tokens all the same)
#pragma unroll
        for (int i = 0; i < 16; i++) amax = max(amax, max(abs_bits(x[v][i][0]), abs_bits(x[v][i][1])));
    const Scale sc = page_scale(amax);
    if (sc.finite && lo && sc.e > sc.old_e) {
        rescale_values(codes, kv.head_dim, kv.page_shift, lo, pow2f(max(sc.old_e - sc.e, -126)), threadIdx.x, kAppendThreads);
        __syncthreads();  // (a word of a value row can hold older and new tokens)
    }
    const float inv = sc.finite ? pow2f(-sc.e) : 0.f;
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const uint32_t u = threadIdx.x + (uint32_t)v * kAppendThreads, d = u % pairs * 2, slot0 = u / pairs * 16;
        if (u >= units || slot0 >= hi || slot0 + 16 <= lo) continue;
#pragma unroll
        for (int c = 0; c < 2; c++) {
            u32x4_t code = {0u, 0u, 0u, 0u};
            if (sc.finite)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    code[i] = pack_fp8(x[v][4 * i][c] * inv, x[v][4 * i + 1][c] * inv, x[v][4 * i + 2][c] * inv, x[v][4 * i + 3][c] * inv);
            uint8_t *at = codes + ((size_t)(d + (uint32_t)c) << kv.page_shift) + slot0;
            if (slot0 >= lo && slot0 + 16 <= hi) {
                *(u32x4_t *)at = code;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 16; i++)
                    if (slot0 + i >= lo && slot0 + i < hi) at[i] = (uint8_t)(code[i / 4] >> (8 * (i % 4)));
            }
        }
    }
}

template <uint32_t LPH>
static void launch_lanes(hipStream_t s, const KvAppendArgs &A, uint32_t page_blocks, dim3 grid) {
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kAppendThreads), 0, s, A, page_blocks); };
    constexpr auto passes = [](uint32_t page_tokens) { return (int)((LPH * page_tokens + kAppendThreads - 1) / kAppendThreads); };
    switch (A.kv.page_shift) {
    case 4: return launch(kv_append_kernel<LPH, passes(16)>);
    case 5: return launch(kv_append_kernel<LPH, passes(32)>);
    case 6: return launch(kv_append_kernel<LPH, passes(64)>);
    default: return launch(kv_append_kernel<LPH, passes(128)>);
    }
}

// Lanes of a head; one new token a sequence: workgroups of a sequence.
static uint32_t lanes_of(const KvArgs &kv) { return kv.head_dim <= 32 ? 4 : kv.head_dim <= 64 ? 8 : kv.head_dim <= 128 ? 16 : 32; }
static uint32_t one_blocks(const KvAppendArgs &A) {
    return ((2 * A.kv.kv_heads + (A.q ? A.q_heads : 0)) * lanes_of(A.kv) + kAppendThreads - 1) / kAppendThreads;
}
// Several: n new tokens touch at most (n + 2 P - 2) / P pages.
static uint64_t page_blocks_of(const KvArgs &kv) {
    const uint64_t P = 1u << kv.page_shift;
    return (kv.tokens + kv.sequences * (2 * P - 2)) / P * 2 * kv.kv_heads;
}
uint64_t kv_append_blocks(const KvAppendArgs &A) {
    return A.kv.max_new == 1 ? (uint64_t)A.kv.sequences * one_blocks(A) : page_blocks_of(A.kv) + (A.q ? A.kv.tokens : 0);
}

hipError_t kv_append_launch(hipStream_t s, const KvAppendArgs &A) {
    const dim3 grid = grid_of(kv_append_blocks(A)), threads(kAppendThreads);
    const uint32_t lanes = lanes_of(A.kv);
    if (A.kv.max_new == 1) {
        const uint32_t blocks = one_blocks(A);
        if (lanes == 4) hipLaunchKernelGGL(kv_append_one_kernel<4>, grid, threads, 0, s, A, blocks);
        else if (lanes == 8) hipLaunchKernelGGL(kv_append_one_kernel<8>, grid, threads, 0, s, A, blocks);
        else if (lanes == 16) hipLaunchKernelGGL(kv_append_one_kernel<16>, grid, threads, 0, s, A, blocks);
        else hipLaunchKernelGGL(kv_append_one_kernel<32>, grid, threads, 0, s, A, blocks);
        return hipGetLastError();
    }
    const uint32_t page_blocks = (uint32_t)page_blocks_of(A.kv);
    if (lanes == 4) launch_lanes<4>(s, A, page_blocks, grid);
    else if (lanes == 8) launch_lanes<8>(s, A, page_blocks, grid);
    else if (lanes == 16) launch_lanes<16>(s, A, page_blocks, grid);
    else launch_lanes<32>(s, A, page_blocks, grid);
    return hipGetLastError();
}

}  // namespace larql
