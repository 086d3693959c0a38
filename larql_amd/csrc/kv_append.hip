// kv_append.hip — new queries, keys and values of a step's sequences: rms norm per head, rotation by position, and keys and values
// as e4m3 codes into the pages of the cache, a power-of-two scale for each page and head.
//
// A workgroup owns one head of one page that gets new tokens, so the page's scale is decided and its codes are written in one
// place, with no atomics: the new elements stay in registers between the largest |x| and the codes.  Where the scale of a page with
// older tokens grows, their codes are rounded again for it (a power of two: exact unless a code becomes subnormal).
#include "kernels.h"
#include "layer.h"

namespace larql {

constexpr uint32_t kAppendThreads = 256;

// 8 channels of one head and token, as four pairs (lo[i], hi[i]) that turn together
struct Quad {
    float lo[4], hi[4];
};

// Channels of the pairs 4g .. 4g+3: (p, p + rot/2) inside the rotated part of a halved layout, else (2p, 2p + 1).
__device__ __forceinline__ bool halved(const KvAppendArgs &A, uint32_t g) { return !A.interleaved && 8 * g < A.rot_dim; }
__device__ __forceinline__ void load_quad(const KvAppendArgs &A, const void *row, int type, size_t at, uint32_t g, Quad &q) {
    if (halved(A, g)) {
        load4(row, type, at + 4 * g, q.lo);
        load4(row, type, at + 4 * g + A.rot_dim / 2, q.hi);
    } else {
        float x[8];
        load8(row, type, at + 8 * g, x);
#pragma unroll
        for (int i = 0; i < 4; i++) q.lo[i] = x[2 * i], q.hi[i] = x[2 * i + 1];
    }
}
__device__ __forceinline__ void store_quad(const KvAppendArgs &A, void *row, int type, size_t at, uint32_t g, const Quad &q) {
    if (halved(A, g)) {
        store4(row, type, at + 4 * g, q.lo);
        store4(row, type, at + 4 * g + A.rot_dim / 2, q.hi);
    } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; i++) x[2 * i] = q.lo[i], x[2 * i + 1] = q.hi[i];
        store8(row, type, at + 8 * g, x);
    }
}

// cos and sin of position * inv_freq[4g + i], times rope_scale.  Far positions lose the angle in 32 bits: whole turns leave in 64.
struct Turn {
    float c[4], s[4];
};
__device__ __forceinline__ void turn_of(const KvAppendArgs &A, int32_t pos, uint32_t g, Turn &t) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const double turns = (double)pos * (double)A.inv_freq[4 * g + i] * 0.15915494309189533577;
        sincospif(2.f * (float)(turns - rint(turns)), &t.s[i], &t.c[i]);
        t.s[i] *= A.rope_scale;
        t.c[i] *= A.rope_scale;
    }
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
    if (kv.max_new == 1) {  // at most one page for each sequence
        s = item;
        const NewTokens t = new_tokens(kv, s);
        j = (uint32_t)(t.len - 1) >> kv.page_shift;
        return t.n == 1 && t.len > 0;
    }
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

// The sequence that row `token` belongs to.
__device__ __forceinline__ bool find_token(const KvArgs &kv, uint32_t token, NewTokens &t) {
    const uint32_t lane = threadIdx.x % 64;
    uint32_t s = 0;
    for (uint32_t base = 0; base < kv.sequences; base += 64) {
        const bool before = base + lane < kv.sequences && kv.q_start[base + lane + 1] <= (int32_t)token;
        s += (uint32_t)__popcll(__ballot(before));
    }
    if (s >= kv.sequences) return false;
    t = new_tokens(kv, s);
    return token >= t.row && token - t.row < t.n;
}

// LPH lanes (8 channels each) serve a token of a head, kAppendThreads / LPH tokens at once, NP times a page.
template <uint32_t LPH, int NP>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(KvAppendArgs A, uint32_t page_blocks) {
    constexpr uint32_t kTokens = kAppendThreads / LPH;
    __shared__ uint32_t part[kAppendThreads / 64];
    const KvArgs &kv = A.kv;
    const uint32_t g = threadIdx.x % LPH;
    const bool in_head = 8 * g < kv.head_dim, turns = 8 * g < A.rot_dim;
    Quad w;
    if (blockIdx.x >= page_blocks) {  // the queries of one token
        const uint32_t token = blockIdx.x - page_blocks;
        NewTokens t;
        if (!find_token(kv, token, t)) return;
        Turn turn;
        if (turns) turn_of(A, t.len - (int32_t)t.n + (int32_t)(token - t.row), g, turn);
        if (A.q_norm && in_head) load_quad(A, A.q_norm, ELEM_F32, 0, g, w);
        for (uint32_t head = threadIdx.x / LPH; head < (A.q_heads + kTokens - 1) / kTokens * kTokens; head += kTokens) {
            Quad q = {};
            const bool live = in_head && head < A.q_heads;
            if (live) load_quad(A, A.q, A.type, token * A.q_stride + (size_t)head * kv.head_dim, g, q);
            if (A.q_norm) norm_quad<LPH>(A, q, w);
            if (turns) rotate(q, turn);
            if (live) store_quad(A, A.q_out, A.type, token * A.q_out_stride + (size_t)head * kv.head_dim, g, q);
        }
        return;
    }
    const uint32_t part_of = blockIdx.x % (2 * kv.kv_heads), head = part_of % kv.kv_heads;
    const bool is_v = part_of >= kv.kv_heads;
    uint32_t s, j;
    if (!find_page(kv, blockIdx.x / (2 * kv.kv_heads), s, j)) return;
    const uint32_t page = kv_page(kv, kv.block_table + (size_t)s * kv.table_width, j << kv.page_shift);
    if (page == ~0u) return;
    const NewTokens t = new_tokens(kv, s);
    const uint32_t P = 1u << kv.page_shift, base = j << kv.page_shift;
    const int32_t first = t.len - (int32_t)t.n;             // position of the sequence's first new token
    const uint32_t lo = (uint32_t)max(first, (int32_t)base) - base, hi = min((uint32_t)t.len - base, P);  // new slots of this page
    float *scale_at = (is_v ? kv.v_scales : kv.k_scales) + (size_t)page * kv.kv_heads + head;
    const float old_scale = lo ? *scale_at : 1.f;

    // pass 1: the new elements, and the largest |x| as bits (a NaN or an infinity above every number)
    const void *src = is_v ? A.v : A.k;
    const size_t stride = is_v ? A.v_stride : A.k_stride;
    const bool with_norm = !is_v && A.k_norm;
    if (with_norm && in_head) load_quad(A, A.k_norm, ELEM_F32, 0, g, w);
    Quad x[NP];
    uint32_t amax = 0;
#pragma unroll
    for (int p = 0; p < NP; p++) {
        const uint32_t slot = (uint32_t)p * kTokens + threadIdx.x / LPH;
        const bool live = in_head && slot >= lo && slot < hi;
        x[p] = {};
        if (live) {
            const size_t at = (t.row + (size_t)((int32_t)(base + slot) - first)) * stride + (size_t)head * kv.head_dim;
            if (is_v) {
                float v[8];
                load8(src, A.type, at + 8 * g, v);
#pragma unroll
                for (int i = 0; i < 4; i++) x[p].lo[i] = v[i], x[p].hi[i] = v[4 + i];
            } else {
                load_quad(A, src, A.type, at, g, x[p]);
            }
        }
        if (with_norm) norm_quad<LPH>(A, x[p], w);
        if (!is_v && turns && live) {
            Turn turn;
            turn_of(A, (int32_t)(base + slot), g, turn);
            rotate(x[p], turn);
        }
        if (live)
#pragma unroll
            for (int i = 0; i < 4; i++)
                amax = max(amax, max(__builtin_bit_cast(uint32_t, x[p].lo[i]) & 0x7FFFFFFFu, __builtin_bit_cast(uint32_t, x[p].hi[i]) & 0x7FFFFFFFu));
    }
    amax = wave_max_u32(amax);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = amax;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kAppendThreads / 64; i++) amax = max(amax, part[i]);

    // 448 = 1.75 * 2^8: the smallest e with |x| <= 448 * 2^e
    int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    bool finite = amax < 0x7F800000u && e <= kScaleMaxExp;
    e = max(e, kScaleMinExp);
    const uint32_t old_bits = __builtin_bit_cast(uint32_t, old_scale) & 0x7FFFFFFFu;
    if (lo) {
        finite = finite && old_bits < 0x7F800000u;
        e = max(e, (int)(old_bits >> 23) - 127);
    }
    uint8_t *codes = (is_v ? kv.v_codes : kv.k_codes) + ((size_t)page * kv.kv_heads + head) * ((size_t)kv.head_dim << kv.page_shift);
    if (finite && lo && e > (int)(old_bits >> 23) - 127) {  // the older tokens' codes, for the larger scale
        const float ratio = pow2f(max((int)(old_bits >> 23) - 127 - e, -126));
        if (is_v) {
            const uint32_t words = (lo + 3) / 4;
            for (uint32_t i = threadIdx.x; i < kv.head_dim * words; i += kAppendThreads) {
                const uint32_t c = i % words;
                uint32_t *at = (uint32_t *)(codes + ((size_t)(i / words) << kv.page_shift)) + c;
                const uint32_t v = *at, keep = lo - 4 * c >= 4 ? 0u : ~0u << (8 * (lo - 4 * c));
                *at = (rescale_fp8(v & ~keep, ratio) & ~keep) | (v & keep);
            }
        } else {
            for (uint32_t i = threadIdx.x; i < lo * kv.head_dim / 4; i += kAppendThreads) {
                uint32_t *at = (uint32_t *)codes + i;
                *at = rescale_fp8(*at, ratio);
            }
        }
    }
    if (threadIdx.x == 0) *scale_at = finite ? pow2f(e) : __builtin_nanf("");
    if (is_v) __syncthreads();  // (a word of a value row can hold older and new tokens)

    // pass 2: the codes
    const float inv = finite ? pow2f(-e) : 0.f;
#pragma unroll
    for (int p = 0; p < NP; p++) {
        const uint32_t slot = (uint32_t)p * kTokens + threadIdx.x / LPH;
        if (!in_head || slot < lo || slot >= hi) continue;
        uint32_t a = 0, b = 0;  // codes of lo[], hi[]
        if (finite) {
            a = pack_fp8(x[p].lo[0] * inv, x[p].lo[1] * inv, x[p].lo[2] * inv, x[p].lo[3] * inv);
            b = pack_fp8(x[p].hi[0] * inv, x[p].hi[1] * inv, x[p].hi[2] * inv, x[p].hi[3] * inv);
        }
        if (is_v) {
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                codes[((size_t)(8 * g + i) << kv.page_shift) + slot] = (uint8_t)(a >> (8 * i));
                codes[((size_t)(8 * g + 4 + i) << kv.page_shift) + slot] = (uint8_t)(b >> (8 * i));
            }
        } else if (halved(A, g)) {
            *(uint32_t *)(codes + (size_t)slot * kv.head_dim + 4 * g) = a;
            *(uint32_t *)(codes + (size_t)slot * kv.head_dim + 4 * g + A.rot_dim / 2) = b;
        } else {  // lo and hi alternate
            const uint32_t c = (a & 0xFFu) | (b & 0xFFu) << 8 | (a & 0xFF00u) << 8 | (b & 0xFF00u) << 16;
            const uint32_t d = (a >> 16 & 0xFFu) | (b >> 16 & 0xFFu) << 8 | (a >> 24) << 16 | (b >> 24) << 24;
            *(u32x2_t *)(codes + (size_t)slot * kv.head_dim + 8 * g) = u32x2_t{c, d};
        }
    }
}

template <uint32_t LPH>
static void launch_lanes(hipStream_t s, const KvAppendArgs &A, uint32_t page_blocks, uint32_t grid) {
    const uint32_t passes = (1u << A.kv.page_shift) * LPH / kAppendThreads;
#define LARQL_APPEND(NP) hipLaunchKernelGGL((kv_append_kernel<LPH, NP>), dim3(grid), dim3(kAppendThreads), 0, s, A, page_blocks)
    if (passes <= 1) LARQL_APPEND(1);
    else if (passes <= 2) LARQL_APPEND(2);
    else if (passes <= 4) LARQL_APPEND(4);
    else if (passes <= 8) LARQL_APPEND(8);
    else LARQL_APPEND(16);
#undef LARQL_APPEND
}

hipError_t kv_append_launch(hipStream_t s, const KvAppendArgs &A) {
    const KvArgs &kv = A.kv;
    const uint64_t P = 1u << kv.page_shift;
    // n new tokens touch at most (n + 2 P - 2) / P pages, one token one
    const uint64_t pages = kv.max_new == 1 ? kv.sequences : (kv.tokens + kv.sequences * (2 * P - 2)) / P;
    const uint64_t page_blocks = pages * 2 * kv.kv_heads, grid = page_blocks + (A.q ? kv.tokens : 0);
    if (grid > 0x7FFFFFFFull) return hipErrorInvalidValue;
    if (grid == 0) return hipSuccess;
    const uint32_t groups = kv.head_dim / 8;
    if (groups <= 4) launch_lanes<4>(s, A, (uint32_t)page_blocks, (uint32_t)grid);
    else if (groups <= 8) launch_lanes<8>(s, A, (uint32_t)page_blocks, (uint32_t)grid);
    else if (groups <= 16) launch_lanes<16>(s, A, (uint32_t)page_blocks, (uint32_t)grid);
    else launch_lanes<32>(s, A, (uint32_t)page_blocks, (uint32_t)grid);
    return hipGetLastError();
}

}  // namespace larql
