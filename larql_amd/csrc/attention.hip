// attention.hip — attention of a step's new tokens over the paged 8-bit cache.
//
// Scores are formed transposed, S^T = K . Q^T, keys down the rows of a matrix instruction and query rows (token, head of the group)
// across its columns: a lane then holds weights of ONE query row for 16 keys of each step, in the order in which the second product
// O^T = V^T . P^T takes its operand, so the weights never leave the registers.  Which key is which row of S^T is free: row 4g + r
// of tile t is key 16g + 4t + r of a step of 64, so lane group g holds keys 16g .. 16g+15 — the 16 bytes that it loads of a value
// channel's row.
//
// Codes are exact in f16.  The key scale enters the scores' factor and the value scale, a power of two 2^e, the exponent:
//   weight 2^(t + e - M), M the running maximum of t + e, times the bare code;  sum of weights: 2^(t + e - M) * 2^-e.
// So neither costs an instruction for each element, and numerators keep their precision whatever the blocks' scales.
#include <algorithm>

#include "kernels.h"
#include "layer.h"

namespace larql {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr uint32_t kStep = 64;          // keys of a step
constexpr uint32_t kAttnThreads = 256;
constexpr uint32_t kAttnWaves = kAttnThreads / 64;
constexpr uint32_t kTile = 16;          // query rows of a workgroup
constexpr uint32_t kTargetItems = 1024; // pieces that long rows are split into, over all heads
constexpr uint32_t kMinSteps = 4;       // steps of a piece at least
constexpr float kLog2E = 1.44269504088896341f;
// Weights are held as 2^(t + e - M + 12) with t + e - M <= 3, so that the f16 pair of an f32 weight keeps 22 bits down to 2^-15 of the
// largest and 2^-37 of it beyond; M only moves where a score leaves that range.
constexpr float kBias = 12.f, kSlack = 3.f;
constexpr float kNoMax = -1e30f;

// A sequence's share of the work: its query rows in tiles, and the steps of keys that any of them sees.
struct Share {
    uint32_t row, n;      // first row of the activations, new tokens
    int32_t len, first;   // keys, position of the first new token
    uint32_t tiles, step_lo, steps;
};
__device__ __forceinline__ Share share_of(const AttentionArgs &A, uint32_t s, uint32_t group) {
    const NewTokens t = new_tokens(A.kv, s);
    Share h;
    h.row = t.row;
    h.n = t.n;
    h.len = (int32_t)min((uint64_t)t.len, (uint64_t)A.kv.table_width << A.kv.page_shift);
    h.first = t.len - (int32_t)t.n;
    h.tiles = (t.n * group + kTile - 1) / kTile;
    const int32_t lo = A.window ? (int32_t)max((int64_t)h.first - (int64_t)A.window + 1, (int64_t)0) : 0;
    h.step_lo = (uint32_t)lo / kStep;
    h.steps = h.n && h.len > lo ? ((uint32_t)h.len + kStep - 1) / kStep - h.step_lo : 0;
    return h;
}

// What the wavefront that serves item `item` of a head works on; false beyond the last.  Every wavefront finds it from the lengths:
// pieces of `chunk` steps, as many as kTargetItems over all heads asks for.
struct Item {
    uint32_t s, tile, piece, pieces, chunk;
};
__device__ __forceinline__ bool find_item(const AttentionArgs &A, uint32_t item, bool by_tile, Item &it, uint32_t &first_item) {
    const uint32_t lane = threadIdx.x % 64, group = A.q_heads / A.kv.kv_heads;
    float units = 0.f;  // (tiles x steps; their sum need not be exact)
    for (uint32_t base = 0; base < A.kv.sequences; base += 64)
        if (base + lane < A.kv.sequences) {
            const Share h = share_of(A, base + lane, group);
            units += (float)h.tiles * (float)h.steps;
        }
    units = wave_fsum(units);
    const uint32_t target = max(kTargetItems / A.kv.kv_heads, 1u);
    const uint32_t chunk = max((uint32_t)ceilf(units / (float)target), kMinSteps);
    first_item = 0;
    for (uint32_t base = 0; base < A.kv.sequences; base += 64) {
        uint32_t tiles = 0, pieces = 1;
        if (base + lane < A.kv.sequences) {
            const Share h = share_of(A, base + lane, group);
            tiles = h.tiles;
            pieces = max((h.steps + chunk - 1) / chunk, 1u);
        }
        const uint32_t weight = by_tile ? tiles : tiles * pieces;
        const uint32_t upto = wave_inclusive_sum(weight), all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        const uint32_t items_upto = by_tile ? wave_inclusive_sum(tiles * pieces) : upto;
        if (item < all) {
            const int at = (int)__builtin_ctzll(__ballot(upto > item));
            it.pieces = (uint32_t)__builtin_amdgcn_readlane((int)pieces, at);
            const uint32_t in = item - (uint32_t)__builtin_amdgcn_readlane((int)(upto - weight), at);
            it.s = base + (uint32_t)at;
            it.tile = by_tile ? in : in / it.pieces;
            it.piece = by_tile ? 0 : in % it.pieces;
            it.chunk = chunk;
            first_item += (uint32_t)__builtin_amdgcn_readlane((int)(items_upto - tiles * pieces), at) + it.tile * it.pieces;
            return true;
        }
        item -= all;
        first_item += (uint32_t)__builtin_amdgcn_readlane((int)items_upto, 63);
    }
    return false;
}

// Items of one head at most: every sequence's last piece may be short.
static uint64_t items_bound(const AttentionArgs &A) {
    const uint64_t group = A.q_heads / A.kv.kv_heads;
    const uint64_t tiles = A.kv.tokens * group / kTile + A.kv.sequences;
    return tiles + std::max(kTargetItems / A.kv.kv_heads, 1u) + 1;
}

// 8 codes as f16
__device__ __forceinline__ f16x8_t codes_f16(u32x2_t v) {
    f16x8_t o;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const f16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)v[i], 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)v[i], 1.f, true);
        o[4 * i] = a[0], o[4 * i + 1] = a[1], o[4 * i + 2] = b[0], o[4 * i + 3] = b[1];
    }
    return o;
}

// Partial results of a piece: [items][kTile][head_dim] weighted sums, then [items][kTile] maxima and sums of weights.
struct Partials {
    float *acc, *ml;
};

template <int NK, bool PAIRS, bool CAP>
__global__ void __launch_bounds__(kAttnThreads, NK > 4 ? 1 : 2) attention_rows_kernel(AttentionArgs A, Partials part) {
    constexpr uint32_t D = NK * 32, kPad = D + 4;
    __shared__ float sh_acc[kAttnWaves][kTile][kPad];
    __shared__ float sh_ml[kAttnWaves][kTile][2];
    const KvArgs &kv = A.kv;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, n = lane % 16, g = lane / 16;
    const uint32_t kvh = blockIdx.y, group = A.q_heads / kv.kv_heads;
    Item it;
    uint32_t first_item;
    if (!find_item(A, blockIdx.x, false, it, first_item)) return;
    const Share sh = share_of(A, it.s, group);

    // The lane's query row: token and head, what it sees, its elements as f16 after a power-of-two scale.
    const uint32_t row = it.tile * kTile + n, tok = row / group, head = kvh * group + row % group;
    const bool live = tok < sh.n;
    const int32_t pos = sh.first + (int32_t)tok;
    const int32_t key_hi = !live ? -1 : (A.causal ? min(pos, sh.len - 1) : sh.len - 1);
    const int32_t key_lo = A.window ? (int32_t)max((int64_t)pos - (int64_t)A.window + 1, (int64_t)0) : 0;
    f16x8_t qh[NK], ql[PAIRS ? NK : 1];
    float factor;
    {
        float q[NK][8];
        uint32_t amax = 0;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const uint32_t d = (k | 1) < NK ? (uint32_t)(k & ~1) * 32 + g * 16 + (uint32_t)(k & 1) * 8 : (uint32_t)k * 32 + g * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) q[k][i] = 0.f;
            if (live) load8(A.q, A.q_type, (size_t)(sh.row + tok) * A.q_stride + (size_t)head * D + d, q[k]);
#pragma unroll
            for (int i = 0; i < 8; i++) amax = max(amax, __builtin_bit_cast(uint32_t, q[k][i]) & 0x7FFFFFFFu);
        }
        amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16, 64));
        amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32, 64));
        // largest |q| to [2^14, 2^15)
        const int e = max((int)(amax >> 23) - 127, -100) - 14;
        const float inv = __builtin_bit_cast(float, (uint32_t)(127 - min(max(e, -126), 126)) << 23);
        factor = A.scale * __builtin_bit_cast(float, (uint32_t)(127 + min(max(e, -126), 126)) << 23);
        if (amax >= 0x7F800000u) factor = __builtin_nanf("");
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float x = amax >= 0x7F800000u ? 0.f : q[k][i] * inv;
                qh[k][i] = (_Float16)x;
                if constexpr (PAIRS) ql[k][i] = (_Float16)(x - (float)qh[k][i]);
            }
        if constexpr (!CAP) factor *= kLog2E;
    }
    // steps that every live row of the tile sees whole need no mask
    int32_t all_hi = live ? key_hi : 0x7FFFFFFF, all_lo = live ? key_lo : 0;
    int32_t any_hi = key_hi, any_lo = live ? key_lo : 0x7FFFFFFF;
#pragma unroll
    for (int m = 1; m < 16; m *= 2) {
        all_hi = min(all_hi, __shfl_xor(all_hi, m, 64));
        all_lo = max(all_lo, __shfl_xor(all_lo, m, 64));
        any_hi = max(any_hi, __shfl_xor(any_hi, m, 64));
        any_lo = min(any_lo, __shfl_xor(any_lo, m, 64));
    }
    all_hi = __builtin_amdgcn_readfirstlane(all_hi), all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    any_hi = __builtin_amdgcn_readfirstlane(any_hi), any_lo = __builtin_amdgcn_readfirstlane(any_lo);

    const int32_t *table = kv.block_table + (size_t)it.s * kv.table_width;
    const uint32_t page_mask = (1u << kv.page_shift) - 1;
    const size_t head_codes = (size_t)D << kv.page_shift;
    f32x4_t acc[2 * NK];
#pragma unroll
    for (int i = 0; i < 2 * NK; i++) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float M = kNoMax, L = 0.f;

    // Steps of this piece that some row sees, every kAttnWaves-th of them this wavefront's.  A step's page numbers are read two steps
    // ahead, its key codes one step ahead (while the step before multiplies values), its value codes while its scores form: a
    // wavefront always has a load of its own 64 x head_dim bytes or more in flight.
    const uint32_t step_end = any_hi < 0 ? 0u : min(min(sh.step_lo + (it.piece + 1) * it.chunk, sh.step_lo + sh.steps), (uint32_t)any_hi / kStep + 1);
    uint32_t step = max(sh.step_lo + it.piece * it.chunk, any_lo == 0x7FFFFFFF ? step_end : (uint32_t)any_lo / kStep) + wave;
    const uint32_t gk = n / 4;  // this lane loads keys of group gk, and values and weights of group g, of a step
    const auto page_of = [&](uint32_t st, uint32_t grp) -> uint32_t {
        const uint32_t key = st * kStep + grp * 16;
        return st >= step_end || (int32_t)key >= sh.len ? ~0u : kv_page(kv, table, key);
    };
    u32x4_t kc[4][(NK + 1) / 2], vc[2 * NK];
    float ks = 0.f, vs = 1.f;
    const auto load_keys = [&](uint32_t st, uint32_t page_k, uint32_t page_v) {
        const uint8_t *kp = kv.k_codes + ((size_t)(page_k == ~0u ? 0u : page_k) * kv.kv_heads + kvh) * head_codes +
                            (size_t)((st * kStep + gk * 16) & page_mask) * D;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int k = 0; k < NK; k += 2) {
                const uint8_t *kr = kp + (size_t)(4 * t + n % 4) * D + k * 32;
                if (k + 1 < NK) {
                    kc[t][k / 2] = *(const u32x4_t *)(kr + g * 16);
                } else {
                    const u32x2_t c = *(const u32x2_t *)(kr + g * 8);
                    kc[t][k / 2] = u32x4_t{c[0], c[1], 0u, 0u};
                }
            }
        const size_t at = (size_t)(page_v == ~0u ? 0u : page_v) * kv.kv_heads + kvh;
        ks = kv.k_scales[at];
        vs = kv.v_scales[at];
    };
    uint32_t page_k = page_of(step, gk), page_v = page_of(step, g);
    if (step < step_end) load_keys(step, page_k, page_v);
    uint32_t next_k = page_of(step + kAttnWaves, gk), next_v = page_of(step + kAttnWaves, g);

    for (; step < step_end; step += kAttnWaves) {
        const int32_t key0 = (int32_t)(step * kStep);
        const bool hole = page_v == ~0u;
        {
            const uint8_t *vp = kv.v_codes + ((size_t)(hole ? 0u : page_v) * kv.kv_heads + kvh) * head_codes + (((uint32_t)key0 + g * 16) & page_mask);
#pragma unroll
            for (int d = 0; d < 2 * NK; d++) vc[d] = *(const u32x4_t *)(vp + ((size_t)(d * 16 + n) << kv.page_shift));
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t S[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            S[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NK; k++) {
                const u32x4_t c = kc[t][k / 2];
                const f16x8_t ka = codes_f16(k % 2 ? u32x2_t{c[2], c[3]} : u32x2_t{c[0], c[1]});
                S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh[k], S[t], 0, 0, 0);
                if constexpr (PAIRS) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql[k], S[t], 0, 0, 0);
            }
        }
        float cur_ks = ks;
        const float cur_vs = vs;
        __builtin_amdgcn_sched_barrier(0);
        page_k = next_k, page_v = next_v;
        if (step + kAttnWaves < step_end) {
            load_keys(step + kAttnWaves, page_k, page_v);
            next_k = page_of(step + 2 * kAttnWaves, gk), next_v = page_of(step + 2 * kAttnWaves, g);
        }
        __builtin_amdgcn_sched_barrier(0);
        // Logarithms (base 2) of the weights times the value scale.  A scale that is not a number makes its tokens' scores NaN.
        const bool odd = !(cur_vs == cur_vs);
        if (odd) cur_ks = __builtin_nanf("");
        const int ev = odd || hole ? 0 : (int)(__builtin_bit_cast(uint32_t, cur_vs) >> 23 & 0xFFu) - 127;
        const float unscale = __builtin_bit_cast(float, (uint32_t)(127 - ev) << 23);
        const float a = factor * cur_ks;
        float x[16];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float v;
                if constexpr (CAP) {
                    // cap * tanh(s / cap) = cap - 2 cap / (exp(2 s / cap) + 1)
                    const float z = __builtin_amdgcn_exp2f(S[t][r] * a * (2.f * kLog2E / A.softcap));
                    v = fmaf(A.softcap - 2.f * A.softcap / (z + 1.f), kLog2E, (float)ev);
                } else {
                    v = fmaf(S[t][r], a, (float)ev);
                }
                x[4 * t + r] = v;
            }
        const bool plain = key0 >= all_lo && key0 + (int32_t)kStep - 1 <= all_hi && __ballot(hole) == 0;
        if (!plain) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int32_t key = key0 + (int32_t)g * 16 + i;
                if (hole || key > key_hi || key < key_lo) x[i] = -__builtin_inff();
            }
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, x[i]);
        if (__ballot(top > M + kSlack)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float next = top > M + kSlack ? top : M;
            const float f = __builtin_amdgcn_exp2f(M - next);
            M = next;
            L *= f;
#pragma unroll
            for (int i = 0; i < 2 * NK; i++) acc[i] *= f;
        }
        f16x8_t ph[2], pl[2];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float p = __builtin_amdgcn_exp2f(x[i] - M + kBias);
            L = fmaf(p, unscale, L);
            ph[i / 8][i % 8] = (_Float16)p;
            if constexpr (PAIRS) pl[i / 8][i % 8] = (_Float16)(p - (float)ph[i / 8][i % 8]);
        }
#pragma unroll
        for (int d = 0; d < 2 * NK; d++) {
            u32x4_t c = vc[d];
            if (!plain) {  // bytes behind the last key may be anything
                const int32_t have = hole ? 0 : sh.len - key0 - (int32_t)g * 16;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int32_t b = have - 4 * i;
                    c[i] = b >= 4 ? c[i] : (b <= 0 ? 0u : c[i] & ~(~0u << (8 * b)));
                }
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const f16x8_t va = codes_f16(u32x2_t{c[2 * u], c[2 * u + 1]});
                acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[u], acc[d], 0, 0, 0);
                if constexpr (PAIRS) acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[u], acc[d], 0, 0, 0);
            }
        }
    }

    // the wavefronts' sums as one
    L += __shfl_xor(L, 16, 64);
    L += __shfl_xor(L, 32, 64);
    if (g == 0) sh_ml[wave][n][0] = M, sh_ml[wave][n][1] = L;
#pragma unroll
    for (int d = 0; d < 2 * NK; d++) *(f32x4_t *)&sh_acc[wave][n][d * 16 + g * 4] = acc[d];
    __syncthreads();
    const uint32_t item = blockIdx.y * gridDim.x + blockIdx.x;
    for (uint32_t i = threadIdx.x; i < kTile * (D / 4); i += kAttnThreads) {
        const uint32_t r = i / (D / 4), d = i % (D / 4) * 4, q = it.tile * kTile + r;
        if (q >= sh.n * group) continue;
        float top = kNoMax;
#pragma unroll
        for (uint32_t w = 0; w < kAttnWaves; w++) top = fmaxf(top, sh_ml[w][r][0]);
        f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kAttnWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(sh_ml[w][r][0] - top);
            l = fmaf(f, sh_ml[w][r][1], l);
            o += *(const f32x4_t *)&sh_acc[w][r][d] * f;
        }
        if (it.pieces > 1) {
            *(f32x4_t *)(part.acc + ((size_t)item * kTile + r) * D + d) = o;
            if (d == 0) part.ml[((size_t)item * kTile + r) * 2] = top, part.ml[((size_t)item * kTile + r) * 2 + 1] = l;
            continue;
        }
        const uint32_t h = kvh * group + q % group;
        if (A.sinks && l != 0.f) l += __builtin_amdgcn_exp2f(A.sinks[h] * kLog2E - top + kBias);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        store4(A.out, A.out_type, (size_t)(sh.row + q / group) * A.out_stride + (size_t)h * D + d, v);
    }
}

// The pieces of split rows as one: a workgroup for each query row of a tile (rows of tiles that are not split leave at once), its
// wavefronts a quarter of the pieces each.
__global__ void __launch_bounds__(kAttnThreads) attention_join_kernel(AttentionArgs A, Partials part, uint32_t items_per_head) {
    __shared__ float sh_acc[kAttnWaves][256], sh_ml[kAttnWaves][2];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, D = A.kv.head_dim;
    const uint32_t kvh = blockIdx.y, group = A.q_heads / A.kv.kv_heads, r = blockIdx.z;
    Item it;
    uint32_t first_item;
    if (!find_item(A, blockIdx.x, true, it, first_item) || it.pieces < 2) return;
    const Share sh = share_of(A, it.s, group);
    const uint32_t q = it.tile * kTile + r;
    if (q >= sh.n * group) return;
    const size_t at = ((size_t)kvh * items_per_head + first_item) * kTile + r;  // row r of the first piece; the next kTile rows on
    float top = kNoMax, l = 0.f;
    f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const uint32_t dim = min(lane * 4, D - 4);
    for (uint32_t p0 = wave; p0 < it.pieces; p0 += 8 * kAttnWaves) {
        float m[8], s[8];
        f32x4_t a[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {  // (beyond the last piece: the last once more, with no weight)
            const uint32_t p = p0 + i * kAttnWaves;
            const size_t x = at + (size_t)min(p, it.pieces - 1) * kTile;
            m[i] = p < it.pieces ? part.ml[2 * x] : kNoMax;
            s[i] = part.ml[2 * x + 1];
            a[i] = *(const f32x4_t *)(part.acc + x * D + dim);
        }
        float next = top;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) next = fmaxf(next, m[i]);
        const float f = __builtin_amdgcn_exp2f(top - next);
        o *= f;
        l *= f;
        top = next;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (p0 + i * kAttnWaves >= it.pieces) break;
            const float w = __builtin_amdgcn_exp2f(m[i] - top);
            l = fmaf(w, s[i], l);
            o += a[i] * w;
        }
    }
    if (lane == 0) sh_ml[wave][0] = top, sh_ml[wave][1] = l;
    if (lane * 4 < D) *(f32x4_t *)&sh_acc[wave][lane * 4] = o;
    __syncthreads();
    if (wave || lane * 4 >= D) return;
#pragma unroll
    for (uint32_t w = 1; w < kAttnWaves; w++) top = fmaxf(top, sh_ml[w][0]);
    l = 0.f;
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t w = 0; w < kAttnWaves; w++) {
        const float f = __builtin_amdgcn_exp2f(sh_ml[w][0] - top);
        l = fmaf(f, sh_ml[w][1], l);
        o += *(const f32x4_t *)&sh_acc[w][lane * 4] * f;
    }
    const uint32_t h = kvh * group + q % group;
    if (A.sinks && l != 0.f) l += __builtin_amdgcn_exp2f(A.sinks[h] * kLog2E - top + kBias);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    store4(A.out, A.out_type, (size_t)(sh.row + q / group) * A.out_stride + (size_t)h * D + lane * 4, v);
}

static size_t items_of(const AttentionArgs &A) { return (size_t)items_bound(A) * A.kv.kv_heads; }
size_t attention_workspace_bytes(const AttentionArgs &A) { return items_of(A) * kTile * (A.kv.head_dim + 2) * sizeof(float) + 16; }

int attention_launches(const AttentionArgs &) { return 2; }

template <int NK>
static void launch_dim(hipStream_t s, const AttentionArgs &A, const Partials &part, dim3 grid) {
    const bool pairs = A.out_type == ELEM_F32, cap = A.softcap > 0.f;
#define LARQL_ATTN(P, C) hipLaunchKernelGGL((attention_rows_kernel<NK, P, C>), grid, dim3(kAttnThreads), 0, s, A, part)
    if (pairs && cap) LARQL_ATTN(true, true);
    else if (pairs) LARQL_ATTN(true, false);
    else if (cap) LARQL_ATTN(false, true);
    else LARQL_ATTN(false, false);
#undef LARQL_ATTN
}

hipError_t attention_launch(hipStream_t s, const AttentionArgs &A, void *workspace) {
    if (A.kv.tokens == 0 || A.kv.sequences == 0) return hipSuccess;
    const uint64_t items = items_bound(A);
    if (items > 0x7FFFFFFFull) return hipErrorInvalidValue;
    const Partials part{(float *)workspace, (float *)workspace + items_of(A) * kTile * A.kv.head_dim};
    const dim3 grid((uint32_t)items, A.kv.kv_heads);
    switch (A.kv.head_dim / 32) {
    case 1: launch_dim<1>(s, A, part, grid); break;
    case 2: launch_dim<2>(s, A, part, grid); break;
    case 3: launch_dim<3>(s, A, part, grid); break;
    case 4: launch_dim<4>(s, A, part, grid); break;
    case 5: launch_dim<5>(s, A, part, grid); break;
    case 6: launch_dim<6>(s, A, part, grid); break;
    case 7: launch_dim<7>(s, A, part, grid); break;
    case 8: launch_dim<8>(s, A, part, grid); break;
    default: return hipErrorInvalidValue;
    }
    const uint64_t group = A.q_heads / A.kv.kv_heads, tiles = A.kv.tokens * group / kTile + A.kv.sequences;
    const uint32_t join_rows = (uint32_t)std::min<uint64_t>(A.kv.max_new * group, kTile);
    hipLaunchKernelGGL(attention_join_kernel, dim3((uint32_t)tiles, A.kv.kv_heads, join_rows), dim3(kAttnThreads), 0, s, A, part, (uint32_t)items);
    return hipGetLastError();
}

}  // namespace larql
