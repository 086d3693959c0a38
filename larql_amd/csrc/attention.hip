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
//
// Measured: one token over 131072 keys of 16/8 heads of 256, f32: 95 us, 5.7 TB/s of codes (reads reach 6.5), and 7 of joining; 32 sequences of 4000
// keys of 32/8 heads of 128: 49 us, 5.3 TB/s.  A prompt of 8192 tokens, causal: 32/8 heads of 128, bf16, 640-700 us, 0.79-0.86 PFLOP/s at a clock of
// 1.95 GHz (a large bf16 product of the library: 1.24); 8/4 heads of 256: bf16 400 us, f32 (twice the matrix instructions) 457.
#include <algorithm>

#include "kernels.h"
#include "layer.h"

namespace larql {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr uint32_t kStep = 64;          // keys of a step
constexpr uint32_t kAttnThreads = 256;
constexpr uint32_t kAttnWaves = kAttnThreads / 64;
constexpr uint32_t kRowsTile = 16;      // query rows of a workgroup of the kernel for few rows
constexpr uint32_t kTilesTile = 128;    // ... for many
// A sequence with at most this many rows for each key/value head goes through the former.  16 sequences of 4000 keys, us through it / through the
// latter: 24 rows 51 / 54 (128 channels, bf16), 85 / 97 (256, f32); 32 rows 51 / 53, 86 / 99; 56 rows 94 / 62, 154 / 106.
constexpr uint32_t kFewRows = 32;
constexpr float kLog2E = 1.44269504088896341f;
// Weights are held as 2^(t + e - M + bias) with t + e - M <= 3; M is whole and only moves where a score leaves that range, so it brings no
// rounding.  f32 results: the bias is small, for the exponent is rounded as a number of its size; an f16 pair keeps 22 bits down to 2^-9 of the
// largest, which is 2^6 at least, and is off by 2^-25 beyond: 2^-31 of it (131072 equal weights 2^-17 of one that weighs as much as they all: 2^-14
// each, at random).  16-bit results: as large as fits; one f16 keeps 11 bits down to 2^-25 of the largest, a pair 22 down to 2^-14, 2^-36 beyond.
constexpr float kLowBias = 7.f, kHighBias = 12.f, kSlack = 3.f;
__device__ __forceinline__ float weight_bias(bool f32_result) { return f32_result ? kLowBias : kHighBias; }
constexpr float kNoMax = -1e30f;

// How one of the two kernels shares its work out.
struct Plan {
    uint32_t tile;                // query rows of a workgroup
    uint32_t rows_min, rows_max;  // sequences with this many rows for each key/value head are its own
    uint32_t target;              // pieces of one head's work that long rows are split into
    uint32_t min_steps;           // steps of a piece at least
    uint32_t split;               // whether rows are split at all
    int fits;                     // how often pieces are made longer to meet the target
};

// Steps of keys that the window lets a tile of a sequence with n new tokens see, at most.  Causal: the window and the tile's tokens, which may
// straddle; else all keys behind the first one's window, so up to n more than the window.
__host__ __device__ __forceinline__ uint64_t window_steps(const AttentionArgs &A, uint32_t tile, uint32_t n) {
    return A.window ? ((uint64_t)A.window + (A.causal ? A.group.of(tile) : n) + 1) / kStep + 2 : ~(uint64_t)0;
}

// A sequence's share of the work: its query rows in tiles, and at most how many steps of keys one of them sees.
struct Share {
    uint32_t row, n;      // first row of the activations, new tokens
    int32_t len, first;   // keys, position of the first new token
    uint32_t tiles, steps;
};
__device__ __forceinline__ Share share_of(const AttentionArgs &A, const Plan &P, uint32_t s) {
    const NewTokens t = new_tokens(A.kv, s);
    Share h;
    h.row = t.row;
    h.n = t.n;
    h.len = (int32_t)min((uint64_t)t.len, (uint64_t)A.kv.table_width << A.kv.page_shift);
    h.first = t.len - (int32_t)t.n;
    const uint32_t rows = t.n * A.group.d;
    h.tiles = rows < P.rows_min || rows > P.rows_max ? 0u : (rows + P.tile - 1) / P.tile;
    h.steps = h.tiles ? ((uint32_t)h.len + kStep - 1) / kStep : 0;
    h.steps = min((uint64_t)h.steps, window_steps(A, P.tile, t.n));
    return h;
}

// What the wavefront that serves item `item` of a head works on; false beyond the last.  Every wavefront finds it from the lengths:
// tiles of sequences in order, the keys that a tile sees in equal pieces, as many as P.target asks for.  Pieces of split tiles
// have places for their partial results, `slot` on; `split_tiles`: items count split tiles instead.  Lengths of more than 64 sequences are read
// once more for each sum and for the search: one token each over 500 keys, 1024 sequences of 8/2 heads of 128 take 65 us (4.1 TB/s), 4096 of 4/1 heads
// 231 (2.3).
struct Item {
    uint32_t s, tile, piece, pieces, slot;
    // the steps of this piece, of those from `first` to before `end` that its tile sees
    __device__ __forceinline__ uint32_t begin_of(uint32_t first, uint32_t end) const { return first + piece * ((end - first + pieces - 1) / pieces); }
    __device__ __forceinline__ uint32_t end_of(uint32_t first, uint32_t end) const {
        return min(first + (piece + 1) * ((end - first + pieces - 1) / pieces), end);
    }
};
__device__ __forceinline__ bool find_item(const AttentionArgs &A, const Plan &P, uint32_t item, bool split_tiles, Item &it, Share &sh) {
    const uint32_t lane = threadIdx.x % 64;
    const auto share_at = [&](uint32_t s) { return s < A.kv.sequences ? share_of(A, P, s) : Share{}; };
    const auto pieces_of = [](const Share &h, uint32_t chunk) { return max(h.steps / chunk + (h.steps % chunk ? 1u : 0u), 1u); };
    const Share first = share_at(lane);  // (read once where 64 sequences are all)
    const auto sum_of = [&](auto f) {  // over the sequences; a sum that need not be exact
        float v = f(first);
        for (uint32_t base = 64; base < A.kv.sequences; base += 64) v += f(share_at(base + lane));
        return wave_fsum(v);
    };
    uint32_t chunk = 0x7FFFFFFFu;  // steps of a piece
    if (P.split) {
        chunk = max((uint32_t)ceilf(sum_of([](const Share &h) { return (float)h.tiles * (float)h.steps; }) / (float)P.target), P.min_steps);
        for (int i = 0; i < P.fits; i++) {  // pieces are whole: longer ones, until the items are as few as asked for
            if (sum_of([&](const Share &h) { return (float)h.tiles * (float)pieces_of(h, chunk); }) <= (float)P.target) break;
            chunk += chunk / 8 + 1;
        }
    }
    it.slot = 0;
    for (uint32_t base = 0; base < A.kv.sequences; base += 64) {
        const Share h = base ? share_at(base + lane) : first;
        const uint32_t tiles = h.tiles, pieces = pieces_of(h, chunk);
        const uint32_t slots = pieces > 1 ? tiles * pieces : 0u, weight = split_tiles ? (pieces > 1 ? tiles : 0u) : tiles * pieces;
        const uint32_t upto = wave_inclusive_sum(weight), all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        const uint32_t slots_upto = P.split ? wave_inclusive_sum(slots) : 0u;
        if (item < all) {
            const int at = (int)__builtin_ctzll(__ballot(upto > item));
            const auto of_it = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
            it.pieces = of_it(pieces);
            const uint32_t in = item - of_it(upto - weight);
            it.s = base + (uint32_t)at;
            it.tile = split_tiles ? in : in / it.pieces;
            it.piece = split_tiles ? 0 : in % it.pieces;
            it.slot += of_it(slots_upto - slots) + it.tile * it.pieces;
            sh.row = of_it(h.row), sh.n = of_it(h.n), sh.len = (int32_t)of_it((uint32_t)h.len), sh.first = (int32_t)of_it((uint32_t)h.first);
            sh.tiles = of_it(tiles), sh.steps = of_it(h.steps);
            return true;
        }
        item -= all;
        it.slot += P.split ? (uint32_t)__builtin_amdgcn_readlane((int)slots_upto, 63) : 0u;
    }
    return false;
}

// The two kernels' plans, and what the host has to know of them: items of one head at most (the last piece of a tile may be
// short), places for partial results (split tiles have at least two pieces: twice the target), and tiles that may be split.
struct Plans {
    Plan rows, tiles;
    bool use_rows, use_tiles;
    static uint64_t tiles_at_most(const AttentionArgs &A, const Plan &P) {
        const uint64_t of_rows = A.kv.tokens * (uint64_t)A.group.d / P.tile + A.kv.sequences;  // (of few rows: a sequence's are few)
        return std::min(of_rows, A.kv.sequences * (((uint64_t)P.rows_max + P.tile - 1) / P.tile));
    }
    static uint64_t items(const AttentionArgs &A, const Plan &P) { return tiles_at_most(A, P) + (P.split ? P.target + 1 : 0); }
    static uint64_t slots(const Plan &P) { return P.split ? 2 * P.target + 2 : 0; }
    static uint64_t split_tiles(const AttentionArgs &A, const Plan &P) { return P.split ? std::min<uint64_t>(P.target + 1, tiles_at_most(A, P)) : 0; }
};
static Plans plans_of(const AttentionArgs &A) {
    const uint64_t group = A.group.d, most = A.kv.max_new * group;
    const auto steps_of = [&](uint32_t tile, uint64_t rows) {  // of a sequence with at most so many rows
        const uint32_t n = (uint32_t)std::min<uint64_t>(A.kv.max_new, rows / group);
        return std::min((((uint64_t)A.kv.table_width << A.kv.page_shift) + kStep - 1) / kStep, window_steps(A, tile, n));
    };
    const uint32_t cus = 256;
    Plans p;
    // Pieces of few rows: as many as workgroups are resident, 2 a compute unit above 128 channels (131072 keys of 256, us with 1, 2, 3, 4 of
    // them: 148, 103, 125, 110, joining included), 3 below (64 sequences, 64 channels, with 2, 3, 4: 38, 34, 37); a wavefront's step each at least.
    p.rows = {kRowsTile, 1, kFewRows, std::max((A.kv.head_dim > 128 ? 2 : 3) * cus / A.kv.kv_heads, 1u), kAttnWaves, 1, 0};
    // Rows so short that the launch of joining costs what it saves stay whole (1000 keys, us whole / split: 32/8 heads of 128 13.4 / 12.8, 16
    // sequences of them 14.6 / 17.2, 64/8 of 64 10.0 / 10.8; 2000 of the first 20.7 / 13.0; 8/4 heads of 256, f32: 500 keys 13.0 / 14.7, 1000 19.1 /
    // 15.0).
    p.rows.split = steps_of(kRowsTile, kFewRows) > (A.kv.head_dim > 128 ? 8u : 16u);
    // Many rows: as many as are resident, unless the tiles by themselves (of which a sequence's last is half full, say) are as many: splitting
    // then is a launch more for nothing (2048 tokens of 32/8 heads of 128: 76 us whole, 88 with it; 16 sequences of 32 tokens, 256 channels,
    // f32: 239 and 165).
    p.tiles = {kTilesTile, kFewRows + 1, 0xFFFFFFFFu, std::max((A.kv.head_dim > 128 ? 1 : 2) * cus / A.kv.kv_heads, 1u), 8, 1, 6};
    p.tiles.split = steps_of(kTilesTile, most) > p.tiles.min_steps && A.kv.tokens * group / p.tiles.tile + A.kv.sequences / 2 < p.tiles.target;
    p.use_tiles = most > kFewRows;
    p.use_rows = !p.use_tiles || A.kv.sequences > 1;
    if (!p.use_rows) p.tiles.rows_min = 1;  // one sequence: one kernel, whatever its number of new tokens turns out to be
    return p;
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

// two weights as f16, or as f16 pairs
template <bool PAIRS>
__device__ __forceinline__ void weights_f16(f32x2_t p, f16x8_t &h, f16x8_t &l, int at) {
    const f16x2_t a = __builtin_convertvector(p, f16x2_t);
    h[at] = a[0], h[at + 1] = a[1];
    if constexpr (PAIRS) {
        const f16x2_t b = __builtin_convertvector(p - __builtin_convertvector(a, f32x2_t), f16x2_t);
        l[at] = b[0], l[at + 1] = b[1];
    }
}

// Weights of one f16 are summed as they enter the matrix instructions, so that a rounding moves numerator and sum alike, unless the value
// scale of one of the turn's blocks is so far (kFar) below the largest met that its weights may be nothing in f16 and still count: those are
// summed in f32.
constexpr int kFar = 8;
__device__ __forceinline__ float weights_sum(const f16x8_t &h) {
    const f16x2_t one = {(_Float16)1.f, (_Float16)1.f};
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) sum = __builtin_amdgcn_fdot2(f16x2_t{h[j], h[j + 1]}, one, sum, false);
    return sum;
}

// Partial results of pieces: [kv_heads][slots][tile][head_dim] weighted sums, and [kv_heads][slots][tile] maxima and sums of weights.
struct Partials {
    float *acc, *ml;
    uint32_t slots;
};

// A result row's end: the sink, the quotient.
__device__ __forceinline__ float inverse_sum(const AttentionArgs &A, float l, float top, uint32_t head) {
    if (A.sinks && l != 0.f) l += __builtin_amdgcn_exp2f(fmaf(A.sinks[head], kLog2E, weight_bias(A.out_type == ELEM_F32) - top));
    return l == 0.f ? 0.f : 1.f / l;
}

// The logarithm (base 2) of a capped score's weight, plus e: cap * tanh(x / cap) = cap - 2 cap / (exp(2 x / cap) + 1), where s a is the
// exponent of that as a power of two (query_scale).  That is off by what 32 bits leave of the cap: for a cap of 64 up to 2^-17 of a weight, little
// beside one f16 of it, not beside a pair.  A score below 0.26 of its cap (kSeriesBelow) can take the series of tanh (next term below 2e-8 of it), so
// that a cap above the scores costs them no precision.  Few rows, which wait for memory, compute both; many rows the series alone where a wavefront's
// scores all allow it, and where weights are one f16 and the cap is at most kLowCap the closed form alone (4096 causal tokens of 32/8 heads
// of 128, us: f16, closed 230, by the scores 235, both 285; f32 with a cap of 50 378, 386, 439, of 5 371, 434, 434).
constexpr float kLowCap = 64.f;
enum class CapBy { WHOLE, SERIES, EITHER };
constexpr float kSeriesBelow = 0.75f;  // of |s a|
template <CapBy BY>
__device__ __forceinline__ float capped(const AttentionArgs &A, float s, float a, float e) {
    const float c = A.softcap * kLog2E, z = s * a;
    const float whole = fmaf(-2.f * c, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(z) + 1.f), c + e);
    if constexpr (BY == CapBy::WHOLE) return whole;
    constexpr float u2 = 0.120113253f;  // (ln 2 / 2)^2: x / cap = z ln 2 / 2
    const float t = z * z;
    const float poly = fmaf(t, fmaf(t, fmaf(t, fmaf(t, u2 * u2 * u2 * u2 * 62.f / 2835.f, u2 * u2 * u2 * -17.f / 315.f), u2 * u2 * 2.f / 15.f), u2 / -3.f), 1.f);
    const float series = fmaf(A.softcap * 0.5f * z, poly, e);
    return BY == CapBy::SERIES || fabsf(z) < kSeriesBelow ? series : whole;
}
// Scores s of a step with hidden keys, whose logarithms are s a + e: a hidden one is -inf, times a factor that is positive; a factor that is
// not (a scale of 0, a block that is no number) goes into the scores that are seen.
struct Seen {
    float factor, offset;
    bool keep;
    __device__ __forceinline__ Seen(float a, float e) : factor(a), offset(e), keep(a > 0.f) {}
    __device__ __forceinline__ float operator()(float s, int hidden) const {
        const float x = keep ? s : fmaf(s, factor, offset);
        return hidden ? -__builtin_inff() : x;
    }
    __device__ __forceinline__ float a() const { return keep ? factor : 1.f; }
    __device__ __forceinline__ float e() const { return keep ? offset : 0.f; }
};

// A query row's elements (spread over lanes 32 apart, and 16 apart where QUARTERS) enter as f16 or f16 pairs after a power-of-two scale that
// brings the largest to [2^14, 2^15): what they are multiplied by, and what scores are.  A row that is not finite gets NaN there.
struct QueryScale {
    float mul, factor;
};
template <int N, bool CAP, bool QUARTERS>
__device__ __forceinline__ QueryScale query_scale(const AttentionArgs &A, const Eight (&q)[N]) {
    uint32_t amax = 0;
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) amax = max(amax, __builtin_bit_cast(uint32_t, q[k][i]) & 0x7FFFFFFFu);
    if constexpr (QUARTERS) amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16, 64));
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32, 64));
    const bool finite = amax < 0x7F800000u;
    const int e = min(max((int)(amax >> 23) - 127 - 14, -114), 114);
    const float inv = finite ? __builtin_bit_cast(float, (uint32_t)(127 - e) << 23) : 0.f;
    const float factor = fabsf(A.scale) * (CAP ? 2.f * kLog2E / A.softcap : kLog2E) * __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
    // (the scale's sign goes into the query: factors of scores are not negative)
    return {A.scale < 0.f ? -inv : inv, finite ? factor : __builtin_nanf("")};
}
template <bool PAIRS>
__device__ __forceinline__ void query_f16(const Eight &q, float mul, f16x8_t &h, f16x8_t &l) {
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        weights_f16<PAIRS>(f32x2_t{mul == 0.f ? 0.f : q[i] * mul, mul == 0.f ? 0.f : q[i + 1] * mul}, h, l, i);
}

// ---- few query rows --------------------------------------------------------------------------------------------------
//
// 16 query rows a workgroup, as the columns of v_mfma_f32_16x16x32_f16; its wavefronts take steps of 64 keys in turn and add up at the
// end.  A wavefront reads its step's codes straight into the registers that the matrix instructions' operands are converted
// from, 64 x head_dim bytes of K and then of V through ONE set of registers: as a part of the keys is multiplied its registers take a part
// of the step's values, and as that is multiplied a part of the next step's keys, so two wavefronts fit a SIMD above 128 channels and three
// below.  The loads do not stay in flight throughout: the two page numbers read in a step are compared where they are read (kv_page), and
// each waits for every load before it, so the step's values have arrived before the next keys are asked for; other wavefronts fill that gap.
// The queries' operands are read from LDS.
// Queries and weights are f16 pairs for every result: memory, not the matrix instructions, is waited for (one token of 131072 keys of 16/8 heads of
// 128 into bf16, 52 us in pairs, 58 as one f16; 64 sequences of 64/8 heads of 64: 34.6, 33.3, of 500 keys each: 12, 11).
template <int NK, bool CAP>
__global__ void __launch_bounds__(kAttnThreads, NK > 4 ? 2 : 3) attention_rows_kernel(AttentionArgs A, Plan P, Partials part) {
    constexpr uint32_t D = NK * 32, kPad = D + 4;
    constexpr int NP = (NK + 1) / 2;  // parts: 64 channels of the keys, 64 channels of the values
    struct Queries {
        f16x8_t q[2][NK][64];
        float factor[16];
    };
    struct Sums {
        float acc[kAttnWaves][kRowsTile][kPad], ml[kAttnWaves][kRowsTile][2];
    };
    __shared__ __align__(16) char shared[sizeof(Queries) > sizeof(Sums) ? sizeof(Queries) : sizeof(Sums)];
    Queries &sq = *(Queries *)shared;
    Sums &ss = *(Sums *)shared;
    const KvArgs &kv = A.kv;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, n = lane % 16, g = lane / 16;
    const uint32_t kvh = blockIdx.y, group = A.group.d;
    Item it;
    Share sh;
    if (!find_item(A, P, blockIdx.x, false, it, sh)) return;
    const uint32_t rows = sh.n * group;

    // The lane's query row, and what it sees.  What all and any of the rows see: the first and the last say it.
    const uint32_t row0 = it.tile * kRowsTile, row = row0 + n;
    const bool live = row < rows;
    const auto hi_of = [&](uint32_t r) { return A.causal ? min(sh.first + (int32_t)A.group.of(r), sh.len - 1) : sh.len - 1; };
    const auto lo_of = [&](uint32_t r) {
        return A.window ? (int32_t)max((int64_t)sh.first + (int64_t)A.group.of(r) - (int64_t)A.window + 1, (int64_t)0) : 0;
    };
    const int32_t key_hi = live ? hi_of(row) : -1, key_lo = lo_of(row);
    const uint32_t last_row = min(row0 + kRowsTile - 1, rows - 1);
    const int32_t all_hi = hi_of(row0), any_hi = hi_of(last_row), any_lo = lo_of(row0), all_lo = lo_of(last_row);

    const uint32_t tile_end = any_hi < any_lo ? 0u : (uint32_t)any_hi / kStep + 1, tile_begin = min((uint32_t)any_lo / kStep, tile_end);
    const uint32_t end = it.end_of(tile_begin, tile_end);
    uint32_t step = it.begin_of(tile_begin, tile_end) + wave;

    const int32_t *table = kv.block_table + (size_t)it.s * kv.table_width;
    const uint32_t page_mask = (1u << kv.page_shift) - 1;
    const size_t head_codes = (size_t)D << kv.page_shift;
    const uint8_t *k_head = kv.k_codes + kvh * head_codes, *v_head = kv.v_codes + kvh * head_codes;
    const uint32_t page_bytes = (uint32_t)(kv.kv_heads * head_codes);
    const uint32_t gk = n / 4;  // this lane loads keys of group gk, and values and weights of group g, of a step
    const auto page_of = [&](uint32_t st, uint32_t grp) -> uint32_t {
        const uint32_t key = st * kStep + grp * 16;
        return st >= end || (int32_t)key >= sh.len ? ~0u : kv_page(kv, table, key);
    };
    u32x4_t ring[NP][4];
    const auto load_keys = [&](const uint8_t *kp, int p) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const uint8_t *kr = kp + (uint32_t)(4 * t) * D + p * 64;
            if (2 * p + 1 < NK) {
                ring[p][t] = *(const u32x4_t *)(kr + g * 16);
            } else {
                const u32x2_t c = *(const u32x2_t *)(kr + g * 8);
                ring[p][t] = u32x4_t{c[0], c[1], 0u, 0u};
            }
        }
    };
    const auto keys_at = [&](uint32_t st, uint32_t page) {
        return k_head + (uint64_t)(page == ~0u ? 0u : page) * page_bytes + (((st * kStep + gk * 16) & page_mask) + n % 4) * D;
    };
    float ks = 0.f, vs = 1.f;
    const auto load_scales = [&](uint32_t page) {
        const size_t at = (size_t)(page == ~0u ? 0u : page) * kv.kv_heads + kvh;
        ks = kv.k_scales[at];
        vs = kv.v_scales[at];
    };
    uint32_t page_k = page_of(step, gk), page_v = page_of(step, g);
    __builtin_amdgcn_sched_barrier(0);
    // The queries' elements, before the keys': each piece is converted by its type where it is loaded, so one is waited for before the next leaves.
    // Channels of the lane's operand k: two operands' lie in one 16-byte piece of a key's row.
    Eight q[NK];
    const uint32_t q_row = live ? row : last_row;
#pragma unroll
    for (int k = 0; k < NK; k++) {
        const uint32_t d = (k | 1) < NK ? (uint32_t)(k & ~1) * 32 + g * 16 + (uint32_t)(k & 1) * 8 : (uint32_t)k * 32 + g * 8;
        q[k] = load8(A.q, A.q_type, (size_t)(sh.row + A.group.of(q_row)) * A.q_stride + (size_t)(kvh * group + A.group.rest(q_row)) * D + d);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (step < end) {
        const uint8_t *kp = keys_at(step, page_k);
#pragma unroll
        for (int p = 0; p < NP; p++) load_keys(kp, p);
        load_scales(page_v);
    }
    uint32_t next_k = page_of(step + kAttnWaves, gk), next_v = page_of(step + kAttnWaves, g);

    // (every wavefront scales the rows, each converts a quarter of the operands)
    const QueryScale f = query_scale<NK, CAP, true>(A, q);
    if (wave == 0 && g == 0) sq.factor[n] = f.factor;
#pragma unroll
    for (int k = 0; k < NK; k++)
        if ((uint32_t)k % kAttnWaves == wave) {
            f16x8_t h, l;
            query_f16<true>(q[k], f.mul, h, l);
            sq.q[0][k][lane] = h;
            sq.q[1][k][lane] = l;
        }
    __syncthreads();
    const float factor = sq.factor[n];

    f32x4_t acc[2 * NK];
#pragma unroll
    for (int i = 0; i < 2 * NK; i++) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float M = kNoMax, L = 0.f;
    for (; step < end; step += kAttnWaves) {
        const int32_t key0 = (int32_t)(step * kStep);
        const bool hole = page_v == ~0u;
        const uint8_t *vp = v_head + (uint64_t)(hole ? 0u : page_v) * page_bytes + ((n << kv.page_shift) + (((uint32_t)key0 + g * 16) & page_mask));
        f32x4_t S[4], odd[4] = {}, low[4] = {};  // (three sums, each of a third of the roundings)
#pragma unroll
        for (int p = 0; p < NP; p++) {
#pragma unroll
            for (int k = 2 * p; k < (2 * p + 2 < NK ? 2 * p + 2 : NK); k++) {
                const f16x8_t qh = sq.q[0][k][lane], ql = sq.q[1][k][lane];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const u32x4_t c = ring[p][t];
                    const f16x8_t ka = codes_f16(k % 2 ? u32x2_t{c[2], c[3]} : u32x2_t{c[0], c[1]});
                    const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
                    f32x4_t &sum = k % 2 ? odd[t] : S[t];
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qh, k < 2 ? zero : sum, 0, 0, 0);
                    low[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, ql, k ? low[t] : zero, 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 4 * p; d < (4 * p + 4 < 2 * NK ? 4 * p + 4 : 2 * NK); d++) ring[p][d % 4] = *(const u32x4_t *)(vp + ((size_t)(16 * d) << kv.page_shift));
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) S[t] += odd[t] + low[t];
        // Logarithms (base 2) of the weights times the value scale.  A scale that is not a number makes its tokens' scores NaN.
        const bool none = !(vs == vs);
        const int ev = none || hole ? 0 : (int)(__builtin_bit_cast(uint32_t, vs) >> 23 & 0xFFu) - 127;
        const float unscale = __builtin_bit_cast(float, (uint32_t)(127 - ev) << 23);
        float a = factor * (none ? __builtin_nanf("") : ks), e = (float)ev;
        const bool plain = key0 >= all_lo && key0 + (int32_t)kStep - 1 <= all_hi && __ballot(hole) == 0;
        if constexpr (CAP) {
#pragma unroll
            for (int i = 0; i < 16; i++) S[i / 4][i % 4] = capped<CapBy::EITHER>(A, S[i / 4][i % 4], a, e);
            a = 1.f, e = 0.f;
        }
        if (!plain) {
            const Seen see(a, e);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int32_t key = key0 + (int32_t)g * 16 + i;
                S[i / 4][i % 4] = see(S[i / 4][i % 4], (int)hole | (int)(key > key_hi) | (int)(key < key_lo));
            }
            a = see.a(), e = see.e();
        }
        float top = S[0][0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, S[i / 4][i % 4]);
        top = fmaf(top, a, e);
        if (__ballot(top > M + kSlack)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float next = top > M + kSlack ? ceilf(top) : M;
            const float f = __builtin_amdgcn_exp2f(M - next);
            M = next;
            L *= f;
#pragma unroll
            for (int i = 0; i < 2 * NK; i++) acc[i] *= f;
        }
        f16x8_t ph[2], pl[2];
        float sum = 0.f;
        const float shift = e - M + weight_bias(A.out_type == ELEM_F32);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const f32x2_t p = {__builtin_amdgcn_exp2f(fmaf(S[i / 4][i % 4], a, shift)), __builtin_amdgcn_exp2f(fmaf(S[i / 4][i % 4 + 1], a, shift))};
            weights_f16<true>(p, ph[i / 8], pl[i / 8], i % 8);
            sum += p[0] + p[1];
        }
        L = fmaf(sum, unscale, L);
        if (!plain) {  // bytes behind the last key may be anything
            const int32_t have = hole ? 0 : sh.len - key0 - (int32_t)g * 16;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int32_t b = have - 4 * i;
                const uint32_t keep = b >= 4 ? ~0u : (b <= 0 ? 0u : ~(~0u << (8 * b)));
#pragma unroll
                for (int d = 0; d < 2 * NK; d++) ring[d / 4][d % 4][i] &= keep;
            }
        }
        page_k = next_k, page_v = next_v;
        const bool more = step + kAttnWaves < end;
        const uint8_t *kp = keys_at(step + kAttnWaves, page_k);
        if (more) {
            load_scales(page_v);
            next_k = page_of(step + 2 * kAttnWaves, gk), next_v = page_of(step + 2 * kAttnWaves, g);
        }
#pragma unroll
        for (int p = 0; p < NP; p++) {
#pragma unroll
            for (int d = 4 * p; d < (4 * p + 4 < 2 * NK ? 4 * p + 4 : 2 * NK); d++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const u32x4_t c = ring[p][d % 4];
                    const f16x8_t va = codes_f16(u32x2_t{c[2 * u], c[2 * u + 1]});
                    acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[u], acc[d], 0, 0, 0);
                    acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[u], acc[d], 0, 0, 0);
                }
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_keys(kp, p);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // the wavefronts' sums as one
    L += __shfl_xor(L, 16, 64);
    L += __shfl_xor(L, 32, 64);
    __syncthreads();  // (the sums lie where the queries did)
    if (g == 0) ss.ml[wave][n][0] = M, ss.ml[wave][n][1] = L;
#pragma unroll
    for (int d = 0; d < 2 * NK; d++) *(f32x4_t *)&ss.acc[wave][n][d * 16 + g * 4] = acc[d];
    __syncthreads();
    const size_t slot = (size_t)kvh * part.slots + it.slot + it.piece;
    for (uint32_t i = threadIdx.x; i < min(rows - row0, kRowsTile) * (D / 4); i += kAttnThreads) {
        const uint32_t r = i / (D / 4), d = i % (D / 4) * 4, q = row0 + r;
        float top = kNoMax;
#pragma unroll
        for (uint32_t w = 0; w < kAttnWaves; w++) top = fmaxf(top, ss.ml[w][r][0]);
        f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kAttnWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(ss.ml[w][r][0] - top);
            l = fmaf(f, ss.ml[w][r][1], l);
            o += *(const f32x4_t *)&ss.acc[w][r][d] * f;
        }
        if (it.pieces > 1) {
            *(f32x4_t *)(part.acc + (slot * kRowsTile + r) * D + d) = o;
            if (d == 0) part.ml[(slot * kRowsTile + r) * 2] = top, part.ml[(slot * kRowsTile + r) * 2 + 1] = l;
            continue;
        }
        const uint32_t h = kvh * group + A.group.rest(q);
        const float inv = inverse_sum(A, l, top, h);
        const f32x4_t v = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        store4(A.out, A.out_type, (size_t)(sh.row + A.group.of(q)) * A.out_stride + (size_t)h * D + d, v);
    }
}

// ---- many query rows -------------------------------------------------------------------------------------------------
//
// 128 query rows a workgroup as the columns of matrix instructions; a turn's codes (64 keys) are converted to f16 once and lie in LDS, two
// turns' worth, rows padded by 16 bytes (an odd number of 16-byte pieces: consecutive rows in other banks).
//   Wide: four wavefronts of 32 rows, v_mfma_f32_32x32x16_f16.  An operand read from LDS feeds 32 columns.
//   Narrow: eight wavefronts of 16 rows, v_mfma_f32_16x16x32_f16, two a SIMD at every head_dim, for twice the reads from LDS: where f16
//     pairs double the multiplications anyway, and above 128 channels, where the wide shape's registers leave one.
// The order of the keys in S^T's rows is free: they are laid out so that a lane holds the weights of 8 consecutive keys for each k step
// of the second product, within one group of 16 keys, so a block's scales are the same for all of them.
template <bool NARROW> struct Shape;
template <> struct Shape<false> {
    static constexpr uint32_t kRows = 32, kWaves = 4, kStepDims = 16, kStepKeys = 16, kTileKeys = 32;  // a k step's channels, keys; keys of a score tile
    typedef f32x16_t Acc;
    static __device__ __forceinline__ Acc mma(f16x8_t a, f16x8_t b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    // the LDS row of a key: bits 2 and 3 exchanged
    static __device__ __forceinline__ uint32_t row_of_key(uint32_t key) { return (key & ~12u) | (key & 4u) << 1 | (key & 8u) >> 1; }
    // score j of a lane's k step c, in its score tiles
    static constexpr int tile(int c, int) { return c / 2; }
    static constexpr int reg(int c, int j) { return c % 2 * 8 + j; }
    static __device__ __forceinline__ uint32_t group(uint32_t c, uint32_t) { return c; }  // of 16 keys
};
template <> struct Shape<true> {
    static constexpr uint32_t kRows = 16, kWaves = 8, kStepDims = 32, kStepKeys = 32, kTileKeys = 16;
    typedef f32x4_t Acc;
    static __device__ __forceinline__ Acc mma(f16x8_t a, f16x8_t b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    // keys 8 g + 4 t + r of 32 to rows 16 t + 4 g + r
    static __device__ __forceinline__ uint32_t row_of_key(uint32_t key) { return (key & ~28u) | (key & 4u) << 2 | (key & 24u) >> 1; }
    static constexpr int tile(int c, int j) { return 2 * c + j / 4; }
    static constexpr int reg(int, int j) { return j % 4; }
    static __device__ __forceinline__ uint32_t group(uint32_t c, uint32_t part) { return 2 * c + part / 2; }
};
constexpr bool tiles_narrow(int nk, bool pairs) { return pairs || nk > 4; }
// A narrow product's order in a wavefront: four reads from LDS ahead of the matrix instructions that use them, `per` for each.
template <int READS, int PER>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < READS - 4; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, PER, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, 4 * PER, 0);
}

enum Cap { CAP_NONE, CAP_LOW, CAP_ANY };  // no cap, one up to kLowCap and weights of one f16, any other
template <int NK, bool QPAIRS, bool PAIRS, Cap CAP>  // f16 pairs: queries, weights
__global__ void __launch_bounds__(Shape<tiles_narrow(NK, PAIRS)>::kWaves * 64, 2)
    attention_tiles_kernel(AttentionArgs A, Plan P, Partials part) {
    typedef Shape<tiles_narrow(NK, PAIRS)> Sh;
    constexpr uint32_t D = NK * 32, kKeys = kStep, kThreads = Sh::kWaves * 64, kKeyPad = D + 8, kValPad = kKeys + 8;
    constexpr int KD = D / Sh::kStepDims, KC = kKeys / Sh::kStepKeys;        // k steps of the two products
    constexpr int ST = kKeys / Sh::kTileKeys, DT = D / Sh::kRows, G = kKeys / 16;  // score tiles, channel tiles, groups of 16 keys
    constexpr int kPieces = (int)((kKeys * D / 16 + kThreads - 1) / kThreads);  // 16-byte pieces of a thread
    constexpr bool kUneven = kKeys * D / 16 % kThreads != 0;
    static_assert(Sh::kRows * Sh::kWaves == kTilesTile, "a workgroup's rows");
    __shared__ __align__(16) _Float16 sh_k[2][kKeys][kKeyPad];
    __shared__ __align__(16) _Float16 sh_v[2][D][kValPad];
    __shared__ float sh_s[2][G][4];  // of each group of 16 keys: key scale, log2 of the value scale, one over it, and whether the turn has a far one
    const KvArgs &kv = A.kv;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, n = lane % Sh::kRows, hi = lane / Sh::kRows;  // column; part of a k step
    const uint32_t block = block_number(), kvh = block % kv.kv_heads, group = A.group.d;  // (neighbours: the heads, one for each XCD's cache)
    Item it;
    Share sh;
    if (!find_item(A, P, block / kv.kv_heads, false, it, sh)) return;
    const uint32_t rows = sh.n * group;
    const uint32_t tile = sh.tiles - 1 - it.tile;  // (the last rows see the most keys: first)

    const uint32_t row = tile * kTilesTile + wave * Sh::kRows + n, tok = A.group.of(row), head = kvh * group + A.group.rest(row);
    const bool live = row < rows;
    const int32_t pos = sh.first + (int32_t)tok;
    const int32_t key_hi = !live ? -1 : (A.causal ? min(pos, sh.len - 1) : sh.len - 1);
    const int32_t key_lo = A.window ? (int32_t)max((int64_t)pos - (int64_t)A.window + 1, (int64_t)0) : 0;
    f16x8_t qh[KD], ql[QPAIRS ? KD : 1];
    float factor;
    {
        Eight q[KD];
#pragma unroll
        for (int k = 0; k < KD; k++) {
            q[k] = {};
            if (live) q[k] = load8(A.q, A.q_type, (size_t)(sh.row + tok) * A.q_stride + (size_t)head * D + (uint32_t)k * Sh::kStepDims + hi * 8);
        }
        const QueryScale f = query_scale<KD, CAP != CAP_NONE, tiles_narrow(NK, PAIRS)>(A, q);
        factor = f.factor;
#pragma unroll
        for (int k = 0; k < KD; k++) query_f16<QPAIRS>(q[k], f.mul, qh[k], ql[QPAIRS ? k : 0]);
    }
    // what all and any of the wavefront's rows see (whole rows of lanes: the first and the last live one say it)
    const uint32_t first_row = tile * kTilesTile + wave * Sh::kRows, last_row = min(first_row + Sh::kRows - 1, rows - 1);
    const bool any_live = first_row < rows;
    const auto hi_of = [&](uint32_t r) { return A.causal ? min(sh.first + (int32_t)A.group.of(r), sh.len - 1) : sh.len - 1; };
    const auto lo_of = [&](uint32_t r) {
        return A.window ? (int32_t)max((int64_t)sh.first + (int64_t)A.group.of(r) - (int64_t)A.window + 1, (int64_t)0) : 0;
    };
    const int32_t all_hi = hi_of(first_row), any_hi = any_live ? hi_of(last_row) : -1;
    const int32_t any_lo = lo_of(first_row), all_lo = lo_of(any_live ? last_row : first_row);
    // the workgroup's steps: those of its piece that any of its rows sees
    const int32_t tile_hi = hi_of(min(tile * kTilesTile + kTilesTile - 1, rows - 1)), tile_lo = lo_of(tile * kTilesTile);
    const uint32_t tile_end = tile_hi < tile_lo ? 0u : (uint32_t)tile_hi / kKeys + 1, tile_begin = min((uint32_t)tile_lo / kKeys, tile_end);
    const uint32_t end = it.end_of(tile_begin, tile_end);
    uint32_t step = it.begin_of(tile_begin, tile_end);

    const int32_t *table = kv.block_table + (size_t)it.s * kv.table_width;
    const uint32_t page_mask = (1u << kv.page_shift) - 1;
    const size_t head_codes = (size_t)D << kv.page_shift;
    // Staging: a piece is 16 channels of a key's row, or 16 keys of a value channel's.
    u32x4_t kc[kPieces], vc[kPieces];
    float ks = 0.f, vs = 0.f;
    int e_top = -1000;  // the largest logarithm of a value scale met
    // The pages of a step, that of group lane % 4 in a lane: read one step before its codes.  (A page number is compared where it is read: behind a
    // step's staging loads that waits for them too, once a turn and before the turn's matrix instructions.)
    const auto pages_of = [&](uint32_t st) -> uint32_t {
        const uint32_t key = st * kKeys + lane % G * 16;
        return st >= end || (int32_t)key >= sh.len ? ~0u : kv_page(kv, table, key);
    };
    // A thread's pieces: where they lie in a page (a page of 128 holds two steps), their groups' lanes.
    const uint32_t page_bytes = (uint32_t)(kv.kv_heads * head_codes);
    const uint8_t *k_head = kv.k_codes + kvh * head_codes, *v_head = kv.v_codes + kvh * head_codes;
    uint32_t odd_pages = 0;  // lanes whose page (of the step in kc, vc) is a hole
    const auto load_step = [&](uint32_t st, uint32_t pages) {
        const uint32_t in_page = (st * kKeys) & page_mask;
        odd_pages = (uint32_t)__ballot(pages == ~0u) & ((1u << G) - 1);
        const uint32_t safe = pages == ~0u ? 0u : pages;
        const uint8_t *vp = v_head + (uint64_t)(uint32_t)__shfl((int)safe, (int)(threadIdx.x % G), 64) * page_bytes +
                            (((threadIdx.x / G) << kv.page_shift) + in_page + ((threadIdx.x % G * 16) & page_mask));
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            const uint32_t p = threadIdx.x + (uint32_t)i * kThreads, key = p / (D / 16);
            const uint32_t page = (uint32_t)__shfl((int)safe, (int)(key / 16 % G), 64);
            if (kUneven && p >= kKeys * D / 16) break;
            kc[i] = *(const u32x4_t *)(k_head + (uint64_t)page * page_bytes + ((in_page + (key & page_mask)) * D + p % (D / 16) * 16));
            vc[i] = *(const u32x4_t *)(vp + ((size_t)(i * (kThreads / G)) << kv.page_shift));
        }
        if (threadIdx.x < G) {
            ks = pages == ~0u ? 0.f : kv.k_scales[(size_t)pages * kv.kv_heads + kvh];
            vs = pages == ~0u ? 0.f : kv.v_scales[(size_t)pages * kv.kv_heads + kvh];
        }
    };
    const auto store_step = [&](uint32_t st, uint32_t buf) {
        if ((int32_t)(st * kKeys + kKeys) > sh.len || odd_pages) {  // codes behind the last key and in holes may be anything: they count as zeros
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                const uint32_t p = threadIdx.x + (uint32_t)i * kThreads, key = p / (D / 16);
                if ((int32_t)(st * kKeys + key) >= sh.len || (odd_pages >> (key / 16 % G) & 1u)) kc[i] = u32x4_t{0u, 0u, 0u, 0u};
                const int32_t have = odd_pages >> (p % G) & 1u ? 0 : sh.len - (int32_t)(st * kKeys + p % G * 16);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int32_t b = have - 4 * j;
                    vc[i][j] = b >= 4 ? vc[i][j] : (b <= 0 ? 0u : vc[i][j] & ~(~0u << (8 * b)));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            const uint32_t p = threadIdx.x + (uint32_t)i * kThreads;
            if (kUneven && p >= kKeys * D / 16) break;
            const uint32_t key = p / (D / 16);
            f16x8_t *kd = (f16x8_t *)&sh_k[buf][Sh::row_of_key(key)][p % (D / 16) * 16];
            kd[0] = codes_f16(u32x2_t{kc[i][0], kc[i][1]});
            kd[1] = codes_f16(u32x2_t{kc[i][2], kc[i][3]});
            f16x8_t *vd = (f16x8_t *)&sh_v[buf][p / G][p % G * 16];
            vd[0] = codes_f16(u32x2_t{vc[i][0], vc[i][1]});
            vd[1] = codes_f16(u32x2_t{vc[i][2], vc[i][3]});
        }
        if (threadIdx.x < G) {
            // A hole's weights are 2^-inf of codes that are zeros.  A scale that is not a number makes its keys' scores NaN.
            const bool hole = vs == 0.f, odd = !(vs == vs);
            const int ev = odd || hole ? 0 : (int)(__builtin_bit_cast(uint32_t, vs) >> 23 & 0xFFu) - 127;
            sh_s[buf][threadIdx.x][0] = odd ? __builtin_nanf("") : ks;
            sh_s[buf][threadIdx.x][1] = hole ? -__builtin_inff() : (float)ev;
            sh_s[buf][threadIdx.x][2] = hole ? 0.f : __builtin_bit_cast(float, (uint32_t)(127 - ev) << 23);
            if constexpr (!PAIRS) {  // whether one of the turn's blocks is far below the largest met (weights_sum)
                int low = hole ? 0x7FFFFFFF : ev;
                e_top = max(e_top, hole ? -1000 : ev);
#pragma unroll
                for (int m = 1; m < (int)G; m *= 2) low = min(low, __shfl_xor(low, m, 64)), e_top = max(e_top, __shfl_xor(e_top, m, 64));
                sh_s[buf][threadIdx.x][3] = low < e_top - kFar ? 1.f : 0.f;
            }
        }
    };

    typename Sh::Acc acc[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) acc[i] = 0.f;
    float M = kNoMax, L = 0.f;
    uint32_t buf = 0;
    uint32_t pages = ~0u;
    if (step < end) {
        const uint32_t pages0 = pages_of(step), pages1 = pages_of(step + 1);
        pages = pages_of(step + 2);
        load_step(step, pages0);
        store_step(step, 0);
        if (step + 1 < end) load_step(step + 1, pages1);
    }
    for (; step < end; step++, buf ^= 1) {
        __syncthreads();
        if (step + 1 < end) store_step(step + 1, buf ^ 1);
        if (step + 2 < end) {
            load_step(step + 2, pages);
            pages = pages_of(step + 3);
        }
        const int32_t key0 = (int32_t)(step * kKeys);
        if (key0 > any_hi || key0 + (int32_t)kKeys <= any_lo) continue;  // (no row of this wavefront sees the step)
        typename Sh::Acc S[ST], zero = 0.f;
#pragma unroll
        for (int k = 0; k < KD; k++) {
#pragma unroll
            for (int t = 0; t < ST; t++) {
                const f16x8_t ka = *(const f16x8_t *)&sh_k[buf][t * Sh::kTileKeys + n][k * Sh::kStepDims + hi * 8];
                S[t] = Sh::mma(ka, qh[k], k ? S[t] : zero);
                if constexpr (QPAIRS) S[t] = Sh::mma(ka, ql[k], S[t]);
            }
        }
        if constexpr (tiles_narrow(NK, PAIRS)) reads_ahead<KD * ST, QPAIRS ? 2 : 1>();
        // x(c, j): the lane's 8 scores of k step c, keys kStepKeys c + 8 hi + j; their logarithm (base 2) with the value scale: x a + e
        float a[KC], e[KC], unscale[KC];
        const bool far = !PAIRS && __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, sh_s[buf][0][3])) != 0;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const uint32_t grp = Sh::group(c, hi);
            a[c] = factor * sh_s[buf][grp][0], e[c] = sh_s[buf][grp][1], unscale[c] = sh_s[buf][grp][2];
        }
#define LARQL_X(c, j) S[Sh::tile(c, j)][Sh::reg(c, j)]
        const bool whole = key0 >= all_lo && key0 + (int32_t)kKeys - 1 <= all_hi;
        if constexpr (CAP != CAP_NONE) {
#pragma unroll
            for (int c = 0; c < KC; c++) {
                float most = 0.f;
                if constexpr (CAP == CAP_ANY)
#pragma unroll
                    for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(LARQL_X(c, j)));
                if (CAP == CAP_ANY && __ballot(most * a[c] >= kSeriesBelow) == 0) {  // (the usual case)
#pragma unroll
                    for (int j = 0; j < 8; j++) LARQL_X(c, j) = capped<CapBy::SERIES>(A, LARQL_X(c, j), a[c], e[c]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) LARQL_X(c, j) = capped<CAP == CAP_ANY ? CapBy::EITHER : CapBy::WHOLE>(A, LARQL_X(c, j), a[c], e[c]);
                }
                a[c] = 1.f, e[c] = 0.f;
            }
        }
        if (!whole) {
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const Seen see(a[c], e[c]);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int32_t key = key0 + c * (int32_t)Sh::kStepKeys + (int32_t)hi * 8 + j;
                    LARQL_X(c, j) = see(LARQL_X(c, j), (int)(key > key_hi) | (int)(key < key_lo));
                }
                a[c] = see.a(), e[c] = see.e();
            }
        }
        float top = kNoMax;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            float m = LARQL_X(c, 0);
#pragma unroll
            for (int j = 1; j < 8; j++) m = fmaxf(m, LARQL_X(c, j));
            top = fmaxf(top, fmaf(m, a[c], e[c]));
        }
        float far_sum = 0.f;
        if (far || __ballot(top > M + kSlack)) {
#pragma unroll
            for (uint32_t d = Sh::kRows; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, (int)d, 64));
            const float next = top > M + kSlack ? ceilf(top) : M;
            const float f = __builtin_amdgcn_exp2f(M - next);
            M = next;
            L *= f;
#pragma unroll
            for (int i = 0; i < DT; i++) acc[i] *= f;
            if (far) {  // (exponentials of its own, hidden from the compiler: those below are to mix with the matrix instructions)
                float top_of = M;
                asm volatile("" : "+v"(top_of));
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; j++) sum += __builtin_amdgcn_exp2f(fmaf(LARQL_X(c, j), a[c], e[c] - top_of + weight_bias(PAIRS)));
                    far_sum = fmaf(sum, unscale[c], far_sum);
                }
            }
        }
        f16x8_t ph[KC], pl[KC];
        float near_sum = 0.f;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const float shift = e[c] - M + weight_bias(PAIRS);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const f32x2_t p = {__builtin_amdgcn_exp2f(fmaf(LARQL_X(c, j), a[c], shift)), __builtin_amdgcn_exp2f(fmaf(LARQL_X(c, j + 1), a[c], shift))};
                weights_f16<PAIRS>(p, ph[c], pl[c], j);
                if constexpr (PAIRS) sum += p[0] + p[1];
            }
            if constexpr (!PAIRS) sum = weights_sum(ph[c]);
            near_sum = fmaf(sum, unscale[c], near_sum);
        }
        L += far ? far_sum : near_sum;
#undef LARQL_X
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const f16x8_t va = *(const f16x8_t *)&sh_v[buf][d * Sh::kRows + n][c * Sh::kStepKeys + hi * 8];
                acc[d] = Sh::mma(va, ph[c], acc[d]);
                if constexpr (PAIRS) acc[d] = Sh::mma(va, pl[c], acc[d]);
            }
        if constexpr (tiles_narrow(NK, PAIRS)) reads_ahead<KC * DT, PAIRS ? 2 : 1>();
    }
#pragma unroll
    for (uint32_t d = Sh::kRows; d < 64; d *= 2) L += __shfl_xor(L, (int)d, 64);
    if (!live) return;
    // acc[d][4 i + j]: channel kRows d + 8 i + 4 hi + j
    constexpr int QUADS = sizeof(typename Sh::Acc) / 16;
    const auto quad = [&](int d, int i) { return f32x4_t{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]}; };
    if (it.pieces > 1) {
        const size_t at = ((size_t)kvh * part.slots + it.slot + it.piece) * kTilesTile + wave * Sh::kRows + n;
        if (hi == 0) part.ml[2 * at] = M, part.ml[2 * at + 1] = L;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < QUADS; i++) *(f32x4_t *)(part.acc + at * D + d * Sh::kRows + i * 8 + hi * 4) = quad(d, i);
        return;
    }
    const float inv = inverse_sum(A, L, M, head);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < QUADS; i++)
            store4(A.out, A.out_type, (size_t)(sh.row + tok) * A.out_stride + (size_t)head * D + d * Sh::kRows + i * 8 + hi * 4, quad(d, i) * inv);
}

// One query row of a split tile: pieces p0, p0 + step, ... as one sum.  `at`: the row in the first piece.
__device__ __forceinline__ void join_pieces(const Partials &part, uint32_t tile, uint32_t D, size_t at, uint32_t pieces, uint32_t p0, uint32_t step, uint32_t dim,
                                            float &top, float &l, f32x4_t &o) {
    top = kNoMax, l = 0.f;
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (; p0 < pieces; p0 += 8 * step) {
        float m[8], s[8];
        f32x4_t a[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {  // (beyond the last piece: the last once more, with no weight)
            const uint32_t p = p0 + i * step;
            const size_t x = at + (size_t)min(p, pieces - 1) * tile;
            m[i] = p < pieces ? part.ml[2 * x] : kNoMax;
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
            if (p0 + i * step >= pieces) break;
            const float w = __builtin_amdgcn_exp2f(m[i] - top);
            l = fmaf(w, s[i], l);
            o += a[i] * w;
        }
    }
}

// The pieces of split rows as one, of both kernels: a workgroup for kJoinRows rows of a split tile, `share` of its wavefronts (1, 2, 4 or 8)
// for a row.
constexpr uint32_t kJoinRows = 16, kJoinWaves = 8;
struct Join {
    Plan plan[2];
    Partials part[2];
    uint32_t split_tiles[2];  // at most
    uint32_t parts[2];        // workgroups of a tile
    uint32_t share;
};
__global__ void __launch_bounds__(kJoinWaves * 64) attention_join_kernel(AttentionArgs A, Join J) {
    __shared__ float sh_acc[kJoinWaves][256], sh_ml[kJoinWaves][2];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, D = A.kv.head_dim, dim = min(lane * 4, D - 4), share = J.share;
    const uint32_t kvh = blockIdx.y, group = A.group.d;
    const uint32_t of_first = J.split_tiles[0] * J.parts[0];
    const bool second = blockIdx.x >= of_first;
    const Plan P = second ? J.plan[1] : J.plan[0];
    const Partials part = second ? J.part[1] : J.part[0];
    const uint32_t at_tile = second ? blockIdx.x - of_first : blockIdx.x, parts = second ? J.parts[1] : J.parts[0], part_of = at_tile % parts;
    Item it;
    Share sh;
    if (!find_item(A, P, at_tile / parts, true, it, sh)) return;
    const uint32_t row0 = (P.tile == kTilesTile ? sh.tiles - 1 - it.tile : it.tile) * P.tile;
    const size_t at = ((size_t)kvh * part.slots + it.slot) * P.tile;
    const uint32_t end = min((part_of + 1) * kJoinRows, min(P.tile, sh.n * group - row0));
    for (uint32_t r0 = part_of * kJoinRows; r0 < end; r0 += kJoinWaves / share) {
        const uint32_t r = r0 + wave / share;
        float top = kNoMax, l = 0.f;
        f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (r < end) join_pieces(part, P.tile, D, at + r, it.pieces, wave % share, share, dim, top, l, o);
        if (share > 1) {
            __syncthreads();  // (the rows before have been read)
            if (lane == 0) sh_ml[wave][0] = top, sh_ml[wave][1] = l;
            if (lane * 4 < D) *(f32x4_t *)&sh_acc[wave][lane * 4] = o;
            __syncthreads();
            if (wave % share) continue;
            for (uint32_t w = wave + 1; w < wave + share; w++) top = fmaxf(top, sh_ml[w][0]);
            l = 0.f;
            o = f32x4_t{0.f, 0.f, 0.f, 0.f};
            for (uint32_t w = wave; w < wave + share; w++) {
                const float f = __builtin_amdgcn_exp2f(sh_ml[w][0] - top);
                l = fmaf(f, sh_ml[w][1], l);
                o += *(const f32x4_t *)&sh_acc[w][dim] * f;
            }
        }
        if (r >= end || lane * 4 >= D) continue;
        const uint32_t q = row0 + r, h = kvh * group + A.group.rest(q);
        const float inv = inverse_sum(A, l, top, h);
        const f32x4_t v = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        store4(A.out, A.out_type, (size_t)(sh.row + A.group.of(q)) * A.out_stride + (size_t)h * D + lane * 4, v);
    }
}

// Partial results of one of the kernels, from `at` on.
static Partials partials_of(const AttentionArgs &A, const Plan &P, float *at, float **end) {
    const size_t rows = Plans::slots(P) * A.kv.kv_heads * P.tile;
    *end = at + rows * (A.kv.head_dim + 2);
    return {at, at + rows * A.kv.head_dim, (uint32_t)Plans::slots(P)};
}
static size_t partial_floats(const AttentionArgs &A, const Plan &P) { return Plans::slots(P) * A.kv.kv_heads * P.tile * (size_t)(A.kv.head_dim + 2); }

uint64_t attention_blocks(const AttentionArgs &A) {
    const Plans p = plans_of(A);
    return std::max(p.use_rows ? Plans::items(A, p.rows) : 0, p.use_tiles ? Plans::items(A, p.tiles) : 0) * A.kv.kv_heads;
}
size_t attention_workspace_bytes(const AttentionArgs &A) {
    const Plans p = plans_of(A);
    return ((p.use_rows ? partial_floats(A, p.rows) : 0) + (p.use_tiles ? partial_floats(A, p.tiles) : 0)) * sizeof(float) + 16;
}
int attention_launches(const AttentionArgs &A) {
    const Plans p = plans_of(A);
    const bool join = (p.use_rows && p.rows.split) || (p.use_tiles && p.tiles.split);
    return (int)p.use_rows + (int)p.use_tiles + (int)join;
}

template <int NK>
static void launch_rows(hipStream_t s, const AttentionArgs &A, const Plan &P, const Partials &part, uint32_t items) {
    const dim3 grid(items, A.kv.kv_heads), threads(kAttnThreads);  // (at most 2 * 2^16 tiles and the target: far below 2^24)
    if (A.softcap > 0.f) hipLaunchKernelGGL((attention_rows_kernel<NK, true>), grid, threads, 0, s, A, P, part);
    else hipLaunchKernelGGL((attention_rows_kernel<NK, false>), grid, threads, 0, s, A, P, part);
}
template <int NK, bool QPAIRS, bool PAIRS>
static void launch_tiles(hipStream_t s, const AttentionArgs &A, const Plan &P, const Partials &part, uint32_t items) {
    const dim3 grid = grid_of((uint64_t)items * A.kv.kv_heads), threads(Shape<tiles_narrow(NK, PAIRS)>::kWaves * 64);
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, threads, 0, s, A, P, part); };
    if (A.softcap == 0.f) return launch(attention_tiles_kernel<NK, QPAIRS, PAIRS, CAP_NONE>);
    if constexpr (!PAIRS)
        if (A.softcap <= kLowCap) return launch(attention_tiles_kernel<NK, QPAIRS, PAIRS, CAP_LOW>);
    launch(attention_tiles_kernel<NK, QPAIRS, PAIRS, CAP_ANY>);
}
// One f16 holds a 16-bit query, but 11 of an f32 query's 24 bits, and what a score loses grows with the score: f32 queries enter as f16 pairs
// whatever the result's type (a causal prompt of 4096 f32 queries, 32/8 heads of 128, into bf16: 242 us for 203; 8/4 of 256 into f16: 195 for 191, and
// 2.6e-4 from 64 bits for 4.6e-4).  Weights of many rows into 16 bits are one f16: pairs, a second product more, would take 782 us for 632 (a causal
// prompt of 8192, 32/8 heads of 128, bf16: 1.65e-3 from 64 bits for 1.66e-3) and 231 for 187 (4096, f16: 2.1e-4 for 2.5e-4).
template <int NK>
static void launch_dim(hipStream_t s, const AttentionArgs &A, const Plan &P, const Partials &part, bool tiles) {
    const uint32_t items = (uint32_t)Plans::items(A, P);
    const bool f32_query = A.q_type == ELEM_F32, f32_result = A.out_type == ELEM_F32;
    if (!tiles) {
        launch_rows<NK>(s, A, P, part, items);
    } else if (f32_result) {
        launch_tiles<NK, true, true>(s, A, P, part, items);
    } else if (f32_query) {
        launch_tiles<NK, true, false>(s, A, P, part, items);
    } else {
        launch_tiles<NK, false, false>(s, A, P, part, items);
    }
}

static hipError_t launch_plan(hipStream_t s, const AttentionArgs &A, const Plan &P, const Partials &part, bool tiles) {
    switch (A.kv.head_dim / 32) {
    case 1: launch_dim<1>(s, A, P, part, tiles); break;
    case 2: launch_dim<2>(s, A, P, part, tiles); break;
    case 3: launch_dim<3>(s, A, P, part, tiles); break;
    case 4: launch_dim<4>(s, A, P, part, tiles); break;
    case 5: launch_dim<5>(s, A, P, part, tiles); break;
    case 6: launch_dim<6>(s, A, P, part, tiles); break;
    case 7: launch_dim<7>(s, A, P, part, tiles); break;
    case 8: launch_dim<8>(s, A, P, part, tiles); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t attention_launch(hipStream_t s, const AttentionArgs &A, void *workspace) {
    const Plans p = plans_of(A);
    float *at = (float *)workspace;
    hipError_t e = hipSuccess;
    Join J = {};
    uint32_t rows = 0;  // of a split tile, at most
    const auto run = [&](const Plan &P, bool tiles) {
        const Partials part = partials_of(A, P, at, &at);
        if (e == hipSuccess) e = launch_plan(s, A, P, part, tiles);
        const int i = tiles ? 0 : 1;
        J.plan[i] = P;
        J.part[i] = part;
        J.split_tiles[i] = (uint32_t)Plans::split_tiles(A, P);
        const uint32_t most = (uint32_t)std::min<uint64_t>((uint64_t)A.kv.max_new * A.group.d, P.tile);
        J.parts[i] = (most + kJoinRows - 1) / kJoinRows;
        if (P.split) rows = std::max(rows, most);
    };
    if (p.use_tiles) run(p.tiles, true);
    if (p.use_rows) run(p.rows, false);
    const uint32_t groups = J.split_tiles[0] * J.parts[0] + J.split_tiles[1] * J.parts[1];
    if (e != hipSuccess || groups == 0) return e;
    J.share = rows <= 1 ? 8 : rows <= 2 ? 4 : rows <= 4 ? 2 : 1;
    hipLaunchKernelGGL(attention_join_kernel, dim3(groups, A.kv.kv_heads), dim3(kJoinWaves * 64), 0, s, A, J);
    return hipGetLastError();
}

}  // namespace larql
