// layer.h — what a decoder layer does between its matrix products (norm.hip, kv_append.hip, attention.hip): arguments of the
// kernels, and what they share on the device.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave.h"

namespace larql {

// A launch takes fewer than 2^32 threads in a dimension of its grid: workgroups beyond kGridRow go into a second one, whose last row may have
// some that are too many.  Their number is below 2^31 (the callers' checks).
constexpr uint32_t kGridRowShift = 20, kGridRow = 1u << kGridRowShift;
constexpr uint64_t kMaxBlocks = 0x7FFFFFFFull;
inline dim3 grid_of(uint64_t blocks) {
    return blocks <= kGridRow ? dim3((uint32_t)blocks) : dim3(kGridRow, (uint32_t)((blocks + kGridRow - 1) >> kGridRowShift));
}
__device__ __forceinline__ uint32_t block_number() { return blockIdx.y << kGridRowShift | blockIdx.x; }

enum ElemType : int32_t { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };
__host__ __device__ constexpr uint32_t elem_bytes(int t) { return t == ELEM_F32 ? 4u : 2u; }

struct NormArgs {  // strides in elements
    const void *block, *residual;
    void *residual_out, *normed;
    const float *gate, *post_weight, *pre_weight;
    size_t block_stride, residual_stride, residual_out_stride, normed_stride, gate_stride;
    int32_t block_type, residual_type, normed_type;
    uint32_t rows, hidden;
    float residual_scale, norm_offset, eps;
    uint32_t vec;  // every row of every operand starts 16-byte aligned and holds whole groups of 8 elements
};
constexpr uint32_t kNormMaxHidden = 32768;
hipError_t residual_norm_launch(hipStream_t s, const NormArgs &A);

// The paged cache and the sequences of a step (larql_hip_kv_cache, larql_hip_kv_batch).
struct KvArgs {
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    const int32_t *kv_len, *block_table, *q_start;
    uint32_t num_pages, kv_heads, head_dim, page_shift;  // page_tokens = 1 << page_shift
    uint32_t sequences, table_width, tokens, max_new;
};
constexpr int kScaleMinExp = -40, kScaleMaxExp = 60;

struct KvAppendArgs {
    KvArgs kv;
    const void *q, *k, *v;
    void *q_out;
    size_t q_stride, q_out_stride, k_stride, v_stride;
    const float *inv_freq, *q_norm, *k_norm;
    int32_t type;
    uint32_t q_heads, rot_dim, interleaved;
    float rope_scale, norm_offset, norm_eps;
};
constexpr size_t kMaxRowStride = 1u << 22;  // elements between tokens
uint64_t kv_append_blocks(const KvAppendArgs &A);  // workgroups of a launch
hipError_t kv_append_launch(hipStream_t s, const KvAppendArgs &A);

// Division by a number that the host knows: (n * mul / 2^32 + n) / 2^shift, exact for every n below 2^31.
struct Divisor {
    uint32_t d, mul, shift;
    static Divisor by(uint32_t d) {
        uint32_t shift = 0;
        while (((uint64_t)1 << shift) < d) shift++;
        return {d, (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1), shift};
    }
    __host__ __device__ uint32_t of(uint32_t n) const { return ((uint32_t)(((uint64_t)n * mul) >> 32) + n) >> shift; }
    __host__ __device__ uint32_t rest(uint32_t n) const { return n - of(n) * d; }
};

struct AttentionArgs {
    KvArgs kv;
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    const float *sinks;
    int32_t q_type, out_type;
    uint32_t q_heads, window, causal;
    Divisor group;  // query heads of a key/value head
    float scale, softcap;
};
uint64_t attention_blocks(const AttentionArgs &A);  // workgroups of its largest launch
size_t attention_workspace_bytes(const AttentionArgs &A);
int attention_launches(const AttentionArgs &A);
hipError_t attention_launch(hipStream_t s, const AttentionArgs &A, void *workspace);

// ---- device ---------------------------------------------------------------------------------------------------------

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t b) { return __builtin_bit_cast(float, b << 16); }
// to nearest even; a NaN stays one
__device__ __forceinline__ uint32_t f32_to_bf16_rne(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return x != x ? (u >> 16) | 0x40u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ uint32_t f32_to_f16_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
__device__ __forceinline__ float f16_bits_to_f32(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }

// element i of a row
__device__ __forceinline__ float load_elem(const void *p, int type, size_t i) {
    if (type == ELEM_F32) return ((const float *)p)[i];
    const uint32_t b = ((const uint16_t *)p)[i];
    return type == ELEM_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}
__device__ __forceinline__ void store_elem(void *p, int type, size_t i, float v) {
    if (type == ELEM_F32) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = (uint16_t)(type == ELEM_BF16 ? f32_to_bf16_rne(v) : f32_to_f16_bits(v));
}
// Groups of elements from an offset at which the address is aligned to the group, at most 16 bytes.  (By value: stores through references that
// both sides of a branch make would keep the array in memory.)
__device__ __forceinline__ f32x4_t unpack4(int type, u32x2_t a) {
    if (type == ELEM_BF16)
        return f32x4_t{bf16_bits_to_f32(a[0]), __builtin_bit_cast(float, a[0] & 0xFFFF0000u), bf16_bits_to_f32(a[1]), __builtin_bit_cast(float, a[1] & 0xFFFF0000u)};
    return f32x4_t{f16_bits_to_f32(a[0] & 0xFFFFu), f16_bits_to_f32(a[0] >> 16), f16_bits_to_f32(a[1] & 0xFFFFu), f16_bits_to_f32(a[1] >> 16)};
}
__device__ __forceinline__ uint32_t pack2(int type, float a, float b) {
    return type == ELEM_BF16 ? f32_to_bf16_rne(a) | f32_to_bf16_rne(b) << 16 : f32_to_f16_bits(a) | f32_to_f16_bits(b) << 16;
}
__device__ __forceinline__ f32x2_t load2(const void *p, int type, uint32_t i) {
    if (type == ELEM_F32) return *(const f32x2_t *)((const float *)p + i);
    const f32x4_t v = unpack4(type, u32x2_t{*(const uint32_t *)((const uint16_t *)p + i), 0u});
    return f32x2_t{v[0], v[1]};
}
__device__ __forceinline__ f32x4_t load4(const void *p, int type, uint32_t i) {
    if (type == ELEM_F32) return *(const f32x4_t *)((const float *)p + i);
    return unpack4(type, *(const u32x2_t *)((const uint16_t *)p + i));
}
__device__ __forceinline__ void store4(void *p, int type, size_t i, f32x4_t v) {
    if (type == ELEM_F32) *(f32x4_t *)((float *)p + i) = v;
    else *(u32x2_t *)((uint16_t *)p + i) = u32x2_t{pack2(type, v[0], v[1]), pack2(type, v[2], v[3])};
}
struct Eight {
    f32x4_t a, b;
    __device__ __forceinline__ float operator[](int i) const { return i < 4 ? a[i] : b[i - 4]; }
};
__device__ __forceinline__ Eight load8(const void *p, int type, size_t i) {
    if (type == ELEM_F32) return {*(const f32x4_t *)((const float *)p + i), *(const f32x4_t *)((const float *)p + i + 4)};
    const u32x4_t v = *(const u32x4_t *)((const uint16_t *)p + i);
    return {unpack4(type, u32x2_t{v[0], v[1]}), unpack4(type, u32x2_t{v[2], v[3]})};
}
__device__ __forceinline__ void store8(void *p, int type, size_t i, const Eight &v) {
    if (type == ELEM_F32) {
        *(f32x4_t *)((float *)p + i) = v.a;
        *(f32x4_t *)((float *)p + i + 4) = v.b;
        return;
    }
    *(u32x4_t *)((uint16_t *)p + i) = u32x4_t{pack2(type, v.a[0], v.a[1]), pack2(type, v.a[2], v.a[3]), pack2(type, v.b[0], v.b[1]), pack2(type, v.b[2], v.b[3])};
}

// The page of a sequence's token at `key` (its table's row at `table`), or ~0: a hole, or beyond the table.
__host__ __device__ __forceinline__ uint32_t kv_page(const KvArgs &kv, const int32_t *table, uint32_t key) {
    const uint32_t j = key >> kv.page_shift;
    if (j >= kv.table_width) return ~0u;
    const uint32_t p = (uint32_t)table[j];
    return p < kv.num_pages ? p : ~0u;
}

// New tokens of sequence s: their first row, or none where the rows do not fit.
struct NewTokens {
    uint32_t row, n;
    int32_t len;  // of the sequence, new tokens included
};
__host__ __device__ __forceinline__ NewTokens new_tokens(const KvArgs &kv, uint32_t s) {
    const int32_t a = kv.q_start[s], b = kv.q_start[s + 1], len = kv.kv_len[s];
    const bool fits = a >= 0 && b >= a && (uint32_t)b <= kv.tokens && (uint32_t)(b - a) <= kv.max_new;
    return {fits ? (uint32_t)a : 0u, fits ? (uint32_t)(b - a) : 0u, len < 0 ? 0 : len};
}

}  // namespace larql
