// norm.hip — the residual between two blocks and the norms around it:
//   h' = h + s * g . rms(b; w_post),  n = rms(h'; w_pre),  rms(x; w) = x / sqrt(mean(x^2) + eps) * (offset + w)
// A row is read once and kept in registers over both reductions, so many rows are bound by memory: 4096 of 3840 (f32 block and stream, bf16
// result) take 39.4 us, 5.6 TB/s of reads and writes (a large copy: 5.0); of 3841, element by element, 48.  A single row is bound by its launch:
// 2.8 us at 2560, the shortest kernel here 2.6.  Few rows with a gate are bound by a chain of waits: block, residual (each converted by its type where
// it is loaded), and behind the first sum the weights and the gate; 77 rows of 2880 in f16 4.4 us.  A thread holds 8 elements where the row's threads
// allow it (fewer waits a row), at most 32.
#include "kernels.h"
#include "layer.h"

namespace larql {

constexpr int kNormChunks = 4;  // groups of 8 elements a thread holds

// Sum of v over the TPR threads of a row.
template <uint32_t TPR>
__device__ __forceinline__ float row_sum(float v, float *part) {
    v = wave_fsum(v);
    if constexpr (TPR > 64) {
        const uint32_t wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) part[wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < TPR / 64; w++) v += part[w];
    }
    return v;
}

// TPR threads serve a row, which holds at most TPR * 8 * NC elements.  VEC: groups of 8 elements by 16-byte accesses; else thread t
// holds elements t, t + TPR, ...
template <uint32_t TPR, int NC, bool VEC>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) residual_norm_kernel(NormArgs A) {
    constexpr uint32_t kRows = TPR < 256 ? (TPR == 64 ? 4 : 1) : 1;
    __shared__ float part[2][16];
    const uint32_t row = block_number() * kRows + threadIdx.x / TPR, t = threadIdx.x % TPR;
    if (row >= A.rows) return;  // (whole waves, and only where a row is one wave's)
    const char *block = A.block ? (const char *)A.block + row * A.block_stride * elem_bytes(A.block_type) : nullptr;
    const char *res = (const char *)A.residual + row * A.residual_stride * elem_bytes(A.residual_type);
    char *res_out = A.residual_out ? (char *)A.residual_out + row * A.residual_out_stride * elem_bytes(A.residual_type) : nullptr;
    char *normed = A.normed ? (char *)A.normed + row * A.normed_stride * elem_bytes(A.normed_type) : nullptr;
    const float *gate = A.gate ? A.gate + row * A.gate_stride : nullptr;
    const auto at = [&](int c, int j) -> uint32_t { return VEC ? (t + (uint32_t)c * TPR) * 8 + (uint32_t)j : t + (uint32_t)(c * 8 + j) * TPR; };
    const auto get = [&](const void *p, int type, int c, float (&o)[8]) {
        if constexpr (VEC) {
            const Eight v = load8(p, type, at(c, 0));
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = at(c, j) < A.hidden ? load_elem(p, type, at(c, j)) : 0.f;
        }
    };
    const auto put = [&](void *p, int type, int c, const float (&v)[8]) {
        if constexpr (VEC) {
            store8(p, type, at(c, 0), Eight{f32x4_t{v[0], v[1], v[2], v[3]}, f32x4_t{v[4], v[5], v[6], v[7]}});
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (at(c, j) < A.hidden) store_elem(p, type, at(c, j), v[j]);
        }
    };
    float b[NC][8] = {}, h[NC][8] = {};
#pragma unroll
    for (int c = 0; c < NC; c++)
        if (at(c, 0) < A.hidden) {
            if (block) get(block, A.block_type, c, b[c]);
            get(res, A.residual_type, c, h[c]);
        }
    const float inv_n = 1.f / (float)A.hidden;
    float scale = A.residual_scale;
    if (block) {
        if (A.post_weight) {
            float sq = 0.f;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int j = 0; j < 8; j++) sq = fmaf(b[c][j], b[c][j], sq);
            scale *= 1.f / sqrtf(row_sum<TPR>(sq, part[0]) * inv_n + A.eps);
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
            if (at(c, 0) < A.hidden) {
                float w[8];
                if (A.post_weight) {
                    get(A.post_weight, ELEM_F32, c, w);
#pragma unroll
                    for (int j = 0; j < 8; j++) b[c][j] *= A.norm_offset + w[j];
                }
                if (gate) {
                    get(gate, ELEM_F32, c, w);
#pragma unroll
                    for (int j = 0; j < 8; j++) b[c][j] *= w[j];
                }
#pragma unroll
                for (int j = 0; j < 8; j++) h[c][j] = fmaf(scale, b[c][j], h[c][j]);
            }
    }
    if (res_out)
#pragma unroll
        for (int c = 0; c < NC; c++)
            if (at(c, 0) < A.hidden) put(res_out, A.residual_type, c, h[c]);
    if (!normed) return;
    float sq = 0.f;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) sq = fmaf(h[c][j], h[c][j], sq);
    const float r = 1.f / sqrtf(row_sum<TPR>(sq, part[1]) * inv_n + A.eps);
#pragma unroll
    for (int c = 0; c < NC; c++)
        if (at(c, 0) < A.hidden) {
            float w[8], o[8];
            if (A.pre_weight) get(A.pre_weight, ELEM_F32, c, w);
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = h[c][j] * r * (A.pre_weight ? A.norm_offset + w[j] : 1.f);
            put(normed, A.normed_type, c, o);
        }
}

template <uint32_t TPR, bool VEC>
static void launch_rows(hipStream_t s, const NormArgs &A) {
    const uint32_t threads = TPR < 256 ? (TPR == 64 ? 256 : TPR) : TPR, rows = threads / TPR;
    const dim3 grid = grid_of((A.rows + rows - 1) / rows);
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, A); };
    if constexpr (TPR == 1024) {  // the most threads: longer rows are more groups a thread
        const uint32_t chunks = (A.hidden + TPR * 8 - 1) / (TPR * 8);
        if (chunks > 2) return launch(residual_norm_kernel<TPR, kNormChunks, VEC>);
        if (chunks > 1) return launch(residual_norm_kernel<TPR, 2, VEC>);
    }
    launch(residual_norm_kernel<TPR, 1, VEC>);
}

template <bool VEC>
static void launch_vec(hipStream_t s, const NormArgs &A) {
    const uint32_t groups = (A.hidden + 7) / 8;
    if (groups <= 64) launch_rows<64, VEC>(s, A);
    else if (groups <= 128) launch_rows<128, VEC>(s, A);
    else if (groups <= 256) launch_rows<256, VEC>(s, A);
    else if (groups <= 512) launch_rows<512, VEC>(s, A);
    else launch_rows<1024, VEC>(s, A);
}

hipError_t residual_norm_launch(hipStream_t s, const NormArgs &A) {
    if (A.vec) launch_vec<true>(s, A);
    else launch_vec<false>(s, A);
    return hipGetLastError();
}

}  // namespace larql
