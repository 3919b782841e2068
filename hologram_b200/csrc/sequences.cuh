// What the calls over several packed sequences share: the sequence a row belongs to, stores rounded to nearest, and the general
// attention kernel that serves every shape.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "numerics.cuh"

namespace {

__device__ __forceinline__ float seq_load(const void* p, uint64_t i, int dtype) {
    if (dtype == HOLO_DTYPE_F32) return ((const float*)p)[i];
    if (dtype == HOLO_DTYPE_BF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
    return __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void seq_store(void* p, uint64_t i, float v, int dtype) {
    if (dtype == HOLO_DTYPE_F32) ((float*)p)[i] = v;
    else if (dtype == HOLO_DTYPE_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
    else ((__half*)p)[i] = __float2half_rn(v);
}

// The last s in [0, n] with starts[s] <= row, or -1. Whatever starts hold, the search ends and reads starts[0 .. n] only; starts[s] <= row
// then holds for what it returns. Empty sequences end where they begin, so the last of equal starts is the one that has the row.
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ starts, uint32_t n, int64_t row) {
    int lo = -1, hi = (int)n;
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (starts[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// Rows [begin, end) of the sequence that has `row`; false when none does.
__device__ __forceinline__ bool sequence_of(const int32_t* __restrict__ starts, uint32_t n, uint32_t rows, uint32_t row, uint32_t* begin, uint32_t* end, uint32_t* which) {
    const int s = find_sequence(starts, n, row);
    if (s < 0 || s >= (int)n) return false;
    const int b = starts[s], e = starts[s + 1];
    if (b < 0 || e <= (int)row) return false;
    *begin = (uint32_t)b;
    *end = min((uint32_t)e, rows);
    *which = (uint32_t)s;
    return true;
}
// One block of the launch looks every sequence's starts over (and its length, where there is one).
__device__ __forceinline__ void check_sequences(const int32_t* starts, const int32_t* lengths, uint32_t n, uint32_t rows, int64_t most, uint32_t* status) {
    bool bad = false;
    for (uint32_t s = threadIdx.x; s < n; s += blockDim.x) {
        const int64_t b = starts ? starts[s] : 0, e = starts ? starts[s + 1] : 1;
        bad |= b < 0 || e < b || e > (starts ? (int64_t)rows : 1);
        if (lengths) bad |= lengths[s] < e - b || lengths[s] > most;
    }
    if (bad) atomicOr(status, HOLO_STATUS_TABLE);
}

constexpr int SEQ_WARPS = 4;
constexpr int SEQ_PER_LANE = 16;      // dims up to 512

// Attention of any shape: a CTA takes one (row, head) after another; its warps take every fourth key, each with a maximum, a sum and a
// context of its own, merged at the end. A lane holds dims lane, lane + 32, ... Only keys that the row sees are read. It serves what the
// tiled kernels do not: dims that are no multiple of 16, rows that are not 16-byte aligned.
template <class Source>
__global__ void __launch_bounds__(SEQ_WARPS * 32)
general_rows_kernel(const __grid_constant__ Source src) {
    extern __shared__ float s_mem[];      // [SEQ_WARPS][vdim + 2]
    holo_pdl_trigger();
    holo_pdl_wait();
    if (blockIdx.x == 0) src.check();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, vdim = src.vdim(), heads = src.heads();
    const uint64_t units = (uint64_t)src.rows() * heads;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t row = (uint32_t)(u / heads), head = (uint32_t)(u % heads);
        typename Source::Place at;
        if (!src.place(row, &at)) continue;
        float q[SEQ_PER_LANE], o[SEQ_PER_LANE];
#pragma unroll
        for (int i = 0; i < SEQ_PER_LANE; ++i) {
            const uint32_t c = lane + 32 * i;
            q[i] = c < src.dim() ? src.q(row, head, c) : 0.0f;
            o[i] = 0.0f;
        }
        float top = -INFINITY, sum = 0.0f;
        for (uint32_t j = at.begin + warp; j < at.end; j += SEQ_WARPS) {
            uint64_t kb, vb;
            float ks, vs;
            src.key(at, head, j, &kb, &vb, &ks, &vs);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < SEQ_PER_LANE; ++i) {
                const uint32_t c = lane + 32 * i;
                if (c < src.dim()) s = fmaf(q[i], src.k(kb + c), s);
            }
            for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            s *= ks * src.scale();
            if (s == -INFINITY) continue;
            // a score that is NaN or +inf makes the row NaN
            const float most = s > top ? s : top, f = expf(top - most), p = expf(s - most);
            top = most;
            sum = sum * f + p;
#pragma unroll
            for (int i = 0; i < SEQ_PER_LANE; ++i) {
                const uint32_t c = lane + 32 * i;
                if (c < vdim) o[i] = fmaf(p, src.v(vb + c) * vs, o[i] * f);
            }
        }
        float* mine = s_mem + warp * (vdim + 2);
#pragma unroll
        for (int i = 0; i < SEQ_PER_LANE; ++i)
            if (lane + 32 * i < vdim) mine[lane + 32 * i] = o[i];
        if (lane == 0) {
            mine[vdim] = top;
            mine[vdim + 1] = sum;
        }
        __syncthreads();
        float most = -INFINITY, total = 0.0f, f[SEQ_WARPS];
        for (int w = 0; w < SEQ_WARPS; ++w) most = fmaxf(most, s_mem[w * (vdim + 2) + vdim]);
#pragma unroll
        for (int w = 0; w < SEQ_WARPS; ++w) {
            const float t = s_mem[w * (vdim + 2) + vdim], l = s_mem[w * (vdim + 2) + vdim + 1];
            f[w] = l == 0.0f ? 0.0f : expf(t - most);
            total += f[w] * l;
        }
        for (uint32_t c = threadIdx.x; c < vdim; c += blockDim.x) {
            float acc = 0.0f;
#pragma unroll
            for (int w = 0; w < SEQ_WARPS; ++w)
                if (f[w] != 0.0f) acc = fmaf(f[w], s_mem[w * (vdim + 2) + c], acc);     // NaN is not 0
            src.store(row, head, c, total == 0.0f ? 0.0f : acc / total);
        }
        __syncthreads();
    }
}
template <class Source>
int32_t launch_general_rows(holo_b200_ctx* ctx, const Source& src, uint64_t units, uint32_t vdim) {
    const uint64_t most = (uint64_t)ctx->sm_count * 16;
    HOLO_CUDA(holo_launch_kernel(ctx, general_rows_kernel<Source>, dim3((uint32_t)(units < most ? units : most)), dim3(SEQ_WARPS * 32),
                                 SEQ_WARPS * (vdim + 2) * sizeof(float), 1, src));
    ctx->launches++;
    return HOLO_OK;
}

}  // namespace
