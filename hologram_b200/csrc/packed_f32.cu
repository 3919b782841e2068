// Attention of packed f32 sequences (the PackedAttention call) on the CUDA cores, for dims in steps of 4 up to 128: f32 products and sums.
//
// A CTA takes 16 * NR packed rows of a head, whatever sequences they belong to, and the keys from its first row's sequence on to the last key
// any of its rows sees; NG groups of NR warps each take every NG-th tile of 64 keys and their results are added at the end. A warp
// holds 16 rows: a thread 4 rows x 8 keys of the scores and 4 rows x D / 8 columns of the context, all as packed pairs (fma.rn.f32x2).
// K arrives while the previous tile's context is added up, V while the scores are computed: one buffer each. Dot products are summed in
// runs of 32 elements. Bound: the FMA rate, and beside it reads of shared memory (12 128-bit reads for 64 packed multiply-adds).
//
// A weight of zero times an infinite or NaN value is NaN: in tiles that some row of a warp does not see whole, keys are added row by row.
#include "sequences.cuh"

namespace {

constexpr int PF_TILE = 64;                 // keys
constexpr int PF_LD = PF_TILE + 8;          // weights: the four rows a warp writes together start 8 banks apart

__device__ __forceinline__ uint64_t twice(float a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(a));
    return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 16 bytes to shared memory, or 16 zero bytes when `take` is false (nothing is read then)
__device__ __forceinline__ void pf_copy(float* dst, const float* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(take ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void pf_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void pf_arrived() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

template <int D, int NR, int NG>
struct PackedF32Layout {
    static constexpr int ROWS = 16 * NR, WARPS = NR * NG, LD = D + 4;
    static constexpr int Q = ROWS * LD, GROUP = PF_TILE * LD + PF_TILE * D, P = WARPS * 16 * PF_LD;
    static constexpr int FLOATS = Q + NG * GROUP + P;
    static_assert(NG * ROWS * (D + 2) <= NG * GROUP, "the groups' results fit in the tiles' memory");
};

template <int D, int NR, int NG>
__global__ void __launch_bounds__(NR * NG * 32, D <= 64 && NR * NG <= 4 ? 3 : 1)
packed_f32_kernel(const __grid_constant__ HoloPackedArgs a) {
    using L = PackedF32Layout<D, NR, NG>;
    extern __shared__ __align__(16) float smem[];
    __shared__ uint2 s_range[L::ROWS];        // keys each row sees; none for rows of no sequence
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = warp / NR, wrow = warp % NR;
    // lanes' bits in the order column, row, column, column, row: 128-bit reads then take two wavefronts
    const uint32_t tx = (lane & 1) | ((lane >> 1) & 6), ty = ((lane >> 1) & 1) | ((lane >> 3) & 2);
    const uint32_t head = blockIdx.x, g = head / (a.heads / a.kv_heads);
    const uint32_t row0 = (gridDim.y - 1 - blockIdx.y) * L::ROWS;      // a long causal sequence: the rows with the most keys first
    float *s_q = smem, *s_k = smem + L::Q + group * L::GROUP, *s_v = s_k + PF_TILE * L::LD;
    float* s_p = smem + L::Q + NG * L::GROUP + warp * 16 * PF_LD;
    holo_pdl_trigger();
    holo_pdl_wait();
    const uint32_t dvec = a.dim / 4, vvec = a.vdim / 4;
    {
        const float* q = (const float*)a.q + (uint64_t)row0 * a.q_ld + (uint64_t)head * a.dim;
        for (uint32_t i = tid; i < L::ROWS * (D / 4); i += L::WARPS * 32) {
            const uint32_t r = i / (D / 4), c = i % (D / 4);
            const bool take = row0 + r < a.rows && c < dvec;
            pf_copy(s_q + r * L::LD + 4 * c, take ? q + (uint64_t)r * a.q_ld + 4 * c : (const float*)a.q, take);
        }
    }
    if (blockIdx.x == 0 && blockIdx.y == 0) check_sequences(a.starts, nullptr, a.sequences, a.rows, 0, a.status);
    if (tid < L::ROWS) {
        uint32_t begin = 0, end = 0, which;
        if (row0 + tid < a.rows && sequence_of(a.starts, a.sequences, a.rows, row0 + tid, &begin, &end, &which)) {
            if (a.causal) end = row0 + tid + 1;
        } else {
            begin = end = 0;
        }
        s_range[tid] = make_uint2(begin, end);
    }
    __syncthreads();
    uint32_t first = 0xffffffffu, last = 0;
    for (uint32_t r = lane; r < L::ROWS; r += 32) {
        const uint2 x = s_range[r];
        if (x.y > x.x) {
            first = min(first, x.x);
            last = max(last, x.y);
        }
    }
    first = __reduce_min_sync(0xffffffffu, first);
    last = __reduce_max_sync(0xffffffffu, last);
    if (last <= first) {        // no row of a sequence
        pf_commit();
        pf_arrived();
        return;
    }
    const uint32_t keys = last - first, tiles = (keys + PF_TILE - 1) / PF_TILE;     // counted from `first`
    const uint32_t gt = tid % (NR * 32);
    auto request = [&](float* dst, uint32_t ld, const float* src, uint32_t src_ld, uint32_t vecs, uint32_t tile) {
#pragma unroll 4
        for (uint32_t i = gt; i < PF_TILE * (D / 4); i += NR * 32) {
            const uint32_t r = i / (D / 4), c = i % (D / 4), key = tile * PF_TILE + r;
            const bool take = key < keys && c < vecs;
            pf_copy(dst + r * ld + 4 * c, take ? src + (uint64_t)(first + key) * src_ld + 4 * c : src, take);
        }
    };
    const float *k_from = (const float*)a.k + (uint64_t)g * a.dim, *v_from = (const float*)a.v + (uint64_t)g * a.vdim;
    auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(NR * 32) : "memory"); };
    if (group < tiles) request(s_k, L::LD, k_from, a.k_ld, dvec, group);
    pf_commit();
    pf_arrived();
    __syncthreads();

    uint64_t o[4][D / 16];
    float top[4], sum[4];
    uint32_t from[4], to[4];        // keys of the thread's rows, counted from `first`
    // keys that all rows of the warp see, and that any does
    uint32_t all_from = 0, all_to = 0xffffffffu, any_from = 0xffffffffu, any_to = 0;
    for (uint32_t r = 0; r < 16; ++r) {
        const uint2 x = s_range[wrow * 16 + r];
        if (x.y <= x.x) continue;
        all_from = max(all_from, x.x - first);
        all_to = min(all_to, x.y - first);
        any_from = min(any_from, x.x - first);
        any_to = max(any_to, x.y - first);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint2 x = s_range[wrow * 16 + ty + 4 * i];
        from[i] = x.y > x.x ? x.x - first : 0u;
        to[i] = x.y > x.x ? x.y - first : 0u;
        top[i] = -INFINITY;
        sum[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[i][c] = 0;
    }
    const float* q = s_q + (wrow * 16 + ty) * L::LD;
    const float* k = s_k + tx * L::LD;
    const uint32_t runs = (a.dim + 31) / 32;
#pragma unroll 1
    for (uint32_t t = group; t < tiles; t += NG) {
        pf_arrived();
        meet();         // this tile's K is here, and everybody in the group has left the last tile's V
        request(s_v, D, v_from, a.v_ld, vvec, t);
        pf_commit();
        const uint32_t at = t * PF_TILE;
        const bool sees = at < any_to && at + PF_TILE > any_from;       // some row of the warp
        if (sees) {
            float s[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < 8; ++x) s[i][x] = 0.0f;
#pragma unroll 1
            for (uint32_t run = 0; run < runs; ++run) {
                uint64_t acc[4][8];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < 8; ++x) acc[i][x] = 0;
#pragma unroll 2
                for (uint32_t c = run * 32; c < run * 32 + 32; c += 4) {
                    ulonglong2 qv[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const ulonglong2*>(q + 4 * i * L::LD + c);
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const ulonglong2 kv = *reinterpret_cast<const ulonglong2*>(k + 8 * x * L::LD + c);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[i][x] = fma_pair(qv[i].y, kv.y, fma_pair(qv[i].x, kv.x, acc[i][x]));
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const float2 e = halves(acc[i][x]);
                        s[i][x] += e.x + e.y;
                    }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float most = -INFINITY;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const uint32_t key = at + tx + 8 * x;
                    s[i][x] = key >= from[i] && key < to[i] ? s[i][x] * a.scale : -INFINITY;
                    most = fmaxf(most, s[i][x]);
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                most = fmaxf(most, top[i]);
                const float f = top[i] == -INFINITY ? 0.0f : expf(top[i] - most);
                top[i] = most;
                float part = 0.0f;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const float w = s[i][x] == -INFINITY ? 0.0f : expf(s[i][x] - most);
                    s_p[(ty + 4 * i) * PF_LD + tx + 8 * x] = w;
                    part += w;
                }
                sum[i] = sum[i] * f + part;
                const uint64_t f2 = twice(f);
#pragma unroll
                for (int c = 0; c < D / 16; ++c) o[i][c] = mul_pair(o[i][c], f2);
            }
        }
        __syncwarp();
        pf_arrived();
        meet();         // V is here, and everybody in the group has left K
        if (t + NG < tiles) request(s_k, L::LD, k_from, a.k_ld, dvec, t + NG);
        pf_commit();
        if (!sees) continue;
        if (at >= all_from && at + PF_TILE <= all_to) {
#pragma unroll 1
            for (uint32_t j = 0; j < PF_TILE; j += 4) {
                float4 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float4*>(s_p + (ty + 4 * i) * PF_LD + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ulonglong2 v[D / 32];
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) v[c] = *reinterpret_cast<const ulonglong2*>(s_v + (j + e) * D + 32 * c + 4 * tx);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint64_t w2 = twice(e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w);
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            o[i][2 * c] = fma_pair(w2, v[c].x, o[i][2 * c]);
                            o[i][2 * c + 1] = fma_pair(w2, v[c].y, o[i][2 * c + 1]);
                        }
                    }
                }
            }
        } else {
            const uint32_t j0 = any_from > at ? (any_from - at) & ~3u : 0u, j1 = min((uint32_t)PF_TILE, any_to - at);
#pragma unroll 1
            for (uint32_t j = j0; j < j1; j += 4) {
                float4 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float4*>(s_p + (ty + 4 * i) * PF_LD + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ulonglong2 v[D / 32];
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) v[c] = *reinterpret_cast<const ulonglong2*>(s_v + (j + e) * D + 32 * c + 4 * tx);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (at + j + e >= from[i] && at + j + e < to[i]) {
                            const uint64_t w2 = twice(e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w);
#pragma unroll
                            for (int c = 0; c < D / 32; ++c) {
                                o[i][2 * c] = fma_pair(w2, v[c].x, o[i][2 * c]);
                                o[i][2 * c + 1] = fma_pair(w2, v[c].y, o[i][2 * c + 1]);
                            }
                        }
                }
            }
        }
        __syncwarp();   // the warp's weights have been read
    }
    // ---- add the groups up: each leaves its rows, maxima and sums in its own tiles' memory ----
    pf_arrived();
    __syncthreads();
    float *s_o = smem + L::Q, *s_ml = s_o + NG * L::ROWS * D;      // [NG][ROWS][D], [NG][ROWS][2]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 4);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 8);
        const uint32_t r = group * L::ROWS + wrow * 16 + ty + 4 * i;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) *reinterpret_cast<ulonglong2*>(s_o + r * D + 32 * c + 4 * tx) = make_ulonglong2(o[i][2 * c], o[i][2 * c + 1]);
        if (tx == 0) {
            s_ml[2 * r] = top[i];
            s_ml[2 * r + 1] = sum[i];
        }
    }
    __syncthreads();
    float* out = (float*)a.out + (uint64_t)row0 * a.ld + (uint64_t)head * a.vdim;
    for (uint32_t i = tid; i < L::ROWS * vvec; i += L::WARPS * 32) {
        const uint32_t r = i / vvec, c = 4 * (i % vvec);
        if (s_range[r].y <= s_range[r].x) continue;
        float most = -INFINITY, total = 0.0f;
#pragma unroll
        for (int n = 0; n < NG; ++n) most = fmaxf(most, s_ml[2 * (n * L::ROWS + r)]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const float l = s_ml[2 * (n * L::ROWS + r) + 1];
            if (l == 0.0f) continue;       // NaN is not 0
            const float f = expf(s_ml[2 * (n * L::ROWS + r)] - most);
            const float4 v = *reinterpret_cast<const float4*>(s_o + (n * L::ROWS + r) * D + c);
            total = fmaf(f, l, total);
            acc = make_float4(fmaf(f, v.x, acc.x), fmaf(f, v.y, acc.y), fmaf(f, v.z, acc.z), fmaf(f, v.w, acc.w));
        }
        const bool nothing = total == 0.0f;       // every score -inf
        *reinterpret_cast<float4*>(out + (uint64_t)r * a.ld + c) =
            nothing ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc.x / total, acc.y / total, acc.z / total, acc.w / total);
    }
}

template <int D, int NR, int NG>
int32_t launch_packed_f32(holo_b200_ctx* ctx, const HoloPackedArgs& a) {
    using L = PackedF32Layout<D, NR, NG>;
    constexpr int SMEM = L::FLOATS * 4;
    static thread_local int configured_device = -1;
    if (configured_device != ctx->device) {
        HOLO_CUDA(cudaFuncSetAttribute(packed_f32_kernel<D, NR, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        configured_device = ctx->device;
    }
    HOLO_CUDA(holo_launch_kernel(ctx, packed_f32_kernel<D, NR, NG>, dim3(a.heads, (a.rows + L::ROWS - 1) / L::ROWS), dim3(L::WARPS * 32), SMEM, 1, a));
    ctx->launches++;
    return HOLO_OK;
}

}  // namespace

int32_t holo_try_packed_f32(holo_b200_ctx* ctx, const HoloPackedArgs& a, bool* taken) {
    *taken = false;
    if (a.dtype != HOLO_DTYPE_F32 || a.dim % 4 != 0 || a.vdim % 4 != 0 || a.dim > 128 || a.vdim > 128) return HOLO_OK;
    if ((((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15u) != 0 || ((a.q_ld | a.k_ld | a.v_ld | a.ld) & 3u) != 0) return HOLO_OK;
    const uint32_t d = a.dim > a.vdim ? a.dim : a.vdim;
    const uint64_t blocks = ((uint64_t)a.rows + 63) / 64;
    if (2 * blocks > 65535) return HOLO_OK;
    *taken = true;
    // where 64-row blocks leave SMs without one: 32-row blocks whose groups share the keys
    const bool small = blocks * a.heads < (uint64_t)ctx->sm_count;
    if (d <= 64) return small ? launch_packed_f32<64, 2, 4>(ctx, a) : launch_packed_f32<64, 4, 1>(ctx, a);
    if (d <= 96) return small ? launch_packed_f32<96, 2, 2>(ctx, a) : launch_packed_f32<96, 4, 2>(ctx, a);
    return small ? launch_packed_f32<128, 2, 2>(ctx, a) : launch_packed_f32<128, 4, 2>(ctx, a);
}
