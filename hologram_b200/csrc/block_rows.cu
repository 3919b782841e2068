// Attention of many rows of each sequence (portions of prompts) over the int8 block cache, for dims in steps of 16 up to 128: f32 rows, and blocks
// whose rows are no multiple of 16 (the others: block_tile.cu).
//
// A CTA takes 128 query rows of a kv head (a row is a new position and a head of the group) and walks the keys in slabs of 64; two warps share
// 16 rows, each with half of a slab's keys and a maximum, sums and a context of its own, joined at the plane's end: sixteen warps hide more
// of each other's latency than eight with whole slabs (373 us against 472 for bf16 portions of 128, 256, 77 and 128 rows, 32 heads over 8 of
// dim 128, behind up to 8000 positions; block_tile.cu, which has taken 16-bit rows over since, takes 109).
// The codes of a slab are copied to a ring (cp.async), turned into f16 once for all warps (exact: integers of 8 bits), while the slab
// before is worked on, and are the operands of mma.sync m16n8k16 with f32 sums. Query rows are scaled by a power of two to a largest value in
// [2^14, 2^15), so that bf16 and f16 queries are exact in f16 (values 2^29 smaller than the largest aside); f32 queries go as two f16 terms,
// which hold 22 bits. Scales of blocks are applied to the scores, and to the weights, w = 2^(s - max) * scale_v relative to a power of two that
// follows the largest scale_v seen, lifted by 2^14; weights are rounded to f16 (by up to 2^-11 of a weight), for an f32 result to two terms.
// Bound: the rate of mma.sync (8 cycles a product and quarter of an SM), a half of what tcgen05 has; the codes would have to be turned into f16
// for it as well. The slabs of all planes form one list that the CTAs share out evenly, as for few rows (block_list.cuh).
#include "block_list.cuh"

namespace {

constexpr int BR_ROWS = 128, BR_SLAB = 64, BR_WARPS = 16, BR_STAGES = 3;
constexpr uint32_t BR_THREADS = BR_WARPS * 32;

struct BlockRowsParams {
    HoloBlockAttnArgs a;
    float* partials;          // [CTAs][2][128 rows][vdim + 2]
    uint32_t* arrivals;       // a counter per CTA, zero between launches
    uint32_t group, q_pitch, k_pitch, v_pitch, q_bytes, tile_bytes, stage_bytes;
    int32_t br_shift;         // -1: block_rows is no power of two
};

constexpr uint32_t PICK01 = 0x4140, PICK23 = 0x4342;

template <int MAXD, bool TWO>
__global__ void __launch_bounds__(BR_THREADS, 1)
block_rows_kernel(const __grid_constant__ BlockRowsParams p) {
    constexpr int KSTEPS = MAXD / 16, CHUNKS = MAXD / 16, UNITS = (BR_SLAB * MAXD / 16 + BR_THREADS - 1) / BR_THREADS, KEYS = BR_SLAB / 2;      // 16-byte units of codes a thread
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_row[BR_ROWS], s_scales[4][2][BR_SLAB];
    __shared__ uint32_t s_last;
    const HoloBlockAttnArgs& a = p.a;
    const HoloBlockCache& c = a.c;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, in_quad = lane & 3;
    const uint32_t rows16 = warp & 7u, half = warp >> 3, group = p.group, dim = c.dim, vdim = c.vdim, br = c.block_rows, k_chunks = dim / 16, v_chunks = vdim / 16;
    const uint32_t q_at = smem_u32(smem), tiles_at = q_at + p.q_bytes, ring_at = tiles_at + 2 * p.tile_bytes;
    uint8_t *tiles_mem = smem + p.q_bytes, *ring_mem = tiles_mem + 2 * p.tile_bytes;
    holo_pdl_trigger();
    holo_pdl_wait();
    if (blockIdx.x == 0) check_sequences(c.starts, c.lengths, c.sequences, c.rows, (int64_t)c.table_ld * br, c.status);
    Share mine;
    if (!find_share<BR_ROWS, BR_SLAB, 2, 6>(c, group, &mine)) return;
    auto block_of = [&](uint32_t pos) { return p.br_shift >= 0 ? pos >> p.br_shift : pos / br; };
    // this thread's units of a slab: (key, unit of its row); keys of -1 do not exist
    int key_k[UNITS], key_v[UNITS];
    uint32_t x_k[UNITS], x_v[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const uint32_t i = tid + u * BR_THREADS;
        key_k[u] = i < BR_SLAB * k_chunks ? (int)(i / k_chunks) : -1;
        x_k[u] = i % k_chunks;
        key_v[u] = i < BR_SLAB * v_chunks ? (int)(i / v_chunks) : -1;
        x_v[u] = i % v_chunks;
    }

    Plane at = mine.first;
#pragma unroll 1
    for (;;) {
        uint32_t s0, s1;
        mine.ends_of(at, &s0, &s1);
        const uint32_t rows = min((uint32_t)BR_ROWS, at.n * group - at.tile * BR_ROWS), sees = keys_of_plane<BR_ROWS>(at, at.tile, group);
        // block numbers of a slab's keys, a slab ahead of the copies
        int id_k[UNITS], id_v[UNITS], id_s = -1;
        auto find = [&](uint32_t slab, int key) {
            const uint32_t pos = slab * BR_SLAB + key;
            if (key < 0 || slab >= s1 || pos >= sees) return -1;
            const int id = c.table[(uint64_t)at.seq * c.table_ld + block_of(pos)];
            if ((uint32_t)id < c.blocks) return id;
            atomicOr(c.status, HOLO_STATUS_TABLE);
            return -1;
        };
        auto find_all = [&](uint32_t slab) {
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                id_k[u] = find(slab, key_k[u]);
                id_v[u] = find(slab, key_v[u]);
            }
            id_s = find(slab, tid < BR_SLAB ? (int)tid : -1);
        };
        auto request = [&](uint32_t slab) {
            if (slab < s1) {
                const uint32_t to = ring_at + (slab - s0) % BR_STAGES * p.stage_bytes, to_v = to + BR_SLAB * dim;
                auto row_of = [&](int id, int key) {
                    const uint32_t pos = slab * BR_SLAB + key;
                    return ((uint64_t)(uint32_t)id * c.kv_heads + at.head) * br + (pos - block_of(pos) * br);
                };
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    if (key_k[u] >= 0) cp_async16(to + 16 * (tid + u * BR_THREADS), id_k[u] < 0 ? c.k_codes : c.k_codes + row_of(id_k[u], key_k[u]) * dim + 16 * x_k[u], id_k[u] >= 0);
                    if (key_v[u] >= 0) cp_async16(to_v + 16 * (tid + u * BR_THREADS), id_v[u] < 0 ? c.v_codes : c.v_codes + row_of(id_v[u], key_v[u]) * vdim + 16 * x_v[u], id_v[u] >= 0);
                }
                if (tid < BR_SLAB) {
                    const uint64_t plane = (uint64_t)(uint32_t)max(id_s, 0) * c.kv_heads + at.head;
                    float(&to_s)[2][BR_SLAB] = s_scales[(slab - s0) & 3u];
                    cp_async4(smem_u32(&to_s[0][tid]), c.k_scales + plane, id_s >= 0);
                    cp_async4(smem_u32(&to_s[1][tid]), c.v_scales + plane, id_s >= 0);
                }
                find_all(slab + 1);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        auto convert = [&](uint32_t slab) {
            if (slab >= s1) return;
            const uint8_t* codes = ring_mem + (slab - s0) % BR_STAGES * p.stage_bytes;
            uint8_t* to = tiles_mem + ((slab - s0) & 1u) * p.tile_bytes;
            auto unit = [&](const uint8_t* from, uint8_t* dst) {
                const uint4 v = *reinterpret_cast<const uint4*>(from);
                const uint32_t w[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
                uint32_t h[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h[2 * e] = codes_to_half<PICK01>(w[e]);
                    h[2 * e + 1] = codes_to_half<PICK23>(w[e]);
                }
                reinterpret_cast<uint4*>(dst)[0] = make_uint4(h[0], h[1], h[2], h[3]);
                reinterpret_cast<uint4*>(dst)[1] = make_uint4(h[4], h[5], h[6], h[7]);
            };
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                if (key_k[u] >= 0) unit(codes + 16 * (tid + u * BR_THREADS), to + key_k[u] * p.k_pitch + 32 * x_k[u]);
                if (key_v[u] >= 0) unit(codes + BR_SLAB * dim + 16 * (tid + u * BR_THREADS), to + BR_SLAB * p.k_pitch + key_v[u] * p.v_pitch + 32 * x_v[u]);
            }
        };
        find_all(s0);
#pragma unroll 1
        for (uint32_t s = 0; s < BR_STAGES; ++s) request(s0 + s);
        // ---- the rows of the plane, a warp its own ----
#pragma unroll 4
        for (uint32_t r = warp * 8; r < warp * 8 + 8; ++r) {
            const uint32_t flat = at.tile * BR_ROWS + r, i = flat / group, head = at.head * group + flat % group;
            float x[MAXD / 32], most = 0.0f;
            bool finite = true;
#pragma unroll
            for (int e = 0; e < MAXD / 32; ++e) {
                const uint32_t d = lane + 32 * e;
                x[e] = r < rows && d < dim ? seq_load(a.q, (uint64_t)(at.first_row + i) * a.q_ld + (uint64_t)head * dim + d, a.dtype) : 0.0f;
                most = fmaxf(most, fabsf(x[e]));
                finite = finite && fabsf(x[e]) < INFINITY;
            }
            most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
            finite = __all_sync(0xffffffffu, finite);
            // 2^e <= most < 2^(e + 1); two factors, since 2^(14 - e) alone may overflow
            const uint32_t bits = __float_as_uint(most);
            const int up = finite && bits ? 14 - (bits >> 23 ? (int)(bits >> 23) - 127 : -118 - __clz((int)bits)) : 0;
            const float f0 = power_of_two(up / 2), f1 = power_of_two(up - up / 2);
#pragma unroll
            for (int e = 0; e < MAXD / 32; ++e) {
                const uint32_t d = lane + 32 * e;
                if (d >= dim) continue;
                const float y = finite ? x[e] * f0 * f1 : 0.0f;
                const __half h = __float2half_rn(y);
                *reinterpret_cast<__half*>(smem + r * p.q_pitch + 2 * d) = h;
                if (TWO) *reinterpret_cast<__half*>(smem + (BR_ROWS + r) * p.q_pitch + 2 * d) = __float2half_rn(y - __half2float(h));
            }
            if (lane == 0) s_row[r] = finite ? a.scale * LOG2E * power_of_two(-(up / 2)) * power_of_two(-(up - up / 2)) : NAN;
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(BR_STAGES - 1) : "memory");
        __syncthreads();
        const bool works = rows16 * 16 < rows;
        const float row_scale[2] = {s_row[rows16 * 16 + quad], s_row[rows16 * 16 + quad + 8]};
        uint32_t limit[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t i = (at.tile * BR_ROWS + min(rows16 * 16 + quad + 8 * x, rows - 1)) / group;
            limit[x] = (uint32_t)max(0, at.length - (int32_t)(at.n - i - 1));
        }
        // keys that all rows of the warp see, and that any does
        const uint32_t common = __reduce_min_sync(0xffffffffu, limit[0]), most_keys = __reduce_max_sync(0xffffffffu, limit[1]);
        float o[CHUNKS][2][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
        int lift = -1000;           // the exponent that value scales are relative to
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[i][0][x] = o[i][1][x] = 0.0f;
        convert(s0);
#pragma unroll 1
        for (uint32_t slab = s0; slab < s1; ++slab) {
            asm volatile("cp.async.wait_group %0;" ::"n"(BR_STAGES - 2) : "memory");
            __syncthreads();        // the next slab's codes are here, this one's f16 are, and everybody has left the one before
            convert(slab + 1);
            request(slab + BR_STAGES);
            if (!works || slab * BR_SLAB + half * KEYS >= most_keys) continue;
            const uint32_t k_at = tiles_at + ((slab - s0) & 1u) * p.tile_bytes + half * KEYS * p.k_pitch;
            const uint32_t v_at = tiles_at + ((slab - s0) & 1u) * p.tile_bytes + BR_SLAB * p.k_pitch + half * KEYS * p.v_pitch;
            const float *ks = s_scales[(slab - s0) & 3u][0] + half * KEYS, *vs = s_scales[(slab - s0) & 3u][1] + half * KEYS;
            float s[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[j][x] = 0.0f;
            // the operands of a step are requested while the products of the step before run
            const uint32_t q_from = q_at + (rows16 * 16 + (lane & 15u)) * p.q_pitch + 16 * (lane >> 4), k_from = k_at + (8 * (lane >> 4) + (lane & 7u)) * p.k_pitch + 16 * ((lane >> 3) & 1u);
            uint32_t q[2][4], q2[2][4], w[2][2][4];
            auto fetch = [&](int k) {
                ldsm4(q_from + 32 * k, q[k & 1]);
                if (TWO) ldsm4(q_from + BR_ROWS * p.q_pitch + 32 * k, q2[k & 1]);
                ldsm4(k_from + 32 * k, w[k & 1][0]);
                ldsm4(k_from + 16 * p.k_pitch + 32 * k, w[k & 1][1]);
            };
            fetch(0);
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
                if (16 * k >= dim) break;
                if (k + 1 < KSTEPS && 16 * (k + 1) < dim) fetch(k + 1);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    mma_f16(s[2 * j], q[k & 1], w[k & 1][j][0], w[k & 1][j][1]);
                    mma_f16(s[2 * j + 1], q[k & 1], w[k & 1][j][2], w[k & 1][j][3]);
                }
                if (TWO)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma_f16(s[2 * j], q2[k & 1], w[k & 1][j][0], w[k & 1][j][1]);
                        mma_f16(s[2 * j + 1], q2[k & 1], w[k & 1][j][2], w[k & 1][j][3]);
                    }
            }
            const uint32_t key0 = slab * BR_SLAB + half * KEYS + 2 * in_quad;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = *reinterpret_cast<const float2*>(ks + 8 * j + 2 * in_quad);
                s[j][0] *= row_scale[0] * f.x; s[j][1] *= row_scale[0] * f.y;
                s[j][2] *= row_scale[1] * f.x; s[j][3] *= row_scale[1] * f.y;
            }
            if (slab * BR_SLAB + half * KEYS + KEYS > common) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (key0 + 8 * j + (x & 1) >= limit[x >> 1]) s[j][x] = -INFINITY;
            }
            float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                most[0] = fmaxf(most[0], fmaxf(s[j][0], s[j][1]));
                most[1] = fmaxf(most[1], fmaxf(s[j][2], s[j][3]));
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                most[x] = fmaxf(most[x], __shfl_xor_sync(0xffffffffu, most[x], 1));
                most[x] = fmaxf(most[x], __shfl_xor_sync(0xffffffffu, most[x], 2));
            }
            const float largest = vs[lane];
            int e = largest > 0.0f && largest < INFINITY ? max((int)(__float_as_uint(largest) >> 23) - 126, -110) : -110;
            e = __reduce_max_sync(0xffffffffu, e);
            if (__any_sync(0xffffffffu, most[0] > top[0] || most[1] > top[1]) || e > lift) {
                const int higher = max(e, lift);
                const float turn = lift == -1000 || lift - higher < -126 ? 0.0f : power_of_two(lift - higher);
                lift = higher;
                float f[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float t = fmaxf(top[x], most[x]);
                    f[x] = top[x] == t ? 1.0f : ex2(top[x] - t);
                    top[x] = t;
                    sum[x] *= f[x];
                    f[x] *= turn;
                }
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        o[i][0][x] *= f[x >> 1];
                        o[i][1][x] *= f[x >> 1];
                    }
            }
            const float t0 = top[0] == -INFINITY ? 0.0f : top[0], t1 = top[1] == -INFINITY ? 0.0f : top[1], raise = power_of_two(min(14 - lift, 127));
            uint32_t u[2][4], u2[2][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = *reinterpret_cast<const float2*>(vs + 8 * j + 2 * in_quad);
                const float e0 = ex2(s[j][0] - t0), e1 = ex2(s[j][1] - t0), e2 = ex2(s[j][2] - t1), e3 = ex2(s[j][3] - t1);
                sum[0] += e0 + e1;
                sum[1] += e2 + e3;
                const float f0 = f.x * raise, f1 = f.y * raise, y0 = e0 * f0, y1 = e1 * f1, y2 = e2 * f0, y3 = e3 * f1;
                u[j >> 1][2 * (j & 1)] = half_pair(y0, y1);
                u[j >> 1][2 * (j & 1) + 1] = half_pair(y2, y3);
                if (TWO) {
                    const float2 h0 = half_values(u[j >> 1][2 * (j & 1)]), h1 = half_values(u[j >> 1][2 * (j & 1) + 1]);
                    u2[j >> 1][2 * (j & 1)] = half_pair(y0 - h0.x, y1 - h0.y);
                    u2[j >> 1][2 * (j & 1) + 1] = half_pair(y2 - h1.x, y3 - h1.y);
                }
            }
            const uint32_t v_from = v_at + (lane & 15u) * p.v_pitch + 16 * (lane >> 4);
            uint32_t v[2][2][4];
            auto fetch_v = [&](int i) {
                ldsm4t(v_from + 32 * i, v[i & 1][0]);
                ldsm4t(v_from + 16 * p.v_pitch + 32 * i, v[i & 1][1]);
            };
            fetch_v(0);
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                if (16 * i >= vdim) break;
                if (i + 1 < CHUNKS && 16 * (i + 1) < vdim) fetch_v(i + 1);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    mma_f16(o[i][0], u[t], v[i & 1][t][0], v[i & 1][t][1]);
                    mma_f16(o[i][1], u[t], v[i & 1][t][2], v[i & 1][t][3]);
                    if (TWO) {
                        mma_f16(o[i][0], u2[t], v[i & 1][t][0], v[i & 1][t][1]);
                        mma_f16(o[i][1], u2[t], v[i & 1][t][2], v[i & 1][t][3]);
                    }
                }
            }
        }
        // ---- the second half's results join the first's, through the memory of queries and tiles ----
        const float back = lift == -1000 ? 0.0f : power_of_two(lift - 14);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
            sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
        }
        float* s_o = reinterpret_cast<float*>(smem);       // [128][vdim + 2]
        __syncthreads();        // queries and tiles have been read
        if (half && works) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float* to = s_o + (rows16 * 16 + quad + 8 * x) * (vdim + 2);
#pragma unroll
                for (int i = 0; i < 2 * CHUNKS; ++i) {
                    if (8 * i >= vdim) break;
                    *reinterpret_cast<float2*>(to + 8 * i + 2 * in_quad) = make_float2(o[i >> 1][i & 1][2 * x] * back, o[i >> 1][i & 1][2 * x + 1] * back);
                }
                if (in_quad == 0) *reinterpret_cast<float2*>(to + vdim) = make_float2(top[x], sum[x]);
            }
        }
        __syncthreads();
        if (!half && works) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float* add = s_o + (rows16 * 16 + quad + 8 * x) * (vdim + 2);
                const float2 ml = *reinterpret_cast<const float2*>(add + vdim);
                const float t = fmaxf(top[x], ml.x);
                // a half that saw nothing has no sum; NaN is not 0
                const float f = sum[x] == 0.0f ? 0.0f : ex2(top[x] - t), g = ml.y == 0.0f ? 0.0f : ex2(ml.x - t);
                sum[x] = fmaf(f, sum[x], g * ml.y);
                top[x] = t;
#pragma unroll
                for (int i = 0; i < 2 * CHUNKS; ++i) {
                    if (8 * i >= vdim) break;
                    const float2 y = *reinterpret_cast<const float2*>(add + 8 * i + 2 * in_quad);
                    float &lo = o[i >> 1][i & 1][2 * x], &hi = o[i >> 1][i & 1][2 * x + 1];
                    lo = fmaf(f * back, lo, g * y.x);
                    hi = fmaf(f * back, hi, g * y.y);
                }
            }
        }
        // ---- every warp has its rows' results ----
        const bool begins = at.at >= mine.lo, whole = begins && at.at + at.slabs <= mine.hi;
        float* partial = p.partials + ((uint64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * BR_ROWS * (vdim + 2);
        auto out_of = [&](uint32_t r) {
            const uint32_t flat = at.tile * BR_ROWS + r;
            return (uint64_t)(at.first_row + flat / group) * a.ld + (uint64_t)(at.head * group + flat % group) * vdim;
        };
        const bool pairs_ok = ((uintptr_t)a.out % 8u) == 0 && a.ld % 2 == 0;      // two values a store
        auto store2 = [&](uint64_t i, float lo, float hi) {
            if (!pairs_ok) {
                seq_store(a.out, i, lo, a.dtype);
                seq_store(a.out, i + 1, hi, a.dtype);
            } else if (a.dtype == HOLO_DTYPE_F32) {
                *reinterpret_cast<float2*>((float*)a.out + i) = make_float2(lo, hi);
            } else {
                *reinterpret_cast<uint32_t*>((uint16_t*)a.out + i) = a.dtype == HOLO_DTYPE_F16 ? half_pair(lo, hi) : pack_bf16(lo, hi);
            }
        };
        if (!half && works) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t r = rows16 * 16 + quad + 8 * x;
                if (r >= rows) continue;
                const float by = whole ? sum[x] == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum[x]) : 1.0f;
                const uint64_t out = out_of(r);
#pragma unroll
                for (int i = 0; i < 2 * CHUNKS; ++i) {
                    if (8 * i >= vdim) break;
                    const float lo = o[i >> 1][i & 1][2 * x] * by, hi = o[i >> 1][i & 1][2 * x + 1] * by;
                    const uint32_t col = 8 * i + 2 * in_quad;
                    if (whole) store2(out + col, lo, hi);
                    else __stcg(reinterpret_cast<float2*>(partial + r * (vdim + 2) + col), make_float2(lo, hi));
                }
                if (!whole && in_quad == 0) __stcg(reinterpret_cast<float2*>(partial + r * (vdim + 2) + vdim), make_float2(top[x], sum[x]));
            }
        }
        if (!whole) {
            // the plane's CTAs, and its counter: that of the CTA it begins in
            const uint32_t from_cta = mine.first_cta(at), count = mine.cta_count(at);
            __syncthreads();
            if (tid == 0) {
                uint32_t n;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(n) : "l"(p.arrivals + from_cta) : "memory");
                s_last = n + 1 == count;
                if (s_last) p.arrivals[from_cta] = 0;
            }
            __syncthreads();
            if (s_last) {
                const uint32_t step = 2 * BR_ROWS * (vdim + 2), own = BR_ROWS * (vdim + 2), pairs = vdim / 2;
                const float* base = p.partials + (uint64_t)from_cta * step;
                auto part = [&](uint32_t w, uint32_t r) { return base + (uint64_t)w * step + (w == 0 ? own : 0u) + r * (vdim + 2); };
                float* s_f = reinterpret_cast<float*>(smem);      // [rows][count]: nothing is on its way any more
                for (uint32_t r = tid; r < rows; r += BR_THREADS) {
                    float m = -INFINITY, l = 0.0f;
                    for (uint32_t w = 0; w < count; ++w) m = fmaxf(m, __ldcg(part(w, r) + vdim));
                    for (uint32_t w = 0; w < count; ++w) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(part(w, r) + vdim));
                        const float f = ml.y == 0.0f ? 0.0f : ex2(ml.x - m);       // NaN is not 0
                        s_f[r * count + w] = f;
                        l = fmaf(f, ml.y, l);
                    }
                    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                    for (uint32_t w = 0; w < count; ++w) s_f[r * count + w] *= inv;
                }
                __syncthreads();
#pragma unroll 4
                for (uint32_t i = tid; i < rows * pairs; i += BR_THREADS) {
                    const uint32_t r = i / pairs, col = 2 * (i % pairs);
                    float2 v = make_float2(0.f, 0.f);
                    for (uint32_t w = 0; w < count; ++w) {
                        const float2 y = __ldcg(reinterpret_cast<const float2*>(part(w, r) + col));
                        const float f = s_f[r * count + w];
                        v = make_float2(fmaf(f, y.x, v.x), fmaf(f, y.y, v.y));
                    }
                    const uint64_t out = out_of(r);
                    store2(out + col, v.x, v.y);
                }
            }
        }
        if (at.at + at.slabs >= mine.hi) break;
        next_plane<BR_ROWS, BR_SLAB>(c, group, &at);
        if (!at.slabs) break;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();        // everybody has left this plane's memory
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int MAXD, bool TWO>
int32_t launch_block_rows(holo_b200_ctx* ctx, BlockRowsParams& p) {
    const uint32_t dim = p.a.c.dim, vdim = p.a.c.vdim;
    // 16-byte units of 8 neighbouring rows on different banks: an odd number of them a row
    p.q_pitch = p.k_pitch = 2 * dim + 16;
    p.v_pitch = 2 * vdim + 16;
    p.q_bytes = (TWO ? 2 : 1) * BR_ROWS * p.q_pitch;
    p.tile_bytes = BR_SLAB * (p.k_pitch + p.v_pitch);
    p.stage_bytes = BR_SLAB * (dim + vdim);
    uint32_t smem = p.q_bytes + 2 * p.tile_bytes + BR_STAGES * p.stage_bytes;
    const uint32_t weights = BR_ROWS * 4 * (uint32_t)ctx->sm_count;       // of a plane's parts
    if (smem < weights) smem = weights;
    if (smem < BR_ROWS * (vdim + 2) * 4) smem = BR_ROWS * (vdim + 2) * 4;       // a half's results
    if (smem > (uint32_t)ctx->smem_optin - 4096) return holo_fail(HOLO_ERR_DISPATCH, "dispatch failed: block_cache_attention needs %u bytes of shared memory", smem);
    static thread_local int configured_device = -1;
    if (configured_device != ctx->device) {
        HOLO_CUDA(cudaFuncSetAttribute(block_rows_kernel<MAXD, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, ctx->smem_optin - 4096));
        configured_device = ctx->device;
    }
    HOLO_CUDA(holo_launch_kernel(ctx, block_rows_kernel<MAXD, TWO>, dim3((uint32_t)ctx->sm_count), dim3(BR_THREADS), smem, 1, p));
    ctx->launches++;
    return HOLO_OK;
}

}  // namespace

// The buffer of partial results, from the first call on
int32_t holo_block_row_partials(holo_b200_ctx* ctx) {
    if (!ctx->block_row_partials) {
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        HOLO_CUDA(cudaStreamIsCapturing(ctx->stream, &capturing));
        if (capturing != cudaStreamCaptureStatusNone)
            return holo_fail(HOLO_ERR_DISPATCH, "dispatch failed: block_cache_attention allocates its buffer on its first call, which cannot be recorded: make one before");
        HOLO_CUDA(cudaMalloc(&ctx->block_row_partials, (uint64_t)ctx->sm_count * 2 * BR_ROWS * (128 + 2) * sizeof(float)));
    }
    return HOLO_OK;
}

int32_t holo_try_block_rows(holo_b200_ctx* ctx, const HoloBlockAttnArgs& a, bool* taken) {
    *taken = false;
    const HoloBlockCache& c = a.c;
    const uint32_t group = a.heads / c.kv_heads;
    if (c.dim % 16 != 0 || c.vdim % 16 != 0 || c.dim > 128 || c.vdim > 128 || (((uintptr_t)c.k_codes | (uintptr_t)c.v_codes) & 15u) != 0) return HOLO_OK;
    // where a sequence has more rows of a head than the few-row kernel takes in three passes over the cache
    if ((uint64_t)c.rows * group <= 24ull * c.sequences) return HOLO_OK;
    // slabs of the whole list of 32 bits
    const uint64_t tiles = ((uint64_t)c.rows * group / BR_ROWS + c.sequences) * c.kv_heads;
    if ((uint64_t)c.rows * a.heads > 0x7fffffffull || tiles > 0x7fffffffull / (((uint64_t)c.table_ld * c.block_rows + BR_SLAB - 1) / BR_SLAB)) return HOLO_OK;
    HOLO_TRY(holo_block_row_partials(ctx));
    *taken = true;
    BlockRowsParams p = {};
    p.a = a;
    p.partials = ctx->block_row_partials;
    p.arrivals = ctx->attn_arrivals;
    p.group = group;
    p.br_shift = -1;
    for (int s = 0; s <= 10; ++s)
        if (c.block_rows == 1u << s) p.br_shift = s;
    const bool small = c.dim <= 64 && c.vdim <= 64;
    if (a.dtype == HOLO_DTYPE_F32) return small ? launch_block_rows<64, true>(ctx, p) : launch_block_rows<128, true>(ctx, p);
    return small ? launch_block_rows<64, false>(ctx, p) : launch_block_rows<128, false>(ctx, p);
}
