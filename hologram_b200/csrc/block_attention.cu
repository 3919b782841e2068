// Attention of few rows of each sequence over the int8 block cache (the BlockCacheAttention call), for dims in steps of 16 up to 256.
//
// The codes are the operands: 16 query rows (a row is a new position and a head of the group) against 32 keys at a time with
// mma.sync m16n8k16 on f16, f32 sums. A code is an integer of 8 bits and so exact in f16; two of them take a byte permute onto 1024's
// exponent and a packed subtraction (1024 + 128 + c - 1152). Every query row is scaled by a power of two to a largest value in
// [2^14, 2^15): bf16 and f16 queries are then exact in f16 (values 2^29 smaller than the largest aside), f32 queries go as two
// f16 terms, which hold 22 bits. The scales of blocks are applied to the scores, and to the weights: w = 2^(s - max) * scale_v, taken
// relative to a power of two that follows the largest scale_v seen, and lifted by 2^14 so that weights 2^28 smaller are still normal f16. A bf16
// result keeps weights of 11 bits (an error of 2^-12, a sixteenth of the result's own rounding); f16 and f32 results take two terms.
//
// Bound for single tokens: HBM, a byte an element. Loaded latency is 2 to 3 us, so 100 KB and more have to be on their way to every SM:
// each of a CTA's four warps has a ring of its own, slabs of 32 keys and their values copied 16 bytes at a time (cp.async),
// and takes every fourth slab, with a maximum, sums and a context of its own; no barrier stands between a warp and its next slab.
// All slabs of the call (sequence by sequence, head by head, 16 rows at a time) form one list that the CTAs share out evenly, so that
// neither short sequences nor few heads leave SMs without work. Where a share begins or ends inside a plane its partial result goes
// to a buffer of the context, and the last of the plane's CTAs to arrive adds them up in the order of the list: nobody waits,
// and no order of arrival shows in the result.
#include "attention_tile.cuh"
#include "sequences.cuh"

namespace {

constexpr int BA_WARPS = 4, BA_SLAB = 32, BA_ROWS = 16;
constexpr uint32_t BA_THREADS = BA_WARPS * 32;

struct BlockAttnParams {
    HoloBlockAttnArgs a;
    float* partials;          // [CTAs][2][16 rows][vdim + 2]
    uint32_t* arrivals;       // a counter per CTA, zero between launches
    uint32_t group, k_pitch, v_pitch, slab_bytes, q_pitch, head_bytes;
    bool aligned_out;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 half_values(uint32_t v) {
    float2 r;
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.f32.f16 %0, l;\ncvt.f32.f16 %1, h;\n}" : "=f"(r.x), "=f"(r.y) : "r"(v));
    return r;
}
// Bytes 0 and 1 (2 and 3; 0 and 2; 1 and 3) of four codes plus 128 as a pair of f16 codes
template <uint32_t PICK>
__device__ __forceinline__ uint32_t codes_to_half(uint32_t biased) {
    const uint32_t raised = __byte_perm(biased, 0x64646464u, PICK);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&raised), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
constexpr uint32_t PICK01 = 0x4140, PICK23 = 0x4342, PICK02 = 0x4240, PICK13 = 0x4341;

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4u : 0u) : "memory");
}

// The list of planes: sequence by sequence, kv head by kv head, 16 rows by 16 rows; `at` counts the slabs of all planes before.
struct Plane {
    uint32_t seq, head, tile, tiles, first_row, n, slabs;
    int64_t length, at;
};
__device__ __forceinline__ uint32_t slabs_of(int64_t length, uint32_t n, uint32_t tile, uint32_t group) {
    const uint32_t rows = min(n, (tile * BA_ROWS + BA_ROWS - 1) / group + 1);      // rows up to the tile's last one
    const int64_t sees = length - n + rows;
    return sees <= 0 ? 0u : (uint32_t)((sees + BA_SLAB - 1) / BA_SLAB);
}
__device__ __forceinline__ void read_sequence(const HoloBlockCache& c, uint32_t group, uint32_t s, Plane* p) {
    int64_t b = s, e = (int64_t)s + 1;
    if (c.starts) {
        b = c.starts[s];
        e = c.starts[s + 1];
        if (b < 0 || e < b || e > c.rows) b = e = 0;
    }
    p->seq = s;
    p->first_row = (uint32_t)b;
    p->n = (uint32_t)(e - b);
    p->length = min((int64_t)c.lengths[s], (int64_t)c.table_ld * c.block_rows);
    p->tiles = (uint32_t)(((uint64_t)p->n * group + BA_ROWS - 1) / BA_ROWS);
    p->head = p->tile = 0;
}
__device__ __forceinline__ int64_t slabs_of_sequence(const HoloBlockCache& c, uint32_t group, uint32_t s) {
    Plane p;
    read_sequence(c, group, s, &p);
    int64_t sum = 0;
    for (uint32_t t = 0; t < p.tiles; ++t) sum += slabs_of(p.length, p.n, t, group);
    return sum * c.kv_heads;
}
// On to the next plane that has slabs; seq == sequences: there is none.
__device__ __forceinline__ void next_plane(const HoloBlockCache& c, uint32_t group, Plane* p) {
    p->at += p->slabs;
    for (;;) {
        if (++p->tile >= p->tiles) {
            p->tile = 0;
            if (++p->head >= c.kv_heads) {
                if (++p->seq >= c.sequences) {
                    p->slabs = 0;
                    return;
                }
                read_sequence(c, group, p->seq, p);
            }
        }
        p->slabs = p->tiles ? slabs_of(p->length, p->n, p->tile, group) : 0u;
        if (p->slabs) return;
        if (!p->tiles) p->head = c.kv_heads - 1;
    }
}

// MODE 0: bf16, 1: f16 (weights as two terms), 2: f32 (queries and weights as two terms)
template <int MODE, int MAXD, int STAGES>
__global__ void __launch_bounds__(BA_THREADS, MAXD <= 128 ? 2 : 1)
block_attention_kernel(const __grid_constant__ BlockAttnParams p) {
    constexpr bool Q2 = MODE == 2, P2 = MODE != 0;
    constexpr int KSTEPS = MAXD / 16, CHUNKS = MAXD / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t s_sum[BA_WARPS + 1];
    __shared__ Plane s_first;
    __shared__ float s_row[BA_ROWS], s_ml[BA_WARPS][BA_ROWS][3];
    __shared__ uint32_t s_last;
    const HoloBlockAttnArgs& a = p.a;
    const HoloBlockCache& c = a.c;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, in_quad = lane & 3;
    const uint32_t group = p.group, dim = c.dim, vdim = c.vdim, br = c.block_rows;
    holo_pdl_trigger();
    holo_pdl_wait();
    if (blockIdx.x == 0) check_sequences(c.starts, c.lengths, c.sequences, c.rows, (int64_t)c.table_ld * br, c.status);

    // ---- this CTA's share of the list ----
    auto block_sum = [&](int64_t v, int64_t* before) {       // the sum over the block, and over the threads before this one
        int64_t run = v;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= (uint32_t)o) run += u;
        }
        __syncthreads();
        if (lane == 31) s_sum[warp] = run;
        __syncthreads();
        int64_t all = 0, base = 0;
        for (int w = 0; w < BA_WARPS; ++w) {
            if (w < (int)warp) base += s_sum[w];
            all += s_sum[w];
        }
        *before = base + run - v;
        return all;
    };
    int64_t total = 0, before = 0, mine = 0;
    for (uint32_t s0 = 0; s0 < c.sequences; s0 += BA_THREADS) {
        mine = s0 + tid < c.sequences ? slabs_of_sequence(c, group, s0 + tid) : 0;
        total += block_sum(mine, &before);
    }
    // a share is one slab a warp at least: fewer CTAs take part in a short list
    const int64_t ctas = min((int64_t)gridDim.x, (total + BA_WARPS - 1) / BA_WARPS);
    if ((int64_t)blockIdx.x >= ctas) return;
    auto share = [&](int64_t cta) { return cta * total / ctas; };
    const int64_t lo = share(blockIdx.x), hi = share((int64_t)blockIdx.x + 1);
    {
        int64_t run = 0;
        for (uint32_t s0 = 0; s0 < c.sequences; s0 += BA_THREADS) {
            int64_t all;
            if (c.sequences > BA_THREADS) {
                mine = s0 + tid < c.sequences ? slabs_of_sequence(c, group, s0 + tid) : 0;
                all = block_sum(mine, &before);
            } else {
                all = total;
            }
            if (lo < run + all) {
                const int64_t at = run + before;
                if (mine && lo >= at && lo < at + mine) {
                    Plane f;
                    read_sequence(c, group, s0 + tid, &f);
                    f.at = at;
                    f.slabs = slabs_of(f.length, f.n, 0, group);
                    const int64_t each = mine / c.kv_heads;
                    f.head = (uint32_t)((lo - at) / each);
                    f.at += f.head * each;
                    while (lo >= f.at + f.slabs && f.tile + 1 < f.tiles) {
                        f.at += f.slabs;
                        f.slabs = slabs_of(f.length, f.n, ++f.tile, group);
                    }
                    s_first = f;
                }
                break;
            }
            run += all;
        }
        __syncthreads();
    }

    // ---- the ring of this warp ----
    const uint32_t ring = smem_u32(smem) + p.head_bytes + warp * STAGES * p.slab_bytes;
    const uint8_t* ring_at = smem + p.head_bytes + warp * STAGES * p.slab_bytes;
    const uint32_t k_chunks = dim / 16, v_chunks = vdim / 16;
    Plane ahead = s_first;          // where the next slab to request lies
    int64_t ahead_slab = lo + warp; // its number in the list
    int ahead_id = -1;
    auto find_ahead = [&]() {
        while (ahead_slab >= ahead.at + ahead.slabs && ahead.at + ahead.slabs < hi) {
            // every plane's slabs begin with the first warp again
            const int64_t begin = ahead.at + ahead.slabs;
            next_plane(c, group, &ahead);
            ahead_slab = begin + warp;
            if (!ahead.slabs) {
                ahead_slab = hi;
                break;
            }
        }
        ahead_id = -1;
        if (ahead_slab < hi) {
            const uint32_t pos = (uint32_t)(ahead_slab - ahead.at) * BA_SLAB + lane;
            const uint32_t rows = min(ahead.n, (ahead.tile * BA_ROWS + BA_ROWS - 1) / group + 1);
            if ((int64_t)pos < ahead.length - ahead.n + rows) {
                ahead_id = c.table[(uint64_t)ahead.seq * c.table_ld + pos / br];
                if (ahead_id < 0 || (uint32_t)ahead_id >= c.blocks) {
                    atomicOr(c.status, HOLO_STATUS_TABLE);
                    ahead_id = -1;
                }
            }
        }
    };
    auto request = [&](uint32_t stage) {
        if (ahead_slab < hi) {
            const uint32_t to = ring + stage * p.slab_bytes, pos = (uint32_t)(ahead_slab - ahead.at) * BA_SLAB + lane;
            const uint32_t plane = (uint32_t)max(ahead_id, 0) * c.kv_heads + ahead.head;
            const uint32_t row = ahead_id < 0 ? 0xffffffffu : plane * br + pos % br;
            for (uint32_t i = lane; i < BA_SLAB * k_chunks; i += 32) {
                const uint32_t key = i / k_chunks, x = i % k_chunks, r = __shfl_sync(0xffffffffu, row, key);
                const uint32_t y = (dim & 127u) == 0 ? x ^ (key & 7u) : x;
                cp_async16(to + key * p.k_pitch + 16 * y, c.k_codes + (r == 0xffffffffu ? 0 : (uint64_t)r * dim + 16 * x), r != 0xffffffffu);
            }
            const uint32_t to_v = to + BA_SLAB * p.k_pitch;
            for (uint32_t i = lane; i < BA_SLAB * v_chunks; i += 32) {
                const uint32_t key = i / v_chunks, x = i % v_chunks, r = __shfl_sync(0xffffffffu, row, key);
                const uint32_t y = (vdim & 127u) == 0 ? x ^ (key & 7u) : x;
                cp_async16(to_v + key * p.v_pitch + 16 * y, c.v_codes + (r == 0xffffffffu ? 0 : (uint64_t)r * vdim + 16 * x), r != 0xffffffffu);
            }
            const uint32_t to_s = to_v + BA_SLAB * p.v_pitch + 4 * lane;
            cp_async4(to_s, c.k_scales + (ahead_id < 0 ? 0 : plane), ahead_id >= 0);
            cp_async4(to_s + 128, c.v_scales + (ahead_id < 0 ? 0 : plane), ahead_id >= 0);
            ahead_slab += BA_WARPS;
            find_ahead();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    find_ahead();
#pragma unroll
    for (int s = 0; s < STAGES; ++s) request(s);

    uint32_t stage = 0;
    Plane at = s_first;
    while (at.at < hi) {
        // ---- one plane: its rows, then the slabs of it that are this CTA's ----
        const uint32_t rows = min((uint32_t)BA_ROWS, at.n * group - at.tile * BA_ROWS);
        for (uint32_t r = warp; r < BA_ROWS; r += BA_WARPS) {
            const uint32_t flat = at.tile * BA_ROWS + r, i = flat / group, head = at.head * group + flat % group;
            float x[MAXD / 32], most = 0.0f;
            bool finite = true;
#pragma unroll
            for (int e = 0; e < MAXD / 32; ++e) {
                const uint32_t d = lane + 32 * e;
                x[e] = r < rows && d < dim ? seq_load(a.q, (uint64_t)(at.first_row + i) * a.q_ld + (uint64_t)head * dim + d, a.dtype) : 0.0f;
                most = fmaxf(most, fabsf(x[e]));
                finite = finite && fabsf(x[e]) < INFINITY;
            }
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            finite = __all_sync(0xffffffffu, finite);
            // 2^e <= most < 2^(e + 1); two factors, since 2^(14 - e) alone may overflow
            const int e2 = finite && most > 0.0f ? ilogbf(most) : 14, up = 14 - e2;
            const float f0 = exp2f((float)(up / 2)), f1 = exp2f((float)(up - up / 2));
#pragma unroll
            for (int e = 0; e < MAXD / 32; ++e) {
                const uint32_t d = lane + 32 * e, c4 = (d & 15u) >> 2, j = d & 3u;
                if (d >= dim) continue;
                // columns as the codes' words have them: products 2c, 2c + 1, 2c + 8, 2c + 9 take dims 4c .. 4c + 3
                const uint32_t col = (d & ~15u) + (j < 2 ? 2 * c4 + j : 8 + 2 * c4 + j - 2);
                const float y = x[e] * f0 * f1;
                const __half h = __float2half_rn(y);
                *reinterpret_cast<__half*>(smem + r * p.q_pitch + 2 * col) = h;
                if (Q2) *reinterpret_cast<__half*>(smem + (BA_ROWS + r) * p.q_pitch + 2 * col) = __float2half_rn(finite ? y - __half2float(h) : 0.0f);
            }
            if (lane == 0) s_row[r] = a.scale * LOG2E * exp2f((float)(-up / 2)) * exp2f((float)(-(up - up / 2)));
        }
        __syncthreads();
        const float row_scale[2] = {s_row[quad], s_row[quad + 8]};
        uint32_t limit[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t r = quad + 8 * x, i = (at.tile * BA_ROWS + min(r, rows - 1)) / group;
            limit[x] = (uint32_t)max((int64_t)0, at.length - at.n + i + 1);
        }
        const uint32_t common = (uint32_t)max((int64_t)0, at.length - at.n + (at.tile * BA_ROWS) / group + 1);      // keys that all rows see
        float o[CHUNKS][2][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
        int lift = -1000;           // the exponent that value scales are relative to
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[i][0][x] = o[i][1][x] = 0.0f;
        const int64_t from = max(lo, at.at), to = min(hi, at.at + at.slabs);
        for (int64_t slab = from + warp; slab < to; slab += BA_WARPS) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t k_at = ring + stage * p.slab_bytes, v_at = k_at + BA_SLAB * p.k_pitch;
            const float* scales = reinterpret_cast<const float*>(ring_at + stage * p.slab_bytes + BA_SLAB * (p.k_pitch + p.v_pitch));
            float s[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[j][x] = 0.0f;
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
                if (16 * k >= dim) break;
                uint32_t q[4], q2[4], w[4];
                ldsm4(smem_u32(smem) + (lane & 15u) * p.q_pitch + 32 * k + 16 * (lane >> 4), q);
                if (Q2) ldsm4(smem_u32(smem) + (BA_ROWS + (lane & 15u)) * p.q_pitch + 32 * k + 16 * (lane >> 4), q2);
                ldsm4(k_at + lane * p.k_pitch + 16 * ((dim & 127u) == 0 ? (uint32_t)k ^ (lane & 7u) : (uint32_t)k), w);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t u = w[j] ^ 0x80808080u, b0 = codes_to_half<PICK01>(u), b1 = codes_to_half<PICK23>(u);
                    mma_f16(s[j], q, b0, b1);
                    if (Q2) mma_f16(s[j], q2, b0, b1);
                }
            }
            const uint32_t key0 = (uint32_t)(slab - at.at) * BA_SLAB;
            float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 ks = *reinterpret_cast<const float2*>(scales + 8 * j + 2 * in_quad);
                s[j][0] *= row_scale[0] * ks.x; s[j][1] *= row_scale[0] * ks.y;
                s[j][2] *= row_scale[1] * ks.x; s[j][3] *= row_scale[1] * ks.y;
            }
            if (key0 + BA_SLAB > common) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (key0 + 8 * j + 2 * in_quad + (x & 1) >= limit[x >> 1]) s[j][x] = -INFINITY;
            }
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
            float largest = scales[32 + lane];
            // a scale that is not finite spoils what it stands for; the others keep their exponent
            int e = largest > 0.0f && largest < INFINITY ? max(ilogbf(largest) + 1, -110) : -110;
            e = __reduce_max_sync(0xffffffffu, e);
            if (__any_sync(0xffffffffu, most[0] > top[0] || most[1] > top[1]) || e > lift) {
                const int up = max(e, lift);
                const float turn = lift == -1000 ? 0.0f : exp2f((float)max(lift - up, -250));
                lift = up;
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
            const float t0 = top[0] == -INFINITY ? 0.0f : top[0], t1 = top[1] == -INFINITY ? 0.0f : top[1];
            const float raise = exp2f((float)(14 - lift));
            uint32_t w[2][4], w2[2][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 vs = *reinterpret_cast<const float2*>(scales + 32 + 8 * j + 2 * in_quad);
                const float e0 = ex2(s[j][0] - t0), e1 = ex2(s[j][1] - t0), e2 = ex2(s[j][2] - t1), e3 = ex2(s[j][3] - t1);
                sum[0] += e0 + e1;
                sum[1] += e2 + e3;
                const float x0 = vs.x * raise, x1 = vs.y * raise;
                const float y0 = e0 * x0, y1 = e1 * x1, y2 = e2 * x0, y3 = e3 * x1;
                w[j >> 1][2 * (j & 1)] = half_pair(y0, y1);
                w[j >> 1][2 * (j & 1) + 1] = half_pair(y2, y3);
                if (P2) {
                    const float2 h0 = half_values(w[j >> 1][2 * (j & 1)]), h1 = half_values(w[j >> 1][2 * (j & 1) + 1]);
                    w2[j >> 1][2 * (j & 1)] = half_pair(y0 - h0.x, y1 - h0.y);
                    w2[j >> 1][2 * (j & 1) + 1] = half_pair(y2 - h1.x, y3 - h1.y);
                }
            }
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                if (16 * i >= vdim) break;
                uint32_t v[4];
                ldsm4t(v_at + lane * p.v_pitch + 16 * ((vdim & 127u) == 0 ? (uint32_t)i ^ (lane & 7u) : (uint32_t)i), v);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t u0 = v[2 * k] ^ 0x80808080u, u1 = v[2 * k + 1] ^ 0x80808080u;
                    const uint32_t even0 = codes_to_half<PICK02>(u0), even1 = codes_to_half<PICK02>(u1), odd0 = codes_to_half<PICK13>(u0), odd1 = codes_to_half<PICK13>(u1);
                    mma_f16(o[i][0], w[k], even0, even1);
                    mma_f16(o[i][1], w[k], odd0, odd1);
                    if (P2) {
                        mma_f16(o[i][0], w2[k], even0, even1);
                        mma_f16(o[i][1], w2[k], odd0, odd1);
                    }
                }
            }
            __syncwarp();       // the slab has been read
            request(stage);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        // ---- the four warps' results, four rows at a time through the memory of the queries ----
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
            sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
            if (in_quad == 0) {
                s_ml[warp][quad + 8 * x][0] = top[x];
                s_ml[warp][quad + 8 * x][1] = sum[x];
                s_ml[warp][quad + 8 * x][2] = lift == -1000 ? 0.0f : exp2f((float)(lift - 14));
            }
        }
        const bool begins = at.at >= lo, ends = at.at + at.slabs <= hi, whole = begins && ends;
        float* partial = p.partials + ((uint64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * BA_ROWS * (vdim + 2);
        float* s_o = reinterpret_cast<float*>(smem);       // [warp][4][vdim]
        const uint32_t columns = vdim / 4;
        auto store4 = [&](uint32_t r, uint32_t col, float4 v) {
            const uint32_t flat = at.tile * BA_ROWS + r;
            const uint64_t index = (uint64_t)(at.first_row + flat / group) * a.ld + (uint64_t)(at.head * group + flat % group) * vdim + col;
            if (p.aligned_out) {
                if (MODE == 2) *reinterpret_cast<float4*>((float*)a.out + index) = v;
                else if (MODE == 1) *reinterpret_cast<uint2*>((uint16_t*)a.out + index) = make_uint2(half_pair(v.x, v.y), half_pair(v.z, v.w));
                else *reinterpret_cast<uint2*>((uint16_t*)a.out + index) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
            } else {
                seq_store(a.out, index, v.x, a.dtype); seq_store(a.out, index + 1, v.y, a.dtype);
                seq_store(a.out, index + 2, v.z, a.dtype); seq_store(a.out, index + 3, v.w, a.dtype);
            }
        };
#pragma unroll 1
        for (uint32_t r0 = 0; r0 < rows; r0 += 4) {
            __syncthreads();        // the queries, or the four rows before, have been read
            if (quad >> 2 == ((r0 >> 2) & 1u)) {
                float* to4 = s_o + (warp * 4 + (quad & 3u)) * vdim + 4 * in_quad;
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i) {
                    if (16 * i >= vdim) break;
                    const int x = r0 >= 8 ? 2 : 0;
                    // the thread's columns 4c, 4c + 2 are in the even product, 4c + 1, 4c + 3 in the odd one
                    *reinterpret_cast<float4*>(to4 + 16 * i) = x ? make_float4(o[i][0][2], o[i][1][2], o[i][0][3], o[i][1][3]) : make_float4(o[i][0][0], o[i][1][0], o[i][0][1], o[i][1][1]);
                }
            }
            __syncthreads();
            for (uint32_t i = tid; i < 4 * columns; i += BA_THREADS) {
                const uint32_t r = r0 + i / columns, col = 4 * (i % columns);
                if (r >= rows) break;
                float m = -INFINITY, l = 0.0f;
#pragma unroll
                for (int w = 0; w < BA_WARPS; ++w) m = fmaxf(m, s_ml[w][r][0]);
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < BA_WARPS; ++w) {
                    const float lw = s_ml[w][r][1], f = lw == 0.0f ? 0.0f : ex2(s_ml[w][r][0] - m), g = f * s_ml[w][r][2];
                    l = fmaf(f, lw, l);
                    if (lw != 0.0f) {
                        const float4 y = *reinterpret_cast<const float4*>(s_o + (w * 4 + r - r0) * vdim + col);
                        v = make_float4(fmaf(g, y.x, v.x), fmaf(g, y.y, v.y), fmaf(g, y.z, v.z), fmaf(g, y.w, v.w));
                    }
                }
                if (whole) {
                    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                    store4(r, col, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                } else {
                    float* row = partial + r * (vdim + 2);
                    __stcg(reinterpret_cast<float2*>(row + col), make_float2(v.x, v.y));
                    __stcg(reinterpret_cast<float2*>(row + col + 2), make_float2(v.z, v.w));
                    if (col == 0) __stcg(reinterpret_cast<float2*>(row + vdim), make_float2(m, l));
                }
            }
        }
        if (!whole) {
            // the CTAs that share the plane, and its counter: that of the CTA it begins in
            auto owner = [&](int64_t slab) {
                int64_t w = slab * ctas / total;
                while (share(w) > slab) --w;
                while (share(w + 1) <= slab) ++w;
                return w;
            };
            const int64_t first = owner(at.at), last = owner(at.at + at.slabs - 1);
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                const uint32_t n = atomicAdd(p.arrivals + first, 1u) + 1;
                s_last = n == (uint32_t)(last - first + 1);
                if (s_last) p.arrivals[first] = 0;
                __threadfence();
            }
            __syncthreads();
            if (s_last) {
                auto of = [&](int64_t cta, uint32_t r) { return p.partials + ((uint64_t)cta * 2 + (cta == first ? 1 : 0)) * BA_ROWS * (vdim + 2) + r * (vdim + 2); };
                for (uint32_t i = tid; i < rows * columns; i += BA_THREADS) {
                    const uint32_t r = i / columns, col = 4 * (i % columns);
                    float m = -INFINITY, l = 0.0f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                    for (int64_t w = first; w <= last; ++w) m = fmaxf(m, __ldcg(of(w, r) + vdim));
#pragma unroll 8
                    for (int64_t w = first; w <= last; ++w) {
                        const float* row = of(w, r);
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(row + vdim)), y0 = __ldcg(reinterpret_cast<const float2*>(row + col)),
                                     y1 = __ldcg(reinterpret_cast<const float2*>(row + col + 2));
                        const float f = ml.y == 0.0f ? 0.0f : ex2(ml.x - m);
                        l = fmaf(f, ml.y, l);
                        v = make_float4(fmaf(f, y0.x, v.x), fmaf(f, y0.y, v.y), fmaf(f, y1.x, v.z), fmaf(f, y1.y, v.w));
                    }
                    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                    store4(r, col, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
            }
        }
        __syncthreads();        // the results have been read: the next plane's queries may come
        next_plane(c, group, &at);
        if (!at.slabs) break;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

constexpr uint32_t BA_MOST_CTAS = 2 * 192;

template <int MODE, int MAXD, int STAGES>
int32_t launch_block_attention(holo_b200_ctx* ctx, BlockAttnParams& p) {
    const uint32_t dim = p.a.c.dim, vdim = p.a.c.vdim;
    // 16-byte units of 8 neighbouring rows on different banks: an odd number of them a row, or units moved by the row's number
    auto pitch = [](uint32_t d) { return d % 128 == 0 || (d / 16) % 2 == 1 ? d : d + 16; };
    p.k_pitch = pitch(dim);
    p.v_pitch = pitch(vdim);
    p.slab_bytes = BA_SLAB * (p.k_pitch + p.v_pitch) + 256;
    p.q_pitch = 2 * dim + 16;
    const uint32_t queries = (MODE == 2 ? 2 : 1) * BA_ROWS * p.q_pitch, merge = BA_WARPS * 4 * vdim * 4;
    p.head_bytes = ((queries > merge ? queries : merge) + 127u) & ~127u;
    const uint32_t smem = p.head_bytes + BA_WARPS * STAGES * p.slab_bytes;
    static thread_local int configured_device = -1;
    static thread_local uint32_t configured = 0;
    if (configured_device != ctx->device || configured < smem) {
        HOLO_CUDA(cudaFuncSetAttribute(block_attention_kernel<MODE, MAXD, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        configured_device = ctx->device;
        configured = smem;
    }
    const uint32_t ctas = (uint32_t)ctx->sm_count * (MAXD <= 128 ? 2 : 1);
    HOLO_CUDA(holo_launch_kernel(ctx, block_attention_kernel<MODE, MAXD, STAGES>, dim3(ctas < BA_MOST_CTAS ? ctas : BA_MOST_CTAS), dim3(BA_THREADS), smem, 1, p));
    ctx->launches++;
    return HOLO_OK;
}
template <int MODE>
int32_t launch_block_attention_dims(holo_b200_ctx* ctx, BlockAttnParams& p) {
    const uint32_t d = p.a.c.dim > p.a.c.vdim ? p.a.c.dim : p.a.c.vdim;
    if (d <= 64) return launch_block_attention<MODE, 64, 5>(ctx, p);
    return d <= 128 ? launch_block_attention<MODE, 128, 3>(ctx, p) : launch_block_attention<MODE, 256, 3>(ctx, p);
}

}  // namespace

int32_t holo_try_block_attention(holo_b200_ctx* ctx, const HoloBlockAttnArgs& a, bool* taken) {
    *taken = false;
    const HoloBlockCache& c = a.c;
    if (c.dim % 16 != 0 || c.vdim % 16 != 0 || c.dim > 256 || c.vdim > 256) return HOLO_OK;
    if ((((uintptr_t)c.k_codes | (uintptr_t)c.v_codes) & 15u) != 0) return HOLO_OK;
    if ((uint64_t)c.blocks * c.kv_heads * c.block_rows >= 0xffffffffull || (uint64_t)c.rows * a.heads > 0x7fffffffull) return HOLO_OK;      // row numbers of 32 bits
    if (!ctx->block_partials) {
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        HOLO_CUDA(cudaStreamIsCapturing(ctx->stream, &capturing));
        if (capturing != cudaStreamCaptureStatusNone)
            return holo_fail(HOLO_ERR_DISPATCH, "dispatch failed: block_cache_attention allocates its buffer on its first call, which cannot be recorded: make one before");
        HOLO_CUDA(cudaMalloc(&ctx->block_partials, (uint64_t)BA_MOST_CTAS * 2 * BA_ROWS * (256 + 2) * sizeof(float)));
    }
    *taken = true;
    BlockAttnParams p = {};
    p.a = a;
    p.partials = ctx->block_partials;
    p.arrivals = ctx->attn_arrivals;
    p.group = a.heads / c.kv_heads;
    const uint32_t es = (uint32_t)holo_dtype_size(a.dtype);
    p.aligned_out = ((uintptr_t)a.out % (4 * es)) == 0 && a.ld % 4 == 0;
    if (a.dtype == HOLO_DTYPE_BF16) return launch_block_attention_dims<0>(ctx, p);
    return a.dtype == HOLO_DTYPE_F16 ? launch_block_attention_dims<1>(ctx, p) : launch_block_attention_dims<2>(ctx, p);
}
