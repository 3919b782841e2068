// Attention of few rows of each sequence over the int8 block cache (the BlockCacheAttention call), for dims in steps of 16 up to 256.
//
// A warp takes four or eight query rows (a row is a new position and a head of the group) against slabs of 32 keys.
// Scores: the codes are the int8 operand of mma.sync m16n8k32 as they lie in memory. A query row is scaled by a power of two to a largest
// value in [2^29, 2^30), rounded to an integer and cut into four digits of base 256, each a row of the product: sums of digits are exact
// integers, joined in f32. That holds a query to 2^-31 of its row's largest value, whatever its type.
// Weights: w = 2^(s - max) * scale_v, f32, relative to a power of two that follows the largest scale_v seen and lifted by 2^14, so that weights 2^28
// below the largest are still normal f16; two f16 terms hold 22 bits. Four rows take both terms in the eight columns of one product; eight rows
// take two products, or, for a bf16 result, the first term alone (2^-11 of a weight, an eighth of the result's own rounding).
// Values: a code is exact in f16; two of them take a byte permute onto 1024's exponent and a packed subtraction (1024 + 128 + c - 1152).
// The product is V^T w^T (m16n8k16): a weight's place among the scores is its place as an operand, nothing is transposed.
//
// Bound for single tokens: HBM, a byte an element. Loaded latency is 2 to 3 us, so 100 KB and more have to be on their way to every SM:
// each of a CTA's four warps has a ring of its own, slabs copied 16 bytes at a time (cp.async), and takes every fourth slab, with a
// maximum, sums and a context of its own; no barrier stands between a warp and its next slab.
// All slabs of the call (sequence by sequence, head by head, four or eight rows at a time) form one list that the CTAs share out evenly, so
// that neither short sequences nor few heads leave SMs without work. Where a share begins or ends inside a plane its partial result goes
// to a buffer of the context, and the last of the plane's CTAs to arrive adds them up in the order of the list: nobody waits,
// and no order of arrival shows in the result.
#include "block_list.cuh"

namespace {

constexpr int BA_WARPS = 4, BA_SLAB = 32, BA_MOST_ROWS = 8;
constexpr uint32_t BA_THREADS = BA_WARPS * 32;

struct BlockAttnParams {
    HoloBlockAttnArgs a;
    float* partials;          // [CTAs][2][8 rows][vdim + 2]
    uint32_t* arrivals;       // a counter per CTA, zero between launches
    uint32_t group, k_pitch, v_pitch, slab_bytes, head_bytes;
    int32_t br_shift;         // -1: block_rows is no power of two
    bool aligned_out;
};

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two CTAs an SM have some 114 KB each: the results of eight rows of 128 columns, 16 KB for four warps, are joined in two passes of 64 columns.
// In one pass a CTA takes 118 KB, an SM holds one, and the list, cut for two, is worked through in two turns. One pass and two, dim 128: 64
// sequences of 4096 positions, 16 heads over 2, 63.2 and 40.3 us, 8 over 1 40.9 and 27.8; two rows of each, 32 over 8, 159 and 102; eight
// sequences of 1000, 16 over 2, 14.5 and 16.5; one of 30000 34.3 and 35.7.
template <int RT, int MAXD, bool EXACT>
constexpr uint32_t BA_PASSES = RT == 2 && MAXD == 128 && EXACT ? 2 : 1;

// RT: four query rows or eight. D: dim and vdim where both are MAXD (their steps are constants then), else 0. SECOND: eight rows' weights
// as two terms.
template <int RT, int MAXD, bool EXACT, bool SECOND, int STAGES, int CTAS>
__global__ void __launch_bounds__(BA_THREADS, CTAS)
block_attention_kernel(const __grid_constant__ BlockAttnParams p) {
    constexpr int R = 4 * RT, KSTEPS = MAXD / 32, CHUNKS = MAXD / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_row[R], s_ml[BA_WARPS][R][3];
    __shared__ uint32_t s_last;
    const HoloBlockAttnArgs& a = p.a;
    const HoloBlockCache& c = a.c;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, in_quad = lane & 3;
    const uint32_t group = p.group, dim = EXACT ? MAXD : c.dim, vdim = EXACT ? MAXD : c.vdim, br = c.block_rows;
    const uint32_t k_pitch = EXACT && MAXD % 128 == 0 ? MAXD : p.k_pitch, v_pitch = EXACT && MAXD % 128 == 0 ? MAXD : p.v_pitch;
    const bool k_turns = EXACT ? MAXD % 128 == 0 : dim % 128 == 0, v_turns = EXACT ? MAXD % 128 == 0 : vdim % 128 == 0;
    holo_pdl_trigger();
    holo_pdl_wait();
    if (blockIdx.x == 0) check_sequences(c.starts, c.lengths, c.sequences, c.rows, (int64_t)c.table_ld * br, c.status);

    Share mine;
    if (!find_share<R, BA_SLAB, BA_WARPS, 8>(c, group, &mine)) return;
    const uint32_t lo = mine.lo, hi = mine.hi;
    const Plane first = mine.first;

    // ---- a plane's rows: requested early, cut into digits when the plane begins ----
    constexpr int OWN = R / BA_WARPS;
    float x[OWN][MAXD / 32];
    auto load_rows = [&](const Plane& f) {
#pragma unroll
        for (int y = 0; y < OWN; ++y) {
            const uint32_t r = warp + BA_WARPS * y, flat = f.tile * R + r, i = flat / group, head = f.head * group + flat % group;
#pragma unroll
            for (int e = 0; e < MAXD / 32; ++e) {
                const uint32_t d = lane + 32 * e;
                x[y][e] = i < f.n && d < dim ? seq_load(a.q, (uint64_t)(f.first_row + i) * a.q_ld + (uint64_t)head * dim + d, a.dtype) : 0.0f;
            }
        }
    };
    load_rows(first);

    // ---- the ring of this warp ----
    const uint32_t ring = smem_u32(smem) + p.head_bytes + warp * STAGES * p.slab_bytes;
    const uint8_t* ring_at = smem + p.head_bytes + warp * STAGES * p.slab_bytes;
    const uint32_t k_chunks = dim / 16, v_chunks = vdim / 16;
    // A whole slab lies in one block where block_rows is a multiple of 32: one number says where its rows are. Rows of the block behind the
    // sequence's last position come along, are masked, and are integers whatever they hold.
    const bool one_block = br % BA_SLAB == 0;
    auto block_of = [&](uint32_t pos) { return p.br_shift >= 0 ? pos >> p.br_shift : pos / br; };
    Plane ahead = first;            // where the next slab to request lies
    uint32_t ahead_slab, ahead_end, ahead_sees, ids_at = 0;
    int ahead_id = -1, ids = -1;    // ids: the blocks from number ids_at on, one a lane
    bool more = true;
    auto load_ids = [&](uint32_t blk) {
        ids_at = blk;
        ids = blk + lane <= block_of(ahead_sees - 1) ? c.table[(uint64_t)ahead.seq * c.table_ld + blk + lane] : -1;
    };
    auto enter_ahead = [&]() {
        mine.ends_of(ahead, &ahead_slab, &ahead_end);
        ahead_slab += warp;
        ahead_sees = keys_of_plane<R>(ahead, ahead.tile, group);
        load_ids(block_of(ahead_slab * BA_SLAB));
    };
    auto find_ahead = [&]() {
        while (ahead_slab >= ahead_end) {
            if (ahead.at + ahead.slabs >= hi) {
                more = false;
                return;
            }
            next_plane<R, BA_SLAB>(c, group, &ahead);
            if (!ahead.slabs) {
                more = false;
                return;
            }
            enter_ahead();
        }
        const uint32_t at_pos = ahead_slab * BA_SLAB, pos = at_pos + (one_block ? 0u : lane);
        if (block_of(min(at_pos + BA_SLAB, ahead_sees) - 1) - ids_at > 31) load_ids(block_of(at_pos));
        const bool there = pos < ahead_sees;
        ahead_id = __shfl_sync(0xffffffffu, ids, there ? block_of(pos) - ids_at : 0u);
        if (!there) ahead_id = -1;
        if ((uint32_t)ahead_id >= c.blocks) {
            if (there) atomicOr(c.status, HOLO_STATUS_TABLE);
            ahead_id = -1;
        }
    };
    auto request = [&](uint32_t stage) {
        if (more) {
            const uint32_t to = ring + stage * p.slab_bytes, to_v = to + BA_SLAB * k_pitch, to_s = to_v + BA_SLAB * v_pitch + 4 * lane;
            const uint32_t pos = ahead_slab * BA_SLAB + (one_block ? 0u : lane);
            const bool take = ahead_id >= 0;
            const uint32_t plane = (uint32_t)max(ahead_id, 0) * c.kv_heads + ahead.head;
            const uint32_t row = plane * br + (pos - block_of(pos) * br);
            if (one_block) {
                const int8_t *k = c.k_codes + (uint64_t)row * dim, *v = c.v_codes + (uint64_t)row * vdim;
                if (EXACT) {
                    constexpr uint32_t CH = MAXD / 16, KEYS = 32 / CH;     // 16-byte units a row, rows a turn
                    const uint32_t key = lane / CH, x = lane % CH;
#pragma unroll
                    for (uint32_t i = 0; i < CH; ++i) {
                        const uint32_t at = key + KEYS * i, y = k_turns ? x ^ (at & 7u) : x;
                        cp_async16(to + at * k_pitch + 16 * y, k + 16 * lane + 512 * i, take);
                        cp_async16(to_v + at * v_pitch + 16 * y, v + 16 * lane + 512 * i, take);
                    }
                } else {
                    for (uint32_t i = lane; i < BA_SLAB * k_chunks; i += 32) {
                        const uint32_t key = i / k_chunks, x = i % k_chunks;
                        cp_async16(to + key * k_pitch + 16 * (k_turns ? x ^ (key & 7u) : x), k + 16 * i, take);
                    }
                    for (uint32_t i = lane; i < BA_SLAB * v_chunks; i += 32) {
                        const uint32_t key = i / v_chunks, x = i % v_chunks;
                        cp_async16(to_v + key * v_pitch + 16 * (v_turns ? x ^ (key & 7u) : x), v + 16 * i, take);
                    }
                }
            } else {
                const uint32_t where = take ? row : 0xffffffffu;
                for (uint32_t i = lane; i < BA_SLAB * k_chunks; i += 32) {
                    const uint32_t key = i / k_chunks, x = i % k_chunks, r = __shfl_sync(0xffffffffu, where, key);
                    cp_async16(to + key * k_pitch + 16 * (k_turns ? x ^ (key & 7u) : x), c.k_codes + (r == 0xffffffffu ? 0 : (uint64_t)r * dim + 16 * x), r != 0xffffffffu);
                }
                for (uint32_t i = lane; i < BA_SLAB * v_chunks; i += 32) {
                    const uint32_t key = i / v_chunks, x = i % v_chunks, r = __shfl_sync(0xffffffffu, where, key);
                    cp_async16(to_v + key * v_pitch + 16 * (v_turns ? x ^ (key & 7u) : x), c.v_codes + (r == 0xffffffffu ? 0 : (uint64_t)r * vdim + 16 * x), r != 0xffffffffu);
                }
            }
            cp_async4(to_s, c.k_scales + plane, take);
            cp_async4(to_s + 128, c.v_scales + plane, take);
            ahead_slab += BA_WARPS;
            find_ahead();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    enter_ahead();
    find_ahead();
#pragma unroll 1
    for (int s = 0; s < STAGES - 1; ++s) request(s);

    uint32_t stage = 0;
    Plane at = first;
#pragma unroll 1
    for (;;) {
        // ---- one plane: its rows' digits, then the slabs of it that are this CTA's ----
        const uint32_t rows = min((uint32_t)R, at.n * group - at.tile * R);
#pragma unroll
        for (int y = 0; y < OWN; ++y) {
            const uint32_t r = warp + BA_WARPS * y;
            float most = 0.0f;
            bool finite = true;
#pragma unroll
            for (int e = 0; e < MAXD / 32; ++e) {
                most = fmaxf(most, fabsf(x[y][e]));
                finite = finite && fabsf(x[y][e]) < INFINITY;
            }
            // magnitudes order as their bits do
            most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
            finite = __all_sync(0xffffffffu, finite);
            // 2^e <= most < 2^(e + 1); two factors, since 2^(29 - e) alone may overflow
            const uint32_t bits = __float_as_uint(most);
            const int up = finite && bits ? 29 - (bits >> 23 ? (int)(bits >> 23) - 127 : -118 - __clz((int)bits)) : 0;
            const float f0 = power_of_two(up / 2), f1 = power_of_two(up - up / 2);
            uint8_t* to = smem + (r >> 2) * 16 * MAXD + (r & 3u) * MAXD + lane;       // digit g of row r is row 4 g + r % 4 of product r / 4
#pragma unroll
            for (int e = 0; e < MAXD / 32; ++e) {
                int v = finite ? __float2int_rn(x[y][e] * f0 * f1) : 0;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int digit = (int)(int8_t)v;
                    to[4 * g * MAXD + 32 * e] = (uint8_t)digit;
                    v = (v - digit) >> 8;
                }
            }
            if (lane == 0) s_row[r] = finite ? a.scale * LOG2E * power_of_two(-(up / 2)) * power_of_two(-(up - up / 2)) : NAN;
        }
        __syncthreads();
        uint32_t q[RT][KSTEPS][4];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x) q[t][k][x] = *reinterpret_cast<const uint32_t*>(smem + t * 16 * MAXD + (quad + 8 * (x & 1)) * MAXD + 32 * k + 16 * (x >> 1) + 4 * in_quad);
        // this lane's row (four rows: in both halves of the warp)
        const uint32_t row = RT == 1 ? quad & 3u : quad, row_at = (at.tile * R + min(row, rows - 1)) / group;
        const float row_scale = s_row[row];
        const uint32_t limit = (uint32_t)max(0, at.length - (int32_t)(at.n - row_at - 1));
        const uint32_t common = (uint32_t)max(0, at.length - (int32_t)(at.n - (at.tile * R) / group - 1));      // keys that all rows see
        float o[CHUNKS][4], top = -INFINITY, sum = 0.0f;
        int lift = -1000;           // the exponent that value scales are relative to
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[i][x] = 0.0f;
        uint32_t from, to;
        mine.ends_of(at, &from, &to);
#pragma unroll 1
        for (uint32_t slab = from + warp; slab < to; slab += BA_WARPS) {
            request(stage == 0 ? STAGES - 1 : stage - 1);      // where the slab before this one was
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t k_at = ring + stage * p.slab_bytes + lane * k_pitch, v_at = ring + stage * p.slab_bytes + BA_SLAB * k_pitch + lane * v_pitch;
            const float* scales = reinterpret_cast<const float*>(ring_at + stage * p.slab_bytes + BA_SLAB * (k_pitch + v_pitch));
            int dots[RT][4][4];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int x = 0; x < 4; ++x) dots[t][j][x] = 0;
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
                if (!EXACT && 32 * k >= dim) break;
                // dims past the last are digits of zero: what stands there does not count
                uint32_t w0[4], w1[4];
                ldsm4(k_at + 16 * (k_turns ? (2 * k) ^ (lane & 7u) : 2 * k), w0);
                ldsm4(k_at + 16 * (k_turns ? (2 * k + 1) ^ (lane & 7u) : 2 * k + 1), w1);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int t = 0; t < RT; ++t) mma_s8(dots[t][j], q[t][k], w0[j], w1[j]);
            }
            const uint32_t key0 = slab * BA_SLAB + 2 * in_quad;
            float s[4][2], most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 ks = *reinterpret_cast<const float2*>(scales + 8 * j + 2 * in_quad);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    // this half's digits (0 and 2, or 1 and 3), then the other half's
                    const float half0 = fmaf((float)dots[0][j][x + 2], 65536.0f, (float)dots[0][j][x]);
                    float v;
                    if (RT == 1) {
                        const float other = __shfl_xor_sync(0xffffffffu, half0, 16);
                        v = lane < 16 ? fmaf(other, 256.0f, half0) : fmaf(half0, 256.0f, other);
                    } else {
                        const float half1 = fmaf((float)dots[RT - 1][j][x + 2], 65536.0f, (float)dots[RT - 1][j][x]);
                        const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? half1 : half0, 16);
                        v = lane < 16 ? fmaf(other, 256.0f, half0) : fmaf(half1, 256.0f, other);
                    }
                    s[j][x] = v * (row_scale * (x ? ks.y : ks.x));
                }
            }
            if ((slab + 1) * BA_SLAB > common) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        if (key0 + 8 * j + x >= limit) s[j][x] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) most = fmaxf(most, fmaxf(s[j][0], s[j][1]));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const float largest = scales[32 + lane];
            int e = largest > 0.0f && largest < INFINITY ? (int)(__float_as_uint(largest) >> 23) - 126 : -110;
            e = max(e, -110);
            if (one_block) e = __shfl_sync(0xffffffffu, e, 0);
            else e = __reduce_max_sync(0xffffffffu, e);
            if (__any_sync(0xffffffffu, most > top) || e > lift) {
                const int higher = max(e, lift);
                const float turn = lift == -1000 ? 0.0f : lift - higher < -126 ? 0.0f : power_of_two(lift - higher);
                lift = higher;
                const float t = fmaxf(top, most), f = top == t ? 1.0f : ex2(top - t);
                top = t;
                sum *= f;
                // columns 2c and 2c + 1 of this lane's context are the rows of quads 2c and 2c + 1
                const float g0 = __shfl_sync(0xffffffffu, f, 8 * in_quad) * turn, g1 = __shfl_sync(0xffffffffu, f, 8 * in_quad + 4) * turn;
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i) {
                    o[i][0] *= g0; o[i][1] *= g1;
                    o[i][2] *= g0; o[i][3] *= g1;
                }
            }
            const float least = top == -INFINITY ? 0.0f : top, raise = power_of_two(min(14 - lift, 127));
            uint32_t w[4], w2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 vs = *reinterpret_cast<const float2*>(scales + 32 + 8 * j + 2 * in_quad);
                const float e0 = ex2(s[j][0] - least), e1 = ex2(s[j][1] - least);
                sum += e0 + e1;
                const float y0 = e0 * (vs.x * raise), y1 = e1 * (vs.y * raise);
                w[j] = half_pair(y0, y1);
                if (RT == 1 || SECOND) {
                    const float2 h = half_values(w[j]);
                    w2[j] = half_pair(y0 - h.x, y1 - h.y);
                    if (RT == 1 && lane >= 16) w[j] = w2[j];       // columns 4 to 7: the second terms
                }
            }
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                if (!EXACT && 16 * i >= vdim) break;
                uint32_t v[4];
                ldsm4t(v_at + 16 * (v_turns ? i ^ (lane & 7u) : i), v);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t u0 = v[2 * k] ^ 0x80808080u, u1 = v[2 * k + 1] ^ 0x80808080u;
                    // rows 0 to 7 of the product are the even dims, 8 to 15 the odd ones
                    const uint32_t m[4] = {codes_to_half<PICK02>(u0), codes_to_half<PICK13>(u0), codes_to_half<PICK02>(u1), codes_to_half<PICK13>(u1)};
                    mma_f16(o[i], m, w[2 * k], w[2 * k + 1]);
                    if (RT == 2 && SECOND) mma_f16(o[i], m, w2[2 * k], w2[2 * k + 1]);
                }
            }
            __syncwarp();       // the slab has been read
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        // ---- the four warps' results, through the memory of the digits ----
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (in_quad == 0 && (RT == 2 || lane < 16)) {
            s_ml[warp][row][0] = top;
            s_ml[warp][row][1] = sum;
            s_ml[warp][row][2] = lift == -1000 ? 0.0f : power_of_two(lift - 14);
        }
        Plane next = at;
        const bool begins = at.at >= lo, ends = at.at + at.slabs <= hi, whole = begins && ends;
        if (at.at + at.slabs < hi) {
            next_plane<R, BA_SLAB>(c, group, &next);
            if (next.slabs) load_rows(next);
        }
        float* partial = p.partials + ((uint64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * R * (vdim + 2);
        float* s_o = reinterpret_cast<float*>(smem);       // [warp][R][columns of a pass]
        constexpr uint32_t PASSES = BA_PASSES<RT, MAXD, EXACT>, STEPS = CHUNKS / PASSES;
        const uint32_t columns = vdim / 4, across = vdim / PASSES;      // units of four; columns of a pass
        auto store4 = [&](uint32_t r, uint32_t col, float4 v) {
            const uint32_t flat = at.tile * R + r;
            const uint64_t index = (uint64_t)(at.first_row + flat / group) * a.ld + (uint64_t)(at.head * group + flat % group) * vdim + col;
            if (p.aligned_out) {
                if (a.dtype == HOLO_DTYPE_F32) *reinterpret_cast<float4*>((float*)a.out + index) = v;
                else if (a.dtype == HOLO_DTYPE_F16) *reinterpret_cast<uint2*>((uint16_t*)a.out + index) = make_uint2(half_pair(v.x, v.y), half_pair(v.z, v.w));
                else *reinterpret_cast<uint2*>((uint16_t*)a.out + index) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
            } else {
                seq_store(a.out, index, v.x, a.dtype); seq_store(a.out, index + 1, v.y, a.dtype);
                seq_store(a.out, index + 2, v.z, a.dtype); seq_store(a.out, index + 3, v.w, a.dtype);
            }
        };
        __syncthreads();        // the digits have been read
#pragma unroll
        for (uint32_t pass = 0; pass < PASSES; ++pass) {
            if (pass) __syncthreads();      // the last pass's have been read
#pragma unroll
            for (uint32_t i = pass * STEPS; i < (pass + 1) * STEPS; ++i) {
                if (!EXACT && 16 * i >= vdim) break;
                float y[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) y[x] = RT == 1 ? o[i][x] + __shfl_xor_sync(0xffffffffu, o[i][x], 2) : o[i][x];
                if (RT == 2 || in_quad < 2) {
                    float* to4 = s_o + (warp * R + 2 * in_quad) * across + 16 * (i - pass * STEPS) + 2 * quad;
                    *reinterpret_cast<float2*>(to4) = make_float2(y[0], y[2]);
                    *reinterpret_cast<float2*>(to4 + across) = make_float2(y[1], y[3]);
                }
            }
            __syncthreads();
            for (uint32_t i = tid; i < rows * (across / 4); i += BA_THREADS) {
                const uint32_t r = i / (across / 4), x = 4 * (i % (across / 4)), col = pass * across + x;
                float m = -INFINITY, l = 0.0f;
#pragma unroll
                for (int w = 0; w < BA_WARPS; ++w) m = fmaxf(m, s_ml[w][r][0]);
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < BA_WARPS; ++w) {
                    const float lw = s_ml[w][r][1];
                    if (lw != 0.0f) {       // NaN is not 0
                        const float f = ex2(s_ml[w][r][0] - m), g = f * s_ml[w][r][2];
                        const float4 y = *reinterpret_cast<const float4*>(s_o + (w * R + r) * across + x);
                        l = fmaf(f, lw, l);
                        v = make_float4(fmaf(g, y.x, v.x), fmaf(g, y.y, v.y), fmaf(g, y.z, v.z), fmaf(g, y.w, v.w));
                    }
                }
                if (whole) {
                    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                    store4(r, col, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                } else {
                    float* to2 = partial + r * (vdim + 2);
                    __stcg(reinterpret_cast<float2*>(to2 + col), make_float2(v.x, v.y));
                    __stcg(reinterpret_cast<float2*>(to2 + col + 2), make_float2(v.z, v.w));
                    if (col == 0) __stcg(reinterpret_cast<float2*>(to2 + vdim), make_float2(m, l));
                }
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
                const float* base = p.partials + (uint64_t)from_cta * 2 * R * (vdim + 2);
                const uint32_t step = 2 * R * (vdim + 2), own = R * (vdim + 2);
                auto part = [&](uint32_t w, uint32_t r) { return base + (uint64_t)w * step + (w == 0 ? own : 0u) + r * (vdim + 2); };
                // the parts' weights first: a warp a row, a part a lane; then a column of all parts at a time
                float* s_f = s_o;         // [R][count]
#pragma unroll 1
                for (uint32_t r = warp; r < rows; r += BA_WARPS) {
                    float m = -INFINITY, l = 0.0f;
#pragma unroll 1
                    for (uint32_t w = lane; w < count; w += 64) {
                        const float2 y0 = __ldcg(reinterpret_cast<const float2*>(part(w, r) + vdim));
                        const float2 y1 = w + 32 < count ? __ldcg(reinterpret_cast<const float2*>(part(w + 32, r) + vdim)) : make_float2(-INFINITY, 0.0f);
                        const float t = fmaxf(m, fmaxf(y0.x, y1.x));
                        s_f[r * count + w] = y0.x;
                        if (w + 32 < count) s_f[r * count + w + 32] = y1.x;
                        // parts that saw nothing have no sum; NaN is not 0
                        if (l != 0.0f) l *= ex2(m - t);
                        if (y0.y != 0.0f) l = fmaf(ex2(y0.x - t), y0.y, l);
                        if (y1.y != 0.0f) l = fmaf(ex2(y1.x - t), y1.y, l);
                        m = t;
                    }
                    float top_m = m;
                    for (int o = 16; o > 0; o >>= 1) top_m = fmaxf(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
                    if (l != 0.0f) l *= ex2(m - top_m);
                    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                    __syncwarp();
                    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                    for (uint32_t w = lane; w < count; w += 32) {
                        const float x0 = s_f[r * count + w];
                        s_f[r * count + w] = l == 0.0f || (x0 == -INFINITY && l == l) ? 0.0f : ex2(x0 - top_m) * inv;
                    }
                }
                __syncthreads();
                for (uint32_t i = tid; i < rows * columns; i += BA_THREADS) {
                    const uint32_t r = i / columns, col = 4 * (i % columns);
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 16
                    for (uint32_t w = 0; w < count; ++w) {
                        const float* of = part(w, r) + col;
                        const float2 y0 = __ldcg(reinterpret_cast<const float2*>(of)), y1 = __ldcg(reinterpret_cast<const float2*>(of + 2));
                        const float f = s_f[r * count + w];
                        v = make_float4(fmaf(f, y0.x, v.x), fmaf(f, y0.y, v.y), fmaf(f, y1.x, v.z), fmaf(f, y1.y, v.w));
                    }
                    store4(r, col, v);
                }
            }
        }
        if (at.at + at.slabs >= hi || !next.slabs) break;
        at = next;
        __syncthreads();        // the results have been read: the next plane's digits may come
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

constexpr uint32_t BA_MOST_CTAS = 3 * 192;

// 16-byte units of 8 neighbouring rows on different banks: an odd number of them a row, or units moved by the row's number
constexpr uint32_t ba_pitch(uint32_t d) { return d % 128 == 0 || (d / 16) % 2 == 1 ? d : d + 16; }
constexpr uint32_t ba_slab_bytes(uint32_t k_pitch, uint32_t v_pitch) { return BA_SLAB * (k_pitch + v_pitch) + 256; }
// the digits; then the warps' results, `columns` of them at a time; then the weights of a plane's parts
constexpr uint32_t ba_head_bytes(uint32_t rt, uint32_t maxd, uint32_t columns, uint32_t ctas) {
    const uint32_t digits = rt * 16 * maxd, merge = BA_WARPS * 4 * rt * columns * 4, weights = 16 * rt * ctas, most = digits > merge ? digits : merge;
    return ((most > weights ? most : weights) + 127u) & ~127u;
}
// what no call of an instance goes beyond
constexpr uint32_t ba_most_bytes(uint32_t rt, uint32_t maxd, uint32_t stages) {
    uint32_t pitch = 0;
    for (uint32_t d = 16; d <= maxd; d += 16) pitch = ba_pitch(d) > pitch ? ba_pitch(d) : pitch;
    return ba_head_bytes(rt, maxd, maxd, BA_MOST_CTAS) + BA_WARPS * stages * ba_slab_bytes(pitch, pitch);
}

template <int RT, int MAXD, bool EXACT, bool SECOND, int STAGES, int CTAS>
int32_t launch_block_attention(holo_b200_ctx* ctx, BlockAttnParams& p) {
    constexpr uint32_t PASSES = BA_PASSES<RT, MAXD, EXACT>;
    // 228 KB an SM, of which every CTA takes 1 KB for itself and has 512 bytes of static variables; the other dims are below these
    static_assert(!EXACT || CTAS * (ba_head_bytes(RT, MAXD, MAXD / PASSES, 148 * CTAS) + BA_WARPS * STAGES * ba_slab_bytes(ba_pitch(MAXD), ba_pitch(MAXD)) + 1536) <= 228 * 1024,
                  "the CTAs that an SM is to hold do not fit");
    const uint32_t ctas = (uint32_t)ctx->sm_count * CTAS < BA_MOST_CTAS ? (uint32_t)ctx->sm_count * CTAS : BA_MOST_CTAS;
    p.k_pitch = ba_pitch(p.a.c.dim);
    p.v_pitch = ba_pitch(p.a.c.vdim);
    p.slab_bytes = ba_slab_bytes(p.k_pitch, p.v_pitch);
    p.head_bytes = ba_head_bytes(RT, MAXD, p.a.c.vdim / PASSES, ctas);
    const uint32_t smem = p.head_bytes + BA_WARPS * STAGES * p.slab_bytes;
    static thread_local int configured_device = -1;
    if (configured_device != ctx->device) {
        // the attribute is the process's: every thread sets the same, whatever sizes its calls have
        HOLO_CUDA(cudaFuncSetAttribute(block_attention_kernel<RT, MAXD, EXACT, SECOND, STAGES, CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ba_most_bytes(RT, MAXD, STAGES)));
        configured_device = ctx->device;
    }
    HOLO_CUDA(holo_launch_kernel(ctx, block_attention_kernel<RT, MAXD, EXACT, SECOND, STAGES, CTAS>, dim3(ctas), dim3(BA_THREADS), smem, 1, p));
    ctx->launches++;
    return HOLO_OK;
}
template <int RT, bool SECOND>
int32_t launch_block_attention_dims(holo_b200_ctx* ctx, BlockAttnParams& p) {
    const HoloBlockCache& c = p.a.c;
    const uint32_t d = c.dim > c.vdim ? c.dim : c.vdim;
    const bool exact = c.dim == c.vdim && (d == 64 || d == 128);
    if (d <= 64) return exact ? launch_block_attention<RT, 64, true, SECOND, 4, 2>(ctx, p) : launch_block_attention<RT, 64, false, SECOND, 4, 2>(ctx, p);
    if (d <= 128) return exact ? launch_block_attention<RT, 128, true, SECOND, 3, 2>(ctx, p) : launch_block_attention<RT, 128, false, SECOND, 3, 2>(ctx, p);
    return launch_block_attention<RT, 256, false, SECOND, 2, 1>(ctx, p);
}

}  // namespace

int32_t holo_try_block_attention(holo_b200_ctx* ctx, const HoloBlockAttnArgs& a, bool* taken) {
    *taken = false;
    const HoloBlockCache& c = a.c;
    if (c.dim % 16 != 0 || c.vdim % 16 != 0 || c.dim > 256 || c.vdim > 256) return HOLO_OK;
    if ((((uintptr_t)c.k_codes | (uintptr_t)c.v_codes) & 15u) != 0) return HOLO_OK;
    // row numbers, and slabs of the whole list, of 32 bits
    const uint64_t tiles = ((uint64_t)c.rows * (a.heads / c.kv_heads) / 4 + c.sequences) * c.kv_heads;
    if ((uint64_t)c.blocks * c.kv_heads * c.block_rows >= 0xffffffffull || (uint64_t)c.rows * a.heads > 0x7fffffffull) return HOLO_OK;
    if (tiles > 0x7fffffffull / (((uint64_t)c.table_ld * c.block_rows + BA_SLAB - 1) / BA_SLAB)) return HOLO_OK;
    if (!ctx->block_partials) {
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        HOLO_CUDA(cudaStreamIsCapturing(ctx->stream, &capturing));
        if (capturing != cudaStreamCaptureStatusNone)
            return holo_fail(HOLO_ERR_DISPATCH, "dispatch failed: block_cache_attention allocates its buffer on its first call, which cannot be recorded: make one before");
        HOLO_CUDA(cudaMalloc(&ctx->block_partials, (uint64_t)BA_MOST_CTAS * 2 * BA_MOST_ROWS * (256 + 2) * sizeof(float)));
    }
    *taken = true;
    BlockAttnParams p = {};
    p.a = a;
    p.partials = ctx->block_partials;
    p.arrivals = ctx->attn_arrivals;
    p.group = a.heads / c.kv_heads;
    p.br_shift = -1;
    for (int s = 0; s <= 10; ++s)
        if (c.block_rows == 1u << s) p.br_shift = s;
    const uint32_t es = (uint32_t)holo_dtype_size(a.dtype);
    p.aligned_out = ((uintptr_t)a.out % (4 * es)) == 0 && a.ld % 4 == 0;
    // four rows where that is a head's whole group of a single token: eight would be half empty
    if (p.group <= 4 && c.rows <= c.sequences) return launch_block_attention_dims<1, false>(ctx, p);
    return a.dtype == HOLO_DTYPE_BF16 ? launch_block_attention_dims<2, false>(ctx, p) : launch_block_attention_dims<2, true>(ctx, p);
}
