// Attention of many rows of each sequence (portions of prompts) over the int8 block cache on tcgen05, for 16-bit queries, dims in steps of
// 16 up to 128 and blocks of a multiple of 16 rows.
//
// A CTA takes 128 query rows of a kv head (a row is a new position and a head of the group) and walks the keys in tiles of 128:
//   warps 8-15 turn the tiles' codes into f16 (exact: integers of 8 bits) in the operands' swizzled layout, half of the warps K, half V, from
//              rings of two that asynchronous copies fill into rings of two; and the query rows, scaled by a power of two to a largest value
//              in [2^14, 2^15): exact in f16 but for values 2^29 smaller than the largest
//   warp 1     tcgen05.mma issuer: S = Q K^T of a tile while the softmax of the one before runs, then O += P V with P read from TMEM
//   warps 4-7  softmax, one thread per row. A block's scales are the same for 16 keys in a row: the key scale is a factor of the scores, the
//              value scale a term of the exponent, w = 2^(s - max + log2 scale_v), and is taken out of the row's sum again. Weights are
//              relative to a power of two above the largest value scale of the CTA's keys and rounded to f16 (by up to 2^-11 of a weight)
// The tiles of all planes form one list that the CTAs share out evenly; parts of a plane are joined as for few rows (block_list.cuh).
// TMEM: S of even tiles at 0, of odd ones at 128, their weights over them, O at 256.
// Bound: the softmax (3700 cycles a tile of 128 x 128, of which 1024 are ex2) and a plane's beginning (12 k cycles: queries, scales, first codes);
// the workers keep up. 109 us for bf16 portions of 128, 256, 77 and 128 rows behind 2048 to 8100 positions, 32 heads over 8 of dim 128.
#include "attention_issue.cuh"
#include "block_list.cuh"

namespace {

constexpr int BT_ROWS = 128, BT_TILE = 128, BT_WARPS = 16, BT_WORKERS = 128;      // threads that turn the codes of keys, and of values
// registers a thread: the workers' and the issuer's leave what the softmax's 128 scores take (their sum is the launch's at most)
constexpr int BT_ISSUER_REGS = 80, BT_SOFTMAX_REGS = 208, BT_WORKER_REGS = 112;
constexpr int BT_PLANE = 3;      // tiles that a plane's beginning and end cost as much as (portions as above, for 0, 2, 3, 4, 6: 134, 118, 110, 110, 113 us)
constexpr float BT_GROWTH = 8.0f;
constexpr int BT_LIFT = 7;
// A row's maximum (an exponent of two) of this size and more is taken off its scores before the exponents of value scales are added. Below, both
// are one sum, 2^-13 off at most, and the scores' product with their factor is fused with it; above, that sum loses the scales'
// exponents and the fused product the rounding that the maximum had, by whole factors of a weight. The test costs 1.5 %.
constexpr float BT_FAR = 0x1p12f;

struct BlockTileParams {
    HoloBlockAttnArgs a;
    float* partials;          // [CTAs][2][vdim + 2][128 rows]: a warp's rows side by side
    uint32_t* arrivals;       // a counter per CTA, zero between launches
    uint32_t group, k_chunks, v_chunks;      // chunks of 64 columns
    int32_t br_shift;
};

constexpr uint32_t PICK01 = 0x4140, PICK23 = 0x4342;

__global__ void __launch_bounds__(BT_WARPS * 32, 1)
block_tile_kernel(const __grid_constant__ BlockTileParams p) {
    extern __shared__ uint8_t smem_raw[];
    const HoloBlockAttnArgs& a = p.a;
    const HoloBlockCache& c = a.c;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - raw);
    const uint32_t k_bytes = p.k_chunks * TILE_CHUNK, v_bytes = p.v_chunks * TILE_CHUNK;
    const uint32_t o_k = k_bytes, o_v = o_k + 2 * k_bytes, o_raw = o_v + 2 * v_bytes, raw_bytes = BT_TILE * (c.dim + c.vdim), o_bars = o_raw + 2 * raw_bytes, bars = base + o_bars;
    const uint32_t bar_q_full = bars, bar_q_empty = bars + 8, bar_k_full = bars + 16, bar_k_empty = bars + 32, bar_v_full = bars + 48, bar_v_empty = bars + 64,
                   bar_s = bars + 192, bar_pa = bars + 208, bar_pb = bars + 224;      // two of each, by tile: nobody is two phases of one ahead
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(sm + o_bars + 120);
    volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(sm + o_bars + 124);
    uint32_t* s_last = reinterpret_cast<uint32_t*>(sm + o_bars + 128);
    int* s_lift = reinterpret_cast<int*>(sm + o_bars + 132);                       // [2], by plane
    uint32_t* s_most = reinterpret_cast<uint32_t*>(sm + o_bars + 144);              // [2][4], by plane
    const uint32_t bar_workers = bars + 176, bar_rows = bars + 184;                  // the eight worker warps meet, the four softmax warps
    float* s_row = reinterpret_cast<float*>(sm + o_bars + 256);                     // [2][128], by plane
    float* s_scale = s_row + 2 * BT_ROWS;                                           // [8][3][8], by tile: key scales; exponents; reciprocals. The keys' workers are up to four tiles ahead of the softmax
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = p.group, dim = c.dim, vdim = c.vdim, br = c.block_rows;
    if (tid == 0) {
        mbar_init(bar_q_full, 4);             // one arrival per worker warp
        mbar_init(bar_q_empty, 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(bar_k_full + 8 * s, 4);
            mbar_init(bar_k_empty + 8 * s, 1);
            mbar_init(bar_v_full + 8 * s, 4);
            mbar_init(bar_v_empty + 8 * s, 1);
            mbar_init(bar_s + 8 * s, 2);      // the scores, and the issuer that has seen the tile's scales
            mbar_init(bar_pa + 8 * s, 4);     // one arrival per softmax warp
            mbar_init(bar_pb + 8 * s, 4);
        }
        mbar_init(bar_workers, 8);
        mbar_init(bar_rows, 4);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    holo_pdl_wait();
    if (blockIdx.x == 0) check_sequences(c.starts, c.lengths, c.sequences, c.rows, (int64_t)c.table_ld * br, c.status);
    Share mine;
    if (!find_share<BT_ROWS, BT_TILE, 4, 4, BT_PLANE>(c, group, &mine)) return;       // the same for every thread
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    holo_pdl_trigger();
    const uint32_t tmem_base = *s_tmem;
    // everybody walks the planes by itself
    auto keys_of = [&](const Plane& f) { return keys_of_plane<BT_ROWS>(f, f.tile, group); };
    auto more = [&](Plane& f) {
        if (f.at + f.slabs >= mine.hi) return false;
        next_plane<BT_ROWS, BT_TILE, BT_PLANE>(c, group, &f);
        return f.slabs != 0 && f.at < mine.hi;
    };

    auto arrive_at = [&](uint32_t bar) {
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
    };
    auto all_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, long_wait(bar, parity, s_abort, c.status)) != 0; };

    if (warp >= 8) {
        // ---------------- workers: codes and queries into operands; warps 8-11 keys, 12-15 values ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BT_WORKER_REGS));
        // eight lanes take the 16-byte units of a row of codes, a warp four rows at a time: unit `unit` of keys 16 j + sub
        const bool values = warp >= 12;
        const uint32_t me = tid & 127u, unit = lane & 7u, sub = (warp & 3u) * 4 + (lane >> 3);
        const int8_t* codes = values ? c.v_codes : c.k_codes;
        const uint32_t d = values ? vdim : dim, raw0 = o_raw + (values ? 2 * BT_TILE * dim : 0u), raw_step = BT_TILE * d;
        const uint32_t to0 = values ? o_v : o_k, to_step = values ? v_bytes : k_bytes, bar_full = values ? bar_v_full : bar_k_full, bar_empty = values ? bar_v_empty : bar_k_empty;
        uint32_t nt = 0, np = 0;
        bool ok = true;
        auto block_of = [&](uint32_t pos) { return p.br_shift >= 0 ? pos >> p.br_shift : pos / br; };
        // 16 codes as 32 bytes of a 128-byte row: the row's 16-byte units stand at their number xor key % 8
        auto turn = [&](uint8_t* tile, uint32_t key, const uint4& v) {
            const uint32_t w[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                h[2 * e] = codes_to_half<PICK01>(w[e]);
                h[2 * e + 1] = codes_to_half<PICK23>(w[e]);
            }
            uint4* to = reinterpret_cast<uint4*>(tile + (unit >> 2) * TILE_CHUNK + key * 128);
            // the lanes of the two chunks begin with different halves: the eight lanes of a row meet all banks
            const uint32_t late = unit >> 2, at = (2 * (unit & 3u) + late) ^ (key & 7u);
            to[at] = late ? make_uint4(h[4], h[5], h[6], h[7]) : make_uint4(h[0], h[1], h[2], h[3]);
            to[at ^ 1u] = late ? make_uint4(h[0], h[1], h[2], h[3]) : make_uint4(h[4], h[5], h[6], h[7]);
        };
        auto arrive = [&](uint32_t bar) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive_at(bar);
        };
        Plane at = mine.first;
        do {
            uint32_t s0, s1;
            mine.ends_of(at, &s0, &s1);
            const uint32_t sees = keys_of(at), rows = min((uint32_t)BT_ROWS, at.n * group - at.tile * BT_ROWS);
            // Sixteen keys in a row lie in one block: lane j < 8 has the number of the block of keys 16 j of a tile, as the table has it
            auto find = [&](uint32_t tile) {
                const uint32_t pos = tile * BT_TILE + 16 * lane;
                return lane < 8 && tile < s1 && pos < sees ? c.table[(uint64_t)at.seq * c.table_ld + block_of(pos)] : -1;
            };
            // where those keys' rows begin in the cache, none: 0xffffffff
            auto rows_of = [&](uint32_t tile, int id) {
                const uint32_t pos = tile * BT_TILE + 16 * lane;
                if (lane >= 8 || tile >= s1 || pos >= sees) return 0xffffffffu;
                if ((uint32_t)id >= c.blocks) {
                    atomicOr(c.status, HOLO_STATUS_TABLE);
                    return 0xffffffffu;
                }
                return ((uint32_t)id * c.kv_heads + at.head) * br + (pos - block_of(pos) * br);
            };
            float ks = 0.0f, vs = 0.0f;
            // the codes of a tile into the ring, each unit by the thread that turns it
            auto request = [&](uint32_t to, uint32_t from) {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const uint32_t row = __shfl_sync(0xffffffffu, from, j);
                    const bool there = row != 0xffffffffu;
                    if (16 * unit < d) cp_async16(base + to + (16 * j + sub) * d + 16 * unit, codes + (there ? (uint64_t)(row + sub) * d + 16 * unit : 0), there);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            auto load_scales = [&](uint32_t from) {
                const bool there = from != 0xffffffffu;
                const uint32_t plane = there ? block_of(from) : 0u;
                ks = there ? c.k_scales[plane] : 0.0f;
                vs = there ? c.v_scales[plane] : 0.0f;
            };
            asm volatile("cp.async.wait_group 0;" ::: "memory");      // what was requested behind the last plane's end
            const int id0 = find(s0), id1 = find(s0 + 1);
            int ahead = find(s0 + 2);
            uint32_t from = rows_of(s0, id0);
            if (!values) load_scales(from);
            request(raw0 + (nt & 1u) * raw_step, from);
            from = rows_of(s0 + 1, id1);
            request(raw0 + (~nt & 1u) * raw_step, from);
            volatile uint32_t* most_of = s_most + 4 * (np & 1u);
            if (values) {
                // the largest value scale of the CTA's part of the plane
                float largest = 0.0f;
                for (uint32_t b = block_of(s0 * BT_TILE) + me, last = block_of(min(s1 * BT_TILE, sees) - 1); b <= last; b += BT_WORKERS) {
                    const int x = c.table[(uint64_t)at.seq * c.table_ld + b];
                    const float f = (uint32_t)x < c.blocks ? c.v_scales[(uint64_t)x * c.kv_heads + at.head] : 0.0f;
                    if (f < INFINITY) largest = fmaxf(largest, f);
                }
                const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));
                if (lane == 0) most_of[warp & 3u] = bits;
            }
            if (!values) {
                // the queries' memory is free when the last plane's last scores are there
                ok = np == 0 || all_wait(bar_q_empty, (np - 1) & 1u);
                if (!ok) break;
                // a thread its query row, on its way while the rest of the plane's beginning is done
                uint4 query[16];
                {
                    const uint32_t flat = at.tile * BT_ROWS + min(me, rows - 1), i = flat / group;
                    const uint16_t* from_q = (const uint16_t*)a.q + (uint64_t)(at.first_row + i) * a.q_ld + (uint64_t)(at.head * group + flat - i * group) * dim;
                    if (((uintptr_t)a.q & 15u) == 0 && (a.q_ld & 7u) == 0) {
#pragma unroll
                        for (int u = 0; u < 16; ++u) query[u] = 8 * u < dim ? *reinterpret_cast<const uint4*>(from_q + 8 * u) : make_uint4(0, 0, 0, 0);
                    } else {
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            uint32_t w[4] = {0, 0, 0, 0};
                            if (8 * u < dim)
#pragma unroll
                                for (int e = 0; e < 4; ++e) w[e] = from_q[8 * u + 2 * e] | (uint32_t)from_q[8 * u + 2 * e + 1] << 16;
                            query[u] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
                // magnitudes order as their bits do, infinities and NaN above all
                uint32_t most = 0;
#pragma unroll
                for (int u = 0; u < 16; ++u)
                    most = __vmaxu2(__vmaxu2(__vmaxu2(most, query[u].x & 0x7fff7fffu), query[u].y & 0x7fff7fffu), __vmaxu2(query[u].z & 0x7fff7fffu, query[u].w & 0x7fff7fffu));
                most = max(most & 0xffffu, most >> 16);
                most = __float_as_uint(a.dtype == HOLO_DTYPE_BF16 ? __uint_as_float(most << 16) : half_values(most).x);
                const bool finite = most < 0x7f800000u;
                // 2^e <= most < 2^(e + 1); two factors, since 2^(14 - e) alone may overflow
                const int up = finite && most ? 14 - (most >> 23 ? (int)(most >> 23) - 127 : -118 - __clz((int)most)) : 0;
                const float f0 = power_of_two(up / 2), f1 = power_of_two(up - up / 2);
                const uint64_t first_factor = pair(f0, f0), second_factor = pair(f1, f1);
                auto scaled = [&](uint32_t v) {
                    const float2 x = a.dtype == HOLO_DTYPE_BF16 ? make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)) : half_values(v);
                    const float2 y = unpair(mul2(mul2(pair(x.x, x.y), first_factor), second_factor));
                    return half_pair(y.x, y.y);
                };
#pragma unroll
                for (int u = 0; u < 16; ++u)
                    if (8 * u < dim)
                        *reinterpret_cast<uint4*>(sm + (u >> 3) * TILE_CHUNK + me * 128 + (((u & 7u) ^ (me & 7u)) << 4)) =
                            finite ? make_uint4(scaled(query[u].x), scaled(query[u].y), scaled(query[u].z), scaled(query[u].w)) : make_uint4(0, 0, 0, 0);
                s_row[(np & 1u) * BT_ROWS + me] = finite ? a.scale * LOG2E * power_of_two(-(up / 2)) * power_of_two(-(up - up / 2)) : NAN;
                arrive(bar_q_full);
            }
            // all have what they keep of the plane before
            arrive_at(bar_workers);
            ok = all_wait(bar_workers, np & 1u);
            if (!ok) break;
            const uint32_t top_bits = max(max(most_of[0], most_of[1]), max(most_of[2], most_of[3]));
            const int lift = max((int)(top_bits >> 23) - 126, -100);       // 2^lift is above it
            if (!values && me == 0) s_lift[np & 1u] = lift;
            ++np;
#pragma unroll 1
            for (uint32_t t = s0; t < s1 && ok; ++t, ++nt) {
                const uint32_t stage = nt & 1u;
                // scales of 16 keys in a row, from the lane that has their block. A value scale 2^-60 of the largest and less is as good
                // as none; its keys' weights still count in the rows' sums
                if (!values && me < 8) {
                    float* to = s_scale + (nt & 7u) * 24 + me;
                    const float x = fmaxf(vs, power_of_two(max(lift - 60, -126)));
                    to[0] = ks;
                    to[8] = __log2f(x) + (float)(BT_LIFT - lift);
                    to[16] = __fdiv_rn(1.0f, x) * power_of_two(lift - BT_LIFT);
                }
                ok = nt < 2 || all_wait(bar_empty + 8 * stage, ((nt >> 1) - 1) & 1u);
                if (!ok) break;
                asm volatile("cp.async.wait_group 1;" ::: "memory");      // all but the last request
                if (16 * unit < d) {
                    uint8_t* to = sm + to0 + stage * to_step;
                    const uint8_t* raw = sm + raw0 + stage * raw_step + 16 * unit;
#pragma unroll 4
                    for (uint32_t j = 0; j < 8; ++j) turn(to, 16 * j + sub, *reinterpret_cast<const uint4*>(raw + (16 * j + sub) * d));
                }
                arrive(bar_full + 8 * stage);
                if (!values) load_scales(from);
                from = rows_of(t + 2, ahead);
                ahead = find(t + 3);
                request(raw0 + stage * raw_step, from);
            }
        } while (ok && more(at));
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BT_ISSUER_REGS));
        const uint32_t elected = lane == 0;
        // D = f32, A and B f16, M = 128; S: both operands K-major, N = 128; O: V is N-major, N = vdim
        const uint32_t idesc_s = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
        const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((vdim >> 3) << 17) | ((128u >> 4) << 24);
        const uint64_t first_q = smem_desc(uniform(base), 16, 1024), first_v = smem_desc(uniform(base + o_v), TILE_CHUNK, 1024);
        const uint32_t desc_q = (uint32_t)first_q, desc_k = (uint32_t)smem_desc(uniform(base + o_k), 16, 1024), high_s = (uint32_t)(first_q >> 32);
        const uint32_t desc_v = (uint32_t)first_v, high_v = (uint32_t)(first_v >> 32), tmem_s = uniform(tmem_base), tmem_o = tmem_s + 256, ub = uniform(bars);
        const uint32_t ksteps = dim / 16;
        uint32_t nk = 0, nv = 0, np = 0;
        bool ok = true;
        auto wait = all_wait;
        Plane at = mine.first;
        do {
            uint32_t s0, s1;
            mine.ends_of(at, &s0, &s1);
            const uint32_t tiles = uniform(s1 - s0), keys = uniform(keys_of(at) - s0 * BT_TILE);
            ok = wait(bar_q_full, np & 1u);
            ++np;
            for (uint32_t t = 0; t <= tiles && ok; ++t) {
                // the scores of key tile t, then the product of key tile t - 1, whose softmax runs meanwhile
                if (t < tiles) {
                    ok = wait(bar_k_full + 8 * (nk & 1u), (nk >> 1) & 1u);
                    if (!ok) break;
                    // where the weights of tile t - 2 are, behind the product that reads them (see product_ss)
                    const uint32_t dk = desc_k + (nk & 1u) * (k_bytes >> 4), to = tmem_s + 128 * (nk & 1u);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {
                        const uint32_t off = (k >> 2) * (TILE_CHUNK >> 4) + 2 * (k & 3u);
                        elected_ss(elected & (uint32_t)(k < ksteps), to, desc_q + off, high_s, dk + off, high_s, idesc_s, k != 0);
                    }
                    elected_commit(elected, ub + 192 + 8 * (nk & 1u));
                    arrive_at(ub + 192 + 8 * (nk & 1u));
                    elected_commit(elected, ub + 32 + 8 * (nk & 1u));
                    if (t + 1 == tiles) elected_commit(elected, ub + 8);
                    ++nk;
                }
                if (t > 0) {
                    const uint32_t dv = desc_v + (nv & 1u) * (v_bytes >> 4), steps = min(8u, (keys - (t - 1) * 128 + 15) / 16), weights = tmem_s + 128 * (nv & 1u);
                    ok = wait(bar_v_full + 8 * (nv & 1u), (nv >> 1) & 1u) && wait(bar_pa + 8 * (nv & 1u), (nv >> 1) & 1u);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) elected_ts(elected & (uint32_t)(k < steps), tmem_o, weights + k * 8, dv + 128 * k, high_v, idesc_o, k | (t > 1));
                    ok = wait(bar_pb + 8 * (nv & 1u), (nv >> 1) & 1u);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (uint32_t k = 4; k < 8; ++k) elected_ts(elected & (uint32_t)(k < steps), tmem_o, weights + k * 8, dv + 128 * k, high_v, idesc_o, 1);
                    elected_commit(elected, ub + 64 + 8 * (nv & 1u));
                    ++nv;
                }
            }
        } while (ok && more(at));
    } else if (warp >= 4) {
        // ---------------- softmax (TMEM lane quarter = warp % 4), then the output ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BT_SOFTMAX_REGS));
        const uint32_t quarter = warp & 3u, lanes = (quarter * 32u) << 16, r = quarter * 32 + lane;
        const uint32_t tmem_first = tmem_base + lanes, tmem_o = tmem_base + 256 + lanes;
        uint32_t nt = 0, np = 0, met = 0;
        bool ok = true;
        // the product of a tile is done (every phase of its barrier is waited for in turn)
        auto product_of = [&](uint32_t tile) { return all_wait(bar_v_empty + 8 * (tile & 1u), (tile >> 1) & 1u); };
        Plane at = mine.first;
        do {
            uint32_t s0, s1;
            mine.ends_of(at, &s0, &s1);
            const uint32_t rows = min((uint32_t)BT_ROWS, at.n * group - at.tile * BT_ROWS);
            const uint32_t i = (at.tile * BT_ROWS + min(r, rows - 1)) / group, limit = (uint32_t)max(0, at.length - (int32_t)(at.n - i - 1));
            const uint32_t common = __reduce_min_sync(0xffffffffu, limit);
            // (the queries' barrier may be a plane ahead of this warp: what the workers left for the plane is read behind its first scores)
            float top = -INFINITY, sum = 0.0f, row_scale = 0.0f, back = 0.0f;
            for (uint32_t t = s0; t < s1; ++t, ++nt) {
                ok = all_wait(bar_s + 8 * (nt & 1u), (nt >> 1) & 1u) && (nt < 2 || product_of(nt - 2));
                if (!ok) break;
                const uint32_t tmem_s = tmem_first + 128 * (nt & 1u);
                if (t == s0) {
                    row_scale = s_row[(np & 1u) * BT_ROWS + r];
                    back = power_of_two(s_lift[np & 1u] - BT_LIFT);
                    if (row_scale != row_scale) sum = NAN;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t v[4][32];
#pragma unroll
                for (int x = 0; x < 4; ++x) tmem_ld32_request(tmem_s + 32 * x, v[x]);
                const float* scale = s_scale + (nt & 7u) * 24;
                auto factor = [&](int g) { return fmaxf(row_scale * scale[g], 1e-37f); };      // above 0: -inf stays -inf
                tmem_ld32_wait(v[0]);
#pragma unroll
                for (int x = 1; x < 4; ++x) tmem_ld32_pass(v[x]);
                const uint32_t key0 = t * BT_TILE;
                if (key0 + 128 > common) {
                    const uint32_t hi = limit > key0 ? limit - key0 : 0u;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t seen = hi <= 32u * x ? 0u : hi >= 32u * x + 32 ? 0xffffffffu : (1u << (hi - 32u * x)) - 1u;
#pragma unroll
                        for (int y = 0; y < 32; ++y)
                            if (!(seen >> y & 1u)) v[x][y] = 0xff800000u;
                    }
                }
                float here = -INFINITY;
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    float m = -INFINITY;
#pragma unroll
                    for (int y = 0; y < 16; y += 2) m = fmaxf(fmaxf(m, __uint_as_float(v[g >> 1][16 * (g & 1) + y])), __uint_as_float(v[g >> 1][16 * (g & 1) + y + 1]));
                    here = fmaxf(here, m * factor(g));
                }
                const bool grows = here > top + BT_GROWTH;
                if (__any_sync(0xffffffffu, grows)) {
                    const float f = grows ? ex2(top - here) : 1.0f;      // 0 from the first scores on
                    if (grows) top = here;
                    sum *= f;
                    if (t > s0) {    // O is at rest when the product before is done; the next waits for this warp
                        ok = product_of(nt - 1);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t f2 = pair(f, f);
                        for (uint32_t x = 0; x < vdim; x += 16) {
                            uint32_t o[16];
                            tmem_ld16(tmem_o + x, o);
#pragma unroll
                            for (int y = 0; y < 8; ++y) {
                                const float2 m = unpair(mul2(pair(__uint_as_float(o[2 * y]), __uint_as_float(o[2 * y + 1])), f2));
                                o[2 * y] = __float_as_uint(m.x);
                                o[2 * y + 1] = __float_as_uint(m.y);
                            }
                            tmem_st16(tmem_o + x, o);
                        }
                    }
                }
                float less = top == -INFINITY ? 0.0f : top;
                float by_row = row_scale, by_least = 1e-37f;
                if (__builtin_expect(fabsf(less) >= BT_FAR, 0)) {
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int y = 0; y < 32; ++y) v[x][y] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(v[x][y]), factor(2 * x + (y >> 4))), less));
                    less = by_row = 0.0f;
                    by_least = 1.0f;      // a factor of 1 is left
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t w[16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int g = 2 * x + h;
                        const float term = scale[8 + g] - less, by = fmaxf(by_row * scale[g], by_least);
                        const uint64_t c2 = pair(by, by), d2 = pair(term, term);
                        uint64_t s2 = 0;
#pragma unroll
                        for (int y = 0; y < 8; ++y) {
                            float2 e = unpair(fma2(pair(__uint_as_float(v[x][16 * h + 2 * y]), __uint_as_float(v[x][16 * h + 2 * y + 1])), c2, d2));
                            e.x = ex2(e.x);
                            e.y = ex2(e.y);
                            s2 = add2(s2, pair(e.x, e.y));
                            w[8 * h + y] = half_pair(e.x, e.y);
                        }
                        const float2 q = unpair(s2);
                        sum = fmaf(q.x + q.y, scale[16 + g], sum);
                    }
                    tmem_st16(tmem_s + x * 16, w);
                    if (x & 1) {      // half of the weights: the products of their keys may begin
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"((x == 1 ? bar_pa : bar_pb) + 8 * (nt & 1u)) : "memory");
                    }
                }
            }
            if (!ok) break;
            ok = product_of(nt - 1);
            ++np;
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool begins = at.at >= mine.lo, whole = begins && at.at + at.slabs <= mine.hi;
            float* partial = p.partials + ((uint64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * BT_ROWS * (vdim + 2) + r;
            const float by = whole ? sum == 0.0f ? 0.0f : __fdiv_rn(back, sum) : back;
            auto out_of = [&](uint32_t row) {
                const uint32_t flat = at.tile * BT_ROWS + row;
                return (uint64_t)(at.first_row + flat / group) * a.ld + (uint64_t)(at.head * group + flat % group) * vdim;
            };
            const bool wide = ((uintptr_t)a.out & 15u) == 0 && (a.ld & 7u) == 0;
            const uint64_t out = r < rows ? out_of(r) : 0;
            auto store16 = [&](uint64_t index, const float (&f)[16]) {
                if (wide) {
                    uint32_t w[8];
#pragma unroll
                    for (int y = 0; y < 8; ++y) w[y] = a.dtype == HOLO_DTYPE_F16 ? half_pair(f[2 * y], f[2 * y + 1]) : pack_bf16(f[2 * y], f[2 * y + 1]);
                    uint4* to = reinterpret_cast<uint4*>((uint16_t*)a.out + index);
                    to[0] = make_uint4(w[0], w[1], w[2], w[3]);
                    to[1] = make_uint4(w[4], w[5], w[6], w[7]);
                } else {
#pragma unroll
                    for (int y = 0; y < 16; ++y) seq_store(a.out, index + y, f[y], a.dtype);
                }
            };
            for (uint32_t x = 0; x < vdim; x += 16) {
                uint32_t o[16];
                tmem_ld16(tmem_o + x, o);
                float f[16];
#pragma unroll
                for (int y = 0; y < 16; ++y) f[y] = __uint_as_float(o[y]) * by;
                if (r >= rows) {
                } else if (!whole) {
#pragma unroll
                    for (int y = 0; y < 16; ++y) __stcg(partial + (x + y) * BT_ROWS, f[y]);
                } else {
                    store16(out + x, f);
                }
            }
            __syncwarp();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (!whole) {
                if (r < rows) {
                    __stcg(partial + vdim * BT_ROWS, top);
                    __stcg(partial + (vdim + 1) * BT_ROWS, sum);
                }
                // the plane's CTAs, and its counter: that of the CTA it begins in
                const uint32_t from_cta = mine.first_cta(at), count = mine.cta_count(at);
                arrive_at(bar_rows);
                ok = all_wait(bar_rows, met++ & 1u);
                if (!ok) break;
                if (r == 0) {
                    uint32_t n;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(n) : "l"(p.arrivals + from_cta) : "memory");
                    *s_last = n + 1 == count;
                    if (n + 1 == count) p.arrivals[from_cta] = 0;
                }
                arrive_at(bar_rows);
                ok = all_wait(bar_rows, met++ & 1u);
                if (!ok) break;
                if (*reinterpret_cast<volatile uint32_t*>(s_last)) {
                    // A thread the weights of its row's parts, which take the place of their maxima; then the four warps take 16 columns of
                    // 32 rows in turn, four parts' values on their way at a time
                    const uint32_t step = 2 * BT_ROWS * (vdim + 2), own = BT_ROWS * (vdim + 2);
                    float* const first = p.partials + (uint64_t)from_cta * step;
                    auto part = [&](uint32_t w) { return first + (uint64_t)w * step + (w == 0 ? own : 0u); };
                    if (r < rows) {
                        float m = -INFINITY, l = 0.0f;
#pragma unroll 8
                        for (uint32_t w = 0; w < count; ++w) m = fmaxf(m, __ldcg(part(w) + vdim * BT_ROWS + r));
#pragma unroll 4
                        for (uint32_t w = 0; w < count; ++w) {
                            float* const of = part(w) + vdim * BT_ROWS + r;
                            const float lw = __ldcg(of + BT_ROWS), f = lw == 0.0f ? 0.0f : ex2(__ldcg(of) - m);      // NaN is not 0
                            l = fmaf(f, lw, l);
                            __stcg(of, f);
                        }
                        __stcg(part(0) + (vdim + 1) * BT_ROWS + r, l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l));
                    }
                    arrive_at(bar_rows);
                    ok = all_wait(bar_rows, met++ & 1u);
                    if (!ok) break;
                    const uint32_t chunks = vdim / 16, tasks = (rows + 31) / 32 * chunks;
#pragma unroll 1
                    for (uint32_t task = quarter; task < tasks; task += 4) {
                        const uint32_t row = task / chunks * 32 + lane, x = task % chunks * 16;
                        if (row >= rows) continue;
                        float acc[16];
#pragma unroll
                        for (int y = 0; y < 16; ++y) acc[y] = 0.0f;
#pragma unroll 4
                        for (uint32_t w = 0; w < count; ++w) {
                            const float *from = part(w) + row, f = __ldcg(from + vdim * BT_ROWS);
#pragma unroll
                            for (int y = 0; y < 16; ++y) acc[y] = fmaf(f, __ldcg(from + (x + y) * BT_ROWS), acc[y]);
                        }
                        const float inv = __ldcg(part(0) + (vdim + 1) * BT_ROWS + row);
#pragma unroll
                        for (int y = 0; y < 16; ++y) acc[y] *= inv;
                        store16(out_of(row) + x, acc);
                    }
                    __syncwarp();
                }
            }
        } while (more(at));
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BT_ISSUER_REGS));
    }
    // everyone meets here, whatever happened above, so that TMEM is always released
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

int32_t launch_block_tile(holo_b200_ctx* ctx, const BlockTileParams& p) {
    const uint32_t smem = 1024 + 3 * p.k_chunks * TILE_CHUNK + 2 * p.v_chunks * TILE_CHUNK + 2 * BT_TILE * (p.a.c.dim + p.a.c.vdim) + 256 + 2 * BT_ROWS * 4 + 8 * 24 * 4;
    static thread_local int configured_device = -1;
    if (configured_device != ctx->device) {
        HOLO_CUDA(cudaFuncSetAttribute(block_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ctx->smem_optin));
        // the roles' registers come out of the launch's: a sum above them would be waited for without end
        cudaFuncAttributes built;
        HOLO_CUDA(cudaFuncGetAttributes(&built, block_tile_kernel));
        if (built.numRegs * BT_WARPS * 32 < 128 * (BT_ISSUER_REGS + BT_SOFTMAX_REGS + 2 * BT_WORKER_REGS))
            return holo_fail(HOLO_ERR_DISPATCH, "dispatch failed: block_cache_attention was built with %d registers a thread, too few to share out", built.numRegs);
        configured_device = ctx->device;
    }
    HOLO_CUDA(holo_launch_kernel(ctx, block_tile_kernel, dim3((uint32_t)ctx->sm_count), dim3(BT_WARPS * 32), smem, 1, p));
    ctx->launches++;
    return HOLO_OK;
}

}  // namespace

int32_t holo_try_block_tile(holo_b200_ctx* ctx, const HoloBlockAttnArgs& a, bool* taken) {
    *taken = false;
    const HoloBlockCache& c = a.c;
    const uint32_t group = a.heads / c.kv_heads;
    if (a.dtype == HOLO_DTYPE_F32 || c.block_rows % 16 != 0) return HOLO_OK;
    if (c.dim % 16 != 0 || c.vdim % 16 != 0 || c.dim > 128 || c.vdim > 128 || (((uintptr_t)c.k_codes | (uintptr_t)c.v_codes) & 15u) != 0) return HOLO_OK;
    // where a sequence has more rows of a head than the few-row kernel takes in two passes over the cache: three take 78 us against 56 here for
    // 8 sequences of 4096 positions (137 against 101 for 32 of 2048, 28 against 28 for one of 4096), two 63 (101, 22)
    if ((uint64_t)c.rows * group <= 16ull * c.sequences) return HOLO_OK;
    // tiles of the whole list of 32 bits
    const uint64_t tiles = ((uint64_t)c.rows * group / BT_ROWS + c.sequences) * c.kv_heads;
    if ((uint64_t)c.rows * a.heads > 0x7fffffffull || tiles > 0x7fffffffull / (((uint64_t)c.table_ld * c.block_rows + BT_TILE - 1) / BT_TILE + BT_PLANE)) return HOLO_OK;
    if ((uint64_t)c.blocks * c.kv_heads * c.block_rows >= 0xffffffffull) return HOLO_OK;      // row numbers of 32 bits
    HOLO_TRY(holo_block_row_partials(ctx));
    *taken = true;
    BlockTileParams p = {};
    p.a = a;
    p.partials = ctx->block_row_partials;
    p.arrivals = ctx->attn_arrivals;
    p.group = group;
    p.k_chunks = (c.dim + 63) / 64;
    p.v_chunks = (c.vdim + 63) / 64;
    p.br_shift = -1;
    for (int s = 0; s <= 10; ++s)
        if (c.block_rows == 1u << s) p.br_shift = s;
    return launch_block_tile(ctx, p);
}
