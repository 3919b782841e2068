// Attention of packed 16-bit sequences (the PackedAttention call) on tcgen05, for dims in steps of 16 up to 128.
//
// Query tiles are 128 rows of the packed rows, whatever sequences they belong to: a row sees the keys [begin, end) of its own sequence, and
// a tile walks the keys from its first row's sequence on in tiles of 128. So the host needs no lengths, and short sequences share
// tiles. A CTA takes one or two neighbouring query tiles of a head after another (persistent: the next tiles' loads and scores run
// while the last ones are stored):
//   warp 0     TMA producer: the query tiles, K and V tiles through rings of two
//   warps 1, 2 tcgen05.mma issuers, one for each query tile: S = Q K^T, then O += P V with P read from TMEM. A wait or a commit costs an
//              issuer 150 to 300 cycles while the tensor core has the shared memory; two of them hide each other's (8192 rows: 353 -> 311 us)
//   warps 4-11 softmax, one group of four warps per query tile, one thread per row: running maximum, exponentials, row sum;
//              a row's O is rescaled in TMEM only when its maximum grows by more than 2^GROWTH
// The weights are rounded to the operands' type (by up to 2^-8 of a weight in bf16, 2^-11 in f16), sums stay f32: a rounded weight moves
// a result by as much as the result's own rounding does, and a second term for the remainder would be half as many products again. Errors
// against 64 bits are 1.1 to 1.4 times those with f32 weights (8192 rows of bf16 0.0020 against 0.0016 of a result, documents of f16 0.00028
// against 0.00021).
// TMEM (512 columns): S at 0 and 128, overwritten by its weights, O at 256 and 384.
// Bound: two products per score on the tensor core (1024 cycles a 128 x 128 tile at dim 128), and 1024 cycles of ex2 beside it. Measured (32
// heads over 8 of dim 128, 8192 rows of seven sequences): 275 us, 0.41 of the burst rate of a large bf16 product; a pair of tiles takes
// some 4500 cycles, of which a thread's softmax is 3200 and the way of its weights to the next scores the rest.
//
// A weight of zero times an infinite or NaN value is NaN, so a value that is not finite spoils its column in every row of the tile. A
// row that ends with results that are not finite is computed again from memory by its own thread (redo_rows), only the keys it sees.
#include "attention_issue.cuh"
#include "sequences.cuh"

namespace {

constexpr int PT_WARPS = 12;
constexpr uint32_t PT_ITEMS = 128;       // items of a CTA that are worked out beforehand
constexpr uint32_t PT_SORTED = 256;      // pairs that are put in the order of their work
constexpr float PT_GROWTH = 8.0f;
constexpr uint32_t PT_STARTS = 4096;      // starts kept in shared memory; more are read where they are

struct PackedTileParams {
    HoloPackedArgs a;
    float to_log2;
    uint32_t nq, k_chunks, v_chunks, pairs, items;
};

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) { return F16 ? pack_half(lo, hi) : pack_bf16(lo, hi); }

// An item: the query tiles of a pair and a head. Tile q walks the key tiles [from[q], to[q]) of 128 keys each, counted from `anchor`;
// left[q]: keys from there to its last one. Pairs come in the order of their work, the most first (many pairs: the last rows
// first, which have the most keys in a causal sequence), and CTAs take items back and forth: within 5 % of always giving the next
// item to the CTA with the least (8192 rows of seven sequences, 1024 items: 104.5 key tiles at most for 99.5 on average; as the rows come 116.5).
struct PackedItem {
    uint32_t row0, head, anchor, tiles, from[2], to[2], left[2];
};

// Keys that some row of a query tile sees, [begin, end); the same for every thread that asks.
struct KeyRange {
    uint32_t begin, end;
};
__device__ __forceinline__ KeyRange keys_of_tile(const HoloPackedArgs& a, const int32_t* starts, uint32_t row0) {
    KeyRange r = {0, 0};
    const int64_t first = max((int64_t)row0, (int64_t)starts[0]), last = min(min((int64_t)row0 + 128, (int64_t)a.rows), (int64_t)starts[a.sequences]) - 1;
    if (first < 0 || last < first) return r;
    const int s0 = find_sequence(starts, a.sequences, first), s1 = find_sequence(starts, a.sequences, last);
    if (s0 < 0 || s0 >= (int)a.sequences || s1 < 0 || s1 >= (int)a.sequences) return r;
    r.begin = (uint32_t)max(starts[s0], 0);
    r.end = a.causal ? (uint32_t)last + 1 : (uint32_t)min((int64_t)starts[s1 + 1], (int64_t)a.rows);
    if (r.end < r.begin || r.begin > first) r.begin = r.end = 0;      // starts that do not ascend
    return r;
}

// Rows of this warp (one a thread, `mine`: it is to be done) over the keys [begin, end), from memory, in one pass with a running maximum of
// its own. All lanes take the same key, so that its elements are one transaction. A value that is not finite has
// the rows of all tiles that read it done again: where 8 heads x 2048 rows of dim 128 read one, 6.8 ms against 40 us.
template <bool F16>
__device__ __noinline__ void redo_rows(const PackedTileParams& p, uint32_t row, uint32_t head, uint32_t begin, uint32_t end, bool mine) {
    const HoloPackedArgs& a = p.a;
    const uint32_t g = head / (a.heads / a.kv_heads), lo = __reduce_min_sync(0xffffffffu, mine ? begin : 0xffffffffu), hi = __reduce_max_sync(0xffffffffu, mine ? end : 0u);
    const uint4* q = reinterpret_cast<const uint4*>((const uint16_t*)a.q + (uint64_t)(mine ? row : 0u) * a.q_ld + (uint64_t)head * a.dim);
    auto wide = [](uint32_t v) { return F16 ? __half22float2(*reinterpret_cast<const __half2*>(&v)) : make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); };
    float acc[128], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int c = 0; c < 128; ++c) acc[c] = 0.0f;
#pragma unroll 1
    for (uint32_t j = lo; j < hi; ++j) {
        if (!mine || j < begin || j >= end) continue;
        const uint4* k = reinterpret_cast<const uint4*>((const uint16_t*)a.k + (uint64_t)j * a.k_ld + (uint64_t)g * a.dim);
        float s = 0.0f;
#pragma unroll 1
        for (uint32_t d = 0; d < a.dim / 8; ++d) {
            const uint4 x = q[d], y = k[d];
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 u = wide(xs[e]), w = wide(ys[e]);
                s = fmaf(u.y, w.y, fmaf(u.x, w.x, s));
            }
        }
        s = __fmul_rn(s, p.to_log2);      // not fused with the subtraction below: a large exponent's rounding cancels
        if (s == -INFINITY) continue;
        if (s > top) {
            const float f = exp2f(__fsub_rn(top, s));
            top = s;
            sum *= f;
#pragma unroll
            for (int c = 0; c < 128; ++c) acc[c] = f == 0.0f ? 0.0f : acc[c] * f;
        }
        const float w = exp2f(__fsub_rn(s, top));
        sum += w;
        const uint4* v = reinterpret_cast<const uint4*>((const uint16_t*)a.v + (uint64_t)j * a.v_ld + (uint64_t)g * a.vdim);
#pragma unroll
        for (int c = 0; c < 16; ++c)
            if (8 * c < a.vdim) {
                const uint4 y = v[c];
                const uint32_t ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 u = wide(ys[e]);
                    acc[8 * c + 2 * e] = fmaf(w, u.x, acc[8 * c + 2 * e]);
                    acc[8 * c + 2 * e + 1] = fmaf(w, u.y, acc[8 * c + 2 * e + 1]);
                }
            }
    }
    __syncwarp();
    if (!mine) return;
    uint32_t* out = reinterpret_cast<uint32_t*>((uint16_t*)a.out + (uint64_t)row * a.ld + (uint64_t)head * a.vdim);
#pragma unroll
    for (int c = 0; c < 64; ++c)
        if (2 * c < a.vdim) out[c] = sum == 0.0f ? 0u : pack16<F16>(__fdiv_rn(acc[2 * c], sum), __fdiv_rn(acc[2 * c + 1], sum));
}

constexpr float PT_WILD = 0x1p22f;     // from here on a fused exponent of the largest score is off by whole units

// KS: dim / 16 where that is 4 or 8, else 0
template <bool F16, int KS>
__global__ void __launch_bounds__(PT_WARPS * 32, 1)
packed_tile_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ PackedTileParams p) {
    // f16 weights are kept 2^7 larger, so that fewer of them fall below f16's smallest steps (2^GROWTH more still fits)
    constexpr float LIFT = F16 ? 7.0f : 0.0f;
    extern __shared__ uint8_t smem_raw[];
    const HoloPackedArgs& a = p.a;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - raw);
    const uint32_t k_bytes = p.k_chunks * TILE_CHUNK, v_bytes = p.v_chunks * TILE_CHUNK;
    const uint32_t s_q = base, s_k = s_q + p.nq * k_bytes, s_v = s_k + 2 * k_bytes, bars = s_v + 2 * v_bytes;
    const uint32_t bar_q_full = bars, bar_q_empty = bars + 8, bar_k_full = bars + 16, bar_k_empty = bars + 32, bar_v_full = bars + 48, bar_v_empty = bars + 64,
                   bar_s = bars + 80, bar_pa = bars + 96, bar_pb = bars + 112, bar_pv = bars + 128;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(sm + (bars - base) + 160);
    volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(sm + (bars - base) + 164);
    PackedItem* s_items = reinterpret_cast<PackedItem*>(sm + (bars - base) + 256);
    uint32_t* s_work = reinterpret_cast<uint32_t*>(sm + (bars - base) + 256 + PT_ITEMS * sizeof(PackedItem));
    uint16_t* s_order = reinterpret_cast<uint16_t*>(s_work + PT_SORTED);
    int32_t* s_starts = reinterpret_cast<int32_t*>(s_order + PT_SORTED);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(bar_q_full, 1);
        mbar_init(bar_q_empty, p.nq);         // one arrival per issuer

        for (int s = 0; s < 2; ++s) {
            mbar_init(bar_k_full + 8 * s, 1);
            mbar_init(bar_k_empty + 8 * s, p.nq);
            mbar_init(bar_v_full + 8 * s, 1);
            mbar_init(bar_v_empty + 8 * s, p.nq);
            mbar_init(bar_s + 8 * s, 1);
            mbar_init(bar_pa + 8 * s, 4);     // one arrival per softmax warp
            mbar_init(bar_pb + 8 * s, 4);
            mbar_init(bar_pv + 8 * s, 1);
        }
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    holo_pdl_wait();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const bool kept = a.sequences < PT_STARTS;
    if (kept)
        for (uint32_t i = threadIdx.x; i <= a.sequences; i += PT_WARPS * 32) s_starts[i] = a.starts[i];
    if (blockIdx.x == 0) check_sequences(a.starts, nullptr, a.sequences, a.rows, 0, a.status);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    holo_pdl_trigger();
    const uint32_t tmem_base = *s_tmem;
    const int32_t* starts = kept ? s_starts : a.starts;

    // (the order does not matter where every item has a CTA of its own)
    const bool sorted = p.pairs <= PT_SORTED && p.items > gridDim.x;
    if (sorted) {
        uint32_t mine = 0;
        if (threadIdx.x < p.pairs) {
            for (uint32_t q = 0; q < p.nq; ++q) {
                const KeyRange r = keys_of_tile(a, starts, (threadIdx.x * p.nq + q) * 128);
                mine = max(mine, r.end - r.begin);
            }
            s_work[threadIdx.x] = mine;
        }
        __syncthreads();
        if (threadIdx.x < p.pairs) {
            uint32_t rank = 0;
            for (uint32_t j = 0; j < p.pairs; ++j) rank += s_work[j] > mine || (s_work[j] == mine && j < threadIdx.x);
            s_order[rank] = (uint16_t)threadIdx.x;
        }
        __syncthreads();
    }
    const uint32_t rounds = (p.items + gridDim.x - 1) / gridDim.x;
    // the item of this CTA's round, or one past the last
    auto number_of = [&](uint32_t round) { return round * gridDim.x + (round & 1u ? gridDim.x - 1 - blockIdx.x : blockIdx.x); };
    auto make_item = [&](uint32_t i) {
        PackedItem it;
        it.head = i % a.heads;
        it.row0 = (sorted ? s_order[i / a.heads] : p.pairs - 1 - i / a.heads) * p.nq * 128;
        KeyRange r[2];
        r[0] = keys_of_tile(a, starts, it.row0);
        r[1] = p.nq == 2 ? keys_of_tile(a, starts, it.row0 + 128) : KeyRange{0, 0};
        it.anchor = r[0].end > r[0].begin ? r[0].begin : r[1].begin;
        it.tiles = 0;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const bool any = r[q].end > r[q].begin && r[q].begin >= it.anchor;
            it.from[q] = any ? (r[q].begin - it.anchor) / 128 : 0u;
            it.to[q] = any ? (r[q].end - it.anchor + 127) / 128 : 0u;
            it.left[q] = r[q].end - it.anchor;
            it.tiles = max(it.tiles, it.to[q]);
        }
        return it;
    };
    // a thread an item
    if (threadIdx.x < PT_ITEMS && threadIdx.x < rounds) {
        const uint32_t i = number_of(threadIdx.x);
        if (i < p.items) s_items[threadIdx.x] = make_item(i);
        else s_items[threadIdx.x].tiles = s_items[threadIdx.x].from[0] = s_items[threadIdx.x].to[0] = s_items[threadIdx.x].from[1] = s_items[threadIdx.x].to[1] = 0;
    }
    __syncthreads();
    auto item_of = [&](uint32_t round) {
        if (round < PT_ITEMS) return s_items[round];
        const uint32_t i = number_of(round);
        if (i < p.items) return make_item(i);
        return PackedItem{};
    };

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            uint32_t nq = 0, nk = 0, nv = 0;       // copies of each kind so far
            bool ok = true;
            for (uint32_t i = 0; i < rounds && ok; ++i) {
                const PackedItem it = item_of(i);
                if (it.tiles == 0) continue;
                const int g = (int)(it.head / (a.heads / a.kv_heads));
                ok = nq == 0 || long_wait(bar_q_empty, (nq - 1) & 1u, s_abort, a.status);
                if (!ok) break;
                mbar_arrive_expect_tx(bar_q_full, p.nq * k_bytes);
                for (uint32_t q = 0; q < p.nq; ++q)
                    for (uint32_t c = 0; c < p.k_chunks; ++c)
                        tma_load_3d(s_q + q * k_bytes + c * TILE_CHUNK, &map_q, (int)(64 * c), (int)it.head, (int)(it.row0 + q * 128), bar_q_full);
                ++nq;
                for (uint32_t t = 0; t < it.tiles; ++t) {
                    ok = nk < 2 || long_wait(bar_k_empty + 8 * (nk & 1u), ((nk >> 1) - 1) & 1u, s_abort, a.status);
                    if (!ok) break;
                    mbar_arrive_expect_tx(bar_k_full + 8 * (nk & 1u), k_bytes);
                    for (uint32_t c = 0; c < p.k_chunks; ++c)
                        tma_load_3d(s_k + (nk & 1u) * k_bytes + c * TILE_CHUNK, &map_k, (int)(64 * c), g, (int)(it.anchor + t * 128), bar_k_full + 8 * (nk & 1u));
                    ++nk;
                    ok = nv < 2 || long_wait(bar_v_empty + 8 * (nv & 1u), ((nv >> 1) - 1) & 1u, s_abort, a.status);
                    if (!ok) break;
                    mbar_arrive_expect_tx(bar_v_full + 8 * (nv & 1u), v_bytes);
                    for (uint32_t c = 0; c < p.v_chunks; ++c)
                        tma_load_3d(s_v + (nv & 1u) * v_bytes + c * TILE_CHUNK, &map_v, (int)(64 * c), g, (int)(it.anchor + t * 128), bar_v_full + 8 * (nv & 1u));
                    ++nv;
                }
            }
            if (!ok) {
                // nothing may still be on its way into this CTA's shared memory when it ends
                for (uint32_t x = 0; nq && x < WAIT_LIMIT && !mbar_try_wait(bar_q_full, (nq - 1) & 1u); ++x) __nanosleep(64);
                for (uint32_t t = nk > 2 ? nk - 2 : 0; t < nk; ++t)
                    for (uint32_t x = 0; x < WAIT_LIMIT && !mbar_try_wait(bar_k_full + 8 * (t & 1), (t >> 1) & 1); ++x) __nanosleep(64);
                for (uint32_t t = nv > 2 ? nv - 2 : 0; t < nv; ++t)
                    for (uint32_t x = 0; x < WAIT_LIMIT && !mbar_try_wait(bar_v_full + 8 * (t & 1), (t >> 1) & 1); ++x) __nanosleep(64);
            }
        }
    } else if (warp <= 2) {
        // ---------------- MMA issuers ----------------
        if (warp <= p.nq) {
            const uint32_t q = uniform(warp - 1), elected = lane == 0;
            // D = f32, A and B of the call's type, M = 128; S: both operands K-major, N = 128; O: V is N-major, N = vdim
            const uint32_t type = F16 ? 0u : (1u << 7) | (1u << 10);
            const uint32_t idesc_s = (1u << 4) | type | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            const uint32_t idesc_o = (1u << 4) | type | (1u << 16) | ((a.vdim >> 3) << 17) | ((128u >> 4) << 24);
            const uint64_t first_q = smem_desc(uniform(s_q + q * k_bytes), 16, 1024), first_v = smem_desc(uniform(s_v), TILE_CHUNK, 1024);
            const uint32_t desc_q = (uint32_t)first_q, desc_k = (uint32_t)smem_desc(uniform(s_k), 16, 1024), high_s = (uint32_t)(first_q >> 32);
            const uint32_t desc_v = (uint32_t)first_v, high_v = (uint32_t)(first_v >> 32), tmem_s = uniform(tmem_base + q * 128), tmem_o = tmem_s + 256, ub = uniform(bars);
            const uint32_t u_s = ub + 80 + 8 * q, u_pv = ub + 128 + 8 * q, u_ke = ub + 32, u_ve = ub + 64, u_qe = ub + 8;
            const uint32_t ksteps = KS ? KS : a.dim / 16;
            uint32_t nq = 0, nk = 0, nv = 0, np = 0;
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, long_wait(bar, parity, s_abort, a.status)); };
            for (uint32_t i = 0; i < rounds && ok; ++i) {
                const PackedItem it = item_of(i);
                const uint32_t from = uniform(it.from[q]), to = uniform(it.to[q]), left = uniform(it.left[q]), tiles = uniform(it.tiles);
                if (tiles == 0) continue;
                ok = wait(bar_q_full, nq & 1u);
                ++nq;
                for (uint32_t t = 0; t <= tiles && ok; ++t) {
                    // the product of key tile t - 1, the scores of key tile t
                    if (t > 0) {
                        ok = wait(bar_v_full + 8 * (nv & 1u), (nv >> 1) & 1u);
                        if (ok && t > from && t <= to) {
                            const uint32_t dv = desc_v + (nv & 1u) * (v_bytes >> 4), more = t - 1 > from;
                            // keys past the last one any row of the tile sees have no weight: whole steps of them are left out
                            const uint32_t steps = min(8u, (left - (t - 1) * 128 + 15) / 16);
                            ok = wait(bar_pa + 8 * q, np & 1u);
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                            for (uint32_t k = 0; k < 4; ++k) elected_ts(elected & (uint32_t)(k < steps), tmem_o, tmem_s + k * 8, dv + 128 * k, high_v, idesc_o, k | more);
                            ok = wait(bar_pb + 8 * q, np & 1u);
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                            for (uint32_t k = 4; k < 8; ++k) elected_ts(elected & (uint32_t)(k < steps), tmem_o, tmem_s + k * 8, dv + 128 * k, high_v, idesc_o, 1);
                            ++np;
                            if (t == to) elected_commit(elected, u_pv);
                        }
                    }
                    if (ok && t < tiles) {
                        ok = wait(bar_k_full + 8 * (nk & 1u), (nk >> 1) & 1u);
                        if (ok && t >= from && t < to) {
                            // the next scores go where the weights are, behind the product that reads them (see product_ss)
                            const uint32_t dk = desc_k + (nk & 1u) * (k_bytes >> 4);
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                            for (uint32_t k = 0; k < (KS ? KS : 8); ++k) {
                                const uint32_t off = (k >> 2) * (TILE_CHUNK >> 4) + 2 * (k & 3u);
                                elected_ss(KS ? elected : elected & (uint32_t)(k < ksteps), tmem_s, desc_q + off, high_s, dk + off, high_s, idesc_s, k != 0);
                            }
                            elected_commit(elected, u_s);
                        }
                    }
                    if (!ok) break;
                    if (t > 0) {
                        elected_commit(elected, u_ve + 8 * (nv & 1u));
                        ++nv;
                    }
                    if (t < tiles) {
                        elected_commit(elected, u_ke + 8 * (nk & 1u));
                        ++nk;
                        if (t + 1 == tiles) elected_commit(elected, u_qe);
                    }
                }
            }
        }
    } else if (warp >= 4) {
        // ---------------- softmax (TMEM lane quarter = warp % 4), then the output ----------------
        const uint32_t q = (warp - 4) >> 2, quarter = warp & 3u, lanes = (quarter * 32u) << 16;
        const uint32_t tmem_s = tmem_base + q * 128 + lanes, tmem_o = tmem_base + 256 + q * 128 + lanes;
        const uint64_t c2 = pair(p.to_log2, p.to_log2);
        uint32_t ns = 0, ndone = 0;
        bool ok = true;
        for (uint32_t i = 0; i < rounds && ok; ++i) {
            const PackedItem it = item_of(i);
            const uint32_t from = q ? it.from[1] : it.from[0], to = q ? it.to[1] : it.to[0];
            if (from == to) continue;
            const uint32_t row = it.row0 + q * 128 + quarter * 32 + lane;
            uint32_t begin = 0, end = 0, which;
            const bool mine = row < a.rows && sequence_of(starts, a.sequences, a.rows, row, &begin, &end, &which);
            if (mine && a.causal) end = row + 1;
            // keys that all rows of the warp see; rows of no sequence do not count
            const uint32_t all_from = __reduce_max_sync(0xffffffffu, mine ? begin : 0u), all_to = __reduce_min_sync(0xffffffffu, mine ? end : 0xffffffffu);
            float top = -INFINITY, sum = 0.0f;
            for (uint32_t t = from; t < to; ++t, ++ns) {
                ok = long_wait(bar_s + 8 * q, ns & 1u, s_abort, a.status) && !*s_abort;
                ok = __all_sync(0xffffffffu, ok);   // the TMEM accesses below are whole-warp instructions
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t v[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32_request(tmem_s + 32 * c, v[c]);
                tmem_ld32_wait(v[0]);
#pragma unroll
                for (int c = 1; c < 4; ++c) tmem_ld32_pass(v[c]);
                const uint32_t key0 = it.anchor + t * 128;
                if (key0 < all_from || key0 + 128 > all_to) {
                    // of the tile's keys this row sees [lo, hi): 32 bits a request
                    const uint32_t lo = begin > key0 ? begin - key0 : 0u, hi = end > key0 ? end - key0 : 0u;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t from_lo = lo <= 32u * c ? 0xffffffffu : lo >= 32u * c + 32 ? 0u : 0xffffffffu << (lo - 32u * c);
                        const uint32_t to_hi = hi <= 32u * c ? 0u : hi >= 32u * c + 32 ? 0xffffffffu : (1u << (hi - 32u * c)) - 1u;
                        const uint32_t sees = from_lo & to_hi;
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (!(sees >> x & 1u)) v[c][x] = 0xff800000u;
                    }
                }
                float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int x = 0; x < 32; x += 2)
#pragma unroll
                    for (int c = 0; c < 4; ++c) most[c] = fmaxf(fmaxf(most[c], __uint_as_float(v[c][x])), __uint_as_float(v[c][x + 1]));
                const float here = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * p.to_log2;
                const bool grows = here > top + PT_GROWTH;
                if (__any_sync(0xffffffffu, grows)) {
                    const float f = grows ? ex2(top - here) : 1.0f;      // 0 from the first scores on
                    if (grows) top = here;
                    sum *= f;
                    if (t > from) {    // the barrier of this tile's scores stands for the product before them too: O is at rest
                        const uint64_t f2 = pair(f, f);
                        for (uint32_t c = 0; c < a.vdim; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(tmem_o + c, o);
#pragma unroll
                            for (int x = 0; x < 8; ++x) {
                                const float2 m = unpair(mul2(pair(__uint_as_float(o[2 * x]), __uint_as_float(o[2 * x + 1])), f2));
                                o[2 * x] = __float_as_uint(m.x);
                                o[2 * x + 1] = __float_as_uint(m.y);
                            }
                            tmem_st16(tmem_o + c, o);
                        }
                    }
                }
                const float less = (top == -INFINITY ? 0.0f : top) - LIFT;
                const uint64_t less2 = pair(-less, -less);
                uint64_t s2[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        float2 e = unpair(fma2(pair(__uint_as_float(v[c][2 * x]), __uint_as_float(v[c][2 * x + 1])), c2, less2));
                        e.x = ex2(e.x);
                        e.y = ex2(e.y);
                        s2[x & 1] = add2(s2[x & 1], pair(e.x, e.y));
                        w[x] = pack16<F16>(e.x, e.y);
                    }
                    tmem_st16(tmem_s + c * 16, w);
                    if (c & 1) {      // half of the weights: the products of their keys may begin
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"((c == 1 ? bar_pa : bar_pb) + 8 * q) : "memory");
                    }
                }
                const float2 s0 = unpair(add2(s2[0], s2[1]));
                sum += s0.x + s0.y;
            }
            ok = ok && long_wait(bar_pv + 8 * q, ndone & 1u, s_abort, a.status) && !*s_abort;
            ++ndone;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float inv = __fdiv_rn(1.0f, sum);
            // every score -inf (a sum of 0 under a finite maximum: exponents of far scores were off, which the row is done again for)
            const bool nothing = sum == 0.0f && top == -INFINITY;
            uint16_t* out = (uint16_t*)a.out + (uint64_t)row * a.ld + (uint64_t)it.head * a.vdim;
            bool finite = true;
            for (uint32_t c = 0; c < a.vdim; c += 16) {
                uint32_t o[16], w[8];
                tmem_ld16(tmem_o + c, o);
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const float lo = __uint_as_float(o[2 * x]) * inv, hi = __uint_as_float(o[2 * x + 1]) * inv;
                    finite = finite && isfinite(lo) && isfinite(hi);
                    w[x] = nothing ? 0u : pack16<F16>(lo, hi);
                }
                if (mine) {
                    reinterpret_cast<uint4*>(out + c)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                    reinterpret_cast<uint4*>(out + c)[1] = make_uint4(w[4], w[5], w[6], w[7]);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            // a row whose maximum is +inf is NaN throughout already
            const bool again = mine && !nothing && fabsf(top) < INFINITY && (!finite || !isfinite(inv) || fabsf(top) >= PT_WILD);
            if (__any_sync(0xffffffffu, again)) redo_rows<F16>(p, row, it.head, begin, end, again);
        }
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

// [rows, heads * width] at pitch ld as (column, head, row), 128 rows of 64 columns a box
int32_t make_packed_map(CUtensorMap* map, const void* ptr, uint32_t width, uint32_t heads, uint32_t rows, uint32_t ld) {
    cuuint64_t dims[3] = {width, heads, rows};
    cuuint64_t strides[2] = {(cuuint64_t)width * 2, (cuuint64_t)ld * 2};
    cuuint32_t box[3] = {64, 1, 128};
    cuuint32_t es[3] = {1, 1, 1};
    const CUresult r = encode_tiled_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return holo_fail(HOLO_ERR_DISPATCH, "dispatch failed: cuTensorMapEncodeTiled (packed attention) returned %d", (int)r);
    return HOLO_OK;
}

template <bool F16, int KS>
int32_t launch_packed_tile(holo_b200_ctx* ctx, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PackedTileParams& p, uint32_t grid, uint32_t smem) {
    static thread_local int configured_device = -1;
    if (configured_device != ctx->device) {
        HOLO_CUDA(cudaFuncSetAttribute(packed_tile_kernel<F16, KS>, cudaFuncAttributeMaxDynamicSharedMemorySize, ctx->smem_optin));
        configured_device = ctx->device;
    }
    HOLO_CUDA(holo_launch_kernel(ctx, packed_tile_kernel<F16, KS>, dim3(grid), dim3(PT_WARPS * 32), smem, 1, mq, mk, mv, p));
    ctx->launches++;
    return HOLO_OK;
}

}  // namespace

int32_t holo_try_packed_tile(holo_b200_ctx* ctx, const HoloPackedArgs& a, bool* taken) {
    *taken = false;
    if (a.dtype == HOLO_DTYPE_F32 || a.dim % 16 != 0 || a.vdim % 16 != 0 || a.dim > 128 || a.vdim > 128) return HOLO_OK;
    // TMA and 16-byte stores want aligned rows
    if ((((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15u) != 0 || ((a.q_ld | a.k_ld | a.v_ld | a.ld) & 7u) != 0) return HOLO_OK;
    const uint64_t tiles = ((uint64_t)a.rows + 127) / 128, pairs = (tiles + 1) / 2;
    if (tiles * a.heads > 0x7fffffffull || encode_tiled_fn() == nullptr) return HOLO_OK;
    PackedTileParams p = {};
    p.a = a;
    p.to_log2 = a.scale * LOG2E;
    p.k_chunks = (a.dim + 63) / 64;
    p.v_chunks = (a.vdim + 63) / 64;
    // two query tiles a CTA share what is read of K and V and hide each other's softmax, where that still gives every SM a CTA
    p.nq = tiles > 1 && pairs * a.heads >= (uint64_t)ctx->sm_count ? 2 : 1;
    p.pairs = (uint32_t)(p.nq == 2 ? pairs : tiles);
    p.items = p.pairs * a.heads;
    CUtensorMap mq, mk, mv;
    HOLO_TRY(make_packed_map(&mq, a.q, a.dim, a.heads, a.rows, a.q_ld));
    HOLO_TRY(make_packed_map(&mk, a.k, a.dim, a.kv_heads, a.rows, a.k_ld));
    HOLO_TRY(make_packed_map(&mv, a.v, a.vdim, a.kv_heads, a.rows, a.v_ld));
    const uint32_t kept = a.sequences < PT_STARTS ? 4 * (a.sequences + 1) : 0;
    const uint32_t smem = 1024 + (p.nq + 2) * p.k_chunks * TILE_CHUNK + 2 * p.v_chunks * TILE_CHUNK + 256 + PT_ITEMS * (uint32_t)sizeof(PackedItem) + 6 * PT_SORTED + ((kept + 15u) & ~15u);
    const uint32_t grid = p.items < (uint32_t)ctx->sm_count ? p.items : (uint32_t)ctx->sm_count;
    *taken = true;
    if (a.dtype == HOLO_DTYPE_F16)
        return a.dim == 128 ? launch_packed_tile<true, 8>(ctx, mq, mk, mv, p, grid, smem)
               : a.dim == 64 ? launch_packed_tile<true, 4>(ctx, mq, mk, mv, p, grid, smem) : launch_packed_tile<true, 0>(ctx, mq, mk, mv, p, grid, smem);
    return a.dim == 128 ? launch_packed_tile<false, 8>(ctx, mq, mk, mv, p, grid, smem)
           : a.dim == 64 ? launch_packed_tile<false, 4>(ctx, mq, mk, mv, p, grid, smem) : launch_packed_tile<false, 0>(ctx, mq, mk, mv, p, grid, smem);
}
