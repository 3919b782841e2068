// What the block cache's attention kernels share: products and codes as operands, and the list of all slabs of a call that its CTAs
// share out.
#pragma once
#include "attention_tile.cuh"
#include "sequences.cuh"

namespace {

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
// Bytes 0 and 2 (1 and 3) of four codes plus 128 as a pair of f16 codes
template <uint32_t PICK>
__device__ __forceinline__ uint32_t codes_to_half(uint32_t biased) {
    const uint32_t raised = __byte_perm(biased, 0x64646464u, PICK);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&raised), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
constexpr uint32_t PICK02 = 0x4240, PICK13 = 0x4341;

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4u : 0u) : "memory");
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
// The list of planes: sequence by sequence, kv head by kv head, R rows by R rows; `at` counts the slabs of all planes before.
struct Plane {
    uint32_t seq, head, tile, tiles, first_row, n, slabs, at;
    int32_t length;
};
template <int R>
__device__ __forceinline__ uint32_t rows_before(const Plane& p, uint32_t tile, uint32_t group) {       // positions up to the tile's last one
    return min(p.n, (tile * R + R - 1) / group + 1);
}
// Positions that the tile's last row sees. None happens to sequences with fewer positions than rows (reported by check_sequences): their planes
// have a slab all the same, whose keys are beyond every row's limit, so that rows that see nothing are stored as zeros.
template <int R>
__device__ __forceinline__ uint32_t keys_of_plane(const Plane& p, uint32_t tile, uint32_t group) {
    return (uint32_t)max(1, p.length - (int32_t)(p.n - rows_before<R>(p, tile, group)));
}
template <int R, int SLAB>
__device__ __forceinline__ uint32_t slabs_of(const Plane& p, uint32_t tile, uint32_t group) {
    return (keys_of_plane<R>(p, tile, group) + SLAB - 1) / SLAB;
}
template <int R>
__device__ __forceinline__ void read_sequence(const HoloBlockCache& c, uint32_t group, uint32_t s, Plane* p) {
    int32_t b = (int32_t)s, e = (int32_t)s + 1;
    if (c.starts) {
        b = c.starts[s];
        e = c.starts[s + 1];
        if (b < 0 || e < b || e > (int32_t)c.rows) b = e = 0;
    }
    p->seq = s;
    p->first_row = (uint32_t)b;
    p->n = (uint32_t)(e - b);
    p->length = max(0, min(c.lengths[s], (int32_t)(c.table_ld * c.block_rows)));
    p->tiles = (p->n * group + R - 1) / R;
    p->head = p->tile = 0;
}
// On to the next plane; slabs == 0: there is none. EXTRA: places of the list behind a plane's slabs that stand for what a
// plane costs a CTA beside them.
template <int R, int SLAB, int EXTRA = 0>
__device__ __forceinline__ void next_plane(const HoloBlockCache& c, uint32_t group, Plane* p) {
    p->at += p->slabs + EXTRA;
    for (;;) {
        if (++p->tile >= p->tiles) {
            p->tile = 0;
            if (++p->head >= c.kv_heads) {
                if (++p->seq >= c.sequences) {
                    p->slabs = 0;
                    return;
                }
                read_sequence<R>(c, group, p->seq, p);
            }
        }
        if (p->tiles) {
            p->slabs = slabs_of<R, SLAB>(*p, p->tile, group);
            return;
        }
        p->head = c.kv_heads - 1;      // no rows: on to the next sequence
    }
}


// A CTA's share of the list: slabs [lo, hi), from plane `first` on. Shares are equal and go from plane to plane, or, where there are few
// planes (`apart`), every plane is cut into pieces of its own, of which this is number `part`, and slabs count within the plane.
struct Share {
    Plane first;
    uint32_t lo, hi, part, unit, each, more_by_one;
    bool apart;
    // the first of the CTAs that share a plane, and how many they are
    __device__ __forceinline__ uint32_t owner(uint32_t slab) const {
        const uint32_t longer = more_by_one * (each + 1);
        return slab < longer ? slab / (each + 1) : more_by_one + (slab - longer) / each;
    }
    __device__ __forceinline__ uint32_t first_cta(const Plane& p) const { return apart ? blockIdx.x - part : owner(p.at); }
    __device__ __forceinline__ uint32_t cta_count(const Plane& p) const { return apart ? (p.slabs + unit - 1) / unit : owner(p.at + p.slabs - 1) - owner(p.at) + 1; }
    // the slabs of a plane that are this CTA's
    __device__ __forceinline__ void ends_of(const Plane& p, uint32_t* s0, uint32_t* s1) const {
        *s0 = lo > p.at ? lo - p.at : 0u;
        *s1 = min(p.slabs, hi - p.at);
    }
};

// Every warp finds the share by itself, one or four sequences a lane at a time; false: there is none for this CTA. A share is LEAST slabs at
// least, so that fewer CTAs take part in a short list. Planes are cut apart where that lengthens a share by less than the SECOND
// slabs that another plane costs a CTA.
template <int R, int SLAB, int LEAST, int SECOND, int EXTRA = 0>
__device__ __forceinline__ bool find_share(const HoloBlockCache& c, uint32_t group, Share* out) {
    const uint32_t lane = threadIdx.x & 31, each = c.sequences <= 32 ? 1u : 4u;      // of a lane
    uint32_t cnt[4], upto = 0, sum = 0, all = 0, planes = 0, unit = 1, extra = 0;
    auto count_chunk = [&](uint32_t s0) {
        Plane seq[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t s = s0 + each * lane + i;
            read_sequence<R>(c, group, min(s, c.sequences - 1), &seq[i]);
            if ((uint32_t)i >= each || s >= c.sequences) seq[i].tiles = 0;
        }
        sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cnt[i] = 0;
#pragma unroll 1
            for (uint32_t t = 0; t < seq[i].tiles; ++t) {
                cnt[i] += (slabs_of<R, SLAB>(seq[i], t, group) + unit - 1) / unit + (EXTRA ? extra : 0u);
            }
            cnt[i] *= c.kv_heads;
            sum += cnt[i];
            planes += seq[i].tiles;
        }
        upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += u;
        }
        all = __shfl_sync(0xffffffffu, upto, 31);
    };
    uint32_t total = 0;
#pragma unroll 1
    for (uint32_t s0 = 0; s0 < c.sequences; s0 += 128) {
        count_chunk(s0);
        total += all;
    }
    planes = __reduce_add_sync(0xffffffffu, planes) * c.kv_heads;
    const uint32_t grid = gridDim.x;
    Share& s = *out;
    s.apart = planes < grid && (uint64_t)total * planes <= (uint64_t)SECOND * grid * (grid - planes);
    s.each = s.more_by_one = s.part = 0;
    uint32_t want;
    if (s.apart) {
        unit = max((total + grid - planes - 1) / (grid - planes), (uint32_t)LEAST);
        want = blockIdx.x;
    } else {
        extra = EXTRA;
        total += EXTRA * planes;
        const uint32_t ctas = min(grid, (total + LEAST - 1) / LEAST);
        if (blockIdx.x >= ctas) return false;
        s.each = total / ctas;
        s.more_by_one = total - s.each * ctas;
        want = blockIdx.x * s.each + min(blockIdx.x, s.more_by_one);
    }
    s.unit = unit;
    uint32_t run = 0, s0 = 0;
    bool found = false;
#pragma unroll 1
    for (;; s0 += 128) {
        if (s.apart || EXTRA || c.sequences > 128) count_chunk(s0);
        found = want < run + all;
        if (found || s0 + 128 >= c.sequences) break;
        run += all;
    }
    if (!found) return false;
    uint32_t at = run + upto - sum, mine = 0, which = 0;
    const uint32_t from = __ffs(__ballot_sync(0xffffffffu, want < run + upto)) - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (mine == 0) {
            if (want < at + cnt[i]) {
                mine = cnt[i];
                which = s0 + each * lane + i;
            } else {
                at += cnt[i];
            }
        }
    which = __shfl_sync(0xffffffffu, which, from);
    at = __shfl_sync(0xffffffffu, at, from);
    mine = __shfl_sync(0xffffffffu, mine, from);
    Plane& f = s.first;
    read_sequence<R>(c, group, min(which, c.sequences - 1), &f);
    const uint32_t a_head = max(mine / c.kv_heads, 1u);
    f.head = min((want - at) / a_head, c.kv_heads - 1);
    f.at = at + f.head * a_head;
    f.slabs = slabs_of<R, SLAB>(f, 0, group);
    for (;;) {
        const uint32_t pieces = (f.slabs + unit - 1) / unit + (EXTRA ? extra : 0u);
        if (want < f.at + pieces || f.tile + 1 >= f.tiles) break;
        f.at += pieces;
        f.slabs = slabs_of<R, SLAB>(f, ++f.tile, group);
    }
    if (s.apart) {
        s.part = want - f.at;
        f.at = 0;
        s.lo = s.part * unit;
        s.hi = min(s.lo + unit, f.slabs);
    } else {
        s.lo = want;
        s.hi = (blockIdx.x + 1) * s.each + min(blockIdx.x + 1, s.more_by_one);
        if (EXTRA && f.at + f.slabs <= want) {      // the share begins behind the plane's slabs
            next_plane<R, SLAB, EXTRA>(c, group, &f);
            if (!f.slabs || f.at >= s.hi) return false;
        }
    }
    return true;
}

}  // namespace
