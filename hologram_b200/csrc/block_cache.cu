// A cache of int8 blocks with one scale for each block and head: writing rows into it, and attention over it.
#include "sequences.cuh"

namespace {

// ---- writing -----------------------------------------------------------------------------------------------------------
// One CTA takes one touched block of one head, keys or values: the largest magnitude of its new rows, the block's scale, the codes of
// earlier rows again where the scale grows, the new codes. Nothing is shared between CTAs, so nothing depends on their order.
// A sequence of n rows touches at most (n - 1) / block_rows + 2 blocks; it owns the launch's items from starts[s] / block_rows + 2 s on,
// a sum that needs no pass over the lengths before it.

// The integer nearest to x / s, ties to even, for s > 0, clamped to +-127. An estimate that is at most one off, and the exact remainder
// of x by it: x - n s is a multiple of the smaller of the two's last places and smaller than 2 s, so fma holds it, or rounds it on the same side of +-s / 2.
__device__ __forceinline__ int nearest_code(float x, float s, float inv) {
    const float n = rintf(x * inv), r = fmaf(-n, s, x), twice = 2.0f * r;
    int i = __float2int_rn(n);
    // further than half a step, or just there from an odd number: the other neighbour
    if (fabsf(twice) > s || (fabsf(twice) == s && (i & 1))) i += r > 0.0f ? 1 : -1;
    return max(-127, min(127, i));
}
// The same in 64 bits for x and s of 31 bits at most, whose remainder is exact there; about = x / s, rounded somehow.
__device__ __forceinline__ int nearest_code(double x, double s, double about) {
    double n = rint(about);
    const double twice = 2.0 * fma(-n, s, x);
    const bool odd = ((int)n & 1) != 0;
    if (twice > s || (twice == s && odd)) n += 1.0;
    if (twice < -s || (twice == -s && odd)) n -= 1.0;
    return max(-127, min(127, (int)n));
}
__device__ __forceinline__ int code_of(float x, float s, float inv) {
    if (s == 0.0f || x != x) return 0;
    if (fabsf(x) == INFINITY) return x > 0.0f ? 127 : -127;
    if (inv == 0.0f) return nearest_code((double)x, (double)s, (double)x / (double)s);      // a scale whose reciprocal may overflow
    return nearest_code(x, s, inv);
}

// Division of numbers below 2^31 by a number that the host knows, by a product: with 2^l >= d and m = floor(2^32 (2^l - d) / d) + 1,
// n / d = (n + floor(m n / 2^32)) / 2^l (Granlund and Montgomery), where the sum fits 32 bits.
struct Divisor {
    uint32_t d, m, l;
    explicit Divisor(uint32_t by) : d(by), l(0) {
        while (1ull << l < by) ++l;
        m = (uint32_t)((((1ull << l) - by) << 32) / by + 1);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return (n + __umulhi(m, n)) >> l; }
};
struct BlockWriteParams {
    HoloBlockWriteArgs a;
    Divisor heads, block, k_across, v_across;      // across: units of a row
    int32_t most;                                  // positions that a sequence may have
};

constexpr int WRITE_THREADS = 128;
constexpr int WRITE_KEPT = 4;       // units of new values a thread keeps from the search for the largest to the coding

// VEC values of a row at a time (8 where rows and pitches allow 16-byte loads of 16-bit types, 4 of f32, else 1), kept as they came
template <int VEC>
struct Unit {
    uint4 raw;
};
template <>
struct Unit<1> {
    float raw;
};
template <int DT, int VEC>
__device__ __forceinline__ Unit<VEC> load_unit(const void* p, uint64_t i) {
    Unit<VEC> u;
    if constexpr (VEC == 1) u.raw = seq_load(p, i, DT);
    else u.raw = *reinterpret_cast<const uint4*>((const uint8_t*)p + i * (16 / VEC));
    return u;
}
template <int DT, int VEC>
__device__ __forceinline__ void values_of(const Unit<VEC>& u, float (&x)[VEC]) {
    if constexpr (VEC == 1) {
        x[0] = u.raw;
    } else {
        const uint32_t w[4] = {u.raw.x, u.raw.y, u.raw.z, u.raw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (DT == HOLO_DTYPE_F32) {
                x[e] = __uint_as_float(w[e]);
            } else if constexpr (DT == HOLO_DTYPE_BF16) {
                x[2 * e] = __uint_as_float(w[e] << 16);
                x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                x[2 * e] = f.x;
                x[2 * e + 1] = f.y;
            }
        }
    }
}
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* to, const int (&code)[VEC]) {
    if (VEC == 1) {
        *to = (int8_t)code[0];
    } else {
        uint32_t w[(VEC + 3) / 4];
#pragma unroll
        for (int e = 0; e < (VEC + 3) / 4; ++e)
            w[e] = __byte_perm(__byte_perm((uint32_t)code[(4 * e) % VEC], (uint32_t)code[(4 * e + 1) % VEC], 0x0040),
                               __byte_perm((uint32_t)code[(4 * e + 2) % VEC], (uint32_t)code[(4 * e + 3) % VEC], 0x0040), 0x5410);
        if (VEC == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[(VEC + 3) / 4 - 1]);
        else *reinterpret_cast<uint32_t*>(to) = w[0];
    }
}

// What a block held in a smaller scale, said in the new one.
__device__ __noinline__ void recode_rows(int8_t* codes, uint32_t n, float before, float now) {
    const double ratio = (double)before / (double)now;
    for (uint32_t i = threadIdx.x; i < n; i += WRITE_THREADS) {
        const double old = (double)codes[i];
        codes[i] = (int8_t)nearest_code(old * (double)before, (double)now, old * ratio);
    }
}
__device__ __noinline__ int any_code(float x, float s, float inv) { return code_of(x, s, inv); }

// 128-thread CTAs, eight to an SM: what a CTA waits for is a chain of loads (starts, length, block number, rows), hidden by the others
template <int DT, int VEC>
__global__ void __launch_bounds__(WRITE_THREADS, 8)
block_write_kernel(const __grid_constant__ BlockWriteParams p) {
    __shared__ uint32_t s_most[WRITE_THREADS / 32];
    const HoloBlockWriteArgs& a = p.a;
    const HoloBlockCache& c = a.c;
    // neighbouring CTAs take the heads of the same rows, whose values lie side by side
    const uint32_t turn = p.heads.of(blockIdx.x), head = blockIdx.x - turn * c.kv_heads, item = turn >> 1, tid = threadIdx.x, br = c.block_rows;
    const bool values = (turn & 1u) != 0;
    holo_pdl_trigger();
    holo_pdl_wait();
    if (blockIdx.x == 0) check_sequences(c.starts, c.lengths, c.sequences, c.rows, p.most, c.status);
    // the sequence that owns the item, and the item's number in it
    uint32_t s, nth;
    int32_t begin, end, length;
    if (c.starts) {
        // the last sequence whose first item is at most `item`: 32 places a round trip
        uint32_t lo = 0, left = c.sequences;
        int32_t from, to = 0, has = 0;
        for (;;) {
            const uint32_t step = (left + 31) / 32, at = lo + min(tid & 31u, (left - 1) / step) * step;
            from = c.starts[at];
            if (step == 1) {        // the last round: what is asked of the sequence comes along
                to = c.starts[at + 1];
                has = c.lengths[at];
            }
            const bool below = (uint64_t)p.block.of((uint32_t)max(from, 0)) + 2ull * at <= item;
            const uint32_t ahead = __ballot_sync(0xffffffffu, below);
            if (ahead == 0) return;         // starts that do not begin at 0
            const int last = 31 - __clz(ahead);
            lo = __shfl_sync(0xffffffffu, at, last);
            if (step == 1) {
                from = __shfl_sync(0xffffffffu, from, last);
                to = __shfl_sync(0xffffffffu, to, last);
                has = __shfl_sync(0xffffffffu, has, last);
                break;
            }
            left = min(step, c.sequences - lo);
        }
        s = lo;
        begin = from;
        end = to;
        length = has;
        if (begin < 0 || end <= begin || end > (int32_t)c.rows) return;
        nth = item - p.block.of((uint32_t)begin) - 2 * s;
    } else {
        s = item;
        begin = (int32_t)s;
        end = begin + 1;
        nth = 0;
        length = c.lengths[s];
    }
    const int32_t count = end - begin;
    if (length < count || length > p.most || nth > p.block.of((uint32_t)count - 1) + 1) return;
    const uint32_t first = (uint32_t)(length - count), j = p.block.of(first) + nth, block_at = j * br;      // positions are below 2^31
    if (block_at >= (uint32_t)length) return;
    const int id = c.table[(uint64_t)s * c.table_ld + j];
    const uint32_t lo = first > block_at ? first - block_at : 0u, hi = min(br, (uint32_t)length - block_at);     // new rows of the block
    const uint32_t d = values ? c.vdim : c.dim, ld = values ? a.v_ld : a.k_ld;
    const void* x = values ? a.v : a.k;
    const uint64_t x0 = (uint64_t)((uint32_t)begin + (block_at + lo - first)) * ld + (uint64_t)head * d;      // the block's row `lo` in the call's rows
    const Divisor& units = values ? p.v_across : p.k_across;
    const uint32_t across = units.d, n = (hi - lo) * across;
    Unit<VEC> kept[WRITE_KEPT];
    auto unit = [&](uint32_t i) {
        const uint32_t row = units.of(i);
        return load_unit<DT, VEC>(x, x0 + (uint64_t)row * ld + (i - row * across) * VEC);
    };
#pragma unroll
    for (int u = 0; u < WRITE_KEPT; ++u)
        if (tid + u * WRITE_THREADS < n) kept[u] = unit(tid + u * WRITE_THREADS);
    // the rows are on their way while the block's number comes
    if (id < 0 || (uint32_t)id >= c.blocks) {
        if (tid == 0) atomicOr(c.status, HOLO_STATUS_TABLE);
        return;
    }
    const uint64_t plane = (uint64_t)id * c.kv_heads + head;
    int8_t* codes = (values ? c.v_codes : c.k_codes) + plane * br * d;
    float* scale = (values ? c.v_scales : c.k_scales) + plane;
    const float before = lo ? *scale : 0.0f;
    // magnitudes order as their bits do, infinities and NaN above all
    uint32_t largest = 0;
    auto look = [&](const Unit<VEC>& u, uint32_t below) {
        if constexpr (VEC == 8) {
            // two 16-bit magnitudes at a time; what is not below becomes 0
            const uint32_t w[4] = {u.raw.x & 0x7fff7fffu, u.raw.y & 0x7fff7fffu, u.raw.z & 0x7fff7fffu, u.raw.w & 0x7fff7fffu};
            uint32_t m = 0;
            if (below == 0xffffffffu) {
                m = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
            } else {
                const uint32_t inf = DT == HOLO_DTYPE_BF16 ? 0x7f807f80u : 0x7c007c00u;
#pragma unroll
                for (int e = 0; e < 4; ++e) m = __vmaxu2(m, w[e] & __vcmpltu2(w[e], inf));
            }
            m = max(m & 0xffffu, m >> 16);
            largest = max(largest, DT == HOLO_DTYPE_BF16 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half((uint16_t)m))));
        } else {
            float v[VEC];
            values_of<DT, VEC>(u, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const uint32_t m = __float_as_uint(v[e]) & 0x7fffffffu;
                if (m < below) largest = max(largest, m);
            }
        }
    };
    auto look_all = [&](uint32_t below) {
#pragma unroll
        for (int u = 0; u < WRITE_KEPT; ++u)
            if (tid + u * WRITE_THREADS < n) look(kept[u], below);
#pragma unroll 1
        for (uint32_t i = tid + WRITE_KEPT * WRITE_THREADS; i < n; i += WRITE_THREADS) look(unit(i), below);
        largest = __reduce_max_sync(0xffffffffu, largest);
        if ((tid & 31) == 0) s_most[tid >> 5] = largest;
        __syncthreads();        // nobody stores the new scale before everybody has read the old one
#pragma unroll
        for (int w = 0; w < WRITE_THREADS / 32; ++w) largest = max(largest, s_most[w]);
    };
    look_all(0xffffffffu);
    const bool finite = largest < 0x7f800000u;
    if (!finite) {
        __syncthreads();
        largest = 0;
        look_all(0x7f800000u);
    }
    const float now = fmaxf(before, __fdiv_rn(__uint_as_float(largest), 127.0f));
    if (lo && now > before) recode_rows(codes, lo * d, before, now);
    const float inv = now < 1.2e-37f ? 0.0f : __fdiv_rn(1.0f, now), half = 0.5f * now;
    const bool plain = finite && inv != 0.0f;
    auto encode = [&](uint32_t i, const Unit<VEC>& u) {
        float v[VEC];
        values_of<DT, VEC>(u, v);
        int code[VEC];
        bool special = !plain;
        if (plain) {
            // |x / now| is 127 at most, but for roundings: a sum with 1.5 * 2^23 has the integer next to it in its low bits, and is it
            // where the remainder (exact, see nearest_code) is below half a step; the few others are left to that
            float most_left = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float m = fmaf(v[e], inv, 12582912.0f), r = fmaf(12582912.0f - m, now, v[e]);
                code[e] = __float_as_int(m);
                most_left = fmaxf(most_left, fabsf(r));
            }
            special = most_left >= half;
        }
        if (special) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) code[e] = any_code(v[e], now, now < 1.2e-37f ? 0.0f : inv);
        }
        store_codes<VEC>(codes + lo * d + i * VEC, code);
    };
#pragma unroll
    for (int u = 0; u < WRITE_KEPT; ++u)
        if (tid + u * WRITE_THREADS < n) encode(tid + u * WRITE_THREADS, kept[u]);
#pragma unroll 1
    for (uint32_t i = tid + WRITE_KEPT * WRITE_THREADS; i < n; i += WRITE_THREADS) encode(i, unit(i));
    if (tid == 0) *scale = now;
}

// ---- attention ---------------------------------------------------------------------------------------------------------

struct CacheSource {
    HoloBlockAttnArgs a;
    struct Place {
        uint32_t begin, end, sequence;
    };
    __device__ uint32_t rows() const { return a.c.rows; }
    __device__ uint32_t heads() const { return a.heads; }
    __device__ uint32_t dim() const { return a.c.dim; }
    __device__ uint32_t vdim() const { return a.c.vdim; }
    __device__ float scale() const { return a.scale; }
    __device__ void check() const { check_sequences(a.c.starts, a.c.lengths, a.c.sequences, a.c.rows, (int64_t)a.c.table_ld * a.c.block_rows, a.c.status); }
    __device__ bool place(uint32_t row, Place* p) const {
        uint32_t from = row, to = row + 1;
        p->sequence = row;
        if (a.c.starts && !sequence_of(a.c.starts, a.c.sequences, a.c.rows, row, &from, &to, &p->sequence)) return false;
        const int64_t most = (int64_t)a.c.table_ld * a.c.block_rows, length = max((int64_t)0, min((int64_t)a.c.lengths[p->sequence], most));
        p->begin = 0;
        p->end = (uint32_t)max((int64_t)0, length - to + row + 1);
        return true;
    }
    __device__ float q(uint32_t row, uint32_t head, uint32_t x) const { return seq_load(a.q, (uint64_t)row * a.q_ld + (uint64_t)head * a.c.dim + x, a.dtype); }
    __device__ void key(const Place& at, uint32_t head, uint32_t j, uint64_t* kb, uint64_t* vb, float* ks, float* vs) const {
        const uint32_t br = a.c.block_rows;
        const int id = a.c.table[(uint64_t)at.sequence * a.c.table_ld + j / br];
        if (id < 0 || (uint32_t)id >= a.c.blocks) {      // a block of zeros
            atomicOr(a.c.status, HOLO_STATUS_TABLE);
            *kb = *vb = 0;
            *ks = *vs = 0.0f;
            return;
        }
        const uint64_t plane = (uint64_t)id * a.c.kv_heads + head / (a.heads / a.c.kv_heads), row = plane * br + j % br;
        *kb = row * a.c.dim;
        *vb = row * a.c.vdim;
        *ks = a.c.k_scales[plane];
        *vs = a.c.v_scales[plane];
    }
    __device__ float k(uint64_t i) const { return (float)a.c.k_codes[i]; }
    __device__ float v(uint64_t i) const { return (float)a.c.v_codes[i]; }
    __device__ void store(uint32_t row, uint32_t head, uint32_t x, float y) const { seq_store(a.out, (uint64_t)row * a.ld + (uint64_t)head * a.c.vdim + x, y, a.dtype); }
};

}  // namespace

int32_t holo_launch_block_cache_write(holo_b200_ctx* ctx, const HoloBlockWriteArgs& a) {
    const uint64_t items = a.c.starts ? (uint64_t)a.c.rows / a.c.block_rows + 2ull * a.c.sequences : a.c.sequences;
    if (items * a.c.kv_heads > 0x3fffffffull) return holo_fail(HOLO_ERR_UNSUPPORTED_OP, "unsupported op: block_cache_write of %u rows, %u heads", a.c.rows, a.c.kv_heads);
    const uint32_t es = (uint32_t)holo_dtype_size(a.dtype), vec = 16 / es;
    const bool wide = ((((uintptr_t)a.k | (uintptr_t)a.v) & 15u) | (a.c.dim | a.c.vdim | a.k_ld | a.v_ld) % vec) == 0 && (((uintptr_t)a.c.k_codes | (uintptr_t)a.c.v_codes) & 7u) == 0;
    const dim3 grid((uint32_t)(items * a.c.kv_heads * 2)), block(WRITE_THREADS);
    const uint32_t per = wide ? vec : 1u;
    const BlockWriteParams p = {a, Divisor(a.c.kv_heads), Divisor(a.c.block_rows), Divisor(a.c.dim / per), Divisor(a.c.vdim / per), (int32_t)(a.c.table_ld * a.c.block_rows)};
    auto launch = [&](auto kernel) { return holo_launch_kernel(ctx, kernel, grid, block, 0, 1, p); };
    cudaError_t e;
    if (a.dtype == HOLO_DTYPE_F32) e = wide ? launch(block_write_kernel<HOLO_DTYPE_F32, 4>) : launch(block_write_kernel<HOLO_DTYPE_F32, 1>);
    else if (a.dtype == HOLO_DTYPE_BF16) e = wide ? launch(block_write_kernel<HOLO_DTYPE_BF16, 8>) : launch(block_write_kernel<HOLO_DTYPE_BF16, 1>);
    else e = wide ? launch(block_write_kernel<HOLO_DTYPE_F16, 8>) : launch(block_write_kernel<HOLO_DTYPE_F16, 1>);
    HOLO_CUDA(e);
    ctx->launches++;
    return HOLO_OK;
}

int32_t holo_launch_block_cache_attention(holo_b200_ctx* ctx, const HoloBlockAttnArgs& a) {
    bool taken;
    HOLO_TRY(holo_try_block_tile(ctx, a, &taken));
    if (taken) return HOLO_OK;
    HOLO_TRY(holo_try_block_rows(ctx, a, &taken));
    if (taken) return HOLO_OK;
    HOLO_TRY(holo_try_block_attention(ctx, a, &taken));
    if (taken) return HOLO_OK;
    CacheSource src = {a};
    return launch_general_rows(ctx, src, (uint64_t)a.c.rows * a.heads, a.c.vdim);
}
