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
    float n = rintf(x * inv);
    const float r = fmaf(-n, s, x), twice = 2.0f * r;
    const bool odd = ((int)n & 1) != 0;
    if (twice > s || (twice == s && odd)) n += 1.0f;
    if (twice < -s || (twice == -s && odd)) n -= 1.0f;
    return max(-127, min(127, __float2int_rn(n)));
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

constexpr int WRITE_THREADS = 128;

__global__ void __launch_bounds__(WRITE_THREADS)
block_write_kernel(const __grid_constant__ HoloBlockWriteArgs a) {
    __shared__ float s_most[WRITE_THREADS / 32];
    const HoloBlockCache& c = a.c;
    const uint32_t item = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, br = c.block_rows;
    const bool values = blockIdx.z != 0;
    holo_pdl_trigger();
    holo_pdl_wait();
    const int64_t most = (int64_t)c.table_ld * br;
    if (item == 0 && head == 0 && !values) check_sequences(c.starts, c.lengths, c.sequences, c.rows, most, c.status);
    // the sequence that owns the item, and the item's number in it
    uint32_t s, nth;
    int64_t begin, count;
    if (c.starts) {
        int lo = -1, hi = (int)c.sequences - 1;
        while (lo < hi) {
            const int mid = lo + (hi - lo + 1) / 2;
            if ((int64_t)(max(c.starts[mid], 0) / (int)br) + 2ll * mid <= (int64_t)item) lo = mid;
            else hi = mid - 1;
        }
        if (lo < 0) return;
        s = (uint32_t)lo;
        begin = c.starts[s];
        const int64_t end = c.starts[s + 1];
        if (begin < 0 || end > c.rows) return;
        count = end - begin;
        nth = item - (uint32_t)(begin / br) - 2 * s;
    } else {
        s = item;
        begin = s;
        count = 1;
        nth = 0;
    }
    const int64_t length = c.lengths[s], first = length - count;
    if (count <= 0 || first < 0 || length > most) return;
    const uint32_t j = (uint32_t)(first / br) + nth;
    const int64_t block_at = (int64_t)j * br;
    if (block_at >= length) return;
    const int id = c.table[(uint64_t)s * c.table_ld + j];
    if (id < 0 || (uint32_t)id >= c.blocks) {
        if (tid == 0) atomicOr(c.status, HOLO_STATUS_TABLE);
        return;
    }
    const uint32_t lo = first > block_at ? (uint32_t)(first - block_at) : 0u, hi = (uint32_t)min((int64_t)br, length - block_at);     // new rows of the block
    const uint32_t d = values ? c.vdim : c.dim, ld = values ? a.v_ld : a.k_ld;
    const void* x = values ? a.v : a.k;
    const uint64_t plane = (uint64_t)id * c.kv_heads + head;
    int8_t* codes = (values ? c.v_codes : c.k_codes) + plane * br * d;
    float* scale = (values ? c.v_scales : c.k_scales) + plane;
    const uint64_t row0 = (uint64_t)(begin + (block_at + lo - first));      // the call's row behind the block's row `lo`
    const uint32_t n = (hi - lo) * d;
    float largest = 0.0f;
    for (uint32_t i = tid; i < n; i += WRITE_THREADS) {
        const float m = fabsf(seq_load(x, (row0 + i / d) * ld + (uint64_t)head * d + i % d, a.dtype));
        if (m < INFINITY) largest = fmaxf(largest, m);
    }
    for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    if ((tid & 31) == 0) s_most[tid >> 5] = largest;
    const float before = lo ? *scale : 0.0f;
    __syncthreads();        // nobody stores the new scale before everybody has read the old one
    for (int w = 0; w < WRITE_THREADS / 32; ++w) largest = fmaxf(largest, s_most[w]);
    const float now = fmaxf(before, __fdiv_rn(largest, 127.0f));
    if (now > before && lo) {
        const double ratio = (double)before / (double)now;
        for (uint32_t i = tid; i < lo * d; i += WRITE_THREADS) {
            const double old = (double)codes[i];
            codes[i] = (int8_t)nearest_code(old * (double)before, (double)now, old * ratio);
        }
    }
    const float inv = now < 1.2e-38f ? 0.0f : __fdiv_rn(1.0f, now);
    for (uint32_t i = tid; i < n; i += WRITE_THREADS)
        codes[lo * d + i] = (int8_t)code_of(seq_load(x, (row0 + i / d) * ld + (uint64_t)head * d + i % d, a.dtype), now, inv);
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
        const int64_t most = (int64_t)a.c.table_ld * a.c.block_rows, sees = (int64_t)a.c.lengths[p->sequence] - to + row + 1;
        p->begin = 0;
        p->end = (uint32_t)max((int64_t)0, min(sees, most));
        return true;
    }
    __device__ float q(uint32_t row, uint32_t head, uint32_t x) const { return seq_load(a.q, (uint64_t)row * a.q_ld + (uint64_t)head * a.c.dim + x, a.dtype); }
    __device__ bool key(const Place& at, uint32_t head, uint32_t j, uint64_t* kb, uint64_t* vb, float* ks, float* vs) const {
        const uint32_t br = a.c.block_rows;
        const int id = a.c.table[(uint64_t)at.sequence * a.c.table_ld + j / br];
        if (id < 0 || (uint32_t)id >= a.c.blocks) {
            atomicOr(a.c.status, HOLO_STATUS_TABLE);
            return false;
        }
        const uint64_t plane = (uint64_t)id * a.c.kv_heads + head / (a.heads / a.c.kv_heads), row = plane * br + j % br;
        *kb = row * a.c.dim;
        *vb = row * a.c.vdim;
        *ks = a.c.k_scales[plane];
        *vs = a.c.v_scales[plane];
        return true;
    }
    __device__ float k(uint64_t i) const { return (float)a.c.k_codes[i]; }
    __device__ float v(uint64_t i) const { return (float)a.c.v_codes[i]; }
    __device__ void store(uint32_t row, uint32_t head, uint32_t x, float y) const { seq_store(a.out, (uint64_t)row * a.ld + (uint64_t)head * a.c.vdim + x, y, a.dtype); }
};

}  // namespace

int32_t holo_launch_block_cache_write(holo_b200_ctx* ctx, const HoloBlockWriteArgs& a) {
    const uint64_t items = a.c.starts ? (uint64_t)a.c.rows / a.c.block_rows + 2ull * a.c.sequences : a.c.sequences;
    if (items > 0x7fffffffull || a.c.kv_heads > 65535) return holo_fail(HOLO_ERR_UNSUPPORTED_OP, "unsupported op: block_cache_write of %u rows, %u heads", a.c.rows, a.c.kv_heads);
    HOLO_CUDA(holo_launch_kernel(ctx, block_write_kernel, dim3((uint32_t)items, a.c.kv_heads, 2), dim3(WRITE_THREADS), 0, 1, a));
    ctx->launches++;
    return HOLO_OK;
}

int32_t holo_launch_block_cache_attention(holo_b200_ctx* ctx, const HoloBlockAttnArgs& a) {
    bool taken;
    HOLO_TRY(holo_try_block_attention(ctx, a, &taken));
    if (taken) return HOLO_OK;
    CacheSource src = {a};
    return launch_general_rows(ctx, src, (uint64_t)a.c.rows * a.heads, a.c.vdim);
}
