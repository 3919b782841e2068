// Rules on logits before a token is chosen (the LogitRules call): penalties for repeated tokens, biases, temperature, grammar masks.
//
// A CTA takes a part of a row's vocabulary. It reads the row's whole history and bias list and keeps, in shared memory, a count and, where
// the row has biases, the last bias entry for every token of its part (integer sums and maxima: no order of threads shows), then
// streams its logits once. Reading the history once for every part costs L2 traffic alone; counting it once for all parts of a row, with
// atomics into the other CTAs' memory through a cluster, took 19.7 us for 64 x 32000 against 9.9, since half of a text's tokens fall
// into one part.
// Bound: HBM for many rows, for few the chain spans -> history -> counts; the logits are requested before the history, so that they arrive
// while it is counted.
#include "sequences.cuh"

namespace {

constexpr int RULES_THREADS = 256;
constexpr int RULES_KEPT = 4;                 // units of logits a thread requests before the counts are there
constexpr int RULES_AHEAD = 8;                // history entries a thread has on their way
constexpr uint32_t RULES_MOST_PART = 8192;    // tokens of a CTA: counts and bias entries are 8 bytes a token
constexpr uint32_t RULES_MOST_ROWS = 65535;      // of a launch (a first row or a third dimension in the kernel takes 64 x 32000 from 9.9 to 13.4 us)
constexpr uint32_t IN_PROMPT = 0x80000000u;   // of a count: the token stands in the prompt; the rest counts it behind the prompt

struct RulesParams {
    HoloLogitRulesArgs a;
    uint32_t part;       // tokens of a CTA, a multiple of 32
};

template <int VEC>
struct RulesUnit {
    uint4 raw;
};
template <>
struct RulesUnit<1> {
    float raw;
};

template <int DT, int VEC>
__global__ void __launch_bounds__(RULES_THREADS)
logit_rules_kernel(const __grid_constant__ RulesParams p) {
    extern __shared__ __align__(16) uint32_t s_words[];     // counts [part], then bias entries + 1 [part]
    const HoloLogitRulesArgs& a = p.a;
    const uint32_t tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * p.part, n = min(p.part, a.vocab - first);
    holo_pdl_trigger();
    holo_pdl_wait();
    // what this thread's first logits are: on their way while the history is counted
    const uint64_t z0 = (uint64_t)row * a.ld + first, o0 = (uint64_t)row * a.out_ld + first;
    RulesUnit<VEC> kept[RULES_KEPT];
    auto load = [&](uint32_t i) {
        RulesUnit<VEC> u;
        if constexpr (VEC == 1) u.raw = seq_load(a.logits, z0 + i, DT);
        else u.raw = *reinterpret_cast<const uint4*>((const uint8_t*)a.logits + (z0 + i) * (16 / VEC));
        return u;
    };
#pragma unroll
    for (int k = 0; k < RULES_KEPT; ++k)
        if ((tid + k * RULES_THREADS) * VEC < n) kept[k] = load((tid + k * RULES_THREADS) * VEC);
    int prompt = 0, total = 0, from = 0, to = 0;
    bool bad = false;
    if (a.history) {
        prompt = a.spans[2 * (uint64_t)row];
        total = a.spans[2 * (uint64_t)row + 1];
        if (prompt < 0 || total < prompt || total > (int)a.history_ld) {
            bad = true;
            prompt = total = 0;
        }
    }
    if (a.bias_ids) {
        from = a.bias_starts[row];
        to = a.bias_starts[row + 1];
        if (from < 0 || to < from || to > (int)a.biases) {
            bad = true;
            from = to = 0;
        }
    }
    const uint32_t* mask = nullptr;
    if (a.masks) {
        const int which = a.mask_of ? a.mask_of[row] : (int)row;
        if (which < -1 || which >= (int)a.mask_rows) bad = true;
        else if (which >= 0) mask = a.masks + (uint64_t)which * a.mask_ld;
    }
    if (bad && tid == 0) atomicOr(a.status, HOLO_STATUS_TABLE);
    float repetition = 1.0f, presence = 0.0f, frequency = 0.0f, temperature = 0.0f;
    if (a.params) {
        const float* f = a.params + 4 * (uint64_t)row;
        repetition = f[0]; presence = f[1]; frequency = f[2]; temperature = f[3];
    }
    const bool counts = total > 0, biases = to > from;
    uint32_t *s_count = s_words, *s_bias = s_words + p.part;
    if (counts || biases) {
        if (counts)
            for (uint32_t i = tid; i < p.part / 4; i += RULES_THREADS) reinterpret_cast<uint4*>(s_count)[i] = make_uint4(0, 0, 0, 0);
        if (biases)
            for (uint32_t i = tid; i < p.part / 4; i += RULES_THREADS) reinterpret_cast<uint4*>(s_bias)[i] = make_uint4(0, 0, 0, 0);
        const int32_t* history = a.history + (uint64_t)row * a.history_ld;
        int32_t ahead[RULES_AHEAD];
        auto fetch = [&](uint32_t i) {
#pragma unroll
            for (int k = 0; k < RULES_AHEAD; ++k) ahead[k] = i + k * RULES_THREADS < (uint32_t)total ? history[i + k * RULES_THREADS] : -1;
        };
        fetch(tid);             // before the memory is clear
        __syncthreads();
        for (uint32_t i = tid; i < (uint32_t)total; i += RULES_AHEAD * RULES_THREADS) {
            int32_t now[RULES_AHEAD];
#pragma unroll
            for (int k = 0; k < RULES_AHEAD; ++k) now[k] = ahead[k];
            fetch(i + RULES_AHEAD * RULES_THREADS);
#pragma unroll
            for (int k = 0; k < RULES_AHEAD; ++k) {
                const uint32_t t = (uint32_t)now[k] - first;        // -1 and other ids outside the part wrap to large numbers
                if (now[k] < 0 || t >= n) continue;
                if (i + k * RULES_THREADS < (uint32_t)prompt) atomicOr(s_count + t, IN_PROMPT);
                else atomicAdd(s_count + t, 1u);
            }
        }
        for (uint32_t i = (uint32_t)from + tid; i < (uint32_t)to; i += RULES_THREADS) {
            const int32_t id = a.bias_ids[i];
            const uint32_t t = (uint32_t)id - first;
            if (id >= 0 && t < n) atomicMax(s_bias + t, i + 1);
        }
        __syncthreads();
    }
    auto one = [&](float z, uint32_t c, uint32_t entry, uint32_t allowed) {
        const uint32_t made = c & ~IN_PROMPT;
        if (c) z = z > 0.0f ? __fdiv_rn(z, repetition) : z * repetition;
        if (made) z -= fmaf(frequency, (float)made, presence);
        if (entry) z += a.bias_values[entry - 1];
        if (temperature > 0.0f && temperature != 1.0f) z = __fdiv_rn(z, temperature);
        return allowed ? z : -INFINITY;
    };
    auto apply = [&](uint32_t i, const RulesUnit<VEC>& u) {
        if constexpr (VEC == 1) {
            const uint32_t bit = mask ? mask[(first + i) >> 5] >> ((first + i) & 31u) & 1u : 1u;
            seq_store(a.out, o0 + i, one(u.raw, counts ? s_count[i] : 0u, biases ? s_bias[i] : 0u, bit), DT);
        } else {
            // the part and its units are multiples of 8 tokens: their bits lie in one word
            const uint32_t bits = mask ? mask[(first + i) >> 5] >> ((first + i) & 31u) : 0xffffffffu;
            uint32_t w[4] = {u.raw.x, u.raw.y, u.raw.z, u.raw.w};
            uint32_t c[VEC], b[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const uint4 x = counts ? *reinterpret_cast<const uint4*>(s_count + i + e) : make_uint4(0, 0, 0, 0);
                const uint4 y = biases ? *reinterpret_cast<const uint4*>(s_bias + i + e) : make_uint4(0, 0, 0, 0);
                c[e] = x.x; c[e + 1] = x.y; c[e + 2] = x.z; c[e + 3] = x.w;
                b[e] = y.x; b[e + 1] = y.y; b[e + 2] = y.z; b[e + 3] = y.w;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (DT == HOLO_DTYPE_F32) {
                    w[e] = __float_as_uint(one(__uint_as_float(w[e]), c[e], b[e], bits >> e & 1u));
                } else if constexpr (DT == HOLO_DTYPE_BF16) {
                    const float lo = one(__uint_as_float(w[e] << 16), c[2 * e], b[2 * e], bits >> (2 * e) & 1u);
                    const float hi = one(__uint_as_float(w[e] & 0xffff0000u), c[2 * e + 1], b[2 * e + 1], bits >> (2 * e + 1) & 1u);
                    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
                    w[e] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                    const __half2 h = __floats2half2_rn(one(f.x, c[2 * e], b[2 * e], bits >> (2 * e) & 1u), one(f.y, c[2 * e + 1], b[2 * e + 1], bits >> (2 * e + 1) & 1u));
                    w[e] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            *reinterpret_cast<uint4*>((uint8_t*)a.out + (o0 + i) * (16 / VEC)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };
#pragma unroll
    for (int k = 0; k < RULES_KEPT; ++k)
        if ((tid + k * RULES_THREADS) * VEC < n) apply((tid + k * RULES_THREADS) * VEC, kept[k]);
    for (uint32_t i = (tid + RULES_KEPT * RULES_THREADS) * VEC; i < n; i += RULES_THREADS * VEC) apply(i, load(i));
}

template <int DT, int VEC>
int32_t launch_logit_rules(holo_b200_ctx* ctx, RulesParams p) {
    const uint32_t smem = p.part * (p.a.bias_ids ? 8 : p.a.history ? 4 : 0);
    static thread_local int configured_device = -1;
    if (configured_device != ctx->device) {
        HOLO_CUDA(cudaFuncSetAttribute(logit_rules_kernel<DT, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(RULES_MOST_PART * 8)));
        configured_device = ctx->device;
    }
    for (;;) {
        HoloLogitRulesArgs& a = p.a;
        const uint32_t n = a.rows < RULES_MOST_ROWS ? a.rows : RULES_MOST_ROWS;
        HOLO_CUDA(holo_launch_kernel(ctx, logit_rules_kernel<DT, VEC>, dim3((a.vocab + p.part - 1) / p.part, n), dim3(RULES_THREADS), smem, 1, p));
        ctx->launches++;
        if (a.rows == n) return HOLO_OK;
        // the rows behind these
        const uint64_t es = holo_dtype_size(a.dtype);
        a.rows -= n;
        a.logits = (const uint8_t*)a.logits + n * es * a.ld;
        a.out = (uint8_t*)a.out + n * es * a.out_ld;
        if (a.history) {
            a.history += (uint64_t)n * a.history_ld;
            a.spans += 2ull * n;
        }
        if (a.params) a.params += 4ull * n;
        if (a.bias_ids) a.bias_starts += n;
        if (a.mask_of) {
            a.mask_of += n;
        } else if (a.masks) {
            a.masks += (uint64_t)n * a.mask_ld;
            a.mask_rows -= n;
        }
    }
}

}  // namespace

int32_t holo_launch_logit_rules(holo_b200_ctx* ctx, const HoloLogitRulesArgs& a) {
    RulesParams p = {};
    p.a = a;
    const uint32_t es = (uint32_t)holo_dtype_size(a.dtype), vec = 16 / es;
    const bool wide = ((((uintptr_t)a.logits | (uintptr_t)a.out) & 15u) | (a.ld | a.out_ld | a.vocab) % vec) == 0;
    // four CTAs an SM if the logits give that many; every thread one unit of logits at least, as many as it keeps at most
    const uint64_t ctas = 4ull * ctx->sm_count, a_row = ctas / a.rows + 1;
    uint64_t part = ((uint64_t)a.vocab + a_row - 1) / a_row;
    const uint64_t least = RULES_THREADS * (wide ? vec : 1u), most = least * RULES_KEPT < RULES_MOST_PART ? least * RULES_KEPT : RULES_MOST_PART;
    part = part < least ? least : part > most ? most : part;
    p.part = (uint32_t)((part + 31) & ~31ull);
    if (a.dtype == HOLO_DTYPE_F32) return wide ? launch_logit_rules<HOLO_DTYPE_F32, 4>(ctx, p) : launch_logit_rules<HOLO_DTYPE_F32, 1>(ctx, p);
    if (a.dtype == HOLO_DTYPE_BF16) return wide ? launch_logit_rules<HOLO_DTYPE_BF16, 8>(ctx, p) : launch_logit_rules<HOLO_DTYPE_BF16, 1>(ctx, p);
    return wide ? launch_logit_rules<HOLO_DTYPE_F16, 8>(ctx, p) : launch_logit_rules<HOLO_DTYPE_F16, 1>(ctx, p);
}
