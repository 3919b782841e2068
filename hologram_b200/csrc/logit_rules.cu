// Rules on logits before a token is chosen (the LogitRules call): penalties for repeated tokens, biases, temperature, grammar masks.
//
// A CTA takes a row's part of the vocabulary: it counts the history's tokens that fall into it in shared memory, notes which bias
// entry each token has (the last that names it: integer maxima, so no order of threads shows), then streams the logits once.
#include "sequences.cuh"

namespace {

constexpr int RULES_THREADS = 256;
constexpr uint32_t RULES_PART = 8192;         // tokens of a CTA
constexpr uint32_t IN_PROMPT = 0x80000000u;   // of a count: the token stands in the prompt; the rest counts it behind the prompt

__global__ void __launch_bounds__(RULES_THREADS)
logit_rules_kernel(const __grid_constant__ HoloLogitRulesArgs a) {
    extern __shared__ uint32_t s_words[];     // counts, then bias entries + 1
    const uint32_t tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * RULES_PART, n = min(RULES_PART, a.vocab - first);
    uint32_t *s_count = s_words, *s_bias = s_words + RULES_PART;
    holo_pdl_trigger();
    holo_pdl_wait();
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
        const float* p = a.params + 4 * (uint64_t)row;
        repetition = p[0]; presence = p[1]; frequency = p[2]; temperature = p[3];
    }
    const bool counts = total > 0, biases = to > from;
    if (counts)
        for (uint32_t i = tid; i < n; i += RULES_THREADS) s_count[i] = 0;
    if (biases)
        for (uint32_t i = tid; i < n; i += RULES_THREADS) s_bias[i] = 0;
    __syncthreads();
    const int32_t* history = a.history + (uint64_t)row * a.history_ld;
    for (int i = (int)tid; i < total; i += RULES_THREADS) {
        const uint32_t t = (uint32_t)history[i] - first;
        if ((uint32_t)history[i] >= first && t < n) {
            if (i < prompt) atomicOr(s_count + t, IN_PROMPT);
            else atomicAdd(s_count + t, 1u);
        }
    }
    for (int i = from + (int)tid; i < to; i += RULES_THREADS) {
        const uint32_t t = (uint32_t)a.bias_ids[i] - first;
        if ((uint32_t)a.bias_ids[i] >= first && t < n) atomicMax(s_bias + t, (uint32_t)i + 1);
    }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += RULES_THREADS) {
        float z = seq_load(a.logits, (uint64_t)row * a.ld + first + i, a.dtype);
        const uint32_t c = counts ? s_count[i] : 0u, made = c & ~IN_PROMPT;
        if (c) z = z > 0.0f ? __fdiv_rn(z, repetition) : z * repetition;
        if (made) z -= fmaf(frequency, (float)made, presence);
        if (biases && s_bias[i]) z += a.bias_values[s_bias[i] - 1];
        if (temperature > 0.0f) z = __fdiv_rn(z, temperature);
        if (mask && !(mask[(first + i) >> 5] >> ((first + i) & 31u) & 1u)) z = -INFINITY;
        seq_store(a.out, (uint64_t)row * a.out_ld + first + i, z, a.dtype);
    }
}

}  // namespace

int32_t holo_launch_logit_rules(holo_b200_ctx* ctx, const HoloLogitRulesArgs& a) {
    if (a.rows > 65535) return holo_fail(HOLO_ERR_UNSUPPORTED_OP, "unsupported op: logit_rules of %u rows", a.rows);
    const uint32_t smem = RULES_PART * 8;
    static thread_local int configured_device = -1;
    if (configured_device != ctx->device) {
        HOLO_CUDA(cudaFuncSetAttribute(logit_rules_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        configured_device = ctx->device;
    }
    HOLO_CUDA(holo_launch_kernel(ctx, logit_rules_kernel, dim3((a.vocab + RULES_PART - 1) / RULES_PART, a.rows), dim3(RULES_THREADS), smem, 1, a));
    ctx->launches++;
    return HOLO_OK;
}
