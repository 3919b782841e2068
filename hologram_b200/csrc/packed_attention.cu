// Attention of whole sequences of different lengths packed one behind another (the PackedAttention call).
#include "sequences.cuh"

namespace {

struct PackedSource {
    HoloPackedArgs a;
    struct Place {
        uint32_t begin, end;
    };
    __device__ uint32_t rows() const { return a.rows; }
    __device__ uint32_t heads() const { return a.heads; }
    __device__ uint32_t dim() const { return a.dim; }
    __device__ uint32_t vdim() const { return a.vdim; }
    __device__ float scale() const { return a.scale; }
    __device__ void check() const { check_sequences(a.starts, nullptr, a.sequences, a.rows, 0, a.status); }
    __device__ bool place(uint32_t row, Place* p) const {
        uint32_t which;
        if (!sequence_of(a.starts, a.sequences, a.rows, row, &p->begin, &p->end, &which)) return false;
        if (a.causal) p->end = row + 1;
        return true;
    }
    __device__ float q(uint32_t row, uint32_t head, uint32_t c) const { return seq_load(a.q, (uint64_t)row * a.q_ld + (uint64_t)head * a.dim + c, a.dtype); }
    __device__ void key(const Place&, uint32_t head, uint32_t j, uint64_t* kb, uint64_t* vb, float* ks, float* vs) const {
        const uint32_t g = head / (a.heads / a.kv_heads);
        *kb = (uint64_t)j * a.k_ld + (uint64_t)g * a.dim;
        *vb = (uint64_t)j * a.v_ld + (uint64_t)g * a.vdim;
        *ks = *vs = 1.0f;
    }
    __device__ float k(uint64_t i) const { return seq_load(a.k, i, a.dtype); }
    __device__ float v(uint64_t i) const { return seq_load(a.v, i, a.dtype); }
    __device__ void store(uint32_t row, uint32_t head, uint32_t c, float x) const { seq_store(a.out, (uint64_t)row * a.ld + (uint64_t)head * a.vdim + c, x, a.dtype); }
};

}  // namespace

int32_t holo_launch_packed_attention(holo_b200_ctx* ctx, const HoloPackedArgs& a) {
    bool taken;
    HOLO_TRY(holo_try_packed_tile(ctx, a, &taken));
    if (taken) return HOLO_OK;
    HOLO_TRY(holo_try_packed_f32(ctx, a, &taken));
    if (taken) return HOLO_OK;
    PackedSource src = {a};
    return launch_general_rows(ctx, src, (uint64_t)a.rows * a.heads, a.vdim);
}
