// kvb_linear.cuh -- what the kernels of linear attention share: the call's view, its sequences and their checks on the device.
#pragma once

#include "kvb_common.cuh"
#include "kvb_linear_plan.hpp"
#include "kvb_ptx.cuh"
#include "kvb_rope.cuh"

namespace kvb {

// Rows [begin, end) of one sequence and the slots its state is read from and written to.
struct Sequence {
    int begin, end, from, to;
    bool valid;
};

struct LinearView {
    float* state;            // [slots][v_heads][head_dim of k][head_dim of v]
    const float* log_decay;  // [v_heads]
    const uint16_t *q, *k, *v;
    uint16_t* out;
    int64_t q_stride, k_stride, v_stride;
    const int32_t *offsets, *reads, *writes;  // offsets null: one token each
    float scale;
    int batch, tokens, slots, v_heads, share, head_dim;
    uint32_t* error_word;

    __device__ __forceinline__ void flag(uint32_t bit) const {
        if (error_word != nullptr && threadIdx.x == 0) atomicOr(error_word, bit);
    }
    __device__ __forceinline__ float* state_of(int slot, int head) const { return state + (static_cast<int64_t>(slot) * v_heads + head) * head_dim * head_dim; }
    // The whole CTA asks.  A sequence is refused, its rows and state left as they are, where its rows are not inside the call's, a slot is not inside
    // the pool, or the slot it writes is one that another sequence of the call reads or writes.
    __device__ __forceinline__ Sequence sequence(int seq) const {
        Sequence s;
        s.begin = offsets != nullptr ? offsets[seq] : seq;
        s.end = offsets != nullptr ? offsets[seq + 1] : seq + 1;
        s.from = reads[seq];
        s.to = writes[seq];
        bool shared = false;
        for (int i = threadIdx.x; i < batch; i += blockDim.x)
            if (i != seq) shared = shared || writes[i] == s.to || reads[i] == s.to || writes[i] == s.from;
        s.valid = allowed(s, __syncthreads_or(shared) != 0);
        return s;
    }
    __device__ __forceinline__ bool allowed(const Sequence& s, bool shared) const {
        const bool rows = s.begin >= 0 && s.end >= s.begin && s.end <= tokens;
        const bool pool = s.from >= 0 && s.from < slots && s.to >= 0 && s.to < slots;
        if (!rows) flag(KVB_ERR_POSITIONS);
        if (!pool || shared) flag(KVB_ERR_SLOT);
        return rows && pool && !shared;
    }
    // exp(log_decay) is 0 .. 1; a head with another one is refused.
    __device__ __forceinline__ bool decay_fits(float log_decay_of_head) const {
        if (log_decay_of_head <= 0.0f) return true;
        flag(KVB_ERR_GEOMETRY);
        return false;
    }
};

// The chunked form: tokens of a segment on this device, and the launches.
inline int linear_segment(int tokens, int batch, int v_heads) { return linear_segment_of(tokens, batch, v_heads, device_sm_count()); }
int linear_chunks(const LinearView& V, bool bf16, bool aligned, void* workspace, cudaStream_t stream);

int check_linear(const kvb_linear* layer, const char* who);

}  // namespace kvb
