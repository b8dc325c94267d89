// kvb_linear.cu -- linear attention with a decay for each head: a state per sequence and head instead of a cache.
//
//   S_t = lambda S_{t-1} + k_t v_t^T,   o_t = scale * q_t S_t,   lambda = exp(log_decay[head])
//
// S is [head_dim of k][head_dim of v] in fp32.  This file has the recurrent form, one token after another: a call of single tokens is
// bound by the state, which is read and written once (64 KB each way for a head of 128 dims).  Measured on B200, graph replay, 32 value heads of 128
// dims: 64 sequences 48 us, 5.6 TB/s, 86 % of a copy; one sequence 2.7 us, the latency of a launch, a read, two sums over warps and a write.
#include <cmath>

#include "kvb_linear.cuh"

namespace kvb {

int check_linear(const kvb_linear* L, const char* who) {
    if (L == nullptr) return fail(KVB_EINVAL, "%s: null layer", who);
    if (L->state == nullptr || L->log_decay == nullptr) return fail(KVB_EINVAL, "%s: null state / log_decay", who);
    if ((reinterpret_cast<uintptr_t>(L->state) & 15u) != 0) return fail(KVB_EINVAL, "%s: the state starts at a 16-byte boundary", who);
    if (L->head_dim != 64 && L->head_dim != 128) return fail(KVB_EINVAL, "%s: head_dim %d unsupported (64 or 128)", who, L->head_dim);
    if (L->qk_heads < 1 || L->v_heads < L->qk_heads || L->v_heads % L->qk_heads != 0 || L->v_heads > 256)
        return fail(KVB_EINVAL, "%s: v_heads %d must be qk_heads (%d) * (1..), at most 256", who, L->v_heads, L->qk_heads);
    if (L->slots < 1) return fail(KVB_EINVAL, "%s: slots %d", who, L->slots);
    if (L->dtype != KVB_DTYPE_F16 && L->dtype != KVB_DTYPE_BF16) return fail(KVB_EINVAL, "%s: dtype %d", who, L->dtype);
    return KVB_OK;
}

namespace {

constexpr int kStepThreads = 256;

// One CTA has kCols columns of the state of one sequence and head, in registers, for all tokens of the sequence; thread (row group, four columns).  The
// rows of q, k (whole) and v (its columns) of a token go through shared memory, asked for a token ahead; the sums over the state's rows by shuffles, then
// shared memory.
template <int D, int kCols, bool kBf16>
__global__ void __launch_bounds__(kStepThreads) step_kernel(LinearView L) {
    constexpr int kVecs = kCols / 4, kGroups = kStepThreads / kVecs, kRows = D / kGroups;
    static_assert(kRows >= 1 && kVecs <= 32 && kGroups * kRows == D, "threads cover the columns");
    __shared__ float qs[D], ks[D], vs[kCols];
    __shared__ float4 sums[kStepThreads / 32][kVecs];
    grid_dependency_wait();
    launch_dependents();
    const int seq = blockIdx.z, head = blockIdx.y, col0 = blockIdx.x * kCols, tid = threadIdx.x;
    const Sequence s = L.sequence(seq);
    if (!s.valid) return;
    const float g = L.log_decay[head], lambda = expf(g);
    if (!L.decay_fits(g)) return;
    const int vec = tid % kVecs, group = tid / kVecs;
    const float* from = L.state_of(s.from, head) + col0 + 4 * vec;
    float* to = L.state_of(s.to, head) + col0 + 4 * vec;
    float4 S[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) S[r] = *reinterpret_cast<const float4*>(from + (group + r * kGroups) * D);
    const int qk_head = head / L.share;
    constexpr int kEach = (2 * D + kCols + kStepThreads - 1) / kStepThreads;  // elements of a token's rows, a thread
    uint16_t row[kEach];
    auto ask = [&](int64_t t) {
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int i = tid + n * kStepThreads;
            if (i < D) row[n] = L.q[t * L.q_stride + qk_head * D + i];
            else if (i < 2 * D) row[n] = L.k[t * L.k_stride + qk_head * D + i - D];
            else if (i < 2 * D + kCols) row[n] = L.v[t * L.v_stride + head * D + col0 + i - 2 * D];
        }
    };
    if (s.begin < s.end) ask(s.begin);
    for (int t = s.begin; t < s.end; ++t) {
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int i = tid + n * kStepThreads;
            if (i < 2 * D + kCols) (i < D ? qs[i] : i < 2 * D ? ks[i - D] : vs[i - 2 * D]) = in_to_f32<kBf16>(row[n]);
        }
        __syncthreads();
        if (t + 1 < s.end) ask(t + 1);
        const float4 v = make_float4(vs[4 * vec], vs[4 * vec + 1], vs[4 * vec + 2], vs[4 * vec + 3]);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const float k = ks[group + r * kGroups], q = qs[group + r * kGroups];
            S[r].x = fmaf(S[r].x, lambda, k * v.x);
            S[r].y = fmaf(S[r].y, lambda, k * v.y);
            S[r].z = fmaf(S[r].z, lambda, k * v.z);
            S[r].w = fmaf(S[r].w, lambda, k * v.w);
            o.x = fmaf(q, S[r].x, o.x);
            o.y = fmaf(q, S[r].y, o.y);
            o.z = fmaf(q, S[r].z, o.z);
            o.w = fmaf(q, S[r].w, o.w);
        }
#pragma unroll
        for (int step = kVecs; step < 32; step <<= 1) {
            o.x += __shfl_xor_sync(0xffffffffu, o.x, step);
            o.y += __shfl_xor_sync(0xffffffffu, o.y, step);
            o.z += __shfl_xor_sync(0xffffffffu, o.z, step);
            o.w += __shfl_xor_sync(0xffffffffu, o.w, step);
        }
        if ((tid & 31) < kVecs) sums[tid >> 5][vec] = o;
        __syncthreads();
        if (tid < kCols) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kStepThreads / 32; ++w) sum += reinterpret_cast<const float*>(sums[w])[tid];
            L.out[static_cast<int64_t>(t) * L.v_heads * D + head * D + col0 + tid] = f32_to_out<kBf16>(sum * L.scale);
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) *reinterpret_cast<float4*>(to + (group + r * kGroups) * D) = S[r];
}

template <int D, int kCols> int launch_step(const LinearView& V, bool bf16, cudaStream_t stream) {
    const dim3 grid(D / kCols, V.v_heads, V.batch);
    KVB_CUDA_OK(launch_early(bf16 ? step_kernel<D, kCols, true> : step_kernel<D, kCols, false>, grid, dim3(kStepThreads), 0, stream, V));
    return KVB_OK;
}

int linear_call(const kvb_linear* layer, const char* who, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                const int32_t* offsets, int batch, int tokens, const int32_t* reads, const int32_t* writes, float scale, void* workspace, void* out, cudaStream_t stream) {
    if (int st = check_linear(layer, who)) return st;
    if (batch < 0 || tokens < 0) return fail(KVB_EINVAL, "%s: batch = %d, tokens = %d", who, batch, tokens);
    if (batch == 0) return KVB_OK;
    if (batch > kMostSequences) return fail(KVB_ERANGE, "%s: batch = %d (at most %d)", who, batch, kMostSequences);
    if (reads == nullptr || writes == nullptr) return fail(KVB_EINVAL, "%s: null slots", who);
    if (tokens > 0 && (q == nullptr || k == nullptr || v == nullptr || out == nullptr)) return fail(KVB_EINVAL, "%s: null q / k / v / out", who);
    const int D = layer->head_dim;
    const int64_t qk_width = static_cast<int64_t>(layer->qk_heads) * D, v_width = static_cast<int64_t>(layer->v_heads) * D;
    if (tokens > 1 && (q_stride < qk_width || k_stride < qk_width || v_stride < v_width)) return fail(KVB_EINVAL, "%s: a row is longer than the distance to the next", who);
    if (tokens > 0) {
        const Span written = span_of(out, sizeof(uint16_t) * static_cast<size_t>(tokens) * v_width);
        const Span state = span_of(layer->state, sizeof(float) * static_cast<size_t>(layer->slots) * layer->v_heads * D * D);
        if (overlap(written, rows_span(q, tokens, q_stride, qk_width)) || overlap(written, rows_span(k, tokens, k_stride, qk_width)) ||
            overlap(written, rows_span(v, tokens, v_stride, v_width)) || overlap(written, state))
            return fail(KVB_EINVAL, "%s: out shares memory with an input or the state", who);
    }
    LinearView V;
    V.state = layer->state;
    V.log_decay = layer->log_decay;
    V.q = static_cast<const uint16_t*>(q);
    V.k = static_cast<const uint16_t*>(k);
    V.v = static_cast<const uint16_t*>(v);
    V.out = static_cast<uint16_t*>(out);
    V.q_stride = q_stride;
    V.k_stride = k_stride;
    V.v_stride = v_stride;
    V.offsets = offsets;
    V.reads = reads;
    V.writes = writes;
    V.scale = scale;
    V.batch = batch;
    V.tokens = tokens;
    V.slots = layer->slots;
    V.v_heads = layer->v_heads;
    V.share = layer->v_heads / layer->qk_heads;
    V.head_dim = D;
    V.error_word = layer->error_word;
    const bool bf = layer->dtype == KVB_DTYPE_BF16;
    // Few tokens a sequence go one after another (verify steps of up to eight rows always): a token costs 0.4 .. 1.1 us, by how many heads and
    // sequences share the device, a call of the chunked form 7 us (64 dims) or 10 a wave of its CTAs, one an SM.  Measured on B200, 32 value heads, us one
    // after another / in chunks at the tokens where they meet: 64 dims 1 sequence 12 6.9 / 6.9, 2 8 7.2 / 6.9, 4 5 7.2 / 7.3, 8 8 13.0 / 13.3; 128 dims 1
    // 17 9.0 / 10.0, 2 11 10.3 / 10.3, 4 7 10.6 / 10.6, 8 10 22.5 / 22.6, 16 12 44.2 / 43.7.  The lines between them lie within 2.5 us of the better form
    // for sequences of equal lengths, and go by the mean: the host has no others.  A prompt of 300 tokens packed with 63 single ones goes one after another,
    // 252 us; 18 and 48 in calls of their own.
    const int64_t units = static_cast<int64_t>(batch) * layer->v_heads, sms = device_sm_count();
    const int few = units <= sms / 3 ? 12 : units <= sms ? 8 : 10;
    if (offsets != nullptr && static_cast<int64_t>(tokens) > static_cast<int64_t>(few) * batch) {
        if (workspace == nullptr) return fail(KVB_EINVAL, "%s: null workspace", who);
        const bool aligned = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 && q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0;
        return linear_chunks(V, bf, aligned, workspace, stream);
    }
    if (D == 128) return static_cast<int64_t>(batch) * layer->v_heads < 2 * device_sm_count() ? launch_step<128, 32>(V, bf, stream) : launch_step<128, 128>(V, bf, stream);
    return static_cast<int64_t>(batch) * layer->v_heads < 2 * device_sm_count() ? launch_step<64, 16>(V, bf, stream) : launch_step<64, 64>(V, bf, stream);
}

}  // namespace
}  // namespace kvb

extern "C" int kvb_linear_decode(const kvb_linear* layer, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride, int batch,
                                 const int32_t* reads_dev, const int32_t* writes_dev, float scale, void* out, void* stream) {
    return kvb::linear_call(layer, "kvb_linear_decode", q, q_stride, k, k_stride, v, v_stride, nullptr, batch, batch, reads_dev, writes_dev, scale, nullptr, out,
                            static_cast<cudaStream_t>(stream));
}

extern "C" int kvb_linear_chunk(const kvb_linear* layer, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                const int32_t* offsets_dev, int batch, int tokens, const int32_t* reads_dev, const int32_t* writes_dev, float scale, void* workspace,
                                void* out, void* stream) {
    using namespace kvb;
    if (batch > 0 && offsets_dev == nullptr) return fail(KVB_EINVAL, "kvb_linear_chunk: null offsets");
    return linear_call(layer, "kvb_linear_chunk", q, q_stride, k, k_stride, v, v_stride, offsets_dev, batch, tokens, reads_dev, writes_dev, scale, workspace, out,
                       static_cast<cudaStream_t>(stream));
}

extern "C" size_t kvb_linear_workspace_bytes(int tokens, int batch, int v_heads, int head_dim) {
    using namespace kvb;
    if (tokens < 1 || batch < 1 || v_heads < 1 || (head_dim != 64 && head_dim != 128)) return kWorkspaceSlack;
    const int segment = linear_segment(tokens, batch, v_heads);
    if (tokens <= segment) return kWorkspaceSlack;
    return sizeof(float) * static_cast<size_t>(linear_units(tokens, batch, segment)) * v_heads * head_dim * head_dim + kWorkspaceSlack;
}
