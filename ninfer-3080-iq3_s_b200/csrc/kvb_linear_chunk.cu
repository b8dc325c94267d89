// kvb_linear_chunk.cu -- linear attention with a decay for each head over prompts, chunk by chunk on the 5th-generation tensor cores.
//
// For a chunk of C = 128 tokens (rows i, j; L of them valid) behind a state S, with lambda = exp(log_decay):
//
//   P_ij  = lambda^(i-j) q_i k_j  (j <= i, else 0)                        scores          C x C
//   o_i   = scale (sum_j P_ij v_j + lambda^(i+1) q_i S)                   inside + before
//   S    <- lambda^L S + sum_j (lambda^(L-1-j) k_j) v_j^T                 the state behind the chunk
//
// Everything but the scores is computed transposed, head dims of v along the M rows of the MMAs: S^T stays in tensor memory as an fp32 accumulator from
// chunk to chunk, and is an A operand there too (two 16-bit numbers an element, whose sum has 16 bits of bf16 or 22 of fp16); only rows of
// tokens as they come from global memory, decayed keys (two 16-bit numbers likewise, so that states keep their precision over long prompts) and P lie in
// shared memory.  P is rounded to the type once, like the output.  Heads of 64 dims fill both halves of the M rows with the same 64.
//
// A sequence is split into segments where there are fewer heads and sequences than SMs: a first launch sums up each segment alone
// (keys and values only, half the reads of the second), the second starts each from the sums before it.
//
// In fp16 the scores of a row and the state's rows are scaled by a power of two to a largest magnitude of 2^14 .. 2^15 before they are rounded, so that
// neither overflows; the scales come out again in the sum of the two parts.  bf16 has the range of fp32.
#include "kvb_linear.cuh"
#include "kvb_tcgen05.cuh"

namespace kvb {
namespace {

constexpr int kC = kLinearChunk;  // tokens of a chunk
constexpr int kComputeWarps = 8, kMmaWarp = 8, kLoadWarps = 4;
constexpr int kComputeThreads = kComputeWarps * 32, kLoadThreads = kLoadWarps * 32;
constexpr int kChunkThreads = kComputeThreads + 32 + kLoadThreads;
constexpr uint32_t kTmemCols = 512;

template <int D> struct LinearSmem {
    static constexpr int kTileBytes = kC * D * 2;  // [D / 64][128 rows][128 bytes], 128-byte swizzle
    alignas(1024) unsigned char q[2][kTileBytes];
    unsigned char k[2][kTileBytes];                // keys, then the first numbers of the decayed keys
    unsigned char v[2][kTileBytes];
    unsigned char x[kC * kC * 2];                  // the second numbers of the decayed keys, then P
    float power[kC];                               // lambda^n
    float before[kC];                              // scale lambda^(i + 1)
    float inside[kC];                              // scale times what P's row i was scaled down by (fp16)
    uint16_t most[2][2][kC];                       // exponents of the largest magnitudes of a row of the state, of P, one a column half (fp16)
    uint64_t full[2], empty[2], keys_ready[2], scores, state_ready, scores_read, state_done, p_ready, out_full, out_read, most_ready[2], drained;
    uint32_t tmem_base;
    int abort_flag;
    int unit[3];
};

struct ChunkCall {
    LinearView V;
    float* sums;   // [unit][head][D][D]: each segment's sum; the last one's place holds the state before the first
    int segment;   // tokens, a multiple of kC
    bool aligned;  // rows of q, k, v keep to 16 bytes
};

// Sequence and segment of the call's unit `unit`, found by one warp; the same for all threads afterwards.  seq = batch: none.
struct Unit {
    int seq, index, count;  // segment `index` of `count`
};
__device__ __forceinline__ int segments_of(const ChunkCall& P, int seq) {
    const int begin = P.V.offsets[seq], end = P.V.offsets[seq + 1];
    const int64_t length = static_cast<int64_t>(end) - begin;
    return length <= 0 || length > P.V.tokens ? 1 : static_cast<int>((length + P.segment - 1) / P.segment);
}
__device__ __forceinline__ Unit unit_of(const ChunkCall& P, int unit, int (&shared)[3]) {
    if (threadIdx.x < 32) {
        int base = 0;
        bool found = false;
        for (int s0 = 0; s0 < P.V.batch; s0 += 32) {
            const int seq = s0 + static_cast<int>(threadIdx.x);
            const int count = seq < P.V.batch ? segments_of(P, seq) : 0;
            int sum = count;  // inclusive
#pragma unroll
            for (int step = 1; step < 32; step <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, step);
                if (static_cast<int>(threadIdx.x) >= step) sum += up;
            }
            const bool mine = unit >= base + sum - count && unit < base + sum;
            if (mine) shared[0] = seq, shared[1] = unit - (base + sum - count), shared[2] = count;
            found = __any_sync(0xffffffffu, mine) || found;
            base += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (!found && threadIdx.x == 0) shared[0] = P.V.batch, shared[1] = shared[2] = 0;
        // sequences that overlap have more segments than the grid has units: what is left out is reported
        if (unit == 0 && base > static_cast<int>(gridDim.x)) P.V.flag(KVB_ERR_POSITIONS);
    }
    __syncthreads();
    return Unit{shared[0], shared[1], shared[2]};
}

// exp(g n): 1 at n = 0, whatever g is.
__device__ __forceinline__ float decay_power(float g, int n) { return n == 0 ? 1.0f : expf(g * static_cast<float>(n)); }

template <bool kBf16> __device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    if constexpr (kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        return pack_half2(a, b);
    }
}
template <bool kBf16> __device__ __forceinline__ float2 unpack_pair(uint32_t w) {
    if constexpr (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return unpack_half2(w);
}
// Instruction descriptor of 16-bit operands of either type (format 0 = f16, 1 = bf16).
template <bool kBf16> __host__ __device__ constexpr uint32_t idesc_16(int m, int n, bool a_mn, bool b_mn) {
    return tc::idesc_f16(m, n, a_mn, b_mn) | (kBf16 ? (1u << 7) | (1u << 10) : 0u);
}
// 2^-e and 2^e for the e that brings magnitudes with this largest exponent field below 2^15; 1 where it is 0's or not finite.
__device__ __forceinline__ float2 down_and_up(int field) {
    const int e = field > 0 && field < 255 ? max(-112, min(112, field - 127 - 14)) : 0;
    return make_float2(__uint_as_float(static_cast<uint32_t>(127 - e) << 23), __uint_as_float(static_cast<uint32_t>(127 + e) << 23));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// Rows of a chunk into a tile, zeros behind the valid ones.
template <int D> __device__ __forceinline__ void load_tile(unsigned char* tile, const uint16_t* rows, int64_t stride, int valid, bool aligned) {
    constexpr int kUnits = D / 8;  // 16 bytes each, of a row
    const int tid = threadIdx.x - kComputeThreads - 32;
    if (aligned) {
        const uint32_t base = smem_u32(tile);
#pragma unroll 8
        for (int u = tid; u < kC * kUnits; u += kLoadThreads) {
            const int row = u / kUnits, c = u % kUnits;
            const bool in = row < valid;
            cp_async16(base + (c >> 3) * (kC * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4), rows + (in ? row : 0) * stride + 8 * c, in ? 16u : 0u);
        }
    } else {
        for (int u = tid; u < kC * kUnits; u += kLoadThreads) {
            const int row = u / kUnits, c = u % kUnits;
            uint32_t w[4] = {0u, 0u, 0u, 0u};
            if (row < valid) {
                const uint16_t* from = rows + row * stride + 8 * c;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = static_cast<uint32_t>(from[2 * e]) | static_cast<uint32_t>(from[2 * e + 1]) << 16;
            }
            *reinterpret_cast<uint4*>(tile + (c >> 3) * (kC * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// Sum of P_ij v_j over j <= i for a value that came out not finite: a value of a later row that is not finite meets a 0 of P in the product.
template <bool kBf16> __device__ __noinline__ float inside_again(const unsigned char* p, int i, const uint16_t* v, int64_t stride) {
    float sum = 0.0f;
    for (int j = 0; j <= i; ++j) {
        const uint16_t w = *reinterpret_cast<const uint16_t*>(p + (j >> 6) * (kC * 128) + i * 128 + ((((j & 63) >> 3) ^ (i & 7)) << 4) + (j & 7) * 2);
        sum = fmaf(in_to_f32<kBf16>(w), in_to_f32<kBf16>(v[j * stride]), sum);
    }
    return sum;
}

// kSums: the first launch, sums of segments; else the outputs and the state behind each sequence.
template <int D, bool kBf16, bool kSums>
__global__ void __launch_bounds__(kChunkThreads, 1) chunk_kernel(const ChunkCall P) {
    using Smem = LinearSmem<D>;
    constexpr int kHalf = D / 2;                    // columns of the state a compute warp has
    constexpr uint32_t kStateCol = 0, kFirstCol = D, kSecondCol = D + D / 2, kScoreCol = 2 * D, kOutCol = 2 * D + kC;
    static_assert(kOutCol + kC <= kTmemCols, "tensor memory");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    grid_dependency_wait();
    launch_dependents();
    const LinearView& V = P.V;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.y;
    const Unit unit = unit_of(P, blockIdx.x, sm.unit);
    if (unit.seq >= V.batch) return;
    if (kSums && unit.count == 1) return;
    const Sequence seq = V.sequence(unit.seq);
    float lambda;
    if (!seq.valid || !V.decay_of(head, &lambda)) return;
    if ((smem_u32(smem_raw) & 1023u) != 0) {  // the swizzle needs it; the launch asks for nothing beside it
        V.flag(KVB_ERR_GEOMETRY);
        return;
    }
    const float g = V.log_decay[head];
    const bool last_segment = unit.index == unit.count - 1;
    const int begin = seq.begin + unit.index * P.segment, end = last_segment ? seq.end : begin + P.segment;
    const int chunks = kSums && last_segment ? 0 : (end - begin + kC - 1) / kC;
    float* const sums = P.sums + (static_cast<int64_t>(blockIdx.x) * V.v_heads + head) * D * D;  // this segment's; earlier ones lie in front
    const int64_t sums_step = static_cast<int64_t>(V.v_heads) * D * D;

    if (warp == kMmaWarp) tc::tmem_alloc(&sm.tmem_base, kTmemCols);
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.full[s], kLoadThreads);
            mbar_init(&sm.empty[s], 1);
            mbar_init(&sm.keys_ready[s], kComputeThreads);
            mbar_init(&sm.most_ready[s], kComputeThreads);
        }
        mbar_init(&sm.scores, 1);
        mbar_init(&sm.state_done, 1);
        mbar_init(&sm.out_full, 1);
        mbar_init(&sm.drained, 1);
        mbar_init(&sm.state_ready, kComputeThreads);
        mbar_init(&sm.scores_read, kComputeThreads);
        mbar_init(&sm.p_ready, kComputeThreads);
        mbar_init(&sm.out_read, kComputeThreads);
        mbar_fence_init();
        sm.abort_flag = 0;
    }
    if (threadIdx.x < kC) {
        const int n = threadIdx.x;
        sm.power[n] = decay_power(g, n);
        sm.before[n] = V.scale * decay_power(g, n + 1);
        sm.inside[n] = V.scale;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sm.tmem_base;
    bool failed = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!failed && !chunk_wait(bar, parity, &sm.abort_flag)) failed = true;
        return !failed;
    };

    if (warp > kMmaWarp) {
        // ---- loads: chunk c into stage c & 1; a chunk is announced once its copies have landed, a chunk later
        const uint16_t* const q = V.q + static_cast<int64_t>(head / V.share) * D;
        const uint16_t* const k = V.k + static_cast<int64_t>(head / V.share) * D;
        const uint16_t* const v = V.v + static_cast<int64_t>(head) * D;
        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1, t = begin + c * kC, valid = min(kC, end - t);
            if (c > 1 && !wait(&sm.empty[st], ((c >> 1) + 1) & 1)) break;
            load_tile<D>(sm.k[st], k + t * V.k_stride, V.k_stride, valid, P.aligned);
            load_tile<D>(sm.v[st], v + t * V.v_stride, V.v_stride, valid, P.aligned);
            if (!kSums) load_tile<D>(sm.q[st], q + t * V.q_stride, V.q_stride, valid, P.aligned);
            cp_async_commit();
            if (c > 0) {
                cp_async_wait<1>();
                fence_proxy_async();
                mbar_arrive(&sm.full[st ^ 1]);
            }
        }
        cp_async_wait<0>();
        fence_proxy_async();
        if (!failed && chunks > 0) mbar_arrive(&sm.full[(chunks - 1) & 1]);
    } else if (warp == kMmaWarp) {
        // ---- MMAs, issued by one thread
        const uint64_t q0 = tc::smem_desc(smem_u32(sm.q[0]), 16, 1024), k0 = tc::smem_desc(smem_u32(sm.k[0]), 16, 1024), p0 = tc::smem_desc(smem_u32(sm.x), 16, 1024);
        // MN-major: the next 64 head dims a tile half further (heads of 64 dims: the same ones again), the next 8 tokens 1024 bytes
        const uint64_t v0 = tc::smem_desc(smem_u32(sm.v[0]), D == 128 ? kC * 128 : 0, 1024);
        const uint64_t key0 = tc::smem_desc(smem_u32(sm.k[0]), kC * 128, 1024);
        const uint64_t second0 = kSums ? tc::smem_desc(smem_u32(sm.q[0]), kC * 128, 1024) : tc::smem_desc(smem_u32(sm.x), kC * 128, 1024);
        constexpr uint32_t kScores = idesc_16<kBf16>(128, kC, false, false), kState = idesc_16<kBf16>(128, D, true, true), kOut = idesc_16<kBf16>(128, kC, true, false);
        auto k_major = [](uint64_t desc, int step) { return tc::desc_at(desc, (step >> 2) * (kC * 128) + (step & 3) * 32); };  // 16 of the K dims further
        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1, at = st * Smem::kTileBytes;
            if (!kSums) {
                if (!wait(&sm.full[st], (c >> 1) & 1)) break;
                if (c > 0 && !wait(&sm.out_read, (c - 1) & 1)) break;
                tc::fence_after_sync();
                if (tc::elect_one()) {
                    const uint64_t a = tc::desc_here(tc::desc_at(q0, at)), b = tc::desc_here(tc::desc_at(k0, at));
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) tc::mma_f16_ss(tmem + kScoreCol, k_major(a, s), k_major(b, s), kScores, s > 0);
                    tc::commit(&sm.scores);
                }
                __syncwarp();
                if (!wait(&sm.state_ready, c & 1)) break;
            }
            if (!wait(&sm.keys_ready[st], (c >> 1) & 1)) break;
            tc::fence_after_sync();
            if (tc::elect_one()) {
                const uint64_t a = tc::desc_here(tc::desc_at(v0, at)), b = tc::desc_here(tc::desc_at(key0, at)), b2 = tc::desc_here(kSums ? tc::desc_at(second0, at) : second0);
#pragma unroll
                for (int s = 0; s < kC / 16; ++s) tc::mma_f16_ss(tmem + kStateCol, tc::desc_at(a, s * 2048), tc::desc_at(b, s * 2048), kState, !kSums || c > 0 || s > 0);
#pragma unroll
                for (int s = 0; s < kC / 16; ++s) tc::mma_f16_ss(tmem + kStateCol, tc::desc_at(a, s * 2048), tc::desc_at(b2, s * 2048), kState, true);
                if (kSums) tc::commit(&sm.empty[st]);
                if (!kSums || c == chunks - 1) tc::commit(&sm.state_done);
            }
            __syncwarp();
            if (kSums) continue;
            if (!wait(&sm.scores_read, c & 1)) break;
            tc::fence_after_sync();
            if (tc::elect_one()) {
                const uint64_t b = tc::desc_here(tc::desc_at(q0, at));
#pragma unroll
                for (int s = 0; s < D / 16; ++s) tc::mma_f16_ts(tmem + kScoreCol, tmem + kFirstCol + 8 * s, k_major(b, s), kScores, s > 0);
#pragma unroll
                for (int s = 0; s < D / 16; ++s) tc::mma_f16_ts(tmem + kScoreCol, tmem + kSecondCol + 8 * s, k_major(b, s), kScores, true);
            }
            __syncwarp();
            if (!wait(&sm.p_ready, c & 1)) break;
            tc::fence_after_sync();
            if (tc::elect_one()) {
                const uint64_t a = tc::desc_here(tc::desc_at(v0, at)), b = tc::desc_here(p0);
#pragma unroll
                for (int s = 0; s < kC / 16; ++s) tc::mma_f16_ss(tmem + kOutCol, tc::desc_at(a, s * 2048), k_major(b, s), kOut, s > 0);
                tc::commit(&sm.out_full);
                tc::commit(&sm.empty[st]);
            }
            __syncwarp();
        }
        if (failed) {  // nothing is freed under MMAs that still run
            if (tc::elect_one()) tc::commit(&sm.drained);
            __syncwarp();
            mbar_wait_bounded(&sm.drained, 0);
        }
    } else {
        // ---- the eight other warps: rows 32 (warp % 4) + lane of tensor memory, columns by warp / 4
        const int quad = warp & 3, side = warp >> 2, row = 32 * quad + lane, dim = row % D, tid = threadIdx.x;
        const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
        const uint32_t state_at = tmem + lanes + kStateCol + side * kHalf;

        if (!kSums || last_segment) {
            // the state before the segment, rows of S^T: from the pool, or the sums of the segments before
            const float* from = V.state_of(seq.from, head);
            if (!kSums && unit.count > 1 && unit.index == 0) from = sums + (unit.count - 1) * sums_step;
#pragma unroll 1
            for (int b = 0; b < kHalf / 32; ++b) {
                uint32_t r[32];
                const int col = side * kHalf + 32 * b;
                if (kSums || unit.index == 0) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(from[(col + e) * D + dim]);
                } else {
                    float f[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) f[e] = 0.0f;
                    for (int s = 0; s < unit.index; ++s) {
                        const float* sum = sums - (unit.index - s) * sums_step;
                        const float w = decay_power(g, (unit.index - 1 - s) * P.segment);
#pragma unroll
                        for (int e = 0; e < 32; ++e) f[e] = fmaf(w, sum[(col + e) * D + dim], f[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(f[e]);
                }
                if (kSums) {  // the last segment's place keeps the state for the second launch, which may write over it
                    if (row < D) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) sums[(col + e) * D + dim] = __uint_as_float(r[e]);
                    }
                } else {
                    tc::tmem_st32(state_at + 32 * b, r);
                }
            }
            tc::tmem_st_wait();
        }
        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1, t = begin + c * kC, valid = min(kC, end - t);
            float up = 1.0f;  // what this row of the state was scaled down by
            if (!kSums) {
                // ---- the state as an operand, and decayed over the chunk
                if (c > 0 && !wait(&sm.state_done, (c - 1) & 1)) break;
                tc::fence_after_sync();
                const float decay = decay_power(g, valid);
                float down = 1.0f;
                if constexpr (!kBf16) {
                    float most = 0.0f;
#pragma unroll 1
                    for (int b = 0; b < kHalf / 32; ++b) {
                        uint32_t r[32];
                        tc::tmem_ld32(state_at + 32 * b, r);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) most = fmaxf(most, fabsf(__uint_as_float(r[e])));
                    }
                    const int mine = static_cast<int>(__float_as_uint(most) >> 23);
                    sm.most[0][side][row] = static_cast<uint16_t>(mine);
                    mbar_arrive(&sm.most_ready[0]);
                    if (!wait(&sm.most_ready[0], c & 1)) break;
                    const float2 s = down_and_up(max(mine, static_cast<int>(sm.most[0][side ^ 1][row])));
                    down = s.x;
                    up = s.y;
                }
#pragma unroll 1
                for (int b = 0; b < kHalf / 32; ++b) {
                    uint32_t r[32], first[16], second[16];
                    tc::tmem_ld32(state_at + 32 * b, r);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float x = __uint_as_float(r[2 * e]), y = __uint_as_float(r[2 * e + 1]);
                        r[2 * e] = __float_as_uint(x * decay);
                        r[2 * e + 1] = __float_as_uint(y * decay);
                        if constexpr (!kBf16) x *= down, y *= down;
                        first[e] = pack_pair<kBf16>(x, y);
                        const float2 f = unpack_pair<kBf16>(first[e]);
                        second[e] = pack_pair<kBf16>(x - f.x, y - f.y);
                    }
                    tc::tmem_st32(state_at + 32 * b, r);
                    tc::tmem_st16(tmem + lanes + kFirstCol + (side * kHalf + 32 * b) / 2, first);
                    tc::tmem_st16(tmem + lanes + kSecondCol + (side * kHalf + 32 * b) / 2, second);
                }
                tc::tmem_st_wait();
                tc::fence_before_sync();
                mbar_arrive(&sm.state_ready);
                if (!wait(&sm.scores, c & 1)) break;  // the keys have been read, too
                tc::fence_after_sync();
            }
            if (!wait(&sm.full[st], (c >> 1) & 1)) break;
            // ---- decayed keys: the first numbers in the keys' place, the second beside them
            {
                unsigned char* const keys = sm.k[st];
                unsigned char* const second = kSums ? sm.q[st] : sm.x;
                constexpr int kEach = kC * D / 8 / kComputeThreads;
#pragma unroll
                for (int n = 0; n < kEach; ++n) {
                    const int u = tid + n * kComputeThreads, j = (u >> 3) & (kC - 1);
                    const float w = kSums ? (j < valid ? decay_power(g, end - 1 - t - j) : 0.0f) : (j < valid ? sm.power[valid - 1 - j] : 0.0f);
                    const uint4 raw = *reinterpret_cast<const uint4*>(keys + 16 * u);
                    const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
                    uint32_t a[4], b[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = unpack_pair<kBf16>(in[e]);
                        const float x = f.x * w, y = f.y * w;
                        a[e] = pack_pair<kBf16>(x, y);
                        const float2 h = unpack_pair<kBf16>(a[e]);
                        b[e] = pack_pair<kBf16>(x - h.x, y - h.y);
                    }
                    *reinterpret_cast<uint4*>(keys + 16 * u) = make_uint4(a[0], a[1], a[2], a[3]);
                    *reinterpret_cast<uint4*>(second + 16 * u) = make_uint4(b[0], b[1], b[2], b[3]);
                }
                fence_proxy_async();
                mbar_arrive(&sm.keys_ready[st]);
            }
            if (kSums) continue;
            // ---- P: row `row`, 64 columns
            uint32_t p[32];
            {
                float most = 0.0f;
                uint32_t s[2][32];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int j0 = 64 * side + 32 * b;
                    if (j0 <= 32 * quad + 31) {  // a block with something on or below the diagonal
                        tc::tmem_ld32(tmem + lanes + kScoreCol + j0, s[b]);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int n = row - j0 - e;
                            const float x = n >= 0 ? __uint_as_float(s[b][e]) * sm.power[n & (kC - 1)] : 0.0f;
                            if constexpr (!kBf16) most = fmaxf(most, fabsf(x));
                            s[b][e] = __float_as_uint(x);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[b][e] = 0u;
                    }
                }
                tc::fence_before_sync();
                mbar_arrive(&sm.scores_read);
                float down = 1.0f;
                if constexpr (!kBf16) {
                    const int mine = static_cast<int>(__float_as_uint(most) >> 23);
                    sm.most[1][side][row] = static_cast<uint16_t>(mine);
                    mbar_arrive(&sm.most_ready[1]);
                    if (!wait(&sm.most_ready[1], c & 1)) break;
                    const float2 f = down_and_up(max(mine, static_cast<int>(sm.most[1][side ^ 1][row])));
                    down = f.x;
                    if (side == 0) sm.inside[row] = V.scale * f.y;
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float x = __uint_as_float(s[e >> 4][2 * (e & 15)]), y = __uint_as_float(s[e >> 4][2 * (e & 15) + 1]);
                    if constexpr (!kBf16) x *= down, y *= down;
                    p[e] = pack_pair<kBf16>(x, y);
                }
            }
            if (!wait(&sm.state_done, c & 1)) break;  // the second numbers of the keys have been read
            {
                unsigned char* const to = sm.x + side * (kC * 128) + row * 128;
#pragma unroll
                for (int u = 0; u < 8; ++u) *reinterpret_cast<uint4*>(to + ((u ^ (row & 7)) << 4)) = make_uint4(p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]);
                fence_proxy_async();
                mbar_arrive(&sm.p_ready);
            }
            if (!kBf16 && !wait(&sm.p_ready, c & 1)) break;  // sm.inside of all rows
            // ---- the outputs: head dim `dim`, 64 tokens (heads of 64 dims, which are there twice: 32)
            if (!wait(&sm.out_full, c & 1)) break;
            tc::fence_after_sync();
            constexpr int kBlocks = D == 128 ? 2 : 1;
            const int i0 = D == 128 ? 64 * side : 64 * side + 32 * (quad >> 1);
            uint16_t* const out = V.out + (static_cast<int64_t>(t) * V.v_heads + head) * D + dim;
            const int64_t out_stride = static_cast<int64_t>(V.v_heads) * D;
#pragma unroll 1
            for (int b = 0; b < kBlocks; ++b) {
                const int i1 = i0 + 32 * b;
                uint32_t r[32], s[32];
                tc::tmem_ld32(tmem + lanes + kOutCol + i1, r);
                tc::tmem_ld32(tmem + lanes + kScoreCol + i1, s);
                tc::tmem_ld_wait();
                float zero = 0.0f;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float in = kBf16 ? V.scale : sm.inside[i1 + e];
                    const float y = fmaf(__uint_as_float(r[e]), in, __uint_as_float(s[e]) * (sm.before[i1 + e] * up));
                    zero = fmaf(y, 0.0f, zero);
                    r[e] = __float_as_uint(y);
                }
                if (!(zero == 0.0f)) {
#pragma unroll 1
                    for (int e = 0; e < 32; ++e) {
                        const int i = i1 + e;
                        uint32_t word = 0;  // r[e], s[e] without an index into registers
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (x == e) word = r[x];
                        if ((word & 0x7F800000u) != 0x7F800000u || i >= valid) continue;
                        uint32_t state_part = 0;
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (x == e) state_part = s[x];
                        const float in = kBf16 ? V.scale : sm.inside[i];
                        const float y = fmaf(inside_again<kBf16>(sm.x, i, V.v + t * V.v_stride + head * D + dim, V.v_stride), in, __uint_as_float(state_part) * (sm.before[i] * up));
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (x == e) r[x] = __float_as_uint(y);
                    }
                }
                if (b == kBlocks - 1) {
                    tc::fence_before_sync();
                    mbar_arrive(&sm.out_read);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (i1 + e < valid) out[(i1 + e) * out_stride] = f32_to_out<kBf16>(__uint_as_float(r[e]));
                __syncwarp();
            }
        }
        // ---- what is left in tensor memory: the state behind the sequence, or the segment's sum
        if (!failed && (kSums ? chunks > 0 : last_segment)) {
            if (kSums && !wait(&sm.state_done, 0)) {
            } else {
                tc::fence_after_sync();
                float* const to = kSums ? sums : V.state_of(seq.to, head);
                const float* const first = V.state_of(seq.from, head);
                const float w = decay_power(g, P.segment);
#pragma unroll 1
                for (int b = 0; b < kHalf / 32; ++b) {
                    uint32_t r[32];
                    const int col = side * kHalf + 32 * b;
                    tc::tmem_ld32(state_at + 32 * b, r);
                    tc::tmem_ld_wait();
                    if (row < D) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float x = __uint_as_float(r[e]);
                            if (kSums && unit.index == 0) x = fmaf(w, first[(col + e) * D + dim], x);
                            to[(col + e) * D + dim] = x;
                        }
                    }
                    __syncwarp();
                }
            }
        }
    }
    if (failed && lane == 0 && V.error_word != nullptr) atomicOr(V.error_word, KVB_ERR_WAIT_TIMEOUT);
    tc::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

template <int D, bool kBf16> int launch_chunks(const ChunkCall& P, int units, cudaStream_t stream) {
    constexpr int smem = static_cast<int>(sizeof(LinearSmem<D>));
    static_assert(smem <= 227 * 1024, "shared memory");
    static OncePerDevice opted;  // per template instance
    KVB_CUDA_OK(opted.run(current_device(), [] {
        const cudaError_t e = cudaFuncSetAttribute(chunk_kernel<D, kBf16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(chunk_kernel<D, kBf16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    }));
    const dim3 grid(units, P.V.v_heads);
    if (P.V.tokens > P.segment) KVB_CUDA_OK(launch_early(chunk_kernel<D, kBf16, true>, grid, dim3(kChunkThreads), smem, stream, P));
    KVB_CUDA_OK(launch_early(chunk_kernel<D, kBf16, false>, grid, dim3(kChunkThreads), smem, stream, P));
    return KVB_OK;
}

}  // namespace

int linear_segment(int tokens, int batch, int v_heads) {
    // segments enough that heads and segments together are as many as the SMs, or as near below as whole segments allow
    const int sequences = batch < 1 ? 1 : batch;
    const int64_t wanted = device_sm_count() / (static_cast<int64_t>(sequences) * v_heads);
    const int64_t split = wanted < 1 ? 1 : wanted;
    const int64_t length = (static_cast<int64_t>(tokens) + sequences - 1) / sequences;
    const int64_t chunks = (length + kC * split - 1) / (kC * split);
    return static_cast<int>((wanted < 2 ? (static_cast<int64_t>(tokens) + kC - 1) / kC : chunks < 1 ? 1 : chunks) * kC);
}
int linear_units(int tokens, int batch, int segment) { return tokens / segment + batch; }

int linear_chunks(const LinearView& V, bool bf16, bool aligned, void* workspace, cudaStream_t stream) {
    ChunkCall P;
    P.V = V;
    P.sums = workspace_base(workspace);
    P.segment = linear_segment(V.tokens, V.batch, V.v_heads);
    P.aligned = aligned;
    const int units = linear_units(V.tokens, V.batch, P.segment);
    if (V.head_dim == 128) return bf16 ? launch_chunks<128, true>(P, units, stream) : launch_chunks<128, false>(P, units, stream);
    return bf16 ? launch_chunks<64, true>(P, units, stream) : launch_chunks<64, false>(P, units, stream);
}

}  // namespace kvb
