// kvb_linear_chunk.cu -- linear attention with a decay for each head over prompts, chunk by chunk on the 5th-generation tensor cores.
//
// For a chunk of C = 64 tokens (rows i, j; L of them valid) behind a state S, with lambda = exp(log_decay):
//
//   P_ij  = lambda^(i-j) q_i k_j  (j <= i, else 0)                        scores          C x C
//   o_i   = scale (sum_j P_ij v_j + lambda^(i+1) q_i S)                   inside + before
//   S    <- lambda^L S + sum_j (lambda^(L-1-j) k_j) v_j^T                 the state behind the chunk
//
// Everything but the scores is computed transposed, head dims of v along the M rows of the MMAs: S^T stays in tensor memory as an fp32 accumulator from
// chunk to chunk, and is an A operand there too; only rows of tokens as they come from global memory, decayed keys and P lie in shared memory.
// Roundings: P, and the state as an operand, to the type, like the output that they are summed up to (both together as much as the output's own
// rounding); decayed keys as two numbers of the type, whose sum has 16 bits of bf16 or 22 of fp16 (2^-36 where these are less), so that states keep their
// precision over long prompts: 4e-6 of the state's norm in bf16 (a third number would take 32 KB of shared memory that are not there), 5e-7 in fp16.
// Heads of 64 dims fill both halves of the M rows with the same 64; the scores' 64 rows are the first of 128, and what the others multiply is not looked at.
//
// Warps by role, so that a chunk's steps run beside its neighbours':
//   state warps   the state as an operand (then decayed over the chunk), decayed keys of the next chunk
//   score warps   P, up to two chunks ahead
//   row warps     outputs
//   an MMA warp   S += K'^T V, and the outputs' part from before
//   another       P V, and scores two chunks ahead
//   a load warp   tiles by TMA, into three stages (16-byte copies by the lanes filled the SM's load queue, where everybody's shared-memory accesses
//                 and arrivals waited behind them)
//   a store warp  outputs, 16 bytes a lane (two bytes a lane from the row warps held those up for 4,000 cycles a chunk, most of it in the fence before
//                 their next accesses for the MMAs, which waits for the thread's stores)
// The loop that cannot be shortened is state -> operand -> two products -> state.
//
// A sequence is split into segments where there are fewer heads and sequences than SMs: a first launch sums up each segment alone
// (keys and values only, half the reads of the second), the second starts each from the sums before it.
//
// Bound by the hand-overs between warps and tensor cores: two loops of about 3,800 cycles a chunk, in which no role's own work is more than an eighth
// (left out one at a time, none shortens a chunk by more than 13 %); the tensor pipe is busy for 22 % of the time, memory for 26.  Measured on B200,
// graph replay, bf16 / fp16: 8,192 tokens of 32 value heads of 128 dims 110 / 138 us (floor 31), 1.9 TB/s of q, k, v, o once; 7 prompts of 9,001 tokens, 24 heads
// of 64 dims 52 / 66 us with states of 16 KB a head (floor 18); 300 tokens 18 / 22 us.  Chunks of 128 tokens, whose products do a half more for the same rows,
// were slower (2,048 tokens of 128 heads 89 ... 106 us, of 64 tokens 77), so were outputs stored by TMA (90).
//
// In fp16 the scores of a row and the state's rows are scaled by a power of two to a largest magnitude of 2^14 .. 2^15 before they are rounded, so that
// neither overflows; the scales come out again in the sum of the two parts.  bf16 has the range of fp32.
#include <cuda.h>

#include "kvb_linear.cuh"
#include "kvb_tcgen05.cuh"

namespace kvb {
namespace {

constexpr int kC = kLinearChunk;  // tokens of a chunk
constexpr int kStages = kLinearStages;
constexpr int kStateWarps = 8, kRowWarps = 8;
// the last eight: warps 0, 1, 4, 5 of them P (rows 0 .. 63 of tensor memory are a warp's by its number mod 4)
constexpr int kLastWarps = kStateWarps + kRowWarps, kStateMmaWarp = kLastWarps + 2, kLoadWarp = kLastWarps + 3, kRowMmaWarp = kLastWarps + 6, kStoreWarp = kLastWarps + 7;
constexpr int kScoreWarps = 4;
constexpr int kChunkThreads = (kLastWarps + 8) * 32;  // 24 warps: six to a scheduler, 80 registers a thread
constexpr uint32_t kTmemCols = 512;

template <int D> struct LinearSmem {
    static constexpr int kTileBytes = kC * D * 2;  // [D / 64][64 rows][128 bytes], 128-byte swizzle
    struct Stage {  // the scores' MMA reads 64 rows behind those of q, too
        unsigned char q[kTileBytes], k[kTileBytes], v[kTileBytes];
    };
    alignas(1024) Stage stage[kStages];    // the keys' place takes the first numbers of the decayed keys once the scores are there
    unsigned char second[2][kTileBytes];   // their second numbers, of two chunks
    unsigned char p[2][kC * kC * 2];       // P of two chunks
    uint32_t out[2][kTileBytes / 4];       // outputs of two chunks, [32 pairs of tokens][D]
    float fade[2][2 * kC + 16];            // fade[s][x] = lambda^(63 - x - s), 0 behind lambda^0; the second copy for aligned pairs from odd x on, 16 banks further
    alignas(16) float before[kC];                      // scale lambda^(i + 1)
    uint8_t inside[2][kC];                 // exponent field of what P's row i was scaled down by (fp16)
    uint8_t up[3][128];                    // exponent field of what a row of the state was scaled down by (fp16)
    uint8_t most_state[2][128], most_p[2][2][kC];  // exponents of the largest magnitudes of a row, one a column half (fp16)
    // chunk c has the one of c mod their number; done: the state's products of a chunk; rows_done: its P V; scores: its scores
    uint64_t full[kStages], done[kStages], rows_done[kStages], scores[kStages], state_ready[3], p_ready[2], keys_ready[2], out_read[2], out_ready[2], out_free[2], most_ready[2], loaded, drained[2];
    uint32_t tmem_base;
    int abort_flag;
    int issued;  // chunks whose tiles were asked for by TMA
    int unit[3];
};

struct ChunkCall {
    CUtensorMap q, k, v;  // [tokens][heads * D], boxes of 64 rows of 64 dims
    LinearView V;
    float* sums;   // [unit][head][D][D]: each segment's sum; the last one's place holds the state before the first
    int segment;   // tokens, a multiple of kC
    bool aligned;  // rows of q, k, v keep to 16 bytes: the maps are there
};

// Which sequence and segment a unit is, and the checks of LinearView::sequence(), for the whole CTA: everything is asked of global memory at once,
// one latency instead of one after another.  Units go by the sequences' lengths, the longest first: what starts in a second wave is short.  `scratch`:
// 4 kMostSequences + 1 words of shared memory.
struct Unit {
    int index, count;  // segment `index` of `count`; count = 0: nothing to do
    Sequence seq;
    float g;           // log_decay of the head
};
__device__ __forceinline__ Unit unit_of(const ChunkCall& P, int unit, int head, int32_t* scratch, int (&found)[3]) {
    const LinearView& V = P.V;
    const int tid = threadIdx.x, lane = tid & 31;
    int32_t *const offsets = scratch, *const reads = scratch + kMostSequences + 1, *const writes = reads + kMostSequences, *const order = writes + kMostSequences;
    static_assert(kMostSequences < kChunkThreads, "a thread a sequence");
    Unit u;
    u.g = V.log_decay[head];
    if (tid <= V.batch) offsets[tid] = V.offsets[tid];
    if (tid < V.batch) {
        reads[tid] = V.reads[tid];
        writes[tid] = V.writes[tid];
    }
    __syncthreads();
    if (tid < V.batch) order[linear_rank(offsets, tid, V.batch)] = tid;
    __syncthreads();
    if (tid < 32) {
        int base = 0;
        bool any = false;
        for (int s0 = 0; s0 < V.batch; s0 += 32) {
            const int seq = s0 + lane < V.batch ? order[s0 + lane] : V.batch;
            const int count = seq < V.batch ? linear_segments(offsets, seq, V.tokens, P.segment) : 0;
            int sum = count;  // inclusive
#pragma unroll
            for (int step = 1; step < 32; step <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, step);
                if (lane >= step) sum += up;
            }
            const bool mine = unit >= base + sum - count && unit < base + sum;
            if (mine) found[0] = seq, found[1] = unit - (base + sum - count), found[2] = count;
            any = __any_sync(0xffffffffu, mine) || any;
            base += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (!any && lane == 0) found[0] = found[1] = found[2] = 0;
        // sequences that share rows have more segments than the grid has units: the ones left alone for it are reported
        if (unit == 0 && base > static_cast<int>(gridDim.y)) V.flag(KVB_ERR_POSITIONS);
    }
    __syncthreads();
    const int seq = found[0];
    u.index = found[1];
    u.count = found[2];
    u.seq.begin = offsets[seq];
    u.seq.end = offsets[seq + 1];
    u.seq.from = reads[seq];
    u.seq.to = writes[seq];
    const bool other = tid < V.batch && tid != seq;
    const bool shared = __syncthreads_or(other && (writes[tid] == u.seq.to || reads[tid] == u.seq.to || writes[tid] == u.seq.from)) != 0;
    u.seq.valid = u.count > 0 && V.allowed(u.seq, shared) && linear_fits(unit, u.index, u.count, static_cast<int>(gridDim.y));
    return u;
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
template <bool kBf16> __device__ __forceinline__ F2 pair_of(uint32_t w) {
    const float2 f = unpack_pair<kBf16>(w);
    return F2(f.x, f.y);
}
template <bool kBf16> __device__ __forceinline__ uint32_t pack_pair(F2 x) {
    const float2 f = x.get();
    return pack_pair<kBf16>(f.x, f.y);
}
__device__ __forceinline__ F2 pair_of_words(uint32_t a, uint32_t b) { return F2(__uint_as_float(a), __uint_as_float(b)); }
// What an infinite key leaves out of its first number is inf - inf: the first number alone has the key then.
template <bool kBf16> __device__ __forceinline__ uint32_t zero_if_nan(uint32_t w) {
    if constexpr (kBf16) {
        const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w);
        return w & __heq2_mask(x, x);
    } else {
        const __half2 x = *reinterpret_cast<const __half2*>(&w);
        return w & __heq2_mask(x, x);
    }
}
// Instruction descriptor of 16-bit operands of either type (format 0 = f16, 1 = bf16).
template <bool kBf16> __host__ __device__ constexpr uint32_t idesc_16(int m, int n, bool a_mn, bool b_mn) {
    return tc::idesc_f16(m, n, a_mn, b_mn) | (kBf16 ? (1u << 7) | (1u << 10) : 0u);
}
// Exponent fields of 2^-e and 2^e for the e that brings magnitudes with this largest exponent field below 2^15; 1 where it is 0's or not finite.
__device__ __forceinline__ float of_field(int field) { return __uint_as_float(static_cast<uint32_t>(field) << 23); }
__device__ __forceinline__ int2 down_and_up(int field) {
    const int e = field > 0 && field < 255 ? max(-112, min(112, field - 127 - 14)) : 0;
    return make_int2(127 - e, 127 + e);
}

// fp16 numbers end at 2^-24, so the second one of a small decayed key would have few bits left: it is held times 2^11 (2^15 at most: the first is off by 16 at most), and
// what it leaves out is 2^-22 of the key or 2^-36, which is 2^-22 of the smallest normal key.  The first launch sums up its products apart; in the second, where tensor
// memory has no room for that, the state is held times 2^11 as well while they are added, and taken back by the MMA that adds the first product.
constexpr int kSecondShift = 11;
constexpr float kSecondTimes = 1 << kSecondShift;

// A box of a tensor map into shared memory, from `row` and the first dim `x` on (a multiple of 64).
__device__ __forceinline__ void prefetch_map(const CUtensorMap& map) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory"); }
__device__ __forceinline__ void tma_load(unsigned char* dst, const CUtensorMap& map, int x, int row, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(&map)), "r"(x), "r"(row), "r"(smem_u32(bar))
                 : "memory");
}
template <int D> __device__ __forceinline__ void load_tile(unsigned char* tile, const CUtensorMap& map, int head, int64_t token, uint64_t* bar) {
#pragma unroll
    for (int half = 0; half < D / 64; ++half) tma_load(tile + half * kC * 128, map, head * D + 64 * half, static_cast<int>(token), bar);
}
// The same by a warp for rows that do not keep to 16 bytes.
template <int D> __device__ __noinline__ void load_tile_by_elements(unsigned char* tile, const uint16_t* rows, int64_t stride, int valid, int lane) {
    constexpr int kUnits = D / 8;
    for (int u = lane; u < kC * kUnits; u += 32) {
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

// Sum of P_ij v_j over j <= i for a value that came out not finite: a value of a later row that is not finite meets a 0 of P in the product.
template <bool kBf16> __device__ __noinline__ float inside_again(const unsigned char* p, int i, const uint16_t* v, int64_t stride) {
    float sum = 0.0f;
    for (int j = 0; j <= i; ++j) {
        const uint16_t w = *reinterpret_cast<const uint16_t*>(p + i * 128 + (((j >> 3) ^ (i & 7)) << 4) + (j & 7) * 2);
        sum = fmaf(in_to_f32<kBf16>(w), in_to_f32<kBf16>(v[j * stride]), sum);
    }
    return sum;
}

// kSums: the first launch, sums of segments; else the outputs and the state behind each sequence.
template <int D, bool kBf16, bool kSums>
__global__ void __launch_bounds__(kChunkThreads, 1) chunk_kernel(const __grid_constant__ ChunkCall P) {
    using Smem = LinearSmem<D>;
    // in the first launch the row warps help with the keys
    constexpr int kKeyWarps = kSums ? kLastWarps : kStateWarps, kKeyThreads = kKeyWarps * 32, kHalf = 4 * D / kKeyWarps;  // kHalf: columns of the state such a warp has
    // kSecondCol: of the first launch in fp16, the products of the keys' second numbers
    constexpr uint32_t kStateCol = 0, kSecondCol = kSums && !kBf16 ? D : 0, kOperandCol = D, kScoreCol = D + D / 2, kBeforeCol = kScoreCol + 2 * kC, kInsideCol = kBeforeCol + 2 * kC;
    static_assert(kInsideCol + kC <= kTmemCols, "tensor memory");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    grid_dependency_wait();
    launch_dependents();
    const LinearView& V = P.V;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.x;
    if (warp == kLoadWarp && lane == 0 && P.aligned) {
        if (!kSums) prefetch_map(P.q);
        prefetch_map(P.k);
        prefetch_map(P.v);
    }
    const Unit unit = unit_of(P, blockIdx.y, head, reinterpret_cast<int32_t*>(sm.out), sm.unit);
    const Sequence& seq = unit.seq;
    if (kSums && unit.count == 1) return;
    if (!seq.valid || !V.decay_fits(unit.g)) return;
    if ((smem_u32(smem_raw) & 1023u) != 0) {  // the swizzle needs it; the launch asks for nothing beside it
        V.flag(KVB_ERR_GEOMETRY);
        return;
    }
    const float g = unit.g;
    const bool last_segment = unit.index == unit.count - 1;
    const int begin = seq.begin + unit.index * P.segment, end = last_segment ? seq.end : begin + P.segment;
    const int chunks = kSums && last_segment ? 0 : (end - begin + kC - 1) / kC;
    float* const sums = P.sums + (static_cast<int64_t>(blockIdx.y) * V.v_heads + head) * D * D;  // this segment's; earlier ones lie in front
    const int64_t sums_step = static_cast<int64_t>(V.v_heads) * D * D;

    if (warp == kStateMmaWarp) tc::tmem_alloc(&sm.tmem_base, kTmemCols);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.done[s], 1);
            mbar_init(&sm.rows_done[s], 1);
            mbar_init(&sm.scores[s], 1);
            mbar_init(&sm.state_ready[s], kStateWarps);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.p_ready[s], kScoreWarps);
            mbar_init(&sm.keys_ready[s], kKeyWarps);
            mbar_init(&sm.out_read[s], kRowWarps);
            mbar_init(&sm.out_ready[s], kRowWarps);
            mbar_init(&sm.out_free[s], 1);
        }
        mbar_init(&sm.most_ready[0], kStateWarps);
        mbar_init(&sm.most_ready[1], kScoreWarps);
        mbar_init(&sm.loaded, kStateWarps + kRowWarps);
        mbar_init(&sm.drained[0], 1);
        mbar_init(&sm.drained[1], 1);
        mbar_fence_init();
        sm.abort_flag = 0;
        sm.issued = 0;
    }
    if (threadIdx.x < 4 * kC) {
        const int copy = threadIdx.x / (2 * kC), x = threadIdx.x % (2 * kC), n = kC - 1 - x - copy;
        sm.fade[copy][x] = n >= 0 ? decay_power(g, n) : 0.0f;
        if (threadIdx.x < kC) sm.before[threadIdx.x] = V.scale * decay_power(g, threadIdx.x + 1);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sm.tmem_base;
    bool failed = false;
    auto wait = [&](uint64_t* bar, int phase) {
        if (!failed && !chunk_wait(bar, static_cast<uint32_t>(phase & 1), &sm.abort_flag)) failed = true;
        return !failed;
    };
    // one arrival a warp, when all its lanes are there (256 a barrier kept shared memory busy)
    auto arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    auto wait2 = [&](uint64_t (&bars)[2], int c) { return wait(&bars[c & 1], c >> 1); };
    auto wait3 = [&](uint64_t (&bars)[3], int c) { return wait(&bars[c % 3], c / 3); };

    if (warp < kLastWarps && (!kSums || last_segment)) {
        // ---- the state before the segment, a quarter of the columns a warp: from the pool, or the sums of the segments before
        const int quad = warp & 3, row = 32 * quad + lane, dim = row % D;
        constexpr int kEach = D / 4;
        const int col = (warp >> 2) * kEach;
        const float* from = V.state_of(seq.from, head);
        if (!kSums && unit.count > 1 && unit.index == 0) from = sums + (unit.count - 1) * sums_step;
#pragma unroll 1
        for (int b = 0; b < kEach; b += 16) {
            const int at = (col + b) * D + dim;
            uint32_t r[16];
            if (kSums || unit.index == 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(from[at + e * D]);
            } else {
                float f[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) f[e] = 0.0f;
#pragma unroll 2
                for (int s = 0; s < unit.index; ++s) {
                    const float* const sum = sums - (unit.index - s) * sums_step + at;
                    const float w = decay_power(g, (unit.index - 1 - s) * P.segment);
#pragma unroll
                    for (int e = 0; e < 16; ++e) f[e] = fmaf(w, sum[e * D], f[e]);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(f[e]);
            }
            if (kSums) {  // the last segment's place keeps the state for the second launch, which may write over it
                if (row < D) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) sums[at + e * D] = __uint_as_float(r[e]);
                }
            } else {
                tc::tmem_st16(tmem + (static_cast<uint32_t>(32 * quad) << 16) + kStateCol + col + b, r);
            }
        }
        if (!kSums) {
            tc::tmem_st_wait();
            tc::fence_before_sync();
            arrive(&sm.loaded);
        }
    }
    if (warp == kLoadWarp) {
        // ---- loads: chunk c into stage c % 3.  Rows behind a sequence's last come with it, whatever they hold: see there.
        const int qk_head = head / V.share;
        for (int c = 0; c < chunks; ++c) {
            const int stage = c % kStages;
            typename Smem::Stage& st = sm.stage[stage];
            const int64_t t = begin + c * kC;
            // the products of the stage's chunk before: the state's, its P V
            if (c >= kStages && (!wait3(sm.done, c - kStages) || (!kSums && !wait3(sm.rows_done, c - kStages)))) break;
            if (P.aligned) {
                if (lane == 0) {
                    mbar_expect_tx(&sm.full[stage], (kSums ? 2 : 3) * Smem::kTileBytes);
                    load_tile<D>(st.k, P.k, qk_head, t, &sm.full[stage]);
                    if (!kSums) load_tile<D>(st.q, P.q, qk_head, t, &sm.full[stage]);
                    load_tile<D>(st.v, P.v, head, t, &sm.full[stage]);
                    sm.issued = c + 1;
                }
            } else {
                const int valid = min(kC, end - static_cast<int>(t));
                load_tile_by_elements<D>(st.k, V.k + t * V.k_stride + qk_head * D, V.k_stride, valid, lane);
                if (!kSums) load_tile_by_elements<D>(st.q, V.q + t * V.q_stride + qk_head * D, V.q_stride, valid, lane);
                load_tile_by_elements<D>(st.v, V.v + t * V.v_stride + head * D, V.v_stride, valid, lane);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.full[stage]);
            }
            __syncwarp();
        }
    } else if (warp == kStoreWarp) {
        // ---- stores
        const bool wide = (reinterpret_cast<uintptr_t>(V.out) & 15u) == 0;
        const int64_t out_stride = static_cast<int64_t>(V.v_heads) * D;
        for (int c = 0; !kSums && c < chunks; ++c) {
            const int64_t t = begin + c * kC;
            const int valid = min(kC, end - static_cast<int>(t));
            if (!wait2(sm.out_ready, c)) break;
            uint16_t* const to = V.out + (t * V.v_heads + head) * D;
            const uint32_t* const words = sm.out[c & 1];  // of a head dim and two tokens
            if (wide) {
                constexpr int kUnits = D / 8, kAtOnce = 2;  // 8 dims a unit; bursts of stores are in everybody's way
#pragma unroll 1
                for (int u0 = lane; u0 < kC / 2 * kUnits; u0 += 32 * kAtOnce) {
                    uint4 r[kAtOnce][2];
#pragma unroll
                    for (int n = 0; n < kAtOnce; ++n) {
                        r[n][0] = reinterpret_cast<const uint4*>(words)[2 * (u0 + 32 * n)];
                        r[n][1] = reinterpret_cast<const uint4*>(words)[2 * (u0 + 32 * n) + 1];
                    }
#pragma unroll
                    for (int n = 0; n < kAtOnce; ++n) {
                        const int row = (u0 + 32 * n) / kUnits * 2, col = (u0 + 32 * n) % kUnits;
                        uint16_t* const at = to + row * out_stride + 8 * col;
                        const uint4 x = r[n][0], y = r[n][1];
                        if (row < valid) *reinterpret_cast<uint4*>(at) = make_uint4(prmt(x.x, x.y, 0x5410), prmt(x.z, x.w, 0x5410), prmt(y.x, y.y, 0x5410), prmt(y.z, y.w, 0x5410));
                        if (row + 1 < valid)
                            *reinterpret_cast<uint4*>(at + out_stride) = make_uint4(prmt(x.x, x.y, 0x7632), prmt(x.z, x.w, 0x7632), prmt(y.x, y.y, 0x7632), prmt(y.z, y.w, 0x7632));
                    }
                }
            } else {
#pragma unroll 1
                for (int u = lane; u < valid * D; u += 32) to[u / D * out_stride + u % D] = static_cast<uint16_t>(words[u / D / 2 * D + u % D] >> (u / D % 2 * 16));
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.out_free[c & 1]);
        }
    } else if (warp == kStateMmaWarp || warp == kRowMmaWarp) {
        // ---- MMAs, issued by one thread of a warp
        // MN-major: the next 64 head dims half a tile further (heads of 64 dims: the same ones again), the next 8 tokens 1024 bytes
        constexpr uint32_t kScores = idesc_16<kBf16>(128, kC, false, false), kState = idesc_16<kBf16>(128, D, true, true), kOut = idesc_16<kBf16>(128, kC, true, false);
        auto rows_desc = [&](const unsigned char* tile) { return tc::smem_desc(smem_u32(tile), 16, 1024); };
        auto dims_desc = [&](const unsigned char* tile) { return tc::smem_desc(smem_u32(tile), D == 128 ? kC * 128 : 0, 1024); };
        auto keys_desc = [&](const unsigned char* tile) { return tc::smem_desc(smem_u32(tile), kC * 128, 1024); };
        auto k_major = [](uint64_t desc, int step) { return tc::desc_at(desc, (step >> 2) * (kC * 128) + (step & 3) * 32); };  // 16 of the K dims further
        if (warp == kStateMmaWarp) {
            for (int c = 0; c < chunks; ++c) {
                const typename Smem::Stage& st = sm.stage[c % kStages];
                if (!wait2(sm.keys_ready, c)) break;
                // what is left of the outputs before the last in tensor memory has been read
                if (!kSums && (!wait3(sm.state_ready, c) || (c > 1 && !wait2(sm.out_read, c - 2)))) break;
                tc::fence_after_sync();
                if (tc::elect_one()) {
                    const uint64_t a = dims_desc(st.v), b = keys_desc(st.k), b2 = keys_desc(sm.second[c & 1]);
                    auto second = [&](int s, bool accumulate) { tc::mma_f16_ss(tmem + kStateCol + kSecondCol, tc::desc_at(a, s * 2048), tc::desc_at(b2, s * 2048), kState, accumulate); };
                    auto first = [&](int s, bool accumulate) { tc::mma_f16_ss(tmem + kStateCol, tc::desc_at(a, s * 2048), tc::desc_at(b, s * 2048), kState, accumulate); };
                    if constexpr (!kBf16 && !kSums) {
#pragma unroll
                        for (int s = 0; s < kC / 16; ++s) second(s, true);
                        tc::mma_f16_ss_scaled<kSecondShift>(tmem + kStateCol, a, b, kState);
#pragma unroll
                        for (int s = 1; s < kC / 16; ++s) first(s, true);
                    } else {
#pragma unroll
                        for (int s = 0; s < kC / 16; ++s) first(s, !kSums || c > 0 || s > 0);
#pragma unroll
                        for (int s = 0; s < kC / 16; ++s) second(s, kBf16 || c > 0 || s > 0);
                    }
                    if (!kSums) {
                        const uint64_t q = rows_desc(st.q);
#pragma unroll
                        for (int s = 0; s < D / 16; ++s) tc::mma_f16_ts(tmem + kBeforeCol + (c & 1) * kC, tmem + kOperandCol + 8 * s, k_major(q, s), kScores, s > 0);
                    }
                    tc::commit(&sm.done[c % 3]);
                }
                __syncwarp();
            }
        } else if (!kSums) {
            for (int n = 0; n < chunks + 2; ++n) {  // P V of chunk n - 2, scores of chunk n
                const int c = n - 2;
                if (c >= 0) {
                    if (!wait2(sm.keys_ready, c) || !wait2(sm.p_ready, c) || (c > 0 && !wait2(sm.out_read, c - 1))) break;  // keys: values behind the last are zeros
                    tc::fence_after_sync();
                    if (tc::elect_one()) {
                        const uint64_t a = dims_desc(sm.stage[c % kStages].v), b = rows_desc(sm.p[c & 1]);
#pragma unroll
                        for (int s = 0; s < kC / 16; ++s) tc::mma_f16_ss(tmem + kInsideCol, tc::desc_at(a, s * 2048), k_major(b, s), kOut, s > 0);
                        tc::commit(&sm.rows_done[c % 3]);
                    }
                    __syncwarp();
                }
                if (n < chunks) {
                    if (!wait3(sm.full, n)) break;
                    tc::fence_after_sync();
                    if (tc::elect_one()) {
                        const uint64_t a = rows_desc(sm.stage[n % kStages].q), b = rows_desc(sm.stage[n % kStages].k);
#pragma unroll
                        for (int s = 0; s < D / 16; ++s) tc::mma_f16_ss(tmem + kScoreCol + (n & 1) * kC, k_major(a, s), k_major(b, s), kScores, s > 0);
                        tc::commit(&sm.scores[n % 3]);
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp < kKeyWarps) {
        // ---- state warps: rows 32 (warp % 4) + lane of S^T, columns by warp / 4
        const int quad = warp & 3, side = warp >> 2, row = 32 * quad + lane, dim = row % D, tid = threadIdx.x;
        const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
        const uint32_t state_at = tmem + lanes + kStateCol + side * kHalf;

        // decayed keys of chunk c, two numbers each
        auto decay_keys = [&](int c) {
            if (!wait3(sm.full, c)) return;
            if (!kSums && !wait3(sm.scores, c)) return;  // the keys themselves have been read
            const int t = begin + c * kC, valid = min(kC, end - t);
            unsigned char* const keys = sm.stage[c % kStages].k;
            unsigned char* const second = sm.second[c & 1];
            constexpr int kEach = kC * D / 8 / kKeyThreads;
#pragma unroll
            for (int n = 0; n < kEach; ++n) {
                const int u = tid + n * kKeyThreads, j = (u >> 3) & (kC - 1);
                const float w = kSums ? decay_power(g, end - 1 - t - j) : sm.fade[0][kC - 1 - max(valid - 1 - j, 0)];
                uint4 raw = *reinterpret_cast<const uint4*>(keys + 16 * u);
                if (j >= valid) raw = make_uint4(0u, 0u, 0u, 0u);
                const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
                uint32_t a[4], b[4];
                if constexpr (kBf16) {
                    // the weight as two numbers, too: the first product rounded, what that left out (exact) and the second product
                    const __nv_bfloat16 first = __float2bfloat16_rn(w);
                    const __nv_bfloat162 w1 = __bfloat162bfloat162(first), w2 = __bfloat162bfloat162(__float2bfloat16_rn(w - __bfloat162float(first)));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const __nv_bfloat162 k = *reinterpret_cast<const __nv_bfloat162*>(&in[e]), x = __hmul2(k, w1), y = __hfma2(k, w2, __hfma2(k, w1, __hneg2(x)));
                        a[e] = *reinterpret_cast<const uint32_t*>(&x);
                        b[e] = zero_if_nan<kBf16>(*reinterpret_cast<const uint32_t*>(&y));
                    }
                } else {  // small weights have too few bits in fp16
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const F2 x = mul2(pair_of<kBf16>(in[e]), F2(w, w));
                        a[e] = pack_pair<kBf16>(x);
                        b[e] = zero_if_nan<kBf16>(pack_pair<kBf16>(mul2(sub2(x, pair_of<kBf16>(a[e])), F2(kSecondTimes, kSecondTimes))));
                    }
                }
                *reinterpret_cast<uint4*>(keys + 16 * u) = make_uint4(a[0], a[1], a[2], a[3]);
                *reinterpret_cast<uint4*>(second + 16 * u) = make_uint4(b[0], b[1], b[2], b[3]);
            }
            if (valid < kC) {  // values behind the sequence's last row meet zeros in P and the keys: they have to be finite
                for (int u = tid; u < kC * D / 8; u += kKeyThreads)
                    if (((u >> 3) & (kC - 1)) >= valid) *reinterpret_cast<uint4*>(sm.stage[c % kStages].v + 16 * u) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async();
            arrive(&sm.keys_ready[c & 1]);
        };
        if (kSums) {
            for (int c = 0; c < chunks && !failed; ++c) {
                if (c > 1 && !wait3(sm.done, c - 2)) break;  // the keys' buffer has been read
                decay_keys(c);
            }
        } else {
            if (chunks > 0) decay_keys(0);
            wait(&sm.loaded, 0);
            tc::fence_after_sync();
            for (int c = 0; c < chunks && !failed; ++c) {
                // the state as an operand, and decayed over the chunk
                if (c > 0 && !wait3(sm.done, c - 1)) break;
                tc::fence_after_sync();
                const float decay = decay_power(g, min(kC, end - begin - c * kC)) * (kBf16 ? 1.0f : kSecondTimes);
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
                    sm.most_state[side][row] = static_cast<uint8_t>(mine);
                    arrive(&sm.most_ready[0]);
                    if (!wait(&sm.most_ready[0], c)) break;
                    const int2 f = down_and_up(max(mine, static_cast<int>(sm.most_state[side ^ 1][row])));
                    down = of_field(f.x);
                    if (side == 0) sm.up[c % 3][row] = static_cast<uint8_t>(f.y);
                }
#pragma unroll 1
                for (int b = 0; b < kHalf / 32; ++b) {
                    uint32_t r[32], operand[16];
                    tc::tmem_ld32(state_at + 32 * b, r);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const F2 x = pair_of_words(r[2 * e], r[2 * e + 1]);
                        operand[e] = pack_pair<kBf16>(kBf16 ? x : mul2(x, F2(down, down)));
                        const float2 y = mul2(x, F2(decay, decay)).get();
                        r[2 * e] = __float_as_uint(y.x);
                        r[2 * e + 1] = __float_as_uint(y.y);
                    }
                    tc::tmem_st32(state_at + 32 * b, r);
                    tc::tmem_st16(tmem + lanes + kOperandCol + (side * kHalf + 32 * b) / 2, operand);
                }
                tc::tmem_st_wait();
                tc::fence_before_sync();
                arrive(&sm.state_ready[c % 3]);
                if (c + 1 < chunks) decay_keys(c + 1);  // their buffer's last reader was done before the state was
            }
        }
        // ---- what is left in tensor memory: the state behind the sequence, or the segment's sum
        if (!failed && chunks > 0) wait3(sm.done, chunks - 1);
        if (!failed && (kSums ? chunks > 0 : last_segment)) {
            tc::fence_after_sync();
            float* const to = kSums ? sums : V.state_of(seq.to, head);
            const float w = decay_power(g, P.segment);
#pragma unroll 1
            for (int b = 0; b < kHalf; b += 16) {
                const int at = (side * kHalf + b) * D + dim;
                uint32_t r[16];
                float first[16];  // asked for ahead of the stores, which might write there for all the compiler knows
                if (kSums && unit.index == 0) {
                    const float* const from = V.state_of(seq.from, head) + at;
#pragma unroll
                    for (int e = 0; e < 16; ++e) first[e] = from[e * D];
                }
                tc::tmem_ld16(state_at + b, r);
                if constexpr (kSecondCol != 0) {
                    uint32_t second[16];
                    tc::tmem_ld16(state_at + kSecondCol + b, second);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(fmaf(__uint_as_float(second[e]), 1.0f / kSecondTimes, __uint_as_float(r[e])));
                }
                tc::tmem_ld_wait();
                if (row < D) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) to[at + e * D] = kSums && unit.index == 0 ? fmaf(w, first[e], __uint_as_float(r[e])) : __uint_as_float(r[e]);
                }
                __syncwarp();
            }
        }
    } else if (!kSums && warp >= kLastWarps) {
        // ---- score warps: rows 0 .. 63 of the scores, 32 columns a warp
        const int quad = warp & 3, side = (warp - kLastWarps) >> 2, row = 32 * quad + lane, j0 = 32 * side;
        for (int c = 0; c < chunks; ++c) {
            if (!wait3(sm.scores, c)) break;
            tc::fence_after_sync();
            uint32_t s[32], p[16];
            float most = 0.0f;
            if (side <= quad) {  // a block with something on or below the diagonal
                tc::tmem_ld32(tmem + (static_cast<uint32_t>(32 * quad) << 16) + kScoreCol + (c & 1) * kC + j0, s);
                const int x0 = kC - 1 - row + j0, below = row - j0;  // columns 0 .. below are on or below the diagonal
                const float2* const fade = reinterpret_cast<const float2*>(sm.fade[x0 & 1] + (x0 & ~1));
                tc::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float2 w = fade[e / 2];
                    const float2 x = mul2(pair_of_words(s[e], s[e + 1]), F2(w.x, w.y)).get();
                    // not a product with 0: a score of a later token need not be finite
                    s[e] = e <= below ? __float_as_uint(x.x) : 0u;
                    s[e + 1] = e + 1 <= below ? __float_as_uint(x.y) : 0u;
                    if constexpr (!kBf16) most = fmaxf(most, fmaxf(fabsf(__uint_as_float(s[e])), fabsf(__uint_as_float(s[e + 1]))));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) s[e] = 0u;
            }
            float down = 1.0f;
            int up = 0;
            if constexpr (!kBf16) {
                const int mine = static_cast<int>(__float_as_uint(most) >> 23);
                sm.most_p[c & 1][side][row] = static_cast<uint8_t>(mine);
                arrive(&sm.most_ready[1]);
                if (!wait(&sm.most_ready[1], c)) break;
                const int2 f = down_and_up(max(mine, static_cast<int>(sm.most_p[c & 1][side ^ 1][row])));
                down = of_field(f.x);
                up = f.y;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const F2 x = pair_of_words(s[2 * e], s[2 * e + 1]);
                p[e] = pack_pair<kBf16>(kBf16 ? x : mul2(x, F2(down, down)));
            }
            if (c > 1 && !wait2(sm.out_read, c - 2)) break;  // nobody looks at P of the chunk before the last, and its scales, any more
            if (!kBf16 && side == 0) sm.inside[c & 1][row] = static_cast<uint8_t>(up);
            unsigned char* const to = sm.p[c & 1] + row * 128;
#pragma unroll
            for (int u = 0; u < 4; ++u) *reinterpret_cast<uint4*>(to + (((4 * side + u) ^ (row & 7)) << 4)) = make_uint4(p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]);
            fence_proxy_async();
            tc::fence_before_sync();
            arrive(&sm.p_ready[c & 1]);
        }
    } else if (!kSums) {
        // ---- row warps: head dim `dim`, 32 tokens (heads of 64 dims, which are there twice: 16), 16 at a time
        const int quad = warp & 3, side = (warp - kStateWarps) >> 2, row = 32 * quad + lane, dim = row % D;
        const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
        constexpr int kTokens = 16, kBlocks = D == 128 ? 2 : 1;
        const int first = D == 128 ? 32 * side : 32 * side + 16 * (quad >> 1);
        for (int c = 0; c < chunks; ++c) {
            const int64_t t = begin + c * kC;
            const int valid = min(kC, end - static_cast<int>(t));
            if (!wait3(sm.done, c) || !wait3(sm.rows_done, c)) break;
            if (!kBf16 && (!wait3(sm.state_ready, c) || !wait2(sm.p_ready, c))) break;  // sm.up, sm.inside of all rows
            if (c > 1 && !wait2(sm.out_free, c - 2)) break;
            tc::fence_after_sync();
            const float up = kBf16 ? 1.0f : of_field(sm.up[c % 3][row]);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int i0 = first + kTokens * b;
                uint32_t r[kTokens], s[kTokens];
                tc::tmem_ld16(tmem + lanes + kInsideCol + i0, r);
                tc::tmem_ld16(tmem + lanes + kBeforeCol + (c & 1) * kC + i0, s);
                tc::tmem_ld_wait();
                F2 zeros(0.0f, 0.0f);
#pragma unroll
                for (int e = 0; e < kTokens; e += 4) {
                    float4 in = make_float4(V.scale, V.scale, V.scale, V.scale);
                    if constexpr (!kBf16) {
                        const uchar4 f = *reinterpret_cast<const uchar4*>(&sm.inside[c & 1][i0 + e]);
                        in = make_float4(V.scale * of_field(f.x), V.scale * of_field(f.y), V.scale * of_field(f.z), V.scale * of_field(f.w));
                    }
                    const float4 before = *reinterpret_cast<const float4*>(&sm.before[i0 + e]);
#pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        F2 part = mul2(pair_of_words(s[e + h], s[e + h + 1]), h ? F2(before.z, before.w) : F2(before.x, before.y));
                        if constexpr (!kBf16) part = mul2(part, F2(up, up));
                        const F2 y = fma2(pair_of_words(r[e + h], r[e + h + 1]), h ? F2(in.z, in.w) : F2(in.x, in.y), part);
                        zeros = fma2(y, F2(0.0f, 0.0f), zeros);
                        r[e + h] = __float_as_uint(y.get().x);
                        r[e + h + 1] = __float_as_uint(y.get().y);
                    }
                }
                if (!(zeros.get().x + zeros.get().y == 0.0f)) {
#pragma unroll 1
                    for (int e = 0; e < kTokens; ++e) {
                        const int i = i0 + e;
                        uint32_t word = 0, part = 0;  // r[e], s[e] without an index into registers
#pragma unroll
                        for (int x = 0; x < kTokens; ++x)
                            if (x == e) word = r[x], part = s[x];
                        if ((word & 0x7F800000u) != 0x7F800000u || i >= valid) continue;
                        const float in = kBf16 ? V.scale : V.scale * of_field(sm.inside[c & 1][i]);
                        const float again = inside_again<kBf16>(sm.p[c & 1], i, V.v + t * V.v_stride + head * D + dim, V.v_stride);
                        const float y = fmaf(again, in, __uint_as_float(part) * sm.before[i] * up);
#pragma unroll
                        for (int x = 0; x < kTokens; ++x)
                            if (x == e) r[x] = __float_as_uint(y);
                    }
                }
                __syncwarp();
                if (b == kBlocks - 1) {
                    tc::fence_before_sync();
                    arrive(&sm.out_read[c & 1]);
                }
                uint32_t* const out = sm.out[c & 1] + i0 / 2 * D + dim;
#pragma unroll
                for (int e = 0; e < kTokens / 2; ++e) out[e * D] = pack_pair<kBf16>(pair_of_words(r[2 * e], r[2 * e + 1]));
            }
            arrive(&sm.out_ready[c & 1]);
        }
    }
    if (failed && lane == 0 && V.error_word != nullptr) atomicOr(V.error_word, KVB_ERR_WAIT_TIMEOUT);
    tc::fence_before_sync();
    // Where any warp gave up, others may have gone through: no copy lands in shared memory, and no MMA runs on tensor memory, that is no longer this CTA's.
    if (__syncthreads_or(failed)) {
        if (warp == kLoadWarp) {
            const int issued = sm.issued;
            for (int c = linear_first_in_flight(issued); c < issued; ++c) mbar_wait_bounded(&sm.full[c % kStages], (c / kStages) & 1);
        } else if (warp == kStateMmaWarp || warp == kRowMmaWarp) {
            uint64_t* const drained = &sm.drained[warp == kRowMmaWarp];
            if (tc::elect_one()) tc::commit(drained);
            __syncwarp();
            mbar_wait_bounded(drained, 0);
        }
        tc::fence_before_sync();
        __syncthreads();
    }
    if (warp == kStateMmaWarp) {
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
    const dim3 grid(P.V.v_heads, units);  // units that are none come last
    if (P.V.tokens > P.segment) KVB_CUDA_OK(launch_early(chunk_kernel<D, kBf16, true>, grid, dim3(kChunkThreads), smem, stream, P));
    KVB_CUDA_OK(launch_early(chunk_kernel<D, kBf16, false>, grid, dim3(kChunkThreads), smem, stream, P));
    return KVB_OK;
}

}  // namespace

namespace {

// The driver's encoder of tensor maps; null where there is none.
decltype(&cuTensorMapEncodeTiled) tensor_map_encoder() {
    static const auto encoder = [] {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult found;
        const bool ok = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(entry) : nullptr;
    }();
    return encoder;
}
bool rows_map(CUtensorMap* map, const void* rows, bool bf16, int64_t width, int64_t tokens, int64_t stride) {
    const auto encode = tensor_map_encoder();
    const cuuint64_t size[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(tokens)}, pitch[1] = {static_cast<cuuint64_t>(stride) * 2};
    const cuuint32_t box[2] = {64, kC}, step[2] = {1, 1};
    return encode != nullptr && encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(rows), size, pitch, box, step,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

int linear_chunks(const LinearView& V, bool bf16, bool aligned, void* workspace, cudaStream_t stream) {
    ChunkCall P{};
    P.V = V;
    P.sums = workspace_base(workspace);
    P.segment = linear_segment(V.tokens, V.batch, V.v_heads);
    const int64_t qk_width = static_cast<int64_t>(V.v_heads) / V.share * V.head_dim, v_width = static_cast<int64_t>(V.v_heads) * V.head_dim;
    P.aligned = aligned && rows_map(&P.q, V.q, bf16, qk_width, V.tokens, V.q_stride) && rows_map(&P.k, V.k, bf16, qk_width, V.tokens, V.k_stride) &&
                rows_map(&P.v, V.v, bf16, v_width, V.tokens, V.v_stride);
    const int units = linear_units(V.tokens, V.batch, P.segment);
    if (V.head_dim == 128) return bf16 ? launch_chunks<128, true>(P, units, stream) : launch_chunks<128, false>(P, units, stream);
    return bf16 ? launch_chunks<64, true>(P, units, stream) : launch_chunks<64, false>(P, units, stream);
}

}  // namespace kvb
