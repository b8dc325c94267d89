// kvb_read.cu -- rows of the cache back as 16-bit keys and values: codes de-quantised, the Walsh-Hadamard rotation undone.
//
//   x = H ((code * scale_axis + zp_axis) * other_axis)   rows of sealed tiles (scale and zero point per dim for K, per token for V)
//   x = H stage                                          rows of the open tile
// in fp32, rounded once.
//
// The rotation of 128 dims is one of 16 (bits 0, 1, 4, 5 of the dim) for each of 8 groups (bits 2, 3, 6), then one of 8 across the groups.  The first
// is a product on the tensor cores, 16 tokens at a time, of codes -- small whole numbers, exact in fp16 -- with the rotation's signs times what
// belongs to the dim (K: the scale, V: the factor; fp16 values as they are): all products exact, sums in fp32.  What is added per dim goes through
// the same product once a tile, with ones for the codes; what belongs to the token is applied to the sums.  The second stays inside a thread:
// lane (4 g + t) has dims 16 t .. + 15 and 64 + 16 t .. + 15 of tokens g and g + 8 ahead of the products and behind them: 32 bytes a store, 128
// of a row a warp.  At 256 dims the two slices are rotated apart and meet in the last sum and difference.
// A CTA goes through tiles of one head of K or V, 16 tokens a warp at a time; the next tile's codes and axes are on their way by bulk copies meanwhile.
//
// Bound by what the L1 passes on, then by memory.  Measured on B200, 131,072 tokens of 4 heads of 128 dims (floor 52 us): 104 us with the rotation in
// shuffles; 114 by products, a tile a CTA and 16 bytes a store; 97 with 32 bytes a store; 88 with CTAs that stay and ask for the next tile ahead; 63 with the
// kinds of rows told apart outside the loop over tokens: 5.4 TB/s, 82 % of a copy.  5,001 rows of 256 dims 9.3 us (floor 4.0): a tile or two a CTA.
#include "kvb_common.cuh"
#include "kvb_ptx.cuh"

#include <type_traits>

namespace kvb {
namespace {

// Probes of the wait for a CTA's n-th tile.  (A test builds the kernel with waits that give up at once while tiles are on their way.)
#ifndef KVB_READ_PROBES
#define KVB_READ_PROBES kSpinLimit
#endif

constexpr int kReadThreads = 128, kReadWarps = kReadThreads / 32;

constexpr int kDimStride = 36;  // of a lane number's 32 dims: four lanes' 8 (16) bytes lie in different banks

template <int D> struct ReadSmem {
    static constexpr int S = Geo<D>::S;
    struct alignas(16) Tile {
        uint8_t code[2 * Geo<D>::kCodePageBytes];
        __half axes[2 * kPage * Geo<D>::kKScaleLeading];  // of the first page, then of the second
    };
    Tile tile[2];
    alignas(16) __half dim_a[S][4][kDimStride];  // K: scale, V: factor of a dim
    alignas(16) __half dim_b[4 * kDimStride * S];  // K: zero point
    alignas(16) float term[S][4][kDimStride];    // what is added per dim, through the first product
    float token_a[S][kTile];                     // K: factor, V: scale of a token
    float token_b[S][kTile];                     // V: zero point
    uint64_t full[2];
    int kind[2];
};
enum { kSkip = 0, kSealed = 1, kOpen = 2 };
// D = A B + C of m16n8k16, C apart from D.
__device__ __forceinline__ void mma_apart(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
// The two codes of byte `byte` of w as halves: one in bits 0 .. 3 under 2^10, one in bits 4 .. 7 under 2^6, less these.
__device__ __forceinline__ uint32_t code_halves(uint32_t w, int byte) {
    return hsub2_u32(lop3_and_or(prmt(w, 0u, 0x4040u | static_cast<uint32_t>(byte) * 0x0101u), 0x00F0000Fu, 0x54006400u), 0x54006400u);
}

// 32 bytes from a lane, to a 32-byte boundary.
__device__ __forceinline__ void store32(void* to, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

template <bool kBf16> __device__ __forceinline__ uint32_t pack_out(float2 y) {
    if constexpr (kBf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(y.x, y.y);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        return pack_half2(y.x, y.y);
    }
}

// Rotation of 8 across the groups.
__device__ __forceinline__ void rotate_groups(F2 (&x)[8][2][2]) {
#pragma unroll
    for (int span = 1; span < 8; span <<= 1)
#pragma unroll
        for (int b = 0; b < 8; b += 2 * span)
#pragma unroll
            for (int e = 0; e < span; ++e)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const F2 lo = x[b + e][j][r], hi = x[b + e + span][j][r];
                        x[b + e][j][r] = add2(lo, hi);
                        x[b + e + span][j][r] = sub2(lo, hi);
                    }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kReadThreads) read_kernel(LayerView L, int begin, int end, const int32_t* __restrict__ total_pos, uint16_t* __restrict__ out_k,
                                                            uint16_t* __restrict__ out_v) {
    using G = Geo<D>;
    using Smem = ReadSmem<D>;
    constexpr int S = G::S, c = G::kAxisCols;
    constexpr float kNorm = D == 256 ? 0.0625f : 0.08838834764831845f;
    static_assert(kReadThreads == kTile, "a thread a token");
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, head = blockIdx.y, which = blockIdx.z;
    const int leading = which ? G::kVScaleLeading : G::kKScaleLeading;
    if (tid == 0) {
        mbar_init(&sm.full[0], 1);
        mbar_init(&sm.full[1], 1);
        mbar_fence_init();
    }
    grid_dependency_wait();
    launch_dependents();
    const int last_tile = (end - 1) / kTile, step = gridDim.x;
    const int32_t* const tbl = L.table();
    int32_t entry0 = LayerView::kNoEntry, entry1 = LayerView::kNoEntry;  // thread 0: the pages of the tile to be asked for next
    auto look_up = [&](int tile) {
        if (tile > last_tile) return;
        entry0 = 2 * tile < L.table_len ? tbl[2 * tile] : LayerView::kNoEntry;
        entry1 = 2 * tile + 1 < L.table_len ? tbl[2 * tile + 1] : LayerView::kNoEntry;
    };
    const int first_tile = begin / kTile + static_cast<int>(blockIdx.x);
    if (tid == 0) look_up(first_tile);
    const int newest = *total_pos;
    auto rows_of = [&](int tile) { return make_int2(max(begin, tile * kTile), min(end - 1, min(newest, tile * kTile + kTile - 1))); };  // first and last to be read
    auto ask = [&](int tile, int buffer) {  // thread 0: the tile's codes and axes
        if (tile > last_tile) return;
        const int32_t page0 = entry0, page1 = entry1;
        look_up(tile + step);
        const int2 rows = rows_of(tile);
        int kind = rows.x > rows.y ? kSkip : tile * kTile + kTile - 1 <= newest ? kSealed : kOpen;
        if (kind == kSealed) {
            if (page0 == LayerView::kNoEntry || page1 == LayerView::kNoEntry) L.flag(KVB_ERR_TABLE_RANGE);
            const int32_t a = L.checked_page(page0), b = L.checked_page(page1);
            if (a < 0 || b < 0) {
                kind = kSkip;  // the tile's rows are left as they are
            } else {
                const uint32_t axes = kPage * leading * 2;
                const uint8_t* const code = (which ? L.v_code : L.k_code);
                const __half* const scale = which ? L.v_scale : L.k_scale;
                typename Smem::Tile& to = sm.tile[buffer];
                mbar_expect_tx(&sm.full[buffer], 2 * (G::kCodePageBytes + axes));
                bulk_g2s(to.code, code + page_head_offset(G::kCodeLeading, L.kv_heads, a, head), G::kCodePageBytes, &sm.full[buffer]);
                bulk_g2s(to.code + G::kCodePageBytes, code + page_head_offset(G::kCodeLeading, L.kv_heads, b, head), G::kCodePageBytes, &sm.full[buffer]);
                bulk_g2s(to.axes, scale + page_head_offset(leading, L.kv_heads, a, head), axes, &sm.full[buffer]);
                bulk_g2s(to.axes + kPage * leading, scale + page_head_offset(leading, L.kv_heads, b, head), axes, &sm.full[buffer]);
            }
        }
        if (kind != kSealed) mbar_arrive(&sm.full[buffer]);
        sm.kind[buffer] = kind;
    };
    if (tid == 0) ask(first_tile, 0);
    __syncthreads();

    // B: column n = 2 t' + p of product j is the dim 2 j + p of a group of lane number t', row the dim that a lane of number t holds: signs by the parity
    // of the common bits
    const uint32_t sign = ((__popc(t & (g >> 1)) & 1) ? 0x80008000u : 0u) ^ ((g & 1) ? 0x80000000u : 0u);
    auto signed_dims = [&](const __half* per_dim, int group) {  // of a group of this lane
        uint2 w = *reinterpret_cast<const uint2*>(per_dim + t * kDimStride + 4 * group);
        w.x ^= sign;
        w.y ^= sign;
        return w;
    };

    int n = 0;
    for (int tile = first_tile; tile <= last_tile; tile += step, ++n) {
        const int buffer = n & 1;
        if (tid == 0) ask(tile + step, buffer ^ 1);
        const bool ok = mbar_wait_lane_bounded(&sm.full[buffer], (n >> 1) & 1, KVB_READ_PROBES);
        if (__syncthreads_or(!ok)) {
            if (tid == 0) {
                L.flag(KVB_ERR_WAIT_TIMEOUT);
                // no copy lands in shared memory that is no longer this CTA's
                mbar_wait_lane_bounded(&sm.full[buffer], (n >> 1) & 1);
                if (tile + step <= last_tile) mbar_wait_lane_bounded(&sm.full[buffer ^ 1], ((n + 1) >> 1) & 1);
            }
            return;
        }
        const int kind = sm.kind[buffer];
        const bool sealed = kind == kSealed;
        if (kind != kSkip) {
            const __half* const axes = sm.tile[buffer].axes;
            for (int d = tid; d < D; d += kReadThreads) {
                const int at = ((d >> 4) & 3) * kDimStride + 4 * (((d >> 2) & 3) | ((d >> 4) & 4)) + (d & 3);
                const __half* row = axes + leading * (d / c) + d % c;
                sm.dim_a[d / kSlice][0][at] = sealed ? row[0] : __float2half_rn(1.0f);
                if (!which) sm.dim_b[d / kSlice * 4 * kDimStride + at] = sealed ? row[c] : __float2half_rn(0.0f);
            }
            const __half* const token = axes + leading * tid + (which ? c : 2 * c);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                sm.token_a[s][tid] = sealed ? __half2float(token[s]) * kNorm : kNorm;
                sm.token_b[s][tid] = sealed && which ? __half2float(token[S + s]) * kNorm : 0.0f;
            }
            __syncthreads();
            // two groups a warp
            constexpr uint32_t kOnes = 0x3C003C00u;
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const int group = 2 * warp + m;
                    const uint2 b = signed_dims(which ? sm.dim_a[s][0] : sm.dim_b + s * 4 * kDimStride, group);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float d[4];
                        mma_apart(d, kOnes, kOnes, kOnes, kOnes, b.x, j ? b.y ^ 0x80008000u : b.y, 0.0f, 0.0f);
                        if (g == 0) *reinterpret_cast<float2*>(&sm.term[s][t][4 * group + 2 * j]) = make_float2(d[0], d[1]);
                    }
                }
            __syncthreads();

            const __half* const stage = L.stage_row(which, tile & 1, head, 0);
            const uint8_t* const code = sm.tile[buffer].code;
            uint16_t* const out = which ? out_v : out_k;
            const bool whole = (reinterpret_cast<uintptr_t>(out) & 31u) == 0;  // 32 bytes a store: 16 leave halves of the L2's sectors
            const int2 rows = rows_of(tile);
            // kAfter: the tokens' parts are applied to the sums (V); kCodes: rows of a sealed tile
            auto run = [&](auto after, auto codes) {
                constexpr bool kAfter = decltype(after)::value, kCodes = decltype(codes)::value;
#pragma unroll 1
                for (int from = 16 * warp; from < kTile; from += 16 * kReadWarps) {
                    const int row0 = from + g, row1 = row0 + 8;  // of the tile
                    if (tile * kTile + from > rows.y || tile * kTile + from + 15 < rows.x) continue;  // the whole warp's
                    auto rotated = [&](int s, F2 (&x)[8][2][2]) {  // slice s of 16 tokens: [group][j][token g, token g + 8], times what belongs to the token
                        const float a0 = sm.token_a[s][row0], a1 = sm.token_a[s][row1], b0 = sm.token_b[s][row0], b1 = sm.token_b[s][row1];
                        uint32_t w[2][4];
#pragma unroll
                        for (int side = 0; side < 2; ++side) {
                            const uint2 r0 = *reinterpret_cast<const uint2*>(code + row0 * G::kCodeLeading + 64 * s + 32 * side + 8 * t);
                            const uint2 r1 = *reinterpret_cast<const uint2*>(code + row1 * G::kCodeLeading + 64 * s + 32 * side + 8 * t);
                            w[0][2 * side] = r0.x;
                            w[0][2 * side + 1] = r0.y;
                            w[1][2 * side] = r1.x;
                            w[1][2 * side + 1] = r1.y;
                        }
#pragma unroll
                        for (int group = 0; group < 8; ++group) {
                            uint32_t a[4];
                            if constexpr (kCodes) {
                                a[0] = code_halves(w[0][group >> 1], 2 * (group & 1));
                                a[1] = code_halves(w[1][group >> 1], 2 * (group & 1));
                                a[2] = code_halves(w[0][group >> 1], 2 * (group & 1) + 1);
                                a[3] = code_halves(w[1][group >> 1], 2 * (group & 1) + 1);
                            } else {
                                const int dim = 128 * s + 16 * t + 4 * (group & 3) + 64 * (group >> 2);
                                const uint2 r0 = *reinterpret_cast<const uint2*>(stage + row0 * D + dim), r1 = *reinterpret_cast<const uint2*>(stage + row1 * D + dim);
                                a[0] = r0.x;
                                a[1] = r1.x;
                                a[2] = r0.y;
                                a[3] = r1.y;
                            }
                            const uint2 b = signed_dims(sm.dim_a[s][0], group);
                            const float4 term = *reinterpret_cast<const float4*>(&sm.term[s][t][4 * group]);
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float t0 = j ? term.z : term.x, t1 = j ? term.w : term.y;
                                float d[4];
                                mma_apart(d, a[0], a[1], a[2], a[3], b.x, j ? b.y ^ 0x80008000u : b.y, kAfter ? 0.0f : t0, kAfter ? 0.0f : t1);
                                x[group][j][0] = mul2(F2(d[0], d[1]), F2(a0, a0));
                                x[group][j][1] = mul2(F2(d[2], d[3]), F2(a1, a1));
                                if constexpr (kAfter) {
                                    x[group][j][0] = fma2(F2(t0, t1), F2(b0, b0), x[group][j][0]);
                                    x[group][j][1] = fma2(F2(t0, t1), F2(b1, b1), x[group][j][1]);
                                }
                            }
                        }
                        rotate_groups(x);
                    };
                    auto store = [&](int s, const F2 (&x)[8][2][2]) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int at = tile * kTile + (half ? row1 : row0);
                            if (at < rows.x || at > rows.y) continue;
                            uint16_t* const to = out + (static_cast<int64_t>(at - begin) * L.kv_heads + head) * D + 128 * s + 16 * t;
#pragma unroll
                            for (int side = 0; side < 2; ++side) {
                                uint32_t o[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const float2 y = x[4 * side + (e >> 1)][e & 1][half].get();
                                    o[e] = pack_out<kBf16>(y);
                                }
                                if (whole) {
                                    store32(to + 64 * side, o);
                                } else {
                                    *reinterpret_cast<uint4*>(to + 64 * side) = make_uint4(o[0], o[1], o[2], o[3]);
                                    *reinterpret_cast<uint4*>(to + 64 * side + 8) = make_uint4(o[4], o[5], o[6], o[7]);
                                }
                            }
                        }
                    };
                    F2 x[8][2][2];
                    rotated(0, x);
                    if constexpr (S == 1) {
                        store(0, x);
                    } else {
                        F2 y[8][2][2];
                        rotated(1, y);
#pragma unroll
                        for (int group = 0; group < 8; ++group)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int r = 0; r < 2; ++r) {
                                    const F2 lo = x[group][j][r], hi = y[group][j][r];
                                    x[group][j][r] = add2(lo, hi);
                                    y[group][j][r] = sub2(lo, hi);
                                }
                        store(0, x);
                        store(1, y);
                    }
                }
            };
            if (!sealed) run(std::true_type{}, std::false_type{});
            else if (which) run(std::true_type{}, std::true_type{});
            else run(std::false_type{}, std::true_type{});
        }
        fence_proxy_async();  // the buffer has been read, and a copy may be asked into it
        __syncthreads();
    }
}

template <int D, bool kBf16>
int launch_read(const LayerView& V, int begin, int tokens, const int32_t* total_pos, void* out_k, void* out_v, cudaStream_t stream) {
    constexpr int smem = static_cast<int>(sizeof(ReadSmem<D>));
    static OncePerDevice opted;  // per template instance
    KVB_CUDA_OK(allow_smem(opted, read_kernel<D, kBf16>, smem));
    // as many CTAs as are resident, a head of K or V each
    const int tiles = (begin + tokens - 1) / kTile - begin / kTile + 1, resident = device_sm_count() * (D == 256 ? 3 : 4) / (2 * V.kv_heads);
    const dim3 grid(tiles < resident ? tiles : resident, V.kv_heads, 2);
    KVB_CUDA_OK(launch_early(read_kernel<D, kBf16>, grid, dim3(kReadThreads), smem, stream, V, begin, begin + tokens, total_pos, static_cast<uint16_t*>(out_k),
                             static_cast<uint16_t*>(out_v)));
    return KVB_OK;
}

}  // namespace
}  // namespace kvb

extern "C" int kvb_read_rows(const kvb_layer* layer, int begin, int tokens, const int32_t* total_pos_dev, void* out_k, void* out_v, void* stream) {
    using namespace kvb;
    if (tokens == 0) return KVB_OK;
    if (int st = check_layer(layer, "kvb_read_rows")) return st;
    if (begin < 0 || tokens < 0 || static_cast<int64_t>(begin) + tokens > INT32_MAX - 2 * kTile) return fail(KVB_EINVAL, "kvb_read_rows: rows %d .. + %d", begin, tokens);
    if (total_pos_dev == nullptr || out_k == nullptr || out_v == nullptr) return fail(KVB_EINVAL, "kvb_read_rows: null position or output");
    if (((reinterpret_cast<uintptr_t>(out_k) | reinterpret_cast<uintptr_t>(out_v)) & 15u) != 0) return fail(KVB_EINVAL, "kvb_read_rows: outputs start at 16-byte boundaries");
    if (layer->stage == nullptr) return fail(KVB_EINVAL, "kvb_read_rows: layer has no stage buffer");
    const size_t bytes = sizeof(uint16_t) * static_cast<size_t>(tokens) * layer->kv_heads * layer->head_dim;
    if (overlap(span_of(out_k, bytes), span_of(out_v, bytes))) return fail(KVB_EINVAL, "kvb_read_rows: the outputs share memory");
    const LayerView V = make_view(*layer);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = layer->dtype == KVB_DTYPE_BF16;
    if (layer->head_dim == 128) return bf ? launch_read<128, true>(V, begin, tokens, total_pos_dev, out_k, out_v, s) : launch_read<128, false>(V, begin, tokens, total_pos_dev, out_k, out_v, s);
    return bf ? launch_read<256, true>(V, begin, tokens, total_pos_dev, out_k, out_v, s) : launch_read<256, false>(V, begin, tokens, total_pos_dev, out_k, out_v, s);
}
