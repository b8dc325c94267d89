// kvb_read.cu -- rows of the cache back as 16-bit keys and values: codes de-quantised, the Walsh-Hadamard rotation undone.
//
//   x = H ((code * scale_axis + zp_axis) * other_axis)   rows of sealed tiles (scale and zero point per dim for K, per token for V)
//   x = H stage                                          rows of the open tile
// in fp32, rounded once.  A CTA has one tile of one head of K or V.  A lane holds 32 neighbouring dims of a row -- one 16-byte load of codes --
// and D / 32 lanes a row, so the strides up to 16 of the rotation stay inside a lane.
#include "kvb_common.cuh"
#include "kvb_ptx.cuh"

namespace kvb {
namespace {

constexpr int kReadThreads = 128;

// Two codes of a byte as floats: 2^23 + code has the code in its last bits.
__device__ __forceinline__ F2 code_pair(uint32_t w, int byte) {
    const uint32_t lo = lop3_and_or(w >> (8 * byte), 15u, 0x4B000000u), hi = lop3_and_or(w >> (8 * byte + 4), 15u, 0x4B000000u);
    return sub2(F2(__uint_as_float(lo), __uint_as_float(hi)), F2(8388608.0f, 8388608.0f));
}
__device__ __forceinline__ F2 half_pair(uint32_t w) {
    const float2 f = unpack_half2(w);
    return F2(f.x, f.y);
}

// 32 neighbouring dims (pairs (x[0], x[1]), ...) of a row on each of kLanes lanes: the rotation, normalised.
template <int D> __device__ __forceinline__ void hadamard_lanes(F2 (&x)[16], int block) {
    constexpr int kLanes = D / 32;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const float2 y = x[e].get();
        x[e] = F2(y.x + y.y, y.x - y.y);
    }
#pragma unroll
    for (int span = 1; span <= 8; span <<= 1)
#pragma unroll
        for (int b = 0; b < 16; b += 2 * span)
#pragma unroll
            for (int e = 0; e < span; ++e) {
                const F2 lo = x[b + e], hi = x[b + e + span];
                x[b + e] = add2(lo, hi);
                x[b + e + span] = sub2(lo, hi);
            }
    constexpr float norm = D == 256 ? 0.0625f : 0.08838834764831845f;
#pragma unroll
    for (int step = 1; step < kLanes; step <<= 1) {
        const float sign = (block & step) == 0 ? 1.0f : -1.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float2 y = x[e].get();
            const F2 peer(__shfl_xor_sync(0xffffffffu, y.x, step), __shfl_xor_sync(0xffffffffu, y.y, step));
            x[e] = fma2(x[e], F2(sign, sign), peer);
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = mul2(x[e], F2(norm, norm));
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kReadThreads) read_kernel(LayerView L, int begin, int end, const int32_t* __restrict__ total_pos, uint16_t* __restrict__ out_k,
                                                            uint16_t* __restrict__ out_v) {
    using G = Geo<D>;
    constexpr int S = G::S, c = G::kAxisCols, kLanes = D / 32, kAtOnce = 32 / kLanes, kPasses = kTile / (kReadThreads / 32 * kAtOnce);
    constexpr int kMostLeading = G::kKScaleLeading;
    __shared__ __align__(16) __half axes[2 * kPage * kMostLeading];  // the scale pages of the tile's two pages
    grid_dependency_wait();
    launch_dependents();
    const int tile = begin / kTile + blockIdx.x, head = blockIdx.y, which = blockIdx.z;
    const int newest = *total_pos;
    const int first = max(begin, tile * kTile), last = min(end - 1, min(newest, tile * kTile + kTile - 1));  // rows of the tile to be read
    if (first > last) return;
    const bool sealed = tile * kTile + kTile - 1 <= newest;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, block = lane % kLanes;
    uint16_t* const out = which ? out_v : out_k;
    auto row_of = [&](int pass) { return (pass * (kReadThreads / 32) + warp) * kAtOnce + lane / kLanes; };  // of the tile
    auto store = [&](int row, F2 (&x)[16]) {
        hadamard_lanes<D>(x, block);
        const int at = tile * kTile + row;
        if (at < first || at > last) return;
        uint4* to = reinterpret_cast<uint4*>(out + (static_cast<int64_t>(at - begin) * L.kv_heads + head) * D + 32 * block);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 y = x[4 * j + e].get();
                w[e] = static_cast<uint32_t>(f32_to_out<kBf16>(y.x)) | static_cast<uint32_t>(f32_to_out<kBf16>(y.y)) << 16;
            }
            to[j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };

    if (!sealed) {
        const __half* const stage = L.stage_row(which, tile & 1, head, 0);
#pragma unroll 1
        for (int pass = 0; pass < kPasses; ++pass) {
            const int row = row_of(pass);
            F2 x[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 w = reinterpret_cast<const uint4*>(stage + row * D + 32 * block)[j];
                x[4 * j] = half_pair(w.x);
                x[4 * j + 1] = half_pair(w.y);
                x[4 * j + 2] = half_pair(w.z);
                x[4 * j + 3] = half_pair(w.w);
            }
            store(row, x);
        }
        return;
    }

    const int32_t* const tbl = L.table();
    const int32_t page0 = L.page_of(tbl, 2 * tile), page1 = L.page_of(tbl, 2 * tile + 1);
    if (page0 < 0 || page1 < 0) return;  // error word already set; the tile's rows are left as they are
    const int leading = which ? G::kVScaleLeading : G::kKScaleLeading;
    {
        const __half* const scale = which ? L.v_scale : L.k_scale;
        const int words = kPage * leading / 8;
        for (int i = threadIdx.x; i < 2 * words; i += kReadThreads) {
            const __half* from = scale + page_head_offset(leading, L.kv_heads, i < words ? page0 : page1, head);
            reinterpret_cast<uint4*>(axes)[i] = reinterpret_cast<const uint4*>(from)[i < words ? i : i - words];
        }
    }
    const uint8_t* const code = which ? L.v_code : L.k_code;
    uint4 raw[kPasses];
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
        const int row = row_of(pass);
        raw[pass] = *reinterpret_cast<const uint4*>(code + page_head_offset(G::kCodeLeading, L.kv_heads, row < kPage ? page0 : page1, head) + (row % kPage) * G::kCodeLeading + 16 * block);
    }
    __syncthreads();
    // what belongs to a dim: K's scale and zero point, V's factor
    F2 scale[16], zp[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int d = 32 * block + 2 * e;
        const __half* row = axes + leading * (d / c) + d % c;
        scale[e] = F2(__half2float(row[0]), __half2float(row[1]));
        if (!which) zp[e] = F2(__half2float(row[c]), __half2float(row[c + 1]));
    }
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
        const int row = row_of(pass);
        const __half* token = axes + leading * row + (which ? c : 2 * c) + (32 * block) / kSlice;
        const float a = __half2float(token[0]), b = which ? __half2float(token[S]) : 0.0f;
        const uint32_t w[4] = {raw[pass].x, raw[pass].y, raw[pass].z, raw[pass].w};
        F2 x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const F2 q = code_pair(w[e / 4], e % 4);
            x[e] = which ? mul2(fma2(q, F2(a, a), F2(b, b)), scale[e]) : mul2(fma2(q, scale[e], zp[e]), F2(a, a));
        }
        store(row, x);
    }
}

template <int D, bool kBf16>
int launch_read(const LayerView& V, int begin, int tokens, const int32_t* total_pos, void* out_k, void* out_v, cudaStream_t stream) {
    const dim3 grid((begin + tokens - 1) / kTile - begin / kTile + 1, V.kv_heads, 2);
    KVB_CUDA_OK(launch_early(read_kernel<D, kBf16>, grid, dim3(kReadThreads), 0, stream, V, begin, begin + tokens, total_pos, static_cast<uint16_t*>(out_k),
                             static_cast<uint16_t*>(out_v)));
    return KVB_OK;
}

}  // namespace
}  // namespace kvb

extern "C" int kvb_read_rows(const kvb_layer* layer, int begin, int tokens, const int32_t* total_pos_dev, void* out_k, void* out_v, void* stream) {
    using namespace kvb;
    if (tokens == 0) return KVB_OK;
    if (int st = check_layer(layer, "kvb_read_rows")) return st;
    if (begin < 0 || tokens < 0 || static_cast<int64_t>(begin) + tokens > INT32_MAX - kTile) return fail(KVB_EINVAL, "kvb_read_rows: rows %d .. + %d", begin, tokens);
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
