// kvb_rope.cu -- rotary positions of rows in global memory, and the frequencies of the usual scalings for long contexts.
//
// Bound by memory: each row is read and written once, 16 bytes an access.  The angles cost about 40 instructions a pair, so a thread keeps
// those of its 8 pairs in registers for several heads of the token; the fewer tokens a call has, the fewer heads a thread takes.
// Measured on B200, graph replay: 8,192 tokens of 28 heads of 128 dims 23.0 us, 5.1 TB/s, 78 % of a copy (the angles of 64 pairs a token in 64 bits
// are the rest); one token 2.4 us.
#include <cmath>

#include "kvb_rope.cuh"

namespace kvb {

int check_rope(const kvb_rope* rope, int head_dim, const char* who) {
    if (rope == nullptr || rope->inv_freq == nullptr) return fail(KVB_EINVAL, "%s: null rope / inv_freq", who);
    if ((reinterpret_cast<uintptr_t>(rope->inv_freq) & 7u) != 0) return fail(KVB_EINVAL, "%s: inv_freq starts at an 8-byte boundary", who);
    if (rope->rotary_dim < 2 || rope->rotary_dim % 2 != 0 || rope->rotary_dim > head_dim)
        return fail(KVB_EINVAL, "%s: rotary_dim %d must be even, 2..head_dim (%d)", who, rope->rotary_dim, head_dim);
    if (rope->interleaved != 0 && rope->interleaved != 1) return fail(KVB_EINVAL, "%s: interleaved = %d", who, rope->interleaved);
    if (!std::isfinite(rope->factor)) return fail(KVB_EINVAL, "%s: factor is not finite", who);
    return KVB_OK;
}

RopeRows rope_rows_of(const kvb_rope& rope, const void* x, void* out, const int32_t* positions, int tokens, int heads, int head_dim, int64_t x_stride,
                      int64_t out_stride, bool wide) {
    RopeRows P;
    P.rope = {rope.inv_freq, rope.factor, rope.rotary_dim, rope.interleaved};
    P.x = static_cast<const uint16_t*>(x);
    P.out = static_cast<uint16_t*>(out);
    P.positions = positions;
    P.x_stride = x_stride;
    P.out_stride = out_stride;
    P.heads = heads;
    P.head_dim = head_dim;
    P.in_a_row = 0;
    const int turning = wide ? (rope.interleaved ? rope.rotary_dim / 8 : rope.rotary_dim / 16) : rope.rotary_dim / 2;
    const int passing = x == out ? 0 : (head_dim - rope.rotary_dim) / (wide ? 8 : 1);  // in place they are there already
    P.units = turning + passing;
    // as many heads a thread as leave 512 threads an SM
    const int64_t per_head = static_cast<int64_t>(tokens) * P.units, want = static_cast<int64_t>(device_sm_count()) * 512;
    const int64_t splits = (want + per_head - 1) / per_head;
    P.splits = static_cast<int>(splits < 1 ? 1 : splits > heads ? heads : splits);
    P.items = per_head * P.splits;
    return P;
}

namespace {

template <bool kBf16, bool kWide> __global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeRows P, bool beside) {
    if (!beside) grid_dependency_wait();
    launch_dependents();
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kRopeThreads + threadIdx.x;
    bool sound = true;
    if (P.in_a_row > 0) {
        const int first = P.positions[0], last = P.positions[P.in_a_row - 1];
        sound = first >= 0 && last - first == P.in_a_row - 1;
    }
    if (sound && item < P.items) rope_item<kBf16, kWide>(P, item);
    // One CTA leaves after the append is over, so that what waits for this grid finds both done; the others make room.  (All of them waiting:
    // 1,024 tokens of 24 heads of 128 dims beside 4 of keys 11.9 us, one 9.0.)
    if (beside && blockIdx.x == 0) grid_dependency_wait();
}

}  // namespace

int launch_rope(const RopeRows& P, bool bf16, bool wide, bool beside, cudaStream_t stream) {
    const int64_t blocks = (P.items + kRopeThreads - 1) / kRopeThreads;
    if (blocks > INT32_MAX) return fail(KVB_ERANGE, "rotary positions: too many rows for one call");
    auto* kernel = wide ? (bf16 ? rope_kernel<true, true> : rope_kernel<false, true>) : (bf16 ? rope_kernel<true, false> : rope_kernel<false, false>);
    KVB_CUDA_OK(launch_early(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kRopeThreads), 0, stream, P, beside));
    return KVB_OK;
}

}  // namespace kvb

extern "C" int kvb_rope_frequencies(int rotary_dim, double base, int scaling, double factor, int original_len, double* inv_freq, float* attention_factor) {
    using namespace kvb;
    if (rotary_dim < 2 || rotary_dim % 2 != 0) return fail(KVB_EINVAL, "kvb_rope_frequencies: rotary_dim %d must be even and positive", rotary_dim);
    if (inv_freq == nullptr || attention_factor == nullptr) return fail(KVB_EINVAL, "kvb_rope_frequencies: null output");
    if (!(base > 1.0) || !std::isfinite(base)) return fail(KVB_EINVAL, "kvb_rope_frequencies: base %g must be above 1", base);
    if (scaling < KVB_ROPE_PLAIN || scaling > KVB_ROPE_YARN) return fail(KVB_EINVAL, "kvb_rope_frequencies: scaling %d", scaling);
    if (scaling != KVB_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor)))
        return fail(KVB_EINVAL, "kvb_rope_frequencies: factor %g must be at least 1", factor);
    if (scaling == KVB_ROPE_YARN && original_len < 1) return fail(KVB_EINVAL, "kvb_rope_frequencies: original_len %d", original_len);
    const double pi = 3.14159265358979323846;
    const int pairs = rotary_dim / 2;
    if (scaling == KVB_ROPE_NTK && rotary_dim > 2) base *= std::pow(factor, rotary_dim / (rotary_dim - 2.0));
    // the pair that makes n turns over the original context
    auto pair_of = [&](double n) { return rotary_dim * std::log(original_len / (n * 2.0 * pi)) / (2.0 * std::log(base)); };
    double low = 0.0, width = 1.0;
    if (scaling == KVB_ROPE_YARN) {
        low = std::fmax(std::floor(pair_of(32.0)), 0.0);
        width = std::fmax(std::fmin(std::ceil(pair_of(1.0)), rotary_dim - 1.0) - low, 1e-3);
    }
    for (int p = 0; p < pairs; ++p) {
        double f = std::pow(base, -2.0 * p / rotary_dim);
        if (scaling == KVB_ROPE_LINEAR) f /= factor;
        if (scaling == KVB_ROPE_YARN) {
            const double ramp = std::fmin(std::fmax((p - low) / width, 0.0), 1.0);
            f = f / factor * ramp + f * (1.0 - ramp);
        }
        inv_freq[p] = f;
    }
    *attention_factor = scaling == KVB_ROPE_YARN ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
    return KVB_OK;
}

extern "C" int kvb_rope_rows(const kvb_rope* rope, const void* x, int64_t x_stride, void* out, int64_t out_stride, const int32_t* positions_dev, int tokens,
                             int heads, int head_dim, int dtype, void* stream) {
    using namespace kvb;
    if (tokens == 0) return KVB_OK;
    if (head_dim < 2 || head_dim > 1024) return fail(KVB_EINVAL, "kvb_rope_rows: head_dim %d (2..1024)", head_dim);
    if (int st = check_rope(rope, head_dim, "kvb_rope_rows")) return st;
    if (x == nullptr || out == nullptr || positions_dev == nullptr) return fail(KVB_EINVAL, "kvb_rope_rows: null x / out / positions");
    if (tokens < 0 || heads < 1) return fail(KVB_EINVAL, "kvb_rope_rows: tokens = %d, heads = %d", tokens, heads);
    if (heads > 4096) return fail(KVB_ERANGE, "kvb_rope_rows: heads = %d (at most 4096)", heads);
    if (dtype != KVB_DTYPE_F16 && dtype != KVB_DTYPE_BF16) return fail(KVB_EINVAL, "kvb_rope_rows: dtype %d", dtype);
    const int64_t width = static_cast<int64_t>(heads) * head_dim;
    if (tokens > 1 && (x_stride < width || out_stride < width)) return fail(KVB_EINVAL, "kvb_rope_rows: a row of %lld elements is longer than the distance to the next", static_cast<long long>(width));
    const bool in_place = x == out && (tokens == 1 || x_stride == out_stride);
    if (!in_place && rows_overlap(x, x_stride, width, out, out_stride, width, tokens)) return fail(KVB_EINVAL, "kvb_rope_rows: out shares memory with x and is not x itself");
    const Span written = rows_span(out, tokens, out_stride, width);
    if (overlap(written, span_of(positions_dev, sizeof(int32_t) * static_cast<size_t>(tokens))) || overlap(written, span_of(rope->inv_freq, sizeof(double) * (rope->rotary_dim / 2))))
        return fail(KVB_EINVAL, "kvb_rope_rows: out shares memory with the positions or frequencies");
    const bool wide = rope_is_wide(*rope, head_dim, x, out, x_stride, out_stride);
    const RopeRows P = rope_rows_of(*rope, x, out, positions_dev, tokens, heads, head_dim, x_stride, out_stride, wide);
    return launch_rope(P, dtype == KVB_DTYPE_BF16, wide, false, static_cast<cudaStream_t>(stream));
}
