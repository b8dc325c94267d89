// kvb_rope.cuh -- rotary positions: the angle of a (position, pair), and the rotation of rows in global memory.
//
// Dims (i, j) of a pair p of a head at position t become
//   y_i = x_i c - x_j s,  y_j = x_j c + x_i s,   c + i s = factor * exp(i t inv_freq[p])
// with (i, j) = (p, p + rotary / 2), or (2 p, 2 p + 1) where neighbouring dims turn together; dims from `rotary` on pass.
#pragma once

#include "kvb_common.cuh"
#include "kvb_ptx.cuh"

namespace kvb {

struct RopeView {
    const double* inv_freq;
    float factor;
    int rotary, interleaved;
};

// factor * (cos, sin) of the angle.  Angles grow to positions of a million radians, where fp32 has no fraction left: the turns are counted and
// reduced in 64 bits (off by 2^-53 of them), and what remains, at most half a turn, is rounded once for CUDA's sincospif.
__device__ __forceinline__ float2 rope_turn(double inv_freq, int position, float factor) {
    constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
    double turns = __dmul_rn(static_cast<double>(position), __dmul_rn(inv_freq, kTurn));
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns), &s, &c);
    return make_float2(__fmul_rn(c, factor), __fmul_rn(s, factor));
}
// The same for positions in a row: turns as 64-bit fractions of one, whose products and sums with whole numbers of positions are exact but for whole
// turns, so that the next position costs an addition.  `step`: turns per position, rounded to 2^-55 of one.
__device__ __forceinline__ uint64_t rope_step(double inv_freq) {
    const double turns = __dmul_rn(inv_freq, 0.15915494309189533577);
    return __double2ull_rz(__dmul_rn(turns - floor(turns), 18446744073709551616.0));
}
__device__ __forceinline__ float2 rope_turn_of(uint64_t phase, float factor) {
    float s, c;
    sincospif(static_cast<float>(static_cast<int32_t>((phase + 0x80000000u) >> 32)) * 0x1p-31f, &s, &c);
    return make_float2(__fmul_rn(c, factor), __fmul_rn(s, factor));
}
__device__ __forceinline__ float turn_first(float x, float peer, float2 t) { return __fmaf_rn(x, t.x, -__fmul_rn(peer, t.y)); }
__device__ __forceinline__ float turn_second(float x, float peer, float2 t) { return __fmaf_rn(x, t.x, __fmul_rn(peer, t.y)); }

// Rows of `heads` heads of each token, [tokens][heads][head_dim] with any distance between tokens.  An item is a unit of a head (8 pairs of
// dims, 4 neighbouring ones, or 8 dims that pass: 16-byte accesses; one pair or one dim where rows or `rotary` are not made for that) of
// one token, for every `splits`-th head: the angles are computed once for those.
struct RopeRows {
    RopeView rope;
    const uint16_t* x;
    uint16_t* out;
    const int32_t* positions;
    int64_t x_stride, out_stride, items;
    int heads, head_dim, units, splits;
    int in_a_row;  // that many positions have to follow one another from 0 or more on, or nothing is written; 0: any positions
};

template <bool kBf16> __device__ __forceinline__ void unpack8_16(uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = in_to_f32<kBf16>(static_cast<uint16_t>(w[e]));
        f[2 * e + 1] = in_to_f32<kBf16>(static_cast<uint16_t>(w[e] >> 16));
    }
}
template <bool kBf16> __device__ __forceinline__ uint4 pack8_16(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = static_cast<uint32_t>(f32_to_out<kBf16>(f[2 * e])) | static_cast<uint32_t>(f32_to_out<kBf16>(f[2 * e + 1])) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Heads of a thread whose loads are under way at once.
constexpr int kRopeAtOnce = 4;

constexpr int kRopeThreads = 128;

template <bool kBf16, bool kWide> __device__ __forceinline__ void rope_item(const RopeRows& P, int64_t item) {
    const int unit = static_cast<int>(item % P.units);
    const int64_t rest = item / P.units;
    const int split = static_cast<int>(rest % P.splits);
    const int64_t token = rest / P.splits;
    const int rotary = P.rope.rotary, half = rotary / 2;
    const bool inter = P.rope.interleaved != 0;
    constexpr int kUnit = kWide ? 8 : 1;                                          // pairs of a turning unit in two halves, dims of one that passes
    const int turning = kWide ? (inter ? rotary / 8 : half / 8) : half;           // units that turn
    const bool turns = unit < turning;
    // first dim of the unit, and of its other half
    const int at = !turns ? rotary + (unit - turning) * kUnit : inter ? (kWide ? 8 : 2) * unit : kUnit * unit;
    const int peer = turns ? (inter ? at + 1 : at + half) : at;
    const uint16_t* x = P.x + token * P.x_stride;
    uint16_t* out = P.out + token * P.out_stride;

    if constexpr (kWide) {
        float2 t[8];
        if (turns) {
            const int position = P.positions[token];
            const int pair = inter ? at / 2 : at;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < 4 || !inter) t[e] = rope_turn(P.rope.inv_freq[pair + e], position, P.rope.factor);
        }
        const bool two = turns && !inter;
        for (int h0 = split; h0 < P.heads; h0 += P.splits * kRopeAtOnce) {
            uint4 a[kRopeAtOnce], b[kRopeAtOnce];
#pragma unroll
            for (int u = 0; u < kRopeAtOnce; ++u) {
                const int h = h0 + u * P.splits;
                if (h >= P.heads) break;
                const uint16_t* row = x + static_cast<int64_t>(h) * P.head_dim;
                a[u] = *reinterpret_cast<const uint4*>(row + at);
                if (two) b[u] = *reinterpret_cast<const uint4*>(row + peer);
            }
#pragma unroll
            for (int u = 0; u < kRopeAtOnce; ++u) {
                const int h = h0 + u * P.splits;
                if (h >= P.heads) break;
                uint16_t* row = out + static_cast<int64_t>(h) * P.head_dim;
                if (turns) {
                    float f[8], g[8];
                    unpack8_16<kBf16>(a[u], f);
                    if (two) {
                        unpack8_16<kBf16>(b[u], g);
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = turn_first(f[e], g[e], t[e]);
                        a[u] = pack8_16<kBf16>(y);
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = turn_second(g[e], f[e], t[e]);
                        *reinterpret_cast<uint4*>(row + peer) = pack8_16<kBf16>(y);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            g[2 * e] = turn_first(f[2 * e], f[2 * e + 1], t[e]);
                            g[2 * e + 1] = turn_second(f[2 * e + 1], f[2 * e], t[e]);
                        }
                        a[u] = pack8_16<kBf16>(g);
                    }
                }
                *reinterpret_cast<uint4*>(row + at) = a[u];
            }
        }
    } else {
        float2 t = make_float2(1.0f, 0.0f);
        if (turns) t = rope_turn(P.rope.inv_freq[unit], P.positions[token], P.rope.factor);
        for (int h = split; h < P.heads; h += P.splits) {
            const uint16_t* from = x + static_cast<int64_t>(h) * P.head_dim;
            uint16_t* row = out + static_cast<int64_t>(h) * P.head_dim;
            const uint16_t a = from[at];
            if (turns) {
                const float f = in_to_f32<kBf16>(a), g = in_to_f32<kBf16>(from[peer]);
                row[at] = f32_to_out<kBf16>(turn_first(f, g, t));
                row[peer] = f32_to_out<kBf16>(turn_second(g, f, t));
            } else {
                row[at] = a;
            }
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
int check_rope(const kvb_rope* rope, int head_dim, const char* who);
// Turns rows, beside the append right before it in the stream where `beside` (kvb_step.hpp): nothing that it touches is the append's.
int launch_rope(const RopeRows& P, bool bf16, bool wide, bool beside, cudaStream_t stream);
// Whether rows, distances and the turning part allow 16-byte accesses.
inline bool rope_is_wide(const kvb_rope& rope, int head_dim, const void* x, const void* out, int64_t x_stride, int64_t out_stride) {
    const int whole = rope.interleaved ? 8 : 16;
    return rope.rotary_dim % whole == 0 && head_dim % 8 == 0 && x_stride % 8 == 0 && out_stride % 8 == 0 &&
           ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
}
RopeRows rope_rows_of(const kvb_rope& rope, const void* x, void* out, const int32_t* positions, int tokens, int heads, int head_dim, int64_t x_stride,
                      int64_t out_stride, bool wide);

// The part of a strided set of rows that a call touches, and whether two of them (rows of `width` elements) share memory: rows one
// distance apart may lie beside each other in the same buffer.
inline Span rows_span(const void* p, int tokens, int64_t stride, int64_t width) { return span_of(p, ((tokens - 1) * stride + width) * sizeof(uint16_t)); }
inline bool rows_overlap(const void* a, int64_t a_stride, int64_t a_width, const void* b, int64_t b_stride, int64_t b_width, int tokens) {
    if (!overlap(rows_span(a, tokens, a_stride, a_width), rows_span(b, tokens, b_stride, b_width))) return false;
    if (tokens == 1 || a_stride != b_stride) return true;
    const int64_t bytes = a_stride * 2, gap = static_cast<int64_t>(reinterpret_cast<intptr_t>(b) - reinterpret_cast<intptr_t>(a));
    const int64_t off = (gap % bytes + bytes) % bytes;
    return off < a_width * 2 || off + b_width * 2 > bytes;
}

}  // namespace kvb
