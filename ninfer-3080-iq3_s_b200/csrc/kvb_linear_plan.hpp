// kvb_linear_plan.hpp -- how the chunked form of linear attention deals the segments of its sequences to the units of its grid and to the places of its
// workspace.  Host and device, no CUDA.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define KVB_LINEAR_PLAN __host__ __device__ __forceinline__
#else
#define KVB_LINEAR_PLAN inline
#endif

namespace kvb {

constexpr int kMostSequences = 256;  // of one call
constexpr int kLinearChunk = 64;     // tokens that the chunked form takes at a time

// Tokens of a segment, for sequences of the average length: what costs least, in chunks of the second launch, by waves of CTAs (one an SM).  A CTA costs 4
// chunks beside its own there (states in and out, the pipeline's start), the first launch 0.45 of a chunk and 2.5.  Measured on B200, 32 value heads of 128
// dims: 2.1 us a chunk in the second launch, 0.9 in the first.  (Lengths that are far apart: 8,192 tokens with 7 single ones are one segment, 274 us; 110 alone.)
inline int linear_segment_of(int tokens, int batch, int v_heads, int sms) {
    const int64_t sequences = batch < 1 ? 1 : batch, units = sequences * v_heads;
    const int64_t length = (static_cast<int64_t>(tokens) + sequences * kLinearChunk - 1) / (sequences * kLinearChunk);
    const int64_t whole = (static_cast<int64_t>(tokens) + kLinearChunk - 1) / kLinearChunk;  // one segment, whichever sequence has the tokens
    auto waves = [&](int64_t ctas) { return static_cast<double>((ctas + sms - 1) / sms); };
    double least = waves(units) * (static_cast<double>(length) + 4.0);
    int64_t segment = whole;
    for (int64_t n = 2; n <= length && n <= 64; ++n) {
        const int64_t chunks = (length + n - 1) / n;
        const double cost = waves(units * n) * (static_cast<double>(chunks) + 4.0) + waves(units * (n - 1)) * (0.45 * static_cast<double>(chunks) + 2.5);
        if (cost < least) least = cost, segment = chunks;
    }
    return static_cast<int>((segment < 1 ? 1 : segment) * kLinearChunk);
}
// Units of the grid, and places of the workspace (a state a head each) where a sequence may have several segments: enough for sequences that do not
// share rows.
inline int linear_units(int tokens, int batch, int segment) { return tokens / segment + batch; }

// Segments of the sequence of rows offsets[seq] .. offsets[seq + 1] - 1; one where it has no rows, or is refused for them.
KVB_LINEAR_PLAN int linear_segments(const int32_t* offsets, int seq, int tokens, int segment) {
    const int64_t length = static_cast<int64_t>(offsets[seq + 1]) - offsets[seq];
    return length <= 0 || length > tokens ? 1 : static_cast<int>((length + segment - 1) / segment);
}
// Where a sequence comes in the order of the units: the longest first, then by number.
KVB_LINEAR_PLAN int linear_rank(const int32_t* offsets, int seq, int batch) {
    const int64_t mine = static_cast<int64_t>(offsets[seq + 1]) - offsets[seq];
    int rank = 0;
    for (int s = 0; s < batch; ++s) {
        const int64_t length = static_cast<int64_t>(offsets[s + 1]) - offsets[s];
        rank += length > mine || (length == mine && s < seq);
    }
    return rank;
}
// A unit that is segment `index` of `count` uses the places of its sequence's units, [unit - index, unit - index + count), and no other: whether these are
// all there.  Sequences that share rows (offsets that fall) have more segments than the grid has units; one whose last units are not there is
// left alone, by all of its units and in both launches.
KVB_LINEAR_PLAN bool linear_fits(int unit, int index, int count, int units) { return unit - index + count <= units; }

// Tiles come chunk by chunk into kLinearStages stages in turn, a stage's next one when the chunk before it there is done with.  Of `issued` chunks that were asked
// for, the first that may still be under way; chunk c's barrier is that of its stage, in phase c / kLinearStages.
constexpr int kLinearStages = 3;
KVB_LINEAR_PLAN int linear_first_in_flight(int issued) { return issued > kLinearStages ? issued - kLinearStages : 0; }

}  // namespace kvb
