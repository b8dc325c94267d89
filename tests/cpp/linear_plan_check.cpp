// The units of linear attention's chunked form: sequences behind one another all fit their grid, each segment one unit; whatever the offsets, no unit that runs
// touches a place outside the workspace.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "kvb_linear_plan.hpp"

using namespace kvb;

static int bad = 0, refused = 0;
static void wrong(const char* what, int tokens, int batch, int at) {
    if (bad++ < 10) std::printf("%s: %d tokens, %d sequences, at %d\n", what, tokens, batch, at);
}

// As the kernel goes: a unit's sequence and segment by the order of the lengths.
static void deal(const std::vector<int32_t>& offsets, int tokens, int v_heads, int sms, bool in_a_row) {
    const int batch = static_cast<int>(offsets.size()) - 1, segment = linear_segment_of(tokens, batch, v_heads, sms), units = linear_units(tokens, batch, segment);
    if (segment < kLinearChunk || segment % kLinearChunk != 0) return wrong("segment", tokens, batch, segment);
    std::vector<int> order(batch, -1);
    for (int s = 0; s < batch; ++s) {
        const int rank = linear_rank(offsets.data(), s, batch);
        if (rank < 0 || rank >= batch || order[rank] >= 0) return wrong("rank", tokens, batch, s);
        order[rank] = s;
    }
    int base = 0;
    bool fits_all = true;
    for (int n = 0; n < batch; ++n) {
        const int s = order[n], count = linear_segments(offsets.data(), s, tokens, segment);
        if (count < 1) return wrong("count", tokens, batch, s);
        const int64_t begin = offsets[s], end = offsets[s + 1];
        const bool valid = begin >= 0 && end >= begin && end <= tokens;
        int running = 0;
        for (int index = 0; index < count; ++index) {
            const int unit = base + index;
            if (unit >= units) continue;  // not in the grid
            const bool fits = linear_fits(unit, index, count, units);
            fits_all = fits_all && fits;
            if (!valid || !fits) continue;
            ++running;
            // its own place, those of the segments before, and for the first one the last's
            for (int place : {unit, unit - index, index > 0 ? unit - 1 : unit, index == 0 ? unit + count - 1 : unit})
                if (place < 0 || place >= units) wrong("place", tokens, batch, place);
            const int64_t from = begin + static_cast<int64_t>(index) * segment, to = index == count - 1 ? end : from + segment;
            if (from > to || to > end || (count > 1 && from == to)) wrong("rows", tokens, batch, unit);
        }
        if (running != 0 && running != count) wrong("a part of a sequence", tokens, batch, s);
        if (base + count > units) fits_all = false;
        base += count;
    }
    if (in_a_row && !fits_all) wrong("does not fit", tokens, batch, base);
    if ((base <= units) != fits_all) wrong("report", tokens, batch, base);
    refused += !fits_all;
}

int main() {
    std::mt19937 rng(1);
    auto below = [&](int n) { return static_cast<int>(rng() % static_cast<uint32_t>(n)); };
    for (int round = 0; round < 6000; ++round) {
        const int batch = 1 + (round % 7 == 0 ? below(kMostSequences) : below(9)), v_heads = 1 << below(9), sms = round % 3 ? 148 : 1 + below(200);
        const int tokens = 1 + below(round % 5 == 0 ? 2000000000 : round % 2 ? 300000 : 9000);
        std::vector<int32_t> offsets(batch + 1);
        for (auto& x : offsets) x = below(tokens) + below(2);
        std::vector<int32_t> sorted = offsets;
        for (size_t i = 1; i < sorted.size(); ++i)
            for (size_t j = i; j > 0 && sorted[j] < sorted[j - 1]; --j) std::swap(sorted[j], sorted[j - 1]);
        deal(sorted, tokens, v_heads, sms, true);
        sorted.front() = 0, sorted.back() = tokens;
        deal(sorted, tokens, v_heads, sms, true);
        deal(offsets, tokens, v_heads, sms, false);
        for (size_t i = 0; i < offsets.size(); ++i) offsets[i] = i % 2 ? tokens : 0;  // every other one has all rows
        deal(offsets, tokens, v_heads, sms, false);
        for (auto& x : offsets)
            if (below(3) == 0) x = below(2) ? INT32_MIN + below(100) : INT32_MAX - below(100);
        deal(offsets, tokens, v_heads, sms, false);
    }
    // two sequences of the same 9,000 rows, 4 heads: the second one's units are not all there
    {
        const std::vector<int32_t> offsets{0, 9000, 0, 9000};
        const int segment = linear_segment_of(9000, 3, 4, 148), units = linear_units(9000, 3, segment), count = linear_segments(offsets.data(), 2, 9000, segment);
        if (count < 2 || !linear_fits(0, 0, count, units) || linear_fits(count, 0, count, units)) wrong("twice the same rows", 9000, 3, count);
    }
    if (refused == 0) wrong("nothing refused", 0, 0, 0);
    std::printf(bad ? "linear plan: %d wrong\n" : "linear plan: ok\n", bad);
    return bad != 0;
}
