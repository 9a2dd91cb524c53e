// Bounds of the paged cache's index arithmetic (neuralnet.cpp_amd/csrc/pages_index.hpp) on the CPU: random
// caches, lengths, chunks, packings (well-formed and not) and tables (with bad ids), walked as the
// kernels walk them. Prints the number of places that are out of bounds or not where they should be.
#include "pages_index.hpp"

#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

using namespace nnhip;

int main()
{
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return (int)std::uniform_int_distribution<int>(lo, hi)(rng); };
    long wrong = 0, seen = 0;
    for (int round = 0; round < 3000; ++round)
    {
        const int shift = pick(3, 10), Hkv = pick(1, 9), num_pages = pick(1, 40), stride = pick(1, 30);
        const long rows = (long)num_pages * Hkv << shift;
        const int capacity = stride << shift;
        std::vector<int32_t> table(stride);
        for (auto& id : table) id = pick(0, 9) ? pick(0, num_pages - 1) : (pick(0, 1) ? num_pages + pick(0, 5) : -pick(1, 9));
        // one decode step: every chunk of a sequence at position p
        const int chunk = 128 << pick(0, 3), p = pick(0, capacity - 1);
        std::vector<int> reads(p + 1, 0);
        for (int t0 = 0; t0 <= p; t0 += chunk)
        {
            const int n = std::min(chunk, p - t0);
            const bool has_new = p - t0 < chunk;
            const int entries = page_entries(t0, t0 + n - (has_new ? 0 : 1), shift), e0 = t0 >> shift;
            wrong += entries < 1 || entries > 1024 / 8 || e0 + entries > stride;
            for (int t = t0; t < t0 + n + (has_new ? 1 : 0); ++t)
            {
                const int e = (t >> shift) - e0;
                wrong += e < 0 || e >= entries;
                ++reads[t];
                const int id = table[e0 + e];
                if (!page_ok(id, num_pages)) continue;
                const size_t row = page_row(id, pick(0, Hkv - 1), t & ((1 << shift) - 1), Hkv, shift);
                wrong += row >= (size_t)rows;
                ++seen;
            }
            wrong += has_new && (p >> shift) - e0 != entries - 1;
        }
        for (int r : reads) wrong += r != 1;
        // a packed call
        const int B = pick(0, 12), M = pick(1, 200), limit = pick(1, capacity);
        std::vector<int32_t> cu(B + 1), pos0(B + 1);
        const bool sane = pick(0, 2) != 0;
        for (int b = 0; b <= B; ++b)
        {
            cu[b] = sane ? pick(0, M) : pick(-5, M + 50);
            pos0[b] = sane ? pick(0, limit) : pick(-3, 2 * limit);
        }
        if (sane) std::sort(cu.begin(), cu.end());
        for (int m = 0; m < M; ++m)
        {
            const int b = packed_sequence(cu.data(), B, m);
            wrong += b < -1 || b >= B;
            if (b >= 0) wrong += cu[b] > m || cu[b + 1] <= m;
            if (sane)
            {
                int want = -1;
                for (int i = 0; i < B; ++i)
                    if (cu[i] <= m && m < cu[i + 1]) want = i;
                wrong += want != b;
            }
            if (b < 0) continue;
            const int pos = packed_position(cu.data(), pos0.data(), b, m, limit);
            wrong += pos < -1 || pos >= limit;
            if (pos >= 0) wrong += pos != pos0[b] + m - cu[b] || (pos >> shift) >= stride;
            ++seen;
        }
    }
    // a large cache: rows past 2^31 elements
    wrong += page_row(2000000, 3, 15, 8, 6) != ((size_t)2000000 * 8 + 3) * 64 + 15;
    std::printf("places %ld wrong %ld\n", seen, wrong);
    return wrong != 0;
}
