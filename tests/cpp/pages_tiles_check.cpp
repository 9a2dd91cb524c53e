// The rows that the paged attention's tiles read (tile_lookup, tile_rows and seen_rows of
// neuralnet.cpp_amd/csrc/pages_index.hpp) on the CPU: random chunks, lengths and page sizes, walked as
// the kernels walk them. Prints the number of reads that are out of bounds or not where they should be.
#include "pages_index.hpp"

#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

using namespace nnhip;

int main()
{
    std::mt19937 rng(11);
    auto pick = [&](int lo, int hi) { return (int)std::uniform_int_distribution<int>(lo, hi)(rng); };
    long wrong = 0, seen = 0;
    for (int round = 0; round < 4000; ++round)
    {
        const int shift = pick(3, 10), page = 1 << shift, stride = pick(1, 3000 / page + 1);
        const int p = pick(0, std::min(stride * page, 3000) - 1);
        // decode: the new token at position p; chunks of a multiple of 64 positions, four waves' tiles of 16 rows in
        // turn, the ids of a tile looked up a turn before (of the first also where the chunk has no cached row)
        const int chunk = pick(0, 1) ? 128 : 64 * pick(2, 20);
        std::vector<int> reads(p + 1, 0);
        for (int t0 = 0; t0 <= p; t0 += chunk)
        {
            const int n = std::min(chunk, p - t0);
            for (int base = 0; base < n + 128; base += 16)
                for (int i = 0; i < 2; ++i)
                {
                    const int look = tile_lookup(t0, base + 8 * i, n);
                    wrong += look < 0 || look > p || (look >> shift) >= stride;
                    if (base >= n) continue;
                    const int at = tile_rows(t0, base + 8 * i, n);
                    // the 8 rows lie in the page looked up, within the table's positions
                    wrong += at < t0 || (at >> shift) != (look >> shift) || ((at + 7) >> shift) != (look >> shift);
                    wrong += (at & (page - 1)) + 7 >= page;
                    for (int r = 0; r < 8; ++r)
                    {
                        const int row = base + 8 * i + r;
                        if (row >= n) continue;   // its score is -infinity
                        wrong += at + r != t0 + row;
                        ++reads[t0 + row];
                        ++seen;
                    }
                }
        }
        for (int t = 0; t < p; ++t) wrong += reads[t] != 1;
        wrong += reads[p] != 0;  // the new token's own row is never read
        // prompts: the last key that an item sees, every tile up to its, one key and runs of four
        for (int kb = 0; kb <= p / 32; ++kb)
            for (int key = 0; key < 32; ++key)
            {
                const int t = 32 * kb + key, one = seen_rows(t, p, 1), run = seen_rows(t & ~3, p, 4) + (t & 3);
                wrong += one < 0 || one > p || (t <= p && one != t);
                wrong += run < 0 || (run >> shift) >= stride || (run >> shift) != (seen_rows(t & ~3, p, 4) >> shift);
                wrong += t <= p && run != t;
                wrong += (run & ~3) > p;  // its page is one that the item sees
                ++seen;
            }
    }
    std::printf("reads %ld wrong %ld\n", seen, wrong);
    return wrong != 0;
}
