// The 8-bit pools' index arithmetic (csrc/pages_index.hpp) on the CPU: every byte of a pool belongs to one element, 16
// positions of a head to one run; and every block of a packed call's tokens to one work-group of 64 columns, as
// k_pages_fill_i8 divides them (columns behind the first 64 included). Prints "wrong N".
#include "pages_index.hpp"

#include <cstdio>
#include <random>
#include <vector>

using namespace nnhip;

int main()
{
    long wrong = 0;
    for (int dk : {64, 128, 256})
        for (int shift : {4, 5, 7})
        {
            const int pages = 3, Hkv = 2, page = 1 << shift;
            std::vector<int> k(pages * Hkv * page * dk), v(k.size());
            for (int id = 0; id < pages; ++id)
                for (int g = 0; g < Hkv; ++g)
                    for (int slot = 0; slot < page; ++slot)
                        for (int d = 0; d < dk; ++d)
                        {
                            const size_t row = page_row(id, g, slot, Hkv, shift), a = key_byte(row, d, dk), b = value_byte(row, d, dk);
                            if (a >= k.size() || b >= v.size()) return std::printf("outside\nwrong 1\n"), 1;
                            ++k[a], ++v[b];
                            const size_t group = row / 16 * 16 * (size_t)dk;
                            wrong += a < group || a >= group + 16 * (size_t)dk || b < group || b >= group + 16 * (size_t)dk;
                            // as the tensors of the handle have them
                            const size_t head = ((size_t)id * Hkv + g) * (page / 16) + slot / 16;
                            wrong += a != ((head * (dk / 16) + d / 16) * 16 + slot % 16) * 16 + d % 16;
                            wrong += b != (head * dk + d) * 16 + slot % 16;
                        }
            for (size_t i = 0; i < k.size(); ++i) wrong += (k[i] != 1) + (v[i] != 1);
        }
    // rows past 2^27 stay exact
    wrong += key_byte((size_t)0x7FFFFFF0u, 255, 256) != (size_t)0x7FFFFFFu * 4096u + 15 * 256 + 15;

    std::mt19937 rng(7);
    for (int turn = 0; turn < 4000; ++turn)
    {
        const int block = 16 << (int)(rng() % 3), B = 1 + (int)(rng() % 20), most = 1 + (int)(rng() % 200);
        std::vector<int> cu{(int)(rng() % 5)}, pos0;
        for (int b = 0; b < B; ++b)
        {
            cu.push_back(cu.back() + (int)(rng() % (most + 1)));
            pos0.push_back((int)(rng() % 300));
        }
        const int M = cu.back() + (int)(rng() % 70) - (turn % 7 == 0 ? 20 : 0), limit = 150 + (int)(rng() % 400);
        std::vector<int> seen(M > 0 ? M : 0);
        for (int m0 = 0; m0 < M; m0 += 64)
        {
            int last_b = -1, last_p = -1;
            for (int lane = 0; lane < 64; ++lane)
            {
                const int m = m0 + lane, b = m < M ? packed_sequence(cu.data(), B, m) : -1;
                int p = b < 0 ? -1 : packed_position(cu.data(), pos0.data(), b, m, limit);
                if (p >= 0 && block_column(m, cu[b], p, block) < m0) p = -1;
                if (p >= 0) ++seen[m];
                if (lane == 63) last_b = b, last_p = p;
            }
            if (last_b < 0 || last_p < 0) continue;
            const int left = block - 1 - (last_p & (block - 1));
            int more = left < limit - 1 - last_p ? left : limit - 1 - last_p;
            const int end = (cu[last_b + 1] < M ? cu[last_b + 1] : M) - (m0 + 64);
            more = end < more ? end : more;
            for (int i = 0; i < more; ++i)
            {
                const int m = m0 + 64 + i;
                if (m >= M || packed_sequence(cu.data(), B, m) != last_b) ++wrong;
                else ++seen[m];
                wrong += block_column(m, cu[last_b], last_p + 1 + i, block) != block_column(m0 + 63, cu[last_b], last_p, block);
            }
            wrong += more > 63;
        }
        for (int m = 0; m < M; ++m)
        {
            const int b = packed_sequence(cu.data(), B, m);
            const int want = b >= 0 && packed_position(cu.data(), pos0.data(), b, m, limit) >= 0;
            wrong += seen[m] != want;
        }
    }
    std::printf("wrong %ld\n", wrong);
    return wrong != 0;
}
