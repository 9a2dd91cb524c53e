// pages_index.hpp — where a position of a paged sequence lies. Plain arithmetic that the kernels share
// with CPU tests (tests/cpp/pages_index_check.cpp, pages_tiles_check.cpp), so that its bounds are checked
// without a GPU.
#pragma once

#include <cstddef>
#include <cstdint>

#ifdef __HIPCC__
#define NNHIP_HD __host__ __device__ __forceinline__
#else
#define NNHIP_HD inline
#endif

namespace nnhip
{

// A table entry that may be followed
NNHIP_HD bool page_ok(int id, int num_pages) { return id >= 0 && id < num_pages; }

// Row (of dk elements) of head g, slot `slot` of page id in a pool (num_pages, Hkv, page_size, dk)
NNHIP_HD size_t page_row(int id, int g, int slot, int Hkv, int shift)
{
    return (((size_t)id * (size_t)Hkv + (size_t)g) << shift) + (size_t)slot;
}

// Position of a chunk (its first position t0, a multiple of 8, n > 0 cached rows) where the decode's tile of
// rows at, at + 1, ... looks up its page: its own, or the chunk's last one (n == 0: the chunk's first).
NNHIP_HD int tile_lookup(int t0, int at, int n) { return t0 + (at < n ? at : n > 0 ? n - 1 : 0); }

// Position of the first of 8 rows that such a tile reads, which lie in that page: its own rows, or those that
// hold the chunk's last one
NNHIP_HD int tile_rows(int t0, int at, int n)
{
    const int last = (n - 1) & ~7;
    return t0 + (at < last ? at : last);
}

// Position whose row(s) the prompt's tile reads for position t: its own, or, for t past the last one that is seen,
// the run of `run` (a power of two, up to 8) positions with that one
NNHIP_HD int seen_rows(int t, int last, int run)
{
    const int end = last & -run;
    return t < end ? t : end;
}

// Table entries that positions [t0, last] of a sequence need, from entry t0 >> shift on (the kernels look theirs up
// one at a time; a count for tests that walk chunks)
NNHIP_HD int page_entries(int t0, int last, int shift) { return (last >> shift) - (t0 >> shift) + 1; }

// The sequence of column m of a packed call: the first b with cu[b + 1] > m, or -1 if it has none
// (whatever cu holds, the result is below B and column m lies in [cu[b], cu[b + 1]))
NNHIP_HD int packed_sequence(const int32_t* cu, int B, int m)
{
    int lo = 0, hi = B;
    while (lo < hi)
    {
        const int mid = lo + ((hi - lo) >> 1);
        if (cu[mid + 1] > m) hi = mid;
        else lo = mid + 1;
    }
    return lo < B && cu[lo] >= 0 && cu[lo] <= m && cu[lo + 1] > m ? lo : -1;
}

// Position of column m in its sequence b, or -1 if it is not in [0, limit)
NNHIP_HD int packed_position(const int32_t* cu, const int32_t* pos0, int b, int m, int limit)
{
    const int p0 = pos0 ? pos0[b] : 0, t = m - cu[b];
    return p0 >= 0 && p0 < limit && t < limit - p0 ? p0 + t : -1;
}

}  // namespace nnhip
