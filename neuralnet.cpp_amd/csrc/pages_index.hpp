// pages_index.hpp — where a position of a paged sequence lies. Plain arithmetic that the kernels share
// with a CPU test (tests/cpp/pages_index_check.cpp), so that its bounds are checked without a GPU.
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

// Table entries that positions [t0, last] of a sequence need, from entry t0 >> shift on
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
