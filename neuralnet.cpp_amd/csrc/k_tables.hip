// k_tables.hip — the page tables of a paged KV cache kept on the GPU: pages for new tokens from a free list, the tokens'
// offsets, positions and slots, and pages given back. A server's step then needs no length on the host, and a captured
// step goes on by itself.
//
// The free list is a stack: free_pages[0 .. free_count - 1], taken from its end. Sequences are served in their order:
// sequence b gets its pages if those of all sequences up to it (that could be served at all) are there, and needs none or
// gets none otherwise. Sums over the sequences are 64-bit: lengths up to 2^30 of 65535 sequences pass 2^31.
//
// One work-group scans the sequences, a run of them to each thread. Latency is what there is to these calls: up to kOneB sequences and
// kOneM tokens the same work-group also writes the table's entries and the tokens, each found by bisection of
// the offsets in LDS; beyond that further launches do, a wave to a sequence and a thread to a token.
#include "pages_split.hpp"

namespace nnhip
{
namespace
{

constexpr int kTbThreads = 1024, kTbWaves = kTbThreads / kWave;
constexpr int kOneB = 256;    // sequences of a call in one launch
constexpr int kOneM = 4096;   // its tokens at most

__device__ __forceinline__ int64_t shfl_up64(int64_t x, int off)
{
    const int lo = __shfl_up((int)(uint32_t)x, off, kWave), hi = __shfl_up((int)(x >> 32), off, kWave);
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

// The sum of x over the threads before this one; total: over all
__device__ __forceinline__ int64_t scan_before(int64_t x, int64_t* wave_s, int64_t& total)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int64_t incl = x;
    for (int off = 1; off < kWave; off <<= 1)
    {
        const int64_t y = shfl_up64(incl, off);
        if (lane >= off) incl += y;
    }
    __syncthreads();  // (wave_s may still be read by an earlier scan)
    if (lane == kWave - 1) wave_s[w] = incl;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kTbWaves; ++i)
    {
        if (i < w) before += wave_s[i];
        total += wave_s[i];
    }
    return before + incl - x;
}

__device__ __forceinline__ int pages_of(int len, int shift) { return (int)(((int64_t)len + (1 << shift) - 1) >> shift); }

struct AssignArgs
{
    int32_t* table;
    int32_t* free_pages;
    int32_t* free_count;
    int32_t* lens;
    const int32_t* add;
    int32_t* cu;
    int32_t* pos0;
    int32_t* pos;
    int32_t* slots;
    int32_t* starts;  // two launches: a sequence's first index of the free list
    int table_stride, shift, num_pages, B, M, run;  // run: sequences of a thread
};

// What a sequence asks for: new tokens, 0 if it cannot be served, and pages
__device__ __forceinline__ int wanted(const AssignArgs& a, int len, int add, int& need)
{
    need = 0;
    const int64_t limit = (int64_t)a.table_stride << a.shift;
    if (len < 0 || add <= 0 || (int64_t)len + add > limit) return 0;
    need = pages_of(len + add, a.shift) - pages_of(len, a.shift);
    return add;
}

// Position and slot of token m, of sequence b, whose columns begin at cu0 and positions at p0
__device__ __forceinline__ void put_token(const int32_t* table, int table_stride, int shift, int num_pages, int m, int b, int p,
                                          int32_t* pos, int32_t* slots)
{
    if (pos) pos[m] = p;
    if (!slots) return;
    int slot = -1;
    if (p >= 0)
    {
        const int id = table[(size_t)b * table_stride + (p >> shift)];
        if (page_ok(id, num_pages)) slot = (id << shift) + (p & ((1 << shift) - 1));
    }
    slots[m] = slot;
}

// The last i of n with x[i] <= at (x not falling, x[0] <= at)
__device__ __forceinline__ int bisect(const int* x, int n, int at)
{
    int lo = 0;
    while (n > 1)
    {
        const int half = n >> 1;
        if (x[lo + half] <= at) lo += half;
        n -= half;
    }
    return lo;
}

template <bool kOne>
__global__ __launch_bounds__(kTbThreads) void k_pages_assign(AssignArgs a)
{
    __shared__ int64_t wave_s[kTbWaves];
    __shared__ int cu_s[kOne ? kOneB : 1], page_s[kOne ? kOneB : 1], len_s[kOne ? kOneB : 1];
    const int b0 = min((int)threadIdx.x * a.run, a.B), b1 = min(b0 + a.run, a.B);
    const int64_t count = min(max(*a.free_count, 0), a.num_pages);
    int64_t need = 0, pages = 0, tokens = 0, total, all_pages, all_tokens;
    for (int b = b0; b < b1; ++b)
    {
        int n;
        wanted(a, a.lens[b], a.add[b], n);
        need += n;
    }
    const int64_t asked = scan_before(need, wave_s, total);
    need = asked;
    for (int b = b0; b < b1; ++b)
    {
        int n;
        const int add = wanted(a, a.lens[b], a.add[b], n);
        need += n;
        if (n == 0 || need <= count) pages += n, tokens += add;
    }
    pages = scan_before(pages, wave_s, all_pages);
    tokens = scan_before(tokens, wave_s, all_tokens);
    need = asked;
    if (threadIdx.x == 0)
    {
        a.cu[0] = 0;
        *a.free_count = (int)(count - all_pages);
    }
    for (int b = b0; b < b1; ++b)
    {
        int n;
        const int len = a.lens[b], add = wanted(a, len, a.add[b], n);
        need += n;
        const bool given = add > 0 && (n == 0 || need <= count);
        if (kOne)
        {
            cu_s[b] = (int)tokens;
            page_s[b] = (int)pages;
            len_s[b] = len;
        }
        else a.starts[b] = (int)(count - 1 - pages);
        if (given)
        {
            pages += n;
            tokens += add;
            a.lens[b] = len + add;
        }
        a.pos0[b] = given ? len : -1;
        a.cu[b + 1] = (int)tokens;
    }
    if constexpr (kOne)
    {
        __syncthreads();
        for (int i = threadIdx.x; i < (int)all_pages; i += kTbThreads)
        {
            const int b = bisect(page_s, a.B, i);
            a.table[(size_t)b * a.table_stride + pages_of(len_s[b], a.shift) + (i - page_s[b])] = a.free_pages[count - 1 - i];
        }
        if (a.pos || a.slots)
        {
            __threadfence_block();
            __syncthreads();  // the table's entries are there
            for (int m = threadIdx.x; m < a.M; m += kTbThreads)
            {
                const bool there = m < (int)all_tokens;
                const int b = there ? bisect(cu_s, a.B, m) : 0;
                put_token(a.table, a.table_stride, a.shift, a.num_pages, m, b, there ? len_s[b] + (m - cu_s[b]) : -1, a.pos, a.slots);
            }
        }
    }
}

// The table's entries, a wave to a sequence
__global__ __launch_bounds__(256) void k_pages_entries(AssignArgs a)
{
    const int b = (int)(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (b >= a.B) return;
    const int len = a.pos0[b], start = a.starts[b];
    if (len < 0) return;
    const int held = pages_of(len, a.shift), n = pages_of(len + (a.cu[b + 1] - a.cu[b]), a.shift) - held;
    for (int i = lane; i < n; i += kWave) a.table[(size_t)b * a.table_stride + held + i] = a.free_pages[start - i];
}

struct SlotArgs
{
    const int32_t* table;
    const int32_t* cu;
    const int32_t* pos0;
    int32_t* pos;
    int32_t* slots;
    int table_stride, shift, num_pages, B, M, limit;
};

__global__ __launch_bounds__(256) void k_pages_slots(SlotArgs a)
{
    const int lane = threadIdx.x & 63, m0 = (int)(blockIdx.x * 256 + (threadIdx.x & ~63u)), m = m0 + lane;
    if (m0 >= a.M) return;
    const int b = wave_sequence(a.cu, a.B, a.M, m0, lane);
    if (m >= a.M) return;
    const int p = b < 0 ? -1 : packed_position(a.cu, a.pos0, b, m, a.limit);
    put_token(a.table, a.table_stride, a.shift, a.num_pages, m, max(b, 0), p, a.pos, a.slots);
}

struct ReleaseArgs
{
    const int32_t* table;
    int32_t* free_pages;
    int32_t* free_count;
    int32_t* lens;
    const int32_t* keep;
    int4* moves;  // two launches: first entry, pages, place of the first in the free list
    int table_stride, shift, num_pages, B, run;
};

// Pages behind the kept length of a sequence: the first entry and how many. kept: the new length
__device__ __forceinline__ int behind(const ReleaseArgs& a, int b, int& first, int& kept)
{
    const int len = a.lens[b];
    kept = min(max(a.keep[b], 0), len);
    first = kept < 0 ? 0 : pages_of(kept, a.shift);
    return len <= 0 ? 0 : min(pages_of(len, a.shift), a.table_stride) - min(first, a.table_stride);
}

// The pages go back in the opposite order of the table's, so that what k_pages_assign took last lies on top again
template <bool kOne>
__global__ __launch_bounds__(kTbThreads) void k_pages_release(ReleaseArgs a)
{
    __shared__ int64_t wave_s[kTbWaves];
    __shared__ int page_s[kOne ? kOneB : 1], first_s[kOne ? kOneB : 1];
    const int b0 = min((int)threadIdx.x * a.run, a.B), b1 = min(b0 + a.run, a.B);
    const int64_t count = min(max(*a.free_count, 0), a.num_pages);
    int64_t pages = 0, total;
    for (int b = b0; b < b1; ++b)
    {
        int first, kept;
        pages += behind(a, b, first, kept);
    }
    pages = scan_before(pages, wave_s, total);
    const int64_t top = min(count + total, (int64_t)a.num_pages);  // (more than the list holds: pages given back twice)
    if (threadIdx.x == 0) *a.free_count = (int)top;
    for (int b = b0; b < b1; ++b)
    {
        int first, kept;
        const int n = behind(a, b, first, kept);
        if (kOne)
        {
            page_s[b] = (int)pages;
            first_s[b] = first;
        }
        else a.moves[b] = make_int4(first, n, (int)(count + total - 1 - pages), 0);
        pages += n;
        if (a.lens[b] >= 0) a.lens[b] = kept;
    }
    if constexpr (kOne)
    {
        __syncthreads();
        for (int64_t i = threadIdx.x; i < total; i += kTbThreads)
        {
            const int b = bisect(page_s, a.B, (int)i);
            const int64_t to = count + total - 1 - i;
            if (to < a.num_pages) a.free_pages[to] = a.table[(size_t)b * a.table_stride + first_s[b] + ((int)i - page_s[b])];
        }
    }
}

__global__ __launch_bounds__(256) void k_pages_return(ReleaseArgs a)
{
    const int b = (int)(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (b >= a.B) return;
    const int4 x = a.moves[b];
    for (int i = lane; i < x.y; i += kWave)
        if (x.z - i >= 0 && x.z - i < a.num_pages) a.free_pages[x.z - i] = a.table[(size_t)b * a.table_stride + x.x + i];
}

}  // namespace

size_t tables_workspace_bytes(size_t B) { return B <= (size_t)kOneB ? 0 : B * sizeof(int4); }

hipError_t launch_pages_assign(hipStream_t st, int32_t* table, size_t table_stride, size_t page_size, size_t num_pages, size_t B,
                               int32_t* free_pages, int32_t* free_count, int32_t* lens, const int32_t* add, int32_t* cu,
                               int32_t* pos0, size_t M, int32_t* pos, int32_t* slots, void* ws)
{
    const AssignArgs a{table, free_pages, free_count, lens, add, cu, pos0, pos, slots, static_cast<int32_t*>(ws),
                       (int)table_stride, log2_of(page_size), (int)num_pages, (int)B, (int)M, (int)ceil_div(B, (size_t)kTbThreads)};
    const bool tokens = M > 0 && (pos || slots), one = B <= (size_t)kOneB;
    AssignArgs first = a;
    const bool together = one && tokens && M <= (size_t)kOneM;
    if (!together) first.pos = first.slots = nullptr;
    if (one) k_pages_assign<true><<<1, kTbThreads, 0, st>>>(first);
    else k_pages_assign<false><<<1, kTbThreads, 0, st>>>(first);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (!one)
    {
        k_pages_entries<<<(unsigned)ceil_div(B, (size_t)4), 256, 0, st>>>(a);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return !tokens || together ? hipSuccess
                               : launch_pages_slots(st, table, table_stride, page_size, num_pages, cu, pos0, B, M, pos, slots);
}

hipError_t launch_pages_slots(hipStream_t st, const int32_t* table, size_t table_stride, size_t page_size, size_t num_pages,
                              const int32_t* cu, const int32_t* pos0, size_t B, size_t M, int32_t* pos, int32_t* slots)
{
    const SlotArgs a{table, cu, pos0, pos, slots, (int)table_stride, log2_of(page_size), (int)num_pages, (int)B, (int)M,
                     (int)(table_stride * page_size)};
    k_pages_slots<<<(unsigned)ceil_div(M, (size_t)256), 256, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_pages_release(hipStream_t st, const int32_t* table, size_t table_stride, size_t page_size, size_t num_pages,
                                size_t B, int32_t* free_pages, int32_t* free_count, int32_t* lens, const int32_t* keep, void* ws)
{
    const ReleaseArgs a{table, free_pages, free_count, lens, keep, static_cast<int4*>(ws), (int)table_stride, log2_of(page_size),
                        (int)num_pages, (int)B, (int)ceil_div(B, (size_t)kTbThreads)};
    if (B <= (size_t)kOneB) k_pages_release<true><<<1, kTbThreads, 0, st>>>(a);
    else
    {
        k_pages_release<false><<<1, kTbThreads, 0, st>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        k_pages_return<<<(unsigned)ceil_div(B, (size_t)4), 256, 0, st>>>(a);
    }
    return hipGetLastError();
}

}  // namespace nnhip
