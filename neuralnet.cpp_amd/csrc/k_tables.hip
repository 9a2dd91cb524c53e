// k_tables.hip — the page tables of a paged KV cache kept on the GPU: pages for new tokens from a free list, the tokens'
// offsets, positions and slots, and pages given back. A server's step then needs no length on the host, and a captured
// step goes on by itself.
//
// The free list is a stack: free_pages[0 .. free_count - 1], taken from its end. Sequences are served in their order:
// sequence b gets its pages if those of all sequences up to it (that could be served at all) are there, and needs none or
// gets none otherwise. Sums over the sequences are 64-bit: lengths up to 2^30 of 65535 sequences pass 2^31.
//
// One work-group scans the sequences, a run of them to each thread. Latency is what there is to these calls: the same
// work-group also writes the table's entries and the tokens, each found by bisection of the offsets in LDS, while they are
// few; beyond that a second launch does, a wave to a sequence and a thread to a token. Pages for new tokens and their way
// back, in one launch and in two: 256 sequences of a token 14.8 and 20.8 us, 1000 of 1 .. 30 15.5 and 17.8, of 1 .. 60
// 19.3 and 17.8, of 900 83 and 22; 16 of 1 .. 2000 15.0 and 18.0, of 1 .. 8000 18.4 and 18.0.
#include "pages_split.hpp"

namespace nnhip
{
namespace
{

constexpr int kTbThreads = 1024, kTbWaves = kTbThreads / kWave;
constexpr int kOneB = 256;    // sequences of a call in one launch, whose pages may be any number
constexpr int kOneT = 1024, kOneM = 16384;  // and where no more than so many tokens ask for pages

__device__ __forceinline__ int64_t shfl_up64(int64_t x, int off)
{
    const int lo = __shfl_up((int)(uint32_t)x, off, kWave), hi = __shfl_up((int)(x >> 32), off, kWave);
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

// The sums of x[k] over the threads before this one; total: over all
template <int N>
__device__ __forceinline__ void scan_before(int64_t (&x)[N], int64_t (*wave_s)[N], int64_t (&total)[N])
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int64_t incl[N];
#pragma unroll
    for (int k = 0; k < N; ++k) incl[k] = x[k];
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k)
        {
            const int64_t y = shfl_up64(incl[k], off);
            if (lane >= off) incl[k] += y;
        }
    if (lane == kWave - 1)
#pragma unroll
        for (int k = 0; k < N; ++k) wave_s[w][k] = incl[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k)
    {
        int64_t before = 0;
        total[k] = 0;
#pragma unroll
        for (int i = 0; i < kTbWaves; ++i)
        {
            const int64_t y = wave_s[i][k];
            if (i < w) before += y;
            total[k] += y;
        }
        x[k] = before + incl[k] - x[k];
    }
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
template <typename T>
__device__ __forceinline__ int bisect(const T* x, int n, T at)
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

// kOne: every sequence in a thread of its own
template <bool kOne>
__global__ __launch_bounds__(kTbThreads) void k_pages_assign(AssignArgs a)
{
    __shared__ int64_t need_s[kTbWaves][1], given_s[kTbWaves][2];
    __shared__ int cu_s[kOne ? kOneT : 1], page_s[kOne ? kOneT : 1], len_s[kOne ? kOneT : 1];
    const int b0 = min((int)threadIdx.x * a.run, a.B), b1 = min(b0 + a.run, a.B);
    const int64_t count = min(max(*a.free_count, 0), a.num_pages);
    int first_len = 0, first_add = 0, first_n = 0;
    if (b0 < b1) first_len = a.lens[b0], first_add = wanted(a, first_len, a.add[b0], first_n);
    // what sequence b asks for: the first one's is in registers
    auto asks = [&](int b, int& len, int& n) {
        len = first_len, n = first_n;
        if (kOne || b == b0) return first_add;
        len = a.lens[b];
        return wanted(a, len, a.add[b], n);
    };
    // on its way during the sums: the id that this thread will put into the table
    int64_t at_id = count - 1 - (int)threadIdx.x;
    const int id = kOne && at_id >= 0 ? a.free_pages[at_id] : 0;
    int64_t need[1] = {0}, given[2] = {0, 0}, asked[1], all[2];
    for (int b = b0; b < b1; ++b)
    {
        int len, n;
        asks(b, len, n);
        need[0] += n;
    }
    scan_before(need, need_s, asked);
    int64_t so_far = need[0];
    for (int b = b0; b < b1; ++b)
    {
        int len, n;
        const int add = asks(b, len, n);
        so_far += n;
        if (n == 0 || so_far <= count) given[0] += n, given[1] += add;
    }
    scan_before(given, given_s, all);
    int64_t pages = given[0], tokens = given[1];
    so_far = need[0];
    if (threadIdx.x == 0)
    {
        a.cu[0] = 0;
        if (a.B > 0) *a.free_count = (int)(count - all[0]);
    }
    for (int b = b0; b < b1; ++b)
    {
        int len, n;
        const int add = asks(b, len, n);
        so_far += n;
        const bool served = add > 0 && (n == 0 || so_far <= count);
        if (kOne)
        {
            cu_s[b] = (int)tokens;
            page_s[b] = (int)pages;
            len_s[b] = len;
        }
        else a.starts[b] = (int)(count - 1 - pages);
        if (served)
        {
            pages += n;
            tokens += add;
            a.lens[b] = len + add;
        }
        a.pos0[b] = served ? len : -1;
        a.cu[b + 1] = (int)tokens;
    }
    if constexpr (kOne)
    {
        __syncthreads();
        for (int i = threadIdx.x; i < (int)all[0]; i += kTbThreads)
        {
            const int b = bisect(page_s, a.B, i);
            a.table[(size_t)b * a.table_stride + pages_of(len_s[b], a.shift) + (i - page_s[b])] =
                i == (int)threadIdx.x ? id : a.free_pages[count - 1 - i];
        }
        if (a.pos || a.slots)
        {
            __threadfence_block();
            __syncthreads();  // the table's entries are there
            for (int m = threadIdx.x; m < a.M; m += kTbThreads)
            {
                const bool there = m < (int)all[1];
                const int b = there ? bisect(cu_s, a.B, m) : 0;
                put_token(a.table, a.table_stride, a.shift, a.num_pages, m, b, there ? len_s[b] + (m - cu_s[b]) : -1, a.pos, a.slots);
            }
        }
    }
}

// The table's entries, a wave to a sequence in the first `blocks` work-groups, and in the others the tokens, whose new
// pages come from the free list (the entries may not be there yet)
__global__ __launch_bounds__(256) void k_pages_entries(AssignArgs a, int blocks)
{
    const int lane = threadIdx.x & 63;
    if ((int)blockIdx.x < blocks)
    {
        const int b = (int)(blockIdx.x * 4 + (threadIdx.x >> 6));
        if (b >= a.B) return;
        const int len = a.pos0[b], start = a.starts[b];
        if (len < 0) return;
        const int held = pages_of(len, a.shift), n = pages_of(len + (a.cu[b + 1] - a.cu[b]), a.shift) - held;
        for (int i = lane; i < n; i += kWave) a.table[(size_t)b * a.table_stride + held + i] = a.free_pages[start - i];
        return;
    }
    const int m0 = (int)((blockIdx.x - blocks) * 256 + (threadIdx.x & ~63u)), m = m0 + lane;
    if (m0 >= a.M) return;
    const int b = wave_sequence(a.cu, a.B, a.M, m0, lane);
    if (m >= a.M) return;
    int p = -1, slot = -1;
    if (b >= 0)
    {
        const int len = a.pos0[b], held = pages_of(len, a.shift);
        p = len + (m - a.cu[b]);
        const int j = p >> a.shift;
        const int id = j >= held ? a.free_pages[a.starts[b] - (j - held)] : a.table[(size_t)b * a.table_stride + j];
        if (page_ok(id, a.num_pages)) slot = (id << a.shift) + (p & ((1 << a.shift) - 1));
    }
    if (a.pos) a.pos[m] = p;
    if (a.slots) a.slots[m] = slot;
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
    __shared__ int64_t pages_s[kTbWaves][1];
    __shared__ int64_t page_s[kOne ? kOneB : 1];  // (of pages in more than one row the sums may be anything: past 2^31, too)
    __shared__ int first_s[kOne ? kOneB : 1];
    const int b0 = min((int)threadIdx.x * a.run, a.B), b1 = min(b0 + a.run, a.B);
    const int64_t count = min(max(*a.free_count, 0), a.num_pages);
    int first_first = 0, first_kept = 0, first_n = 0;
    if (b0 < b1) first_n = behind(a, b0, first_first, first_kept);
    // sequence b's: the first one's is in registers
    auto gives = [&](int b, int& first, int& kept) {
        first = first_first, kept = first_kept;
        return kOne || b == b0 ? first_n : behind(a, b, first, kept);
    };
    int64_t before[1] = {0}, all[1];
    for (int b = b0; b < b1; ++b)
    {
        int first, kept;
        before[0] += gives(b, first, kept);
    }
    scan_before(before, pages_s, all);
    int64_t pages = before[0];
    const int64_t total = all[0];
    const int64_t top = min(count + total, (int64_t)a.num_pages);  // (more than the list holds: pages given back twice)
    if (threadIdx.x == 0) *a.free_count = (int)top;
    for (int b = b0; b < b1; ++b)
    {
        int first, kept;
        const int n = gives(b, first, kept);
        if (kOne)
        {
            page_s[b] = pages;
            first_s[b] = first;
        }
        else a.moves[b] = make_int4(first, n, (int)min(count + total - 1 - pages, (int64_t)0x7FFFFFFF), 0);
        pages += n;
        if (kept >= 0) a.lens[b] = kept;
    }
    if constexpr (kOne)
    {
        __syncthreads();
        for (int64_t i = count + total - top + threadIdx.x; i < total; i += kTbThreads)
        {
            const int b = bisect(page_s, a.B, i);
            a.free_pages[count + total - 1 - i] = a.table[(size_t)b * a.table_stride + first_s[b] + (int)(i - page_s[b])];
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

// Pages for the new tokens in one launch? (tokens: M bounds the pages)
static bool assign_one(size_t B, size_t M, bool tokens) { return tokens ? B <= (size_t)kOneT && M <= (size_t)kOneM : B <= (size_t)kOneB; }

size_t pages_assign_workspace_bytes(size_t B, size_t M, bool tokens) { return assign_one(B, M, tokens) ? 0 : B * sizeof(int32_t); }

size_t pages_release_workspace_bytes(size_t B) { return B <= (size_t)kOneB ? 0 : B * sizeof(int4); }

hipError_t launch_pages_assign(hipStream_t st, int32_t* table, size_t table_stride, size_t page_size, size_t num_pages, size_t B,
                               int32_t* free_pages, int32_t* free_count, int32_t* lens, const int32_t* add, int32_t* cu,
                               int32_t* pos0, size_t M, int32_t* pos, int32_t* slots, void* ws)
{
    const AssignArgs a{table, free_pages, free_count, lens, add, cu, pos0, pos, slots, static_cast<int32_t*>(ws),
                       (int)table_stride, log2_of(page_size), (int)num_pages, (int)B, (int)M, (int)ceil_div(B, (size_t)kTbThreads)};
    const bool tokens = M > 0 && (pos || slots);
    if (assign_one(B, M, tokens))
    {
        k_pages_assign<true><<<1, kTbThreads, 0, st>>>(a);
        return hipGetLastError();
    }
    k_pages_assign<false><<<1, kTbThreads, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const size_t entries = ceil_div(B, (size_t)4), places = tokens ? ceil_div(M, (size_t)256) : 0;
    k_pages_entries<<<(unsigned)(entries + places), 256, 0, st>>>(a, (int)entries);
    return hipGetLastError();
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
