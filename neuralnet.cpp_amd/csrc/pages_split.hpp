// pages_split.hpp — what the kernels of the paged caches share (k_pages.hip, k_pages_i8.hip): the decode attention's
// arguments, its cut into chunks of positions and the join of their records, and the sequences of packed columns.
#pragma once

#include "common.hpp"
#include "pages_index.hpp"

namespace nnhip
{
namespace
{

constexpr int kPgThreads = 256;  // 4 waves
constexpr int kPgWaves = kPgThreads / kWave;
constexpr int kPgMaxR = 8;       // query heads of a work-group
constexpr int kPgRec = 16;       // tail of a record: maximum[8], sum[8]
constexpr int kPgMinChunk = 128;  // positions of a work-group at least (a multiple of 64)
constexpr int kPgEvenB = 1024;   // sequences up to which the chunks are sized by the lengths

struct PagesArgs
{
    const float* q;
    const float* k;
    const float* v;
    const int32_t* pos;
    const float* cosT;
    const float* sinT;
    void* kc;
    void* vc;
    const int32_t* table;
    const float* slopes;
    float* part;
    int2* places;  // even > 0: each sequence's first record and its chunks' size, for the join
    float* out;
    int B, H, Hkv, R, groups, RG;  // R = H / Hkv heads of a KV head, in `groups` groups of at most RG
    int shift;                     // log2(page_size)
    int table_stride, num_pages, len_bound;
    int chunk, nchunk;             // even == 0: chunks of every sequence
    int even;                      // > 0: chunks sized by the lengths (see find_item), about `even` of them
    float scale2;  // scale * log2(e)
    float capi;    // scale / softcap
    float cap2;    // softcap * log2(e), 0 without a cap
    int tokens;
};

// Two rounded products and a rounded sum per output, as the contiguous cache's append rotates.
__device__ __forceinline__ void pg_rope(float x0, float x1, float cs, float sn, float& y0, float& y1)
{
    y0 = __fadd_rn(__fmul_rn(x0, cs), __fmul_rn(-x1, sn));
    y1 = __fadd_rn(__fmul_rn(x1, cs), __fmul_rn(x0, sn));
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140, kDppRor4 = 0x124,
              kDppRor8 = 0x128, kDppBcast = 0x150;  // kDppBcast + n: lane n of each row of 16

// A barrier for LDS data only: loads of the pools stay in flight across it
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // vmcnt and expcnt at their maxima, lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Where a work-group works: chunk c of `chunk` positions of sequence b, whose new token has position p;
// `first` = the sequence's first record. b < 0: nothing to do.
struct PagesItem
{
    int b, c, chunk, first, p;
};

__device__ __forceinline__ int pages_len(const PagesArgs& a, int p) { return p < 0 || p >= a.len_bound ? 0 : p + 1; }

// Item `item` of a call. With lengths spread from 1 to 16 K, chunks of one size for len_bound leave a few
// long work-groups and thousands of empty ones (37 sequences of 1 .. 16384 over 2 KV heads: 63 us against 26
// when this was measured, 19.4 now), so every wave sizes the chunks by the lengths themselves: with D = a.even
// the smallest multiple of 64 that is at least sum(len) / D, which makes at most D + B chunks. Every
// work-group of the call finds the same ones; the first of a sequence leaves its place for the join.
__device__ __forceinline__ PagesItem find_item(const PagesArgs& a, int item)
{
    const int lane = threadIdx.x & 63;
    uint32_t total = 0;  // below 2^31
    for (int b = lane; b < a.B; b += kWave) total += (uint32_t)pages_len(a, a.pos[b]);
    for (int off = 1; off < min(a.B, kWave); off <<= 1) total += (uint32_t)__shfl_xor((int)total, off, kWave);
    total = (uint32_t)__builtin_amdgcn_readfirstlane((int)total);
    const int chunk = max(kPgMinChunk, (int)(64 * (((total + 63) / 64 + (uint32_t)a.even - 1) / (uint32_t)a.even)));
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave)
    {
        const int b = b0 + lane, p = b < a.B ? a.pos[b] : -1;
        const int n = b < a.B ? max(1, (int)(((uint32_t)pages_len(a, p) + (uint32_t)chunk - 1) / (uint32_t)chunk)) : 0;
        const int live = min(a.B - b0, kWave);
        int incl = n;
        for (int off = 1; off < live; off <<= 1)
        {
            const int x = __shfl_up(incl, off, kWave);
            if (lane >= off) incl += x;
        }
        const int sum = __builtin_amdgcn_readlane(incl, live - 1);
        const unsigned long long here = __builtin_amdgcn_ballot_w64(b < a.B && before + incl > item);
        if (here != 0)
        {
            const int l = __builtin_ctzll(here);
            const int first = before + __builtin_amdgcn_readlane(incl - n, l);
            return {b0 + l, item - first, chunk, first, __builtin_amdgcn_readlane(p, l)};
        }
        before += sum;
    }
    return {-1, 0, chunk, 0, -1};
}

// out of one (sequence, head) from its chunks' records: sum_c 2^(m_c - m) acc_c / sum_c 2^(m_c - m) l_c, in the order
// of the records: the same in every call of the same sizes and positions. A launch of its own: a join by the
// last work-group to arrive would need the records written back from one XCD's L2 before another's reads.
template <int DK>
__global__ __launch_bounds__(kPgThreads) void k_pages_join(PagesArgs a)
{
    constexpr int L = DK / 4, G = kPgThreads / L;  // lanes of a record's row, records side by side
    __shared__ float4 acc_s[G][L];
    __shared__ float m_s[G], l_s[G];
    const int h = blockIdx.x, b = blockIdx.y;
    const int2 place = a.even ? a.places[b] : make_int2(b * a.nchunk, a.chunk);
    const PagesItem it{b, 0, place.y, place.x, a.pos[b]};
    const int p = it.p;
    if (p < 0 || p >= a.len_bound) return;  // the chunks' kernel wrote those
    const int g = h / a.R, r0 = h - g * a.R, hg = r0 / a.RG, r = r0 - hg * a.RG;
    const int nch = p / it.chunk + 1, HG = a.Hkv * a.groups;
    const size_t step = (size_t)HG * (a.RG * DK + kPgRec);
    const float* rec = a.part + ((size_t)it.first * HG + g * a.groups + hg) * (size_t)(a.RG * DK + kPgRec);
    const int tid = threadIdx.x, i = tid % L, gr = tid / L;
    float m = -__builtin_inff(), l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int U = 4;  // records on their way together
    for (int c0 = gr; c0 < nch; c0 += U * G)
    {
        float mc[U], lc[U];
        float4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int c = c0 + u * G;
            const float* at = rec + (size_t)(c < nch ? c : c0) * step;
            mc[u] = at[a.RG * DK + r];
            lc[u] = at[a.RG * DK + 8 + r];
            x[u] = reinterpret_cast<const float4*>(at + r * DK)[i];
            if (c >= nch) mc[u] = -__builtin_inff(), lc[u] = 0.0f, x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        float to = m;
#pragma unroll
        for (int u = 0; u < U; ++u) to = fmaxf(to, mc[u]);
        const float f = m == to ? 1.0f : __builtin_amdgcn_exp2f(m - to);
        l *= f, acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const float e = mc[u] == to ? 1.0f : __builtin_amdgcn_exp2f(mc[u] - to);
            l = __builtin_fmaf(e, lc[u], l);
            acc.x = __builtin_fmaf(e, x[u].x, acc.x), acc.y = __builtin_fmaf(e, x[u].y, acc.y);
            acc.z = __builtin_fmaf(e, x[u].z, acc.z), acc.w = __builtin_fmaf(e, x[u].w, acc.w);
        }
        m = to;
    }
    acc_s[gr][i] = acc;
    if (i == 0) m_s[gr] = m, l_s[gr] = l;
    __syncthreads();
    if (gr != 0) return;
    float top = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < G; ++k) top = fmaxf(top, m_s[k]);
    float sum = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < G; ++k)
    {
        const float e = m_s[k] == top ? 1.0f : __builtin_amdgcn_exp2f(m_s[k] - top);
        const float4 x = acc_s[k][i];
        sum = __builtin_fmaf(e, l_s[k], sum);
        y.x = __builtin_fmaf(e, x.x, y.x), y.y = __builtin_fmaf(e, x.y, y.y);
        y.z = __builtin_fmaf(e, x.z, y.z), y.w = __builtin_fmaf(e, x.w, y.w);
    }
    const size_t st = a.tokens ? 1 : (size_t)a.B;
    float* o = a.out + (a.tokens ? ((size_t)b * a.H + h) * DK + 4 * i : ((size_t)h * DK + 4 * i) * a.B + b);
    const float inv = sum == 0.0f ? 1.0f : sum;
    o[0] = y.x / inv, o[st] = y.y / inv, o[2 * st] = y.z / inv, o[3 * st] = y.w / inv;
}

// Chunks of a call at most, over all sequences
inline size_t pages_items(size_t B, size_t len_bound, size_t chunk, size_t even)
{
    const size_t all = B * ceil_div(len_bound, chunk);
    return even && even + B < all ? even + B : all;
}

constexpr int kPfTok = 64;  // tokens of a work-group (16 x 1111 .. 2048 tokens, 5 heads of 128, f16: 46.5 us, 32: 50.4)

// The sequence of column m0 + lane, or -1:
// packed_sequence's in two round trips for up to 64 sequences, for the wave at once.
__device__ __forceinline__ int wave_sequence(const int32_t* cu, int B, int M, int m0, int lane)
{
    // the first b with cu[b + 1] > m0, by 64ths
    int lo = 0, n = B;
    while (n > 0)
    {
        const int step = (n + kWave - 1) / kWave;
        const int at = lo + min((lane + 1) * step, n) - 1;
        const unsigned long long above = __builtin_amdgcn_ballot_w64(cu[at + 1] > m0);
        if (above == 0)
        {
            lo += n;
            break;
        }
        const int k = __builtin_ctzll(above) * step;
        lo += k;
        if (step == 1) break;
        n = min(step, n - k);
    }
    if (lo >= B) return -1;
    const int m = m0 + (lane & (kPfTok - 1));
    // the ends of the sequences from there on that lie in the block: of every lane, those behind column M too
    const int end = lo + 1 + lane <= B ? cu[lo + 1 + lane] : 0x7FFFFFFF;
    const int ends = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= m0 + kPfTok - 1));
    int b = lo;
    for (int i = 0; i < ends; ++i) b += __builtin_amdgcn_readlane(end, i) <= m ? 1 : 0;
    if (m >= M) return -1;
    if (ends == kWave) return packed_sequence(cu, B, m);  // (64 sequences that end here, and more maybe)
    return b < B && cu[b] >= 0 && cu[b] <= m && cu[b + 1] > m ? b : -1;
}

// Block of columns of work-group `at` of `blocks` (issued to the 8 XCDs in turn): an XCD takes a run of them, so that lines
// of the L2 that two neighbouring blocks share are in one
__device__ __forceinline__ int xcd_run(int at, int blocks)
{
    const int each = blocks >> 3, over = blocks & 7, xcd = at & 7;
    return xcd * each + min(xcd, over) + (at >> 3);
}

inline int log2_of(size_t v)
{
    int n = 0;
    while ((size_t(1) << n) < v) ++n;
    return n;
}

// Query heads of a KV head in groups of at most 8 (dk = 256: 4, whose registers are as many), as even as they go
inline size_t pages_groups(size_t R, size_t dk) { return ceil_div(R, (size_t)(dk == 256 ? 4 : kPgMaxR)); }

// How a call is cut: chunks of `chunk` positions (nchunk to a sequence), or with even > 0 about `even` of a
// size that the kernels find
struct PagesCut
{
    size_t chunk, nchunk, even;
};

inline PagesCut pages_cut(size_t B, size_t Hkv, size_t R, size_t dk, size_t len_bound, size_t num_cus)
{
    const size_t HG = Hkv * pages_groups(R, dk);
    // chunks that fill the GPU: two work-groups to a CU, and not one more, which a CU would take as a third (4
    // sequences of 128 K over 8 KV heads: 512 work-groups 234 us, 528 269, 768 241, 256 302; 1 x 32768 over 5
    // heads 23.4, 25.2 with 768)
    const size_t want = 2 * num_cus / HG;
    if (len_bound <= kPgMinChunk) return {kPgMinChunk, 1, 0};
    if (B <= kPgEvenB && B * len_bound < (size_t(1) << 31)) return {kPgMinChunk, 0, want > 2 * B ? want - B : B};
    size_t chunk = kPgMinChunk;
    while (B * ceil_div(len_bound, chunk) > 2 * want && chunk < len_bound) chunk *= 2;
    return {chunk, ceil_div(len_bound, chunk), 0};
}

// Floats of a call's records
inline size_t pages_records(size_t B, size_t Hkv, size_t groups, size_t RG, size_t dk, size_t len_bound, const PagesCut& cut)
{
    return pages_items(B, len_bound, cut.chunk, cut.even) * Hkv * groups * (RG * dk + kPgRec);
}

}  // namespace
}  // namespace nnhip
