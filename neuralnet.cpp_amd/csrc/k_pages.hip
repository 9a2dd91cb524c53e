// k_pages.hip — the paged KV cache: keys and values of sequences of unlike lengths in pages of a
// common pool, found through a page table. Here its fill from packed prompts and the attention of
// one new token per sequence; the attention of packed prompts is k_prefill.hip's.
//
// Layouts (device):
//   pools   (num_pages, Hkv, page_size, dk) f32 or f16, keys and values apart: a page holds page_size
//           consecutive positions of one sequence, and one head's rows of a page lie in one run
//   table   (B, table_stride) int32: entry (b, i) = the page of positions [i * page_size, (i + 1) *
//           page_size) of sequence b. Entries past a sequence's length are never read.
//   q, out  (H*dk, n) or token-major (n, H*dk); k, v the same with Hkv heads
//
// No id of the table is followed before it is checked against num_pages: a sequence with a bad one
// among its positions gets NaN outputs, and a bad page is never written.
#include "common.hpp"
#include "pages_index.hpp"

#include <cmath>
#include <type_traits>
#include <utility>

namespace nnhip
{
namespace
{

constexpr int kPgThreads = 256;  // 4 waves
constexpr int kPgWaves = kPgThreads / kWave;
constexpr int kPgU = 4;          // rows of a group of 16 lanes in flight together
constexpr int kPgTile = 16;      // rows of a wave's tile: 4 groups x kPgU
constexpr int kPgMaxR = 8;       // query heads of a work-group
constexpr int kPgRec = 16;       // tail of a record: maximum[8], sum[8]
constexpr int kPgMinChunk = 128;  // positions of a work-group at least (a multiple of 64)
constexpr int kPgEvenB = 1024;   // sequences up to which the chunks are sized by the lengths
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
constexpr float kPgLazy = 8.0f;  // log2 growth of a maximum before its sums are rescaled

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

template <typename F, int... I>
__device__ __forceinline__ void static_for_each(F&& f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}

// f(0), ..., f(N - 1) with constants
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f)
{
    static_for_each(f, std::make_integer_sequence<int, N>{});
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140, kDppRor4 = 0x124,
              kDppRor8 = 0x128, kDppBcast = 0x150;  // kDppBcast + n: lane n of each row of 16

// The sums over 16 lanes of N values per lane, spread over the lanes: a level halves the lanes that
// share a value, and while there are two values or more each lane passes one half of them on and
// keeps the other. Lane 8 b3 + 4 b2 + 2 b1 + b0 ends with the values (16 / N of them, at least one)
// from index N b3 / 2 + N b2 / 4 + ... on. 3 (N - 1) instructions against 4 N for every sum in every lane.
template <int A, int CTRL, int BIT, int N>
__device__ __forceinline__ void fold_level(float (&x)[N], int lane)
{
    if constexpr (A >= 2)
    {
        const bool up = (lane & BIT) != 0;
#pragma unroll
        for (int i = 0; i < A / 2; ++i)
        {
            const float send = up ? x[i] : x[i + A / 2], keep = up ? x[i + A / 2] : x[i];
            x[i] = keep + dpp<CTRL>(send);
        }
    }
    else x[0] += dpp<CTRL>(x[0]);
}

constexpr int half_of(int n) { return n > 1 ? n / 2 : 1; }

template <int N>
__device__ __forceinline__ void fold16(float (&x)[N], int lane)
{
    constexpr int N1 = half_of(N), N2 = half_of(N1), N3 = half_of(N2);
    fold_level<N, kDppMirror, 8>(x, lane);
    fold_level<N1, kDppHalfMirror, 4>(x, lane);
    fold_level<N2, kDppXor2, 2>(x, lane);
    fold_level<N3, kDppXor1, 1>(x, lane);
}

template <int LANE>
__device__ __forceinline__ float bcast16(float x)
{
    return dpp<kDppBcast + LANE>(x);
}

// a's upper half of the lanes (odd rows of 16) against b's lower half (even rows), then their sum
__device__ __forceinline__ float fold32(float a, float b)
{
    const auto z = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    const uint32_t x = z[0], y = z[1];  // (a bit cast of a vector's element takes the first one)
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
__device__ __forceinline__ float fold16_rows(float a, float b)
{
    const auto z = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    const uint32_t x = z[0], y = z[1];
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}

// E elements of a cache row as a lane loads them: loads of W elements, 16 lanes side by side
template <int DK, typename CT>
struct PagesRow
{
    static constexpr int E = DK / 16;
    static constexpr int W = sizeof(CT) == 4 ? 4 : (E < 8 ? E : 8);
    static constexpr int N = E / W;               // loads
    static constexpr int WORDS = W * (int)sizeof(CT) / 4;
    typedef uint32_t Vec __attribute__((ext_vector_type(WORDS)));
    Vec x[N];
    static __device__ __forceinline__ int dim(int e, int j) { return 16 * W * (e / W) + W * j + e % W; }
    __device__ __forceinline__ void load(const CT* row, int j)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(row + 16 * W * i + W * j));
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = Vec(0u);
    }
    __device__ __forceinline__ float get(int e) const
    {
        constexpr int H = sizeof(CT) == 4 ? 1 : 2;  // elements in a word
        const uint32_t word = x[e / W][e % W / H];
        if constexpr (H == 1) return __builtin_bit_cast(float, word);
        else
        {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            return (float)__builtin_bit_cast(h2, word)[e & 1];
        }
    }
};

// Lanes of 16 that hold head h's maximum, and the weight of row u and head h (k_pages_attn)
template <bool kDots, int RT>
constexpr int head_lane(int h)
{
    return kDots ? h : RT >= 4 ? h / (RT / 4) : 2 * h;
}
template <bool kDots, int RT>
constexpr int score_lane(int u, int h)
{
    return kDots ? 8 * (u / 2) + h : 4 * u + head_lane<false, RT>(h);
}

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

// Attention of one new token per sequence. Work-group = (chunk of positions, KV head and group of at most 8
// of its query heads, sequence); a group of 16 lanes takes one row of dk at a time, 4 rows on their way
// together, so a wave's tile is 16 rows; its four waves take the chunk's tiles in turn. A tile lies in one
// page, or in two of 8 rows: its addresses are the wave's.
// No wave waits for another before the chunk's end: each group of 16 lanes keeps running maxima, sums
// and weighted values of its own rows. q stays in registers (each lane the elements of its columns).
//   scores   each lane multiplies its columns, the sums over 16 lanes come out spread over them
//            (fold16): lane 4u + s holds row u's score of head(s) s, so that the cap, the bias and the
//            exponential are computed once per score. 8 heads over f16 pools: 16 keys by (8 queries in two
//            f16 parts) is one 16x16x32 product for 32 dimensions, in place of 220 of 390 VALU
//            instructions a tile of dk 64 (37 sequences of 1 .. 16384 over 2 KV heads of 64: 25.6 -> 20.8 us with the
//            join). 4 heads fill half of it, and the rows in lines of 64 bytes cost more than the
//            instructions (64 x 2000 over 5 heads of 128: 71 -> 77 us), so they stay with the VALU;
//   values   the probability of (row u, head h) is broadcast within the 16 lanes by a DPP move.
// A head's reference maximum moves only when it has grown by 2^8.
// The chunk that holds the new position writes its rotated key and its value to the page (no other
// work-group reads that row) and adds them to its sums as one more row.
// Bound by HBM where the caches are large (4 x 60000 .. 131072 positions, 8 heads of 128, f16: 231 us with the
// join, 6.4 TB/s of the bytes it cannot do without; a large copy reaches 4.9 read and written together);
// by the chain of round trips position -> page -> rows, about 7 us in the kernel and 4 in the join,
// where they are small (16 x 2112, 5 heads of 128, f32: 34.0 us, 5 TB/s; 1 x 100: 7.5 us, one launch). 8 heads to a
// KV head of 64: by both, and the VALU instructions of the values (128 multiply-adds a tile).
template <int DK, int RT, bool kFinal, typename CT>
__global__ __launch_bounds__(kPgThreads) void k_pages_attn(PagesArgs a)
{
    using Row = PagesRow<DK, CT>;
    constexpr int E = Row::E, HALF = DK / 2, NV = RT / 4 > 1 ? RT / 4 : 1;  // scores per lane
    constexpr bool kDots = sizeof(CT) == 2 && RT == 8;   // scores by matrix products
    constexpr int NM = kDots ? 1 : NV;                   // heads per lane
    constexpr int KC = DK / 32;                          // kDots: steps of a score
    constexpr int NS = kPgU * RT, QI = (RT * HALF + kPgThreads - 1) / kPgThreads;  // query pairs per thread
    __shared__ __align__(16) float q_s[RT * DK];
    __shared__ float new_s[2][DK];
    __shared__ float ml_s[2][kPgWaves * 4][RT];
    __shared__ float red_s[kPgWaves][RT * DK];
    __shared__ float tot_s[2][RT];
    __shared__ int bad_s[kPgWaves];

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, grp = lane >> 4;
    const int HG = a.Hkv * a.groups;
    const int gh = blockIdx.x % HG, item = blockIdx.x / HG;
    const int g = gh / a.groups, hg = gh - g * a.groups;
    const PagesItem it = !kFinal && a.even ? find_item(a, item)
                                           : PagesItem{item / a.nchunk, item % a.nchunk, a.chunk, item - item % a.nchunk,
                                                       a.pos[item / a.nchunk]};
    if (it.b < 0) return;
    const int b = it.b, c = it.c, p = it.p;
    const int h0 = g * a.R + hg * a.RG;            // first query head
    const int R = min(a.RG, a.R - hg * a.RG);      // query heads here (<= RT)
    // the query pairs, on their way while the rest finds its place
    const size_t in_step = a.tokens ? 1 : (size_t)a.B;
    float qx[QI][2];
#pragma unroll
    for (int u = 0; u < QI; ++u)
    {
        const int e = tid + u * kPgThreads, r = min(e / HALF, R - 1), i = e % HALF;
        const float* q = a.q + (a.tokens ? ((size_t)b * a.H + h0 + r) * DK : (size_t)(h0 + r) * DK * a.B + b);
        qx[u][0] = q[i * in_step];
        qx[u][1] = q[(i + HALF) * in_step];
    }
    const size_t out_step = a.tokens ? 1 : (size_t)a.B;
    float* const out = a.out + (a.tokens ? ((size_t)b * a.H + h0) * DK : (size_t)h0 * DK * a.B + b);
    if (p < 0 || p >= a.len_bound)
    {
        // no token: zeros; a position past the bound: NaN
        if (c == 0)
            for (int e = tid; e < R * DK; e += kPgThreads) out[e * out_step] = p < 0 ? 0.0f : __builtin_nanf("");
        return;
    }
    if (!kFinal && a.even && c == 0 && gh == 0 && tid == 0) a.places[b] = make_int2(it.first, it.chunk);
    const int t0 = c * it.chunk;
    if (t0 > p) return;
    const int n = min(it.chunk, p - t0);           // cached rows here
    const bool has_new = p - t0 < it.chunk;

    // ---- the wave's first tile: its page ids
    const int32_t* const table = a.table + (size_t)b * a.table_stride;
    bool bad = false;
    int ids[2];
    auto load_ids = [&](int base) {
#pragma unroll
        for (int i = 0; i < 2; ++i) ids[i] = table[tile_lookup(t0, base + 8 * i, n) >> a.shift];
    };
    load_ids(w * kPgTile);
    const int new_id = has_new ? table[p >> a.shift] : 0;
    const int slot_mask = (1 << a.shift) - 1;
    const CT* const kc = static_cast<const CT*>(a.kc);
    const CT* const vc = static_cast<const CT*>(a.vc);
    Row kr[kDots ? 1 : kPgU], vr[kPgU];
    v8h km[kDots ? KC : 1];
    auto load = [&](int base) {
        size_t at[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            const int id = __builtin_amdgcn_readfirstlane(ids[i]);
            const bool in = page_ok(id, a.num_pages);
            bad |= !in;
            // rows 8 i .. 8 i + 7 of the tile; those behind the chunk's last row are in the same page as its
            // last 8 rows, or read those (their score is -inf)
            at[i] = page_row(in ? id : 0, g, tile_rows(t0, base + 8 * i, n) & slot_mask, a.Hkv, a.shift) * DK;
        }
        load_ids(base + kPgWaves * kPgTile);
        if constexpr (kDots)
        {
            const CT* k = kc + (j & 8 ? at[1] : at[0]) + (j & 7) * DK + 8 * grp;
            const CT* v = vc + (grp & 2 ? at[1] : at[0]) + 4 * (grp & 1) * DK;
#pragma unroll
            for (int i = 0; i < KC; ++i) km[i] = __builtin_nontemporal_load(reinterpret_cast<const v8h*>(k + 32 * i));
#pragma unroll
            for (int u = 0; u < kPgU; ++u) vr[u].load(v + u * DK, j);
        }
        else
        {
#pragma unroll
            for (int u = 0; u < kPgU; ++u) kr[u].load(kc + at[u / 2] + (4 * (u & 1) + grp) * DK, j);
#pragma unroll
            for (int u = 0; u < kPgU; ++u) vr[u].load(vc + at[u / 2] + (4 * (u & 1) + grp) * DK, j);
        }
    };

    // ---- rotated queries, the new key and value
#pragma unroll
    for (int u = 0; u < QI; ++u)
    {
        const int e = tid + u * kPgThreads, r = e / HALF, i = e % HALF;
        float y0 = qx[u][0], y1 = qx[u][1];
        if (a.cosT) pg_rope(y0, y1, a.cosT[(size_t)p * HALF + i], a.sinT[(size_t)p * HALF + i], y0, y1);
        if (e < RT * HALF)
        {
            // (heads past R stay 0)
            q_s[r * DK + i] = r < R ? y0 : 0.0f;
            q_s[r * DK + i + HALF] = r < R ? y1 : 0.0f;
        }
    }
    if (has_new && tid < HALF)
    {
        const size_t at = a.tokens ? ((size_t)b * a.Hkv + g) * DK : (size_t)g * DK * a.B + b;
        const float* k = a.k + at;
        const float* v = a.v + at;
        float y0 = k[tid * in_step], y1 = k[(tid + HALF) * in_step];
        if (a.cosT) pg_rope(y0, y1, a.cosT[(size_t)p * HALF + tid], a.sinT[(size_t)p * HALF + tid], y0, y1);
        // as the cache holds them (f16: rounded to nearest)
        new_s[0][tid] = (float)(CT)y0;
        new_s[0][tid + HALF] = (float)(CT)y1;
        new_s[1][tid] = (float)(CT)v[tid * in_step];
        new_s[1][tid + HALF] = (float)(CT)v[(tid + HALF) * in_step];
    }
    if (w * kPgTile < n) load(w * kPgTile);  // the first tile, on its way during the rest
    lds_barrier();
    if (has_new)
    {
        const bool in = page_ok(new_id, a.num_pages);
        bad |= !in;
        if (hg == 0 && in)
        {
            const size_t at = page_row(new_id, g, p & slot_mask, a.Hkv, a.shift) * DK;
            for (int i = tid; i < 2 * DK; i += kPgThreads)
                const_cast<CT*>(i < DK ? kc : vc)[at + (size_t)(i & (DK - 1))] = (CT)new_s[i / DK][i & (DK - 1)];
        }
    }

    // This lane's scores: row (lane / 4) % 4 of its 16 lanes' four and heads hs .. hs + NV - 1; kDots: two rows from
    // 2 (lane / 8 % 2) on, and head hs = lane % 8.
    const int hs = kDots ? j & 7 : RT >= 4 ? (j & 3) * NV : RT == 2 ? (j & 3) >> 1 : 0, ur = j >> 2;
    auto row_at = [&](int i) { return kDots ? 4 * grp + 2 * (j >> 3) + i : 4 * ur + grp; };  // in the tile
    float q[kDots ? 1 : RT][kDots ? 1 : E];
    // kDots: columns 0 .. 7 of the products are the heads' queries in f16, columns 8 .. 15 what that leaves,
    // q = (hi + lo 2^-11) 2^(e - 14): 22 bits of every element down to 2^-29 of its head's largest, and of
    // smaller ones what is above 2^-51 of that. The products of f16 keys with them are exact, their sums f32.
    const bool lo_col = (j & 8) != 0;
    v8h qm[kDots ? KC : 1];
    float unit = 1.0f;
    if constexpr (kDots)
    {
        float x[KC][8];
        uint32_t mx = 0;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                x[c][i] = q_s[hs * DK + 32 * c + 8 * grp + i];
                mx = max(mx, __builtin_bit_cast(uint32_t, x[c][i]) & 0x7FFFFFFFu);
            }
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, kWave));
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, kWave));
        const int e = min(max((int)(mx >> 23) - 127, -85), 127);
        const float up = __builtin_bit_cast(float, (uint32_t)(127 + 14 - e) << 23);  // the largest is below 2^15
        unit = __builtin_bit_cast(float, (uint32_t)(127 - 14 + e) << 23);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                const float y = x[c][i] * up;
                const _Float16 hi = (_Float16)y;
                const float rest = y - (float)hi;  // (NaN beside an infinity, which hi says)
                qm[c][i] = lo_col ? (_Float16)(rest == rest ? rest * 0x1p11f : 0.0f) : hi;
            }
    }
    else
    {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int e = 0; e < E; ++e) q[r][e] = q_s[r * DK + Row::dim(e, j)];
    }
    // 16 keys' products with the lane's column, of which it has four rows; then the scores of two of them: a hi
    // lane and its lo lane exchange the others. An infinite key times a part that is 0, or whose sign is not its
    // element's, can make NaN of an infinite sum: NaN from such keys, the tile's first `rows`, comes again from the
    // queries as they are. (The look at each tile's sums takes 1 to 2 % of a call: 16 x 16384, 16 heads over 2 of
    // 64 32.4 -> 32.9 us, of 128 51.7 -> 52.8. One look at the wave's sums, and then all its rows again, took as much.)
    auto dots = [&](const v8h(&k)[kDots ? KC : 1], float(&x)[NV], int rows) {
        typedef float v4f __attribute__((ext_vector_type(4)));
        v4f d = v4f{};
#pragma unroll
        for (int c = 0; c < (kDots ? KC : 1); ++c) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[c], qm[c], d, 0, 0, 0);
        const float y[4] = {d[0], d[1], d[2], d[3]};
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            const float got = dpp<kDppRor8>(lo_col ? y[i] : y[2 + i]);
            x[i] = lo_col ? __builtin_fmaf(y[2 + i], 0x1p-11f, got) : __builtin_fmaf(got, 0x1p-11f, y[i]);
        }
        if (__builtin_amdgcn_ballot_w64(__builtin_isunordered(x[0], x[NV - 1])) == 0) return;
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < (kDots ? KC : 1); ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, (uint32_t)(__builtin_bit_cast(uint16_t, (_Float16)k[c][i]) & 0x7FFFu));
        if (__builtin_amdgcn_ballot_w64(j < rows && top >= 0x7C00u) == 0) return;
        const float up = 1.0f / unit;  // a power of 2
#pragma unroll 1
        for (int r = 0; r < RT; ++r)
        {
            // lane j of every 16: row j's product with head r
            float d = 0.0f;
#pragma unroll
            for (int c = 0; c < (kDots ? KC : 1); ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) d = __builtin_fmaf((float)k[c][i], q_s[r * DK + 32 * c + 8 * grp + i], d);
            d += __shfl_xor(d, 16, kWave);
            d += __shfl_xor(d, 32, kWave);
#pragma unroll
            for (int i = 0; i < NV; ++i)
            {
                const float at = __shfl(d, row_at(i), kWave);
                if (r == hs && x[i] != x[i]) x[i] = at * up;
            }
        }
    };
    // over the lanes of 16 that hold the same heads
    auto same_max = [&](float x) {
        x = fmaxf(x, dpp<kDppRor8>(x));
        return kDots ? x : fmaxf(x, dpp<kDppRor4>(x));
    };
    auto same_sum = [&](float x) {
        x += dpp<kDppRor8>(x);
        return kDots ? x : x + dpp<kDppRor4>(x);
    };
    // (kDots: a product past f32's range would make a score of 0 NaN; any other score is past the cap, or the
    // range, with the largest float, too)
    auto held = [](float x) { return x > 3.40282347e38f ? 3.40282347e38f : x < -3.40282347e38f ? -3.40282347e38f : x; };
    const float scale2 = held(a.scale2 * unit), capi = held(a.capi * unit);
    float slope2[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) slope2[i] = a.slopes && hs + i < R ? a.slopes[h0 + hs + i] * 1.44269504f : 0.0f;
    auto shape = [&](float dot, int i, int t) {
        float x = a.cap2 > 0.0f ? a.cap2 * tanh_any(dot * capi) : dot * scale2;
        if (a.slopes) x = __builtin_fmaf(slope2[kDots ? 0 : i], (float)(t - p), x);
        return x;
    };

    float acc[RT][E], m[NM], l[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) m[i] = -__builtin_inff(), l[i] = 0.0f;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = 0.0f;

    auto tile = [&](int base, v8h(&km)[kDots ? KC : 1], Row(&vr)[kPgU]) {
        const bool part = base + kPgTile > n;  // rows behind the chunk's last one
        float x[NV], top[NM];
        if constexpr (kDots) dots(km, x, n - base);
        else
        {
            float s[NS];
#pragma unroll
            for (int u = 0; u < kPgU; ++u)
#pragma unroll
                for (int r = 0; r < RT; ++r)
                {
                    float d = kr[u].get(0) * q[r][0];
#pragma unroll
                    for (int e = 1; e < E; ++e) d = __builtin_fmaf(kr[u].get(e), q[r][e], d);
                    s[u * RT + r] = d;
                }
            fold16(s, lane);
#pragma unroll
            for (int i = 0; i < NV; ++i) x[i] = s[i];
        }
        bool grown = false;
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            const int tl = base + row_at(i);
            x[i] = shape(x[i], i, t0 + tl);
            if (part && tl >= n) x[i] = -__builtin_inff();
            if (kDots && i > 0) top[0] = fmaxf(top[0], x[i]);
            else top[kDots ? 0 : i] = x[i];
        }
#pragma unroll
        for (int i = 0; i < NM; ++i)
        {
            top[i] = same_max(top[i]);
            grown |= top[i] > m[i] + kPgLazy;
        }
        if (__builtin_amdgcn_ballot_w64(grown) != 0)
        {
            float corr[NM];
#pragma unroll
            for (int i = 0; i < NM; ++i)
            {
                const float to = top[i] > m[i] + kPgLazy ? top[i] : m[i];
                corr[i] = m[i] == to ? 1.0f : __builtin_amdgcn_exp2f(m[i] - to);
                l[i] *= corr[i];
                m[i] = to;
            }
            static_for<RT>([&](auto r) {
                constexpr int h = decltype(r)::value;
                const float f = bcast16<head_lane<kDots, RT>(h)>(corr[h % NM]);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[h][e] *= f;
            });
        }
        float pr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
        {
            // no score above -inf yet: nothing to add (and no -inf - -inf)
            pr[i] = x[i] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x[i] - m[kDots ? 0 : i]);
            l[kDots ? 0 : i] += pr[i];
        }
        if (part)  // whatever is there: 0 * it has to be 0
#pragma unroll
            for (int u = 0; u < kPgU; ++u)
                if (base + (kDots ? 4 * grp + u : 4 * u + grp) >= n) vr[u].zero();
        static_for<kPgU>([&](auto uu) {
            constexpr int u = decltype(uu)::value;
            static_for<RT>([&](auto r) {
                constexpr int h = decltype(r)::value;
                const float f = bcast16<score_lane<kDots, RT>(u, h)>(pr[kDots ? u % NV : h % NV]);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[h][e] = __builtin_fmaf(f, vr[u].get(e), acc[h][e]);
            });
        });
    };
    // (kDots: the next tile's rows are on their way during a tile, 3 .. 7 % of the call; where a tile takes the VALU
    // longer that changes nothing, since the other waves' are)
    for (int base = w * kPgTile; base < n; base += kPgWaves * kPgTile)
    {
        if constexpr (kDots)
        {
            v8h km_now[KC];
            Row vr_now[kPgU];
#pragma unroll
            for (int i = 0; i < KC; ++i) km_now[i] = km[i];
#pragma unroll
            for (int u = 0; u < kPgU; ++u) vr_now[u] = vr[u];
            if (base + kPgWaves * kPgTile < n) load(base + kPgWaves * kPgTile);
            tile(base, km_now, vr_now);
        }
        else
        {
            if (base != w * kPgTile) load(base);
            tile(base, km, vr);
        }
    }

    // ---- the new position: one more row, of the first group of the wave whose turn it is
    if (has_new && w == (n + kPgTile - 1) / kPgTile % kPgWaves)
    {
        float x[NV];
        if constexpr (kDots)
        {
            v8h k[KC];
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) k[c][i] = (_Float16)new_s[0][32 * c + 8 * grp + i];
            dots(k, x, kPgTile);
        }
        else
        {
            float s[NS];
#pragma unroll
            for (int u = 0; u < kPgU; ++u)
#pragma unroll
                for (int r = 0; r < RT; ++r)
                {
                    float d = 0.0f;
#pragma unroll
                    for (int e = 0; e < E; ++e) d = __builtin_fmaf(new_s[0][Row::dim(e, j)], q[r][e], d);
                    s[u * RT + r] = d;
                }
            fold16(s, lane);
#pragma unroll
            for (int i = 0; i < NV; ++i) x[i] = s[i];
        }
        float corr[NM], pr[NM];
#pragma unroll
        for (int i = 0; i < NM; ++i)
        {
            x[i] = grp == 0 ? shape(x[i], i, p) : -__builtin_inff();
            const float to = x[i] > m[i] ? x[i] : m[i];
            corr[i] = m[i] == to ? 1.0f : __builtin_amdgcn_exp2f(m[i] - to);
            pr[i] = x[i] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x[i] - to);
            // every row of lanes holds the same score: it counts once
            l[i] = l[i] * corr[i] + ((kDots ? j < RT : ur == 0) ? pr[i] : 0.0f);
            m[i] = to;
        }
        static_for<RT>([&](auto r) {
            constexpr int h = decltype(r)::value;
            const float f = bcast16<head_lane<kDots, RT>(h)>(corr[h % NM]);
            const float y = bcast16<head_lane<kDots, RT>(h)>(pr[h % NM]);
#pragma unroll
            for (int e = 0; e < E; ++e)
                acc[h][e] = __builtin_fmaf(y, grp == 0 ? new_s[1][Row::dim(e, j)] : 0.0f, acc[h][e] * f);
        });
    }

    // ---- join: maxima and sums of the 16 groups of lanes, then their weighted values
#pragma unroll
    for (int i = 0; i < NM; ++i)
    {
        l[i] = same_sum(l[i]);
        if (kDots ? j < RT : ur == 0)
        {
            ml_s[0][4 * w + grp][hs + i] = m[i];
            ml_s[1][4 * w + grp][hs + i] = l[i];
        }
    }
    if (lane == 0) bad_s[w] = bad;
    __syncthreads();
    constexpr int N = RT * E;
    float y[N];
#pragma unroll
    for (int r = 0; r < RT; ++r)
    {
        // lane j of every 16: group j's maximum and sum
        const float mj = ml_s[0][j][r], own = ml_s[0][4 * w + grp][r];
        float top = mj;
        top = fmaxf(top, dpp<kDppRor8>(top));
        top = fmaxf(top, dpp<kDppRor4>(top));
        top = fmaxf(top, dpp<kDppXor2>(top));
        top = fmaxf(top, dpp<kDppXor1>(top));
        if (w == r % kPgWaves)
        {
            float sum = ml_s[1][j][r] * (mj == top ? 1.0f : __builtin_amdgcn_exp2f(mj - top));
            sum += dpp<kDppRor8>(sum);
            sum += dpp<kDppRor4>(sum);
            sum += dpp<kDppXor2>(sum);
            sum += dpp<kDppXor1>(sum);
            if (lane == 0) tot_s[0][r] = top, tot_s[1][r] = sum;
        }
        // (a NaN among the scores leaves its sum and values NaN, not the maximum)
        const float f = own == top ? 1.0f : __builtin_amdgcn_exp2f(own - top);
#pragma unroll
        for (int e = 0; e < E; ++e) y[r * E + e] = acc[r][e] * f;
    }
    // over the wave's four groups: each swap exchanges halves of two registers between halves of the
    // lanes, and their sum holds one value in each half
    static_assert(N % 4 == 0, "a quarter of the values per group of lanes");
#pragma unroll
    for (int i = 0; i < N / 2; ++i) y[i] = fold32(y[i], y[i + N / 2]);
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
    {
        const int at = i + (grp >> 1) * (N / 2) + (grp & 1) * (N / 4);
        red_s[w][at / E * DK + Row::dim(at % E, j)] = fold16_rows(y[i], y[i + N / 4]);
    }
    __syncthreads();
    bad = (bad_s[0] | bad_s[1] | bad_s[2] | bad_s[3]) != 0;
    float* const rec = a.part + ((size_t)(it.first + c) * HG + gh) * (size_t)(a.RG * DK + kPgRec);
    for (int e = tid; e < R * DK; e += kPgThreads)
    {
        const int r = e / DK;
        const float sum = bad ? __builtin_nanf("") : tot_s[1][r];
        const float v = (red_s[0][e] + red_s[1][e]) + (red_s[2][e] + red_s[3][e]);
        if constexpr (kFinal) out[e * out_step] = sum == 0.0f ? 0.0f : v / sum;
        else
        {
            rec[e] = v;
            if (e % DK == 0)
            {
                rec[a.RG * DK + r] = tot_s[0][r];
                rec[a.RG * DK + 8 + r] = sum;
            }
        }
    }
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
size_t pages_items(size_t B, size_t len_bound, size_t chunk, size_t even)
{
    const size_t all = B * ceil_div(len_bound, chunk);
    return even && even + B < all ? even + B : all;
}

template <int DK, int RT, typename CT>
hipError_t launch_pages_rt(hipStream_t st, const PagesArgs& a)
{
    const dim3 grid((unsigned)(pages_items(a.B, a.len_bound, a.chunk, a.even) * a.Hkv * a.groups));
    if (a.nchunk == 1)
    {
        k_pages_attn<DK, RT, true, CT><<<grid, kPgThreads, 0, st>>>(a);
        return hipGetLastError();
    }
    k_pages_attn<DK, RT, false, CT><<<grid, kPgThreads, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_pages_join<DK><<<dim3((unsigned)a.H, (unsigned)a.B), kPgThreads, 0, st>>>(a);
    return hipGetLastError();
}

template <int DK, typename CT>
hipError_t launch_pages_dk(hipStream_t st, const PagesArgs& a)
{
    if (a.RG == 1) return launch_pages_rt<DK, 1, CT>(st, a);
    if (a.RG == 2) return launch_pages_rt<DK, 2, CT>(st, a);
    if (DK == 256 || a.RG <= 4) return launch_pages_rt<DK, 4, CT>(st, a);
    if constexpr (DK != 256) return launch_pages_rt<DK, 8, CT>(st, a);
}

// ------------------------------------------------------------------ fill from packed prompts

constexpr int kPfTok = 64;  // tokens of a work-group (16 x 1111 .. 2048 tokens, 5 heads of 128, f16: 46.5 us, 32: 50.4)

struct FillArgs
{
    const float* k;
    const float* v;
    const int32_t* cu;
    const int32_t* pos0;
    const float* cosT;
    const float* sinT;
    void* kc;
    void* vc;
    const int32_t* table;
    int M, B, Hkv, shift, table_stride, num_pages, limit;  // limit: positions from here on are not written
};

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

// Work-group = (64 tokens, KV head, keys or values): the head's dk feature rows of those tokens read
// along tokens, turned through LDS and written as rows of pages, keys rotated at their positions. Bound by
// HBM; a work-group lives for its chain of round trips, so the features are on their way while the chain
// sequence -> position -> page and rotation is followed, the same in each wave (by bisection in each thread
// behind the features 56.5 us, 44.4 so: 16 x 1111 .. 2048 tokens, 5 heads of 128, f16, 4.4 TB/s).
// Tokens of no sequence, positions outside the table or the rope tables and pages outside the pool are
// not written.
template <int DK, typename CT>
__global__ __launch_bounds__(256) void k_pages_fill(FillArgs a)
{
    constexpr int HALF = DK / 2, NR = 256 / kPfTok, U = DK / NR;
    constexpr int J = HALF / 2, NT = 256 / J, N = kPfTok / NT;  // threads of a token, tokens at a time, times
    __shared__ float x_s[DK][kPfTok + 1];
    const int tid = threadIdx.x, lane = tid & 63, g = blockIdx.y;
    const bool keys = blockIdx.z == 0;
    const int m0 = blockIdx.x * kPfTok;
    const int c = tid % kPfTok, i0 = tid / kPfTok;
    const float* src = (keys ? a.k : a.v) + (size_t)(g * DK + i0) * (size_t)a.M + (size_t)min(m0 + c, a.M - 1);
    const int b = wave_sequence(a.cu, a.B, a.M, m0, lane);
    const int at = b < 0 ? -1 : packed_position(a.cu, a.pos0, b, m0 + (lane & (kPfTok - 1)), a.limit);
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = src[(size_t)(NR * u) * (size_t)a.M];
    int to = -1;
    if (at >= 0)
    {
        const int id = a.table[(size_t)b * a.table_stride + (at >> a.shift)];
        if (page_ok(id, a.num_pages)) to = (int)page_row(id, g, at & ((1 << a.shift) - 1), a.Hkv, a.shift);
    }
    // a thread stores features (j, j + 1) and (j + dk / 2, j + 1 + dk / 2) of its tokens
    const int j = 2 * (tid % J), c0 = tid / J;
    typedef float v2f __attribute__((ext_vector_type(2), aligned(4)));
    v2f cs[N], sn[N];
    int row[N];
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
        row[n] = __shfl(to, c0 + NT * n, kWave);
        const size_t r = (size_t)max(__shfl(at, c0 + NT * n, kWave), 0) * HALF + (size_t)j;
        if (keys && a.cosT)
        {
            cs[n] = *reinterpret_cast<const v2f*>(a.cosT + r);
            sn[n] = *reinterpret_cast<const v2f*>(a.sinT + r);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) x_s[i0 + NR * u][c] = x[u];
    __syncthreads();
    typedef CT v2 __attribute__((ext_vector_type(2)));
    CT* const dst = static_cast<CT*>(keys ? a.kc : a.vc);
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
        const int cn = c0 + NT * n;
        if (row[n] < 0) continue;
        float y[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
        {
            const float x0 = x_s[j + e][cn], x1 = x_s[j + e + HALF][cn];
            y[0][e] = x0, y[1][e] = x1;
            if (keys && a.cosT) pg_rope(x0, x1, cs[n][e], sn[n][e], y[0][e], y[1][e]);
        }
        CT* o = dst + (size_t)row[n] * DK + j;
        *reinterpret_cast<v2*>(o) = v2{(CT)y[0][0], (CT)y[0][1]};
        *reinterpret_cast<v2*>(o + HALF) = v2{(CT)y[1][0], (CT)y[1][1]};
    }
}

template <typename CT>
hipError_t launch_pages_fill_ct(hipStream_t st, const FillArgs& a, size_t dk)
{
    const dim3 grid((unsigned)ceil_div(a.M, kPfTok), (unsigned)a.Hkv, 2);
    if (dk == 64) k_pages_fill<64, CT><<<grid, 256, 0, st>>>(a);
    else if (dk == 128) k_pages_fill<128, CT><<<grid, 256, 0, st>>>(a);
    else if (dk == 256) k_pages_fill<256, CT><<<grid, 256, 0, st>>>(a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

int log2_of(size_t v)
{
    int n = 0;
    while ((size_t(1) << n) < v) ++n;
    return n;
}

}  // namespace

// Query heads of a KV head in groups of at most 8 (dk = 256: 4, whose registers are as many), as even as they go
static size_t pages_groups(size_t R, size_t dk) { return ceil_div(R, (size_t)(dk == 256 ? 4 : kPgMaxR)); }

// How a call is cut: chunks of `chunk` positions (nchunk to a sequence), or with even > 0 about `even` of a
// size that the kernels find
struct PagesCut
{
    size_t chunk, nchunk, even;
};

static PagesCut pages_cut(size_t B, size_t Hkv, size_t R, size_t dk, size_t len_bound, size_t num_cus)
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
static size_t pages_records(size_t B, size_t Hkv, size_t groups, size_t RG, size_t dk, size_t len_bound, const PagesCut& cut)
{
    return pages_items(B, len_bound, cut.chunk, cut.even) * Hkv * groups * (RG * dk + kPgRec);
}

size_t pages_workspace_bytes(size_t B, size_t H, size_t Hkv, size_t dk, size_t len_bound, size_t num_cus)
{
    const size_t R = H / Hkv, groups = pages_groups(R, dk);
    const PagesCut cut = pages_cut(B, Hkv, R, dk, len_bound, num_cus);
    if (cut.nchunk == 1) return 0;
    return pages_records(B, Hkv, groups, ceil_div(R, groups), dk, len_bound, cut) * sizeof(float) + (cut.even ? B * sizeof(int2) : 0);
}

hipError_t launch_pages_attn(hipStream_t st, const nnhip_kv_pages& kv, const float* q, const float* k, const float* v,
                             size_t B, size_t H, const int32_t* pos, size_t len_bound, const float* cosT,
                             const float* sinT, float scale, float softcap, const float* slopes, bool tokens,
                             float* part, float* out, size_t num_cus)
{
    constexpr double kLog2e = 1.4426950408889634;
    const size_t R = H / kv.Hkv, dk = kv.dk, groups = pages_groups(R, dk);
    const PagesCut cut = pages_cut(B, kv.Hkv, R, dk, len_bound, num_cus);
    const bool cap = softcap > 0.0f;
    PagesArgs a{q, k, v, pos, cosT, sinT, kv.k, kv.v, kv.table, slopes, part,
                reinterpret_cast<int2*>(part + (cut.even ? pages_records(B, kv.Hkv, groups, ceil_div(R, groups), dk, len_bound, cut) : 0)),
                out, (int)B, (int)H, (int)kv.Hkv, (int)R,
                (int)groups, (int)ceil_div(R, groups), log2_of(kv.page_size), (int)kv.table_stride, (int)kv.num_pages,
                (int)len_bound, (int)cut.chunk, (int)cut.nchunk, (int)cut.even, (float)(scale * kLog2e),
                cap ? scale / softcap : 0.0f, cap ? (float)(softcap * kLog2e) : 0.0f, tokens ? 1 : 0};
    if (kv.f16)
    {
        if (kv.dk == 64) return launch_pages_dk<64, _Float16>(st, a);
        if (kv.dk == 128) return launch_pages_dk<128, _Float16>(st, a);
        if (kv.dk == 256) return launch_pages_dk<256, _Float16>(st, a);
        return hipErrorInvalidValue;
    }
    if (kv.dk == 64) return launch_pages_dk<64, float>(st, a);
    if (kv.dk == 128) return launch_pages_dk<128, float>(st, a);
    if (kv.dk == 256) return launch_pages_dk<256, float>(st, a);
    return hipErrorInvalidValue;
}

hipError_t launch_pages_fill(hipStream_t st, const nnhip_kv_pages& kv, const float* k, const float* v, size_t M,
                             const int32_t* cu, const int32_t* pos0, size_t B, const float* cosT, const float* sinT,
                             size_t limit)
{
    FillArgs a{k, v, cu, pos0, cosT, sinT, kv.k, kv.v, kv.table, (int)M, (int)B, (int)kv.Hkv, log2_of(kv.page_size),
               (int)kv.table_stride, (int)kv.num_pages, (int)limit};
    return kv.f16 ? launch_pages_fill_ct<_Float16>(st, a, kv.dk) : launch_pages_fill_ct<float>(st, a, kv.dk);
}

}  // namespace nnhip
