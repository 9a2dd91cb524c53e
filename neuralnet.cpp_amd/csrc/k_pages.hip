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
#include "pages_split.hpp"

#include <cmath>
#include <type_traits>
#include <utility>

namespace nnhip
{
namespace
{

constexpr int kPgU = 4;          // rows of a group of 16 lanes in flight together
constexpr int kPgTile = 16;      // rows of a wave's tile: 4 groups x kPgU
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
constexpr float kPgLazy = 8.0f;  // log2 growth of a maximum before its sums are rescaled
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

}  // namespace

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
