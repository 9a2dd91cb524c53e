// prompt_spans.hpp — what the attention kernels of packed prompts share (k_prefill.hip, k_prefill_i8.hip):
// their arguments, the queries of a wave, the cut of a call's work into equal spans and the join of the items
// that spans share.
#pragma once

#include "common.hpp"
#include "pages_index.hpp"

namespace nnhip
{
namespace
{

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kPQ = 32;   // queries per wave of the attention, tokens per block of the cache fill
constexpr int kPK = 32;   // keys per tile

__device__ __forceinline__ __amdgpu_buffer_rsrc_t pf_rsrc(const void* base, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ float4 ld_f4(__amdgpu_buffer_rsrc_t r, uint32_t off)
{
    return __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

// (x0, x1) = (x[j], x[j + dk/2]) -> x*cos + rotate_half(x)*sin: two rounded products and a
// rounded sum per output, as the decode append does.
__device__ __forceinline__ void pf_rope(float x0, float x1, float cs, float sn, float& y0, float& y1)
{
    y0 = __fadd_rn(__fmul_rn(x0, cs), __fmul_rn(-x1, sn));
    y1 = __fadd_rn(__fmul_rn(x1, cs), __fmul_rn(x0, sn));
}

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kPWaves = 8;             // waves of a work-group: R heads x (8 / R) blocks of 32 queries
constexpr int kPThreads = 64 * kPWaves;
constexpr int kPWaveShift = 3, kPQShift = 5, kPKShift = 5;  // their logarithms
static_assert(kPWaves == 1 << kPWaveShift && kPQ == 1 << kPQShift && kPK == 1 << kPKShift, "");
constexpr int kPExpMax = 48;           // scalings beyond 2^+-48 take the f32 products
constexpr float kPLazy = 8.0f;         // log2 growth of a query's maximum before its sums are rescaled

struct PrefillArgs
{
    const float* q;
    const void* kc;  // caches of CT elements
    const void* vc;
    const float* cosT;
    const float* sinT;
    float* out;
    int B, T, H, Hkv, R, pos0, max_len, nqb;
    float scale;
    float scale2;  // |scale| * log2(e)
    int f32;       // 1: the f32 products throughout (a scale outside [2^-20, 2^20])
    int M;         // columns of q and out (paged; otherwise B * T)
    int groups;    // work-groups that share a KV head's queries: R heads each
    // paged: B packed sequences of at most T tokens, whose keys and values lie in pages
    const int32_t* table;
    const int32_t* cu;      // columns cu[b] .. cu[b + 1] - 1 are sequence b's
    const int32_t* starts;  // position of its first token, or null for 0
    const int32_t* prefix;  // positions before prefix[b] are visible to all its queries, or null
    const float* slopes;
    int table_stride, num_pages, shift, limit;  // limit: positions from here on have no place
    float cap2, capi2;      // softcap * log2(e) and its inverse, 0 without
    float* part;            // spans: records of the items that several work-groups share
    int spans;              // work-groups that take spans of all tiles (see prompt_cut); 0: one item each
};

// The two halves of two f32 values scaled into f16's range: x = hi + lo up to 2^-23 |x| or 2^-25
__device__ __forceinline__ void split2(float x0, float x1, v2h& hi, v2h& lo)
{
    hi = __builtin_convertvector(v2f{x0, x1}, v2h);
    // x - hi, exact, from the packed half in place (the compiler widens it with an instruction first)
    const uint32_t u = __builtin_bit_cast(uint32_t, hi);
    float l0, l1;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(l0) : "v"(u), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(l1) : "v"(u), "v"(x1));
    lo = __builtin_convertvector(v2f{l0, l1}, v2h);
}

// 2^e for |e| <= 126
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23); }

// The exponent that brings values whose largest bit pattern is mx (sign cleared) into [2^14, 2^15):
// kPExpMax for all-zero values. Outside +-kPExpMax (infinities and NaN among it) the f32 products run.
__device__ __forceinline__ int f16_exp(uint32_t mx) { return mx == 0 ? kPExpMax : 14 + 127 - (int)(mx >> 23); }

// A lane's value and that of the lane 32 away
__device__ __forceinline__ float max_halves(float x)
{
    const auto z = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t a = z[0], b = z[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// Where a wave works: query head, first query, the lane's query
struct PrefillWave
{
    int b, g, head, t0, qt, qpos;
    bool live;  // the wave has queries
};

// What depends on the sequence: its tokens, its first column and position, the columns of q, the last key
// that the lane's query sees and the last ones that all and any of the wave's queries see. Equal prompts
// at one position have it in the arguments.
template <bool kPaged>
struct PrefillSeq
{
    __device__ __forceinline__ int n(const PrefillArgs& a) const { return a.T; }
    __device__ __forceinline__ int col0(const PrefillArgs& a, const PrefillWave& w) const { return w.b * a.T; }
    __device__ __forceinline__ int pos0(const PrefillArgs& a) const { return a.pos0; }
    __device__ __forceinline__ int cols(const PrefillArgs& a) const { return a.B * a.T; }
    __device__ __forceinline__ int sight(const PrefillWave& w) const { return w.qpos; }
    __device__ __forceinline__ int from(const PrefillArgs& a, const PrefillWave& w) const { return a.pos0 + w.t0; }
    __device__ __forceinline__ int to(const PrefillArgs& a, const PrefillWave& w) const { return a.pos0 + w.t0 + kPQ - 1; }
};
template <>
struct PrefillSeq<true>
{
    int n_, col0_, pos0_, pre;  // pre: keys that every query sees
    __device__ __forceinline__ int n(const PrefillArgs&) const { return n_; }
    __device__ __forceinline__ int col0(const PrefillArgs&, const PrefillWave&) const { return col0_; }
    __device__ __forceinline__ int pos0(const PrefillArgs&) const { return pos0_; }
    __device__ __forceinline__ int cols(const PrefillArgs& a) const { return a.M; }
    __device__ __forceinline__ int sight(const PrefillWave& w) const { return max(w.qpos, pre - 1); }
    __device__ __forceinline__ int from(const PrefillArgs&, const PrefillWave& w) const { return max(pos0_ + w.t0, pre - 1); }
    __device__ __forceinline__ int to(const PrefillArgs&, const PrefillWave& w) const { return max(pos0_ + w.t0 + kPQ - 1, pre - 1); }
};

// The lane's query: values x[c][0][e] of its dimensions 2Gc + Gh + e below DK/2 and x[c][1][e] of those DK/2
// further. Lanes past the last token repeat it (they are never stored).
template <int DK, int G>
struct PrefillQuery
{
    static constexpr int HALF = DK / 2, NG = HALF / (2 * G);
    float x[NG][2][G];
    template <bool kPaged>
    __device__ __forceinline__ void load(const PrefillArgs& a, const PrefillWave& w, const PrefillSeq<kPaged>& seq, int h)
    {
        const int M = seq.cols(a);
        const __amdgpu_buffer_rsrc_t rq = pf_rsrc(a.q, (uint32_t)((size_t)a.H * DK * (size_t)M * 4u));
        const int qt = min(w.qt, seq.n(a) - 1);
        const uint32_t q_at = (uint32_t)(((size_t)(w.head * DK + G * h) * (size_t)M + (size_t)(seq.col0(a, w) + qt)) * 4u);
#pragma unroll
        for (int c = 0; c < NG; ++c)
#pragma unroll
            for (int e = 0; e < G; ++e)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    x[c][q][e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rq, q_at, (2 * G * c + e + HALF * q) * M * 4, 0));
    }
    // f(c, e, rotated values), with cs(c, i) and sn(c, i) = the tables at dimensions 2Gc + Gh + 4i .. + 3
    template <typename C, typename S, typename F>
    __device__ __forceinline__ void rotate(const PrefillArgs& a, C&& cs, S&& sn, F&& f) const
    {
        if (!a.cosT)
        {
#pragma unroll
            for (int c = 0; c < NG; ++c)
#pragma unroll
                for (int e = 0; e < G; ++e) f(c, e, x[c][0][e], x[c][1][e]);
            return;
        }
#pragma unroll
        for (int c = 0; c < NG; ++c)
#pragma unroll
            for (int i = 0; i < G / 4; ++i)
            {
                const float4 c4 = cs(c, i), s4 = sn(c, i);
                const float cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    float y0, y1;
                    pf_rope(x[c][0][4 * i + e], x[c][1][4 * i + e], cv[e], sv[e], y0, y1);
                    f(c, 4 * i + e, y0, y1);
                }
            }
    }
};

__device__ __forceinline__ uint32_t rope_bytes(const PrefillArgs& a, int half)
{
    return a.cosT ? (uint32_t)((size_t)a.max_len * half * 4u) : 0u;  // (paged: max_len = limit)
}

// out[head*DK + i][m] = y(d, v) for the lane's query: element v of block d belongs to row
// r = 8(v/4) + 4h + v%4 of the block; dim(d, r) is its dimension
template <int DK, bool kPaged, typename D, typename Y>
__device__ __forceinline__ void store_out(const PrefillArgs& a, const PrefillWave& w, const PrefillSeq<kPaged>& seq, int h,
                                          D&& dim, Y&& y)
{
    if (w.qt >= seq.n(a)) return;
    const int M = seq.cols(a), m = seq.col0(a, w) + w.qt;
#pragma unroll
    for (int d = 0; d < DK / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v)
            a.out[(size_t)(w.head * DK + dim(d, 8 * (v >> 2) + 4 * h + (v & 3))) * (size_t)M + (size_t)m] = y(d, v);
}

// A record (prompt_record) of the wave's part of an item: y(d, v) as store_out's, the lane's reference maximum and
// sum. Lanes l and l + 32 hold other dimensions of one query.
template <int DK, typename D, typename Y>
__device__ __forceinline__ void store_record(float* rec, int tid, D&& dim, Y&& y, float m, float l)
{
    const int h = (tid >> 5) & 1, row = (tid >> 6) * 32 + (tid & 31);
#pragma unroll
    for (int d = 0; d < DK / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) rec[(size_t)dim(d, 8 * (v >> 2) + 4 * h + (v & 3)) * (32 * kPWaves) + row] = y(d, v);
    if (h == 0)
    {
        rec[(size_t)DK * (32 * kPWaves) + row] = m;
        rec[(size_t)(DK + 1) * (32 * kPWaves) + row] = l;
    }
}

// log2 of the heads of a work-group, which are 1, 2, 4 or 8
__device__ __forceinline__ int log2_heads(const PrefillArgs& a) { return __builtin_ctz(a.R); }

// What a work-group works on: a block of qn = 32 (8 / R) queries of R heads (from `first`, of KV head g) of
// sequence b. Paged: with the sequence.
struct PrefillItem
{
    int b, g, first, qb;
    PrefillSeq<true> seq;
};

// The place of thread tid in an item, and the last key that the item sees
template <bool kPaged>
__device__ __forceinline__ void seat(const PrefillArgs& a, const PrefillItem& it, int tid, PrefillWave& w,
                                     PrefillSeq<kPaged>& seq, int& last_key)
{
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rs = log2_heads(a), qn = kPQ << (kPWaveShift - rs);  // queries of the work-group
    w.b = it.b;
    w.g = it.g;
    w.head = it.first + (wave & (a.R - 1));
    w.t0 = it.qb * qn + (wave >> rs) * kPQ;
    w.qt = w.t0 + (tid & 31);
    if constexpr (kPaged) seq = it.seq;
    w.qpos = seq.pos0(a) + w.qt;
    w.live = w.t0 < seq.n(a);
    last_key = seq.pos0(a) + min(it.qb * qn + qn, seq.n(a)) - 1;
    if constexpr (kPaged) last_key = max(last_key, seq.pre - 1);
}

// ---- paged: packed sequences

// Sequence b as its arguments say; false if it does not fit them (it gets NaN)
__device__ __forceinline__ bool packed_seq(const PrefillArgs& a, int b, PrefillSeq<true>& seq)
{
    const int col0 = a.cu[b], pos0 = a.starts ? a.starts[b] : 0;
    const int64_t n = (int64_t)a.cu[b + 1] - col0;
    if (col0 < 0 || col0 + n > a.M || n > a.T || pos0 < 0 || pos0 >= a.limit || n > a.limit - pos0) return false;
    seq = {(int)n, col0, pos0, a.prefix ? max(0, min(a.prefix[b], pos0 + (int)n)) : 0};
    return true;
}

// NaN in the columns that are there of the heads from `first` on, by thread `at` of `step`
template <int DK>
__device__ void store_nan(const PrefillArgs& a, int b, int first, int heads, int at, int step)
{
    const int64_t c1 = min((int64_t)a.cu[b + 1], (int64_t)a.M);
    for (int64_t c = (int64_t)max(a.cu[b], 0) + at; c < c1; c += step)
        for (int i = 0; i < heads * DK; ++i) a.out[(size_t)(first * DK + i) * (size_t)a.M + (size_t)c] = __builtin_nanf("");
}

// Work of the whole call in tiles of 32 keys, for work-groups that take equal spans of it: blocks of queries
// differ in their keys by any factor, and a chunk of a long prompt has fewer of them than the GPU has CUs
// (4 x 1024 queries of 20 heads: 270 for 256 CUs, the last 14 of which took as long as all others). The order
// is (head group, sequence, block of queries, tile); an item counts kOver tiles more than it has, which
// its queries and outputs cost. A cut within the first or last kSnap tiles of an item moves to its edge, and
// where no item has more than kShort tiles, to its start. Every work-group finds its two cuts.
struct PromptCut
{
    int gh, b, qb, t;
};
constexpr int kOver = 3, kSnap = 2, kShort = 4, kSpanMin = 2;
constexpr int kOverI8 = 5;  // over 8-bit pages, whose tiles take less (8 x 77 .. 1900 of 64: 69 us, with 3 73, 8 75; 4 x 700 .. 1024 at 6144 435, 438, 436)

__device__ __forceinline__ int prompt_blocks(const PrefillArgs& a, int n)
{
    const int qs = kPQShift + kPWaveShift - log2_heads(a);  // log2 of a block's queries
    return (n + (1 << qs) - 1) >> qs;
}

// Tiles of block qb
__device__ __forceinline__ int prompt_tiles(const PrefillArgs& a, const PrefillSeq<true>& q, int qb)
{
    const int qs = kPQShift + kPWaveShift - log2_heads(a);
    return (max(q.pos0_ + min((qb + 1) << qs, q.n_), q.pre) + kPK - 1) >> kPKShift;
}

// Tiles of blocks 0 .. qb - 1 with `over` each: A + j u for block j - 1, but at least P, and the last block's own
__device__ __forceinline__ int64_t prompt_before(const PrefillArgs& a, const PrefillSeq<true>& q, int qb, int over = kOver)
{
    const int us = kPWaveShift - log2_heads(a);  // log2 of u
    const int nq = prompt_blocks(a, q.n_), A = (q.pos0_ + kPK - 1) >> kPKShift, P = (q.pre + kPK - 1) >> kPKShift;
    const int full = min(qb, nq - 1);
    const int k = max(0, min(full, ((P - A + (1 << us) - 1) >> us) - 1));
    int64_t f = (int64_t)k * P + (int64_t)(full - k) * (A + over) + (int64_t)k * over +
                (((int64_t)full * (full + 1) - (int64_t)k * (k + 1)) >> 1 << us);
    if (qb == nq && nq > 0) f += prompt_tiles(a, q, nq - 1) + over;
    return f;
}

// Work of sequence b (0 past the last, or if it does not fit)
__device__ __forceinline__ int64_t prompt_work(const PrefillArgs& a, int b, int& most, int over = kOver)
{
    PrefillSeq<true> q;
    most = 0;
    if (b >= a.B || !packed_seq(a, b, q) || q.n_ <= 0) return 0;
    const int nq = prompt_blocks(a, q.n_);
    most = prompt_tiles(a, q, nq - 1);
    return prompt_before(a, q, nq, over);
}

__device__ __forceinline__ int64_t read_lane64(int64_t x, int l)
{
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, l);
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)x >> 32), l) << 32) | lo);
}

// The cut before span `span` of `spans` (or the call's end), found by a wave. kFew: where two tiles to a span are enough for
// the whole call, what an item costs beside its tiles is left out, so that the tiles spread over as many work-groups as they
// can (8-bit pages, 20 heads of 128: 3 x 5 .. 40 queries behind 200 positions 23 us, with it 26; 32 behind 200 18 and 22, behind 1000 25 and 24)
// found, if not null: the cut's sequence, where there is one
template <bool kFew = false>
__device__ __forceinline__ PromptCut prompt_cut(const PrefillArgs& a, int spans, int span, PrefillSeq<true>* found = nullptr)
{
    const int lane = threadIdx.x & 63;
    constexpr int kItem = kFew ? kOverI8 : kOver;
    int over = kItem;
    int64_t own = 0, sum = 0;
    int most = 0, blocks = 0;
    PrefillSeq<true> mine{};  // the lane's sequence, of up to 64
    for (int b = lane; b < a.B; b += kWave)
    {
        int m;
        own = prompt_work(a, b, m, kItem);
        sum += own;
        most = max(most, m);
        if constexpr (kFew)
        {
            if (packed_seq(a, b, mine) && mine.n_ > 0) blocks += prompt_blocks(a, mine.n_);
        }
    }
    for (int off = 1; off < min(a.B, kWave); off <<= 1)
    {
        sum += __shfl_xor(sum, off, kWave);
        most = max(most, __shfl_xor(most, off, kWave));
        if constexpr (kFew) blocks += __shfl_xor(blocks, off, kWave);
    }
    int64_t head = read_lane64(sum, 0);  // tiles of a head group
    if constexpr (kFew)
    {
        const int64_t bare = head - (int64_t)kItem * __builtin_amdgcn_readfirstlane(blocks);
        if (bare * (a.Hkv * a.groups) <= (int64_t)kSpanMin * spans)
        {
            over = 0;
            head = bare;
            int m;
            if (a.B <= kWave) own = prompt_work(a, lane, m, 0);
        }
    }
    const int64_t total = head * (a.Hkv * a.groups);  // of all
    most = __builtin_amdgcn_readfirstlane(most);
    const bool small = total < 0x7FFFFFFF - spans;  // (a 64-bit division is a hundred instructions)
    int64_t per = small ? (int64_t)((uint32_t)((int)total + spans - 1) / (uint32_t)spans) : (total + spans - 1) / spans;
    int snap = 1 << 30;
    if (most > kShort)
    {
        per = max(per, (int64_t)max(kSpanMin + min(over, kOver), (most + over) / 32));  // at most about 32 spans to an item
        snap = kSnap;
    }
    // where tile x of the call lies
    const int64_t x = span * per;
    if (x >= total) return {a.Hkv * a.groups, 0, 0, 0};
    const int gh = small ? (int)((uint32_t)x / (uint32_t)head) : (int)(x / head);
    int64_t y = x - gh * head;
    for (int b0 = 0; b0 < a.B; b0 += kWave)
    {
        int m;
        if (a.B > kWave) own = prompt_work(a, b0 + lane, m, over);
        int64_t incl = own;
        const int live = min(a.B - b0, kWave);
        for (int off = 1; off < live; off <<= 1)
        {
            const int64_t t = __shfl_up(incl, off, kWave);
            if (lane >= off) incl += t;
        }
        const unsigned long long here = __builtin_amdgcn_ballot_w64(lane < live && incl > y);
        if (here == 0)
        {
            y -= read_lane64(incl, live - 1);
            continue;
        }
        const int l = __builtin_ctzll(here), b = b0 + l;
        y -= read_lane64(incl - own, l);
        PrefillSeq<true> q;
        if (kFew && a.B <= kWave)
            q = {__builtin_amdgcn_readlane(mine.n_, l), __builtin_amdgcn_readlane(mine.col0_, l), __builtin_amdgcn_readlane(mine.pos0_, l),
                 __builtin_amdgcn_readlane(mine.pre, l)};
        else packed_seq(a, b, q);
        if (found) *found = q;
        // the last block whose tiles begin at or before y: of 64 candidates at a time
        int qb = 0;
        for (int n = prompt_blocks(a, q.n_); n > 1;)
        {
            const int step = (n + kWave - 1) / kWave;
            const bool at_or_before = lane * step < n && prompt_before(a, q, qb + lane * step, over) <= y;
            const int k = step * (__builtin_popcountll(__builtin_amdgcn_ballot_w64(at_or_before)) - 1);
            qb += k;
            n = min(step, n - k);
        }
        const int tiles = prompt_tiles(a, q, qb);
        int t = (int)(y - prompt_before(a, q, qb, over)) - over;
        if (t < snap) t = 0;
        else if (tiles - t < snap) return {gh, b, qb + 1, 0};
        return {gh, b, qb, t};
    }
    return {a.Hkv * a.groups, 0, 0, 0};
}

__device__ __forceinline__ PromptCut uniform(const PromptCut& x)
{
    return {__builtin_amdgcn_readfirstlane(x.gh), __builtin_amdgcn_readfirstlane(x.b), __builtin_amdgcn_readfirstlane(x.qb),
            __builtin_amdgcn_readfirstlane(x.t)};
}

__device__ __forceinline__ bool cut_before(const PromptCut& x, const PromptCut& y)
{
    if (x.gh != y.gh) return x.gh < y.gh;
    if (x.b != y.b) return x.b < y.b;
    return x.qb != y.qb ? x.qb < y.qb : x.t < y.t;
}

__device__ __forceinline__ bool cut_same_item(const PromptCut& x, const PromptCut& y) { return x.gh == y.gh && x.b == y.b && x.qb == y.qb; }

// Record `slot` of span g: an item's outputs before the division, as [dk][256] by dimension and lane of a work-group's
// waves, then its reference maxima and its sums [256] each. Slot 0: the span's first item, begun by another
// span; slot 1: its last, begun here.
template <int DK>
__device__ __forceinline__ float* prompt_record(const PrefillArgs& a, int g, int slot)
{
    return a.part + ((size_t)g * 2 + slot) * (size_t)((DK + 2) * 32 * kPWaves);
}

// The cuts before each of the spans, behind their records
template <int DK>
__device__ __forceinline__ PromptCut* prompt_cuts(const PrefillArgs& a, int spans)
{
    return reinterpret_cast<PromptCut*>(prompt_record<DK>(a, spans, 0));
}

// The items that several spans share: work-group g joins the one that the cut before span g is the first to
// fall into, from its records: sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, N dimensions of its 256 queries.
// Span g - 1 wrote slot 1, those from g on that begin within the item slot 0: fewer than 64 (prompt_cut's per).
template <int DK, int N = 16, int U = 1>
__global__ __launch_bounds__(32 * kPWaves) void k_prompt_join(PrefillArgs a)
{
    const int g = blockIdx.x + 1, d0 = blockIdx.y * N, row = threadIdx.x, lane = row & 63;
    const PromptCut* const cuts = prompt_cuts<DK>(a, a.spans);
    const PromptCut at = cuts[g], last = cuts[g - 1], later = cuts[min(g + lane, a.spans - 1)];
    if (at.gh >= a.Hkv * a.groups || at.t == 0 || (cut_same_item(at, last) && last.t > 0)) return;
    const unsigned long long within = __builtin_amdgcn_ballot_w64(g + lane < a.spans && cut_same_item(at, later));
    const int n = 1 + __builtin_popcountll(within);
    PrefillSeq<true> q;
    packed_seq(a, at.b, q);
    const int wave = row >> 5, qt = at.qb * kPQ * (kPWaves / a.R) + wave / a.R * kPQ + (row & 31);
    if (qt >= q.n_) return;
    float top = -__builtin_inff(), den = 0.0f, y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = 0.0f;
    // (the records of U spans on their way together, joined in their order: 32 records 9.7 us with 2, 12.4 one by one)
    for (int s0 = 0; s0 < n; s0 += U)
    {
        float x[U][N], m[U], l[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int s = min(s0 + u, n - 1);
            const float* rec = prompt_record<DK>(a, g - 1 + s, s == 0 ? 1 : 0) + row;
#pragma unroll
            for (int i = 0; i < N; ++i) x[u][i] = rec[(size_t)(d0 + i) * (32 * kPWaves)];
            m[u] = rec[(size_t)DK * (32 * kPWaves)], l[u] = rec[(size_t)(DK + 1) * (32 * kPWaves)];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            // (selections, not a branch, which the loads would be moved behind)
            const bool there = u == 0 || s0 + u < n;
            const float to = fmaxf(top, m[u]);
            const float old = top == to ? 1.0f : __builtin_amdgcn_exp2f(top - to);
            const float now = m[u] == to ? 1.0f : __builtin_amdgcn_exp2f(m[u] - to);
            den = there ? __builtin_fmaf(l[u], now, den * old) : den;
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = there ? __builtin_fmaf(x[u][i], now, y[i] * old) : y[i];
            top = there ? to : top;
        }
    }
    float* out = a.out + (size_t)((at.gh * a.R + wave % a.R) * DK + d0) * (size_t)a.M + (size_t)(q.col0_ + qt);
#pragma unroll
    for (int i = 0; i < N; ++i) out[(size_t)i * (size_t)a.M] = den == 0.0f ? 0.0f : y[i] / den;
}

}  // namespace
}  // namespace nnhip
