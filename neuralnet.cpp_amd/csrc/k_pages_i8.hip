// k_pages_i8.hip — the paged KV cache in 8 bits: int8 codes and one f32 scale for every `block` positions of a head.
// Its fill from packed prompts, the values read back, and the attention of one new token per sequence with the
// append; the attention of packed prompts is k_prefill_i8.hip's.
//
// Layouts (device), as the pools of k_pages.hip by pages (num_pages, Hkv, page_size, dk), but for each 16 positions:
//   keys    (dk / 16, 16 positions, 16 dimensions) bytes: a wave's 16-byte loads of 16 positions are one run, and
//           each is an operand of the int8 MFMA as it stands (16 positions x 64 dimensions)
//   values  (dk, 16 positions) bytes: 16 positions of a dimension are an operand of the product with the weights
//   scales  (num_pages, Hkv, page_size / block) f32, keys and values apart
//
// A block's scale is s = fl(max|x| fl(1/127)) over its tokens and the head's dk dimensions, a code quantize_one(x, s)
// (token_quant.hpp): the engine's activations are held the same way. A token that joins a block whose scale is smaller
// raises it, and the older codes q become quantize_one(fl(q s_old), s): each time at most half a step of the new
// scale is added to what they are off.
#include "pages_split.hpp"
#include "token_quant.hpp"

#include <cmath>
#include <type_traits>

namespace nnhip
{
namespace
{

// The pools of a cache and their scales
struct PoolsI8
{
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    int bshift;  // log2(block)
};

typedef int32_t v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));

// Order between a wave's own LDS accesses of different lanes
__device__ __forceinline__ void wave_lds_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The scale of a block that goes on: `before` unless the new tokens' s is larger. A NaN stays, as an infinity does (s is never NaN): the
// block's positions keep standing for NaN, and the new tokens' codes are 0.
__device__ __forceinline__ float joined_scale(float s, float before) { return s > before ? s : before; }

// A block whose scale has grown: its first row, the positions that it had, and both scales
struct Regrown
{
    int row, n;
    float before, after;
};

// The older codes of `count` blocks of `groups` 16s of positions again under their larger scales, of(i) the i-th: thread
// `at` of `step`, four 16-byte pieces on their way together. Of values, only the bytes of those positions are written.
template <typename Of>
__device__ __forceinline__ void requantize(int8_t* pool, int count, int groups, int dk, bool keys, int at, int step, Of&& of)
{
    constexpr int U = 4;
    const int per = groups * dk;
    for (int i0 = at; i0 < count * per; i0 += U * step)
    {
        u32x4 x[U];
        int live[U];
        u32x4* to[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int i = i0 + u * step;
            live[u] = 0;
            if (i >= count * per) continue;
            const Regrown r = of(i / per);
            const int piece = i % per, first = piece / dk * 16;  // position of the piece's group
            live[u] = keys ? (first + (piece & 15) < r.n ? 16 : 0) : min(16, r.n - first);
            to[u] = reinterpret_cast<u32x4*>(pool + ((size_t)r.row >> 4) * (size_t)(16 * dk)) + piece;
            if (live[u] > 0) x[u] = *to[u];
        }
#pragma unroll 1
        for (int u = 0; u < U; ++u)
        {
            // (one body for the four: the code is fetched once)
            u32x4 y = u == 0 ? x[0] : u == 1 ? x[1] : u == 2 ? x[2] : x[3];
            const int n = u == 0 ? live[0] : u == 1 ? live[1] : u == 2 ? live[2] : live[3];
            u32x4* const out = u == 0 ? to[0] : u == 1 ? to[1] : u == 2 ? to[2] : to[3];
            if (n <= 0) continue;
            const Regrown r = of((i0 + u * step) / per);
#pragma unroll
            for (int w = 0; w < 4; ++w)
            {
                uint32_t z = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    const int c = (int8_t)(y[w] >> (8 * e));
                    z |= (uint32_t)(uint8_t)quantize_one(__fmul_rn((float)c, r.before), r.after) << (8 * e);
                }
                y[w] = z;
            }
            if (n == 16) *out = y;
            else
                for (int e = 0; e < n; ++e)
                    reinterpret_cast<int8_t*>(out)[e] = (int8_t)((e < 8 ? (e < 4 ? y[0] : y[1]) : (e < 12 ? y[2] : y[3])) >> (8 * (e & 3)));
        }
    }
}

// ------------------------------------------------------------------ fill from packed prompts

constexpr int kFillThreads = 512;  // of a work-group that takes 64 columns

struct FillI8Args
{
    const float* k;
    const float* v;
    const int32_t* cu;
    const int32_t* pos0;
    const float* cosT;
    const float* sinT;
    PoolsI8 pools;
    const int32_t* table;
    int M, B, Hkv, shift, table_stride, num_pages, limit;  // limit: positions from here on are not written
};

// Work-group = (64 columns, KV head, keys or values) and the blocks whose first token of this call lies in them, the
// last of which may end up to 63 columns further: each block's largest value is known to one work-group, and every
// element is read once. Lane = column, wave = an eighth of the dimension pairs (j, j + dk / 2); the values stay in
// registers between the search for the blocks' maxima and their codes. Values go through LDS as bytes, up to 16 positions of
// a dimension at a time. For few tokens of each of many sequences: bound by latency, so by eight waves (16 x 1 .. 8 tokens of 5
// heads of 128: 8.2 us).
// Tokens of no sequence, positions outside the table or the rope tables and pages outside the pool are not written.
template <int DK>
__global__ __launch_bounds__(kFillThreads) void k_pages_fill_i8(FillI8Args a)
{
    constexpr int HALF = DK / 2, NP = DK / 16;  // pairs of a thread
    constexpr int kCols = 2 * kPfTok, kPitch = kCols + 4;
    __shared__ uint32_t top_s[kPfTok];   // by the block's first column: its largest magnitude (bits)
    __shared__ int row_s[kCols];         // row of a column's token, -1 if it is not this work-group's
    __shared__ uint8_t head_s[kCols], run_s[kCols];  // columns that begin a group of 16 positions, in order, and the group's
    __shared__ Regrown grown_s[kPfTok];  // blocks whose scale has grown
    __shared__ __align__(16) uint8_t code_s[DK * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = blockIdx.y;
    const bool keys = blockIdx.z == 0;
    const int m0 = blockIdx.x * kPfTok, block = 1 << a.pools.bshift;
    if (tid < kPfTok) top_s[tid] = 0u;

    // the lane's column and the one 64 further, which is part of this work-group where the last block goes on there
    int pos[2], row[2] = {-1, -1}, first[2] = {-1, -1}, older[2] = {0, 0};
    const int b = wave_sequence(a.cu, a.B, a.M, m0, lane);
    pos[0] = b < 0 ? -1 : packed_position(a.cu, a.pos0, b, m0 + lane, a.limit);
    if (pos[0] >= 0)
    {
        const int cu0 = a.cu[b], head = block_column(m0 + lane, cu0, pos[0], block);
        if (head < m0) pos[0] = -1;
        else
        {
            first[0] = head - m0;
            older[0] = (pos[0] & (block - 1)) - (m0 + lane - head);  // positions of the block before the call's
        }
    }
    const int b_last = __builtin_amdgcn_readlane(b, 63), pos_last = __builtin_amdgcn_readlane(pos[0], 63);
    int more = 0;
    if (b_last >= 0 && pos_last >= 0)
    {
        const int left = block - 1 - (pos_last & (block - 1));  // of the block, behind column 63
        more = min(min(left, a.limit - 1 - pos_last), min(a.cu[b_last + 1], a.M) - (m0 + kPfTok));
    }
    pos[1] = lane < more ? pos_last + 1 + lane : -1;
    first[1] = __builtin_amdgcn_readlane(first[0], 63);
    older[1] = __builtin_amdgcn_readlane(older[0], 63);
    const bool any[2] = {true, more > 0};

    const float* const src = (keys ? a.k : a.v) + (size_t)(g * DK + w * NP) * (size_t)a.M;
    float x[2][2][NP];
    auto load = [&](int e) {
        const int m = min(m0 + kPfTok * e + lane, a.M - 1);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < NP; ++i) x[e][q][i] = src[(size_t)(HALF * q + i) * (size_t)a.M + (size_t)m];
    };
    load(0);
    if (any[1]) load(1);
    float s_old[2] = {0.0f, 0.0f};
    float* const scales = keys ? a.pools.ks : a.pools.vs;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (pos[e] >= 0)
        {
            const int id = a.table[(size_t)(e ? b_last : b) * a.table_stride + (pos[e] >> a.shift)];
            if (page_ok(id, a.num_pages)) row[e] = (int)page_row(id, g, pos[e] & ((1 << a.shift) - 1), a.Hkv, a.shift);
            if (row[e] >= 0 && older[e] > 0) s_old[e] = scales[row[e] >> a.pools.bshift];
        }
    v4fu cs[2][NP / 4], sn[2][NP / 4];
    const bool turn = keys && a.cosT;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (turn && any[e])
#pragma unroll
            for (int i = 0; i < NP / 4; ++i)
            {
                const size_t at = (size_t)max(pos[e], 0) * HALF + (size_t)(w * NP + 4 * i);
                cs[e][i] = *reinterpret_cast<const v4fu*>(a.cosT + at);
                sn[e][i] = *reinterpret_cast<const v4fu*>(a.sinT + at);
            }
    __syncthreads();  // top_s is clear
    float top[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 2; ++e)
    {
        if (!any[e]) break;
        if (turn)
#pragma unroll
            for (int i = 0; i < NP; ++i) pg_rope(x[e][0][i], x[e][1][i], cs[e][i / 4][i & 3], sn[e][i / 4][i & 3], x[e][0][i], x[e][1][i]);
#pragma unroll
        for (int i = 0; i < NP; ++i) top[e] = fmaxf(top[e], fmaxf(fabsf(x[e][0][i]), fabsf(x[e][1][i])));
        if (row[e] >= 0) atomicMax(&top_s[first[e]], __builtin_bit_cast(uint32_t, top[e]));
        if (w == 0) row_s[kPfTok * e + lane] = row[e];
    }
    if (!any[1] && w == 0) row_s[kPfTok + lane] = -1;
    __syncthreads();
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (row[e] >= 0)
        {
            s[e] = __fmul_rn(__builtin_bit_cast(float, top_s[first[e]]), 1.0f / 127.0f);
            if (older[e] > 0) s[e] = joined_scale(s[e], s_old[e]);
            if (w == 0 && kPfTok * e + lane == first[e]) scales[row[e] >> a.pools.bshift] = s[e];
        }
    int8_t* const pool = keys ? a.pools.k : a.pools.v;

    // ---- older codes of blocks whose scale has grown (each has its first token of this call in the first 64 columns)
    const bool regrown = row[0] >= 0 && first[0] == lane && older[0] > 0 && s[0] > s_old[0];
    const unsigned long long grown = __builtin_amdgcn_ballot_w64(regrown);
    if (grown != 0)
    {
        if (w == 0 && regrown)
            grown_s[__builtin_popcountll(grown & ((1ull << lane) - 1))] = Regrown{row[0] - older[0], older[0], s_old[0], s[0]};
        __syncthreads();
        requantize(pool, __builtin_popcountll(grown), block >> 4, DK, keys, tid, kFillThreads, [&](int i) { return grown_s[i]; });
    }

    // ---- codes: 4 of a quarter's dimensions in a word
    uint32_t code[2][2][NP / 4];
#pragma unroll
    for (int e = 0; e < 2; ++e)
    {
        if (!any[e]) break;
        const float r = quant_rcp(s[e]);
        bool amb = false;
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < NP; i += 4)
            {
                uint32_t y = 0;
#pragma unroll
                for (int n = 0; n < 4; ++n) y |= (uint32_t)(uint8_t)quantize_code(x[e][q][i + n], r, amb) << (8 * n);
                code[e][q][i / 4] = y;
            }
        if (amb && row[e] >= 0)
        {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < NP; i += 4)
                {
                    uint32_t y = 0;
#pragma unroll
                    for (int n = 0; n < 4; ++n) y |= (uint32_t)(uint8_t)quantize_one(x[e][q][i + n], s[e]) << (8 * n);
                    code[e][q][i / 4] = y;
                }
        }
    }
    if (keys)
    {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (any[e] && row[e] >= 0)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                {
                    typedef uint32_t Piece __attribute__((ext_vector_type(NP / 4)));
                    Piece y;
#pragma unroll
                    for (int i = 0; i < NP / 4; ++i) y[i] = code[e][q][i];
                    *reinterpret_cast<Piece*>(pool + key_byte((size_t)row[e], HALF * q + w * NP, DK)) = y;
                }
        return;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (any[e])
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    code_s[(HALF * q + w * NP + i) * kPitch + kPfTok * e + lane] = (uint8_t)(code[e][q][i / 4] >> (8 * (i & 3)));
    // the columns that begin a group of 16 positions and how many go on with it, found by every wave alike
    unsigned long long begins[2], stops[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
    {
        const int c = kPfTok * e + lane, before = c > 0 ? row_s[c - 1] : -1;
        const bool head = row[e] >= 0 && !(before >= 0 && before == row[e] - 1 && (row[e] & 15) != 0);
        begins[e] = __builtin_amdgcn_ballot_w64(head);
        stops[e] = begins[e] | __builtin_amdgcn_ballot_w64(row[e] < 0);
    }
    const int heads = __builtin_popcountll(begins[0]) + __builtin_popcountll(begins[1]);
    if (w == 0)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (begins[e] >> lane & 1)
            {
                const int i = __builtin_popcountll(begins[e] & ((1ull << lane) - 1)) + (e ? __builtin_popcountll(begins[0]) : 0);
                const unsigned long long own = lane < 63 ? stops[e] >> (lane + 1) : 0;
                int n = own ? __builtin_ctzll(own) + 1 : 64 - lane;
                if (!own && e == 0) n += stops[1] ? __builtin_ctzll(stops[1]) : 64;
                head_s[i] = (uint8_t)(kPfTok * e + lane);
                run_s[i] = (uint8_t)n;
            }
    __syncthreads();
#pragma unroll 2
    for (int i = tid; i < heads * DK; i += kFillThreads)
    {
        const int h = i / DK, d = i % DK, c = head_s[h], n = run_s[h];
        const uint8_t* const from = code_s + d * kPitch + c;
        int8_t* const to = pool + value_byte((size_t)row_s[c], d, DK);
        if (n == 16)
        {
            u32x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[e] = from[4 * e] | (uint32_t)from[4 * e + 1] << 8 | (uint32_t)from[4 * e + 2] << 16 | (uint32_t)from[4 * e + 3] << 24;
            *reinterpret_cast<u32x4*>(to) = y;
        }
        else
            for (int e = 0; e < n; ++e) to[e] = (int8_t)from[e];
    }
}

// The window of 64 positions with number `item` of a call, in the order of the sequences: sequence b (-1: none is left), its
// first position of the window, its column and position of the first token, its tokens that have a place.
struct FillWindow
{
    int b, from, col0, pos0, n;
};

__device__ __forceinline__ FillWindow find_window(const FillI8Args& a, int item)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave)
    {
        const int b = b0 + lane;
        int col0 = 0, p0 = 0, n = 0;
        if (b < a.B)
        {
            col0 = a.cu[b];
            const int64_t end = min(a.cu[b + 1], a.M);
            p0 = a.pos0 ? a.pos0[b] : 0;
            if (col0 >= 0 && p0 >= 0 && p0 < a.limit) n = (int)max((int64_t)0, min(end - col0, (int64_t)(a.limit - p0)));
        }
        const int windows = n > 0 ? ((p0 + n - 1) >> 6) - (p0 >> 6) + 1 : 0;
        int incl = windows;
        for (int off = 1; off < kWave; off <<= 1)
        {
            const int x = __shfl_up(incl, off, kWave);
            if (lane >= off) incl += x;
        }
        const unsigned long long here = __builtin_amdgcn_ballot_w64(before + incl > item);
        if (here != 0)
        {
            const int l = __builtin_ctzll(here);
            p0 = __builtin_amdgcn_readlane(p0, l);
            return {b0 + l, ((p0 >> 6) + item - before - __builtin_amdgcn_readlane(incl - windows, l)) << 6,
                    __builtin_amdgcn_readlane(col0, l), p0, __builtin_amdgcn_readlane(n, l)};
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return {-1, 0, 0, 0, 0};
}

// The same for long prompts: work-group = (window of 64 positions of a sequence, KV head, keys or values), lane = position. A
// window holds whole blocks and groups, so maxima are those of neighbouring lanes, and the values' bytes are
// turned 4 x 4 between the lanes of a quad, which leaves words of 4 positions for LDS. 16 x 1111 .. 2048 tokens of 5 heads of
// 128: 51 us, 3.1 TB/s, where a copy's 32 us are the floor. A lane takes one column, so rows are read in runs of 256 bytes that
// begin anywhere; and the work-groups past the last window lie on the last XCDs, with nothing to do there (a quarter of them at
// 16 x 300 tokens, 14.2 us, half at 64 x 128, 24.4).
template <int DK>
__global__ __launch_bounds__(256, DK == 256 ? 3 : 5) void k_windows_fill_i8(FillI8Args a)
{
    constexpr int HALF = DK / 2, NP = DK / 8;  // pairs of a thread
    constexpr int kPitch = 80;                 // bytes of a dimension's 64 positions in LDS
    __shared__ float top_s[4][4];
    __shared__ __align__(16) uint8_t code_s[DK * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = blockIdx.y;
    const bool keys = blockIdx.z == 0;
    const FillWindow at = find_window(a, xcd_run(blockIdx.x, gridDim.x));
    if (at.b < 0) return;
    const int pos = at.from + lane, block = 1 << a.pools.bshift, end = at.pos0 + at.n;
    const bool in = pos >= at.pos0 && pos < end;
    const int seen = min(max(pos, at.pos0), end - 1);  // (lanes without a token read another's)
    const float* const src = (keys ? a.k : a.v) + (size_t)(g * DK + w * NP) * (size_t)a.M + (size_t)(at.col0 + seen - at.pos0);
    float x[2][NP];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < NP; ++i) x[q][i] = src[(size_t)(HALF * q + i) * (size_t)a.M];
    const bool turn = keys && a.cosT;
    v4fu cs[NP / 4], sn[NP / 4];
    if (turn)
#pragma unroll
        for (int i = 0; i < NP / 4; ++i)
        {
            const size_t r = (size_t)seen * HALF + (size_t)(w * NP + 4 * i);
            cs[i] = *reinterpret_cast<const v4fu*>(a.cosT + r);
            sn[i] = *reinterpret_cast<const v4fu*>(a.sinT + r);
        }
    // the lane's row: of a block that has older positions, of those, too
    const int start = pos & -block;  // of the lane's block
    const bool held = pos < end && start + block > at.pos0;  // the block has a token of the call, or may have
    int row = -1;
    if (pos < end)
    {
        const int id = a.table[(size_t)at.b * a.table_stride + (pos >> a.shift)];
        if (page_ok(id, a.num_pages)) row = (int)page_row(id, g, pos & ((1 << a.shift) - 1), a.Hkv, a.shift);
    }
    const bool goes_on = held && row >= 0 && start < at.pos0;
    float* const scales = keys ? a.pools.ks : a.pools.vs;
    const float s_old = goes_on ? scales[row >> a.pools.bshift] : 0.0f;
    if (turn)
#pragma unroll
        for (int i = 0; i < NP; ++i) pg_rope(x[0][i], x[1][i], cs[i / 4][i & 3], sn[i / 4][i & 3], x[0][i], x[1][i]);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) top = fmaxf(top, fmaxf(fabsf(x[0][i]), fabsf(x[1][i])));
    if (!in) top = 0.0f;
    top = fmaxf(top, dpp<kDppXor1>(top));
    top = fmaxf(top, dpp<kDppXor2>(top));
    top = fmaxf(top, dpp<kDppHalfMirror>(top));
    top = fmaxf(top, dpp<kDppMirror>(top));
    if (block > 16) top = fmaxf(top, __shfl_xor(top, 16, kWave));
    if (block > 32) top = fmaxf(top, __shfl_xor(top, 32, kWave));
    if ((lane & 15) == 0) top_s[w][lane >> 4] = top;
    __syncthreads();
    top = fmaxf(fmaxf(top_s[0][lane >> 4], top_s[1][lane >> 4]), fmaxf(top_s[2][lane >> 4], top_s[3][lane >> 4]));
    float s = __fmul_rn(top, 1.0f / 127.0f);
    if (goes_on) s = joined_scale(s, s_old);
    const bool begins = in && row >= 0 && (pos == at.pos0 || pos == start);  // the block's first token of the call
    if (w == 0 && begins) scales[row >> a.pools.bshift] = s;
    int8_t* const pool = keys ? a.pools.k : a.pools.v;
    // older codes, of the block that the sequence goes on with
    const unsigned long long grown = __builtin_amdgcn_ballot_w64(begins && goes_on && s > s_old);
    if (grown != 0)
    {
        const int l = __builtin_ctzll(grown), n = at.pos0 & (block - 1);
        const Regrown r{__builtin_amdgcn_readlane(row, l) - n, n, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s_old), l)),
                        __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), l))};
        requantize(pool, 1, (n + 15) >> 4, DK, keys, tid, 256, [&](int) { return r; });
    }
    const float rcp = quant_rcp(s);
    uint32_t code[2][NP / 4];
    bool amb = false;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < NP; i += 4)
        {
            uint32_t y = 0;
#pragma unroll
            for (int n = 0; n < 4; ++n) y |= (uint32_t)(uint8_t)quantize_code(x[q][i + n], rcp, amb) << (8 * n);
            code[q][i / 4] = y;
        }
    if (amb && in)
    {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < NP; i += 4)
            {
                uint32_t y = 0;
#pragma unroll
                for (int n = 0; n < 4; ++n) y |= (uint32_t)(uint8_t)quantize_one(x[q][i + n], s) << (8 * n);
                code[q][i / 4] = y;
            }
    }
    if (keys)
    {
        if (in && row >= 0)
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < NP; i += NP < 16 ? NP : 16)
                {
                    int8_t* const to = pool + key_byte((size_t)row, HALF * q + w * NP + i, DK);
                    if constexpr (NP < 16) *reinterpret_cast<uint2*>(to) = make_uint2(code[q][0], code[q][1]);
                    else
                        *reinterpret_cast<u32x4*>(to) = u32x4{code[q][i / 4], code[q][i / 4 + 1], code[q][i / 4 + 2], code[q][i / 4 + 3]};
                }
        return;
    }
    const uint32_t sel1 = lane & 1 ? 0x03070105u : 0x06020400u, sel2 = lane & 2 ? 0x03020706u : 0x05040100u;
    auto exchanged = [](uint32_t x, auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xF, 0xF, true); };
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < NP / 4; ++i)
        {
            uint32_t y = code[q][i];
            y = __builtin_amdgcn_perm(exchanged(y, std::integral_constant<int, kDppXor1>{}), y, sel1);
            y = __builtin_amdgcn_perm(exchanged(y, std::integral_constant<int, kDppXor2>{}), y, sel2);
            // dimension 4 i + lane % 4 of the quad's positions
            *reinterpret_cast<uint32_t*>(code_s + (HALF * q + w * NP + 4 * i + (lane & 3)) * kPitch + (lane & ~3)) = y;
        }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < 4 * DK; i += 256)
    {
        const int d = i % DK, group = i / DK;  // (a wave's pieces are of one group)
        const int first = max(at.pos0 - at.from - 16 * group, 0), n = min(end - at.from - 16 * group, 16);
        // the row of the group's last position, which has a place if any of its positions has
        const int r = __shfl(row, 16 * group + max(min(n, 16), 1) - 1, kWave);
        if (first >= n || r < 0) continue;
        const u32x4 y = *reinterpret_cast<const u32x4*>(code_s + d * kPitch + 16 * group);
        int8_t* const to = pool + value_byte((size_t)(r & ~15), d, DK);
        if (n - first == 16) *reinterpret_cast<u32x4*>(to) = y;
        else
            for (int e = first; e < n; ++e) to[e] = (int8_t)((e < 8 ? (e < 4 ? y[0] : y[1]) : (e < 12 ? y[2] : y[3])) >> (8 * (e & 3)));
    }
}

// ------------------------------------------------------------------ values read back

constexpr int kReadCols = 256;

struct ReadI8Args
{
    PoolsI8 pools;
    const int32_t* table;
    const int32_t* cu;
    const int32_t* pos0;
    float* k;
    float* v;
    int M, B, Hkv, shift, table_stride, num_pages, limit;
    int parts;  // work-groups that share a head's dimensions
};

// Work-group = (256 columns, KV head and `parts`-th of its dimensions, keys or values), wave = 64 columns, lane = column,
// 16 dimensions at a time: of keys, the column's piece of them; of values, the pieces (16 positions of a dimension) of the
// groups that the columns lie in, 8 groups at a time, turned through LDS. (Codes of values taken from the pool one by one, or in words of four columns,
// are bound by the addresses: 47 and 39 us at 16 x 1111 .. 2048 tokens, 16 x 28 .. 35 tokens 17.) code * scale is one
// rounded product. Bound by the f32 columns that it writes: 16 x 1111 .. 2048 tokens of 5 heads of 128 30 us, 5.4 TB/s.
template <int DK>
__global__ __launch_bounds__(256) void k_pages_read_i8(ReadI8Args a)
{
    constexpr int kPiece = 16, kGroup = 16 * kPiece + 16;  // bytes of a piece and of a group's 16 in LDS
    __shared__ __align__(16) uint8_t piece_s[4][8 * kGroup];
    __shared__ int group_s[4][64];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = blockIdx.y / a.parts, part = blockIdx.y - g * a.parts, d0 = part * (DK / a.parts), d1 = d0 + DK / a.parts;
    const bool keys = blockIdx.z == 0;
    const int m0 = (xcd_run(blockIdx.x, gridDim.x) * 4 + w) * kPfTok, m = m0 + lane;
    if (m0 >= a.M) return;
    const int b = wave_sequence(a.cu, a.B, a.M, m0, lane);
    const int pos = b < 0 ? -1 : packed_position(a.cu, a.pos0, b, m, a.limit);
    int row = 0;
    float s = __builtin_nanf("");  // a position that has no place
    if (pos >= 0)
    {
        const int id = a.table[(size_t)b * a.table_stride + (pos >> a.shift)];
        if (page_ok(id, a.num_pages))
        {
            row = (int)page_row(id, g, pos & ((1 << a.shift) - 1), a.Hkv, a.shift);
            s = (keys ? a.pools.ks : a.pools.vs)[row >> a.pools.bshift];
        }
    }
    float* const out = (keys ? a.k : a.v) + (size_t)(g * DK) * (size_t)a.M + (size_t)m;
    if (keys)
    {
        const u32x4* const from = reinterpret_cast<const u32x4*>(a.pools.k + key_byte((size_t)row, 0, DK));
        u32x4 x = from[d0];  // (256 bytes, 16 pieces, from one 16 dimensions to the next)
#pragma unroll 1
        for (int d = d0; d < d1; d += 16)
        {
            const u32x4 y = x;
            if (d + 16 < d1) x = from[d + 16];
            if (b >= 0)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    out[(size_t)(d + i) * (size_t)a.M] = __fmul_rn((float)(int8_t)(y[i / 4] >> (8 * (i & 3))), s);
        }
        return;
    }
    // the groups of the wave's columns: a column begins one where the one before lies in another
    const int own = row >> 4;
    const int before = __shfl_up(own, 1, kWave);  // (every lane takes part: lane 1 reads lane 0's)
    const bool head = lane == 0 || before != own;
    const unsigned long long heads = __builtin_amdgcn_ballot_w64(head);
    const int at = __builtin_popcountll(heads & ((2ull << lane) - 1)) - 1, n = __builtin_popcountll(heads);
    if (head) group_s[w][at] = own;
    wave_lds_fence();
#pragma unroll 1
    for (int first = 0; first < n; first += 8)
    {
        const u32x4* from[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            from[u] = reinterpret_cast<const u32x4*>(a.pools.v) + (size_t)group_s[w][min(first + 4 * u + (lane >> 4), n - 1)] * DK + (lane & 15);
        const bool mine = at >= first && at < first + 8 && b >= 0;
        const uint8_t* const code = piece_s[w] + (mine ? (at - first) * kGroup + (row & 15) : 0);
        uint8_t* const to = piece_s[w] + (lane >> 4) * kGroup + (lane & 15) * kPiece;
        u32x4 x[2] = {from[0][d0], from[1][d0]};
#pragma unroll 1
        for (int d = d0; d < d1; d += 16)
        {
            *reinterpret_cast<u32x4*>(to) = x[0];
            *reinterpret_cast<u32x4*>(to + 4 * kGroup) = x[1];
            if (d + 16 < d1) x[0] = from[0][d + 16], x[1] = from[1][d + 16];
            wave_lds_fence();
            int8_t c[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) c[i] = (int8_t)code[i * kPiece];
            wave_lds_fence();
            if (mine)
#pragma unroll
                for (int i = 0; i < 16; ++i) out[(size_t)(d + i) * (size_t)a.M] = __fmul_rn((float)c[i], s);
        }
    }
}

// ------------------------------------------------------------------ attention of one new token per sequence

// What the append of a token has left: the scales of its block, and whether older codes have changed
struct Appended
{
    float s[2];
    bool regrown;
};

// The new token of a sequence, by one wave: its rotated key and its value of KV head g at position p. begin() gets its elements
// (element i at k[i * step]) and its block's scales on their way; end() writes it to its page (row `row`, -1: a page outside
// the pool, and nothing is written), and its codes, keys' and values', to LDS.
template <int DK>
struct Append
{
    static constexpr int HALF = DK / 2, N = (HALF + 63) / 64;
    float x[2][2][N], cs[N], sn[N], s_old[2];  // keys, values; the halves
    __device__ __forceinline__ void begin(const PoolsI8& pools, const float* k, const float* v, size_t step, const float* cosT,
                                          const float* sinT, int p, int row)
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
            const int i = min(lane + 64 * n, HALF - 1);
            x[0][0][n] = k[i * step], x[0][1][n] = k[(i + HALF) * step];
            x[1][0][n] = v[i * step], x[1][1][n] = v[(i + HALF) * step];
            if (cosT) cs[n] = cosT[(size_t)p * HALF + (size_t)i], sn[n] = sinT[(size_t)p * HALF + (size_t)i];
        }
        const bool goes_on = row >= 0 && (p & ((1 << pools.bshift) - 1)) != 0;
        s_old[0] = goes_on ? pools.ks[row >> pools.bshift] : 0.0f;
        s_old[1] = goes_on ? pools.vs[row >> pools.bshift] : 0.0f;
    }
    __device__ __forceinline__ Appended end(const PoolsI8& pools, bool turn, int p, int row, uint8_t (*codes)[DK])
    {
        const int lane = threadIdx.x & 63, into = p & ((1 << pools.bshift) - 1);
        if (turn)
#pragma unroll
            for (int n = 0; n < N; ++n) pg_rope(x[0][0][n], x[0][1][n], cs[n], sn[n], x[0][0][n], x[0][1][n]);
        Appended got{{0.0f, 0.0f}, false};
#pragma unroll 1
        for (int q = 0; q < 2; ++q)
        {
            float y[2][N];
            float top = 0.0f;
#pragma unroll
            for (int n = 0; n < N; ++n)
            {
                y[0][n] = q ? x[1][0][n] : x[0][0][n], y[1][n] = q ? x[1][1][n] : x[0][1][n];
                top = fmaxf(top, fmaxf(fabsf(y[0][n]), fabsf(y[1][n])));
            }
            const uint32_t bits = wave_max(__builtin_bit_cast(uint32_t, top));
            const float before = q ? s_old[1] : s_old[0];
            float s = __fmul_rn(__builtin_bit_cast(float, bits), 1.0f / 127.0f);
            if (into > 0) s = joined_scale(s, before);
            (q ? got.s[1] : got.s[0]) = s;
            int8_t* const pool = q ? pools.v : pools.k;
            if (row >= 0 && into > 0 && s > before)
            {
                got.regrown = true;
                requantize(pool, 1, (into + 15) >> 4, DK, q == 0, lane, 64, [&](int) { return Regrown{row - into, into, before, s}; });
            }
            if (row >= 0 && lane == 0 && (into == 0 || s > before)) (q ? pools.vs : pools.ks)[row >> pools.bshift] = s;
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (lane + 64 * n < HALF)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
                        const int d = lane + 64 * n + HALF * h;
                        const int8_t c = (int8_t)quantize_one(y[h][n], s);
                        if (row >= 0) pool[q ? value_byte((size_t)row, d, DK) : key_byte((size_t)row, d, DK)] = c;
                        codes[q][d] = (uint8_t)c;
                    }
        }
        return got;
    }
};

// The append by itself, for calls whose attention reads a KV head by more than one work-group a chunk
template <int DK>
__global__ __launch_bounds__(64) void k_pages_append_i8(PagesArgs a, PoolsI8 pools)
{
    __shared__ uint8_t codes[2][DK];
    const int g = blockIdx.x, b = blockIdx.y, p = a.pos[b];
    if (p < 0 || p >= a.len_bound) return;
    const size_t at = a.tokens ? ((size_t)b * a.Hkv + g) * DK : (size_t)g * DK * a.B + b;
    const int id = a.table[(size_t)b * a.table_stride + (p >> a.shift)];
    const int row = page_ok(id, a.num_pages) ? (int)page_row(id, g, p & ((1 << a.shift) - 1), a.Hkv, a.shift) : -1;
    Append<DK> append;
    append.begin(pools, a.k + at, a.v + at, a.tokens ? 1 : (size_t)a.B, a.cosT, a.sinT, p, row);
    append.end(pools, a.cosT != nullptr, p, row, codes);
}

constexpr int kI8Tile = 64;       // positions of a wave's tile
constexpr float kI8Room = 4.0f;   // log2 units between a new reference maximum and the largest score
constexpr int kI8Pitch = 80;      // bytes of a row of weights' digits in LDS (64 positions)

// X as four signed base-256 digits, X = sum d_i 256^i, the bytes of the result (|X| < 2^31 - 2^23.01)
__device__ __forceinline__ uint32_t digits(uint32_t X) { return (X + 0x80808080u) ^ 0x80808080u; }

// The exponent field that scales a query whose largest element has these bits
__device__ __forceinline__ int query_field(uint32_t top) { return max((int)(top >> 23), 30); }

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_bits(uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}

__device__ __forceinline__ float pow2_field(int field) { return __builtin_bit_cast(float, (uint32_t)field << 23); }

// Attention of one new token per sequence: work-groups as k_pages_attn's (a chunk of positions of a sequence, a KV head
// and a group of at most 4 NS of its query heads; its W waves take the chunk's tiles in turn), records and join the
// same. Both products run on the int8 MFMA with the codes as they lie in the pools:
//   scores  a head's rotated query as 30-bit fixed point under its largest element, |X| < 2^30, in four
//           signed base-256 digits: rows 4 h + i of a 16 x 64 operand for four heads, against 16 positions' keys. Every
//           partial sum is exact in int32, and a lane finds the four digit sums of one head and position in its
//           registers; s = (256 a3 + a2) 2^16 + (256 a1 + a0) is rounded as an f32.
//   values  the weights of a tile, times their blocks' scales, as 30-bit fixed point under the head's largest such product (a power
//           of two above it) in the same digits, through LDS to the columns of an operand; the digits' sums over
//           the tile's 64 positions are exact, and each is added to an f32 sum of its own, joined at the end. (Under the
//           reference of the whole wave thousands of small weights beside a large one were lost, under the tile's largest
//           scale those beside a large value without weight.)
// So neither codes are converted nor multiplied by their scales one by one: 330 VALU instructions a tile of 64
// positions for 4 heads of 128 (counted at 8), where multiply-adds on widened elements would take 1300.
// A head's reference maximum moves when a score passes it, to 4 above that score (weights are 2^-4 at most then and
// 1 at most later).
// The chunk that holds the new position writes its key and value, by the wave that reads them (no other wave reads that
// block), and takes their codes into its operands from LDS: its tile is on its way meanwhile, and is read again only
// where the block's older codes have changed (16 x 64 .. 4200, alone: 21.7 us where no block's scale is raised, 40.0 where every one is).
// A block whose scale is not finite (its tokens had an infinity) stands for NaN, and so does a query with one.
// 6 x 50000 .. 131072 positions, 8 heads to each of 4 KV heads of 128: 101 us, 5.9 TB/s, bound by HBM; 16 x 64 .. 4200, 4 to each of
// 5: 12.0 us and 4.0 for the join, 1 x 100: 7.4, bound by the chain of round trips from position to page to rows to output.
// Heads of 256 go 4 at a time, for their registers: where a KV head has more, each 4 read all codes again, and the token is
// appended in a launch of its own (16 x 4000 .. 16000 over 1 KV head, 76 MB: 4 heads 33 us, 8 heads 47).
template <int DK, int NS, int W, bool kFinal>
__global__ __launch_bounds__(64 * W) void k_pages_attn_i8(PagesArgs a, PoolsI8 pools, int append)
{
    constexpr int HALF = DK / 2, RT = 4 * NS, KC = DK / 64, ND = DK / 16, T = 64 * W;
    constexpr int QI = (RT * HALF + T - 1) / T;  // query pairs per thread
    constexpr int kDigits = DK + 4;              // words of a head's digits in LDS
    __shared__ __align__(16) uint32_t dig_s[RT * kDigits];
    __shared__ uint32_t top_s[RT];               // each head's largest element (bits)
    __shared__ __align__(16) uint8_t w_s[W][NS][16 * kI8Pitch];
    __shared__ __align__(16) uint8_t new_s[2][DK];
    __shared__ float ml_s[2][W][RT];
    __shared__ __align__(16) float red_s[W][RT * DK];
    __shared__ int bad_s[W];

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, grp = lane >> 4;
    const int HG = a.Hkv * a.groups;
    const int gh = blockIdx.x % HG, item = blockIdx.x / HG;
    const int g = gh / a.groups, hg = gh - g * a.groups;
    if (tid < RT) top_s[tid] = 0u;
    const PagesItem it = !kFinal && a.even ? find_item(a, item)
                                           : PagesItem{item / a.nchunk, item % a.nchunk, a.chunk, item - item % a.nchunk,
                                                       a.pos[item / a.nchunk]};
    if (it.b < 0) return;
    const int b = it.b, c = it.c, p = it.p;
    const int h0 = g * a.R + hg * a.RG;        // first query head
    const int R = min(a.RG, a.R - hg * a.RG);  // query heads here (<= RT)
    const size_t io_step = a.tokens ? 1 : (size_t)a.B;
    float qx[QI][2];
#pragma unroll
    for (int u = 0; u < QI; ++u)
    {
        const int e = tid + u * T, r = min(e / HALF, R - 1), i = e % HALF;
        const float* q = a.q + (a.tokens ? ((size_t)b * a.H + h0 + r) * DK : (size_t)(h0 + r) * DK * a.B + b);
        qx[u][0] = q[i * io_step];
        qx[u][1] = q[(i + HALF) * io_step];
    }
    float* const out = a.out + (a.tokens ? ((size_t)b * a.H + h0) * DK : (size_t)h0 * DK * a.B + b);
    if (p < 0 || p >= a.len_bound)
    {
        // no token: zeros; a position past the bound: NaN
        if (c == 0)
            for (int e = tid; e < R * DK; e += T) out[e * io_step] = p < 0 ? 0.0f : __builtin_nanf("");
        return;
    }
    if (!kFinal && a.even && c == 0 && gh == 0 && tid == 0) a.places[b] = make_int2(it.first, it.chunk);
    const int t0 = c * it.chunk;
    if (t0 > p) return;
    const int last = min(p, t0 + it.chunk - 1);  // the chunk's last position

    // ---- the tiles: a lane looks up the page of group lane % 4 of 16 positions
    const int32_t* const table = a.table + (size_t)b * a.table_stride;
    const int slot_mask = (1 << a.shift) - 1;
    bool bad = false;
    int id;
    auto load_id = [&](int t) { id = table[min(t + 16 * (lane & 3), last) >> a.shift]; };
    u32x4 kf[4][KC], vf[ND];
    float ks = 0.0f, vs = 0.0f;
    auto load = [&](int t) {
        const int at = t + 16 * (lane & 3);
        const bool in = page_ok(id, a.num_pages);
        bad |= !in;
        // groups behind the last position read the last one's rows (their scores are -inf)
        const int row = (int)(page_row(in ? id : 0, g, min(at, last & ~15) & slot_mask, a.Hkv, a.shift) >> 4);
        ks = pools.ks[row >> (pools.bshift - 4)];
        vs = pools.vs[row >> (pools.bshift - 4)];
        if (at > last) ks = vs = 0.0f;
        load_id(t + W * kI8Tile);
#pragma unroll
        for (int n = 0; n < 4; ++n)
        {
            const u32x4* k = reinterpret_cast<const u32x4*>(pools.k + (size_t)__builtin_amdgcn_readlane(row, n) * (16 * DK)) + lane;
#pragma unroll
            for (int i = 0; i < KC; ++i) kf[n][i] = __builtin_nontemporal_load(k + 64 * i);
        }
        const u32x4* v = reinterpret_cast<const u32x4*>(pools.v + (size_t)__shfl(row, grp, kWave) * (16 * DK)) + j;
#pragma unroll
        for (int i = 0; i < ND; ++i) vf[i] = __builtin_nontemporal_load(v + 16 * i);
    };
    const int first = t0 + w * kI8Tile, new_tile = p & -kI8Tile;
    // whether this wave appends the token
    const bool own = append && p == last && first <= new_tile && (new_tile - first) % (W * kI8Tile) == 0;
    load_id(first);
    const int new_id = own ? table[p >> a.shift] : 0;
    float cs[QI], sn[QI];
    if (a.cosT)
#pragma unroll
        for (int u = 0; u < QI; ++u)
        {
            const size_t r = (size_t)p * HALF + (size_t)((tid + u * T) % HALF);
            cs[u] = a.cosT[r], sn[u] = a.sinT[r];
        }
    if (first <= last) load(first);  // on its way during the rest
    Append<DK> token;
    Appended done{{0.0f, 0.0f}, false};
    const int new_row = own && page_ok(new_id, a.num_pages) ? (int)page_row(new_id, g, p & slot_mask, a.Hkv, a.shift) : -1;
    if (own)
    {
        const size_t at = a.tokens ? ((size_t)b * a.Hkv + g) * DK : (size_t)g * DK * a.B + b;
        token.begin(pools, a.k + at, a.v + at, io_step, a.cosT, a.sinT, p, new_row);
    }

    // ---- rotated queries, as digits
    lds_barrier();  // top_s is clear
#pragma unroll
    for (int u = 0; u < QI; ++u)
    {
        const int r = (tid + u * T) / HALF;
        if (a.cosT) pg_rope(qx[u][0], qx[u][1], cs[u], sn[u], qx[u][0], qx[u][1]);
        uint32_t mx = max(__builtin_bit_cast(uint32_t, qx[u][0]) & 0x7FFFFFFFu, __builtin_bit_cast(uint32_t, qx[u][1]) & 0x7FFFFFFFu);
        mx = max(mx, dpp_bits<kDppXor1>(mx));
        mx = max(mx, dpp_bits<kDppXor2>(mx));
        mx = max(mx, dpp_bits<kDppHalfMirror>(mx));
        mx = max(mx, dpp_bits<kDppMirror>(mx));
        if (j == 0 && r < R) atomicMax(&top_s[r], mx);
    }
    lds_barrier();
#pragma unroll
    for (int u = 0; u < QI; ++u)
    {
        const int e = tid + u * T, r = e / HALF, i = e % HALF;
        if (r >= RT) continue;
        const float up = pow2_field(283 - query_field(top_s[r]));  // brings the largest below 2^30
        // (heads past R: 0)
        dig_s[r * kDigits + i] = r < R ? digits((uint32_t)(int)__builtin_rintf(qx[u][0] * up)) : 0u;
        dig_s[r * kDigits + i + HALF] = r < R ? digits((uint32_t)(int)__builtin_rintf(qx[u][1] * up)) : 0u;
    }
    lds_barrier();
    u32x4 qd[NS][KC];
    float unit[NS], slope2[NS];  // of head 4 s + lane / 16
    // (a product past f32's range would make a score of 0 NaN; any other score is past the cap, or the range, with the
    // largest float, too)
    auto held = [](float x) { return fminf(fmaxf(x, -3.40282347e38f), 3.40282347e38f); };
    const uint32_t sel = (uint32_t)(j & 3) | (uint32_t)((j & 3) + 4) << 8;
#pragma unroll
    for (int s = 0; s < NS; ++s)
    {
        const uint32_t* const q = dig_s + (4 * s + (j >> 2)) * kDigits + 16 * grp;
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n)
            {
                const u32x4 x = *reinterpret_cast<const u32x4*>(q + 64 * i + 4 * n);
                qd[s][i][n] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(x[3], x[2], sel), __builtin_amdgcn_perm(x[1], x[0], sel), 0x05040100u);
            }
        const uint32_t mx = top_s[4 * s + grp];
        const float to = (a.cap2 > 0.0f ? a.capi : a.scale2) * pow2_field(query_field(mx) - 29);
        unit[s] = mx >= 0x7F800000u ? __builtin_nanf("") : held(to);
        slope2[s] = a.slopes && 4 * s + grp < R ? a.slopes[h0 + 4 * s + grp] * 1.44269504f : 0.0f;
    }
    if (own) done = token.end(pools, a.cosT != nullptr, p, new_row, new_s);

    v4f acc[NS][ND];
    float m[NS], l[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s)
    {
        m[s] = -__builtin_inff(), l[s] = 0.0f;
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[s][i] = v4f{};
    }
    for (int t = first; t <= last; t += W * kI8Tile)
    {
        if (t != first) load(t);  // (the next tile's on its way during a tile was up to 4 % slower, its registers there or not)
        if (own && t == new_tile)
        {
            if (done.regrown)
            {
                __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
                load_id(t);
                load(t);
            }
            // the token's codes, and its block's scales
            wave_lds_fence();
            const int n_new = (p - t) >> 4, at = p & 15;
#pragma unroll
            for (int n = 0; n < 4; ++n)
                if (n == n_new && j == at)
#pragma unroll
                    for (int i = 0; i < KC; ++i) kf[n][i] = *reinterpret_cast<const u32x4*>(new_s[0] + 64 * i + 16 * grp);
            const uint32_t keep = ~(0xFFu << (8 * (at & 3)));
#pragma unroll
            for (int i = 0; i < ND; ++i)
            {
                const uint32_t x = (uint32_t)new_s[1][16 * i + j] << (8 * (at & 3));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (grp == n_new && e == at >> 2) vf[i][e] = (vf[i][e] & keep) | x;
            }
            const int mine = t + 16 * (lane & 3);
            if (mine >> pools.bshift == p >> pools.bshift && mine <= last) ks = done.s[0], vs = done.s[1];
        }
        // a power of two above the tile's largest scale of values
        float top_v = fmaxf(vs, dpp<kDppXor1>(vs));
        top_v = fmaxf(top_v, dpp<kDppXor2>(top_v));
        const bool odd = __builtin_amdgcn_ballot_w64(!(fabsf(vs) < 0x1p125f)) != 0;  // (no write makes one from there on)
        const int ev = min(max(__builtin_amdgcn_readfirstlane((int)(__builtin_bit_cast(uint32_t, top_v) >> 23)), 31), 252);
        const float down = odd ? 0.0f : pow2_field(253 - ev);                  // 2^(126 - ev) times a scale is at most 1
        float kg[4], vg[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
        {
            kg[n] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks), n));
            vg[n] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs), n)) * down;
        }
        const bool part = t + kI8Tile - 1 > last;
        float back[NS];  // of head 4 s + j / 4
#pragma unroll
        for (int s = 0; s < NS; ++s)
        {
            float x[4];
            float top = -__builtin_inff(), far = 0.0f;
#pragma unroll
            for (int n = 0; n < 4; ++n)
            {
                v4i d = v4i{};
#pragma unroll
                for (int i = 0; i < KC; ++i)
                    d = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, qd[s][i]), __builtin_bit_cast(v4i, kf[n][i]), d, 0, 0, 0);
                const int hi = (int)((uint32_t)d[3] << 8) + d[2], lo = (int)((uint32_t)d[1] << 8) + d[0];
                float f = unit[s] * kg[n];
                f = kg[n] < __builtin_inff() && f == f ? held(f) : __builtin_nanf("");
                x[n] = __builtin_fmaf((float)hi, 65536.0f, (float)lo) * f;
                far = fmaxf(far, fabsf(x[n]));
            }
            if (a.cap2 > 0.0f)
            {
                // scores rarely reach the cap: a few terms where none does (a NaN does not show, and stays one)
                const bool near = __builtin_amdgcn_ballot_w64(far > 0.25f) == 0;
#pragma unroll
                for (int n = 0; n < 4; ++n) x[n] = a.cap2 * (near ? tanh_below_quarter(x[n]) : tanh_any(x[n]));
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
            {
                const int at = t + 16 * n + j;
                if (a.slopes) x[n] = __builtin_fmaf(slope2[s], (float)(at - p), x[n]);
                if (part && at > last) x[n] = -__builtin_inff();
                top = fmaxf(top, x[n]);
            }
            top = fmaxf(top, dpp<kDppRor8>(top));
            top = fmaxf(top, dpp<kDppRor4>(top));
            top = fmaxf(top, dpp<kDppXor2>(top));
            top = fmaxf(top, dpp<kDppXor1>(top));
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > m[s]) != 0, 0))
            {
                const float to = top > m[s] ? top + kI8Room : m[s];
                float corr = m[s] == to ? 1.0f : __builtin_amdgcn_exp2f(m[s] - to);
                asm volatile("" : "+v"(corr));  // (or every product is computed whether the branch is taken or not)
                l[s] *= corr;
                m[s] = to;
                const float f = __shfl(corr, (j >> 2) * 16, kWave);
#pragma unroll
                for (int i = 0; i < ND; ++i) acc[s][i] *= f;
            }
            uint32_t most = 0;  // (bits, of products that are at least 0, or NaN)
#pragma unroll
            for (int n = 0; n < 4; ++n)
            {
                // no score above -inf yet: nothing to add (and no -inf - -inf)
                const float pr = x[n] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x[n] - m[s]);
                l[s] += pr;
                x[n] = pr * vg[n];
                most = max(most, __builtin_bit_cast(uint32_t, x[n]));
            }
            most = max(most, dpp_bits<kDppRor8>(most));
            most = max(most, dpp_bits<kDppRor4>(most));
            most = max(most, dpp_bits<kDppXor2>(most));
            most = max(most, dpp_bits<kDppXor1>(most));
            const int ew = min(max((int)(most >> 23), 29), 127);
            const float up = pow2_field(283 - ew);  // brings the largest below 2^30
            // 2^(ev - 126) 2^(ew - 126) 2^-30
            back[s] = __shfl(__builtin_ldexpf(1.0f, ew + ev - 282), (j >> 2) * 16, kWave);
            if (odd) back[s] = __builtin_nanf("");
            uint8_t* const to = w_s[w][s] + 4 * grp * kI8Pitch + j;
#pragma unroll
            for (int n = 0; n < 4; ++n)
            {
                const uint32_t d = digits((uint32_t)__builtin_fmaf(x[n], up, 0.5f));
#pragma unroll
                for (int i = 0; i < 4; ++i) to[i * kI8Pitch + 16 * n] = (uint8_t)(d >> (8 * i));
            }
        }
        wave_lds_fence();
#pragma unroll
        for (int s = 0; s < NS; ++s)
        {
            const v4i wd = *reinterpret_cast<const v4i*>(w_s[w][s] + j * kI8Pitch + 16 * grp);
#pragma unroll
            for (int i = 0; i < ND; ++i)
            {
                const v4i d = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, vf[i]), wd, v4i{}, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[s][i][e] = __builtin_fmaf((float)d[e], back[s], acc[s][i][e]);
            }
        }
        wave_lds_fence();
    }

    // ---- join of the waves
#pragma unroll
    for (int s = 0; s < NS; ++s)
    {
        l[s] += dpp<kDppRor8>(l[s]);
        l[s] += dpp<kDppRor4>(l[s]);
        l[s] += dpp<kDppXor2>(l[s]);
        l[s] += dpp<kDppXor1>(l[s]);
        if (j == 0) ml_s[0][w][4 * s + grp] = m[s], ml_s[1][w][4 * s + grp] = l[s];
    }
    const bool any_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) bad_s[w] = any_bad;
    lds_barrier();
    auto top_of = [&](int h) {
        float top = ml_s[0][0][h];
#pragma unroll
        for (int i = 1; i < W; ++i) top = fmaxf(top, ml_s[0][i][h]);
        return top;
    };
    const float digit = pow2_field(127 + 8 * (j & 3));
#pragma unroll
    for (int s = 0; s < NS; ++s)
    {
        const int h = 4 * s + (j >> 2);
        const float mine = ml_s[0][w][h], top = top_of(h);
        const float f = (mine == top ? 1.0f : __builtin_amdgcn_exp2f(mine - top)) * digit;
#pragma unroll
        for (int i = 0; i < ND; ++i)
        {
            v4f y = acc[s][i] * f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                y[e] += dpp<kDppXor1>(y[e]);
                y[e] += dpp<kDppXor2>(y[e]);
            }
            if ((i & 3) == (j & 3)) *reinterpret_cast<v4f*>(&red_s[w][h * DK + 16 * i + 4 * grp]) = y;
        }
    }
    lds_barrier();
    int lost = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) lost |= bad_s[i];
    float* const rec = a.part + ((size_t)(it.first + c) * HG + gh) * (size_t)(a.RG * DK + kPgRec);
    for (int e = tid; e < R * DK; e += T)
    {
        const int r = e / DK;
        const float top = top_of(r);
        float sum = 0.0f, y = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i)
        {
            sum += ml_s[1][i][r] * (ml_s[0][i][r] == top ? 1.0f : __builtin_amdgcn_exp2f(ml_s[0][i][r] - top));
            y += red_s[i][e];
        }
        if (lost) sum = __builtin_nanf("");
        if constexpr (kFinal) out[e * io_step] = sum == 0.0f ? 0.0f : y / sum;
        else
        {
            rec[e] = y;
            if (e % DK == 0)
            {
                rec[a.RG * DK + r] = top;
                rec[a.RG * DK + 8 + r] = sum;
            }
        }
    }
}

// A sequence by one work-group, up to so many positions: no records, and no join. Of eight waves from 256 positions on
// (four of dk = 256, whose tile takes half of a SIMD's registers). With the token read back, alone and split, us: 16 x 400 of
// 20 heads over 5 of 128 13.4 and 17.1, 16 x 900 17.5 and 19.1, 64 x 900 of 16 over 2 of 64 16.9 and 21.9, 16 x 1500 20.1 and 20.4,
// 16 x 2500 25.9 and 24.7, 1 x 2000 of 8 over 1 22 and 17. Of 256, which fall behind sooner where there are few: 16 x 400 of 8 over 1 18.9 and 20.4
// (eight waves 23.2), 16 x 1000 26.1 and 21.2, 64 x 1000 28.8 and 39.5.
constexpr size_t kI8Solo = 1024;

inline PagesCut cut_i8(size_t B, size_t Hkv, size_t R, size_t dk, size_t len_bound, size_t num_cus)
{
    const bool few = dk == 256 && 2 * B * Hkv * pages_groups(R, dk) < num_cus;
    return len_bound <= (few ? kI8Solo / 2 : kI8Solo) ? PagesCut{round_up(len_bound, kI8Tile), 1, 0} : pages_cut(B, Hkv, R, dk, len_bound, num_cus);
}

template <int DK, int NS>
hipError_t launch_attn_i8(hipStream_t st, const PagesArgs& a, const PoolsI8& pools)
{
    const bool alone = a.k && a.groups > 1;
    if (alone)
    {
        k_pages_append_i8<DK><<<dim3((unsigned)a.Hkv, (unsigned)a.B), 64, 0, st>>>(a, pools);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const int append = a.k && !alone;
    const dim3 grid((unsigned)(pages_items(a.B, a.len_bound, a.chunk, a.even) * a.Hkv * a.groups));
    if (a.nchunk == 1)
    {
        constexpr int W = DK == 256 ? 4 : 8;
        if (a.len_bound <= 4 * kI8Tile) k_pages_attn_i8<DK, NS, 4, true><<<grid, 256, 0, st>>>(a, pools, append);
        else k_pages_attn_i8<DK, NS, W, true><<<grid, 64 * W, 0, st>>>(a, pools, append);
        return hipGetLastError();
    }
    k_pages_attn_i8<DK, NS, 4, false><<<grid, 256, 0, st>>>(a, pools, append);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_pages_join<DK><<<dim3((unsigned)a.H, (unsigned)a.B), kPgThreads, 0, st>>>(a);
    return hipGetLastError();
}

PoolsI8 pools_of(const nnhip_kv_pages_i8& kv)
{
    return {static_cast<int8_t*>(kv.k), static_cast<int8_t*>(kv.v), kv.k_scale, kv.v_scale, log2_of(kv.block)};
}

}  // namespace

size_t pages_workspace_bytes_i8(size_t B, size_t H, size_t Hkv, size_t dk, size_t len_bound, size_t num_cus)
{
    const size_t R = H / Hkv, groups = pages_groups(R, dk);
    const PagesCut cut = cut_i8(B, Hkv, R, dk, len_bound, num_cus);
    if (cut.nchunk == 1) return 0;
    return pages_records(B, Hkv, groups, ceil_div(R, groups), dk, len_bound, cut) * sizeof(float) + (cut.even ? B * sizeof(int2) : 0);
}

hipError_t launch_pages_attn_i8(hipStream_t st, const nnhip_kv_pages_i8& kv, const float* q, const float* k, const float* v,
                                size_t B, size_t H, const int32_t* pos, size_t len_bound, const float* cosT,
                                const float* sinT, float scale, float softcap, const float* slopes, bool tokens,
                                float* part, float* out, size_t num_cus)
{
    constexpr double kLog2e = 1.4426950408889634;
    const size_t R = H / kv.Hkv, dk = kv.dk, groups = pages_groups(R, dk);
    const PagesCut cut = cut_i8(B, kv.Hkv, R, dk, len_bound, num_cus);
    const bool cap = softcap > 0.0f;
    PagesArgs a{q, k, v, pos, cosT, sinT, kv.k, kv.v, kv.table, slopes, part,
                reinterpret_cast<int2*>(part + (cut.even ? pages_records(B, kv.Hkv, groups, ceil_div(R, groups), dk, len_bound, cut) : 0)),
                out, (int)B, (int)H, (int)kv.Hkv, (int)R,
                (int)groups, (int)ceil_div(R, groups), log2_of(kv.page_size), (int)kv.table_stride, (int)kv.num_pages,
                (int)len_bound, (int)cut.chunk, (int)cut.nchunk, (int)cut.even, (float)(scale * kLog2e),
                cap ? scale / softcap : 0.0f, cap ? (float)(softcap * kLog2e) : 0.0f, tokens ? 1 : 0};
    const PoolsI8 pools = pools_of(kv);
    if (dk == 256) return launch_attn_i8<256, 1>(st, a, pools);
    if (dk == 128) return a.RG <= 4 ? launch_attn_i8<128, 1>(st, a, pools) : launch_attn_i8<128, 2>(st, a, pools);
    if (dk == 64) return a.RG <= 4 ? launch_attn_i8<64, 1>(st, a, pools) : launch_attn_i8<64, 2>(st, a, pools);
    return hipErrorInvalidValue;
}

hipError_t launch_pages_fill_i8(hipStream_t st, const nnhip_kv_pages_i8& kv, const float* k, const float* v, size_t M,
                                const int32_t* cu, const int32_t* pos0, size_t B, const float* cosT, const float* sinT,
                                size_t limit)
{
    const FillI8Args a{k, v, cu, pos0, cosT, sinT, pools_of(kv), kv.table, (int)M, (int)B, (int)kv.Hkv, log2_of(kv.page_size),
                       (int)kv.table_stride, (int)kv.num_pages, (int)limit};
    // sequences of 128 tokens or more on average (the lengths are on the device: one long prompt among many short ones goes by
    // columns): windows of their positions, of which there are at most M / 64 + 2 B (by
    // windows and by columns, with the values read back, us: 16 x 64 tokens of 5 heads of 128 15.0 and 13.4, x 128 18.9 and 18.5, x 300 22.7 and 27.8)
    if (M >= 2 * kPfTok * B)
    {
        const dim3 grid((unsigned)(M / kPfTok + 2 * B), (unsigned)kv.Hkv, 2);
        if (kv.dk == 64) k_windows_fill_i8<64><<<grid, 256, 0, st>>>(a);
        else if (kv.dk == 128) k_windows_fill_i8<128><<<grid, 256, 0, st>>>(a);
        else if (kv.dk == 256) k_windows_fill_i8<256><<<grid, 256, 0, st>>>(a);
        else return hipErrorInvalidValue;
        return hipGetLastError();
    }
    const dim3 grid((unsigned)ceil_div(M, kPfTok), (unsigned)kv.Hkv, 2);
    if (kv.dk == 64) k_pages_fill_i8<64><<<grid, kFillThreads, 0, st>>>(a);
    else if (kv.dk == 128) k_pages_fill_i8<128><<<grid, kFillThreads, 0, st>>>(a);
    else if (kv.dk == 256) k_pages_fill_i8<256><<<grid, kFillThreads, 0, st>>>(a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_pages_read_i8(hipStream_t st, const nnhip_kv_pages_i8& kv, size_t M, const int32_t* cu, const int32_t* pos0,
                                size_t B, float* k, float* v, size_t num_cus)
{
    ReadI8Args a{pools_of(kv), kv.table, cu, pos0, k, v, (int)M, (int)B, (int)kv.Hkv, log2_of(kv.page_size),
                       (int)kv.table_stride, (int)kv.num_pages, (int)(kv.table_stride * kv.page_size), 1};
    // few columns: a head's dimensions shared by more work-groups, which do not wait 16 after 16 of them (a block of 32
    // behind 16 sequences: 4.4 us, by whole heads 9.7; from two work-groups to a CU on nothing is gained)
    const size_t blocks = ceil_div(M, kReadCols);
    while ((size_t)a.parts < kv.dk / 16 && blocks * kv.Hkv * 2 * (size_t)a.parts < 2 * num_cus) a.parts *= 2;
    const dim3 grid((unsigned)blocks, (unsigned)(kv.Hkv * (size_t)a.parts), 2);
    if (kv.dk == 64) k_pages_read_i8<64><<<grid, 256, 0, st>>>(a);
    else if (kv.dk == 128) k_pages_read_i8<128><<<grid, 256, 0, st>>>(a);
    else if (kv.dk == 256) k_pages_read_i8<256><<<grid, 256, 0, st>>>(a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace nnhip
