// k_prefill_i8.hip — attention of packed prompts over a paged KV cache in 8 bits (k_pages_i8.hip's pools): unlike
// lengths, positions and prefixes, a tanh cap and a bias on the scores, as k_prefill.hip's over f32 and f16 pages.
//
// A work-group = 8 waves = (R heads of a KV head) x (8 / R blocks of 32 queries); lane l holds query l % 32 of its wave
// throughout. Tiles of 64 keys are staged in LDS (double buffered, one barrier a tile) as f16, which holds every code
// as it is: keys as rows of dk, values as rows of 64 keys, in the order in which the weights of a query lie in its
// lane. The codes are widened once for the 256 queries (5 instructions for 4 of them), and no code is multiplied by its scale:
//   S^T = K . Q^T  with each query in two f16 parts, q 2^e = hi + lo to 2^-23 of it (and 2^-40 of the query's
//                  largest): two v_mfma_f32_32x32x16_f16 a step, whose products are exact; a key's scale is a factor of
//                  the 16 scores that share it, folded into the exponential's argument with the softmax scale;
//   O^T += V^T . P^T  with the weights in two f16 parts, 2^8 .. 2^15 at their largest: 2^-22 of every weight down to 2^-10 .. 2^-17
//                  of the largest, and 2^-33 .. 2^-40 of the largest below; over more than 8192 keys a tile far below the
//                  largest is weighed under its own. Of the scale of 16 values 2^k, a power of two, goes into their
//                  codes as they are widened, the rest, in 1 .. 2, into the weights by its logarithm in the same argument. O is in
//                  units of a power of two that the largest scale of a tile stays within 2^+-5 of: where it leaves that range,
//                  O moves to another unit first. Groups 2^-14 or more below it are summed apart, and so are those of a tile whose unit
//                  is 2^100 or more above that of a query which does not see the tile's large ones: each query's O has a unit of its
//                  own then. So no scale costs the weights bits, and none that a query does not see costs it anything.
// O^T stays in the accumulators over all tiles; a query's reference maximum moves when its maximum has grown by
// 2^6, by a whole power of two. Sums and softmax are f32. The next tile is converted by half of the waves before their
// products and by the other half behind them, so that every SIMD has one of each. A tile that every query of the wave sees
// goes in one piece, a group's weights between the last group's products (in two halves, each step by itself: 477 us for 446).
// Work-groups take equal spans of all tiles and join the items they share (prompt_spans.hpp).
// 4 x 700 .. 1024 queries at 6144, 20 heads over 5 of 128: 434 us and 20 for the join, 1.06 PFLOP/s of products (a large
// library product of f16: 1.16); the matrix cores are busy for half of the cycles and the VALU's 10 instructions a score, most of them the f32
// exponential and the weights' splitting, take most of the rest. 8 x 77 .. 1900 of 16 over 2 of 64, capped and biased: 69 us and 9, of which the
// VALU (23 instructions a score) takes about half and the matrix cores 15 %: a CU has one work-group, so an item's start, 4 to 5 us
// before its first product, has nothing beside it, and nearly every span ends in a record.
// A query that holds an infinity or a NaN gets NaN, and so does one that sees a block whose scale is not finite.
#include "prompt_spans.hpp"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace nnhip
{
namespace
{

struct ScalesI8
{
    const float* k;
    const float* v;
    int bshift;  // log2(positions of a scale)
};

constexpr int kI8Keys = 64;      // keys of a tile, two halves of kPK
constexpr float kI8Up = 8.0f;    // log2 of the largest weight when a reference maximum is new
constexpr float kI8Lazy = 6.0f;  // log2 growth of a query's maximum before its sums are rescaled: weights are at most 2^15 then
// f16 holds a weight to 2^-25, 2^-32 of the largest before: up to kI8Many tiles of 32 keys (8192 keys) all that is lost is 2^-19 of the largest
// weight at most. Over more of them a tile whose largest weight is more than kI8Deep log2 units below the reference is weighed under that
// weight. (Where a few queries of one wave do so, all wait for it: 4 x 700 .. 1024 at 6144, which has none with more, 432 us, with
// every tile looked at 448, from 4 units on 637.)
constexpr int kI8Many = 256;
constexpr float kI8Deep = 7.0f;
constexpr int kI8Near = 5;       // the largest scale of a tile's values is within 2^+-5 of O's unit
constexpr int kI8Low = -14;      // the least power of two that codes are multiplied by: they stay normal f16 values
constexpr int kI8Far = 100;      // O moves up by at most 2^100 to a unit whose scale its query need not see: it stays a normal f32 value
constexpr int kI8Fall = 60;      // and a unit lies at most 2^60 below the largest: O, below 2^57 in its unit over 2^30 keys, stays finite

constexpr int kJoin = 8;         // dimensions of a work-group that joins (17 records: 16 25.7 us, 8 24.8, 4 25.0)

template <int DK>
struct TileI8
{
    // rows are padded by 16 bytes: 16 lanes' accesses of consecutive rows fall on all banks
    static constexpr int kKPitch = DK * 2 + 16, kVPitch = kI8Keys * 2 + 16;
    static constexpr int kV = kI8Keys * kKPitch, kBuf = kV + DK * kVPitch;
    static constexpr int kTPitch = DK * 2 + 16;  // rows of the cos / sin tables, before the first tile
    static constexpr int kTables = 2 * 32 * kPWaves * kTPitch;
    static constexpr int kMain = 2 * kBuf > kTables ? 2 * kBuf : kTables;
    static constexpr int kScales = kMain;          // [4][2][4]: of four tiles' keys and values
    static constexpr int kFound = kMain + 128;     // [8]
    static constexpr int kBytes = kMain + 160;
};

// Four codes times 2^k as f16, f = 2^k, off = -1152 2^k: the byte code + 128 under the exponent of 1024 is 1152 + code
__device__ __forceinline__ u32x2 widen_codes(uint32_t x, v2h f, v2h off)
{
    const uint32_t u = x ^ 0x80808080u;
    const v2h a = __builtin_elementwise_fma(__builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)), f, off);
    const v2h b = __builtin_elementwise_fma(__builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)), f, off);
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
__device__ __forceinline__ u32x2 widen_codes(uint32_t x)
{
    const uint32_t u = x ^ 0x80808080u;
    const v2h off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const v2h a = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
    const v2h b = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

// The exponent field of a scale that counts, or 0: zeros, and what is not finite
__device__ __forceinline__ int scale_field(uint32_t bits) { return (bits >> 23) == 255 ? 0 : (int)(bits >> 23); }

// The power of two that goes into the codes of a group whose scale has that field, where O's unit is `unit`
__device__ __forceinline__ int code_power(int field, int unit) { return field == 0 ? 0 : min(max(field - unit, kI8Low), kI8Near); }

// Attention of an item over its tiles of 32 keys k0 .. k1 - 1; rec: into a record instead of the output
template <int DK, bool kShaped>
__device__ __forceinline__ void attend_i8(const PrefillArgs& a, const ScalesI8& sc, const PrefillItem& item, uint8_t* smem,
                                          int k0, int k1, float* rec, bool distance)
{
    using Tile = TileI8<DK>;
    constexpr int NC = DK / 16;  // MFMA steps over the head dimension
    constexpr int ND = DK / 32;  // 32-row blocks of O^T
    constexpr int NPC = 4 * DK;  // 16-byte pieces of a tile's keys, or values
    float* const scales = reinterpret_cast<float*>(smem + Tile::kScales);
    int* const found_s = reinterpret_cast<int*>(smem + Tile::kFound);

    // (opaque per item, so that no thread-index arithmetic stays alive across the items)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, h = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    PrefillWave w;
    PrefillSeq<true> seq;
    int last_key;
    seat(a, item, tid, w, seq, last_key);
    // Where at most half of the waves have queries, the others take the second half of each tile for them (6 x 5 .. 30
    // queries of 16 heads behind 2000 positions, 8 KV heads: 42.5 us without, 37.5)
    const int pair = kPWaves / 2, queries = kPQ << (kPWaveShift - log2_heads(a));  // of the work-group
    const bool shared = a.R < kPWaves && seq.n(a) - item.qb * queries <= queries / 2;
    const bool second = shared && wave >= pair;
    if (second)
    {
        w.t0 -= queries / 2;
        w.qt -= queries / 2;
        w.qpos -= queries / 2;
        w.live = w.t0 < seq.n(a);
    }
    const int end_key = min(last_key, k1 * kPK - 1);  // the last key of these tiles

    // ---- staging: a wave's pieces are of one group of 16 positions
    const int group = wave * 64 % NPC / DK;
    const bool has_k = DK == 128 || wave < 4, has_v = DK == 128 || wave >= 4;
    const int piece = tid % DK;  // within its group
    bool bad = false;
    int id;
    auto at_group = [&](int kb) { return min(kb * kPK + 16 * group, end_key & ~15); };
    auto load_id = [&](int kb) { id = a.table[(size_t)w.b * a.table_stride + (at_group(kb) >> a.shift)]; };
    u32x4 raw_k, raw_v;
    auto load_raw = [&](int kb) {
        const int page = __builtin_amdgcn_readfirstlane(id);
        const bool in = page_ok(page, a.num_pages);
        bad |= !in;
        const size_t row = page_row(in ? page : 0, w.g, at_group(kb) & ((1 << a.shift) - 1), a.Hkv, a.shift);
        const size_t off = (row >> 4) * (size_t)(16 * DK) + (size_t)(16 * piece);
        if (has_k) raw_k = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.kc) + off);
        if (has_v) raw_v = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(a.vc) + off);
        if (kb + 2 < k1) load_id(kb + 2);
    };
    // scales: the first four waves read those of a group each, a tile before its codes are widened
    auto at_scale = [&](int kb) { return min(kb * kPK + 16 * wave, end_key & ~15); };
    auto scale_id = [&](int kb) { return a.table[(size_t)w.b * a.table_stride + (at_scale(kb) >> a.shift)]; };
    auto load_scales = [&](int kb, int id, float(&s)[2]) {
        const int page = __builtin_amdgcn_readfirstlane(id);
        const size_t row = page_row(page_ok(page, a.num_pages) ? page : 0, w.g, at_scale(kb) & ((1 << a.shift) - 1), a.Hkv, a.shift);
        const bool there = kb * kPK + 16 * wave <= end_key;  // (behind the last key: whatever is there)
        s[0] = there ? sc.k[row >> sc.bshift] : 0.0f;
        s[1] = there ? sc.v[row >> sc.bshift] : 0.0f;
    };
    auto slot_of = [&](int kb) { return scales + ((kb - k0) >> 1 & 3) * 8; };
    auto post_scales = [&](int kb, const float(&s)[2]) {
        if (lane < 2) slot_of(kb)[4 * lane + wave] = lane ? s[1] : s[0];
    };
    // the unit of O for a tile whose scales are posted, where it was `unit` before and `top` at most so far
    auto next_unit = [&](int kb, int unit, int& top) {
        int field = scale_field(__builtin_bit_cast(uint32_t, slot_of(kb)[4 + (lane & 3)]));
        field = max(field, __builtin_amdgcn_update_dpp(0, field, 0xB1, 0xF, 0xF, true));  // lane ^ 1
        field = max(field, __builtin_amdgcn_update_dpp(0, field, 0x4E, 0xF, 0xF, true));  // lane ^ 2
        field = __builtin_amdgcn_readfirstlane(field);
        if (field == 0) return unit;
        top = max(top, field);
        return field > unit + kI8Near || field < unit - kI8Near ? max(field, top - kI8Fall) : unit;
    };
    auto convert = [&](int kb, int par, int unit) {
        uint8_t* const buf = smem + par * Tile::kBuf;
        if (has_k)
        {
            // 16 dimensions (chunk piece / 16) of position piece % 16
            uint8_t* const dst = buf + (16 * group + (piece & 15)) * Tile::kKPitch + 32 * (piece >> 4);
            const u32x2 x = widen_codes(raw_k[0]), y = widen_codes(raw_k[1]), z = widen_codes(raw_k[2]), t = widen_codes(raw_k[3]);
            *reinterpret_cast<u32x4*>(dst) = u32x4{x[0], x[1], y[0], y[1]};
            *reinterpret_cast<u32x4*>(dst + 16) = u32x4{z[0], z[1], t[0], t[1]};
        }
        if (has_v)
        {
            // 16 positions of dimension `piece`, as S^T's accumulators hold them: 0..3 and 8..11, then 4..7 and 12..15
            const uint32_t bits = (uint32_t)__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, slot_of(kb)[4 + group]));
            const int field = scale_field(bits);  // (0: values below 2^-119, or NaN, which their weights are then)
            const _Float16 to = field == 0 ? (_Float16)0.0f : (_Float16)pow2(code_power(field, unit)), down = (_Float16)-1152.0f * to;
            const v2h f = {to, to}, off = {down, down};
            uint8_t* const dst = buf + Tile::kV + piece * Tile::kVPitch + 32 * group;
            const u32x2 x = widen_codes(raw_v[0], f, off), y = widen_codes(raw_v[1], f, off), z = widen_codes(raw_v[2], f, off),
                        t = widen_codes(raw_v[3], f, off);
            *reinterpret_cast<u32x4*>(dst) = u32x4{x[0], x[1], z[0], z[1]};
            *reinterpret_cast<u32x4*>(dst + 16) = u32x4{y[0], y[1], t[0], t[1]};
        }
    };

    // ---- everything that the first tile waits for on its way together: rows of the cos / sin tables, page ids,
    // queries, then (with the ids) keys and values
    const int qn = kPQ << (kPWaveShift - log2_heads(a));
    constexpr int TC = DK / 8, TU = 32 * kPWaves * TC / kPThreads;  // 16-byte chunks of a row, those of a thread at most
    float4 tc[TU], ts[TU];
    if (a.cosT)
    {
        const __amdgpu_buffer_rsrc_t rc = pf_rsrc(a.cosT, rope_bytes(a, DK / 2)), rs = pf_rsrc(a.sinT, rope_bytes(a, DK / 2));
        const uint32_t t_at = (uint32_t)(seq.pos0(a) + item.qb * qn) * (uint32_t)(DK * 2) + (uint32_t)tid * 16u;
#pragma unroll
        for (int i = 0; i < TU; ++i)
            if (i * kPThreads < qn * TC)
            {
                tc[i] = ld_f4(rc, t_at + (uint32_t)(i * kPThreads * 16));
                ts[i] = ld_f4(rs, t_at + (uint32_t)(i * kPThreads * 16));
            }
    }
    load_id(k0);
    int sid = wave < 4 ? scale_id(k0) : 0, sid2 = wave < 4 && k0 + 2 < k1 ? scale_id(k0 + 2) : 0;
    PrefillQuery<DK, 8> query;
    if (w.live) query.load(a, w, seq, h);
    if (a.cosT)
    {
#pragma unroll
        for (int i = 0; i < TU; ++i)
        {
            const int ct = tid + i * kPThreads;
            if (ct >= qn * TC) break;
            uint8_t* dst = smem + ct / TC * Tile::kTPitch + 16 * (ct % TC);
            *reinterpret_cast<float4*>(dst) = tc[i];
            *reinterpret_cast<float4*>(dst + qn * Tile::kTPitch) = ts[i];
        }
    }
    __syncthreads();
    load_raw(k0);
    float s_now[2], s_next[2];
    if (wave < 4)
    {
        load_scales(k0, sid, s_now);
        if (k0 + 2 < k1) load_scales(k0 + 2, sid2, s_next);
        if (k0 + 4 < k1) sid = scale_id(k0 + 4);
    }

    // ---- the lane's rotated query in halves: step c holds dimensions 16c + 8h + 0..7, scaled by 2^eq
    v8h qh[NC], ql[NC];
    float f = 0.0f;  // 2^-eq |scale| log2(e), or over the cap
    if (w.live)
    {
        float qv[DK / 2];
        uint32_t mx = 0;
        const uint8_t* tab = smem + (min(w.qt, seq.n(a) - 1) - item.qb * qn) * Tile::kTPitch + 32 * h;
        auto table = [&](const uint8_t* t, int c, int i) { return *reinterpret_cast<const float4*>(t + 64 * c + 16 * i); };
        query.rotate(a, [&](int c, int i) { return table(tab, c, i); }, [&](int c, int i) { return table(tab + qn * Tile::kTPitch, c, i); },
                     [&](int c, int e, float y0, float y1) {
            qv[8 * c + e] = y0;
            qv[8 * (c + NC / 2) + e] = y1;
            mx = max(mx, max(__builtin_bit_cast(uint32_t, y0) & 0x7FFFFFFFu, __builtin_bit_cast(uint32_t, y1) & 0x7FFFFFFFu));
        });
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, kWave));
        const int eq = min(f16_exp(mx), 120);  // (infinities and NaN: -114, and they stay what they are)
        const float sq = a.scale < 0.0f ? -pow2(eq) : pow2(eq);
        f = pow2(-eq) * (a.cap2 > 0.0f ? a.scale2 * a.capi2 : a.scale2);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 8; e += 2)
            {
                v2h x, y;
                split2(qv[8 * c + e] * sq, qv[8 * c + e + 1] * sq, x, y);
                qh[c][e] = x[0], qh[c][e + 1] = x[1];
                ql[c][e] = y[0], ql[c][e + 1] = y[1];
            }
    }
    v16f o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = v16f{};
    float m_ref = -__builtin_inff(), l_run = 0.0f;  // log2 units; l_run: this lane half's keys
    const float slope2 = kShaped && a.slopes ? a.slopes[w.head] * 1.44269504f : 0.0f;
    float steps[16];  // the bias of a half's keys, from its first on (as many registers, at one work-group to a CU)
    if constexpr (kShaped)
    {
#pragma unroll
        for (int v = 0; v < 16; ++v) steps[v] = slope2 * (float)(8 * (v >> 2) + (v & 3));
    }
    if (wave < 4)
    {
        post_scales(k0, s_now);
        if (k0 + 2 < k1) post_scales(k0 + 2, s_next);
    }
    __syncthreads();  // the tables have been read; the first two tiles' scales are there
    int unit_top = 0, unit = next_unit(k0, 127, unit_top);  // tiles are added to O in units of 2^(unit - 127)
    int lane_unit = unit;                                   // and what the lane has of O is in units of 2^(lane_unit - 127)
    bool settled = true;                                    // the same in every lane
    convert(k0, 0, unit);
    if (k0 + 2 < k1) load_raw(k0 + 2);
    // scores s of a half, with their keys' scales: capped, and their bias from the half's first key on
    auto shape = [&](v16f& s, float k0, float k1) {
        float kf[2] = {k0, k1};
                        if (a.cap2 > 0.0f)
                        {
                            // scores rarely reach the cap: a polynomial of few terms where none does
                            float top = 0.0f;  // (a NaN does not show, and stays one in each form)
#pragma unroll
                            for (int v = 0; v < 16; ++v)
                            {
                                s[v] *= kf[v >> 3];
                                top = fmaxf(top, fabsf(s[v]));
                            }
                            if (__builtin_amdgcn_ballot_w64(top > 0.25f) == 0)
                            {
#pragma unroll
                                for (int v = 0; v < 16; ++v) s[v] = __builtin_fmaf(tanh_below_quarter(s[v]), a.cap2, steps[v]);
                            }
                            else if (__builtin_amdgcn_ballot_w64(top > 1.0f) == 0)
                            {
#pragma unroll
                                for (int v = 0; v < 16; ++v) s[v] = __builtin_fmaf(tanh_below1(s[v]), a.cap2, steps[v]);
                            }
                            else
                            {
#pragma unroll
                                for (int v = 0; v < 16; ++v) s[v] = __builtin_fmaf(tanh_any(s[v]), a.cap2, steps[v]);
                            }
                        }
                        else
                        {
                            // (an opaque factor: or this is computed whether the branch is taken or not)
                            asm volatile("" : "+v"(kf[0]), "+v"(kf[1]));
#pragma unroll
                            for (int v = 0; v < 16; ++v) s[v] = __builtin_fmaf(s[v], kf[v >> 3], steps[v]);
                        }
    };
    // a score's factor, of a key's scale: within f32's range, as a score of 0 is 0 under any finite scale (any other is past the
    // cap, or the range, with the largest float, too). Scales are below 2^122, so only large queries get there
    auto factor = [&](float scale) { return scale < __builtin_inff() ? fminf(f * scale, 3.40282347e38f) : __builtin_nanf(""); };
    const bool many = k1 - k0 > kI8Many;
    const bool large = __builtin_amdgcn_ballot_w64(!(f < 32.0f)) != 0;
    const uint32_t k_at = (uint32_t)(l32 * Tile::kKPitch + 16 * h), v_at = (uint32_t)(Tile::kV + l32 * Tile::kVPitch + 16 * h);
    int par = 0;
    for (int kb = k0; kb < k1; kb += 2, par ^= 1)
    {
        __syncthreads();  // tile kb is in LDS; the other buffer is free
        const bool more = kb + 2 < k1;
        const int unit_next = more ? next_unit(kb + 2, unit, unit_top) : unit;
        if (more && wave < 4)
        {
            convert(kb + 2, par ^ 1, unit_next);
            if (kb + 4 < k1)
            {
                load_raw(kb + 4);  // in flight during this tile's products
                load_scales(kb + 4, sid, s_next);
                if (kb + 6 < k1) sid = scale_id(kb + 6);
            }
        }
        const uint8_t* const buf = smem + par * Tile::kBuf;
        const float* const ts4 = slot_of(kb);
        // Where every query sees the whole tile, no unit moves, every scale counts and no query is large: both halves at once, a group's weights beside the
        // last group's products with the values
        bool whole = !shared && !large && w.live && kb + 1 < k1 && (kb + 2) * kPK - 1 <= (kShaped ? seq.pos0(a) + w.t0 : seq.from(a, w)) &&
                     settled;
        float lv4[4];
        // (keys two steps ahead of their products, of both halves in turn)
        auto keys = [&](int half, int c) { return *reinterpret_cast<const v8h*>(buf + k_at + half * kPK * Tile::kKPitch + 32 * c); };
        constexpr int kDeep = 2;
        v8h k[2][kDeep];
        if (whole)
        {
#pragma unroll
            for (int i = 0; i < 2 * kDeep; ++i) k[i & 1][i >> 1] = keys(i & 1, i >> 1);
            const float scale = ts4[4 + (lane & 3)];
            const int e = scale_field(__builtin_bit_cast(uint32_t, scale));
            const float lv = __builtin_amdgcn_logf(scale) - (float)(e - 127);
            whole = __builtin_amdgcn_ballot_w64(e == 0 || e - unit < kI8Low || e - unit > kI8Near) == 0;
#pragma unroll
            for (int t = 0; t < 4; ++t) lv4[t] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, lv), t));
        }
        if (whole)
        {
            v16f s[2] = {v16f{}, v16f{}};
#pragma unroll
            for (int c = 0; c < NC; ++c)
            {
                const v8h x = k[0][c % kDeep], y = k[1][c % kDeep];
                if (c + kDeep < NC) k[0][c % kDeep] = keys(0, c + kDeep), k[1][c % kDeep] = keys(1, c + kDeep);
                s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ql[c], s[0], 0, 0, 0);
                s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, ql[c], s[1], 0, 0, 0);
                s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qh[c], s[0], 0, 0, 0);
                s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, qh[c], s[1], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            float kf[4], away[2] = {0.0f, 0.0f}, top = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < 4; ++t) kf[t] = f * ts4[t];
            if constexpr (kShaped)
            {
#pragma unroll
                for (int half = 0; half < 2; ++half)
                {
                    shape(s[half], kf[2 * half], kf[2 * half + 1]);
                    away[half] = slope2 * (float)((kb + half) * kPK + 4 * h - w.qpos);
                    kf[2 * half] = kf[2 * half + 1] = 1.0f;
                }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
            {
                float most = s[t >> 1][8 * (t & 1)];
#pragma unroll
                for (int v = 1; v < 8; ++v) most = fmaxf(most, s[t >> 1][8 * (t & 1) + v]);
                top = fmaxf(top, kShaped ? most + away[t >> 1] : most * kf[t]);
            }
            const float mx = __builtin_ceilf(max_halves(top));
            whole = !many || __builtin_amdgcn_ballot_w64(mx < m_ref - kI8Deep) == 0;
            if (__builtin_expect(whole, 1))
            {
                const bool grown = mx > m_ref + kI8Lazy;
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(grown) != 0, 0))
                {
                    const float m_new = grown ? mx : m_ref;
                    float corr = grown ? __builtin_amdgcn_exp2f(m_ref - m_new) : 1.0f;
                    asm volatile("" : "+v"(corr));
                    l_run *= corr;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int v = 0; v < 16; ++v) o[d][v] *= corr;
                    m_ref = m_new;
                }
                float base[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) base[half] = kI8Up + (m_ref == -__builtin_inff() ? 0.0f : away[half] - m_ref);
                // weights of group t + 1 between the products of group t: a pair of keys beside 8 / ND products
                v8h pa[2], pb[2];
                float sum = 0.0f;
                auto pair = [&](int t, int v) {
                    const float off = base[t >> 1] + lv4[t];
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t >> 1][8 * (t & 1) + v], kf[t], off));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t >> 1][8 * (t & 1) + v + 1], kf[t], off));
                    sum += p0;
                    sum += p1;
                    v2h x, y;
                    split2(p0, p1, x, y);
                    pa[t & 1][v] = x[0], pa[t & 1][v + 1] = x[1];
                    pb[t & 1][v] = y[0], pb[t & 1][v + 1] = y[1];
                    if (v == 6)
                    {
                        l_run = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(-lv4[t]), l_run);
                        sum = 0.0f;
                    }
                };
                auto values = [&](int i) { return *reinterpret_cast<const v8h*>(buf + v_at + 32 * (i % ND) * Tile::kVPitch + 32 * (i / ND)); };
                v8h x = values(0);
#pragma unroll
                for (int v = 0; v < 8; v += 2) pair(0, v);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                    {
                        const v8h y = x;
                        if (t * ND + d + 1 < 4 * ND) x = values(t * ND + d + 1);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, pb[t & 1], o[d], 0, 0, 0);
                        if (t < 3)
#pragma unroll
                            for (int v = 8 / ND * d; v < 8 / ND * (d + 1); v += 2) pair(t + 1, v);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, pa[t & 1], o[d], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
#pragma unroll 1
        for (int half = whole ? 2 : 0; half < 2; ++half)
        {
            const int key0 = (kb + half) * kPK;
            if (!w.live || kb + half >= k1 || key0 > seq.to(a, w) || (shared && half != (int)second)) continue;
            v16f s = v16f{};
#pragma unroll
            for (int c = 0; c < NC; ++c)
            {
                const v8h k = *reinterpret_cast<const v8h*>(buf + k_at + half * kPK * Tile::kKPitch + 32 * c);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[c], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[c], s, 0, 0, 0);
            }
            float kf[2], vs[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
            {
                kf[t] = factor(ts4[2 * half + t]);
                vs[t] = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, ts4[4 + 2 * half + t])));
            }
            const bool masked = key0 + kPK - 1 > seq.from(a, w);
            float away = 0.0f;  // the bias of the half's first key, the steps from there apart
            if constexpr (kShaped)
            {
                shape(s, kf[0], kf[1]);
                const float first = (float)(key0 + 4 * h - w.qpos);
                away = slope2 * first;
                if (distance && key0 + kPK - 1 > seq.pos0(a) + w.t0)
                {
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (first + (float)(8 * (v >> 2) + (v & 3)) > 0.0f) s[v] = __builtin_fmaf(-2.0f, steps[v] + away, s[v]);
                }
                kf[0] = kf[1] = 1.0f;
            }
            else if (masked)
            {
                // (opaque factors here too)
                asm volatile("" : "+v"(kf[0]), "+v"(kf[1]));
#pragma unroll
                for (int v = 0; v < 16; ++v) s[v] *= kf[v >> 3];
                kf[0] = kf[1] = 1.0f;
            }
            if (masked)
            {
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (key0 + 8 * (v >> 2) + 4 * h + (v & 3) > seq.sight(w)) s[v] = -__builtin_inff();
            }
            float top[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
            {
                top[t] = s[8 * t];
#pragma unroll
                for (int v = 1; v < 8; ++v) top[t] = fmaxf(top[t], s[8 * t + v]);
                top[t] *= kf[t];
            }
            const float mx = __builtin_ceilf(max_halves(fmaxf(top[0], top[1]) + away));
            // the reference of a query moves only when its maximum has grown by 2^6 (or is new)
            const bool grown = mx > m_ref + kI8Lazy;
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(grown) != 0, 0))
            {
                const float m_new = grown ? mx : m_ref;
                float corr = grown ? __builtin_amdgcn_exp2f(m_ref - m_new) : 1.0f;
                asm volatile("" : "+v"(corr));
                l_run *= corr;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] *= corr;
                m_ref = m_new;
            }
            const float base = kI8Up + (m_ref == -__builtin_inff() ? 0.0f : away - m_ref);
            const bool deep = many && __builtin_amdgcn_ballot_w64(mx < m_ref - kI8Deep && mx > -__builtin_inff()) != 0;
            if (__builtin_expect(!settled, 0))
            {
                // O to the tile's unit, unless that is far above the lane's: its query may not see what has raised it
                const bool far = lane_unit - unit < -kI8Far;
                int by = far ? 0 : lane_unit - unit;
                asm volatile("" : "+v"(by));
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] = __builtin_ldexpf(o[d][v], by);
                if (!far) lane_unit = unit;
                settled = __builtin_amdgcn_ballot_w64(far) == 0;
            }
            int apart = 0;  // bit t: group t's sums are not added to O as they are
#pragma unroll
            for (int t = 0; t < 2; ++t)
            {
                // what the codes have not got of their scale (0 and what is not finite: nothing)
                const uint32_t bits = __builtin_bit_cast(uint32_t, vs[t]);
                const int e = scale_field(bits);
                const float lv = e == 0 ? 0.0f : __builtin_amdgcn_logf(vs[t]) - (float)(e - 127);
                if (__builtin_expect((bits >> 23) == 255, 0) && key0 + 16 * t <= seq.sight(w)) l_run = __builtin_nanf("");
                const bool here = settled && !deep && (e == 0 || e - unit == code_power(e, unit));
                const float off = here ? base + lv : -__builtin_inff();
                apart |= here ? 0 : 1 << t;
                float sum = 0.0f;
                v8h pa, pb;
#pragma unroll
                for (int v = 0; v < 8; v += 2)
                {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * t + v], kf[t], off));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * t + v + 1], kf[t], off));
                    sum += p0;
                    sum += p1;
                    v2h x, y;
                    split2(p0, p1, x, y);
                    pa[v] = x[0], pa[v + 1] = x[1];
                    pb[v] = y[0], pb[v + 1] = y[1];
                }
                l_run = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(-lv), l_run);
#pragma unroll
                for (int d = 0; d < ND; ++d)
                {
                    const v8h x = *reinterpret_cast<const v8h*>(buf + v_at + 32 * d * Tile::kVPitch + 32 * (2 * half + t));
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pb, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pa, o[d], 0, 0, 0);
                }
            }
            // A group whose scale is far below the largest of its tile, which some queries may not see, or some lane's unit far below,
            // or the largest weight of 32 keys far below the reference, over many keys: weights times 2^up, under a reference of their own,
            // and their sums, in units of 2^(own - up - 127), to each lane's own unit, which becomes the group's where the
            // query sees that, and it is 2^20 larger or the lane has nothing yet
            const float up = deep && mx < m_ref - kI8Deep && mx > -__builtin_inff() ? fminf(m_ref - mx, 400.0f) : 0.0f;
#pragma unroll 1
            for (int t = 0; __builtin_expect(apart >> t != 0, 0); ++t)
            {
                if (!(apart >> t & 1)) continue;
                settled = false;
                const float scale = t ? vs[1] : vs[0], by = t ? kf[1] : kf[0];
                const int e = scale_field(__builtin_bit_cast(uint32_t, scale)), own = e == 0 ? unit : e - code_power(e, unit);
                const float lv = e == 0 ? 0.0f : __builtin_amdgcn_logf(scale) - (float)(e - 127);
                uint32_t any = 0;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) any |= __builtin_bit_cast(uint32_t, o[d][v]);
                int to = own - (int)up - lane_unit;
                const int move = (to > 20 || any << 1 == 0) && key0 + 16 * t <= seq.sight(w) ? to : 0;
                lane_unit += move;
                to -= move;
                float sum = 0.0f;
                v8h pa, pb;
#pragma unroll
                for (int v = 0; v < 8; v += 2)
                {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(t ? s[8 + v] : s[v], by, base + up + lv));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(t ? s[9 + v] : s[v + 1], by, base + up + lv));
                    sum += p0;
                    sum += p1;
                    v2h x, y;
                    split2(p0, p1, x, y);
                    pa[v] = x[0], pa[v + 1] = x[1];
                    pb[v] = y[0], pb[v + 1] = y[1];
                }
                l_run = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(-lv - up), l_run);
#pragma unroll
                for (int d = 0; d < ND; ++d)
                {
                    const v8h x = *reinterpret_cast<const v8h*>(buf + v_at + 32 * d * Tile::kVPitch + 32 * (2 * half + t));
                    v16f y = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pb, v16f{}, 0, 0, 0);
                    y = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pa, y, 0, 0, 0);
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] = __builtin_ldexpf(o[d][v], -move) + __builtin_ldexpf(y[v], to);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if (more && wave >= 4)
        {
            convert(kb + 2, par ^ 1, unit_next);
            if (kb + 4 < k1) load_raw(kb + 4);
        }
        if (more)
        {
            settled &= unit == unit_next;
            unit = unit_next;
            if (wave < 4 && kb + 4 < k1) post_scales(kb + 4, s_next);
        }
    }
    l_run += __shfl_xor(l_run, 32);
    const bool any_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) found_s[wave] = any_bad;
    __syncthreads();
    int found = 0;
#pragma unroll
    for (int i = 0; i < kPWaves; ++i) found |= found_s[i];
    if (found) l_run = __builtin_nanf("");
    int power = lane_unit - 127;  // of two, that O is in units of
    if ((rec || shared) && power > 0)
    {
        // large values, whose sums would pass f32's range: O and its sum to below 2^-8 of the values, 64 records' to below the
        // values themselves (where they are joined before the division; small ones would lose bits)
        const int field = (int)(__builtin_bit_cast(uint32_t, l_run) >> 23), by = l_run > 0.0f && field < 255 ? field - 126 + 8 : 0;
        l_run = __builtin_ldexpf(l_run, -by);
        m_ref += (float)by;
        power -= by;
    }
    if (shared)
    {
        // the second halves' outputs, maxima and sums through LDS (every wave is past its tiles)
        float* const at = reinterpret_cast<float*>(smem) + (wave & (pair - 1)) * (16 * ND + 2) * kWave + lane;
        if (second && w.live)
        {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) at[(16 * d + v) * kWave] = __builtin_ldexpf(o[d][v], power);
            at[16 * ND * kWave] = m_ref;
            at[(16 * ND + 1) * kWave] = l_run;
        }
        __syncthreads();
        if (!second && w.live)
        {
            const float m = at[16 * ND * kWave], to = fmaxf(m_ref, m);
            const float own = m_ref == to ? 1.0f : __builtin_amdgcn_exp2f(m_ref - to);
            const float other = m == to ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            l_run = __builtin_fmaf(at[(16 * ND + 1) * kWave], other, l_run * own);
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    o[d][v] = __builtin_fmaf(at[(16 * d + v) * kWave], other, __builtin_ldexpf(o[d][v], power) * own);
            power = 0;
            m_ref = to;
        }
        __syncthreads();  // the next item may write there
        w.live &= !second;
    }
    auto dim = [](int d, int i) { return 32 * d + i; };
    if (!w.live) return;
    if (rec)
    {
        store_record<DK>(rec, tid, dim, [&](int d, int v) { return __builtin_ldexpf(o[d][v], power); }, m_ref, l_run);
        return;
    }
    // (nothing visible above -infinity: 0)
    const float inv = l_run == 0.0f ? 1.0f : 1.0f / l_run;
    store_out<DK>(a, w, seq, h, dim, [&](int d, int v) { return __builtin_ldexpf(o[d][v] * inv, power); });
}

// The items of a work-group of a call of packed prompts, one after the other: attend(item, first tile, end, record or
// null). One item each, heaviest first (the last queries attend over the most keys) and a step further per block of
// queries, or a long sequence's work-groups, per_qb apart, would all fall on one or two of the 8 XCDs; or spans.
template <int DK, typename F>
__device__ __forceinline__ void prompt_items(const PrefillArgs& a, uint8_t* smem, F&& attend)
{
    PrefillItem it;
    const int groups = a.groups, HG = a.Hkv * groups;
    const int per_qb = a.B * HG, back = (int)blockIdx.x / per_qb;
    const int bg = ((int)blockIdx.x + back) % per_qb;
    const int g = blockIdx.x;
    PromptCut at, end;
    if (a.spans)
    {
        // the span's two cuts by a wave each, while the others look for sequences that do not fit
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        struct Found
        {
            PromptCut cut;
            PrefillSeq<true> seq;
        };
        Found* const cuts = reinterpret_cast<Found*>(smem);
        if (wave < 2)
        {
            PrefillSeq<true> seq{};
            const PromptCut cut = prompt_cut<true>(a, a.spans, g + wave, &seq);
            if ((threadIdx.x & 63) == 0)
            {
                cuts[wave] = {cut, seq};
                if (wave == 0) prompt_cuts<DK>(a, a.spans)[g] = cut;
            }
        }
        else
            for (int b = g; b < a.B; b += a.spans)
                if (PrefillSeq<true> any; !packed_seq(a, b, any)) store_nan<DK>(a, b, 0, a.H, (int)threadIdx.x - 2 * kWave, kPThreads - 2 * kWave);
        __syncthreads();
        at = uniform(cuts[0].cut);
        end = uniform(cuts[1].cut);
        const PrefillSeq<true> q = cuts[0].seq;
        it.seq = {__builtin_amdgcn_readfirstlane(q.n_), __builtin_amdgcn_readfirstlane(q.col0_), __builtin_amdgcn_readfirstlane(q.pos0_),
                  __builtin_amdgcn_readfirstlane(q.pre)};
        __syncthreads();
    }
    else
    {
        at = {bg % HG, bg / HG, a.nqb - 1 - back, 0};
        if (!packed_seq(a, at.b, it.seq))
        {
            store_nan<DK>(a, at.b, at.gh * a.R, a.R, at.qb * kPThreads + (int)threadIdx.x, a.nqb * kPThreads);
            return;
        }
        if (at.qb >= prompt_blocks(a, it.seq.n_)) return;
        end = {at.gh, at.b, at.qb + 1, 0};
    }
    bool known = true;  // it.seq is at.b's
    while (cut_before(at, end))
    {
        // the next sequence with a block left
        const bool there = at.b < a.B;
        if (!there || !(known || packed_seq(a, at.b, it.seq)) || at.qb >= prompt_blocks(a, it.seq.n_))
        {
            at = there ? PromptCut{at.gh, at.b + 1, 0, 0} : PromptCut{at.gh + 1, 0, 0, 0};
            known = false;
            continue;
        }
        const int tiles = prompt_tiles(a, it.seq, at.qb), to = cut_same_item(at, end) ? end.t : tiles;
        it.b = at.b;
        it.g = at.gh / groups;
        it.first = at.gh * a.R;
        it.qb = at.qb;
        float* rec = at.t == 0 && to == tiles ? nullptr : prompt_record<DK>(a, g, at.t > 0 ? 0 : 1);
        attend(it, at.t, to, rec);
        known = true;
        at = {at.gh, at.b, at.qb + 1, 0};
    }
}

template <int DK, bool kShaped>
__global__ __launch_bounds__(kPThreads) void k_attn_prefill_i8(PrefillArgs a, ScalesI8 sc, int distance)
{
    extern __shared__ __align__(16) uint8_t smem[];
    prompt_items<DK>(a, smem, [&](const PrefillItem& it, int k0, int k1, float* rec) {
        attend_i8<DK, kShaped>(a, sc, it, smem, k0, k1, rec, distance != 0);
    });
}

template <int DK, bool kShaped>
hipError_t launch_prefill_i8_dk(hipStream_t st, const PrefillArgs& a, const ScalesI8& sc, bool distance)
{
    constexpr int lds = TileI8<DK>::kBytes;
    static std::atomic<uint64_t> set{0};  // a bit per device
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    if (device > 63 || !(set.load() >> device & 1))
    {
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_attn_prefill_i8<DK, kShaped>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        if (device <= 63) set.fetch_or(uint64_t(1) << device);
    }
    const unsigned blocks = a.spans ? (unsigned)a.spans : (unsigned)(a.nqb * a.B * a.Hkv * a.groups);
    hipLaunchKernelGGL((k_attn_prefill_i8<DK, kShaped>), dim3(blocks), dim3(kPThreads), lds, st, a, sc, distance ? 1 : 0);
    if (a.spans > 1)
    {
        e = hipGetLastError();
        if (e != hipSuccess) return e;
        k_prompt_join<DK, kJoin, 2><<<dim3((unsigned)a.spans - 1, DK / kJoin), 32 * kPWaves, 0, st>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_pages_prefill_i8(hipStream_t st, const nnhip_kv_pages_i8& kv, const float* q, size_t M, const int32_t* cu,
                                   const int32_t* pos0, size_t B, size_t t_bound, size_t H, const float* cosT,
                                   const float* sinT, size_t limit, float scale, float softcap, const float* slopes,
                                   const int32_t* prefix, bool distance, float* out, void* ws, size_t num_cus)
{
    // a KV head's R query heads in work-groups of 8, 4, 2 or 1
    const size_t heads = H / kv.Hkv, R = heads % 8 == 0 ? 8 : heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
    const double cap2 = softcap * 1.4426950408889634;
    PrefillArgs a{q, kv.k, kv.v, cosT, sinT, out, (int)B, (int)t_bound, (int)H, (int)kv.Hkv, (int)R, 0,
                  (int)limit, (int)std::max<size_t>(1, ceil_div(std::min(t_bound, limit), kPQ * (kPWaves / R))), scale,
                  (float)(std::fabs(scale) * 1.4426950408889634), 0,
                  (int)M, (int)(heads / R), kv.table, cu, pos0, prefix, slopes, (int)kv.table_stride, (int)kv.num_pages,
                  0, (int)limit, (float)cap2, softcap > 0.0f ? (float)(1.0 / cap2) : 0.0f,
                  static_cast<float*>(ws), (int)pages_prefill_spans(limit, num_cus)};
    while ((size_t(1) << a.shift) < kv.page_size) ++a.shift;
    ScalesI8 sc{kv.k_scale, kv.v_scale, 0};
    while ((size_t(1) << sc.bshift) < kv.block) ++sc.bshift;
    if (cap2 > 0.0 || slopes)
        return kv.dk == 64 ? launch_prefill_i8_dk<64, true>(st, a, sc, distance) : launch_prefill_i8_dk<128, true>(st, a, sc, distance);
    return kv.dk == 64 ? launch_prefill_i8_dk<64, false>(st, a, sc, distance) : launch_prefill_i8_dk<128, false>(st, a, sc, distance);
}

}  // namespace nnhip
