// k_prefill.hip — batched prefill of the decoder's attention: T new tokens for each of B
// sequences at positions pos0 .. pos0 + T - 1 in one pass, instead of T decode steps.
//
// Reference: GPTModel::generate fills the KV cache by calling forward_step once per context
// token (include/neuralnet.cpp/compute_layer_gpt.hpp:774-794); each call rotates the new key
// at its position, appends key and value to the caches and attends over positions [0, pos]
// (AttentionBase::forward_step, compute_layer_attention.hpp:1003-1091). The same results for
// all T tokens at once:
//   * k_kv_fill writes the T rotated keys and values of every sequence into cache rows
//     pos0 .. pos0 + T - 1 (RoPE as the decode append: two rounded products and a rounded sum);
//   * k_attn_prefill gives token t the softmax attention over cache rows [0, pos0 + t] (causal),
//     query head h reading KV head h / (H / Hkv).
//
// Layouts (device, f32): q (H*dk, M), k / v (Hkv*dk, M) and out (H*dk, M) feature-major with
// token column m = b*T + t (the BitLinear outputs of the B*T tokens); caches (B, max_len,
// Hkv*dk) as the decode step's; cos / sin (max_len, dk/2).
//
// k_attn_prefill: the fp32 MFMA's rate (157 TFLOP/s) bounded this attention (101 of it at 4 x 2048
// tokens), and the f16 and bf16 MFMAs run 16 times as fast. So its products run on those with every
// f32 operand as a sum of parts, whose products are exact in f32:
//   * S = K . Q^T: two f16 halves, x 2^e = hi + lo to 2^-23 of x, where e brings the largest value of a
//     query or of a tile of K to 2^14..2^15 (f16 caches: K as it is). What is below 2^-40 of that is
//     lost, less than 2^-21 of a score in all where scores cannot reach 2^18. low x low, at most
//     2^-22 of a term, is left out: three MFMAs per product with f32 caches, two with f16 caches.
//   * O = P . V: three bf16 parts, x = b0 + b1 + b2 exactly and without a scale, two for f16 caches' V.
//     The probability of a key and the size of its value have nothing to do with each other, so
//     neither may cost the other bits: no exponent shared by a tile or a sequence holds both (f16
//     halves of V under one scale lost a channel 1e-7 of the others to 1e-4, 1e-10 altogether).
//     Products b_i b_j with i + j > 2, at most 2^-24 of a term, are left out: six and five MFMAs.
// Sums, softmax and output are f32. Against float64, 1024 tokens of 20 heads over 5 KV heads of 128,
// f32 / f16 caches: 2.3e-7 / 2.0e-7 off in norm (f32 products: 3.9e-7 both).
// What the parts cannot hold (infinities, NaN, a query's or K tile's largest value outside 2^+-48,
// outputs below 2^-100, largest values whose scores could reach 2^18) sends the work-group to the f32
// products (attend_f32).
//
// Work-group = 8 waves = (the R = H / Hkv heads of KV head g) x (8 / R blocks of 32 queries) of
// sequence b; all waves share each 32-key tile of K and V, staged in LDS as planes of parts (double
// buffered, one barrier per tile): the next tile is converted from registers while the one after
// it is loaded. A wave computes S^T = K . Q^T (32 keys x 32 queries) and O^T += V^T . P^T, where
// lane l holds query l % 32 throughout: its 16 elements v of S^T are keys 8(v/4) + 4(l/32) + v%4,
// and V^T is staged with its keys in that order, so P^T is an operand as it stands. Row 32d + r of
// V^T is dimension (DK/32) r + d, which lets a staging lane load contiguous dimensions and its
// stores fall on all banks. K rows and V^T rows are padded to odd multiples of 16 bytes.
// Softmax in log2 units with the hardware exp2; a query's reference maximum moves only when it has
// grown by 2^8 (probabilities are at most 2^8), so the sums are rarely rescaled.
// Work-groups are issued heaviest first (the last query blocks attend over the most keys).
// V's four waves convert their part of the next tile behind their products, K's before them: every SIMD
// has one wave of each, and one's VALU phases fall on the other's MFMA phases (4 x 2048 tokens f32 caches
// 389 -> 367 us, f16 280 -> 273, back to back on one box; 350 and 269 with the steps below).
// Measured before that (calls back to back in a graph, us, f32 products / here): f32 caches 4 x 2048 tokens
// 809 / 398, 3 x 1111 at 517 411 / 202, 16 x 2048 3088 / 1498, 1 x 64 22.5 / 17.7; f16 caches 817 / 293,
// 421 / 146, 3153 / 1121, 22.7 / 15.9. Two f16 halves for P and V too (at the cost above) took 295 and
// 198 us at 4 x 2048.
//
// Over pages (kPaged): packed sequences of unlike lengths, each at its own position, whose rows are found
// through a page table read a tile ahead; a prefix that all queries see, a tanh cap and a bias on the scores,
// linear in the position or (kDistance; the two differ for keys ahead of the query, inside a prefix) in the
// distance. Any H / Hkv: a KV head's heads go in groups of 8, 4, 2 or 1.
//   * Work-groups take equal spans of all tiles of the call (prompt_cut) and join the blocks of queries
//     they share; a plain work-group per block of queries left most CUs idle behind a long sequence, or
//     behind the 14 blocks beyond 256 (4 x 700 .. 1024 tokens at 6144, f16: 1087 -> 754 us).
//   * f16 caches: V as it is in f16 products with the weights in two f16 parts, p = a + b 2^-11, under a reference of
//     the tile's own: every weight to 2^-22 of itself down to 2^-29 of the largest of its 32 keys, and to
//     2^-51 of that one below; two MFMAs instead of five and no splitting of V (688 -> 579 us). Weights of
//     one tile share an exponent with each other here, never with values; where heavy keys' values are 0, and
//     lost bits could show, the f32 products run.
//   * A block of queries costs about four tiles besides its own: its queries (128 KB for dk 128, into one CU), their
//     rotation and splitting, and the check at its end. What it waits for is on its way together.
// 4 x 700 .. 1024 tokens at position 6144, 20 heads over 5 of 128, f16: 555 us with the join (20), 410 TFLOP/s of the
// attention's own products; 8 x 77 .. 1900 tokens, 16 heads over 2 of 64, f32, capped and biased: 105 .. 114 us.
// Bound by the VALU and MFMA work of a tile, which two waves to a SIMD overlap in part.
// Caches of f16 elements (compute = F16): the fill rounds the rotated keys and the values to the
// nearest f16 (ties to even), as the decode append does.
#include "prompt_spans.hpp"

#include <algorithm>
#include <cmath>

namespace nnhip
{
namespace
{

// Four cache elements at byte offset off as floats (f32, or f16 widened exactly)
template <typename CT>
__device__ __forceinline__ float4 ld_c4(__amdgpu_buffer_rsrc_t r, uint32_t off)
{
    if constexpr (sizeof(CT) == 4) return ld_f4(r, off);
    else
    {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        const h4 h = __builtin_bit_cast(h4, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
        return make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
    }
}

// ------------------------------------------------------------------ cache fill

// Block = (32 tokens, KV head g): the head's dk feature rows of k and v for the 32 tokens are
// read along tokens (coalesced), transposed through LDS and written as cache rows (coalesced
// along features), the keys rotated at their positions. Bound by HBM: each element read and written
// once; every load of a thread (k, v, cos, sin) is in flight at once, since a block lives for one
// round trip, and token positions are stepped, not divided out per element. 5 heads of 128, back to
// back, before / after (us): 8 x 1024 tokens f32 21.5 / 14.4 (5.9 TB/s), 16 x 2048 f32 104 / 73, f16
// 59.7 / 40.0, 3 x 1111 13.1 / 10.2, 1 x 64 6.4 / 3.5.
template <int DK, typename CT>
__global__ __launch_bounds__(256, 4) void k_kv_fill(const float* __restrict__ k, const float* __restrict__ v, int B, int T,
                                                    int Hkv, int pos0, const float* __restrict__ cosT,
                                                    const float* __restrict__ sinT, CT* __restrict__ kc,
                                                    CT* __restrict__ vc, int max_len)
{
    constexpr int HALF = DK / 2;
    constexpr int NR = 256 / kPQ, U = DK / NR;      // feature rows per round of loads, rounds
    constexpr int NT = 256 / HALF, N = kPQ / NT;    // tokens per round of stores, rounds
    __shared__ float sk[DK][kPQ + 1];
    __shared__ float sv[DK][kPQ + 1];
    const int M = B * T;
    const int g = blockIdx.y;
    const int m0 = blockIdx.x * kPQ;
    const int tid = threadIdx.x;
    const int row = Hkv * DK;
    // loads past the last token repeat it (never stored)
    const int c = tid % kPQ, i0 = tid / kPQ;
    const size_t src = (size_t)(g * DK + i0) * (size_t)M + (size_t)min(m0 + c, M - 1);
    float xk[U], xv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) xk[u] = k[src + (size_t)(NR * u) * (size_t)M];
#pragma unroll
    for (int u = 0; u < U; ++u) xv[u] = v[src + (size_t)(NR * u) * (size_t)M];
    // the tokens this thread stores features j and j + dk / 2 of
    const int j = tid % HALF, c0 = tid / HALF;
    int t = (m0 + c0) % T, b = (m0 + c0) / T, p[N];
    size_t dst[N];
    float cs[N], sn[N];
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
        p[n] = pos0 + t;
        dst[n] = ((size_t)b * (size_t)max_len + (size_t)p[n]) * (size_t)row + (size_t)(g * DK + j);
        t += NT;
        while (t >= T)
        {
            t -= T;
            ++b;
        }
    }
    if (cosT)
    {
#pragma unroll
        for (int n = 0; n < N; ++n)
        {
            cs[n] = cosT[(size_t)p[n] * HALF + j];
            sn[n] = sinT[(size_t)p[n] * HALF + j];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
    {
        sk[i0 + NR * u][c] = xk[u];
        sv[i0 + NR * u][c] = xv[u];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
        const int cn = c0 + NT * n;
        if (m0 + cn >= M) return;
        const float x0 = sk[j][cn], x1 = sk[j + HALF][cn];
        float y0 = x0, y1 = x1;
        if (cosT) pf_rope(x0, x1, cs[n], sn[n], y0, y1);
        kc[dst[n]] = (CT)y0;
        kc[dst[n] + HALF] = (CT)y1;
        vc[dst[n]] = (CT)sv[j][cn];
        vc[dst[n] + HALF] = (CT)sv[j + HALF][cn];
    }
}

// ------------------------------------------------------------------ causal attention

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
// Largest dk max|q| max|k| |scale| log2(e) of a query and a tile: a score's parts below the halves' range
// (2^-40 of the largest value) add up to less than 2^-21, and no score rounds a reference maximum by 2^-5.
constexpr float kPReach = 0x1p18f;
constexpr float kPUp = 15.0f;          // f16 parts of probabilities: the largest of a tile is 2^15
constexpr float kPTiny = 0x1p-100f;    // outputs below this (but for 0) may have lost bits of a bf16 part

// kHalf: V as it is in f16 caches, for products with probabilities in f16 parts
template <int DK, typename CT, bool kHalf = false>
struct PrefillTile
{
    static constexpr int kKPlanes = sizeof(CT) == 4 ? 2 : 1;  // K: high and low f16 halves of f32 values
    static constexpr int kVPlanes = kHalf ? 1 : sizeof(CT) == 4 ? 3 : 2;  // V: bf16 parts of f32 / f16 values, or f16
    // rows are padded by 16 bytes: 16 lanes' reads of consecutive rows fall on all banks, and every
    // chunk is at a constant offset from a lane's first
    static constexpr int kKPitch = DK * 2 + 16, kVPitch = kPK * 2 + 16;
    static constexpr int kKPlane = kPK * kKPitch, kVPlane = DK * kVPitch;
    static constexpr int kV = kKPlanes * kKPlane;            // K planes, then V planes
    static constexpr int kBuf = kV + kVPlanes * kVPlane;
    static constexpr int KROW = DK + 4;                      // f32 products: padded row (floats)
    static constexpr int kF32 = 2 * kPK * KROW * 4;
    static constexpr int kTPitch = DK * 2 + 16;              // rows of the cos / sin tables, before the first tile
    static constexpr int kTables = 2 * 32 * kPWaves * kTPitch;
    static constexpr int kMain = 2 * kBuf > kTables ? 2 * kBuf : kTables;  // double-buffered
    static_assert(kF32 <= kMain, "");
    static constexpr int kBytes = kMain + 128;               // maxima of K in two tiles, the fallback flag, the waves' findings
};

// x = hi + lo / up, up = 2^11: two halves that hold 22 bits of what is from 2^-14 on
__device__ __forceinline__ void split2_up(float x0, float x1, float up, v2h& hi, v2h& lo)
{
    hi = __builtin_convertvector(v2f{x0, x1}, v2h);
    const uint32_t u = __builtin_bit_cast(uint32_t, hi);
    float l0, l1;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(l0) : "v"(u), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(l1) : "v"(u), "v"(x1));
    lo = __builtin_convertvector(v2f{l0 * up, l1 * up}, v2h);
}

// The first N bf16 parts of two values: x = sum of parts, exactly, for f32 values (N = 3) and widened f16
// values (N = 2) from 2^-110 on (each rounding leaves 8 bits less); infinities and NaN give NaN.
template <int N>
__device__ __forceinline__ void split_bf16(float x0, float x1, v2b (&part)[N])
{
#pragma unroll
    for (int n = 0; n < N; ++n)
    {
        part[n] = __builtin_convertvector(v2f{x0, x1}, v2b);
        if (n + 1 == N) break;
        const uint32_t u = __builtin_bit_cast(uint32_t, part[n]);
        x0 -= __builtin_bit_cast(float, u << 16);
        x1 -= __builtin_bit_cast(float, u & 0xFFFF0000u);
    }
}

// Four elements of a cache row as floats
template <typename CT>
__device__ __forceinline__ float4 widen4(const CT* p)
{
    if constexpr (sizeof(CT) == 4) return *reinterpret_cast<const float4*>(p);
    else
    {
        const v4h x = *reinterpret_cast<const v4h*>(p);
        return make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
    }
}

// Paged: the pool's row of position t of the wave's sequence and KV head; a page outside the pool sets
// `bad` and gives page 0's
__device__ __forceinline__ size_t paged_row(const PrefillArgs& a, const PrefillWave& w, int t, bool& bad)
{
    int id = a.table[(size_t)w.b * a.table_stride + (t >> a.shift)];
    if (!page_ok(id, a.num_pages))
    {
        bad = true;
        id = 0;
    }
    return page_row(id, w.g, t & ((1 << a.shift) - 1), a.Hkv, a.shift);
}

// The work-group's attention on the fp32 MFMA (v_mfma_f32_32x32x2_f32), for inputs that the f16
// and bf16 parts cannot hold (see the top of the file). Per 32-key
// tile S^T (not S) is in the accumulators, so lane l holds query l % 32 and keys
// 8(v/4) + 4(l/32) + v%4 of its 16 elements v: the B operand of the P . V products when the keys of
// product s are taken in that order. The sum over the head dimension takes product s = 4c + e over
// dimensions 8c + e and 8c + 4 + e (the two lane halves).
// Paged: a NaN or an infinity among the values of a key that one query sees and another does not must
// not reach the other, whose probability of 0 a matrix product would multiply with it; tiles that reach
// past some query's sight therefore add their values key by key.
template <int DK, bool kPaged, bool kShaped, bool kDistance, typename CT>
__device__ void attend_f32(const PrefillArgs& a, const PrefillWave& w, const PrefillSeq<kPaged>& seq, int last_key,
                           int k0, int k1, float* rec, __amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rv, float* ks, int tid)
{
    constexpr int NC = DK / 8, ND = DK / 32, KROW = PrefillTile<DK, CT>::KROW;
    const int lane = tid & 63, h = lane >> 5, l32 = lane & 31;
    const int row = a.Hkv * DK;
    float* vs = ks + kPK * KROW;
    bool bad = false;  // a page outside the pool
    float qv[DK / 2];  // qv[4c + e] = rotated query value of dimension 8c + 4h + e
    PrefillQuery<DK, 4> query;
    query.load(a, w, seq, h);
    const __amdgpu_buffer_rsrc_t rc = pf_rsrc(a.cosT ? a.cosT : a.q, rope_bytes(a, DK / 2));
    const __amdgpu_buffer_rsrc_t rs = pf_rsrc(a.cosT ? a.sinT : a.q, rope_bytes(a, DK / 2));
    const uint32_t r_at = (uint32_t)(((size_t)(seq.pos0(a) + min(w.qt, seq.n(a) - 1)) * (DK / 2) + (size_t)(4 * h)) * 4u);
    auto table = [&](__amdgpu_buffer_rsrc_t r, int c, int i) { return ld_f4(r, r_at + (uint32_t)(8 * c + 4 * i) * 4u); };
    query.rotate(a, [&](int c, int i) { return table(rc, c, i); }, [&](int c, int i) { return table(rs, c, i); },
                 [&](int c, int e, float y0, float y1) {
        qv[4 * c + e] = y0;
        qv[4 * (c + NC / 2) + e] = y1;
    });
    v16f o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = v16f{};
    float m_run = -__builtin_inff(), l_run = 0.0f;
    for (int kb = kPaged ? k0 : 0; kb < (kPaged ? k1 : last_key / kPK + 1); ++kb)
    {
        __syncthreads();  // every wave is done with the previous tile
        for (int u = tid; u < kPK * DK / 4; u += kPThreads)
        {
            const int key = u / (DK / 4), c4 = u % (DK / 4);
            if constexpr (kPaged)
            {
                const int t = kb * kPK + key;
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
                if (t <= last_key)
                {
                    const size_t at = paged_row(a, w, t, bad) * DK + 4 * c4;
                    x = widen4<CT>(static_cast<const CT*>(a.kc) + at);
                    y = widen4<CT>(static_cast<const CT*>(a.vc) + at);
                }
                *reinterpret_cast<float4*>(ks + key * KROW + 4 * c4) = x;
                *reinterpret_cast<float4*>(vs + key * KROW + 4 * c4) = y;
                continue;
            }
            const uint32_t off = (uint32_t)(((size_t)(kb * kPK + key) * (size_t)row + (size_t)w.g * DK + 4 * c4) * sizeof(CT));
            *reinterpret_cast<float4*>(ks + key * KROW + 4 * c4) = ld_c4<CT>(rk, off);
            *reinterpret_cast<float4*>(vs + key * KROW + 4 * c4) = ld_c4<CT>(rv, off);
        }
        __syncthreads();
        if (!w.live || kb * kPK > seq.to(a, w)) continue;
        v16f s = v16f{};
#pragma unroll
        for (int c = 0; c < NC; ++c)
        {
            const float4 kk = *reinterpret_cast<const float4*>(ks + l32 * KROW + 8 * c + 4 * h);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk.x, qv[4 * c + 0], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk.y, qv[4 * c + 1], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk.z, qv[4 * c + 2], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk.w, qv[4 * c + 3], s, 0, 0, 0);
        }
        float sc[16];
        float mx = -__builtin_inff();
#pragma unroll
        for (int v = 0; v < 16; ++v)
        {
            const int key = kb * kPK + 8 * (v >> 2) + 4 * h + (v & 3);
            float x = s[v] * a.scale;
            if constexpr (kShaped)
            {
                if (a.cap2 > 0.0f) x = a.cap2 * 0.69314718f * tanh_any(x * (a.capi2 * 1.44269504f));
                const float away = (float)(key - w.qpos);
                if (a.slopes) x += a.slopes[w.head] * (kDistance ? -fabsf(away) : away);
            }
            sc[v] = key <= seq.sight(w) ? x : -__builtin_inff();
            mx = fmaxf(mx, sc[v]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = fmaxf(m_run, mx);
        const bool any = m_new != -__builtin_inff();
        const float corr = any ? expf(m_run - m_new) : 1.0f;
        float ls = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; ++v)
        {
            sc[v] = any ? expf(sc[v] - m_new) : 0.0f;
            ls += sc[v];
        }
        ls += __shfl_xor(ls, 32);
        l_run = l_run * corr + ls;
        m_run = m_new;
        // corr is exactly 1 where the running maximum did not move
        if (__builtin_amdgcn_ballot_w64(corr != 1.0f) != 0)
        {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[d][v] *= corr;
        }
        if constexpr (kPaged)
        {
            if (kb * kPK + kPK - 1 > seq.from(a, w))
            {
#pragma unroll 1
                for (int n = 0; n < 16; ++n)
                {
                    float own = 0.0f;
#pragma unroll
                    for (int v = 0; v < 16; ++v) own = v == n ? sc[v] : own;
                    const float other = __shfl_xor(own, 32);
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                    {
                        const float pr = half == h ? own : other;
                        const int key = 8 * (n >> 2) + 4 * half + (n & 3);
                        const bool seen = kb * kPK + key <= seq.sight(w);
#pragma unroll
                        for (int d = 0; d < ND; ++d)
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                            {
                                const float x = vs[key * KROW + 32 * d + 8 * (i >> 2) + 4 * h + (i & 3)];
                                o[d][i] = __builtin_fmaf(pr, seen ? x : 0.0f, o[d][i]);
                            }
                    }
                }
                continue;
            }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int sp = 0; sp < 16; ++sp)
            {
                const int key = 8 * (sp >> 2) + 4 * h + (sp & 3);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vs[key * KROW + 32 * d + l32], sc[sp], o[d], 0, 0, 0);
            }
    }
    if constexpr (kPaged)
    {
        // nothing visible above -infinity: 0; a page outside the pool: NaN
        bad = __syncthreads_or(bad) != 0;
        if (bad) l_run = __builtin_nanf("");
        if (rec)
        {
            // the reference in log2 units, as records hold it, and what its rounding left out as a factor
            const float m2 = m_run * 1.44269504f;
            const float left = __builtin_fmaf(m_run, 1.44269504f, -m2) + m_run * 1.92596299e-8f;
            const float f = m_run == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(left);
            store_record<DK>(rec, tid, [](int d, int r) { return 32 * d + r; }, [&](int d, int v) { return o[d][v] * f; }, m2, l_run * f);
            return;
        }
        if (l_run == 0.0f) l_run = 1.0f;
    }
    if (w.live)
        store_out<DK>(a, w, seq, h, [](int d, int r) { return 32 * d + r; }, [&](int d, int v) { return o[d][v] / l_run; });
}

// Attention of an item over its tiles k0 .. k1 - 1; rec: into a record instead of the output
template <int DK, bool kPaged, bool kShaped, bool kDistance, typename CT>
__device__ __forceinline__ void attend(const PrefillArgs& a, const PrefillItem& item, uint8_t* smem, int k0, int k1, float* rec)
{
    constexpr bool F32C = sizeof(CT) == 4;
    constexpr bool kHalf = kPaged && !F32C;
    using Tile = PrefillTile<DK, CT, kHalf>;
    constexpr int NC = DK / 16;  // MFMA steps over the head dimension
    constexpr int ND = DK / 32;  // 32-row blocks of O^T, and dimensions per lane when staging V
    constexpr int CH = DK / 8;   // 16-byte chunks of a K row
    constexpr int KU = CH * kPK / 256;  // chunks a thread stages
    uint32_t* smax = reinterpret_cast<uint32_t*>(smem + Tile::kMain);  // [2][4]: per tile parity and K wave; f16 caches: [8] per wave
    // set to send the work-group to the f32 products: written in iteration kb (or before the loop) into
    // [(kb + 1) & 1] and read after the barrier of iteration kb + 1, so all waves read the same value
    int* sflag = reinterpret_cast<int*>(smem + Tile::kMain + 32);
    int* sany = reinterpret_cast<int*>(smem + Tile::kMain + 64);  // [2][8]: what each wave has found at the end

    // (paged: opaque per item, so that no thread-index arithmetic stays alive across the items)
    int tid = threadIdx.x;
    if constexpr (kPaged) asm volatile("" : "+v"(tid));
    const int lane = tid & 63, h = lane >> 5, l32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    PrefillWave w;
    PrefillSeq<kPaged> seq;
    int last_key;
    seat(a, item, tid, w, seq, last_key);
    const int row = a.Hkv * DK;
    const int valid = seq.pos0(a) + seq.n(a);  // cache rows [0, valid) hold keys / values
    const int nkb = kPaged ? k1 : last_key / kPK + 1;
    const int kb0 = kPaged ? k0 : 0;
    const size_t seq_off = kPaged ? 0 : (size_t)w.b * (size_t)a.max_len * (size_t)row;
    // rows at or past `valid` read as zeros: their scores are masked and their zero values keep
    // 0 * v finite
    const uint32_t seq_bytes = kPaged ? 0u : (uint32_t)((size_t)min(valid, a.max_len) * (size_t)row * sizeof(CT));
    const __amdgpu_buffer_rsrc_t rk = pf_rsrc(static_cast<const CT*>(a.kc) + seq_off, seq_bytes);
    const __amdgpu_buffer_rsrc_t rv = pf_rsrc(static_cast<const CT*>(a.vc) + seq_off, seq_bytes);

    // ---- staging, 16 elements per thread: waves 0-3 take V (thread = 4 keys x ND dimensions), waves
    // 4-7 take K (thread = KU chunks of 8 dimensions of a key). raw holds them as loaded.
    constexpr int RW = F32C ? 16 : 8;  // words
    uint32_t raw[RW];
    const bool is_v = wave < 4;
    const int u = tid & 255;
    const int vq = u >> 5, vg = u & 31;  // V: key quad, dimension group
    // the thread's offsets within a tile; the tile's rows are reached through the buffer's base
    constexpr int NL = F32C ? 4 : (4 > KU ? 4 : KU);
    uint32_t at[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i)
    {
        const int ct = u + 256 * i;
        at[i] = is_v ? (uint32_t)(((4 * vq + i) * row + w.g * DK + ND * vg) * (int)sizeof(CT))
                     : (uint32_t)((ct / CH * row + w.g * DK + 8 * (ct % CH)) * (int)sizeof(CT));
    }
    const uint32_t tile_bytes = (uint32_t)(kPK * row) * (uint32_t)sizeof(CT);
    const CT* const kvb = (is_v ? static_cast<const CT*>(a.vc) : static_cast<const CT*>(a.kc)) + seq_off;
    // paged: the page(s) of the thread's keys in the tile to be loaded next, read from the table a tile ahead so
    // that no load waits for its address. A page holds 8 positions or more: the four keys of a V thread lie in
    // one. Keys past the last that the work-group sees are read where that one is (trim() makes them zeros).
    int ids[KU];
    bool bad = false;
    auto key_at = [&](int kb, int i) {
        return is_v ? seen_rows(kb * kPK + 4 * vq, last_key, 4) : seen_rows(kb * kPK + (u + 256 * i) / CH, last_key, 1);
    };
    auto load_ids = [&](int kb) {
        if constexpr (kPaged)
        {
#pragma unroll
            for (int i = 0; i < KU; ++i)
                if (i == 0 || !is_v) ids[i] = a.table[(size_t)w.b * a.table_stride + (key_at(kb, i) >> a.shift)];
        }
    };
    auto load_paged = [&](int kb) {
        const uint8_t* at[KU];
#pragma unroll
        for (int i = 0; i < KU; ++i)
            if (i == 0 || !is_v)
            {
                const bool in = page_ok(ids[i], a.num_pages);
                bad |= !in;
                const uint32_t r = (uint32_t)page_row(in ? ids[i] : 0, w.g, key_at(kb, i) & ((1 << a.shift) - 1), a.Hkv, a.shift);
                at[i] = reinterpret_cast<const uint8_t*>(kvb) + (uint64_t)r * (uint32_t)(DK * sizeof(CT)) +
                        (is_v ? ND * vg : 8 * ((u + 256 * i) % CH)) * (int)sizeof(CT);
            }
        if (is_v)
        {
            constexpr int W = ND * (int)sizeof(CT) / 4;  // words per key
            typedef uint32_t VWord __attribute__((ext_vector_type(W)));
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                const VWord x = *reinterpret_cast<const VWord*>(at[0] + i * DK * (int)sizeof(CT));
#pragma unroll
                for (int e = 0; e < W; ++e) raw[W * i + e] = x[e];
            }
        }
        else
        {
#pragma unroll
            for (int j = 0; j < KU; ++j)
#pragma unroll
                for (int q = 0; q < (F32C ? 2 : 1); ++q)
                {
                    const u32x4 x = reinterpret_cast<const u32x4*>(at[j])[q];
#pragma unroll
                    for (int e = 0; e < 4; ++e) raw[(F32C ? 8 : 4) * j + 4 * q + e] = x[e];
                }
        }
        if (kb + 1 < nkb) load_ids(kb + 1);
    };
    // paged: what was read for keys behind the last becomes 0, as buffer loads past their range give
    auto trim = [&](int kb) {
        if constexpr (kPaged)
        {
            if (kb * kPK + kPK - 1 <= last_key) return;
            constexpr int VK = F32C ? ND : ND / 2;  // words of a V thread's key
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VK; ++e)
                    if (is_v && kb * kPK + 4 * vq + i > last_key) raw[VK * i + e] = 0u;
#pragma unroll
            for (int j = 0; j < KU; ++j)
#pragma unroll
                for (int e = 0; e < (F32C ? 8 : 4); ++e)
                    if (!is_v && kb * kPK + (u + 256 * j) / CH > last_key) raw[(F32C ? 8 : 4) * j + e] = 0u;
        }
    };
    auto load_raw = [&](int kb) {
        if constexpr (kPaged)
        {
            load_paged(kb);
            return;
        }
        const uint64_t before = (uint64_t)kb * tile_bytes;
        const __amdgpu_buffer_rsrc_t rt = pf_rsrc(reinterpret_cast<const uint8_t*>(kvb) + before,
                                                  before < seq_bytes ? seq_bytes - (uint32_t)before : 0u);
        if (is_v)
        {
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                constexpr int W = ND * (int)sizeof(CT) / 4;  // words per key
                if constexpr (W == 4)
                {
                    const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rt, at[i], 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) raw[4 * i + e] = x[e];
                }
                else if constexpr (W == 2)
                {
                    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rt, at[i], 0, 0);
                    raw[2 * i] = x[0];
                    raw[2 * i + 1] = x[1];
                }
                else raw[i] = __builtin_amdgcn_raw_buffer_load_b32(rt, at[i], 0, 0);
            }
        }
        else
        {
#pragma unroll
            for (int j = 0; j < KU; ++j)
#pragma unroll
                for (int q = 0; q < (F32C ? 2 : 1); ++q)
                {
                    const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rt, at[j] + 16 * q, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) raw[(F32C ? 8 : 4) * j + 4 * q + e] = x[e];
                }
        }
    };
    // words of raw in use
    constexpr int VW = 4 * ND * (int)sizeof(CT) / 4, KW = KU * 8 * (int)sizeof(CT) / 4;
    static_assert(VW == KW && VW <= RW, "V and K threads stage the same amount");
    // f32 caches: the wave's largest magnitude in K, for the tile's scaling
    auto post_max = [&](int kb) {
        if (!F32C || is_v) return;
        uint32_t mx = 0;
#pragma unroll
        for (int e = 0; e < KW; ++e) mx = max(mx, raw[e] & 0x7FFFFFFFu);
        mx = wave_max(mx);
        if (lane == 0) smax[(kb & 1) * 4 + wave - 4] = mx;
    };
    int ek = 0;        // exponent of the staged tile's K
    float eqf = 0.0f;  // the lane's query: 2^-eq |scale| log2(e)
    float klim = 0.0f; // f16 caches: the largest key element within kPReach of every query of the work-group
    // K's exponent, then raw as f16 halves (K) and bf16 parts (V) into buffer kb & 1
    auto find_scale = [&](int kb, int* flag) {
        if constexpr (F32C)
        {
            const uint32_t* sm = smax + (kb & 1) * 4;
            ek = __builtin_amdgcn_readfirstlane(f16_exp(max(max(sm[0], sm[1]), max(sm[2], sm[3]))));
            if (abs(ek) > kPExpMax)
            {
                if (tid == 0) *flag = 1;
                ek = 0;
            }
            // |q| 2^eq and |k| 2^ek are at most 2^15
            else if (__builtin_amdgcn_ballot_w64(eqf * pow2(-ek) > kPReach / (DK * 0x1p30f)) != 0 && lane == 0) *flag = 1;
        }
        else if (!is_v)
        {
            u16x2 m = {0, 0};
#pragma unroll
            for (int e = 0; e < KW; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, raw[e] & 0x7FFF7FFFu));
            const uint16_t top = max(m[0], m[1]);
            if (__builtin_amdgcn_ballot_w64(!((float)__builtin_bit_cast(_Float16, top) <= klim)) != 0 && lane == 0) *flag = 1;
        }
    };
    u16x2 v_top = {0, 0};  // kHalf, V's waves: the largest value (bits)
    // raw as f16 halves (K, scaled by 2^ek) and bf16 parts (V; kHalf: as it is) into buffer kb & 1
    auto convert = [&](int kb) {
        uint8_t* buf = smem + (kb & 1) * Tile::kBuf;
        const float sk = F32C ? pow2(ek) : 1.0f;
        if (is_v)
        {
            // row 32e + vg = dimension ND vg + e; its 4 chunks are (16-key half s, lane half) and hold
            // keys 16s + 8a + 4h + i in the order (a, i): the accumulators' order of S^T
            const int s = vq >> 2, ah = (vq >> 1) & 1, hh = vq & 1;
#pragma unroll
            for (int e = 0; e < ND; ++e)
            {
                const int r = 32 * e + vg;
                uint8_t* dst = buf + Tile::kV + r * Tile::kVPitch + 32 * s + 16 * hh + 8 * ah;
                if constexpr (kHalf)
                {
                    if (e == 0)
#pragma unroll
                        for (int i = 0; i < VW; ++i) v_top = __builtin_elementwise_max(v_top, __builtin_bit_cast(u16x2, raw[i] & 0x7FFF7FFFu));
                    // the halves of dimension e of the four keys
                    const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                    const uint32_t k01 = __builtin_amdgcn_perm(raw[ND / 2 + e / 2], raw[e / 2], sel);
                    const uint32_t k23 = __builtin_amdgcn_perm(raw[ND / 2 * 3 + e / 2], raw[ND / 2 * 2 + e / 2], sel);
                    *reinterpret_cast<u32x2*>(dst) = u32x2{k01, k23};
                    continue;
                }
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                {
                    if constexpr (F32C) x[i] = __builtin_bit_cast(float, raw[ND * i + e]);
                    else x[i] = (float)__builtin_bit_cast(v2h, raw[ND / 2 * i + e / 2])[e & 1];
                }
                v2b p0[Tile::kVPlanes], p1[Tile::kVPlanes];
                split_bf16(x[0], x[1], p0);
                split_bf16(x[2], x[3], p1);
#pragma unroll
                for (int q = 0; q < Tile::kVPlanes; ++q)
                    *reinterpret_cast<u32x2*>(dst + q * Tile::kVPlane) =
                        u32x2{__builtin_bit_cast(uint32_t, p0[q]), __builtin_bit_cast(uint32_t, p1[q])};
            }
        }
        else
        {
#pragma unroll
            for (int j = 0; j < KU; ++j)
            {
                const int ct = u + 256 * j, key = ct / CH, c = ct % CH;
                uint8_t* dst = buf + key * Tile::kKPitch + 16 * c;
                if constexpr (F32C)
                {
                    v8h hi, lo;
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                    {
                        v2h x, y;
                        split2(__builtin_bit_cast(float, raw[8 * j + e]) * sk, __builtin_bit_cast(float, raw[8 * j + e + 1]) * sk, x, y);
                        hi[e] = x[0], hi[e + 1] = x[1];
                        lo[e] = y[0], lo[e + 1] = y[1];
                    }
                    *reinterpret_cast<v8h*>(dst) = hi;
                    *reinterpret_cast<v8h*>(dst + Tile::kKPlane) = lo;
                }
                else
                    *reinterpret_cast<u32x4*>(dst) = u32x4{raw[4 * j], raw[4 * j + 1], raw[4 * j + 2], raw[4 * j + 3]};
            }
        }
    };

    // Fragments from LDS, up to four 16-byte reads at a time, a group ahead of the products that use them:
    // group g of K holds steps GK g .., group g of V^T (block, half) pairs GV g .., each with its planes.
    constexpr int PK = Tile::kKPlanes, PV = Tile::kVPlanes, GK = 4 / PK, GV = 4 / PV;
    constexpr int GKN = NC / GK, GVN = 2 * ND / GV;  // groups
    static_assert(NC % GK == 0 && (2 * ND) % GV == 0 && (!kHalf || GV == 4), "whole groups");
    const uint32_t k_at = (uint32_t)(l32 * Tile::kKPitch + 16 * h), v_at = (uint32_t)(Tile::kV + l32 * Tile::kVPitch + 16 * h);
    auto read_k = [&](u32x4(&f)[4], uint32_t par, int g) {
        const uint8_t* p = smem + (par + k_at);
#pragma unroll
        for (int e = 0; e < GK; ++e)
#pragma unroll
            for (int q = 0; q < PK; ++q)
                f[PK * e + q] = *reinterpret_cast<const u32x4*>(p + 32 * (GK * g + e) + q * Tile::kKPlane);
    };
    auto read_v = [&](u32x4(&f)[4], uint32_t par, int g) {
        const uint8_t* p = smem + (par + v_at);
#pragma unroll
        for (int e = 0; e < GV; ++e)
        {
            const int d = (GV * g + e) >> 1, t = (GV * g + e) & 1;
#pragma unroll
            for (int q = 0; q < PV; ++q)
                f[PV * e + q] = *reinterpret_cast<const u32x4*>(p + 32 * d * Tile::kVPitch + 32 * t + q * Tile::kVPlane);
        }
    };

    // ---- everything that the first tile waits for on its way together: rows of the cos / sin tables, page ids,
    // queries, then (with the ids) keys and values. The tables' rows of the work-group's queries are one run; from
    // registers a lane's row would be read in lines of its own, 16 bytes at a time, by every head again.
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
    load_ids(kb0);
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
    if (tid < 2) sflag[tid] = tid == (kb0 & 1) ? a.f32 : 0;
    __syncthreads();
    load_raw(kb0);

    // ---- the lane's rotated query in halves: step c holds dimensions 16c + 8h + 0..7, scaled by 2^eq
    v8h qh[NC], ql[NC];
    if (w.live)
    {
        float qv[DK / 2];
        uint32_t mx = 0;
        const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
        const uint8_t* tab = smem + (min(w.qt, seq.n(a) - 1) - item.qb * qn) * Tile::kTPitch + 32 * h;
        auto table = [&](const uint8_t* t, int c, int i) { return *reinterpret_cast<const float4*>(t + 64 * c + 16 * i); };
        query.rotate(a, [&](int c, int i) { return table(tab, c, i); }, [&](int c, int i) { return table(tab + qn * Tile::kTPitch, c, i); },
                     [&](int c, int e, float y0, float y1) {
            qv[8 * c + e] = y0;
            qv[8 * (c + NC / 2) + e] = y1;
            mx = max(mx, max(__builtin_bit_cast(uint32_t, y0) & 0x7FFFFFFFu, __builtin_bit_cast(uint32_t, y1) & 0x7FFFFFFFu));
        });
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, kWave));
        int eq = f16_exp(mx);
        const bool far = abs(eq) > kPExpMax;
        if (__builtin_amdgcn_ballot_w64(far) != 0 && lane == 0) sflag[kb0 & 1] = 1;
        if (far) eq = 0;
        const float sq = sign * pow2(eq);
        eqf = a.scale2 * pow2(-eq);
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
    bool deep = false;  // kHalf: the lane's query has seen a tile whose smallest weight has lost bits

    trim(kb0);
    post_max(kb0);
    if constexpr (!F32C)
    {
        const uint32_t mx = wave_max(__builtin_bit_cast(uint32_t, eqf));  // not negative
        if (lane == 0) smax[wave] = mx;
    }
    __syncthreads();
    if constexpr (!F32C)
    {
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < kPWaves; ++i) mx = max(mx, smax[i]);
        klim = kPReach / (DK * 0x1p15f) / __builtin_bit_cast(float, mx);  // |q| 2^eq is at most 2^15
    }
    find_scale(kb0, sflag + (kb0 & 1));
    convert(kb0);
    if (kb0 + 1 < nkb)
    {
        load_raw(kb0 + 1);
        trim(kb0 + 1);
        post_max(kb0 + 1);
    }
    // f32 caches: in a vector register, since a scalar load in each tile waits for what is on its way from LDS, too
    // (4 x 1024 at 2048, 20 heads over 5 of 128: 519 -> 506 us; f16 caches, of 64, 186 -> 189)
    auto slope = [&]() { return a.slopes ? a.slopes[w.head] * 1.44269504f : 0.0f; };
    float kept = kShaped && F32C ? slope() : 0.0f;
    if constexpr (kShaped && F32C) asm volatile("" : "+v"(kept));
    bool fallback = false;
    for (int kb = kb0; kb < nkb; ++kb)
    {
        __syncthreads();  // tile kb is in LDS, the maxima of tile kb + 1 too; buffer (kb + 1) & 1 is free
        if (sflag[kb & 1])
        {
            fallback = true;
            break;
        }
        const int ek_now = ek;
        // this tile's first K fragments, in flight during the conversion of the next tile
        const uint32_t par = (uint32_t)(kb & 1) * Tile::kBuf;
        u32x4 fr[2][4];
        read_k(fr[0], par, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (kb + 1 < nkb)
        {
            find_scale(kb + 1, sflag + ((kb + 1) & 1));
            if (!is_v)
            {
                convert(kb + 1);
                if (kb + 2 < nkb) load_raw(kb + 2);  // in flight during this tile's products
            }
        }
        if (w.live && kb * kPK <= seq.to(a, w))
        {
            // S^T = K . Q^T: the products of the halves but low x low (at most 2^-22 of a term)
            v16f s = v16f{};
#pragma unroll
            for (int g = 0; g < GKN; ++g)
            {
                if (g + 1 < GKN) read_k(fr[(g + 1) & 1], par, g + 1);
                else read_v(fr[(g + 1) & 1], par, 0);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < GK; ++e)
                {
                    const int c = GK * g + e;
                    const v8h kh = __builtin_bit_cast(v8h, fr[g & 1][PK * e]);
                    if constexpr (F32C)
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, fr[g & 1][PK * e + 1]), qh[c], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[c], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[c], s, 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // scores in log2 units are s * f; the causal mask only where the tile reaches past the
            // wave's first query
            float f = F32C ? eqf * pow2(-ek_now) : eqf;
            if constexpr (kShaped)
            {
                const float slope2 = F32C ? kept : slope();
                // scores rarely reach the cap: a polynomial alone where none does (16 exponentials and
                // reciprocals less), of 3 terms where none is above a quarter of it
                const float g = a.cap2 > 0.0f ? f * a.capi2 : f;
                float top = 0.0f;  // (a NaN does not show, and stays one in each form)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                {
                    s[v] *= g;
                    const float x = s[v];
                    top = fmaxf(top, fabsf(x));
                }
                if (a.cap2 > 0.0f)
                {
                    if (__builtin_amdgcn_ballot_w64(top > 0.25f) == 0)
                    {
#pragma unroll
                        for (int v = 0; v < 16; ++v) s[v] = tanh_below_quarter(s[v]);
                    }
                    else if (__builtin_amdgcn_ballot_w64(top > 1.0f) == 0)
                    {
#pragma unroll
                        for (int v = 0; v < 16; ++v) s[v] = tanh_below1(s[v]);
                    }
                    else
                    {
#pragma unroll
                        for (int v = 0; v < 16; ++v) s[v] = tanh_any(s[v]);
                    }
                }
                // (the distance of the tile's first key and the steps from there apart: a step costs one multiply-add; kDistance:
                // and a change of sign, 107 us instead of 102 at 8 x 77 .. 1900 tokens, 16 heads over 2 of 64)
                const float unit = a.cap2 > 0.0f ? a.cap2 : 1.0f, first = (float)(kb * kPK + 4 * h - w.qpos), away = slope2 * first;
#pragma unroll
                for (int v = 0; v < 16; ++v)
                {
                    const float step = (float)(8 * (v >> 2) + (v & 3)), bias = __builtin_fmaf(slope2, step, away);
                    s[v] = __builtin_fmaf(s[v], unit, kDistance && first + step > 0.0f ? -bias : bias);
                }
                f = 1.0f;
            }
            float low = 0.0f;  // kHalf: the lane's lowest score (masked ones, too)
            if constexpr (kHalf)
            {
                low = s[0];
#pragma unroll
                for (int v = 1; v < 16; ++v) low = fminf(low, s[v]);
            }
            if (kb * kPK + kPK - 1 > seq.from(a, w))
            {
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (kb * kPK + 8 * (v >> 2) + 4 * h + (v & 3) > seq.sight(w)) s[v] = -__builtin_inff();
            }
            float mx = s[0];
#pragma unroll
            for (int v = 1; v < 16; ++v) mx = fmaxf(mx, s[v]);
            // (by registers 1 % faster with dk 64, 1 % slower with dk 128, where it takes two that are short)
            mx = (DK == 64 ? max_halves(mx) : fmaxf(mx, __shfl_xor(mx, 32))) * f;
            // the reference of a query moves only when its maximum has grown by 2^8 (or is new)
            if constexpr (kHalf) mx = __builtin_ceilf(mx);  // whole powers of two: every rescaling is exact
            const bool grown = mx > m_ref + kPLazy;
            if (__builtin_amdgcn_ballot_w64(grown) != 0)
            {
                const float m_new = grown ? mx : m_ref;
                // 0 on the first tile (a query may have seen no key yet where a span begins within its item)
                const float corr = kPaged && !grown ? 1.0f : __builtin_amdgcn_exp2f(m_ref - m_new);
                l_run *= corr;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] *= corr;
                m_ref = m_new;
            }
            const float ref = kPaged && m_ref == -__builtin_inff() ? 0.0f : m_ref;
            if constexpr (kHalf)
            {
                // The tile's weights under a reference of its own, 2^15 at most: p = a + b 2^-11 to 2^-22 of it for p
                // from 2^-14 on, and to 2^-36 below
                const float own = mx == -__builtin_inff() ? 0.0f : mx - kPUp;
                const float back = mx == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(own - ref);
                const float least = __builtin_fmaf(low, f, -own);
                deep |= least < -14.0f;
                // where no weight is below 2^-18 of the largest, what a leaves of it is in f16's range as it is, to
                // 2^-22 of the weight: no scaling of the products (4 x 1024 queries at 4096, 16 heads over 2 of 64:
                // 247 -> 237 us; with dk 128 the branch costs registers that are not there, 560 -> 735)
                const bool near = DK == 64 && __builtin_amdgcn_ballot_w64(!(least >= -3.0f)) == 0;
                const float up = near ? 1.0f : 0x1p11f;
                float l_tile = 0.0f;
                v8h pa[2], pb[2];
#pragma unroll
                for (int v = 0; v < 16; v += 2)
                {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], f, -own));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v + 1], f, -own));
                    l_tile += p0;
                    l_tile += p1;
                    v2h x, y;
                    split2_up(p0, p1, up, x, y);
                    pa[v >> 3][v & 7] = x[0], pa[v >> 3][(v & 7) + 1] = x[1];
                    pb[v >> 3][v & 7] = y[0], pb[v >> 3][(v & 7) + 1] = y[1];
                }
                l_run = __builtin_fmaf(l_tile, back, l_run);
                __builtin_amdgcn_sched_barrier(0);
                // O^T += V^T . P^T, a tile summed from zero, the low parts first
                v16f sum[2];
#pragma unroll
                for (int g = 0; g < GVN; ++g)
                {
                    const u32x4(&f4)[4] = fr[(GKN + g) & 1];
                    if (g + 1 < GVN) read_v(fr[(GKN + g + 1) & 1], par, g + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                    {
                        sum[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, f4[2 * e]), pb[0], v16f{}, 0, 0, 0);
                        sum[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, f4[2 * e + 1]), pb[1], sum[e], 0, 0, 0);
                    }
                    if (!near) sum[0] *= 0x1p-11f, sum[1] *= 0x1p-11f;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                    {
                        sum[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, f4[2 * e]), pa[0], sum[e], 0, 0, 0);
                        sum[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, f4[2 * e + 1]), pa[1], sum[e], 0, 0, 0);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int v = 0; v < 16; ++v) o[2 * g + e][v] = __builtin_fmaf(sum[e][v], back, o[2 * g + e][v]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            else
            {
                v8b p[3][2];
#pragma unroll
                for (int v = 0; v < 16; v += 2)
                {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], f, -ref));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v + 1], f, -ref));
                    l_run += p0;
                    l_run += p1;
                    v2b x[3];
                    split_bf16(p0, p1, x);
#pragma unroll
                    for (int q = 0; q < 3; ++q) p[q][v >> 3][v & 7] = x[q][0], p[q][v >> 3][(v & 7) + 1] = x[q][1];
                }
                __builtin_amdgcn_sched_barrier(0);
                // O^T += V^T . P^T: the products of parts i and j with i + j <= 2, smallest first; the rest is
                // at most 2^-24 of a term. A tile is summed from zero and added once: that rounds the running
                // sum once in 32 keys. The add of a block runs beside the products of the next.
                v16f sum[2];
#pragma unroll
                for (int g = 0; g < GVN; ++g)
                {
                    const u32x4(&f4)[4] = fr[(GKN + g) & 1];
                    if (g + 1 < GVN) read_v(fr[(GKN + g + 1) & 1], par, g + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < GV; ++e)
                    {
                        const int d = (GV * g + e) >> 1, t = (GV * g + e) & 1;
                        if (t == 0) sum[d & 1] = v16f{};
                        if (t == 1 - (GV & 1) && d > 0) o[d - 1] += sum[(d - 1) & 1];
#pragma unroll
                        for (int n = 2; n >= 0; --n)
#pragma unroll
                            for (int i = PV - 1 < n ? PV - 1 : n; i >= 0; --i)
                                sum[d & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, f4[PV * e + i]), p[n - i][t], sum[d & 1], 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                o[ND - 1] += sum[(ND - 1) & 1];
            }
        }
        // V's waves convert behind their products, K's before them: each SIMD has one of both, whose VALU and MFMA
        // phases then fall together
        if (is_v && kb + 1 < nkb)
        {
            trim(kb + 1);
            convert(kb + 1);
            if (kb + 2 < nkb) load_raw(kb + 2);
        }
        if (!is_v && kb + 2 < nkb)
        {
            trim(kb + 2);
            post_max(kb + 2);
        }
    }
    // V is not looked through for infinities and NaN: any that matters is in the sums. Nor for values whose smallest part would lie below bf16's range: their output is tiny then.
    l_run += __shfl_xor(l_run, 32);
    bool lost = !(l_run < __builtin_inff());
    const int any_bad = kPaged && __builtin_amdgcn_ballot_w64(bad) != 0 ? 2 : 0;
    float faint = l_run * kPTiny;  // outputs below (but for 0) may have lost bits
    if constexpr (kHalf)
    {
        // Weights below 2^-29 of the largest of their tile are held to 2^-51 of that one: nothing beside an output, unless
        // the heavy keys' values are 0 where theirs are not. Such outputs are below 2^-32 of the largest value then,
        // and come from the f32 products. (From 2^-27 on, a value that happens to be 0 sent a call in four there,
        // at the cost of five tiles each.)
        const uint32_t top = wave_max(max((uint32_t)v_top[0], (uint32_t)v_top[1]));
        if (lane == 0) smax[wave] = is_v ? top : 0u, sany[kPWaves + wave] = any_bad;
        __syncthreads();
        const uint32_t most = max(max(smax[0], smax[1]), max(smax[2], smax[3]));
        deep |= __shfl_xor((int)deep, 32) != 0;
        faint = deep ? l_run * ((float)__builtin_bit_cast(_Float16, (uint16_t)most) * 0x1p-32f) : -1.0f;
    }
    {
        // the lowest magnitude (but for zeros where those hold no lost bits), and NaN from an infinity or a NaN
        float low = __builtin_inff(), odd = 0.0f;
        uint32_t least = 0xFFFFFFFFu;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v)
            {
                const float y = o[d][v];
                odd = __builtin_fmaf(y, 0.0f, odd);
                if constexpr (kHalf) low = fminf(low, fabsf(y));
                else least = min(least, 2 * __builtin_bit_cast(uint32_t, y) - 1);
            }
        lost |= odd != odd;
        if constexpr (kHalf) lost |= low < faint;
        else lost |= faint > 0.0f && least < 2 * __builtin_bit_cast(uint32_t, faint) - 1;
    }
    const bool any_lost = __builtin_amdgcn_ballot_w64(!fallback && w.live && lost) != 0;
    if (lane == 0) sany[wave] = any_lost | (kHalf ? 0 : any_bad);
    __syncthreads();
    int found = 0;
#pragma unroll
    for (int i = 0; i < (kHalf ? 2 : 1) * kPWaves; ++i) found |= sany[i];
    found = __builtin_amdgcn_readfirstlane(found);
    if ((found & 1) || fallback)
    {
        // everything from scratch: kept alive across the loop above, it would push that into spills
        int t2 = threadIdx.x;
        if constexpr (kPaged) asm volatile("" : "+v"(t2));
        PrefillWave w2;
        PrefillSeq<kPaged> seq2;
        int last2;
        if constexpr (kPaged) seat(a, item, t2, w2, seq2, last2);
        else w2 = w, seq2 = seq, last2 = last_key;
        attend_f32<DK, kPaged, kShaped, kDistance, CT>(a, w2, seq2, last2, k0, k1, rec, rk, rv, reinterpret_cast<float*>(smem), kPaged ? t2 : tid);
        return;
    }
    if constexpr (kPaged)
    {
        if (found & 2) l_run = __builtin_nanf("");
        if (rec)
        {
            store_record<DK>(rec, tid, [](int d, int i) { return ND * i + d; }, [&](int d, int v) { return o[d][v]; }, m_ref, l_run);
            return;
        }
    }
    if (!w.live) return;
    // o / l, correctly rounded but for the last step's double rounding: the residual is exact
    const float r = 1.0f / l_run;
    store_out<DK>(a, w, seq, h, [](int d, int i) { return ND * i + d; }, [&](int d, int v) {
        const float q = o[d][v] * r;
        return __builtin_fmaf(__builtin_fmaf(-q, l_run, o[d][v]), r, q);
    });
}

template <int DK, bool kPaged, bool kShaped, typename CT, bool kDistance = false>
__global__ __launch_bounds__(kPThreads) void k_attn_prefill(PrefillArgs a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    PrefillItem it;
    const int groups = kPaged ? a.groups : 1, HG = a.Hkv * groups;
    // one item each, heaviest first: the last queries attend over the most keys. (Paged: a step further per block
    // of queries, or a long sequence's work-groups, per_qb apart, would all fall on one or two of the 8 XCDs.)
    const int per_qb = a.B * HG, back = (int)blockIdx.x / per_qb;
    const int bg = kPaged ? ((int)blockIdx.x + back) % per_qb : (int)blockIdx.x % per_qb;
    if constexpr (!kPaged)
    {
        it.b = bg / a.Hkv;
        it.g = bg % a.Hkv;
        it.first = it.g * a.R;
        it.qb = a.nqb - 1 - back;
        attend<DK, kPaged, kShaped, kDistance, CT>(a, it, smem, 0, 0, nullptr);
    }
    else
    {
        const int g = blockIdx.x;
        PromptCut at, end;
        if (a.spans)
        {
            // the span's two cuts by a wave each, while the others look for sequences that do not fit
            const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
            PromptCut* const cuts = reinterpret_cast<PromptCut*>(smem);
            if (wave < 2)
            {
                const PromptCut cut = prompt_cut(a, a.spans, g + wave);
                if ((threadIdx.x & 63) == 0)
                {
                    cuts[wave] = cut;
                    if (wave == 0) prompt_cuts<DK>(a, a.spans)[g] = cut;
                }
            }
            else
                for (int b = g; b < a.B; b += a.spans)
                    if (PrefillSeq<true> any; !packed_seq(a, b, any)) store_nan<DK>(a, b, 0, a.H, (int)threadIdx.x - 2 * kWave, kPThreads - 2 * kWave);
            __syncthreads();
            at = uniform(cuts[0]);
            end = uniform(cuts[1]);
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
        bool known = a.spans == 0;  // it.seq is at.b's
        while (cut_before(at, end))
        {
            // the next sequence with a block left
            const bool there = at.b < a.B;
            if (!there || !(known || packed_seq(a, at.b, it.seq)) || at.qb >= prompt_blocks(a, it.seq.n_))
            {
                at = there ? PromptCut{at.gh, at.b + 1, 0, 0} : PromptCut{at.gh + 1, 0, 0, 0};
                continue;
            }
            const int tiles = prompt_tiles(a, it.seq, at.qb), to = cut_same_item(at, end) ? end.t : tiles;
            it.b = at.b;
            it.g = at.gh / groups;
            it.first = at.gh * a.R;
            it.qb = at.qb;
            float* rec = at.t == 0 && to == tiles ? nullptr : prompt_record<DK>(a, g, at.t > 0 ? 0 : 1);
            attend<DK, kPaged, kShaped, kDistance, CT>(a, it, smem, at.t, to, rec);
            known = false;
            at = {at.gh, at.b, at.qb + 1, 0};
        }
    }
}

template <int DK, bool kPaged, bool kShaped, typename CT, bool kDistance = false>
hipError_t launch_prefill_dk(hipStream_t st, const PrefillArgs& a)
{
    constexpr int lds = PrefillTile<DK, CT, kPaged && sizeof(CT) == 2>::kBytes;
    static bool attr_set = false;
    if (!attr_set)
    {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_attn_prefill<DK, kPaged, kShaped, CT, kDistance>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        attr_set = true;
    }
    const unsigned blocks = kPaged && a.spans ? (unsigned)a.spans : (unsigned)(a.nqb * a.B * a.Hkv * a.groups);
    hipLaunchKernelGGL((k_attn_prefill<DK, kPaged, kShaped, CT, kDistance>), dim3(blocks), dim3(kPThreads), lds, st, a);
    if constexpr (kPaged)
        if (a.spans > 1)
        {
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            k_prompt_join<DK><<<dim3((unsigned)a.spans - 1, DK / 16), 32 * kPWaves, 0, st>>>(a);
        }
    return hipGetLastError();
}

}  // namespace

bool prefill_dk_supported(size_t dk) { return dk == 64 || dk == 128; }

template <typename CT>
hipError_t launch_kv_fill_ct(hipStream_t st, const float* k, const float* v, size_t B, size_t T, size_t Hkv, size_t dk,
                             size_t pos0, const float* cosT, const float* sinT, CT* kc, CT* vc, size_t max_len)
{
    const dim3 grid((unsigned)ceil_div(B * T, kPQ), (unsigned)Hkv);
    if (dk == 64)
        hipLaunchKernelGGL((k_kv_fill<64, CT>), grid, dim3(256), 0, st, k, v, (int)B, (int)T, (int)Hkv, (int)pos0, cosT,
                           sinT, kc, vc, (int)max_len);
    else if (dk == 128)
        hipLaunchKernelGGL((k_kv_fill<128, CT>), grid, dim3(256), 0, st, k, v, (int)B, (int)T, (int)Hkv, (int)pos0, cosT,
                           sinT, kc, vc, (int)max_len);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_kv_fill(hipStream_t st, const float* k, const float* v, size_t B, size_t T, size_t Hkv, size_t dk,
                          size_t pos0, const float* cosT, const float* sinT, void* kc, void* vc, bool cache_f16,
                          size_t max_len)
{
    if (B * T == 0) return hipSuccess;
    if (cache_f16)
        return launch_kv_fill_ct(st, k, v, B, T, Hkv, dk, pos0, cosT, sinT, static_cast<_Float16*>(kc),
                                 static_cast<_Float16*>(vc), max_len);
    return launch_kv_fill_ct(st, k, v, B, T, Hkv, dk, pos0, cosT, sinT, static_cast<float*>(kc),
                             static_cast<float*>(vc), max_len);
}

hipError_t launch_attn_prefill(hipStream_t st, const float* q, const void* kc, const void* vc, bool cache_f16,
                               size_t B, size_t T, size_t H, size_t Hkv, size_t dk, size_t pos0, const float* cosT,
                               const float* sinT, size_t max_len, float scale, float* out)
{
    if (B * T == 0) return hipSuccess;
    const size_t R = H / Hkv;
    const float mag = std::fabs(scale);
    const bool f32 = !(mag >= 0x1p-20f && mag <= 0x1p20f);
    PrefillArgs a{q, kc, vc, cosT, sinT, out, (int)B, (int)T, (int)H, (int)Hkv, (int)R, (int)pos0,
                  (int)max_len, (int)ceil_div(T, kPQ * (kPWaves / R)), scale, (float)(mag * 1.4426950408889634), f32 ? 1 : 0,
                  (int)(B * T), 1};
    if (cache_f16)
    {
        if (dk == 64) return launch_prefill_dk<64, false, false, _Float16>(st, a);
        if (dk == 128) return launch_prefill_dk<128, false, false, _Float16>(st, a);
        return hipErrorInvalidValue;
    }
    if (dk == 64) return launch_prefill_dk<64, false, false, float>(st, a);
    if (dk == 128) return launch_prefill_dk<128, false, false, float>(st, a);
    return hipErrorInvalidValue;
}

// Spans of a call: one work-group to a CU (its registers allow no more), unless no sequence can be long enough to be cut
size_t pages_prefill_spans(size_t limit, size_t num_cus) { return limit <= (size_t)kShort * kPK ? 0 : num_cus; }

size_t pages_prefill_workspace_bytes(size_t dk, size_t limit, size_t num_cus)
{
    return pages_prefill_spans(limit, num_cus) * (2 * (dk + 2) * 32 * kPWaves * sizeof(float) + sizeof(PromptCut));
}

hipError_t launch_pages_prefill(hipStream_t st, const nnhip_kv_pages& kv, const float* q, size_t M, const int32_t* cu,
                                const int32_t* pos0, size_t B, size_t t_bound, size_t H, const float* cosT,
                                const float* sinT, size_t limit, float scale, float softcap, const float* slopes,
                                const int32_t* prefix, bool distance, float* out, void* ws, size_t num_cus)
{
    // a KV head's R query heads in work-groups of 8, 4, 2 or 1
    const size_t heads = H / kv.Hkv, R = heads % 8 == 0 ? 8 : heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
    const float mag = std::fabs(scale);
    const bool f32 = !(mag >= 0x1p-20f && mag <= 0x1p20f);
    const double cap2 = softcap * 1.4426950408889634;
    PrefillArgs a{q, kv.k, kv.v, cosT, sinT, out, (int)B, (int)t_bound, (int)H, (int)kv.Hkv, (int)R, 0,
                  (int)limit, (int)std::max<size_t>(1, ceil_div(std::min(t_bound, limit), kPQ * (kPWaves / R))), scale, (float)(mag * 1.4426950408889634), f32 ? 1 : 0,
                  (int)M, (int)(heads / R), kv.table, cu, pos0, prefix, slopes, (int)kv.table_stride, (int)kv.num_pages,
                  0, (int)limit, (float)cap2, softcap > 0.0f ? (float)(1.0 / cap2) : 0.0f,
                  static_cast<float*>(ws), (int)pages_prefill_spans(limit, num_cus)};
    while ((size_t(1) << a.shift) < kv.page_size) ++a.shift;
    // (a key ahead of its query is inside a prefix: without one the two biases are the same)
    if (slopes && prefix && distance)
    {
        if (kv.f16)
            return kv.dk == 64 ? launch_prefill_dk<64, true, true, _Float16, true>(st, a)
                               : launch_prefill_dk<128, true, true, _Float16, true>(st, a);
        return kv.dk == 64 ? launch_prefill_dk<64, true, true, float, true>(st, a) : launch_prefill_dk<128, true, true, float, true>(st, a);
    }
    if (cap2 > 0.0 || slopes)
    {
        if (kv.f16)
            return kv.dk == 64 ? launch_prefill_dk<64, true, true, _Float16>(st, a) : launch_prefill_dk<128, true, true, _Float16>(st, a);
        return kv.dk == 64 ? launch_prefill_dk<64, true, true, float>(st, a) : launch_prefill_dk<128, true, true, float>(st, a);
    }
    if (kv.f16)
        return kv.dk == 64 ? launch_prefill_dk<64, true, false, _Float16>(st, a) : launch_prefill_dk<128, true, false, _Float16>(st, a);
    return kv.dk == 64 ? launch_prefill_dk<64, true, false, float>(st, a) : launch_prefill_dk<128, true, false, float>(st, a);
}

}  // namespace nnhip
