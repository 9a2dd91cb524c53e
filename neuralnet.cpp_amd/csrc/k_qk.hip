// k_qk.hip — RMSNorm of every head of queries and keys and the rotation at each token's position, in one pass:
//   y = (x * rinv) * gain,  rinv = 1 / sqrt(sum x^2 * fl(1/dk) + eps) over the head's dk elements,
//   (y[j], y[j + dk/2]) turned by the angle of pair j at the token's position,
// each step rounded as nnhip_rmsnorm and the caches' rotation round it; the sum's order is the kernel's own. Bound
// by HBM (8 bytes an element); in the caller's two passes it would be 16.
#include "pages_split.hpp"
#include "token_quant.hpp"

#include <algorithm>

namespace nnhip
{
namespace
{

typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));

struct QkArgs
{
    const float* x[2];     // queries, keys
    float* y[2];
    const float* gain[2];  // (dk), or null
    int heads[2];
    const int32_t* pos;
    const float* cosT;
    const float* sinT;
    int M, rope_len;
    int per;               // heads of a work-group (columns)
    float eps;
};

// A pair of elements, normalized and rotated
__device__ __forceinline__ void qk_pair(float& x0, float& x1, float rinv, float g0, float g1, bool rope, float c, float s)
{
    x0 = __fmul_rn(__fmul_rn(x0, rinv), g0);
    x1 = __fmul_rn(__fmul_rn(x1, rinv), g1);
    if (rope) pg_rope(x0, x1, c, s, x0, x1);
}

// Token-major: dk / 8 lanes to a head, four pairs each. 16 tokens of 20 + 5 heads of 128: 3.0 us, a launch's latency.
template <int DK>
__global__ __launch_bounds__(256) void k_qk_tokens(QkArgs a)
{
    constexpr int L = DK / 8, HALF = DK / 2;
    const int all = a.heads[0] + a.heads[1];
    const int64_t unit = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;  // (token, head)
    const int i = threadIdx.x % L;
    if (unit >= (int64_t)a.M * all) return;
    const int m = (int)(unit / all), hh = (int)(unit - (int64_t)m * all), z = hh >= a.heads[0], head = z ? hh - a.heads[0] : hh;
    const size_t at = ((size_t)m * a.heads[z] + head) * DK + (size_t)(4 * i);
    v4fu x0 = *reinterpret_cast<const v4fu*>(a.x[z] + at), x1 = *reinterpret_cast<const v4fu*>(a.x[z] + at + HALF);
    const int p = a.pos ? a.pos[m] : 0;
    v4fu g0 = {1.0f, 1.0f, 1.0f, 1.0f}, g1 = g0, c = g0, s = g0;
    if (a.gain[z])
    {
        g0 = *reinterpret_cast<const v4fu*>(a.gain[z] + 4 * i);
        g1 = *reinterpret_cast<const v4fu*>(a.gain[z] + 4 * i + HALF);
    }
    const bool rope = a.cosT != nullptr, past = rope && p >= a.rope_len;
    if (p < 0) return;
    if (rope && !past)
    {
        c = *reinterpret_cast<const v4fu*>(a.cosT + (size_t)p * HALF + 4 * i);
        s = *reinterpret_cast<const v4fu*>(a.sinT + (size_t)p * HALF + 4 * i);
    }
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = __builtin_fmaf(x1[e], x1[e], __builtin_fmaf(x0[e], x0[e], sum));
#pragma unroll
    for (int off = 1; off < L; off <<= 1) sum += __shfl_xor(sum, off, kWave);
    const float rinv = past ? __builtin_nanf("") : rms_inv_of(sum, 1.0f / DK, a.eps);
#pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        float u = x0[e], v = x1[e];
        qk_pair(u, v, rinv, g0[e], g1[e], rope && !past, c[e], s[e]);
        x0[e] = u, x1[e] = v;
    }
    *reinterpret_cast<v4fu*>(a.y[z] + at) = x0;
    *reinterpret_cast<v4fu*>(a.y[z] + at + HALF) = x1;
}

// Feature-major: work-group = 128 columns of `per` heads, lane = two columns, wave = an eighth of the dimension pairs, whose
// cosines and sines stay in registers over the heads. Neighbouring blocks of columns go to one XCD: rows do not begin at the
// lines of the L2, and a line that two blocks share is written back once. 16 x 1111 .. 2048 tokens of 20 + 5 heads of 128: 148 us,
// 4.4 TB/s (a copy: 4.9); 64 columns in any order 193, with the next head's elements on their way during a head 150, non-temporal 164 .. 171.
template <int DK>
__global__ __launch_bounds__(512) void k_qk_columns(QkArgs a)
{
    constexpr int HALF = DK / 2, NP = DK / 16;
    typedef float v2fu __attribute__((ext_vector_type(2), aligned(4)));
    __shared__ float2 sum_s[2][8][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = xcd_run(blockIdx.x, gridDim.x) * 128 + 2 * lane;
    // the last columns: pairs that end at column M - 1 or a column of its own
    const int mc = min(m, max(a.M - 2, 0));
    const int shift = m - mc;  // 0; 1: the lane's first column is the pair's second; more: none
    const int all = a.heads[0] + a.heads[1], h0 = (int)blockIdx.y * a.per, h1 = min(h0 + a.per, all);
    const size_t step = (size_t)a.M;
    auto offset = [&](int hh) {
        return ((size_t)((hh >= a.heads[0] ? hh - a.heads[0] : hh) * DK + w * NP)) * step + (size_t)mc;
    };
    v2fu x[2][NP];
    auto load = [&](int hh) {
        const float* const src = a.x[hh >= a.heads[0]] + offset(hh);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < NP; ++i)
            {
                const float* const at = src + (size_t)(HALF * q + i) * step;
                if (a.M > 1) x[q][i] = *reinterpret_cast<const v2fu*>(at);
                else x[q][i] = v2fu{at[0], 0.0f};
            }
    };
    load(h0);
    const bool rope = a.cosT != nullptr;
    bool past[2], live[2];
    float c[2][NP], s[2][NP];
#pragma unroll
    for (int e = 0; e < 2; ++e)
    {
        const int at = mc + e, p = a.pos ? a.pos[min(at, a.M - 1)] : 0;
        past[e] = rope && p >= a.rope_len;
        live[e] = at < a.M && e >= shift && shift < 2 && p >= 0;
        if (rope)
        {
            const size_t r = (size_t)(past[e] ? 0 : max(p, 0)) * HALF + (size_t)(w * NP);
#pragma unroll
            for (int i = 0; i < NP; i += 4)
            {
                const v4fu y = *reinterpret_cast<const v4fu*>(a.cosT + r + i), z = *reinterpret_cast<const v4fu*>(a.sinT + r + i);
#pragma unroll
                for (int k = 0; k < 4; ++k) c[e][i + k] = y[k], s[e][i + k] = z[k];
            }
        }
    }
    for (int hh = h0; hh < h1; ++hh)
    {
        const int z = hh >= a.heads[0];
        if (hh != h0) load(hh);
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < NP; ++i) sum[e] = __builtin_fmaf(x[1][i][e], x[1][i][e], __builtin_fmaf(x[0][i][e], x[0][i][e], sum[e]));
        float2(&part)[8][64] = sum_s[hh & 1];
        part[w][lane] = make_float2(sum[0], sum[1]);
        lds_barrier();
        sum[0] = sum[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            const float2 y = part[i][lane];
            sum[0] += y.x, sum[1] += y.y;
        }
        float rinv[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) rinv[e] = past[e] ? __builtin_nanf("") : rms_inv_of(sum[e], 1.0f / DK, a.eps);
        float* const dst = a.y[z] + offset(hh);
        const float* const gain = a.gain[z] ? a.gain[z] + w * NP : nullptr;
#pragma unroll
        for (int i = 0; i < NP; ++i)
        {
            const float g0 = gain ? gain[i] : 1.0f, g1 = gain ? gain[i + HALF] : 1.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e)
            {
                float u = x[0][i][e], v = x[1][i][e];
                qk_pair(u, v, rinv[e], g0, g1, rope, rope ? c[e][i] : 1.0f, rope ? s[e][i] : 0.0f);
                x[0][i][e] = u, x[1][i][e] = v;
            }
            float* const lo = dst + (size_t)i * step;
            float* const hi = dst + (size_t)(HALF + i) * step;
            if (live[0] && live[1])
            {
                *reinterpret_cast<v2fu*>(lo) = x[0][i];
                *reinterpret_cast<v2fu*>(hi) = x[1][i];
            }
            else
            {
                if (live[0]) lo[0] = x[0][i][0], hi[0] = x[1][i][0];
                if (live[1]) lo[1] = x[0][i][1], hi[1] = x[1][i][1];
            }
        }
    }
}

template <int DK>
hipError_t launch_qk_dk(hipStream_t st, QkArgs a, bool tokens, size_t num_cus)
{
    const size_t all = (size_t)a.heads[0] + (size_t)a.heads[1];
    if (tokens) k_qk_tokens<DK><<<(unsigned)ceil_div((size_t)a.M * all, (size_t)(256 / (DK / 8))), 256, 0, st>>>(a);
    else
    {
        // heads of a work-group: as many (up to 5: a head's share of the rotation's tables is a fifth of its elements
        // then; 16 x 1111 .. 2048 tokens: 5 149.9 us, 3 152.4, 7 160.4) as leave three work-groups to a CU
        const size_t blocks = ceil_div((size_t)a.M, (size_t)128);
        size_t per = 5;
        while (per > 1 && blocks * ceil_div(all, per) < 3 * num_cus) --per;
        a.per = (int)per;
        k_qk_columns<DK><<<dim3((unsigned)blocks, (unsigned)ceil_div(all, per)), 512, 0, st>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_qk_norm_rope(hipStream_t st, const float* q, const float* k, size_t M, size_t H, size_t Hkv, size_t dk,
                               const float* gq, const float* gk, float eps, const int32_t* pos, const float* cosT,
                               const float* sinT, size_t rope_len, bool tokens, float* q_out, float* k_out, size_t num_cus)
{
    const QkArgs a{{q, k}, {q_out, k_out}, {gq, gk}, {q ? (int)H : 0, k ? (int)Hkv : 0}, pos, cosT, sinT, (int)M,
                   (int)std::min<size_t>(rope_len, 0x7FFFFFFF), 1, eps};
    if (dk == 64) return launch_qk_dk<64>(st, a, tokens, num_cus);
    if (dk == 128) return launch_qk_dk<128>(st, a, tokens, num_cus);
    if (dk == 256) return launch_qk_dk<256>(st, a, tokens, num_cus);
    return hipErrorInvalidValue;
}

}  // namespace nnhip
