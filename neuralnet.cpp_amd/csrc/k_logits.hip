// k_logits.hip — penalties for repeated tokens, biases and grammar masks on a batch's logits, and the
// greedy choice behind them, in one pass over the logits.
//
// Reference: the greedy rule of compute_layer_base.hpp:1152-1160 (k_argmax of k_decode.hip); the
// reference has no rules before it.
#include "common.hpp"
#include "pages_index.hpp"

#include <algorithm>

namespace nnhip
{
namespace
{

constexpr int kLgSlices = 64; // at most, of a row

// What a slice of a row found: its best value (index -1: none), and its first allowed token as
// 2 * index + (its value is NaN)
struct LogitBest
{
    float v;
    int i;
    uint32_t first;
    uint32_t pad;
};

struct LogitArgs
{
    const float* x;
    nnhip_logit_rules r;
    float* out;
    int32_t* ids;
    int32_t* pos;
    LogitBest* part;
    int V, slices;
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // dword-aligned 16-byte accesses
typedef int32_t i32x4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void take(LogitBest& a, const LogitBest& o)
{
    if (o.i >= 0 && (a.i < 0 || o.v > a.v || (o.v == a.v && o.i < a.i)))
    {
        a.v = o.v;
        a.i = o.i;
    }
    a.first = min(a.first, o.first);
}

__device__ __forceinline__ LogitBest wave_best(LogitBest a)
{
    for (int off = 32; off >= 1; off >>= 1)
    {
        LogitBest o;
        o.v = __shfl_xor(a.v, off, kWave);
        o.i = __shfl_xor(a.i, off, kWave);
        o.first = (uint32_t)__shfl_xor((int)a.first, off, kWave);
        take(a, o);
    }
    return a;
}

// The reference's loop starts from the first allowed token: a NaN there is never replaced.
__device__ __forceinline__ void choose(const LogitArgs& a, int b, const LogitBest& best)
{
    const int id = best.first == 0xFFFFFFFFu ? -1 : (best.first & 1u) ? (int)(best.first >> 1) : best.i;
    a.ids[b] = id;
    if (id < 0 || (a.pos && a.pos[b] < 0)) return;
    if (a.r.count_choice && a.r.counts) a.r.counts[(size_t)b * a.V + id] += 1;
    if (a.pos) a.pos[b] += 1;
}

// Work-group = a slice of row b in groups of 4 logits. Bound by HBM: logits, counts, biases and masks
// read once, the adjusted logits written once (256 rows of 131071 with every rule: 82.3 us, 4.9 TB/s, a large
// copy's rate), and by a round trip where rows are short (16 x 10000: 6.7 us a call).
template <int T, int U>
__global__ __launch_bounds__(T) void k_logits_adjust(LogitArgs a)
{
    __shared__ LogitBest best_s[T / kWave];
    const int b = blockIdx.y, tid = threadIdx.x, V = a.V;
    const int groups = (V + 3) / 4;
    const int per = (groups + a.slices - 1) / a.slices;
    const int i0 = blockIdx.x * per, i1 = min(groups, i0 + per);
    const float* x = a.x + (size_t)b * V;
    const int32_t* counts = a.r.counts ? a.r.counts + (size_t)b * V : nullptr;
    const float* bias = a.r.bias ? a.r.bias + (size_t)b * a.r.bias_stride : nullptr;
    const uint32_t* allowed = a.r.allowed ? a.r.allowed + (size_t)b * a.r.allowed_stride : nullptr;
    float* out = a.out ? a.out + (size_t)b * V : nullptr;
    const float rep = counts && a.r.repeat ? a.r.repeat[b] : 1.0f;
    const float freq = counts && a.r.frequency ? a.r.frequency[b] : 0.0f;
    const float pres = counts && a.r.presence ? a.r.presence[b] : 0.0f;
    LogitBest best{-__builtin_inff(), -1, 0xFFFFFFFFu, 0u};

    auto one = [&](float y, int c, float bi, bool ok, int v) {
        if (c > 0)
        {
            if (a.r.repeat) y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
            if (a.r.frequency) y = __fsub_rn(y, __fmul_rn(freq, (float)c));
            if (a.r.presence) y = __fsub_rn(y, pres);
        }
        if (bias) y = __fadd_rn(y, bi);
        if (!ok) return -__builtin_inff();
        best.first = min(best.first, 2u * (uint32_t)v + (y != y ? 1u : 0u));
        if (y == y && (best.i < 0 || y > best.v))
        {
            best.v = y;
            best.i = v;
        }
        return y;
    };

    for (int base = i0 + tid; base < i1; base += T * U)
    {
        f32x4u xv[U], bv[U];
        i32x4u cv[U];
        uint32_t word[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int v = 4 * (base + u * T);
            xv[u] = f32x4u(0.0f), bv[u] = f32x4u(0.0f), cv[u] = i32x4u(0), word[u] = 0xFFFFFFFFu;
            if (base + u * T >= i1) continue;
            if (v + 4 <= V)
            {
                xv[u] = *reinterpret_cast<const f32x4u*>(x + v);
                if (counts) cv[u] = *reinterpret_cast<const i32x4u*>(counts + v);
                if (bias) bv[u] = *reinterpret_cast<const f32x4u*>(bias + v);
            }
            else
                for (int e = 0; e < 4; ++e)
                    if (v + e < V)
                    {
                        xv[u][e] = x[v + e];
                        if (counts) cv[u][e] = counts[v + e];
                        if (bias) bv[u][e] = bias[v + e];
                    }
            if (allowed) word[u] = allowed[v >> 5] >> (v & 31);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
        {
            const int v = 4 * (base + u * T);
            if (base + u * T >= i1) continue;
            f32x4u y;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v + e < V) y[e] = one(xv[u][e], cv[u][e], bv[u][e], (word[u] >> e) & 1u, v + e);
            if (out)
            {
                if (v + 4 <= V) __builtin_nontemporal_store(y, reinterpret_cast<f32x4u*>(out + v));
                else
                    for (int e = 0; e < 4; ++e)
                        if (v + e < V) out[v + e] = y[e];
            }
        }
    }
    if (!a.ids) return;
    best = wave_best(best);
    if ((tid & 63) == 0) best_s[tid >> 6] = best;
    __syncthreads();
    if (tid >= kWave) return;
    best = tid < T / kWave ? best_s[tid] : LogitBest{-__builtin_inff(), -1, 0xFFFFFFFFu, 0u};
    best = wave_best(best);
    if (tid != 0) return;
    if (a.slices == 1) choose(a, b, best);
    else a.part[(size_t)b * a.slices + blockIdx.x] = best;
}

__global__ __launch_bounds__(kWave) void k_logits_choose(LogitArgs a)
{
    const int b = blockIdx.x, tid = threadIdx.x;
    LogitBest best{-__builtin_inff(), -1, 0xFFFFFFFFu, 0u};
    if (tid < a.slices) best = a.part[(size_t)b * a.slices + tid];
    best = wave_best(best);
    if (tid == 0) choose(a, b, best);
}

// One thread per token; the adds are of whole numbers, so their order does not show.
__global__ __launch_bounds__(256) void k_token_counts(const int32_t* ids, int M, const int32_t* cu, int B, int V,
                                                      int32_t* counts)
{
    const int m = blockIdx.x * 256 + threadIdx.x;
    if (m >= M) return;
    const int b = packed_sequence(cu, B, m), id = ids[m];
    if (b >= 0 && id >= 0 && id < V) atomicAdd(counts + (size_t)b * V + id, 1);
}

}  // namespace

// Rows of up to 16384 logits: one work-group of 1024 threads with 4 groups of 4 logits each on their way,
// so that a row is one round trip and one launch (10000 logits with every rule: 6.4 us a call, 7.8 with the
// kernel of long rows). Longer ones: slices of 4096 or more, up to 16 work-groups of 512 threads to a CU
// (256 rows of 131071: 4 to a CU 91.9 us, 8 86.7, 16 83.1; 1024 threads and 4 groups, one to a CU, 94), and a
// second launch that joins them.
constexpr size_t kLgRow = 16384;
constexpr size_t kLgPerCu = 16;

size_t logits_slices(size_t V, size_t B, size_t num_cus)
{
    if (V <= kLgRow) return 1;
    const size_t most = std::min<size_t>(kLgSlices, V / 4096);
    return std::max<size_t>(1, std::min(most, kLgPerCu * num_cus / B));
}

size_t logits_workspace_bytes(size_t V, size_t B, size_t num_cus)
{
    const size_t s = logits_slices(V, B, num_cus);
    return s <= 1 ? 0 : B * s * sizeof(LogitBest);
}

hipError_t launch_logits_adjust(hipStream_t st, const float* logits, size_t V, size_t B, const nnhip_logit_rules& rules,
                                float* out, int32_t* ids, int32_t* pos, void* ws, size_t num_cus)
{
    const size_t s = logits_slices(V, B, num_cus);
    LogitArgs a{logits, rules, out, ids, pos, static_cast<LogitBest*>(ws), (int)V, (int)s};
    if (V <= kLgRow) k_logits_adjust<1024, 4><<<dim3((unsigned)s, (unsigned)B), 1024, 0, st>>>(a);
    else k_logits_adjust<512, 2><<<dim3((unsigned)s, (unsigned)B), 512, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || s == 1 || !ids) return e;
    k_logits_choose<<<dim3((unsigned)B), kWave, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_token_counts(hipStream_t st, const int32_t* ids, size_t M, const int32_t* cu, size_t B, size_t V,
                               int32_t* counts)
{
    k_token_counts<<<dim3((unsigned)ceil_div(M, 256)), 256, 0, st>>>(ids, (int)M, cu, (int)B, (int)V, counts);
    return hipGetLastError();
}

}  // namespace nnhip
