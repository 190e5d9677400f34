// Log probabilities of given tokens under rows of logits, with each row's entropy and its top alternatives
// (ql_token_logprobs). No counterpart in the reference, whose sampler reads the logits on the host.
//
//   lse = m + ln sum e^(x - m),  log p(t) = x_t - lse,  H = ln S - (sum (x - m) e^(x - m)) / S,  S = sum e^(x - m)
// with m the row's largest logit, so nothing cancels however large the logits are; -inf logits (a mask) add nothing. A
// row without any other: log p = -inf, H = 0. Alternatives are ordered by value, equal ones by index.
#include <cmath>

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"

namespace ql {

namespace {

constexpr int kThreads = 1024;

// A logit's order and place as one unsigned number: larger logits first, of equal ones the lower index. NaN above all.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index)
{
    uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    b = x != x ? 0xFFFFFFFFu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return (uint64_t)b << 32 | (uint32_t)~index;
}

__device__ __forceinline__ float reduce_max(float v, float* lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int i = 1; i < kThreads / 64; i++) v = fmaxf(v, lds[i]);
    return v;
}

__device__ __forceinline__ float reduce_sum(float v, float* lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int i = 1; i < kThreads / 64; i++) v += lds[i];
    return v;
}

// one workgroup per row
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(const LogprobArgs a)
{
    __shared__ float red[kThreads / 64];
    __shared__ uint64_t best[kThreads / 64];
    const int row = blockIdx.x, V = a.V, tid = threadIdx.x;
    const float* x = a.logits + (size_t)row * a.stride;
    float m = -INFINITY;
    bool nan = false;
    for (int i = tid; i < V; i += kThreads) {
        m = fmaxf(m, x[i]);
        nan |= x[i] != x[i];
    }
    m = reduce_max(m, red);
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f, t = 0.f;
    for (int i = tid; i < V; i += kThreads) {
        const float d = x[i] - ref, e = expf(d);
        s += e;
        t += d == -INFINITY ? 0.f : d * e;
    }
    s = reduce_sum(s, red);
    t = reduce_sum(t, red);
    if (__syncthreads_or(nan)) s = t = NAN;
    const float ls = logf(s);
    const bool none = s == 0.f;
    if (tid == 0 && a.entropy) a.entropy[row] = none ? 0.f : ls - t / s;
    for (int i = tid; i < a.n_tok; i += kThreads) {
        const int tok = a.tokens[(size_t)row * a.n_tok + i];
        a.logprob[(size_t)row * a.n_tok + i] = tok < 0 || tok >= V ? 0.f : none ? -INFINITY : x[tok] - ref - ls;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top_k; k++) {
        uint64_t b = 0;
        for (int i = tid; i < V; i += kThreads) {
            const uint64_t key = order_key(x[i], i);
            if (key < last && key > b) b = key;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)b, o);
            b = b > other ? b : other;
        }
        __syncthreads();
        if ((tid & 63) == 0) best[tid >> 6] = b;
        __syncthreads();
        for (int i = 0; i < kThreads / 64; i++) b = b > best[i] ? b : best[i];
        last = b;
        if (tid == 0) {
            const int id = k < V ? (int)~(uint32_t)b : -1;
            a.top_id[(size_t)row * a.top_k + k] = id;
            a.top_logprob[(size_t)row * a.top_k + k] = id < 0 || none ? -INFINITY : x[id] - ref - ls;
        }
    }
}

}  // namespace

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t stream)
{
    hipLaunchKernelGGL(token_logprobs_kernel, dim3(a.M), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ql
