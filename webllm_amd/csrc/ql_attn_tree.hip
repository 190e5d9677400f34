// Attention of a tree of drafted tokens over the KV cache (ql_attention_tree), and of any few rows over a long or half cache.
//
//   out[m, h] = sum_s p_s V[s] / sum_s p_s,  p_s = exp(q[m, h] . K[s] / sqrt(D) - max)
// over the cache's past positions and the drafted rows j (at past + j) whose bit is set in row m's mask. A row that sees
// nothing is zero; what it does not see it takes nothing from, not even 0 * V.
#include <cmath>

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"

namespace ql {

namespace {

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// one wave per (row, head): 64 keys a step, a lane's own key for the scores, its own values of D for the sums
template <typename T>
__global__ __launch_bounds__(64) void attn_tree_row_kernel(const TreeArgs a)
{
    __shared__ float q[256];
    const int h = blockIdx.x, m = blockIdx.y, lane = threadIdx.x, D = a.D;
    const size_t row = (size_t)m * a.H + h, row_len = (size_t)a.KV * D;
    const T* k = static_cast<const T*>(a.k) + (size_t)(h / a.G) * D;
    const T* v = static_cast<const T*>(a.v) + (size_t)(h / a.G) * D;
    for (int d = lane; d < D; d += 64) q[d] = a.q[row * D + d];
    __syncthreads();
    float mx = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < a.past + a.M; s0 += 64) {
        const int s = s0 + lane, j = s - a.past;
        bool seen = s < a.past + a.M;
        if (seen && j >= 0) seen = a.mask ? a.mask[(size_t)m * a.words + (j >> 6)] >> (j & 63) & 1 : j <= m;
        float sc = -INFINITY;
        if (seen) {
            sc = 0.f;
            for (int d = 0; d < D; d++) sc = fmaf(q[d], (float)k[(size_t)s * row_len + d], sc);
            sc *= a.scale;
        }
        float bm = sc;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor(bm, o));
        const float mn = fmaxf(mx, bm), ref = mn == -INFINITY ? 0.f : mn, al = ex2(mx - ref);
        const float p = seen ? ex2(sc - ref) : 0.f;
        float sum = p;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        l = l * al + sum;
        mx = mn;
        for (int i = 0; i < 4; i++) acc[i] *= al;
        const uint64_t vis = __ballot(seen);
        for (int c = 0; c < 64; c++) {
            if (!(vis >> c & 1)) continue;
            const float pc = __shfl(p, c);
            for (int i = 0; i < 4; i++)
                if (lane + 64 * i < D) acc[i] = fmaf(pc, (float)v[(size_t)(s0 + c) * row_len + lane + 64 * i], acc[i]);
        }
    }
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < D) a.out[row * D + lane + 64 * i] = l == 0.f ? 0.f : acc[i] / l;
}

}  // namespace

hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t stream)
{
    if (a.half) hipLaunchKernelGGL(attn_tree_row_kernel<_Float16>, dim3(a.H, a.M), dim3(64), 0, stream, a);
    else hipLaunchKernelGGL(attn_tree_row_kernel<float>, dim3(a.H, a.M), dim3(64), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ql
