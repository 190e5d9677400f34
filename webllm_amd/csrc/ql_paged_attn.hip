// Attention of a batch's rows over their sequences' pages (ql_paged_attention):
//   out[m, h] = sum_t p_t V[t] / sum_t p_t,  p_t = exp(q[m, h] . K[t] / sqrt(D) - max)   over the tokens t up to the row's own.
//
// A workgroup a (row, head); its four waves take blocks of 64 tokens in turn, a lane a token's score, then a lane its columns; running
// maximum and sum; the waves' states are merged through LDS.
#include <type_traits>

#include "ql_paged.h"

namespace ql {

namespace {

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

template <bool F8>
__device__ __forceinline__ float value_at(const void* p, size_t i)
{
    if (F8) return __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(p)[i], 0);
    return (float)static_cast<const _Float16*>(p)[i];
}

template <bool F8, typename Q>
__global__ __launch_bounds__(256) void paged_row_kernel(const PagedAttnArgs a)
{
    typedef PagedLayout<F8 ? 1 : 2> Lay;
    __shared__ float q[256], p[4][64], st[2][4], part[4][256];
    const int h = blockIdx.x, m = blockIdx.y, kvh = h / a.G, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = a.D;
    const PagedBatch& b = a.b;
    int s;
    PagedSeq seq;
    if (!paged_row(b, m, s, seq)) return;
    const int last = seq.len - seq.n + m - seq.row0;
    const size_t row = ((size_t)m * a.H + h) * D;
    if (tid < D) q[tid] = (float)static_cast<const Q*>(a.q)[row + tid];
    __syncthreads();
    float mx = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t0 = 64 * wave; t0 <= last; t0 += 256) {
        const int t = t0 + lane, page = paged_page(b, s, t0), in_page = t0 & ((1 << b.log_page) - 1);
        if (page < 0) continue;
        const size_t head = (size_t)page * a.KV + kvh, base = (head << b.log_page) * D, sc0 = (head << (b.log_page - 4)) + (in_page >> 4);
        float sc = -INFINITY;
        if (t <= last) {
            sc = 0.f;
            for (int d = 0; d < D; d++) sc = fmaf(q[d], value_at<F8>(a.k, base + Lay::k_at(D, in_page + lane, d / Lay::kUnit) + d % Lay::kUnit), sc);
            sc *= a.scale * (F8 ? a.k_scale[sc0 + lane / 16] : 1.f);
        }
        float bm = sc;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) bm = fmaxf(bm, __shfl_xor(bm, o));
        const float mn = fmaxf(mx, bm), ref = mn == -INFINITY ? 0.f : mn, al = ex2(mx - ref);
        mx = mn;
        const float e = t <= last ? ex2(sc - ref) : 0.f;
        float sum = e;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        l = l * al + sum;
        p[wave][lane] = e * (F8 ? a.v_scale[sc0 + lane / 16] : 1.f);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = lane + 64 * i;
            acc[i] *= al;
            if (d < D)
                for (int k = 0; k < 64 && t0 + k <= last; k++)
                    acc[i] = fmaf(p[wave][k], value_at<F8>(a.v, base + Lay::v_at(D, in_page + k / 4 * 4, d) + k % 4), acc[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    if (lane == 0) st[0][wave] = mx, st[1][wave] = l;
#pragma unroll
    for (int i = 0; i < 4; i++) part[wave][lane + 64 * i] = acc[i];
    __syncthreads();
    if (tid >= D) return;
    float top = st[0][0], total = 0.f, o = 0.f;
    for (int w = 1; w < 4; w++) top = fmaxf(top, st[0][w]);
    for (int w = 0; w < 4; w++) {
        const float f = st[0][w] == -INFINITY ? (st[1][w] != st[1][w] ? st[1][w] : 0.f) : ex2(st[0][w] - top);
        if (f == 0.f) continue;
        total += f * st[1][w];
        o += f * part[w][tid];
    }
    o = total == 0.f ? 0.f : o / total;
    static_cast<Q*>(a.out)[row + tid] = (Q)o;
}

}  // namespace

uint64_t plan_paged_attention(PagedAttnArgs*, size_t) { return 0; }

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream)
{
    const dim3 grid(a.H, a.b.M);
    if (a.k_scale) {
        if (a.half) hipLaunchKernelGGL((paged_row_kernel<true, _Float16>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((paged_row_kernel<true, float>), grid, dim3(256), 0, stream, a);
    } else {
        if (a.half) hipLaunchKernelGGL((paged_row_kernel<false, _Float16>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((paged_row_kernel<false, float>), grid, dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace ql
