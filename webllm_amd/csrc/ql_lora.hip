// Low-rank adapters of a batch's rows beside a shared projection (ql_lora_add): y = base + s_a (x . A_a^T) . B_a^T, a = ids[row].
//
// A workgroup a row and projection: t = x . A^T goes to LDS, a wave a rank at a time, then a thread four columns of y.
#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"

namespace ql {

namespace {

__global__ __launch_bounds__(256) void lora_row_kernel(const LoraArgs a)
{
    __shared__ float t[kLoraMaxRank];
    const int m = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const LoraArgs::One p = a.p[blockIdx.y];
    const int id = ld_global(a.ids + m);
    const bool has = (uint32_t)id < (uint32_t)p.n;
    if (!has && p.base == p.y) return;
    if (has) {
        const float s = p.scale ? ld_global(p.scale + id) : 1.f;
        for (int r = tid >> 6; r < p.rank; r += 4) {
            const uint16_t* A = p.a + ((size_t)id * p.rank + r) * p.K;
            float sum = 0.f;
            for (int k = 8 * lane; k < p.K; k += 512) {
                const f16x8 w = __builtin_bit_cast(f16x8, ld_global(reinterpret_cast<const u32x4*>(A + k)));
                float x[8];
                load8(p.x, a.half, (size_t)m * p.K + k, x);
#pragma unroll
                for (int e = 0; e < 8; e++) sum = fmaf(x[e], (float)w[e], sum);
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
            if (lane == 0) t[r] = sum * s;
        }
    }
    __syncthreads();
    for (int n = 4 * tid; n < p.N; n += 1024) {
        f32x4 y = ld_global(reinterpret_cast<const f32x4*>(p.base + (size_t)m * p.N + n));
        if (has)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint16_t* B = p.b + ((size_t)id * p.N + n + e) * p.rank;
                float sum = 0.f;
                for (int r = 0; r < p.rank; r += 8) {
                    const f16x8 w = __builtin_bit_cast(f16x8, ld_global(reinterpret_cast<const u32x4*>(B + r)));
#pragma unroll
                    for (int i = 0; i < 8; i++) sum = fmaf(t[r + i], (float)w[i], sum);
                }
                y[e] += sum;
            }
        st_global(reinterpret_cast<f32x4*>(p.y + (size_t)m * p.N + n), y);
    }
}

}  // namespace

uint64_t plan_lora(LoraArgs*, size_t) { return 0; }

hipError_t launch_lora(const LoraArgs& a, hipStream_t stream)
{
    hipLaunchKernelGGL(lora_row_kernel, dim3(a.M, a.count), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ql
