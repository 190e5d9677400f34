// Norms of the query and key heads, position rotation and cache store of a pass's rows (ql_qk_norm_rope), and the
// table of angles it reads (ql_rope_table). The reference rotates on its own (src/gpu/kernels/rope,
// src/reference/qwen-ref.ts ropeHalfRef) and stores keys and values with kv_store after it.
//
//   x' = x / sqrt(mean(x^2) + eps) * w          per head of q and k, where a norm weight is given
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * theta^(-2 i / rot), for the pairs
//       (x'[i], x'[i + rot / 2]), or (x'[2 i], x'[2 i + 1]) where interleaved; values from rot on stay
// q goes to fp32 rows, k (rotated) and v to the cache rows slot0 + m, fp32 or rounded once to fp16.
//
// A lane has eight values of a head, whole pairs of them, so nothing but the head's sum of squares (a
// butterfly over the 8 to 32 lanes of the head) crosses lanes, and q may be rotated in place. The angles come from
// the table, since t in fp32 is off by position * 2^-24 and fp64 sines a row cost more than 4 rot bytes from L2.
// Bytes: q, k and v read once, q, k and v written once: 2048 rows (28 / 4 heads of 128, norms, fp32) 13.2 us, 5.8 TB/s; up to some
// 24 rows one launch and a chain of loads, 4.4 us.
#include <cmath>

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"

namespace ql {

namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// GS: lanes per head (D / 8 rounded up to a power of two); HALF: the cache is fp16
template <int GS, bool HALF>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const RopeArgs a)
{
    const uint32_t unit = (blockIdx.x * 256u + threadIdx.x) / GS, l = threadIdx.x % GS;
    const uint32_t heads = a.H + 2 * a.KV;
    const uint32_t row = unit / heads, h = unit - row * heads;
    if (row >= (uint32_t)a.M) return;
    const int pos = ld_global(a.pos + row);
    if ((uint32_t)pos >= (uint32_t)a.max_pos || 8 * l >= (uint32_t)a.D) return;   // a padding row; no values of the head
    const bool is_q = h < (uint32_t)a.H, is_v = h >= (uint32_t)(a.H + a.KV);
    const uint32_t head = is_q ? h : is_v ? h - a.H - a.KV : h - a.H;
    const float* x = is_q ? a.q + (size_t)row * a.q_stride : is_v ? a.v + (size_t)row * a.v_stride : a.k + (size_t)row * a.k_stride;
    x += (size_t)head * a.D;
    const bool turn = !is_v && 8 * l < (uint32_t)a.rot, split = turn && !a.interleaved;
    const uint32_t i0 = split ? 4 * l : 8 * l, i1 = split ? 4 * l + a.rot / 2 : 8 * l + 4;
    f32x4 x0 = ld_global(reinterpret_cast<const f32x4*>(x + i0)), x1 = ld_global(reinterpret_cast<const f32x4*>(x + i1));
    f32x4 c = {1.f, 1.f, 1.f, 1.f}, s = {0.f, 0.f, 0.f, 0.f};
    if (turn) {
        const float* t = a.table + (size_t)pos * a.rot + 4 * l;
        c = ld_global(reinterpret_cast<const f32x4*>(t));
        s = ld_global(reinterpret_cast<const f32x4*>(t + a.rot / 2));
    }
    const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    if (w) {                                             // the same for every lane of a head
        const f32x4 w0 = ld_global(reinterpret_cast<const f32x4*>(w + i0)), w1 = ld_global(reinterpret_cast<const f32x4*>(w + i1));
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) ss = fmaf(x0[e], x0[e], ss);
#pragma unroll
        for (int e = 0; e < 4; e++) ss = fmaf(x1[e], x1[e], ss);
        const int lanes = a.D / 8;
        float total = ss;
        if (lanes == GS) {
#pragma unroll
            for (int o = GS / 2; o > 0; o >>= 1) total += __shfl_xor(total, o);
        } else {
            // a head of other than a power of two lanes: the lanes without values have left
            total = 0.f;
            const int first = (threadIdx.x & 63) - l;
            for (int i = 0; i < lanes; i++) total += __shfl(ss, first + i);
        }
        const float r = 1.0f / sqrtf(total / (float)a.D + a.eps);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x0[e] = x0[e] * r * w0[e];
            x1[e] = x1[e] * r * w1[e];
        }
    }
    f32x4 y0 = x0, y1 = x1;
    if (split) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y0[e] = x0[e] * c[e] - x1[e] * s[e];
            y1[e] = x1[e] * c[e] + x0[e] * s[e];
        }
    } else if (turn) {
        y0 = f32x4{x0[0] * c[0] - x0[1] * s[0], x0[1] * c[0] + x0[0] * s[0], x0[2] * c[1] - x0[3] * s[1], x0[3] * c[1] + x0[2] * s[1]};
        y1 = f32x4{x1[0] * c[2] - x1[1] * s[2], x1[1] * c[2] + x1[0] * s[2], x1[2] * c[3] - x1[3] * s[3], x1[3] * c[3] + x1[2] * s[3]};
    }
    if (is_q) {
        float* o = a.q_out + ((size_t)row * a.H + head) * a.D;
        st_global(reinterpret_cast<f32x4*>(o + i0), y0);
        st_global(reinterpret_cast<f32x4*>(o + i1), y1);
    } else {
        const size_t at = ((size_t)(a.slot0 + row) * a.KV + head) * a.D;
        if (HALF) {
            _Float16* o = static_cast<_Float16*>(is_v ? a.v_cache : a.k_cache) + at;
            st_global(reinterpret_cast<f16x4*>(o + i0), __builtin_convertvector(y0, f16x4));
            st_global(reinterpret_cast<f16x4*>(o + i1), __builtin_convertvector(y1, f16x4));
        } else {
            float* o = static_cast<float*>(is_v ? a.v_cache : a.k_cache) + at;
            st_global(reinterpret_cast<f32x4*>(o + i0), y0);
            st_global(reinterpret_cast<f32x4*>(o + i1), y1);
        }
    }
}

// one pair's angle a thread, in fp64, its cosine and sine rounded once
__global__ __launch_bounds__(256) void rope_table_kernel(float* table, int max_pos, int rot, double log_theta)
{
    const long long u = (long long)blockIdx.x * 256 + threadIdx.x;
    const int half = rot / 2, pos = (int)(u / half), i = (int)(u - (long long)pos * half);
    if (pos >= max_pos) return;
    double s, c;
    sincos((double)pos * exp(-2.0 * i / rot * log_theta), &s, &c);
    float* t = table + (size_t)pos * rot + i;
    st_global(t, (float)c);
    st_global(t + half, (float)s);
}

template <int GS>
void launch_rope_gs(const RopeArgs& a, hipStream_t stream)
{
    const dim3 grid((unsigned)(((long long)a.M * (a.H + 2 * a.KV) * GS + 255) / 256));
    if (a.half) hipLaunchKernelGGL((qk_norm_rope_kernel<GS, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<GS, false>), grid, dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_qk_norm_rope(const RopeArgs& a, hipStream_t stream)
{
    const int lanes = a.D / 8;
    if (lanes <= 1) launch_rope_gs<1>(a, stream);
    else if (lanes <= 2) launch_rope_gs<2>(a, stream);
    else if (lanes <= 4) launch_rope_gs<4>(a, stream);
    else if (lanes <= 8) launch_rope_gs<8>(a, stream);
    else if (lanes <= 16) launch_rope_gs<16>(a, stream);
    else launch_rope_gs<32>(a, stream);
    return hipGetLastError();
}

hipError_t launch_rope_table(float* table, int max_pos, int rot, double theta, hipStream_t stream)
{
    const long long n = (long long)max_pos * (rot / 2);
    hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, table, max_pos, rot, std::log(theta));
    return hipGetLastError();
}

}  // namespace ql
