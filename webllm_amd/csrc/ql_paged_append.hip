// Norms and rotation of a batch's query and key heads, and keys and values appended to their sequences' pages (ql_paged_append).
//
//   x' = x / sqrt(mean(x^2) + eps) * w,  (a, b) -> (a cos t - b sin t, b cos t + a sin t)   as ql_rope.hip, at the row's token
//   e4m3: a group of 16 tokens of a head has p = 2^e, the least e >= -120 with max |x| <= 448 2^e over the tokens that the
//   pass brings, or the group's own p where it has earlier tokens and that is larger; x / p rounded once.
// A power of two leaves the values' own exponents to carry their sizes: a group that grows moves its earlier tokens by whole
// binades, which only rounds what falls below e4m3's normal range again, so a cache depends on how its tokens came in passes by
// those alone.
//
// A workgroup has the query heads of one row, or one group of 16 tokens of a kv head's K or V; LN lanes have a head, a lane whole pairs
// of it. A group's values are put into LDS in the cache's type and go out in pieces of 16 bytes of K (columns of a token) or of
// four tokens of V's column, or token by token where a group is not whole.
//
// Bound by memory where there is much: 4096 rows of 28 / 4 heads of 128 to e4m3 pages and fp16 q, 111 MB, 23.4 us, 4.7 TB/s (a copy: 5.2). A pass of single
// tokens is one launch: 64 rows with norms 4.6 us (4.9 in the kernel's trace), four rows of 14 / 2 heads of 64 4.3 to 4.6. A group, and not a row, is a workgroup's, since its
// tokens share a scale, and V's tokens their 16 bytes.
#include <type_traits>

#include "ql_paged.h"

namespace ql {

namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr float kMaxFinite = 3.4028235e38f;
constexpr int kLeast = -120;

// the least power of two p >= 2^kLeast with top <= 448 p
__device__ __forceinline__ float f8_power(float top)
{
    if (!(top > 0.f)) return ldexpf(1.f, kLeast);
    int ex;
    const float m = frexpf(top, &ex);                  // top = m 2^ex, 448 = 0.875 2^9
    return ldexpf(1.f, max(kLeast, m <= 0.875f ? ex - 9 : ex - 8));
}

__device__ __forceinline__ float finite_or_nan(float x) { return fabsf(x) <= kMaxFinite ? x : __builtin_nanf(""); }

__device__ __forceinline__ uint32_t f8_of4(f32x4 x)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(finite_or_nan(x[0]), finite_or_nan(x[1]), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(finite_or_nan(x[2]), finite_or_nan(x[3]), w, true);
}

__device__ __forceinline__ uint32_t f8_scaled(uint32_t w, float r)
{
    const f32x4 x = {__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * r, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * r, __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * r,
                     __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * r};
    return f8_of4(x);
}

// A lane's values of a head: item k has four from at[2 k] and four from at[2 k + 1], whole pairs
template <int LN, int ITEMS>
struct Head {
    f32x4 y[2 * ITEMS];
    int at[2 * ITEMS];                                 // -1: none

    __device__ __forceinline__ void places(const RopeArgs& a, bool turns, int l)
    {
#pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            const int it = l + LN * k;
            const bool split = turns && 8 * it < a.rot && !a.interleaved;
            at[2 * k] = 8 * it >= a.D ? -1 : split ? 4 * it : 8 * it;
            at[2 * k + 1] = 8 * it >= a.D ? -1 : split ? 4 * it + a.rot / 2 : 8 * it + 4;
        }
    }
    __device__ __forceinline__ void load(const float* x)
    {
#pragma unroll
        for (int k = 0; k < 2 * ITEMS; k++) y[k] = at[k] >= 0 ? ld_global(reinterpret_cast<const f32x4*>(x + at[k])) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // every lane of the head takes part
    __device__ __forceinline__ void norm(const float* w, int D, float eps)
    {
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < 2 * ITEMS; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) ss = fmaf(y[k][e], y[k][e], ss);
#pragma unroll
        for (int o = LN / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        const float r = 1.0f / sqrtf(ss / (float)D + eps);
#pragma unroll
        for (int k = 0; k < 2 * ITEMS; k++) {
            if (at[k] < 0) continue;
            const f32x4 wk = ld_global(reinterpret_cast<const f32x4*>(w + at[k]));
#pragma unroll
            for (int e = 0; e < 4; e++) y[k][e] = y[k][e] * r * wk[e];
        }
    }
    __device__ __forceinline__ void turn(const RopeArgs& a, int pos, int l)
    {
#pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            const int it = l + LN * k;
            if (8 * it >= a.rot) continue;
            const float* t = a.table + (size_t)pos * a.rot + 4 * it;
            const f32x4 c = ld_global(reinterpret_cast<const f32x4*>(t)), s = ld_global(reinterpret_cast<const f32x4*>(t + a.rot / 2));
            const f32x4 x0 = y[2 * k], x1 = y[2 * k + 1];
            if (!a.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    y[2 * k][e] = x0[e] * c[e] - x1[e] * s[e];
                    y[2 * k + 1][e] = x1[e] * c[e] + x0[e] * s[e];
                }
            } else {
                y[2 * k] = f32x4{x0[0] * c[0] - x0[1] * s[0], x0[1] * c[0] + x0[0] * s[0], x0[2] * c[1] - x0[3] * s[1], x0[3] * c[1] + x0[2] * s[1]};
                y[2 * k + 1] = f32x4{x1[0] * c[2] - x1[1] * s[2], x1[1] * c[2] + x1[0] * s[2], x1[2] * c[3] - x1[3] * s[3], x1[3] * c[3] + x1[2] * s[3]};
            }
        }
    }
};

template <int LN, int ITEMS, bool F8>
__global__ __launch_bounds__(16 * LN) void paged_append_kernel(const PagedAppendArgs a)
{
    typedef typename std::conditional<F8, uint8_t, _Float16>::type T;
    typedef PagedLayout<sizeof(T)> Lay;
    constexpr int kThreads = 16 * LN, kStride = 8 * LN * ITEMS + 16 / (int)sizeof(T);
    __shared__ __attribute__((aligned(16))) T tile[16 * kStride];
    __shared__ float most[kThreads / 64];
    const int tid = threadIdx.x, l = tid % LN, token = tid / LN, D = a.r.D, KV = a.r.KV;
    const PagedBatch& b = a.b;
    const int groups = a.jobs * 2 * KV;
    Head<LN, ITEMS> x;
    if ((int)blockIdx.x >= groups) {                    // a row's query heads
        const int row = blockIdx.x - groups;
        int s;
        PagedSeq q;
        if (!paged_row(b, row, s, q)) return;
        const int pos = q.len - q.n + row - q.row0;
        x.places(a.r, true, l);
        for (int h0 = 0; h0 < a.r.H; h0 += 16) {        // lanes of a head that is not there go along: norm() needs them
            const int h = min(h0 + token, a.r.H - 1);
            x.load(a.r.q + (size_t)row * a.r.q_stride + (size_t)h * D);
            if (a.r.q_norm) x.norm(a.r.q_norm, D, a.r.eps);
            x.turn(a.r, pos, l);
            if (h0 + token >= a.r.H) continue;
            const size_t to = ((size_t)row * a.r.H + h) * D;
#pragma unroll
            for (int k = 0; k < 2 * ITEMS; k++) {
                if (x.at[k] < 0) continue;
                if (a.q_half) st_global(reinterpret_cast<f16x4*>(static_cast<_Float16*>(a.q_out) + to + x.at[k]), __builtin_convertvector(x.y[k], f16x4));
                else st_global(reinterpret_cast<f32x4*>(static_cast<float*>(a.q_out) + to + x.at[k]), x.y[k]);
            }
        }
        return;
    }
    const int job = blockIdx.x / (2 * KV), rest = blockIdx.x - job * (2 * KV), h = rest >> 1;
    const bool is_v = rest & 1;
    int s, g;
    PagedSeq q;
    auto count = [](const PagedSeq& q) { return (q.len - 1) / 16 - (q.len - q.n) / 16 + 1; };
    if (!PagedUnits(b, count).find(job, s, g, q)) return;
    const int t0 = ((q.len - q.n) / 16 + g) * 16;       // the group's first token
    const int start = max(q.len - q.n - t0, 0), end = min(q.len - t0, 16);   // of it the pass brings start .. end - 1
    const int page = paged_page(b, s, t0);
    if (page < 0) return;
    const int in_page = t0 & ((1 << b.log_page) - 1);
    const size_t head = (size_t)page * KV + h;
    T* const cache = static_cast<T*>(is_v ? a.r.v_cache : a.r.k_cache) + (head << b.log_page) * D;
    float* const scale = F8 ? (is_v ? a.v_scale : a.k_scale) + (head << (b.log_page - 4)) + (in_page >> 4) : nullptr;
    const float before = F8 && start > 0 ? ld_global(scale) : 0.f;

    const bool mine = token >= start && token < end;
    const int t = t0 + token;
    const size_t row = (size_t)(q.row0 + min(max(t - (q.len - q.n), 0), q.n - 1));
    x.places(a.r, !is_v, l);
    x.load((is_v ? a.r.v + row * a.r.v_stride : a.r.k + row * a.r.k_stride) + (size_t)h * D);
    if (!is_v) {
        if (a.r.k_norm) x.norm(a.r.k_norm, D, a.r.eps);
        x.turn(a.r, min(max(t, q.len - q.n), q.len - 1), l);
    }
    float power = 1.f;
    bool grows = false;
    if constexpr (F8) {
        float top = 0.f;
        if (mine)
#pragma unroll
            for (int k = 0; k < 2 * ITEMS; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = fabsf(x.y[k][e]);
                    top = fmaxf(top, y <= kMaxFinite ? y : 0.f);
                }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if ((tid & 63) == 0) most[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 64; w++) top = fmaxf(top, most[w]);
        power = start > 0 ? fmaxf(before, f8_power(top)) : f8_power(top);
        grows = start > 0 && power != before;
        if (tid == 0 && (start == 0 || grows)) st_global(scale, power);
    }
    if (mine) {
        const float inv = 1.f / power;
#pragma unroll
        for (int k = 0; k < 2 * ITEMS; k++) {
            if (x.at[k] < 0) continue;
            T* to = tile + token * kStride + x.at[k];
            if constexpr (F8) *reinterpret_cast<uint32_t*>(to) = f8_of4(f32x4{x.y[k][0] * inv, x.y[k][1] * inv, x.y[k][2] * inv, x.y[k][3] * inv});
            else *reinterpret_cast<f16x4*>(to) = __builtin_convertvector(x.y[k], f16x4);
        }
    }
    __syncthreads();
    const float ratio = grows ? before / power : 1.f;
    if (!is_v) {
        for (int u = tid; u < 16 * (D / Lay::kUnit); u += kThreads) {
            const int tok = u & 15, unit = u >> 4;
            u32x4* to = reinterpret_cast<u32x4*>(cache + Lay::k_at(D, in_page + tok, unit));
            if (tok >= start && tok < end) {
                st_global(to, *reinterpret_cast<const u32x4*>(tile + tok * kStride + unit * Lay::kUnit));
            } else if (F8 && grows && tok < start) {
                u32x4 w = ld_global(to);
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = f8_scaled(w[e], ratio);
                st_global(to, w);
            }
        }
    } else {
        for (int u = tid; u < 4 * D; u += kThreads) {
            const int d = (u >> 6) * 16 + (u & 15), tok = (u >> 4 & 3) * 4;
            T* to = cache + Lay::v_at(D, in_page + tok, d);
            if (tok >= end || (tok + 4 <= start && !grows)) continue;
            T y[4];
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = tile[(tok + r) * kStride + d];
            if (tok >= start && tok + 4 <= end) {
                if constexpr (F8) st_global(reinterpret_cast<uint32_t*>(to), (uint32_t)y[0] | (uint32_t)y[1] << 8 | (uint32_t)y[2] << 16 | (uint32_t)y[3] << 24);
                else st_global(reinterpret_cast<f16x4*>(to), f16x4{y[0], y[1], y[2], y[3]});
                continue;
            }
            if constexpr (F8) {
                const uint32_t moved = grows ? f8_scaled(ld_global(reinterpret_cast<const uint32_t*>(to)), ratio) : 0;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if (tok + r >= start && tok + r < end) st_global(to + r, y[r]);
                    else if (grows && tok + r < start) st_global(to + r, (uint8_t)(moved >> (8 * r)));
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (tok + r >= start && tok + r < end) st_global(to + r, y[r]);
            }
        }
    }
}

template <int LN, int ITEMS>
void launch(const PagedAppendArgs& a, hipStream_t stream)
{
    const dim3 grid((unsigned)(a.jobs * 2 * a.r.KV + a.r.M));
    if (a.k_scale) hipLaunchKernelGGL((paged_append_kernel<LN, ITEMS, true>), grid, dim3(16 * LN), 0, stream, a);
    else hipLaunchKernelGGL((paged_append_kernel<LN, ITEMS, false>), grid, dim3(16 * LN), 0, stream, a);
}

}  // namespace

hipError_t launch_paged_append(PagedAppendArgs a, hipStream_t stream)
{
    // n rows in a row touch (n - 1) / 16 + 2 groups at most, and one row one
    a.jobs = (int)std::min<long long>(a.b.M, a.b.M / 16 + 2ll * a.b.S);
    if (a.r.D <= 64) launch<8, 1>(a, stream);
    else if (a.r.D <= 128) launch<16, 1>(a, stream);
    else launch<16, 2>(a, stream);
    return hipGetLastError();
}

}  // namespace ql
