// Low-rank adapters of a batch's rows beside a shared projection (ql_lora_add): y = base + s_a (x . A_a^T) . B_a^T, a = ids[row].
//
// lora_row_kernel, few rows: a workgroup of sixteen waves has a row of a projection and a range of its columns. t = x . A^T first: a wave has
// four ranks, so that x is read once for them, and a part of K, the parts' sums meet in LDS; then a thread has a column of y, and B's row of it. The
// workgroups of one row's column ranges each make t for themselves: A comes from L2, and a second launch would cost more.
//
// Many rows, two launches: lora_down_kernel makes t of 16 rows, eight waves a part of K each, on the matrix cores, T^T = A x^T
// (lane = row, registers = ranks), for all projections that read one x; lora_up_kernel has 64 rows and a range of columns, y^T = B t^T. Rows of
// several adapters in one tile: it is gone through once for each adapter, and a row takes its own. fp32 x enters as two fp16 parts (22 bits) under the
// exponent of the row's 32 columns at a time; t likewise under the row's.
#include <algorithm>

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"
#include "ql_lanes.h"

namespace ql {

namespace {

constexpr int kRowWaves = 16;
constexpr float kMaxFinite = 3.4028235e38f;

template <bool HALF>
__global__ __launch_bounds__(64 * kRowWaves) void lora_row_kernel(const LoraArgs a)
{
    __shared__ float part[kRowWaves][4], t[kLoraMaxRank];
    const int m = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const LoraArgs::One p = a.p[blockIdx.y];
    const int id = ld_global(a.ids + m);
    const bool has = (uint32_t)id < (uint32_t)p.n;
    if (!has && p.base == p.y) return;
    const int cols = (p.N / 4 + (int)gridDim.z - 1) / (int)gridDim.z * 4, n0 = blockIdx.z * cols, n1 = min(p.N, n0 + cols);
    const float* base = p.base + (size_t)m * p.N;
    float* y = p.y + (size_t)m * p.N;
    if (!has) {
        for (int n = n0 + tid; n < n1; n += 64 * kRowWaves) st_global(y + n, ld_global(base + n));
        return;
    }
    const float s = p.scale ? ld_global(p.scale + id) : 1.f;
    const int groups = p.rank / 4;
    for (int g0 = 0; g0 < groups; g0 += kRowWaves) {
        // `here` groups of four ranks, `parts` waves each
        const int here = min(groups - g0, kRowWaves), parts = kRowWaves / here, grp = wave % here, k = wave / here;
        const int seg = ((p.K + parts - 1) / parts + 511) / 512 * 512, k1 = min(p.K, (k + 1) * seg);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        if (k < parts) {
            const uint16_t* A = p.a + ((size_t)id * p.rank + 4 * (g0 + grp)) * p.K;
#pragma unroll 4
            for (int i = k * seg + 8 * lane; i < k1; i += 512) {
                float x[8];
                load8(p.x, HALF, (size_t)m * p.K + i, x);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const f16x8 w = __builtin_bit_cast(f16x8, ld_global(reinterpret_cast<const u32x4*>(A + (size_t)r * p.K + i)));
#pragma unroll
                    for (int e = 0; e < 8; e++) sum[r] = fmaf(x[e], (float)w[e], sum[r]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) sum[r] = wave_sum(sum[r], lane);
            if (lane == 0)
#pragma unroll
                for (int r = 0; r < 4; r++) part[wave][r] = sum[r];
        }
        __syncthreads();
        if (tid < 4 * here) {
            float v = part[tid >> 2][tid & 3];
            for (int k = 1; k < parts; k++) v += part[(tid >> 2) + k * here][tid & 3];
            t[4 * g0 + tid] = v * s;
        }
        __syncthreads();
    }
#pragma unroll 2
    for (int n = n0 + tid; n < n1; n += 64 * kRowWaves) {
        const uint16_t* B = p.b + ((size_t)id * p.N + n) * p.rank;
        const float b = ld_global(base + n);
        float sum = 0.f;
#pragma unroll 2
        for (int r = 0; r < p.rank; r += 8) {
            const f16x8 w = __builtin_bit_cast(f16x8, ld_global(reinterpret_cast<const u32x4*>(B + r)));
#pragma unroll
            for (int i = 0; i < 8; i++) sum = fmaf(t[r + i], (float)w[i], sum);
        }
        st_global(y + n, b + sum);
    }
}

// ---- many rows

constexpr int kDownWaves = 8, kDownTiles = 12;   // waves of a workgroup; tiles of 16 ranks that it makes at once
constexpr int kUpRows = 64, kUpCols = 256;

// the ranks of all projections that read one x, in tiles of 16: tile u is of projection p[u], its first rank r[u]
struct LoraDown {
    LoraArgs a;
    const void* x;
    int K, tiles;
    short p[kDownTiles], r[kDownTiles];
};

// the other rows' adapters of a tile come later: those of `left` that are the first one's
__device__ __forceinline__ uint64_t next_adapter(int id, uint64_t left, int& which)
{
    which = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    return left & __ballot(id == which);
}

// x's two parts: hi + 2^-11 lo of x * s
__device__ __forceinline__ void split_f16(const float (&x)[8], float s, f16x8& hi, f16x8& lo)
{
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float y = x[e] * s;
        hi[e] = (_Float16)y;
        lo[e] = (_Float16)((y - (float)hi[e]) * 2048.f);
    }
}
// the power of two that brings mx to [2^14, 2^15)
__device__ __forceinline__ float scale_of(float mx) { return mx > 0.f && mx <= kMaxFinite ? ldexpf(1.f, min(100, 14 - ilogbf(mx))) : 1.f; }

template <bool HALF>
__global__ __launch_bounds__(64 * kDownWaves) void lora_down_kernel(const LoraDown d)
{
    __shared__ f32x4 part[kDownWaves][kDownTiles][64];
    const int m0 = 16 * blockIdx.x, tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = min(m0 + i16, d.a.M - 1), id = m0 + i16 < d.a.M ? ld_global(d.a.ids + m) : -1;
    int most = 0;
    for (int u = 0; u < d.tiles; u++) most = max(most, d.a.p[d.p[u]].n);
    uint64_t left = __ballot((uint32_t)id < (uint32_t)most) & 0xFFFF;
    const int steps = (d.K + 31) / 32, per = (steps + kDownWaves - 1) / kDownWaves, s0 = wave * per, s1 = min(steps, s0 + per);
    while (left) {
        int which;
        const uint64_t mine = next_adapter(id, left, which);
        left &= ~mine;
        f32x4 acc[kDownTiles];
#pragma unroll
        for (int u = 0; u < kDownTiles; u++) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int st = s0; st < s1; st++) {
            const int k = 32 * st + 8 * g;
            const bool in = k < d.K;
            f16x8 hi, lo;
            float up = 1.f;
            if constexpr (HALF) {
                hi = in ? __builtin_bit_cast(f16x8, ld_global(reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(d.x) + (size_t)m * d.K + k))) : f16x8{};
            } else {
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (in) load8(d.x, 0, (size_t)m * d.K + k, x);
                float mx = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[e]));
                mx = pair_max<32>(pair_max<16>(mx));
                const float s = scale_of(mx);
                up = 1.f / s;
                split_f16(x, s, hi, lo);
            }
#pragma unroll
            for (int u = 0; u < kDownTiles; u++) {
                if (u >= d.tiles) continue;
                const LoraArgs::One& p = d.a.p[d.p[u]];
                const int r = d.r[u] + i16;
                const bool there = in && r < p.rank && which < p.n;
                const f16x8 w = there ? __builtin_bit_cast(f16x8, ld_global(reinterpret_cast<const u32x4*>(p.a + ((size_t)which * p.rank + r) * p.K + k))) : f16x8{};
                if constexpr (HALF) {
                    acc[u] = mfma_16x16x32_f16(w, hi, acc[u]);
                } else {
                    f32x4 o = {0.f, 0.f, 0.f, 0.f}, ol = {0.f, 0.f, 0.f, 0.f};
                    ol = mfma_16x16x32_f16(w, lo, ol);
                    o = mfma_16x16x32_f16(w, hi, o);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[u][e] = fmaf(fmaf(ol[e], 1.f / 2048.f, o[e]), up, acc[u][e]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kDownTiles; u++)
            if (u < d.tiles) part[wave][u][lane] = acc[u];
        __syncthreads();
        for (int u = wave; u < d.tiles; u += kDownWaves) {
            const LoraArgs::One& p = d.a.p[d.p[u]];
            f32x4 v = part[0][u][lane];
#pragma unroll
            for (int k = 1; k < kDownWaves; k++) v += part[k][u][lane];
            if (!(mine >> i16 & 1) || which >= p.n || d.r[u] + 4 * g >= p.rank) continue;
            const float s = p.scale ? ld_global(p.scale + which) : 1.f;
            float* t = d.a.ws + d.a.t_off[d.p[u]] + (size_t)m * p.rank + d.r[u] + 4 * g;
            st_global(reinterpret_cast<f32x4*>(t), f32x4{v[0] * s, v[1] * s, v[2] * s, v[3] * s});
        }
        __syncthreads();
    }
}

template <int STEPS>
__global__ __launch_bounds__(256) void lora_up_kernel(const LoraArgs a, const int proj)
{
    const LoraArgs::One& p = a.p[proj];
    const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m0 = kUpRows * blockIdx.y, n0 = kUpCols * blockIdx.x + 64 * wave;
    const float* t = a.ws + a.t_off[proj];
#pragma unroll 1
    for (int mt = 0; mt < kUpRows / 16; mt++) {
        const int m = m0 + 16 * mt + i16;
        if (m0 + 16 * mt >= a.M) break;
        const bool row = m < a.M;
        const int id = row ? ld_global(a.ids + m) : -1;
        const bool has = (uint32_t)id < (uint32_t)p.n;
        if (!__any(has) && p.base == p.y) continue;
        f32x4 y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = n0 + 16 * j + 4 * g;
            y[j] = row && n < p.N ? ld_global(reinterpret_cast<const f32x4*>(p.base + (size_t)m * p.N + n)) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
        f16x8 hi[STEPS], lo[STEPS];
        float mx = 0.f, x[STEPS][8];
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[st][e] = 0.f;
            if (has && 32 * st + 8 * g < p.rank) load8(t, 0, (size_t)m * p.rank + 32 * st + 8 * g, x[st]);
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[st][e]));
        }
        mx = pair_max<32>(pair_max<16>(mx));
        const float s = scale_of(mx), up = 1.f / s;
#pragma unroll
        for (int st = 0; st < STEPS; st++) split_f16(x[st], s, hi[st], lo[st]);
        uint64_t left = __ballot(has) & 0xFFFF;
        while (left) {
            int which;
            const uint64_t mine = next_adapter(id, left, which);
            left &= ~mine;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int n = n0 + 16 * j + i16;
                f32x4 o = {0.f, 0.f, 0.f, 0.f}, ol = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < STEPS; st++) {
                    const int r = 32 * st + 8 * g;
                    const f16x8 w = n < p.N && r < p.rank ? __builtin_bit_cast(f16x8, ld_global(reinterpret_cast<const u32x4*>(p.b + ((size_t)which * p.N + n) * p.rank + r))) : f16x8{};
                    ol = mfma_16x16x32_f16(w, lo[st], ol);
                    o = mfma_16x16x32_f16(w, hi[st], o);
                }
                if (mine >> i16 & 1)
#pragma unroll
                    for (int e = 0; e < 4; e++) y[j][e] = fmaf(fmaf(ol[e], 1.f / 2048.f, o[e]), up, y[j][e]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = n0 + 16 * j + 4 * g;
            if (row && n < p.N && (has || p.base != p.y)) st_global(reinterpret_cast<f32x4*>(p.y + (size_t)m * p.N + n), y[j]);
        }
    }
}

}  // namespace

uint64_t plan_lora(LoraArgs* a, size_t ws_bytes)
{
    a->rows = 0;
    if (a->M <= kLoraRowMax) return 0;
    int64_t ranks = 0;
    for (int i = 0; i < a->count; i++) ranks += a->p[i].rank;
    // as many rows at once as have room
    a->rows = (int)std::min<int64_t>(a->M, (int64_t)(ws_bytes / sizeof(float)) / ranks / kUpRows * kUpRows);
    for (int64_t i = 0, at = 0; i < a->count; i++) {
        a->t_off[i] = at;
        at += (int64_t)a->rows * a->p[i].rank;
    }
    return ranks * a->rows * sizeof(float);
}

namespace {

hipError_t launch_tiled(const LoraArgs& a, hipStream_t stream)
{
    const dim3 tiles((a.M + 15) / 16);
    bool done[kMaxBatch] = {};
    for (int i = 0; i < a.count; i++) {
        if (done[i]) continue;
        LoraDown d;
        d.a = a;
        d.x = a.p[i].x;
        d.K = a.p[i].K;
        d.tiles = 0;
        auto flush = [&] {
            if (a.half) hipLaunchKernelGGL(lora_down_kernel<true>, tiles, dim3(64 * kDownWaves), 0, stream, d);
            else hipLaunchKernelGGL(lora_down_kernel<false>, tiles, dim3(64 * kDownWaves), 0, stream, d);
            d.tiles = 0;
        };
        for (int k = i; k < a.count; k++) {
            if (done[k] || a.p[k].x != d.x || a.p[k].K != d.K) continue;
            done[k] = true;
            for (int r = 0; r < a.p[k].rank; r += 16) {
                if (d.tiles == kDownTiles) flush();
                d.p[d.tiles] = (short)k;
                d.r[d.tiles++] = (short)r;
            }
        }
        if (d.tiles) flush();
    }
    for (int i = 0; i < a.count; i++) {
        const dim3 grid((a.p[i].N + kUpCols - 1) / kUpCols, (a.M + kUpRows - 1) / kUpRows);
        if (a.p[i].rank <= 32) hipLaunchKernelGGL(lora_up_kernel<1>, grid, dim3(256), 0, stream, a, i);
        else if (a.p[i].rank <= 64) hipLaunchKernelGGL(lora_up_kernel<2>, grid, dim3(256), 0, stream, a, i);
        else hipLaunchKernelGGL(lora_up_kernel<4>, grid, dim3(256), 0, stream, a, i);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_lora(const LoraArgs& a, hipStream_t stream)
{
    if (!a.rows) {
        int most = 0;
        for (int i = 0; i < a.count; i++) most = std::max(most, a.p[i].N);
        const int split = std::max(1, std::min(512 / (a.M * a.count), most / 1024));
        if (a.half) hipLaunchKernelGGL(lora_row_kernel<true>, dim3(a.M, a.count, split), dim3(64 * kRowWaves), 0, stream, a);
        else hipLaunchKernelGGL(lora_row_kernel<false>, dim3(a.M, a.count, split), dim3(64 * kRowWaves), 0, stream, a);
        return hipGetLastError();
    }
    LoraArgs some = a;
    for (int m = 0; m < a.M; m += a.rows) {
        some.M = std::min(a.rows, a.M - m);
        some.ids = a.ids + m;
        for (int i = 0; i < a.count; i++) {
            some.p[i].x = static_cast<const char*>(a.p[i].x) + (size_t)m * a.p[i].K * (a.half ? 2 : 4);
            some.p[i].base = a.p[i].base + (size_t)m * a.p[i].N;
            some.p[i].y = a.p[i].y + (size_t)m * a.p[i].N;
        }
        const hipError_t e = launch_tiled(some, stream);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ql
