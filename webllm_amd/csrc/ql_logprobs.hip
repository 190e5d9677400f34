// Log probabilities of given tokens under rows of logits, with each row's entropy and its top alternatives
// (ql_token_logprobs). No counterpart in the reference, whose sampler reads the logits on the host.
//
//   lse = m + ln sum e^(x - m),  log p(t) = x_t - lse,  H = ln S - (sum (x - m) e^(x - m)) / S,  S = sum e^(x - m)
// with m the row's largest logit, so nothing cancels however large the logits are; -inf logits (a mask) add nothing. A
// row without any other: log p = -inf, H = 0. Alternatives are ordered by value, equal ones by index.
// S = n + R: the n logits that are m are counted, R is the sum of the others' terms. A sure row's R is far below the last bit of an
// fp32 S, and its log probability and entropy are made of nothing else: ln S = ln n + ln(1 + R / n).
//
// logprob_scan_kernel reads the logits, once: a wave has a unit of 1024 of a row in registers, and leaves the unit's (m, R, sum (x - m)
// e^(x - m), n) and, where alternatives are wanted, the largest (value, index) of each of its four parts of 256. No LDS, no barrier.
// logprob_row_kernel joins a row's units, and finds the top k exactly from the parts' largest: a part whose largest is not
// among the k largest of those has none of the top k (k others are larger), so the k parts that are hold them all, and what
// lies below the smallest of those k is left out. Where more than 256 are left (a masked row's are all alike) the same is done once
// more with the threads' largest, of eight each, which leaves 8 k at most; the rest is sorted.
// Bound: 4 bytes a logit from memory: 512 rows of 151936 take 55.7 us, 5.6 TB/s. With few rows the two launches and their chains
// of loads: 1 row 7.2 us, with alternatives 9.6; 24 rows 8.0, with 20 alternatives 13.9, and 17.8 where a row is masked whole
// (22.2 with one sort of all that is alike).
#include <algorithm>
#include <cmath>

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"
#include "ql_lanes.h"

namespace ql {

namespace {

constexpr int kUnit = 1024, kPart = 256, kParts = kUnit / kPart;   // logits of a wave, of its 16-lane rows
constexpr int kWaves = 16;                                          // of a row's workgroup where alternatives are wanted
constexpr float kLog2e = 1.4426950408889634f, kMaxFinite = 3.4028235e38f;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // rows start at any multiple of 4 bytes

// A logit's order and place as one unsigned number: larger logits first, of equal ones the lower index. NaN above all; 0: none.
__device__ __forceinline__ uint32_t order_bits(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    return x != x ? 0xFFFFFFFFu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint64_t key)
{
    const uint32_t h = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, h & 0x80000000u ? h ^ 0x80000000u : ~h);
}
__device__ __forceinline__ uint64_t key_of(uint32_t bits, uint32_t index) { return (uint64_t)bits << 32 | (uint32_t)~index; }
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// four logits from index i on; those past the row's end are -inf
__device__ __forceinline__ f32x4 load4(const float* x, int i, int V)
{
    if (i + 3 < V) {
        const f32x4u v = *QL_GLOBAL(const f32x4u, x + i);
        return f32x4{v.x, v.y, v.z, v.w};
    }
    f32x4 v;
#pragma unroll
    for (int c = 0; c < 4; c++) v[c] = i + c < V ? ld_global(x + i + c) : -INFINITY;
    return v;
}

template <bool TOP>
__global__ __launch_bounds__(256) void logprob_scan_kernel(const LogprobArgs a)
{
    const int lane = threadIdx.x & 63, unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    const size_t row = blockIdx.y;
    if (unit >= a.units) return;
    const float* x = a.logits + row * a.stride;
    const int i0 = unit * kUnit + 4 * lane;
    f32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) v[u] = load4(x, i0 + kPart * u, a.V);
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int c = 0; c < 4; c++) mx = fmaxf(mx, v[u][c]);
    const float m = wave_max(mx, lane), ref = m == -INFINITY ? 0.f : m;
    float s = 0.f, t = 0.f;
    int n = 0;                                            // the wave's
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float d = v[u][c] - ref, e = __builtin_amdgcn_exp2f(d * kLog2e);
            n += __popcll(__ballot(d == 0.f));
            s += d == 0.f ? 0.f : e;
            t = fmaf(fmaxf(d, -kMaxFinite), e, t);        // -inf: e is 0
        }
    s = wave_sum(s, lane);
    t = wave_sum(t, lane);
    if (lane == 0) st_global(reinterpret_cast<f32x4*>(a.stat) + row * a.units + unit, f32x4{m, s, t, (float)n});
    if (TOP) {
        uint32_t best = 0, at = 0;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int i = i0 + kPart * u + c;
                const uint32_t b = i < a.V ? order_bits(v[u][c]) : 0u;
                if (b > best) {
                    best = b;
                    at = i;
                }
            }
        uint64_t key = best ? key_of(best, at) : 0;
        key = larger(key, lane_xor64<8>(key, lane));
        key = larger(key, lane_xor64<4>(key, lane));
        key = larger(key, lane_xor64<2>(key, lane));
        key = larger(key, lane_xor64<1>(key, lane));
        if ((lane & 15) == 0) st_global(a.best + (row * a.units + unit) * kParts + (lane >> 4), key);
    }
}

// a step of a bitonic network: with the lane ^ J, descending where `down`
template <int J>
__device__ __forceinline__ uint64_t merge_step(uint64_t v, int lane, bool down)
{
    const uint64_t o = lane_xor64<J>(v, lane);
    return ((lane & J) == 0) == down ? larger(v, o) : (v > o ? o : v);
}
template <int J>
__device__ __forceinline__ uint64_t merge_from(uint64_t v, int lane, bool down)
{
    v = merge_step<J>(v, lane, down);
    if constexpr (J > 1) v = merge_from<J / 2>(v, lane, down);
    return v;
}
// descending over the wave's lanes
template <int K = 2>
__device__ __forceinline__ uint64_t sort64(uint64_t v, int lane)
{
    v = merge_from<K / 2>(v, lane, (lane & K) == 0);
    if constexpr (K < 64) v = sort64<2 * K>(v, lane);
    return v;
}
// the largest 64 of two descending lists; b is the second one's from its end
__device__ __forceinline__ uint64_t merge64(uint64_t a, uint64_t b_reversed, int lane)
{
    return merge_from<32>(larger(a, b_reversed), lane, true);
}

// The largest 64 of n keys, descending over wave 0's lanes: each wave sorts 64 at a time, the waves' lists are merged
// through `list` [kWaves][64]. Every thread of the workgroup comes here.
template <bool FEW = false, typename F>
__device__ __forceinline__ uint64_t largest64(F key, int n, int k, uint64_t* list, int wave, int lane)
{
    uint64_t mine = 0;
    for (int i0 = 64 * wave; i0 < n; i0 += 64 * kWaves) {
        const uint64_t v = i0 + lane < n ? key(i0 + lane) : 0;
        if (i0 == 64 * wave) {
            mine = sort64(v, lane);
        } else {
            const uint64_t last = (uint64_t)__shfl((unsigned long long)mine, k - 1);
            if (__any(v > last)) {
                const uint64_t w = sort64(v, lane);
                mine = merge64(mine, (uint64_t)__shfl((unsigned long long)w, 63 - lane), lane);
            }
        }
    }
    const int lists = min(kWaves, (n + 63) / 64);
    if (FEW && lists > 4 && lists * k <= 64) {            // their first k are one list more: 1 row, 5 alternatives 10.2 -> 9.8 us (20: 10.5 -> 10.6)
        if (wave < lists && lane < k) list[wave * k + lane] = mine;
        __syncthreads();
        if (wave == 0) mine = sort64(lane < lists * k ? list[lane] : 0, lane);
        __syncthreads();
        return mine;
    }
    if (wave < lists) list[64 * wave + lane] = mine;
    __syncthreads();
    for (int half = kWaves / 2; half > 0; half >>= 1) {
        if (half >= lists) continue;                      // the same for every thread
        if (wave < half && wave + half < lists) {
            mine = merge64(mine, list[64 * (wave + half) + 63 - lane], lane);
            list[64 * wave + lane] = mine;
        }
        __syncthreads();
    }
    return mine;
}

// A row's units joined by one wave: its largest logit and ln S, and the tokens' log probabilities and the entropy. The logarithm, the
// division and the last subtractions are in 64 bits: what is rounded before them are the sums.
__device__ __forceinline__ void join_units(const LogprobArgs& a, size_t row, int lane, float& ref, double& ls, bool& none)
{
    constexpr int kFirst = 4;                             // units a lane has at once, the first with the first token's logit
    const f32x4* st = reinterpret_cast<const f32x4*>(a.stat) + row * a.units;
    const float* x = a.logits + row * a.stride;
    const f32x4 empty = {-INFINITY, 0.f, 0.f, 0.f};
    f32x4 u[kFirst];
#pragma unroll
    for (int i = 0; i < kFirst; i++) u[i] = lane + 64 * i < a.units ? ld_global(st + lane + 64 * i) : empty;
    auto logit = [&](int i, bool& there) {
        const int tok = ld_global(a.tokens + row * a.n_tok + i);
        there = tok >= 0 && tok < a.V;
        return there ? ld_global(x + tok) : 0.f;
    };
    bool there = false;
    const float xt = lane < a.n_tok ? logit(lane, there) : 0.f;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kFirst; i++) m = fmaxf(m, u[i].x);
    for (int i = lane + 64 * kFirst; i < a.units; i += 64) m = fmaxf(m, ld_global(st + i).x);
    m = wave_max(m, lane);
    ref = m == -INFINITY ? 0.f : m;
    float n = 0.f, s = 0.f, t = 0.f;
    auto add = [&](const f32x4& u) {
        const float d = u.x == -INFINITY ? 0.f : u.x - ref, e = __builtin_amdgcn_exp2f(d * kLog2e), all = u.y + u.w;
        n += d == 0.f ? u.w : 0.f;                        // the unit's largest are the row's
        s = d == 0.f ? s + u.y : fmaf(all, e, s);
        t += e == 0.f ? 0.f : fmaf(d, all, u.z) * e;      // d may be too far down for d * all
    };
#pragma unroll
    for (int i = 0; i < kFirst; i++) add(u[i]);
    for (int i = lane + 64 * kFirst; i < a.units; i += 64) add(ld_global(st + i));
    n = wave_sum(n, lane);
    s = wave_sum(s, lane);
    t = wave_sum(t, lane);
    none = n + s == 0.f;
    const bool sure = s < n * 0x1p-20f;                   // ln(1 + r) = r - r^2 / 2 to 2^-41 of itself
    const double all = (double)n + s, r = sure ? s / n : 0.f;
    ls = log(sure ? (double)n : all) + (r - 0.5 * r * r);
    if (lane == 0 && a.entropy) st_global(a.entropy + row, none ? 0.f : (float)(ls - t / all));
    auto put = [&](int i, bool there, float x) {
        st_global(a.logprob + row * a.n_tok + i, !there ? 0.f : none ? -INFINITY : (float)((double)x - ref - ls));
    };
    if (lane < a.n_tok) put(lane, there, xt);
    for (int i = lane + 64; i < a.n_tok; i += 64) {
        const float xi = logit(i, there);
        put(i, there, xi);
    }
}

__global__ __launch_bounds__(64) void logprob_row_kernel(const LogprobArgs a)
{
    float ref;
    double ls;
    bool none;
    join_units(a, blockIdx.x, threadIdx.x, ref, ls, none);
}

__global__ __launch_bounds__(64 * kWaves) void logprob_top_kernel(const LogprobArgs a)
{
    constexpr int kOwn = (kLogprobMaxTop + kWaves - 1) / kWaves, kKeysOwn = 4 * kOwn;   // parts of a wave, logits of a thread
    constexpr int kFound = kLogprobMaxTop * kKeysOwn;
    __shared__ uint64_t list[64 * kWaves], found[kFound];
    __shared__ double row_max, row_ls;
    __shared__ int count[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.top_k;
    const size_t row = blockIdx.x;
    if (wave == kWaves - 1) {
        float ref;
        double ls;
        bool none;
        join_units(a, row, lane, ref, ls, none);
        if (lane == 0) {
            row_max = ref;
            row_ls = none ? INFINITY : ls;                // a row of no probability: every alternative's is -inf
            count[0] = count[1] = 0;
        }
    }
    const int parts = a.units * kParts;
    const uint64_t* best = a.best + row * parts;
    const uint64_t p = largest64<true>([&](int i) { return ld_global(best + i); }, parts, k, list, wave, lane);
    if (wave == 0) list[lane] = p;
    __syncthreads();
    const float* x = a.logits + row * a.stride;
    uint64_t e[kKeysOwn], most = 0;
#pragma unroll
    for (int o = 0; o < kOwn; o++) {
        const uint64_t key = wave + o * kWaves < k ? list[wave + o * kWaves] : 0;
        const uint32_t at = ~(uint32_t)key;               // a part: 64 neighbours of each 256 of its unit
        const int i0 = (at & ~(kUnit - 1u)) + kPart * (lane >> 4) + (at & 192u) + 4 * (lane & 15);
        const f32x4 v = key ? load4(x, i0, a.V) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; c++) {
            e[4 * o + c] = key && i0 + c < a.V ? key_of(order_bits(v[c]), i0 + c) : 0;
            most = larger(most, e[4 * o + c]);
        }
    }
    uint64_t least = list[k - 1] ? list[k - 1] : 1;
    // the wave's logits from `least` on, and their place behind the other waves'
    auto place = [&](int* total) {
        int mine = 0;
#pragma unroll
        for (int c = 0; c < kKeysOwn; c++) mine += __popcll(__ballot(e[c] >= least));
        int base = 0;
        if (lane == 0 && mine) base = atomicAdd(total, mine);
        return __builtin_amdgcn_readfirstlane(base);
    };
    int base = place(&count[0]);
    __syncthreads();
    int n = count[0];
    if (n > kFound) {                                     // many are alike: once more, from the threads' largest
        largest64([&](int) { return most; }, 64 * kWaves, k, list, wave, lane);
        least = list[k - 1];
        base = place(&count[1]);
        __syncthreads();
        n = count[1];
    }
#pragma unroll
    for (int c = 0; c < kKeysOwn; c++) {
        const uint64_t in = __ballot(e[c] >= least);
        if (e[c] >= least) found[base + __popcll(in & ((1ull << lane) - 1))] = e[c];
        base += __popcll(in);
    }
    __syncthreads();
    const uint64_t top = largest64([&](int i) { return found[i]; }, n, k, list, wave, lane);
    if (wave == 0 && lane < k) {
        st_global(a.top_id + row * k + lane, top ? (int)~(uint32_t)top : -1);
        st_global(a.top_logprob + row * k + lane, !top || row_ls == INFINITY ? -INFINITY : (float)(value_of(top) - row_max - row_ls));
    }
}

}  // namespace

hipError_t launch_token_logprobs(LogprobArgs a, void* ws, size_t ws_bytes, hipStream_t stream)
{
    a.units = (a.V + kUnit - 1) / kUnit;
    const size_t per = token_logprobs_bytes(1, a.V);
    const int rows = (int)std::min<size_t>(a.M, ws_bytes / per);          // more rows go through the workspace in turn
    a.stat = static_cast<float*>(ws);
    a.best = reinterpret_cast<uint64_t*>(static_cast<char*>(ws) + (size_t)rows * a.units * 16);
    const int M = a.M;
    for (int m = 0; m < M; m += rows) {
        a.M = std::min(rows, M - m);
        const dim3 grid((a.units + 3) / 4, a.M);
        if (a.top_k) {
            hipLaunchKernelGGL(logprob_scan_kernel<true>, grid, dim3(256), 0, stream, a);
            hipLaunchKernelGGL(logprob_top_kernel, dim3(a.M), dim3(64 * kWaves), 0, stream, a);
        } else {
            hipLaunchKernelGGL(logprob_scan_kernel<false>, grid, dim3(256), 0, stream, a);
            hipLaunchKernelGGL(logprob_row_kernel, dim3(a.M), dim3(64), 0, stream, a);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        a.logits += (size_t)a.M * a.stride;
        a.tokens += (size_t)a.M * a.n_tok;
        a.logprob += (size_t)a.M * a.n_tok;
        if (a.entropy) a.entropy += a.M;
        a.top_id += (size_t)a.M * a.top_k;
        a.top_logprob += (size_t)a.M * a.top_k;
    }
    return hipSuccess;
}

// a unit's sums and its parts' largest
uint64_t token_logprobs_bytes(int M, int V) { return (uint64_t)M * ((V + kUnit - 1) / kUnit) * (16 + 8 * kParts); }

}  // namespace ql
