// Attention of a tree of drafted tokens over the KV cache (ql_attention_tree), and of any few rows over a long or half cache.
//
//   out[m, h] = sum_s p_s V[s] / sum_s p_s,  p_s = exp(q[m, h] . K[s] / sqrt(D) - max)
// over the cache's past positions and the drafted rows j (at past + j) whose bit is set in row m's mask. A row that sees
// nothing is zero; what it does not see it takes nothing from, not even 0 * V.
//
// attn_tree_kernel: a workgroup has 16 NT (row, head) pairs of one kv head and a range of key blocks; its four waves take
// the blocks in turn, so that K and V go from memory to the registers of one wave, with no shared memory and no barrier
// on the way, and each is split into parts once for 16 NT pairs. Scores are computed transposed, S^T = K Q^T (lane = pair, registers =
// keys), which leaves a lane with the B fragment of O^T = V^T P^T. V's fragment needs eight keys of one column in a lane: a lane loads
// four (fp16: eight) neighbouring columns of eight keys, and the tile of MFMA j takes the j-th of each, so the tile's
// columns are 4 i + j, and nothing crosses lanes. The softmax keeps its running maximum and sum in fp32; the waves' states are
// merged through LDS, the key ranges' (where the pairs do not fill the chip) by attn_tree_merge_*.
//
// fp32 caches: an operand enters as three bf16 parts, 24 bits with fp32's own range, so no value depends on its neighbours' size; a
// product is the six largest of the nine (v_mfma_f32_16x16x32_bf16: 6/16 of the fp32 MFMA's time).
// fp16 caches: K and V enter as they are; q as hi + 2^-11 lo under its row's exponent, in two sums; P as hi + lo of 2^14 P. Two products.
//
// What the parts cannot carry is not finite: an infinity's remainder is a NaN, and 0 * V is one where V is not. A wave whose sums
// end that way does its blocks again on the VALU from q, K and V themselves, skipping what a pair does not see (again()).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"

namespace ql {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kTreeWorkgroups = 512;     // two per CU
constexpr int kTreeMaxSplit = 128;
constexpr float kPScale = 16384.f;       // fp16 parts of P: 2^14 P
constexpr float kMaxFinite = 3.4028235e38f;

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return mfma_16x16x32_f16(a, b, c); }
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// x = p[0] + p[1] + p[2], each the nearest bf16 of what the ones before leave
__device__ __forceinline__ void split_bf16(const float (&x)[8], bf16x8 (&p)[3])
{
#pragma unroll
    for (int e = 0; e < 8; e++) {
        p[0][e] = (__bf16)x[e];
        const float r = x[e] - (float)p[0][e];
        p[1][e] = (__bf16)r;
        p[2][e] = (__bf16)(r - (float)p[1][e]);
    }
}

// the six products of three parts, the small ones first; the largest is the caller's
__device__ __forceinline__ f32x4 small_products(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x4 c)
{
    c = mfma(a[2], b[0], c);
    c = mfma(a[0], b[2], c);
    c = mfma(a[1], b[1], c);
    c = mfma(a[1], b[0], c);
    return mfma(a[0], b[1], c);
}

template <typename T, int DP, int NT, bool FULL>
struct TreeTile {
    static constexpr bool kHalf = std::is_same<T, _Float16>::value;
    static constexpr int kKeys = 32;                        // keys of a block
    static constexpr bool kAhead = DP <= 128;               // a block's K is loaded before the last one's V is used, V before K is
    static constexpr int kNK = kKeys / 16, kNH = kKeys / 32;
    static constexpr int kTD = DP / 32, kDT = DP / 16;
    static constexpr int kParts = kHalf ? 2 : 3;            // of q
    static constexpr int kCols = kHalf && DP >= 128 ? 8 : 4;   // columns of V a lane loads at once
    static constexpr int kChunk = 16 * kCols, kNC = DP / kChunk;   // columns of a load, loads of a row
    static constexpr int kRows = 16 * NT;
    typedef typename std::conditional<kHalf, f16x8, bf16x8>::type Frag;
    typedef typename std::conditional<kHalf, typename std::conditional<kCols == 8, u32x4, u32x2>::type, f32x4>::type VRaw;
    static constexpr int kQBytes = kTD * NT * kParts * 64 * 16;
    static constexpr int kMergeStride = kChunk + 4;
    static constexpr int kMergeBytes = 4 * kRows * kMergeStride * 4;
    static constexpr int kLds = kQBytes > kMergeBytes ? kQBytes : kMergeBytes;
    // the column of tile (c, j), index i
    static __device__ __forceinline__ int col(int c, int j, int i) { return kChunk * c + kCols * i + j; }
    // the column of element e of step t of a K or Q fragment, group g
    static __device__ __forceinline__ int kcol(int t, int g, int e) { return kHalf ? 32 * t + 8 * g + e : 32 * t + 16 * (e >> 2) + 4 * g + (e & 3); }
};

// A block's first key, its number of keys, and which of them pair row m sees.
struct TreeBlock {
    int base, n, j0;                                        // j0: the first drafted row, or -1 in the context
};
template <int KEYS>
__device__ __forceinline__ TreeBlock tree_block(const TreeArgs& a, int b, int past_blocks)
{
    TreeBlock k;
    if (b < past_blocks) {
        k.base = b * KEYS;
        k.n = min(KEYS, a.past - k.base);
        k.j0 = -1;
    } else {
        k.j0 = (b - past_blocks) * KEYS;
        k.base = a.past + k.j0;
        k.n = min(KEYS, a.M - k.j0);
    }
    return k;
}
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }
__device__ __forceinline__ uint64_t seen_bits(const TreeArgs& a, const TreeBlock& k, int m)
{
    if (k.j0 < 0) return low_bits(k.n);
    const uint64_t w = a.mask ? ld_global(a.mask + (size_t)m * a.words + (k.j0 >> 6)) >> (k.j0 & 63) : low_bits(m - k.j0 + 1);
    return w & low_bits(k.n);
}

// The wave's blocks on the VALU, in the layout of the kernel below.
template <typename T, int DP, int NT, bool FULL>
__device__ __attribute__((noinline)) void tree_again(const TreeArgs& a, int kvh, int first, int end, int past_blocks, const int (&qrow)[NT], const int (&qm)[NT],
                                                     float (&mr)[NT], float (&l)[NT], f32x4 (&acc)[DP / 16][NT])
{
    using C = TreeTile<T, DP, NT, FULL>;
    const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
    const size_t row_len = (size_t)a.KV * a.D;
    const T* kb = static_cast<const T*>(a.k) + (size_t)kvh * a.D;
    const T* vb = static_cast<const T*>(a.v) + (size_t)kvh * a.D;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        mr[nt] = -INFINITY;
        l[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < C::kDT; d++) acc[d][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int b = first; b < end; b += 4) {
        const TreeBlock blk = tree_block<C::kKeys>(a, b, past_blocks);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const uint64_t seen = seen_bits(a, blk, qm[nt]);
            const float* q = a.q + (size_t)qrow[nt] * a.D;
            // four of the block's keys per lane and 16; then each lane takes all of them to its columns
#pragma unroll 1
            for (int kt = 0; kt < C::kNK; kt++) {
                float s[4], bm = -INFINITY;
#pragma unroll 1
                for (int r = 0; r < 4; r++) {
                    const int i = 16 * kt + 4 * g + r;
                    float sc = -INFINITY;
                    if (seen >> i & 1) {
                        const T* k = kb + (size_t)(blk.base + i) * row_len;
                        sc = 0.f;
                        for (int d = 0; d < a.D; d++) sc = fmaf(q[d], (float)k[d], sc);
                        sc *= a.scale;
                    }
                    s[0] = r == 0 ? sc : s[0];
                    s[1] = r == 1 ? sc : s[1];
                    s[2] = r == 2 ? sc : s[2];
                    s[3] = r == 3 ? sc : s[3];
                    bm = fmaxf(bm, sc);
                }
                bm = fmaxf(bm, __shfl_xor(bm, 16));
                bm = fmaxf(bm, __shfl_xor(bm, 32));
                const float mn = fmaxf(mr[nt], bm), ref = mn == -INFINITY ? 0.f : mn, al = ex2(mr[nt] - ref);
                mr[nt] = mn;
                l[nt] *= al;
#pragma unroll
                for (int d = 0; d < C::kDT; d++) acc[d][nt] *= al;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    s[r] = seen >> (16 * kt + 4 * g + r) & 1 ? ex2(s[r] - ref) : 0.f;
                    l[nt] += s[r];
                }
#pragma unroll 1
                for (int key = 0; key < 16; key++) {
                    const int r = key & 3;
                    const float mine = r == 0 ? s[0] : r == 1 ? s[1] : r == 2 ? s[2] : s[3];
                    const float p = __shfl(mine, 16 * (key >> 2) + i16);
                    if (!(seen >> (16 * kt + key) & 1)) continue;      // differs between lanes, but not between the four of a pair
                    const T* v = vb + (size_t)(blk.base + 16 * kt + key) * row_len;
#pragma unroll
                    for (int c = 0; c < C::kNC; c++)
#pragma unroll
                        for (int j = 0; j < C::kCols; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int d = C::col(c, j, 4 * g + e);
                                if (FULL || d < a.D) acc[c * C::kCols + j][nt][e] = fmaf(p, (float)v[d], acc[c * C::kCols + j][nt][e]);
                            }
                }
            }
        }
    }
}

template <typename T, int DP, int NT, bool FULL>
__global__ __launch_bounds__(256, 2) void attn_tree_kernel(const TreeArgs a)
{
    using C = TreeTile<T, DP, NT, FULL>;
    using Frag = typename C::Frag;
    __shared__ __attribute__((aligned(16))) char lds[C::kLds];
    __shared__ float qscale[C::kRows], stat[2][4][C::kRows];
    const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % a.KV, split = blockIdx.x / a.KV, rg = blockIdx.y;
    const int R = a.M * a.G, D = a.D, last_key = a.past + a.M - 1;
    const int past_blocks = (a.past + C::kKeys - 1) / C::kKeys, blocks = past_blocks + (a.M + C::kKeys - 1) / C::kKeys;
    const int per = (blocks + a.nsplit - 1) / a.nsplit;
    const int b0 = min(blocks, split * per), b1 = min(blocks, b0 + per);
    const size_t row_len = (size_t)a.KV * D;
    const T* kb = static_cast<const T*>(a.k) + (size_t)kvh * D;
    const T* vb = static_cast<const T*>(a.v) + (size_t)kvh * D;
    auto pair_row = [&](int r, int& m) {                    // pair r of this kv head as a row of q and out
        m = r / a.G;
        return m * a.H + kvh * a.G + (r - m * a.G);
    };

    // K of the wave's first block is on its way while q's parts are made
    typename std::conditional<C::kHalf, u32x4, f32x4>::type kraw[C::kNK][C::kTD * (C::kHalf ? 1 : 2)];
    auto load_k = [&](const TreeBlock& blk, int from, int to) {
#pragma unroll
        for (int kt = from; kt < to; kt++) {
            const T* p = kb + (size_t)min(blk.base + 16 * kt + i16, last_key) * row_len;
#pragma unroll
            for (int t = 0; t < C::kTD; t++)
                if constexpr (C::kHalf) {
                    const int d = 32 * t + 8 * g;
                    kraw[kt][t] = FULL || d < D ? ld_global(reinterpret_cast<const u32x4*>(p + d)) : u32x4{0, 0, 0, 0};
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int d = 32 * t + 16 * h + 4 * g;
                        kraw[kt][2 * t + h] = FULL || d < D ? ld_global(reinterpret_cast<const f32x4*>(p + d)) : f32x4{0.f, 0.f, 0.f, 0.f};
                    }
                }
        }
    };
    int b = b0 + wave;
    TreeBlock blk = tree_block<C::kKeys>(a, min(b, blocks - 1), past_blocks);
    if (C::kAhead && b < b1) load_k(blk, 0, C::kNK);

    // q's parts as fragments in LDS: unit (t, nt, part), lane (i, g)
    Frag* qf = reinterpret_cast<Frag*>(lds);
    if (C::kHalf) {
        constexpr int P = 256 / C::kRows;                   // threads a row
        int m;
        const float* q = a.q + (size_t)pair_row(min(rg * C::kRows + tid / P, R - 1), m) * D;
        float mx = 0.f;
        for (int d = 4 * (tid % P); d < D; d += 4 * P) {
            const f32x4 x = ld_global(reinterpret_cast<const f32x4*>(q + d));
            mx = fmaxf(fmaxf(mx, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
        }
#pragma unroll
        for (int o = 1; o < P; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        if (tid % P == 0) qscale[tid / P] = mx > 0.f && mx <= kMaxFinite ? ldexpf(1.f, min(100, 14 - ilogbf(mx))) : 1.f;
        __syncthreads();
    }
    for (int u = tid; u < C::kTD * NT * 64; u += 256) {
        const int ln = u & 63, t = (u >> 6) / NT, nt = (u >> 6) % NT, row = 16 * nt + (ln & 15);
        int m;
        const float* q = a.q + (size_t)pair_row(min(rg * C::kRows + row, R - 1), m) * D;
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int d = C::kcol(t, ln >> 4, 4 * h);
            const f32x4 y = FULL || d < D ? ld_global(reinterpret_cast<const f32x4*>(q + d)) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * h + e] = y[e];
        }
        Frag* dst = qf + (size_t)(u >> 6) * C::kParts * 64 + ln;
        if constexpr (C::kHalf) {
            const float s = qscale[row];
            f16x8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = x[e] * s;
                hi[e] = (_Float16)y;
                lo[e] = (_Float16)((y - (float)hi[e]) * 2048.f);
            }
            dst[0] = hi;
            dst[64] = lo;
        } else {
            bf16x8 p[3];
            split_bf16(x, p);
            dst[0] = p[0];
            dst[64] = p[1];
            dst[128] = p[2];
        }
    }
    int qrow[NT], qm[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) qrow[nt] = pair_row(min(rg * C::kRows + 16 * nt + i16, R - 1), qm[nt]);
    __syncthreads();

    f32x4 acc[C::kDT][NT];
    float mr[NT], l[NT], f[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        mr[nt] = -INFINITY;
        l[nt] = 0.f;
        f[nt] = C::kHalf ? fmaxf(a.scale / qscale[16 * nt + i16], 1.17549435e-38f) : a.scale;
#pragma unroll
        for (int d = 0; d < C::kDT; d++) acc[d][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int first = b;
    for (; b < b1; b += 4) {
        typename C::VRaw vraw[C::kNH][8][C::kNC];           // [32 keys][element of the fragment][columns]
        auto load_v = [&](const TreeBlock& blk, int c0, int c1) {
#pragma unroll
            for (int h = 0; h < C::kNH; h++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const T* p = vb + (size_t)min(blk.base + 32 * h + 16 * (e >> 2) + 4 * g + (e & 3), last_key) * row_len;
#pragma unroll
                    for (int c = c0; c < c1; c++) {
                        const int d = C::kChunk * c + C::kCols * i16;
                        if (FULL || d < D) vraw[h][e][c] = ld_global(reinterpret_cast<const typename C::VRaw*>(p + d));
                        else vraw[h][e][c] = typename C::VRaw{};
                    }
                }
        };
        f32x4 s[C::kNK][NT];
#pragma unroll
        for (int kt = 0; kt < C::kNK; kt++) {
            if (!C::kAhead) load_k(blk, kt, kt + 1);
            if (C::kAhead && kt == 1) {
                __builtin_amdgcn_sched_barrier(0);          // not before the first keys' registers are free
                load_v(blk, 0, C::kNC);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (C::kHalf) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < C::kTD; t++) {
                        const f16x8* q = qf + (size_t)(t * NT + nt) * 128 + lane;
                        const f16x8 k = __builtin_bit_cast(f16x8, kraw[kt][t]);
                        lo = mfma(k, q[64], lo);
                        hi = mfma(k, q[0], hi);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) s[kt][nt][r] = fmaf(lo[r], 1.f / 2048.f, hi[r]);
                }
            } else {
                // the small products first: the sum takes its full size only in the last ones, and half of those apart
                bf16x8 kh[C::kTD];
                f32x4 lo[NT], hi[NT];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) lo[nt] = hi[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 0; t < C::kTD; t++) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = kraw[kt][2 * t + (e >> 2)][e & 3];
                    bf16x8 kp[3];
                    split_bf16(x, kp);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const bf16x8* q = qf + (size_t)(t * NT + nt) * 192 + lane;
                        const bf16x8 qp[3] = {q[0], q[64], q[128]};
                        lo[nt] = small_products(kp, qp, lo[nt]);
                    }
                    kh[t] = kp[0];
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int t = 0; t < C::kTD; t++) {
                        const bf16x8 q = qf[(size_t)(t * NT + nt) * 192 + lane];
                        if (t < C::kTD / 2) lo[nt] = mfma(kh[t], q, lo[nt]);
                        else hi[nt] = mfma(kh[t], q, hi[nt]);
                    }
                    s[kt][nt] = lo[nt] + hi[nt];
                }
            }
        }
        const TreeBlock now = blk;
        if (b + 4 < b1) {
            blk = tree_block<C::kKeys>(a, b + 4, past_blocks);
            if (C::kAhead) {
                __builtin_amdgcn_sched_barrier(0);
                load_k(blk, 0, C::kNK);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (now.j0 >= 0 || now.n < C::kKeys) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint64_t seen = seen_bits(a, now, qm[nt]) >> (4 * g);
#pragma unroll
                for (int kt = 0; kt < C::kNK; kt++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (!(seen >> (16 * kt + r) & 1)) s[kt][nt][r] = -INFINITY;
            }
        }
        Frag pf[C::kNH][NT][C::kParts];
        float al[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float bm = s[0][nt][0];
#pragma unroll
            for (int kt = 0; kt < C::kNK; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) bm = fmaxf(bm, s[kt][nt][r]);
            bm = fmaxf(bm, __shfl_xor(bm, 16));
            bm = fmaxf(bm, __shfl_xor(bm, 32));
            const float mn = fmaxf(mr[nt], bm * f[nt]), ref = mn == -INFINITY ? 0.f : mn;
            al[nt] = ex2(mr[nt] - ref);
            mr[nt] = mn;
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < C::kNH; h++) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    p[e] = ex2(fmaf(s[2 * h + (e >> 2)][nt][e & 3], f[nt], -ref));
                    sum += p[e];
                }
                if constexpr (C::kHalf) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float y = p[e] * kPScale;
                        pf[h][nt][0][e] = (_Float16)y;
                        pf[h][nt][1][e] = (_Float16)(y - (float)pf[h][nt][0][e]);
                    }
                } else {
                    split_bf16(p, pf[h][nt]);
                }
            }
            l[nt] = l[nt] * al[nt] + sum;
        }
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) moved = moved || al[nt] != 1.f;
        if (__any(moved))
#pragma unroll
            for (int d = 0; d < C::kDT; d++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) acc[d][nt] *= al[nt];
        // a block's sums start from zero and are added to the others by the VALU: the matrix unit carries no long sum
#pragma unroll
        for (int c = 0; c < C::kNC; c++) {
            if (!C::kAhead) load_v(now, c, c + 1);
#pragma unroll
            for (int j = 0; j < C::kCols; j++) {
                f32x4 o[NT];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) o[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (C::kHalf) {
                    f16x8 v[C::kNH];
#pragma unroll
                    for (int h = 0; h < C::kNH; h++) {
                        u32x4 w;
#pragma unroll
                        for (int e = 0; e < 4; e++)         // column j of keys 2 e and 2 e + 1
                            w[e] = __builtin_amdgcn_perm(vraw[h][2 * e + 1][c][j / 2], vraw[h][2 * e][c][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
                        v[h] = __builtin_bit_cast(f16x8, w);
                    }
#pragma unroll
                    for (int part = 1; part >= 0; part--)
#pragma unroll
                        for (int h = 0; h < C::kNH; h++)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) o[nt] = mfma(v[h], pf[h][nt][part], o[nt]);
                } else {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = vraw[0][e][c][j];
                    bf16x8 vp[3];
                    split_bf16(x, vp);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) o[nt] = mfma(vp[0], pf[0][nt][0], small_products(vp, pf[0][nt], o[nt]));
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) acc[c * C::kCols + j][nt] += o[nt];
            }
        }
    }
    float odd = 0.f;                                        // NaN if a sum is not finite
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        odd = fmaf(l[nt], 0.f, odd);
#pragma unroll
        for (int d = 0; d < C::kDT; d++)
#pragma unroll
            for (int r = 0; r < 4; r++) odd = fmaf(acc[d][nt][r], 0.f, odd);
    }
    const bool redo = __any(odd != 0.f);
    if (redo) {                                             // through copies: the sums themselves stay in registers
        int row[NT], m[NT];
        float mx[NT], sum[NT];
        f32x4 o[C::kDT][NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            row[nt] = qrow[nt];
            m[nt] = qm[nt];
        }
        tree_again<T, DP, NT, FULL>(a, kvh, first, b1, past_blocks, row, m, mx, sum, o);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            mr[nt] = mx[nt];
            l[nt] = sum[nt];
#pragma unroll
            for (int d = 0; d < C::kDT; d++) acc[d][nt] = o[d][nt];
        }
    }

    // the four waves' states
    const float unit = C::kHalf && !redo ? 1.f / kPScale : 1.f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        l[nt] += __shfl_xor(l[nt], 16);
        l[nt] += __shfl_xor(l[nt], 32);
        if (g == 0) {
            stat[0][wave][16 * nt + i16] = mr[nt];
            stat[1][wave][16 * nt + i16] = l[nt];
        }
    }
    __syncthreads();                                        // also: q's parts are no longer read
    float* merge = reinterpret_cast<float*>(lds);
    float w[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = 16 * nt + i16;
        const float mx = fmaxf(fmaxf(stat[0][0][r], stat[0][1][r]), fmaxf(stat[0][2][r], stat[0][3][r]));
        w[nt] = mr[nt] == -INFINITY ? 0.f : ex2(mr[nt] - mx) * unit;
        if (mr[nt] == -INFINITY && l[nt] != l[nt]) w[nt] = 1.f;   // scores that are all NaN
    }
#pragma unroll
    for (int c = 0; c < C::kNC; c++) {
        if (c) __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float* dst = merge + (size_t)(wave * C::kRows + 16 * nt + i16) * C::kMergeStride;
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int j = 0; j < C::kCols; j += 4) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = w[nt] == 0.f ? 0.f : acc[c * C::kCols + j + e][nt][r] * w[nt];
                    *reinterpret_cast<f32x4*>(dst + C::kCols * (4 * g + r) + j) = v;
                }
        }
        __syncthreads();
        for (int u = tid; u < C::kRows * (C::kChunk / 4); u += 256) {
            const int row = u / (C::kChunk / 4), c4 = u % (C::kChunk / 4), d = C::kChunk * c + 4 * c4, r = rg * C::kRows + row;
            if (r >= R || (!FULL && d >= D)) continue;
            f32x4 sum = *reinterpret_cast<const f32x4*>(merge + (size_t)row * C::kMergeStride + 4 * c4);
#pragma unroll
            for (int k = 1; k < 4; k++) sum += *reinterpret_cast<const f32x4*>(merge + (size_t)(k * C::kRows + row) * C::kMergeStride + 4 * c4);
            const float mx = fmaxf(fmaxf(stat[0][0][row], stat[0][1][row]), fmaxf(stat[0][2][row], stat[0][3][row]));
            float total = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float lk = stat[1][k][row], mk = stat[0][k][row];
                total += mk == -INFINITY ? (lk != lk ? lk : 0.f) : lk * ex2(mk - mx);
            }
            int m;
            const size_t at = pair_row(r, m);
            if (a.nsplit == 1) {
                const float inv = total == 0.f ? 0.f : 1.f / total;
                st_global(reinterpret_cast<f32x4*>(a.out + at * D + d), f32x4{sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv});
            } else {
                const size_t slot = at * a.nsplit + split;
                st_global(reinterpret_cast<f32x4*>(a.ws + slot * D + d), sum);
                if (d == 0) {
                    float* st = a.ws + (size_t)a.M * a.H * a.nsplit * D + 2 * slot;
                    st_global(st, mx);
                    st_global(st + 1, total);
                }
            }
        }
    }
}

// out = sum_i acc_i 2^(m_i - m) / sum_i l_i 2^(m_i - m) over the key ranges, a workgroup a row: the ranges' weights in
// LDS, then thread (part p, four columns c) adds ranges p, p + P, ... in order, and the P parts are added in order
__global__ __launch_bounds__(256) void attn_tree_merge_kernel(const TreeArgs a)
{
    __shared__ float wgt[kTreeMaxSplit];
    __shared__ f32x4 part[256];
    const size_t row = (size_t)blockIdx.y * a.H + blockIdx.x;
    const int t = threadIdx.x, S = a.nsplit, D = a.D;
    if (t < 64) {
        const float* st = a.ws + (size_t)a.M * a.H * S * D + 2 * row * S;
        float mi[2], li[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int i = t + 64 * r;
            mi[r] = i < S ? ld_global(st + 2 * i) : -INFINITY;
            li[r] = i < S ? ld_global(st + 2 * i + 1) : 0.f;
        }
        float mx = fmaxf(mi[0], mi[1]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        float e[2], l = 0.f;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            e[r] = mi[r] == -INFINITY ? (li[r] != li[r] ? li[r] : 0.f) : ex2(mi[r] - mx);
            l += li[r] * e[r];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
#pragma unroll
        for (int r = 0; r < 2; r++) wgt[t + 64 * r] = l == 0.f ? 0.f : e[r] / l;
    }
    __syncthreads();
    const int nc = D / 4, P = 256 / nc, c = t % nc, p = t / nc;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (p < P) {
        const f32x4* src = reinterpret_cast<const f32x4*>(a.ws + row * S * D) + c;
#pragma unroll 4
        for (int i = p; i < S; i += P) {
            const float w = wgt[i];
            const f32x4 v = ld_global(src + (size_t)i * nc);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(w, v[e], o[e]);
        }
    }
    part[t] = o;
    __syncthreads();
    if (t < nc) {
        f32x4 r = part[t];
        for (int k = 1; k < P; k++) r += part[k * nc + t];
        st_global(reinterpret_cast<f32x4*>(a.out + row * D) + t, r);
    }
}

typedef void (*TreeFn)(TreeArgs);

template <typename T>
TreeFn tree_fn(int D, int nt)
{
    if (D == 64) return nt == 2 ? attn_tree_kernel<T, 64, 2, true> : attn_tree_kernel<T, 64, 1, true>;
    if (D == 128) return nt == 2 ? attn_tree_kernel<T, 128, 2, true> : attn_tree_kernel<T, 128, 1, true>;
    if (D == 256) return attn_tree_kernel<T, 256, 1, true>;
    if (D < 64) return attn_tree_kernel<T, 64, 1, false>;
    if (D < 128) return attn_tree_kernel<T, 128, 1, false>;
    return attn_tree_kernel<T, 256, 1, false>;
}

}  // namespace

uint64_t plan_attention_tree(TreeArgs* a, size_t ws_bytes)
{
    const int R = a->M * a->G, keys = 32;
    a->nt = (a->D == 64 || a->D == 128) && R > 16 ? 2 : 1;
    a->groups = (R + 16 * a->nt - 1) / (16 * a->nt);
    const int blocks = (a->past + keys - 1) / keys + (a->M + keys - 1) / keys;
    const size_t one = (size_t)a->M * a->H * (a->D + 2) * sizeof(float);
    // key ranges up to two workgroups a CU, of at least a block a wave, as many as the workspace holds
    const int s = std::max(1, std::min({kTreeWorkgroups / (a->groups * a->KV), (blocks + 3) / 4, kTreeMaxSplit, (int)std::min<size_t>(kTreeMaxSplit, ws_bytes / one)}));
    const int per = (blocks + s - 1) / s;
    a->nsplit = (blocks + per - 1) / per;
    return a->nsplit == 1 ? 0 : a->nsplit * one;
}

hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t stream)
{
    const TreeFn fn = a.half ? tree_fn<_Float16>(a.D, a.nt) : tree_fn<float>(a.D, a.nt);
    hipLaunchKernelGGL(fn, dim3(a.nsplit * a.KV, a.groups), dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1) return e;
    hipLaunchKernelGGL(attn_tree_merge_kernel, dim3(a.H, a.M), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace ql
