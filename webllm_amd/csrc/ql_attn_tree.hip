// Attention of a tree of drafted tokens over the KV cache (ql_attention_tree), and of any few rows over a long or half cache.
//
//   out[m, h] = sum_s p_s V[s] / sum_s p_s,  p_s = exp(q[m, h] . K[s] / sqrt(D) - max)
// over the cache's past positions and the drafted rows j (at past + j) whose bit is set in row m's mask. A row that sees
// nothing is zero; what it does not see it takes nothing from, not even 0 * V.
//
// attn_tree_kernel: a workgroup has 16 NT (row, head) pairs of one kv head and a range of key blocks; its four or eight waves take
// the blocks in turn, so that K and V go from memory to the registers of one wave, with no barrier
// on the way, and each is split into parts once for 16 NT pairs. Scores are computed transposed, S^T = K Q^T (lane = pair, registers =
// keys), which leaves a lane with the B fragment of O^T = V^T P^T. V's fragment needs eight keys of one column in a lane: a lane loads
// four (fp16: eight) neighbouring columns of eight keys, and the tile of MFMA j takes the j-th of each, so the tile's
// columns are 4 i + j, and nothing crosses lanes. The softmax keeps its running reference and sum in fp32; the waves' states are
// merged through LDS, the key ranges' (where the pairs do not fill the chip) by attn_tree_merge_kernel. Contexts of fewer keys than
// a block: attn_tree_row_kernel, a wave a (row, head).
//
// fp32 caches: an operand enters as three bf16 parts, 24 bits with fp32's own range, so no value depends on its neighbours' size; a
// product is the six largest of the nine (v_mfma_f32_16x16x32_bf16: 6/16 of the fp32 MFMA's time).
// fp16 caches: K and V enter as they are; q as hi + 2^-11 lo under its row's exponent, in two sums; P as hi + lo of 2^8 P. Two products.
// P's parts hold 22 bits of a weight down to 2^-10 of the running reference, below that to half a step of 2^-24, 2^-33 of the reference: T
// keys of a wave are off by T 2^-33 of the largest |V| at most, a sixteenth of what their T / 32 fp32 additions may be. Finer parts,
// and what 256 rows after 8000 keys took for 91.0 us: lo as 2^-11 lo in a sum of its own (2^-44 of the reference) 96.0, a reference
// raised at 2^1 in place of 2^7 and 2^14 P (2^-39) 93.9, at 2^3 and 2^12 P (2^-37) 91.8.
//
// What the parts cannot carry is not finite: an infinity's remainder is a NaN, and 0 * V is one where V is not. A wave whose sums
// end that way does its blocks again on the VALU from q, K and V themselves, skipping what a pair does not see (tree_again).
//
// us, of them the merge, and what bounds it (28 / 4 heads of 128): 1 row after 32000 fp16 keys 17.1, 4, memory (65.5 MB; fp32 35.2); 24 rows
// after 4000 fp32 keys 23.3, 4, the parts' VALU work and the matrix unit in turn, on CUs that have one or two workgroups;
// 256 after 8000 fp16 keys 86.4, 5, issue: two waves a SIMD fit its registers, the VALU is busy half of the
// cycles, the matrix unit 28 %; fp32 205.8. 14 / 2 heads of 64: 5 rows after 300 fp32 keys 7.4, one launch and its chain of loads.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"
#include "ql_lanes.h"

namespace ql {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kTreeMaxSplit = 128;
constexpr int kKeys = kTreeKeys;         // keys of a block
constexpr float kRaise = 7.f;            // log2 that scores may rise above the running reference before it is raised
constexpr float kPScale = 256.f;         // fp16 parts of P: 2^8 P, at most 2^15
constexpr float kMaxFinite = 3.4028235e38f;

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return mfma_16x16x32_f16(a, b, c); }
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// x = p[0] + p[1] + p[2], exactly: each part the first eight bits of what the ones before leave (5.5 instructions a value; the
// nearest ones instead of the first took 8.4, since conversions come in pairs)
__device__ __forceinline__ void split_bf16(const float (&x)[8], bf16x8 (&p)[3])
{
    u32x4 w[3];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        uint32_t b[2][3];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            float r = x[2 * e + k];
#pragma unroll
            for (int i = 0; i < 3; i++) {
                b[k][i] = __builtin_bit_cast(uint32_t, r);
                if (i < 2) r -= __builtin_bit_cast(float, b[k][i] & 0xFFFF0000u);
            }
        }
#pragma unroll
        for (int i = 0; i < 3; i++) w[i][e] = __builtin_amdgcn_perm(b[1][i], b[0][i], 0x07060302u);
    }
#pragma unroll
    for (int i = 0; i < 3; i++) p[i] = __builtin_bit_cast(bf16x8, w[i]);
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

template <typename T, int DP, int NT, bool FULL, int WAVES>
struct TreeTile {
    static constexpr bool kHalf = std::is_same<T, _Float16>::value;
    static constexpr bool kAhead = DP <= 128;               // a block's K is loaded before the last one's V is used, V before K is
    static constexpr int kNK = kKeys / 16;
    static constexpr int kTD = DP / 32, kDT = DP / 16;
    static constexpr int kParts = kHalf ? 2 : 3;            // of q
    static constexpr int kCols = kHalf && DP >= 128 ? 8 : 4;   // columns of V a lane loads at once
    static constexpr int kChunk = 16 * kCols, kNC = DP / kChunk;   // columns of a load, loads of a row
    static constexpr int kRows = 16 * NT;
    typedef typename std::conditional<kHalf, f16x8, bf16x8>::type Frag;
    typedef typename std::conditional<kHalf, typename std::conditional<kCols == 8, u32x4, u32x2>::type, f32x4>::type VRaw;
    static constexpr int kQBytes = kTD * NT * kParts * 64 * 16;
    static constexpr int kMergeStride = kChunk + 4;
    static constexpr int kMergeBytes = WAVES * kRows * kMergeStride * 4;
    // K of kAhead: 16 bytes a lane, whole rows; units of a row, rows of a load, loads of 16 keys, a row's bytes in LDS
    static constexpr int kRowUnits = DP * (int)sizeof(T) / 16, kLoadRows = 64 / kRowUnits, kLoads = 16 / kLoadRows;
    static constexpr int kTurnStride = 16 * kRowUnits + 16;
    static constexpr int kTurnBytes = kAhead ? 16 * kTurnStride : 0;
    static constexpr int kLoopBytes = kQBytes + WAVES * kTurnBytes;
    static constexpr int kLds = kLoopBytes > kMergeBytes ? kLoopBytes : kMergeBytes;
    // the column of element e of step t of a K or Q fragment, group g
    static __device__ __forceinline__ int kcol(int t, int g, int e) { return kHalf ? 32 * t + 8 * g + e : 32 * t + 16 * (e >> 2) + 4 * g + (e & 3); }
};

// A block of up to 32 keys, all of them in the context or all drafted. It is read as the 32 keys from `at` on, which all
// exist (the call has that many): where the last keys are fewer, those before them come along unseen.
struct TreeBlock {
    int base, n, j0, at;                                    // j0: the first drafted row, or -1 in the context
};
__device__ __forceinline__ TreeBlock tree_block(const TreeArgs& a, int b, int past_blocks)
{
    TreeBlock k;
    if (b < past_blocks) {
        k.base = b * kKeys;
        k.n = min(kKeys, a.past - k.base);
        k.j0 = -1;
    } else {
        k.j0 = (b - past_blocks) * kKeys;
        k.base = a.past + k.j0;
        k.n = min(kKeys, a.M - k.j0);
    }
    k.at = min(k.base, a.past + a.M - kKeys);
    return k;
}
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : (1ull << n) - 1; }   // n < 64
// which of the keys from k.base on query row m sees
__device__ __forceinline__ uint64_t seen_bits(const TreeArgs& a, const TreeBlock& k, int m)
{
    if (k.j0 < 0) return low_bits(k.n);
    const uint64_t w = a.mask ? ld_global(a.mask + (size_t)m * a.words + (k.j0 >> 6)) >> (k.j0 & 63) : low_bits(min(m - k.j0 + 1, kKeys));
    return w & low_bits(k.n);
}
// the row of q and out of pair r of kv head kvh, and its query row m
__device__ __forceinline__ int pair_row(const TreeArgs& a, int kvh, int r, int& m)
{
    r = min(r, a.M * a.G - 1);
    m = (int)(((float)r + 0.5f) * a.inv_g);                 // r / G, exact: r < 2^20
    return m * a.H + kvh * a.G + (r - m * a.G);
}

// The wave's blocks on the VALU, in the layout of the kernel below.
// Blocks first, first + step, ... before `end`; a lane's columns come COLS at a time.
template <typename T, int DP, int NT, bool FULL, int COLS>
__device__ __forceinline__ void tree_again(const TreeArgs& a, int kvh, int r0, int first, int end, int step, int past_blocks, float (&mr)[NT], float (&l)[NT],
                                           f32x4 (&acc)[DP / 16][NT])
{
    const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
    const size_t row_len = (size_t)a.KV * a.D;
    const T* kb = static_cast<const T*>(a.k) + (size_t)kvh * a.D;
    const T* vb = static_cast<const T*>(a.v) + (size_t)kvh * a.D;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        mr[nt] = -INFINITY;
        l[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < DP / 16; d++) acc[d][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int b = first; b < end; b += step) {
        const TreeBlock blk = tree_block(a, b, past_blocks);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            int m;
            const float* q = a.q + (size_t)pair_row(a, kvh, r0 + 16 * nt + i16, m) * a.D;
            const uint64_t seen = seen_bits(a, blk, m);
            // four of the block's keys per lane and 16; then each lane takes all of them to its columns
#pragma unroll 1
            for (int kt = 0; kt < kKeys / 16; kt++) {
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
                bm = pair_max<32>(pair_max<16>(bm));
                const float mn = fmaxf(mr[nt], bm), ref = mn == -INFINITY ? 0.f : mn, al = ex2(mr[nt] - ref);
                mr[nt] = mn;
                l[nt] *= al;
#pragma unroll
                for (int d = 0; d < DP / 16; d++) acc[d][nt] *= al;
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
                    for (int c = 0; c < DP / (16 * COLS); c++)
#pragma unroll
                        for (int j = 0; j < COLS; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int d = 16 * COLS * c + COLS * (4 * g + e) + j;
                                if (FULL || d < a.D) acc[c * COLS + j][nt][e] = fmaf(p, (float)v[d], acc[c * COLS + j][nt][e]);
                            }
                }
            }
        }
    }
}

template <typename T, int DP, int NT, bool FULL, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void attn_tree_kernel(const TreeArgs a)
{
    using C = TreeTile<T, DP, NT, FULL, WAVES>;
    using Frag = typename C::Frag;
    __shared__ __attribute__((aligned(16))) char lds[C::kLds];
    __shared__ float qmax[C::kHalf ? C::kTD : 1][C::kRows], stat[2][WAVES][C::kRows], row_inv[C::kRows];
    __shared__ int row_at[C::kRows];
    const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups go to the eight XCDs in turn. The groups of pairs that read the same keys, (kv head, range) number p, are to
    // share one's L2: x = 8 * group + p % 8, y = p / 8. A kv head's keys lie in a few of the L2's channels (row stride), so an
    // XCD has ranges of all the kv heads (of one only: 24 rows after 4000 keys 44 us for 33).
    const int p = 8 * blockIdx.y + (blockIdx.x & 7), rg = blockIdx.x >> 3;
    if (p >= a.KV * a.nsplit) return;
    const int kvh = __builtin_amdgcn_readfirstlane((int)(((float)p + 0.5f) * a.inv_nsplit)), split = p - kvh * a.nsplit;   // exact: p < 2^19
    const int R = a.M * a.G, D = a.D;
    const int past_blocks = a.past_blocks, blocks = a.blocks, b0 = split * a.per, b1 = min(blocks, b0 + a.per);
    const size_t row_len = (size_t)a.KV * D;
    const T* kb = static_cast<const T*>(a.k) + (size_t)kvh * D;
    const T* vb = static_cast<const T*>(a.v) + (size_t)kvh * D;

    // q's fragments (t, nt): a wave has some whole, lane (i, g) eight values of pair i's row
    constexpr int kUnits = (C::kTD * NT + WAVES - 1) / WAVES;
    float qv[kUnits][8];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const int u = wave + WAVES * k, t = u / NT, nt = u % NT;
        int m;
        const float* q = a.q + (size_t)pair_row(a, kvh, rg * C::kRows + 16 * nt + i16, m) * D;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int d = C::kcol(t, g, 4 * h);
            const f32x4 y = u < C::kTD * NT && (FULL || d < D) ? ld_global(reinterpret_cast<const f32x4*>(q + d)) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; e++) qv[k][4 * h + e] = y[e];
        }
    }
    // K of the wave's first block is on its way while q's parts are made
    typedef typename std::conditional<C::kHalf, u32x4, f32x4>::type KRaw;
    KRaw kraw[C::kNK][C::kTD * (C::kHalf ? 1 : 2)];
    // from an address that the whole wave shares and a lane's own offset
    const uint32_t row_bytes = (uint32_t)(row_len * sizeof(T));
    const uint32_t k_lane = C::kAhead ? lane / C::kRowUnits * row_bytes + 16 * (lane % C::kRowUnits)
                                      : (uint32_t)i16 * row_bytes + (C::kHalf ? 8 : 4) * g * (uint32_t)sizeof(T);
    const uint32_t v_lane = 4u * g * row_bytes + C::kCols * i16 * (uint32_t)sizeof(T);
    auto load_k = [&](const TreeBlock& blk, int from, int to) {
        const char* base = reinterpret_cast<const char*>(kb + (size_t)blk.at * row_len);
#pragma unroll
        for (int kt = from; kt < to; kt++) {
            const char* p = base + (size_t)(16 * kt) * row_bytes;
            if constexpr (C::kAhead) {
#pragma unroll
                for (int r = 0; r < C::kLoads; r++)
                    kraw[kt][r] = FULL || 16 / (int)sizeof(T) * (lane % C::kRowUnits) < D ? ld_global(reinterpret_cast<const KRaw*>(p + (size_t)(C::kLoadRows * r) * row_bytes + k_lane))
                                                                                          : KRaw{};
                continue;
            }
#pragma unroll
            for (int t = 0; t < C::kTD; t++)
                if constexpr (C::kHalf) {
                    kraw[kt][t] = FULL || 32 * t + 8 * g < D ? ld_global(reinterpret_cast<const u32x4*>(p + 64 * t + k_lane)) : u32x4{0, 0, 0, 0};
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        kraw[kt][2 * t + h] = FULL || 32 * t + 16 * h + 4 * g < D ? ld_global(reinterpret_cast<const f32x4*>(p + 128 * t + 64 * h + k_lane))
                                                                                 : f32x4{0.f, 0.f, 0.f, 0.f};
                }
        }
    };
    // A fragment is 16 keys' rows, 64 bytes of each: K is loaded as whole rows, which the L1 serves faster, and turned in a part of
    // LDS that is the wave's own (5 rows after 300 keys 8.1 -> 7.4 us, 24 after 4000 25.2 -> 23.6, fp16 17.3 -> 15.1, 16 after 200
    // 7.0 -> 5.9; 256 after 8000 in fp32, where LDS is busy with q's parts, 207 either way).
    char* const turn = lds + C::kQBytes + wave * C::kTurnBytes;
    auto turn_k = [&](int kt) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < C::kLoads; r++)
            *reinterpret_cast<KRaw*>(turn + (lane / C::kRowUnits + C::kLoadRows * r) * C::kTurnStride + 16 * (lane % C::kRowUnits)) = kraw[kt][r];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    auto turned = [&](int r) { return *reinterpret_cast<const KRaw*>(turn + i16 * C::kTurnStride + 16 * g + 64 * r); };
    auto drop_k = [&](int from, int to) {                   // no value: the last block's is not carried along
#pragma unroll
        for (int kt = from; kt < to; kt++)
#pragma unroll
            for (auto& x : kraw[kt]) x = __builtin_nondeterministic_value(x);
    };
    int b = b0 + wave;
    TreeBlock blk = tree_block(a, min(b, blocks - 1), past_blocks);
    if (C::kAhead && b < b1) load_k(blk, 0, C::kNK);

    // q's parts as fragments in LDS: (t, nt, part), lane (i, g)
    Frag* qf = reinterpret_cast<Frag*>(lds);
    if (C::kHalf) {
#pragma unroll
        for (int k = 0; k < kUnits; k++) {
            const int u = wave + WAVES * k;
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(qv[k][e]));
            mx = pair_max<32>(pair_max<16>(mx));
            if (g == 0 && u < C::kTD * NT) qmax[u / NT][16 * (u % NT) + i16] = mx;
        }
        __syncthreads();
    }
    // a row's power of two: its largest value to [2^14, 2^15)
    auto q_scale = [&](int row) {
        float mx = 0.f;
#pragma unroll
        for (int t = 0; t < C::kTD; t++) mx = fmaxf(mx, qmax[t][row]);
        return mx > 0.f && mx <= kMaxFinite ? ldexpf(1.f, min(100, 14 - ilogbf(mx))) : 1.f;
    };
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const int u = wave + WAVES * k;
        if (u >= C::kTD * NT) break;
        Frag* dst = qf + (size_t)u * C::kParts * 64 + lane;
        if constexpr (C::kHalf) {
            const float s = q_scale(16 * (u % NT) + i16);
            f16x8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = qv[k][e] * s;
                hi[e] = (_Float16)y;
                lo[e] = (_Float16)((y - (float)hi[e]) * 2048.f);
            }
            dst[0] = hi;
            dst[64] = lo;
        } else {
            bf16x8 p[3];
            split_bf16(qv[k], p);
            dst[0] = p[0];
            dst[64] = p[1];
            dst[128] = p[2];
        }
    }
    int qm[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) pair_row(a, kvh, rg * C::kRows + 16 * nt + i16, qm[nt]);
    __syncthreads();

    f16x8 qr[NT][C::kTD][2];                                // fp16 caches leave the registers for q
    if constexpr (C::kHalf && C::kAhead)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int t = 0; t < C::kTD; t++)
#pragma unroll
                for (int i = 0; i < 2; i++) qr[nt][t][i] = qf[(size_t)((t * NT + nt) * 2 + i) * 64 + lane];
    f32x4 acc[C::kDT][NT];
    float mr[NT], l[NT], f[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        mr[nt] = -INFINITY;
        l[nt] = 0.f;
        f[nt] = C::kHalf ? fmaxf(a.scale / q_scale(16 * nt + i16), 1.17549435e-38f) : a.scale;
#pragma unroll
        for (int d = 0; d < C::kDT; d++) acc[d][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int first = b;
    for (; b < b1; b += WAVES) {
        typename C::VRaw vraw[8][C::kNC];                   // [element of the fragment][columns]
        auto load_v = [&](const TreeBlock& blk, int c0, int c1) {
            const char* base = reinterpret_cast<const char*>(vb + (size_t)blk.at * row_len);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const char* p = base + (size_t)(16 * (e >> 2) + (e & 3)) * row_bytes;      // 4 g keys more in group g
#pragma unroll
                for (int c = c0; c < c1; c++) {
                    if (FULL || C::kChunk * c + C::kCols * i16 < D)
                        vraw[e][c] = ld_global(reinterpret_cast<const typename C::VRaw*>(p + C::kChunk * c * sizeof(T) + v_lane));
                    else vraw[e][c] = typename C::VRaw{};
                }
            }
        };
        const bool more = b + WAVES < b1;
        const TreeBlock next = tree_block(a, more ? b + WAVES : b, past_blocks);
        const bool all_seen = blk.j0 < 0 && blk.n == kKeys;
        uint32_t seen[NT];                                  // bit 16 kt + r: key 16 kt + 4 g + r; asked for before it is needed
        if (!all_seen)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) seen[nt] = (uint32_t)(seen_bits(a, blk, qm[nt]) << (blk.base - blk.at)) >> (4 * g);
        f32x4 s[C::kNK][NT];
#pragma unroll
        for (int kt = 0; kt < C::kNK; kt++) {
            if (!C::kAhead) load_k(blk, kt, kt + 1);
            if (C::kAhead && kt == 1) {
                __builtin_amdgcn_sched_barrier(0);          // not before the first keys' registers are free
                load_v(blk, 0, 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (C::kAhead) turn_k(kt);
            if constexpr (C::kHalf) {
                f16x8 keys[C::kTD];
#pragma unroll
                for (int t = 0; t < C::kTD; t++) keys[t] = __builtin_bit_cast(f16x8, C::kAhead ? turned(t) : kraw[kt][t]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < C::kTD; t++) {
                        if constexpr (!C::kAhead) {
#pragma unroll
                            for (int i = 0; i < 2; i++) qr[nt][t][i] = qf[(size_t)((t * NT + nt) * 2 + i) * 64 + lane];
                        }
                        lo = mfma(keys[t], qr[nt][t][1], lo);
                        hi = mfma(keys[t], qr[nt][t][0], hi);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) s[kt][nt][r] = fmaf(lo[r], 1.f / 2048.f, hi[r]);
                }
            } else {
                // the small products first: the sum takes its full size only in the last ones, and half of those apart
                bf16x8 kh[C::kTD], qh[C::kTD][NT];
                f32x4 lo[NT], hi[NT];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) lo[nt] = hi[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
                f32x4 y[2];                                 // the next step's, on their way from LDS
                auto key = [&](int r) { return C::kAhead ? turned(r) : kraw[kt][r]; };
                y[0] = key(0), y[1] = key(1);
#pragma unroll
                for (int t = 0; t < C::kTD; t++) {
                    const float x[8] = {y[0].x, y[0].y, y[0].z, y[0].w, y[1].x, y[1].y, y[1].z, y[1].w};
                    if (t + 1 < C::kTD) y[0] = key(2 * t + 2), y[1] = key(2 * t + 3);
                    bf16x8 qp[NT][3];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int i = 0; i < 3; i++) qp[nt][i] = qf[(size_t)((t * NT + nt) * 3 + i) * 64 + lane];
                    __builtin_amdgcn_sched_barrier(0);      // asked for before the parts are made (256 rows after 8000: 207 -> 203 us)
                    bf16x8 kp[3];
                    split_bf16(x, kp);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) lo[nt] = small_products(kp, qp[nt], lo[nt]);
                    kh[t] = kp[0];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) qh[t][nt] = qp[nt][0];
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int t = 0; t < C::kTD; t++) {
                        const bf16x8 q = qh[t][nt];
                        if (t < C::kTD / 2) lo[nt] = mfma(kh[t], q, lo[nt]);
                        else hi[nt] = mfma(kh[t], q, hi[nt]);
                    }
                    s[kt][nt] = lo[nt] + hi[nt];
                }
            }
        }
        if (C::kAhead && C::kNC > 1) {
            __builtin_amdgcn_sched_barrier(0);
            load_v(blk, 1, C::kNC);
            __builtin_amdgcn_sched_barrier(0);
        }
        const TreeBlock now = blk;
        blk = next;
        if (!all_seen)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int kt = 0; kt < C::kNK; kt++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (!(seen[nt] >> (16 * kt + r) & 1)) s[kt][nt][r] = -INFINITY;
        // The exponentials are taken from a reference, a maximum of earlier blocks, and the sums rescaled only where a score has
        // risen far above it: a maximum over 32 pairs rises a little in almost every block (256 rows after 8000 keys: fp32 212
        // -> 207 us, fp16 92.2 -> 90.8).
        float bm[NT];
        bool up = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            bm[nt] = s[0][nt][0];
#pragma unroll
            for (int kt = 0; kt < C::kNK; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) bm[nt] = fmaxf(bm[nt], s[kt][nt][r]);
            bm[nt] = pair_max<32>(pair_max<16>(bm[nt])) * f[nt];
            up = up || bm[nt] > mr[nt] + kRaise;
        }
        if (__any(up))
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float mn = fmaxf(mr[nt], bm[nt]), al = ex2(mr[nt] - (mn == -INFINITY ? 0.f : mn));
                mr[nt] = mn;
                l[nt] *= al;
#pragma unroll
                for (int d = 0; d < C::kDT; d++) acc[d][nt] *= al;
            }
        Frag pf[NT][C::kParts];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const float ref = mr[nt] == -INFINITY ? 0.f : mr[nt];
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[e] = ex2(fmaf(s[e >> 2][nt][e & 3], f[nt], -ref));
                l[nt] += p[e];
            }
            if constexpr (C::kHalf) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float y = p[e] * kPScale;
                    pf[nt][0][e] = (_Float16)y;
                    pf[nt][1][e] = (_Float16)(y - (float)pf[nt][0][e]);
                }
            } else {
                split_bf16(p, pf[nt]);
            }
        }
        // a block's sums start from zero and are added to the others by the VALU: the matrix unit carries no long sum
#pragma unroll
        for (int c = 0; c < C::kNC; c++) {
            if (!C::kAhead) load_v(now, c, c + 1);
            if (C::kAhead && c < 2) {                       // the next K: in halves, the second in the first columns' registers
                constexpr bool whole = C::kNC == 1;
                __builtin_amdgcn_sched_barrier(0);
                if (c == 0 && more) load_k(blk, 0, whole ? 2 : 1);
                else if (c == 0) drop_k(0, whole ? 2 : 1);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j = 0; j < C::kCols; j++) {
                f32x4 o[NT];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) o[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (C::kHalf) {
                    u32x4 w;
#pragma unroll
                    for (int e = 0; e < 4; e++)             // column j of keys 2 e and 2 e + 1
                        w[e] = __builtin_amdgcn_perm(vraw[2 * e + 1][c][j / 2], vraw[2 * e][c][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
                    const f16x8 v = __builtin_bit_cast(f16x8, w);
#pragma unroll
                    for (int part = 1; part >= 0; part--)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) o[nt] = mfma(v, pf[nt][part], o[nt]);
                } else {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = vraw[e][c][j];
                    bf16x8 vp[3];
                    split_bf16(x, vp);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) o[nt] = mfma(vp[0], pf[nt][0], small_products(vp, pf[nt], o[nt]));
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) acc[c * C::kCols + j][nt] += o[nt];
                if (!C::kHalf) __builtin_amdgcn_sched_barrier(0);   // parts of more tiles at once would spill
            }
        }
        if (C::kAhead && C::kNC > 1) {
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_k(blk, 1, 2);
            else drop_k(1, 2);
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
    if (redo) tree_again<T, DP, NT, FULL, C::kCols>(a, kvh, rg * C::kRows, first, b1, WAVES, past_blocks, mr, l, acc);

    // the waves' states
    const float unit = C::kHalf && !redo ? 1.f / kPScale : 1.f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        l[nt] = pair_sum<32>(pair_sum<16>(l[nt]));
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
        float mx = stat[0][0][r];
#pragma unroll
        for (int k = 1; k < WAVES; k++) mx = fmaxf(mx, stat[0][k][r]);
        w[nt] = mr[nt] == -INFINITY ? (l[nt] != l[nt] ? 1.f : 0.f) : ex2(mr[nt] - mx) * unit;   // NaN: no score is a number
    }
    if (tid < C::kRows) {                                   // what a row's sums are divided by, or its state, and its place
        const int r = rg * C::kRows + tid;
        float mx = stat[0][0][tid];
#pragma unroll
        for (int k = 1; k < WAVES; k++) mx = fmaxf(mx, stat[0][k][tid]);
        float total = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; k++) {
            const float lk = stat[1][k][tid], mk = stat[0][k][tid];
            total += mk == -INFINITY ? (lk != lk ? lk : 0.f) : lk * ex2(mk - mx);
        }
        int m;
        const int at = pair_row(a, kvh, r, m);
        row_at[tid] = r < R ? at : -1;
        row_inv[tid] = a.nsplit > 1 ? 1.f : total == 0.f ? 0.f : 1.f / total;
        if (a.nsplit > 1 && r < R) {
            f32x2* st = reinterpret_cast<f32x2*>(a.ws + (size_t)a.M * a.H * a.nsplit * D) + (size_t)at * a.nsplit + split;
            st_global(st, f32x2{mx, total});
        }
    }
    float* const out = a.nsplit > 1 ? a.ws + (size_t)split * D : a.out;
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
#pragma unroll
        for (int u = tid; u < C::kRows * (C::kChunk / 4); u += 64 * WAVES) {
            const int row = u / (C::kChunk / 4), c4 = u % (C::kChunk / 4), d = C::kChunk * c + 4 * c4, at = row_at[row];
            if (at < 0 || (!FULL && d >= D)) continue;
            f32x4 sum = *reinterpret_cast<const f32x4*>(merge + (size_t)row * C::kMergeStride + 4 * c4);
#pragma unroll
            for (int k = 1; k < WAVES; k++) sum += *reinterpret_cast<const f32x4*>(merge + (size_t)(k * C::kRows + row) * C::kMergeStride + 4 * c4);
            const float inv = row_inv[row];
            st_global(reinterpret_cast<f32x4*>(out + (size_t)at * a.nsplit * D + d), f32x4{sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv});
        }
    }
}

// Fewer keys than a block: one wave per (row, head), a lane's own key for the scores, its own values of D for the sums
template <typename T>
__global__ __launch_bounds__(64) void attn_tree_row_kernel(const TreeArgs a)
{
    __shared__ float q[256];
    const int h = blockIdx.x, m = blockIdx.y, lane = threadIdx.x, D = a.D, T0 = a.past + a.M, j = lane - a.past;
    const size_t row = (size_t)m * a.H + h, row_len = (size_t)a.KV * D;
    const T* k = static_cast<const T*>(a.k) + (size_t)(h / a.G) * D;
    const T* v = static_cast<const T*>(a.v) + (size_t)(h / a.G) * D;
    for (int d = lane; d < D; d += 64) q[d] = ld_global(a.q + row * D + d);
    __syncthreads();
    bool seen = lane < T0;
    if (seen && j >= 0) seen = a.mask ? ld_global(a.mask + (size_t)m * a.words) >> j & 1 : j <= m;
    float sc = -INFINITY;
    if (seen) {
        sc = 0.f;
#pragma unroll 8
        for (int d = 0; d < D; d++) sc = fmaf(q[d], (float)k[(size_t)lane * row_len + d], sc);
        sc *= a.scale;
    }
    float mx = sc;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    const float p = seen ? ex2(sc - (mx == -INFINITY ? 0.f : mx)) : 0.f;
    float l = p, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    const uint64_t all = __ballot(seen);
    for (int s = 0; s < T0; s++) {
        if (!(all >> s & 1)) continue;
        const float w = __shfl(p, s);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < D) acc[i] = fmaf(w, (float)v[(size_t)s * row_len + lane + 64 * i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < D) st_global(a.out + row * D + lane + 64 * i, l == 0.f ? 0.f : acc[i] / l);
}

// out = sum_i acc_i 2^(m_i - m) / sum_i l_i 2^(m_i - m) over the key ranges. A workgroup has `rows` rows and a power of two `parts` of threads a
// column of each: the ranges' weights go to LDS, a wave a row, then thread (row, part p, four columns c) adds ranges p, p + parts, ... in
// order, and the parts are added in order.
constexpr int kMergeFirst = 4;                              // ranges a thread has asked for before the weights are there
__global__ __launch_bounds__(256) void attn_tree_merge_kernel(const TreeArgs a, int rows, int log_parts)
{
    __shared__ float wgt[512];                              // rows * nsplit: 4 * (256 / (D / 4)), or one row's
    __shared__ f32x4 part[256];
    const int t = threadIdx.x, lane = t & 63, S = a.nsplit, D = a.D, R = a.M * a.H, row0 = blockIdx.x * rows;
    const int nc = D / 4, slot = t / nc, c = t - slot * nc, parts = 1 << log_parts, r = slot >> log_parts, p = slot - (r << log_parts);
    const size_t row = (size_t)row0 + r;
    const bool here = r < rows && row < (size_t)R;
    const f32x4* src = reinterpret_cast<const f32x4*>(a.ws + row * S * D) + c;
    f32x4 v[kMergeFirst];
#pragma unroll
    for (int k = 0; k < kMergeFirst; k++) v[k] = here && p + k * parts < S ? ld_global(src + (size_t)(p + k * parts) * nc) : f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = t >> 6; i < rows && row0 + i < R; i += 4) {
        const f32x2* st = reinterpret_cast<const f32x2*>(a.ws + (size_t)R * S * D) + (size_t)(row0 + i) * S;
        f32x2 s[2];
#pragma unroll
        for (int k = 0; k < 2; k++) s[k] = lane + 64 * k < S ? ld_global(st + lane + 64 * k) : f32x2{-INFINITY, 0.f};
        const float mx = wave_max(fmaxf(s[0].x, s[1].x), lane);
        float e[2], l = 0.f;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const float mi = s[k].x, li = s[k].y;
            e[k] = mi == -INFINITY ? (li != li ? li : 0.f) : ex2(mi - mx);
            l += li * e[k];
        }
        l = wave_sum(l, lane);
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (lane + 64 * k < S) wgt[i * S + lane + 64 * k] = l == 0.f ? 0.f : e[k] / l;
    }
    __syncthreads();
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (here) {
        const float* w = wgt + r * S;
#pragma unroll
        for (int k = 0; k < kMergeFirst; k++) {
            const float wk = p + k * parts < S ? w[p + k * parts] : 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(wk, v[k][e], o[e]);
        }
#pragma unroll 4
        for (int i = p + kMergeFirst * parts; i < S; i += parts) {
            const f32x4 x = ld_global(src + (size_t)i * nc);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = fmaf(w[i], x[e], o[e]);
        }
    }
    if (parts > 1) {
        part[t] = o;
        __syncthreads();
    }
    if (here && p == 0) {
        for (int k = 1; k < parts; k++) o += part[t + k * nc];
        st_global(reinterpret_cast<f32x4*>(a.out + row * D) + c, o);
    }
}

typedef void (*TreeFn)(TreeArgs);

template <typename T>
TreeFn tree_fn(int D, int nt, int waves)
{
    if (D == 64) return waves == 8 ? attn_tree_kernel<T, 64, 1, true, 8> : nt == 2 ? attn_tree_kernel<T, 64, 2, true, 4> : attn_tree_kernel<T, 64, 1, true, 4>;
    if (D == 128) return waves == 8 ? attn_tree_kernel<T, 128, 1, true, 8> : nt == 2 ? attn_tree_kernel<T, 128, 2, true, 4> : attn_tree_kernel<T, 128, 1, true, 4>;
    if (D == 256) return waves == 8 ? attn_tree_kernel<T, 256, 1, true, 8> : attn_tree_kernel<T, 256, 1, true, 4>;
    if (D < 64) return waves == 8 ? attn_tree_kernel<T, 64, 1, false, 8> : attn_tree_kernel<T, 64, 1, false, 4>;
    if (D < 128) return waves == 8 ? attn_tree_kernel<T, 128, 1, false, 8> : attn_tree_kernel<T, 128, 1, false, 4>;
    return waves == 8 ? attn_tree_kernel<T, 256, 1, false, 8> : attn_tree_kernel<T, 256, 1, false, 4>;
}

}  // namespace

uint64_t plan_attention_tree(TreeArgs* a, size_t ws_bytes)
{
    const int R = a->M * a->G;
    a->nsplit = 1;
    if (a->past + a->M < kKeys) return 0;
    // 32 pairs a workgroup where those fill the chip three times (fp16: eight) with ranges of a block a wave: a block is then split
    // into parts half as often, but a wave's own chain is longer. Also where 16 would be more than two workgroups a CU (fp16: and 32
    // fill it four times). 16 against 32, in us (28 / 4 heads of 128): 16 rows after 4000 keys 18.9, 19.5, 24 after 4000 26.1, 23.6,
    // fp16 24 after 8000 19.8, 21.1, 64 after 8000 32.8, 31.1, 256 after none 15.5, 21.2; 14 / 2 heads of 64: 256 after 200 22.8,
    // 15.1, fp16 256 after 200 11.5, 13.7, after 2000 35.9, 19.6. About the border in fp32, by `full`: 576 21.7, 22.4 (24 after 3000), 640
    // 22.2, 22.7 (20 after 4000), 672 22.3, 23.4 (32 after 3000), 744 26.0, 23.2 (24 after 3900), 748 22.4, 23.9 (48 after 2000), 756 25.9, 22.4
    // (12 after 8000), 868 26.6, 24.5 (32 after 3900), 960 26.7, 24.1 (20 after 6000), 1056 27.6, 29.5 (48 after 3000), 1364 34.8, 34.9 (48 after
    // 4000): `full` is a measure of the work, and what decides between 700 and 1100 is how evenly the ranges lie on the CUs.
    const long full = (long)((R + 31) / 32) * a->KV * ((a->past + a->M + 4 * kKeys - 1) / (4 * kKeys));
    const int per_xcd = (R + 15) / 16 * ((a->KV + 7) / 8);              // workgroups of 16 pairs, in a range
    const bool crowded = per_xcd > 64, wide = a->half ? full >= (crowded ? 1024 : 2048) : full >= 768 || crowded;
    a->nt = (a->D == 64 || a->D == 128) && wide ? 2 : 1;
    a->past_blocks = (a->past + kKeys - 1) / kKeys;
    const int blocks = a->blocks = a->past_blocks + (a->M + kKeys - 1) / kKeys;
    // Short contexts: one range of 8 waves and no merge launch, while an XCD, which then has whole kv heads only, has a workgroup
    // a CU (fp16: two) and a wave has one block (keys of 512 bytes), two or (128 bytes) four, and more where the merge would have
    // many rows. Eight waves against four with ranges, in us: 14 / 2 heads of 64: 5 rows after 300 keys (fp32) 7.4, 8.5, 5 after 800
    // (fp16) 7.2, 8.4; 28 / 4 heads of 128: 8 after 200 (fp32) 8.9, 10.8, 64 after 200 11.7, 13.6, 64 after 450 (fp16) 8.5, 12.3, 128
    // after 100 (fp16) 11.2, 13.3; beyond these limits 8 after 300 (fp32) 11.3, 10.4, 8 after 700 (fp16) 8.9, 8.4, 128 after 100
    // (fp32) 17.6, 16.3.
    const int key_bytes = (a->D <= 64 ? 64 : a->D <= 128 ? 128 : 256) * (a->half ? 2 : 4);
    a->waves = 4;
    if (blocks > 4 && per_xcd <= (a->half ? 64 : 32) && blocks <= std::max(8, 4096 / key_bytes) + per_xcd / 8) a->waves = 8, a->nt = 1;
    a->groups = (R + 16 * a->nt - 1) / (16 * a->nt);
    const size_t one = (size_t)a->M * a->H * (a->D + 2) * sizeof(float);
    const int fit = (int)std::min<size_t>(kTreeMaxSplit, ws_bytes / one);
    // key ranges that keep every XCD's 32 CUs within `each` workgroups: a (kv head, range)'s groups are on one of them
    auto ranges = [&](int each) { return 8 * (32 * each / a->groups) / a->KV; };
    // up to two workgroups a CU, at least a block a wave, as many as the workspace holds
    const int s = a->waves == 8 ? 1 : std::max(1, std::min({ranges(2), (blocks + 3) / 4, fit}));
    a->per = ((blocks + s - 1) / s + a->waves - 1) / a->waves * a->waves;            // as many for each of the waves
    a->nsplit = (blocks + a->per - 1) / a->per;
    a->inv_nsplit = 1.f / a->nsplit;
    a->inv_g = 1.f / a->G;
    return a->nsplit == 1 ? 0 : a->nsplit * one;
}

hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t stream)
{
    if (a.past + a.M < kKeys) {
        if (a.half) hipLaunchKernelGGL(attn_tree_row_kernel<_Float16>, dim3(a.H, a.M), dim3(64), 0, stream, a);
        else hipLaunchKernelGGL(attn_tree_row_kernel<float>, dim3(a.H, a.M), dim3(64), 0, stream, a);
        return hipGetLastError();
    }
    const TreeFn fn = a.half ? tree_fn<_Float16>(a.D, a.nt, a.waves) : tree_fn<float>(a.D, a.nt, a.waves);
    hipLaunchKernelGGL(fn, dim3(8 * a.groups, (a.KV * a.nsplit + 7) / 8), dim3(64 * a.waves), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1) return e;
    // a thread's columns of four ranges, more where a row has more than the workgroup's; rows as fit (a row a workgroup: 256 rows
    // after 8000 keys, two ranges, 9.2 us of 90)
    const int slots = 256 / (a.D / 4);
    int log_parts = 0;
    while (kMergeFirst << log_parts < a.nsplit && 2 << log_parts <= slots) log_parts++;
    const int rows = slots >> log_parts;
    hipLaunchKernelGGL(attn_tree_merge_kernel, dim3((a.M * a.H + rows - 1) / rows), dim3(256), 0, stream, a, rows, log_parts);
    return hipGetLastError();
}

}  // namespace ql
