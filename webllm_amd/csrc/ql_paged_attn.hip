// Attention of a batch's rows over their sequences' pages (ql_paged_attention):
//   out[m, h] = sum_t p_t V[t] / sum_t p_t,  p_t = exp(q[m, h] . K[t] / sqrt(D) - max)   over the tokens t up to the row's own.
//
// Sequences of up to 64 (row, head) pairs a kv head (`few`), paged_decode: a workgroup has 16 pairs and a range of blocks (32 tokens of an fp16 cache, 64 of an e4m3
// one: the tokens of V that lie together); its four waves take the blocks in turn, K and V from memory to one wave's registers. The cache lies as the matrix
// instructions take it: a load is 16 bytes a lane and 1 KB in a row. Scores are computed transposed, S^T = K Q^T (lane = pair, registers = tokens), and what a lane
// then has of P is the B fragment of O^T = V^T P^T, with nothing crossing lanes: tile kt of S is the block's tokens 16 kt + 4 g + r (g: lane / 16, r: register), and
// the tokens of V that a lane reads together are 16 b + 4 g + r. Softmax in fp32 with a running reference, raised by leaps only; the waves' states meet in LDS.
// Sequences differ in length, so the blocks of all of them, one behind the other, are dealt to the workgroups in equal ranges (two workgroups a CU); a workgroup goes
// through the sequences that its range meets, and paged_merge joins the parts of those that are cut. Every workgroup finds its range from the tables by itself:
// lengths stay on the device. Up to max_len 1024 each tile of 16 pairs is one workgroup's, and there is no second launch.
// Bound by memory: 64 requests of up to 8000 tokens, e4m3, 28 / 4 heads of 128, 299 MB, 69 us, 4.3 TB/s (61 to 63 in the first launch's trace, 6 the merge's);
// one of 60000 tokens, fp16, 123 MB, 33 us, 26 of them the first launch (4.7 TB/s) and 7 the merge. 1.02 of the bytes cross the memory's bus. Four requests of 300
// tokens, 14 / 2 heads of 64: 5.5 us, a launch and its chain of loads. Blocks of 64 tokens of fp16 take 41 us for the one request's 33 (registers go to memory).
//
// Sequences of more rows, paged_prompt: 64 or 128 pairs of a kv head a workgroup, 16 or 32 a wave, which read the tokens, 64 at a time, from LDS; the next 64
// come there from memory meanwhile, past the registers. Tiles are dealt the longest first, and in parts of their tokens where they are few; paged_join joins those.
// 9000 tokens of five prompts, fp16, 28 / 4 heads of 128: 166 to 174 us, 139 GFLOP, 800 to 840 TFLOP/s, where an 8192^3 product of the library reaches 1185. The matrix unit is busy
// 37 % of the cycles (at 1.9 GHz), the VALU (an exponential, a product and a conversion for each score) 40 %: two waves a SIMD overlap them in part. Slower or no faster:
// 64 pairs a wave (its sums in the accumulators' registers are moved for every product), 32 tokens a step, scores one step ahead of the products, an order of
// instructions given to the compiler. 24 requests of up to 4000 tokens beside 700 rows of two prompts of up to 4200, e4m3: 78 us, 28 GFLOP; 71 the first
// launch, whose prompts' workgroups begin as the decoding ones end (512, all that the device holds at D = 128) and have 10 to 20 blocks each, where 13.4 would be equal
// (every tile has as many parts as another); each wave makes e4m3 fp16 for itself.
//
// Numbers: K and V enter as they are (e4m3 is exact in fp16); K's scales multiply scores, V's its values as they become fp16, in units of a running power of two, which is
// exact where scales lie up to 2^15 apart in a block, often 2^21 (v_reference). A probability keeps its own range that way: it would leave fp16's under the scale of a group far
// below another one, also in rows that do not see the other. fp32 rows: q as hi + 2^-11 lo under its row's exponent, in two sums; P as hi + lo of 2^8 P: about 22 bits, down
// to 2^-33 of the row's largest. fp16 rows: q as it is, 2^8 P rounded once, which costs a result up to half a step of its own type (2.5e-4 relative over the prompts,
// 2.1e-4 for fp32 arithmetic rounded once). A product of an infinity's parts is a NaN, and 0 * V is one where V is not finite: a wave whose sums end that way, or
// whose scales lie further apart than its units reach, does its blocks again on the VALU from q, K and V themselves, skipping what a pair does not see (paged_again).
#include <algorithm>
#include <type_traits>

#include "ql_lanes.h"
#include "ql_paged.h"

namespace ql {

namespace {

constexpr int kBlock = 64;               // tokens of a block of a prompt's kernel; pages are whole blocks
constexpr int kPairs = 16;
constexpr int kDecodeWaves = 4;
constexpr int kPromptParts = 512;         // workgroups up to which the tiles of many rows are done in parts of their tokens
constexpr int kPromptMost = 32;           // parts of a tile at most
constexpr float kRaise = 7.f;            // log2 that scores may rise above the running reference before it is raised
constexpr float kPLog = 8.f, kPScale = 256.f;   // parts of P: 2^8 P, at most 2^15
constexpr float kMaxFinite = 3.4028235e38f;

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// The larger of two, NaN if one is: one instruction (fmaxf first makes numbers of what may be signalling). A NaN score leaves the reference as it is and
// makes its row's sums NaN by its own weight.
__device__ __forceinline__ float maxi(float a, float b) { return __builtin_elementwise_maximum(a, b); }
template <int O>
__device__ __forceinline__ float pair_maxi(float v)
{
    const u32pair p = lane_pair<O>(__builtin_bit_cast(uint32_t, v));
    const uint32_t x = p.x, y = p.y;
    return maxi(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}

template <bool F8>
__device__ __forceinline__ float value_at(const void* p, size_t i)
{
    if (F8) return __builtin_amdgcn_cvt_f32_fp8(ld_global(static_cast<const uint8_t*>(p) + i), 0);
    return (float)ld_global(static_cast<const _Float16*>(p) + i);
}

// eight e4m3 values, exactly, four and four times a power of two 2^-15 .. 2^7 or zero
__device__ __forceinline__ f16x8 f8_to_f16(uint32_t lo, uint32_t hi, float s = 1.f, float t = 1.f)
{
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, s, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, t, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, t, true);
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// What a workgroup goes through: pairs r0 .. r0 + 15 of sequence s, blocks b0 .. b1 - 1 of nb
struct Piece {
    int s, r0, b0, b1, nb;
    PagedSeq q;
};

__device__ __forceinline__ bool few(const PagedAttnArgs& a, const PagedSeq& q) { return q.n * a.G <= a.few; }
__device__ __forceinline__ int tiles_of(const PagedAttnArgs& a, const PagedSeq& q) { return (q.n * a.G + kPairs - 1) / kPairs; }
template <int BLOCK>
__device__ __forceinline__ int blocks_of(const PagedSeq& q) { return (q.len + BLOCK - 1) / BLOCK; }
// the blocks of a range of the `ranges` that `total` are dealt in, a multiple of the workgroup's waves
template <int WAVES>
__device__ __forceinline__ long long per_range(const PagedAttnArgs& a, long long total) { return ((total + a.ranges - 1) / a.ranges + WAVES - 1) / WAVES * WAVES; }

// A wave's blocks on the VALU, into the sums' own layout: lane (i, g) has pair i, columns 16 ct + 4 g + r. The four lanes of a pair share a dot product.
template <bool F8, typename Q, int CT, int BLOCK>
__device__ __forceinline__ void paged_again(const PagedAttnArgs& a, const Piece& p, int kvh, size_t q_row, int last, int first, int step, float& mr, float& l, f32x4 (&acc)[CT])
{
    typedef PagedLayout<F8 ? 1 : 2> Lay;
    const int g = threadIdx.x >> 4 & 3, D = a.D;
    const Q* q = static_cast<const Q*>(a.q) + q_row;
    mr = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int c = 0; c < CT; c++) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int b = first; b < p.b1; b += step) {
        const int t0 = b * BLOCK, page = paged_page(a.b, p.s, t0), in_page = t0 & ((1 << a.b.log_page) - 1);
        if (page < 0) continue;
        const size_t head = (size_t)page * a.KV + kvh, base = (head << a.b.log_page) * D, sc0 = (head << (a.b.log_page - 4)) + (in_page >> 4);
#pragma unroll 1
        for (int i = 0; i < BLOCK && t0 + i < p.q.len; i++) {
            const bool seen = t0 + i <= last;
            float sc = 0.f;
#pragma unroll 1
            for (int d = g * (D / 4); d < (g + 1) * (D / 4); d++) sc = fmaf((float)q[d], value_at<F8>(a.k, base + Lay::k_at(D, in_page + i, d / Lay::kUnit) + d % Lay::kUnit), sc);
            sc = pair_sum<32>(pair_sum<16>(sc)) * (a.scale * (F8 ? ld_global(a.k_scale + sc0 + i / 16) : 1.f));
            if (!seen) sc = -INFINITY;
            const float mn = fmaxf(mr, sc), ref = mn == -INFINITY ? 0.f : mn, al = ex2(mr - ref), e = seen ? ex2(sc - ref) : 0.f;
            mr = mn;
            l = l * al + (g == 0 ? e : 0.f);
            const float ev = e * (F8 ? ld_global(a.v_scale + sc0 + i / 16) : 1.f);
#pragma unroll
            for (int c = 0; c < CT; c++) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    acc[c][r] *= al;
                    if (seen && 16 * c < D) acc[c][r] = fmaf(ev, value_at<F8>(a.v, base + Lay::v_at(D, in_page + i / 4 * 4, 16 * c + 4 * g + r) + i % 4), acc[c][r]);
                }
            }
        }
    }
}

template <bool F8, typename Q, int DP>
struct DecodeTile {
    static constexpr bool kHalf = std::is_same<Q, _Float16>::value;
    static constexpr int kParts = kHalf ? 1 : 2;                 // of q and of P
    static constexpr int kUnits = DP / (F8 ? 64 : 32);           // 16-byte loads of a token's K, of 16 tokens
    static constexpr int kSteps = DP / 32;                       // matrix instructions along D
    static constexpr int kCT = DP / 16;                          // tiles of 16 columns
    static constexpr int kVB = F8 ? 1 : 2;                       // parts of a block whose tokens of V lie together
    static constexpr int kMerge = DP + 4;                        // floats of a row of the merge buffer
    static constexpr int kMergeBytes = kDecodeWaves * kPairs * (kMerge + 2) * 4 + kPairs * 8;
    // the column of element e of step t of a K or Q fragment, lane group g
    static __device__ __forceinline__ int col(int t, int g) { return F8 ? 64 * (t >> 1) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g; }
};

// q's fragments of the lane's pair; returns what scores are multiplied by
template <typename C, typename Q>
__device__ __forceinline__ float load_q(const Q* q, int g, int D, float scale, f16x8 (&qf)[C::kSteps][C::kParts])
{
    if constexpr (C::kHalf) {
#pragma unroll
        for (int t = 0; t < C::kSteps; t++) {
            const int d = C::col(t, g);
            qf[t][0] = d < D ? __builtin_bit_cast(f16x8, ld_global(reinterpret_cast<const u32x4*>(q + d))) : f16x8{};
        }
        return scale;
    } else {
        f32x4 x[C::kSteps][2];
        float mx = 0.f;
#pragma unroll
        for (int t = 0; t < C::kSteps; t++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int d = C::col(t, g) + 4 * k;
                x[t][k] = d < D ? ld_global(reinterpret_cast<const f32x4*>(q + d)) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(x[t][k][e]));
            }
        mx = pair_max<32>(pair_max<16>(mx));
        // the row's power of two: its largest value to [2^14, 2^15)
        const float s = mx > 0.f && mx <= kMaxFinite ? ldexpf(1.f, min(100, 14 - ilogbf(mx))) : 1.f;
#pragma unroll
        for (int t = 0; t < C::kSteps; t++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = x[t][e >> 2][e & 3] * s;
                const _Float16 hi = (_Float16)y;
                qf[t][0][e] = hi;
                qf[t][1][e] = (_Float16)((y - (float)hi) * 2048.f);
            }
        return fmaxf(scale / s, 1.17549435e-38f);
    }
}

// Sums are kept in units of a power of two, ref, that follows the blocks' scales of V: 2^-6 of a largest one. far: scales lie where the unit's products and sums do not
// reach, and the wave's blocks are done again.
struct ValueUnit {
    float ref = 0.f, low = INFINITY;                        // low: the smallest unit so far
    bool far = false;
};
// rv: a block's scales in units of u.ref, which V is multiplied by as it becomes fp16: at most 2^6, and exact from 2^-15 on, 2^-15 of the block's largest at least. Probabilities
// stay as they are, so that a row has its accuracy from the tokens that it sees. Groups whose scale is smaller still are `late`, rv zero: zeros (under 2^-120), or far. Scales of
// 2^-100 and less, and of a block more than 2^-32 below the unit's, move no unit. A wave that is far takes some hundred times as long (64 rows after 2000 tokens, 28 / 4
// heads of 128, 27 us and 3.0 ms; with a quarter of the groups zeros 26). Returns what the sums so far are multiplied by. Groups from lim on have no token, and
// scales that may hold anything.
__device__ __forceinline__ float v_reference(const float (&vs)[4], int lim, ValueUnit& u, float (&rv)[4], uint32_t& late)
{
    float top = 0.f, al = 1.f;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (16 * i < lim) top = fmaxf(top, vs[i]);
    if (top > 0x1p-100f && (top > u.ref * 0x1p6f || (top < u.ref && top > u.ref * 0x1p-26f))) {
        const float ref = top * 0x1p-6f;
        al = u.ref / ref;
        u.ref = ref;
        u.low = fminf(u.low, ref);
        u.far |= u.low < ref * 0x1p-100f;
    }
    const float inv = u.ref > 0.f ? 1.f / u.ref : 0.f;
    late = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        rv[i] = 16 * i < lim ? vs[i] * inv : 0.f;
        if (rv[i] < 0x1p-15f) {
            rv[i] = 0.f;
            if (16 * i < lim) late |= 1u << i;
        }
    }
    late = __builtin_amdgcn_readfirstlane(late);
    return al;
}
// whether any value of the late groups is not zero, group i being word i of v
__device__ __forceinline__ uint32_t v_late(u32x4 v, uint32_t late)
{
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (late >> i & 1) any |= v[i] & 0x7F7F7F7F;
    return any;
}

// which of word j of part h of V's fragment are of tokens before lim: four tokens of group j (e4m3), or two of group 2 h + j / 2
template <bool F8>
__device__ __forceinline__ uint32_t v_there(int lim, int h, int j, int g)
{
    constexpr int kIn = F8 ? 4 : 2;
    const int n = min(max(lim - (F8 ? 16 * j + 4 * g : 32 * h + 16 * (j >> 1) + 4 * g + 2 * (j & 1)), 0), kIn);
    return n == kIn ? ~0u : (1u << (n * (32 / kIn))) - 1;
}

// 16 bytes a lane to LDS, a wave's in a row from `to`
__device__ __forceinline__ void load_to_lds(const void* from, void* to)
{
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
#endif
}

template <bool F8, typename Q, int DP, int WAVES, bool FULL>
__device__ __forceinline__ void paged_decode(const PagedAttnArgs& a, float* merge, int wg)
{
    using C = DecodeTile<F8, Q, DP>;
    typedef PagedLayout<F8 ? 1 : 2> Lay;
    constexpr int kKT = F8 ? 4 : 2, kTokens = 16 * kKT;    // tiles of 16 tokens, tokens of a block: V's that lie together
    // all of LDS is one variable of the kernel's: with several, the compiler takes the reads of LDS in paged_prompt to meet the loads on their way there
    auto& stat = *reinterpret_cast<float(*)[2][WAVES][kPairs]>(merge + WAVES * kPairs * C::kMerge);
    float* const row_inv = merge + WAVES * kPairs * (C::kMerge + 2);
    int* const row_at = reinterpret_cast<int*>(row_inv + kPairs);
    const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4, D = FULL ? DP : a.D;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PagedBatch& b = a.b;
    const int kvh = wg % a.KV, w = wg / a.KV;

    // this workgroup's range [at, end) of all sequences' blocks, or of their tiles where each is done whole (a.whole)
    auto count = [&](const PagedSeq& q) { return few(a, q) ? tiles_of(a, q) * (a.whole ? 1 : blocks_of<kTokens>(q)) : 0; };
    PagedUnits units(b, count);
    long long at = w, end = w + 1;
    if (!a.whole) {
        const long long total = units.total(), per = per_range<WAVES>(a, total);
        at = w * per;
        end = min(at + per, total);
    }
    while (at < end) {
        Piece p;
        int local;
        if (!units.find(at, p.s, local, p.q)) return;
        p.nb = blocks_of<kTokens>(p.q);
        if (a.whole) {
            p.r0 = kPairs * local;
            p.b0 = 0;
            p.b1 = p.nb;
            at++;
        } else {
            const int tile = local / p.nb;
            p.r0 = kPairs * tile;
            p.b0 = local - tile * p.nb;
            p.b1 = (int)min((long long)p.nb, p.b0 + (end - at));
            at += p.b1 - p.b0;
        }
        const int R = p.q.n * a.G, r = min(p.r0 + i16, R - 1), row = r / a.G;
        const size_t q_row = ((size_t)(p.q.row0 + row) * a.H + kvh * a.G + (r - row * a.G)) * D;
        const int last = p.q.len - p.q.n + row;             // the lane's pair sees the tokens up to it
        const int all = p.q.len - p.q.n;                    // every row of the sequence sees the tokens up to it

        f16x8 qf[C::kSteps][C::kParts];
        const float f = load_q<C>(static_cast<const Q*>(a.q) + q_row, g, D, a.scale, qf);
        f32x4 acc[C::kCT];
        float mr = -INFINITY, l = 0.f;
#pragma unroll
        for (int c = 0; c < C::kCT; c++) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};

        // The wave's blocks first, first + WAVES, ...; lane j knows the page of number (base + j) of them
        const int first = p.b0 + wave, mine = first < p.b1 ? (p.b1 - first + WAVES - 1) / WAVES : 0;
        int pages = 0;
        u32x4 kraw[kKT][C::kUnits], vraw[C::kCT];
        float ks[4], vs[4];
        ValueUnit vu;
        struct At {
            size_t head;
            int in_page, t0, lim;                           // lim: tokens of the block that a row may see
        };
        auto block = [&](int k) {
            if ((k & 63) == 0) pages = k + lane < mine ? paged_page(b, p.s, (first + (k + lane) * WAVES) * kTokens) : -1;
            const int page = __builtin_amdgcn_readlane(pages, k & 63);
            At x;
            x.t0 = (first + k * WAVES) * kTokens;
            x.in_page = x.t0 & ((1 << b.log_page) - 1);
            x.lim = page < 0 ? 0 : min(kTokens, p.q.len - x.t0);
            x.head = (size_t)max(page, 0) * a.KV + kvh;
            return x;
        };
        auto load_k = [&](const At& x) {
            const u32x4* k = reinterpret_cast<const u32x4*>(static_cast<const char*>(a.k) + ((x.head << b.log_page) + x.in_page) * D * (F8 ? 1 : 2));
#pragma unroll
            for (int kt = 0; kt < kKT; kt++)
#pragma unroll
                for (int c = 0; c < C::kUnits; c++) {
                    const int unit = 4 * c + g;             // D / kUnit units of 16 tokens
                    kraw[kt][c] = unit * Lay::kUnit < D ? ld_global(k + kt * 16 * (D / Lay::kUnit) + unit * 16 + i16) : u32x4{0, 0, 0, 0};
                }
            if constexpr (F8) {
                const float* s = a.k_scale + (x.head << (b.log_page - 4)) + (x.in_page >> 4);
                const float* v = a.v_scale + (x.head << (b.log_page - 4)) + (x.in_page >> 4);
#pragma unroll
                for (int i = 0; i < 4; i++) ks[i] = ld_global(s + i), vs[i] = ld_global(v + i);
            }
        };
        auto load_v = [&](const At& x) {
            const u32x4* v = reinterpret_cast<const u32x4*>(static_cast<const char*>(a.v) + ((x.head << b.log_page) + x.in_page) * D * (F8 ? 1 : 2));
#pragma unroll
            for (int c = 0; c < C::kCT; c++)
                if (16 * c < D) vraw[c] = ld_global(v + c * 64 + lane);
        };
        At now = block(0);
        if (mine > 0) load_k(now);
        for (int k = 0; k < mine; k++) {
            const At x = now;
            load_v(x);
            float fk[4], vb[4];
            if constexpr (F8)
#pragma unroll
                for (int i = 0; i < 4; i++) fk[i] = f * ks[i], vb[i] = vs[i];
            f32x4 s[kKT];
#pragma unroll
            for (int kt = 0; kt < kKT; kt++) {
                f32x4 hi = {0.f, 0.f, 0.f, 0.f}, lo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 0; t < C::kSteps; t++) {
                    f16x8 y;
                    if constexpr (F8) {
                        const u32x4 w = kraw[kt][t >> 1];
                        y = t & 1 ? f8_to_f16(w[2], w[3]) : f8_to_f16(w[0], w[1]);
                    } else {
                        y = __builtin_bit_cast(f16x8, kraw[kt][t]);
                    }
                    if constexpr (!C::kHalf) lo = mfma_16x16x32_f16(y, qf[t][1], lo);
                    hi = mfma_16x16x32_f16(y, qf[t][0], hi);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) s[kt][i] = (C::kHalf ? hi[i] : fmaf(lo[i], 1.f / 2048.f, hi[i])) * (F8 ? fk[kt] : f);
            }
            if (k + 1 < mine) {
                now = block(k + 1);
                load_k(now);
            }
            if (x.lim < kTokens || x.t0 + kTokens - 1 > all) {
                const int see = min(x.lim, last - x.t0 + 1);
#pragma unroll
                for (int kt = 0; kt < kKT; kt++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (16 * kt + 4 * g + i >= see) s[kt][i] = -INFINITY;
            }
            float bm = s[0][0];
#pragma unroll
            for (int kt = 0; kt < kKT; kt++)
#pragma unroll
                for (int i = 0; i < 4; i++) bm = maxi(bm, s[kt][i]);
            bm = pair_maxi<32>(pair_maxi<16>(bm));
            if (__any(bm > mr + kRaise)) {
                const float mn = fmaxf(mr, bm), al = ex2(mr - (mn == -INFINITY ? 0.f : mn));
                mr = mn;
                l *= al;
#pragma unroll
                for (int c = 0; c < C::kCT; c++) acc[c] *= al;
            }
            float rv[4];
            uint32_t late = 0;
            if constexpr (F8) {
                const float al = v_reference(vb, x.lim, vu, rv, late);
                if (al != 1.f)
#pragma unroll
                    for (int c = 0; c < C::kCT; c++) acc[c] *= al;
            }
            const float ref = mr == -INFINITY ? 0.f : mr;
            f16x8 pf[kKT / 2][C::kParts];
#pragma unroll
            for (int kt = 0; kt < kKT; kt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = ex2(s[kt][i] - ref);
                    l += e;
                    const float y = e * kPScale;
                    const _Float16 hi = (_Float16)y;
                    pf[kt >> 1][0][4 * (kt & 1) + i] = hi;
                    if constexpr (!C::kHalf) pf[kt >> 1][1][4 * (kt & 1) + i] = (_Float16)(y - (float)hi);
                }
            if (x.lim < kTokens)                            // what no row sees may hold anything: zero
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t keep = v_there<F8>(x.lim, 0, j, g);
#pragma unroll
                    for (int c = 0; c < C::kCT; c++) vraw[c][j] &= keep;
                }
            if (late) {
                uint32_t any = 0;
#pragma unroll
                for (int c = 0; c < C::kCT; c++)
                    if (16 * c < D) any |= v_late(vraw[c], late);
                vu.far |= __any(any != 0);
            }
            // a block's sums start from zero and are added to the others by the VALU: the matrix unit carries no long sum
#pragma unroll
            for (int c = 0; c < C::kCT; c++) {
                if (16 * c >= D) continue;
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < kKT / 2; h++) {
                    f16x8 v;
                    if constexpr (F8) v = f8_to_f16(vraw[c][2 * h], vraw[c][2 * h + 1], rv[2 * h], rv[2 * h + 1]);
                    else v = __builtin_bit_cast(f16x8, vraw[c]);
#pragma unroll
                    for (int part = C::kParts - 1; part >= 0; part--) o = mfma_16x16x32_f16(v, pf[h][part], o);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) acc[c][i] += o[i];
            }
        }
        float odd = l * 0.f;                                // NaN if a sum is not finite
#pragma unroll
        for (int c = 0; c < C::kCT; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) odd = fmaf(acc[c][i], 0.f, odd);
        const bool redo = __any(odd != 0.f) || vu.far;
        if (redo) paged_again<F8, Q, C::kCT, kTokens>(a, p, kvh, q_row, last, first, WAVES, mr, l, acc);

        // the waves' states
        const float unit = redo ? 1.f : F8 ? vu.ref / kPScale : 1.f / kPScale;
        l = pair_sum<32>(pair_sum<16>(l));
        __syncthreads();                                    // the last piece's are read
        if (g == 0) {
            stat[0][wave][i16] = mr;
            stat[1][wave][i16] = l;
        }
        __syncthreads();
        float mx = stat[0][0][i16];
#pragma unroll
        for (int k = 1; k < WAVES; k++) mx = fmaxf(mx, stat[0][k][i16]);
        const float wt = mr == -INFINITY ? (l != l ? 1.f : 0.f) : ex2(mr - mx) * unit;   // NaN: no score is a number
#pragma unroll
        for (int c = 0; c < C::kCT; c++) {
            f32x4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = wt == 0.f ? 0.f : acc[c][i] * wt;
            *reinterpret_cast<f32x4*>(merge + (wave * kPairs + i16) * C::kMerge + 16 * c + 4 * g) = v;
        }
        const bool cut = p.b0 > 0 || p.b1 < p.nb;
        float* const part = a.ws + ((size_t)wg * 2 + (p.b0 == 0)) * (kPairs * (D + 2));
        if (tid < kPairs) {
            float top = stat[0][0][tid], total = 0.f;
#pragma unroll
            for (int k = 1; k < WAVES; k++) top = fmaxf(top, stat[0][k][tid]);
#pragma unroll
            for (int k = 0; k < WAVES; k++) {
                const float lk = stat[1][k][tid], mk = stat[0][k][tid];
                total += mk == -INFINITY ? (lk != lk ? lk : 0.f) : lk * ex2(mk - top);
            }
            row_at[tid] = p.r0 + tid < R ? 1 : 0;
            row_inv[tid] = cut ? 1.f : total == 0.f ? 0.f : 1.f / total;
            if (cut) st_global(reinterpret_cast<f32x2*>(part + kPairs * D) + tid, f32x2{top, total});
        }
        __syncthreads();
        for (int u = tid; u < kPairs * (D / 4); u += 64 * WAVES) {
            const int pair = u / (D / 4), d = 4 * (u - pair * (D / 4));
            if (!row_at[pair]) continue;
            f32x4 sum = *reinterpret_cast<const f32x4*>(merge + pair * C::kMerge + d);
#pragma unroll
            for (int k = 1; k < WAVES; k++) sum += *reinterpret_cast<const f32x4*>(merge + (k * kPairs + pair) * C::kMerge + d);
            const float inv = row_inv[pair];
            sum = f32x4{sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
            if (cut) {
                st_global(reinterpret_cast<f32x4*>(part + pair * D + d), sum);
            } else {
                const int rr = p.r0 + pair, m = rr / a.G;
                paged_out(static_cast<Q*>(a.out) + ((size_t)(p.q.row0 + m) * a.H + kvh * a.G + (rr - m * a.G)) * D + d, sum);
            }
        }
    }
}

// The parts of the pairs whose blocks more than one workgroup had: out = sum_i acc_i 2^(m_i - m) / sum_i l_i 2^(m_i - m). A workgroup has `pairs` of a tile's
// pairs; the parts lie with the workgroups of the kv head in a row, the first part in its workgroup's second place, the others in their first. A wave
// makes a pair's weights, then thread (slot, pair, four columns) adds parts slot, slot + slots, ... in order, and the slots are added in order.
constexpr int kMergeWeights = 4096;
template <typename Q, int WAVES, int BLOCK>
__device__ __forceinline__ void paged_merge(const PagedAttnArgs& a, float (&wgt)[kMergeWeights], f32x4 (&sums)[256], int wg)
{
    const PagedBatch& b = a.b;
    const int per_tile = kPairs / a.merge_pairs, kvh = wg % a.KV, rest = wg / a.KV, unit = rest / per_tile, pair0 = (rest - unit * per_tile) * a.merge_pairs;
    const int tid = threadIdx.x, lane = tid & 63, D = a.D;
    // the tile, and how many blocks lie before it and in all
    long long total = 0, before = 0;
    int tiles = 0, s = -1, tile = 0;
    PagedSeq q = {0, 0, 0};
    for (int s0 = 0; s0 < b.S; s0 += 64) {
        PagedSeq me = {0, 0, 0};
        if (s0 + lane < b.S) me = paged_seq(b, s0 + lane);
        const int ct = me.n && few(a, me) ? tiles_of(a, me) : 0, cb = ct ? ct * blocks_of<BLOCK>(me) : 0;
        const int ut = wave_upto(ct), ub = wave_upto(cb);
        if (s < 0 && unit < tiles + __builtin_amdgcn_readlane(ut, 63)) {
            const int at = __builtin_ctzll(__ballot(tiles + ut > unit));
            s = s0 + at;
            q = {__builtin_amdgcn_readlane(me.row0, at), __builtin_amdgcn_readlane(me.n, at), __builtin_amdgcn_readlane(me.len, at)};
            tile = unit - tiles - (__builtin_amdgcn_readlane(ut, at) - __builtin_amdgcn_readlane(ct, at));
            before = total + __builtin_amdgcn_readlane(ub, at) - __builtin_amdgcn_readlane(cb, at) + (long long)tile * blocks_of<BLOCK>(q);
        }
        tiles += __builtin_amdgcn_readlane(ut, 63);
        total += __builtin_amdgcn_readlane(ub, 63);
    }
    if (s < 0) return;
    const int r0 = kPairs * tile + pair0, pairs = min(min(a.merge_pairs, kPairs - pair0), q.n * a.G - r0);
    const long long per = per_range<WAVES>(a, total);
    const int w0 = (int)(before / per), w1 = (int)((before + blocks_of<BLOCK>(q) - 1) / per), n = w1 - w0 + 1;
    if (n == 1 || pairs <= 0) return;
    const size_t stride = (size_t)kPairs * (D + 2);
    auto part = [&](int i) { return a.ws + ((size_t)((w0 + i) * a.KV + kvh) * 2 + (i == 0)) * stride; };
    for (int p = tid >> 6; p < pairs; p += 4) {
        float mx = -INFINITY, l = 0.f;
        for (int i = lane; i < n; i += 64) mx = fmaxf(mx, ld_global(part(i) + kPairs * D + 2 * (pair0 + p)));
        mx = wave_max(mx, lane);
        for (int i = lane; i < n; i += 64) {
            const f32x2 st = ld_global(reinterpret_cast<const f32x2*>(part(i) + kPairs * D) + pair0 + p);
            const float mi = st.x, li = st.y, e = mi == -INFINITY ? (li != li ? 1.f : 0.f) : ex2(mi - mx);   // NaN: no score is a number
            wgt[p * n + i] = e;
            l += e == 0.f ? 0.f : li * e;
        }
        l = wave_sum(l, lane);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        for (int i = lane; i < n; i += 64) wgt[p * n + i] *= inv;
    }
    __syncthreads();
    const int nc = D / 4, items = pairs * nc, slots = max(1, 256 / items), slot = tid / items;
    for (int it = tid - slot * items; it < items; it += 256) {        // more than one round only where a slot is the whole workgroup
        const int p = it / nc, c = it - p * nc;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        if (slot < slots)
#pragma unroll 4
            for (int i = slot; i < n; i += slots) {
                const float wi = wgt[p * n + i];
                const f32x4 x = ld_global(reinterpret_cast<const f32x4*>(part(i) + (pair0 + p) * D) + c);
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = wi == 0.f ? o[k] : fmaf(wi, x[k], o[k]);
            }
        if (slots > 1) {
            sums[tid] = o;
            __syncthreads();
        }
        if (slot > 0) break;
        if (slots > 1)
            for (int i = 1; i < slots; i++) o += sums[it + i * items];
        const int rr = r0 + p, m = rr / a.G;
        paged_out(static_cast<Q*>(a.out) + ((size_t)(q.row0 + m) * a.H + kvh * a.G + (rr - m * a.G)) * D + 4 * c, o);
    }
}

// Sequences of many rows: a workgroup has 64 NT (row, head) pairs of one kv head, 16 NT a wave, and goes through their tokens, 64 at a time, which all its waves
// read from LDS; the next 64 are on their way there meanwhile, as they lie in memory. Scores, softmax and products as above.
// Their tiles come the longest first where a wave's lanes hold all sequences, and in parts of their tokens where there are few of them; paged_join joins
// the parts.
struct PromptTiles {
    const PagedAttnArgs& a;
    const int rows;                                         // pairs of a tile
    struct Count {
        const PagedAttnArgs& a;
        int rows;
        __device__ __forceinline__ int operator()(const PagedSeq& q) const { return few(a, q) ? 0 : (q.n * a.G + rows - 1) / rows; }
    };
    PagedUnits<Count> units;
    long long total;
    int most;                                               // parts of a tile at most

    __device__ __forceinline__ PromptTiles(const PagedAttnArgs& a, int rows) : a(a), rows(rows), units(a.b, Count{a, rows})
    {
        total = units.total();
        most = total > 0 ? (int)max(1ll, min(kPromptParts / (total * a.KV), (long long)kPromptMost)) : 1;
    }
    // tile number j as a piece, whole; in how many parts it is done
    __device__ __forceinline__ bool find(long long j, Piece& p, int& parts)
    {
        if (j >= total) return false;
        int tile;
        if (a.b.S > 64) {
            if (!units.find(total - 1 - j, p.s, tile, p.q)) return false;
        } else {
            const PagedSeq me = units.me;
            const int mine = units.c, all = me.len - me.n;
            // the lane's sequence's tiles of less than x blocks: those whose last row's token lies before block x - 1
            auto below = [&](int x) {
                const int y = (x - 1) * kBlock - all;
                return y <= 0 ? 0 : y >= me.n ? mine : min(mine, y * a.G / rows);
            };
            auto from = [&](int x) { return (int)total - __builtin_amdgcn_readlane(wave_upto(below(x)), 63); };   // all tiles of x blocks or more
            int lo = 1, hi = (a.b.max_len + kBlock - 1) / kBlock + 1;
            while (hi - lo > 1) {
                const int x = (lo + hi) >> 1;
                if (from(x) > j) lo = x;
                else hi = x;
            }
            const int first = below(lo), c = below(lo + 1) - first, upto = wave_upto(c), k = (int)j - from(lo + 1), at = __builtin_ctzll(__ballot(upto > k));
            p.s = at;
            p.q = {__builtin_amdgcn_readlane(me.row0, at), __builtin_amdgcn_readlane(me.n, at), __builtin_amdgcn_readlane(me.len, at)};
            tile = __builtin_amdgcn_readlane(first, at) + k - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(c, at));
        }
        p.r0 = rows * tile;
        p.nb = (p.q.len - p.q.n + (min(p.r0 + rows, p.q.n * a.G) - 1) / a.G) / kBlock + 1;
        p.b0 = 0;
        p.b1 = p.nb;
        parts = max(1, min(most, p.nb / 4));
        return true;
    }
};

template <bool F8, typename Q, int DP, int NT>
struct PromptTile {
    using C = DecodeTile<F8, Q, DP>;
    static constexpr int kWaves = 4, kRows = 16 * NT * kWaves;
    static constexpr int kBytes = kBlock * DP * (F8 ? 1 : 2);    // of K or V of a block
    static constexpr int kLds = 4 * kBytes > C::kMergeBytes ? 2 * kBytes : C::kMergeBytes / 2;   // half of what a workgroup of either kind has
};

template <bool F8, typename Q, int DP, int NT, bool FULL>
__device__ __forceinline__ void paged_prompt(const PagedAttnArgs& a, char (&lds)[2][PromptTile<F8, Q, DP, NT>::kLds], int wg)
{
    using C = DecodeTile<F8, Q, DP>;
    using T = PromptTile<F8, Q, DP, NT>;
    typedef PagedLayout<F8 ? 1 : 2> Lay;
    const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4, D = FULL ? DP : a.D;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PagedBatch& b = a.b;
    const int kvh = wg % a.KV;
    Piece p;
    int parts;
    {
        PromptTiles tiles(a, T::kRows);
        const int number = wg / a.KV, part = number % tiles.most;
        if (!tiles.find(number / tiles.most, p, parts) || part >= parts) return;
        p.b0 = (int)((long long)p.nb * part / parts);
        p.b1 = (int)((long long)p.nb * (part + 1) / parts);
    }
    const int R = p.q.n * a.G, all = p.q.len - p.q.n;       // every row sees the tokens up to `all`
    const int low = all + p.r0 / a.G;                       // every row of the tile sees the tokens up to it

    size_t q_row[NT];
    int last[NT];
    f16x8 qf[NT][C::kSteps][C::kParts];
    float f[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = min(p.r0 + 16 * (NT * wave + nt) + i16, R - 1), row = r / a.G;
        q_row[nt] = ((size_t)(p.q.row0 + row) * a.H + kvh * a.G + (r - row * a.G)) * D;
        last[nt] = all + row;
        f[nt] = load_q<C>(static_cast<const Q*>(a.q) + q_row[nt], g, D, a.scale, qf[nt]);
    }
    const _Float16 one = (_Float16)1.f;
    const f16x8 ones = {one, one, one, one, one, one, one, one};
    f32x4 acc[C::kCT][NT], ls[NT];                          // ls, l: the sums of P, of fp16 rows by the matrix unit, in every register
    float mr[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        mr[nt] = -INFINITY;
        l[nt] = 0.f;
        ls[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C::kCT; c++) acc[c][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int pages = 0;
    float ks[4], vs[4];
    ValueUnit vu;
    const int chunks = D * (F8 ? 1 : 2) / 16;               // of 1 KB, of K or V of a block
    auto page_of = [&](int k) {
        const int r = (k - p.b0) & 63;
        if (r == 0) pages = k + lane < p.b1 ? paged_page(b, p.s, (k + lane) * kBlock) : -1;
        return __builtin_amdgcn_readlane(pages, r);
    };
    auto fetch = [&](int k, int page) {
        char* const to = lds[k & 1];
        const int in_page = (k * kBlock) & ((1 << b.log_page) - 1);
        const size_t head = (size_t)max(page, 0) * a.KV + kvh, at = ((head << b.log_page) + in_page) * D * (F8 ? 1 : 2);
        // an address that the wave shares, the lane's own part of it, and an LDS address per KB
        const uint32_t mine = 16 * lane;
        const char* const kp = static_cast<const char*>(a.k) + at;
        const char* const vp = static_cast<const char*>(a.v) + at;
#pragma unroll
        for (int c = 0; c < (DP * (F8 ? 1 : 2) / 16 + T::kWaves - 1) / T::kWaves; c++) {
            const int u = wave + T::kWaves * c;
            if ((FULL && DP * (F8 ? 1 : 2) / 16 % T::kWaves == 0) || u < chunks) {
                load_to_lds(kp + u * 1024 + mine, to + u * 1024);
                load_to_lds(vp + u * 1024 + mine, to + T::kBytes + u * 1024);
            }
        }
        if constexpr (F8) {
            const float* ss = a.k_scale + (head << (b.log_page - 4)) + (in_page >> 4);
            const float* sv = a.v_scale + (head << (b.log_page - 4)) + (in_page >> 4);
#pragma unroll
            for (int i = 0; i < 4; i++) ks[i] = ld_global(ss + i), vs[i] = ld_global(sv + i);
        }
    };
    int page = page_of(p.b0);
    fetch(p.b0, page);
    for (int k = p.b0; k < p.b1; k++) {
        char* const from = lds[k & 1];
        const int t0 = k * kBlock, lim = page < 0 ? 0 : min(kBlock, p.q.len - t0);
        // this block has arrived, and every wave is done with the one that the next takes the place of
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x70);                   // vmcnt(0) lgkmcnt(0), in a form that the compiler counts
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (lim < kBlock) {                                 // V that no row sees may hold anything: zero
            for (int u = tid; u < 4 * chunks * 16; u += 64 * T::kWaves) {
                u32x4* w = reinterpret_cast<u32x4*>(from + T::kBytes) + u;
                const int h = F8 ? 0 : u / (4 * D);
#pragma unroll
                for (int j = 0; j < 4; j++) (*w)[j] &= v_there<F8>(lim, h, j, u >> 4 & 3);
            }
            __syncthreads();
        }
        float kss[4], vss[4];
        if constexpr (F8)
#pragma unroll
            for (int i = 0; i < 4; i++) kss[i] = 16 * i < lim ? ks[i] : 1.f, vss[i] = vs[i];   // groups without a token may hold anything
        if (k + 1 < p.b1) {
            page = page_of(k + 1);
            fetch(k + 1, page);
        }
        const u32x4* const kl = reinterpret_cast<const u32x4*>(from) + lane;
        const u32x4* const vl = reinterpret_cast<const u32x4*>(from + T::kBytes) + lane;
        f32x4 s[4][NT];
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            f32x4 hi[NT], lo[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) hi[nt] = lo[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < C::kUnits; c++) {
                const u32x4 w = (4 * c + g) * Lay::kUnit < D ? kl[kt * (D / Lay::kUnit) * 16 + c * 64] : u32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < (F8 ? 2 : 1); j++) {
                    const f16x8 y = F8 ? f8_to_f16(w[2 * j], w[2 * j + 1]) : __builtin_bit_cast(f16x8, w);
                    const int t = F8 ? 2 * c + j : c;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        if constexpr (!C::kHalf) lo[nt] = mfma_16x16x32_f16(y, qf[nt][t][1], lo[nt]);
                        hi[nt] = mfma_16x16x32_f16(y, qf[nt][t][0], hi[nt]);
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[kt][nt][i] = C::kHalf ? hi[nt][i] : fmaf(lo[nt][i], 1.f / 2048.f, hi[nt][i]);
        }
        if (lim < kBlock || t0 + kBlock - 1 > low)          // some row sees not all
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const int see = min(lim, last[nt] - t0 + 1) - 4 * g;
#pragma unroll
                for (int kt = 0; kt < 4; kt++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (16 * kt + i >= see) s[kt][nt][i] = -INFINITY;
            }
        float bm[NT];
        bool up = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float mk[4];
#pragma unroll
            for (int kt = 0; kt < 4; kt++) mk[kt] = maxi(maxi(s[kt][nt][0], s[kt][nt][1]), maxi(s[kt][nt][2], s[kt][nt][3])) * (F8 ? kss[kt] : 1.f);
            bm[nt] = pair_maxi<32>(pair_maxi<16>(maxi(maxi(mk[0], mk[1]), maxi(mk[2], mk[3])))) * f[nt];
            up = up || bm[nt] > mr[nt] + kRaise;
        }
        if (__any(up))
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float mn = fmaxf(mr[nt], bm[nt]), al = ex2(mr[nt] - (mn == -INFINITY ? 0.f : mn));
                mr[nt] = mn;
                l[nt] *= al;
                ls[nt] *= al;
#pragma unroll
                for (int c = 0; c < C::kCT; c++) acc[c][nt] *= al;
            }
        float rv[4];
        if constexpr (F8) {
            uint32_t late;
            const float al = v_reference(vss, lim, vu, rv, late);
            if (al != 1.f)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < C::kCT; c++) acc[c][nt] *= al;
            if (late) {
                uint32_t any = 0;
#pragma unroll
                for (int c = 0; c < C::kCT; c++)
                    if (16 * c < D) any |= v_late(vl[c * 64], late);
                vu.far |= __any(any != 0);
            }
        }
        f16x8 pf[2][NT][C::kParts];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const float ref = (mr[nt] == -INFINITY ? 0.f : mr[nt]) - kPLog;
#pragma unroll
            for (int kt = 0; kt < 4; kt++) {
                const float fk = F8 ? f[nt] * kss[kt] : f[nt];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = ex2(fmaf(s[kt][nt][i], fk, -ref));
                    if constexpr (C::kHalf) {
                        pf[kt >> 1][nt][0][4 * (kt & 1) + i] = (_Float16)e;
                    } else {
                        l[nt] += e;
                        const _Float16 hi = (_Float16)e;
                        pf[kt >> 1][nt][0][4 * (kt & 1) + i] = hi;
                        pf[kt >> 1][nt][1][4 * (kt & 1) + i] = (_Float16)(e - (float)hi);
                    }
                }
            }
        }
        if constexpr (C::kHalf)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int h = 0; h < 2; h++) ls[nt] = mfma_16x16x32_f16(ones, pf[h][nt][0], ls[nt]);   // of P as it is rounded
#pragma unroll
        for (int c = 0; c < C::kCT; c++) {
            if (16 * c >= D) continue;
            u32x4 w[C::kVB];
#pragma unroll
            for (int h = 0; h < C::kVB; h++) w[h] = vl[h * 4 * D + c * 64];
            // fp32 rows: a block's sums start from zero and are added to the others by the VALU: the matrix unit carries no long sum
            f32x4 o[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) o[nt] = C::kHalf ? acc[c][nt] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f16x8 v = F8 ? f8_to_f16(w[0][2 * h], w[0][2 * h + 1], rv[2 * h], rv[2 * h + 1]) : __builtin_bit_cast(f16x8, w[F8 ? 0 : h]);
#pragma unroll
                for (int part = C::kParts - 1; part >= 0; part--)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) o[nt] = mfma_16x16x32_f16(v, pf[h][nt][part], o[nt]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) acc[c][nt] = C::kHalf ? o[nt] : acc[c][nt] + o[nt];
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float odd = (C::kHalf ? ls[nt][0] : l[nt]) * 0.f;   // NaN if a sum is not finite
        f32x4 mine[C::kCT];
#pragma unroll
        for (int c = 0; c < C::kCT; c++) {
            mine[c] = acc[c][nt];
#pragma unroll
            for (int i = 0; i < 4; i++) odd = fmaf(mine[c][i], 0.f, odd);
        }
        float unit = (F8 ? vu.ref : 1.f) / kPScale, total = (C::kHalf ? ls[nt][0] : pair_sum<32>(pair_sum<16>(l[nt]))) * (1.f / kPScale);
        if (__any(odd != 0.f) || vu.far) {
            paged_again<F8, Q, C::kCT, kBlock>(a, p, kvh, q_row[nt], last[nt], p.b0, 1, mr[nt], l[nt], mine);
            unit = 1.f;
            total = pair_sum<32>(pair_sum<16>(l[nt]));
        }
        const int pair = 16 * (NT * wave + nt) + i16;
        if (parts > 1) {                                    // a part's sums and state
            float* const ws = a.ws + a.prompt_ws + (size_t)wg * (T::kRows * (D + 2));
#pragma unroll
            for (int c = 0; c < C::kCT; c++)
                if (16 * c < D) st_global(reinterpret_cast<f32x4*>(ws + pair * D + 16 * c + 4 * g), f32x4{mine[c][0] * unit, mine[c][1] * unit, mine[c][2] * unit, mine[c][3] * unit});
            if (g == 0) st_global(reinterpret_cast<f32x2*>(ws + T::kRows * D) + pair, f32x2{mr[nt], total});
        } else {
            const float inv = total == 0.f ? 0.f : unit / total;
            const bool there = p.r0 + pair < R;
#pragma unroll
            for (int c = 0; c < C::kCT; c++)
                if (there && 16 * c < D) paged_out(static_cast<Q*>(a.out) + q_row[nt] + 16 * c + 4 * g, f32x4{mine[c][0] * inv, mine[c][1] * inv, mine[c][2] * inv, mine[c][3] * inv});
        }
    }
}

// The parts of a tile of many rows likewise: a workgroup has a.join_pairs of a tile's pairs.
template <typename Q, int ROWS>
__device__ __forceinline__ void paged_join(const PagedAttnArgs& a, float (&all)[kMergeWeights], int wg)
{
    auto& wgt = reinterpret_cast<float(&)[32][kPromptMost]>(all);
    const int per_tile = ROWS / a.join_pairs;
    const int kvh = wg % a.KV, rest = wg / a.KV, tile = rest / per_tile, tid = threadIdx.x, D = a.D, pair0 = a.join_pairs * (rest % per_tile);
    Piece p;
    int parts;
    PromptTiles tiles(a, ROWS);
    if (tiles.most == 1 || !tiles.find(tile, p, parts) || parts == 1) return;
    const int R = p.q.n * a.G, pairs = min(a.join_pairs, R - p.r0 - pair0);
    if (pairs <= 0) return;
    auto part = [&](int i) { return a.ws + a.prompt_ws + (size_t)((tile * tiles.most + i) * a.KV + kvh) * (ROWS * (D + 2)); };
    if (tid < pairs) {
        f32x2 st[kPromptMost];
        float mx = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < kPromptMost; i++) {
            st[i] = i < parts ? ld_global(reinterpret_cast<const f32x2*>(part(i) + ROWS * D) + pair0 + tid) : f32x2{-INFINITY, 0.f};
            mx = fmaxf(mx, st[i].x);
        }
#pragma unroll
        for (int i = 0; i < kPromptMost; i++) {
            const float mi = st[i].x, li = st[i].y, e = mi == -INFINITY ? (li != li ? 1.f : 0.f) : ex2(mi - mx);   // NaN: no score is a number
            l += e == 0.f ? 0.f : li * e;
            st[i].x = e;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < kPromptMost; i++) wgt[tid][i] = st[i].x * inv;
    }
    __syncthreads();
    const int nc = D / 4;
    for (int u = tid; u < pairs * nc; u += 256) {
        const int pair = u / nc, c = u - pair * nc;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int i = 0; i < parts; i++) {
            const float w = wgt[pair][i];
            const f32x4 x = ld_global(reinterpret_cast<const f32x4*>(part(i) + (pair0 + pair) * D) + c);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = w == 0.f ? o[e] : fmaf(w, x[e], o[e]);
        }
        const int r = p.r0 + pair0 + pair, m = r / a.G;
        paged_out(static_cast<Q*>(a.out) + ((size_t)(p.q.row0 + m) * a.H + kvh * a.G + (r - m * a.G)) * D + 4 * c, o);
    }
}

// Both kinds of parts in one launch
template <typename Q, int WAVES, int BLOCK, int ROWS>
__global__ __launch_bounds__(256) void paged_parts_kernel(const PagedAttnArgs a)
{
    __shared__ float wgt[kMergeWeights];
    __shared__ f32x4 sums[256];
    if ((int)blockIdx.x < a.merge) paged_merge<Q, WAVES, BLOCK>(a, wgt, sums, blockIdx.x);
    else paged_join<Q, ROWS>(a, wgt, blockIdx.x - a.merge);
}

// One launch for both: the first a.decode workgroups have the sequences of few rows. Where these are as many as the device holds at once (two a CU at D = 128), the others begin
// as they end; both kinds are at work together only where they are fewer.
template <bool F8, typename Q, int DP, int NT, bool FULL>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void paged_attention_kernel(const PagedAttnArgs a)
{
    using T = PromptTile<F8, Q, DP, NT>;
    __shared__ __attribute__((aligned(16))) char lds[2][T::kLds];
    if ((int)blockIdx.x < a.decode) paged_decode<F8, Q, DP, kDecodeWaves, FULL>(a, reinterpret_cast<float*>(lds[0]), blockIdx.x);
    else paged_prompt<F8, Q, DP, NT, FULL>(a, lds, blockIdx.x - a.decode);
}
template <bool F8, typename Q, int DP, bool FULL>
__global__ __launch_bounds__(64 * kDecodeWaves, DP > 128 ? 1 : 2) void paged_decode_kernel(const PagedAttnArgs a)
{
    __shared__ __attribute__((aligned(16))) char lds[DecodeTile<F8, Q, DP>::kMergeBytes];
    paged_decode<F8, Q, DP, kDecodeWaves, FULL>(a, reinterpret_cast<float*>(lds), blockIdx.x);
}

}  // namespace

// at most 512 * 2 * 16 * (D + 2) floats of the few and 512 * rows * (D + 2) of the many: 51 MB
uint64_t plan_paged_attention(PagedAttnArgs* a)
{
    const long long pairs = (long long)a->b.M * a->G;
    // Tiles of 16 pairs read the tokens each for themselves, tiles of 64 or 128 once but through LDS. Few as 4 tiles or fewer, against all as many, in us (28 / 4 heads of
    // 128, fp32 rows): 16 sequences of 8 rows (56 pairs) after 2000 tokens 31, 43, e4m3 26, 42; of 16 rows (112 pairs) 80, 39 and 50, 41
    a->few = 4 * kPairs;
    a->units = (int)std::min<long long>(4ll * a->b.S, a->b.S + pairs / kPairs);
    // Whole tiles of sequences that are short, or not very long and many, against ranges and their second launch, which lengths far apart need: one row after 500 tokens
    // 8.2, 10.5, after 1000 11.3, 10.6; 64 after 2048 43, 49, e4m3 25, 32, of 100 to 2048 20, 35; one after 2000 17.6, 11; one of 2048 and 63 of 200 18, 15 to 20
    a->whole = a->b.max_len <= 1024 || (a->b.max_len <= 2048 && (long long)a->b.S * a->KV >= 128);
    a->ranges = std::max(1, 512 / a->KV);
    // the merge's workgroups: some hundreds, their weights in LDS
    a->merge_pairs = 1;
    while (a->merge_pairs < kPairs && (long long)a->units * a->KV * (kPairs / a->merge_pairs) > 512 && 2 * a->merge_pairs * a->ranges <= kMergeWeights) a->merge_pairs *= 2;
    const bool merge = !a->whole && a->ranges > 1;
    a->merge = merge ? a->units * a->KV * (kPairs / a->merge_pairs) : 0;
    a->decode = (a->whole ? a->units : a->ranges) * a->KV;
    a->prompt_ws = merge ? (size_t)a->ranges * a->KV * 2 * kPairs * (a->D + 2) : 0;
    a->prompt = a->join = a->join_pairs = 0;
    // Tiles of 64 pairs (registers allow no more over D = 128) where those of 128 would leave much of the device without work: few of them, and few tokens to part. 128 and 64
    // pairs, fp32 rows (fp16 rows), in us: 64 rows 14, 8.4 (10, 6.8); 1000 of one prompt 55, 40 (40, 30); 1500 78, 56 (53, 41); 300 after 8000 97, 101 (64, 72);
    // 8 x 300 41, 42 (29, 32); 4 x 128 after 4000 90, 87 (59, 61, e4m3 66, 77)
    const long long full = pairs * a->KV / 128, tokens = a->b.max_len - std::min(a->b.max_rows, a->b.max_len) / 2;
    a->rows = a->D > 128 || (full <= 384 && full * tokens <= (a->half ? 4 : 7) << 16) ? 64 : 128;
    uint64_t bytes = a->prompt_ws * sizeof(float);
    if ((long long)a->b.max_rows * a->G > a->few) {
        const int rows = a->rows;
        // tiles of whole rows, and one more of each sequence of so many rows that it is none of the few
        const long long tiles = pairs / rows + std::min<long long>(a->b.S, pairs / a->few) + 1;
        a->prompt = (int)std::max<long long>(tiles * a->KV, kPromptParts);
        // tiles are done in parts where they have eight blocks and there are so few that two parts of each are no more than kPromptParts
        if (a->b.max_len > 7 * kBlock && kPromptParts / a->KV >= 2) {
            a->join_pairs = tiles * a->KV > 64 ? 32 : 8;      // few tiles have many parts: more workgroups for them
            a->join = (int)std::min<long long>(tiles, kPromptParts / a->KV / 2) * a->KV * (rows / a->join_pairs);
            bytes += (uint64_t)kPromptParts * rows * (a->D + 2) * sizeof(float);
        }
    }
    return bytes;
}

namespace {

template <bool F8, typename Q, int DP, int NT, bool FULL>
hipError_t launch(const PagedAttnArgs& a, hipStream_t stream)
{
    if (a.prompt) hipLaunchKernelGGL((paged_attention_kernel<F8, Q, DP, NT, FULL>), dim3(a.decode + a.prompt), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((paged_decode_kernel<F8, Q, DP, FULL>), dim3(a.decode), dim3(256), 0, stream, a);
    if (a.merge + a.join) hipLaunchKernelGGL((paged_parts_kernel<Q, kDecodeWaves, F8 ? 64 : 32, 64 * NT>), dim3(a.merge + a.join), dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <bool F8, typename Q, int NT>
hipError_t launch_nt(const PagedAttnArgs& a, hipStream_t stream)
{
    if (a.D == 64) return launch<F8, Q, 64, NT, true>(a, stream);
    if (a.D == 128) return launch<F8, Q, 128, NT, true>(a, stream);
    if (a.D < 64) return launch<F8, Q, 64, NT, false>(a, stream);
    return launch<F8, Q, 128, NT, false>(a, stream);
}

template <bool F8, typename Q>
hipError_t launch_d(const PagedAttnArgs& a, hipStream_t stream)
{
    if (a.D == 256) return launch<F8, Q, 256, 1, true>(a, stream);
    if (a.D > 128) return launch<F8, Q, 256, 1, false>(a, stream);
    return a.rows == 64 ? launch_nt<F8, Q, 1>(a, stream) : launch_nt<F8, Q, 2>(a, stream);
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream)
{
    if (a.k_scale) return a.half ? launch_d<true, _Float16>(a, stream) : launch_d<true, float>(a, stream);
    return a.half ? launch_d<false, _Float16>(a, stream) : launch_d<false, float>(a, stream);
}

}  // namespace ql
