// Low-rank adapters of a batch's rows beside a shared projection (ql_lora_add): y = base + s_a (x . A_a^T) . B_a^T, a = ids[row].
//
// lora_row_kernel, few rows: a workgroup of sixteen waves has a row of a projection and a range of its columns. t = x . A^T first: a wave has
// four ranks, so that x is read once for them, and a part of K, the parts' sums meet in LDS; then a thread has a column of y, and B's row of it. The
// workgroups of one row's column ranges each make t for themselves: A comes from L2, and a second launch would cost more.
//
// Four rows of 3 adapters of rank 8 beside q/k/v of 896 columns 4.6 us, 64 rows of 24 of rank 16 beside those of 3584 8.4 us (15 MB): a launch, a chain of two
// products and their loads from L2, where rows of one adapter read it each for themselves.
//
// Many rows, two launches: lora_down_kernel makes t of 16 or 32 rows, four waves a part of K each, on the matrix cores, T^T = A x^T
// (lane = row, registers = ranks), for all projections that read one x; lora_up_kernel has 16 rows and 64 columns a wave, Y = T B^T. Rows of
// several adapters in one tile: it is gone through once for each adapter, and a row takes its own. fp32 x enters as two fp16 parts (22 bits) under the
// exponent of the row's 64 columns at a time; t likewise under the row's.
// 4096 rows, 4 adapters of rank 64 beside q/k/v of 3584 columns, fp16 x, 188 MB: 66 us. The second launch, 37 us, is at 4.1 TB/s of base and y; the first, 30, at
// 10 TB/s of A and x from L2, which its tiles read again (a tile of 64 rows whose waves share A in LDS needs K in parts for as many workgroups, and the parts' sums
// cost the second launch 20 us; rank groups of the same rows on one XCD brought 5).
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
    // (lanes that share a column, so that a load is a stretch of memory: no faster at rank 64, and 100 rows of rank 16 to 18944 columns 32 us for 20)
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

constexpr int kDownWaves = 4, kDownGroup = 4;      // waves of a workgroup; most tiles of 16 ranks that it makes
constexpr int kDownTiles = 24;                     // of a launch
constexpr int kUpRows = 32, kUpCols = 256;         // rows of a pass are a multiple of the first launch's; columns of a workgroup of the second
constexpr int kTwoTiles = 1024;                    // rows from which the first launch's A serves two tiles of 16 rows

// The ranks of all projections that read one x, in tiles of 16
struct LoraDown {
    struct Tile {
        const uint16_t* a;         // row of the tile's first rank, of adapter 0
        const float* scale;
        float* t;                  // its first rank's column of t [rows, rank]
        long long step;            // values from an adapter to the next
        int ranks, rank, n;        // ranks of the tile, of the projection; adapters
        size_t part;               // values from a part of K's t to the next
    } tile[kDownTiles];
    const void* x;
    const int32_t* ids;
    int K, M, tiles, most, parts;  // most: adapters of the projection that has most; parts of K, of workgroups each
};

// The adapters of RT tiles of 16 rows, one after the other: bit 16 t + i of `left` is row i of tile t, whose adapter lane i knows in id[t]
template <int RT>
__device__ __forceinline__ uint64_t rows_with(const int (&id)[RT], int which)
{
    uint64_t m = 0;
#pragma unroll
    for (int t = 0; t < RT; t++) m |= (__ballot(id[t] == which) & 0xFFFF) << (16 * t);
    return m;
}
template <int RT>
__device__ __forceinline__ uint64_t rows_below(const int (&id)[RT], int n)
{
    uint64_t m = 0;
#pragma unroll
    for (int t = 0; t < RT; t++) m |= (__ballot((uint32_t)id[t] < (uint32_t)n) & 0xFFFF) << (16 * t);
    return m;
}
template <int RT>
__device__ __forceinline__ int first_adapter(const int (&id)[RT], uint64_t left)
{
    const int r = __builtin_ctzll(left);
    int which = 0;
#pragma unroll
    for (int t = 0; t < RT; t++)
        if (r >> 4 == t) which = __builtin_amdgcn_readlane(id[t], r & 15);
    return which;
}
// 16 bytes a lane to LDS, a wave's in a row from `to`
__device__ __forceinline__ void load_to_lds(const void* from, void* to)
{
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
#endif
}
// what a wave has asked for of memory and LDS is there
__device__ __forceinline__ void wave_arrived()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x70);                       // vmcnt(0) lgkmcnt(0), in a form that the compiler counts
    asm volatile("" ::: "memory");
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

// Of a step of 64 columns: a lane's 16 columns of row i16 of x from `x`, as parts under `1 / up`. Columns that are not there are zeros.
template <bool HALF>
__device__ __forceinline__ void x_parts(const char* x, int i16, int g, const bool (&in)[2], f16x8 (&hi)[2], f16x8 (&lo)[2], float& up)
{
    up = 1.f;
    if constexpr (HALF) {
#pragma unroll
        for (int h = 0; h < 2; h++) hi[h] = in[h] ? *reinterpret_cast<const f16x8*>(x + ((2 * g + h) ^ (i16 & 7)) * 16) : f16x8{};
    } else {
        float v[2][8], mx = 0.f;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const f32x4 y = *reinterpret_cast<const f32x4*>(x + ((4 * g + q) ^ i16) * 16);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[q >> 1][4 * (q & 1) + e] = in[q >> 1] ? y[e] : 0.f;
                mx = fmaxf(mx, fabsf(v[q >> 1][4 * (q & 1) + e]));
            }
        }
        mx = pair_max<32>(pair_max<16>(mx));
        const float s = scale_of(mx);
        up = 1.f / s;
#pragma unroll
        for (int h = 0; h < 2; h++) split_f16(v[h], s, hi[h], lo[h]);
    }
}
// A wave has a quarter of K, 64 columns at a time. Fragments are 16 rows' 16 bytes, which as loads would be a line a lane: rows come whole into a part of LDS that is
// the wave's own, 128 bytes of eight rows a load, and are turned there (4096 rows of rank 64, fp16, both launches: 221 -> 85 us); the next 64 columns are on their way
// meanwhile. The 16-byte pieces of row r lie in the order c ^ (r % 8), so that a fragment's reads meet no bank twice.
template <bool HALF, int TILES, int RT>
struct DownLds {
    static constexpr int kXRow = HALF ? 128 : 256;               // bytes of a row of x, of 64 columns
    static constexpr int kStep = TILES * 2048 + RT * 16 * kXRow; // of a wave's step
    static constexpr int kEnd = kDownWaves * RT * TILES * 1024;  // of the waves' sums
    static constexpr int kBytes = 2 * kDownWaves * kStep > kEnd ? 2 * kDownWaves * kStep : kEnd;
};

template <bool HALF, int TILES, int RT>
__global__ __launch_bounds__(64 * kDownWaves) void lora_down_kernel(const LoraDown d)
{
    using L = DownLds<HALF, TILES, RT>;
    __shared__ __attribute__((aligned(16))) char lds[2][L::kBytes / 2];
    // The groups of ranks of the same rows come one after the other on one XCD, so that x comes from its L2 for all but the first. Of fewer rows an XCD has a range, and few
    // adapters then; of more it has every eighth tile, since ranges meet on memory's channels (4 adapters of rank 64 in runs, q/k/v, fp16 and fp32 x, ranges against tiles in
    // turn, us: 512 rows 22, 25; 1024 26, 28 and 40, 41; 1500 33, 34 and 52, 46; 4096 68, 67 and 101, 90)
    const int groups = (d.tiles + TILES - 1) / TILES, per_xcd = gridDim.x / (8 * groups), xcd = blockIdx.x % 8, in_xcd = blockIdx.x / 8, at = in_xcd / groups;
    const int m0 = 16 * RT * (d.M > kTwoTiles ? 8 * at + xcd : per_xcd * xcd + at), u0 = TILES * (in_xcd - at * groups);
    const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
    if (m0 >= d.M) return;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) id[t] = m0 + 16 * t + i16 < d.M ? ld_global(d.ids + m0 + 16 * t + i16) : -1;
    uint64_t left = rows_below(id, d.most);
    const int steps = (d.K + 63) / 64, per = (steps + d.parts * kDownWaves - 1) / (d.parts * kDownWaves);
    const int s0 = (blockIdx.z * kDownWaves + wave) * per, s1 = min(steps, s0 + per);
    // of the loads, a lane's row and piece
    const int ar = lane >> 3, ac = (lane & 7) ^ ar, xr = HALF ? ar : lane >> 4, xp = HALF ? 8 : 4;
    while (left) {
        const int which = first_adapter(id, left);
        const uint64_t mine = left & rows_with(id, which);
        left &= ~mine;
        const uint16_t* w[TILES][2];
#pragma unroll
        for (int u = 0; u < TILES; u++) {                   // a rank or tile that is not there: another one, not stored
            const LoraDown::Tile& t = d.tile[min(u0 + u, d.tiles - 1)];
#pragma unroll
            for (int h = 0; h < 2; h++) w[u][h] = t.a + (which < t.n ? which : 0) * t.step + (size_t)min(8 * h + ar, t.ranks - 1) * d.K;
        }
        auto fetch = [&](int st, int buf) {
            char* const to = lds[buf] + wave * L::kStep;
            const int ka = 64 * st + 8 * ac, k = ka < d.K ? ka : 0;          // beyond K: what is there, not used
#pragma unroll
            for (int u = 0; u < TILES; u++)
#pragma unroll
                for (int h = 0; h < 2; h++) load_to_lds(w[u][h] + k, to + u * 2048 + h * 1024);
#pragma unroll
            for (int j = 0; j < RT * 16 / xp; j++) {
                const int r = j * xp + xr, m = min(m0 + r, d.M - 1);
                const int c = HALF ? ac : (lane & 15) ^ (r & 15), kx = 64 * st + (HALF ? 8 : 4) * c, kk = kx < d.K ? kx : 0;
                load_to_lds(static_cast<const char*>(d.x) + ((size_t)m * d.K + kk) * (HALF ? 2 : 4), to + TILES * 2048 + j * 1024);
            }
        };
        f32x4 acc[TILES][RT];
#pragma unroll
        for (int u = 0; u < TILES; u++)
#pragma unroll
            for (int t = 0; t < RT; t++) acc[u][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s0 < s1) fetch(s0, s0 & 1);
        for (int st = s0; st < s1; st++) {
            wave_arrived();
            if (st + 1 < s1) fetch(st + 1, (st + 1) & 1);
            const char* const from = lds[st & 1] + wave * L::kStep;
            const int k = 64 * st + 16 * g;
            const bool in[2] = {k < d.K, k + 8 < d.K};      // K is a multiple of eight
            f16x8 hi[RT][2], lo[RT][2];
            float up[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) x_parts<HALF>(from + TILES * 2048 + (16 * t + i16) * L::kXRow, i16, g, in, hi[t], lo[t], up[t]);
#pragma unroll
            for (int u = 0; u < TILES; u++) {
                f16x8 w[2];                                 // beyond K zeros on both sides: 0 * NaN
#pragma unroll
                for (int h = 0; h < 2; h++) w[h] = in[h] ? *reinterpret_cast<const f16x8*>(from + u * 2048 + i16 * 128 + ((2 * g + h) ^ (i16 & 7)) * 16) : f16x8{};
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    if constexpr (HALF) {
#pragma unroll
                        for (int h = 0; h < 2; h++) acc[u][t] = mfma_16x16x32_f16(w[h], hi[t][h], acc[u][t]);
                    } else {
                        f32x4 o = {0.f, 0.f, 0.f, 0.f}, ol = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            ol = mfma_16x16x32_f16(w[h], lo[t][h], ol);
                            o = mfma_16x16x32_f16(w[h], hi[t][h], o);
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[u][t][e] = fmaf(fmaf(ol[e], 1.f / 2048.f, o[e]), up[t], acc[u][t][e]);
                    }
                }
            }
        }
        // the waves' parts, where their steps lay
        f32x4* const part = reinterpret_cast<f32x4*>(lds);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < TILES; u++)
#pragma unroll
            for (int t = 0; t < RT; t++) part[((wave * TILES + u) * RT + t) * 64 + lane] = acc[u][t];
        __syncthreads();
        for (int v = wave; v < min(TILES, d.tiles - u0) * RT; v += kDownWaves) {
            const int u = v / RT, row = 16 * (v - u * RT) + i16;
            const LoraDown::Tile& t = d.tile[u0 + u];
            f32x4 sum = part[v * 64 + lane];
#pragma unroll
            for (int k = 1; k < kDownWaves; k++) sum += part[(k * TILES * RT + v) * 64 + lane];
            if ((mine >> row & 1) && which < t.n && 4 * g < t.ranks) {
                const float s = t.scale ? ld_global(t.scale + which) : 1.f;
                st_global(reinterpret_cast<f32x4*>(t.t + blockIdx.z * t.part + (size_t)(m0 + row) * t.rank + 4 * g), f32x4{sum[0] * s, sum[1] * s, sum[2] * s, sum[3] * s});
            }
        }
        __syncthreads();
    }
}

// Y = T B^T: lane = column, registers = rows 4 g + r. A workgroup has 16 rows and 256 columns of a projection, a wave 64 of them in four tiles, tile j's column i
// being 4 i + j: a lane's four results of a row are 16 bytes, a row's 256 in a row (columns 16 j + i, 64 bytes: 45 us for 38; 32 rows a workgroup, of which the registers leave half as many: 38 for 37, 64: 59). The projections' columns lie one behind
// the other in blockIdx.x. An adapter's B of the 256 columns is one stretch of memory: it goes to LDS as it lies, but for the order of a row's pieces,
// c ^ (n / 4 % their number) where that is a power of two.
template <int STEPS>
__global__ __launch_bounds__(256, 2) void lora_up_kernel(const LoraArgs a)
{
    __shared__ __attribute__((aligned(16))) char lds[kUpCols * STEPS * 64];
    const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int proj = 0, xb = blockIdx.x;
    while (xb >= (a.p[proj].N + kUpCols - 1) / kUpCols) xb -= (a.p[proj++].N + kUpCols - 1) / kUpCols;
    const LoraArgs::One& p = a.p[proj];
    const int m0 = 16 * blockIdx.y, n0 = kUpCols * xb, cols = min(kUpCols, p.N - n0), pieces = p.rank / 8, nl = 64 * wave + 4 * i16;
    const int turn = pieces & (pieces - 1) ? 0 : min(pieces, 8) - 1;
    const bool apart = p.base != p.y;
    const int id[1] = {m0 + i16 < a.M ? ld_global(a.ids + m0 + i16) : -1};
    uint64_t left = rows_below(id, p.n);
    const uint32_t all = (uint32_t)left;
    if (!left && !apart) return;
    auto fetch = [&](int which) {
        const char* const B = reinterpret_cast<const char*>(p.b + ((size_t)which * p.N + n0) * p.rank);
        const int all_pieces = cols * pieces;
        for (int u = tid; u < (all_pieces + 63) / 64 * 64; u += 256) {
            const int at = min(u, all_pieces - 1), n = at / pieces, c = at - n * pieces;
            load_to_lds(B + (n * pieces + (c ^ (n >> 2 & turn))) * 16, lds + (u - lane) * 16);
        }
    };
    int which = 0;
    if (left) fetch(which = first_adapter(id, left));
    f32x4 y[4];                                             // rows 4 g + r, the lane's four columns
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int m = m0 + 4 * g + r;
        y[r] = m < a.M && nl < cols ? ld_global(reinterpret_cast<const f32x4*>(p.base + (size_t)m * p.N + n0 + nl)) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float mx = 0.f, v[STEPS][8];
    const float* const t = a.ws + a.t_off[proj];
#pragma unroll
    for (int st = 0; st < STEPS; st++) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[st][e] = 0.f;
        if ((all >> i16 & 1) && 32 * st + 8 * g < p.rank) {
            const size_t at = (size_t)(m0 + i16) * p.rank + 32 * st + 8 * g;
            load8(t, 0, at, v[st]);
            for (int k = 1; k < a.parts[proj]; k++) {       // the other parts of K, in order
                float w[8];
                load8(t, 0, (size_t)k * a.M * p.rank + at, w);
#pragma unroll
                for (int e = 0; e < 8; e++) v[st][e] += w[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(v[st][e]));
    }
    mx = pair_max<32>(pair_max<16>(mx));
    const float s = scale_of(mx), up = 1.f / s;
    f16x8 hi[STEPS], lo[STEPS];
#pragma unroll
    for (int st = 0; st < STEPS; st++) split_f16(v[st], s, hi[st], lo[st]);
    float up_of[4];                                         // of the rows that the lane's results are of
#pragma unroll
    for (int r = 0; r < 4; r++) up_of[r] = __shfl(up, 4 * g + r);
    while (left) {
        const uint64_t mine = left & rows_with(id, which);
        left &= ~mine;
        wave_arrived();
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = nl + j;
            f32x4 o = {0.f, 0.f, 0.f, 0.f}, ol = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < STEPS; st++) {
                const int c = 4 * st + g;
                const f16x8 w = n < cols && c < pieces ? *reinterpret_cast<const f16x8*>(lds + (n * pieces + (c ^ (n >> 2 & turn))) * 16) : f16x8{};
                ol = mfma_16x16x32_f16(lo[st], w, ol);
                o = mfma_16x16x32_f16(hi[st], w, o);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) y[r][j] = mine >> (4 * g + r) & 1 ? fmaf(fmaf(ol[r], 1.f / 2048.f, o[r]), up_of[r], y[r][j]) : y[r][j];
        }
        __syncthreads();
        if (left) fetch(which = first_adapter(id, left));
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int m = m0 + 4 * g + r;
        if (m < a.M && nl < cols && ((all >> (4 * g + r) & 1) || apart)) st_global(reinterpret_cast<f32x4*>(p.y + (size_t)m * p.N + n0 + nl), y[r]);
    }
}

}  // namespace

uint64_t plan_lora(LoraArgs* a, size_t ws_bytes)
{
    a->rows = 0;
    int rank = 0;
    for (int i = 0; i < a->count; i++) rank = std::max(rank, a->p[i].rank);
    if (a->M <= kLoraRowMax || (long long)a->M * rank <= kLoraRowRanks) return 0;
    // K in parts where the tiles of 16 rows and up to four of 16 ranks that read one x are few: two steps of 64 a wave at least
    int64_t values = 0;                                     // of t, a row
    for (int i = 0; i < a->count; i++) {
        int tiles = 0;
        for (int k = 0; k < a->count; k++)
            if (a->p[k].x == a->p[i].x && a->p[k].K == a->p[i].K) tiles += (a->p[k].rank + 15) / 16;
        const int groups = (a->M + 15) / 16 * ((tiles + kDownGroup - 1) / kDownGroup);
        a->parts[i] = std::max(1, std::min({512 / groups, 16, a->p[i].K / (64 * 2 * kDownWaves)}));
        values += a->p[i].rank * a->parts[i];
    }
    // as many rows at once as have room
    a->rows = (int)std::min<int64_t>(a->M, (int64_t)(ws_bytes / sizeof(float)) / values / kUpRows * kUpRows);
    for (int64_t i = 0, at = 0; i < a->count; i++) {
        a->t_off[i] = at;
        at += (int64_t)a->rows * a->p[i].rank * a->parts[i];
    }
    return values * a->rows * sizeof(float);
}

namespace {

template <bool HALF>
void launch_down(const LoraDown& d, hipStream_t stream)
{
    auto go = [&](auto kernel, int tiles, int rt) {
        const int rows = (d.M + 16 * rt - 1) / (16 * rt);
        hipLaunchKernelGGL(kernel, dim3((rows + 7) / 8 * 8 * ((d.tiles + tiles - 1) / tiles), 1, d.parts), dim3(64 * kDownWaves), 0, stream, d);
    };
    // 32 rows where they still fill the device (q/k/v of rank 64, fp16, both launches, 16 and 32 rows: 4096 rows 72.5, 67.5 us, 1024 30.1, 29.0; fp32 89.9, 102.6)
    if (HALF && d.M >= kTwoTiles && d.tiles > 1) go(lora_down_kernel<HALF, 3, HALF ? 2 : 1>, 3, HALF ? 2 : 1);
    else if (d.tiles == 1) go(lora_down_kernel<HALF, 1, 1>, 1, 1);
    else if (d.tiles <= 3 || d.tiles == 5) go(lora_down_kernel<HALF, 3, 1>, 3, 1);
    else go(lora_down_kernel<HALF, kDownGroup, 1>, kDownGroup, 1);
}

void launch_up(const LoraArgs& a, hipStream_t stream)
{
    int cols = 0, rank = 0;
    for (int i = 0; i < a.count; i++) {
        cols += (a.p[i].N + kUpCols - 1) / kUpCols;
        rank = std::max(rank, a.p[i].rank);
    }
    const dim3 grid(cols, (a.M + 15) / 16);
    if (rank <= 32) hipLaunchKernelGGL(lora_up_kernel<1>, grid, dim3(256), 0, stream, a);
    else if (rank <= 64) hipLaunchKernelGGL(lora_up_kernel<2>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(lora_up_kernel<4>, grid, dim3(256), 0, stream, a);
}

hipError_t launch_tiled(const LoraArgs& a, hipStream_t stream)
{
    bool done[kMaxBatch] = {};
    for (int i = 0; i < a.count; i++) {
        if (done[i]) continue;
        LoraDown d;
        d.x = a.p[i].x;
        d.ids = a.ids;
        d.K = a.p[i].K;
        d.M = a.M;
        d.parts = a.parts[i];
        d.tiles = d.most = 0;
        auto flush = [&] {
            if (a.half) launch_down<true>(d, stream);
            else launch_down<false>(d, stream);
            d.tiles = d.most = 0;
        };
        for (int k = i; k < a.count; k++) {
            const LoraArgs::One& p = a.p[k];
            if (done[k] || p.x != d.x || p.K != d.K) continue;
            done[k] = true;
            for (int r = 0; r < p.rank; r += 16) {
                if (d.tiles == kDownTiles) flush();
                d.tile[d.tiles++] = {p.a + (size_t)r * p.K, p.scale, a.ws + a.t_off[k] + r, (long long)p.rank * p.K, std::min(16, p.rank - r), p.rank, p.n, (size_t)a.M * p.rank};
                d.most = std::max(d.most, p.n);
            }
        }
        if (d.tiles) flush();
    }
    launch_up(a, stream);
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
