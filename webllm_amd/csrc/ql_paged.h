// Device side of a batch's tables and of paged caches, shared by the append and the attention.
#pragma once

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"

namespace ql {

// A sequence's rows in the batch and its tokens with them; n = 0: it has none, or its tables say what they may not.
struct PagedSeq {
    int row0, n, len;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int s)
{
    const int r0 = ld_global(b.row_start + s), r1 = ld_global(b.row_start + s + 1), len = ld_global(b.kv_len + s);
    const bool ok = r0 >= 0 && r1 >= r0 && r1 <= b.M && r1 - r0 <= b.max_rows && len >= r1 - r0 && len <= b.max_len;
    return {r0, ok ? r1 - r0 : 0, len};
}

// Unit number j of the units that the sequences have, count(sequence) of each, in order: its sequence s and its number in it. Every
// lane of a wave takes part and gets the same; false beyond the last one.
template <typename F>
__device__ __forceinline__ bool paged_unit(const PagedBatch& b, long long j, F count, int& s, int& local, PagedSeq& q)
{
    const int lane = threadIdx.x & 63;
    long long before = 0;
    for (int s0 = 0; s0 < b.S; s0 += 64) {
        PagedSeq me = {0, 0, 0};
        if (s0 + lane < b.S) me = paged_seq(b, s0 + lane);
        const int c = me.n ? count(me) : 0;
        int upto = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(upto, o);
            if (lane >= o) upto += t;
        }
        const uint64_t past = __ballot(before + upto > j);
        if (past) {
            const int at = __builtin_ctzll(past);
            s = s0 + at;
            local = (int)(j - before) - (__shfl(upto, at) - __shfl(c, at));
            q = {__shfl(me.row0, at), __shfl(me.n, at), __shfl(me.len, at)};
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
}

// The units of all sequences, or of those before the first `upto`
template <typename F>
__device__ __forceinline__ long long paged_total(const PagedBatch& b, F count, int upto = kPagedMaxSeqs)
{
    const int lane = threadIdx.x & 63, S = min(b.S, upto);
    long long total = 0;
    for (int s0 = 0; s0 < S; s0 += 64) {
        PagedSeq me = {0, 0, 0};
        if (s0 + lane < S) me = paged_seq(b, s0 + lane);
        int c = me.n ? count(me) : 0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
        total += c;
    }
    return total;
}

// The sequence of a row, for a whole wave; false: padding.
__device__ __forceinline__ bool paged_row(const PagedBatch& b, int row, int& s, PagedSeq& q)
{
    const int lane = threadIdx.x & 63;
    s = 0;
    for (int s0 = 0; s0 < b.S; s0 += 64) s += __popcll(__ballot(s0 + lane < b.S && ld_global(b.row_start + 1 + min(s0 + lane, b.S - 1)) <= row));
    if (s >= b.S) return false;
    q = paged_seq(b, s);
    return row >= q.row0 && row < q.row0 + q.n;
}

// The page of token t of sequence s, or -1
__device__ __forceinline__ int paged_page(const PagedBatch& b, int s, int t)
{
    const int p = ld_global(b.pages + (size_t)s * b.max_pages + (t >> b.log_page));
    return (uint32_t)p < (uint32_t)b.n_page ? p : -1;
}

__device__ __forceinline__ void paged_out(float* to, f32x4 x) { st_global(reinterpret_cast<f32x4*>(to), x); }
__device__ __forceinline__ void paged_out(_Float16* to, f32x4 x)
{
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    st_global(reinterpret_cast<f16x4*>(to), __builtin_convertvector(x, f16x4));
}

// Layout (of one kv head's part of a page, in values of SIZE bytes)
template <int SIZE>
struct PagedLayout {
    static constexpr int kUnit = 16 / SIZE;        // values of 16 bytes
    static constexpr int kTokens = 64 / SIZE;      // tokens of V that lie together
    // 16 bytes of token t of K, columns 16 / SIZE * unit and on
    static __device__ __forceinline__ size_t k_at(int D, int t, int unit) { return (size_t)(t >> 4) * (16 * D) + (unit * 16 + (t & 15)) * kUnit; }
    // V's column d of tokens t .. t + 3, t a multiple of 4
    static __device__ __forceinline__ size_t v_at(int D, int t, int d)
    {
        return (size_t)(t / kTokens) * (kTokens * D) + (((d >> 4) * 4 + (t >> 2 & 3)) * 16 + (d & 15)) * kUnit + (t % kTokens >> 4) * 4;
    }
};

}  // namespace ql
