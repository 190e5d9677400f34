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

// inclusive sums over a wave: rows of 16 by shifts, then the rows before
__device__ __forceinline__ int wave_upto(int v)
{
    v += (int)__builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8: nothing comes in at a row's start
    v += (int)__builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += (int)__builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += (int)__builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += (int)__builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // the last of a row to the next, rows 1 and 3
    v += (int)__builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // that of the first half to the second
    return v;
}

// The units that the sequences have, count(sequence) of each, in order. Every lane of a wave takes part and gets the same; a lane knows a sequence
// of the 64 that were looked at last, so that tables of up to 64 are read once.
template <typename F>
struct PagedUnits {
    const PagedBatch& b;
    F count;
    PagedSeq me;
    int c, upto, s0 = 0;
    long long before = 0;

    __device__ __forceinline__ PagedUnits(const PagedBatch& b, F count) : b(b), count(count) { load(); }
    __device__ __forceinline__ void load()
    {
        const int s = s0 + (threadIdx.x & 63);
        me = {0, 0, 0};
        if (s < b.S) me = paged_seq(b, s);
        c = me.n ? count(me) : 0;
        upto = wave_upto(c);
    }
    __device__ __forceinline__ int here() const { return __builtin_amdgcn_readlane(upto, 63); }
    __device__ __forceinline__ bool next()
    {
        if (s0 + 64 >= b.S) return false;
        before += here();
        s0 += 64;
        load();
        return true;
    }
    __device__ __forceinline__ long long total()
    {
        while (next()) {}
        return before + here();
    }
    // unit number j: its sequence s and its number in it; false beyond the last one
    __device__ __forceinline__ bool find(long long j, int& s, int& local, PagedSeq& q)
    {
        if (j < before) {
            s0 = 0;
            before = 0;
            load();
        }
        while (j >= before + here())
            if (!next()) return false;
        const int at = __builtin_ctzll(__ballot(before + upto > j));
        s = s0 + at;
        local = (int)(j - before) - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(c, at));
        q = {__builtin_amdgcn_readlane(me.row0, at), __builtin_amdgcn_readlane(me.n, at), __builtin_amdgcn_readlane(me.len, at)};
        return true;
    }
};

// The sequence of a row, for a whole wave; false: padding. Where the table ascends it is the first that ends behind the row; an entry that it may not have can miscount, so
// a row that this one does not have is looked for in all (a row that no sequence ends behind is in none).
__device__ __forceinline__ bool paged_row(const PagedBatch& b, int row, int& s, PagedSeq& q)
{
    const int lane = threadIdx.x & 63;
    s = 0;
    for (int s0 = 0; s0 < b.S; s0 += 64) s += __popcll(__ballot(s0 + lane < b.S && ld_global(b.row_start + 1 + min(s0 + lane, b.S - 1)) <= row));
    if (s >= b.S) return false;
    q = paged_seq(b, s);
    if (__builtin_expect(!(row >= q.row0 && row < q.row0 + q.n), 0)) {
        s = b.S;
        for (int s0 = 0; s0 < b.S && s == b.S; s0 += 64) {
            PagedSeq me = {0, 0, 0};
            if (s0 + lane < b.S) me = paged_seq(b, s0 + lane);
            const uint64_t has = __ballot(row >= me.row0 && row < me.row0 + me.n);
            if (has) s = s0 + __builtin_ctzll(has);
        }
        if (s == b.S) return false;
        q = paged_seq(b, s);
    }
    return true;
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
