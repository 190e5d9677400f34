// Rows of cache regions moved (ql_kv_move): dst[dst_row + i] = src[src_row + rows[i]] (rows = 0, 1, .. where no list is given)
// in every region, a K or V cache of one layer. Forks a sequence (a prefix into another cache) and keeps a tree's
// accepted path (rows gathered in place).
//
// kv_copy_kernel: source and destination rows do not overlap; 16 bytes a thread and step, two loads in flight, loads and stores
//   past the caches: 115 MB copied in 38.3 us, 6.0 TB/s of reads and writes (cached 41.6; four in flight 39.5 and 43.2; eight 40.6 and 45.2).
// kv_gather_kernel: a region onto itself, up to kMoveInPlaceRows rows. A workgroup has a strip of columns of all n
//   rows and holds it in registers (kHold pieces of 16 bytes a thread) until every load of the strip has arrived, so any
//   list is right, also one that names a row twice or out of order.
// An index outside the source leaves its destination row as it was.
// Bytes: each row read once and written once.
#include <algorithm>

#include "ql_device.h"
#include "ql_digits.h"
#include "ql_internal.h"

namespace ql {

namespace {

constexpr int kUnroll = 2;
constexpr int kHold = 4;
static_assert(kMoveInPlaceRows <= 256 * kHold, "a strip of one column piece fits a workgroup's registers");

__device__ __forceinline__ long long source_row(const MoveArgs& a, uint32_t i)
{
    const long long at = a.rows ? ld_global(a.rows + i) : (long long)i, r = a.src_row + at;
    return at >= 0 && r < a.src_max_t ? r : -1;
}

__global__ __launch_bounds__(256) void kv_copy_kernel(const MoveArgs a)
{
    const uint32_t units = (uint32_t)a.n * a.row16;
    const char* src = a.region[blockIdx.y].src;
    char* dst = a.region[blockIdx.y].dst;
    const uint32_t u0 = blockIdx.x * (256u * kUnroll) + threadIdx.x;
    u32x4 v[kUnroll];
    long long r[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; k++) {
        const uint32_t u = u0 + 256u * k, i = u / a.row16, c = u - i * a.row16;
        r[k] = u < units ? source_row(a, i) : -1;
        if (r[k] >= 0) v[k] = ld_stream(reinterpret_cast<const u32x4*>(src + ((size_t)r[k] * a.row16 + c) * 16));
    }
#pragma unroll
    for (int k = 0; k < kUnroll; k++) {
        const uint32_t u = u0 + 256u * k;
        if (r[k] >= 0) __builtin_nontemporal_store(v[k], QL_GLOBAL(u32x4, reinterpret_cast<u32x4*>(dst + ((size_t)a.dst_row * a.row16 + u) * 16)));
    }
}

__global__ __launch_bounds__(256) void kv_gather_kernel(const MoveArgs a)
{
    const char* src = a.region[blockIdx.y].src;
    char* dst = a.region[blockIdx.y].dst;
    const uint32_t c0 = blockIdx.x * a.strip, width = min((uint32_t)a.strip, (uint32_t)a.row16 - c0), units = (uint32_t)a.n * width;
    u32x4 v[kHold];
    long long r[kHold];
#pragma unroll
    for (int k = 0; k < kHold; k++) {
        const uint32_t u = threadIdx.x + 256u * k, i = u / width, c = c0 + (u - i * width);
        r[k] = u < units ? source_row(a, i) : -1;
        if (r[k] >= 0) v[k] = ld_global(reinterpret_cast<const u32x4*>(src + ((size_t)r[k] * a.row16 + c) * 16));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // every row is in registers before one is overwritten
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kHold; k++) {
        const uint32_t u = threadIdx.x + 256u * k, i = u / width, c = c0 + (u - i * width);
        if (r[k] >= 0) st_global(reinterpret_cast<u32x4*>(dst + ((size_t)(a.dst_row + i) * a.row16 + c) * 16), v[k]);
    }
}

}  // namespace

hipError_t launch_kv_move(MoveArgs& a, hipStream_t stream)
{
    if (a.in_place) {
        a.strip = std::max(1, std::min(a.row16, 256 * kHold / a.n));
        hipLaunchKernelGGL(kv_gather_kernel, dim3((a.row16 + a.strip - 1) / a.strip, a.count), dim3(256), 0, stream, a);
    } else {
        const long long units = (long long)a.n * a.row16;
        hipLaunchKernelGGL(kv_copy_kernel, dim3((unsigned)((units + 256 * kUnroll - 1) / (256 * kUnroll)), a.count), dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace ql
