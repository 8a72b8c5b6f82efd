// What the kernels of the page tables share: sums over a workgroup, the stack's size, the checks of a call's tables.
#pragma once

#include "qwfn_common.h"
#include "qwfn_paged.h"

#include <algorithm>

namespace qwfn {
namespace {

constexpr int PT_THREADS = 1024;       // of a scan
constexpr int PT_WAVES   = PT_THREADS / 64;
constexpr int64_t PT_MAX_SEQ = 65536;

// What a scan leaves for the second launch.
struct pt_req {
    int32_t past;      // extend: tokens held; trim: first column given back
    int32_t have;      // extend: pages held; trim: pages given back
    int32_t at;        // the call's pages of the requests before this one
    int32_t served;
};
struct pt_head {
    int32_t n_free;    // at the start of the call, clipped
    int32_t total;     // extend: listed tokens (cu_new[n_seq])
    int32_t pad[2];
};

__device__ __forceinline__ int64_t shfl_up64(int64_t v, int d) { return __shfl_up((long long) v, d); }

// Inclusive sums of two values over the workgroup's threads, in thread order.
struct pair64 { int64_t x, y; };
__device__ __forceinline__ pair64 block_scan(pair64 v, pair64 (*part)[PT_WAVES]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t x = shfl_up64(v.x, d), y = shfl_up64(v.y, d);
        if (lane >= d) { v.x += x; v.y += y; }
    }
    if (lane == 63) (*part)[w] = v;
    __syncthreads();
    for (int i = 0; i < w; i++) { v.x += (*part)[i].x; v.y += (*part)[i].y; }
    return v;
}

__device__ __forceinline__ int64_t ceil_div(int64_t a, int32_t b) { return (int64_t) (((uint32_t) a + (uint32_t) b - 1u) / (uint32_t) b); }

// The stack's size, clipped.
__device__ __forceinline__ int32_t stack_size(const int32_t * n_free, int32_t cap, bool & bad) {
    const int32_t n = *n_free, x = n < 0 ? 0 : n > cap ? cap : n;
    bad |= x != n;
    return x;
}

inline int scan_threads(int32_t n_seq) { return std::min(PT_THREADS, (n_seq + 63) / 64 * 64); }

inline int check_table_shape(const char * op, int32_t n_seq, int32_t page_size, int64_t table_stride, int32_t max_pages) {
    const std::string o(op);
    if (n_seq < 1 || n_seq > PT_MAX_SEQ) return set_error(QWFN_EINVAL, o + ": n_seq must lie in [1, 65536]");
    if (page_size < 1 || max_pages < 1 || (int64_t) page_size * max_pages > 0x7fffffff)
        return set_error(QWFN_EINVAL, o + ": page_size and max_pages must be positive, their product below 2^31");
    if (table_stride < max_pages) return set_error(QWFN_EINVAL, o + ": table rows overlap (table_stride < max_pages)");
    if (table_stride > 0x7fffffff) return set_error(QWFN_EINVAL, o + ": table_stride must be below 2^31");
    return QWFN_OK;
}

inline int check_tables(const char * op, int32_t n_seq, int32_t page_size, int64_t table_stride, int32_t max_pages,
                        int32_t free_cap, const void * ws, size_t ws_bytes) {
    const std::string o(op);
    if (int rc = check_table_shape(op, n_seq, page_size, table_stride, max_pages)) return rc;
    if (free_cap < 0) return set_error(QWFN_EINVAL, o + ": free_cap must not be negative");
    if (!ws || ws_bytes < qwfn_paged_workspace_size(n_seq))
        return set_error(QWFN_ENOMEM, o + ": ws must hold qwfn_paged_workspace_size bytes");
    if (!is_aligned(ws, 16)) return set_error(QWFN_EALIGN, o + ": ws must be 16-byte aligned");
    return QWFN_OK;
}

// Every span 4-byte aligned and present, and no `out` over another span; in-place pairs are passed once.
inline int check_spans(const char * op, const span * in, int n_in, const span * out, int n_out) {
    for (int i = 0; i < n_in + n_out; i++) {
        const span & s = i < n_in ? in[i] : out[i - n_in];
        if (!is_aligned(s.p, 4)) return set_error(QWFN_EALIGN, std::string(op) + ": " + s.name + " must be 4-byte aligned");
    }
    return check_overlaps(op, in, n_in, out, n_out);
}

}  // namespace
}  // namespace qwfn
