// Pages that requests hold together, and the steps that move a cache's rows: qwfn_paged_fork,
// _release, _compact, _copy, and of a drafted tree qwfn_tree_masks and qwfn_paged_accept.
// With P tokens a page and shared[p] = holders of page p less one:
//   fork     columns c < n / P of the parent's row, shared[p] += 1 each; the rest n % P on a new page
//   release  back_p = columns given back that hold p; free where back_p > shared[p], else
//            shared[p] -= back_p; the free ones by rank onto the stack
//   compact  live page p >= n_live with k live ones in [n_live, p) -> the k-th free page below n_live
//   accept   row B + i <- row B + t_i, t_i the i-th bit of the leaf's mask
//
// The tables move a few KB to a MB, so they are bound by launches and by chains of load, scan and
// store. Counters are only ever added to and taken from by integer atomics, whose order does not
// change what they end at; where a result has an order (the stack, the moves) it comes from ranks in a
// bitmap of the pages, so a call repeats bit for bit. The copies are bound by the rows, read and
// written once.
#include "paged_tables.h"

#include <algorithm>

namespace qwfn {
namespace {

constexpr int SH_THREADS = 256;
constexpr int64_t SH_MAX_GRID = 16384;
constexpr int CP_CACHES = 64;          // tensors of a launch

typedef uint32_t unit16 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int32_t clip_to(int32_t x, int32_t top, bool & bad) {
    const int32_t y = x < 0 ? 0 : x > top ? top : x;
    bad |= y != x;
    return y;
}
__device__ __forceinline__ void report(uint32_t * status, bool bad, uint32_t bit) {
    if (__ballot(bad) && (threadIdx.x & 63) == 0) atomicOr(status, bit);
}
__device__ __forceinline__ bool in_pool(int32_t p, int32_t n_pages) { return (uint32_t) p < (uint32_t) n_pages; }

// ---------------------------------------------------------------- fork

struct fork_args {
    const int32_t * from; const int32_t * n_tok; const int32_t * n_kv;
    int32_t *       table; int64_t t_stride;
    const int32_t * shared; const int32_t * free_pages;
    const int32_t * n_free; int32_t * n_free_out; int32_t * n_kv_out; int32_t * shared_out; int32_t * moves;
    const int32_t * states; int32_t * state_moves;
    int32_t         n_seq, page, room, n_pages, free_cap;      // room: max_pages * page
    pt_req *        req;               // parent, whole pages, the new page, 1 served | 2 with a new page
    uint32_t *      status;
};

// Block 0: which requests are served, by a running sum of the new pages; the others copy shared.
__global__ __launch_bounds__(PT_THREADS) void k_fork_scan(fork_args a) {
    __shared__ pair64 part[2][PT_WAVES];
    __shared__ int64_t last;
    const int tid = threadIdx.x;
    if (blockIdx.x > 0) {
        for (int64_t i = (int64_t) (blockIdx.x - 1) * blockDim.x + tid; i < a.n_pages; i += (int64_t) (gridDim.x - 1) * blockDim.x)
            a.shared_out[i] = a.shared[i];
        return;
    }
    bool bad = false;
    const int32_t n_free = stack_size(a.n_free, a.free_cap, bad);
    int64_t carry = 0, given = 0;
    for (int64_t b0 = 0; b0 < a.n_seq; b0 += blockDim.x) {
        const int64_t b = b0 + tid;
        const bool in = b < a.n_seq;
        const int32_t own = in ? clip_to(a.n_kv[b], a.room, bad) : 0, f = in ? a.from[b] : -1;
        bool fits = f >= 0 && f < a.n_seq && own == 0;
        int32_t n = 0, n_f = 0;
        if (fits) {
            bool dull = false;                 // (the parent's own thread reports its length)
            n_f = clip_to(a.n_kv[f], a.room, dull);
            n = a.n_tok ? a.n_tok[b] : n_f;
            fits = a.from[f] < 0 && n >= 0 && n <= n_f;
        }
        const int32_t full = fits ? n / a.page : 0, rest = fits ? n - full * a.page : 0, need = rest > 0;
        const int64_t c = carry + block_scan({need, 0}, &part[0]).x;
        const bool served = fits && (need == 0 || c <= n_free);
        bad |= f >= 0 && !served;
        if (served) given += need;
        if (in) {
            a.n_kv_out[b] = served ? n : own;
            int32_t fresh = -1, src = 0, dst = 0, cnt = 0;
            if (served && need) {
                fresh = a.free_pages[n_free - c];
                const int32_t old = a.table[(int64_t) f * a.t_stride + full];
                if (in_pool(old, a.n_pages) && in_pool(fresh, a.n_pages)) {
                    src = old * a.page;
                    dst = fresh * a.page;
                    cnt = rest;
                } else {
                    bad = true;
                }
            }
            int32_t * m = a.moves + 3 * b;
            m[0] = src; m[1] = dst; m[2] = cnt;
            if (a.state_moves) {
                int32_t s = 0, d = 0, one = 0;
                if (served && n == n_f) {
                    s = a.states ? a.states[f] : f;
                    d = a.states ? a.states[b] : (int32_t) b;
                    one = s >= 0 && d >= 0;
                    if (!one) s = d = 0;
                }
                int32_t * sm = a.state_moves + 3 * b;
                sm[0] = s; sm[1] = d; sm[2] = one;
            }
            a.req[b] = pt_req{f, full, fresh, served ? (need ? 3 : 1) : 0};
        }
        if (tid == (int) blockDim.x - 1) last = c;
        __syncthreads();
        carry = last;
        __syncthreads();
    }
    const pair64 g = block_scan({given, 0}, &part[1]);
    if (tid == (int) blockDim.x - 1) *a.n_free_out = n_free - (int32_t) g.x;
    report(a.status, bad, DEVERR_PAGES);
}

// The table rows of the forks, a workgroup each.
__global__ __launch_bounds__(SH_THREADS) void k_fork_rows(fork_args a) {
    for (int64_t b = blockIdx.x; b < a.n_seq; b += gridDim.x) {
        const pt_req r = a.req[b];
        if (!r.served) continue;
        const int32_t * src = a.table + (int64_t) r.past * a.t_stride;
        int32_t * dst = a.table + b * a.t_stride;
        bool bad = false;
        for (int32_t c = threadIdx.x; c < r.have; c += SH_THREADS) {
            const int32_t p = src[c];
            dst[c] = p;
            if (in_pool(p, a.n_pages)) atomicAdd(a.shared_out + p, 1);
            else bad = true;
        }
        if (threadIdx.x == 0 && (r.served & 2)) dst[r.have] = r.at;
        report(a.status, bad, DEVERR_PAGES);
    }
}

// ---------------------------------------------------------------- release

struct release_args {
    const int32_t * keep; const int32_t * n_kv;
    const int32_t * table; int64_t t_stride;
    const int32_t * shared; int32_t * free_pages;
    const int32_t * n_free; int32_t * n_free_out; int32_t * n_kv_out; int32_t * shared_out;
    int32_t         n_seq, page, room, n_pages, free_cap, words;
    pt_head *       head;
    pt_req *        req;               // first column given back, how many
    uint32_t *      bits;              // [words]: pages that become free
    uint32_t *      status;
};

// What each request gives back, by the counts as they are before the call; counts copied, bits cleared.
__global__ __launch_bounds__(SH_THREADS) void k_release_mark(release_args a) {
    const int64_t i0 = (int64_t) blockIdx.x * SH_THREADS + threadIdx.x, step = (int64_t) gridDim.x * SH_THREADS;
    bool bad = false;
    for (int64_t b = i0; b < a.n_seq; b += step) {
        const int32_t n = clip_to(a.n_kv[b], a.room, bad), k_in = a.keep[b];
        int32_t keep = k_in < 0 ? 0 : k_in > n ? n : k_in;
        int32_t first = (int32_t) ceil_div(keep, a.page);
        if (keep < n && keep % a.page != 0) {
            const int32_t p = a.table[b * a.t_stride + first - 1];
            if (in_pool(p, a.n_pages) && a.shared[p] > 0) {
                bad = true;
                keep = n;
                first = (int32_t) ceil_div(n, a.page);
            }
        }
        a.n_kv_out[b] = keep;
        a.req[b] = pt_req{first, (int32_t) ceil_div(n, a.page) - first, 0, 1};
    }
    for (int64_t i = i0; i < a.words; i += step) a.bits[i] = 0;
    for (int64_t i = i0; i < a.n_pages; i += step) {
        const int32_t s = a.shared[i];
        bad |= s < 0;
        if (s < 0 || a.shared_out != a.shared) a.shared_out[i] = s < 0 ? 0 : s;
    }
    if (i0 == 0) *a.head = pt_head{stack_size(a.n_free, a.free_cap, bad), 0, {0, 0}};
    report(a.status, bad, DEVERR_PAGES);
}

// A wave per request: each page that it gives back counts one less, and is free with the last of its holders. RD_BATCH pages of a
// lane are on their way together, for a step is a load and two atomics after each other (512 requests of up to 1024 pages: 14 us
// one at a time).
constexpr int RD_BATCH = 8;

__global__ __launch_bounds__(SH_THREADS) void k_release_drop(release_args a) {
    const int lane = threadIdx.x & 63;
    for (int64_t b = (int64_t) blockIdx.x * (SH_THREADS / 64) + (threadIdx.x >> 6); b < a.n_seq; b += (int64_t) gridDim.x * (SH_THREADS / 64)) {
        const pt_req r = a.req[b];
        const int32_t * src = a.table + b * a.t_stride + r.past;
        bool bad = false;
        for (int32_t c = lane; c < r.have; c += 64 * RD_BATCH) {
            int32_t p[RD_BATCH], was[RD_BATCH];
#pragma unroll
            for (int i = 0; i < RD_BATCH; i++) p[i] = src[c + 64 * i < r.have ? c + 64 * i : c];
#pragma unroll
            for (int i = 0; i < RD_BATCH; i++) {
                const bool on = c + 64 * i < r.have, ok = on && in_pool(p[i], a.n_pages);
                bad |= on && !ok;
                was[i] = 1;
                if (ok) was[i] = atomicSub(a.shared_out + p[i], 1);
            }
#pragma unroll
            for (int i = 0; i < RD_BATCH; i++) {
                if (was[i] == 0) atomicOr(a.bits + (p[i] >> 5), 1u << (p[i] & 31));
                bad |= was[i] < 0;
            }
        }
        report(a.status, bad, DEVERR_PAGES);
    }
}

// A thread per word of the bitmap; every workgroup counts the bits before its own for itself, a launch less than with their sums
// from one. The counting grows with the pool's square, which shows in pools of tens of millions: 2^24 pages, half of them given back
// by 64 requests, take 4.7 ms, 2^26 take 23.
__global__ __launch_bounds__(SH_THREADS) void k_release_push(release_args a) {
    __shared__ pair64 part[2][PT_WAVES];
    __shared__ int64_t sum;
    const int tid = threadIdx.x;
    const int64_t w0 = (int64_t) blockIdx.x * SH_THREADS;
    int64_t before = 0;
#pragma unroll 8
    for (int64_t i = tid; i < w0; i += SH_THREADS) before += __popc(a.bits[i]);
    before = block_scan({before, 0}, &part[0]).x;
    if (tid == SH_THREADS - 1) sum = before;
    __syncthreads();
    uint32_t w = w0 + tid < a.words ? a.bits[w0 + tid] : 0u;
    const int64_t end = sum + block_scan({__popc(w), 0}, &part[1]).x;
    const int32_t n_free = a.head->n_free;
    int64_t at = n_free + end - __popc(w);
    bool bad = false;
    while (w) {
        const int32_t p = (int32_t) (w0 + tid) * 32 + __builtin_ctz(w);
        w &= w - 1;
        a.shared_out[p] = 0;
        if (at < a.free_cap) a.free_pages[at] = p;
        else bad = true;
        at++;
    }
    if (blockIdx.x == gridDim.x - 1 && tid == SH_THREADS - 1)
        *a.n_free_out = (int32_t) (n_free + end < a.free_cap ? n_free + end : a.free_cap);
    report(a.status, bad, DEVERR_PAGES);
}

// ---------------------------------------------------------------- compact

struct compact_args {
    const int32_t * n_kv; const int32_t * table; int64_t t_stride;
    const int32_t * shared; const int32_t * free_pages; const int32_t * n_free;
    int32_t *       table_out; int32_t * shared_out; int32_t * free_out; int32_t * n_free_out; int32_t * page_map;
    int32_t *       moves; int32_t * n_moves;
    int32_t         n_seq, page, room, max_pages, n_pages, free_cap, words;
    pt_head *       head;              // n_free: live pages; total: moves
    uint32_t *      bits;              // [words]: free pages
    int32_t *       rank;              // [words]: free pages before the word's
    uint32_t *      status;
};

__device__ __forceinline__ bool page_free(const compact_args & a, int32_t p) { return a.bits[p >> 5] >> (p & 31) & 1; }
// free pages before p (p < n_pages)
__device__ __forceinline__ int32_t free_before(const compact_args & a, int32_t p) {
    return a.rank[p >> 5] + __popc(a.bits[p >> 5] & ((1u << (p & 31)) - 1u));
}

__global__ __launch_bounds__(SH_THREADS) void k_compact_clear(compact_args a) {
    for (int64_t i = (int64_t) blockIdx.x * SH_THREADS + threadIdx.x; i < a.words; i += (int64_t) gridDim.x * SH_THREADS) a.bits[i] = 0;
}
__global__ __launch_bounds__(SH_THREADS) void k_compact_bits(compact_args a) {
    bool bad = false;
    const int32_t n = stack_size(a.n_free, a.free_cap, bad);
    for (int64_t i = (int64_t) blockIdx.x * SH_THREADS + threadIdx.x; i < n; i += (int64_t) gridDim.x * SH_THREADS) {
        const int32_t p = a.free_pages[i];
        if (!in_pool(p, a.n_pages)) bad = true;
        else bad |= atomicOr(a.bits + (p >> 5), 1u << (p & 31)) >> (p & 31) & 1;
    }
    report(a.status, bad, DEVERR_PAGES);
}
__global__ __launch_bounds__(PT_THREADS) void k_compact_rank(compact_args a) {
    __shared__ pair64 part[PT_WAVES];
    __shared__ int32_t last, moves;
    const int tid = threadIdx.x;
    int32_t carry = 0;
    for (int64_t w0 = 0; w0 < a.words; w0 += PT_THREADS) {
        const int64_t w = w0 + tid;
        const int32_t n = w < a.words ? __popc(a.bits[w]) : 0;
        const int32_t end = carry + (int32_t) block_scan({n, 0}, &part).x;
        if (w < a.words) a.rank[w] = end - n;
        if (tid == PT_THREADS - 1) last = end;
        __syncthreads();
        carry = last;
        __syncthreads();
    }
    // the free pages below n_live
    const int32_t n_live = a.n_pages - carry;
    if (tid == 0) moves = n_live < a.n_pages ? free_before(a, n_live) : 0;
    __syncthreads();
    if (tid == 0) {
        *a.head = pt_head{n_live, moves, {0, 0}};
        *a.n_moves = moves;
        *a.n_free_out = carry;
    }
}
// A thread per page: both ends of the moves by rank, the stack, the map and the counts of pages that stay.
__global__ __launch_bounds__(SH_THREADS) void k_compact_moves(compact_args a) {
    const pt_head h = *a.head;
    const int32_t n_live = h.n_free;
    for (int64_t i = (int64_t) blockIdx.x * SH_THREADS + threadIdx.x; i < a.n_pages; i += (int64_t) gridDim.x * SH_THREADS) {
        const int32_t p = (int32_t) i;
        if (page_free(a, p)) {
            a.page_map[p] = -1;
            if (p < n_live) {
                int32_t * m = a.moves + 3 * (int64_t) free_before(a, p);
                m[1] = p * a.page;
                m[2] = a.page;
            } else {
                a.shared_out[p] = 0;
            }
        } else if (p < n_live) {
            a.page_map[p] = p;
            if (a.shared_out != a.shared) a.shared_out[p] = a.shared[p];
        } else {
            a.moves[3 * (int64_t) (p - n_live - (free_before(a, p) - h.total))] = p * a.page;
        }
        if (p < a.n_pages - n_live) a.free_out[p] = a.n_pages - 1 - p;
    }
}
// The first workgroups a request's columns each, the others the moved pages.
__global__ __launch_bounds__(SH_THREADS) void k_compact_finish(compact_args a, int32_t rows) {
    const pt_head h = *a.head;
    const int tid = threadIdx.x;
    if ((int) blockIdx.x >= rows) {
        for (int64_t k = (int64_t) ((int) blockIdx.x - rows) * SH_THREADS + tid; k < h.total; k += (int64_t) ((int) gridDim.x - rows) * SH_THREADS) {
            const int32_t s = a.moves[3 * k] / a.page, d = a.moves[3 * k + 1] / a.page;
            a.page_map[s] = d;
            a.shared_out[d] = a.shared[s];
            a.shared_out[s] = 0;
        }
        return;
    }
    bool bad = false;
    for (int64_t b = blockIdx.x; b < a.n_seq; b += rows) {
        const int32_t n = clip_to(a.n_kv[b], a.room, bad), cols = (int32_t) ceil_div(n, a.page);
        for (int32_t c = tid; c < cols; c += SH_THREADS) {
            int32_t p = a.table[b * a.t_stride + c];
            if (!in_pool(p, a.n_pages) || page_free(a, p)) {
                bad = true;
            } else if (p >= h.n_free) {
                p = a.moves[3 * (int64_t) (p - h.n_free - (free_before(a, p) - h.total)) + 1] / a.page;
            }
            a.table_out[b * a.t_stride + c] = p;
        }
    }
    report(a.status, bad, DEVERR_PAGES);
}

// ---------------------------------------------------------------- copies

struct copy_args {
    char *          cache[CP_CACHES];
    size_t          nb1;               // bytes between rows
    const int32_t * moves; const int32_t * n_moves; int32_t cap;
    int32_t         max_rows, upr;     // units of a row
    int64_t         n_rows;
    uint32_t *      status;
};

// A thread per unit of T (16 bytes where rows are whole ones) of a move's rows, blockIdx.y the tensor: every load of a
// workgroup is in flight before its first store. The units of a move with fewer than max_rows rows stay empty. They have no
// order, so a move whose rows go over each other is refused; one onto its own place is none.
template <typename T>
__global__ __launch_bounds__(SH_THREADS) void k_paged_copy(copy_args a) {
    bool bad = false;
    const int32_t n = a.n_moves ? clip_to(*a.n_moves, a.cap, bad) : a.cap;
    char * const cache = a.cache[blockIdx.y];
    const uint32_t per = (uint32_t) a.max_rows * (uint32_t) a.upr;         // below 2^31
    const int64_t total = (int64_t) n * per, step = (int64_t) gridDim.x * SH_THREADS;
    for (int64_t u0 = (int64_t) blockIdx.x * SH_THREADS; u0 < total; u0 += step) {
        const int64_t m0 = u0 / per;
        const uint32_t x = (uint32_t) (u0 - m0 * per) + threadIdx.x, k = x / per, u = x - k * per;
        const int64_t m = m0 + k;
        if (m >= n) continue;
        const int32_t s = a.moves[3 * m], d = a.moves[3 * m + 1], rows = a.moves[3 * m + 2];
        if (rows == 0) continue;
        if (rows < 0 || rows > a.max_rows || s < 0 || d < 0 || s + (int64_t) rows > a.n_rows || d + (int64_t) rows > a.n_rows ||
            (s != d && (s < d ? d - s : s - d) < rows)) {
            bad = true;
            continue;
        }
        const uint32_t r = u / (uint32_t) a.upr, c = u - r * (uint32_t) a.upr;
        if ((int32_t) r < rows && s != d)
            *(T *) (cache + (size_t) (d + r) * a.nb1 + (size_t) c * sizeof(T)) =
                *(const T *) (cache + (size_t) (s + r) * a.nb1 + (size_t) c * sizeof(T));
    }
    report(a.status, bad, DEVERR_SET_ROWS_INDEX);
}

// ---------------------------------------------------------------- trees

// A wave per request, a lane per node: masks and depths by doubling, 6 steps up to 64 nodes deep.
__global__ __launch_bounds__(SH_THREADS) void k_tree_masks(const int32_t * parents, const int32_t * n_tree, const int32_t * n_past,
                                                           int32_t n_seq, int32_t T, uint64_t * masks, int32_t * pos, uint32_t * status) {
    const int lane = threadIdx.x & 63;
    for (int64_t b = (int64_t) blockIdx.x * (SH_THREADS / 64) + (threadIdx.x >> 6); b < n_seq; b += (int64_t) gridDim.x * (SH_THREADS / 64)) {
        bool bad = false;
        const int32_t n = n_tree ? clip_to(n_tree[b], T, bad) : T;
        const bool on = lane < n;
        int32_t up = on ? parents[b * T + lane] : -1;
        if (up < -1 || up >= lane) {
            bad |= on;
            up = -1;
        }
        uint64_t mask = on ? 1ull << lane : 0ull;
        int32_t depth = up >= 0;
#pragma unroll
        for (int i = 0; i < 6; i++) {
            const int from = up >= 0 ? up : lane;
            const uint64_t m = __shfl((unsigned long long) mask, from);
            const int32_t d = __shfl(depth, from), u = __shfl(up, from);
            if (up >= 0) {
                mask |= m;
                depth += d;
                up = u;
            }
        }
        if (lane < T) {
            masks[b * T + lane] = mask;
            if (pos) pos[b * T + lane] = on ? (n_past ? n_past[b] : 0) + depth : -1;
        }
        report(status, bad, DEVERR_PAGES);
    }
}

struct accept_args {
    char *          cache[CP_CACHES];
    size_t          nb1;
    const int32_t * table; int64_t t_stride;
    const int32_t * n_kv; const int32_t * n_tree; const uint64_t * masks; const int32_t * leaf;
    int32_t *       n_keep; int32_t * cu; int32_t * path;
    int64_t         n_rows;
    int32_t         n_seq, T, page, room, n_caches, upr;
    uint32_t *      status;
};
struct tree_path { int32_t base; uint64_t bits; };

__device__ __forceinline__ tree_path path_of(const accept_args & a, int64_t b, bool & bad) {
    const int32_t n = clip_to(a.n_kv[b], a.room, bad), most = a.T < n ? a.T : n;
    const int32_t nt = a.n_tree ? clip_to(a.n_tree[b], most, bad) : most;
    const int32_t leaf = a.leaf[b];
    if (leaf < -1 || leaf >= nt) bad = true;
    if (leaf < 0 || leaf >= nt) return {n - nt, 0ull};
    const uint64_t live = nt < 64 ? (1ull << nt) - 1 : ~0ull;
    return {n - nt, a.masks[b * a.T + leaf] & live};
}

// blockIdx.y < n_caches: a wave moves a request's rows in one tensor, a lane a unit of every row, from the first accepted
// node to the last: 8 rows loaded, then stored. Row i goes to a place before row i + 1's source, so a lane that goes in this
// order never reads a unit that it has written. blockIdx.y == n_caches: lengths; its first workgroup the path lists.
constexpr int AC_AHEAD = 8;

template <typename T>
__global__ __launch_bounds__(SH_THREADS) void k_paged_accept(accept_args a) {
    __shared__ pair64 part[2][PT_WAVES];
    __shared__ int32_t last;
    const int tid = threadIdx.x, lane = tid & 63;
    bool bad = false;
    if ((int) blockIdx.y == a.n_caches) {
        if (blockIdx.x > 0) return;
        int32_t carry = 0;
        for (int64_t b0 = 0; b0 < a.n_seq; b0 += SH_THREADS) {
            const int64_t b = b0 + tid;
            tree_path p{0, 0ull};
            if (b < a.n_seq) p = path_of(a, b, bad);
            const int32_t m = __popcll(p.bits);
            if (b < a.n_seq) a.n_keep[b] = p.base + m;
            if (!a.cu) continue;
            const int32_t end = carry + (int32_t) block_scan({m, 0}, &part[0]).x;
            if (b < a.n_seq) {
                a.cu[b + 1] = end;
                if (b == 0) a.cu[0] = 0;
                int32_t at = end - m;
                if (a.path)
                    for (uint64_t w = p.bits; w; w &= w - 1) a.path[at++] = (int32_t) (b * a.T) + __builtin_ctzll(w);
            }
            if (tid == SH_THREADS - 1) last = end;
            __syncthreads();
            carry = last;
            __syncthreads();
        }
        if (a.path)
            for (int64_t i = carry + tid; i < (int64_t) a.n_seq * a.T; i += SH_THREADS) a.path[i] = 0;
        report(a.status, bad, DEVERR_PAGES);
        return;
    }
    char * const cache = a.cache[blockIdx.y];
    const int32_t n_pages = (int32_t) (a.n_rows / a.page);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int64_t b = (int64_t) blockIdx.x * (SH_THREADS / 64) + wave; b < a.n_seq; b += (int64_t) gridDim.x * (SH_THREADS / 64)) {
        bool dull = false;
        const tree_path p = path_of(a, b, dull);
        const int32_t count = __popcll(p.bits);
        // the lane's token of the tree: its row, and whether it is on the path
        int32_t row = -1;
        if (lane < a.T && (p.bits >> lane & 1 || lane < count)) {
            const int32_t token = p.base + lane, col = token / a.page, page = a.table[b * a.t_stride + col];
            if (in_pool(page, n_pages)) row = page * a.page + token - col * a.page;
            else bad = true;
        }
        uint64_t left = p.bits;
        int32_t i = 0;
        while (left && __builtin_ctzll(left) == i) {               // nodes that are where they go
            left &= left - 1;
            i++;
        }
        while (left) {
            int32_t src[AC_AHEAD], dst[AC_AHEAD];
            int n = 0;
#pragma unroll
            for (int j = 0; j < AC_AHEAD; j++) {
                src[j] = dst[j] = -1;
                if (left) {
                    src[j] = __builtin_amdgcn_readlane(row, __builtin_ctzll(left));
                    dst[j] = __builtin_amdgcn_readlane(row, i + j);
                    left &= left - 1;
                    n++;
                }
            }
            i += n;
            for (int32_t c = lane; c < a.upr; c += 64) {
                T x[AC_AHEAD];
#pragma unroll
                for (int j = 0; j < AC_AHEAD; j++)         // (row 0 where there is none to load: no branch stands between the loads)
                    x[j] = *(const T *) (cache + (size_t) (src[j] < 0 ? 0 : src[j]) * a.nb1 + (size_t) c * sizeof(T));
#pragma unroll
                for (int j = 0; j < AC_AHEAD; j++)
                    if (src[j] >= 0 && dst[j] >= 0) *(T *) (cache + (size_t) dst[j] * a.nb1 + (size_t) c * sizeof(T)) = x[j];
            }
        }
    }
    report(a.status, bad, DEVERR_PAGES);
}

// ---------------------------------------------------------------- host

// What _fork, _release and _compact check alike; `need` the workspace's bytes.
int check_pool(const char * op, int32_t n_seq, int32_t page_size, int64_t table_stride, int32_t max_pages, int32_t n_pages,
               int32_t free_cap, const void * ws, size_t ws_bytes, size_t need, const char * size_fn) {
    const std::string o(op);
    if (int rc = check_tables(op, n_seq, page_size, table_stride, max_pages, free_cap, ws, SIZE_MAX)) return rc;
    if (n_pages < 1 || (int64_t) n_pages * page_size > 0x7fffffff)
        return set_error(QWFN_EINVAL, o + ": n_pages must be positive, n_pages * page_size below 2^31");
    if (ws_bytes < need) return set_error(QWFN_ENOMEM, o + ": ws must hold " + size_fn + " bytes");
    return QWFN_OK;
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }
int64_t words_of(int32_t n_pages) { return ((int64_t) n_pages + 31) / 32; }
unsigned grid_for(int64_t n, int64_t per) { return (unsigned) std::max<int64_t>(1, std::min<int64_t>((n + per - 1) / per, SH_MAX_GRID)); }

// Bytes from a tensor's first row to behind its last.
size_t view_bytes_rows(const qwfn_tensor & t, size_t row) { return (size_t) (t.ne[1] - 1) * t.nb[1] + row; }

// The tensors whose rows a call moves: one type, shape and stride, rows contiguous, none over another.
struct row_set { size_t row, nb1; int64_t n_rows; size_t unit; };
int check_caches(const char * op, const qwfn_tensor * caches, int32_t n_caches, row_set * out) {
    const std::string o(op);
    if (n_caches < 0 || (n_caches > 0 && !caches)) return set_error(QWFN_EINVAL, o + ": caches is NULL or n_caches negative");
    *out = row_set{0, 0, 0, 16};
    for (int32_t i = 0; i < n_caches; i++) {
        const qwfn_tensor & t = caches[i], & f = caches[0];
        if (!t.data) return set_error(QWFN_EINVAL, o + ": a cache is NULL");
        const size_t es = t.type == QWFN_TYPE_BF16 ? 2 : type_size(t.type);
        const int64_t blk = type_blck(t.type);
        if (es == 0) return set_error(QWFN_EINVAL, o + ": caches must be f32, f16, bf16, i32 or q8_0");
        if (t.ne[0] < 1 || t.ne[1] < 1 || t.ne[2] != 1 || t.ne[3] != 1 || t.ne[0] % blk)
            return set_error(QWFN_EINVAL, o + ": caches must be [ne0, n_rows]");
        if (t.ne[0] > INT64_C(1) << 40 || t.ne[1] > 0x7fffffff) return set_error(QWFN_ENOTSUP, o + ": at most 2^31 - 1 rows of 2^40 values");
        const size_t row = (size_t) (t.ne[0] / blk) * es;
        if (t.nb[0] != es) return set_error(QWFN_EINVAL, o + ": cache rows must be contiguous");
        if (t.ne[1] > 1 && t.nb[1] < row) return set_error(QWFN_EINVAL, o + ": cache rows overlap");
        if (t.type != f.type || t.ne[0] != f.ne[0] || t.ne[1] != f.ne[1] || t.nb[1] != f.nb[1])
            return set_error(QWFN_EINVAL, o + ": caches must have one type, shape and row stride");
        *out = row_set{row, t.nb[1], t.ne[1], out->unit};
        while (out->unit > 2 && (!is_aligned(t.data, out->unit) || t.nb[1] % out->unit || row % out->unit)) out->unit /= out->unit == 16 ? 4 : 2;
        if (!is_aligned(t.data, out->unit) || t.nb[1] % out->unit || row % out->unit)
            return set_error(QWFN_EALIGN, o + ": caches and their rows must be 2-byte aligned");
        for (int32_t j = 0; j < i; j++)
            if (overlaps(t.data, view_bytes_rows(t, row), caches[j].data, view_bytes_rows(caches[j], row)))
                return set_error(QWFN_EINVAL, o + ": caches overlap");
    }
    if (n_caches > 0 && out->row / out->unit > 0x3fffffff) return set_error(QWFN_ENOTSUP, o + ": rows too long");
    return QWFN_OK;
}

}  // namespace
}  // namespace qwfn

using namespace qwfn;

extern "C" int qwfn_paged_fork(const int32_t * from, const int32_t * n_tok, const int32_t * n_kv, int32_t n_seq,
                               int32_t page_size, int32_t * table, int64_t table_stride, int32_t max_pages,
                               const int32_t * shared, int32_t n_pages, const int32_t * free_pages, int32_t free_cap,
                               const int32_t * n_free, int32_t * n_free_out, int32_t * n_kv_out, int32_t * shared_out,
                               int32_t * moves, const int32_t * states, int32_t * state_moves, void * ws, size_t ws_bytes,
                               void * stream) {
    return ::qwfn::abi_call("paged_fork", [&]() -> int {
        if (!from || !n_kv || !table || !shared || !free_pages || !n_free || !n_free_out || !n_kv_out || !shared_out || !moves)
            return set_error(QWFN_EINVAL, "paged_fork: NULL pointer");
        const size_t need = qwfn_paged_workspace_size(n_seq);
        if (int rc = check_pool("paged_fork", n_seq, page_size, table_stride, max_pages, n_pages, free_cap, ws, ws_bytes, need,
                                "qwfn_paged_workspace_size")) return rc;
        const size_t per = (size_t) n_seq * 4, tab = ((size_t) (n_seq - 1) * table_stride + max_pages) * 4, pg = (size_t) n_pages * 4;
        const span in[] = {{from, per, "from"}, {n_tok, per, "n_tok"}, {n_kv_out == n_kv ? nullptr : n_kv, per, "n_kv"},
                           {shared_out == shared ? nullptr : shared, pg, "shared"}, {free_pages, (size_t) free_cap * 4, "free_pages"},
                           {n_free_out == n_free ? nullptr : n_free, 4, "n_free"}, {states, per, "states"}};
        const span out[] = {{table, tab, "table"}, {n_free_out, 4, "n_free_out"}, {n_kv_out, per, "n_kv_out"},
                            {shared_out, pg, "shared_out"}, {moves, 3 * per, "moves"}, {state_moves, 3 * per, "state_moves"},
                            {ws, need, "ws"}};
        if (int rc = check_spans("paged_fork", in, 7, out, 7)) return rc;
        fork_args a{};
        if (int rc = status_word(&a.status)) return rc;
        a.from = from; a.n_tok = n_tok; a.n_kv = n_kv; a.table = table; a.t_stride = table_stride; a.shared = shared;
        a.free_pages = free_pages; a.n_free = n_free; a.n_free_out = n_free_out; a.n_kv_out = n_kv_out; a.shared_out = shared_out;
        a.moves = moves; a.states = states; a.state_moves = state_moves;
        a.n_seq = n_seq; a.page = page_size; a.room = max_pages * page_size; a.n_pages = n_pages; a.free_cap = free_cap;
        a.req = (pt_req *) ((char *) ws + sizeof(pt_head));
        const int threads = scan_threads(n_seq);
        const unsigned copy = shared_out == shared ? 0 : grid_for(n_pages, 4 * threads);
        hipLaunchKernelGGL(k_fork_scan, dim3(1 + copy), dim3(threads), 0, as_stream(stream), a);
        if (int rc = hip_check(hipGetLastError(), "paged_fork launch")) return rc;
        hipLaunchKernelGGL(k_fork_rows, dim3(grid_for(n_seq, 1)), dim3(SH_THREADS), 0, as_stream(stream), a);
        return hip_check(hipGetLastError(), "paged_fork launch");
    });
}

extern "C" size_t qwfn_paged_release_workspace_size(int32_t n_seq, int32_t n_pages) {
    const size_t req = qwfn_paged_workspace_size(n_seq);
    return req == 0 || n_pages < 1 ? 0 : round16(req) + (size_t) words_of(n_pages) * 4;
}

extern "C" int qwfn_paged_release(const int32_t * n_keep, const int32_t * n_kv, int32_t n_seq, int32_t page_size,
                                  const int32_t * table, int64_t table_stride, int32_t max_pages, const int32_t * shared,
                                  int32_t n_pages, int32_t * free_pages, int32_t free_cap, const int32_t * n_free,
                                  int32_t * n_free_out, int32_t * n_kv_out, int32_t * shared_out, void * ws, size_t ws_bytes,
                                  void * stream) {
    return ::qwfn::abi_call("paged_release", [&]() -> int {
        if (!n_keep || !n_kv || !table || !shared || !free_pages || !n_free || !n_free_out || !n_kv_out || !shared_out)
            return set_error(QWFN_EINVAL, "paged_release: NULL pointer");
        const size_t need = qwfn_paged_release_workspace_size(n_seq, n_pages);
        if (int rc = check_pool("paged_release", n_seq, page_size, table_stride, max_pages, n_pages, free_cap, ws, ws_bytes, need,
                                "qwfn_paged_release_workspace_size")) return rc;
        if (free_cap < n_pages) return set_error(QWFN_EINVAL, "paged_release: free_cap must be at least n_pages");
        const size_t per = (size_t) n_seq * 4, tab = ((size_t) (n_seq - 1) * table_stride + max_pages) * 4, pg = (size_t) n_pages * 4;
        const span in[] = {{n_keep, per, "n_keep"}, {n_kv_out == n_kv ? nullptr : n_kv, per, "n_kv"}, {table, tab, "table"},
                           {shared_out == shared ? nullptr : shared, pg, "shared"}, {n_free_out == n_free ? nullptr : n_free, 4, "n_free"}};
        const span out[] = {{free_pages, (size_t) free_cap * 4, "free_pages"}, {n_free_out, 4, "n_free_out"},
                            {n_kv_out, per, "n_kv_out"}, {shared_out, pg, "shared_out"}, {ws, need, "ws"}};
        if (int rc = check_spans("paged_release", in, 5, out, 5)) return rc;
        release_args a{};
        if (int rc = status_word(&a.status)) return rc;
        a.keep = n_keep; a.n_kv = n_kv; a.table = table; a.t_stride = table_stride; a.shared = shared; a.free_pages = free_pages;
        a.n_free = n_free; a.n_free_out = n_free_out; a.n_kv_out = n_kv_out; a.shared_out = shared_out;
        a.n_seq = n_seq; a.page = page_size; a.room = max_pages * page_size; a.n_pages = n_pages; a.free_cap = free_cap;
        a.words = (int32_t) words_of(n_pages);
        a.head = (pt_head *) ws; a.req = (pt_req *) ((char *) ws + sizeof(pt_head));
        a.bits = (uint32_t *) ((char *) ws + round16(qwfn_paged_workspace_size(n_seq)));
        const hipStream_t s = as_stream(stream);
        hipLaunchKernelGGL(k_release_mark, dim3(grid_for(std::max(n_seq, n_pages), SH_THREADS)), dim3(SH_THREADS), 0, s, a);
        if (int rc = hip_check(hipGetLastError(), "paged_release launch")) return rc;
        hipLaunchKernelGGL(k_release_drop, dim3(grid_for(n_seq, SH_THREADS / 64)), dim3(SH_THREADS), 0, s, a);
        if (int rc = hip_check(hipGetLastError(), "paged_release launch")) return rc;
        hipLaunchKernelGGL(k_release_push, dim3((unsigned) ((a.words + SH_THREADS - 1) / SH_THREADS)), dim3(SH_THREADS), 0, s, a);
        return hip_check(hipGetLastError(), "paged_release launch");
    });
}

extern "C" size_t qwfn_paged_compact_workspace_size(int32_t n_pages) {
    return n_pages < 1 ? 0 : sizeof(pt_head) + 2 * round16((size_t) words_of(n_pages) * 4);
}

extern "C" int qwfn_paged_compact(const int32_t * n_kv, int32_t n_seq, int32_t page_size, const int32_t * table,
                                  int64_t table_stride, int32_t max_pages, const int32_t * shared, int32_t n_pages,
                                  const int32_t * free_pages, int32_t free_cap, const int32_t * n_free, int32_t * table_out,
                                  int32_t * shared_out, int32_t * free_out, int32_t * n_free_out, int32_t * page_map,
                                  int32_t * moves, int32_t * n_moves, void * ws, size_t ws_bytes, void * stream) {
    return ::qwfn::abi_call("paged_compact", [&]() -> int {
        if (!n_kv || !table || !shared || !free_pages || !n_free || !table_out || !shared_out || !free_out || !n_free_out ||
            !page_map || !moves || !n_moves)
            return set_error(QWFN_EINVAL, "paged_compact: NULL pointer");
        const size_t need = qwfn_paged_compact_workspace_size(n_pages);
        if (int rc = check_pool("paged_compact", n_seq, page_size, table_stride, max_pages, n_pages, free_cap, ws, ws_bytes, need,
                                "qwfn_paged_compact_workspace_size")) return rc;
        if (free_cap < n_pages) return set_error(QWFN_EINVAL, "paged_compact: free_cap must be at least n_pages");
        const size_t per = (size_t) n_seq * 4, tab = ((size_t) (n_seq - 1) * table_stride + max_pages) * 4, pg = (size_t) n_pages * 4;
        const size_t cap = (size_t) free_cap * 4, mv = ((size_t) n_pages + 1) / 2 * 12;
        const span in[] = {{n_kv, per, "n_kv"}, {table_out == table ? nullptr : table, tab, "table"},
                           {shared_out == shared ? nullptr : shared, pg, "shared"},
                           {free_out == free_pages ? nullptr : free_pages, cap, "free_pages"},
                           {n_free_out == n_free ? nullptr : n_free, 4, "n_free"}};
        const span out[] = {{table_out, tab, "table_out"}, {shared_out, pg, "shared_out"}, {free_out, cap, "free_out"},
                            {n_free_out, 4, "n_free_out"}, {page_map, pg, "page_map"}, {moves, mv, "moves"},
                            {n_moves, 4, "n_moves"}, {ws, need, "ws"}};
        if (int rc = check_spans("paged_compact", in, 5, out, 8)) return rc;
        compact_args a{};
        if (int rc = status_word(&a.status)) return rc;
        a.n_kv = n_kv; a.table = table; a.t_stride = table_stride; a.shared = shared; a.free_pages = free_pages; a.n_free = n_free;
        a.table_out = table_out; a.shared_out = shared_out; a.free_out = free_out; a.n_free_out = n_free_out; a.page_map = page_map;
        a.moves = moves; a.n_moves = n_moves;
        a.n_seq = n_seq; a.page = page_size; a.room = max_pages * page_size; a.max_pages = max_pages; a.n_pages = n_pages;
        a.free_cap = free_cap; a.words = (int32_t) words_of(n_pages);
        a.head = (pt_head *) ws; a.bits = (uint32_t *) ((char *) ws + sizeof(pt_head));
        a.rank = (int32_t *) ((char *) a.bits + round16((size_t) a.words * 4));
        const hipStream_t s = as_stream(stream);
        hipLaunchKernelGGL(k_compact_clear, dim3(grid_for(a.words, SH_THREADS)), dim3(SH_THREADS), 0, s, a);
        if (int rc = hip_check(hipGetLastError(), "paged_compact launch")) return rc;
        hipLaunchKernelGGL(k_compact_bits, dim3(grid_for(n_pages, SH_THREADS)), dim3(SH_THREADS), 0, s, a);
        if (int rc = hip_check(hipGetLastError(), "paged_compact launch")) return rc;
        hipLaunchKernelGGL(k_compact_rank, dim3(1), dim3(PT_THREADS), 0, s, a);
        if (int rc = hip_check(hipGetLastError(), "paged_compact launch")) return rc;
        hipLaunchKernelGGL(k_compact_moves, dim3(grid_for(n_pages, SH_THREADS)), dim3(SH_THREADS), 0, s, a);
        if (int rc = hip_check(hipGetLastError(), "paged_compact launch")) return rc;
        const unsigned rows = grid_for(n_seq, 1);
        hipLaunchKernelGGL(k_compact_finish, dim3(rows + grid_for((n_pages + 1) / 2, SH_THREADS)), dim3(SH_THREADS), 0, s, a, (int32_t) rows);
        return hip_check(hipGetLastError(), "paged_compact launch");
    });
}

extern "C" int qwfn_paged_copy(const qwfn_tensor * caches, int32_t n_caches, const int32_t * moves, int32_t cap,
                               const int32_t * n_moves, int32_t max_rows, void * stream) {
    return ::qwfn::abi_call("paged_copy", [&]() -> int {
        row_set rs;
        if (int rc = check_caches("paged_copy", caches, n_caches, &rs)) return rc;
        if (cap < 0 || (cap > 0 && !moves)) return set_error(QWFN_EINVAL, "paged_copy: moves is NULL or cap negative");
        if (max_rows < 1) return set_error(QWFN_EINVAL, "paged_copy: max_rows must be positive");
        if (!is_aligned(moves, 4) || !is_aligned(n_moves, 4)) return set_error(QWFN_EALIGN, "paged_copy: moves and n_moves must be 4-byte aligned");
        if (n_caches == 0 || cap == 0) return QWFN_OK;
        if ((int64_t) max_rows * (int64_t) (rs.row / rs.unit) > 0x7fffff00) return set_error(QWFN_ENOTSUP, "paged_copy: max_rows rows of 2^31 units or more");
        for (int32_t i = 0; i < n_caches; i++) {
            const span in[] = {{moves, (size_t) cap * 12, "moves"}, {n_moves, 4, "n_moves"}};
            const span out[] = {{caches[i].data, view_bytes_rows(caches[i], rs.row), "a cache"}};
            if (int rc = check_overlaps("paged_copy", in, 2, out, 1)) return rc;
        }
        copy_args a{};
        if (int rc = status_word(&a.status)) return rc;
        a.nb1 = rs.nb1; a.moves = moves; a.n_moves = n_moves; a.cap = cap; a.max_rows = max_rows; a.n_rows = rs.n_rows;
        a.upr = (int32_t) (rs.row / rs.unit);
        for (int32_t c0 = 0; c0 < n_caches; c0 += CP_CACHES) {
            const int n = std::min(n_caches - c0, CP_CACHES);
            for (int i = 0; i < n; i++) a.cache[i] = (char *) caches[c0 + i].data;
            const int64_t units = (int64_t) cap * max_rows * a.upr;
            const int64_t most = std::max<int64_t>(1, SH_MAX_GRID / n);
            const dim3 grid((unsigned) std::min<int64_t>((units + SH_THREADS - 1) / SH_THREADS, most), (unsigned) n), blk(SH_THREADS);
            if (rs.unit == 16)     hipLaunchKernelGGL(k_paged_copy<unit16>, grid, blk, 0, as_stream(stream), a);
            else if (rs.unit == 4) hipLaunchKernelGGL(k_paged_copy<uint32_t>, grid, blk, 0, as_stream(stream), a);
            else                   hipLaunchKernelGGL(k_paged_copy<uint16_t>, grid, blk, 0, as_stream(stream), a);
            if (int rc = hip_check(hipGetLastError(), "paged_copy launch")) return rc;
        }
        return QWFN_OK;
    });
}

extern "C" int qwfn_tree_masks(const int32_t * parents, const int32_t * n_tree, const int32_t * n_past, int32_t n_seq, int32_t T,
                               uint64_t * masks, int32_t * pos, void * stream) {
    return ::qwfn::abi_call("tree_masks", [&]() -> int {
        if (!parents || !masks) return set_error(QWFN_EINVAL, "tree_masks: NULL pointer");
        if (n_seq < 1 || n_seq > PT_MAX_SEQ) return set_error(QWFN_EINVAL, "tree_masks: n_seq must lie in [1, 65536]");
        if (T < 1 || T > 64) return set_error(QWFN_ENOTSUP, "tree_masks: T must lie in [1, 64]");
        if (!is_aligned(masks, 8)) return set_error(QWFN_EALIGN, "tree_masks: masks must be 8-byte aligned");
        const size_t per = (size_t) n_seq * 4;
        const span in[] = {{parents, per * T, "parents"}, {n_tree, per, "n_tree"}, {n_past, per, "n_past"}};
        const span out[] = {{masks, 2 * per * T, "masks"}, {pos, per * T, "pos"}};
        if (int rc = check_spans("tree_masks", in, 3, out, 2)) return rc;
        uint32_t * status = nullptr;
        if (int rc = status_word(&status)) return rc;
        hipLaunchKernelGGL(k_tree_masks, dim3(grid_for(n_seq, SH_THREADS / 64)), dim3(SH_THREADS), 0, as_stream(stream), parents, n_tree,
                           n_past, n_seq, T, masks, pos, status);
        return hip_check(hipGetLastError(), "tree_masks launch");
    });
}

extern "C" int qwfn_paged_accept(const qwfn_tensor * caches, int32_t n_caches, const int32_t * table, int64_t table_stride,
                                 int32_t max_pages, int32_t page_size, const int32_t * n_kv, const int32_t * n_tree,
                                 const uint64_t * masks, const int32_t * leaf, int32_t n_seq, int32_t T, int32_t * n_keep,
                                 int32_t * cu_path, int32_t * path, void * stream) {
    return ::qwfn::abi_call("paged_accept", [&]() -> int {
        row_set rs;
        if (int rc = check_caches("paged_accept", caches, n_caches, &rs)) return rc;
        if (n_caches > CP_CACHES) return set_error(QWFN_ENOTSUP, "paged_accept: at most 64 caches");
        if (!table || !n_kv || !masks || !leaf || !n_keep) return set_error(QWFN_EINVAL, "paged_accept: NULL pointer");
        if (path && !cu_path) return set_error(QWFN_EINVAL, "paged_accept: path without cu_path");
        if (T < 1 || T > 64) return set_error(QWFN_ENOTSUP, "paged_accept: T must lie in [1, 64]");
        if (int rc = check_table_shape("paged_accept", n_seq, page_size, table_stride, max_pages)) return rc;
        if (!is_aligned(masks, 8)) return set_error(QWFN_EALIGN, "paged_accept: masks must be 8-byte aligned");
        const size_t per = (size_t) n_seq * 4, tab = ((size_t) (n_seq - 1) * table_stride + max_pages) * 4;
        const span in[] = {{table, tab, "table"}, {n_kv, per, "n_kv"}, {n_tree, per, "n_tree"}, {masks, 2 * per * T, "masks"},
                           {leaf, per, "leaf"}};
        const span out[] = {{n_keep, per, "n_keep"}, {cu_path, per + 4, "cu_path"}, {path, per * T, "path"}};
        if (int rc = check_spans("paged_accept", in, 5, out, 3)) return rc;
        for (int32_t i = 0; i < n_caches; i++) {
            const span all[] = {in[0], in[1], in[2], in[3], in[4], out[0], out[1], out[2]};
            const span one[] = {{caches[i].data, view_bytes_rows(caches[i], rs.row), "a cache"}};
            if (int rc = check_overlaps("paged_accept", all, 8, one, 1)) return rc;
        }
        accept_args a{};
        if (int rc = status_word(&a.status)) return rc;
        for (int32_t i = 0; i < n_caches; i++) a.cache[i] = (char *) caches[i].data;
        a.nb1 = rs.nb1; a.n_rows = rs.n_rows; a.upr = (int32_t) (rs.row / rs.unit);
        a.table = table; a.t_stride = table_stride; a.n_kv = n_kv; a.n_tree = n_tree; a.masks = masks; a.leaf = leaf;
        a.n_keep = n_keep; a.cu = cu_path; a.path = path;
        a.n_seq = n_seq; a.T = T; a.page = page_size; a.room = max_pages * page_size; a.n_caches = n_caches;
        const dim3 grid(grid_for(n_seq, SH_THREADS / 64), (unsigned) n_caches + 1), blk(SH_THREADS);
        if (rs.unit == 16)     hipLaunchKernelGGL(k_paged_accept<unit16>, grid, blk, 0, as_stream(stream), a);
        else if (rs.unit == 4) hipLaunchKernelGGL(k_paged_accept<uint32_t>, grid, blk, 0, as_stream(stream), a);
        else                   hipLaunchKernelGGL(k_paged_accept<uint16_t>, grid, blk, 0, as_stream(stream), a);
        return hip_check(hipGetLastError(), "paged_accept launch");
    });
}
