// Page tables of the paged KV cache, built on the GPU from request lengths:
// qwfn_paged_extend hands out pages and lists the new tokens' cache rows,
// qwfn_paged_trim takes pages back. With P tokens a page:
//   have = ceil(past / P), need = ceil((past + new) / P) - have
//   c = inclusive sum of need over the requests; the i-th page of request b is
//   free[n_free - 1 - (c_b - need_b + i)]
//   token t of request b: p = past_b + t, row table[b][p / P] * P + p % P
// and back: back = ceil(n_kv / P) - ceil(keep / P), to free[n_free + (sum of back
// before b) + i].
//
// A few KB to a MB move, so the calls are bound by launches and the chain load ->
// scan -> store, not by bytes. The prefix sums need every request. In place
// (lengths, the stack's size) one workgroup has to have read everything before it
// writes: k_extend_scan / k_trim_scan, whose results k_extend_lists / k_trim_pages use
// in a second launch. The scan writes the lists of a decoding step itself (a thread per
// request for the first tokens, a wave together for the rest), up to EXT_FEW tokens a
// request on average: 256 requests with one token each 4.2 us, one launch. Not in place,
// up to 1024 requests, every workgroup makes the sums for itself and one launch does
// (k_extend_once, k_trim_once): 24 prompts of 50000 tokens together 4.0 us for 6.3, 512
// requests of which 102 give back all their pages 4.4 for 6.9, and 3 us less of the
// host's time a call.
#include "qwfn_common.h"
#include "qwfn_paged.h"

#include <algorithm>

namespace qwfn {
namespace {

constexpr int PT_THREADS = 1024;       // of a scan
constexpr int PT_WAVES   = PT_THREADS / 64;
constexpr int EXT_FEW    = 8;          // tokens a request, on average, that the scan's workgroup still writes itself
constexpr int ROW_THREADS = 256;       // of the second launches
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

struct ext_args {
    const int32_t * past; const int32_t * fresh;
    int32_t *       table; int64_t t_stride;
    const int32_t * free_pages; int32_t free_cap;
    const int32_t * n_free; int32_t * n_free_out;
    int32_t *       n_kv; int32_t * cu; int32_t * slots; int32_t * pos; int32_t * seq;
    int64_t         n_tok;
    int32_t         n_seq, page, max_pages, pad_slot;
    int32_t         lists;             // the scan writes the lists and the table
    const int32_t * states; int32_t * state_slots;        // NULL: slot b; not wanted
    pt_head *       head;
    pt_req *        req;
    uint32_t *      status;
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

// Entry i of the lists: token t of request b. The first token of a new page writes its column.
__device__ __forceinline__ void list_token(const ext_args & a, int64_t i, int32_t b, const pt_req & r, int32_t n_free, int64_t t) {
    int32_t slot = a.pad_slot, pos = -1;
    if (r.served) {
        const uint32_t p = (uint32_t) (r.past + t), c = p / (uint32_t) a.page, at = p - c * (uint32_t) a.page;
        int32_t * entry = a.table + (int64_t) b * a.t_stride + c;
        int32_t page;
        if ((int32_t) c >= r.have) {
            page = a.free_pages[n_free - 1 - (r.at + ((int32_t) c - r.have))];
            if (at == 0) *entry = page;
        } else {
            page = *entry;
        }
        if (page >= 0 && (int64_t) page * a.page + at <= 0x7fffffff) {
            slot = page * a.page + (int32_t) at;
            pos = (int32_t) p;
        } else {
            atomicOr(a.status, DEVERR_PAGES);
        }
    }
    a.slots[i] = slot;
    if (a.pos) a.pos[i] = pos;
    if (a.seq) a.seq[i] = b;
}

// The stack's size, clipped.
__device__ __forceinline__ int32_t stack_size(const int32_t * n_free, int32_t cap, bool & bad) {
    const int32_t n = *n_free, x = n < 0 ? 0 : n > cap ? cap : n;
    bad |= x != n;
    return x;
}

// Request b's entry of state_slots: its slot, or -2 - its slot where the step adds nothing to its state. A negative slot is
// none to mark.
__device__ __forceinline__ void put_state(const ext_args & a, int64_t b, bool runs) {
    if (!a.state_slots) return;
    const int32_t s = a.states ? a.states[b] : (int32_t) b;
    a.state_slots[b] = s < 0 || runs ? s : (int32_t) (0xfffffffeu - (uint32_t) s);
}

// Request b, a thread each, behind requests whose new tokens and needs sum to `before`.
struct ext_sums { pt_req r; int64_t total, cu0, cu1, need, c; };
__device__ __forceinline__ ext_sums extend_sums(const ext_args & a, int64_t b, int32_t n_free, pair64 before,
                                                pair64 (*part)[PT_WAVES], bool & bad) {
    const bool in = b < a.n_seq;
    const int32_t past_in = in ? a.past[b] : 0, new_in = in ? a.fresh[b] : 0;
    const int32_t past = past_in < 0 ? 0 : past_in, fresh = new_in < 0 ? 0 : new_in;
    bad |= past != past_in || fresh != new_in;
    ext_sums x;
    x.total = (int64_t) past + fresh;
    const int64_t have = ceil_div(past, a.page);
    // the lists first: a request's tokens have to lie below n_tok
    x.cu1 = before.x + block_scan({fresh, 0}, &part[0]).x;
    x.cu0 = x.cu1 - fresh;
    const bool fits = x.total <= (int64_t) a.max_pages * a.page && x.cu1 <= a.n_tok;
    x.need = in && fits ? ceil_div(x.total, a.page) - have : 0;
    x.c = before.y + block_scan({x.need, 0}, &part[1]).x;
    x.r = {past, (int32_t) have, (int32_t) (x.c - x.need < INT32_MAX ? x.c - x.need : INT32_MAX), in && fits && (x.need == 0 || x.c <= n_free)};
    bad |= in && !x.r.served;
    return x;
}

__global__ __launch_bounds__(PT_THREADS) void k_extend_scan(ext_args a) {
    __shared__ pair64 part[2][PT_WAVES];
    __shared__ pair64 last;
    const int tid = threadIdx.x, lane = tid & 63;
    bool bad = false;
    const int32_t n_free = stack_size(a.n_free, a.free_cap, bad);
    pair64 carry{0, 0};
    int64_t given = 0;                       // pages handed out by this thread's requests
    for (int64_t b0 = 0; b0 < a.n_seq; b0 += blockDim.x) {
        const int64_t b = b0 + tid;
        const bool in = b < a.n_seq;
        const ext_sums x = extend_sums(a, b, n_free, carry, part, bad);
        const pt_req r = x.r;
        const int64_t cu0 = x.cu0, cu1 = x.cu1;
        if (in) {
            if (r.served) given += x.need;
            a.n_kv[b] = r.served ? (int32_t) x.total : r.past;
            put_state(a, b, r.served && cu1 > cu0);
            if (b == 0) a.cu[0] = 0;
            a.cu[b + 1] = (int32_t) (cu1 < a.n_tok ? cu1 : a.n_tok);
            a.req[b] = r;
        }
        if (a.lists) {
            // each thread the first tokens of its request, then the waves the rest together
            const int64_t end = cu1 < a.n_tok ? cu1 : a.n_tok;
            const int64_t n = in && cu0 < end ? end - cu0 : 0;
            for (int64_t t = 0; t < n && t < 4; t++) list_token(a, cu0 + t, (int32_t) b, r, n_free, t);
            uint64_t more = __ballot(n > 4);
            while (more) {
                const int src = __builtin_ctzll(more);
                more &= more - 1;
                const pt_req q{__shfl(r.past, src), __shfl(r.have, src), __shfl(r.at, src), __shfl(r.served, src)};
                const int64_t at = __shfl((long long) cu0, src), cnt = __shfl((long long) n, src);
                const int32_t bs = (int32_t) (b - lane + src);
                for (int64_t t = 4 + lane; t < cnt; t += 64) list_token(a, at + t, bs, q, n_free, t);
            }
        }
        // the running sums: the last thread's
        if (tid == (int) blockDim.x - 1) last = {cu1, x.c};
        __syncthreads();
        carry = last;
        __syncthreads();
    }
    const int64_t listed = carry.x < a.n_tok ? carry.x : a.n_tok;
    if (a.lists)
        for (int64_t i = listed + tid; i < a.n_tok; i += blockDim.x) {
            a.slots[i] = a.pad_slot;
            if (a.pos) a.pos[i] = -1;
            if (a.seq) a.seq[i] = -1;
        }
    const pair64 g = block_scan({given, 0}, &part[0]);
    if (tid == (int) blockDim.x - 1) {
        *a.n_free_out = n_free - (int32_t) g.x;
        *a.head = pt_head{n_free, (int32_t) listed, {0, 0}};
    }
    if (__ballot(bad) && lane == 0) atomicOr(a.status, DEVERR_PAGES);
}

// A thread per token: its request by bisection of cu_new.
__global__ __launch_bounds__(ROW_THREADS) void k_extend_lists(ext_args a) {
    const int64_t i = (int64_t) blockIdx.x * ROW_THREADS + threadIdx.x;
    if (i >= a.n_tok) return;
    const pt_head h = *a.head;
    if (i >= h.total) {
        a.slots[i] = a.pad_slot;
        if (a.pos) a.pos[i] = -1;
        if (a.seq) a.seq[i] = -1;
        return;
    }
    int32_t lo = 0, hi = a.n_seq - 1;        // the last request whose list starts at or before i
    while (lo < hi) {
        const int32_t mid = (lo + hi + 1) >> 1;
        if (a.cu[mid] <= i) lo = mid;
        else hi = mid - 1;
    }
    list_token(a, i, lo, a.req[lo], h.n_free, i - a.cu[lo]);
}

// Both in one launch, for lengths and a stack size that are not updated in place: every workgroup has the sums of all
// requests for itself, the first writes the lengths, and a thread takes a token.
__global__ __launch_bounds__(PT_THREADS) void k_extend_once(ext_args a) {
    __shared__ pair64 part[2][PT_WAVES];
    __shared__ pt_req req[PT_THREADS];
    __shared__ int32_t cu[PT_THREADS + 1];
    const int tid = threadIdx.x;
    bool bad = false;
    const int32_t n_free = stack_size(a.n_free, a.free_cap, bad);
    const ext_sums x = extend_sums(a, tid, n_free, {0, 0}, part, bad);
    const int32_t end = (int32_t) (x.cu1 < a.n_tok ? x.cu1 : a.n_tok);
    if (tid == 0) cu[0] = 0;
    cu[tid + 1] = end;
    req[tid] = x.r;
    if (blockIdx.x == 0) {
        if (tid < a.n_seq) {
            a.n_kv[tid] = x.r.served ? (int32_t) x.total : x.r.past;
            put_state(a, tid, x.r.served && x.cu1 > x.cu0);
            if (tid == 0) a.cu[0] = 0;
            a.cu[tid + 1] = end;
        }
        const pair64 g = block_scan({x.r.served ? x.need : 0, 0}, &part[0]);
        if (tid == (int) blockDim.x - 1) *a.n_free_out = n_free - (int32_t) g.x;
        if (__ballot(bad) && (tid & 63) == 0) atomicOr(a.status, DEVERR_PAGES);
    }
    __syncthreads();
    const int32_t listed = cu[a.n_seq];
    const int64_t i = (int64_t) blockIdx.x * blockDim.x + tid;
    if (i >= a.n_tok) return;
    if (i >= listed) {
        a.slots[i] = a.pad_slot;
        if (a.pos) a.pos[i] = -1;
        if (a.seq) a.seq[i] = -1;
        return;
    }
    int32_t lo = 0, hi = a.n_seq - 1;
    while (lo < hi) {
        const int32_t mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= i) lo = mid;
        else hi = mid - 1;
    }
    list_token(a, i, lo, req[lo], n_free, i - cu[lo]);
}

struct trim_args {
    const int32_t * keep; const int32_t * n_kv;
    const int32_t * table; int64_t t_stride;
    int32_t *       free_pages; int32_t free_cap;
    const int32_t * n_free; int32_t * n_free_out; int32_t * n_kv_out;
    int32_t         n_seq, page, max_pages;
    pt_head *       head;
    pt_req *        req;
    uint32_t *      status;
};

// Request b, a thread each, behind requests that give back `before` pages.
struct trim_sums { int32_t n, keep, first, back, served; int64_t c; };
__device__ __forceinline__ trim_sums sum_trim(const trim_args & a, int64_t b, int32_t n_free, int64_t before, pair64 (*part)[PT_WAVES],
                                              bool & bad) {
    const bool in = b < a.n_seq;
    const int32_t room = a.max_pages * a.page, n_in = in ? a.n_kv[b] : 0, k_in = in ? a.keep[b] : 0;
    trim_sums x;
    x.n = n_in < 0 ? 0 : n_in > room ? room : n_in;
    bad |= x.n != n_in;
    x.keep = k_in < 0 ? 0 : k_in > x.n ? x.n : k_in;
    x.first = (int32_t) ceil_div(x.keep, a.page);
    x.back = (int32_t) ceil_div(x.n, a.page) - x.first;
    x.c = before + block_scan({x.back, 0}, part).x;
    x.served = in && (x.back == 0 || x.c <= a.free_cap - n_free);
    bad |= in && !x.served;
    return x;
}

__global__ __launch_bounds__(PT_THREADS) void k_trim_scan(trim_args a) {
    __shared__ pair64 part[PT_WAVES];
    __shared__ int64_t last;
    const int tid = threadIdx.x, lane = tid & 63;
    bool bad = false;
    const int32_t n_free = stack_size(a.n_free, a.free_cap, bad);
    int64_t carry = 0, given = 0;
    for (int64_t b0 = 0; b0 < a.n_seq; b0 += blockDim.x) {
        const int64_t b = b0 + tid;
        const trim_sums x = sum_trim(a, b, n_free, carry, &part, bad);
        const int32_t back = x.back, first = x.first, served = x.served;
        const int64_t c = x.c;
        if (b < a.n_seq) {
            a.n_kv_out[b] = served ? x.keep : x.n;
            if (served) given += back;
            a.req[b] = pt_req{first, served ? back : 0, (int32_t) (c - back < INT32_MAX ? c - back : INT32_MAX), served};
            // the first pages here, more than that by the second launch
            if (served)
                for (int32_t i = 0; i < back && i < 2; i++)
                    a.free_pages[n_free + (c - back) + i] = a.table[b * a.t_stride + first + i];
        }
        if (tid == (int) blockDim.x - 1) last = c;
        __syncthreads();
        carry = last;
        __syncthreads();
    }
    const pair64 g = block_scan({given, 0}, &part);
    if (tid == (int) blockDim.x - 1) {
        *a.n_free_out = n_free + (int32_t) g.x;
        *a.head = pt_head{n_free, 0, {0, 0}};
    }
    if (__ballot(bad) && lane == 0) atomicOr(a.status, DEVERR_PAGES);
}

// Pages 2 .. of the requests that give back more than two: a wave per request.
__global__ __launch_bounds__(ROW_THREADS) void k_trim_pages(trim_args a) {
    const int64_t b = (int64_t) blockIdx.x * (ROW_THREADS / 64) + (threadIdx.x >> 6);
    if (b >= a.n_seq) return;
    const pt_req r = a.req[b];
    const int32_t * src = a.table + b * a.t_stride + r.past;
    int32_t * dst = a.free_pages + a.head->n_free + (int64_t) r.at;
    for (int32_t i = 2 + (threadIdx.x & 63); i < r.have; i += 64) dst[i] = src[i];
}

// Both in one launch, for lengths and a stack size that are not updated in place: every workgroup has the sums of all
// requests for itself, the first writes the lengths, and a wave takes a request's pages.
__global__ __launch_bounds__(PT_THREADS) void k_trim_once(trim_args a) {
    __shared__ pair64 part[PT_WAVES];
    __shared__ int32_t first[PT_THREADS], back[PT_THREADS], at[PT_THREADS];
    const int tid = threadIdx.x, lane = tid & 63;
    bool bad = false;
    const int32_t n_free = stack_size(a.n_free, a.free_cap, bad);
    const trim_sums x = sum_trim(a, tid, n_free, 0, &part, bad);
    const int32_t given = x.served ? x.back : 0;
    first[tid] = x.first;
    back[tid] = given;
    at[tid] = (int32_t) (x.c - x.back < INT32_MAX ? x.c - x.back : INT32_MAX);
    __syncthreads();
    if (blockIdx.x == 0) {
        if (tid < a.n_seq) a.n_kv_out[tid] = x.served ? x.keep : x.n;
        const pair64 g = block_scan({given, 0}, &part);
        if (tid == (int) blockDim.x - 1) *a.n_free_out = n_free + (int32_t) g.x;
        if (__ballot(bad) && lane == 0) atomicOr(a.status, DEVERR_PAGES);
    }
    const int waves = (int) (blockDim.x >> 6);
    for (int b = (int) blockIdx.x * waves + (tid >> 6); b < a.n_seq; b += (int) gridDim.x * waves) {
        const int32_t * src = a.table + b * a.t_stride + first[b];
        for (int32_t i = lane; i < back[b]; i += 64) a.free_pages[(int64_t) n_free + at[b] + i] = src[i];
    }
}

int scan_threads(int32_t n_seq) { return std::min(PT_THREADS, (n_seq + 63) / 64 * 64); }

int check_tables(const char * op, int32_t n_seq, int32_t page_size, int64_t table_stride, int32_t max_pages,
                 int32_t free_cap, const void * ws, size_t ws_bytes) {
    const std::string o(op);
    if (n_seq < 1 || n_seq > PT_MAX_SEQ) return set_error(QWFN_EINVAL, o + ": n_seq must lie in [1, 65536]");
    if (page_size < 1 || max_pages < 1 || (int64_t) page_size * max_pages > 0x7fffffff)
        return set_error(QWFN_EINVAL, o + ": page_size and max_pages must be positive, their product below 2^31");
    if (table_stride < max_pages) return set_error(QWFN_EINVAL, o + ": table rows overlap (table_stride < max_pages)");
    if (table_stride > 0x7fffffff) return set_error(QWFN_EINVAL, o + ": table_stride must be below 2^31");
    if (free_cap < 0) return set_error(QWFN_EINVAL, o + ": free_cap must not be negative");
    if (!ws || ws_bytes < qwfn_paged_workspace_size(n_seq))
        return set_error(QWFN_ENOMEM, o + ": ws must hold qwfn_paged_workspace_size bytes");
    if (!is_aligned(ws, 16)) return set_error(QWFN_EALIGN, o + ": ws must be 16-byte aligned");
    return QWFN_OK;
}

// Every span 4-byte aligned and present, and no `out` over another span; in-place pairs are passed once.
int check_spans(const char * op, const span * in, int n_in, const span * out, int n_out) {
    for (int i = 0; i < n_in + n_out; i++) {
        const span & s = i < n_in ? in[i] : out[i - n_in];
        if (!is_aligned(s.p, 4)) return set_error(QWFN_EALIGN, std::string(op) + ": " + s.name + " must be 4-byte aligned");
    }
    return check_overlaps(op, in, n_in, out, n_out);
}

int extend(const int32_t * n_past, const int32_t * n_new, int32_t n_seq, int32_t page_size, int32_t * table, int64_t table_stride,
           int32_t max_pages, const int32_t * free_pages, int32_t free_cap, const int32_t * n_free, int32_t * n_free_out,
           int32_t * n_kv, int32_t * cu_new, int32_t * slots, int32_t * pos, int32_t * seq, int64_t n_tok, int32_t pad_slot,
           const int32_t * states, int32_t * state_slots, void * ws, size_t ws_bytes, void * stream) {
    if (!n_past || !n_new || !table || !free_pages || !n_free || !n_free_out || !n_kv || !cu_new || (!slots && n_tok))
        return set_error(QWFN_EINVAL, "paged_extend: NULL pointer");
    if (int rc = check_tables("paged_extend", n_seq, page_size, table_stride, max_pages, free_cap, ws, ws_bytes))
        return rc;
    if (n_tok < 0 || n_tok > 0x7fffffff) return set_error(QWFN_EINVAL, "paged_extend: n_tok must lie in [0, 2^31)");
    const size_t per = (size_t) n_seq * 4, tok = (size_t) n_tok * 4;
    const size_t tab = ((size_t) (n_seq - 1) * table_stride + max_pages) * 4;
    const span in[] = {{n_kv == n_past ? nullptr : n_past, per, "n_past"}, {n_new, per, "n_new"},
                       {free_pages, (size_t) free_cap * 4, "free_pages"}, {states, per, "states"},
                       {n_free_out == n_free ? nullptr : n_free, 4, "n_free"}};
    const span out[] = {{table, tab, "table"}, {n_free_out, 4, "n_free_out"}, {n_kv, per, "n_kv"},
                        {cu_new, per + 4, "cu_new"}, {slots, tok, "slots"}, {pos, tok, "pos"}, {seq, tok, "seq"},
                        {state_slots, per, "state_slots"}, {ws, qwfn_paged_workspace_size(n_seq), "ws"}};
    if (int rc = check_spans("paged_extend", in, 5, out, 9)) return rc;
    ext_args a{};
    if (int rc = status_word(&a.status)) return rc;
    a.past = n_past; a.fresh = n_new; a.table = table; a.t_stride = table_stride;
    a.free_pages = free_pages; a.free_cap = free_cap; a.n_free = n_free; a.n_free_out = n_free_out;
    a.n_kv = n_kv; a.cu = cu_new; a.slots = slots; a.pos = pos; a.seq = seq; a.n_tok = n_tok;
    a.states = states; a.state_slots = state_slots;
    a.n_seq = n_seq; a.page = page_size; a.max_pages = max_pages; a.pad_slot = pad_slot;
    a.head = (pt_head *) ws; a.req = (pt_req *) ((char *) ws + sizeof(pt_head));
    a.lists = n_tok <= (int64_t) EXT_FEW * n_seq;
    if (!a.lists && n_seq <= PT_THREADS && n_kv != n_past && n_free_out != n_free) {
        const int threads = std::max(scan_threads(n_seq), ROW_THREADS);
        hipLaunchKernelGGL(k_extend_once, dim3((unsigned) ((n_tok + threads - 1) / threads)), dim3(threads), 0, as_stream(stream), a);
        return hip_check(hipGetLastError(), "paged_extend launch");
    }
    hipLaunchKernelGGL(k_extend_scan, dim3(1), dim3(scan_threads(n_seq)), 0, as_stream(stream), a);
    if (int rc = hip_check(hipGetLastError(), "paged_extend launch")) return rc;
    if (a.lists) return QWFN_OK;
    hipLaunchKernelGGL(k_extend_lists, dim3((unsigned) ((n_tok + ROW_THREADS - 1) / ROW_THREADS)), dim3(ROW_THREADS), 0,
                       as_stream(stream), a);
    return hip_check(hipGetLastError(), "paged_extend launch");
}

}  // namespace
}  // namespace qwfn

using namespace qwfn;

extern "C" size_t qwfn_paged_workspace_size(int32_t n_seq) {
    return n_seq < 1 || n_seq > PT_MAX_SEQ ? 0 : sizeof(pt_head) + (size_t) n_seq * sizeof(pt_req);
}

extern "C" int qwfn_paged_extend(const int32_t * n_past, const int32_t * n_new, int32_t n_seq, int32_t page_size,
                                 int32_t * table, int64_t table_stride, int32_t max_pages, const int32_t * free_pages,
                                 int32_t free_cap, const int32_t * n_free, int32_t * n_free_out, int32_t * n_kv,
                                 int32_t * cu_new, int32_t * slots, int32_t * pos, int32_t * seq, int64_t n_tok,
                                 int32_t pad_slot, void * ws, size_t ws_bytes, void * stream) {
    return ::qwfn::abi_call("paged_extend", [&]() -> int {
        return extend(n_past, n_new, n_seq, page_size, table, table_stride, max_pages, free_pages, free_cap, n_free, n_free_out,
                      n_kv, cu_new, slots, pos, seq, n_tok, pad_slot, nullptr, nullptr, ws, ws_bytes, stream);
    });
}

extern "C" int qwfn_paged_extend_states(const int32_t * n_past, const int32_t * n_new, int32_t n_seq, int32_t page_size,
                                        int32_t * table, int64_t table_stride, int32_t max_pages, const int32_t * free_pages,
                                        int32_t free_cap, const int32_t * n_free, int32_t * n_free_out, int32_t * n_kv,
                                        int32_t * cu_new, int32_t * slots, int32_t * pos, int32_t * seq, int64_t n_tok,
                                        int32_t pad_slot, const int32_t * states, int32_t * state_slots, void * ws,
                                        size_t ws_bytes, void * stream) {
    return ::qwfn::abi_call("paged_extend", [&]() -> int {
        if (!state_slots) return set_error(QWFN_EINVAL, "paged_extend: NULL pointer");
        return extend(n_past, n_new, n_seq, page_size, table, table_stride, max_pages, free_pages, free_cap, n_free, n_free_out,
                      n_kv, cu_new, slots, pos, seq, n_tok, pad_slot, states, state_slots, ws, ws_bytes, stream);
    });
}

extern "C" int qwfn_paged_trim(const int32_t * n_keep, const int32_t * n_kv, int32_t n_seq, int32_t page_size,
                               const int32_t * table, int64_t table_stride, int32_t max_pages, int32_t * free_pages,
                               int32_t free_cap, const int32_t * n_free, int32_t * n_free_out, int32_t * n_kv_out,
                               void * ws, size_t ws_bytes, void * stream) {
    return ::qwfn::abi_call("paged_trim", [&]() -> int {
        if (!n_keep || !n_kv || !table || !free_pages || !n_free || !n_free_out || !n_kv_out)
            return set_error(QWFN_EINVAL, "paged_trim: NULL pointer");
        if (int rc = check_tables("paged_trim", n_seq, page_size, table_stride, max_pages, free_cap, ws, ws_bytes))
            return rc;
        const size_t per = (size_t) n_seq * 4, tab = ((size_t) (n_seq - 1) * table_stride + max_pages) * 4;
        const span in[] = {{n_keep, per, "n_keep"}, {n_kv_out == n_kv ? nullptr : n_kv, per, "n_kv"}, {table, tab, "table"},
                           {n_free_out == n_free ? nullptr : n_free, 4, "n_free"}};
        const span out[] = {{free_pages, (size_t) free_cap * 4, "free_pages"}, {n_free_out, 4, "n_free_out"},
                            {n_kv_out, per, "n_kv_out"}, {ws, qwfn_paged_workspace_size(n_seq), "ws"}};
        if (int rc = check_spans("paged_trim", in, 4, out, 4)) return rc;
        trim_args a{};
        if (int rc = status_word(&a.status)) return rc;
        a.keep = n_keep; a.n_kv = n_kv; a.table = table; a.t_stride = table_stride;
        a.free_pages = free_pages; a.free_cap = free_cap; a.n_free = n_free; a.n_free_out = n_free_out; a.n_kv_out = n_kv_out;
        a.n_seq = n_seq; a.page = page_size; a.max_pages = max_pages;
        a.head = (pt_head *) ws; a.req = (pt_req *) ((char *) ws + sizeof(pt_head));
        if (n_seq <= PT_THREADS && n_kv_out != n_kv && n_free_out != n_free) {
            const int threads = scan_threads(n_seq), waves = threads / 64;
            hipLaunchKernelGGL(k_trim_once, dim3((unsigned) ((n_seq + waves - 1) / waves)), dim3(threads), 0, as_stream(stream), a);
            return hip_check(hipGetLastError(), "paged_trim launch");
        }
        hipLaunchKernelGGL(k_trim_scan, dim3(1), dim3(scan_threads(n_seq)), 0, as_stream(stream), a);
        if (int rc = hip_check(hipGetLastError(), "paged_trim launch")) return rc;
        hipLaunchKernelGGL(k_trim_pages, dim3((unsigned) ((n_seq + ROW_THREADS / 64 - 1) / (ROW_THREADS / 64))),
                           dim3(ROW_THREADS), 0, as_stream(stream), a);
        return hip_check(hipGetLastError(), "paged_trim launch");
    });
}
