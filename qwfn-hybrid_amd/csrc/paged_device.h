// What the attention kernels over pages share: their arguments, loads and stores of the three types, LDS DMA, and the run
// of key tiles that a workgroup takes.
#pragma once

#include "fattn_device.h"
#include "q8_device.h"
#include "qwfn_common.h"
#include "qwfn_paged.h"

#include <algorithm>

namespace qwfn {

// x / d for x < 2^31 by a multiplication: m = floor(2^(31 + s) / d) + 1, s = ceil(log2 d), is off by at
// most d <= 2^s, and x (m d - 2^(31 + s)) < 2^(31 + s) keeps the quotient whole.
struct fast_div { uint32_t d, m, s; };
inline fast_div make_div(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) s++;
    return {d, (uint32_t) (((1ull << (31 + s)) / d) + 1), s};
}
struct pa_args {
    const char *    q; size_t q_nb1, q_nb2, q_nb3;
    const char *    k; const char * v;
    uint32_t        nb1;               // bytes of a cache row
    size_t          nb2;               // and of a head's offset
    int64_t         n_pages;
    const int32_t * table; int64_t t_stride;
    const int32_t * n_kv;
    int64_t         max_kv;            // max_pages * page
    fast_div        page;
    const char *    gate; char * dst;
    int32_t         type;              // of q, gate and dst
    int32_t         n_seq, T, nh, nh_kv, rep, R, x86;
    int32_t         runs;              // runs the tiles are cut into, at most
    fast_div        f_runs, f_inner, f_kv, f_rep;      // runs, blocks of a run, KV heads, rep
    float           c;                 // scale * log2(e): scores are in log2 units
    float *         part_o;            // [run + request][nh_kv][R][D]; k_paged_tree's: [..][nh_kv][tile of 32 rows][as its registers lie]
    float2 *        part_ml;           // [run + request][nh_kv][R]
    int2 *          span;              // [request] (a tree's: [row group][request]): its first and last run
    // trees: nodes of a request (or NULL), what each sees, query rows of a row group
    const int32_t * n_tree; const uint64_t * masks;
    int32_t         group; fast_div f_group;
    uint32_t *      status;
};

// The attention of a tree with 32 query rows a wave (paged_tree.hip): the rows of a workgroup, workgroups of a CU, and the launch.
int tree_rows(int64_t D);
int launch_tree_attn(const pa_args & a, int64_t D, int groups, hipStream_t s);

namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int PA_WAVES = 4;
constexpr int PA_THREADS = PA_WAVES * 64;
constexpr int PA_TILE = 32;            // keys of a tile
constexpr int PA_MIN_TILES = PA_WAVES; // of a run: one a wave
constexpr int PA_LEAD = 8;             // tiles that a request counts more than it has
constexpr int PA_CUS = 256;            // two workgroups a CU (registers)
constexpr int PA_MAX_ROWS = 64;        // query rows per KV head
constexpr int PA_MAX_TREE_ROWS = 1024;
constexpr int PA_NARROW_ROWS = 64, PA_WIDE_ROWS = 512, PA_WIDE_TILES = 48;      // plan_paged
constexpr float PA_LOG2E = 1.4426950408889634f;
constexpr float PA_SLACK = 6.f;        // log2 by which M may lie below its request
constexpr int PA_BIAS = 8;             // P dv < 2^PA_BIAS at M
constexpr float PA_IBIAS = 12582912.f; // 1.5 2^23: an integer below 2^22 added to its bits is added to its value
constexpr int PA_IBITS = 0x4b400000;   // (a block's dot is at most 32 128 128 = 2^19)

__device__ __forceinline__ uint32_t div_by(uint32_t x, fast_div f) { return f.s == 0 ? x : __umulhi(x, f.m) >> (f.s - 1); }

// One wave-wide LDS DMA: lane i copies its UB bytes to LDS[at + UB i]. Inline asm, so that the compiler neither
// moves memory operations across it nor waits for it: the kernel's own counts do. (m0 is read one wait state after
// its write at the earliest; the compiler keeps nothing in it here.)
template <int UB> __device__ __forceinline__ void pa_dma(uint64_t from, uint32_t at) {
    if constexpr (UB == 16)
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(from), "s"(at) : "memory");
    else
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(from), "s"(at) : "memory");
}
// The same from `from` + delta (delta the same for all lanes); the sum stands in m0's wait state.
template <int UB> __device__ __forceinline__ void pa_dma_plus(uint64_t from, uint64_t delta, uint32_t at) {
    uint64_t sum;
    if constexpr (UB == 16)
        asm volatile("s_mov_b32 m0, %3\n\tv_lshl_add_u64 %0, %1, 0, %2\n\tglobal_load_lds_dwordx4 %0, off"
                     : "=&v"(sum) : "v"(from), "s"(delta), "s"(at) : "memory");
    else
        asm volatile("s_mov_b32 m0, %3\n\tv_lshl_add_u64 %0, %1, 0, %2\n\tglobal_load_lds_dword %0, off"
                     : "=&v"(sum) : "v"(from), "s"(delta), "s"(at) : "memory");
}
// Waits until at most N vector-memory operations are in flight, or for this wave's LDS operations.
template <int N> __device__ __forceinline__ void pa_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
__device__ __forceinline__ void pa_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t pa_lds(const void * p) { return (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) void *) p; }

__device__ __forceinline__ void load4(const char * p, int32_t type, float x[4]) {
    if (type == QWFN_TYPE_F32) {
        const float4 f = *(const float4 *) p;
        x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
    } else {
        const uint2 u = *(const uint2 *) p;
        const uint32_t h[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
        for (int i = 0; i < 4; i++)
            x[i] = type == QWFN_TYPE_F16 ? dev::f16_bits_to_f32((uint16_t) h[i]) : __builtin_bit_cast(float, h[i] << 16);
    }
}
// bf16 of x, to nearest even; a NaN stays one
__device__ __forceinline__ uint32_t bf16_bits(float x) { return __builtin_bit_cast(uint16_t, (__bf16) x); }
__device__ __forceinline__ void store4(char * p, int32_t type, const float x[4]) {
    if (type == QWFN_TYPE_F32) {
        *(float4 *) p = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = type == QWFN_TYPE_F16 ? dev::f32_to_f16_bits(x[i]) : bf16_bits(x[i]);
        *(uint2 *) p = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
}
// l: the row's sum of weights. 0 where its query saw nothing (or is no node): x is 0 then and stays 0 whatever the gate holds, NaN
// in a padded batch. TYPE: a.type where it is known (-1: it is not).
template <int TYPE = -1>
__device__ __forceinline__ void finish4(const pa_args & a, size_t elem, float x[4], float l) {
    const int32_t type = TYPE >= 0 ? TYPE : a.type;
    const size_t es = type == QWFN_TYPE_F32 ? 4 : 2;
    if (a.gate && l != 0.f) {
        float g[4];
        load4(a.gate + elem * es, type, g);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = x[i] / (1.f + expf(-g[i]));
    }
    store4(a.dst + elem * es, type, x);
}

// Largest over lanes l and l ^ 32, l and l ^ 16, a row of 16, without LDS.
__device__ __forceinline__ uint32_t umax_halves(uint32_t x) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    unsigned p = r[0], q = r[1];
    asm volatile("" : "+v"(p), "+v"(q));
    return max(p, q);
}
__device__ __forceinline__ uint32_t umax_rows(uint32_t x) {           // lanes l and l ^ 16
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    unsigned p = r[0], q = r[1];
    asm volatile("" : "+v"(p), "+v"(q));
    return max(p, q);
}
__device__ __forceinline__ uint32_t umax_row(uint32_t x) {            // the 16 lanes of a row
    x = max(x, dev::dpp_u32<dev::DPP_QUAD_1032>(x));
    x = max(x, dev::dpp_u32<dev::DPP_QUAD_2301>(x));
    x = max(x, dev::dpp_u32<dev::DPP_HALF_MIRROR>(x));
    return max(x, dev::dpp_u32<0x140>(x));                            // row_mirror
}

// A block's run of the tiles of all requests: the request it starts in and its length, the tile there, the
// tiles left, its place, how many tiles a run has. A request counts PA_LEAD tiles more than it has, in front of
// its own (off starts at -PA_LEAD): what its queries and its output cost the workgroup that begins it. 48 ragged
// requests without that: 99 us for 91, the workgroups with two requests last.
struct pa_run { int32_t b, n, off, left, pos, per; };

__device__ __forceinline__ int32_t clip_len(const pa_args & a, int32_t n) { return n <= 0 ? 0 : n < a.max_kv ? n : (int32_t) a.max_kv; }
__device__ __forceinline__ int32_t tiles_of(int32_t n) { return (int32_t) (((uint32_t) n + PA_TILE - 1) / PA_TILE); }
template <int LEAD> __device__ __forceinline__ int32_t cost_of(int32_t n) { return n > 0 ? tiles_of(n) + LEAD : 0; }
template <int ROUND> __device__ __forceinline__ int32_t run_len(const pa_args & a, int32_t total) {
    const int32_t per = ((int32_t) div_by((uint32_t) (total + a.runs - 1), a.f_runs) + ROUND - 1) / ROUND * ROUND;
    return per < ROUND ? ROUND : per;                       // whole rounds of the waves
}

// A tree's nodes in the cache, and the keys that row group rg of request b goes through: none where it has no node.
__device__ __forceinline__ int32_t tree_nodes(const pa_args & a, int32_t b, int32_t n) {
    const int32_t t = a.n_tree ? a.n_tree[b] : a.T, most = n < a.T ? n : a.T;
    return t <= 0 ? 0 : t < most ? t : most;
}
__device__ __forceinline__ int32_t tree_len(const pa_args & a, int32_t b, int rg) {
    const int32_t n = clip_len(a, a.n_kv[b]);
    return tree_nodes(a, b, n) * a.rep > rg * a.group ? n : 0;
}
// The 32 keys from `key0` that a node sees, `base` tokens before the tree.
__device__ __forceinline__ uint32_t tree_sees(uint64_t mask, int32_t key0, int32_t base) {
    const int32_t rel = key0 - base;
    if (rel >= 64) return 0u;
    if (rel >= 0) return (uint32_t) (mask >> rel);
    return rel <= -32 ? 0xffffffffu : (uint32_t) (mask << -rel) | ((1u << -rel) - 1u);
}

// Where run g starts, requests of len(b) keys. Up to 64 requests: a lane each, every wave on its own. More: every thread sums
// the tiles of a few requests.
template <int WAVES, int ROUND, int LEAD, typename Len>
__device__ __forceinline__ pa_run find_run(const pa_args & a, int g, int32_t * sh, Len len) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    pa_run r{0, 0, 0, 0, 0, 0};
    if (a.n_seq <= 64) {
        const int32_t n = lane < a.n_seq ? len(lane) : 0, t = cost_of<LEAD>(n);
        int32_t incl = t;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int32_t x = __shfl_up(incl, d);
            if (lane >= d) incl += x;
        }
        const int32_t total = __builtin_amdgcn_readlane(incl, 63);
        r.per = run_len<ROUND>(a, total);
        const int64_t start = (int64_t) g * r.per;
        if (start < total) {
            r.b = __builtin_popcountll(__ballot(incl <= (int32_t) start));
            r.n = __builtin_amdgcn_readlane(n, r.b);
            r.off = (int32_t) start - __builtin_amdgcn_readlane(incl - t, r.b) - LEAD;
            r.left = total - (int32_t) start < r.per ? total - (int32_t) start : r.per;
            r.pos = (int32_t) start;
        }
        return r;
    }
    const int c = (a.n_seq + (WAVES * 64) - 1) / (WAVES * 64);
    int32_t sum = 0;
    for (int i = 0; i < c; i++) {
        const int b = tid * c + i;
        if (b < a.n_seq) sum += cost_of<LEAD>(len(b));
    }
    int32_t incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int32_t x = __shfl_up(incl, d);
        if (lane >= d) incl += x;
    }
    if (lane == 63) sh[w] = incl;
    __syncthreads();
    int32_t before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        const int32_t x = sh[i];
        if (i < w) before += x;
        total += x;
    }
    incl += before;
    r.per = run_len<ROUND>(a, total);
    const int64_t start = (int64_t) g * r.per;
    if (start >= incl - sum && start < incl) {
        int32_t at = incl - sum;
        for (int i = 0; i < c; i++) {
            const int b = tid * c + i;
            const int32_t n = b < a.n_seq ? len(b) : 0, t = cost_of<LEAD>(n);
            if (start >= at && start < at + t) {
                sh[WAVES] = b;
                sh[WAVES + 1] = n;
                sh[WAVES + 2] = (int32_t) (start - at);
            }
            at += t;
        }
    }
    __syncthreads();
    if (start < total) {
        r.b = __builtin_amdgcn_readfirstlane(sh[WAVES]);
        r.n = __builtin_amdgcn_readfirstlane(sh[WAVES + 1]);
        r.off = __builtin_amdgcn_readfirstlane(sh[WAVES + 2]) - LEAD;
        r.left = __builtin_amdgcn_readfirstlane(total - start < r.per ? (int32_t) (total - start) : r.per);
        r.pos = (int32_t) start;
    }
    return r;
}

}  // namespace
}  // namespace qwfn
