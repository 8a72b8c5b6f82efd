// Decode attention over a paged q8_0 cache: many requests of different lengths,
// T newest tokens each, keys found through block tables.
//
//   s_j = c sum_b dq_b dk_jb (qq_b . kq_jb)      q requantised to q8_0, integer dots
//   out = sum_j 2^(s_j - M) dv_j vq_j / sum_j 2^(s_j - M),   c = scale log2(e)
//
// What bounds it: the rows, n_kv * 34 D / 32 bytes of K and of V a KV head, read
// once (at 8 query heads a KV head 7.5 operations a byte).
//
// Work: the requests' keys in tiles of 32, all requests' tiles in one row; each
// workgroup takes an equal run of it for one KV head and one tile of 16 query
// rows, whatever the lengths are (they are known on the device only). A run that
// crosses a request's end is cut there. A request inside one run is finished by its
// workgroup; the parts of the others go to the workspace as (O, M, l) and
// k_paged_merge joins them in the order of the runs, so results repeat bit for bit.
// The KV heads and row groups of one run are blocks next to each other on one XCD:
// the cache lines that two heads share come from one L2, and so do the rows that more
// than 16 query rows need again (a workgroup of 32 query rows leaves one wave a SIMD:
// 3 tokens of 8 requests with 12295 keys took 62 us that way and 52 this way, and 25 and 19
// at 2 requests with 3000 keys). The rows of two row groups go from the L2 to the LDS twice:
// those 8 requests 214 MB in 46 us, the 4.7 TB/s of one group's long requests.
//
// Inside a workgroup the 4 waves take every fourth tile of the run, each on its
// own: no barrier, and no wave waits for another's data. A tile's rows come by LDS
// DMA into the wave's part of the LDS, one buffer for K and one for V: K of the
// next tile is sent for when the scores are done, V when the products are. The table
// entries go the same way, two tiles ahead, so that every vector-memory operation of the
// loop is one whose place in the order is known, and a wait leaves just the later
// ones in flight.
//   S^T = K Q^T   v_mfma_i32_16x16x64_i8 a q8_0 block: A is the 64-byte window of the
//                 row (from a 16-byte boundary) that holds the block's 32 quants, B
//                 the query's quants at the same place of a window that is zero
//                 elsewhere, so whatever else the row's window holds adds nothing.
//   O^T = V^T P^T v_mfma_f32_16x16x32_f16: the accumulators of S^T are the B operand as
//                 they lie (the sum over keys takes them in the order of the
//                 registers). V's int8 are exact in f16; P dv enters as an f16 pair hi
//                 + lo (22 bits; one f16 alone is 3e-4 off).
// The reference M of a row is its running maximum, moved up by the exponent of the
// largest dv of the tile and down by 8: P dv then lies below 2^8 whatever the
// scales of V are, and 33 bits of range lie below it in f16. It follows a rise
// of up to 2^6 late (P dv < 2^15), so O is rescaled rarely.
#include "fattn_device.h"
#include "q8_device.h"
#include "qwfn_common.h"
#include "qwfn_paged.h"

#include <algorithm>
#include <cmath>

namespace qwfn {
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
constexpr float PA_LOG2E = 1.4426950408889634f;
constexpr float PA_SLACK = 6.f;        // log2 by which M may lie below its request
constexpr int PA_BIAS = 8;             // P dv < 2^PA_BIAS at M
constexpr float PA_IBIAS = 12582912.f; // 1.5 2^23: an integer below 2^22 added to its bits is added to its value
constexpr int PA_IBITS = 0x4b400000;   // (a block's dot is at most 32 128 128 = 2^19)

// x / d for x < 2^31 by a multiplication: m = floor(2^(31 + s) / d) + 1, s = ceil(log2 d), is off by at
// most d <= 2^s, and x (m d - 2^(31 + s)) < 2^(31 + s) keeps the quotient whole.
struct fast_div { uint32_t d, m, s; };
fast_div make_div(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) s++;
    return {d, (uint32_t) (((1ull << (31 + s)) / d) + 1), s};
}
__device__ __forceinline__ uint32_t div_by(uint32_t x, fast_div f) { return f.s == 0 ? x : __umulhi(x, f.m) >> (f.s - 1); }

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
    float *         part_o;            // [run + request][nh_kv][R][D]
    float2 *        part_ml;           // [run + request][nh_kv][R]
    int2 *          span;              // [request]: its first and last run
    uint32_t *      status;
};

template <int D> struct pa_cfg {
    static constexpr int NBLK = D / QK;
    static constexpr int SEG = NBLK * QBLOCK;            // bytes of a head row
    // a row goes to LDS in units of a DMA lane, 16 bytes where a head row is whole ones; UPR of them a row
    // (rows from 16-byte boundaries), the last UPR - UV only fill
    static constexpr int UB = SEG % 16 == 0 ? 16 : 4, UV = SEG / UB;
    static constexpr int LS = (SEG + 15) / 16 * 16, UPR = LS / UB;        // bytes of a row in LDS
    static constexpr int UNITS = PA_TILE * UPR, DMAS = (UNITS + 63) / 64;
    static constexpr int UMUL = 65536 / UPR + 1;         // i / UPR = i UMUL >> 16 for i < UNITS
    static constexpr int ROWS = PA_TILE * LS;            // of a tensor's tile in LDS
    static constexpr int OROW = D + 4;                   // floats of a row of O in LDS: rows from other banks
    // of a wave: a tile of K and of V, row addresses, table entries (a lane each), each key's largest dv, K's and V's scales
    static constexpr int OA = 2 * ROWS, OE = OA + PA_TILE * 8, OM = OE + 256, OS = OM + 2 * PA_TILE;
    static constexpr int WAVE = OS + 2 * NBLK * PA_TILE * 2;
    static constexpr int IMG = 16 * NBLK * 64;           // the query windows
    static constexpr int QI = NBLK / 2;                  // 4-value groups a thread quantises
    static_assert(IMG + 16 * NBLK * 4 <= ROWS && WAVE >= 16 * OROW * 4 && WAVE % 16 == 0, "the query images fit, and a wave's O in its part");
    static_assert((UNITS - 1) * (UMUL * UPR - 65536) < 65536, "the division is exact");
    static_assert((QBLOCK * (NBLK - 1) + 2) / 16 * 16 + 64 <= LS + 64, "a window ends in the next row, or V's first");
};
constexpr int pa_win(int b) { return (QBLOCK * b + 2) / 16; }              // first 16 bytes of block b's window

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
__device__ __forceinline__ void finish4(const pa_args & a, size_t elem, float x[4]) {
    const size_t es = a.type == QWFN_TYPE_F32 ? 4 : 2;
    if (a.gate) {
        float g[4];
        load4(a.gate + elem * es, a.type, g);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = x[i] / (1.f + expf(-g[i]));
    }
    store4(a.dst + elem * es, a.type, x);
}

// B operands of a V block: x = p d of the lane's 8 keys (p[u], d[u] packed) as f16 pairs, hi toward zero, lo = p d - hi from
// one fused step each. One asm: a single pair of wait states before the MFMA (fattn_device.h) for all of it.
__device__ __forceinline__ void hilo(const float (&p)[2][4], const uint2 (&d)[2], v4u & hi, v4u & lo) {
    uint32_t h0, h1, h2, h3, l0, l1, l2, l3;
    float x, y;
#define QWFN_HILO(H, L, P0, P1, DV)                                                        \
    "v_fma_mix_f32 %8, " P0 ", " DV ", 0 op_sel:[0,0,0] op_sel_hi:[0,1,0]\n\t"             \
    "v_fma_mix_f32 %9, " P1 ", " DV ", 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]\n\t"             \
    "v_cvt_pkrtz_f16_f32 " H ", %8, %9\n\t"                                               \
    "v_fma_mixlo_f16 " L ", " P0 ", " DV ", -" H " op_sel:[0,0,0] op_sel_hi:[0,1,1]\n\t"   \
    "v_fma_mixhi_f16 " L ", " P1 ", " DV ", -" H " op_sel:[0,1,1] op_sel_hi:[0,1,1]\n\t"
    asm(QWFN_HILO("%0", "%4", "%10", "%11", "%18") QWFN_HILO("%1", "%5", "%12", "%13", "%19")
        QWFN_HILO("%2", "%6", "%14", "%15", "%20") QWFN_HILO("%3", "%7", "%16", "%17", "%21")
        "s_nop 1"
        : "=&v"(h0), "=&v"(h1), "=&v"(h2), "=&v"(h3), "=&v"(l0), "=&v"(l1), "=&v"(l2), "=&v"(l3), "=&v"(x), "=&v"(y)
        : "v"(p[0][0]), "v"(p[0][1]), "v"(p[0][2]), "v"(p[0][3]), "v"(p[1][0]), "v"(p[1][1]), "v"(p[1][2]), "v"(p[1][3]),
          "v"(d[0].x), "v"(d[0].y), "v"(d[1].x), "v"(d[1].y));
#undef QWFN_HILO
    hi = v4u{h0, h1, h2, h3};
    lo = v4u{l0, l1, l2, l3};
}
// A operands: dims 2m (a0) and 2m + 1 (a1) of 8 keys from the bytes of v, int8 to f16 (exact).
__device__ __forceinline__ void cvt_v8(const uint32_t (&v)[2][4], v4u & a0, v4u & a1) {
    uint32_t x0, x1, x2, x3, y0, y1, y2, y3;
#define QWFN_SDWA(D, S, DSEL, UNUSED, SSEL) "v_cvt_f16_i16_sdwa " D ", sext(" S ") dst_sel:" DSEL " dst_unused:" UNUSED " src0_sel:" SSEL "\n\t"
#define QWFN_LOW(D, S, B) QWFN_SDWA(D, S, "WORD_0", "UNUSED_PAD", B)
#define QWFN_HIGH(D, S, B) QWFN_SDWA(D, S, "WORD_1", "UNUSED_PRESERVE", B)
    asm(QWFN_LOW("%0", "%8", "BYTE_0") QWFN_LOW("%1", "%10", "BYTE_0") QWFN_LOW("%2", "%12", "BYTE_0") QWFN_LOW("%3", "%14", "BYTE_0")
        QWFN_HIGH("%0", "%9", "BYTE_0") QWFN_HIGH("%1", "%11", "BYTE_0") QWFN_HIGH("%2", "%13", "BYTE_0") QWFN_HIGH("%3", "%15", "BYTE_0")
        QWFN_LOW("%4", "%8", "BYTE_1") QWFN_LOW("%5", "%10", "BYTE_1") QWFN_LOW("%6", "%12", "BYTE_1") QWFN_LOW("%7", "%14", "BYTE_1")
        QWFN_HIGH("%4", "%9", "BYTE_1") QWFN_HIGH("%5", "%11", "BYTE_1") QWFN_HIGH("%6", "%13", "BYTE_1") QWFN_HIGH("%7", "%15", "BYTE_1")
        "s_nop 1"
        : "=&v"(x0), "=&v"(x1), "=&v"(x2), "=&v"(x3), "=&v"(y0), "=&v"(y1), "=&v"(y2), "=&v"(y3)
        : "v"(v[0][0]), "v"(v[0][1]), "v"(v[0][2]), "v"(v[0][3]), "v"(v[1][0]), "v"(v[1][1]), "v"(v[1][2]), "v"(v[1][3]));
#undef QWFN_LOW
#undef QWFN_HIGH
#undef QWFN_SDWA
    a0 = v4u{x0, x1, x2, x3};
    a1 = v4u{y0, y1, y2, y3};
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
__device__ __forceinline__ int32_t cost_of(int32_t n) { return n > 0 ? tiles_of(n) + PA_LEAD : 0; }
__device__ __forceinline__ int32_t run_len(const pa_args & a, int32_t total) {
    const int32_t per = ((int32_t) div_by((uint32_t) (total + a.runs - 1), a.f_runs) + PA_WAVES - 1) / PA_WAVES * PA_WAVES;
    return per < PA_MIN_TILES ? PA_MIN_TILES : per;         // whole rounds of the waves
}

// Where run g starts. Up to 64 requests: a lane each, every wave on its own. More: every thread sums the tiles of
// a few requests.
__device__ __forceinline__ pa_run find_run(const pa_args & a, int g, int32_t * sh) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    pa_run r{0, 0, 0, 0, 0, 0};
    if (a.n_seq <= 64) {
        const int32_t n = lane < a.n_seq ? clip_len(a, a.n_kv[lane]) : 0, t = cost_of(n);
        int32_t incl = t;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int32_t x = __shfl_up(incl, d);
            if (lane >= d) incl += x;
        }
        const int32_t total = __builtin_amdgcn_readlane(incl, 63);
        r.per = run_len(a, total);
        const int64_t start = (int64_t) g * r.per;
        if (start < total) {
            r.b = __builtin_popcountll(__ballot(incl <= (int32_t) start));
            r.n = __builtin_amdgcn_readlane(n, r.b);
            r.off = (int32_t) start - __builtin_amdgcn_readlane(incl - t, r.b) - PA_LEAD;
            r.left = total - (int32_t) start < r.per ? total - (int32_t) start : r.per;
            r.pos = (int32_t) start;
        }
        return r;
    }
    const int c = (a.n_seq + PA_THREADS - 1) / PA_THREADS;
    int32_t sum = 0;
    for (int i = 0; i < c; i++) {
        const int b = tid * c + i;
        if (b < a.n_seq) sum += cost_of(clip_len(a, a.n_kv[b]));
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
    for (int i = 0; i < PA_WAVES; i++) {
        const int32_t x = sh[i];
        if (i < w) before += x;
        total += x;
    }
    incl += before;
    r.per = run_len(a, total);
    const int64_t start = (int64_t) g * r.per;
    if (start >= incl - sum && start < incl) {
        int32_t at = incl - sum;
        for (int i = 0; i < c; i++) {
            const int b = tid * c + i;
            const int32_t n = b < a.n_seq ? clip_len(a, a.n_kv[b]) : 0, t = cost_of(n);
            if (start >= at && start < at + t) {
                sh[PA_WAVES] = b;
                sh[PA_WAVES + 1] = n;
                sh[PA_WAVES + 2] = (int32_t) (start - at);
            }
            at += t;
        }
    }
    __syncthreads();
    if (start < total) {
        r.b = __builtin_amdgcn_readfirstlane(sh[PA_WAVES]);
        r.n = __builtin_amdgcn_readfirstlane(sh[PA_WAVES + 1]);
        r.off = __builtin_amdgcn_readfirstlane(sh[PA_WAVES + 2]) - PA_LEAD;
        r.left = __builtin_amdgcn_readfirstlane(total - start < r.per ? (int32_t) (total - start) : r.per);
        r.pos = (int32_t) start;
    }
    return r;
}

template <int D>
__global__ __launch_bounds__(PA_THREADS, 2) void k_paged_attn(pa_args a) {
    using C = pa_cfg<D>;
    constexpr int NBLK = C::NBLK, ND = C::DMAS;
    __shared__ __attribute__((aligned(16))) uint8_t lds[PA_WAVES * C::WAVE];
    __shared__ float2 ml[PA_WAVES][16];
    __shared__ int32_t sh[PA_WAVES + 3];
    const int tid = threadIdx.x;
    int lane = tid & 63, ln = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // blocks -> (run, KV head, row group): those of one run follow each other on one XCD
    const uint32_t j = blockIdx.x >> 3, jq = div_by(j, a.f_inner), hr = j - jq * a.f_inner.d;
    const int g = (int) jq * 8 + (int) (blockIdx.x & 7), rg = (int) div_by(hr, a.f_kv), kvh = (int) hr - rg * a.nh_kv;
    pa_run run = find_run(a, g, sh);

    uint8_t * const my = lds + wave * C::WAVE;
    uint64_t * const addr = (uint64_t *) (my + C::OA);
    const int32_t * const entry = (const int32_t *) (my + C::OE);
    uint16_t * const vtop = (uint16_t *) (my + C::OM);
    uint16_t * const kscl = (uint16_t *) (my + C::OS);
    uint16_t * const vscl = kscl + NBLK * PA_TILE;
    const uint32_t at_k = pa_lds(my), at_v = at_k + C::ROWS, at_e = at_k + C::OE;
    // the query image: in the first wave's V, sent for when the image is read
    uint8_t * const image = lds + C::ROWS;
    const char * kh = a.k + (size_t) kvh * a.nb2;
    const char * vh = a.v + (size_t) kvh * a.nb2;
    const uint64_t v_k = (uint64_t) (vh - kh);
    const size_t es = a.type == QWFN_TYPE_F32 ? 4 : 2;
    // element of dst (and gate) of row r's first value
    auto element = [&](int b, int r) {
        const uint32_t t = div_by((uint32_t) r, a.f_rep), h = (uint32_t) (kvh * a.rep + r) - t * (uint32_t) a.rep;
        return (((size_t) b * a.T + t) * a.nh + h) * D;
    };

    while (run.left > 0) {
        const int b = run.b;
        const int32_t n = run.n, tiles = tiles_of(n);
        if (run.off < 0) {                                 // the tiles in front count, no more
            const int32_t lead = -run.off < run.left ? -run.off : run.left;
            run.off += lead;
            run.left -= lead;
            run.pos += lead;
            if (run.left == 0) break;
        }
        const int32_t nt = tiles - run.off < run.left ? tiles - run.off : run.left;   // tiles of this part
        const bool whole = nt == tiles;
        const int32_t * table = a.table + (int64_t) b * a.t_stride;

        // the table entries of a tile's keys (lanes l and l + 32 the same), clipped to the part's last key
        const int32_t end = (run.off + nt) * PA_TILE < n ? (run.off + nt) * PA_TILE : n;
        auto entries = [&](int t) {
            int32_t key = (run.off + t) * PA_TILE + (lane & 31);
            key = key < end ? key : end - 1;
            pa_dma<4>((uint64_t) (uintptr_t) (table + div_by((uint32_t) key, a.page)), at_e);
        };
        // the addresses of the tile's rows of K, and which of its keys exist
        auto rows_of = [&](int t) -> uint32_t {
            const int32_t key = (run.off + t) * PA_TILE + (lane & 31), page = entry[lane];
            const bool in = t < nt && key < end, ok = in && (uint32_t) page < (uint32_t) a.n_pages;
            if (in && !ok) atomicOr(a.status, DEVERR_GET_ROWS_INDEX);
            const uint32_t slot = ok ? (uint32_t) page * a.page.d + ((uint32_t) key - div_by((uint32_t) key, a.page) * a.page.d) : 0u;
            if (lane < PA_TILE) addr[lane] = (uint64_t) (uintptr_t) kh + (uint64_t) slot * a.nb1;
            return (uint32_t) __ballot(ok);
        };
        // a lane's units of the tile's rows: K's addresses, V's are v_k further
        uint64_t from[ND];
        auto units = [&](auto fn) {
#pragma unroll
            for (int i = 0; i < ND; i++) {
                const int x = lane + 64 * i;
                if (64 * (i + 1) <= C::UNITS || x < C::UNITS) fn(i, x);
            }
        };
        auto send_k = [&](uint32_t at) {
            units([&](int i, int x) {
                const int key = (x * C::UMUL) >> 16, u = x - key * C::UPR;
                from[i] = addr[key] + (uint64_t) (uint32_t) ((u < C::UV ? u : C::UV - 1) * C::UB);
            });
            units([&](int i, int) { pa_dma<C::UB>(from[i], at + 64 * C::UB * i); });
        };
        auto send_v = [&](uint32_t at) { units([&](int i, int) { pa_dma_plus<C::UB>(from[i], v_k, at + 64 * C::UB * i); }); };
        __syncthreads();                                   // the LDS of the part before is read
        // query values on their way: 8 lanes a q8_0 block
        float qx[C::QI][4];
        const int sub = tid & 7;
#pragma unroll
        for (int i = 0; i < C::QI; i++) {
            const int x = (tid >> 3) + 32 * i, r = x / NBLK, blk = x % NBLK;
            int rr = 16 * rg + r;
            rr = rr < a.R ? rr : a.R - 1;
            const uint32_t t = div_by((uint32_t) rr, a.f_rep), h = (uint32_t) (kvh * a.rep + rr) - t * (uint32_t) a.rep;
            load4(a.q + (size_t) t * a.q_nb1 + (size_t) h * a.q_nb2 + (size_t) b * a.q_nb3 + (size_t) (blk * QK + sub * 4) * es,
                  a.type, qx[i]);
        }
        uint32_t live = 0, live_next = 0;                  // the tile's keys that exist
        if (wave < nt) {
            entries(wave);
            pa_wait<0>();
            live = rows_of(wave);
        }
        // (they have come with the entries: a wait for them behind the rows' DMA would wait for the rows too)
#pragma unroll
        for (int i = 0; i < C::QI; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) asm volatile("" : "+v"(qx[i][k]));
        if (wave < nt) {
            wave_lds_sync();
            send_k(at_k);
            entries(wave + PA_WAVES);
        }
        // the query image: rows requantised, each block at its place of a window that is zero elsewhere
#pragma unroll
        for (int i = 0; i < C::QI; i++)
            *(uint2 *) (image + ((tid >> 3) + 32 * i) * 64 + sub * 8) = make_uint2(0u, 0u);
        wave_lds_sync();                                   // a block's 8 lanes zero its window, then write into it
        float * const dql = (float *) (image + C::IMG);
#pragma unroll
        for (int i = 0; i < C::QI; i++) {
            const int x = (tid >> 3) + 32 * i, blk = x % NBLK;
            uint16_t d16;
            float dq;
            const uint32_t q4 = dev::q8_quantize_lane4(qx[i], a.x86 != 0, &d16, &dq);
            uint16_t * qp = (uint16_t *) (image + x * 64 + (QBLOCK * blk + 2) % 16 + sub * 4);
            qp[0] = (uint16_t) q4;
            qp[1] = (uint16_t) (q4 >> 16);
            if (sub == 0) dql[x] = dq;
        }
        __syncthreads();
        v4i qw[NBLK];
        float dq[NBLK];                                    // dq c to 22 bits: PA_IBIAS dq is exact
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++) {
            qw[blk] = *(const v4i *) (image + (ln * NBLK + blk) * 64 + 16 * lg);
            const uint32_t x = __builtin_bit_cast(uint32_t, dql[ln * NBLK + blk] * a.c);
            dq[blk] = __builtin_bit_cast(float, (x + 2u) & ~3u);
        }
        __syncthreads();

        v4f O[NBLK][2] = {};
        float M = -INFINITY, l = 0.f;
        // the lane's row sees keys below it
        const int32_t limit = n - a.T + (int32_t) div_by((uint32_t) (16 * rg + ln), a.f_rep) + 1;
        if (wave < nt) {
            pa_wait_lds();
            send_v(at_v);
        }
        // in flight at the top, in this order: K of the tile, the entries of the next, V of the tile
        for (int t = wave; t < nt; t += PA_WAVES) {
            // the lane's places are computed anew in every tile: kept over the loop they cost 40 registers, spilled
            asm volatile("" : "+v"(lane), "+v"(ln), "+v"(lg));
            const int32_t key0 = (run.off + t) * PA_TILE;
            const bool masked = live != 0xffffffffu || key0 + PA_TILE > n - a.T + 1;
            pa_wait<ND + 1>();
            const uint8_t * const kt = my, * const vt = kt + C::ROWS;
            {   // K's scales by block and key
                const int key = lane & 31, half = lane >> 5;
#pragma unroll
                for (int i = 0; i < NBLK / 2; i++) {
                    const int blk = half * (NBLK / 2) + i;
                    kscl[blk * PA_TILE + key] = *(const uint16_t *) (kt + key * C::LS + QBLOCK * blk);
                }
            }
            wave_lds_sync();

            // S^T: lane (row ln, keys 16 u + 4 lg + r). An integer dot comes out of the MFMA on top of the bits of
            // PA_IBIAS, so it is PA_IBIAS + dot as a float, and one fused step makes dot dq of it.
            float s[2][4] = {};
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint8_t * kl = kt + (16 * u + ln) * C::LS + 16 * lg;
#pragma unroll
                for (int blk = 0; blk < NBLK; blk++) {
                    const v4i kw = *(const v4i *) (kl + 16 * pa_win(blk));
                    const uint2 dk = *(const uint2 *) (kscl + blk * PA_TILE + 16 * u + 4 * lg);
                    const v4i d = __builtin_amdgcn_mfma_i32_16x16x64_i8(kw, qw[blk], v4i{PA_IBITS, PA_IBITS, PA_IBITS, PA_IBITS}, 0, 0, 0);
                    const int d0 = d[0], d1 = d[1], d2 = d[2], d3 = d[3];
                    const float f = dq[blk], nb = -PA_IBIAS * f;
                    s[u][0] = fma_f16lo(dk.x, __fmaf_rn(__builtin_bit_cast(float, d0), f, nb), s[u][0]);
                    s[u][1] = fma_f16hi(dk.x, __fmaf_rn(__builtin_bit_cast(float, d1), f, nb), s[u][1]);
                    s[u][2] = fma_f16lo(dk.y, __fmaf_rn(__builtin_bit_cast(float, d2), f, nb), s[u][2]);
                    s[u][3] = fma_f16hi(dk.y, __fmaf_rn(__builtin_bit_cast(float, d3), f, nb), s[u][3]);
                }
            }
            const bool more = t + PA_WAVES < nt;
            pa_wait<ND>();
            if (more) {                                    // the next tile's K
                live_next = rows_of(t + PA_WAVES);
                wave_lds_sync();
                pa_wait_lds();
                send_k(at_k);
                entries(t + 2 * PA_WAVES);
                pa_wait<ND + 1>();
            } else {
                pa_wait<0>();
            }
            // V's scales; its largest of each key and of the tile. One that is not finite counts as 0 here and in
            // the products, and is added by itself below.
            uint32_t dmax = 0;
            bool odd = false;
            {
                const int key = lane & 31, half = lane >> 5;
                const bool on = live >> key & 1;
#pragma unroll
                for (int i = 0; i < NBLK / 2; i++) {
                    const int blk = half * (NBLK / 2) + i;
                    const uint32_t dv = *(const uint16_t *) (vt + key * C::LS + QBLOCK * blk), mag = dv & 0x7fffu;
                    const bool fine = on && mag < 0x7c00u;
                    vscl[blk * PA_TILE + key] = (uint16_t) (fine ? dv : 0u);
                    dmax = max(dmax, fine ? mag : 0u);
                    odd |= on && mag >= 0x7c00u;
                }
                dmax = umax_halves(dmax);
                if (half == 0) vtop[key] = (uint16_t) dmax;
            }
            dmax = umax_rows(umax_row(dmax));
            wave_lds_sync();
            float p[2][4];
            uint32_t top_d = dmax;
            if (masked) {
                top_d = 0;                                 // of the keys that the row sees
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int k = 16 * u + 4 * lg + r;
                        if (!(live >> k & 1) || key0 + k >= limit) s[u][r] = -INFINITY;
                        else top_d = max(top_d, (uint32_t) vtop[k]);
                    }
                top_d = umax_halves(umax_rows(top_d));
            }
            float top = vmax(vmax(s[0][0], s[0][1]), vmax(s[0][2], s[0][3]));
            top = vmax(top, vmax(vmax(s[1][0], s[1][1]), vmax(s[1][2], s[1][3])));
            top = xmax_lanes16_32(top);
            const int e = (int) (top_d >> 10) < 1 ? 1 : (int) (top_d >> 10);      // d < 2^(e - 14)
            const float ref = top + (float) (e - 14 - PA_BIAS);
            if (__ballot(ref > M + PA_SLACK)) {
                const float to = fmaxf(M, ref);
                const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - to);
                M = to;
                l *= f;
#pragma unroll
                for (int blk = 0; blk < NBLK; blk++) { O[blk][0] *= f; O[blk][1] *= f; }
            }
            const float m = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    p[u][r] = __builtin_amdgcn_exp2f(s[u][r] - m);       // 2^-inf = 0
                    l += p[u][r];
                }
            // O^T: A lane (dims 2 ln + e of the block, keys 4 lg + r of both halves)
#pragma unroll
            for (int blk = 0; blk < NBLK; blk++) {
                const uint8_t * vl = vt + 4 * lg * C::LS + QBLOCK * blk + 2 + 2 * ln;
                uint32_t av[2][4];
                uint2 dv[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
#pragma unroll
                    for (int r = 0; r < 4; r++) av[u][r] = *(const uint16_t *) (vl + (16 * u + r) * C::LS);
                    dv[u] = *(const uint2 *) (vscl + blk * PA_TILE + 16 * u + 4 * lg);
                }
                v4u a0, a1;
                cvt_v8(av, a0, a1);
                const v8h A0 = __builtin_bit_cast(v8h, a0), A1 = __builtin_bit_cast(v8h, a1);
                v4u bh, bl;
                hilo(p, dv, bh, bl);
                const v8h H = __builtin_bit_cast(v8h, bh), L = __builtin_bit_cast(v8h, bl);
                O[blk][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A0, H, O[blk][0], 0, 0, 0);
                O[blk][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A1, H, O[blk][1], 0, 0, 0);
                O[blk][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A0, L, O[blk][0], 0, 0, 0);
                O[blk][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A1, L, O[blk][1], 0, 0, 0);
            }
            if (__builtin_expect(__ballot(odd) != 0, 0)) {
                // blocks of V whose scale is not finite, for the rows that see their key
                for (int k = 0; k < PA_TILE; k++) {
                    const int from = (k >> 2 & 3) * 16 + ln;
                    float pk = 0.f;
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float y = __shfl(p[u][r], from);
                            if (k == 16 * u + (k & 12) + r) pk = y;
                        }
#pragma unroll
                    for (int blk = 0; blk < NBLK; blk++) {
                        const uint8_t * vb = vt + k * C::LS + QBLOCK * blk;
                        const uint16_t d = *(const uint16_t *) vb;
                        if ((d & 0x7fffu) < 0x7c00u || !(live >> k & 1)) continue;
#pragma unroll
                        for (int e2 = 0; e2 < 2; e2++)
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                if (pk != 0.f)
                                    O[blk][e2][r] += pk * dev::f16_bits_to_f32(d) * (float) *(const int8_t *) (vb + 2 + 2 * (4 * lg + r) + e2);
                    }
                }
            }
            if (more) {
                pa_wait_lds();
                send_v(at_v);
            }
            live = live_next;
        }
        pa_wait<0>();

        // the waves' parts meet in LDS: O[row][dim] of each
        const float ls = sum_lanes16_32(l);
        __syncthreads();
        float * ob = (float *) (lds + wave * C::WAVE) + ln * C::OROW;
#pragma unroll
        for (int blk = 0; blk < NBLK; blk++)
#pragma unroll
            for (int r = 0; r < 4; r += 2)
                *(float4 *) (ob + QK * blk + 8 * lg + 2 * r) =
                    make_float4(O[blk][0][r], O[blk][1][r], O[blk][0][r + 1], O[blk][1][r + 1]);
        if (lg == 0) ml[wave][ln] = make_float2(M, ls);
        __syncthreads();
        const int r = tid >> 4, rr = 16 * rg + r;
        float2 e[PA_WAVES];
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < PA_WAVES; w++) { e[w] = ml[w][r]; mm = fmaxf(mm, e[w].x); }
#pragma unroll
        for (int w = 0; w < PA_WAVES; w++) {
            e[w].x = e[w].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(e[w].x - mm);
            ll += e[w].x * e[w].y;                         // a NaN stays one
        }
        if (rr < a.R) {
            const size_t elem = element(b, rr), part = ((size_t) (g + b) * a.nh_kv + kvh) * a.R + rr;
            const float inv = ll > 0.f ? 1.f / ll : ll == ll ? 0.f : ll;
#pragma unroll
            for (int i = 0; i < D / 64; i++) {
                const int d0 = 4 * (tid & 15) + 64 * i;
                float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < PA_WAVES; w++) {
                    const float4 x = *(const float4 *) ((const float *) (lds + w * C::WAVE) + r * C::OROW + d0);
                    if (e[w].x != 0.f) {
                        o[0] += e[w].x * x.x; o[1] += e[w].x * x.y; o[2] += e[w].x * x.z; o[3] += e[w].x * x.w;
                    }
                }
                if (whole) {
#pragma unroll
                    for (int k = 0; k < 4; k++) o[k] *= inv;
                    finish4(a, elem + d0, o);
                } else {
                    *(float4 *) (a.part_o + part * D + d0) = make_float4(o[0], o[1], o[2], o[3]);
                }
            }
            if (!whole && (tid & 15) == 0) a.part_ml[part] = make_float2(mm, ll);
        }
        if (run.off == 0 && hr == 0 && tid == 0) a.span[b] = make_int2(g, (run.pos + tiles - 1) / run.per);
        run.left -= nt;
        run.pos += nt;
        run.off = -PA_LEAD;
        if (run.left > 0)
            do run.n = clip_len(a, a.n_kv[++run.b]);
            while (run.n == 0);
    }
    // requests without a key, and lengths that were clipped
    for (int b = g; b < a.n_seq; b += (int) (gridDim.x / a.f_inner.d)) {
        const int32_t n = a.n_kv[b];
        if (n != clip_len(a, n) && tid == 0) atomicOr(a.status, DEVERR_GET_ROWS_INDEX);
        if (n > 0) continue;
        const float z[4] = {0.f, 0.f, 0.f, 0.f};
        for (int r = tid >> 4; r < 16; r += PA_THREADS / 16)
            if (16 * rg + r < a.R)
#pragma unroll
                for (int i = 0; i < D / 64; i++) store4(a.dst + (element(b, 16 * rg + r) + 4 * (tid & 15) + 64 * i) * es, a.type, z);
        if (hr == 0 && tid == 0) a.span[b] = make_int2(0, 0);
    }
}

// The parts of a request joined, log-sum-exp weights: GROUPS groups of 16 lanes a query row and 64 of its dims,
// each taking every GROUPS-th part, PM_BATCH of them in flight. A wave (4 groups) where a request has a few parts, a
// workgroup (16) where it has many. Requests of one part are done.
constexpr int PM_BATCH = 8;

template <int D, int GROUPS>
__global__ __launch_bounds__(256) void k_paged_merge(pa_args a) {
    __shared__ float4 acc[16][16];
    __shared__ float2 gl[16];
    const int sub = GROUPS == 16 ? 0 : (int) threadIdx.x >> 6;
    const int64_t unit = GROUPS == 16 ? (int64_t) blockIdx.x : (int64_t) blockIdx.x * 4 + sub;
    const int quarter = (int) (unit % (D / 64));
    const uint32_t row = (uint32_t) (unit / (D / 64)), bk = row / (uint32_t) a.R, r = row - bk * (uint32_t) a.R;
    const uint32_t b = div_by(bk, a.f_kv), kvh = bk - b * (uint32_t) a.nh_kv;
    const bool on = b < (uint32_t) a.n_seq;
    const int2 sp = on ? a.span[b] : make_int2(0, 0);
    if (GROUPS == 16 && sp.x == sp.y) return;
    const int g = (int) (threadIdx.x >> 4) % GROUPS, q = threadIdx.x & 15;
    float M = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (sp.x != sp.y) {
        const size_t step = (size_t) a.nh_kv * a.R;
        const size_t p0 = ((size_t) (sp.x + (int) b) * a.nh_kv + kvh) * a.R + r;
        const float * po = a.part_o + p0 * D + 64 * quarter + 4 * q;
        const int n = sp.y - sp.x + 1;
        for (int s0 = g; s0 < n; s0 += GROUPS * PM_BATCH) {
            float2 e[PM_BATCH];
            float4 x[PM_BATCH];
            float to = M;
#pragma unroll
            for (int i = 0; i < PM_BATCH; i++) {
                const int s = s0 + i * GROUPS < n ? s0 + i * GROUPS : s0;
                e[i] = a.part_ml[p0 + s * step];
                x[i] = *(const float4 *) (po + s * step * D);
            }
#pragma unroll
            for (int i = 0; i < PM_BATCH; i++) {
                if (s0 + i * GROUPS >= n) e[i] = make_float2(-INFINITY, 0.f);
                to = fmaxf(to, e[i].x);
            }
            const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - to);
            o.x *= f; o.y *= f; o.z *= f; o.w *= f;
            l *= f;
#pragma unroll
            for (int i = 0; i < PM_BATCH; i++) {
                const float w = e[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(e[i].x - to);
                l += w * e[i].y;                           // a NaN stays one
                if (w != 0.f) { o.x += w * x[i].x; o.y += w * x[i].y; o.z += w * x[i].z; o.w += w * x[i].w; }
            }
            M = to;
        }
    }
    const int slot = sub * GROUPS % 16 + g;
    acc[slot][q] = o;
    if (q == 0) gl[slot] = make_float2(M, l);
    __syncthreads();
    if (g == 0 && sp.x != sp.y) {
        float mm = -INFINITY, ll = 0.f;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < GROUPS; i++) mm = fmaxf(mm, gl[slot + i].x);
#pragma unroll
        for (int i = 0; i < GROUPS; i++) {
            const float w = gl[slot + i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(gl[slot + i].x - mm);
            const float4 v = acc[slot + i][q];
            ll += w * gl[slot + i].y;
            if (w != 0.f) { x[0] += w * v.x; x[1] += w * v.y; x[2] += w * v.z; x[3] += w * v.w; }
        }
        const float inv = ll > 0.f ? 1.f / ll : ll == ll ? 0.f : ll;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] *= inv;
        const uint32_t t = div_by(r, a.f_rep), h = kvh * (uint32_t) a.rep + r - t * (uint32_t) a.rep;
        finish4(a, (((size_t) b * a.T + t) * a.nh + h) * D + 64 * quarter + 4 * q, x);
    }
}

// ---------------------------------------------------------------- host

struct pa_plan {
    int32_t groups, runs;              // row groups
    size_t  off_o, off_ml, bytes;
};

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Runs: as many as fill the CUs; no more than the longest requests could need. (Run g is on XCD g mod 8. Their number is
// whole rounds of the 8 XCDs where heads and row groups divide 64; 85 runs, of 2 heads in 3 groups, leave some XCDs with 11
// for the others' 10.)
pa_plan plan_paged(int64_t D, int64_t T, int64_t nh, int64_t nh_kv, int64_t n_seq, int64_t max_kv) {
    pa_plan p;
    const int64_t R = T * (nh / nh_kv);
    p.groups = (int32_t) ((R + 15) / 16);
    const int64_t most = (n_seq * ((max_kv + PA_TILE - 1) / PA_TILE + PA_LEAD) + PA_MIN_TILES - 1) / PA_MIN_TILES;
    p.runs = (int32_t) std::max<int64_t>(1, std::min<int64_t>(2 * PA_CUS / (nh_kv * p.groups), most));
    const size_t parts = (size_t) (p.runs + n_seq) * nh_kv * R;
    p.off_o = round256((size_t) n_seq * sizeof(int2));
    p.off_ml = p.off_o + round256(parts * D * sizeof(float));
    p.bytes = p.off_ml + round256(parts * sizeof(float2));
    return p;
}

int check_paged(const qwfn_tensor * q, const qwfn_tensor * k, const qwfn_tensor * v, int32_t max_pages, int32_t page_size,
                pa_plan * pl) {
    const char * op = "flash_attn_ext_paged";
    auto err = [&](int code, const char * what) { return set_error2(code, op, what); };
    if (!q || !q->data || !k || !k->data || !v || !v->data) return err(QWFN_EINVAL, ": q, k or v is NULL");
    if (q->type != QWFN_TYPE_F32 && q->type != QWFN_TYPE_F16 && q->type != QWFN_TYPE_BF16)
        return err(QWFN_EINVAL, ": q must be f32, f16 or bf16");
    if (k->type != QWFN_TYPE_Q8_0 || v->type != QWFN_TYPE_Q8_0) return err(QWFN_EINVAL, ": k and v must be q8_0");
    for (int i = 0; i < 4; i++)
        if (q->ne[i] < 1 || k->ne[i] < 1) return err(QWFN_EINVAL, ": empty tensor");
    const int64_t D = q->ne[0], T = q->ne[1], nh = q->ne[2], B = q->ne[3], nh_kv = k->ne[2];
    if (D != 64 && D != 128 && D != 256) return err(QWFN_ENOTSUP, ": head size must be 64, 128 or 256");
    if (k->ne[0] != D) return err(QWFN_EINVAL, ": q and k head sizes differ");
    if (k->ne[3] != 1) return err(QWFN_ENOTSUP, ": k and v are one pool (ne[3] == 1)");
    if (nh % nh_kv) return err(QWFN_EINVAL, ": n_head must be a multiple of n_head_kv");
    if (T > PA_MAX_ROWS || T * (nh / nh_kv) > PA_MAX_ROWS)
        return err(QWFN_ENOTSUP, ": at most 64 query rows per KV head (T * n_head / n_head_kv)");
    if (nh_kv > 128) return err(QWFN_ENOTSUP, ": at most 128 KV heads");
    if (page_size < 1 || max_pages < 1 || (int64_t) page_size * max_pages > 0x7fffffff - 2 * PA_TILE * PA_WAVES)
        return err(QWFN_EINVAL, ": page_size and max_pages must be positive, their product below 2^31 - 256");
    if (B > 65536 || B * ((int64_t) page_size * max_pages / PA_TILE + 1 + PA_LEAD) > 0x7ffff000)
        return err(QWFN_ENOTSUP, ": at most 65536 requests and 2^31 tiles of 32 keys");
    // (a wave of the merge a row and 64 dims, and a launch has below 2^32 threads)
    if (B * nh * T * (D / 64) >= 1 << 26) return err(QWFN_ENOTSUP, ": too many query rows");
    if (k->ne[1] < page_size) return err(QWFN_EINVAL, ": the pool holds no whole page");
    if (k->ne[1] > 0x7fffffff) return err(QWFN_ENOTSUP, ": a pool of at most 2^31 - 1 rows");
    *pl = plan_paged(D, T, nh, nh_kv, B, (int64_t) page_size * max_pages);
    return QWFN_OK;
}

template <int D>
int launch_paged(const pa_args & a, const pa_plan & p, hipStream_t s) {
    const dim3 grid((unsigned) ((int64_t) (a.runs + 7) / 8 * 8 * a.nh_kv * p.groups));
    hipLaunchKernelGGL(k_paged_attn<D>, grid, dim3(PA_THREADS), 0, s, a);
    if (int rc = hip_check(hipGetLastError(), "flash_attn_ext_paged launch")) return rc;
    // the requests' parts: on average runs / n_seq each, with long requests among short ones more
    const int64_t units = (int64_t) a.n_seq * a.nh_kv * a.R * (D / 64);
    if (a.runs > 16 * (int64_t) a.n_seq)
        hipLaunchKernelGGL((k_paged_merge<D, 16>), dim3((unsigned) units), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((k_paged_merge<D, 4>), dim3((unsigned) ((units + 3) / 4)), dim3(256), 0, s, a);
    return hip_check(hipGetLastError(), "flash_attn_ext_paged launch");
}

}  // namespace
}  // namespace qwfn

using namespace qwfn;

extern "C" size_t qwfn_fattn_workspace_size_paged(const qwfn_tensor * q, const qwfn_tensor * k, const qwfn_tensor * v,
                                                  int32_t max_pages, int32_t page_size) {
    return ::qwfn::abi_value<size_t>("fattn_workspace_size_paged", 0, [&]() -> size_t {
        pa_plan pl;
        return check_paged(q, k, v, max_pages, page_size, &pl) ? 0 : pl.bytes;
    });
}

extern "C" int qwfn_flash_attn_ext_q8_0_paged(const qwfn_tensor * q, const qwfn_tensor * k, const qwfn_tensor * v,
                                              const int32_t * table, int64_t table_stride, int32_t max_pages,
                                              int32_t page_size, const int32_t * n_kv, float scale, const qwfn_tensor * gate,
                                              const qwfn_tensor * dst, int variant, void * ws, size_t ws_bytes,
                                              void * stream) {
    return ::qwfn::abi_call("flash_attn_ext_paged", [&]() -> int {
        auto err = [&](int code, const char * what) { return set_error2(code, "flash_attn_ext_paged", what); };
        pa_plan pl;
        if (int rc = check_paged(q, k, v, max_pages, page_size, &pl)) return rc;
        if (!table || !n_kv || !dst || !dst->data) return err(QWFN_EINVAL, ": table, n_kv or dst is NULL");
        if (!std::isfinite(scale)) return err(QWFN_EINVAL, ": scale must be finite");
        if (variant != QWFN_Q8_REF && variant != QWFN_Q8_X86) return err(QWFN_EINVAL, ": unknown rounding variant");
        const int64_t D = q->ne[0], T = q->ne[1], nh = q->ne[2], B = q->ne[3], nh_kv = k->ne[2];
        const size_t es = q->type == QWFN_TYPE_F32 ? 4 : 2, seg = (size_t) D / QK * QBLOCK, al = (size_t) D / 16;
        for (int i = 0; i < 4; i++)
            if (v->ne[i] != k->ne[i] || (i < 3 && v->nb[i] != k->nb[i]))
                return err(QWFN_EINVAL, ": k and v must have the same shape and strides");
        if (k->nb[0] != QBLOCK) return err(QWFN_EINVAL, ": k and v nb[0] must be 34");
        if (!is_aligned(k->data, al) || !is_aligned(v->data, al) || k->nb[1] % al || k->nb[2] % al)
            return err(QWFN_EALIGN, ": k and v rows and strides must be aligned to head size / 16 bytes");
        if (k->nb[1] > 0xffffffffu) return err(QWFN_ENOTSUP, ": a row stride of 2^32 bytes or more");
        // heads inside a row, or rows inside a head
        if (k->nb[1] < (size_t) (nh_kv - 1) * k->nb[2] + seg && k->nb[2] < (size_t) (k->ne[1] - 1) * k->nb[1] + seg)
            return err(QWFN_EINVAL, ": k and v rows or heads overlap");
        if (k->nb[1] < seg || (nh_kv > 1 && k->nb[2] < seg)) return err(QWFN_EINVAL, ": k and v rows or heads overlap");
        if (q->nb[0] != es) return err(QWFN_EINVAL, ": q rows must be contiguous");
        if (!is_aligned(q->data, 16) || q->nb[1] % 16 || q->nb[2] % 16 || q->nb[3] % 16)
            return err(QWFN_EALIGN, ": q must be 16-byte aligned");
        const int64_t ne[4] = {D, nh, T, B};
        for (int g = 0; g < 2; g++) {
            const qwfn_tensor * t = g ? gate : dst;
            if (!t) continue;
            if (!t->data || t->type != q->type) return err(QWFN_EINVAL, g ? ": gate must have q's type" : ": dst must have q's type");
            size_t nb = es;
            for (int i = 0; i < 4; i++) {
                if (t->ne[i] != ne[i] || t->nb[i] != nb)
                    return err(QWFN_EINVAL, g ? ": gate must be contiguous [D, n_head, T, n_seq]" : ": dst must be contiguous [D, n_head, T, n_seq]");
                nb *= (size_t) ne[i];
            }
            if (!is_aligned(t->data, 16)) return err(QWFN_EALIGN, g ? ": gate must be 16-byte aligned" : ": dst must be 16-byte aligned");
        }
        if (table_stride < max_pages && B > 1) return err(QWFN_EINVAL, ": table rows overlap (table_stride < max_pages)");
        if (table_stride > 0x7fffffff) return err(QWFN_EINVAL, ": table_stride must be below 2^31");
        if (!is_aligned(table, 4) || !is_aligned(n_kv, 4)) return err(QWFN_EALIGN, ": table and n_kv must be 4-byte aligned");
        if (ws && !is_aligned(ws, 16)) return err(QWFN_EALIGN, ": ws must be 16-byte aligned");
        if (ws && ws_bytes < pl.bytes) return err(QWFN_ENOMEM, ": ws smaller than qwfn_fattn_workspace_size_paged");
        // (a request's queries are read by several workgroups, and one of them may be done before another begins)
        const size_t rows = tensor_extent(dst);
        const span in[] = {{q->data, tensor_extent(q), "q"}, {k->data, view_bytes(*k), "k"}, {v->data, view_bytes(*v), "v"},
                           {gate && gate->data != dst->data ? gate->data : nullptr, rows, "gate"},
                           {table, ((size_t) (B - 1) * table_stride + max_pages) * 4, "table"}, {n_kv, (size_t) B * 4, "n_kv"}};
        const span out[] = {{dst->data, rows, "dst"}, {ws, pl.bytes, "ws"}};
        if (int rc = check_overlaps("flash_attn_ext_paged", in, 6, out, 2)) return rc;
        if (!ws) {
            size_t got = 0;
            if (int rc = library_workspace(pl.bytes, pl.bytes, as_stream(stream), &ws, &got)) return rc;
        }
        pa_args a{};
        if (int rc = status_word(&a.status)) return rc;
        a.q = (const char *) q->data; a.q_nb1 = q->nb[1]; a.q_nb2 = q->nb[2]; a.q_nb3 = q->nb[3];
        a.k = (const char *) k->data; a.v = (const char *) v->data; a.nb1 = (uint32_t) k->nb[1]; a.nb2 = k->nb[2];
        a.n_pages = k->ne[1] / page_size;
        a.table = table; a.t_stride = table_stride; a.n_kv = n_kv; a.max_kv = (int64_t) max_pages * page_size;
        a.page = make_div((uint32_t) page_size);
        a.gate = gate ? (const char *) gate->data : nullptr; a.dst = (char *) dst->data; a.type = q->type;
        a.n_seq = (int32_t) B; a.T = (int32_t) T; a.nh = (int32_t) nh; a.nh_kv = (int32_t) nh_kv;
        a.rep = (int32_t) (nh / nh_kv); a.R = a.T * a.rep; a.x86 = variant == QWFN_Q8_X86;
        a.f_runs = make_div((uint32_t) pl.runs); a.f_inner = make_div((uint32_t) (nh_kv * pl.groups));
        a.f_kv = make_div((uint32_t) nh_kv); a.f_rep = make_div((uint32_t) a.rep);
        a.runs = pl.runs; a.c = scale * PA_LOG2E;
        a.span = (int2 *) ws; a.part_o = (float *) ((char *) ws + pl.off_o); a.part_ml = (float2 *) ((char *) ws + pl.off_ml);
        switch (D) {
            case 64:  return launch_paged<64>(a, pl, as_stream(stream));
            case 128: return launch_paged<128>(a, pl, as_stream(stream));
            default:  return launch_paged<256>(a, pl, as_stream(stream));
        }
    });
}
