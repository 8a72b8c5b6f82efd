// Linear attention with a decay per head over a ragged batch:
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
// per value head, state S [dk][dv] in F32 (q and k of key head h / (n_v / n_k)).
//
// Token by token (k_linear_step): columns of S are independent. A workgroup takes 64
// columns of one head of one sequence, thread (row group rg, column quad cq) the
// rows rg + 16 i; the state stays in registers for the sequence's tokens and is
// read and written once. The output's sum over rows is finished across the lanes
// (permlane swaps) and the waves (LDS), in a fixed order, one barrier a token.
// What bounds it: the state, 8 dk dv bytes a head and sequence (64 sequences of one
// bf16 token, 48 heads of 128: 407 MB in 82 us, 5.0 TB/s, a copy's rate). Calls of
// more than a few tokens a sequence run in chunks (below).
#include "fattn_device.h"
#include "qwfn_common.h"
#include "qwfn_state.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace qwfn {
namespace {

constexpr int LA_THREADS = 256;
constexpr int LA_COLS = 64;            // columns of a workgroup
constexpr int LA_TC = 8;               // tokens whose q and k are brought in at once
constexpr int64_t LA_BLOCKS = 0xffffff;    // of a launch: below 2^32 threads

struct la_args {
    const char * q; const char * k; const char * v; char * out;
    int64_t      q_nb1, q_nb2, k_nb1, k_nb2, v_nb1, v_nb2;      // bytes between heads and tokens
    const float * g; int64_t g_ts;
    const int32_t * cu; const int32_t * slots;
    const float * s_in; float * s_out;
    float        scale;
    int32_t      type, n_seq, max_len, n_slots, n_tok, n_k, n_v, rep, dk, dv, ct;
    uint32_t *   status;
};

// 4 consecutive values of type T at p
__device__ __forceinline__ float4 la_load4(const char * p, int32_t type) {
    if (type == QWFN_TYPE_F32) return *(const float4 *) p;
    const uint2 u = *(const uint2 *) p;
    if (type == QWFN_TYPE_BF16)
        return make_float4(__builtin_bit_cast(float, u.x << 16), __builtin_bit_cast(float, u.x & 0xffff0000u),
                           __builtin_bit_cast(float, u.y << 16), __builtin_bit_cast(float, u.y & 0xffff0000u));
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const v2h a = __builtin_bit_cast(v2h, u.x), b = __builtin_bit_cast(v2h, u.y);
    return make_float4((float) a[0], (float) a[1], (float) b[0], (float) b[1]);
}
__device__ __forceinline__ uint32_t la_pack2(float x, float y, int32_t type) {
    if (type == QWFN_TYPE_BF16)
        return (uint32_t) __builtin_bit_cast(uint16_t, (__bf16) x) | (uint32_t) __builtin_bit_cast(uint16_t, (__bf16) y) << 16;
    return (uint32_t) __builtin_bit_cast(uint16_t, (_Float16) x) | (uint32_t) __builtin_bit_cast(uint16_t, (_Float16) y) << 16;
}
__device__ __forceinline__ void la_store4(char * p, int32_t type, float4 x) {
    if (type == QWFN_TYPE_F32) *(float4 *) p = x;
    else *(uint2 *) p = make_uint2(la_pack2(x.x, x.y, type), la_pack2(x.z, x.w, type));
}

// Sequence b: its first token and its length, its state's slot (-1: none), and the slot of a sequence that is left out
// (then len is 0; -1: none).
struct la_seq { int32_t t0, len, slot, held; };
__device__ __forceinline__ la_seq la_sequence(const la_args & a, int b, bool report) {
    auto clip = [&](int32_t x) { return x < 0 ? 0 : x > a.n_tok ? a.n_tok : x; };
    const int32_t c0 = a.cu[b], c1 = a.cu[b + 1], lo = clip(c0), hi = clip(c1);
    int32_t len = hi - lo, slot = a.slots ? a.slots[b] : b;
    bool bad = lo != c0 || hi != c1 || len < 0 || len > a.max_len;
    len = len < 0 ? 0 : len > a.max_len ? a.max_len : len;
    int32_t held = -1;
    if (slot < 0 || slot >= a.n_slots) {
        if (slot < -1 && -2 - slot < a.n_slots) {
            held = -2 - slot;
            len = 0;
        } else {
            bad |= slot != -1;
        }
        slot = -1;
    }
    if (bad && report) atomicOr(a.status, DEVERR_SET_ROWS_INDEX);
    return {lo, len, slot, held};
}

// The state of head h of a sequence that is left out, from one buffer to the other: thread i of n.
__device__ __forceinline__ void la_carry(const la_args & a, int32_t held, int h, int i, int n) {
    if (held < 0 || a.s_in == a.s_out) return;
    const size_t head = ((size_t) held * a.n_v + h) * a.dk * a.dv;
    for (int e = i; 4 * e < a.dk * a.dv; e += n)
        *(float4 *) (a.s_out + head + 4 * e) = a.s_in ? *(const float4 *) (a.s_in + head + 4 * e) : make_float4(0.f, 0.f, 0.f, 0.f);
}

template <int DK>
__global__ __launch_bounds__(LA_THREADS) void k_linear_step(la_args a) {
    constexpr int RPT = DK / 16;               // rows of a thread
    __shared__ float kq[LA_TC][2][DK];
    __shared__ float4 red[2][LA_THREADS / 64][16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, cq = tid & 15, rg = tid >> 4;
    const int cb = blockIdx.x % a.ct, h = blockIdx.x / a.ct % a.n_v, b = blockIdx.x / a.ct / a.n_v;
    const la_seq s = la_sequence(a, b, tid == 0 && cb == 0 && h == 0);
    if (s.len == 0) {
        la_carry(a, s.held, h, cb * LA_THREADS + tid, a.ct * LA_THREADS);
        return;
    }
    const int c = cb * LA_COLS + 4 * cq;
    const bool on = c < a.dv;                  // dv is a multiple of 16
    const size_t state = (size_t) a.n_v * a.dk * a.dv;
    const size_t sh = (size_t) h * a.dk * a.dv + c;
    float4 S[RPT];
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        const int r = rg + 16 * i;
        S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on && s.slot >= 0 && a.s_in && r < a.dk) S[i] = *(const float4 *) (a.s_in + s.slot * state + sh + (size_t) r * a.dv);
    }
    const int es = a.type == QWFN_TYPE_F32 ? 4 : 2;
    const char * qh = a.q + (int64_t) (h / a.rep) * a.q_nb1, * kh = a.k + (int64_t) (h / a.rep) * a.k_nb1;
    const char * vh = a.v + (int64_t) h * a.v_nb1 + (int64_t) c * es;
    char * oh = a.out + ((int64_t) h * a.dv + c) * es;
    const int64_t o_ts = (int64_t) a.n_v * a.dv * es;
    for (int t0 = 0; t0 < s.len; t0 += LA_TC) {
        const int nt = s.len - t0 < LA_TC ? s.len - t0 : LA_TC;
        if (t0 > 0) __syncthreads();
        for (int u = tid; u < nt * 2 * (DK / 4); u += LA_THREADS) {
            const int e4 = u % (DK / 4), x = u / (DK / 4), tt = x >> 1;
            const int64_t t = s.t0 + t0 + tt;
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (4 * e4 < a.dk) f = la_load4((x & 1 ? qh + t * a.q_nb2 : kh + t * a.k_nb2) + 4 * e4 * es, a.type);
            *(float4 *) &kq[tt][x & 1][4 * e4] = f;
        }
        __syncthreads();
        for (int tt = 0; tt < nt; tt++) {
            const int64_t t = s.t0 + t0 + tt;
            const float e = expf(a.g[t * a.g_ts + h]);
            const float4 v = on ? la_load4(vh + t * a.v_nb2, a.type) : make_float4(0.f, 0.f, 0.f, 0.f);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < RPT; i++) {
                const float kr = kq[tt][0][rg + 16 * i], qr = kq[tt][1][rg + 16 * i];
                S[i].x = __fmaf_rn(kr, v.x, S[i].x * e); S[i].y = __fmaf_rn(kr, v.y, S[i].y * e);
                S[i].z = __fmaf_rn(kr, v.z, S[i].z * e); S[i].w = __fmaf_rn(kr, v.w, S[i].w * e);
                if (rg + 16 * i < a.dk) {
                    o.x = __fmaf_rn(S[i].x, qr, o.x); o.y = __fmaf_rn(S[i].y, qr, o.y);
                    o.z = __fmaf_rn(S[i].z, qr, o.z); o.w = __fmaf_rn(S[i].w, qr, o.w);
                }
            }
            o.x = sum_lanes16_32(o.x); o.y = sum_lanes16_32(o.y); o.z = sum_lanes16_32(o.z); o.w = sum_lanes16_32(o.w);
            if (lane < 16) red[tt & 1][w][cq] = o;
            __syncthreads();
            if (tid < 16 && on) {
                float4 x = red[tt & 1][0][cq];
#pragma unroll
                for (int i = 1; i < LA_THREADS / 64; i++) {
                    const float4 y = red[tt & 1][i][cq];
                    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
                }
                la_store4(oh + t * o_ts, a.type, make_float4(x.x * a.scale, x.y * a.scale, x.z * a.scale, x.w * a.scale));
            }
        }
    }
    if (on && s.slot >= 0) {
#pragma unroll
        for (int i = 0; i < RPT; i++) {
            const int r = rg + 16 * i;
            if (r < a.dk) *(float4 *) (a.s_out + s.slot * state + sh + (size_t) r * a.dv) = S[i];
        }
    }
}

// ---------------------------------------------------------------- in chunks
//
// Chunks of C tokens as matrix products, G the sum of g from the chunk's start
// (inclusive), S the state before it:
//   o_i = scale (e^{G_i} S^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j)
//   S'  = e^{G_C} S + sum_j k_j (e^{G_C - G_j} v_j)^T
// on the bf16 matrix cores (v_mfma_f32_16x16x32_bf16), F32 accumulators. A value
// enters as NT bf16 terms, each the rounded rest of the ones before: bf16 is one
// term, f16 two (its 11 bits exactly), f32 three (24 bits exactly); a product keeps
// the pairs of terms that reach NT terms' accuracy. The state's update always
// takes three terms of e^{G_C - G_j} v_j, so the state stays an F32 sum whatever the
// type; on the way to an output the state and the weighted scores are rounded to NT
// terms, two at least (2^-16 of each: an output is off by its own rounding, 1.7e-3 of the
// result in bf16, whether its tokens run in chunks or one by one; with one term it was
// 2.3e-3, and 4096 tokens took 101 us for 113, replayed from a graph).
// G and its differences are F64: a chunk's strong decays leave the weak ones exact.
// A decay below e^-1000 counts as e^-1000, which is 0 in F32, so -inf is exact.
//
// A workgroup takes 32 columns a wave, its state in the waves' accumulators: lane m
// of wave w, tile u holds column 32 w + 8 (m >> 2) + 4 u + (m & 3), rows
// 32 (t / 2) + 8 (l >> 4) + 4 (t & 1) + r of 16-row tile t. So the state is the A
// operand of S^T q as it lies, two tiles the 32 rows of a block in their order, and
// O^T has 8 consecutive columns of a token in a lane: no data moves between the
// products but the scores, which the waves share through LDS. q, k and v lie in LDS as
// in memory, by rows; k^T and v^T are read by the transposing LDS reads, so each
// value is stored once (with written transposes F32 of dk 128 had one workgroup a CU
// instead of two, and 16 ragged F16 sequences of 32 heads of 64 took 122 us for 102).
// bf16 goes to LDS as it is, by LDS DMA into two buffers, a chunk ahead: no registers
// hold it and a chunk has two barriers. f16 and f32 are taken apart on the way, the
// next chunk waits in registers, and a chunk has three.
// What bounds it: 4096 bf16 tokens of 48 heads of 128 move 134 MB of q, k, v and o and
// the parts' states another 190 MB, 63 us at the rate of a copy, and take 104 in calls one
// after another; the vector units are busy 45 % of the last launch (the state's scaling and
// its roundings), the matrix cores 21 %, the rest are the waits between a chunk's
// dependent products.
//
// A non-finite v_j must not reach tokens before j: a chunk that holds one takes its
// scores times v by plain sums over j <= i. (The rest of a term of an infinity is NaN, so an
// infinity comes out as NaN in its column where the recurrence may leave an infinity.)
//
// A long sequence is cut into parts that run at once: k_linear_chunks<.., true> leaves
// each part's own contribution U to the state and its decay in the workspace,
// k_linear_join makes the state before each part of them, and the third launch runs
// the parts from there.
typedef __bf16   v8b __attribute__((ext_vector_type(8)));
typedef __bf16   v2b __attribute__((ext_vector_type(2)));
typedef uint32_t v4w __attribute__((ext_vector_type(4)));
typedef uint32_t v2w __attribute__((ext_vector_type(2)));

constexpr int LC_WCOLS = 32;           // columns of a wave
constexpr double LC_LOG2E = 1.4426950408889634;
constexpr float LC_FLOOR = -1000.f;

struct lc_args {
    la_args   a;
    int32_t   L;                       // tokens of a part, a multiple of the chunk; 0: sequences are whole
    int32_t   parts;                   // that the workspace has room for
    int32_t   KT, US;                  // row tiles of a state, values of one in the workspace
    float *   U;                       // [part][n_v][wave's columns][row tile][column tile][lane][4], as the lanes hold them
    double *  G;                       // [part][n_v]: log2 of the part's decay
};

constexpr int LC_C = 32;               // tokens of a chunk: the sum of one MFMA

template <int NT, int DK, int NW> struct lc_cfg {
    static constexpr int KT = DK / 16, KB = DK / 32;
    static constexpr int COLS = LC_WCOLS * NW, THREADS = 64 * NW;
    static constexpr int OT = NT == 1 ? 2 : NT;          // terms of the state and of the scores on their way to an output
    static constexpr int ES = NT == 3 ? 4 : 2;           // bytes of a value
    static constexpr int LPU = NT == 3 ? 2 : 1;          // 16-byte loads of 8 values
    static constexpr bool DMA = NT == 1;                 // bf16 goes to LDS as it is
    // a staged unit: 8 values of a token; a thread's units of q and of k, and of v
    static constexpr int KU = LC_C * (DK / 8) / THREADS, VU = LC_C * (COLS / 8) / THREADS;
    static constexpr int QK = LC_C * DK * 2, V = LC_C * COLS * 2, P = LC_C * LC_C * 2;     // bytes of a term
    static constexpr int OQ = 0, OK = OQ + NT * QK, OV = OK + NT * QK, BUF = OV + NT * V, OP = (DMA ? 2 : 1) * BUF, LDS = OP + OT * P;
    // workgroups of a CU: by LDS, and three waves a SIMD (168 registers each), two with a chunk in registers, one with a
    // state of 256 rows
    static constexpr int WAVES = DK == 256 ? 4 : DMA ? 12 : 8;
    static constexpr int PER_CU = 160 * 1024 / (LDS + 1280) < WAVES / NW ? 160 * 1024 / (LDS + 1280) : WAVES / NW;
    static constexpr int WAVES_EU = (PER_CU * NW + 3) / 4;
    static_assert(KU * THREADS == LC_C * (DK / 8) && VU * THREADS == LC_C * (COLS / 8), "whole units a thread");
    static_assert(LDS + 2048 <= 160 * 1024, "LDS of a CU");
};

// Byte of a 16-byte unit in the rows of q, k and v ([token][W values]): the 16 rows of a row read, and the 4 rows by 4
// units of 16 lanes of a transposing read, lie in different banks.
template <int W> __device__ __forceinline__ int lc_place(int row) {       // exclusive or of a row's units
    return W == 64 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3);
}
template <int W> __device__ __forceinline__ int lc_row(int row, int unit) { return row * (W * 2) + ((unit ^ lc_place<W>(row)) * 16); }
// Byte of a 16-byte unit in the scores ([token i][token j]).
__device__ __forceinline__ int lc_score(int row, int unit) { return row * (LC_C * 2) + ((unit ^ (row >> 1 & 3)) * 16); }
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
    return __builtin_bit_cast(uint32_t, v2b{(__bf16) x, (__bf16) y});
}
// x and y as NT bf16 terms, packed by term
template <int NT> __device__ __forceinline__ void bf16_terms(float x, float y, uint32_t (&t)[NT]) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
        t[i] = bf16_pair(x, y);
        if (i + 1 < NT) {
            x -= __builtin_bit_cast(float, t[i] << 16);
            y -= __builtin_bit_cast(float, t[i] & 0xffff0000u);
        }
    }
}
// Lane m of 16-lane group g: column 8 (m >> 2) + 4 half + (m & 3) of the 32 columns from unit 4 ub, of the 8 rows from
// `row` (8 g from a 32-row block): ds_read_b64_tr_b16 takes 4 rows of 16 values, 4 a lane, and gives a lane a column.
template <int W> __device__ __forceinline__ v4w lc_transposed(uint8_t * rows, int row, int ub, int half, int m) {
    typedef int16_t v4h __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4h * lp;
    const int r = row + (m >> 2), u = 4 * ub + (m & 3);
    const v2w x = __builtin_bit_cast(v2w, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp) (rows + lc_row<W>(r, u) + 8 * half)));
    const v2w y = __builtin_bit_cast(v2w, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp) (rows + lc_row<W>(r + 4, u) + 8 * half)));
    return v4w{x[0], x[1], y[0], y[1]};
}
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __builtin_bit_cast(float, u & 0xffff0000u); }
__device__ __forceinline__ v4f mfma_bf16(v4w x, v4w y, v4f z) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, x), __builtin_bit_cast(v8b, y), z, 0, 0, 0);
}
// sum over the pairs of terms whose product reaches NT terms' accuracy, the small ones first
template <int NX, int NY, int NT> __device__ __forceinline__ v4f mfma_terms(const v4w (&x)[NX], const v4w (&y)[NY], v4f z) {
#pragma unroll
    for (int s = NT - 1; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < NX; i++)
            if (s - i >= 0 && s - i < NY) z = mfma_bf16(x[i], y[s - i], z);
    return z;
}

// A part of a sequence: its first token and length, how many parts of the sequence come before and after,
// its place in the workspace, the state's slot, and that of a sequence that is left out (of no tokens: only where
// sequences are whole).
struct lc_part { int32_t b, t0, len, before, after, index, slot, held; };

// Part `want` of the batch, parts in order of the sequences (by_seq: the first part of sequence `want`). Offsets that descend may let sequences share tokens and so
// have more parts than the workspace: a sequence whose parts pass it is left out, by every launch alike.
__device__ lc_part find_part(const lc_args & x, int want, bool by_seq, bool report, int threads, int32_t * sh) {
    const la_args & a = x.a;
    lc_part p{want, 0, 0, 0, 0, want, -1, -1};
    if (x.L > 0) {
        // every thread counts the parts of a few sequences
        const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = (a.n_seq + threads - 1) / threads;
        int32_t sum = 0;
        for (int i = 0; i < c; i++) {
            const int b = tid * c + i;
            if (b < a.n_seq) sum += (la_sequence(a, b, report).len + x.L - 1) / x.L;
        }
        int32_t incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int32_t y = __shfl_up(incl, d);
            if (lane >= d) incl += y;
        }
        if (lane == 63) sh[w] = incl;
        if (tid == 0) sh[8] = -1;
        __syncthreads();
        for (int i = 0; i < w; i++) incl += sh[i];
        if (by_seq ? want / c == tid : want >= incl - sum && want < incl) {
            int32_t at = incl - sum;
            for (int i = 0; i < c; i++) {
                const int b = tid * c + i;
                const int32_t n = b < a.n_seq ? (la_sequence(a, b, false).len + x.L - 1) / x.L : 0;
                if ((by_seq ? b == want && n > 0 : want >= at && want < at + n) && at + n <= x.parts) {
                    const la_seq s = la_sequence(a, b, false);
                    sh[8] = b; sh[9] = by_seq ? 0 : want - at; sh[14] = by_seq ? at : want; sh[10] = n; sh[11] = s.t0; sh[12] = s.len; sh[13] = s.slot;
                }
                at += n;
            }
        }
        __syncthreads();
        auto get = [&](int i) { return __builtin_amdgcn_readfirstlane(sh[i]); };
        p.b = get(8);
        if (p.b < 0) return p;
        p.before = get(9);
        p.after = get(10) - p.before - 1;
        p.t0 = get(11) + p.before * x.L;
        p.len = p.after > 0 ? x.L : get(12) - p.before * x.L;
        p.slot = get(13);
        p.index = get(14);
        return p;
    }
    const la_seq s = la_sequence(a, want, report && threadIdx.x == 0);
    return {want, s.t0, s.len, 0, 0, want, s.slot, s.held};
}

// STATES: only what the part adds to the state, to the workspace.
template <int NT, int DK, int NW, bool STATES>
__global__ __launch_bounds__(64 * NW, (lc_cfg<NT, DK, NW>::WAVES_EU)) void k_linear_chunks(lc_args x) {
    using F = lc_cfg<NT, DK, NW>;
    constexpr int C = LC_C, OT = F::OT;
    __shared__ __attribute__((aligned(256))) uint8_t lds[F::LDS];
    // by the chunk's parity: log2 of the decay from the chunk's start, scale 2^G, 2^(G_end - G), 2^G_end
    __shared__ double G[2][C];
    __shared__ float eG[2][C], wG[2][C], eEnd[2];
    __shared__ int32_t sh[15];
    const la_args & a = x.a;
    int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the heads of a key head on one XCD, key heads and parts in turn on all of them
    const int share = a.rep * a.ct, near = (int) blockIdx.x >> 3;
    const int blk = (near / share * 8 + (int) (blockIdx.x & 7)) * share + near % share;
    const int cb = blk % a.ct, h = blk / a.ct % a.n_v, want = blk / a.ct / a.n_v;
    if (want >= x.parts) return;
    const lc_part part = find_part(x, want, false, !STATES && (x.L > 0 ? blk == 0 : cb == 0 && h == 0), F::THREADS, sh);
    if (part.b < 0) return;
    if (part.len <= 0) {
        la_carry(a, part.held, h, cb * F::THREADS + tid, a.ct * F::THREADS);
        return;
    }
    if (STATES && part.after == 0) return;

    const int hk = h / a.rep, c0 = cb * F::COLS;
    const char * qh = a.q + (int64_t) hk * a.q_nb1, * kh = a.k + (int64_t) hk * a.k_nb1;
    const char * vh = a.v + (int64_t) h * a.v_nb1;
    // Unit i of the thread: 16 bytes of LDS at 16 (tid + THREADS i) of the tensor, its token, its 8 values from `e8`.
    // Its place behind the chunk's first token has 32 bits (the host checks the strides): loads are a uniform base and
    // an offset.
    struct unit { int token, e8; };
    auto q_unit = [&](int i) { const int u = tid + F::THREADS * i, t = u / (DK / 8); return unit{t, 8 * (u % (DK / 8) ^ lc_place<DK>(t))}; };
    auto v_unit = [&](int i) {
        const int u = tid + F::THREADS * i, t = u / (F::COLS / 8);
        return unit{t, c0 + 8 * (u % (F::COLS / 8) ^ lc_place<F::COLS>(t))};
    };
    uint32_t oq[F::KU], ok[F::KU], ov[F::VU];
#pragma unroll
    for (int i = 0; i < F::KU; i++) {
        const unit u = q_unit(i);
        oq[i] = (uint32_t) (u.token * a.q_nb2 + u.e8 * F::ES);
        ok[i] = (uint32_t) (u.token * a.k_nb2 + u.e8 * F::ES);
    }
#pragma unroll
    for (int i = 0; i < F::VU; i++) {
        const unit u = v_unit(i);
        ov[i] = (uint32_t) (u.token * a.v_nb2 + u.e8 * F::ES);
    }
    const bool plain = a.dk == DK && c0 + F::COLS <= a.dv;
    auto get = [&](auto & r, const char * base, const auto & off, auto unit_of, int t0, int d) {
        constexpr int N = sizeof(r) / sizeof(r[0]);
        if (plain && t0 + C <= part.len) {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int j = 0; j < F::LPU; j++) r[i][j] = *(const v4w *) (base + off[i] + 16 * j);
        } else {                                  // zeros past the part, the head's rows and columns
#pragma unroll
            for (int i = 0; i < N; i++) {
                const unit u = unit_of(i);
#pragma unroll
                for (int j = 0; j < F::LPU; j++) {
                    r[i][j] = v4w{0, 0, 0, 0};
                    if (u.e8 + j * (8 / F::LPU) < d && t0 + u.token < part.len) r[i][j] = *(const v4w *) (base + off[i] + 16 * j);
                }
            }
        }
    };
    // 8 values of a staged token as NT terms of 4 packed pairs
    auto terms = [&](const v4w (&r)[F::LPU], uint32_t (&o)[NT][4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t t[NT];
            if constexpr (NT == 1) {
                t[0] = r[0][i];
            } else if constexpr (NT == 2) {
                typedef _Float16 v2h __attribute__((ext_vector_type(2)));
                const uint32_t y = r[0][i];        // (a bit cast of a vector's element itself takes element 0)
                const v2h f = __builtin_bit_cast(v2h, y);
                bf16_terms<NT>((float) f[0], (float) f[1], t);
            } else {
                const uint32_t y0 = r[i >> 1][2 * (i & 1)], y1 = r[i >> 1][2 * (i & 1) + 1];
                bf16_terms<NT>(__builtin_bit_cast(float, y0), __builtin_bit_cast(float, y1), t);
            }
#pragma unroll
            for (int n = 0; n < NT; n++) o[n][i] = t[n];
        }
    };
    auto put = [&](const auto & r, int at, int size) {
        constexpr int N = sizeof(r) / sizeof(r[0]);
#pragma unroll
        for (int i = 0; i < N; i++) {
            uint32_t o[NT][4];
            terms(r[i], o);
#pragma unroll
            for (int n = 0; n < NT; n++) *(v4w *) (lds + at + n * size + 16 * (tid + F::THREADS * i)) = v4w{o[n][0], o[n][1], o[n][2], o[n][3]};
        }
    };
    auto q_at = [&](int t0) { return qh + (int64_t) (part.t0 + t0) * a.q_nb2; };
    auto k_at = [&](int t0) { return kh + (int64_t) (part.t0 + t0) * a.k_nb2; };
    auto v_at = [&](int t0) { return vh + (int64_t) (part.t0 + t0) * a.v_nb2; };
    // bf16: a chunk to the buffer at `to`, under way when the call returns but for ragged chunks
    auto send = [&](int t0, int to) {
        if (plain && t0 + C <= part.len) {
            const uint32_t at = lds_address(lds) + to + 1024 * w;
            if (!STATES) {
#pragma unroll
                for (int i = 0; i < F::KU; i++) lds_dma16(q_at(t0), oq[i], at + F::OQ + 16 * F::THREADS * i);
            }
#pragma unroll
            for (int i = 0; i < F::KU; i++) lds_dma16(k_at(t0), ok[i], at + F::OK + 16 * F::THREADS * i);
#pragma unroll
            for (int i = 0; i < F::VU; i++) lds_dma16(v_at(t0), ov[i], at + F::OV + 16 * F::THREADS * i);
        } else {
            v4w rk[F::KU][F::LPU], rv[F::VU][F::LPU];
            if (!STATES) {
                get(rk, q_at(t0), oq, q_unit, t0, a.dk);
                put(rk, to + F::OQ, F::QK);
            }
            get(rk, k_at(t0), ok, q_unit, t0, a.dk);
            put(rk, to + F::OK, F::QK);
            get(rv, v_at(t0), ov, v_unit, t0, a.dv);
            put(rv, to + F::OV, F::V);
        }
    };
    // f16 and f32: the next chunk waits in registers, and is taken apart on its way to LDS
    v4w rq[F::DMA ? 1 : F::KU][F::LPU], rk[F::DMA ? 1 : F::KU][F::LPU], rv[F::DMA ? 1 : F::VU][F::LPU];
    auto load = [&](int t0) {
        if (!STATES) get(rq, q_at(t0), oq, q_unit, t0, a.dk);
        get(rk, k_at(t0), ok, q_unit, t0, a.dk);
        get(rv, v_at(t0), ov, v_unit, t0, a.dv);
    };
    // The part's chunks in their order; backwards for STATES, where a chunk's weights then hold all the decay behind it and
    // the sum is never scaled (these parts are whole chunks).
    auto place = [&](int t0) { return STATES ? part.len - C - t0 : t0; };
    // the decays of a chunk, by the last wave (which has no scores to make); the next chunk's g is loaded ahead
    float gt = 0.f;
    double after = 0.;                     // STATES: of the chunks behind
    auto load_g = [&](int t0) {
        int t = place(t0) + (lane & (C - 1));
        t = t < part.len ? t : part.len - 1;
        gt = a.g[(int64_t) (part.t0 + (t < 0 ? 0 : t)) * a.g_ts + h];
    };
    auto decays = [&](int t0) {
        const int at = t0 / C & 1;
        float x = place(t0) + lane < part.len && lane < C ? gt : 0.f;
        x = x < LC_FLOOR ? LC_FLOOR : x;
        double s = (double) x * LC_LOG2E;
#pragma unroll
        for (int d = 1; d < C; d <<= 1) {
            const double y = __shfl_up(s, d);
            if (lane >= d) s += y;
        }
        const double end = __shfl(s, C - 1);
        if constexpr (STATES) {
            if (lane < C) wG[at][lane] = __builtin_amdgcn_exp2f((float) (end - s + after));
            after += end;
        } else if (lane < C) {
            G[at][lane] = s;
            eG[at][lane] = __builtin_amdgcn_exp2f((float) s) * a.scale;
            wG[at][lane] = __builtin_amdgcn_exp2f((float) (end - s));
            if (lane == 0) eEnd[at] = __builtin_amdgcn_exp2f((float) end);
        }
    };
    if (w == NW - 1) load_g(0);
    if constexpr (F::DMA) send(place(0), 0);
    else load(place(0));

    // the state of the lane: [row tile][column tile] of rows 32 (t / 2) + 8 g + 4 (t % 2) + r
    v4f S[F::KT][2];
    const size_t hs = (size_t) a.dk * a.dv, per = (size_t) a.n_v * hs;
    int col[2];
#pragma unroll
    for (int u = 0; u < 2; u++) col[u] = c0 + LC_WCOLS * w + 8 * (m >> 2) + 4 * u + (m & 3);
    const bool live = c0 + LC_WCOLS * w < a.dv;            // the wave has columns
    const bool whole = a.dk == DK && c0 + LC_WCOLS * (w + 1) <= a.dv;      // no row or column past the head's
    // the lane's values of a state in the workspace
    auto in_u = [&](size_t index, int t, int u) -> v4f & {
        return *(v4f *) (x.U + (index * a.n_v + h) * x.US + ((((size_t) cb * NW + w) * F::KT + t) * 2 + u) * 256 + 4 * lane);
    };
    auto each = [&](auto fn) {                             // fn(value, its element, element of a head's state)
        auto all = [&](auto inside) {
#pragma unroll
            for (int t = 0; t < F::KT; t++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int row = 32 * (t >> 1) + 8 * g + 4 * (t & 1) + r;
                        if (inside(row, col[u])) fn(S[t][u], r, (size_t) row * a.dv + col[u]);
                    }
        };
        // (without a condition the loads are all in flight at once)
        if (whole) all([](int, int) { return true; });
        else       all([&](int row, int c) { return row < a.dk && c < a.dv; });
    };
#pragma unroll
    for (int t = 0; t < F::KT; t++) S[t][0] = S[t][1] = v4f{0.f, 0.f, 0.f, 0.f};
    if (!STATES) {
        // (in place the last part may be done before the first begins: it finds its state in the workspace too)
        if (part.before > 0 || (part.after > 0 && a.s_in == a.s_out)) {
            const int at = part.before > 0 ? part.index - 1 : part.index + part.after;
#pragma unroll
            for (int t = 0; t < F::KT; t++)
#pragma unroll
                for (int u = 0; u < 2; u++) S[t][u] = in_u(at, t, u);
        } else if (part.slot >= 0 && a.s_in) {
            const float * s0 = a.s_in + part.slot * per + h * hs;
            each([&](v4f & s, int r, size_t e) { s[r] = s0[e]; });
        }
        // the scores of the tokens behind the first 16 stay 0 in their rows
        for (int i = tid; i < OT * F::P / 16; i += F::THREADS) *(v4w *) (lds + F::OP + 16 * i) = v4w{0, 0, 0, 0};
    }
    if (w == NW - 1) {
        decays(0);
        load_g(C);
    }

    for (int t0 = 0; t0 < part.len; t0 += C) {
        // the thread's places are computed anew in every chunk: kept over the loop they cost registers, spilled
        asm volatile("" : "+v"(tid), "+v"(lane), "+v"(m), "+v"(g));
        const int even = t0 / C & 1, buf = F::DMA ? even * F::BUF : 0;
        if constexpr (F::DMA) {
            wait_vmem();
        } else {
            if (!STATES) put(rq, F::OQ, F::QK);
            put(rk, F::OK, F::QK);
            put(rv, F::OV, F::V);
        }
        __syncthreads();
        if (w == NW - 1 && t0 + C < part.len) {
            decays(t0 + C);
            load_g(t0 + 2 * C);
        }
        if constexpr (F::DMA) {
            if (t0 + C < part.len) send(place(t0 + C), F::BUF - buf);
        } else if (STATES && t0 + C < part.len) {
            load(place(t0 + C));
        }
        v4w vx[2][NT];                         // v^T of the wave's columns
        auto load_v = [&]() {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int t = 0; t < NT; t++) vx[u][t] = lc_transposed<F::COLS>(lds + buf + F::OV + t * F::V, 8 * g, w, u, m);
        };
        if constexpr (!STATES) {
            // the scores, 16 x 16 tiles of tokens (j rows, i columns): the three with j <= i
            constexpr int PT = NW == 2 ? 2 : 1;
#pragma unroll
            for (int x = 0; x < PT; x++) {
                const int n = w + NW * x;
                if (n >= 3) break;
                const int it = n > 0, jt = n > 1;
                v4f p{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kb = 0; kb < F::KB; kb++) {
                    v4w kx[NT], qx[NT];
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        kx[t] = *(const v4w *) (lds + buf + F::OK + t * F::QK + lc_row<DK>(16 * jt + m, 4 * kb + g));
                        qx[t] = *(const v4w *) (lds + buf + F::OQ + t * F::QK + lc_row<DK>(16 * it + m, 4 * kb + g));
                    }
                    p = mfma_terms<NT, NT, NT>(kx, qx, p);
                }
                const int i = 16 * it + m;
                const double gi = G[even][i];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = 16 * jt + 4 * g + r;
                    p[r] = j <= i ? p[r] * (__builtin_amdgcn_exp2f((float) (gi - G[even][j])) * a.scale) : 0.f;
                }
                uint32_t lo[OT], hi[OT];
                bf16_terms<OT>(p[0], p[1], lo);
                bf16_terms<OT>(p[2], p[3], hi);
#pragma unroll
                for (int t = 0; t < OT; t++)
                    *(v2w *) (lds + F::OP + t * F::P + lc_score(i, 2 * jt + (g >> 1)) + 8 * (g & 1)) = v2w{lo[t], hi[t]};
            }
            // S^T q
            v4f o[2][2] = {};
            if (live) {
#pragma unroll
                for (int kb = 0; kb < F::KB; kb++) {
                    v4w sx[2][OT];
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const v4f & s = S[2 * kb + (i >> 1)][u];
                            uint32_t t[OT];
                            bf16_terms<OT>(s[2 * (i & 1)], s[2 * (i & 1) + 1], t);
#pragma unroll
                            for (int n = 0; n < OT; n++) sx[u][n][i] = t[n];
                        }
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        v4w qx[NT];
#pragma unroll
                        for (int t = 0; t < NT; t++) qx[t] = *(const v4w *) (lds + buf + F::OQ + t * F::QK + lc_row<DK>(16 * i + m, 4 * kb + g));
                        o[i][0] = mfma_terms<OT, NT, OT>(sx[0], qx, o[i][0]);
                        o[i][1] = mfma_terms<OT, NT, OT>(sx[1], qx, o[i][1]);
                    }
                }
            }
            if constexpr (!F::DMA) {
                if (t0 + C < part.len) load(t0 + C);       // (here the scores' and S^T q's registers are free)
            }
            __syncthreads();                   // the scores
            if (live) {
                load_v();
                float odd = 0.f;               // NaN with a non-finite v (times 0)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t y = vx[u][0][i];
                        odd = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, y), v2b{}, odd, false);
                    }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float e = eG[even][16 * i + m];
                    o[i][0] *= e;
                    o[i][1] *= e;
                }
                if (__ballot(odd != odd) == 0) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        v4w px[OT];
#pragma unroll
                        for (int t = 0; t < OT; t++) px[t] = *(const v4w *) (lds + F::OP + t * F::P + lc_score(16 * i + m, g));
                        o[i][0] = mfma_terms<NT, OT, OT>(vx[0], px, o[i][0]);
                        o[i][1] = mfma_terms<NT, OT, OT>(vx[1], px, o[i][1]);
                    }
                } else {
                    auto sum = [&](int at, int size, int terms) {
                        float f = 0.f;
                        for (int n = 0; n < terms; n++) f += __builtin_bit_cast(float, (uint32_t) *(const uint16_t *) (lds + at + n * size) << 16);
                        return f;
                    };
                    for (int j = 0; j <= 16 + m; j++) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            if (j > 16 * i + m) continue;
                            const float p = sum(F::OP + lc_score(16 * i + m, j >> 3) + 2 * (j & 7), F::P, OT);
#pragma unroll
                            for (int u = 0; u < 2; u++)
#pragma unroll
                                for (int r = 0; r < 4; r++) {
                                    const float v = sum(buf + F::OV + lc_row<F::COLS>(j, 4 * w + g) + 8 * u + 2 * r, F::V, NT);
                                    o[i][u][r] = __fmaf_rn(p, v, o[i][u][r]);
                                }
                        }
                    }
                }
                // 8 columns of a token
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int t = t0 + 16 * i + m, c = c0 + LC_WCOLS * w + 8 * g;
                    if (t < part.len && c < a.dv) {
                        char * p = a.out + ((int64_t) (part.t0 + t) * a.n_v * a.dv + (int64_t) h * a.dv + c) * F::ES;
                        const v4f y0 = o[i][0], y1 = o[i][1];
                        if constexpr (NT == 3) {
                            *(v4f *) p = y0;
                            *(v4f *) (p + 16) = y1;
                        } else {
                            const int type = NT == 1 ? QWFN_TYPE_BF16 : QWFN_TYPE_F16;
                            *(v4w *) p = v4w{la_pack2(y0[0], y0[1], type), la_pack2(y0[2], y0[3], type),
                                             la_pack2(y1[0], y1[1], type), la_pack2(y1[2], y1[3], type)};
                        }
                    }
                }
            }
        } else {
            load_v();
        }
        // the state at the chunk's end
        if (live) {
            v4w vw[2][3];
            float wt[8], cend = 1.f;
            if (!STATES) cend = eEnd[even];
#pragma unroll
            for (int i = 0; i < 8; i++) wt[i] = wG[even][8 * g + i];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float lo = 0.f, hi = 0.f;
#pragma unroll
                    for (int t = NT - 1; t >= 0; t--) { lo += bf16_lo(vx[u][t][i]); hi += bf16_hi(vx[u][t][i]); }
                    uint32_t t3[3];
                    bf16_terms<3>(lo * wt[2 * i], hi * wt[2 * i + 1], t3);
#pragma unroll
                    for (int t = 0; t < 3; t++) vw[u][t][i] = t3[t];
                }
            // (TG row tiles at a time: a sum's products are 2 TG MFMAs apart)
            constexpr int TG = 4;
#pragma unroll
            for (int t0g = 0; t0g < F::KT; t0g += TG) {
                v4w kx[TG][NT];
#pragma unroll
                for (int t = 0; t < TG; t++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        kx[t][n] = lc_transposed<DK>(lds + buf + F::OK + n * F::QK, 8 * g, (t0g + t) >> 1, t & 1, m);
#pragma unroll
                for (int t = t0g; t < t0g + TG; t++)
                    if (!STATES) { S[t][0] *= cend; S[t][1] *= cend; }
#pragma unroll
                for (int d = 2; d >= 0; d--)
#pragma unroll
                    for (int n = 0; n < NT && n <= d; n++)
#pragma unroll
                        for (int t = 0; t < TG; t++)
#pragma unroll
                            for (int u = 0; u < 2; u++) S[t0g + t][u] = mfma_bf16(kx[t][n], vw[u][d - n], S[t0g + t][u]);
            }
        }
        if constexpr (!F::DMA) __syncthreads();
    }
    if constexpr (STATES) {
#pragma unroll
        for (int t = 0; t < F::KT; t++)
#pragma unroll
            for (int u = 0; u < 2; u++) in_u(part.index, t, u) = S[t][u];
        if (tid == F::THREADS - 64 && cb == 0) x.G[(size_t) part.index * a.n_v + h] = after;
    } else if (part.after == 0 && part.slot >= 0) {
        float * so = a.s_out + part.slot * per + h * hs;
        each([&](v4f & s, int r, size_t e) { so[e] = s[r]; });
    }
}

// The states behind the parts of a sequence (but the last), in the place of their U: S = 2^G_p S + U_p; in place the
// state before the first part in the last one's. A thread per 4 elements of a head's state; the parts' values are loaded
// LJ_AHEAD at a time.
constexpr int LJ_AHEAD = 4;

__global__ __launch_bounds__(LA_THREADS) void k_linear_join(lc_args x) {
    __shared__ int32_t sh[15];
    const la_args & a = x.a;
    const int blocks = (x.US / 4 + LA_THREADS - 1) / LA_THREADS;
    const int eb = blockIdx.x % blocks, h = blockIdx.x / blocks % a.n_v;
    const int b = blockIdx.x / blocks / a.n_v;
    const lc_part part = find_part(x, b, true, false, LA_THREADS, sh);
    if (part.b < 0) {
        la_carry(a, la_sequence(a, b, false).held, h, eb * LA_THREADS + threadIdx.x, blocks * LA_THREADS);
        return;
    }
    if (part.after == 0) return;
    const int e = eb * LA_THREADS + threadIdx.x;
    if (4 * e >= x.US) return;
    v4f s{0.f, 0.f, 0.f, 0.f};
    if (part.slot >= 0 && a.s_in) {
        const int lane = e & 63, m = lane & 15, g = lane >> 4, u = e >> 6 & 1, t = (e >> 7) % x.KT, w = (e >> 7) / x.KT;
        const int col = LC_WCOLS * w + 8 * (m >> 2) + 4 * u + (m & 3), row = 32 * (t >> 1) + 8 * g + 4 * (t & 1);
        const float * s0 = a.s_in + ((int64_t) part.slot * a.n_v + h) * a.dk * a.dv + col;
        if (col < a.dv && row < a.dk)              // (dk is a multiple of 16)
#pragma unroll
            for (int r = 0; r < 4; r++) s[r] = s0[(int64_t) (row + r) * a.dv];
    }
    const int64_t per = (int64_t) x.US * a.n_v;
    float * up = x.U + ((int64_t) part.index * a.n_v + h) * x.US + 4 * (int64_t) e;
    if (a.s_in == a.s_out) *(v4f *) (up + part.after * per) = s;
    const double * gp = x.G + (int64_t) part.index * a.n_v + h;
    for (int p0 = 0; p0 < part.after; p0 += LJ_AHEAD) {
        v4f u[LJ_AHEAD];
        float f[LJ_AHEAD];
#pragma unroll
        for (int i = 0; i < LJ_AHEAD; i++) {
            const int p = p0 + i < part.after ? p0 + i : part.after - 1;
            u[i] = *(const v4f *) (up + p * per);
            f[i] = __builtin_amdgcn_exp2f((float) gp[(int64_t) p * a.n_v]);
        }
#pragma unroll
        for (int i = 0; i < LJ_AHEAD; i++) {
            if (p0 + i >= part.after) break;
            s = s * f[i] + u[i];
            *(v4f *) (up + (p0 + i) * per) = s;
        }
    }
}

// ---------------------------------------------------------------- host

int check_heads(const qwfn_tensor * t, int32_t type, const char * name, bool packed) {
    auto err = [&](int code, const char * what) { return set_error(code, std::string("linear_attn: ") + name + what); };
    if (!t || (!t->data && t->ne[2] != 0)) return err(QWFN_EINVAL, " is NULL");        // (no tokens, no address)
    if (t->type != type) return err(QWFN_EINVAL, " must be f32, f16 or bf16, one type for q, k, v and dst");
    const size_t es = type == QWFN_TYPE_F32 ? 4 : 2;
    if (t->ne[0] < 1 || t->ne[1] < 1 || t->ne[2] < 0 || t->ne[3] != 1) return err(QWFN_EINVAL, " must be [d, n_heads, n_tok]");
    if (t->nb[0] != es) return err(QWFN_EINVAL, " rows must be contiguous");
    if (!is_aligned(t->data, 16) || t->nb[1] % 16 || t->nb[2] % 16) return err(QWFN_EALIGN, " must be 16-byte aligned, its strides too");
    if (packed && ((t->ne[1] > 1 && t->nb[1] != t->ne[0] * es) || (t->ne[2] > 1 && t->nb[2] != t->ne[0] * t->ne[1] * es))) return err(QWFN_EINVAL, " must be contiguous");
    if (t->ne[1] > 1 && t->nb[1] < t->ne[0] * es) return err(QWFN_EINVAL, " heads overlap");
    return QWFN_OK;
}

int check_linear(const qwfn_tensor * q, const qwfn_tensor * v, int32_t n_seq, int32_t max_len) {
    if (!q || !v) return set_error(QWFN_EINVAL, "linear_attn: q or v is NULL");
    const int32_t type = q->type;
    if (type != QWFN_TYPE_F32 && type != QWFN_TYPE_F16 && type != QWFN_TYPE_BF16)
        return set_error(QWFN_EINVAL, "linear_attn: q must be f32, f16 or bf16");
    if (int rc = check_heads(q, type, "q", false)) return rc;
    if (int rc = check_heads(v, type, "v", false)) return rc;
    if (q->ne[0] % 16 || v->ne[0] % 16 || q->ne[0] > 256 || v->ne[0] > 512)
        return set_error(QWFN_ENOTSUP, "linear_attn: dk and dv must be multiples of 16, dk at most 256, dv at most 512");
    if (v->ne[1] % q->ne[1]) return set_error(QWFN_EINVAL, "linear_attn: n_v_heads must be a multiple of n_k_heads");
    if (v->ne[2] != q->ne[2]) return set_error(QWFN_EINVAL, "linear_attn: q and v must have the same tokens");
    if (n_seq < 1 || n_seq > 65535 || v->ne[1] > 1024) return set_error(QWFN_EINVAL, "linear_attn: n_seq must lie in [1, 65535], n_v_heads at most 1024");
    if (max_len < 1) return set_error(QWFN_EINVAL, "linear_attn: max_len must be positive");
    if (q->ne[2] > 0x7fffffff) return set_error(QWFN_ENOTSUP, "linear_attn: at most 2^31 - 1 tokens");
    return QWFN_OK;
}

struct lc_plan {
    bool    step;                      // token by token
    int32_t NT, DK, NW, ct, L, US;
    int64_t parts;                     // blocks along the tokens, at most
    size_t  off_g, bytes;
};

template <int NT> int per_cu(int DK, int NW) {
    if (DK == 64) return NW == 2 ? lc_cfg<NT, 64, 2>::PER_CU : lc_cfg<NT, 64, 4>::PER_CU;
    if (DK == 128) return NW == 2 ? lc_cfg<NT, 128, 2>::PER_CU : lc_cfg<NT, 128, 4>::PER_CU;
    if constexpr (NT < 3) if (NW == 2) return lc_cfg<NT, 256, 2>::PER_CU;
    return lc_cfg<NT, 256, 4>::PER_CU;
}

// Parts of a sequence: as many as fill the CUs once with two waves a SIMD, so that no workgroup waits for another (4096
// bf16 tokens of 48 heads of 128, with one term of the state and the scores: 99 us in 10 parts, 120 in 5, 121 in 16, three
// waves a SIMD: a part's state goes through the workspace three times), but no shorter than LC_MIN_PART tokens: a part costs
// a second pass over its k and v (two f32 sequences of 509: 78 us with parts of 128, 93 of 256).
constexpr int64_t LC_CUS = 256, LC_MIN_PART = 128;

lc_plan plan_linear(const qwfn_tensor * q, const qwfn_tensor * v, int32_t n_seq, int32_t max_len) {
    lc_plan p{};
    const int64_t dk = q->ne[0], dv = v->ne[0], n_v = v->ne[1], n_tok = q->ne[2];
    p.NT = q->type == QWFN_TYPE_BF16 ? 1 : q->type == QWFN_TYPE_F16 ? 2 : 3;
    p.DK = dk <= 64 ? 64 : dk <= 128 ? 128 : 256;
    // Short calls go token by token: 1.2 us a token and 4 sequences (16 bf16 heads of 128 for 48), against a chunk whatever it
    // holds: 11.9 us and 11.3 at 4 bf16 tokens, 14.9 and 13.6 at 6 of f16, 16.8 and 15.3 at 8 of f32; 9.6, 10.2 and 10.1
    // against 11.3, 13.6 and 15.3 at 2. At 64 sequences the sides meet at 6 f16 and 8 f32 tokens, and 4 bf16 tokens take 84
    // against 95.
    p.step = max_len <= 2 + 2 * p.NT || n_tok == 0;
    if (p.step) return p;
    p.NW = dv <= 2 * LC_WCOLS && (p.NT < 3 || p.DK < 256) ? 2 : 4;         // (256 rows of F32 for two waves are spilled)
    p.ct = (int32_t) ((dv + LC_WCOLS * p.NW - 1) / (LC_WCOLS * p.NW));
    const int64_t longest = std::min<int64_t>(max_len, n_tok), C = LC_C;
    const int per = p.NT == 1 ? per_cu<1>(p.DK, p.NW) : p.NT == 2 ? per_cu<2>(p.DK, p.NW) : per_cu<3>(p.DK, p.NW);
    const int64_t room = LC_CUS * std::min(per, 8 / p.NW) / (n_v * p.ct);
    // A sequence's last part is half of one on average (16 ragged f16 sequences: 75.8 us with the n_seq / 2, 73.8 without). So
    // a batch of more than about 2 room sequences is not cut, however long one of them is: with 48 heads of 128 (room 10)
    // from 18 sequences on.
    const int64_t whole = std::max<int64_t>(1, room - n_seq / 2);
    const int64_t L = (std::max<int64_t>(LC_MIN_PART, (n_tok + whole - 1) / whole) + C - 1) / C * C;
    p.parts = n_seq;
    if (L < longest) {
        p.L = (int32_t) L;
        p.parts = n_seq + n_tok / L;
        p.US = p.DK * LC_WCOLS * p.NW * p.ct;
        p.off_g = (size_t) p.parts * n_v * p.US * sizeof(float);
        p.bytes = p.off_g + (size_t) p.parts * n_v * sizeof(double);
    }
    return p;
}

template <int NT, int DK, int NW>
int launch_chunks(const lc_args & x, const lc_plan & p, hipStream_t s) {
    const int64_t share = (int64_t) x.a.rep * p.ct;                // (whole rounds of the 8 XCDs)
    const dim3 grid((unsigned) ((p.parts * x.a.n_k + 7) / 8 * 8 * share)), blk(64 * NW);
    if (p.L > 0) {
        hipLaunchKernelGGL((k_linear_chunks<NT, DK, NW, true>), grid, blk, 0, s, x);
        if (int rc = hip_check(hipGetLastError(), "linear_attn launch")) return rc;
        const int64_t blocks = (x.US / 4 + LA_THREADS - 1) / LA_THREADS;
        hipLaunchKernelGGL(k_linear_join, dim3((unsigned) (x.a.n_seq * x.a.n_v * blocks)), dim3(LA_THREADS), 0, s, x);
        if (int rc = hip_check(hipGetLastError(), "linear_attn launch")) return rc;
    }
    hipLaunchKernelGGL((k_linear_chunks<NT, DK, NW, false>), grid, blk, 0, s, x);
    return hip_check(hipGetLastError(), "linear_attn launch");
}
template <int NT>
int launch_type(const lc_args & x, const lc_plan & p, hipStream_t s) {
    if (p.DK == 64)  return p.NW == 2 ? launch_chunks<NT, 64, 2>(x, p, s) : launch_chunks<NT, 64, 4>(x, p, s);
    if (p.DK == 128) return p.NW == 2 ? launch_chunks<NT, 128, 2>(x, p, s) : launch_chunks<NT, 128, 4>(x, p, s);
    if constexpr (NT < 3) if (p.NW == 2) return launch_chunks<NT, 256, 2>(x, p, s);
    return launch_chunks<NT, 256, 4>(x, p, s);
}

}  // namespace
}  // namespace qwfn

using namespace qwfn;

extern "C" size_t qwfn_linear_attn_workspace_size(const qwfn_tensor * q, const qwfn_tensor * v, int32_t n_seq, int32_t max_len) {
    return ::qwfn::abi_value<size_t>("linear_attn_workspace_size", 0, [&]() -> size_t {
        return check_linear(q, v, n_seq, max_len) ? 0 : plan_linear(q, v, n_seq, max_len).bytes;
    });
}

extern "C" int qwfn_linear_attn(const qwfn_tensor * q, const qwfn_tensor * k, const qwfn_tensor * v, const float * g,
                                int64_t g_token_stride, const int32_t * cu, int32_t n_seq, int32_t max_len,
                                const int32_t * slots, int32_t n_slots, const float * state_in, float * state_out,
                                float scale, const qwfn_tensor * dst, void * ws, size_t ws_bytes, void * stream) {
    return ::qwfn::abi_call("linear_attn", [&]() -> int {
        if (int rc = check_linear(q, v, n_seq, max_len)) return rc;
        if (int rc = check_heads(k, q->type, "k", false)) return rc;
        if (int rc = check_heads(dst, q->type, "dst", true)) return rc;
        for (int i = 0; i < 3; i++)
            if (k->ne[i] != q->ne[i]) return set_error(QWFN_EINVAL, "linear_attn: q and k must have the same shape");
        for (int i = 0; i < 3; i++)
            if (dst->ne[i] != v->ne[i]) return set_error(QWFN_EINVAL, "linear_attn: dst must have v's shape");
        if ((!g && q->ne[2] != 0) || !cu || !state_out) return set_error(QWFN_EINVAL, "linear_attn: g, cu or state_out is NULL");
        const int64_t n_v = v->ne[1], dk = q->ne[0], dv = v->ne[0], n_tok = q->ne[2];
        if (g_token_stride != 0 && g_token_stride < n_v) return set_error(QWFN_EINVAL, "linear_attn: g_token_stride must be 0 or at least n_v_heads");
        if (n_slots < 1 || (!slots && n_slots < n_seq)) return set_error(QWFN_EINVAL, "linear_attn: too few state slots");
        if (!std::isfinite(scale)) return set_error(QWFN_EINVAL, "linear_attn: scale must be finite");
        if (!is_aligned(g, 4) || !is_aligned(cu, 4) || !is_aligned(slots, 4) || !is_aligned(state_in, 16) || !is_aligned(state_out, 16))
            return set_error(QWFN_EALIGN, "linear_attn: states 16-byte aligned, g, cu and slots 4");
        const size_t states = (size_t) n_slots * n_v * dk * dv * 4;
        if (state_in && state_in != state_out && (uintptr_t) state_in < (uintptr_t) state_out + states &&
            (uintptr_t) state_out < (uintptr_t) state_in + states)
            return set_error(QWFN_EINVAL, "linear_attn: state_in and state_out must be equal or not overlap");
        if (n_tok == 0 && (!slots || state_in == state_out)) return QWFN_OK;
        if ((q->nb[2] | k->nb[2] | v->nb[2]) >> 24) return set_error(QWFN_ENOTSUP, "linear_attn: token strides of 2^24 bytes or more");
        const lc_plan pl = plan_linear(q, v, n_seq, max_len);
        const int64_t ct = (dv + LA_COLS - 1) / LA_COLS;       // token by token
        const int64_t blocks = pl.step ? n_seq * n_v * ct : (pl.parts + 8) * n_v * std::max<int64_t>(pl.ct, pl.US / (4 * LA_THREADS) + 1);
        if (blocks > LA_BLOCKS) return set_error(QWFN_ENOTSUP, "linear_attn: too many sequences and heads");
        if (pl.bytes > 0 && (!ws || ws_bytes < pl.bytes))
            return set_error(QWFN_ENOMEM, "linear_attn: ws must hold qwfn_linear_attn_workspace_size bytes");
        if (!is_aligned(ws, 16)) return set_error(QWFN_EALIGN, "linear_attn: ws must be 16-byte aligned");
        const span in[] = {{q->data, tensor_extent(q), "q"}, {k->data, tensor_extent(k), "k"}, {v->data, tensor_extent(v), "v"},
                           {g, n_tok > 0 ? (size_t) ((n_tok - 1) * g_token_stride + n_v) * 4 : 0, "g"}, {cu, (size_t) (n_seq + 1) * 4, "cu"},
                           {slots, (size_t) n_seq * 4, "slots"}, {state_in != state_out ? state_in : nullptr, states, "state_in"}};
        const span out[] = {{dst->data, tensor_extent(dst), "dst"}, {state_out, states, "state_out"}, {ws, pl.bytes, "ws"}};
        if (int rc = check_overlaps("linear_attn", in, 7, out, 3)) return rc;
        la_args a{};
        if (int rc = status_word(&a.status)) return rc;
        a.q = (const char *) q->data; a.k = (const char *) k->data; a.v = (const char *) v->data; a.out = (char *) dst->data;
        a.q_nb1 = (int64_t) q->nb[1]; a.q_nb2 = (int64_t) q->nb[2]; a.k_nb1 = (int64_t) k->nb[1]; a.k_nb2 = (int64_t) k->nb[2];
        a.v_nb1 = (int64_t) v->nb[1]; a.v_nb2 = (int64_t) v->nb[2];
        a.g = g; a.g_ts = g_token_stride; a.cu = cu; a.slots = slots; a.s_in = state_in; a.s_out = state_out; a.scale = scale;
        a.type = q->type; a.n_seq = n_seq; a.max_len = max_len; a.n_slots = n_slots; a.n_tok = (int32_t) n_tok;
        a.n_k = (int32_t) q->ne[1]; a.n_v = (int32_t) n_v; a.rep = a.n_v / a.n_k; a.dk = (int32_t) dk; a.dv = (int32_t) dv;
        if (!pl.step) {
            a.ct = pl.ct;
            const lc_args x{a, pl.L, (int32_t) pl.parts, pl.DK / 16, pl.US, (float *) ws, (double *) ((char *) ws + pl.off_g)};
            return pl.NT == 1 ? launch_type<1>(x, pl, as_stream(stream)) : pl.NT == 2 ? launch_type<2>(x, pl, as_stream(stream))
                                                                                      : launch_type<3>(x, pl, as_stream(stream));
        }
        a.ct = (int32_t) ct;
        const dim3 grid((unsigned) blocks), blk(LA_THREADS);
        if (dk <= 64)       hipLaunchKernelGGL(k_linear_step<64>, grid, blk, 0, as_stream(stream), a);
        else if (dk <= 128) hipLaunchKernelGGL(k_linear_step<128>, grid, blk, 0, as_stream(stream), a);
        else                hipLaunchKernelGGL(k_linear_step<256>, grid, blk, 0, as_stream(stream), a);
        return hip_check(hipGetLastError(), "linear_attn launch");
    });
}
