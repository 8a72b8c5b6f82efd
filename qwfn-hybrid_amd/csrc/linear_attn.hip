// Linear attention with a decay per head over a ragged batch:
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
// per value head, state S [dk][dv] in F32 (q and k of key head h / (n_v / n_k)).
//
// Token by token (k_linear_step): columns of S are independent. A workgroup takes 64
// columns of one head of one sequence, thread (row group rg, column quad cq) the
// rows rg + 16 i; the state stays in registers for the sequence's tokens and is
// read and written once. The output's sum over rows is finished across the lanes
// (permlane swaps) and the waves (LDS), in a fixed order, one barrier a token.
// What bounds it: the state, 8 dk dv bytes a head and sequence.
#include "fattn_device.h"
#include "qwfn_common.h"
#include "qwfn_state.h"

#include <algorithm>
#include <cmath>

namespace qwfn {
namespace {

constexpr int LA_THREADS = 256;
constexpr int LA_COLS = 64;            // columns of a workgroup
constexpr int LA_TC = 8;               // tokens whose q and k are brought in at once

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

// Sequence b: its first token and its length, and its state's slot (-1: none).
struct la_seq { int32_t t0, len, slot; };
__device__ __forceinline__ la_seq la_sequence(const la_args & a, int b, bool report) {
    auto clip = [&](int32_t x) { return x < 0 ? 0 : x > a.n_tok ? a.n_tok : x; };
    const int32_t c0 = a.cu[b], c1 = a.cu[b + 1], lo = clip(c0), hi = clip(c1);
    int32_t len = hi - lo, slot = a.slots ? a.slots[b] : b;
    bool bad = lo != c0 || hi != c1 || len < 0 || len > a.max_len;
    len = len < 0 ? 0 : len > a.max_len ? a.max_len : len;
    if (slot < 0 || slot >= a.n_slots) {
        bad |= slot != -1;
        slot = -1;
    }
    if (bad && report) atomicOr(a.status, DEVERR_SET_ROWS_INDEX);
    return {lo, len, slot};
}

template <int DK>
__global__ __launch_bounds__(LA_THREADS) void k_linear_step(la_args a) {
    constexpr int RPT = DK / 16;               // rows of a thread
    __shared__ float kq[LA_TC][2][DK];
    __shared__ float4 red[2][LA_THREADS / 64][16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, cq = tid & 15, rg = tid >> 4;
    const int cb = blockIdx.x % a.ct, h = blockIdx.x / a.ct % a.n_v, b = blockIdx.x / a.ct / a.n_v;
    const la_seq s = la_sequence(a, b, tid == 0 && cb == 0 && h == 0);
    if (s.len == 0) return;
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

// ---------------------------------------------------------------- host

int check_heads(const qwfn_tensor * t, int32_t type, const char * name, bool packed) {
    auto err = [&](int code, const char * what) { return set_error(code, std::string("linear_attn: ") + name + what); };
    if (!t || !t->data) return err(QWFN_EINVAL, " is NULL");
    if (t->type != type) return err(QWFN_EINVAL, " must be f32, f16 or bf16, one type for q, k, v and dst");
    const size_t es = type == QWFN_TYPE_F32 ? 4 : 2;
    if (t->ne[0] < 1 || t->ne[1] < 1 || t->ne[2] < 0 || t->ne[3] != 1) return err(QWFN_EINVAL, " must be [d, n_heads, n_tok]");
    if (t->nb[0] != es) return err(QWFN_EINVAL, " rows must be contiguous");
    if (!is_aligned(t->data, 16) || t->nb[1] % 16 || t->nb[2] % 16) return err(QWFN_EALIGN, " must be 16-byte aligned, its strides too");
    if (packed && (t->nb[1] != t->ne[0] * es || t->nb[2] != t->ne[0] * t->ne[1] * es)) return err(QWFN_EINVAL, " must be contiguous");
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

}  // namespace
}  // namespace qwfn

using namespace qwfn;

extern "C" size_t qwfn_linear_attn_workspace_size(const qwfn_tensor * q, const qwfn_tensor * v, int32_t n_seq, int32_t max_len) {
    return ::qwfn::abi_value<size_t>("linear_attn_workspace_size", 0, [&]() -> size_t {
        if (check_linear(q, v, n_seq, max_len)) return 0;
        return 0;
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
        if (!g || !cu || !state_out) return set_error(QWFN_EINVAL, "linear_attn: g, cu or state_out is NULL");
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
        if (n_tok == 0) return QWFN_OK;
        la_args a{};
        if (int rc = status_word(&a.status)) return rc;
        a.q = (const char *) q->data; a.k = (const char *) k->data; a.v = (const char *) v->data; a.out = (char *) dst->data;
        a.q_nb1 = (int64_t) q->nb[1]; a.q_nb2 = (int64_t) q->nb[2]; a.k_nb1 = (int64_t) k->nb[1]; a.k_nb2 = (int64_t) k->nb[2];
        a.v_nb1 = (int64_t) v->nb[1]; a.v_nb2 = (int64_t) v->nb[2];
        a.g = g; a.g_ts = g_token_stride; a.cu = cu; a.slots = slots; a.s_in = state_in; a.s_out = state_out; a.scale = scale;
        a.type = q->type; a.n_seq = n_seq; a.max_len = max_len; a.n_slots = n_slots; a.n_tok = (int32_t) n_tok;
        a.n_k = (int32_t) q->ne[1]; a.n_v = (int32_t) n_v; a.rep = a.n_v / a.n_k; a.dk = (int32_t) dk; a.dv = (int32_t) dv;
        a.ct = (int32_t) ((dv + LA_COLS - 1) / LA_COLS);
        const int64_t blocks = (int64_t) n_seq * n_v * a.ct;
        if (blocks > 0x7fffffff) return set_error(QWFN_ENOTSUP, "linear_attn: too many sequences and heads");
        const dim3 grid((unsigned) blocks), blk(LA_THREADS);
        if (dk <= 64)       hipLaunchKernelGGL(k_linear_step<64>, grid, blk, 0, as_stream(stream), a);
        else if (dk <= 128) hipLaunchKernelGGL(k_linear_step<128>, grid, blk, 0, as_stream(stream), a);
        else                hipLaunchKernelGGL(k_linear_step<256>, grid, blk, 0, as_stream(stream), a);
        return hip_check(hipGetLastError(), "linear_attn launch");
    });
}
