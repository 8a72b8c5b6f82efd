// Attention of a tree of drafted tokens over a paged q8_0 cache, for many query rows a KV head:
//
//   s_j = c sum_b dq_b dk_jb (qq_b . kq_jb)      q requantised to q8_0, integer dots
//   out = sum_j 2^(s_j - M) v_j / sum_j 2^(s_j - M),   v_j = dv_jb vq_j,   c = scale log2(e)
//
// over the tokens before the tree and the nodes in the query's mask. A tree of 64 nodes at 8 heads a KV head has 512 rows:
// 960 operations a byte of the cache, so the vector and matrix units bound it, not the rows.
//
// Work: as in k_paged_attn the requests' key tiles of 32 stand in one row, cut into equal runs; a workgroup takes one run for
// one KV head and 32 query rows a wave, two waves a SIMD. Its waves share a tile: its rows come by LDS DMA two tiles ahead, and
// each wave converts 4 keys (D below 256, 4 waves: 8) for all the rows, between the matrix instructions of the tile before:
//   K   quants to 16-byte units [block][half][key], the A operands of v_mfma_i32_32x32x32_i8, a whole q8_0 block each
//   V   to f16 pairs hi + lo of vq dv 2^(22 - e), e the exponent of the key's largest dv (dv < 2^(e - 14)), transposed: a
//       unit holds 8 keys of one dim, in the order in which S^T leaves them in the registers
//   S^T = K Q^T: a lane has one query row and 16 keys. The shift of V enters S as e - 22, where it starts, so that
//       P = 2^(s + e - 22 - M) times the stored V is 2^(s - M) v, and the sum takes P 2^(22 - e). The reference M is the
//       running maximum of the shifted scores less 8, so P lies below 2^8 (2^14 before M follows), as in k_paged_attn.
//   O^T = V^T P^T, v_mfma_f32_32x32x16_f16: P, an f16 pair too, is the B operand as it lies; hi hi + hi lo + lo hi, 2^-22, for
//       every type (one f16 each would be 2^-10 off of the sum of p |v|, which bf16's own rounding hides only where the value is
//       as large as that sum)
// Scaling V instead of P dv once a block keeps 20 vector instructions a score out of the loop (8 blocks of D 256). O takes 128
// registers of D 256, so the queries' scales and five of their blocks lie in LDS.
//
// 8 requests of 12295 tokens, 64 nodes, 16 heads, f32: 258 us with the parts' merge (about 20) on one card, 274 on another, passes
// one after another (bursts of ten and kernels under the profiler take up to a tenth more), 0.38 to 0.40 P operations/s: the vector
// units are busy for 58 % of the cycles, the matrix units for 31 %. A tile takes a wave 9900 cycles on average: 2700 the
// scores, 800 the softmax, 3800 the product with the next tile's conversion, 900 addresses, 1700 at the barrier (2600 of the
// waves that come to the scores first, 750 of the others). D 256 spills 6 vector registers.
// 16 ragged requests, 32 nodes, 16 heads, bf16: 130 us; V and P as one f16 each 115.
// Slower: one half of the waves a phase behind the other with two barriers a tile, so that a product stands beside scores
// (292 us), 4 waves of 64 rows with the registers of a whole SIMD (spills), operands of the product read further ahead (spills),
// the conversion before the scores (291 us). Of D 128 and 64 two workgroups of 4 waves share a CU, each lane with a key's 4
// values: 4 requests of 9001 tokens, 24 nodes, 8 KV heads of 128, f16, 76 us; with 8 waves, half of their lanes idle, 112.
#include "paged_device.h"

#include <type_traits>
#include <utility>

namespace qwfn {
namespace {

typedef int      v16i __attribute__((ext_vector_type(16)));
typedef float    v16f __attribute__((ext_vector_type(16)));
typedef uint16_t v2us __attribute__((ext_vector_type(2)));

constexpr int TA_LEAD = 4;             // tiles that a request counts more than it has
constexpr int TA_E0 = 22;              // a key's dv are stored times 2^(TA_E0 - e), below 2^8

template <int D, int WAVES> struct ta_cfg {
    static constexpr int PER_CU = 8 / WAVES, THREADS = 64 * WAVES, ROWS = 32 * WAVES;      // workgroups a CU, by registers
    // of 4 keys of a tile, a wave, D / 4 lanes each
    static constexpr int GROUPS = 8 / WAVES;
    static_assert(GROUPS * D <= 256, "a lane for each");
    static constexpr int NBLK = D / QK, SEG = NBLK * QBLOCK;
    static constexpr int UB = SEG % 16 == 0 ? 16 : 4, UV = SEG / UB;      // DMA units, as in k_paged_attn
    static constexpr int LS = (SEG + 15) / 16 * 16, UPR = LS / UB;
    // a wave brings in its groups' rows of K and V
    static constexpr int UNITS = GROUPS * 8 * UPR, DMAS = (UNITS + 63) / 64;
    static constexpr int UMUL = 65536 / UPR + 1;
    static constexpr int GROUP = GROUPS * 8 * LS, RAW = WAVES * GROUP;
    // an image: K, V, K's scales, the keys' shifts and their inverses
    static constexpr int OV = NBLK * 1024, OS = OV + 2 * NBLK * 2048, OE = OS + NBLK * PA_TILE * 2, OW = OE + PA_TILE * 4, IMG = OW + PA_TILE * 4;
    static constexpr int OI = RAW, OA = OI + 2 * IMG;
    // and of the queries the scales [wave][block][row] and, of D 256, the later blocks [wave][block][lane], which the registers do not hold
    static constexpr int QREG = NBLK == 8 ? 3 : NBLK, OQ = OA + ROWS * NBLK * 4, LDS = OQ + WAVES * (NBLK - QREG) * 1024;
    static_assert((UNITS - 1) * (UMUL * UPR - 65536) < 65536, "all keys, the division is exact");
    static_assert(RAW % 16 == 0 && OV % 16 == 0 && OS % 16 == 0 && OE % 16 == 0 && IMG % 16 == 0, "aligned");
    static_assert(WAVES * NBLK * 1024 <= OA, "the queries fit");
    static_assert(PER_CU * (LDS + 128) <= 160 * 1024, "LDS of a CU");
};

// The workgroup's LDS writes are done, then all its waves are here. (Not __syncthreads: DMA stays in flight over it.)
__device__ __forceinline__ void block_sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float max_halves(float x) {                    // lanes l and l ^ 32
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    unsigned p = r[0], q = r[1];
    asm volatile("" : "+v"(p), "+v"(q));
    return vmax(__builtin_bit_cast(float, p), __builtin_bit_cast(float, q));
}
__device__ __forceinline__ float sum_halves(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    unsigned p = r[0], q = r[1];
    asm volatile("" : "+v"(p), "+v"(q));
    return __builtin_bit_cast(float, p) + __builtin_bit_cast(float, q);
}
__device__ __forceinline__ uint32_t pk_max(uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2us, x), __builtin_bit_cast(v2us, y)));
}
// the larger of lanes l and l ^ 8, l ^ 16 or l ^ 32, of both halves of a dword
template <int BIT> __device__ __forceinline__ uint32_t pk_max_lanes(uint32_t x) {
    if constexpr (BIT == 8) return pk_max(x, dev::dpp_u32<0x128>(x));     // row_ror:8
    const auto r = BIT == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false) : __builtin_amdgcn_permlane32_swap(x, x, false, false);
    unsigned p = r[0], q = r[1];
    asm volatile("" : "+v"(p), "+v"(q));
    return pk_max(p, q);
}

__device__ __forceinline__ uint32_t pk_f16(float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y)); }
// x and y as f16: hi cut off, lo the rest.
__device__ __forceinline__ void split2(float x, float y, uint32_t & hi, uint32_t & lo) {
    hi = pk_f16(x, y);
    float x1, y1;                                          // (the compiler takes two instructions each)
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(x1) : "v"(hi), "v"(x));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y1) : "v"(hi), "v"(y));
    lo = pk_f16(x1, y1);
}
template <int B> __device__ __forceinline__ float byte_f32(uint32_t w) { return (float) (int8_t) (w >> (8 * B)); }

__device__ __forceinline__ v16f mfma_f16(v4u x, v4u y, v16f z) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), z, 0, 0, 0);
}

template <typename F, int... X> __device__ __forceinline__ void for_blocks(F & fn, std::integer_sequence<int, X...>) {
    (fn(std::integral_constant<int, X>{}), ...);
}

template <int D, int TYPE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void k_paged_tree(pa_args a) {
    using C = ta_cfg<D, WAVES>;
    constexpr int NBLK = C::NBLK;
    __shared__ __attribute__((aligned(16))) uint8_t lds[C::LDS];
    __shared__ int32_t sh[WAVES + 3], odd[4];
    int tid = threadIdx.x;
#define lane (tid & 63)
#define ln (tid & 31)
#define half (tid >> 5 & 1)
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // blocks -> (run, KV head, row group): those of one run follow each other on one XCD
    const uint32_t jb = blockIdx.x >> 3, jq = div_by(jb, a.f_inner), hr = jb - jq * a.f_inner.d;
    const int g = (int) jq * 8 + (int) (blockIdx.x & 7), rg = (int) div_by(hr, a.f_kv), kvh = (int) hr - rg * a.nh_kv;
    auto length = [&](int32_t b) { return tree_len(a, b, rg); };
    pa_run run = find_run<WAVES, 1, TA_LEAD>(a, g, sh, length);

    const uint32_t at_raw = pa_lds(lds) + wave * C::GROUP;
    const char * kh = a.k + (size_t) kvh * a.nb2;
    const char * vh = a.v + (size_t) kvh * a.nb2;
    const uint64_t v_k = (uint64_t) (vh - kh);
    constexpr size_t es = TYPE == QWFN_TYPE_F32 ? 4 : 2;
    // the lane's query row
    struct place { int row; uint32_t node, head; };
    auto query = [&]() {
        const int row = rg * C::ROWS + 32 * wave + ln, at = row < a.R ? row : a.R - 1;
        const uint32_t node = div_by((uint32_t) at, a.f_rep);
        return place{row, node, (uint32_t) (kvh * a.rep + at) - node * (uint32_t) a.rep};
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
        const int32_t nodes = tree_nodes(a, b, n), base = n - nodes;
        asm volatile("" : "+v"(tid));
        const bool busy = rg * C::ROWS + 32 * wave < nodes * a.rep;                   // the wave has a row

        const int32_t end = (run.off + nt) * PA_TILE < n ? (run.off + nt) * PA_TILE : n;
        // (the divisor's parts from scalar registers each time: kept in vector ones over the loop they are spilled)
        auto page_of = [&](uint32_t key) {
            uint32_t m = a.page.m, sh1 = a.page.s;
            asm volatile("" : "+s"(m), "+s"(sh1));
            return sh1 == 0 ? key : __umulhi(key, m) >> (sh1 - 1);
        };
        // a tile's table entries (lanes l and l + 32 the same key), clipped to the part's last key
        auto entries = [&](int t) -> int32_t {
            int32_t key = (run.off + t) * PA_TILE + ln;
            key = key < end ? key : end - 1;
            return table[page_of((uint32_t) key)];
        };
        // the DMAs of the wave's keys of tile t, from its entries; which of the tile's keys exist
        auto send = [&](int t, int32_t page, uint32_t at) -> uint32_t {
            const int32_t key = (run.off + t) * PA_TILE + ln;
            const bool in = t < nt && key < end, ok = in && (uint32_t) page < (uint32_t) a.n_pages;
            if (in && !ok) atomicOr(a.status, DEVERR_GET_ROWS_INDEX);
            const uint32_t slot = ok ? (uint32_t) page * a.page.d + ((uint32_t) key - page_of((uint32_t) key) * a.page.d) : 0u;
            uint64_t from[C::DMAS];
#pragma unroll
            for (int i = 0; i < C::DMAS; i++) {
                const int x = lane + 64 * i, row = (x * C::UMUL) >> 16, u = x - row * C::UPR;
                const uint32_t sl = (uint32_t) __shfl((int) slot, 4 * (wave + WAVES * (row >> 3)) + (row & 3));
                from[i] = (uint64_t) (uintptr_t) kh + (uint64_t) sl * a.nb1 + (uint32_t) ((u < C::UV ? u : C::UV - 1) * C::UB) + (row & 4 ? v_k : 0ull);
            }
            if (t < nt)
#pragma unroll
                for (int i = 0; i < C::DMAS; i++)
                    if (64 * (i + 1) <= C::UNITS || lane + 64 * i < C::UNITS) pa_dma<C::UB>(from[i], at + 64 * C::UB * i);
            return (uint32_t) __ballot(ok);
        };
        block_sync();                                      // the LDS of the part before is read
        if (tid < 4) odd[tid] = 0;
        int32_t page = entries(0), page1 = entries(1);
        v4i qw[C::QREG];
        uint8_t * const ql = lds + C::OQ + wave * ((NBLK - C::QREG) * 1024);
        float * const dq = (float *) (lds + C::OA) + wave * (NBLK * 32);      // [block][row], dq c to 22 bits: PA_IBIAS dq is exact
        {
            const place me = query();
            // the lane's 16 values of each block of its row; those that the short rounding does not hold for (q8_device.h) by the
            // LDS, a block at a time
            const char * qp = a.q + (size_t) me.node * a.q_nb1 + (size_t) me.head * a.q_nb2 + (size_t) b * a.q_nb3 + (size_t) (16 * half) * es;
            auto values = [&](int blk, float (&x)[16], dev::q8_scale & sc) -> bool {
#pragma unroll
                for (int i = 0; i < 4; i++) load4(qp + (size_t) (QK * blk + 4 * i) * es, TYPE, x + 4 * i);
                uint32_t am = 0;
#pragma unroll
                for (int i = 0; i < 16; i++) am = max(am, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
                am = umax_halves(am);
                sc = dev::q8_block_scale(__builtin_bit_cast(float, am), a.x86 != 0);
                return am >= dev::Q8_AMAX_NORMAL_MIN && am < 0x7f800000u;
            };
            bool normal = a.x86 != 0;
#pragma unroll
            for (int blk = 0; blk < NBLK; blk++) {
                float x[16];
                dev::q8_scale sc;
                normal &= values(blk, x, sc);
                v4i w;
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = (int) dev::q8_pack4_x86_normal(x + 4 * i, sc.id);
                if (blk < C::QREG) qw[blk < C::QREG ? blk : 0] = w;
                else *(v4i *) (ql + (blk - C::QREG) * 1024 + lane * 16) = w;
                const float d = dev::f16_bits_to_f32(dev::f32_to_f16_bits(sc.d));
                dq[blk * 32 + ln] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, d * a.c) + 2u) & ~3u);
            }
            if (__ballot(!normal)) {
                uint8_t * const my = lds + wave * (NBLK * 1024);
#pragma unroll 1
                for (int blk = 0; blk < NBLK; blk++) {
                    float x[16];
                    dev::q8_scale sc;
                    values(blk, x, sc);
                    v4i w;
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = (int) dev::q8_pack4(x + 4 * i, sc.id, a.x86 != 0);
                    *(v4i *) (my + blk * 1024 + lane * 16) = w;
                }
                wave_lds_sync();
#pragma unroll
                for (int blk = 0; blk < NBLK; blk++) {
                    const v4i w = *(const v4i *) (my + blk * 1024 + lane * 16);
                    if (blk < C::QREG) qw[blk < C::QREG ? blk : 0] = w;
                    else *(v4i *) (ql + (blk - C::QREG) * 1024 + lane * 16) = w;
                }
                wave_lds_sync();
            }
#pragma unroll
            for (int blk = 0; blk < C::QREG; blk++) asm volatile("" : "+v"(qw[blk]));
        }
        block_sync();
        uint32_t live = send(0, page, at_raw);
        page = entries(2);

        v16f O[NBLK] = {};
        float M = -INFINITY, l = 0.f;
        v16i ib;
#pragma unroll
        for (int i = 0; i < 16; i++) ib[i] = PA_IBITS;

        // ---- the wave's keys of a tile into its images, C::GROUPS groups in steps that stand between matrix instructions: a lane 4
        // values of each of its group's keys' K, then of their V (of D 64 and 128 not always all lanes)
        struct { uint32_t w[4], w2[4], dv[4]; float d[4]; } cv;
#define cl (lane & (D / 4 - 1))
        constexpr bool all = D * C::GROUPS == 256;
        auto cv_read = [&](int first) {                    // (a scale by the dword that holds it)
            const int blk = cl >> 3, j = lane & 7, at = QBLOCK * blk + (blk & 1 ? 2 : 0), which = C::GROUPS == 1 ? 0 : lane / (D / 4);
            const uint8_t * raw = lds + wave * C::GROUP + (first + 8 * which) * C::LS + at;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                cv.w[k] = *(const uint32_t *) (raw + 4 * j + k * C::LS);
                cv.w2[k] = *(const uint32_t *) (raw + 4 * j + 4 + k * C::LS);
                cv.dv[k] = *(const uint32_t *) (raw - (blk & 1 ? 4 : 0) + k * C::LS);
            }
        };
        auto cv_align = [&]() {
            const uint32_t sh8 = lane & 8 ? 0u : 2u, sh16 = lane & 8 ? 16u : 0u;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                cv.w[k] = __builtin_amdgcn_alignbyte(cv.w2[k], cv.w[k], sh8);
                cv.dv[k] = __builtin_amdgcn_ubfe(cv.dv[k], sh16, 16);
            }
        };
        auto convert = [&](auto X, int t, uint32_t alive, uint8_t * img) {
            constexpr int x = X.value;
            if (!all && lane >= C::GROUPS * (D / 4)) return;
            const int blk = cl >> 3, j = lane & 7, group = wave + (C::GROUPS == 1 ? 0 : WAVES * (lane / (D / 4)));
            if constexpr (x == 0) cv_read(0);
            if constexpr (x == 1) {
                // K: word j & 3 of unit (block, half j >> 2, key), units of a plane turned by the plane's number
                cv_align();
#pragma unroll
                for (int k = 0; k < 4; k++)
                    *(uint32_t *) (img + (cl >> 2) * 512 + ((4 * group + k + (cl >> 2)) & 31) * 16 + (j & 3) * 4) = cv.w[k];
                if (j == 0) *(uint2 *) (img + C::OS + (blk * PA_TILE + 4 * group) * 2) = make_uint2(cv.dv[0] | cv.dv[1] << 16, cv.dv[2] | cv.dv[3] << 16);
                cv_read(4);
            }
            if constexpr (x == 2) {
                cv_align();
                bool bad = false;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const bool on = alive >> (4 * group + k) & 1, fine = (cv.dv[k] & 0x7fffu) < 0x7c00u;
                    bad |= on && !fine;
                    cv.dv[k] = on && fine ? cv.dv[k] : 0u;
                }
                if (bad) odd[t & 3] = 1;
            }
            if constexpr (x == 3) {
                uint32_t m[2], e[4];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    m[k] = (cv.dv[2 * k] | cv.dv[2 * k + 1] << 16) & 0x7fff7fffu;
                    m[k] = pk_max_lanes<8>(m[k]);
                    if constexpr (D >= 128) m[k] = pk_max_lanes<16>(m[k]);
                    if constexpr (D >= 256) m[k] = pk_max_lanes<32>(m[k]);
                }
                auto up = [](uint32_t e1) { return __builtin_bit_cast(float, (127 + TA_E0 - e1) << 23); };
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    e[k] = k & 1 ? m[k / 2] >> 26 : m[k / 2] >> 10 & 31u;
                    e[k] = e[k] < 1 ? 1u : e[k];
                    cv.d[k] = dev::f16_bits_to_f32((uint16_t) cv.dv[k]) * up(e[k]);
                }
                const uint32_t mine = cl & 2 ? (cl & 1 ? e[3] : e[2]) : (cl & 1 ? e[1] : e[0]);
                if (cl < 4) {
                    *(float *) (img + C::OE + 4 * (4 * group + cl)) = (float) ((int) mine - TA_E0);
                    *(float *) (img + C::OW + 4 * (4 * group + cl)) = up(mine);
                }
            }
            if constexpr (x >= 4) {
                // V, dim x - 4 of the lane's: keys 16 s + 4 h + 8 y + r are halves y of unit 2 s + h
                constexpr int B = x - 4;
                uint8_t * out = img + C::OV + (blk * 4 + 2 * (group >> 2) + (group & 1)) * 512 + j * 16 + (group >> 1 & 1) * 8;
                float f[4];
#pragma unroll
                for (int k = 0; k < 4; k++) f[k] = byte_f32<B>(cv.w[k]) * cv.d[k];
                uint2 hi, lo;
                split2(f[0], f[1], hi.x, lo.x);
                split2(f[2], f[3], hi.y, lo.y);
                *(uint2 *) (out + B * 128) = hi;
                *(uint2 *) (out + NBLK * 2048 + B * 128) = lo;
            }
        };
        // the steps from 1 of block X of NBLK
        auto convert_some = [&](auto X, int t, uint32_t alive, uint8_t * img) {
            constexpr int N = 8 / NBLK;
            auto step = [&](auto S) {
                if constexpr (1 + N * decltype(X)::value + S.value < 8)
                    convert(std::integral_constant<int, 1 + N * decltype(X)::value + S.value>{}, t, alive, img);
            };
            for_blocks(step, std::make_integer_sequence<int, N>{});
        };
        constexpr std::integral_constant<int, 0> step0;
        auto each_block = [&](auto fn) {
            for_blocks(fn, std::make_integer_sequence<int, NBLK>{});
        };

        // ---- S^T of a row tile, a block a step: the block's matrix instruction, and the sums of the one before
        typedef _Float16 v4h __attribute__((ext_vector_type(4)));
        struct kread { v4i kw, qw; v4h dk[2][4]; float dq[2]; } kr;
        float s[16];
        auto qk_read = [&](int blk, const uint8_t * img) {
            kr.kw = *(const v4i *) (img + (2 * blk + half) * 512 + ((ln + 2 * blk + half) & 31) * 16);
            if (blk >= C::QREG) kr.qw = *(const v4i *) (ql + (blk - C::QREG) * 1024 + lane * 16);
        };
        auto qk_scales = [&](int blk, const uint8_t * img) {
            kr.dq[blk & 1] = dq[blk * 32 + ln];
#pragma unroll
            for (int x = 0; x < 4; x++) kr.dk[blk & 1][x] = *(const v4h *) (img + C::OS + (blk * PA_TILE + 8 * x + 4 * half) * 2);
        };
        auto qk_begin = [&](const uint8_t * img) {
            qk_read(0, img);
            qk_scales(0, img);
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const v4f e = *(const v4f *) (img + C::OE + (8 * x + 4 * half) * 4);
#pragma unroll
                for (int r = 0; r < 4; r++) s[4 * x + r] = e[r];
            }
        };
        auto qk_sums = [&](int blk, const v16i & dots) {
            const float f = kr.dq[blk & 1];
            const float nb = -PA_IBIAS * f;
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int d = dots[4 * x + r];
                    s[4 * x + r] = __fmaf_rn((float) kr.dk[blk & 1][x][r], __fmaf_rn(__builtin_bit_cast(float, d), f, nb), s[4 * x + r]);
                }
        };
        auto qk_dots = [&](int blk) {
            return __builtin_amdgcn_mfma_i32_32x32x32_i8(kr.kw, blk < C::QREG ? qw[blk < C::QREG ? blk : 0] : kr.qw, ib, 0, 0, 0);
        };

        // blocks of V whose scale is not finite, for the rows that see their key (their values from the cache again)
        auto rare_v = [&](const float (&p)[16], int t, uint32_t alive, const uint8_t * img) {
#pragma unroll 1
            for (int k = 0; k < PA_TILE; k++) {
                if (!(alive >> k & 1)) continue;
                const uint32_t key = (uint32_t) ((run.off + t) * PA_TILE + k), pg = page_of(key);
                const char * vr = vh + (uint64_t) ((uint32_t) table[pg] * a.page.d + (key - pg * a.page.d)) * a.nb1;
                float pk = 0.f;
#pragma unroll
                for (int i = 0; i < 16; i++) pk = 4 * (k >> 3) + (k & 3) == i ? p[i] : pk;
                pk = __shfl(pk, ln + 32 * (k >> 2 & 1)) * *(const float *) (img + C::OW + 4 * k);
#pragma unroll
                for (int blk = 0; blk < NBLK; blk++) {
                    const uint16_t d = *(const uint16_t *) (vr + QBLOCK * blk);
                    if ((__builtin_amdgcn_readfirstlane(d) & 0x7fff) < 0x7c00) continue;
                    const float pd = pk * dev::f16_bits_to_f32(d);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float y = pd * (float) *(const int8_t *) (vr + QBLOCK * blk + 2 + 16 * half + 4 * (i & 3) + (i >> 2));
                        O[blk][i] += pk != 0.f ? y : 0.f;
                    }
                }
            }
        };

        // ---- the softmax step of a row tile: P in ph, pl
        v4u ph[2], pl[2];
        auto softmax = [&](int t, uint32_t alive, bool rare, const uint8_t * img) {
            const int32_t key0 = (run.off + t) * PA_TILE;
            float (&sr)[16] = s;
            float p[16];
            if (alive != 0xffffffffu || key0 + PA_TILE > base) {
                const place me = query();                // (read here: kept over the loop the masks cost registers)
                const uint64_t mask = me.row < a.R && (int32_t) me.node < nodes ? a.masks[(int64_t) b * a.T + me.node] : 0;
                const uint32_t sees = (alive & tree_sees(mask, key0, base)) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!(sees >> (8 * (i >> 2) + (i & 3)) & 1)) sr[i] = -INFINITY;
            }
            float top = vmax(vmax(vmax(sr[0], sr[1]), vmax(sr[2], sr[3])), vmax(vmax(sr[4], sr[5]), vmax(sr[6], sr[7])));
            top = vmax(top, vmax(vmax(vmax(sr[8], sr[9]), vmax(sr[10], sr[11])), vmax(vmax(sr[12], sr[13]), vmax(sr[14], sr[15]))));
            const float ref = max_halves(top) - (float) PA_BIAS;
            if (__ballot(ref > M + PA_SLACK)) {
                const float to = fmaxf(M, ref);
                const float f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - to);
                M = to;
                l *= f;
#pragma unroll
                for (int blk = 0; blk < NBLK; blk++) O[blk] *= f;
            }
            const float m0 = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const v4f w = *(const v4f *) (img + C::OW + (8 * x + 4 * half) * 4);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    p[4 * x + r] = __builtin_amdgcn_exp2f(sr[4 * x + r] - m0);       // 2^-inf = 0
                    l = __fmaf_rn(p[4 * x + r], w[r], l);
                }
            }
#pragma unroll
            for (int st = 0; st < 2; st++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t hi, lo;
                    split2(p[8 * st + 2 * k], p[8 * st + 2 * k + 1], hi, lo);
                    ph[st][k] = hi;
                    pl[st][k] = lo;
                }
            if (__builtin_expect(rare, 0)) rare_v(p, t, alive, img);
        };

        // ---- O^T of a row tile, a block a step
        v4u va[2][2];                                      // (half a block ahead: a whole one costs 16 registers)
        auto pv_read = [&](int blk, int st, const uint8_t * img) {
#pragma unroll
            for (int x = 0; x < 2; x++) va[st][x] = *(const v4u *) (img + C::OV + half * 512 + ln * 16 + x * (NBLK * 2048) + (blk * 4 + 2 * st) * 512);
        };
        auto pv_half = [&](int blk, int st) {
            O[blk] = mfma_f16(va[st][0], ph[st], O[blk]);
            O[blk] = mfma_f16(va[st][0], pl[st], O[blk]);
            O[blk] = mfma_f16(va[st][1], ph[st], O[blk]);
        };
        // Tile t is multiplied from one image while t + 1 becomes the other and the rows of t + 2 are on their way. A wave converts
        // the keys that it has brought in itself, so one barrier a tile is for the images alone.
        pa_wait<0>();
        convert(step0, 0, live, lds + C::OI);
        each_block([&](auto X) { convert_some(X, 0, live, lds + C::OI); });
        pa_wait_lds();
        uint32_t next = send(1, page1, at_raw);
        block_sync();
        for (int t = 0; t < nt; t++) {
            asm volatile("" : "+v"(tid));                  // the lane's places are computed anew: kept over the loop they cost registers
            const uint8_t * const img = lds + C::OI + (t & 1) * C::IMG;
            if (tid == 0) odd[(t + 2) & 3] = 0;
            uint8_t * const img1 = lds + C::OI + (~t & 1) * C::IMG;
            if (busy) {
                __builtin_amdgcn_s_setprio(2);             // (before another wave's product: it needs the matrix cores between)
                qk_begin(img);
                each_block([&](auto X) {
                    constexpr int blk = X.value;
                    const v16i d = qk_dots(blk);
                    if constexpr (blk + 1 < NBLK) {
                        qk_read(blk + 1, img);
                        qk_scales(blk + 1, img);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    qk_sums(blk, d);
                    __builtin_amdgcn_sched_barrier(0);
                });
                pa_wait<0>();
                convert(step0, t + 1, next, img1);
                pv_read(0, 0, img);
                softmax(t, live, odd[t & 3] != 0, img);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                // the product, and the next tile's images between
                each_block([&](auto X) {
                    constexpr int blk = X.value;
                    pv_read(blk, 1, img);
                    __builtin_amdgcn_sched_barrier(0);
                    pv_half(blk, 0);
                    convert_some(X, t + 1, next, img1);
                    if constexpr (blk + 1 < NBLK) pv_read(blk + 1, 0, img);
#pragma unroll
                    for (int i = 0; i < 3; i++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    pv_half(blk, 1);
                    __builtin_amdgcn_sched_barrier(0);
                });
            } else {
                pa_wait<0>();
                convert(step0, t + 1, next, img1);
                each_block([&](auto X) { convert_some(X, t + 1, next, img1); });
            }
            pa_wait_lds();
            const uint32_t after = send(t + 2, page, at_raw);
            page = entries(t + 3);
            block_sync();
            live = next;
            next = after;
        }
        pa_wait<0>();

        // dim 16 half + 4 x + y of a block in O[blk][4 y + x]
        asm volatile("" : "+v"(tid));
        {
            const place to = query();
            const float ll = sum_halves(l);
            const bool alive = to.row < a.R && (int32_t) to.node < nodes;
            const size_t elem = (((size_t) b * a.T + to.node) * a.nh + to.head) * D + 16 * half;
            const size_t part = ((size_t) (g + b) * a.nh_kv + kvh) * a.R + to.row;
            const float inv = !alive ? 0.f : ll > 0.f ? 1.f / ll : ll == ll ? 0.f : ll;
            if (whole && to.row < a.R) {
#pragma unroll
                for (int blk = 0; blk < NBLK; blk++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        float o[4];
#pragma unroll
                        for (int y = 0; y < 4; y++) o[y] = alive ? O[blk][4 * y + x] * inv : 0.f;
                        finish4<TYPE>(a, elem + QK * blk + 4 * x, o, alive ? ll : 0.f);
                    }
            } else if (to.row < a.R) {
                if (half == 0) a.part_ml[part] = alive ? make_float2(M, ll) : make_float2(-INFINITY, 0.f);
                // (as the registers lie, k_tree_merge takes them so: a store writes 1 KB in one piece)
                const int tile = rg * (C::ROWS / 32) + wave;
                float * po = a.part_o + (((size_t) (g + b) * a.nh_kv + kvh) * ((a.R + 31) / 32) + tile) * (32 * D) + lane * 4;
                if (alive)
#pragma unroll
                    for (int blk = 0; blk < NBLK; blk++)
#pragma unroll
                        for (int x = 0; x < 4; x++)
                            *(float4 *) (po + (blk * 4 + x) * 256) = make_float4(O[blk][x], O[blk][4 + x], O[blk][8 + x], O[blk][12 + x]);
            }
        }
        if (run.off == 0 && kvh == 0 && tid == 0) a.span[rg * a.n_seq + b] = make_int2(g, (run.pos + tiles - 1) / run.per);
        run.left -= nt;
        run.pos += nt;
        run.off = -TA_LEAD;
        if (run.left > 0)
            do run.n = length(++run.b);
            while (run.n == 0);
    }
    // requests without a node in the group or without a key, and numbers that were clipped
    for (int b = g; b < a.n_seq; b += (int) (gridDim.x / a.f_inner.d)) {
        const int32_t n = a.n_kv[b];
        bool wrong = n != clip_len(a, n);
        if (a.n_tree) wrong |= a.n_tree[b] != tree_nodes(a, b, clip_len(a, n));
        if (wrong && tid == 0) atomicOr(a.status, DEVERR_GET_ROWS_INDEX);
        if (length(b) > 0) continue;
        const float z[4] = {0.f, 0.f, 0.f, 0.f};
        for (int x = tid; x < C::ROWS * (D / 4); x += C::THREADS) {
            const int r = rg * C::ROWS + x / (D / 4);
            if (r >= a.R) break;
            const uint32_t t = div_by((uint32_t) r, a.f_rep), h = (uint32_t) (kvh * a.rep + r) - t * (uint32_t) a.rep;
            store4(a.dst + ((((size_t) b * a.T + t) * a.nh + h) * D + 4 * (x % (D / 4))) * es, TYPE, z);
        }
        if (kvh == 0 && tid == 0) a.span[rg * a.n_seq + b] = make_int2(0, 0);
    }
#undef lane
#undef ln
#undef half
#undef cl
}

template <int D, int WAVES>
void launch(const pa_args & a, int groups, hipStream_t s) {
    const dim3 grid((unsigned) ((int64_t) (a.runs + 7) / 8 * 8 * a.nh_kv * groups)), blk(64 * WAVES);
    if (a.type == QWFN_TYPE_BF16)     hipLaunchKernelGGL((k_paged_tree<D, QWFN_TYPE_BF16, WAVES>), grid, blk, 0, s, a);
    else if (a.type == QWFN_TYPE_F16) hipLaunchKernelGGL((k_paged_tree<D, QWFN_TYPE_F16, WAVES>), grid, blk, 0, s, a);
    else                              hipLaunchKernelGGL((k_paged_tree<D, QWFN_TYPE_F32, WAVES>), grid, blk, 0, s, a);
}

}  // namespace

// Of D 256 the images and the queries leave no LDS for a second workgroup of a CU.
int tree_rows(int64_t D) { return D == 256 ? 256 : 128; }
int launch_tree_attn(const pa_args & a, int64_t D, int groups, hipStream_t s) {
    if (D == 256)      launch<256, 8>(a, groups, s);
    else if (D == 128) launch<128, 4>(a, groups, s);
    else               launch<64, 4>(a, groups, s);
    return hip_check(hipGetLastError(), "flash_attn_ext_paged_tree launch");
}

}  // namespace qwfn
