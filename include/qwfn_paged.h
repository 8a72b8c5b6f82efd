/*
 * qwfn_paged.h -- C ABI of the paged q8_0 KV cache: many requests of different
 * lengths in one pool of fixed-size pages, for batched decoding.
 *
 * The reference serves one sequence per cache, so nothing here has a
 * counterpart in it; the cache rows are the ones of qwfn_kv.h. A pool is one K
 * and one V cache tensor (q8_0 [kv_dim, n_rows], token-major rows); page p holds
 * rows p * page_size .. p * page_size + page_size - 1. Token j of request b lies
 * in row ("slot") table[b][j / page_size] * page_size + j % page_size. The block
 * tables are I32 [n_seq][max_pages] rows in device memory; entries past a
 * request's ceil(length / page_size) pages are never read and may hold anything.
 * Free pages are a stack free_pages[0 .. n_free) in device memory.
 *
 * A decoding step: qwfn_paged_extend makes room and lists the new tokens' slots
 * (qwfn_paged_extend_states those of recurrent states too);
 * qwfn_set_rows_q8_0_kv (qwfn_kv.h) with idx = slots appends their K and V rows
 * in every layer; qwfn_flash_attn_ext_q8_0_paged attends; qwfn_paged_trim gives
 * back the pages of finished requests and rejected drafts. For a prompt,
 * qwfn_get_rows_i32 over a request's slots gathers its rows into a contiguous
 * cache for qwfn_flash_attn_ext_q8_0.
 *
 * Conventions are those of qwfn_kv.h. Lengths, tables and lists are device
 * memory, so a whole step can be captured into a graph and replayed.
 */
#ifndef QWFN_PAGED_H
#define QWFN_PAGED_H

#include "qwfn_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Workspace of qwfn_paged_extend and qwfn_paged_trim for n_seq requests. Calls
 * that run at the same time need distinct workspaces; the contents need not be
 * kept between calls. */
size_t qwfn_paged_workspace_size(int32_t n_seq);

/* Room for n_new[b] more tokens behind the n_past[b] of each request b < n_seq,
 * and the lists that a step over the new tokens needs. With P = page_size:
 *   need_b = ceil((n_past + n_new) / P) - ceil(n_past / P)   pages
 *   request b is served if its n_past + n_new tokens fit max_pages pages, its new
 *   tokens lie below n_tok, and need_b = 0 or the needs of the requests up to and
 *   including b, those left out that fail the first two tests, sum to at most
 *   n_free. A request that is not served keeps its length and takes no page.
 *   pages come off the top of the stack in order of the requests: the i-th page
 *   that the call hands out is free_pages[n_free - 1 - i].
 * Writes:
 *   table[b]     the new columns of the served requests, nothing else
 *   n_free_out   n_free less the pages handed out (may be n_free itself)
 *   n_kv         I32 [n_seq]: n_past + n_new where served, else n_past (may be
 *                n_past itself)
 *   cu_new       I32 [n_seq + 1]: the tokens of request b are cu_new[b] ..
 *                cu_new[b + 1] - 1 of the lists below, served or not; at most n_tok
 *   slots        I32 [n_tok]: the cache row of each new token, pad_slot for a token
 *                whose request is not served and for entries past cu_new[n_seq]
 *                (-1, which qwfn_set_rows_* skip with bit 0 of the device status,
 *                or a row the caller keeps for this)
 *   pos          I32 [n_tok] or NULL: each token's position, -1 where slots has
 *                pad_slot
 *   seq          I32 [n_tok] or NULL: each token's request, -1 past cu_new[n_seq]
 * Any request not served, a negative n_past or n_new (taken as 0) and an n_free
 * outside [0, free_cap] (clipped) set bit 2 of qwfn_device_status. A table entry
 * of a partly filled page that names no row below 2^31 gives pad_slot and sets
 * the same bit. n_seq <= 65536, max_pages * page_size and table_stride (entries
 * from one request's row to the next) < 2^31; apart from the two
 * in-place pairs no output may overlap an input or another output. One launch;
 * two where n_tok is more than 8 tokens a request and a pair is in place or n_seq
 * above 1024. */
int qwfn_paged_extend(const int32_t * n_past, const int32_t * n_new, int32_t n_seq, int32_t page_size, int32_t * table,
                      int64_t table_stride, int32_t max_pages, const int32_t * free_pages, int32_t free_cap,
                      const int32_t * n_free, int32_t * n_free_out, int32_t * n_kv, int32_t * cu_new, int32_t * slots,
                      int32_t * pos, int32_t * seq, int64_t n_tok, int32_t pad_slot, void * ws, size_t ws_bytes,
                      void * stream);

/* The same, and for recurrent layers beside the cache (qwfn_linear_attn of
 * qwfn_state.h, which takes cu_new) the state slots of the step:
 *   states       I32 [n_seq] or NULL: the request's state slot, -1 for none (NULL: b)
 *   state_slots  I32 [n_seq]: that slot where the request is served and has new
 *                tokens, else -2 - slot, which leaves the request out there and
 *                keeps its state (a negative slot is passed on as it is)
 * cu_new lists the tokens of requests that are not served too: with other slots a
 * layer would add them to states whose request stays where it was, and once more
 * when it is asked again. */
int qwfn_paged_extend_states(const int32_t * n_past, const int32_t * n_new, int32_t n_seq, int32_t page_size, int32_t * table,
                             int64_t table_stride, int32_t max_pages, const int32_t * free_pages, int32_t free_cap,
                             const int32_t * n_free, int32_t * n_free_out, int32_t * n_kv, int32_t * cu_new, int32_t * slots,
                             int32_t * pos, int32_t * seq, int64_t n_tok, int32_t pad_slot, const int32_t * states,
                             int32_t * state_slots, void * ws, size_t ws_bytes, void * stream);

/* The inverse: request b keeps its first n_keep[b] tokens (a negative count as 0,
 * one above n_kv[b] as n_kv[b]; 0 ends the request), and the pages behind them go
 * onto the stack in order of the requests, each request's in order of its
 * columns. n_kv_out I32 [n_seq]: the tokens kept (may be n_kv itself); n_free_out
 * may be n_free itself. The table is only read: its columns past the kept pages
 * become unused. A request whose pages would pass free_cap (counting those of
 * the requests before it) keeps its length and its pages and sets bit 2 of
 * qwfn_device_status, as do a negative n_kv, one above max_pages * page_size
 * (taken as 0 and as that) and an n_free outside [0, free_cap]. One launch; two
 * where a pair is in place or n_seq above 1024. */
int qwfn_paged_trim(const int32_t * n_keep, const int32_t * n_kv, int32_t n_seq, int32_t page_size, const int32_t * table,
                    int64_t table_stride, int32_t max_pages, int32_t * free_pages, int32_t free_cap,
                    const int32_t * n_free, int32_t * n_free_out, int32_t * n_kv_out, void * ws, size_t ws_bytes,
                    void * stream);

/* Attention of each request's last T tokens over its pages, the keys split over
 * the workgroups by the lengths on the device and joined by a second launch:
 *   q    F32, F16 or BF16 [D, T, n_head, n_seq] (rows contiguous, 16-byte aligned)
 *   k, v Q8_0 [D, n_rows, n_head_kv, 1] views of the pool (nb[1] the row stride,
 *        nb[2] the head's offset), n_rows / page_size pages
 *   n_kv device I32 [n_seq]: query t of request b is its token n_kv[b] - T + t and
 *        sees the tokens up to itself; a query before the first token gives 0, and
 *        so does a request of length 0 (a padded batch)
 *   dst  [D, n_head, T, n_seq] contiguous, 16-byte aligned, q's type, not
 *        overlapping q
 *   gate NULL or dst's type and shape: dst = attention * sigmoid(gate); may be dst
 * D 64, 128 or 256; n_head a multiple of n_head_kv, T * n_head / n_head_kv <= 64;
 * head rows and strides aligned to D / 16 bytes. Arithmetic as
 * qwfn_flash_attn_ext_q8_0: Q requantised to q8_0 with `variant`, exact integer
 * dots, F32 online softmax and accumulation, one rounding to dst's type. A length
 * outside [0, max_pages * page_size] is clipped to it, a table entry outside the
 * pool masks its page's keys; both set bit 1 of qwfn_device_status. Results do
 * not depend on the other requests of the batch beyond float rounding (the
 * split points), and repeat bit for bit on the same inputs.
 * ws: at least qwfn_fattn_workspace_size_paged bytes, 16-byte aligned, or NULL for
 * the library's buffer (see qwfn_flash_attn_ext_q8_0). dst and ws overlap no other tensor
 * but dst the gate. */
size_t qwfn_fattn_workspace_size_paged(const qwfn_tensor * q, const qwfn_tensor * k, const qwfn_tensor * v,
                                       int32_t max_pages, int32_t page_size);
int qwfn_flash_attn_ext_q8_0_paged(const qwfn_tensor * q, const qwfn_tensor * k, const qwfn_tensor * v,
                                   const int32_t * table, int64_t table_stride, int32_t max_pages, int32_t page_size,
                                   const int32_t * n_kv, float scale, const qwfn_tensor * gate, const qwfn_tensor * dst,
                                   int variant, void * ws, size_t ws_bytes, void * stream);

#ifdef __cplusplus
}
#endif
#endif
