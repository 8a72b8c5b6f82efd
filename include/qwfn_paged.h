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
 *   gate NULL or dst's type and shape: dst = attention * sigmoid(gate); may be dst.
 *        Rows that are 0 stay 0 whatever it holds there
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

/* --------------------------------------------------------- shared pages
 *
 * Requests may hold pages together: shared[p] (I32 [n_pages], device memory, 0
 * for a pool that starts) counts the requests that hold page p besides one, so
 * qwfn_paged_extend, whose pages nobody else holds, has nothing to write there.
 * Only whole pages are shared: the page that a request writes into is its own. A
 * pool whose requests share pages gives them back by qwfn_paged_release, not by
 * qwfn_paged_trim. shared_out, n_kv_out, n_free_out, table_out and free_out may be
 * the array that they continue; apart from that no output overlaps an input or another
 * output. n_seq <= 65536, max_pages * page_size, n_pages * page_size and
 * table_stride < 2^31. */

/* Requests that begin as copies of others (samples of one prompt, beams, a cached
 * prefix): request b with from[b] = f >= 0 gets f's first n = n_tok[b] tokens
 * (n_tok NULL: all). It is served if f < n_seq is itself not forked in this call
 * (from[f] < 0), n_kv[b] is 0, 0 <= n <= n_kv[f], and n % page_size is 0 or a page is
 * left: the requests that need one get them in order, the i-th
 * free_pages[n_free - 1 - i]. Then, with F = n / page_size, r = n % page_size:
 *   table[b][0 .. F)  f's, each page counted once more in shared_out
 *   table[b][F]       the new page, if r > 0
 *   moves[b]          I32 {source row, destination row, r} of qwfn_paged_copy, which
 *                     brings the rest over in every layer; {0, 0, 0} where r = 0
 *   state_moves[b]    (NULL: not wanted) {states[f], states[b], 1} for the recurrent
 *                     states, if n = n_kv[f] and both slots are at least 0, else
 *                     {0, 0, 0}; states NULL: request b has slot b
 *   n_kv_out[b]       n; n_kv[b] for every request that is not served
 * A request with from[b] >= 0 that is not served sets bit 2 of qwfn_device_status,
 * as do a negative n_kv, one above max_pages * page_size (taken as 0 and as that), an
 * n_free outside [0, free_cap] (clipped) and a shared page outside the pool (copied,
 * not counted; its rest not moved). ws: qwfn_paged_workspace_size bytes. */
int qwfn_paged_fork(const int32_t * from, const int32_t * n_tok, const int32_t * n_kv, int32_t n_seq, int32_t page_size,
                    int32_t * table, int64_t table_stride, int32_t max_pages, const int32_t * shared, int32_t n_pages,
                    const int32_t * free_pages, int32_t free_cap, const int32_t * n_free, int32_t * n_free_out,
                    int32_t * n_kv_out, int32_t * shared_out, int32_t * moves, const int32_t * states, int32_t * state_moves,
                    void * ws, size_t ws_bytes, void * stream);

/* qwfn_paged_trim for pages that may be shared: request b keeps its first n_keep[b]
 * tokens (0 ends it). Each page behind them counts one request less in shared_out;
 * those that nobody holds any more go onto the stack, the lowest first. A request
 * that would keep a part of a shared page (whose next token would be written into
 * the others' page) keeps its length and its pages and sets bit 2 of
 * qwfn_device_status; so do lengths and an n_free as in qwfn_paged_trim, a negative
 * shared (taken as 0), and a page outside the pool (left out). free_cap at least n_pages;
 * pages beyond it (of tables that hold one page more often than shared says) set the bit
 * and are lost. */
size_t qwfn_paged_release_workspace_size(int32_t n_seq, int32_t n_pages);
int qwfn_paged_release(const int32_t * n_keep, const int32_t * n_kv, int32_t n_seq, int32_t page_size, const int32_t * table,
                       int64_t table_stride, int32_t max_pages, const int32_t * shared, int32_t n_pages, int32_t * free_pages,
                       int32_t free_cap, const int32_t * n_free, int32_t * n_free_out, int32_t * n_kv_out,
                       int32_t * shared_out, void * ws, size_t ws_bytes, void * stream);

/* Closes the pool's holes. The pages that are not on the stack are live, n_live of
 * them; the live pages from n_live on move to the free pages below it, the k-th to the
 * k-th. Writes:
 *   page_map    I32 [n_pages]: where a live page is now, -1 for a free one (tables
 *               of other requests over the same pool are renamed by it)
 *   table_out   the ceil(n_kv / page_size) columns of every request, renamed (an entry
 *               outside the pool, or on the stack, is kept and sets bit 2 of
 *               qwfn_device_status)
 *   shared_out  of the pages where they are now, 0 from n_live on
 *   free_out    [0 .. n_pages - n_live): the pages from n_live on, the lowest on top
 *   moves       I32 [n_moves][3] of qwfn_paged_copy: {source row, destination row,
 *               page_size}, room for (n_pages + 1) / 2 of them; n_moves I32 [1]
 * An n_free outside [0, free_cap], a stack entry outside the pool, one that is there twice
 * and lengths as in qwfn_paged_trim set bit 2 too. free_cap at least n_pages. */
size_t qwfn_paged_compact_workspace_size(int32_t n_pages);
int qwfn_paged_compact(const int32_t * n_kv, int32_t n_seq, int32_t page_size, const int32_t * table, int64_t table_stride,
                       int32_t max_pages, const int32_t * shared, int32_t n_pages, const int32_t * free_pages, int32_t free_cap,
                       const int32_t * n_free, int32_t * table_out, int32_t * shared_out, int32_t * free_out,
                       int32_t * n_free_out, int32_t * page_map, int32_t * moves, int32_t * n_moves, void * ws,
                       size_t ws_bytes, void * stream);

/* Rows copied inside each of n_caches tensors (the K and V of all layers, or the
 * recurrent states with a slot a row): for every move {s, d, n} of the list rows
 * s .. s + n - 1 go to d .. d + n - 1. caches: host array of tensors [ne0, n_rows] of one
 * type, shape and row stride, rows contiguous, none over another. moves: device I32
 * [cap][3]; n_moves: device I32 [1], how many of them count, or NULL for all cap. No
 * row that a move writes may be read or written by another. A move with n = 0 or s = d
 * is none; one with n outside [0, max_rows], rows outside the tensor or rows that go
 * over each other (0 < |s - d| < n) is left out and sets bit 0 of qwfn_device_status, as
 * does an n_moves outside [0, cap] (clipped). One launch for up to 64 tensors. */
int qwfn_paged_copy(const qwfn_tensor * caches, int32_t n_caches, const int32_t * moves, int32_t cap, const int32_t * n_moves,
                    int32_t max_rows, void * stream);

/* ------------------------------------------------ trees of drafted tokens
 *
 * A verify step over a tree: request b has T' = n_tree[b] <= T <= 64 drafted tokens
 * (nodes; n_tree NULL: T, or all where it has fewer), its newest T' tokens in the cache (extend them as usual).
 * A request that the extend does not serve has none there: give it 0 nodes, as n_tree = n_kv - n_past
 * does, or its last tokens count as nodes, which qwfn_paged_accept moves and drops.
 * Node t's parent precedes it; masks[b][t] (64-bit words, [n_seq][T]) has the bit of
 * every node that t sees, t itself among them. Per step: qwfn_tree_masks; per
 * attention layer qwfn_flash_attn_ext_q8_0_paged_tree, per recurrent layer
 * qwfn_linear_attn_tree (qwfn_state.h); then qwfn_paged_accept keeps one path,
 * qwfn_paged_trim (or _release) with its n_keep gives back the rest, and
 * qwfn_linear_attn over the rows of path (qwfn_get_rows_i32) with cu_path brings
 * the recurrent states forward. */

/* parents I32 [n_seq][T]: -1 for a child of the context's last token, else an earlier
 * node (another value counts as -1 and sets bit 2 of qwfn_device_status).
 *   masks  the node and its ancestors; 0 for t >= n_tree[b]
 *   pos    I32 [n_seq][T] or NULL: n_past[b] + the number of t's ancestors, for the
 *          rope; -1 for t >= n_tree[b]. n_past NULL: 0
 * An n_tree outside [0, T] is clipped and sets the bit. */
int qwfn_tree_masks(const int32_t * parents, const int32_t * n_tree, const int32_t * n_past, int32_t n_seq, int32_t T,
                    uint64_t * masks, int32_t * pos, void * stream);

/* qwfn_flash_attn_ext_q8_0_paged with queries that are nodes of a tree: q [D, T, n_head,
 * n_seq]; query t < n_tree[b] of request b sees the n_kv[b] - n_tree[b] tokens before the
 * tree and the nodes in masks[b][t] (any bits; those from n_tree[b] on count for
 * nothing), a query that sees nothing and queries from n_tree[b] on give 0. Arguments,
 * limits and arithmetic as there, but T <= 64 and T * n_head / n_head_kv <= 1024. An n_tree
 * outside [0, min(T, n_kv[b])] is clipped and sets bit 1 of qwfn_device_status. */
size_t qwfn_fattn_workspace_size_paged_tree(const qwfn_tensor * q, const qwfn_tensor * k, const qwfn_tensor * v,
                                            int32_t max_pages, int32_t page_size);
int qwfn_flash_attn_ext_q8_0_paged_tree(const qwfn_tensor * q, const qwfn_tensor * k, const qwfn_tensor * v,
                                        const int32_t * table, int64_t table_stride, int32_t max_pages, int32_t page_size,
                                        const int32_t * n_kv, const int32_t * n_tree, const uint64_t * masks, float scale,
                                        const qwfn_tensor * gate, const qwfn_tensor * dst, int variant, void * ws,
                                        size_t ws_bytes, void * stream);

/* The path from the context to node leaf[b] (-1: nothing is accepted), which is
 * masks[b][leaf[b]], m nodes t_0 < t_1 < ..: with B = n_kv[b] - n_tree[b] token B + t_i becomes
 * token B + i in every cache (as in qwfn_paged_copy: tensors [ne0, n_rows], at most 64).
 *   n_keep   I32 [n_seq]: B + m, for qwfn_paged_trim / _release
 *   cu_path  I32 [n_seq + 1] or NULL: the sums of m before each request
 *   path     I32 [n_seq * T] or NULL (NULL if cu_path is): b * T + t_i at cu_path[b] + i; 0
 *            behind cu_path[n_seq]
 * A leaf outside [-1, n_tree[b]) counts as -1, an n_tree outside [0, min(T, n_kv)] and an
 * n_kv outside [0, max_pages * page_size] are clipped, a row whose page lies outside the
 * caches is not moved; each sets bit 2 of qwfn_device_status. One launch. */
int qwfn_paged_accept(const qwfn_tensor * caches, int32_t n_caches, const int32_t * table, int64_t table_stride,
                      int32_t max_pages, int32_t page_size, const int32_t * n_kv, const int32_t * n_tree,
                      const uint64_t * masks, const int32_t * leaf, int32_t n_seq, int32_t T, int32_t * n_keep,
                      int32_t * cu_path, int32_t * path, void * stream);

#ifdef __cplusplus
}
#endif
#endif
