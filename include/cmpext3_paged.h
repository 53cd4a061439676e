/*
 * cmpext3_paged.h -- C ABI of the paged key-value cache on MI355X (gfx950):
 * appending new tokens' keys and values to the pages of their sequences (with
 * the rotary position embedding applied on the way), attention of new tokens
 * over those pages, and the choice of the pages worth attending to.
 *
 * A cache is a pool of pages, k_pages and v_pages [num_pages, H_kv, page_size,
 * D], and for each of B sequences a row of page numbers:
 *
 *   page_table [B, table_width] int32, row stride table_stride (elements):
 *       token j of sequence b lies in page page_table[b, j / page_size], slot
 *       j % page_size.
 *   seq_lens   [B] int32: the tokens each sequence holds, the call's new ones
 *       among them.  0 (or less): no sequence in this place of the batch.
 *   new_lens   [B] int32, or null: how many of the call's S columns hold new
 *       tokens; column i < n = min(new_lens[b], S, seq_lens[b]) is token
 *       seq_lens[b] - n + i, the columns after them are padding.  Null: S.
 *
 * Strides are in ELEMENTS over the first three dims of a tensor; the last is
 * contiguous.  Head dims are whole 16-byte chunks up to 256 elements (a
 * multiple of 8 for f16 / bf16, of 4 for f32, else CMPEXT3_E_HEAD_DIM), and every
 * base pointer and stride of a dim with more than one index is a multiple of
 * 16 bytes (else CMPEXT3_E_ALIGN).  Any page size runs; the attention reads pages in
 * tiles of 16 slots, so a multiple of 16 wastes nothing.
 *
 * Lengths and page numbers live on the device and are checked there: a page
 * number outside [0, num_pages), or a sequence longer than its table row, is
 * never followed.  What such a token would have written is left out, and the
 * rows of output that depend on it are NaN.
 *
 * All calls launch on `stream`, allocate nothing, wait for nothing on the
 * host, and return CMPEXT3_OK or a code of cmpext3_attn.h (nothing launched,
 * except for CMPEXT3_E_LAUNCH).  They are serving forms; none has a gradient.
 *
 * Reference: none (WifiLast/torch-cmp-patch has no key-value cache; its
 * attention takes one contiguous tensor per call, src/main.cpp:1603-1774).
 */
#ifndef CMPEXT3_PAGED_H
#define CMPEXT3_PAGED_H

#include "cmpext3_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Append: k, v [B, H_kv, S, D] into the pages, and the queries of the same
 * tokens (q [B, H, S, D], or null) rotated into q_out.
 *
 *   cos, sin : [table_rows, rot / 2] f32, row stride rot_stride (elements), or
 *              null (no rotation; q must then be null).  Keys and queries are
 *              rotated in their first `rot` dims by the angles of row
 *              positions[b, i] ([B, S] int32, contiguous) or, with positions
 *              null, of the token's own place in its sequence: the pairs are
 *              (d, d + rot / 2), or (2 d, 2 d + 1) when `interleaved`;
 *              (x, y) -> (x cos - y sin, y cos + x sin) in f32, rounded once.
 *   key_bounds : [num_pages, H_kv, 2, D], or null: the lowest and the highest value of
 *              each channel over a page's keys, as stored (kb_str over the
 *              first three dims).  A token in slot 0 begins its page's bounds
 *              anew, later ones widen them; NaN keys leave them as they are.
 *
 * Only the slots of the new tokens are written (and their pages' bounds); the
 * padding columns of q_out are zero, and a row of q_out whose token has no
 * valid page or no row in the tables is NaN (that token is not stored).
 * Tokens of one call must go to different slots, and with key_bounds different
 * sequences' to different pages.  q_out is memory of
 * its own.
 */
int cmpext3_paged_append(const void* k, const void* v, const void* q, void* q_out,
                         void* k_pages, void* v_pages, void* key_bounds,
                         int dtype, int B, int H, int H_kv, int S, int D, int num_pages, int page_size,
                         const int64_t k_str[3], const int64_t v_str[3],
                         const int64_t q_str[3], const int64_t qo_str[3],
                         const int64_t kp_str[3], const int64_t vp_str[3], const int64_t kb_str[3],
                         const int32_t* page_table, int table_width, int64_t table_stride,
                         const int32_t* seq_lens, const int32_t* new_lens, const int32_t* positions,
                         const float* cos, const float* sin, int table_rows, int rot, int64_t rot_stride,
                         int interleaved, hipStream_t stream);

/*
 * Attention of the new tokens, o = softmax(scale * q K^T) V over the pages of
 * their sequences: q, o [B, H, S, D] with S <= 16 (a decode step, or a short
 * block of tokens), query head h on K/V head h / (H / H_kv).  Column i sees its
 * own token and the tokens before it; a padding column, and every column of a
 * place without a sequence, gives zeros.  The slots behind a sequence's last
 * token are not read.
 *
 *   selected : [B, H_kv, n_selected] int32, contiguous, or null (all pages):
 *              the sequence's pages (as columns of its table row) that each
 *              K/V head attends to, in any order, none twice; negative
 *              entries are left out.  An entry that is no page of the sequence
 *              makes the head's rows NaN.
 *   workspace, workspace_bytes : as in cmpext3_attn_fwd_ws (16-byte aligned,
 *              its first CMPEXT3_WORKSPACE_COUNTER_BYTES zero before its first
 *              use and left zero by every launch); with less than
 *              cmpext3_paged_attn_workspace_size bytes, or null, no sequence
 *              is split over workgroups.  The two give equal results within
 *              rounding; each is bit-identical from one call to the next.
 */
int cmpext3_paged_attn(const void* q, const void* k_pages, const void* v_pages, void* o,
                       int dtype, int B, int H, int H_kv, int S, int D, int num_pages, int page_size,
                       const int64_t q_str[3], const int64_t kp_str[3], const int64_t vp_str[3],
                       const int64_t o_str[3],
                       const int32_t* page_table, int table_width, int64_t table_stride,
                       const int32_t* seq_lens, const int32_t* new_lens,
                       const int32_t* selected, int n_selected, float scale,
                       void* workspace, size_t workspace_bytes, hipStream_t stream);

/*
 * Workspace bytes with which cmpext3_paged_attn splits sequences over
 * workgroups (0 for invalid arguments or nothing to do).  Host-only.
 */
size_t cmpext3_paged_attn_workspace_size(int dtype, int B, int H, int H_kv, int S, int D, int page_size,
                                         int table_width, int n_selected);

/*
 * Page choice for one new token of each sequence (q [B, H, 1, D]): the score of
 * a page for K/V head k is the sum over its query heads h and the channels d of
 * max(q_hd lo_d, q_hd hi_d), lo and hi the page's key_bounds: no key of the
 * page has a larger sum of products with the head group's queries.  It is summed in 64 bits as Q+_d hi_d
 * + Q-_d lo_d with the sums Q+, Q- of the queries' positive and negative values;
 * a part that is 0 adds nothing, whatever its bound.  selected [B, H_kv, n_selected] int32 (contiguous) receives, in ascending order, the sequence's
 * last page and its n_selected - 1 best others (equal scores: the lower page;
 * a NaN score, and a page outside the pool, counts as the highest), or all of
 * its pages followed by -1.
 *
 *   workspace : 16-byte aligned, at least cmpext3_paged_select_workspace_size
 *               bytes (else CMPEXT3_E_INVALID); its contents do not matter and
 *               are overwritten (so it is not the attention's, whose counters
 *               have to stay zero).  Calls that run one after another may share
 *               it, from any thread.
 */
int cmpext3_paged_select(const void* q, const void* key_bounds, int32_t* selected,
                         int dtype, int B, int H, int H_kv, int D, int num_pages, int page_size,
                         const int64_t q_str[3], const int64_t kb_str[3],
                         const int32_t* page_table, int table_width, int64_t table_stride,
                         const int32_t* seq_lens, int n_selected,
                         void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Workspace bytes of cmpext3_paged_select (0 for invalid arguments).  Host-only. */
size_t cmpext3_paged_select_workspace_size(int B, int H_kv, int table_width);

#ifdef __cplusplus
}
#endif

#endif /* CMPEXT3_PAGED_H */
