/*
 * lcr_batch.h — C-ABI kernel layer for serving several requests at once over
 * one paged KV cache.
 *
 * The launchers of lcr_kernels.h serve one sequence: its positions follow each
 * other, its page table is filled by the host, its logits give one token. These
 * run a step of many sequences, each with tokens of its own (one token, drafted
 * tokens to verify, a chunk of a prompt), with every length on the device, so
 * that a captured step replays for other lengths:
 *
 *   lcr_batch_map                  the sequences' lengths -> page tables, row
 *                                  starts, and each row's position and slot
 *   lcr_batch_norm_rope_write_kv   norm of each query and key head, rotation,
 *                                  keys and values into their slots
 *   lcr_batch_attention            each sequence's rows over its pages
 *   lcr_batch_verify               drafted tokens against the target's logits
 *
 * No counterpart in the reference, which serves one sequence.
 *
 * The rows of a step are the sequences' new tokens one after another: sequence
 * b has rows row_starts[b] .. row_starts[b + 1] - 1. The buffers may hold more
 * rows behind the last sequence's; those have slot and position -1 and are
 * neither read nor written (lcr_batch_verify may read their target_logits, to no
 * effect). A sequence may have no rows. A call of some of a step's sequences takes
 * its row starts from the first of them on; rows before that stay as they were,
 * as those behind the last.
 *
 * Conventions (element pointers, streams, status, error text) are those of
 * lcr_kernels.h. Nothing here allocates or waits; arrays named on the device
 * are read when the kernels run, in stream order. A workspace holds nothing
 * between calls and may hold anything before one; two calls that can run at
 * the same time (other streams, other replays) need one each. Outputs may not
 * overlap inputs or the workspace.
 *
 * What the device finds wrong in its arrays (a page outside the pool, a token
 * outside the vocabulary) cannot fail the call; each entry says what then
 * comes out. No such value makes a kernel read or write out of bounds. Of row
 * starts that do not ascend, as lcr_batch_map's do, nothing is said but that:
 * the outputs may hold anything, or what they held.
 */
#ifndef LCR_BATCH_H_
#define LCR_BATCH_H_

#include <stddef.h>
#include <stdint.h>

#include "lcr_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Sequences of one call. */
#define LCR_BATCH_MAX_SEQUENCES 4096

/* The page tables and rows of a step, from the sequences' lengths.
 *
 * Sequence b has lengths[b] positions in the cache, gets new_tokens[b] more,
 * and has mapped[b] pages in its table page_tables[b * table_stride ...] (pages
 * of page_size positions; more than its length needs are kept, as a sequence
 * has whose drafts were rejected). The pages it lacks are taken from the end of
 * free_pages[0 .. free_count[0] - 1] (free_count is clamped to free_capacity),
 * in sequence order.
 *
 * Sequences are placed in order up to the first that cannot be: pages lacking,
 * more than max_rows rows in all, more positions than table_stride pages hold,
 * or a negative entry in lengths, new_tokens or mapped. That sequence and all
 * behind it get no rows and no pages, for the caller to try again.
 *
 * A batch of 0 is a step without rows: row_starts[0], positions, slots and counts
 * are written as for any other, the sequences' arrays are not looked at and may
 * be NULL. (Nothing is done where one of those outputs or free_count is NULL.)
 *
 * Out: row_starts[batch + 1]; positions[max_rows] and slots[max_rows], with
 * slot = page * page_size + position % page_size, both -1 behind the last row
 * (slots also where the page is outside 0 .. pool_pages - 1); lengths_out and
 * mapped_out[batch], both counted with the new tokens (unchanged for a
 * sequence that was not placed); counts[0] sequences placed, counts[1] pages
 * left in free_pages; page_tables gets the new pages.
 * The outputs feed the next call in exchange for its inputs: lengths_out (or
 * lengths + what lcr_batch_verify kept), mapped_out, counts + 1. */
int lcr_batch_map(int32_t* row_starts, int32_t* positions, int32_t* slots, int32_t* lengths_out,
                  int32_t* mapped_out, int32_t* counts, int32_t* page_tables, const int32_t* lengths,
                  const int32_t* new_tokens, const int32_t* mapped, const int32_t* free_pages,
                  const int32_t* free_count, int batch, int max_rows, int table_stride, int page_size,
                  int pool_pages, int free_capacity, void* stream);

/* For each row t with a slot: RMSNorm over each query and key head, half-split
 * RoPE at positions[t], the query into q_out[t][num_heads][head_dim], key and
 * value into the cache at slots[t].
 *   y = x * (1 / sqrt(mean(x^2) + eps)) * weight   (y = x where the weight is NULL)
 *   out[i] = y[i] cos - y[i + d/2] sin, out[i + d/2] = y[i + d/2] cos + y[i] sin
 * in fp32 throughout, rounded once. q, k and v point at row 0's first head;
 * rows are src_row_stride elements apart (parts of one fused projection).
 * q_norm and k_norm: [head_dim] element weights, or NULL. rope_table as
 * lcr_rope_table writes it, for positions 0 .. table_positions - 1.
 * Of the view, page_table is not used. head_dim is even, at most 512.
 * A row whose slot is outside the pool's pool_pages pages or whose position is
 * outside the table is left alone, its query too. Slots differ from row to
 * row. */
int lcr_batch_norm_rope_write_kv(void* q_out, const lcr_kv_view* view, const void* q, const void* k,
                                 const void* v, const void* q_norm, const void* k_norm, float eps,
                                 const float* rope_table, int table_positions, const int32_t* positions,
                                 const int32_t* slots, int tokens, int num_heads, int pool_pages,
                                 int src_row_stride, void* stream);

/* Causal GQA attention of each sequence's rows over its pages.
 * Row i of sequence b's n rows is at position lengths[b] - n + i (lengths
 * counts the new tokens, whose keys and values are in the cache) and sees
 * positions 0 .. its own:  out = softmax(scale q . k) v, statistics and sums in
 * fp32. On the matrix cores the weights exp(s - max) are rounded to the element
 * type, for the value product and for their sum alike: by half a step each, and
 * in fp16 by 2^-32 of the row's largest where that is more.
 *   q:   [tokens] rows q_row_stride elements apart, [num_heads][head_dim] each
 *   out: [tokens][num_heads][head_dim]
 * view->page_table: [batch][table_stride]. max_new: no sequence has more rows
 * than that (its further rows come out as zeros). head_dim is at most 256;
 * 64 and 128 with 16-byte aligned rows run on the matrix cores, and
 * fastest with a page_size that is a multiple of 16. Tables hold up to 2^30
 * positions.
 * Infinities and NaN in places that a row does not see leave it as it is; of a
 * value that it sees, its element becomes infinite or NaN, also where the weight
 * rounds to 0. Scores, scale q . k, may be up to 2^26 in size (beyond that a row
 * may come out as NaN).
 * A row that sees no position (lengths[b] < n) is zeros. Positions behind
 * table_stride pages do not exist. A sequence with a page outside 0 ..
 * pool_pages - 1 among those it reads may come out as NaN.
 * With a workspace of lcr_batch_attention_workspace_bytes (16-byte aligned)
 * tables of more than 768 to 1024 positions have their keys split over the device;
 * without one (NULL, 0, or a smaller one) nothing is split, which is one launch
 * less for sequences known to be short. Where a sequence is
 * split depends on the lengths of all, and the rounding of its sums with it; the
 * same call gives the same bits. */
int lcr_batch_attention(void* out, const void* q, const lcr_kv_view* view, const int32_t* row_starts,
                        const int32_t* lengths, int batch, int tokens, int max_new, int num_heads,
                        int heads_per_kv, int table_stride, int pool_pages, int q_row_stride, float scale,
                        void* workspace, size_t workspace_bytes, void* stream);

size_t lcr_batch_attention_workspace_bytes(int batch, int tokens, int max_new, int num_heads,
                                           int heads_per_kv, int head_dim);

/* Drafted tokens against the target's distribution.
 * Sequence b has n rows of target_logits: behind its last token and behind each
 * of n - 1 drafted tokens; draft_ids[row] is the token drafted behind that row,
 * draft_logits[row] what it was drawn from (NULL: drafted without a
 * distribution, so q below is 1 at the drafted token). Of a sequence's last
 * row neither is read. Rows are logits_stride floats apart, at most 65535. At most
 * max_draft drafts are taken (itself at most 2^30).
 *   temperature T = temperatures[b] > 0: p = softmax(target / T), q =
 *     softmax(draft / T); the draft x of row i is kept iff
 *     accept_uniforms[row] * q(x) < p(x). Behind the first one not kept comes a
 *     token drawn from max(p - q, 0), behind n - 1 kept ones a token drawn from
 *     the last row's p: the first index whose running sum exceeds
 *     sample_uniforms[b] times the whole sum. (From p where max(p - q, 0) is 0
 *     everywhere.) Sums are in fp64, exponentials to 2e-13 of their value: whole
 *     draws hang on intervals of the running sum narrower than fp32 resolves. A
 *     probability of less than 2^-1020 of its row's largest is 0.
 *     Logits that top-k, top-p or a grammar leave out are -inf in the rows given.
 *   T <= 0 or NaN: p is 1 at the largest logit (ties to the lowest index), a
 *     draft is kept iff it is that index.
 * A NaN logit counts as -inf. Where a row's largest logit is not finite, its p
 * is 1 at the lowest index of that value, its q 1 at the drafted token. A draft
 * outside the vocabulary is not kept.
 * out_ids[batch][max_draft + 1]: the kept drafts, the drawn token, then -1;
 * out_counts[batch]: how many (0 for a sequence without rows).
 * The workspace (lcr_batch_verify_workspace_bytes, 16-byte aligned) is needed. */
int lcr_batch_verify(int32_t* out_ids, int32_t* out_counts, const float* target_logits,
                     const float* draft_logits, const int32_t* draft_ids, const int32_t* row_starts,
                     const float* temperatures, const float* accept_uniforms, const float* sample_uniforms,
                     int batch, int rows, int max_draft, int vocab, int logits_stride, void* workspace,
                     size_t workspace_bytes, void* stream);

size_t lcr_batch_verify_workspace_bytes(int batch, int rows, int vocab);

#ifdef __cplusplus
}
#endif

#endif /* LCR_BATCH_H_ */
