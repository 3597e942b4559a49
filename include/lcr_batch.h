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
 *   lcr_batch_logprobs             what an answer says beside its tokens: their log
 *                                  probabilities, entropies, likeliest ids
 *
 * and, over a cache of 8-bit numbers with a scale for every 16 positions of a
 * head (lcr_kv8_view), in place of the second and third:
 *
 *   lcr_batch_norm_rope_write_kv8
 *   lcr_batch_attention_kv8
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

/* Alternatives of a row, at most. */
#define LCR_BATCH_MAX_ALTERNATIVES 32

/* Log probabilities of given tokens, with their rows' entropies and likeliest ids.
 * Of row t of the logits (rows are logits_stride floats apart), p = softmax(logits):
 *   logprobs[t]      log p of token_ids[t]; -inf for an id past the vocabulary
 *   ranks[t]         how many ids have a larger logit than it (0: the likeliest;
 *                    vocab for an id past the vocabulary)
 *   entropies[t]     -sum p log p, in nats
 *   top_ids[t][top], top_logprobs[t][top]
 *                    the ids of the largest logits in descending order, equal ones
 *                    by ascending id, and their log p; top is at most
 *                    LCR_BATCH_MAX_ALTERNATIVES. Logits of -inf are no alternatives:
 *                    where fewer than top others are left, -1 and -inf behind them.
 * A row whose token id is negative is left out: nothing of it is read or written.
 * token_ids NULL: no tokens are given, logprobs and ranks are not written, and no
 * row is left out. logprobs, ranks and entropies may each be NULL for what is not
 * wanted, and with top 0 the last two.
 * Weights are fp32, summed in fp32 sixteen at a time and in fp64 beyond that; the
 * logarithm is fp64.
 * A NaN logit counts as -inf, whose p is 0. Where a row's largest logit is not
 * finite, p is 1 at the lowest index of that value, as for lcr_batch_verify.
 * With a workspace of lcr_batch_logprobs_workspace_bytes (16-byte aligned) few rows
 * are split over the device, in two launches; without one (NULL, 0, or a smaller
 * one) a row is read by one compute unit. The same call gives the same bits. */
int lcr_batch_logprobs(float* logprobs, int32_t* ranks, float* entropies, int32_t* top_ids, float* top_logprobs,
                       const float* logits, const int32_t* token_ids, int rows, int top, int vocab,
                       int logits_stride, void* workspace, size_t workspace_bytes, void* stream);

size_t lcr_batch_logprobs_workspace_bytes(int rows, int top, int vocab);

/* ---- a cache of 8-bit numbers -------------------------------------------- */

/* Positions of a block: those of a head that share a scale. */
#define LCR_KV8_BLOCK 16

/* One layer of a paged cache of e4m3 numbers (four bits of exponent, three of
 * mantissa, no infinities). Positions lie in blocks of 16, a block in a page
 * (page_size is a multiple of 16), and block n of a page's head is
 *   16 head_dim bytes from page * page_stride + head * head_stride + n * 16 head_dim on,
 *   a scale at     page * scale_page_stride + head * scale_head_stride + n
 * in keys and key_scales, values and value_scales. In a block, dim i of position t
 * (of 16) is byte
 *   t head_dim + i                          of its keys,
 *   (t / 4) 4 head_dim + 4 i + t % 4        of its values: four positions side by
 *                                           side, as matrix instructions take them.
 * It stands for its number times the block's scale, a power of two. That is a value
 * of the library's element type itself, so that the cache is a 16-bit one whose
 * values were rounded. head_dim is a multiple of 16, at most 256. Strides are in
 * bytes and in floats, and multiples of 16 bytes for the numbers, which begin on 16
 * bytes. page_table as in lcr_kv_view. */
typedef struct lcr_kv8_view {
  void* keys;
  void* values;
  float* key_scales;
  float* value_scales;
  const int32_t* page_table;
  int page_size;
  int page_stride;
  int head_stride;
  int scale_page_stride;
  int scale_head_stride;
  int num_kv_heads;
  int head_dim;
} lcr_kv8_view;

/* lcr_batch_norm_rope_write_kv with keys and values appended to an 8-bit cache.
 * A row's slot, as lcr_batch_map gives it, is its position's place in the pool.
 * A block's scale is the least power of two with which its largest number is at
 * most 448, and at least 2^-117 (fp16: 2^-15). Writing to a block's position 0
 * begins the block: its scale is that of the positions written in this call, and what
 * it held counts for nothing. Writing to others keeps the block's scale if it
 * suffices; otherwise the numbers that it holds are rounded to the larger one, in
 * place. However often that happens, a number is off by less than one step of the
 * last scale's grid at its size. Scales do not fall before a block is begun again
 * (also not when drafts that raised them are rejected).
 * Keys are normed and rotated in fp64 and rounded to fp32, where scales are
 * decided, so that one at the edge of a power of two does not hang on the order
 * of sums; queries as for the 16-bit cache. An infinity or a NaN is held as NaN and
 * does not count for the scale; finite values past the largest product that the
 * element type holds (61440 in fp16, 1.875 * 2^127 in bf16) are held as that.
 * All rows of a call whose slots lie in one block have to be among 16 rows that
 * follow each other, as those of a sequence are; slots differ from row to row. Of
 * blocks for which that is not so, nothing is said but that nothing out of bounds
 * is touched. A call takes up to 2^26 - 4 heads, of queries, keys and values of all
 * rows together. */
int lcr_batch_norm_rope_write_kv8(void* q_out, const lcr_kv8_view* view, const void* q, const void* k,
                                  const void* v, const void* q_norm, const void* k_norm, float eps,
                                  const float* rope_table, int table_positions, const int32_t* positions,
                                  const int32_t* slots, int tokens, int num_heads, int pool_pages,
                                  int src_row_stride, void* stream);

/* lcr_batch_attention over an 8-bit cache: of the values that the cache stands for,
 * the same results, to the rounding of sums, with the same arguments, limits and
 * workspace rules (head_dim a multiple of 16 up to 256; 64 and 128 run on the matrix
 * cores). There too the weights exp(s - max) are rounded to the element type on the
 * matrix cores, for the value product and for their sum alike: by half a step each,
 * and in fp16 by 2^-32 of the row's largest where that is more. Statistics and sums are
 * fp32. Pages may be of any size that a table holds, also past 2^32 bytes. Positions that no row of a sequence sees may hold anything, scales
 * included, and numbers that a row does not see leave it as it is; a NaN that it sees
 * makes its element NaN, also where the weight rounds to 0. */
int lcr_batch_attention_kv8(void* out, const void* q, const lcr_kv8_view* view, const int32_t* row_starts,
                            const int32_t* lengths, int batch, int tokens, int max_new, int num_heads,
                            int heads_per_kv, int table_stride, int pool_pages, int q_row_stride, float scale,
                            void* workspace, size_t workspace_bytes, void* stream);

size_t lcr_batch_attention_kv8_workspace_bytes(int batch, int tokens, int max_new, int num_heads,
                                               int heads_per_kv, int head_dim);

#ifdef __cplusplus
}
#endif

#endif /* LCR_BATCH_H_ */
