/* styx_serve.h -- batched decoding over a paged KV cache, C ABI.
 *
 * The operators a server needs beside the batched MoE block
 * (styx_moe_block_batch) to decode many sequences at once: K / V rows in
 * pages that sequences share one pool of, attention of one new token per
 * sequence over its pages, a bound on the cache by accumulated attention
 * weight, and sampling.  The reference decodes one sequence over a flat f32
 * cache and picks greedily (crates/model/src/moe.rs:1780-2140,
 * crates/model/examples/generate_moe.rs:29); the arithmetic of each row is
 * its own (RmsNorm per head, NEOX RoPE, softmax(scale q.K) V, q head h reads
 * kv head h / (n_heads / n_kv_heads)).
 *
 * Activations are f32; the cache is f32, f16 or bf16.  Lengths, page tables
 * and per-sequence settings are device memory, so a step can be recorded
 * once as a graph and replayed as they change.  Error codes, streams and
 * styx_last_error() as in styx_moe.h: what the host can see is refused with
 * STYX_EINVAL before anything is queued; a row, page or length that only the
 * device can see to be out of range is skipped and reported by
 * styx_check_device_error.
 */
#ifndef STYX_SERVE_H
#define STYX_SERVE_H

#include <stdint.h>

#include "styx_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of a paged cache (ggml type ids; f32 is STYX_F32 = 0) */
#define STYX_F16 1
#define STYX_BF16 30

/* Row r of sequence b lies in page table[b * table_stride + r / page_size]
 * of the two pools; in it kv head j's row is at element
 *   page * page_stride + (j * page_size + r % page_size) * head_dim
 * (a page holds one head's rows together).  Page ids are < n_pages; entries
 * past a sequence's rows are not read.  A sequence with lens[b] = 0 is an
 * empty slot.  Layers may share a pool and its tables with other k / v.  table
 * and lens may change between calls (of one stream, or ordered by an event), not
 * while one runs. */
typedef struct styx_paged_kv {
    void *k, *v;               /* pools, 16-byte aligned */
    int64_t page_stride;       /* elements from page to page, rows 16-byte aligned */
    const int32_t *table;      /* device [n_seqs][table_stride] */
    const int32_t *lens;       /* device [n_seqs]: rows in use */
    int32_t dtype;             /* STYX_F32, STYX_F16 or STYX_BF16 */
    int32_t n_pages;
    int32_t page_size;         /* rows, a power of two, <= 4096 */
    int32_t n_kv_heads;
    int32_t head_dim;          /* <= 256, a multiple of 8 (f32: of 4) */
    int32_t n_seqs;
    int32_t max_pages;         /* table entries of a sequence in use at most */
    int32_t table_stride;      /* >= max_pages */
} styx_paged_kv;

/* For token t < n_tokens of sequence seq[t] (NULL: t), at rotary position
 * pos[t], into the sequence's row row[t] (NULL: lens - 1, the newest row of
 * the length that the step's attention reads):
 *   q_out[t][h]   = RoPE(RMSNorm(q[t][h]) * q_norm)      f32 [n_heads][head_dim]
 *   K row (j)     = RoPE(RMSNorm(k[t][j]) * k_norm)      rounded to the cache's type
 *   V row (j)     = v[t][j]                              rounded to the cache's type
 * q / k / v rows are q_stride / k_stride / v_stride floats apart (slices of
 * one projection's output, for instance); a NULL norm is left out; NEOX
 * pairs (i, i + head_dim / 2), theta = pos * freq_base^(-2i/head_dim).  A
 * token whose row is negative (a slot of length 0 among them) writes no row
 * and a zero q_out; a row past max_pages * page_size or a page outside the
 * pool is skipped and reported.  n_heads may be 0 (no q); q_out, 16-byte
 * aligned, may not overlap q, k or v (nor what lies between their tokens).
 * Two tokens with one (sequence, row) leave either's row. */
int styx_paged_append(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, int n_tokens, int n_heads,
                      const float *q, int64_t q_stride, const float *k, int64_t k_stride, const float *v,
                      int64_t v_stride, const float *q_norm, const float *k_norm, float eps, float freq_base,
                      const int32_t *pos, const int32_t *seq, const int32_t *row, float *q_out);

/* out[b][h] = sum_r p[r] V[r], p = softmax over the rows r of sequence b
 * with lens[b] - window <= r < lens[b] (window 0: all rows) of
 * scale * q[b][h] . K[r]; zeros where a sequence has no rows.  q and out f32
 * [n_seqs][n_heads][head_dim], 16-byte aligned; n_heads a multiple of
 * n_kv_heads.  Rows outside the window or past the length are never used,
 * whatever they hold.
 * A NaN in a head's q or in a row of K that is seen, or a score of +inf, makes
 * the head's output (and its lse and weights) NaN.
 *   lse (may be NULL): f32 [n_seqs][n_heads], log sum_r e^(scale q.K[r]),
 *     -inf where there are no rows.
 *   acc_out (may be NULL): f32 [n_seqs][n_kv_heads][acc_stride], the
 *     accumulated attention weight of every row r < lens[b]:
 *       acc_out[r] = (r == lens[b] - 1 ? 0 : acc[r]) + sum of p[r] over the
 *     kv head's q heads (acc of the newest row is not read, so a row enters
 *     with nothing to be cleared first).  acc_out may be acc, and out may be
 *     q; no other overlap of these.
 * The workspace (styx_paged_attend_workspace_bytes, 256-byte aligned) holds
 * the splits' partial sums and their counters, and with acc a score of 4 bytes
 * for every q head of every row that the table has room for (n_seqs x n_heads x
 * max_pages x page_size): initialise it once.  Calls
 * that share one must not run at the same time. */
int styx_paged_attend_workspace_bytes(styx_ctx *ctx, const styx_paged_kv *kv, int n_heads, int with_acc,
                                      uint64_t *out);
int styx_paged_attend_workspace_init(styx_ctx *ctx, styx_stream stream, void *workspace, uint64_t workspace_bytes);
int styx_paged_attend(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, int n_heads, const float *q,
                      float scale, int window, float *out, float *lse, const float *acc, float *acc_out,
                      int64_t acc_stride, void *workspace, uint64_t workspace_bytes);

/* Brings every sequence down to at most `budget` rows, per kv head.  Of the
 * n = lens[b] rows those stay that come first by
 *   protected rows: pos[r] >= next_pos[b] - n_recent or pos[r] < n_sink,
 *   then the larger accumulated weight acc[r] (NaN counts as the lowest),
 *   then the lower r.
 * A row that stays but lies at or beyond the budget moves into the place of
 * one below it that leaves (the i-th such row into the i-th such place): its
 * K and V rows in the pools, its weight and position.  acc and pos are
 * [n_seqs][n_kv_heads][stride] (f32, int32) with pos[r] the position of the
 * token in row r, next_pos[n_seqs] the position the next token will have.
 * acc_out, pos_out (same shape, the first min(n, budget) of each line
 * written) and lens_out[b] = min(n, budget) are new arrays: the inputs,
 * kv->lens among them, are left as they are, so the call may be repeated.
 * n_recent + n_sink <= budget.  After it the pages past
 * lens_out can go back to the pool. */
int styx_paged_evict_workspace_bytes(const styx_paged_kv *kv, int budget, uint64_t *out);
int styx_paged_evict(styx_ctx *ctx, styx_stream stream, const styx_paged_kv *kv, const float *acc,
                     const int32_t *pos, const int32_t *next_pos, int64_t stride, int budget, int n_recent,
                     int n_sink, float *acc_out, int32_t *pos_out, int32_t *lens_out, void *workspace,
                     uint64_t workspace_bytes);

/* One token for each of n_rows rows of logits (f32, row_stride floats
 * apart), from given uniform numbers u in [0, 1).  With m the row's maximum
 *   w[i] = exp((x[i] - m) * (1 / temperature))        in f32,
 *   W[i] = floor(w[i] * 2^40)                           whole numbers, so that
 * every sum below is exact and the same in any order;
 *   top_k: the k first tokens by (larger x, lower index); 0 or less: all;
 *   top_p: of those, in that order, the fewest whose W reach
 *          rint(p * 2^24) / 2^24 of their sum (one at least);
 *   min_p: of those, w[i] >= min_p (above 1, or NaN: as 1, the maximum and its
 *          equals stay);
 *   token: the first kept i with sum of kept W up to and with i >
 *          floor(floor(u 2^24) S / 2^24), S the sum of all kept;
 *   logprob = (x - m) / temperature - log(S / 2^40).
 * temperature <= 0 (or NaN) takes the maximum (lowest index among equals;
 * logprob 0).
 * NaN logits count as -inf.  A row with nothing to draw from (all -inf)
 * gives token -1 and logprob -inf.  temperature, top_k, top_p, min_p: device
 * arrays of n_rows, each NULL for 1, all, 1 and 0; logprob may be NULL.
 * n_vocab <= 2^22.  token and logprob may not overlap the inputs or each
 * other; either may be u. */
int styx_sample(styx_ctx *ctx, styx_stream stream, const float *logits, int64_t row_stride, int n_rows, int n_vocab,
                const float *u, const float *temperature, const int32_t *top_k, const float *top_p,
                const float *min_p, int32_t *token, float *logprob);

#ifdef __cplusplus
}
#endif
#endif
