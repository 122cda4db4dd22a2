/*
 * nsparse_lm.h -- sparse products whose pattern a language model chooses row by row (C ABI).
 *
 * libnsparse.{d,s} multiplies matrices whose pattern is given.  In a language model the pattern is chosen
 * while the model runs, and the products are in 16 or 32 bits:
 *   - attention over blocks of keys: a cheap score selects `width` blocks for every query (the symbolic phase: a
 *     row of block indexes), attention runs over the listed blocks only (the numeric phase: a sampled product, a
 *     softmax, a product), and its gradient runs over the pattern and its transpose;
 *   - tokens sorted by expert: a router lists `top` experts a token; the tokens are brought together expert by
 *     expert (product with the pattern's transpose) and back with weights (product with the pattern).
 *
 * libnsparse_lm.so is one library for all types: they are arguments.  It depends on the HIP runtime only.
 *
 * Rules of every entry point
 *   - Pointers are device pointers on the current device; a NULL of a required one is refused.
 *   - Work is queued on `stream` (a hipStream_t, NULL: the null stream) and the call returns at once: no
 *     synchronisation, no allocation, no memset node.  It may be captured into a graph.
 *   - Nothing is kept between calls.  Scratch memory is the caller's (`workspace`, of the size the query function
 *     names); two calls that may run at the same time need two workspaces.
 *   - Returns 0; a negative NSPARSE_LM_E* code for refused arguments, nothing queued; or a positive hipError_t.
 *     nsparse_lm_last_error_string() is the calling thread's last message.
 *   - Results do not depend on timing: no floating-point atomics.
 *   - Sums, softmax statistics and gradients are accumulated in 32 bits (the block means and the scores near a
 *     selection's border in 64) and rounded once; the probabilities and their gradients are rounded to the
 *     inputs' type on the way into the second product, which adds an error of about the outputs' own rounding.
 */
#ifndef NSPARSE_AMD_NSPARSE_LM_H
#define NSPARSE_AMD_NSPARSE_LM_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { NSPARSE_LM_F32 = 0, NSPARSE_LM_F16 = 1, NSPARSE_LM_BF16 = 2 };

enum {
    NSPARSE_LM_EARG = -1,      /* a NULL pointer, a size out of range, sizes that contradict each other */
    NSPARSE_LM_ETYPE = -2,     /* unknown type */
    NSPARSE_LM_EALIGN = -3,    /* a base pointer or stride that is not a multiple of 16 bytes */
    NSPARSE_LM_EWORKSPACE = -4 /* workspace missing or too small */
};

int nsparse_lm_last_error(void);
const char *nsparse_lm_last_error_string(void);
/* "gfx950 <hash of csrc/lm and this header>" */
const char *nsparse_lm_build_info(void);

/* ---- attention over selected blocks --------------------------------------------------------------------------
 * q      [q_rows, heads, head_dim]            query row t, head h at q + t * q_stride[0] + h * q_stride[1]
 * k, v   [k_rows, kv_heads, head_dim]         key row r, head g at k + r * k_stride[1] + g * k_stride[2]
 *        or, with page_size > 0, a paged cache [k_rows pages, page_size, kv_heads, head_dim]; page n begins at
 *        k + n * k_stride[0].
 * Strides are in elements, the head dimension is contiguous; bases and strides are multiples of 16 bytes.
 * heads is a multiple of kv_heads; query head h reads key head h / (heads / kv_heads).
 *
 * Sequences.  cu_q / cu_k: int[n_seq + 1], sequence s has the rows [cu[s], cu[s+1]).  Without them every sequence has
 * q_rows / n_seq query rows and k_rows / n_seq key rows (both divide).  q_len / k_len: int[n_seq], optional:
 * only that many of a sequence's rows count (a padded batch).  Paged: k_len and page_table are required, key j of sequence s is
 * row j % page_size of page page_table[s * table_stride + j / page_size].  Query i of a sequence has position
 * len_k - len_q + i; with causal != 0 it attends to keys j <= position, else to all len_k keys.
 * Output rows of queries that no sequence has (behind cu_q[n_seq], or i >= q_len) are left as they were.
 * cu_q and cu_k ascend.  Numbers in these arrays are clamped to the buffers' sizes; where they contradict each other the
 * results mean nothing, but nothing outside the buffers is read or written.  A page outside [0, k_rows) hides its keys.
 *
 * Pattern.  idx int[q_rows, kv_heads, width]: the blocks (of `block` keys, numbered inside the sequence) that the query's
 * heads of group g attend to.  An entry counts only if it is not negative, lies inside the sequence and is greater
 * than every entry before it in its row; others are skipped (so -1 ends a row, and a block listed twice counts once).
 * A query with no key left gets out = 0 and lse = -inf, and gradients 0.  Whatever stands in keys and values that a query does not see
 * (NaN included) does not reach its outputs; a query whose own q or dout is no number spoils dk and dv of the blocks that it lists.
 *
 * Block means.  One row [kv_heads, head_dim] a block, in the keys' type, contiguous.  The row of block b of sequence s:
 *   paged     page * (page_size / block) + block inside the page       k_rows * page_size / block rows
 *   cu_k      cu_k[s] / block + s + b                                   k_rows / block + n_seq rows
 *   else      s * ceil(k_rows / n_seq / block) + b
 * Sequences that share a page share its rows: they have to hold the same keys of a block whose mean a call computes (else one of
 * their means stands there, which one is open).
 */
typedef struct nsparse_lm_attn {
    int dtype;                  /* of q, k, v, out, dout, dq, dk, dv, means */
    int heads, kv_heads;        /* heads % kv_heads == 0, heads / kv_heads <= 1024 */
    int head_dim;               /* a multiple of 8, at most 256 */
    int block;                  /* keys a block: 16, 32, 64, 128 or 256 */
    int width;                  /* entries of a pattern row: 1 .. 256 */
    int causal;
    int n_seq;
    int page_size;              /* 0, or a multiple of block */
    int first, local;           /* selection: the first and the last eligible blocks always taken; see select_blocks */
    float scale;                /* of q.k in the softmax; at most 2.3e38 */
    long long q_rows, k_rows;   /* a sequence has at most 2^31 - 4097 keys; q_rows x heads is limited alike */
    long long table_stride;     /* entries of page_table a sequence */
    const int *cu_q, *cu_k, *q_len, *k_len, *page_table;
    long long q_stride[2];      /* row, head */
    long long k_stride[3];      /* page, row, head */
    long long v_stride[3];
} nsparse_lm_attn;

/* Rows of the block-mean array (see above), or a negative code. */
long long nsparse_lm_mean_rows(const nsparse_lm_attn *a);
/* means[row of (s, b)] = mean of the block's keys that lie inside the sequence.  last > 0: only the blocks that hold
 * the last `last` keys of each sequence (a serving step that appended them); rows of other blocks are left as
 * they were. */
int nsparse_lm_block_means(const nsparse_lm_attn *a, const void *k, void *means, int last, void *stream);
/* idx <- for every query and key head the blocks it selects, ascending, -1 behind.  Score of a block: the group's
 * queries, summed, times its mean (NaN: lowest).  Eligible are the blocks up to the query's own (causal) or all; always taken are
 * the first `first` and, with causal, the last `local` of them (local >= 1: the own block's mean would
 * show later keys; first + local <= width; without causal local is 0), the rest by score, the lower index on a tie.
 * k_rows, cu_k ... describe the keys as above; k itself is not read. */
int nsparse_lm_select_blocks(const nsparse_lm_attn *a, const void *q, const void *means, int *idx, void *stream);
/* out [q_rows, heads, head_dim] and lse float[q_rows, heads] (natural logarithm of the sum of exp; may be NULL), contiguous. */
int nsparse_lm_block_attention(const nsparse_lm_attn *a, const void *q, const void *k, const void *v, const int *idx,
                               void *out, float *lse, void *stream);
/* Gradients; out, lse, dout as the forward laid them out; dq like out; dk, dv [k_rows, kv_heads, head_dim] contiguous, key rows
 * that no query reads get 0, key rows outside every sequence are left as they were.  Not for paged caches.  The second form adds what
 * comes back through lse: dlse float[q_rows, heads], NULL for none; what it holds for a query without a key does not count. */
long long nsparse_lm_block_attention_bwd_workspace(const nsparse_lm_attn *a);
int nsparse_lm_block_attention_bwd(const nsparse_lm_attn *a, const void *q, const void *k, const void *v, const int *idx,
                                   const void *out, const float *lse, const void *dout, void *dq, void *dk, void *dv,
                                   void *workspace, long long workspace_bytes, void *stream);
int nsparse_lm_block_attention_lse_bwd(const nsparse_lm_attn *a, const void *q, const void *k, const void *v, const int *idx,
                                       const void *out, const float *lse, const void *dout, const float *dlse, void *dq, void *dk,
                                       void *dv, void *workspace, long long workspace_bytes, void *stream);

/* ---- tokens sorted by expert -----------------------------------------------------------------------------------
 * ids int[tokens, top]: entry e = t * top + j names an expert; ids outside [0, experts) are dropped (padding, experts
 * of another device).  Stable: entries of one expert keep their order; an expert named twice by a token counts twice.
 *   offsets int[experts + 1]   sorted rows [offsets[e], offsets[e+1]) belong to expert e
 *   order   int[tokens * top]  sorted row -> entry; rows behind offsets[experts] are left as they were
 *   place   int[tokens * top]  entry -> sorted row, -1 where dropped
 * tokens * top < 2^31 - 4096, experts <= 4096, channels <= 2^28. */
long long nsparse_lm_route_workspace(long long tokens, int top, int experts);
int nsparse_lm_route(const int *ids, long long tokens, int top, int experts, int *offsets, int *order, int *place,
                     void *workspace, long long workspace_bytes, void *stream);
/* Where a place is read, one outside [0, tokens * top) counts as dropped.
 * xs[place[t,j], :] = x[t, :]; rows of xs behind the last expert's are left as they were.  x, xs: contiguous rows of `channels`. */
int nsparse_lm_gather_tokens(int dtype, const void *x, const int *place, long long tokens, int top, int channels, void *xs,
                             void *stream);
/* out[t, :] = sum_j w[t,j] y[place[t,j], :], dropped entries left out (none left: 0).  w float[tokens, top], or NULL for ones: then this
 * is the gradient of gather_tokens. */
int nsparse_lm_combine_tokens(int dtype, const void *y, const int *place, const float *w, long long tokens, int top, int channels,
                              void *out, void *stream);
/* dy[place[t,j], :] = w[t,j] dout[t, :], dw[t,j] = dout[t, :] . y[place[t,j], :] (0 where dropped); rows of dy behind the last expert's
 * are left as they were.  w NULL: ones, and dw may be NULL. */
int nsparse_lm_combine_tokens_bwd(int dtype, const void *dout, const void *y, const int *place, const float *w, long long tokens,
                                  int top, int channels, void *dy, float *dw, void *stream);

#ifdef __cplusplus
}
#endif
#endif
