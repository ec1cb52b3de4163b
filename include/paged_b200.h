/* paged_b200.h — C ABI of libggml-b200.so for decoding several continuations of one prompt (beams, samples, conversations behind one system
 * prompt) over a paged cache: a step's keys and values appended with their rotation, attention that reads shared positions once, the choice of a
 * request's best continuations, and the tables, lengths and pages that follow them.
 *
 * The reference serves sequences over one unified cache and picks tokens on the host (crates/llama/src/kv_cache.rs:1887-1917); these calls have no
 * counterpart there.  They stand beside b200_rope + b200_set_rows_f16, b200_flash_attn_ext, b200_argmax and b200_get_rows of ggml_b200.h and keep their
 * manner: device pointers and sizes, a ggml status code as the result with b200_last_error() for the text, nothing aborts.  All calls
 * run on `stream`, may be captured, allocate nothing and read lengths, positions, tables and parents on the device, so that a captured step can be
 * replayed while these change.  Memory is the current device's, or pinned or managed: an operand on another device or in pageable memory is refused.  A workspace belongs to one call at a time: calls that
 * may run side by side, in two streams or two captured graphs, need one each.  Its contents mean nothing between calls.
 *
 * An index that the host cannot see (a page, a sequence, a position beyond the table, a parent) is looked at on the device: what it
 * would have read or written is left out and b200_kernel_error() reports code 7 afterwards.  Waits inside a kernel are bounded: one that runs out (b200_debug_attn_wait
 * makes it) leaves its rows of dst as they were and reports code 4. */
#ifndef PAGED_B200_H
#define PAGED_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* One layer's cache: pages of page_size positions, [page][position][key head][d] 16-bit floats, keys and values alike.  Position p of sequence s is
 * position p % page_size of page tables[s * table_ld + p / page_size]. */
struct b200_paged_cache {
    int32_t type;            /* B200_TYPE_F16 or B200_TYPE_BF16 */
    int32_t page_size;       /* 16, 32, 64, 128 or 256 */
    int64_t n_pages;
    int64_t n_head_kv, d;    /* d: a multiple of 16 up to 1024 (attention: 64 or 128) */
    void *k, *v;             /* 16-byte aligned */
    int64_t page_stride;     /* bytes from page to page, a multiple of 16; 0: the pages lie back to back */
    const int32_t *tables;   /* [n_seq][table_ld] */
    int64_t table_ld, n_seq;
};

/* Keys and values of n_tok tokens into the cache, keys (and queries) turned to their positions on the way: what ROPE of q and k and two SET_ROWS do
 * in four nodes (crates/llama/src/graph_arch.rs:171-190, 1173-1240).  Token t belongs at position pos[t] of sequence seq[t] (seq null: sequence t);
 * a negative position is a padding token: nothing of it is written.  Every value is computed in F32 and rounded once.  n_dims
 * channels of a head rotate, in pairs (2 i, 2 i + 1) (mode 0, NORMAL) or (i, i + n_dims / 2) (mode 2, NEOX); the others are copied.  rope: (cos, sin)
 * rows by position as b200_rope_table makes them (pair i of a row at 2 i and 2 i + 1), rope_ld floats apart.  Strides are bytes per
 * token and per head.  Queries (n_head 0: none) go to q_out in the cache's type; q_out may be q where types and strides are the same.  Two tokens
 * of one call at the same position of a sequence: what stands there afterwards is channels of either. */
struct b200_paged_append_args {
    struct b200_paged_cache cache;
    int64_t n_tok;
    const int32_t *pos, *seq;
    int32_t x_type;          /* of q, k and v: B200_TYPE_F32, F16 or BF16 */
    int32_t n_head;
    const void *k;           int64_t k_nb1, k_nb2;
    const void *v;           int64_t v_nb1, v_nb2;
    const void *q;           int64_t q_nb1, q_nb2;
    void *q_out;             int64_t q_out_nb1, q_out_nb2;
    const float *rope;       int64_t rope_rows, rope_ld;
    int32_t n_dims;          /* even; 0: nothing rotates */
    int32_t mode;
};
int b200_paged_append(const struct b200_paged_append_args *args, void *stream);

/* Attention of one row (token) per sequence over its cached positions 0 .. lens[s] - 1:
 *   dst[s][h] = sum_p w_p v_p / (sum_p w_p + exp(sinks[h])),  w_p = exp(scale q k_p)
 * Sequences stand in groups: group g is sequences group_first[g] .. group_first[g + 1] - 1 (group_first[0] = 0, group_first[n_group] = n_seq), and of
 * sequence s the first shared[s] positions are read through the table of its group's first sequence, once for the whole group; the others through its
 * own table.  n_group 0 (group_first and shared null): nothing is shared.  lens[s] <= 0: a row of zeros; a row whose weights are all zero too.
 * Positions that a row does not see may hold anything.  q and dst are of the cache's type; scores, weights' sums and outputs are F32 until the
 * last rounding, weights enter the second product with 16 bits.  dst may be q where their strides are the same, else they must not overlap.  max_len, max_shared and max_group (most sequences of a group) shape the launch: larger
 * values on the device are served all the same, only less evenly. */
struct b200_prefix_attn_args {
    struct b200_paged_cache cache;   /* d 64 or 128 */
    int64_t n_seq;                   /* rows; at most cache.n_seq */
    int32_t n_head;                  /* a multiple of cache.n_head_kv */
    int32_t n_group;
    const void *q;           int64_t q_nb1, q_nb2;      /* bytes per row, per head: multiples of 16 */
    void *dst;               int64_t dst_nb1, dst_nb2;
    const int32_t *lens, *shared, *group_first;
    const float *sinks;              /* [n_head], finite or -inf (no sink); or null */
    float scale;
    int32_t max_len, max_shared, max_group;
    void *workspace;                 /* b200_prefix_attn_workspace_nbytes(args) bytes, 256-byte aligned */
    size_t workspace_nbytes;
};
size_t b200_prefix_attn_workspace_nbytes(const struct b200_prefix_attn_args *args);   /* 0: the call would be refused, or needs none */
int b200_prefix_attn(const struct b200_prefix_attn_args *args, void *stream);

/* The k best continuations of every request: candidate (b, w) scores scores[b] + log softmax(logits[b])[w], and a beam that has ended (done[b] != 0)
 * has one candidate, (b, end_token) with scores[b].  They come in descending order of their scores, held in 64 bits until they are stored; equal ones
 * by beam, then by logit, then by token.  A logit that is NaN or -inf, and a beam whose score is NaN or -inf, has no candidates; several logits of +inf share the
 * whole probability.  Where fewer than k candidates are left, the rest are score -inf, token -1, parent -1.  out_scores may be scores where k is n_beam;
 * any other overlap of the outputs or the workspace with an operand is refused. */
struct b200_beam_select_args {
    int32_t logits_type;             /* B200_TYPE_F32, F16 or BF16 */
    int32_t n_request, n_beam, k;    /* n_beam 1 .. 64, k 1 .. 128 */
    int64_t n_vocab, logits_ld;      /* elements from row to row; row request * n_beam + beam */
    const void *logits;
    const float *scores;             /* [n_request][n_beam] */
    const uint8_t *done;             /* [n_request][n_beam] or null */
    int32_t end_token;
    float *out_scores;               /* [n_request][k] */
    int32_t *out_tokens, *out_parents;
    void *workspace;                 /* b200_beam_select_workspace_nbytes(args) bytes, 256-byte aligned */
    size_t workspace_nbytes;
};
size_t b200_beam_select_workspace_nbytes(const struct b200_beam_select_args *args);   /* 0: the call would be refused */
int b200_beam_select(const struct b200_beam_select_args *args, void *stream);

/* What the sequences of a request hold, moved to the beams that were chosen: new beam j continues old beam parents[j] (both counted within the request; a
 * negative parent: j is not in use).  Nothing is copied that a table can say: the first child of a parent takes over its row of the table; the others, in
 * ascending order, take the rows of beams without a child, in ascending order, and the parent's pages are copied into theirs; beams not in use take what is left.
 *   row_of[j]           the old beam whose row (pages, state slot) new beam j has now
 *   tables_out[j]       = tables_in[row_of[j]],  lens_out[j] = lens_in[parents[j]], 0 for a beam not in use
 *   pages               where j took another row than its parent's: every page index i with i * page_size < lens_in[parent] and different ids in the
 *                       two rows, in every pool
 * At one index the rows of a request either all name the same page (a shared prefix) or every one its own.  Recurrent states are pools too: a state
 * slot is a page, page_size 1, lens 1, table_ld 1.  Inputs and outputs must not overlap. */
struct b200_beam_reorder_args {
    int32_t n_request, n_beam;       /* n_beam 1 .. 64 */
    const int32_t *parents;          /* [n_request][n_beam] */
    const int32_t *tables_in;        /* [n_request * n_beam][table_ld] */
    int32_t *tables_out;
    int64_t table_ld;
    const int32_t *lens_in;          /* [n_request * n_beam] */
    int32_t *lens_out, *row_of;      /* row_of may be null */
    int32_t page_size, n_pools;
    int64_t n_pages;
    int64_t page_bytes, page_stride; /* of every pool, multiples of 16; page_stride 0: page_bytes */
    void *const *pools;              /* host array of n_pools device pointers, 16-byte aligned */
};
int b200_beam_reorder(const struct b200_beam_reorder_args *args, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* PAGED_B200_H */
