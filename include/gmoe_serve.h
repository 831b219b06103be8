/*
 * gmoe_serve.h -- the operators of a serving step over several requests, on device buffers
 * (libgmoe.so): page tables and slot maps from the requests' lengths, a paged latent cache
 * in 4 bits with the MLA attention that reads it, and log probabilities of given tokens with
 * entropy and top alternatives. gmoe_model_step (gmoe_model.h) runs a whole model on them.
 *
 * glm.c serves one sequence with an fp32 cache (infer.c:843-844, 1012-1058) and samples from
 * its logits on the host (infer.c:1218-1252); these have no counterpart there.
 *
 * Every pointer is device memory of the caller's on GPU `device`, the current device or
 * not; a call leaves the current device as it was. Nothing is allocated and nothing is kept
 * from one call for the next: a call is enqueued on `stream` (a hipStream_t as void*, NULL =
 * default stream of `device`) and may be captured into a graph. Arguments that the host can
 * see are checked before anything is enqueued; lengths, slots, pages and token ids are device
 * data, and what a kernel does with those out of range is said at each. Return codes and gmoe_last_error()
 * as in gmoe.h. Two calls may overlap when neither writes what the other reads or writes,
 * workspaces included.
 */
#ifndef GMOE_SERVE_H
#define GMOE_SERVE_H

#include <stddef.h>
#include <stdint.h>

#include "gmoe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- page tables and slot maps ------------------------------------------------------------
 * A cache is a pool of pages of page_size positions. A request's table row names the page of
 * each page_size of its positions, and slot page * page_size + position % page_size is the
 * position's row of the pool. */

#define GMOE_MAX_REQUESTS 4096
#define GMOE_MAX_STEP_TOKENS (1 << 19)
#define GMOE_MAX_TABLE (1 << 19)

typedef struct gmoe_batch {
    int32_t n_requests;        /* R: 1..GMOE_MAX_REQUESTS */
    int32_t max_tokens;        /* T: tokens that request, position and slot hold, 1..GMOE_MAX_STEP_TOKENS */
    int32_t max_pages;         /* entries of a table row, 1..GMOE_MAX_TABLE */
    int32_t page_size;         /* a power of two, 1..65536 */
    const int32_t *seen;       /* [R] positions cached before the step */
    const int32_t *fresh;      /* [R] tokens the step adds (0: the request is idle) */
    const int32_t *free_pages; /* [*n_free] pages no request holds, taken from the end */
    const int32_t *n_free;     /* [1] */
    int32_t *table;            /* [R][max_pages] */
    int32_t *offsets;          /* [R + 1] each request's first token in the step */
    int32_t *context;          /* [R] positions cached after the step: seen + fresh, 0 where the request is short */
    int32_t *request;          /* [T] the token's request, -1 past the last token */
    int32_t *position;         /* [T] its position in the request, -1 past the last token or of a short request */
    int32_t *slot;             /* [T] its row of the pool, -1 likewise */
    int32_t *totals;           /* [3] tokens, pages taken, short requests */
} gmoe_batch;

/* From seen, fresh, free_pages, n_free and the table's entries for the positions already
 * cached (pages 0 .. ceil(seen / page_size) - 1 of each row): writes the entries of the pages
 * that the step's tokens begin, and every other array. With need = ceil((seen + fresh) /
 * page_size) - ceil(seen / page_size), pages go to the requests in order: the request whose
 * pages follow n others takes free_pages[*n_free - 1 - n], free_pages[*n_free - 2 - n], ...
 * A request is short, takes no page and gets no slots when its tokens end past T, its pages
 * pass max_pages, a length is negative or past 2^30, or it needs pages and its needs and
 * those of the requests before it pass *n_free (then every later one that needs a page is
 * short too). The call changes none of seen, fresh, free_pages and n_free, so that it may be
 * repeated: the caller counts the pages taken (the last totals[1] of free_pages) and the
 * tokens seen. Tokens past T are left out of offsets (each at most T) and totals. */
int gmoe_page_maps(int device, const gmoe_batch *b, void *stream);

/* ---- a latent cache in 4 bits -------------------------------------------------------------
 * A position's row: kv_lora_rank + rope_dim values, the rope part padded with zeros to whole
 * blocks of 32 columns (the OCP microscaling layout: e2m1 elements, one power-of-two scale a
 * block). First the codes, two a byte, the even column in the low half: 1 sign bit over
 * magnitudes 0, 1/2, 1, 3/2, 2, 3, 4, 6; then one byte a block, the scale 2^(byte - 127);
 * then zeros to a multiple of 16 bytes (gmoe_kv4_row_bytes): 320 for 512 + 64 values. The
 * scale is the power of two that brings the block's largest magnitude into (3.5, 7], held to
 * 2^-23 .. 2^13 so that fp16 holds every value; a value is rounded to the nearest magnitude,
 * ties to the even code, at most 6. A block with an infinity or NaN has scale byte 255 and
 * stands for NaN. */
typedef struct gmoe_kv4 {
    void *rows;                /* [n_pages * page_size] rows of one layer, 16-byte aligned */
    int32_t kv_lora_rank;      /* a multiple of 32, 32..512 */
    int32_t rope_dim;          /* even, 2..64 */
    int32_t n_pages, page_size; /* n_pages * page_size < 2^31; page_size as in gmoe_batch */
} gmoe_kv4;

/* Bytes of a row; 0 for ranks outside the above. */
size_t gmoe_kv4_row_bytes(int kv_lora_rank, int rope_dim);

/* The n tokens' rows into their slots: token t's entry comp + t * ld_comp (kv_lora_rank floats)
 * and rope part pe + t * ld_pe (rope_dim floats), distances in floats. A token whose slot is
 * outside the pool is left out. Slots inside it must differ: of two equal ones the row is a
 * mixture. n = 0 does nothing. */
int gmoe_kv4_append(int device, const gmoe_kv4 *c, int n, const float *comp, int64_t ld_comp, const float *pe,
                    int64_t ld_pe, const int32_t *slot, void *stream);

/* The values that the rows of n slots stand for, laid out as gmoe_kv4_append takes them
 * (comp or pe may be NULL); zeros for a slot outside the pool. */
int gmoe_kv4_read(int device, const gmoe_kv4 *c, int n, const int32_t *slot, float *comp, int64_t ld_comp, float *pe,
                  int64_t ld_pe, void *stream);

/* The queries of a step's tokens, in the latent space, and where their heads' results go. */
typedef struct gmoe_kv4_heads {
    int32_t n_heads;           /* H: 1..256 */
    float scale;               /* of the scores (infer.c:992) */
    const float *q_abs;        /* token t, head h: q_abs + t * ld_q_abs + h * kv_lora_rank */
    int64_t ld_q_abs;
    const float *q_pe;         /* q_pe + t * ld_q_pe + h * rope_dim */
    int64_t ld_q_pe;
    float *out;                /* out + t * ld_out + h * kv_lora_rank */
    int64_t ld_out;
    void *work;                /* gmoe_kv4_attend_workspace bytes, 16-byte aligned, of any content */
    size_t work_bytes;
} gmoe_kv4_heads;

/* The attention of the step's tokens over their requests' cached positions (infer.c:1017-1058
 * on the paged form): for token t at position p of its request and head h, over positions
 * 0 .. p, out = sum_j softmax_j(scale (q_abs . comp_j + q_pe . pe_j)) comp_j. Reads of b the
 * sizes, table, offsets (at most max_tokens, rising) and context, as gmoe_page_maps leaves them; the
 * step's own rows are appended first. A position whose page is outside the pool is not attended; a token that
 * attends none (a short request's) gets zeros. Tokens past offsets[R] are not written. fp32
 * in and out; scores, exponentials and sums in fp32. */
int gmoe_kv4_attend(int device, const gmoe_kv4 *c, const gmoe_batch *b, const gmoe_kv4_heads *h, void *stream);

/* Bytes of gmoe_kv4_heads.work for n_heads heads and kv_lora_rank; 0 outside the ranges above. */
size_t gmoe_kv4_attend_workspace(int n_heads, int kv_lora_rank);

/* ---- log probabilities --------------------------------------------------------------------- */

#define GMOE_TOP_MAX 64

typedef struct gmoe_logprobs_args {
    int32_t n, vocab;          /* rows 0..2^24 (0 does nothing), columns 1..2^24 */
    int32_t n_given, top;      /* given tokens (>= 0) and alternatives (0..GMOE_TOP_MAX) a row */
    const float *logits;       /* row i: logits + i * ld, ld >= vocab floats */
    int64_t ld;
    const int32_t *given;      /* [n][n_given] token ids */
    float *logprob;            /* [n][n_given] */
    float *entropy;            /* [n], or NULL */
    int32_t *top_id;           /* [n][top] */
    float *top_logprob;        /* [n][top] */
    void *work;                /* gmoe_logprobs_workspace bytes, 16-byte aligned, of any content */
    size_t work_bytes;
} gmoe_logprobs_args;

/* Per row, of the softmax p of its logits x: ln p of each given token, the entropy -sum p ln p
 * (natural logarithms), and the `top` most likely tokens with their ln p, the most likely first,
 * the lower id first among equal logits. A logit of -inf has p = 0: its ln p is -inf, it adds
 * nothing to the entropy, and it is an alternative only after every other token. A row of -inf
 * alone has ln p = -inf, entropy 0 and ids -1; one with a NaN or +inf has NaN and ids -1. A given id
 * outside the vocabulary has NaN; alternatives past the vocabulary's size have id -1 and -inf.
 * ln p and the entropy keep their relative precision where one token has nearly all of p. */
int gmoe_logprobs(int device, const gmoe_logprobs_args *a, void *stream);

/* Bytes of gmoe_logprobs_args.work for these sizes (0 where they need none or are out of range). */
size_t gmoe_logprobs_workspace(int n, int vocab, int top);

#ifdef __cplusplus
}
#endif

#endif
