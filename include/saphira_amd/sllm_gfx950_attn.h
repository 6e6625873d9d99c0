/*
 * sllm_gfx950_attn.h -- attention for many sequences on MI355X: a paged cache,
 * a step's attention over it, and causal attention over packed prompts.
 *
 * Device operators beside the projections of sllm_gfx950.h: they take device
 * pointers, enqueue on the library's stream (sllm_gfx950_stream) and return a
 * status; sllm_gfx950_last_error() has the message. Lengths are known on the
 * host, so what depends on them alone (which workgroup takes which rows and
 * keys, the page tables) is laid out once, in a batch or a prompt plan, and
 * serves every layer of a step.
 *
 * Rows are [token][head][head_dim]; a row's head_dim values are adjacent, and
 * pointers and row strides are multiples of 16 bytes. head_dim is a multiple
 * of 8, at most 128; n_head is a multiple of n_head_kv, and query head h reads
 * KV head h / (n_head / n_head_kv). Scores, softmax sums and sums of products
 * are held in f32. The weights that multiply the values are rounded to the
 * cache's type, so a 16-bit result's error is up to 1.4 times what rounding it
 * alone leaves; f32 rows over an f16 cache keep 22 bits of weights and of
 * queries (of elements below 2^-17 of a row's largest, all but 2^-39 of that). The
 * sum of weights times values overflows where that with weights of at most 1 does:
 * values times their number beyond f32's range; values below 2^-118 may lose bits.
 *
 * Calls may come from several threads, whichever device each has current: a
 * cache's calls exclude each other, and everything runs in call order on the
 * one stream. Memory that another stream writes or reads is the caller's to
 * order with the library's stream.
 *
 * batch_store, batch_attend and prompt_attend are launches alone and may be
 * captured into a graph. What takes pages or lays out work (batch_create,
 * seq_fork, seq_copy, pages_compact, prompt_create) is refused while the stream
 * is captured. What is freed or destroyed during a capture keeps its memory until
 * a later call can wait for the stream; the capture goes on.
 */
#ifndef SAPHIRA_AMD_SLLM_GFX950_ATTN_H
#define SAPHIRA_AMD_SLLM_GFX950_ATTN_H

#include <saphira_amd/sllm_gfx950.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define SLLM_GFX950_F32  0
#define SLLM_GFX950_F16  1
#define SLLM_GFX950_BF16 2

#define SLLM_GFX950_ATTN_MAX_HEAD_DIM 128
#define SLLM_GFX950_ATTN_MAX_HEADS    1024
#define SLLM_GFX950_ATTN_MAX_SEQS     65536       /* of one cache, batch or prompt plan */
#define SLLM_GFX950_ATTN_MAX_TOKENS   (1 << 22)   /* new tokens of a batch, query or key rows of a prompt plan */
#define SLLM_GFX950_ATTN_MAX_ROWS     (1 << 24)   /* new tokens x query heads of a batch */
#define SLLM_GFX950_ATTN_MAX_LEN      (1 << 28)   /* positions of a sequence */

/* ------------------------------------------------------------------ */
/* a paged cache                                                       */
/* ------------------------------------------------------------------ */

/*
 * n_pages pages of page_tokens positions each (a power of two, 16 to 1024),
 * for n_layer layers; a page is at most 4 GiB. One allocation of sllm_gfx950_pages_bytes bytes:
 *
 *   [page][layer][K, V][KV head][position in the page][head_dim]
 *
 * mem: that much device memory of the caller's, 16-byte aligned, kept until
 * the cache is freed and its batches are destroyed; NULL: the cache allocates it. Its contents are not
 * cleared; what no store has written is never part of a result.
 *
 * A sequence is a number of positions and the pages that hold them, in order.
 * Pages are handed out lowest free number first. Pages that several sequences
 * hold are read-only by construction: only whole pages are shared, and a
 * sequence that would write into one (it was truncated into it) first gets a
 * copy of its own.
 */
typedef struct sllm_gfx950_pages_desc {
    int32_t n_layer, n_head_kv, head_dim, page_tokens, n_pages;
    int32_t dtype;           /* of the cache */
    void   *mem;
} sllm_gfx950_pages_desc;

typedef struct sllm_gfx950_pages sllm_gfx950_pages;

/* bytes of such a cache; 0 for a description that pages_new refuses */
size_t  sllm_gfx950_pages_bytes(const sllm_gfx950_pages_desc *d);
int     sllm_gfx950_pages_new(const sllm_gfx950_pages_desc *d, sllm_gfx950_pages **out);
/* after the work that uses it; batches still open keep what they need until
 * they are destroyed */
void    sllm_gfx950_pages_free(sllm_gfx950_pages *p);
void   *sllm_gfx950_pages_mem(const sllm_gfx950_pages *p);
/* pages held by a sequence or an open batch */
int32_t sllm_gfx950_pages_in_use(const sllm_gfx950_pages *p);

/* an empty sequence */
int     sllm_gfx950_seq_new(sllm_gfx950_pages *p, int32_t *seq);
/*
 * n new sequences that go on from the first n_tokens positions of src: whole
 * pages are shared, the page that position n_tokens falls into is copied for
 * each (its first n_tokens % page_tokens positions, every layer; the rest of
 * the new page keeps its bytes). It takes what has been stored so far: a store
 * into src's positions that comes later shows in both where the page is shared.
 */
int     sllm_gfx950_seq_fork(sllm_gfx950_pages *p, int32_t src, int32_t n_tokens, int32_t n, int32_t *seqs);
/* a new sequence for each of n, with copies of all its positions in pages of its own */
int     sllm_gfx950_seq_copy(sllm_gfx950_pages *p, const int32_t *src, int32_t n, int32_t *seqs);
/* drop the positions from n_tokens on; pages that nobody holds any more are free again */
int     sllm_gfx950_seq_truncate(sllm_gfx950_pages *p, int32_t seq, int32_t n_tokens);
/* end n sequences: all of them, or none where one is unknown or named twice */
int     sllm_gfx950_seq_free(sllm_gfx950_pages *p, const int32_t *seqs, int32_t n);
/* positions of a sequence, or a negative status */
int32_t sllm_gfx950_seq_len(sllm_gfx950_pages *p, int32_t seq);
/*
 * The page numbers of n sequences, one behind another, into pages[cap]; returns
 * how many there are (written only where they fit), or a negative status.
 */
int32_t sllm_gfx950_seq_tables(sllm_gfx950_pages *p, const int32_t *seqs, int32_t n, int32_t *pages, int32_t cap);
/*
 * Move pages so that those in use are numbers 0 .. in_use - 1: the pages in use
 * above that, in rising order, go to the free numbers below it, in rising
 * order, whole. Refused while a batch is open. *n_moved (or NULL): how many.
 */
int     sllm_gfx950_pages_compact(sllm_gfx950_pages *p, int32_t *n_moved);

/* ------------------------------------------------------------------ */
/* a step of a batch                                                   */
/* ------------------------------------------------------------------ */

/*
 * n sequences, each named once, get n_new[i] >= 0 new positions at their ends
 * (pages are taken; SLLM_GFX950_ERR_NOMEM where there are too few, and nothing
 * is changed). The step's rows are those positions, sequence by sequence. Then,
 * for each layer, store writes the rows' keys and values and attend reads them.
 *
 * act_dtype is the type of every row given or returned: the cache's, or f32
 * over an f16 cache (rounded to nearest by store; queries are not rounded).
 *
 * A batch holds its pages until it is destroyed, whatever happens to its
 * sequences meanwhile; the next batch of a sequence that was truncated may
 * write into the last of them. Its launches may be captured into a graph, which
 * is valid while the batch lives. They share the batch's memory for partial
 * results: graphs of one batch are replayed one after the other.
 */
typedef struct sllm_gfx950_batch sllm_gfx950_batch;

int  sllm_gfx950_batch_create(sllm_gfx950_pages *p, const int32_t *seqs, const int32_t *n_new, int32_t n,
                              int32_t n_head, int32_t act_dtype, sllm_gfx950_batch **out);
void sllm_gfx950_batch_destroy(sllm_gfx950_batch *b);
int32_t sllm_gfx950_batch_rows(const sllm_gfx950_batch *b);

/*
 * k, v: [rows][n_head_kv][head_dim], rows k_stride / v_stride elements apart
 * (0: n_head_kv * head_dim).
 */
int  sllm_gfx950_batch_store(sllm_gfx950_batch *b, int32_t layer, const void *k, size_t k_stride, const void *v,
                             size_t v_stride);
/*
 * out = softmax(scale q . k) v for q and out [rows][n_head][head_dim]: a row
 * sees its sequence's positions up to its own. Whole pages that several of the
 * batch's sequences share are read once for all of them. scale > 0; strides as
 * above (0: n_head * head_dim). out overlaps neither q nor the cache.
 */
int  sllm_gfx950_batch_attend(sllm_gfx950_batch *b, int32_t layer, const void *q, size_t q_stride, float scale,
                              void *out, size_t out_stride);

/* ------------------------------------------------------------------ */
/* whole prompts                                                       */
/* ------------------------------------------------------------------ */

/*
 * Causal attention over n_seq packed sequences: sequence i has q_len[i] query
 * rows and k_len[i] key rows (k_len NULL: as many), one sequence behind the
 * other, and its query row j sees key rows 0 .. j + k_len[i] - q_len[i]. A row
 * that sees none is 0. Every length may be 0. A plan serves any number of calls,
 * one after the other or captured into graphs, which are valid while it lives.
 */
typedef struct sllm_gfx950_prompt_desc {
    int32_t dtype, n_head, n_head_kv, head_dim, n_seq;
    const int32_t *q_len, *k_len;
} sllm_gfx950_prompt_desc;

typedef struct sllm_gfx950_prompt sllm_gfx950_prompt;

/*
 * Device tensors of one call and their strides in elements, between tokens and
 * between heads (0 for both of a tensor: packed). out overlaps no input.
 */
typedef struct sllm_gfx950_prompt_io {
    const void *q, *k, *v;
    void       *out;
    float       scale;       /* > 0 */
    size_t      q_tok, q_head, k_tok, k_head, v_tok, v_head, out_tok, out_head;
} sllm_gfx950_prompt_io;

int  sllm_gfx950_prompt_create(const sllm_gfx950_prompt_desc *d, sllm_gfx950_prompt **out);
int  sllm_gfx950_prompt_attend(sllm_gfx950_prompt *p, const sllm_gfx950_prompt_io *io);
void sllm_gfx950_prompt_destroy(sllm_gfx950_prompt *p);

#ifdef __cplusplus
}
#endif

#endif /* SAPHIRA_AMD_SLLM_GFX950_ATTN_H */
