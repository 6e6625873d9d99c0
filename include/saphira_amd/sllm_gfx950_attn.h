/*
 * sllm_gfx950_attn.h -- attention for many sequences on MI355X: a paged cache, plain
 * or in 8 bits, a step's attention over it, rotary positions, causal attention over packed
 * prompts, and the selection of beams.
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
 * batch_store, batch_rope_store, batch_read, batch_attend, rope_rows, prompt_attend
 * and beam_select are launches alone and may be captured into a graph. What takes pages
 * or lays out work (batch_create, seq_fork, seq_copy, seq_reorder, pages_compact, rope_new,
 * prompt_create, beam_new) is refused while the stream is captured. What is freed or destroyed during a capture keeps its memory until
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
/* of a cache alone: 8 bits and a scale for each row (a position's keys or values of a head) */
#define SLLM_GFX950_I8   4           /* -127 .. 127 */
#define SLLM_GFX950_E4M3 5           /* floating-point: 4 bits of exponent, 3 of mantissa, up to 448 */

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
 * I8 and E4M3 (head_dim a multiple of 16): a KV head's keys or values of a page are its
 * positions' codes, then a scale byte for each. A code stands for code * 2^(byte - 127): the
 * smallest such power of two, 2^-126 or more (E4M3: 2^-117), that 127 (448) times it is at
 * least the row's largest magnitude; codes are rounded to nearest, ties to even. So a row
 * depends on its own values alone, whatever comes before or after it or with it, and what it
 * stands for is exact in f32 and bf16. A row of which something is not finite, or over
 * 127 * 2^120, stands for NaN throughout (its byte is 255).
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
/*
 * Beams that go on from other beams: seqs[i], each named once, becomes what
 * seqs[parent[i]] was (0 <= parent[i] < n), all at one time. Whole pages are shared; the
 * page that a sequence ends in is kept by itself, or else by the first that goes on from
 * it, and copied for each other, in pages that are free then. SLLM_GFX950_ERR_NOMEM where
 * these are too few, and nothing is changed. It takes what has been stored so far: a store
 * that comes later, through a batch made before, shows in whichever sequences hold its page then,
 * the first that went on from it among them, and not in the copies.
 */
int     sllm_gfx950_seq_reorder(sllm_gfx950_pages *p, const int32_t *seqs, const int32_t *parent, int32_t n);
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
 * over an f16 cache (rounded to nearest by store; queries are not rounded), or
 * any of the three over 8 bits. Over 8 bits keys and values are what their codes
 * stand for, queries keep all their bits, and weights 24 (f32) or 16 (f16, bf16); but the 8 of
 * bf16 where more than 64 rows of bf16 see the same keys and there is work enough to go
 * through them 128 at a time.
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
 * The keys and values of a layer read back as rows of act_dtype, every position of
 * the batch's sequences, old and new, sequence by sequence: k, v [batch_positions][n_head_kv]
 * [head_dim], strides as above. Rounded to nearest where act_dtype holds less (f16 of 8 bits).
 * k and v overlap neither each other nor the cache. At most SLLM_GFX950_ATTN_MAX_LEN positions
 * and 2^23 pages, a shared page once for each sequence.
 */
int64_t sllm_gfx950_batch_positions(const sllm_gfx950_batch *b);
int  sllm_gfx950_batch_read(sllm_gfx950_batch *b, int32_t layer, void *k, size_t k_stride, void *v, size_t v_stride);
/*
 * out = softmax(scale q . k) v for q and out [rows][n_head][head_dim]: a row
 * sees its sequence's positions up to its own. Whole pages that several of the
 * batch's sequences share are read once for all of them. scale > 0; strides as
 * above (0: n_head * head_dim). out overlaps neither q nor the cache.
 */
int  sllm_gfx950_batch_attend(sllm_gfx950_batch *b, int32_t layer, const void *q, size_t q_stride, float scale,
                              void *out, size_t out_stride);

/* ------------------------------------------------------------------ */
/* rotary positions                                                    */
/* ------------------------------------------------------------------ */

/*
 * The first n_rot of a head's dimensions, a multiple of 8, are pairs that turn by
 * position times a frequency: (a, b) becomes magnitude (a cos - b sin, b cos + a sin).
 * Pair i is dimensions i and i + n_rot / 2 (HALVES) or 2 i and 2 i + 1 (PAIRS), and turns by
 * freq[i], or base^(-2 i / n_rot), radians a position. For long contexts:
 *
 *   LINEAR  the frequency divided by factor
 *   NTK     base times factor^(n_rot / (n_rot - 2))
 *   PARTS   with turns = original * frequency / (2 pi): as it is from `fast` turns on,
 *           divided by factor below `slow`, and between them in proportion
 *
 * A position times a frequency is reduced to a part of a turn that is exact to 2^-30 of one at any
 * position of 32 bits (of frequencies over a turn a position to as many times that; over 2^20
 * radians they are refused). From there on f32: sine and cosine are off by at most 2^-22 beside
 * that, and rows are rounded once.
 */
enum { SLLM_GFX950_ROPE_HALVES, SLLM_GFX950_ROPE_PAIRS };
enum { SLLM_GFX950_ROPE_PLAIN, SLLM_GFX950_ROPE_LINEAR, SLLM_GFX950_ROPE_NTK, SLLM_GFX950_ROPE_PARTS };

typedef struct sllm_gfx950_rope_desc {
    int32_t head_dim, n_rot, layout, scaling;
    double  base, factor;            /* factor > 0 where there is scaling */
    double  original, fast, slow;    /* PARTS: slow < fast */
    double  magnitude;               /* 0: 1 */
    const double *freq;              /* n_rot / 2, or NULL; not with NTK */
} sllm_gfx950_rope_desc;

typedef struct sllm_gfx950_rope sllm_gfx950_rope;

/* rope_new is refused while the stream is captured */
int  sllm_gfx950_rope_new(const sllm_gfx950_rope_desc *d, sllm_gfx950_rope **out);
/* (graphs that turn rows by it are valid while it lives) */
void sllm_gfx950_rope_free(sllm_gfx950_rope *r);

/*
 * Rows of q [n_rows][n_head][head_dim] and, or NULL, k [n_rows][n_head_kv][head_dim], row i
 * at position pos[i] (device memory; below 0 too), into q_out and k_out: where they come from
 * (same pointer and stride), or memory that overlaps nothing the call reads (rows with different
 * strides overlap where the memory from their first to their last does). Strides in
 * elements, multiples of 16 bytes, 0: packed. back: turned the other way, which is the
 * gradient of what the call did.
 */
typedef struct sllm_gfx950_rope_io {
    int32_t dtype, n_rows, n_head, n_head_kv, back;
    const int32_t *pos;
    const void *q, *k;
    void       *q_out, *k_out;
    size_t      q_stride, q_out_stride, k_stride, k_out_stride;
} sllm_gfx950_rope_io;
int  sllm_gfx950_rope_rows(sllm_gfx950_rope *r, const sllm_gfx950_rope_io *io);

/*
 * A batch's rows at their own positions in one launch: queries turned into q_out (q
 * itself, or apart from q, k and v), keys turned and stored, values stored, as
 * rope_rows and batch_store would (but that turned keys are not rounded to act_dtype before they
 * are to the cache's type).
 */
int  sllm_gfx950_batch_rope_store(sllm_gfx950_batch *b, int32_t layer, sllm_gfx950_rope *r, const void *q, size_t q_stride, void *q_out,
                                  size_t q_out_stride, const void *k, size_t k_stride, const void *v, size_t v_stride);

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

/* ------------------------------------------------------------------ */
/* beams                                                               */
/* ------------------------------------------------------------------ */

/*
 * For each of n_group requests with n_beam beams: the n_pick best of their continuations
 * scores[b] + logits[b][t] - log(sum over t of exp(logits[b][t])), best first. Within a beam
 * they are ordered by logit, between beams by that value, compared in 64 bits; what is alike by the
 * lower beam and the lower token. The sum's terms are of 32 bits: the logarithm is off by at most
 * 2^-24 (17.5 + 4.25 times how far a logit lies below the largest, on average by probability),
 * under 2^-17, and is the same bits for the same row wherever in a plan's calls it lies; so beams
 * nearer to each other than that may come in either order. A NaN logit counts as -infinity. A beam
 * whose score is not finite, or of which a logit is +infinity or all are -infinity, has nothing
 * but -infinity.
 *
 * At most 64 beams and 64 picks, n_beam * n_pick at most 2048 and n_pick at most n_beam * n_vocab;
 * n_vocab at most 2^24, n_group * n_beam at most 2^20. dtype is the logits' type.
 *
 * A plan serves any number of calls, one after the other or captured into graphs, which are
 * valid while it lives and share its memory: graphs of one plan are replayed one after the other.
 */
#define SLLM_GFX950_BEAM_MAX 64      /* beams, picks */

typedef struct sllm_gfx950_beam_desc {
    int32_t n_group, n_beam, n_vocab, n_pick, dtype;
} sllm_gfx950_beam_desc;

typedef struct sllm_gfx950_beam sllm_gfx950_beam;

/* refused while the stream is captured */
int  sllm_gfx950_beam_new(const sllm_gfx950_beam_desc *d, sllm_gfx950_beam **out);
void sllm_gfx950_beam_free(sllm_gfx950_beam *p);
/*
 * Device memory: logits [n_group * n_beam][n_vocab], 16-byte aligned, rows `stride` elements
 * apart (0: n_vocab); scores [n_group][n_beam]; ended [n_group][n_beam] or NULL: below 0, or
 * the token that a beam ended with, which is then its one continuation, at its own
 * score (its logits are not read). Out: score, beam (0 .. n_beam - 1: seq_reorder's parent) and token of
 * each pick, [n_group][n_pick], which overlap nothing that is read, nor each other.
 */
int  sllm_gfx950_beam_select(sllm_gfx950_beam *p, const void *logits, size_t stride, const float *scores, const int32_t *ended,
                             float *out_scores, int32_t *out_beam, int32_t *out_token);

#ifdef __cplusplus
}
#endif

#endif /* SAPHIRA_AMD_SLLM_GFX950_ATTN_H */
