/*
 * attn_layout.h -- what attn.c hands to the kernels of attn_kernels.hip: the
 * argument structs and the device tables, one definition for both sides.
 */
#ifndef SLLM_ATTN_LAYOUT_H
#define SLLM_ATTN_LAYOUT_H

#include <stdint.h>

/* rows (query token x head of one KV head) that a workgroup takes: the four
 * waves on different keys of the same 16, or with 16 or 32 rows each */
#define ATT_FEW_ROWS  16
#define ATT_HALF_ROWS 64
#define ATT_MANY_ROWS 128
#define ATT_THREADS   256
enum { ATT_FEW, ATT_HALF, ATT_MANY };

#define ATT_DIRECT    0xffffffffu    /* att_item.part: rows go to the output */
#define ATT_TOKENS    0xffffffffu    /* att_item.list: tokens in order */
#define ATT_SEE_ALL   (1 << 30)      /* att_item.vis0: every key of the range */

/*
 * One workgroup's share: n_rows rows of a segment (a run of keys and the tokens
 * that read it), from row t0 * group + h0 on, against its keys key0 .. key1. Row
 * r is token r / group and head r % group of KV head `head`; token t is row
 * tok0 + t of the query tensor, or what list[list + t] names, and sees the
 * keys below vis0 + t.
 */
typedef struct att_item {
    uint32_t t0, n_rows, tok0, list;
    int32_t  vis0;
    uint32_t key0, key1;
    uint32_t kv;            /* paged: where the segment's page numbers start; packed: the first key's row */
    uint32_t head;
    uint32_t part;          /* row of the partial results that the first row's go to, or ATT_DIRECT */
    uint16_t mode, h0;      /* ATT_FEW .. ATT_MANY */
    uint32_t order;         /* the order they came in */
} att_item;

typedef struct att_args {
    const void     *q;
    void           *out;
    const uint8_t  *k, *v;           /* paged: the layer's keys and values in page 0 */
    const uint32_t *tables;
    const uint32_t *list;
    const att_item *items;
    float          *part_o;          /* [row][head_dim padded] sums of p v */
    float          *part_ml;         /* [row][2]: the running maximum (log2) and the sum of p */
    uint64_t        q_tok, q_head, out_tok, out_head;    /* bytes */
    uint64_t        k_tok, k_head, v_tok, v_head;        /* bytes */
    uint64_t        page_bytes;
    uint32_t        page_shift, hd, group, n_items;
    float           c;               /* scale * log2(e) */
    float           per_group;       /* 1 / group */
    uint32_t        block_bytes, pad;    /* 8 bits: a KV head's keys or values in a page */
} att_args;

/* the partial results of a token: those of n_split splits of a segment, whose
 * rows are n_rows apart from split to split and n_split * n_rows from KV head
 * to KV head */
typedef struct att_seg {
    uint32_t part0, n_rows, n_split, row_off;
} att_seg;

/* a new token of a batch: where its sequence's page numbers start and its
 * position (the store); the segments of its sequence and its number in the step
 * (the join; n_seg 0: its rows are in the output already) */
typedef struct att_tok {
    uint32_t table, pos, seg0, n_seg, t;
    uint32_t pad[3];
} att_tok;

typedef struct att_join_args {
    void           *out;
    const float    *part_o, *part_ml;
    const att_tok  *toks;
    const att_seg  *segs;
    uint64_t        out_tok;         /* bytes */
    uint32_t        hd, group, n_head, pad;
} att_join_args;

typedef struct att_store_args {
    const void     *k, *v;
    uint8_t        *ck, *cv;         /* the layer's keys and values in page 0 */
    const uint32_t *tables;
    const att_tok  *toks;
    uint64_t        k_tok, v_tok;    /* bytes */
    uint64_t        page_bytes;
    uint32_t        page_shift, hd, n_head_kv, n_tok;
} att_store_args;

/* what rows are held as (att_rows_args.held, att_read_args.held) */
enum { ATT_HELD_F32, ATT_HELD_F16, ATT_HELD_BF16, ATT_HELD_I8, ATT_HELD_E4M3 };
/* the scale byte of a row of 8 bits: 2^(byte - 127); ATT_NAN_ROW: something in it is not finite */
#define ATT_NAN_ROW   255u

/*
 * Rows of one type on their way: queries and keys turned by their position (or,
 * half 0, as they are) into q_out and k_out, or keys and values into the cache.
 * A row is n_head, n_head_kv heads of hd values; NULL: there are none of these.
 */
typedef struct att_rows_args {
    const void     *q, *k, *v;
    void           *q_out, *k_out;   /* k_out NULL: to the cache */
    uint8_t        *ck, *cv;         /* the layer's keys and values in page 0 */
    const uint32_t *tables;
    const att_tok  *toks;            /* positions, or NULL: */
    const int32_t  *pos;
    const uint64_t *freq;            /* [half] turns a position, modulo 1, times 2^64 */
    uint64_t        q_tok, k_tok, v_tok, qo_tok, ko_tok;     /* bytes */
    uint64_t        page_bytes;
    uint32_t        n_tok, n_head, n_head_kv, hd, half, pairs, back;     /* pairs: 2i, 2i + 1; else i, i + half */
    uint32_t        held, page_shift, block_bytes, waves;    /* waves a token */
    float           magnitude;
} att_rows_args;

/* a batch's sequences: where the page numbers of each start, and its first position's row in what is read back */
typedef struct att_seq { uint32_t table, row0; } att_seq;

typedef struct att_read_args {
    void           *k, *v;
    const uint8_t  *ck, *cv;
    const uint32_t *tables;
    const att_seq  *seqs;            /* n_seq of them, then one past the last */
    uint64_t        k_tok, v_tok;    /* bytes */
    uint64_t        page_bytes;
    uint32_t        n_seq, hd, n_head_kv, held, page_shift, block_bytes;
} att_read_args;
#define ATT_READ_UNITS 4u            /* pieces of 8 values that a thread reads back */

/*
 * The best continuations of beams: each workgroup of the first launch takes a part of a row of
 * logits, `chunk` of them, and leaves its sum of exponentials and its best n_pick keys in order; the
 * second launch joins them, a group a workgroup.
 */
#define BEAM_MAX_LIST  2048u         /* n_beam * n_pick */
#define BEAM_MAX_PARTS 64u           /* of a row: a lane each in the join, as picks are in both */
#define BEAM_JOIN_THREADS 512u
#define BEAM_VALUES    8u            /* of a thread at a time */
#define BEAM_TILE      (ATT_THREADS * BEAM_VALUES)
typedef struct att_beam_args {
    const void    *logits;
    const float   *scores;
    const int32_t *ended;            /* or NULL */
    float         *out;
    int32_t       *beam, *token;
    double        *sums;             /* [row][chunk][2]: a reference near the largest logit, the sum of exponentials relative to it */
    uint64_t      *keys;             /* [row][chunk][n_pick] */
    uint64_t       stride;           /* bytes */
    uint32_t       n_beam, n_vocab, n_pick, n_chunk, chunk, pad;
} att_beam_args;

typedef struct att_pair { uint32_t src, dst, rows; } att_pair;
#define ATT_PAIRS 320

/* blocks of block_bytes (a KV head's keys or values of a page in one layer),
 * of each the first rows * row_bytes */
typedef struct att_copy_args {
    uint8_t  *mem;
    uint64_t  page_bytes;
    uint32_t  block_bytes, row_bytes, n_blocks, n_pairs;
    att_pair  pair[ATT_PAIRS];
    uint32_t  scales;                /* 8 bits: where a block's scale bytes start, of which rows are copied too */
    const att_pair *list;            /* the pairs, where they are more than `pair` has room for */
} att_copy_args;

#define ATT_COPY_CHUNKS 1024u        /* 16-byte pieces a workgroup */

#if defined(__cplusplus)
static_assert(sizeof(att_item) == 48 && sizeof(att_args) == 176 && sizeof(att_copy_args) <= 4096, "attn_layout.h");
#else
_Static_assert(sizeof(att_item) == 48 && sizeof(att_args) == 176 && sizeof(att_copy_args) <= 4096, "attn_layout.h");
#endif

#endif /* SLLM_ATTN_LAYOUT_H */
