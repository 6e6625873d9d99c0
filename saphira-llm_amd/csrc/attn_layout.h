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

typedef struct att_pair { uint32_t src, dst, rows; } att_pair;
#define ATT_PAIRS 320

/* blocks of block_bytes (a KV head's keys or values of a page in one layer),
 * of each the first rows * row_bytes */
typedef struct att_copy_args {
    uint8_t  *mem;
    uint64_t  page_bytes;
    uint32_t  block_bytes, row_bytes, n_blocks, n_pairs;
    att_pair  pair[ATT_PAIRS];
} att_copy_args;

#define ATT_COPY_CHUNKS 1024u        /* 16-byte pieces a workgroup */

#if defined(__cplusplus)
static_assert(sizeof(att_item) == 48 && sizeof(att_args) == 168 && sizeof(att_copy_args) <= 4096, "attn_layout.h");
#else
_Static_assert(sizeof(att_item) == 48 && sizeof(att_args) == 168 && sizeof(att_copy_args) <= 4096, "attn_layout.h");
#endif

#endif /* SLLM_ATTN_LAYOUT_H */
