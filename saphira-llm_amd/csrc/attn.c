/*
 * attn.c -- the paged cache, a step's batch and the prompt plan of
 * sllm_gfx950_attn.h: host side of attn_kernels.hip.
 *
 * Which pages a sequence holds is known here alone, so every page number that a
 * kernel reads comes from a table built and checked here. A batch lays out the
 * step once: the sequences' page tables, the runs of pages that several of them
 * share, and which workgroup takes which rows against which keys.
 */
#define _POSIX_C_SOURCE 200809L

#include "shim_internal.h"
#include "attn_layout.h"

#include <saphira_amd/sllm_gfx950_attn.h>

#include <math.h>
#include <pthread.h>
#include <stdlib.h>
#include <string.h>

#define ATT_NEED_OPEN()                                                                  \
    do {                                                                                 \
        if (!sllm_shim_is_open()) return sllm_shim_fail(SLLM_GFX950_ERR_NO_DEVICE, "library not open"); \
    } while (0)

/*
 * The library's device is the current one for the rest of the call and the
 * caller's is afterwards: memory is taken on the current device, and a caller
 * may have another one current, or be a thread that never set one.
 */
typedef struct device_scope { int was, moved; } device_scope;

static int device_enter(device_scope *s) {
    if (!sllm_shim_is_open()) return sllm_shim_fail(SLLM_GFX950_ERR_NO_DEVICE, "library not open");
    hipError_t e = hipGetDevice(&s->was);
    if (e != hipSuccess) return sllm_shim_hip_fail(e, "hipGetDevice");
    if (s->was == sllm_shim_device()) return SLLM_GFX950_OK;
    e = hipSetDevice(sllm_shim_device());
    if (e != hipSuccess) return sllm_shim_hip_fail(e, "hipSetDevice");
    s->moved = 1;
    return SLLM_GFX950_OK;
}
static void device_leave(device_scope *s) { if (s->moved) hipSetDevice(s->was); }

#define ATT_ON_DEVICE()                                                                  \
    device_scope scope __attribute__((cleanup(device_leave))) = { 0, 0 };                \
    do {                                                                                 \
        const int scope_st = device_enter(&scope);                                       \
        if (scope_st != SLLM_GFX950_OK) return scope_st;                                 \
    } while (0)

#define FAIL_ARG(...)   sllm_shim_fail(SLLM_GFX950_ERR_ARG, __VA_ARGS__)
#define FAIL_NOMEM(...) sllm_shim_fail(SLLM_GFX950_ERR_NOMEM, __VA_ARGS__)

#define LOG2E 1.44269504088896340736

static int held8(int32_t dtype) { return dtype == SLLM_GFX950_I8 || dtype == SLLM_GFX950_E4M3; }
static uint32_t type_size(int32_t dtype) { return dtype == SLLM_GFX950_F32 ? 4u : held8(dtype) ? 1u : 2u; }
static int bad_type(int32_t dtype) { return dtype != SLLM_GFX950_F32 && dtype != SLLM_GFX950_F16 && dtype != SLLM_GFX950_BF16; }

/* the kernels' instances for rows and a cache of these types (shim_internal.h), or -1 */
static int type_pair(int32_t act, int32_t cache) {
    if (held8(cache)) return SLLM_ATTN_HELD8 + 3 * (cache == SLLM_GFX950_E4M3) + act;
    if (act == cache) return act == SLLM_GFX950_F32 ? 0 : act == SLLM_GFX950_F16 ? 2 : 3;
    return act == SLLM_GFX950_F32 && cache == SLLM_GFX950_F16 ? 1 : -1;
}

static int bad_heads(int32_t n_head, int32_t n_head_kv, int32_t head_dim) {
    return n_head_kv < 1 || n_head < n_head_kv || n_head > SLLM_GFX950_ATTN_MAX_HEADS || n_head % n_head_kv != 0 ||
           head_dim < 8 || head_dim > SLLM_GFX950_ATTN_MAX_HEAD_DIM || head_dim % 8 != 0;
}

/* device memory, and the pinned memory that what is in it is sent from (`sent`: the
 * copy out of `pin` is done) */
typedef struct buffer {
    uint8_t   *dev, *pin;
    size_t     dev_bytes, pin_bytes;
    hipEvent_t sent;
} buffer;

static void buffer_drop(buffer *b) {
    if (b->dev) hipFree(b->dev);
    if (b->pin) hipHostFree(b->pin);
    if (b->sent) hipEventDestroy(b->sent);
    memset(b, 0, sizeof *b);
}

/* What was released while the stream was captured: waiting for the stream would end the
 * capture. The next call that may wait frees it, or close. */
static struct { pthread_mutex_t mtx; buffer *v; size_t n, cap; } g_later = { PTHREAD_MUTEX_INITIALIZER, NULL, 0, 0 };

static void release_later(void) {
    pthread_mutex_lock(&g_later.mtx);
    if (g_later.n > 0) {
        if (sllm_shim_is_open()) hipStreamSynchronize(sllm_shim_stream());
        for (size_t i = 0; i < g_later.n; ++i) buffer_drop(&g_later.v[i]);
        free(g_later.v);
        g_later.v = NULL;
        g_later.n = g_later.cap = 0;
    }
    pthread_mutex_unlock(&g_later.mtx);
}

void sllm_shim_attn_close(void) { release_later(); }

/* Frees n buffers once what is on the stream is done with them. */
static void release(buffer *b, int n) {
    hipStreamCaptureStatus is = hipStreamCaptureStatusNone;
    if (sllm_shim_is_open() && hipStreamIsCapturing(sllm_shim_stream(), &is) == hipSuccess && is != hipStreamCaptureStatusNone) {
        pthread_mutex_lock(&g_later.mtx);
        for (int i = 0; i < n; ++i) {
            if (g_later.n == g_later.cap) {
                const size_t cap = g_later.cap ? g_later.cap * 2 : 16;
                buffer *v = realloc(g_later.v, cap * sizeof *v);
                if (v == NULL) break;                    /* (it stays until the process ends) */
                g_later.v = v;
                g_later.cap = cap;
            }
            g_later.v[g_later.n++] = b[i];
        }
        pthread_mutex_unlock(&g_later.mtx);
        memset(b, 0, (size_t) n * sizeof *b);
        return;
    }
    release_later();
    if (sllm_shim_is_open()) hipStreamSynchronize(sllm_shim_stream());
    for (int i = 0; i < n; ++i) buffer_drop(&b[i]);
}

/* What changes who holds which page runs once, on the host: a graph would replay
 * its copies into pages that are others' by then. */
static int not_in_capture(const char *who) {
    hipStreamCaptureStatus is = hipStreamCaptureStatusNone;
    const hipError_t e = hipStreamIsCapturing(sllm_shim_stream(), &is);
    if (e != hipSuccess) return sllm_shim_hip_fail(e, "hipStreamIsCapturing");
    if (is != hipStreamCaptureStatusNone) return FAIL_ARG("%s: the stream is being captured", who);
    release_later();
    return SLLM_GFX950_OK;
}

/* what the kernels of rows call a cache's type */
static uint32_t held_as(int32_t dtype) {
    return dtype == SLLM_GFX950_F32 ? ATT_HELD_F32 : dtype == SLLM_GFX950_F16 ? ATT_HELD_F16 : dtype == SLLM_GFX950_BF16 ? ATT_HELD_BF16 :
           dtype == SLLM_GFX950_I8 ? ATT_HELD_I8 : ATT_HELD_E4M3;
}

static int misaligned(const void *p) { return ((uintptr_t) p & 15u) != 0; }

/* ------------------------------------------------------------------ */
/* the cache                                                           */
/* ------------------------------------------------------------------ */

typedef struct sequence {
    int32_t  used, len;
    int32_t  n_pages, cap;
    int32_t *page;
    uint32_t mark;                   /* the call that named it last (pool's stamp) */
} sequence;

/* a batch's buffer is kept by the cache for the next batch */
#define KEPT_BUFFERS 4

struct sllm_gfx950_pages {
    pthread_mutex_t mtx;
    sllm_gfx950_pages_desc d;
    uint8_t   *mem;
    int        own_mem, gone;        /* gone: freed, batches still open */
    uint64_t   page_bytes, layer_bytes;
    uint32_t   page_shift, block_bytes, row_bytes;
    /* who holds a page: sequences, and open batches */
    int32_t   *refs, *holds;
    int32_t    n_free, low;          /* low: no free page below it */
    sequence  *seq;
    int32_t    n_seq, cap_seq, low_seq;
    uint32_t   stamp;
    int32_t    open;                 /* batches */
    buffer     kept[KEPT_BUFFERS];
    int        n_kept;
};

static uint64_t desc_page_bytes(const sllm_gfx950_pages_desc *d) {
    /* (8 bits: a scale byte for each row) */
    const uint64_t row = (uint64_t) d->head_dim * type_size(d->dtype) + (uint64_t) held8(d->dtype);
    return (uint64_t) d->n_layer * 2u * (uint64_t) d->n_head_kv * (uint64_t) d->page_tokens * row;
}

static int bad_desc(const sllm_gfx950_pages_desc *d) {
    return d == NULL || (bad_type(d->dtype) && !held8(d->dtype)) || (held8(d->dtype) && d->head_dim % 16 != 0) || bad_heads(d->n_head_kv, d->n_head_kv, d->head_dim) || d->n_layer < 1 ||
           d->n_layer > 65536 || d->page_tokens < 16 || d->page_tokens > 1024 || (d->page_tokens & (d->page_tokens - 1)) != 0 ||
           d->n_pages < 1 || d->n_pages > (1 << 28) || desc_page_bytes(d) > 1ull << 32;
}

size_t sllm_gfx950_pages_bytes(const sllm_gfx950_pages_desc *d) {
    return bad_desc(d) ? 0 : (size_t) (desc_page_bytes(d) * (uint64_t) d->n_pages);
}

int sllm_gfx950_pages_new(const sllm_gfx950_pages_desc *d, sllm_gfx950_pages **out) {
    ATT_ON_DEVICE();
    if (out == NULL) return FAIL_ARG("pages_new: NULL out");
    *out = NULL;
    if (bad_desc(d)) return FAIL_ARG("pages_new: sizes, page length or type outside what a cache takes");
    if (misaligned(d->mem)) return FAIL_ARG("pages_new: mem is not 16-byte aligned");
    sllm_gfx950_pages *p = calloc(1, sizeof *p);
    int32_t *counts = calloc((size_t) d->n_pages * 2, sizeof *counts);
    if (p == NULL || counts == NULL) {
        free(p);
        free(counts);
        return FAIL_NOMEM("pages_new: %d pages", d->n_pages);
    }
    p->d = *d;
    p->refs = counts;
    p->holds = counts + d->n_pages;
    p->n_free = d->n_pages;
    p->page_bytes = desc_page_bytes(d);
    p->layer_bytes = p->page_bytes / (uint64_t) d->n_layer;
    p->row_bytes = (uint32_t) d->head_dim * type_size(d->dtype);
    p->block_bytes = (uint32_t) d->page_tokens * (p->row_bytes + (uint32_t) held8(d->dtype));
    while ((1 << p->page_shift) < d->page_tokens) ++p->page_shift;
    p->mem = d->mem;
    if (p->mem == NULL) {
        const hipError_t e = hipMalloc((void **) &p->mem, (size_t) (p->page_bytes * (uint64_t) d->n_pages));
        if (e != hipSuccess) {
            free(p);
            free(counts);
            return sllm_shim_hip_fail(e, "hipMalloc(pages)");
        }
        p->own_mem = 1;
    }
    pthread_mutex_init(&p->mtx, NULL);
    *out = p;
    return SLLM_GFX950_OK;
}

static void pages_drop(sllm_gfx950_pages *p) {
    buffer own = { .dev = p->mem };
    release(p->kept, p->n_kept);
    if (p->own_mem) release(&own, 1);
    for (int32_t i = 0; i < p->n_seq; ++i) free(p->seq[i].page);
    free(p->seq);
    free(p->refs);
    pthread_mutex_destroy(&p->mtx);
    free(p);
}

void sllm_gfx950_pages_free(sllm_gfx950_pages *p) {
    if (p == NULL) return;
    pthread_mutex_lock(&p->mtx);
    p->gone = 1;
    const int32_t open = p->open;
    pthread_mutex_unlock(&p->mtx);
    if (open == 0) pages_drop(p);
}

void *sllm_gfx950_pages_mem(const sllm_gfx950_pages *p) { return p ? p->mem : NULL; }
int32_t sllm_gfx950_pages_in_use(const sllm_gfx950_pages *p) {
    if (p == NULL) return 0;
    pthread_mutex_t *mtx = (pthread_mutex_t *) &p->mtx;
    pthread_mutex_lock(mtx);
    const int32_t n = p->d.n_pages - p->n_free;
    pthread_mutex_unlock(mtx);
    return n;
}

/* (the cache's lock is held by everything below that takes or gives pages) */

static int32_t take_page(sllm_gfx950_pages *p) {         /* (n_free > 0) */
    while (p->refs[p->low] != 0 || p->holds[p->low] != 0) ++p->low;
    --p->n_free;
    p->refs[p->low] = 1;
    return p->low++;
}

static void maybe_free(sllm_gfx950_pages *p, int32_t page) {
    if (p->refs[page] != 0 || p->holds[page] != 0) return;
    ++p->n_free;
    if (page < p->low) p->low = page;
}

static void give_page(sllm_gfx950_pages *p, int32_t page) {
    --p->refs[page];
    maybe_free(p, page);
}

static sequence *find(sllm_gfx950_pages *p, int32_t s) {
    return s >= 0 && s < p->n_seq && p->seq[s].used ? &p->seq[s] : NULL;
}

static int32_t pages_for(const sllm_gfx950_pages *p, int32_t len) {
    return (int32_t) (((uint32_t) len + (1u << p->page_shift) - 1u) >> p->page_shift);
}

static int reserve(sequence *s, int32_t n) {             /* room for n page numbers; 0: no memory */
    if (n <= s->cap) return 1;
    int32_t cap = s->cap < 16 ? 16 : s->cap;
    while (cap < n) cap += cap / 2;
    int32_t *page = realloc(s->page, (size_t) cap * sizeof *page);
    if (page == NULL) return 0;
    s->page = page;
    s->cap = cap;
    return 1;
}

/* n empty sequences into ids; 0: no memory (none is made) */
static int new_sequences(sllm_gfx950_pages *p, int32_t n, int32_t *ids) {
    int32_t at = p->low_seq, got = 0;
    while (got < n) {
        while (at < p->n_seq && p->seq[at].used) ++at;
        if (at == p->cap_seq) {
            const int32_t cap = p->cap_seq ? p->cap_seq * 2 : 64;
            sequence *seq = cap > SLLM_GFX950_ATTN_MAX_SEQS ? NULL : realloc(p->seq, (size_t) cap * sizeof *seq);
            if (seq == NULL) break;
            memset(seq + p->cap_seq, 0, (size_t) (cap - p->cap_seq) * sizeof *seq);
            p->seq = seq;
            p->cap_seq = cap;
        }
        if (at == p->n_seq) ++p->n_seq;
        p->seq[at].used = 1;
        p->seq[at].len = p->seq[at].n_pages = 0;
        ids[got++] = at;
    }
    if (got < n) {
        while (got-- > 0) p->seq[ids[got]].used = 0;
        return 0;
    }
    if (n > 0) p->low_seq = at + 1;
    return 1;
}

static void end_sequence(sllm_gfx950_pages *p, int32_t id) {
    sequence *s = &p->seq[id];
    for (int32_t i = 0; i < s->n_pages; ++i) give_page(p, s->page[i]);
    s->used = s->len = s->n_pages = 0;
    if (id < p->low_seq) p->low_seq = id;
}

/* copies of pages, in as few launches as they fit */
typedef struct copies {
    const sllm_gfx950_pages *p;
    att_copy_args a;
    uint32_t most;                   /* rows of the pair with the most */
    int      st;
} copies;

static void copies_start(copies *c, const sllm_gfx950_pages *p) {
    c->p = p;
    c->a.mem = p->mem;
    c->a.page_bytes = p->page_bytes;
    c->a.block_bytes = p->block_bytes;
    c->a.row_bytes = p->row_bytes;
    c->a.n_blocks = (uint32_t) (p->page_bytes / p->block_bytes);
    c->a.scales = held8(p->d.dtype) ? (uint32_t) p->d.page_tokens * p->row_bytes : 0;
    c->a.list = NULL;
    c->a.n_pairs = c->most = 0;
    c->st = SLLM_GFX950_OK;
}

static int copies_flush(copies *c) {
    if (c->st == SLLM_GFX950_OK && c->a.n_pairs > 0) {
        const uint64_t chunks = ((uint64_t) c->most * c->a.row_bytes / 16u + (c->a.scales ? (c->most + 15u) / 16u : 0u)) * c->a.n_blocks;
        void *args[] = { &c->a };
        c->st = sllm_shim_launch(sllm_shim_attn_function(c->a.scales ? SLLM_ATTN_COPY8 : SLLM_ATTN_COPY),
                                 (uint32_t) ((chunks + ATT_COPY_CHUNKS - 1) / ATT_COPY_CHUNKS), c->a.n_pairs, ATT_THREADS, 0, args);
    }
    c->a.n_pairs = c->most = 0;
    return c->st;
}

static void copies_add(copies *c, int32_t src, int32_t dst, int32_t rows) {
    if (c->a.n_pairs == ATT_PAIRS) copies_flush(c);
    c->a.pair[c->a.n_pairs++] = (att_pair) { (uint32_t) src, (uint32_t) dst, (uint32_t) rows };
    if ((uint32_t) rows > c->most) c->most = (uint32_t) rows;
}

int sllm_gfx950_seq_new(sllm_gfx950_pages *p, int32_t *seq) {
    ATT_NEED_OPEN();
    if (p == NULL || seq == NULL) return FAIL_ARG("seq_new: NULL");
    pthread_mutex_lock(&p->mtx);
    const int ok = new_sequences(p, 1, seq);
    pthread_mutex_unlock(&p->mtx);
    return ok ? SLLM_GFX950_OK : FAIL_NOMEM("seq_new: no room for another sequence");
}

int sllm_gfx950_seq_fork(sllm_gfx950_pages *p, int32_t src, int32_t n_tokens, int32_t n, int32_t *seqs) {
    ATT_ON_DEVICE();
    if (p == NULL || n < 0 || (n > 0 && seqs == NULL)) return FAIL_ARG("seq_fork: NULL or a count below 0");
    if (n > SLLM_GFX950_ATTN_MAX_SEQS) return FAIL_ARG("seq_fork: %d copies", n);
    pthread_mutex_lock(&p->mtx);
    int st = not_in_capture("seq_fork");
    const sequence *s = find(p, src);
    if (st != SLLM_GFX950_OK) { }
    else if (s == NULL) st = FAIL_ARG("seq_fork: no sequence %d", src);
    else if (n_tokens < 0 || n_tokens > s->len) st = FAIL_ARG("seq_fork: %d of %d positions", n_tokens, s->len);
    const int32_t whole = n_tokens >> p->page_shift, rows = n_tokens & (p->d.page_tokens - 1);
    if (st == SLLM_GFX950_OK && rows && n > p->n_free) st = FAIL_NOMEM("seq_fork: %d pages wanted, %d free", n, p->n_free);
    if (st == SLLM_GFX950_OK && !new_sequences(p, n, seqs)) st = FAIL_NOMEM("seq_fork: no room for %d sequences", n);
    int32_t got = 0;
    if (st == SLLM_GFX950_OK) {
        copies c;
        copies_start(&c, p);
        for (; got < n && st == SLLM_GFX950_OK; ++got) {
            s = &p->seq[src];                            /* (new_sequences may have moved them) */
            sequence *f = &p->seq[seqs[got]];
            if (!reserve(f, whole + 1)) { st = FAIL_NOMEM("seq_fork: page table"); break; }
            if (whole > 0) memcpy(f->page, s->page, (size_t) whole * sizeof *f->page);
            for (int32_t i = 0; i < whole; ++i) ++p->refs[f->page[i]];
            f->n_pages = whole;
            f->len = n_tokens;
            if (rows) {
                const int32_t to = take_page(p);
                f->page[f->n_pages++] = to;
                copies_add(&c, s->page[whole], to, rows);
            }
        }
        if (st == SLLM_GFX950_OK) st = copies_flush(&c);
        if (st != SLLM_GFX950_OK) for (int32_t i = 0; i < n; ++i) end_sequence(p, seqs[i]);
    }
    pthread_mutex_unlock(&p->mtx);
    return st;
}

int sllm_gfx950_seq_copy(sllm_gfx950_pages *p, const int32_t *src, int32_t n, int32_t *seqs) {
    ATT_ON_DEVICE();
    if (p == NULL || n < 0 || (n > 0 && (src == NULL || seqs == NULL))) return FAIL_ARG("seq_copy: NULL or a count below 0");
    if (n > SLLM_GFX950_ATTN_MAX_SEQS) return FAIL_ARG("seq_copy: %d copies", n);
    int32_t *ids = malloc((size_t) (n ? n : 1) * sizeof *ids);      /* (src and seqs may be one array) */
    if (ids == NULL) return FAIL_NOMEM("seq_copy: %d sequences", n);
    pthread_mutex_lock(&p->mtx);
    int st = not_in_capture("seq_copy");
    int64_t want = 0;
    for (int32_t i = 0; i < n && st == SLLM_GFX950_OK; ++i) {
        const sequence *s = find(p, src[i]);
        if (s == NULL) st = FAIL_ARG("seq_copy: no sequence %d", src[i]);
        else want += s->n_pages;
    }
    if (st == SLLM_GFX950_OK && want > p->n_free) st = FAIL_NOMEM("seq_copy: %lld pages wanted, %d free", (long long) want, p->n_free);
    if (st == SLLM_GFX950_OK && !new_sequences(p, n, ids)) st = FAIL_NOMEM("seq_copy: no room for %d sequences", n);
    if (st == SLLM_GFX950_OK) {
        copies c;
        copies_start(&c, p);
        for (int32_t i = 0; i < n && st == SLLM_GFX950_OK; ++i) {
            const sequence *s = &p->seq[src[i]];
            sequence *f = &p->seq[ids[i]];
            if (!reserve(f, s->n_pages)) { st = FAIL_NOMEM("seq_copy: page table"); break; }
            for (int32_t j = 0; j < s->n_pages; ++j) {
                f->page[f->n_pages++] = take_page(p);
                const int32_t left = s->len - (j << p->page_shift);
                copies_add(&c, s->page[j], f->page[j], left < p->d.page_tokens ? left : p->d.page_tokens);
            }
            f->len = s->len;
        }
        if (st == SLLM_GFX950_OK) st = copies_flush(&c);
        if (st == SLLM_GFX950_OK) memcpy(seqs, ids, (size_t) n * sizeof *ids);
        else for (int32_t i = 0; i < n; ++i) end_sequence(p, ids[i]);
    }
    pthread_mutex_unlock(&p->mtx);
    free(ids);
    return st;
}

int sllm_gfx950_seq_truncate(sllm_gfx950_pages *p, int32_t seq, int32_t n_tokens) {
    ATT_NEED_OPEN();
    if (p == NULL) return FAIL_ARG("seq_truncate: NULL");
    pthread_mutex_lock(&p->mtx);
    int st = SLLM_GFX950_OK;
    sequence *s = find(p, seq);
    if (s == NULL) st = FAIL_ARG("seq_truncate: no sequence %d", seq);
    else if (n_tokens < 0 || n_tokens > s->len) st = FAIL_ARG("seq_truncate: %d of %d positions", n_tokens, s->len);
    else {
        const int32_t keep = pages_for(p, n_tokens);
        while (s->n_pages > keep) give_page(p, s->page[--s->n_pages]);
        s->len = n_tokens;
    }
    pthread_mutex_unlock(&p->mtx);
    return st;
}

/* every one of n sequences there and named once (p->stamp is this call's) */
static int check_names(sllm_gfx950_pages *p, const int32_t *seqs, int32_t n, const char *who) {
    ++p->stamp;
    for (int32_t i = 0; i < n; ++i) {
        sequence *s = find(p, seqs[i]);
        if (s == NULL) return FAIL_ARG("%s: no sequence %d", who, seqs[i]);
        if (s->mark == p->stamp) return FAIL_ARG("%s: sequence %d twice", who, seqs[i]);
        s->mark = p->stamp;
    }
    return SLLM_GFX950_OK;
}

static int buffer_get(sllm_gfx950_pages *p, buffer *b, size_t dev_bytes, size_t pin_bytes);
static void buffer_put(sllm_gfx950_pages *p, buffer *b);

/* n copies in one launch, so that all are on their way or none: what a reorder writes may be
 * pages that it takes back where it fails. (n under ATTN_MAX_SEQS, a grid's most in y.) */
static int copies_at_once(sllm_gfx950_pages *p, const att_pair *pair, uint32_t n) {
    copies c;
    copies_start(&c, p);
    if (n <= ATT_PAIRS) {
        for (uint32_t i = 0; i < n; ++i) copies_add(&c, (int32_t) pair[i].src, (int32_t) pair[i].dst, (int32_t) pair[i].rows);
        return copies_flush(&c);
    }
    buffer b;
    int st = buffer_get(p, &b, n * sizeof *pair, n * sizeof *pair);
    if (st != SLLM_GFX950_OK) return st;
    memcpy(b.pin, pair, n * sizeof *pair);
    hipError_t e = hipMemcpyAsync(b.dev, b.pin, n * sizeof *pair, hipMemcpyHostToDevice, sllm_shim_stream());
    if (e == hipSuccess) e = hipEventRecord(b.sent, sllm_shim_stream());
    if (e != hipSuccess) {
        hipStreamSynchronize(sllm_shim_stream());
        buffer_drop(&b);
        return sllm_shim_hip_fail(e, "seq_reorder");
    }
    for (uint32_t i = 0; i < n; ++i) if (pair[i].rows > c.most) c.most = pair[i].rows;
    c.a.list = (const att_pair *) b.dev;
    c.a.n_pairs = n;
    st = copies_flush(&c);
    buffer_put(p, &b);
    return st;
}

static void hold_page(sllm_gfx950_pages *p, int32_t page) {      /* (one that may be free) */
    if (p->refs[page]++ == 0 && p->holds[page] == 0) --p->n_free;
}

/* The new pages of seqs[i]: its parent's, `was` their old tables (at[i] .. at[i + 1]); the page
 * that the parent ends in goes to keeper[parent] alone. hold: they are taken up, else given back. */
static void reorder_pages(sllm_gfx950_pages *p, const int32_t *parent, const int32_t *keeper, const int32_t *was, const int32_t *at,
                          const int32_t *len, int32_t i, int hold) {
    const int32_t q = parent[i], whole = len[q] >> p->page_shift, n = keeper[q] == i ? at[q + 1] - at[q] : whole;
    for (int32_t j = 0; j < n; ++j) {
        if (hold) hold_page(p, was[at[q] + j]);
        else give_page(p, was[at[q] + j]);
    }
}

int sllm_gfx950_seq_reorder(sllm_gfx950_pages *p, const int32_t *seqs, const int32_t *parent, int32_t n) {
    ATT_ON_DEVICE();
    if (p == NULL || n < 0 || (n > 0 && (seqs == NULL || parent == NULL))) return FAIL_ARG("seq_reorder: NULL or a count below 0");
    if (n > SLLM_GFX950_ATTN_MAX_SEQS) return FAIL_ARG("seq_reorder: %d sequences", n);
    for (int32_t i = 0; i < n; ++i) {
        if (parent[i] < 0 || parent[i] >= n) return FAIL_ARG("seq_reorder: sequence %d of %d goes on from %d", i, n, parent[i]);
    }
    int32_t *work = malloc(((size_t) n * 3 + 1) * sizeof *work), *was = NULL;
    att_pair *pairs = NULL;
    if (work == NULL) return FAIL_NOMEM("seq_reorder: %d sequences", n);
    int32_t *keeper = work, *len = work + n, *at = work + 2 * (size_t) n;
    pthread_mutex_lock(&p->mtx);
    int st = not_in_capture("seq_reorder");
    if (st == SLLM_GFX950_OK) st = check_names(p, seqs, n, "seq_reorder");
    int64_t total = 0, need = 0;
    if (st == SLLM_GFX950_OK) {
        for (int32_t i = 0; i < n; ++i) {
            keeper[i] = -1;
            len[i] = p->seq[seqs[i]].len;
            total += p->seq[seqs[i]].n_pages;
        }
        for (int32_t i = n - 1; i >= 0; --i) if (keeper[parent[i]] != parent[i]) keeper[parent[i]] = i;     /* itself, or the first */
        for (int32_t i = 0; i < n; ++i) need += keeper[parent[i]] != i && (len[parent[i]] & (p->d.page_tokens - 1)) != 0;
        if (total > INT32_MAX) st = FAIL_ARG("seq_reorder: too many pages");
        else if ((was = malloc((size_t) (total ? total : 1) * sizeof *was)) == NULL || (pairs = malloc((size_t) (need ? need : 1) * sizeof *pairs)) == NULL) {
            st = FAIL_NOMEM("seq_reorder: %lld pages", (long long) total);
        }
    }
    if (st == SLLM_GFX950_OK) {
        at[0] = 0;
        for (int32_t i = 0; i < n; ++i) {
            const sequence *s = &p->seq[seqs[i]];
            if (s->n_pages > 0) memcpy(was + at[i], s->page, (size_t) s->n_pages * sizeof *was);
            at[i + 1] = at[i] + s->n_pages;
        }
        for (int32_t i = 0; i < n && st == SLLM_GFX950_OK; ++i) {
            if (!reserve(&p->seq[seqs[i]], at[parent[i] + 1] - at[parent[i]])) st = FAIL_NOMEM("seq_reorder: page table");
        }
    }
    if (st == SLLM_GFX950_OK) {
        /* what is held on, then what nobody holds any more: that may be enough for the copies.
         * (What a copy reads is held, so no copy writes it.) */
        for (int32_t i = 0; i < n; ++i) if (parent[i] != i) reorder_pages(p, parent, keeper, was, at, len, i, 1);
        for (int32_t i = 0; i < n; ++i) if (parent[i] != i) for (int32_t j = at[i]; j < at[i + 1]; ++j) give_page(p, was[j]);
        int32_t got = 0;
        if (need > p->n_free) st = FAIL_NOMEM("seq_reorder: %lld pages wanted, %d free", (long long) need, p->n_free);
        else {
            uint32_t n_pairs = 0;
            for (; got < n; ++got) {
                const int32_t q = parent[got], whole = len[q] >> p->page_shift, rows = len[q] & (p->d.page_tokens - 1);
                sequence *s = &p->seq[seqs[got]];
                if (q == got) continue;
                s->n_pages = at[q + 1] - at[q];
                s->len = len[q];
                if (s->n_pages > 0) memcpy(s->page, was + at[q], (size_t) s->n_pages * sizeof *was);
                if (rows && keeper[q] != got) {
                    s->page[whole] = take_page(p);
                    pairs[n_pairs++] = (att_pair) { (uint32_t) was[at[q] + whole], (uint32_t) s->page[whole], (uint32_t) rows };
                }
            }
            st = copies_at_once(p, pairs, n_pairs);
        }
        if (st != SLLM_GFX950_OK) {                      /* as it was */
            for (int32_t i = 0; i < got; ++i) {
                const int32_t q = parent[i], whole = len[q] >> p->page_shift;
                if (q != i && keeper[q] != i && (len[q] & (p->d.page_tokens - 1)) != 0) give_page(p, p->seq[seqs[i]].page[whole]);
            }
            for (int32_t i = 0; i < n; ++i) if (parent[i] != i) for (int32_t j = at[i]; j < at[i + 1]; ++j) hold_page(p, was[j]);
            for (int32_t i = 0; i < n; ++i) if (parent[i] != i) reorder_pages(p, parent, keeper, was, at, len, i, 0);
            for (int32_t i = 0; i < got; ++i) {
                sequence *s = &p->seq[seqs[i]];
                if (parent[i] == i) continue;
                s->n_pages = at[i + 1] - at[i];
                s->len = len[i];
                if (s->n_pages > 0) memcpy(s->page, was + at[i], (size_t) s->n_pages * sizeof *was);
            }
        }
    }
    pthread_mutex_unlock(&p->mtx);
    free(work);
    free(was);
    free(pairs);
    return st;
}

int sllm_gfx950_seq_free(sllm_gfx950_pages *p, const int32_t *seqs, int32_t n) {
    ATT_NEED_OPEN();
    if (p == NULL || n < 0 || (n > 0 && seqs == NULL)) return FAIL_ARG("seq_free: NULL or a count below 0");
    pthread_mutex_lock(&p->mtx);
    const int st = check_names(p, seqs, n, "seq_free");
    for (int32_t i = 0; i < n && st == SLLM_GFX950_OK; ++i) end_sequence(p, seqs[i]);
    pthread_mutex_unlock(&p->mtx);
    return st;
}

int32_t sllm_gfx950_seq_len(sllm_gfx950_pages *p, int32_t seq) {
    ATT_NEED_OPEN();
    if (p == NULL) return FAIL_ARG("seq_len: NULL");
    pthread_mutex_lock(&p->mtx);
    const sequence *s = find(p, seq);
    const int32_t len = s ? s->len : FAIL_ARG("seq_len: no sequence %d", seq);
    pthread_mutex_unlock(&p->mtx);
    return len;
}

int32_t sllm_gfx950_seq_tables(sllm_gfx950_pages *p, const int32_t *seqs, int32_t n, int32_t *pages, int32_t cap) {
    ATT_NEED_OPEN();
    if (p == NULL || n < 0 || (n > 0 && seqs == NULL) || cap < 0 || (cap > 0 && pages == NULL)) return FAIL_ARG("seq_tables: NULL or a count below 0");
    pthread_mutex_lock(&p->mtx);
    int64_t total = 0;
    for (int32_t i = 0; i < n && total >= 0; ++i) {
        const sequence *s = find(p, seqs[i]);
        total = s ? total + s->n_pages : FAIL_ARG("seq_tables: no sequence %d", seqs[i]);
    }
    if (total > INT32_MAX) total = FAIL_ARG("seq_tables: too many pages");
    if (total >= 0 && total <= cap) {
        for (int32_t i = 0; i < n; ++i) {
            const sequence *s = &p->seq[seqs[i]];
            if (s->n_pages > 0) memcpy(pages, s->page, (size_t) s->n_pages * sizeof *pages);
            pages += s->n_pages;
        }
    }
    pthread_mutex_unlock(&p->mtx);
    return (int32_t) total;
}

int sllm_gfx950_pages_compact(sllm_gfx950_pages *p, int32_t *n_moved) {
    ATT_ON_DEVICE();
    if (n_moved) *n_moved = 0;
    if (p == NULL) return FAIL_ARG("pages_compact: NULL");
    pthread_mutex_lock(&p->mtx);
    int st = not_in_capture("pages_compact");
    const int32_t n_used = p->d.n_pages - p->n_free;
    /* where each page above n_used goes */
    int32_t *to = NULL, moved = 0;
    if (st != SLLM_GFX950_OK) { }
    else if (p->open > 0) st = FAIL_ARG("pages_compact: %d batches are open", p->open);
    else if ((to = malloc((size_t) p->d.n_pages * sizeof *to)) == NULL) st = FAIL_NOMEM("pages_compact: %d pages", p->d.n_pages);
    if (st == SLLM_GFX950_OK) {
        copies c;
        copies_start(&c, p);
        int32_t hole = 0;
        for (int32_t i = n_used; i < p->d.n_pages; ++i) {
            if (p->refs[i] == 0) continue;
            while (p->refs[hole] != 0) ++hole;           /* (as many holes below n_used as pages above it) */
            to[i] = hole++;
            ++moved;
            copies_add(&c, i, to[i], p->d.page_tokens);
        }
        st = copies_flush(&c);
    }
    if (st == SLLM_GFX950_OK && moved > 0) {
        for (int32_t i = 0; i < p->n_seq; ++i) {
            sequence *s = &p->seq[i];
            for (int32_t j = 0; j < s->n_pages; ++j) if (s->page[j] >= n_used) s->page[j] = to[s->page[j]];
        }
        for (int32_t i = n_used; i < p->d.n_pages; ++i) {
            if (p->refs[i] == 0) continue;
            p->refs[to[i]] = p->refs[i];
            p->refs[i] = 0;
        }
        p->low = n_used;
    }
    free(to);
    pthread_mutex_unlock(&p->mtx);
    if (st == SLLM_GFX950_OK && n_moved) *n_moved = moved;
    return st;
}

/* ------------------------------------------------------------------ */
/* a batch                                                             */
/* ------------------------------------------------------------------ */

/* workgroups of a launch: their threads fit 32 bits */
#define MAX_ITEMS ((size_t) 1 << 23)

typedef struct items { att_item *v; size_t n, cap; } items;

static att_item *items_add(items *x) {
    if (x->n == x->cap) {
        const size_t cap = x->cap ? x->cap * 2 : 256;
        att_item *v = realloc(x->v, cap * sizeof *v);
        if (v == NULL) return NULL;
        x->v = v;
        x->cap = cap;
    }
    return &x->v[x->n++];
}

struct sllm_gfx950_batch {
    sllm_gfx950_pages *p;
    int32_t   n_head, act, pair;
    int32_t   n_seq;
    int64_t   n_pos;                 /* positions of its sequences, old and new */
    uint32_t  n_tok, n_pages;
    uint32_t  n_items;
    uint32_t  join;                  /* the most partial results that a row has */
    buffer    buf;
    size_t    off_tables, off_list, off_toks, off_segs, off_seqs, off_part_o, off_part_ml;     /* (its items are at 0) */
    int32_t  *held;                  /* the pages it holds */
    int32_t   n_held;
};

/* a run of keys and the tokens of the sequences that read it (order[lo .. hi)) */
typedef struct segment {
    int32_t  lo, hi;
    int32_t  page0, n_keys;          /* from page page0 of each of their tables */
    uint32_t n_tok, list, part0, n_split, split;
    uint32_t mode;
} segment;

typedef struct plan {
    const sllm_gfx950_pages *p;
    const int32_t *seqs, *n_new;
    int32_t  *order, n_order;        /* sequences with new tokens, like tables side by side */
    int32_t  *common;                /* whole pages that order[i] shares with order[i - 1] */
    uint32_t *tok0, *table;          /* of sequence i: its first row, where its page numbers start */
    segment  *seg;
    int32_t   n_seg;
    uint32_t  n_list;
} plan;

/* fewer shared keys than this are read by each sequence for itself: a segment
 * of their own costs a row a partial result more */
#define MIN_SHARED 128

/* The runs of order[lo .. hi), which share their pages below `from`. At most two
 * per sequence: one of its own, and one at each place where it parts from its
 * neighbour. A range is gone through once for each depth in pages at which some of
 * it part, so a sequence no more often than it has shared pages: less work than
 * copying its page numbers is, also for a chain of forks. */
static void find_segments(plan *x, int32_t lo, int32_t hi, int32_t from) {
    while (hi - lo > 1) {
        int32_t common = INT32_MAX;
        for (int32_t i = lo + 1; i < hi; ++i) if (x->common[i] < common) common = x->common[i];
        if (((int64_t) (common - from) << x->p->page_shift) >= MIN_SHARED) {
            segment *s = &x->seg[x->n_seg++];
            *s = (segment) { .lo = lo, .hi = hi, .page0 = from, .n_keys = (common - from) << x->p->page_shift };
            from = common;
        }
        /* the groups that go on together beyond `common`: the largest in this
         * loop, so that calls go no deeper than the logarithm of their number */
        int32_t big_lo = lo, big_hi = lo, start = lo;
        for (int32_t i = lo + 1; i <= hi; ++i) {
            if (i < hi && x->common[i] != common) continue;
            if (i - start > big_hi - big_lo) {
                big_lo = start;
                big_hi = i;
            }
            start = i;
        }
        start = lo;
        for (int32_t i = lo + 1; i <= hi; ++i) {
            if (i < hi && x->common[i] != common) continue;
            if (start != big_lo) find_segments(x, start, i, from);
            start = i;
        }
        lo = big_lo;
        hi = big_hi;
    }
    const sequence *s = &x->p->seq[x->seqs[x->order[lo]]];
    x->seg[x->n_seg++] = (segment) { .lo = lo, .hi = hi, .page0 = from, .n_keys = s->len - (from << x->p->page_shift) };
}

static __thread const plan *g_sort;                      /* for qsort */

static int by_table(const void *a, const void *b) {
    const int32_t ia = *(const int32_t *) a, ib = *(const int32_t *) b;
    const sequence *s = &g_sort->p->seq[g_sort->seqs[ia]], *t = &g_sort->p->seq[g_sort->seqs[ib]];
    const int32_t n = s->n_pages < t->n_pages ? s->n_pages : t->n_pages;
    for (int32_t i = 0; i < n; ++i) if (s->page[i] != t->page[i]) return s->page[i] < t->page[i] ? -1 : 1;
    return ia < ib ? -1 : ia > ib;
}

static const uint32_t k_rows[] = { ATT_FEW_ROWS, ATT_HALF_ROWS, ATT_MANY_ROWS };      /* by mode */

/* A segment's rows: f32 takes two tiles of few before half of many (8 sequences
 * behind 4096 shared positions, 32 rows: 18.7 us against 24.8), 16 bits one (12.6
 * for half of many, 13.0 for two of few). */
static uint32_t mode_of(uint32_t rows, int32_t dtype, int32_t act) {
    if (held8(dtype) && act == SLLM_GFX950_F32) return rows <= ATT_FEW_ROWS ? ATT_FEW : ATT_HALF;    /* (held8_body) */
    const uint32_t few = dtype == SLLM_GFX950_F32 ? 2 * ATT_FEW_ROWS : ATT_FEW_ROWS;
    return rows <= few ? ATT_FEW : rows <= ATT_HALF_ROWS ? ATT_HALF : ATT_MANY;
}

/*
 * A split's keys. Few rows: the work is cut so that 25/32 of the CUs have a
 * workgroup each, or where that makes splits of over LONG_SPLIT keys, so that
 * all have two, which the memory wants; but never below what one step of the
 * four waves takes. Many rows: 25/32 of the CUs, at least 128 keys: their
 * partial results weigh more. Measured with head_dim 128 over splits of 64 to
 * 2048 keys (us, at the rule and at the best of them): one sequence of 8192
 * positions, bf16 12.1 / 12.0, 64 of about 1000 28.0 / 26.9, 8 of 4096 to 65536
 * 62.8 / 62.8; 64 behind 4096 shared ones 22.8 / 22.5, behind 16384 36.4 / 36.1.
 */
#define SPLIT_KEYS 64u
#define LONG_SPLIT 512u

static uint32_t seg_tiles(const segment *s, uint32_t group) {
    return (s->n_tok * group + k_rows[s->mode] - 1) / k_rows[s->mode];
}

/*
 * 8 bits: where tiles of 128 rows have fewer keys than this a CU, they are made two of 64:
 * twice the workgroups, but each key is turned into bf16 twice as often (and weights of bf16 rows are
 * of 16 bits, not 8). us, 64 rows / 128, 64 sequences behind a shared prefix, 20 heads over 5, by keys a CU:
 *
 *                       160           195           234           273           312           371           430
 *   bf16 128 int8   25.7 / 25.9   27.6 / 27.9   30.2 / 29.0   31.9 / 30.5   35.1 / 31.9   38.6 / 33.1   43.5 / 34.4
 *   bf16 128 e4m3   24.0 / 25.2   25.5 / 27.1   27.7 / 28.2   29.2 / 29.4   31.6 / 30.3   34.8 / 31.5   39.1 / 32.8
 *   f16  128 int8   27.0 / 29.6   28.8 / 32.6   31.7 / 34.5   33.3 / 36.5   36.9 / 38.3   40.6 / 40.6   45.6 / 42.9
 *   f16  128 e4m3   25.4 / 28.2   27.0 / 31.2   29.6 / 32.8   30.6 / 34.4   33.5 / 36.6   36.9 / 38.2   41.3 / 40.2
 *   bf16  64 int8   20.7 / 18.8   22.2 / 20.4   25.5 / 21.6   26.7 / 23.2   29.5 / 24.6   32.5 / 26.5   36.4 / 28.2
 *   bf16  64 e4m3   18.7 / 17.5   19.9 / 19.4   22.3 / 20.3   23.5 / 21.7   25.6 / 22.7   27.9 / 24.2   31.0 / 25.7
 *   f16   64 int8   21.3 / 20.8   22.8 / 22.5   26.1 / 24.0   27.5 / 25.9   30.5 / 27.4   33.4 / 29.7   37.5 / 31.8
 *   f16   64 e4m3   20.1 / 19.8   21.4 / 21.4   24.1 / 22.7   25.4 / 24.2   27.9 / 25.5   30.4 / 27.4   34.0 / 29.3
 *
 * and of few keys, 128 new positions behind 900 (70 a CU) bf16 int8 18.1 / 20.6, 14.7 / 15.4 with heads of 64; drafts of 5
 * behind 1000, 32 heads over 8 (150) 28.7 / 29.5 and 25.0 / 24.5, f16 30.3 / 36.7 and 25.8 / 27.3. int8 and e4m3 cross near
 * enough to each other to have one border.
 */
static uint32_t held8_half_keys(int32_t head_dim, int32_t act) {
    if (head_dim <= 64) return act == SLLM_GFX950_F16 ? 170u : 130u;
    return act == SLLM_GFX950_F16 ? 380u : 220u;
}

static uint32_t split_keys(const plan *x, uint32_t group, uint32_t n_head_kv, int many, uint32_t step) {
    uint64_t work = 0;
    for (int32_t i = 0; i < x->n_seg; ++i) {
        const segment *s = &x->seg[i];
        if ((s->mode >= ATT_HALF) == many) work += (uint64_t) seg_tiles(s, group) * (uint64_t) s->n_keys * n_head_kv;
    }
    const uint64_t cu = (uint64_t) sllm_shim_cu();
    uint64_t keys = work / (cu * 25 / 32 + 1) + 1;
    if (!many && keys > LONG_SPLIT) {
        keys = work / (2 * cu) * 17 / 16;                /* (more than an even share: splits are not all of one length) */
        if (keys < LONG_SPLIT) keys = LONG_SPLIT;
    }
    const uint64_t least = many ? 128 : 4 * step;
    if (keys < least) keys = least;
    keys = (keys + SPLIT_KEYS - 1) / SPLIT_KEYS * SPLIT_KEYS;
    return keys > (1u << 28) ? 1u << 28 : (uint32_t) keys;
}

static uint64_t item_keys(const att_item *a) { return a->key1 > a->key0 ? a->key1 - a->key0 : 0; }

/* Workgroups start in this order: many rows first, then the longest, so that what
 * starts last is short. (Giving each XCD, workgroup i % 8, sequences of its own, so
 * that its L2 holds their keys, gained 2 % for 24 prompts of up to 2048 rows, but its
 * uneven ends lost 13 % for four and 40 % for 64 sequences behind a shared prefix.) */
static int by_work(const void *a, const void *b) {
    const att_item *x = a, *y = b;
    if (x->mode != y->mode) return x->mode > y->mode ? -1 : 1;
    if (item_keys(x) != item_keys(y)) return item_keys(x) > item_keys(y) ? -1 : 1;
    return x->order < y->order ? -1 : x->order > y->order;
}

static void order_work(items *x) {
    for (size_t i = 0; i < x->n; ++i) x->v[i].order = (uint32_t) i;
    if (x->n > 0) qsort(x->v, x->n, sizeof *x->v, by_work);
}

static size_t align256(size_t x) { return (x + 255) & ~(size_t) 255; }

static int buffer_get(sllm_gfx950_pages *p, buffer *b, size_t dev_bytes, size_t pin_bytes) {
    memset(b, 0, sizeof *b);
    for (int i = 0; i < p->n_kept; ++i) {
        if (p->kept[i].dev_bytes >= dev_bytes && p->kept[i].pin_bytes >= pin_bytes) {
            *b = p->kept[i];
            p->kept[i] = p->kept[--p->n_kept];
            const hipError_t e = hipEventSynchronize(b->sent);
            if (e == hipSuccess) return SLLM_GFX950_OK;
            buffer_drop(b);
            return sllm_shim_hip_fail(e, "hipEventSynchronize(batch)");
        }
    }
    /* a quarter more than asked for: the next steps' tables are a little longer */
    dev_bytes += dev_bytes / 4;
    pin_bytes += pin_bytes / 4;
    hipError_t e = hipMalloc((void **) &b->dev, dev_bytes);
    const char *what = "hipMalloc(batch)";
    if (e == hipSuccess) { e = hipHostMalloc((void **) &b->pin, pin_bytes, hipHostMallocDefault); what = "hipHostMalloc(batch)"; }
    if (e == hipSuccess) { e = hipEventCreateWithFlags(&b->sent, hipEventDisableTiming); what = "hipEventCreate(batch)"; }
    b->dev_bytes = dev_bytes;
    b->pin_bytes = pin_bytes;
    if (e == hipSuccess) return SLLM_GFX950_OK;
    buffer_drop(b);
    return sllm_shim_hip_fail(e, what);
}

static void buffer_put(sllm_gfx950_pages *p, buffer *b) {
    if (b->dev == NULL) return;
    if (p->n_kept == KEPT_BUFFERS) {                     /* the smallest goes */
        int least = 0;
        for (int i = 1; i < p->n_kept; ++i) if (p->kept[i].dev_bytes < p->kept[least].dev_bytes) least = i;
        if (p->kept[least].dev_bytes < b->dev_bytes) {
            const buffer t = p->kept[least];
            p->kept[least] = *b;
            *b = t;
        }
        release(b, 1);
        return;
    }
    p->kept[p->n_kept++] = *b;
    memset(b, 0, sizeof *b);
}

/* The step's segments, work items and tables into the batch's buffer. */
static int lay_out(sllm_gfx950_batch *b, plan *x, int32_t n, const int32_t *len0) {
    sllm_gfx950_pages *p = b->p;
    const uint32_t kv = (uint32_t) p->d.n_head_kv, group = (uint32_t) b->n_head / kv;
    const uint32_t hd_pad = p->d.head_dim <= 64 ? 64 : 128;
    items it = { 0 };
    int st = SLLM_GFX950_OK;

    /* like tables side by side, and how far each goes with the one before it:
     * in whole pages of positions that were there before the step */
    for (int32_t i = 0; i < n; ++i) if (x->n_new[i] > 0) x->order[x->n_order++] = i;
    g_sort = x;
    qsort(x->order, (size_t) x->n_order, sizeof *x->order, by_table);
    for (int32_t i = 1; i < x->n_order; ++i) {
        const int32_t ia = x->order[i - 1], ib = x->order[i];
        const sequence *s = &p->seq[x->seqs[ia]], *t = &p->seq[x->seqs[ib]];
        int32_t most = (len0[ia] < len0[ib] ? len0[ia] : len0[ib]) >> p->page_shift, c = 0;
        while (c < most && s->page[c] == t->page[c]) ++c;
        x->common[i] = c;
    }
    if (x->n_order > 0) find_segments(x, 0, x->n_order, 0);
    uint64_t n_list = 0, many = 0;
    for (int32_t i = 0; i < x->n_seg; ++i) {
        segment *s = &x->seg[i];
        for (int32_t j = s->lo; j < s->hi; ++j) s->n_tok += (uint32_t) x->n_new[x->order[j]];
        s->list = ATT_TOKENS;
        if (s->hi - s->lo > 1) { s->list = (uint32_t) n_list; n_list += s->n_tok; }
        s->mode = mode_of(s->n_tok * group, p->d.dtype, b->act);
        if (s->mode == ATT_MANY) many += (uint64_t) seg_tiles(s, group) * (uint64_t) s->n_keys * kv;
    }
    if (held8(p->d.dtype) && many < (uint64_t) sllm_shim_cu() * held8_half_keys(p->d.head_dim, b->act)) {
        for (int32_t i = 0; i < x->n_seg; ++i) if (x->seg[i].mode == ATT_MANY) x->seg[i].mode = ATT_HALF;
    }
    /* segments of each sequence, and those with one part alone */
    uint32_t *seg_count = calloc((size_t) n + 1, sizeof *seg_count), *seg_at = calloc((size_t) n + 1, sizeof *seg_at);
    uint32_t *parts = calloc((size_t) n + 1, sizeof *parts);
    uint8_t *alone = calloc((size_t) n + 1, 1);
    if (seg_count == NULL || seg_at == NULL || parts == NULL || alone == NULL) { st = FAIL_NOMEM("batch_create: tables"); goto out; }
    const uint32_t step = p->d.dtype == SLLM_GFX950_F32 ? 16 : 32;
    const uint32_t split[2] = { split_keys(x, group, kv, 0, step), split_keys(x, group, kv, 1, step) };
    uint64_t n_part = 0, n_segs = 0, n_pages = 0;
    for (int32_t i = 0; i < x->n_seg; ++i) {
        segment *s = &x->seg[i];
        s->n_split = ((uint32_t) s->n_keys + split[s->mode >= ATT_HALF] - 1) / split[s->mode >= ATT_HALF];
        s->split = ((uint32_t) s->n_keys + s->n_split - 1) / s->n_split;        /* evenly */
        s->split = (s->split + SPLIT_KEYS - 1) / SPLIT_KEYS * SPLIT_KEYS;
        s->n_split = ((uint32_t) s->n_keys + s->split - 1) / s->split;
        for (int32_t j = s->lo; j < s->hi; ++j) ++seg_count[x->order[j]];
    }
    for (int32_t i = 0; i < x->n_seg; ++i) {
        segment *s = &x->seg[i];
        const int32_t q = x->order[s->lo];
        alone[q] = s->hi - s->lo == 1 && seg_count[q] == 1 && s->n_split == 1;
        if (alone[q]) { seg_count[q] = 0; continue; }
        s->part0 = (uint32_t) n_part;
        n_part += (uint64_t) kv * s->n_split * s->n_tok * group;
        if (n_part > 0xfffffff0ull) { st = FAIL_ARG("batch_create: too many rows and splits"); goto out; }
    }
    for (int32_t i = 0; i < n; ++i) {
        seg_at[i] = (uint32_t) n_segs;
        n_segs += seg_count[i];
        seg_count[i] = 0;
        n_pages += (uint64_t) p->seq[x->seqs[i]].n_pages;
    }
    for (int32_t i = 0; i < x->n_seg; ++i) {
        const segment *s = &x->seg[i];
        for (int32_t j = s->lo; j < s->hi; ++j) if (!alone[x->order[j]]) parts[x->order[j]] += s->n_split;
    }
    b->join = 0;
    for (int32_t i = 0; i < n; ++i) if (parts[i] > b->join) b->join = parts[i];

    /* the work */
    for (int32_t i = 0; i < x->n_seg && st == SLLM_GFX950_OK; ++i) {
        const segment *s = &x->seg[i];
        const int32_t q = x->order[s->lo];
        const uint32_t rows = s->n_tok * group, tile = k_rows[s->mode];
        const int own = s->hi - s->lo == 1;
        const int32_t vis0 = own ? len0[q] - (s->page0 << p->page_shift) + 1 : ATT_SEE_ALL;
        for (uint32_t hk = 0; hk < kv * s->n_split && st == SLLM_GFX950_OK; ++hk) {
            const uint32_t h = hk / s->n_split, k = hk % s->n_split, key0 = k * s->split;
            for (uint32_t r = 0; r < rows; r += tile) {
                const uint32_t nr = rows - r < tile ? rows - r : tile;
                const uint64_t sees = (uint64_t) vis0 + (r + nr - 1) / group;
                uint32_t key1 = (uint32_t) s->n_keys < key0 + s->split ? (uint32_t) s->n_keys : key0 + s->split;
                if (key1 > sees) key1 = (uint32_t) sees;
                att_item *a = items_add(&it);
                if (a == NULL) { st = FAIL_NOMEM("batch_create: work items"); break; }
                *a = (att_item) { r / group, nr, own ? x->tok0[q] : 0, s->list, vis0, key0, key1, x->table[q] + (uint32_t) s->page0, h,
                                  alone[q] ? ATT_DIRECT : s->part0 + hk * rows + r, (uint16_t) s->mode, (uint16_t) (r % group), 0 };
            }
        }
    }
    if (st == SLLM_GFX950_OK && it.n > MAX_ITEMS) st = FAIL_ARG("batch_create: too much work for a launch");
    if (st != SLLM_GFX950_OK) goto out;
    order_work(&it);

    b->n_items = (uint32_t) it.n;
    size_t at = align256(it.n * sizeof(att_item));
    b->off_tables = at;  at = align256(at + n_pages * 4);
    b->off_list = at;    at = align256(at + n_list * 4);
    b->off_toks = at;    at = align256(at + (size_t) b->n_tok * sizeof(att_tok));
    b->off_segs = at;    at = align256(at + n_segs * sizeof(att_seg));
    b->off_seqs = at;    at = align256(at + ((size_t) n + 1) * sizeof(att_seq));
    const size_t sent = at;
    b->off_part_ml = at; at = align256(at + n_part * 8);
    b->off_part_o = at;  at = align256(at + n_part * hd_pad * 4);
    if ((st = buffer_get(p, &b->buf, at + 256, sent + 256)) != SLLM_GFX950_OK) goto out;

    uint8_t *to = b->buf.pin;
    if (it.n > 0) memcpy(to, it.v, it.n * sizeof(att_item));
    uint32_t *tables = (uint32_t *) (to + b->off_tables), *list = (uint32_t *) (to + b->off_list);
    att_tok *toks = (att_tok *) (to + b->off_toks);
    att_seg *segs = (att_seg *) (to + b->off_segs);
    for (int32_t i = 0; i < x->n_seg; ++i) {
        const segment *s = &x->seg[i];
        uint32_t t = 0;
        for (int32_t j = s->lo; j < s->hi; ++j) {
            const int32_t q = x->order[j];
            if (!alone[q]) segs[seg_at[q] + seg_count[q]++] = (att_seg) { s->part0, s->n_tok * group, s->n_split, t * group };
            for (int32_t k = 0; k < x->n_new[q] && s->list != ATT_TOKENS; ++k) list[s->list + t + (uint32_t) k] = x->tok0[q] + (uint32_t) k;
            t += (uint32_t) x->n_new[q];
        }
    }
    att_seq *seqs = (att_seq *) (to + b->off_seqs);
    uint64_t row0 = 0;
    for (int32_t i = 0; i < n; ++i) {
        seqs[i] = (att_seq) { x->table[i], (uint32_t) row0 };        /* (past 32 bits: batch_read refuses) */
        row0 += (uint64_t) p->seq[x->seqs[i]].len;
    }
    seqs[n] = (att_seq) { (uint32_t) n_pages, (uint32_t) row0 };
    b->n_seq = n;
    b->n_pos = (int64_t) row0;
    b->n_pages = (uint32_t) n_pages;
    for (int32_t i = 0; i < n; ++i) {
        const sequence *s = &p->seq[x->seqs[i]];
        if (s->n_pages > 0) memcpy(tables + x->table[i], s->page, (size_t) s->n_pages * 4);
        for (int32_t t = 0; t < x->n_new[i]; ++t) {
            toks[x->tok0[i] + (uint32_t) t] = (att_tok) { x->table[i], (uint32_t) (len0[i] + t), seg_at[i], seg_count[i], (uint32_t) t, { 0 } };
        }
    }
    if (sent > 0) {
        hipError_t e = hipMemcpyAsync(b->buf.dev, b->buf.pin, sent, hipMemcpyHostToDevice, sllm_shim_stream());
        if (e == hipSuccess) e = hipEventRecord(b->buf.sent, sllm_shim_stream());
        if (e != hipSuccess) {
            hipStreamSynchronize(sllm_shim_stream());
            buffer_drop(&b->buf);
            st = sllm_shim_hip_fail(e, "batch_create");
        }
    }
out:
    free(it.v);
    free(seg_count);
    free(seg_at);
    free(parts);
    free(alone);
    return st;
}

int sllm_gfx950_batch_create(sllm_gfx950_pages *p, const int32_t *seqs, const int32_t *n_new, int32_t n, int32_t n_head,
                             int32_t act_dtype, sllm_gfx950_batch **out) {
    ATT_ON_DEVICE();
    if (out == NULL) return FAIL_ARG("batch_create: NULL out");
    *out = NULL;
    if (p == NULL || n < 0 || n > SLLM_GFX950_ATTN_MAX_SEQS || (n > 0 && (seqs == NULL || n_new == NULL))) {
        return FAIL_ARG("batch_create: NULL, or %d sequences", n);
    }
    if (bad_heads(n_head, p->d.n_head_kv, p->d.head_dim)) return FAIL_ARG("batch_create: %d query heads over %d", n_head, p->d.n_head_kv);
    const int pair = bad_type(act_dtype) ? -1 : type_pair(act_dtype, p->d.dtype);
    if (pair < 0) return FAIL_ARG("batch_create: rows of type %d over a cache of type %d", act_dtype, p->d.dtype);
    int st = not_in_capture("batch_create");
    if (st != SLLM_GFX950_OK) return st;

    const size_t n1 = (size_t) n + 1;
    sllm_gfx950_batch *b = calloc(1, sizeof *b);
    int32_t *work = malloc(n1 * 5 * sizeof *work);
    uint32_t *uwork = malloc(n1 * 2 * sizeof *uwork);
    segment *seg = calloc(n1 * 2, sizeof *seg);
    plan x = { .p = p, .seqs = seqs, .n_new = n_new, .seg = seg };
    if (b == NULL || work == NULL || uwork == NULL || seg == NULL) {
        st = FAIL_NOMEM("batch_create: %d sequences", n);
        goto out;
    }
    int32_t *len0 = work, *pages0 = work + n1, *last0 = work + 2 * n1;
    x.order = work + 3 * n1;
    x.common = work + 4 * n1;
    x.tok0 = uwork;
    x.table = uwork + n1;
    b->p = p;
    b->n_head = n_head;
    b->act = act_dtype;
    b->pair = pair;

    pthread_mutex_lock(&p->mtx);
    int64_t want = 0, tokens = 0, held = 0;
    st = check_names(p, seqs, n, "batch_create");
    for (int32_t i = 0; i < n && st == SLLM_GFX950_OK; ++i) {
        sequence *s = &p->seq[seqs[i]];
        if (n_new[i] < 0 || (int64_t) s->len + n_new[i] > SLLM_GFX950_ATTN_MAX_LEN) {
            st = FAIL_ARG("batch_create: %d new positions for sequence %d of %d", n_new[i], seqs[i], s->len);
            break;
        }
        const int32_t pages = pages_for(p, s->len + n_new[i]);
        const int own_last = s->len % p->d.page_tokens == 0 || p->refs[s->page[s->n_pages - 1]] == 1 || n_new[i] == 0;
        want += pages - s->n_pages + !own_last;
        x.tok0[i] = (uint32_t) tokens;
        x.table[i] = (uint32_t) held;
        tokens += n_new[i];
        held += pages;
        len0[i] = s->len;
        pages0[i] = s->n_pages;
        last0[i] = own_last ? -1 : s->page[s->n_pages - 1];
        if (tokens > SLLM_GFX950_ATTN_MAX_TOKENS || held > INT32_MAX) st = FAIL_ARG("batch_create: too many new positions or pages");
        else if (!reserve(s, pages)) st = FAIL_NOMEM("batch_create: page table");
    }
    if (st == SLLM_GFX950_OK && tokens * n_head > SLLM_GFX950_ATTN_MAX_ROWS) st = FAIL_ARG("batch_create: too many rows");
    if (st == SLLM_GFX950_OK && want > p->n_free) st = FAIL_NOMEM("batch_create: %lld pages wanted, %d free", (long long) want, p->n_free);
    if (st == SLLM_GFX950_OK && (b->held = malloc((size_t) (held ? held : 1) * sizeof *b->held)) == NULL) st = FAIL_NOMEM("batch_create: pages held");
    if (st == SLLM_GFX950_OK) {
        copies c;
        copies_start(&c, p);
        b->n_tok = (uint32_t) tokens;
        for (int32_t i = 0; i < n; ++i) {
            sequence *s = &p->seq[seqs[i]];
            if (last0[i] >= 0) {                         /* it would write into a page that others hold */
                s->page[s->n_pages - 1] = take_page(p);
                copies_add(&c, last0[i], s->page[s->n_pages - 1], s->len % p->d.page_tokens);
            }
            s->len += n_new[i];
            const int32_t pages = pages_for(p, s->len);
            while (s->n_pages < pages) s->page[s->n_pages++] = take_page(p);
        }
        st = copies_flush(&c);
        if (st == SLLM_GFX950_OK) st = lay_out(b, &x, n, len0);
        for (int32_t i = 0; i < n; ++i) {
            sequence *s = &p->seq[seqs[i]];
            if (st != SLLM_GFX950_OK) {                  /* as it was */
                while (s->n_pages > pages0[i]) give_page(p, s->page[--s->n_pages]);
                if (last0[i] >= 0) {
                    give_page(p, s->page[s->n_pages - 1]);
                    s->page[s->n_pages - 1] = last0[i];
                }
                s->len = len0[i];
                continue;
            }
            if (last0[i] >= 0) give_page(p, last0[i]);
            for (int32_t j = 0; j < s->n_pages; ++j) {
                ++p->holds[s->page[j]];
                b->held[b->n_held++] = s->page[j];
            }
        }
        if (st == SLLM_GFX950_OK) ++p->open;
    }
    pthread_mutex_unlock(&p->mtx);
out:
    free(work);
    free(uwork);
    free(seg);
    if (st != SLLM_GFX950_OK) {
        if (b != NULL) free(b->held);
        free(b);
        return st;
    }
    *out = b;
    return SLLM_GFX950_OK;
}

void sllm_gfx950_batch_destroy(sllm_gfx950_batch *b) {
    if (b == NULL) return;
    sllm_gfx950_pages *p = b->p;
    pthread_mutex_lock(&p->mtx);
    for (int32_t i = 0; i < b->n_held; ++i) {
        --p->holds[b->held[i]];
        maybe_free(p, b->held[i]);
    }
    buffer_put(p, &b->buf);
    const int last = --p->open == 0 && p->gone;
    pthread_mutex_unlock(&p->mtx);
    if (last) pages_drop(p);
    free(b->held);
    free(b);
}

int32_t sllm_gfx950_batch_rows(const sllm_gfx950_batch *b) { return b ? (int32_t) b->n_tok : 0; }

/* n rows of `row` bytes, `tok` bytes apart */
typedef struct rows_at { const void *p; uint64_t tok, row; int64_t n; } rows_at;

/* whether any of their bytes are the same, as far as can be told from their ends and, where
 * they are equally far apart, from their places between */
static int overlap(const rows_at *a, const rows_at *b) {
    if (a->p == NULL || b->p == NULL || a->n == 0 || b->n == 0) return 0;
    const uint64_t x = (uint64_t) (uintptr_t) a->p, y = (uint64_t) (uintptr_t) b->p;
    if (x + (uint64_t) (a->n - 1) * a->tok + a->row <= y || y + (uint64_t) (b->n - 1) * b->tok + b->row <= x) return 0;
    if (a->tok != b->tok && a->n > 1 && b->n > 1) return 1;
    const uint64_t tok = a->n > 1 ? a->tok : b->tok, off = x < y ? (y - x) % tok : (tok - (x - y) % tok) % tok;      /* of b behind a row of a */
    return off < a->row || off + b->row > tok;
}

/* Waves of a CU that rows are spread over before a wave takes more of a token's (us at 16 / 32 /
 * 64: 4099 tokens of 40 heads of 96 17.4 / 16.3 / 16.3; 64 and 18355 tokens alike). */
#define ROWS_WAVES 32u

/* Rows on their way (att_rows_args): a token's heads are gone through by one wave, or where
 * there are few tokens by several. */
static int rows_go(att_rows_args *a, int32_t dtype) {
    const uint32_t at_once = a->hd > 64 ? 4 : 8, rows = (a->q ? a->n_head : 0) + (a->k ? a->n_head_kv : 0) + (a->v ? a->n_head_kv : 0);
    const uint32_t most = (rows + at_once - 1) / at_once, places = (uint32_t) sllm_shim_cu() * ROWS_WAVES;
    a->waves = (places + a->n_tok - 1) / a->n_tok;
    if (a->waves > most) a->waves = most;
    void *args[] = { a };
    const uint64_t waves = (uint64_t) a->n_tok * a->waves;
    return sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_ROWS + dtype), (uint32_t) ((waves + ATT_THREADS / 64 - 1) / (ATT_THREADS / 64)), 1,
                            ATT_THREADS, 0, args);
}

/* bytes between a tensor's rows of `width` elements; 0: not what a call takes */
static uint64_t row_bytes(size_t stride, uint64_t width, uint32_t size) {
    if (stride == 0) stride = (size_t) width;
    if (stride > (1u << 28) || stride < width || stride * size % 16u != 0) return 0;
    return (uint64_t) stride * size;
}

/* A batch's rows into the cache, turned or not: a has where they are and how they turn. */
static int launch_rows(sllm_gfx950_batch *b, int32_t layer, att_rows_args *a) {
    const sllm_gfx950_pages *p = b->p;
    uint8_t *layer_mem = p->mem + (uint64_t) layer * p->layer_bytes;
    a->ck = layer_mem;
    a->cv = layer_mem + (uint64_t) p->d.n_head_kv * p->block_bytes;
    a->tables = (const uint32_t *) (b->buf.dev + b->off_tables);
    a->toks = (const att_tok *) (b->buf.dev + b->off_toks);
    a->page_bytes = p->page_bytes;
    a->page_shift = p->page_shift;
    a->block_bytes = p->block_bytes;
    a->n_tok = b->n_tok;
    a->n_head = (uint32_t) b->n_head;
    a->n_head_kv = (uint32_t) p->d.n_head_kv;
    a->hd = (uint32_t) p->d.head_dim;
    a->held = held_as(p->d.dtype);
    return rows_go(a, b->act);
}

int sllm_gfx950_batch_store(sllm_gfx950_batch *b, int32_t layer, const void *k, size_t k_stride, const void *v, size_t v_stride) {
    ATT_ON_DEVICE();
    if (b == NULL) return FAIL_ARG("batch_store: NULL");
    sllm_gfx950_pages *p = b->p;
    if (layer < 0 || layer >= p->d.n_layer) return FAIL_ARG("batch_store: layer %d of %d", layer, p->d.n_layer);
    const uint32_t kv = (uint32_t) p->d.n_head_kv, hd = (uint32_t) p->d.head_dim, size = type_size(b->act);
    const uint64_t kt = row_bytes(k_stride, (uint64_t) kv * hd, size), vt = row_bytes(v_stride, (uint64_t) kv * hd, size);
    if (kt == 0 || vt == 0) return FAIL_ARG("batch_store: stride");
    if (b->n_tok == 0) return SLLM_GFX950_OK;
    if (k == NULL || v == NULL || misaligned(k) || misaligned(v)) return FAIL_ARG("batch_store: NULL or misaligned rows");
    if (held8(p->d.dtype)) {
        att_rows_args r = { .k = k, .v = v, .k_tok = kt, .v_tok = vt };
        return launch_rows(b, layer, &r);
    }
    uint8_t *layer_mem = p->mem + (uint64_t) layer * p->layer_bytes;
    att_store_args a = { k, v, layer_mem, layer_mem + (uint64_t) kv * p->block_bytes,
                         (const uint32_t *) (b->buf.dev + b->off_tables), (const att_tok *) (b->buf.dev + b->off_toks), kt, vt, p->page_bytes, p->page_shift, hd, kv, b->n_tok };
    void *args[] = { &a };
    const uint64_t threads = (uint64_t) b->n_tok * (hd / 8u);
    return sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_STORE + (b->pair < 2 ? b->pair : 2)),
                            (uint32_t) ((threads + ATT_THREADS - 1) / ATT_THREADS), 2u * kv, ATT_THREADS, 0, args);
}

int64_t sllm_gfx950_batch_positions(const sllm_gfx950_batch *b) { return b ? b->n_pos : 0; }

int sllm_gfx950_batch_read(sllm_gfx950_batch *b, int32_t layer, void *k, size_t k_stride, void *v, size_t v_stride) {
    ATT_ON_DEVICE();
    if (b == NULL) return FAIL_ARG("batch_read: NULL");
    const sllm_gfx950_pages *p = b->p;
    if (layer < 0 || layer >= p->d.n_layer) return FAIL_ARG("batch_read: layer %d of %d", layer, p->d.n_layer);
    const uint32_t kv = (uint32_t) p->d.n_head_kv, hd = (uint32_t) p->d.head_dim, size = type_size(b->act);
    const uint64_t width = (uint64_t) kv * hd, kt = row_bytes(k_stride, width, size), vt = row_bytes(v_stride, width, size);
    if (kt == 0 || vt == 0) return FAIL_ARG("batch_read: stride");
    if (b->n_pos > SLLM_GFX950_ATTN_MAX_LEN || b->n_pages > MAX_ITEMS) return FAIL_ARG("batch_read: %lld positions", (long long) b->n_pos);
    if (b->n_pos == 0) return SLLM_GFX950_OK;
    if (k == NULL || v == NULL || misaligned(k) || misaligned(v)) return FAIL_ARG("batch_read: NULL or misaligned rows");
    const rows_at ko = { k, kt, width * size, b->n_pos }, vo = { v, vt, width * size, b->n_pos };
    if (overlap(&ko, &vo)) return FAIL_ARG("batch_read: rows of k and v overlap");
    const uint8_t *layer_mem = p->mem + (uint64_t) layer * p->layer_bytes;
    att_read_args a = { k, v, layer_mem, layer_mem + (uint64_t) kv * p->block_bytes, (const uint32_t *) (b->buf.dev + b->off_tables),
                        (const att_seq *) (b->buf.dev + b->off_seqs), kt, vt, p->page_bytes, (uint32_t) b->n_seq, hd, kv, held_as(p->d.dtype),
                        p->page_shift, p->block_bytes };
    void *args[] = { &a };
    const uint64_t units = (uint64_t) p->d.page_tokens * (hd / 8u) * 2u * kv;
    const uint32_t per = ATT_THREADS * ATT_READ_UNITS;
    return sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_READ + b->act), b->n_pages, (uint32_t) ((units + per - 1) / per), ATT_THREADS, 0, args);
}

static int bad_scale(float scale) { return !(scale > 0.0f) || isinf((float) ((double) scale * LOG2E)); }

int sllm_gfx950_batch_attend(sllm_gfx950_batch *b, int32_t layer, const void *q, size_t q_stride, float scale, void *out,
                             size_t out_stride) {
    ATT_ON_DEVICE();
    if (b == NULL) return FAIL_ARG("batch_attend: NULL");
    sllm_gfx950_pages *p = b->p;
    if (layer < 0 || layer >= p->d.n_layer) return FAIL_ARG("batch_attend: layer %d of %d", layer, p->d.n_layer);
    const uint32_t kv = (uint32_t) p->d.n_head_kv, hd = (uint32_t) p->d.head_dim, size = type_size(b->act);
    const uint64_t qt = row_bytes(q_stride, (uint64_t) b->n_head * hd, size), ot = row_bytes(out_stride, (uint64_t) b->n_head * hd, size);
    if (qt == 0 || ot == 0) return FAIL_ARG("batch_attend: stride");
    if (bad_scale(scale)) return FAIL_ARG("batch_attend: scale %g", (double) scale);
    if (b->n_tok == 0) return SLLM_GFX950_OK;
    if (q == NULL || out == NULL || misaligned(q) || misaligned(out)) return FAIL_ARG("batch_attend: NULL or misaligned rows");
    const uint32_t wide = hd > 64, group = (uint32_t) b->n_head / kv;
    uint8_t *dev = b->buf.dev;
    const uint8_t *layer_mem = p->mem + (uint64_t) layer * p->layer_bytes;
    att_args a = { .q = q, .out = out, .k = layer_mem, .v = layer_mem + (uint64_t) kv * p->block_bytes,
                   .items = (const att_item *) dev, .n_items = b->n_items, .tables = (const uint32_t *) (dev + b->off_tables), .list = (const uint32_t *) (dev + b->off_list),
                   .part_o = (float *) (dev + b->off_part_o), .part_ml = (float *) (dev + b->off_part_ml),
                   .q_tok = qt, .q_head = (uint64_t) hd * size, .out_tok = ot, .out_head = (uint64_t) hd * size,
                   .page_bytes = p->page_bytes, .page_shift = p->page_shift, .hd = hd, .group = group,
                   .per_group = 1.0f / (float) group, .c = (float) ((double) scale * LOG2E), .block_bytes = p->block_bytes };
    /* the partial results are one set of memory: a call's launches stay together */
    pthread_mutex_lock(&p->mtx);
    int st = SLLM_GFX950_OK;
    void *args[] = { &a };
    st = sllm_shim_launch(sllm_shim_attn_function(b->pair >= SLLM_ATTN_HELD8 ? SLLM_ATTN_ATTEND8 + (b->pair - SLLM_ATTN_HELD8) * 2 + (int) wide :
                                                  SLLM_ATTN_ATTEND + b->pair * 2 + (int) wide), a.n_items, 1, ATT_THREADS, 0, args);
    if (st == SLLM_GFX950_OK && b->join > 0) {
        att_join_args j = { out, a.part_o, a.part_ml, (const att_tok *) (dev + b->off_toks), (const att_seg *) (dev + b->off_segs), ot,
                            hd, group, (uint32_t) b->n_head, 0 };
        void *jargs[] = { &j };
        /* a workgroup a row, or where none has more than eight partial results a wave
         * (us, a wave / a workgroup: 5120 rows of up to 4, 26.5 / 29.8; 8 sequences of
         * over 16 parts a row 16.9 / 12.1; 5 to 16 parts alike) */
        const int whole = b->join > 8;
        const uint32_t heads = (uint32_t) b->n_head, gy = whole ? heads : (heads + ATT_THREADS / 64 - 1) / (ATT_THREADS / 64);
        st = sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_JOIN + 6 * whole + b->act * 2 + (int) wide),
                              b->n_tok, gy, ATT_THREADS, 0, jargs);
    }
    pthread_mutex_unlock(&p->mtx);
    return st;
}

/* ------------------------------------------------------------------ */
/* whole prompts                                                       */
/* ------------------------------------------------------------------ */

struct sllm_gfx950_prompt {
    int32_t  dtype, n_head, n_head_kv, head_dim;
    uint64_t n_q, n_k;               /* rows */
    uint32_t n_items;
    att_item *items;                 /* device */
};

/*
 * The rows of a plan's workgroups. Smaller ones read the keys more often but are
 * more, and each is done sooner: what counts is all work against the longest row
 * tile's, in tiles of keys, of which starting a workgroup costs about eight. Many
 * rows take 1.1 us a tile with two workgroups a CU and 0.85 alone (16 bits; f32 4.3
 * and 2.8 for half the keys), half as many 0.73 and 0.69 (2.3 and 1.9); few rows
 * go through their keys with four waves at once. Measured, us at few / half / many:
 * bf16, one prompt of 128 rows 6.0 / 6.6 / 8.8, 512 16.5 / 13.8 / 18.1, 2048
 * 104 / 44 / 55, 4096 376 / 127 / 108, four of up to 2048 123 / 45 / 55, 64 of up
 * to 200 70 / 27 / 23; f32, 512 30 / 48 / 85, 2048 217 / 237 / 357, 4096
 * 782 / 765 / 862, four of up to 2048 254 / 239 / 367 and, longer, 606 / 502 / 490.
 */
static uint32_t prompt_mode(const sllm_gfx950_prompt_desc *d, uint32_t group) {
    const int wide = d->dtype == SLLM_GFX950_F32;
    const int64_t tile = wide ? 16 : 32;
    uint64_t all = 0, longest = 0;
    for (int32_t i = 0; i < d->n_seq; ++i) {
        const int64_t nq = d->q_len[i], nk = d->k_len ? d->k_len[i] : nq, rows = nq * group;
        for (int64_t r = 0; r < rows; r += ATT_MANY_ROWS) {
            const int64_t end = (r + ATT_MANY_ROWS < rows ? r + ATT_MANY_ROWS : rows) - 1, keys = end / group + nk - nq + 1;
            const uint64_t tiles = keys > 0 ? (uint64_t) ((keys + tile - 1) / tile) : 0;
            all += (tiles + 8) * (uint32_t) d->n_head_kv;
            if (tiles > longest) longest = tiles;
        }
    }
    const uint64_t cu = (uint64_t) sllm_shim_cu();
    if (all * 32 < cu * (wide ? 25 : 8) * longest) return ATT_FEW;
    return all * 8 < cu * (wide ? 11 : 9) * (longest + 8) ? ATT_HALF : ATT_MANY;
}

int sllm_gfx950_prompt_create(const sllm_gfx950_prompt_desc *d, sllm_gfx950_prompt **out) {
    ATT_ON_DEVICE();
    if (out == NULL) return FAIL_ARG("prompt_create: NULL out");
    *out = NULL;
    if (d == NULL || bad_type(d->dtype) || bad_heads(d->n_head, d->n_head_kv, d->head_dim) || d->n_seq < 0 ||
        d->n_seq > SLLM_GFX950_ATTN_MAX_SEQS || (d->n_seq > 0 && d->q_len == NULL)) {
        return FAIL_ARG("prompt_create: type, heads, head dimension or sequences outside what a plan takes");
    }
    int st = not_in_capture("prompt_create");
    if (st != SLLM_GFX950_OK) return st;
    sllm_gfx950_prompt *p = calloc(1, sizeof *p);
    items it = { 0 };
    if (p == NULL) return FAIL_NOMEM("prompt_create");
    p->dtype = d->dtype;
    p->n_head = d->n_head;
    p->n_head_kv = d->n_head_kv;
    p->head_dim = d->head_dim;
    const uint32_t group = (uint32_t) (d->n_head / d->n_head_kv);
    uint64_t whole = 0;
    for (int32_t i = 0; i < d->n_seq; ++i) {
        if (d->q_len[i] > 0) whole += ((uint64_t) d->q_len[i] * group + ATT_MANY_ROWS - 1) / ATT_MANY_ROWS * (uint32_t) d->n_head_kv;
    }
    /* (so many that smaller ones might not fit a launch) */
    const uint32_t mode = whole > MAX_ITEMS / (ATT_MANY_ROWS / ATT_FEW_ROWS) ? ATT_MANY : prompt_mode(d, group);
    for (int32_t i = 0; i < d->n_seq && st == SLLM_GFX950_OK; ++i) {
        const int32_t nq = d->q_len[i], nk = d->k_len ? d->k_len[i] : nq;
        if (nq < 0 || nk < 0 || p->n_q + (uint64_t) nq > SLLM_GFX950_ATTN_MAX_TOKENS || p->n_k + (uint64_t) nk > SLLM_GFX950_ATTN_MAX_TOKENS) {
            st = FAIL_ARG("prompt_create: sequence %d of %d and %d rows, or too many", i, nq, nk);
            break;
        }
        if (whole > MAX_ITEMS) { st = FAIL_ARG("prompt_create: too many rows"); break; }
        const uint32_t rows = (uint32_t) nq * group;
        const uint32_t own = mode_of(rows, d->dtype, d->dtype) == ATT_FEW ? ATT_FEW : mode, tile = k_rows[own];
        for (int32_t h = 0; h < d->n_head_kv && st == SLLM_GFX950_OK; ++h) {
            for (uint32_t r = 0; r < rows; r += tile) {
                const uint32_t n = rows - r < tile ? rows - r : tile;
                const int32_t last = (int32_t) ((r + n - 1) / group) + nk - nq + 1;    /* keys that the last row sees */
                att_item *a = items_add(&it);
                if (a == NULL) { st = FAIL_NOMEM("prompt_create: work items"); break; }
                *a = (att_item) { r / group, n, (uint32_t) p->n_q, ATT_TOKENS, nk - nq + 1, 0, last > 0 ? (uint32_t) last : 0,
                                  (uint32_t) p->n_k, (uint32_t) h, ATT_DIRECT, (uint16_t) own, (uint16_t) (r % group), 0 };
            }
        }
        p->n_q += (uint64_t) nq;
        p->n_k += (uint64_t) nk;
        if (st == SLLM_GFX950_OK && it.n > MAX_ITEMS) st = FAIL_ARG("prompt_create: too many rows");
    }
    if (st == SLLM_GFX950_OK && it.n > 0) {
        order_work(&it);
        p->n_items = (uint32_t) it.n;
        hipError_t e = hipMalloc((void **) &p->items, it.n * sizeof *it.v);
        if (e != hipSuccess) { p->items = NULL; st = sllm_shim_hip_fail(e, "hipMalloc(prompt plan)"); }
        else {
            e = hipMemcpyAsync(p->items, it.v, it.n * sizeof *it.v, hipMemcpyHostToDevice, sllm_shim_stream());
            if (e == hipSuccess) e = hipStreamSynchronize(sllm_shim_stream());
            if (e != hipSuccess) st = sllm_shim_hip_fail(e, "prompt_create");
        }
    }
    free(it.v);
    if (st != SLLM_GFX950_OK) {
        if (p->items) hipFree(p->items);
        free(p);
        return st;
    }
    *out = p;
    return SLLM_GFX950_OK;
}

void sllm_gfx950_prompt_destroy(sllm_gfx950_prompt *p) {
    if (p == NULL) return;
    buffer own = { .dev = (uint8_t *) p->items };
    if (p->items) release(&own, 1);
    free(p);
}

/* A tensor [n][heads][hd] with strides tok and head in elements, 0 and 0: packed.
 * Bytes into *t and *h; 0: not what a call takes (32 rows of a tile are apart by
 * less than 2^32 bytes). */
static int strides(size_t tok, size_t head, uint64_t heads, uint64_t hd, uint32_t size, uint64_t *t, uint64_t *h) {
    if (tok == 0 && head == 0) {
        tok = (size_t) (heads * hd);
        head = (size_t) hd;
    }
    if (tok > (1u << 25) || (uint64_t) head > 1ull << 40 || tok * size % 16u != 0 || head * size % 16u != 0) return 0;
    *t = (uint64_t) tok * size;
    *h = (uint64_t) head * size;
    return 1;
}

int sllm_gfx950_prompt_attend(sllm_gfx950_prompt *p, const sllm_gfx950_prompt_io *io) {
    ATT_ON_DEVICE();
    if (p == NULL || io == NULL) return FAIL_ARG("prompt_attend: NULL");
    if (bad_scale(io->scale)) return FAIL_ARG("prompt_attend: scale %g", (double) io->scale);
    const uint32_t size = type_size(p->dtype), hd = (uint32_t) p->head_dim;
    att_args a = { .q = io->q, .out = io->out, .k = io->k, .v = io->v, .items = p->items, .hd = hd,
                   .group = (uint32_t) (p->n_head / p->n_head_kv), .per_group = 1.0f / (float) (p->n_head / p->n_head_kv),
                   .n_items = p->n_items, .c = (float) ((double) io->scale * LOG2E) };
    if (!strides(io->q_tok, io->q_head, (uint64_t) p->n_head, hd, size, &a.q_tok, &a.q_head) ||
        !strides(io->k_tok, io->k_head, (uint64_t) p->n_head_kv, hd, size, &a.k_tok, &a.k_head) ||
        !strides(io->v_tok, io->v_head, (uint64_t) p->n_head_kv, hd, size, &a.v_tok, &a.v_head) ||
        !strides(io->out_tok, io->out_head, (uint64_t) p->n_head, hd, size, &a.out_tok, &a.out_head)) {
        return FAIL_ARG("prompt_attend: strides");
    }
    /* rows of out apart: heads within a token, or tokens within a head */
    const uint64_t row = (uint64_t) hd * size;
    const int by_tok = a.out_head >= row && (p->n_q <= 1 || a.out_tok >= (uint64_t) (p->n_head - 1) * a.out_head + row);
    const int by_head = a.out_tok >= row && (p->n_head == 1 || a.out_head >= (p->n_q ? (p->n_q - 1) : 0) * a.out_tok + row);
    if (!by_tok && !by_head) return FAIL_ARG("prompt_attend: rows of out overlap");
    if (p->n_items == 0) return SLLM_GFX950_OK;
    if (io->q == NULL || io->out == NULL || misaligned(io->q) || misaligned(io->k) || misaligned(io->v) || misaligned(io->out) ||
        (p->n_k > 0 && (io->k == NULL || io->v == NULL))) {
        return FAIL_ARG("prompt_attend: NULL or misaligned rows");
    }
    const int type = p->dtype == SLLM_GFX950_F32 ? 0 : p->dtype == SLLM_GFX950_F16 ? 1 : 2;
    void *args[] = { &a };
    return sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_PROMPT + type * 2 + (hd > 64)), p->n_items, 1, ATT_THREADS, 0, args);
}

/* ------------------------------------------------------------------ */
/* rotary positions                                                    */
/* ------------------------------------------------------------------ */

struct sllm_gfx950_rope {
    int32_t   head_dim, n_rot, pairs;
    float     magnitude;
    uint64_t *freq;                  /* device */
};

/* The turns a position of pair i, modulo 1, times 2^64: a position times that, modulo 2^64, is its
 * angle to 2^-64 of a turn a position, however far it is. */
static int rope_turns(const sllm_gfx950_rope_desc *d, uint64_t *to) {
    const long double two_pi = 6.283185307179586476925286766559L;
    const long double base = d->scaling == SLLM_GFX950_ROPE_NTK ? d->base * powl(d->factor, (long double) d->n_rot / (d->n_rot - 2)) : d->base;
    for (int32_t i = 0; i < d->n_rot / 2; ++i) {
        long double f = d->freq ? d->freq[i] : powl(base, -2.0L * i / d->n_rot);
        if (d->scaling == SLLM_GFX950_ROPE_LINEAR) f /= d->factor;
        if (d->scaling == SLLM_GFX950_ROPE_PARTS) {
            long double keep = (d->original * f / two_pi - d->slow) / ((long double) d->fast - d->slow);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * keep + f / d->factor * (1 - keep);
        }
        if (!(fabsl(f) <= 1048576.0L)) return 0;
        long double t = f / two_pi;
        t -= floorl(t);
        t = ldexpl(t, 64);
        to[i] = t >= 18446744073709551615.0L ? UINT64_MAX : (uint64_t) t;
    }
    return 1;
}

int sllm_gfx950_rope_new(const sllm_gfx950_rope_desc *d, sllm_gfx950_rope **out) {
    ATT_ON_DEVICE();
    if (out == NULL) return FAIL_ARG("rope_new: NULL out");
    *out = NULL;
    if (d == NULL || bad_heads(1, 1, d->head_dim) || d->n_rot < 8 || d->n_rot > d->head_dim || d->n_rot % 8 != 0 ||
        (d->layout != SLLM_GFX950_ROPE_HALVES && d->layout != SLLM_GFX950_ROPE_PAIRS)) {
        return FAIL_ARG("rope_new: head dimension, dimensions that turn, or their layout");
    }
    if (d->scaling < SLLM_GFX950_ROPE_PLAIN || d->scaling > SLLM_GFX950_ROPE_PARTS || !isfinite((float) d->magnitude) ||
        (d->freq == NULL && !(d->base > 0 && isfinite(d->base))) ||
        (d->scaling != SLLM_GFX950_ROPE_PLAIN && !(d->factor > 0 && isfinite(d->factor))) || (d->scaling == SLLM_GFX950_ROPE_NTK && d->freq != NULL) ||
        (d->scaling == SLLM_GFX950_ROPE_PARTS && !(d->original > 0 && isfinite(d->original) && isfinite(d->slow) && d->fast > d->slow && isfinite(d->fast)))) {
        return FAIL_ARG("rope_new: base, frequencies or scaling");
    }
    int st = not_in_capture("rope_new");
    if (st != SLLM_GFX950_OK) return st;
    uint64_t turns[SLLM_GFX950_ATTN_MAX_HEAD_DIM / 2];
    if (!rope_turns(d, turns)) return FAIL_ARG("rope_new: a frequency over 2^20 or not finite");
    sllm_gfx950_rope *r = calloc(1, sizeof *r);
    if (r == NULL) return FAIL_NOMEM("rope_new");
    r->head_dim = d->head_dim;
    r->n_rot = d->n_rot;
    r->pairs = d->layout == SLLM_GFX950_ROPE_PAIRS;
    r->magnitude = d->magnitude == 0 ? 1.0f : (float) d->magnitude;
    const size_t bytes = (size_t) (d->n_rot / 2) * sizeof *turns;
    hipError_t e = hipMalloc((void **) &r->freq, bytes);
    const char *what = "hipMalloc(rope)";
    if (e != hipSuccess) r->freq = NULL;
    else {
        what = "rope_new";
        e = hipMemcpyAsync(r->freq, turns, bytes, hipMemcpyHostToDevice, sllm_shim_stream());
        if (e == hipSuccess) e = hipStreamSynchronize(sllm_shim_stream());
    }
    if (e != hipSuccess) {
        if (r->freq) hipFree(r->freq);
        free(r);
        return sllm_shim_hip_fail(e, what);
    }
    *out = r;
    return SLLM_GFX950_OK;
}

void sllm_gfx950_rope_free(sllm_gfx950_rope *r) {
    if (r == NULL) return;
    buffer own = { .dev = (uint8_t *) r->freq };
    release(&own, 1);
    free(r);
}

static void rope_args(const sllm_gfx950_rope *r, att_rows_args *a) {
    a->freq = r->freq;
    a->half = (uint32_t) r->n_rot / 2;
    a->pairs = (uint32_t) r->pairs;
    a->magnitude = r->magnitude;
}

/* where rows may go: to where they come from, or apart from all that is read */
static int bad_target(const rows_at *out, const rows_at *own, const rows_at *other, const rows_at *third) {
    if ((out->p != own->p || out->tok != own->tok) && overlap(out, own)) return 1;
    return overlap(out, other) || overlap(out, third);
}

int sllm_gfx950_rope_rows(sllm_gfx950_rope *r, const sllm_gfx950_rope_io *io) {
    ATT_ON_DEVICE();
    if (r == NULL || io == NULL) return FAIL_ARG("rope_rows: NULL");
    if (bad_type(io->dtype) || io->n_rows < 0 || io->n_rows > SLLM_GFX950_ATTN_MAX_TOKENS || io->n_head < 1 || io->n_head > SLLM_GFX950_ATTN_MAX_HEADS ||
        (io->k != NULL && (io->n_head_kv < 1 || io->n_head_kv > SLLM_GFX950_ATTN_MAX_HEADS))) {
        return FAIL_ARG("rope_rows: type, rows or heads");
    }
    const uint32_t size = type_size(io->dtype), hd = (uint32_t) r->head_dim;
    const uint64_t qw = (uint64_t) io->n_head * hd, kw = io->k ? (uint64_t) io->n_head_kv * hd : hd;
    const uint64_t qt = row_bytes(io->q_stride, qw, size), qo = row_bytes(io->q_out_stride, qw, size);
    const uint64_t kt = io->k ? row_bytes(io->k_stride, kw, size) : 1, ko = io->k ? row_bytes(io->k_out_stride, kw, size) : 1;
    if (qt == 0 || qo == 0 || kt == 0 || ko == 0) return FAIL_ARG("rope_rows: stride");
    if (io->n_rows == 0) return SLLM_GFX950_OK;
    if (io->q == NULL || io->q_out == NULL || io->pos == NULL || (io->k != NULL) != (io->k_out != NULL) || misaligned(io->q) || misaligned(io->q_out) ||
        misaligned(io->k) || misaligned(io->k_out) || ((uintptr_t) io->pos & 3u) != 0) {
        return FAIL_ARG("rope_rows: NULL or misaligned rows or positions");
    }
    const rows_at q = { io->q, qt, qw * size, io->n_rows }, k = { io->k, kt, kw * size, io->n_rows }, pos = { io->pos, 4, 4, io->n_rows };
    const rows_at qo_at = { io->q_out, qo, qw * size, io->n_rows }, ko_at = { io->k_out, ko, kw * size, io->n_rows };
    if (bad_target(&qo_at, &q, &k, &pos) || bad_target(&ko_at, &k, &q, &pos) || overlap(&qo_at, &ko_at)) return FAIL_ARG("rope_rows: rows overlap");
    att_rows_args a = { .q = io->q, .k = io->k, .q_out = io->q_out, .k_out = io->k_out, .pos = io->pos, .q_tok = qt, .k_tok = kt, .qo_tok = qo, .ko_tok = ko,
                        .n_tok = (uint32_t) io->n_rows, .n_head = (uint32_t) io->n_head, .n_head_kv = (uint32_t) io->n_head_kv, .hd = hd,
                        .back = io->back != 0 };
    rope_args(r, &a);
    return rows_go(&a, io->dtype);
}

int sllm_gfx950_batch_rope_store(sllm_gfx950_batch *b, int32_t layer, sllm_gfx950_rope *r, const void *q, size_t q_stride, void *q_out, size_t q_out_stride,
                                 const void *k, size_t k_stride, const void *v, size_t v_stride) {
    ATT_ON_DEVICE();
    if (b == NULL || r == NULL) return FAIL_ARG("batch_rope_store: NULL");
    const sllm_gfx950_pages *p = b->p;
    if (layer < 0 || layer >= p->d.n_layer) return FAIL_ARG("batch_rope_store: layer %d of %d", layer, p->d.n_layer);
    if (r->head_dim != p->d.head_dim) return FAIL_ARG("batch_rope_store: heads of %d and %d", r->head_dim, p->d.head_dim);
    const uint32_t kv = (uint32_t) p->d.n_head_kv, hd = (uint32_t) p->d.head_dim, size = type_size(b->act);
    const uint64_t qw = (uint64_t) b->n_head * hd, kw = (uint64_t) kv * hd;
    const uint64_t qt = row_bytes(q_stride, qw, size), qo = row_bytes(q_out_stride, qw, size), kt = row_bytes(k_stride, kw, size), vt = row_bytes(v_stride, kw, size);
    if (qt == 0 || qo == 0 || kt == 0 || vt == 0) return FAIL_ARG("batch_rope_store: stride");
    if (b->n_tok == 0) return SLLM_GFX950_OK;
    if (q == NULL || q_out == NULL || k == NULL || v == NULL || misaligned(q) || misaligned(q_out) || misaligned(k) || misaligned(v)) {
        return FAIL_ARG("batch_rope_store: NULL or misaligned rows");
    }
    const rows_at out = { q_out, qo, qw * size, b->n_tok }, qr = { q, qt, qw * size, b->n_tok }, kr = { k, kt, kw * size, b->n_tok }, vr = { v, vt, kw * size, b->n_tok };
    if (bad_target(&out, &qr, &kr, &vr)) return FAIL_ARG("batch_rope_store: rows overlap");
    att_rows_args a = { .q = q, .k = k, .v = v, .q_out = q_out, .q_tok = qt, .k_tok = kt, .v_tok = vt, .qo_tok = qo };
    rope_args(r, &a);
    return launch_rows(b, layer, &a);
}

/* ------------------------------------------------------------------ */
/* beams                                                               */
/* ------------------------------------------------------------------ */

struct sllm_gfx950_beam {
    pthread_mutex_t mtx;
    sllm_gfx950_beam_desc d;
    uint32_t  n_chunk, chunk;
    uint8_t  *mem;                   /* keys, then sums */
    size_t    off_sums;
};

/* A row's parts: as many as give every CU BEAM_GROUPS workgroups, of whole tiles, but no more than
 * the join has lanes. (us, 256 rows of 128256 at 2 / 4 / 8 / 16 of them: bf16, 16 picks 28.9 / 26.2 /
 * 30.5 / 30.8, 1 pick 24.5 / 23.2 / 26.6 / 27.2, 64 picks 59 / 56 / 52 / 45; f32 32.3 / 34.4 / 37.8 / 39.7;
 * 1024 rows of 32000 27.5 / 26.4 / 28.4 / 28.6. One number for all: 64 picks of few rows would like more, f32 fewer.) */
#define BEAM_GROUPS 4u

static void beam_chunks(sllm_gfx950_beam *p) {
    const uint32_t rows = (uint32_t) (p->d.n_group * p->d.n_beam), tiles = ((uint32_t) p->d.n_vocab + BEAM_TILE - 1) / BEAM_TILE;
    uint32_t n = ((uint32_t) sllm_shim_cu() * BEAM_GROUPS + rows - 1) / rows;
    if (n > BEAM_MAX_PARTS) n = BEAM_MAX_PARTS;
    const uint32_t each = (tiles + n - 1) / n;
    p->chunk = each * BEAM_TILE;
    p->n_chunk = (tiles + each - 1) / each;
}

int sllm_gfx950_beam_new(const sllm_gfx950_beam_desc *d, sllm_gfx950_beam **out) {
    ATT_ON_DEVICE();
    if (out == NULL) return FAIL_ARG("beam_new: NULL out");
    *out = NULL;
    if (d == NULL || bad_type(d->dtype) || d->n_group < 1 || d->n_beam < 1 || d->n_beam > SLLM_GFX950_BEAM_MAX || d->n_vocab < 1 || d->n_vocab > 1 << 24 ||
        d->n_pick < 1 || d->n_pick > SLLM_GFX950_BEAM_MAX || d->n_beam * d->n_pick > (int32_t) BEAM_MAX_LIST ||
        (int64_t) d->n_pick > (int64_t) d->n_beam * d->n_vocab || (int64_t) d->n_group * d->n_beam > 1 << 20) {
        return FAIL_ARG("beam_new: type, groups, beams, vocabulary or picks outside what a plan takes");
    }
    int st = not_in_capture("beam_new");
    if (st != SLLM_GFX950_OK) return st;
    sllm_gfx950_beam *p = calloc(1, sizeof *p);
    if (p == NULL) return FAIL_NOMEM("beam_new");
    p->d = *d;
    beam_chunks(p);
    const size_t parts = (size_t) d->n_group * (size_t) d->n_beam * p->n_chunk;
    p->off_sums = align256(parts * (size_t) d->n_pick * sizeof(uint64_t));
    const hipError_t e = hipMalloc((void **) &p->mem, p->off_sums + parts * 2 * sizeof(double));
    if (e != hipSuccess) {
        free(p);
        return sllm_shim_hip_fail(e, "hipMalloc(beams)");
    }
    pthread_mutex_init(&p->mtx, NULL);
    *out = p;
    return SLLM_GFX950_OK;
}

void sllm_gfx950_beam_free(sllm_gfx950_beam *p) {
    if (p == NULL) return;
    buffer own = { .dev = p->mem };
    release(&own, 1);
    pthread_mutex_destroy(&p->mtx);
    free(p);
}

int sllm_gfx950_beam_select(sllm_gfx950_beam *p, const void *logits, size_t stride, const float *scores, const int32_t *ended, float *out_scores,
                            int32_t *out_beam, int32_t *out_token) {
    ATT_ON_DEVICE();
    if (p == NULL || logits == NULL || scores == NULL || out_scores == NULL || out_beam == NULL || out_token == NULL) return FAIL_ARG("beam_select: NULL");
    const uint32_t size = type_size(p->d.dtype), rows = (uint32_t) (p->d.n_group * p->d.n_beam);
    if (stride == 0) stride = (size_t) p->d.n_vocab;
    if (stride < (size_t) p->d.n_vocab || stride > (1u << 28)) return FAIL_ARG("beam_select: stride");
    if (misaligned(logits) || (((uintptr_t) scores | (uintptr_t) ended | (uintptr_t) out_scores | (uintptr_t) out_beam | (uintptr_t) out_token) & 3u) != 0) {
        return FAIL_ARG("beam_select: misaligned");
    }
    const uint64_t in = (uint64_t) rows * 4u, picks = (uint64_t) p->d.n_group * (uint64_t) p->d.n_pick * 4u, width = (uint64_t) p->d.n_vocab * size;
    const rows_at outs[3] = { { out_scores, picks, picks, 1 }, { out_beam, picks, picks, 1 }, { out_token, picks, picks, 1 } };
    const rows_at ins[3] = { { logits, (uint64_t) stride * size, width, rows }, { scores, in, in, 1 }, { ended, in, in, 1 } };
    for (int i = 0; i < 3; ++i) {
        for (int j = 0; j < 3; ++j) {
            if (overlap(&outs[i], &ins[j]) || (j < i && overlap(&outs[i], &outs[j]))) return FAIL_ARG("beam_select: what is written overlaps");
        }
    }
    att_beam_args a = { logits, scores, ended, out_scores, out_beam, out_token, (double *) (p->mem + p->off_sums), (uint64_t *) p->mem,
                        (uint64_t) stride * size, (uint32_t) p->d.n_beam, (uint32_t) p->d.n_vocab, (uint32_t) p->d.n_pick, p->n_chunk, p->chunk, 0 };
    void *args[] = { &a };
    /* the plan's memory is one: a call's launches stay together */
    pthread_mutex_lock(&p->mtx);
    int st = sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_BEAM + p->d.dtype), p->n_chunk * rows, 1, ATT_THREADS, 0, args);
    if (st == SLLM_GFX950_OK) st = sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_BEAM_JOIN), (uint32_t) p->d.n_group, 1, BEAM_JOIN_THREADS, 0, args);
    pthread_mutex_unlock(&p->mtx);
    return st;
}
