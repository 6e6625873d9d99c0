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

static uint32_t type_size(int32_t dtype) { return dtype == SLLM_GFX950_F32 ? 4u : 2u; }
static int bad_type(int32_t dtype) { return dtype != SLLM_GFX950_F32 && dtype != SLLM_GFX950_F16 && dtype != SLLM_GFX950_BF16; }

/* the kernels' instances for rows and a cache of these types (shim_internal.h), or -1 */
static int type_pair(int32_t act, int32_t cache) {
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
    return (uint64_t) d->n_layer * 2u * (uint64_t) d->n_head_kv * (uint64_t) d->page_tokens * (uint64_t) d->head_dim * type_size(d->dtype);
}

static int bad_desc(const sllm_gfx950_pages_desc *d) {
    return d == NULL || bad_type(d->dtype) || bad_heads(d->n_head_kv, d->n_head_kv, d->head_dim) || d->n_layer < 1 ||
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
    p->block_bytes = (uint32_t) d->page_tokens * p->row_bytes;
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
    c->a.n_pairs = c->most = 0;
    c->st = SLLM_GFX950_OK;
}

static int copies_flush(copies *c) {
    if (c->st == SLLM_GFX950_OK && c->a.n_pairs > 0) {
        const uint64_t chunks = (uint64_t) c->most * c->a.row_bytes / 16u * c->a.n_blocks;
        void *args[] = { &c->a };
        c->st = sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_COPY),
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
    int32_t   n_head, pair;
    uint32_t  n_tok;
    uint32_t  n_items;
    uint32_t  join;                  /* the most partial results that a row has */
    buffer    buf;
    size_t    off_tables, off_list, off_toks, off_segs, off_part_o, off_part_ml;     /* (its items are at 0) */
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
static uint32_t mode_of(uint32_t rows, int32_t dtype) {
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
    uint64_t n_list = 0;
    for (int32_t i = 0; i < x->n_seg; ++i) {
        segment *s = &x->seg[i];
        for (int32_t j = s->lo; j < s->hi; ++j) s->n_tok += (uint32_t) x->n_new[x->order[j]];
        s->list = ATT_TOKENS;
        if (s->hi - s->lo > 1) { s->list = (uint32_t) n_list; n_list += s->n_tok; }
        s->mode = mode_of(s->n_tok * group, p->d.dtype);
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

/* bytes between a tensor's rows of `width` elements; 0: not what a call takes */
static uint64_t row_bytes(size_t stride, uint64_t width, uint32_t size) {
    if (stride == 0) stride = (size_t) width;
    if (stride > (1u << 28) || stride < width || stride * size % 16u != 0) return 0;
    return (uint64_t) stride * size;
}

int sllm_gfx950_batch_store(sllm_gfx950_batch *b, int32_t layer, const void *k, size_t k_stride, const void *v, size_t v_stride) {
    ATT_ON_DEVICE();
    if (b == NULL) return FAIL_ARG("batch_store: NULL");
    sllm_gfx950_pages *p = b->p;
    if (layer < 0 || layer >= p->d.n_layer) return FAIL_ARG("batch_store: layer %d of %d", layer, p->d.n_layer);
    const uint32_t kv = (uint32_t) p->d.n_head_kv, hd = (uint32_t) p->d.head_dim, size = b->pair <= 1 ? 4u : 2u;
    const uint64_t kt = row_bytes(k_stride, (uint64_t) kv * hd, size), vt = row_bytes(v_stride, (uint64_t) kv * hd, size);
    if (kt == 0 || vt == 0) return FAIL_ARG("batch_store: stride");
    if (b->n_tok == 0) return SLLM_GFX950_OK;
    if (k == NULL || v == NULL || misaligned(k) || misaligned(v)) return FAIL_ARG("batch_store: NULL or misaligned rows");
    uint8_t *layer_mem = p->mem + (uint64_t) layer * p->layer_bytes;
    att_store_args a = { k, v, layer_mem, layer_mem + (uint64_t) kv * p->block_bytes,
                         (const uint32_t *) (b->buf.dev + b->off_tables), (const att_tok *) (b->buf.dev + b->off_toks), kt, vt, p->page_bytes, p->page_shift, hd, kv, b->n_tok };
    void *args[] = { &a };
    const uint64_t threads = (uint64_t) b->n_tok * (hd / 8u);
    return sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_STORE + (b->pair < 2 ? b->pair : 2)),
                            (uint32_t) ((threads + ATT_THREADS - 1) / ATT_THREADS), 2u * kv, ATT_THREADS, 0, args);
}

static int bad_scale(float scale) { return !(scale > 0.0f) || isinf((float) ((double) scale * LOG2E)); }

int sllm_gfx950_batch_attend(sllm_gfx950_batch *b, int32_t layer, const void *q, size_t q_stride, float scale, void *out,
                             size_t out_stride) {
    ATT_ON_DEVICE();
    if (b == NULL) return FAIL_ARG("batch_attend: NULL");
    sllm_gfx950_pages *p = b->p;
    if (layer < 0 || layer >= p->d.n_layer) return FAIL_ARG("batch_attend: layer %d of %d", layer, p->d.n_layer);
    const uint32_t kv = (uint32_t) p->d.n_head_kv, hd = (uint32_t) p->d.head_dim, size = b->pair <= 1 ? 4u : 2u;
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
                   .per_group = 1.0f / (float) group, .c = (float) ((double) scale * LOG2E) };
    /* the partial results are one set of memory: a call's launches stay together */
    pthread_mutex_lock(&p->mtx);
    int st = SLLM_GFX950_OK;
    void *args[] = { &a };
    st = sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_ATTEND + b->pair * 2 + (int) wide), a.n_items, 1, ATT_THREADS, 0, args);
    if (st == SLLM_GFX950_OK && b->join > 0) {
        att_join_args j = { out, a.part_o, a.part_ml, (const att_tok *) (dev + b->off_toks), (const att_seg *) (dev + b->off_segs), ot,
                            hd, group, (uint32_t) b->n_head, 0 };
        void *jargs[] = { &j };
        /* a workgroup a row, or where none has more than eight partial results a wave
         * (us, a wave / a workgroup: 5120 rows of up to 4, 26.5 / 29.8; 8 sequences of
         * over 16 parts a row 16.9 / 12.1; 5 to 16 parts alike) */
        const int whole = b->join > 8;
        const uint32_t heads = (uint32_t) b->n_head, gy = whole ? heads : (heads + ATT_THREADS / 64 - 1) / (ATT_THREADS / 64);
        st = sllm_shim_launch(sllm_shim_attn_function(SLLM_ATTN_JOIN + 6 * whole + (b->pair < 2 ? 0 : b->pair - 1) * 2 + (int) wide),
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
        const uint32_t own = mode_of(rows, d->dtype) == ATT_FEW ? ATT_FEW : mode, tile = k_rows[own];
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
