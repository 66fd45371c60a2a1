/*
 * si_kvpages.c -- paged KV bookkeeping and a multi-layer decode stack over
 * the MI355X C ABI.  Neither exists in the reference, which runs one layer
 * with one contiguous cache (qwen_one_layer.c:237-281); this is the next
 * step after a single layer: many sequences of unequal, growing length
 * decoding together through a stack of layers, each layer's K/V in its own
 * page pool, one page table shared by all layers (every layer holds the
 * same positions of a sequence).
 */
#define _GNU_SOURCE
#include "si_host.h"

#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <hip/hip_runtime_api.h>

static void die(const char *message) {
    fprintf(stderr, "error: %s\n", message);
    exit(1);
}

static void check(int rc, const char *what) {
    if (rc != SI_OK) {
        fprintf(stderr, "error: %s: %s\n", what, si_last_error());
        exit(1);
    }
}

static void hip_check(hipError_t e, const char *what) {
    if (e != hipSuccess) {
        fprintf(stderr, "error: %s: %s\n", what, hipGetErrorString(e));
        exit(1);
    }
}

/* ------------------------------------------------------------------ */
/* page bookkeeping                                                    */
/* ------------------------------------------------------------------ */

struct si_kv_pages {
    int npages, page_size, max_seqs, max_pages;
    int most;       /* pages that the pools have, 0: the caller's concern */
    int *free_list; /* stack of free page ids */
    int nfree;
    int *seqs;      /* per page: sequences that hold it, */
    int *reads;     /* and pending copies that read it; free when both are 0 */
    int *table;     /* [max_seqs][max_pages] page ids (unused entries 0) */
    int *npg;       /* pages held per sequence, -1 = sequence slot unused */
    int *len;       /* positions per sequence */
    int *src, *dst; /* pending copies; at most npages, as no page is written twice */
    int ncopies;
    int sorted;     /* the free list is to be sorted when the copies are done */
};

si_kv_pages_t *si_kv_pages_create(int npages, int page_size, int max_seqs, int max_pages) {
    if (npages < 1 || page_size < 1 || (page_size & (page_size - 1)) || max_seqs < 1 ||
        max_pages < 1)
        die("si_kv_pages_create: bad sizes (page_size must be a power of two)");
    si_kv_pages_t *p = calloc(1, sizeof *p);
    if (!p) die("Out of memory");
    p->npages = npages;
    p->page_size = page_size;
    p->max_seqs = max_seqs;
    p->max_pages = max_pages;
    p->free_list = malloc(sizeof(int) * (size_t)npages);
    p->table = calloc((size_t)max_seqs * max_pages, sizeof(int));
    p->npg = malloc(sizeof(int) * (size_t)max_seqs);
    p->len = calloc((size_t)max_seqs, sizeof(int));
    p->seqs = calloc((size_t)npages, sizeof(int));
    p->reads = calloc((size_t)npages, sizeof(int));
    p->src = malloc(sizeof(int) * (size_t)npages);
    p->dst = malloc(sizeof(int) * (size_t)npages);
    if (!p->free_list || !p->table || !p->npg || !p->len || !p->seqs || !p->reads || !p->src ||
        !p->dst)
        die("Out of memory");
    /* lowest ids on top of the stack: a fresh pool hands out 0, 1, 2, ... */
    for (int i = 0; i < npages; ++i) p->free_list[i] = npages - 1 - i;
    p->nfree = npages;
    for (int i = 0; i < max_seqs; ++i) p->npg[i] = -1;
    return p;
}

void si_kv_pages_destroy(si_kv_pages_t *p) {
    if (!p) return;
    free(p->free_list);
    free(p->table);
    free(p->npg);
    free(p->len);
    free(p->seqs);
    free(p->reads);
    free(p->src);
    free(p->dst);
    free(p);
}

static void check_seq(const si_kv_pages_t *p, int seq) {
    if (seq < 0 || seq >= p->max_seqs || p->npg[seq] < 0) die("si_kv_pages: unknown sequence");
}

int si_kv_seq_add(si_kv_pages_t *p) {
    for (int i = 0; i < p->max_seqs; ++i)
        if (p->npg[i] < 0) {
            p->npg[i] = 0;
            p->len[i] = 0;
            return i;
        }
    return -1;
}

static int take_page(si_kv_pages_t *p) {
    const int pg = p->free_list[--p->nfree];
    p->seqs[pg] = 1;
    return pg;
}

/* Returns a page that nothing holds any more, and drops the copy into it (one
 * at most): its source is held by one copy less. */
static void release_page(si_kv_pages_t *p, int pg) {
    if (p->seqs[pg] || p->reads[pg]) return;
    p->free_list[p->nfree++] = pg;
    for (int i = 0; i < p->ncopies; ++i)
        if (p->dst[i] == pg) {
            const int src = p->src[i];
            --p->ncopies;
            p->src[i] = p->src[p->ncopies];
            p->dst[i] = p->dst[p->ncopies];
            --p->reads[src];
            release_page(p, src); /* itself no copy's target: see si_kv_seq_grow */
            return;
        }
}

static void drop_page(si_kv_pages_t *p, int pg) {
    --p->seqs[pg];
    release_page(p, pg);
}

/* pages of len positions (len + page_size may pass an int) */
static int pages_of(const si_kv_pages_t *p, int len) {
    return (int)(((long long)len + p->page_size - 1) / p->page_size);
}

int si_kv_seq_grow(si_kv_pages_t *p, int seq, int len) {
    check_seq(p, seq);
    const int old = p->len[seq];
    if (len < old) die("si_kv_seq_grow: sequences only grow");
    const long long need = pages_of(p, len);
    int *row = p->table + (size_t)seq * p->max_pages;
    /* positions are about to be written into the last one's page: where another
     * sequence holds it too, into a copy */
    int *last = row + old / p->page_size;
    const int shared = len > old && old % p->page_size && p->seqs[*last] > 1;
    if (need > p->max_pages || need - p->npg[seq] + shared > p->nfree)
        return -1; /* nothing taken */
    if (shared) {
        int from = *last;
        /* copies run at once: of a page that is itself a pending copy, what that reads */
        for (int i = 0; i < p->ncopies; ++i)
            if (p->dst[i] == from) {
                from = p->src[i];
                break;
            }
        --p->seqs[*last];
        *last = take_page(p);
        ++p->reads[from];
        p->src[p->ncopies] = from;
        p->dst[p->ncopies++] = *last;
    }
    while (p->npg[seq] < need) row[p->npg[seq]++] = take_page(p);
    p->len[seq] = len;
    return 0;
}

int si_kv_seq_fork(si_kv_pages_t *p, int seq) {
    check_seq(p, seq);
    const int to = si_kv_seq_add(p);
    if (to < 0) return -1;
    const int *from = p->table + (size_t)seq * p->max_pages;
    int *row = p->table + (size_t)to * p->max_pages;
    p->len[to] = p->len[seq];
    /* the pages with its positions (a sequence may hold more, after a prepare
     * that failed) */
    p->npg[to] = pages_of(p, p->len[seq]);
    for (int i = 0; i < p->npg[to]; ++i) {
        row[i] = from[i];
        ++p->seqs[row[i]];
    }
    return to;
}

void si_kv_seq_truncate(si_kv_pages_t *p, int seq, int len) {
    check_seq(p, seq);
    if (len < 0 || len > p->len[seq]) die("si_kv_seq_truncate: length outside 0..its own");
    int *row = p->table + (size_t)seq * p->max_pages;
    const int keep = pages_of(p, len);
    while (p->npg[seq] > keep) {
        const int i = --p->npg[seq];
        drop_page(p, row[i]);
        row[i] = 0;
    }
    p->len[seq] = len;
}

void si_kv_seq_free(si_kv_pages_t *p, int seq) {
    check_seq(p, seq);
    int *row = p->table + (size_t)seq * p->max_pages;
    /* returned in reverse order, so the next sequence reuses them in order */
    for (int i = p->npg[seq] - 1; i >= 0; --i) {
        drop_page(p, row[i]);
        row[i] = 0;
    }
    p->npg[seq] = -1;
    p->len[seq] = 0;
}

int si_kv_copies(const si_kv_pages_t *p, const int **src, const int **dst) {
    *src = p->src;
    *dst = p->dst;
    return p->ncopies;
}

static int descending(const void *a, const void *b) { return *(const int *)b - *(const int *)a; }

void si_kv_copies_done(si_kv_pages_t *p) {
    while (p->ncopies > 0) {
        const int src = p->src[--p->ncopies];
        --p->reads[src];
        release_page(p, src);
    }
    if (p->sorted) qsort(p->free_list, (size_t)p->nfree, sizeof(int), descending);
    p->sorted = 0;
}

int si_kv_compact(si_kv_pages_t *p) {
    if (p->ncopies) die("si_kv_compact: copies are pending");
    const int used = p->npages - p->nfree;
    int *to = malloc(sizeof(int) * (size_t)p->npages);
    if (!to) die("Out of memory");
    /* each held page past the first `used` ids to a free one among them */
    int low = 0;
    for (int pg = 0; pg < p->npages; ++pg) {
        to[pg] = pg;
        if (pg < used || p->seqs[pg] == 0) continue;
        while (p->seqs[low]) ++low; /* < used: as many are free there as held past it */
        to[pg] = low;
        p->seqs[low] = p->seqs[pg];
        p->seqs[pg] = 0;
        p->reads[pg] = 1;
        p->src[p->ncopies] = pg;
        p->dst[p->ncopies++] = low;
    }
    p->nfree = 0;
    for (int pg = p->npages - 1; pg >= 0; --pg)
        if (!p->seqs[pg] && !p->reads[pg]) p->free_list[p->nfree++] = pg;
    for (int i = 0; i < p->max_seqs; ++i)
        for (int j = 0; j < p->npg[i]; ++j) {
            int *e = p->table + (size_t)i * p->max_pages + j;
            *e = to[*e];
        }
    free(to);
    p->sorted = p->ncopies > 0;
    return used;
}

int si_kv_pages_resize(si_kv_pages_t *p, int npages) {
    if (npages < 1) die("si_kv_pages_resize: npages must be >= 1");
    if (p->most && npages > p->most) return -1;
    for (int pg = npages; pg < p->npages; ++pg)
        if (p->seqs[pg] || p->reads[pg]) return -1;
    if (npages > p->npages) {
        int **arrays[] = {&p->free_list, &p->seqs, &p->reads, &p->src, &p->dst};
        for (int i = 0; i < 5; ++i) {
            int *n = realloc(*arrays[i], sizeof(int) * (size_t)npages);
            if (!n) die("Out of memory");
            *arrays[i] = n;
        }
        for (int pg = p->npages; pg < npages; ++pg) p->seqs[pg] = p->reads[pg] = 0;
    }
    p->npages = npages;
    p->nfree = 0;
    for (int pg = npages - 1; pg >= 0; --pg)
        if (!p->seqs[pg] && !p->reads[pg]) p->free_list[p->nfree++] = pg;
    return 0;
}

int si_kv_seq_len(const si_kv_pages_t *p, int seq) {
    check_seq(p, seq);
    return p->len[seq];
}

int si_kv_pages_free(const si_kv_pages_t *p) { return p->nfree; }

const int *si_kv_page_table(const si_kv_pages_t *p) { return p->table; }

/* ------------------------------------------------------------------ */
/* multi-layer decode stack                                            */
/* ------------------------------------------------------------------ */

struct si_stack {
    si_shape_t shape;
    int nlayers, max_seqs, max_ctx, page_size, npages, format;
    int device;     /* current when it was created: its pools' and tables' */
    size_t page_bytes;
    si_workspace_t *ws;
    si_layer_t **layers;
    uint16_t **kpool, **vpool;
    si_kv_pages_t *pages;
    int *dev_table; /* [max_seqs][max_pages], batch order of the last prepare */
    int *dev_ctx;   /* [max_seqs] */
    int *host_table, *host_ctx;
    float *act[2];  /* ping-pong activations between layers */
    int nseq;       /* rows of the last prepare */
    void *stream;   /* stream of the last si_stack_decode */
    int pending;    /* a decode was enqueued since the last prepare */
    int streams;    /* and another before it, on another stream */
    int captured;   /* a decode was captured: its replays run on any stream, unseen */
};

si_stack_t *si_stack_create(const si_shape_t *s, const si_layer_host_t *layers, int nlayers,
                            int max_seqs, int max_ctx, int npages, int page_size) {
    return si_stack_create_kv(s, layers, nlayers, max_seqs, max_ctx, npages, page_size, SI_KV_F16);
}

si_stack_t *si_stack_create_kv(const si_shape_t *s, const si_layer_host_t *layers, int nlayers,
                               int max_seqs, int max_ctx, int npages, int page_size, int format) {
    if (nlayers < 1 || max_seqs < 1 || max_ctx < 1) die("si_stack_create: bad sizes");
    if (format != SI_KV_F16 && format != SI_KV_Q4) die("si_stack_create: unknown K/V format");
    if (format == SI_KV_Q4 && !si_kv4_page_bytes(s, page_size))
        die("si_stack_create: a 4-bit cache's page_size must be a power of two in 16..65536");
    si_stack_t *st = calloc(1, sizeof *st);
    if (!st) die("Out of memory");
    st->shape = *s;
    st->nlayers = nlayers;
    st->max_seqs = max_seqs;
    st->max_ctx = max_ctx;
    st->page_size = page_size;
    st->npages = npages;
    hip_check(hipGetDevice(&st->device), "hipGetDevice");
    const int max_pages = (max_ctx + page_size - 1) / page_size;
    st->pages = si_kv_pages_create(npages, page_size, max_seqs, max_pages);
    st->pages->most = npages;
    check(si_workspace_create(s, max_seqs, max_ctx, &st->ws), "si_workspace_create");
    st->layers = calloc((size_t)nlayers, sizeof *st->layers);
    st->kpool = calloc((size_t)nlayers, sizeof *st->kpool);
    st->vpool = calloc((size_t)nlayers, sizeof *st->vpool);
    if (!st->layers || !st->kpool || !st->vpool) die("Out of memory");
    st->format = format;
    st->page_bytes = format == SI_KV_Q4
                         ? si_kv4_page_bytes(s, page_size)
                         : (size_t)page_size * s->kvheads * s->hdim * sizeof(uint16_t);
    const size_t pool = (size_t)npages * st->page_bytes;
    for (int l = 0; l < nlayers; ++l) {
        check(si_layer_create_in(st->ws, &layers[l], &st->layers[l]), "si_layer_create_in");
        hip_check(hipMalloc((void **)&st->kpool[l], pool), "hipMalloc(K pool)");
        hip_check(hipMalloc((void **)&st->vpool[l], pool), "hipMalloc(V pool)");
    }
    hip_check(hipMalloc((void **)&st->dev_table, sizeof(int) * (size_t)max_seqs * max_pages),
              "hipMalloc(page table)");
    hip_check(hipMalloc((void **)&st->dev_ctx, sizeof(int) * (size_t)max_seqs), "hipMalloc");
    const size_t act = sizeof(float) * (size_t)max_seqs * s->hidden;
    hip_check(hipMalloc((void **)&st->act[0], act), "hipMalloc(activations)");
    hip_check(hipMalloc((void **)&st->act[1], act), "hipMalloc(activations)");
    st->host_table = calloc((size_t)max_seqs * max_pages, sizeof(int));
    st->host_ctx = calloc((size_t)max_seqs, sizeof(int));
    if (!st->host_table || !st->host_ctx) die("Out of memory");
    return st;
}

void si_stack_destroy(si_stack_t *st) {
    if (!st) return;
    for (int l = 0; l < st->nlayers; ++l) {
        si_layer_destroy(st->layers[l]);
        (void)hipFree(st->kpool[l]);
        (void)hipFree(st->vpool[l]);
    }
    si_workspace_destroy(st->ws);
    (void)hipFree(st->dev_table);
    (void)hipFree(st->dev_ctx);
    (void)hipFree(st->act[0]);
    (void)hipFree(st->act[1]);
    si_kv_pages_destroy(st->pages);
    free(st->layers);
    free(st->kpool);
    free(st->vpool);
    free(st->host_table);
    free(st->host_ctx);
    free(st);
}

si_kv_pages_t *si_stack_pages(si_stack_t *st) { return st->pages; }
uint16_t *si_stack_k_pool(si_stack_t *st, int layer) { return st->kpool[layer]; }
uint16_t *si_stack_v_pool(si_stack_t *st, int layer) { return st->vpool[layer]; }
si_layer_t *si_stack_layer(si_stack_t *st, int layer) { return st->layers[layer]; }
const int *si_stack_dev_table(const si_stack_t *st) { return st->dev_table; }
const int *si_stack_dev_ctx(const si_stack_t *st) { return st->dev_ctx; }
int si_stack_nseq(const si_stack_t *st) { return st->nseq; }

/* Makes `device` current, if it is not: the one that was. */
static int switch_device(int device) {
    int was = device;
    hip_check(hipGetDevice(&was), "hipGetDevice");
    if (was != device) hip_check(hipSetDevice(device), "hipSetDevice");
    return was;
}

/* The previous step's kernels, which read the pools and the device table. */
static void wait_decode(si_stack_t *st) {
    const int was = switch_device(st->device); /* (a null stream is the current device's) */
    if (st->captured || st->streams)
        hip_check(hipDeviceSynchronize(), "si_stack: wait");
    else if (st->pending)
        hip_check(hipStreamSynchronize((hipStream_t)st->stream), "si_stack: wait");
    switch_device(was);
    st->pending = st->streams = 0;
}

static int is_capturing(void *stream) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    return stream && hipStreamIsCapturing((hipStream_t)stream, &s) == hipSuccess &&
           s != hipStreamCaptureStatusNone;
}

/* The bookkeeping's copies in every pool (after wait_decode), and until done. */
static void run_copies(si_stack_t *st) {
    const int *src, *dst;
    const int n = si_kv_copies(st->pages, &src, &dst);
    if (n == 0) return;
    void **pools = malloc(sizeof(void *) * 2 * (size_t)st->nlayers);
    if (!pools) die("Out of memory");
    for (int l = 0; l < st->nlayers; ++l) {
        pools[2 * l] = st->kpool[l];
        pools[2 * l + 1] = st->vpool[l];
    }
    const int was = switch_device(st->device);
    check(si_kv_copy_pages(pools, 2 * st->nlayers, st->page_bytes, st->npages, src, dst, n, NULL),
          "si_kv_copy_pages");
    free(pools);
    hip_check(hipStreamSynchronize(NULL), "si_stack: page copies");
    switch_device(was);
    si_kv_copies_done(st->pages);
}

int si_stack_fork(si_stack_t *st, int seq) { return si_kv_seq_fork(st->pages, seq); }

int si_stack_compact(si_stack_t *st) {
    wait_decode(st);
    run_copies(st);
    const int used = si_kv_compact(st->pages);
    run_copies(st);
    st->nseq = 0; /* the device table is the old one */
    return used;
}

int si_stack_prepare(si_stack_t *st, const int *seqs, int nseq) {
    if (nseq < 1 || nseq > st->max_seqs) die("si_stack_prepare: nseq outside 1..max_seqs");
    /* the previous step's kernels read the device table and contexts this
     * call rewrites: wait for them */
    wait_decode(st);
    for (int i = 0; i < nseq; ++i)
        for (int j = 0; j < i; ++j)
            if (seqs[i] == seqs[j]) die("si_stack_prepare: a sequence appears twice");
    si_kv_pages_t *p = st->pages;
    for (int i = 0; i < nseq; ++i) {
        const int len = si_kv_seq_len(p, seqs[i]) + 1;
        if (len > st->max_ctx) die("si_stack_prepare: a sequence exceeds max_ctx");
        if (si_kv_seq_grow(p, seqs[i], len) != 0) {
            /* roll back this call's growth so the caller can preempt; the
             * device table and contexts still describe the previous step, so
             * no decode may run until a prepare succeeds */
            for (int j = 0; j < i; ++j) p->len[seqs[j]] -= 1;
            st->nseq = 0;
            return -1;
        }
    }
    run_copies(st);
    for (int i = 0; i < nseq; ++i) {
        memcpy(st->host_table + (size_t)i * p->max_pages,
               p->table + (size_t)seqs[i] * p->max_pages, sizeof(int) * (size_t)p->max_pages);
        st->host_ctx[i] = p->len[seqs[i]];
    }
    hip_check(hipMemcpy(st->dev_table, st->host_table, sizeof(int) * (size_t)nseq * p->max_pages,
                        hipMemcpyHostToDevice), "upload page table");
    hip_check(hipMemcpy(st->dev_ctx, st->host_ctx, sizeof(int) * (size_t)nseq,
                        hipMemcpyHostToDevice), "upload contexts");
    st->nseq = nseq;
    return 0;
}

void si_stack_decode(si_stack_t *st, const float *x, float *out, int flags, void *stream) {
    if (st->nseq < 1) die("si_stack_decode: no si_stack_prepare call");
    const int capturing = is_capturing(stream);
    int max_ctx = 1;
    for (int i = 0; i < st->nseq; ++i)
        if (st->host_ctx[i] > max_ctx) max_ctx = st->host_ctx[i];
    /* the contexts of its replays are any */
    if (capturing && st->format == SI_KV_Q4) max_ctx = st->max_ctx;
    const float *in = x;
    for (int l = 0; l < st->nlayers; ++l) {
        float *o = l == st->nlayers - 1 ? out : st->act[l & 1];
        if (st->format == SI_KV_Q4)
            check(si_layer_decode_kv4(st->layers[l], in, st->nseq, (uint8_t *)st->kpool[l],
                                      (uint8_t *)st->vpool[l], st->npages, st->page_size,
                                      st->dev_table, st->pages->max_pages, st->dev_ctx, max_ctx,
                                      max_ctx, o, flags, stream),
                  "si_layer_decode_kv4");
        else
            check(si_layer_decode_paged(st->layers[l], in, st->nseq, st->kpool[l], st->vpool[l],
                                        st->npages, st->page_size, st->dev_table,
                                        st->pages->max_pages, st->dev_ctx, max_ctx, max_ctx, o,
                                        flags, stream),
                  "si_layer_decode_paged");
        in = o;
    }
    if (capturing) {
        st->captured = 1;
        return;
    }
    if (st->pending && st->stream != stream) st->streams = 1;
    st->stream = stream;
    st->pending = 1;
}
