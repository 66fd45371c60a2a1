"""The decode stack's host side (si_kvpages.c) on the CPU: compiled beside stand-ins for the HIP
runtime and the layers, which write down the order of what the stack asks of them.  A stream's
work counts as running until something waits for it."""
import os
import subprocess

import pytest

import si_amd

STUBS = r"""
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <hip/hip_runtime_api.h>
#include "si_host.h"

static int device, running[8], capturing, last_max, copies, copy_device, waits;
#define ID(s) ((int)(size_t)(s))   /* streams 1, 2, ..; the null stream 0 */
static void fail(const char *what) { printf("%s\n", what); exit(2); }
static void none_running(const char *what) {
    for (int i = 0; i < 8; ++i) if (running[i]) fail(what);
}
hipError_t hipGetDevice(int *d) { *d = device; return hipSuccess; }
hipError_t hipSetDevice(int d) { device = d; return hipSuccess; }
hipError_t hipMalloc(void **p, size_t n) { *p = calloc(n + 16, 1); return hipSuccess; }
hipError_t hipFree(void *p) { free(p); return hipSuccess; }
hipError_t hipMemcpy(void *d, const void *s, size_t n, hipMemcpyKind k) {
    (void)k; none_running("the tables were written below a running step"); memcpy(d, s, n);
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t s) {
    if (s || device == 0) running[ID(s)] = 0;   /* a null stream is the current device's */
    return hipSuccess;
}
hipError_t hipDeviceSynchronize(void) {
    if (device == 0) memset(running, 0, sizeof running);
    ++waits; return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus *c) {
    *c = capturing && ID(s) == capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
const char *hipGetErrorString(hipError_t e) { (void)e; return "error"; }
const char *si_last_error(void) { return "error"; }
int si_workspace_create(const si_shape_t *s, int n, int m, si_workspace_t **w) {
    (void)s; (void)n; (void)m; *w = NULL; return SI_OK;
}
int si_workspace_destroy(si_workspace_t *w) { (void)w; return SI_OK; }
int si_layer_create_in(si_workspace_t *w, const si_layer_host_t *h, si_layer_t **l) {
    (void)w; (void)h; *l = NULL; return SI_OK;
}
int si_layer_destroy(si_layer_t *l) { (void)l; return SI_OK; }
size_t si_kv4_page_bytes(const si_shape_t *s, int ps) { return (size_t)s->kvheads * ps * s->hdim / 16 * 9; }
static void decode(int max_ctx, void *stream) {
    last_max = max_ctx;
    if (ID(stream) != capturing || !capturing) running[ID(stream)] = 1;
}
int si_layer_decode_kv4(si_layer_t *l, const float *x, int nseq, uint8_t *k, uint8_t *v, int npages,
                        int ps, const int *pages, int mp, const int *ctx, int context, int max_ctx,
                        float *out, int flags, void *stream) {
    (void)l; (void)x; (void)nseq; (void)k; (void)v; (void)npages; (void)ps; (void)pages; (void)mp;
    (void)ctx; (void)context; (void)out; (void)flags; decode(max_ctx, stream); return SI_OK;
}
int si_layer_decode_paged(si_layer_t *l, const float *x, int nseq, uint16_t *k, uint16_t *v,
                          int npages, int ps, const int *pages, int mp, const int *ctx, int context,
                          int max_ctx, float *out, int flags, void *stream) {
    (void)l; (void)x; (void)nseq; (void)k; (void)v; (void)npages; (void)ps; (void)pages; (void)mp;
    (void)ctx; (void)context; (void)out; (void)flags; decode(max_ctx, stream); return SI_OK;
}
int si_kv_copy_pages(void *const *pools, int np, size_t pb, int npages, const int *src,
                     const int *dst, int n, void *stream) {
    (void)pools; (void)np; (void)pb; (void)src; (void)dst;
    none_running("pages were copied below a running step");
    for (int i = 0; i < n; ++i) if (src[i] >= npages || dst[i] >= npages) fail("past the pool");
    copies += n; copy_device = device; running[ID(stream)] = 1; return SI_OK;
}
#define S(i) ((void *)(size_t)(i))
#define CHECK(x) do { if (!(x)) fail(#x); } while (0)
int main(int argc, char **argv) {
    (void)argc;
    si_shape_t sh = {0};
    sh.hidden = 64; sh.qheads = 2; sh.kvheads = 2; sh.hdim = 32;
    static si_layer_host_t lay[1];
    const int format = atoi(argv[1]);
    si_stack_t *st = si_stack_create_kv(&sh, lay, 1, 4, 96, 12, 16, format);
    si_kv_pages_t *pg = si_stack_pages(st);
    int seqs[2] = {si_kv_seq_add(pg), 0};
    float x[64], out[64];
    for (int i = 0; i < 5; ++i) {
        CHECK(si_stack_prepare(st, seqs, 1) == 0);
        si_stack_decode(st, x, out, 0, S(1));
    }
#ifdef BODY
    BODY
#endif
    si_stack_destroy(st);
    puts("ok");
    return 0;
}
"""

BODIES = {
    # a captured step's replays run on streams that the stack was never given
    "replays": """
    CHECK(si_stack_prepare(st, seqs, 1) == 0);
    capturing = 3;
    si_stack_decode(st, x, out, 0, S(3));
    capturing = 0;
    running[4] = 1;                               /* a replay */
    seqs[1] = si_stack_fork(st, seqs[0]);
    CHECK(si_stack_prepare(st, seqs, 2) == 0 && copies == 1);
    running[5] = 1;
    si_kv_seq_free(pg, seqs[0]);
    si_stack_compact(st);
    running[4] = 1;
    CHECK(si_stack_prepare(st, seqs + 1, 1) == 0);
""",
    # contexts grow between a captured 4-bit step's replays
    "capture": """
    CHECK(si_stack_prepare(st, seqs, 1) == 0);
    si_stack_decode(st, x, out, 0, S(1));
    CHECK(last_max == 6);
    capturing = 3;
    si_stack_decode(st, x, out, 0, S(3));
    CHECK(last_max == (format == SI_KV_Q4 ? 96 : 6));
    capturing = 0;
    si_stack_decode(st, x, out, 0, S(1));
    CHECK(last_max == 6);
""",
    # the caller's current device is another one
    "device": """
    si_stack_decode(st, x, out, 0, S(0));
    si_stack_prepare(st, seqs, 1);
    si_stack_decode(st, x, out, 0, S(0));
    device = 1;
    seqs[1] = si_stack_fork(st, seqs[0]);
    CHECK(si_stack_prepare(st, seqs, 2) == 0);
    CHECK(copies == 1 && copy_device == 0 && device == 1);
    running[4] = 1;
    capturing = 3;
    si_stack_decode(st, x, out, 0, S(3));
    capturing = 0;
    CHECK(si_stack_prepare(st, seqs, 2) == 0 && device == 1);
    si_kv_seq_free(pg, seqs[0]);
    copy_device = -1;
    si_stack_compact(st);
    CHECK((copy_device == 0 || copy_device == -1) && device == 1);
""",
    # the stack's pools stay as they are: its bookkeeping may set pages aside, no more
    "resize": """
    CHECK(si_kv_pages_resize(pg, 13) == -1 && si_kv_pages_free(pg) == 11);
    CHECK(si_kv_pages_resize(pg, 2) == 0 && si_kv_pages_free(pg) == 1);
    CHECK(si_kv_pages_resize(pg, 1 << 20) == -1 && si_kv_pages_free(pg) == 1);
    CHECK(si_kv_pages_resize(pg, 12) == 0 && si_kv_pages_free(pg) == 11);
    CHECK(si_kv_seq_grow(pg, seqs[0], 96) == 0 && si_kv_pages_free(pg) == 6);
    for (int i = 0; i < 6; ++i) CHECK(si_kv_page_table(pg)[i] < 12);
""",
    "streams": """
    si_stack_decode(st, x, out, 0, S(2));         /* the same step again, on another stream */
    seqs[1] = si_stack_fork(st, seqs[0]);
    CHECK(si_stack_prepare(st, seqs, 2) == 0 && copies == 1);
    si_stack_decode(st, x, out, 0, S(1));
    const int before = waits;
    CHECK(si_stack_prepare(st, seqs, 2) == 0);    /* one stream again: it alone is waited for */
    CHECK(waits == before);
""",
}


def _run(tmp_path, body, fmt):
    src, exe = tmp_path / "stack.c", tmp_path / "stack"
    src.write_text(STUBS.replace("#ifdef BODY\n    BODY\n#endif\n", body))
    host = os.path.join(si_amd.PKG, "host", "si_kvpages.c")
    subprocess.run(["gcc", "-O1", "-std=gnu11", "-D__HIP_PLATFORM_AMD__",
                    "-I", si_amd.INCLUDE_DIR, "-I/opt/rocm/include", str(src), host, "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe), str(fmt)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


@pytest.mark.parametrize("fmt", [si_amd.SI_KV_F16, si_amd.SI_KV_Q4])
@pytest.mark.parametrize("what", list(BODIES))
def test_stack(tmp_path, what, fmt):
    _run(tmp_path, BODIES[what], fmt)
