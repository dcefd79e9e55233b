"""Forks and compaction of a model's cache where calls of the device fail: sequences hold what they held, and go on. The host side is the framework's own, compiled
here over a device in host memory whose calls fail when told to; a model's cache holds the tokens themselves."""
import ctypes as C
import os
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
HOST = ROOT / "c-ml_b200" / "host"

FAKE = r"""
#include <stdlib.h>
#include <string.h>
#include "cml_lm_internal.h"
int fail_in = -1, calls = 0;                             /* the device call that fails, counted from the next one on */
static int failed(void) { calls++; return fail_in >= 0 && fail_in-- == 0; }
const char* cmlb200_last_error(void) { return "told to"; }
int cmlb200_malloc(void** p, size_t n) { *p = calloc(1, n ? n : 1); return *p ? 0 : -1; }
int cmlb200_free(void* p) { free(p); return 0; }
int cmlb200_host_alloc_pinned(void** p, size_t n) { return cmlb200_malloc(p, n); }
int cmlb200_host_free_pinned(void* p) { free(p); return 0; }
int cmlb200_memset(void* p, int v, size_t n, void* st) { (void)st; memset(p, v, n); return 0; }
int cmlb200_memcpy_h2d(void* d, const void* s, size_t n, void* st) { (void)st; if (failed()) return -1; memcpy(d, s, n); return 0; }
int cmlb200_memcpy_d2h(void* d, const void* s, size_t n, void* st) { (void)st; memcpy(d, s, n); return 0; }
int cmlb200_stream_create(void** s) { *s = NULL; return 0; }
int cmlb200_stream_destroy(void* s) { (void)s; return 0; }
int cmlb200_stream_sync(void* s) { (void)s; return failed() ? -1 : 0; }            /* (says so after the work is done) */
static void copy(const cmlb200_pages* p, int from, int to) {
    for (int k = 0; k < p->pools; k++) memcpy((char*)p->pool[k].base + (size_t)to * p->pool[k].stride, (char*)p->pool[k].base + (size_t)from * p->pool[k].stride, p->pool[k].bytes);
}
int cmlb200_pages_copy(const cmlb200_pages* p, const int* m, int n, void* st) {
    (void)st;
    if (failed()) return -1;
    for (int i = 0; i < n; i++) {
        copy(p, m[2 * i], m[2 * i + 1]);
        for (int e = 0; p->table && e < p->slots * p->table_ld; e++) if (p->table[e] == m[2 * i]) p->table[e] = m[2 * i + 1];
    }
    return 0;
}
int cmlb200_pages_fork(const cmlb200_pages* p, const int* f, int n, void* st) {
    (void)st;
    if (failed()) return -1;
    for (int i = 0; i < n; i++, f += 4) {
        int *a = p->table + f[0] * p->table_ld, *b = p->table + f[1] * p->table_ld;
        memcpy(b, a, (size_t)f[2] * sizeof(int));
        if (f[3] >= 0) { copy(p, a[f[2]], f[3]); b[f[2]] = f[3]; }
    }
    return 0;
}
/* ---- a model whose cache is its tokens, and whose slots count them ---- */
static int *pool, *counts, g_slots;
static const int* g_table;
static int g_ld;
static void* fake_load(const char* p, const CMLJson* c, const CMLLMOptions* o, CMLLMInfo* info) { (void)p; (void)c; (void)o; info->vocab = 1000; return malloc(1); }
static void fake_free(void* m) { free(m); free(pool); free(counts); pool = counts = NULL; }
static int fake_pools_make(void* m, int blocks, int size, int slots, int ld) {
    (void)m;
    pool = calloc((size_t)blocks * (size_t)size, sizeof(int));
    counts = calloc((size_t)slots, sizeof(int));
    g_ld = ld;
    g_slots = slots;
    return 0;
}
static int fake_forward(void* m, const CMLLMBatch* b, void* st) {
    (void)m; (void)st;
    g_table = b->d_table;
    for (int r = 0; r < b->rows; r++) {
        const int p = b->d_pos[r], s = b->d_slot[r];
        pool[b->d_table[s * b->table_ld + p / 16] * 16 + p % 16] = b->d_tokens[r];
        counts[s] = p + 1;
    }
    return 0;
}
static int fake_head(void* m, const int* rows, int n, float* l, void* st) { (void)m; (void)rows; (void)n; (void)l; (void)st; return 0; }
static int fake_pools(void* m, int per_slot, cmlb200_page_pool* p, int max) {
    (void)m;
    if (max) { cmlb200_page_pool x = {per_slot ? (void*)counts : (void*)pool, per_slot ? 4 : 64, per_slot ? 4 : 64}; *p = x; }
    return 1;
}
static int fake_check(void* m, const CMLLMBatch* b) { (void)m; (void)b; return 0; }
static const CMLLMClass kFake = {.architecture = "Fake", .load = fake_load, .free = fake_free, .make_pools = fake_pools_make, .forward = fake_forward, .head = fake_head, .pools = fake_pools,
                                 .check = fake_check};
__attribute__((constructor)) static void reg(void) { cml_lm_register(&kFake); }
/* what the device would read of a sequence */
int held(int slot, int n, int* out) {
    for (int i = 0; i < n; i++) out[i] = pool[g_table[slot * g_ld + i / 16] * 16 + i % 16];
    return counts[slot];
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory, pkg):
    folder = tmp_path_factory.mktemp("fake")
    (folder / "fake.c").write_text(FAKE)
    flags = ["-std=c11", "-O1", "-fPIC", "-D_GNU_SOURCE", f"-I{ROOT / 'include'}", f"-I{HOST}", "-I/usr/local/cuda/include"]
    run = lambda *cmd: subprocess.run(cmd, check=True, capture_output=True, text=True)
    objects = []
    for src in (folder / "fake.c", HOST / "cml_lm.c", HOST / "cml_paged.c", HOST / "cml_json.c"):
        objects.append(str(folder / (src.stem + ".o")))
        run(os.environ.get("CC", "gcc"), *flags, "-c", str(src), "-o", objects[-1])
    # everything else that they refer to is not reached here
    known = {x.split()[-1] for x in run("nm", "--defined-only", *objects).stdout.splitlines() if len(x.split()) == 3}
    wanted = {x.split()[-1] for x in run("nm", "-u", *objects).stdout.splitlines() if " U " in f" {x.strip()} "}
    stubs = sorted(n for n in wanted - known if n.startswith(("cml", "tensor")))
    (folder / "stubs.c").write_text("".join(f"long {n}(void) {{ return 0; }}\n" for n in stubs))
    objects.append(str(folder / "stubs.o"))
    run(os.environ.get("CC", "gcc"), "-fPIC", "-c", str(folder / "stubs.c"), "-o", objects[-1])
    run(os.environ.get("CC", "gcc"), "-shared", "-o", str(folder / "fake.so"), *objects, "-lpthread", "-lm")
    so = C.CDLL(str(folder / "fake.so"))
    for n in ("cml_lm_load", "cml_lm_free", "cml_lm_sequence_open", "cml_lm_sequence_close", "cml_lm_sequence_fork", "cml_lm_compact", "cml_lm_step", "cml_lm_blocks_free", "cml_lm_sequence_length"):
        getattr(so, n).argtypes, getattr(so, n).restype = getattr(pkg.lib, n).argtypes, getattr(pkg.lib, n).restype
    (folder / "config.json").write_text('{"architecture": "Fake"}')
    so.folder = str(folder).encode()
    return so


class Model:
    def __init__(self, lib, pkg, tokens=800, sequences=6):
        self.L, self.pkg, self.lines = lib, pkg, {}
        self.fail, self.calls = C.c_int.in_dll(lib, "fail_in"), C.c_int.in_dll(lib, "calls")
        self.fail.value = -1
        self.h = lib.cml_lm_load(lib.folder, pkg.LMOptions(6, tokens, sequences, 0, 0))
        assert self.h

    def open(self, tokens):
        s = self.L.cml_lm_sequence_open(self.h)
        assert s >= 0
        self.lines[s] = []
        self.feed(s, tokens)
        return s

    def feed(self, s, tokens):
        t = np.ascontiguousarray(tokens, np.int32)
        assert self.L.cml_lm_step(self.h, self.pkg.LMEntry(s, t.ctypes.data, len(t), None, 0), 1, None) == 0
        self.lines[s] = self.lines[s] + list(tokens)

    def end(self, s):
        assert self.L.cml_lm_sequence_close(self.h, s) == 0
        del self.lines[s]

    def check(self):
        for s, want in self.lines.items():
            out = np.zeros(len(want), np.int32)
            assert self.L.held(s, len(want), C.c_void_p(out.ctypes.data)) == len(want) == self.L.cml_lm_sequence_length(self.h, s)
            assert out.tolist() == want

    def busy(self):
        """A pool with holes, a fork among the sequences."""
        r = np.random.default_rng(1)
        some = lambda n: r.integers(1, 1000, n).tolist()
        seqs = [self.open(some(n)) for n in (100, 37, 90)]
        for s in seqs:
            self.feed(s, some(20))
        child = self.L.cml_lm_sequence_fork(self.h, seqs[2])
        self.lines[child] = list(self.lines[seqs[2]])
        self.feed(child, some(2))
        self.end(seqs[0])
        self.check()
        return seqs[1:] + [child], some


def test_compaction(lib, pkg):
    m = Model(lib, pkg)
    seqs, some = m.busy()
    assert lib.cml_lm_compact(m.h) > 0
    m.check()
    m.open(some(60))
    m.check()
    lib.cml_lm_free(m.h)


def test_compaction_that_fails_at_any_call(lib, pkg):
    made = 0
    for n in range(20):
        m = Model(lib, pkg)
        seqs, some = m.busy()
        free = lib.cml_lm_blocks_free(m.h)
        m.fail.value = n
        rc = lib.cml_lm_compact(m.h)
        failed, m.fail.value = m.fail.value < 0, -1
        if not failed:
            assert rc > 0
            made = n
        else:
            assert rc == -1
        m.check()
        assert lib.cml_lm_blocks_free(m.h) == free
        new = m.open(some(200))                         # takes blocks that would be somebody's, were the two sides of two minds
        for s in seqs:
            m.feed(s, some(30))
        m.check()
        assert lib.cml_lm_compact(m.h) >= 0
        m.end(new)
        m.check()
        lib.cml_lm_free(m.h)
        if not failed:
            break
    assert made >= 3                                    # an upload, the copies, a wait


def test_fork_that_fails_at_any_call(lib, pkg):
    for n in range(20):
        m = Model(lib, pkg)
        seqs, some = m.busy()
        free = lib.cml_lm_blocks_free(m.h)
        m.fail.value = n
        child = lib.cml_lm_sequence_fork(m.h, seqs[0])
        failed, m.fail.value = m.fail.value < 0, -1
        assert (child < 0) == failed
        if failed:
            assert lib.cml_lm_blocks_free(m.h) == free
            child = lib.cml_lm_sequence_fork(m.h, seqs[0])
        m.lines[child] = list(m.lines[seqs[0]])
        for s in (*seqs, child):
            m.feed(s, some(30))
        m.open(some(100))
        m.check()
        lib.cml_lm_free(m.h)
        if not failed:
            assert n >= 4
            break
