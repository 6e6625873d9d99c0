"""The host side of sllm_gfx950_attn.h on the CPU, against the HIP stand-in of
tests/fakehip (kernels do nothing there): what is refused, with what left as it
was; the pages of sequences against a plain model of them; every HIP call
failing in turn; how a step's work is laid out."""
import ctypes
import os
import subprocess
import sys
from ctypes import byref, c_char_p, c_int, c_int32, c_long, c_uint, c_void_p

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE_DIR = os.path.join(ROOT, "tests", "fakehip")
FAKE_NAME = "libsllm_gfx950_fakehip_san.so" if os.environ.get("SLLM_FAKEHIP_SAN") else "libsllm_gfx950_fakehip.so"
ARG, NOMEM, NO_DEVICE, HIP = -1, -2, -60, -61
F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def L(amd):
    import fcntl
    with open(os.path.join(FAKE_DIR, ".build.lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        r = subprocess.run(["make", "-s", "-C", FAKE_DIR, FAKE_NAME], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    lib = amd._bind(os.path.join(FAKE_DIR, FAKE_NAME), amd.PROTOTYPES)
    for name, res, args in (("fakehip_fail", None, [c_char_p, c_int, c_uint]), ("fakehip_clear", None, []),
                            ("fakehip_fired", c_int, []), ("fakehip_live", c_long, []), ("fakehip_launches", c_char_p, []),
                            ("fakehip_current", None, [c_int]), ("fakehip_capture", None, [c_int])):
        getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    # no cache yet: every call says that there is no device
    d = amd.PagesDesc(1, 1, 64, 16, 4, F32, None)
    p, one = c_void_p(), c_int32()
    for st in (lib.sllm_gfx950_pages_new(byref(d), byref(p)), lib.sllm_gfx950_seq_new(None, byref(one)),
               lib.sllm_gfx950_seq_fork(None, 0, 0, 0, None), lib.sllm_gfx950_seq_copy(None, None, 0, None),
               lib.sllm_gfx950_seq_truncate(None, 0, 0), lib.sllm_gfx950_seq_free(None, None, 0),
               lib.sllm_gfx950_seq_len(None, 0), lib.sllm_gfx950_seq_tables(None, None, 0, None, 0),
               lib.sllm_gfx950_pages_compact(None, None), lib.sllm_gfx950_batch_create(None, None, None, 0, 1, 0, byref(p)),
               lib.sllm_gfx950_batch_store(None, 0, None, 0, None, 0), lib.sllm_gfx950_batch_attend(None, 0, None, 0, 1.0, None, 0),
               lib.sllm_gfx950_prompt_create(None, byref(p)), lib.sllm_gfx950_prompt_attend(None, None)):
        assert st == NO_DEVICE
    assert lib.sllm_gfx950_open(0) == 0
    yield lib
    lib.sllm_gfx950_close()
    assert lib.fakehip_live() == 0


def I(*v):
    return (c_int32 * max(len(v), 1))(*v)


class Cache:
    def __init__(self, amd, L, n_pages=20, page=16, kv=2, d=64, layers=2, dtype=F32):
        self.L, self.p, self.page = L, c_void_p(), page
        desc = amd.PagesDesc(layers, kv, d, page, n_pages, dtype, None)
        assert L.sllm_gfx950_pages_new(byref(desc), byref(self.p)) == 0

    def new(self):
        s = c_int32()
        assert self.L.sllm_gfx950_seq_new(self.p, byref(s)) == 0
        return s.value

    def batch(self, seqs, n_new, n_head=4, act=F32, status=0):
        b = c_void_p()
        st = self.L.sllm_gfx950_batch_create(self.p, I(*seqs), I(*n_new), len(seqs), n_head, act, byref(b))
        assert st == status, (st, self.err())
        return b

    def grow(self, seqs, n_new):
        self.L.sllm_gfx950_batch_destroy(self.batch(seqs, n_new))

    def fork(self, s, n_tokens, n, status=0):
        out = I(*[-7] * n)
        st = self.L.sllm_gfx950_seq_fork(self.p, s, n_tokens, n, out)
        assert st == status, (st, self.err())
        return list(out[:n])

    def table(self, s):
        out = I(*[-7] * 500)
        n = self.L.sllm_gfx950_seq_tables(self.p, I(s), 1, out, 500)
        assert n >= 0
        return list(out[:n])

    def state(self, seqs):
        return self.L.sllm_gfx950_pages_in_use(self.p), [(self.L.sllm_gfx950_seq_len(self.p, s), self.table(s)) for s in seqs]

    def err(self):
        return self.L.sllm_gfx950_last_error().decode()

    def close(self):
        self.L.sllm_gfx950_pages_free(self.p)


@pytest.mark.parametrize("field,value", [("n_layer", 0), ("n_head_kv", 0), ("n_head_kv", 1025), ("head_dim", 0), ("head_dim", 12),
                                         ("head_dim", 136), ("page_tokens", 8), ("page_tokens", 24), ("page_tokens", 2048),
                                         ("n_pages", 0), ("dtype", 3), ("dtype", -1), ("mem", 8), ("n_layer", 65537)])
def test_caches_that_are_refused(amd, L, field, value):
    d = amd.PagesDesc(2, 2, 64, 16, 4, F16, None)
    assert L.sllm_gfx950_pages_bytes(byref(d)) == 4 * 2 * 2 * 2 * 16 * 64 * 2
    setattr(d, field, value)
    p, live = c_void_p(1), L.fakehip_live()
    assert L.sllm_gfx950_pages_new(byref(d), byref(p)) == ARG and not p.value
    assert L.sllm_gfx950_last_error() and L.fakehip_live() == live
    if field != "mem":
        assert L.sllm_gfx950_pages_bytes(byref(d)) == 0
    big = amd.PagesDesc(60000, 1000, 128, 1024, 4, F32, None)       # a page over 4 GiB
    assert L.sllm_gfx950_pages_new(byref(big), byref(p)) == ARG
    assert L.sllm_gfx950_pages_new(None, byref(p)) == ARG and L.sllm_gfx950_pages_new(byref(d), None) == ARG


def test_sequences_that_are_refused(amd, L):
    c = Cache(amd, L)
    a, b = c.new(), c.new()
    c.grow([a, b], [40, 16])
    was = c.state([a, b])
    out = I(0, 0, 0)
    for st in (L.sllm_gfx950_seq_fork(c.p, 7, 0, 1, out), L.sllm_gfx950_seq_fork(c.p, -1, 0, 1, out),
               L.sllm_gfx950_seq_fork(c.p, a, 41, 1, out), L.sllm_gfx950_seq_fork(c.p, a, -1, 1, out),
               L.sllm_gfx950_seq_fork(c.p, a, 4, -1, out), L.sllm_gfx950_seq_fork(c.p, a, 4, 1, None),
               L.sllm_gfx950_seq_copy(c.p, I(a, 9), 2, out), L.sllm_gfx950_seq_copy(c.p, None, 1, out),
               L.sllm_gfx950_seq_truncate(c.p, a, 41), L.sllm_gfx950_seq_truncate(c.p, a, -1),
               L.sllm_gfx950_seq_truncate(c.p, 5, 0), L.sllm_gfx950_seq_free(c.p, I(a, a), 2),
               L.sllm_gfx950_seq_free(c.p, I(b, 3), 2), L.sllm_gfx950_seq_free(c.p, None, 1), L.sllm_gfx950_seq_len(c.p, 2),
               L.sllm_gfx950_seq_tables(c.p, I(a, 2), 2, out, 3), L.sllm_gfx950_seq_tables(c.p, I(a), 1, None, 3)):
        assert st == ARG
    assert L.sllm_gfx950_seq_fork(c.p, a, 33, 20, I(*range(20))) == NOMEM           # a page for each
    assert L.sllm_gfx950_seq_copy(c.p, I(*[a] * 6), 6, I(*range(6))) == NOMEM
    assert L.sllm_gfx950_seq_tables(c.p, I(a, b), 2, out, 3) == 4 and list(out) == [0, 0, 0]    # they do not fit
    assert c.state([a, b]) == was
    # a page that only partly belongs to the fork costs one; whole pages cost none
    f = c.fork(a, 32, 3)
    assert c.state([a, b]) == was and all(c.table(x) == was[1][0][1][:2] for x in f)
    c.close()


def test_batches_that_are_refused(amd, L):
    c = Cache(amd, L)
    a, b = c.new(), c.new()
    c.grow([a], [10])
    was = c.state([a, b])
    x = c_void_p(1)
    for seqs, new, heads, act in (([a, a], [1, 1], 4, F32), ([a, 5], [1, 1], 4, F32), ([a], [-1], 4, F32), ([a], [1], 3, F32),
                                  ([a], [1], 0, F32), ([a], [1], 2048, F32), ([a], [1], 4, F16), ([a], [1], 4, 3),
                                  ([a, b], [1 << 22, 1], 4, F32), ([a], [(1 << 28) - 5], 4, F32)):
        assert L.sllm_gfx950_batch_create(c.p, I(*seqs), I(*new), len(seqs), heads, act, byref(x)) == ARG and not x.value
    assert L.sllm_gfx950_batch_create(c.p, None, I(1), 1, 4, F32, byref(x)) == ARG
    assert L.sllm_gfx950_batch_create(c.p, I(a), I(1), -1, 4, F32, byref(x)) == ARG
    assert L.sllm_gfx950_batch_create(None, I(a), I(1), 1, 4, F32, byref(x)) == ARG
    assert L.sllm_gfx950_batch_create(c.p, I(a), I(1), 1, 4, F32, None) == ARG
    c.batch([a, b], [300, 20], status=NOMEM)
    assert c.state([a, b]) == was
    # a batch's own calls
    b1 = c.batch([a, b], [3, 0])
    assert L.sllm_gfx950_batch_rows(b1) == 3
    mem = c_void_p()
    assert L.sllm_gfx950_malloc(byref(mem), 1 << 16) == 0
    m = (mem.value + 15) // 16 * 16
    bad = [L.sllm_gfx950_batch_store(b1, 2, m, 0, m, 0), L.sllm_gfx950_batch_store(b1, -1, m, 0, m, 0),
           L.sllm_gfx950_batch_store(b1, 0, None, 0, m, 0), L.sllm_gfx950_batch_store(b1, 0, m, 0, m + 4, 0),
           L.sllm_gfx950_batch_store(b1, 0, m, 127, m, 0), L.sllm_gfx950_batch_store(b1, 0, m, 130, m, 0),
           L.sllm_gfx950_batch_store(b1, 0, m, 0, m, 1 << 40)]
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        bad.append(L.sllm_gfx950_batch_attend(b1, 0, m, 0, scale, m, 0))
    bad += [L.sllm_gfx950_batch_attend(b1, 0, None, 0, 1.0, m, 0), L.sllm_gfx950_batch_attend(b1, 0, m, 0, 1.0, m + 8, 0),
            L.sllm_gfx950_batch_attend(b1, 5, m, 0, 1.0, m, 0), L.sllm_gfx950_batch_attend(b1, 0, m, 255, 1.0, m, 0),
            L.sllm_gfx950_batch_attend(b1, 0, m, 0, 1.0, m, 64), L.sllm_gfx950_pages_compact(c.p, None)]
    assert bad == [ARG] * len(bad)
    assert L.sllm_gfx950_batch_store(b1, 1, m, 128, m, 132) == 0 and L.sllm_gfx950_batch_attend(b1, 1, m, 256, 1.0, m, 0) == 0
    # nothing to do, nothing needed
    b2 = c.batch([], [])
    assert L.sllm_gfx950_batch_store(b2, 0, None, 0, None, 0) == 0 and L.sllm_gfx950_batch_attend(b2, 0, None, 0, 1.0, None, 0) == 0
    L.sllm_gfx950_batch_destroy(b1)
    L.sllm_gfx950_batch_destroy(b2)
    assert L.sllm_gfx950_pages_compact(c.p, None) == 0
    L.sllm_gfx950_free(mem)
    c.close()


def test_prompts_that_are_refused(amd, L):
    q, k = I(5, 6), I(5, 9)
    ptr = lambda a: ctypes.cast(a, c_void_p)  # noqa: E731
    x = c_void_p(1)
    for over in ({"dtype": 4}, {"n_head": 3}, {"n_head_kv": 0}, {"head_dim": 20}, {"head_dim": 256}, {"n_seq": -1}, {"q_len": None},
                 {"q_len": ptr(I(5, -1))}, {"k_len": ptr(I(-5, 1))}, {"q_len": ptr(I(1 << 22, 1))}):
        d = amd.PromptDesc(F16, 4, 2, 64, 2, ptr(q), ptr(k))
        for n, v in over.items():
            setattr(d, n, v)
        assert L.sllm_gfx950_prompt_create(byref(d), byref(x)) == ARG and not x.value, over
    d = amd.PromptDesc(F16, 4, 2, 64, 2, ptr(q), ptr(k))
    assert L.sllm_gfx950_prompt_create(None, byref(x)) == ARG and L.sllm_gfx950_prompt_create(byref(d), None) == ARG
    assert L.sllm_gfx950_prompt_create(byref(d), byref(x)) == 0
    mem = c_void_p()
    assert L.sllm_gfx950_malloc(byref(mem), 1 << 16) == 0
    m = (mem.value + 15) // 16 * 16

    def call(**over):
        io = amd.PromptIO(m, m + 8192, m + 16384, m + 32768, 0.125)
        for n, v in over.items():
            setattr(io, n, v)
        return L.sllm_gfx950_prompt_attend(x, byref(io))

    assert call() == 0
    for over in ({"scale": 0.0}, {"scale": float("nan")}, {"q": None}, {"k": None}, {"v": m + 2}, {"out": None}, {"out": m + 8},
                 {"q_tok": 257, "q_head": 64}, {"k_tok": 128, "k_head": 4}, {"out_tok": 128, "out_head": 64},
                 {"out_tok": 256, "out_head": 32}, {"out_tok": 8, "out_head": 64}, {"v_tok": 1 << 33, "v_head": 64}):
        assert call(**over) == ARG, over
    assert call(out_tok=64, out_head=64 * 11) == 0 and call(q_tok=0, q_head=64) == 0    # [head][token]; one row for all tokens
    assert L.sllm_gfx950_prompt_attend(None, None) == ARG
    L.sllm_gfx950_prompt_destroy(x)
    # no sequences, or none with rows
    for lens in ((), (0, 0)):
        a = I(*lens)
        d = amd.PromptDesc(F32, 4, 2, 64, len(lens), ptr(a) if lens else None, None)
        assert L.sllm_gfx950_prompt_create(byref(d), byref(x)) == 0
        assert call(q=None, k=None, v=None, out=None) == 0
        L.sllm_gfx950_prompt_destroy(x)
    L.sllm_gfx950_free(mem)


class Pages:
    """Who holds which page, said plainly."""

    def __init__(self, n, page):
        self.n, self.page, self.seq = n, page, {}

    def used(self):
        return {p for _, t in self.seq.values() for p in t}

    def take(self):
        used = self.used()
        return next(i for i in range(self.n) if i not in used)

    def step(self, seqs, n_new):
        """(copies on write first, then new pages, sequence by sequence)"""
        shared = {s: sum(self.seq[s][1][-1:] == t[len(self.seq[s][1]) - 1:len(self.seq[s][1])] for _, t in self.seq.values())
                  for s in seqs if self.seq[s][0] % self.page}
        held = self.used()

        def take():
            i = next(i for i in range(self.n) if i not in held)
            held.add(i)
            return i

        for s, n in zip(seqs, n_new):
            length, t = self.seq[s]
            t = list(t)
            if n and shared.get(s, 0) > 1:
                t[-1] = take()
            length += n
            while len(t) * self.page < length:
                t.append(take())
            self.seq[s] = (length, t)

    def compact(self):
        used = sorted(self.used())
        n = len(used)
        holes = [i for i in range(n) if i not in used]
        to = dict(zip([p for p in used if p >= n], holes))
        self.seq = {s: (k, [to.get(p, p) for p in t]) for s, (k, t) in self.seq.items()}
        return len(to)


@pytest.mark.parametrize("seed", range(6))
def test_pages_against_a_plain_model(amd, L, seed):
    r, n_pages, page = np.random.RandomState(seed), 60, 16
    c, m = Cache(amd, L, n_pages, page, kv=1, layers=1), Pages(n_pages, page)
    for _ in range(500):
        live = sorted(m.seq)
        free = n_pages - len(m.used())
        assert L.sllm_gfx950_pages_in_use(c.p) == len(m.used())
        what, pick = r.randint(8), live[r.randint(len(live))] if live else None
        if what == 0 or pick is None:
            m.seq[c.new()] = (0, [])
        elif what <= 2:
            seqs = [int(s) for s in r.permutation(live)[:r.randint(1, 5)]]
            n_new = [int(r.choice([0, 1, 5, 16, 33])) for _ in seqs]
            if free > 20:
                c.grow(seqs, n_new)
                m.step(seqs, n_new)
        elif what == 3 and len(live) < 20:
            keep, n = int(r.randint(0, m.seq[pick][0] + 1)), int(r.randint(0, 4))
            want = n if keep % page else 0
            out = c.fork(pick, keep, n, status=NOMEM if want > free else 0)
            for f in out if want <= free else []:
                t = m.seq[pick][1][:keep // page]
                m.seq[f] = (keep, t)
                if keep % page:
                    m.seq[f] = (keep, t + [m.take()])
        elif what == 4 and len(live) < 20:
            out = I(0)
            st = L.sllm_gfx950_seq_copy(c.p, I(pick), 1, out)
            assert st == (NOMEM if len(m.seq[pick][1]) > free else 0)
            if st == 0:
                m.seq[out[0]] = (m.seq[pick][0], [])
                for _ in m.seq[pick][1]:
                    m.seq[out[0]][1].append(m.take())
        elif what == 5:
            keep = int(r.randint(0, m.seq[pick][0] + 1))
            assert L.sllm_gfx950_seq_truncate(c.p, pick, keep) == 0
            m.seq[pick] = (keep, m.seq[pick][1][:-(-keep // page)])
        elif what == 6:
            assert L.sllm_gfx950_seq_free(c.p, I(pick), 1) == 0
            del m.seq[pick]
        elif r.randint(4) == 0:
            moved = c_int32()
            assert L.sllm_gfx950_pages_compact(c.p, byref(moved)) == 0
            assert moved.value == m.compact()
        for s, (n, t) in m.seq.items():
            assert L.sllm_gfx950_seq_len(c.p, s) == n and c.table(s) == t, s
    c.close()


def test_an_open_batch_holds_its_pages(amd, L):
    c = Cache(amd, L)
    a, b = c.new(), c.new()
    c.grow([a], [50])
    batch = c.batch([a], [1])
    assert L.sllm_gfx950_seq_free(c.p, I(a), 1) == 0
    assert L.sllm_gfx950_pages_in_use(c.p) == 4
    c.grow([b], [20])
    assert c.table(b) == [4, 5]                     # not a's, which the batch may still write
    L.sllm_gfx950_batch_destroy(batch)
    assert L.sllm_gfx950_pages_in_use(c.p) == 2
    # a cache freed under a batch goes when the batch does
    batch = c.batch([b], [1])
    live = L.fakehip_live()
    c.close()
    assert L.fakehip_live() == live
    L.sllm_gfx950_batch_destroy(batch)
    assert L.fakehip_live() < live


def test_a_sequence_truncated_into_a_shared_page_gets_its_own(amd, L):
    c = Cache(amd, L)
    a = c.new()
    c.grow([a], [64])
    x, y = c.fork(a, 64, 2)
    assert L.sllm_gfx950_seq_truncate(c.p, x, 40) == 0 and L.sllm_gfx950_seq_truncate(c.p, y, 40) == 0
    L.fakehip_clear()
    c.grow([x, y], [1, 0])
    assert c.table(x) == [0, 1, 4] and c.table(y) == [0, 1, 2] and c.table(a) == [0, 1, 2, 3]
    assert b"sllm_k_attn_copy" in L.fakehip_launches()
    c.close()


def launches(L):
    out = {}
    for x in L.fakehip_launches().decode().split():
        name, grid = x.rsplit(":", 1)
        out[name] = out.get(name, 0) + int(grid)
    return out


def test_how_a_step_is_laid_out(amd, L):
    """Shared pages are one segment for all who share them: its workgroups do not
    grow with their number."""
    c = Cache(amd, L, 600, 16, kv=2, d=64, layers=1)
    a = c.new()
    c.grow([a], [1000])
    mem = c_void_p()
    assert L.sllm_gfx950_malloc(byref(mem), 1 << 20) == 0
    m = (mem.value + 15) // 16 * 16

    def step(seqs, n_new, heads=8):
        b = c.batch(seqs, n_new, heads)
        L.fakehip_clear()
        assert L.sllm_gfx950_batch_attend(b, 0, m, 0, 1.0, m, 0) == 0
        got = launches(L)
        L.sllm_gfx950_batch_destroy(b)
        return got

    alone = c.new()
    assert step([alone], [1]) == {"sllm_k_attend_f32_64": 2}         # one part: straight to the output
    got = step([a], [1])
    assert any(k.startswith("sllm_k_attn_join_f32_64") for k in got) and got["sllm_k_attend_f32_64"] > 2
    counts = []
    for n in (8, 16, 32):
        kids = c.fork(a, 1000, n)
        # each has keys of its own from position 992 on, once for each KV head
        counts.append(step(kids, [1] * n)["sllm_k_attend_f32_64"] - 2 * n)
        assert L.sllm_gfx950_seq_free(c.p, I(*kids), n) == 0
    assert all(0 < x <= 64 for x in counts), counts
    assert step([alone], [100]) == {"sllm_k_attend_f32_64": 8}       # 400 rows of each KV head: four tiles
    L.sllm_gfx950_free(mem)
    c.close()


def test_every_failed_hip_call(amd, L):
    """Out of memory: -2, any other failure: -61; nothing is kept, sequences and
    pages are as before, and the same call then works."""
    c = Cache(amd, L, 400)
    a, b, gap = c.new(), c.new(), c.new()
    c.grow([gap, a, b], [16, 100, 20])
    assert L.sllm_gfx950_seq_free(c.p, I(gap), 1) == 0
    kid = c.fork(a, 96, 1)[0]
    assert L.sllm_gfx950_seq_truncate(c.p, kid, 90) == 0
    big = c.batch([b], [900])
    mem = c_void_p()
    assert L.sllm_gfx950_malloc(byref(mem), 1 << 22) == 0
    m = (mem.value + 15) // 16 * 16
    q = I(5, 300)
    io = amd.PromptIO(m, m, m, m + (1 << 21), 1.0)
    plan = c_void_p()
    pd = amd.PromptDesc(F32, 4, 2, 64, 2, ctypes.cast(q, c_void_p), None)
    assert L.sllm_gfx950_prompt_create(byref(pd), byref(plan)) == 0
    seqs = [a, b, kid]
    sizes = [1]

    def pages_new():
        p = c_void_p()
        d = amd.PagesDesc(1, 1, 64, 16, 4, F32, None)
        return L.sllm_gfx950_pages_new(byref(d), byref(p)), lambda: L.sllm_gfx950_pages_free(p)

    def fork():
        out = I(0, 0)
        return L.sllm_gfx950_seq_fork(c.p, a, 50, 2, out), lambda: L.sllm_gfx950_seq_free(c.p, out, 2)

    def copy():
        out = I(0)
        return L.sllm_gfx950_seq_copy(c.p, I(a), 1, out), lambda: L.sllm_gfx950_seq_free(c.p, out, 1)

    def batch():
        x = c_void_p()
        # a copy on write among it; more heads than the last that worked, so that no kept buffer is enough
        st = L.sllm_gfx950_batch_create(c.p, I(*seqs), I(1500, 3, 1), 3, 4 * sizes[0], F32, byref(x))

        def undo():
            sizes[0] *= 4
            L.sllm_gfx950_batch_destroy(x)
            for s, n in ((a, 100), (b, 920), (kid, 90)):
                assert L.sllm_gfx950_seq_truncate(c.p, s, n) == 0
        return st, undo

    def prompt():
        x = c_void_p()
        return L.sllm_gfx950_prompt_create(byref(pd), byref(x)), lambda: L.sllm_gfx950_prompt_destroy(x)

    nothing = lambda: None  # noqa: E731
    calls = {"pages_new": pages_new, "fork": fork, "copy": copy, "batch": batch, "prompt": prompt,
             "store": lambda: (L.sllm_gfx950_batch_store(big, 0, m, 0, m, 0), nothing),
             "attend": lambda: (L.sllm_gfx950_batch_attend(big, 0, m, 0, 1.0, m, 0), nothing),
             "prompt_attend": lambda: (L.sllm_gfx950_prompt_attend(plan, byref(io)), nothing)}
    points = {}
    for name, call in calls.items():
        for fn, err, want in ((b"hipMalloc", 2, NOMEM), (b"hipHostMalloc", 2, NOMEM), (b"*", 1, HIP)):
            k = 0
            while True:
                was = c.state(seqs)
                live = L.fakehip_live()
                L.fakehip_fail(fn, err, k)
                st, undo = call()
                fired = L.fakehip_fired()
                L.fakehip_clear()
                if not fired:
                    assert st == 0, (name, c.err())
                    undo()
                    break
                assert st == want and L.sllm_gfx950_last_error(), (name, fn, k, st)
                assert c.state(seqs) == was and L.fakehip_live() <= live, (name, fn, k)
                k += 1
            points[name, fn] = k
    assert all(points[n, b"*"] > 0 for n in calls) and points["batch", b"hipMalloc"] > 0 and points["batch", b"hipHostMalloc"] > 0
    L.sllm_gfx950_batch_destroy(big)
    # compaction that fails moves nothing
    was = c.state(seqs)
    L.fakehip_fail(b"hipModuleLaunchKernel", 1, 0)
    assert L.sllm_gfx950_pages_compact(c.p, None) == HIP and c.state(seqs) == was
    L.fakehip_clear()
    assert L.sllm_gfx950_pages_compact(c.p, None) == 0 and c.state(seqs) != was
    L.sllm_gfx950_prompt_destroy(plan)
    L.sllm_gfx950_free(mem)
    c.close()


def test_another_current_device(amd, L):
    """Memory and launches are the library's device's whichever is current, and the
    caller's is current again afterwards."""
    L.fakehip_current(1)
    try:
        c = Cache(amd, L, 40)
        a = c.new()
        c.grow([a], [40])
        kid = c.fork(a, 37, 1)[0]
        b = c.batch([a, kid], [3, 1])
        mem = (c_int32 * 4096)()
        m = (ctypes.addressof(mem) + 15) // 16 * 16
        assert L.sllm_gfx950_batch_store(b, 0, m, 0, m, 0) == 0
        assert L.sllm_gfx950_batch_attend(b, 0, m, 0, 1.0, m, 0) == 0
        L.sllm_gfx950_batch_destroy(b)
        out, plan, q = I(0), c_void_p(), I(5)
        assert L.sllm_gfx950_seq_copy(c.p, I(a), 1, out) == 0
        assert L.sllm_gfx950_seq_free(c.p, I(a), 1) == 0 and L.sllm_gfx950_pages_compact(c.p, None) == 0
        d = amd.PromptDesc(F32, 4, 2, 64, 1, ctypes.cast(q, c_void_p), None)
        assert L.sllm_gfx950_prompt_create(byref(d), byref(plan)) == 0
        assert L.sllm_gfx950_prompt_attend(plan, byref(amd.PromptIO(m, m, m, m, 1.0))) == 0
        x = c_void_p()
        assert L.sllm_gfx950_malloc(byref(x), 16) != 0           # device 1 still is the current one
        L.sllm_gfx950_prompt_destroy(plan)
        c.close()
    finally:
        L.fakehip_current(0)


def test_pages_do_not_change_hands_in_a_capture(amd, L):
    """What takes pages or lays out work is refused while the stream is captured,
    with everything as it was; a batch's own launches are not."""
    c = Cache(amd, L, 40)
    a, gone = c.new(), c.new()
    c.grow([gone, a], [20, 40])
    assert L.sllm_gfx950_seq_free(c.p, I(gone), 1) == 0
    b = c.batch([a], [1])
    was, live = c.state([a]), L.fakehip_live()
    mem = (c_int32 * 4096)()
    m = (ctypes.addressof(mem) + 15) // 16 * 16
    L.fakehip_capture(1)
    try:
        c.batch([a], [1], status=ARG)
        c.fork(a, 33, 2, status=ARG)
        out, plan, q = I(0), c_void_p(), I(5)
        assert L.sllm_gfx950_seq_copy(c.p, I(a), 1, out) == ARG and "captured" in c.err()
        d = amd.PromptDesc(F32, 4, 2, 64, 1, ctypes.cast(q, c_void_p), None)
        assert L.sllm_gfx950_prompt_create(byref(d), byref(plan)) == ARG and not plan.value
        assert L.sllm_gfx950_batch_store(b, 0, m, 0, m, 0) == 0
        assert L.sllm_gfx950_batch_attend(b, 0, m, 0, 1.0, m, 0) == 0
        L.sllm_gfx950_batch_destroy(b)
        assert L.sllm_gfx950_pages_compact(c.p, None) == ARG and "captured" in c.err()
        assert c.state([a]) == was and L.fakehip_live() == live
    finally:
        L.fakehip_capture(0)
    assert L.sllm_gfx950_pages_compact(c.p, None) == 0 and c.state([a]) != was
    c.close()


def test_prompts_of_more_rows_than_32_bits_count(amd, L):
    """4 Mi tokens x 1024 heads of one KV head: refused, not taken as none."""
    q, plan = I(1 << 22), c_void_p()
    for heads in (1024, 512):
        d = amd.PromptDesc(F32, heads, 1, 64, 1, ctypes.cast(q, c_void_p), None)
        assert L.sllm_gfx950_prompt_create(byref(d), byref(plan)) == ARG and not plan.value


def test_a_long_row_beside_many_short_prompts(amd, L):
    """Small tiles for the one's sake would be more than a launch takes."""
    n = 30000
    q, k = I(1, *[64] * n), I(1 << 21, *[64] * n)
    plan = c_void_p()
    d = amd.PromptDesc(F32, 128, 16, 64, n + 1, ctypes.cast(q, c_void_p), ctypes.cast(k, c_void_p))
    assert L.sllm_gfx950_prompt_create(byref(d), byref(plan)) == 0, L.sllm_gfx950_last_error()
    L.sllm_gfx950_prompt_destroy(plan)


def test_threads_on_one_cache(amd, L):
    """Calls from several threads exclude each other: no page is lost."""
    import threading
    c = Cache(amd, L, 600)
    base = c.new()
    c.grow([base], [100])
    bad = []

    def work(i):
        try:
            for _ in range(30):
                s = c.fork(base, 90 + i, 2)
                b = c.batch(s, [20, i])
                assert L.sllm_gfx950_seq_truncate(c.p, s[0], 64) == 0
                assert L.sllm_gfx950_seq_free(c.p, I(*s), 2) == 0
                L.sllm_gfx950_batch_destroy(b)
        except AssertionError as e:
            bad.append(e)

    t = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for x in t:
        x.start()
    for x in t:
        x.join()
    assert not bad and L.sllm_gfx950_pages_in_use(c.p) == 7 and c.table(base) == list(range(7))
    c.close()


def test_under_asan_and_ubsan():
    """This file's other tests against the sanitizer build."""
    if os.environ.get("SLLM_FAKEHIP_SAN"):
        pytest.skip("this is that run")
    asan = subprocess.run(["gcc", "-print-file-name=libasan.so"], capture_output=True, text=True).stdout.strip()
    if not os.path.isabs(asan) or not os.path.exists(asan):
        pytest.skip("gcc's AddressSanitizer runtime is not installed")
    env = dict(os.environ, SLLM_FAKEHIP_SAN="1", UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1",
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1",
               LD_PRELOAD=asan + (":" + os.environ["LD_PRELOAD"] if os.environ.get("LD_PRELOAD") else ""))
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", os.path.abspath(__file__)],
                       cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0 and "AddressSanitizer" not in out and "runtime error:" not in out, out[-5000:]
