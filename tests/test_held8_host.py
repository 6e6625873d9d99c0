"""The host side of a cache of 8 bits, of rotary positions and of reordered sequences
(sllm_gfx950_attn.h) on the CPU, against the HIP stand-in of tests/fakehip: what is
refused, with what left as it was; the pages of reordered sequences against a plain
model; every HIP call failing in turn; which kernels run."""
import ctypes
import os
import random
import subprocess
import sys
from ctypes import byref, c_int32, c_void_p

import numpy as np
import pytest

from test_attn_host import ARG, BF16, F16, F32, HIP, NOMEM, ROOT, Cache, I, L  # noqa: F401  (the fixture)

I8, E4M3 = 4, 5


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_caches(amd, L, dtype):
    d = amd.PagesDesc(2, 3, 80, 16, 4, dtype, None)
    assert L.sllm_gfx950_pages_bytes(byref(d)) == 4 * 2 * 2 * 3 * 16 * 81
    for field, value in (("head_dim", 72), ("head_dim", 8), ("head_dim", 144), ("page_tokens", 8), ("dtype", 6), ("dtype", 3)):
        bad = amd.PagesDesc(2, 3, 80, 16, 4, dtype, None)
        setattr(bad, field, value)
        p = c_void_p(1)
        assert L.sllm_gfx950_pages_bytes(byref(bad)) == 0
        assert L.sllm_gfx950_pages_new(byref(bad), byref(p)) == ARG and not p.value


@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_batches(amd, L, dtype):
    c = Cache(amd, L, dtype=dtype)
    a, b = c.new(), c.new()
    for act in (F32, F16, BF16):
        x = c.batch([a, b], [3, 1], act=act)
        assert L.sllm_gfx950_batch_positions(x) == sum(L.sllm_gfx950_seq_len(c.p, s) for s in (a, b))
        L.sllm_gfx950_batch_destroy(x)
    was = c.state([a, b])
    for act in (I8, E4M3, 3, -1):
        c.batch([a], [1], act=act, status=ARG)
    assert c.state([a, b]) == was
    c.close()
    for dt in (F32, F16, BF16):                     # 8 bits are of a cache alone
        c = Cache(amd, L, dtype=dt)
        for act in (I8, E4M3):
            c.batch([c.new()], [1], act=act, status=ARG)
        c.close()
    p = c_void_p()
    one = I(4)
    for dt in (I8, E4M3):
        desc = amd.PromptDesc(dt, 4, 2, 64, 1, ctypes.cast(one, c_void_p), None)
        assert L.sllm_gfx950_prompt_create(byref(desc), byref(p)) == ARG


def test_which_kernels_run(amd, L):
    mem = (ctypes.c_uint8 * (1 << 16))()
    at = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    for dtype, name in ((I8, "i8"), (E4M3, "e4m3")):
        for d, wide in ((64, 64), (80, 128)):
            for act, rows in ((F32, "f32"), (F16, "f16"), (BF16, "bf16")):
                c = Cache(amd, L, dtype=dtype, d=d)
                s = c.new()
                b = c.batch([s], [20], act=act)
                L.fakehip_clear()
                assert L.sllm_gfx950_batch_store(b, 1, at, 0, at, 0) == 0
                assert L.sllm_gfx950_batch_attend(b, 1, at, 0, 1.0, at + 32768, 0) == 0
                assert L.sllm_gfx950_batch_read(b, 1, at, 0, at + 32768, 0) == 0
                got = [x.split(":")[0] for x in L.fakehip_launches().decode().split()]
                assert got == [f"sllm_k_attn_rows_{rows}", f"sllm_k_attend_{rows}{name}_{wide}", f"sllm_k_attn_read_{rows}"]
                L.fakehip_clear()
                c.fork(s, 19, 1)
                assert L.fakehip_launches().decode().split()[0].startswith("sllm_k_attn_copy8:")
                L.sllm_gfx950_batch_destroy(b)
                c.close()


def test_reads_that_are_refused(amd, L):
    c = Cache(amd, L, dtype=I8)                     # 2 layers, 2 heads of 64
    s = c.new()
    b = c.batch([s], [20], act=F16)
    mem = (ctypes.c_uint8 * (1 << 16))()
    at = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    k, v = at, at + 20 * 256
    L.fakehip_clear()
    for args in ((-1, k, 0, v, 0), (2, k, 0, v, 0), (0, None, 0, v, 0), (0, k, 0, None, 0), (0, k + 2, 0, v, 0), (0, k, 0, v + 8, 0),
                 (0, k, 120, v, 0), (0, k, 0, v, 132), (0, k, 0, k, 0), (0, k, 0, v - 16, 0), (0, k, 256, k + 240, 256)):
        assert L.sllm_gfx950_batch_read(b, *args) == ARG, args
    assert L.sllm_gfx950_batch_read(None, 0, k, 0, v, 0) == ARG
    assert L.fakehip_launches() == b""
    assert L.sllm_gfx950_batch_read(b, 0, k, 256, k + 256, 256) == 0        # one beside the other
    L.sllm_gfx950_batch_destroy(b)
    e = c.batch([c.new()], [0], act=F16)
    assert L.sllm_gfx950_batch_read(e, 0, None, 0, None, 0) == 0 and L.sllm_gfx950_batch_positions(e) == 0
    L.sllm_gfx950_batch_destroy(e)
    c.close()


def rope_desc(amd, **how):
    d = dict(head_dim=64, n_rot=64, layout=0, scaling=0, base=10000.0, factor=0.0, original=0.0, fast=0.0, slow=0.0, magnitude=0.0, freq=None)
    d.update(how)
    return amd.RopeDesc(*d.values())


def new_rope(amd, L, **how):
    r = c_void_p()
    d = rope_desc(amd, **how)
    assert L.sllm_gfx950_rope_new(byref(d), byref(r)) == 0
    return r


@pytest.mark.parametrize("how", [dict(head_dim=0), dict(head_dim=60), dict(head_dim=136), dict(n_rot=0), dict(n_rot=4), dict(n_rot=72), dict(n_rot=12),
                                 dict(n_rot=-8), dict(layout=2), dict(layout=-1), dict(scaling=4), dict(scaling=-1), dict(base=0.0), dict(base=-1.0),
                                 dict(base=float("nan")), dict(base=float("inf")), dict(scaling=1), dict(scaling=1, factor=-2.0),
                                 dict(scaling=2, factor=float("inf")), dict(scaling=3, factor=2.0), dict(scaling=3, factor=2.0, original=8.0, fast=1.0, slow=1.0),
                                 dict(scaling=3, factor=2.0, original=float("nan"), fast=2.0, slow=1.0), dict(magnitude=float("inf")),
                                 dict(magnitude=float("nan")), dict(magnitude=1e39), dict(scaling=1, factor=1e-7)])
def test_ropes_that_are_refused(amd, L, how):
    r, live = c_void_p(1), L.fakehip_live()
    d = rope_desc(amd, **how)
    assert L.sllm_gfx950_rope_new(byref(d), byref(r)) == ARG and not r.value
    assert L.fakehip_live() == live


def test_more_ropes_that_are_refused(amd, L):
    r = c_void_p()
    d = rope_desc(amd)
    assert L.sllm_gfx950_rope_new(None, byref(r)) == ARG and L.sllm_gfx950_rope_new(byref(d), None) == ARG
    f = np.ones(32)
    ok = rope_desc(amd, freq=f.ctypes.data, base=0.0)
    assert L.sllm_gfx950_rope_new(byref(ok), byref(r)) == 0
    L.sllm_gfx950_rope_free(r)
    ntk = rope_desc(amd, freq=f.ctypes.data, scaling=2, factor=2.0)
    assert L.sllm_gfx950_rope_new(byref(ntk), byref(r)) == ARG
    for bad in (np.inf, -np.inf, np.nan, 2.0 ** 20 * 1.0001, -1e300):
        f[7] = bad
        assert L.sllm_gfx950_rope_new(byref(ok), byref(r)) == ARG
    L.fakehip_capture(1)
    assert L.sllm_gfx950_rope_new(byref(d), byref(r)) == ARG
    L.fakehip_capture(0)
    L.sllm_gfx950_rope_free(None)


def test_frequencies_as_turns(amd, L):
    """The table as it is uploaded (device memory is host memory here), against integers."""
    from fractions import Fraction
    turn = Fraction("6.28318530717958647692528676655900576839433879875021164194988918461563281257241799725606965")
    f = np.array([1.0, 2 * np.pi, -1.0, 1e-9, 0.0, 1e6, 3.5, 6.283185307179587])
    r = new_rope(amd, L, head_dim=16, n_rot=16, freq=f.ctypes.data)
    # struct sllm_gfx950_rope: three ints, a float, the table
    table = np.ctypeslib.as_array(ctypes.cast(ctypes.cast(r.value + 16, ctypes.POINTER(c_void_p))[0], ctypes.POINTER(ctypes.c_uint64)), (8,))
    for x, got in zip(f, table):
        want = Fraction(float(x)) / turn % 1 * 2 ** 64
        off = abs(int(got) - want)
        # a quotient of 64 bits: half a step of it where it is above 1, and what is cut off
        assert min(off, 2 ** 64 - off) <= 2 + abs(float(x)) / 6.28, x
    L.sllm_gfx950_rope_free(r)


def test_rows_that_are_refused(amd, L):
    r = new_rope(amd, L)
    mem = (ctypes.c_uint8 * (1 << 18))()
    at = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    n, q, qo, k, ko, pos = 10, at, at + (1 << 14), at + (2 << 14), at + (3 << 14), at + (4 << 14)

    def call(**how):
        d = dict(dtype=F32, n_rows=n, n_head=4, n_head_kv=2, back=0, pos=pos, q=q, k=k, q_out=qo, k_out=ko, qs=0, qos=0, ks=0, kos=0)
        d.update(how)
        io = amd.RopeIO(*d.values())
        return L.sllm_gfx950_rope_rows(r, byref(io))

    L.fakehip_clear()
    for how in (dict(dtype=I8), dict(dtype=3), dict(n_rows=-1), dict(n_rows=(1 << 22) + 1), dict(n_head=0), dict(n_head=2048), dict(n_head_kv=0),
                dict(pos=None), dict(pos=pos + 2), dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(q=q + 4), dict(q_out=qo + 8),
                dict(k=k + 4), dict(k_out=ko + 4), dict(qs=255), dict(qos=258), dict(ks=100), dict(kos=1 << 29), dict(q_out=q + 16),
                dict(q_out=q, qos=512), dict(q_out=k), dict(k_out=q), dict(k_out=qo), dict(k_out=q + 512), dict(q_out=pos), dict(k_out=pos - 16),
                dict(qs=512, qos=512, q_out=q + 1008)):
        assert call(**how) == ARG, how
    io = amd.RopeIO()
    assert L.sllm_gfx950_rope_rows(None, byref(io)) == ARG and L.sllm_gfx950_rope_rows(r, None) == ARG
    assert L.fakehip_launches() == b""
    for how in (dict(), dict(q_out=q), dict(q_out=q, k_out=k), dict(n_rows=0, q=None, q_out=None, pos=None), dict(k=None, k_out=None, n_head_kv=0),
                dict(q=q, q_out=q, qs=384, qos=384, k=q + 1024, k_out=q + 1024, ks=384, kos=384),        # heads of one tensor, in place
                dict(qs=512, qos=512, q_out=q + 1024)):
        assert call(**how) == 0, how
    L.sllm_gfx950_rope_free(r)


def test_rows_on_their_way_that_are_refused(amd, L):
    c = Cache(amd, L, dtype=I8)
    b = c.batch([c.new()], [10], act=F32)
    r, other = new_rope(amd, L), new_rope(amd, L, head_dim=128)
    mem = (ctypes.c_uint8 * (1 << 18))()
    at = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    q, qo, k, v = at, at + (1 << 14), at + (2 << 14), at + (3 << 14)
    L.fakehip_clear()
    for args in ((-1, r, q, 0, qo, 0, k, 0, v, 0), (2, r, q, 0, qo, 0, k, 0, v, 0), (0, None, q, 0, qo, 0, k, 0, v, 0), (0, other, q, 0, qo, 0, k, 0, v, 0),
                 (0, r, None, 0, qo, 0, k, 0, v, 0), (0, r, q, 0, None, 0, k, 0, v, 0), (0, r, q, 0, qo, 0, None, 0, v, 0), (0, r, q, 0, qo, 0, k, 0, None, 0),
                 (0, r, q + 4, 0, qo, 0, k, 0, v, 0), (0, r, q, 0, qo, 0, k, 0, v + 8, 0), (0, r, q, 255, qo, 0, k, 0, v, 0), (0, r, q, 0, qo, 258, k, 0, v, 0),
                 (0, r, q, 0, qo, 0, k, 100, v, 0), (0, r, q, 0, q + 64, 0, k, 0, v, 0), (0, r, q, 0, k, 0, k, 0, v, 0), (0, r, q, 0, v - 1024, 0, k, 0, v, 0),
                 (0, r, q, 0, q, 512, k, 0, v, 0)):
        assert L.sllm_gfx950_batch_rope_store(b, *args) == ARG, args
    assert L.sllm_gfx950_batch_rope_store(None, 0, r, q, 0, qo, 0, k, 0, v, 0) == ARG
    assert L.fakehip_launches() == b""
    assert L.sllm_gfx950_batch_rope_store(b, 0, r, q, 0, qo, 0, k, 0, k, 0) == 0
    assert L.sllm_gfx950_batch_rope_store(b, 0, r, q, 0, q, 0, k, 0, v, 0) == 0
    L.sllm_gfx950_batch_destroy(b)
    e = c.batch([c.new()], [0], act=F32)
    assert L.sllm_gfx950_batch_rope_store(e, 0, r, None, 0, None, 0, None, 0, None, 0) == 0
    L.sllm_gfx950_batch_destroy(e)
    c.close()
    for x in (r, other):
        L.sllm_gfx950_rope_free(x)


def test_reorders_that_are_refused(amd, L):
    c = Cache(amd, L, n_pages=8)
    ids = [c.new() for _ in range(3)]
    c.grow(ids, [20, 40, 16])                       # 2, 3 and 1 pages
    was = c.state(ids)
    for seqs, parents in (([ids[0], ids[0]], [0, 1]), ([ids[0], 9], [0, 1]), (ids, [0, 1, 3]), (ids, [0, -1, 2])):
        assert L.sllm_gfx950_seq_reorder(c.p, I(*seqs), I(*parents), len(seqs)) == ARG
    assert L.sllm_gfx950_seq_reorder(c.p, None, I(0), 1) == ARG and L.sllm_gfx950_seq_reorder(c.p, I(ids[0]), None, 1) == ARG
    assert L.sllm_gfx950_seq_reorder(c.p, I(*ids), I(0, 1, 2), -1) == ARG and L.sllm_gfx950_seq_reorder(None, None, None, 0) == ARG
    L.fakehip_capture(1)
    assert L.sllm_gfx950_seq_reorder(c.p, I(*ids), I(0, 0, 0), 3) == ARG
    L.fakehip_capture(0)
    assert c.state(ids) == was
    assert L.sllm_gfx950_seq_reorder(c.p, None, None, 0) == 0
    assert L.sllm_gfx950_seq_reorder(c.p, I(*ids), I(0, 1, 2), 3) == 0 and c.state(ids) == was
    # 8 pages of which 6 are in use: two batches hold on to the rest, so that nothing gets free
    hold = c.batch(ids, [0, 0, 0])
    more = c.new()
    c.grow([more], [32])
    was = c.state(ids + [more])
    assert L.sllm_gfx950_seq_reorder(c.p, I(*ids, more), I(1, 1, 1, 3), 4) == NOMEM and c.state(ids + [more]) == was
    L.sllm_gfx950_batch_destroy(hold)
    assert L.sllm_gfx950_seq_reorder(c.p, I(*ids, more), I(1, 1, 1, 3), 4) == 0
    assert [L.sllm_gfx950_seq_len(c.p, s) for s in ids] == [40] * 3
    c.close()


@pytest.mark.parametrize("seed", range(6))
def test_reordered_pages_against_a_model(amd, L, seed):
    """Tables, lengths and pages in use: pages freed before any is taken, the lowest first."""
    r = random.Random(seed)
    c = Cache(amd, L, n_pages=120, dtype=I8)
    n, page = 7, 16
    ids = [c.new() for _ in range(n)]
    tables, lens = [[] for _ in range(n)], [0] * n

    def free():
        used = {x for t in tables for x in t}
        return [x for x in range(120) if x not in used]

    for _ in range(60):
        if r.random() < 0.5:
            new = [r.randint(0, 20) for _ in range(n)]
            # (a page that a table ends in is held by others only where it was truncated into: not here)
            c.grow(ids, new)
            room = free()
            for i in range(n):
                lens[i] += new[i]
                while len(tables[i]) * page < lens[i]:
                    tables[i].append(room.pop(0))
            if max(lens) > 150:
                for i in range(n):
                    assert L.sllm_gfx950_seq_truncate(c.p, ids[i], 0) == 0
                    tables[i], lens[i] = [], 0
        else:
            parent = [r.randrange(n) if r.random() < 0.6 else i for i in range(n)]
            assert L.sllm_gfx950_seq_reorder(c.p, I(*ids), I(*parent), n) == 0
            keeper = [next((i for i in [q] + list(range(n)) if parent[i] == q), None) for q in range(n)]
            old, was = tables, lens
            tables, lens = [list(old[p]) for p in parent], [was[p] for p in parent]
            takes = [i for i in range(n) if keeper[parent[i]] != i and lens[i] % page]
            for i in takes:
                tables[i].pop()
            room = free()
            for i in takes:
                tables[i].append(room.pop(0))
        assert c.state(ids) == (len({x for t in tables for x in t}), list(zip(lens, tables)))
    c.close()


def test_another_device_is_current(amd, L):
    """Memory is taken and kernels run on the library's device, and the caller's is current again."""
    mem = (ctypes.c_uint8 * (1 << 17))()
    at = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    L.fakehip_current(1)
    c = Cache(amd, L, dtype=I8)
    ids = [c.new(), c.new()]
    c.grow(ids, [20, 5])
    b = c.batch(ids, [1, 1])
    r = new_rope(amd, L)
    io = amd.RopeIO(F32, 4, 4, 2, 0, at, at + 4096, None, at + 16384, None, 0, 0, 0, 0)
    p = c_void_p()
    d = amd.BeamDesc(1, 2, 100, 4, F32)
    L.fakehip_clear()
    assert L.sllm_gfx950_rope_rows(r, byref(io)) == 0
    assert L.sllm_gfx950_batch_rope_store(b, 0, r, at, 0, at, 0, at + 16384, 0, at + 32768, 0) == 0
    assert L.sllm_gfx950_batch_store(b, 0, at, 0, at, 0) == 0 and L.sllm_gfx950_batch_read(b, 0, at, 0, at + 65536, 0) == 0
    assert L.sllm_gfx950_seq_reorder(c.p, I(*ids), I(0, 0), 2) == 0
    assert L.sllm_gfx950_beam_new(byref(d), byref(p)) == 0
    assert L.sllm_gfx950_beam_select(p, at, 0, at + 8192, None, at + 9216, at + 10240, at + 11264) == 0
    assert len(L.fakehip_launches().split()) == 7
    L.sllm_gfx950_beam_free(p)
    L.sllm_gfx950_rope_free(r)
    L.sllm_gfx950_batch_destroy(b)
    c.close()
    L.fakehip_current(0)


def test_what_ends_in_a_capture(amd, L):
    """Ropes and beams' plans that end while the stream is captured keep their memory until a call
    that may wait; the capture is not broken."""
    L.fakehip_broken.restype = ctypes.c_int
    r, p = new_rope(amd, L), c_void_p()
    d = amd.BeamDesc(1, 2, 100, 4, F32)
    assert L.sllm_gfx950_beam_new(byref(d), byref(p)) == 0
    live, broken = L.fakehip_live(), L.fakehip_broken()
    L.fakehip_capture(1)
    L.sllm_gfx950_rope_free(r)
    L.sllm_gfx950_beam_free(p)
    assert L.fakehip_live() == live and L.fakehip_broken() == broken
    L.fakehip_capture(0)
    L.sllm_gfx950_rope_free(new_rope(amd, L))
    assert L.fakehip_live() == live - 2


def test_every_hip_call_fails_once(amd, L):
    """Whatever call fails, its status comes back, what was there is as it was, and nothing is left."""
    mem = (ctypes.c_uint8 * (1 << 17))()
    at = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    c = Cache(amd, L, dtype=E4M3)
    ids = [c.new(), c.new(), c.new()]
    c.grow(ids, [20, 5, 33])
    b = c.batch(ids, [1, 1, 1])
    r = new_rope(amd, L)
    out = c_void_p()
    desc = rope_desc(amd)
    io = amd.RopeIO(F32, 4, 4, 2, 0, at, at + 4096, None, at + 16384, None, 0, 0, 0, 0)
    calls = [lambda: L.sllm_gfx950_rope_new(byref(desc), byref(out)), lambda: L.sllm_gfx950_rope_rows(r, byref(io)),
             lambda: L.sllm_gfx950_batch_rope_store(b, 0, r, at, 0, at, 0, at + 16384, 0, at + 32768, 0),
             lambda: L.sllm_gfx950_batch_store(b, 0, at, 0, at, 0), lambda: L.sllm_gfx950_batch_read(b, 0, at, 0, at + 65536, 0),
             lambda: L.sllm_gfx950_seq_reorder(c.p, I(*ids), I(2, 2, 0), 3)]
    for call in calls:
        for skip in range(50):
            was, live = c.state(ids), L.fakehip_live()
            L.fakehip_fail(b"*", 999, skip)
            st = call()
            fired = L.fakehip_fired()
            L.fakehip_clear()
            if not fired:
                assert st == 0
                break
            assert st == HIP, (skip, st)
            assert c.state(ids) == was and L.fakehip_live() == live
        else:
            raise AssertionError("it never succeeds")
    L.sllm_gfx950_rope_free(out)
    L.sllm_gfx950_rope_free(r)
    L.sllm_gfx950_batch_destroy(b)
    c.close()


def test_under_sanitizers():
    """This file's other tests with the library's C sources built under ASan and UBSan."""
    if os.environ.get("SLLM_FAKEHIP_SAN"):
        pytest.skip("this is that run")
    asan = subprocess.run(["gcc", "-print-file-name=libasan.so"], capture_output=True, text=True).stdout.strip()
    if not os.path.isabs(asan) or not os.path.exists(asan):
        pytest.skip("gcc's AddressSanitizer runtime is not installed")
    env = dict(os.environ, SLLM_FAKEHIP_SAN="1", UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1",
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1",
               LD_PRELOAD=asan + (":" + os.environ["LD_PRELOAD"] if os.environ.get("LD_PRELOAD") else ""))
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", os.path.abspath(__file__)], cwd=ROOT, env=env,
                       capture_output=True, text=True, timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0 and "AddressSanitizer" not in out and "runtime error:" not in out, out[-5000:]
