"""Caches, batches and prompt plans that end while the stream is captured, against
the HIP stand-in of tests/fakehip: nothing is waited for or freed until it is not."""
import ctypes
import os
import subprocess
import sys
from ctypes import byref, c_int, c_void_p

import pytest

from test_attn_host import F32, I, ROOT, Cache, L  # noqa: F401  (the fixture)


@pytest.fixture
def ends(amd, L):  # noqa: F811
    """A cache of its own memory with six open batches, the library's kept buffers full,
    and a prompt plan; and what ends them all."""
    L.fakehip_broken.restype, L.fakehip_broken.argtypes = c_int, []
    c = Cache(amd, L, 60)
    seqs = [c.new() for _ in range(6)]
    batches = [c.batch([s], [10 * (i + 1)]) for i, s in enumerate(seqs)]
    plan, q = c_void_p(), I(5)
    d = amd.PromptDesc(F32, 4, 2, 64, 1, ctypes.cast(q, c_void_p), None)
    assert L.sllm_gfx950_prompt_create(byref(d), byref(plan)) == 0

    def end():
        for b in batches:
            L.sllm_gfx950_batch_destroy(b)
        L.sllm_gfx950_prompt_destroy(plan)
        c.close()
    return end


def in_capture(L, end):  # noqa: F811
    live, broken = L.fakehip_live(), L.fakehip_broken()
    L.fakehip_capture(1)
    try:
        end()
    finally:
        L.fakehip_capture(0)
    assert L.fakehip_broken() == broken and L.fakehip_live() == live
    return live


def test_what_ends_in_a_capture_is_freed_by_the_next_call(amd, L, ends):  # noqa: F811
    base = in_capture(L, ends)
    c = Cache(amd, L, 4)
    c.fork(c.new(), 0, 1)
    # the six batches' device and pinned memory and events, the cache's memory, the plan's
    assert L.fakehip_live() == base - 6 * 3 - 2 + 1
    c.close()
    assert L.fakehip_live() == base - 6 * 3 - 2


def test_or_by_the_next_end(amd, L, ends):  # noqa: F811
    c = Cache(amd, L, 4)
    base = in_capture(L, ends)
    c.close()
    assert L.fakehip_live() == base - 6 * 3 - 3


def test_a_cache_that_goes_with_its_last_batch(amd, L):  # noqa: F811
    L.fakehip_broken.restype, L.fakehip_broken.argtypes = c_int, []
    base = L.fakehip_live()
    c = Cache(amd, L, 4)
    b = c.batch([c.new()], [3])
    c.close()
    in_capture(L, lambda: L.sllm_gfx950_batch_destroy(b))
    c = Cache(amd, L, 4)
    c.close()
    assert L.fakehip_live() == base


def test_or_by_close(amd, L, ends):  # noqa: F811
    """(the library is closed and opened again)"""
    in_capture(L, ends)
    L.sllm_gfx950_close()
    assert L.fakehip_live() == 0
    assert L.sllm_gfx950_open(0) == 0


def test_under_asan_and_ubsan():
    """This file's other tests, and those of the tables, against the sanitizer build."""
    if os.environ.get("SLLM_FAKEHIP_SAN"):
        pytest.skip("this is that run")
    asan = subprocess.run(["gcc", "-print-file-name=libasan.so"], capture_output=True, text=True).stdout.strip()
    if not os.path.isabs(asan) or not os.path.exists(asan):
        pytest.skip("gcc's AddressSanitizer runtime is not installed")
    env = dict(os.environ, SLLM_FAKEHIP_SAN="1", UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1",
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1",
               LD_PRELOAD=asan + (":" + os.environ["LD_PRELOAD"] if os.environ.get("LD_PRELOAD") else ""))
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", os.path.abspath(__file__),
                        os.path.join(here, "test_attn_tables_host.py")], cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0 and "AddressSanitizer" not in out and "runtime error:" not in out, out[-5000:]
