"""The host side of the beams' selection (sllm_gfx950_attn.h) on the CPU, against the HIP
stand-in of tests/fakehip: what is refused, every HIP call failing in turn, the parts of a row."""
import ctypes
from ctypes import byref, c_void_p

import pytest

from test_attn_host import ARG, F32, HIP, L  # noqa: F401  (the fixture)


def new(amd, L, g, b, v, k, dtype=F32, status=0):
    p = c_void_p(1)
    d = amd.BeamDesc(g, b, v, k, dtype)
    assert L.sllm_gfx950_beam_new(byref(d), byref(p)) == status, (g, b, v, k, dtype)
    return p


@pytest.mark.parametrize("what", [(0, 1, 9, 1), (1, 0, 9, 1), (1, 65, 900, 1), (1, 1, 0, 1), (1, 1, (1 << 24) + 1, 1), (1, 1, 9, 0), (1, 1, 900, 65),
                                  (1, 33, 900, 64), (1, 2, 3, 7), ((1 << 20) + 1, 1, 9, 1), (1 << 19, 3, 9, 1), (-1, 1, 9, 1), (1, 1, 9, 1, 3),
                                  (1, 1, 9, 1, 4), (1, 1, 9, 1, -1)])
def test_plans_that_are_refused(amd, L, what):
    live = L.fakehip_live()
    assert not new(amd, L, *what, status=ARG).value and L.fakehip_live() == live


def test_calls_that_are_refused(amd, L):
    p = c_void_p()
    d = amd.BeamDesc(1, 1, 9, 1, F32)
    assert L.sllm_gfx950_beam_new(None, byref(p)) == ARG and L.sllm_gfx950_beam_new(byref(d), None) == ARG
    L.fakehip_capture(1)
    new(amd, L, 1, 1, 9, 1, status=ARG)
    L.fakehip_capture(0)
    p = new(amd, L, 2, 4, 100, 8)
    mem = (ctypes.c_uint8 * (1 << 16))()
    x = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    s, e, o, b, t = (x + 8192 + 1024 * i for i in range(5))
    L.fakehip_clear()
    for args in ((None, 0, s, e, o, b, t), (x, 0, None, e, o, b, t), (x, 0, s, e, None, b, t), (x, 0, s, e, o, None, t), (x, 0, s, e, o, b, None),
                 (x, 99, s, e, o, b, t), (x, (1 << 28) + 1, s, e, o, b, t), (x + 4, 0, s, e, o, b, t), (x, 0, s + 2, e, o, b, t), (x, 0, s, e + 1, o, b, t),
                 (x, 0, s, e, o + 2, b, t), (x, 0, s, e, s, b, t), (x, 0, s, e, o, e, t), (x, 0, s, e, o, b, x + 3196), (x, 0, s, e, o, o, t),
                 (x, 0, s, e, o, b, b + 60)):
        assert L.sllm_gfx950_beam_select(p, *args) == ARG, args
    assert L.sllm_gfx950_beam_select(None, x, 0, s, e, o, b, t) == ARG
    assert L.fakehip_launches() == b""
    assert L.sllm_gfx950_beam_select(p, x, 0, s, None, o, b, t) == 0
    assert L.sllm_gfx950_beam_select(p, x, 164, s, e, x + 464, b, t) == 0             # between rows
    L.sllm_gfx950_beam_free(p)
    L.sllm_gfx950_beam_free(None)


def test_every_hip_call_fails_once(amd, L):
    mem = (ctypes.c_uint8 * (1 << 16))()
    x = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    p, out = new(amd, L, 2, 4, 100, 8), c_void_p()
    d = amd.BeamDesc(2, 4, 100, 8, F32)
    for call in (lambda: L.sllm_gfx950_beam_new(byref(d), byref(out)),
                 lambda: L.sllm_gfx950_beam_select(p, x, 0, x + 8192, None, x + 9216, x + 10240, x + 11264)):
        for skip in range(20):
            live = L.fakehip_live()
            L.fakehip_fail(b"*", 999, skip)
            st = call()
            fired = L.fakehip_fired()
            L.fakehip_clear()
            if not fired:
                assert st == 0
                break
            assert st == HIP and L.fakehip_live() == live
        else:
            raise AssertionError("it never succeeds")
    L.sllm_gfx950_beam_free(out)
    L.sllm_gfx950_beam_free(p)


@pytest.mark.parametrize("g,b,v,k", [(1, 1, 1, 1), (1, 4, 128256, 8), (32, 8, 128256, 16), (1, 1, 1 << 24, 64), (1 << 20, 1, 5000, 64), (1, 32, 300000, 64)])
def test_parts_of_a_row(amd, L, g, b, v, k):
    """Every logit is in a part, no part is empty, and the join has a lane for each."""
    p = new(amd, L, g, b, v, k)
    mem = (ctypes.c_uint8 * 64)()
    at = ctypes.addressof(mem)
    x, far = (at + 15) // 16 * 16, 1 << 46
    L.fakehip_clear()
    assert L.sllm_gfx950_beam_select(p, x, 0, far, None, 2 * far, 3 * far, 4 * far) == 0      # (nothing is read or written there)
    name, groups = L.fakehip_launches().decode().split()[0].split(":")
    assert name == "sllm_k_beam_f32"
    parts, tiles = int(groups) // (g * b), -(-v // 2048)
    assert int(groups) == parts * g * b and 1 <= parts <= min(tiles, 64)
    assert -(-tiles // -(-tiles // parts)) == parts
    L.sllm_gfx950_beam_free(p)
