"""How many rows of a step over a cache of 8 bits share a workgroup (sllm_gfx950_attn.h), on
the CPU: the work items as they are laid out. What the GPU tests of 128 rows run is asserted
here, so that another choice of when to take them does not leave those tests without any."""
import ctypes
from ctypes import c_uint32, c_void_p

import numpy as np
import pytest

import held8_tiles as tiles
from test_attn_host import BF16, F16, F32, Cache, L  # noqa: F401  (the fixture)

ITEM = np.dtype([("t0", "u4"), ("n_rows", "u4"), ("tok0", "u4"), ("list", "u4"), ("vis0", "i4"), ("key0", "u4"), ("key1", "u4"),
                 ("kv", "u4"), ("head", "u4"), ("part", "u4"), ("mode", "u2"), ("h0", "u2"), ("order", "u4")])
FEW, HALF, MANY = 0, 1, 2
KT = 32                                             # keys of a tile


def items(amd, L, shape, act, dtype):
    heads, kv, d, page, lens, n_new, prefix = shape
    pages = -(-prefix // page) + sum(-(-n // page) + 1 for n in lens) + 2
    c = Cache(amd, L, n_pages=pages, page=page, kv=kv, d=d, layers=1, dtype=dtype)
    base = c.new()
    grow = lambda seqs, new: L.sllm_gfx950_batch_destroy(c.batch(seqs, new, n_head=heads))      # noqa: E731
    grow([base], [prefix])
    ids = c.fork(base, prefix, len(lens))
    grow(ids, [n - m for n, m in zip(lens, n_new)])
    b = c.batch(ids, n_new, n_head=heads, act=act)
    mem = (ctypes.c_uint8 * 64)()
    at = ctypes.addressof(mem) + (-ctypes.addressof(mem)) % 16
    assert L.sllm_gfx950_batch_attend(b, 0, at, 0, 1.0, at + 16, 0) == 0
    L.fakehip_items.restype, L.fakehip_n_items.restype = c_void_p, c_uint32
    n = L.fakehip_n_items()
    got = np.frombuffer(ctypes.string_at(L.fakehip_items(), n * ITEM.itemsize), ITEM).copy()
    L.sllm_gfx950_batch_destroy(b)
    c.close()
    return got


@pytest.mark.parametrize("dtype", [4, 5])
@pytest.mark.parametrize("act", [F16, BF16])
def test_what_the_gpu_tests_of_128_rows_run(amd, L, act, dtype):
    """Every shape has tiles of 128 rows; together they have whole and part tiles of rows, ranges
    of odd and even numbers of tiles of keys, of one, of many, and ranges that end within a tile."""
    all_of = []
    for name, shape in tiles.MANY.items():
        x = items(amd, L, shape, act, dtype)
        x = x[x["mode"] == MANY]
        assert len(x), name
        all_of.append(x[x["key1"] > x["key0"]])
    x = np.concatenate(all_of)
    n = (x["key1"] + KT - 1) // KT - x["key0"] // KT
    assert {0, 1} == set(n % 2) and n.min() <= 2 and n.max() >= 8, sorted(set(n))
    assert (x["key1"] % KT != 0).any() and (x["key1"] % KT == 0).any()
    assert (x["n_rows"] == 128).any() and (x["n_rows"] < 65).any() and ((x["n_rows"] > 64) & (x["n_rows"] < 128)).any()
    assert (x["list"] == 0xffffffff).any() and (x["list"] != 0xffffffff).any()
    assert (x["h0"] != 0).any()                     # a tile of rows that starts within a token


@pytest.mark.parametrize("dtype", [4, 5])
@pytest.mark.parametrize("act", [F32, F16, BF16])
def test_64_rows_where_there_is_little_work(amd, L, act, dtype):
    for name, shape in tiles.HALF.items():
        x = items(amd, L, shape, act, dtype)
        assert set(x["mode"]) <= {FEW, HALF} and (x["mode"] == HALF).any(), name
    for name, shape in tiles.MANY.items() if act == F32 else ():     # f32 rows: 64 at most
        assert set(items(amd, L, shape, act, dtype)["mode"]) <= {FEW, HALF}, name


@pytest.mark.parametrize("dtype", [4, 5])
@pytest.mark.parametrize("act", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_one_border_between_them(amd, L, act, dtype, d):
    """More keys of the same rows: 64 rows at a time, then 128 from some number on."""
    modes = [set(items(amd, L, (40, 40, d, 64, [n], [70], 0), act, dtype)["mode"]) for n in range(100, 4000, 130)]
    assert all(len(m) == 1 for m in modes)
    modes = [m.pop() for m in modes]
    assert modes == sorted(modes) and modes[0] == HALF and modes[-1] == MANY
