"""Attention over a cache of 8 bits 128 rows a workgroup (sllm_gfx950_attn.h) on the GPU,
every row and head against 64 bits: held8_tiles.py has the shapes, and
test_held8_tiles_host.py asserts that they are laid out so."""
import math

import numpy as np
import pytest
import torch

import attn_oracle as ora
import held8_oracle as h8
import held8_rows as rows8
import held8_tiles as tiles

pytestmark = pytest.mark.gpu

ACTS = ["float16", "bfloat16"]
UP = {"float16": 2.0 ** -16, "bfloat16": 2.0 ** -8}


def normal(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


def run(amd, dev, act, dtype, shape, bad=None):
    """A step: rows out, the queries, and the keys and values of each sequence as they were given.
    bad: (part, position of sequence 0, KV head) that has an infinite element."""
    heads, kv, d, page, lens, n_new, prefix = shape
    T = ora.TYPES[act]
    pages = -(-prefix // page) + sum(-(-n // page) + 1 for n in lens) + 2
    c = amd.PagedCache(dev, 1, kv, d, page, pages, dtype)

    def store(ids, new, rows):
        b = c.batch(ids, new, heads, act)
        if b.rows:
            bufs = [dev.put(ora.bits(torch.cat([r[i] for r in rows]))) for i in range(2)]
            b.store(0, bufs[0].ptr, bufs[1].ptr)
            dev.sync()
            for x in bufs:
                x.free()
        return b

    shared = [normal(900 + i, prefix, kv, d).to(T) for i in range(2)]
    own = [[normal(10 * s + i, n, kv, d).to(T) for i in range(2)] for s, n in enumerate(lens)]
    if bad:
        own[0][bad[0]][bad[1], bad[2], 5] = math.inf
    base = c.new()
    store([base], [prefix], [shared]).close()
    ids = c.fork(base, prefix, len(lens))
    store(ids, [n - m for n, m in zip(lens, n_new)], [[x[:n - m] for x in o] for o, n, m in zip(own, lens, n_new)]).close()
    b = store(ids, n_new, [[x[n - m:] for x in o] for o, n, m in zip(own, lens, n_new)])
    n = b.rows
    q = normal(7, n, heads, d).to(T)
    bq, bo, got = dev.put(ora.bits(q)), dev.put(ora.bits(torch.full((n + 1, heads, d), 7.0, dtype=T))), []
    for _ in range(2):                                           # the same call, the same bits
        b.attend(0, bq.ptr, bo.ptr, d ** -0.5)
        dev.sync()
        y = ora.from_bits(bo.download(np.int16, (n + 1) * heads * d), act).view(n + 1, heads, d)
        assert (y[n] == 7).all()
        got.append(y[:n].clone())
    assert torch.equal(got[0].view(torch.int16), got[1].view(torch.int16))
    b.close()
    c.close()
    bq.free(), bo.free()
    return got[0], q, shared, own


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("name", list(tiles.MANY))
def test_every_row(amd, dev, act, dtype, name):
    shape = tiles.MANY[name]
    heads, kv, d, page, lens, n_new, prefix = shape
    got, q, shared, own = run(amd, dev, act, dtype, shape)
    front, at = [h8.held(x.double().numpy(), dtype) for x in shared], 0
    for o, n, m in zip(own, lens, n_new):
        k, v = (np.concatenate([f, h8.held(x.double().numpy(), dtype)]) for f, x in zip(front, o))
        want, tol = rows8.attend(q[at:at + m].double().numpy(), k, v, prefix + n - m + 1 + np.arange(m), d ** -0.5, act, UP[act])
        ora.check(got[at:at + m], want, tol, f"{name}: {m} of {len(k)}")
        at += m


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("name", ["a head a KV head, one tile of rows", "a padded head", "a prompt from its start"])
@pytest.mark.parametrize("part", [0, 1])
def test_what_is_not_finite_reaches_those_who_see_it(amd, dev, act, dtype, name, part):
    """A row of NaN among the new positions: whoever does not see it has the result to the bit."""
    shape = tiles.MANY[name]
    heads, kv, _, _, lens, n_new, _ = shape
    at = lens[0] - n_new[0] // 2
    clean = run(amd, dev, act, dtype, shape)[0]
    got = run(amd, dev, act, dtype, shape, (part, at, 1))[0]
    seen = torch.zeros(sum(n_new), heads, dtype=torch.bool)
    seen[at - (lens[0] - n_new[0]):n_new[0], heads // kv:2 * heads // kv] = True
    assert torch.isnan(got[seen].float()).all() and torch.isfinite(clean.float()).all()
    assert torch.equal(got[~seen], clean[~seen])
