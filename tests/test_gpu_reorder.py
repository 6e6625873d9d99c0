"""Reorders of more sequences than one launch's arguments name copies for (sllm_gfx950_attn.h)
on the GPU: what each then reads back."""
import numpy as np
import pytest
import torch

import held8_oracle as h8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "int8"])
@pytest.mark.parametrize("n", [320, 321, 322, 999])
def test_many_sequences(amd, dev, dtype, n):
    kv, d, page, layers = 2, 32, 16, 2
    r = np.random.default_rng(n)
    lens = [int(r.integers(1, 40)) for _ in range(n)]
    pages = sum(-(-x // page) for x in lens)
    c = amd.PagedCache(dev, layers, kv, d, page, 2 * pages + n, dtype)
    ids = [c.new() for _ in range(n)]
    b = c.batch(ids, lens, kv, "float32")
    rows = [[torch.randn(sum(lens), kv, d) for _ in range(2)] for _ in range(layers)]
    for layer in range(layers):
        bufs = [dev.put(x.numpy()) for x in rows[layer]]
        b.store(layer, bufs[0].ptr, bufs[1].ptr)
        dev.sync()
        for x in bufs:
            x.free()
    b.close()
    hold = (lambda x: x) if dtype == "float32" else (lambda x: torch.from_numpy(h8.held(x.double().numpy(), dtype)).float())
    held = [[torch.split(hold(x), lens) for x in layer] for layer in rows]
    now = list(range(n))
    for turn in range(3):
        parent = [int(r.integers(0, n)) if turn < 2 else now.index(now[0]) for _ in range(n)]
        c.reorder(ids, parent)
        now = [now[p] for p in parent]
        b = c.batch(ids, [0] * n, kv, "float32")
        out = [dev.alloc(b.positions * kv * d * 4) for _ in range(2)]
        for layer in range(layers):
            b.read(layer, out[0].ptr, out[1].ptr)
            dev.sync()
            for i in range(2):
                want = torch.cat([held[layer][i][s] for s in now])
                assert torch.equal(torch.from_numpy(out[i].download(np.float32, want.numel())).view_as(want), want), (turn, layer, i)
        b.close()
        for x in out:
            x.free()
    c.close()


@pytest.mark.parametrize("dtype", ["float32", "int8"])
@pytest.mark.parametrize("stays", [False, True])
def test_a_store_through_a_batch_made_before(amd, dev, dtype, stays):
    """It shows where its page went, whole pages to all and the last to one, and not in the
    copies, which have what was stored when they were made."""
    kv, d, page = 1, 32, 16
    c = amd.PagedCache(dev, 1, kv, d, page, 40, dtype)
    ids = [c.new() for _ in range(4)]
    lens = [20, 3, 3, 3]
    hold = (lambda x: x) if dtype == "float32" else (lambda x: torch.from_numpy(h8.held(x.double().numpy(), dtype)).float())

    def store(b, x):
        buf = dev.put(x.numpy())
        b.store(0, buf.ptr, buf.ptr)
        dev.sync()
        buf.free()

    first, second = torch.randn(sum(lens), kv, d), torch.randn(sum(lens), kv, d)
    b = c.batch(ids, lens, kv, "float32")
    store(b, first)
    c.reorder(ids, [0, 0, 0, 0] if stays else [1, 0, 0, 0])      # goes on from sequence 0: itself and three, or three others
    store(b, second)
    b.close()
    b = c.batch(ids, [0] * 4, kv, "float32")
    out = [dev.alloc(b.positions * kv * d * 4) for _ in range(2)]
    b.read(0, out[0].ptr, out[1].ptr)
    dev.sync()
    old, new = hold(first), hold(second)
    kept = new[:20]
    copied = torch.cat([new[:16], old[16:20]])
    want = torch.cat([kept] + [copied] * 3) if stays else torch.cat([new[20:23], kept, copied, copied])
    for x in out:
        assert torch.equal(torch.from_numpy(x.download(np.float32, want.numel())).view_as(want), want)
        x.free()
    b.close()
    c.close()


def test_as_many_sequences_as_a_cache_holds(amd, dev):
    """65536 beams that go on from one, in pages that the call frees."""
    n, kv, d, page = 65536, 1, 16, 16
    c = amd.PagedCache(dev, 1, kv, d, page, n, "int8")
    ids = [c.new() for _ in range(n)]
    b = c.batch(ids, [3] * n, kv, "float32")
    rows = torch.randn(3 * n, kv, d)
    buf = dev.put(rows.numpy())
    b.store(0, buf.ptr, buf.ptr)
    b.close()
    c.reorder(ids, [77] * n)
    assert c.in_use() == n
    b = c.batch(ids, [0] * n, kv, "float32")
    out = [dev.alloc(3 * n * kv * d * 4) for _ in range(2)]
    b.read(0, out[0].ptr, out[1].ptr)
    dev.sync()
    want = torch.from_numpy(h8.held(rows[231:234].double().numpy(), "int8")).float().expand(n, 3, kv, d)
    for x in out:
        assert torch.equal(torch.from_numpy(x.download(np.float32, rows.numel())).view(n, 3, kv, d), want)
        x.free()
    b.close()
    c.close()
    buf.free()
