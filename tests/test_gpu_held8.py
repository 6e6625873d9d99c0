"""Keys and values held in 8 bits (sllm_gfx950_attn.h) on the GPU: what is written, byte
for byte; what is read back; attention over it, against 64 bits (held8_oracle.py has the
tolerances); pages of such a cache that are shared, copied and moved."""
import math

import numpy as np
import pytest
import torch

import attn_oracle as ora
import held8_oracle as h8

pytestmark = pytest.mark.gpu

ACTS = list(ora.TYPES)


def normal(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


def spread(seed, *shape):
    """Rows of all magnitudes, with rows of zeros, and rows whose largest is just at, below and over a scale's room."""
    x = normal(seed, *shape)
    r = np.random.default_rng(seed)
    rows = x.view(-1, shape[-1])
    for i in range(rows.shape[0]):
        kind = r.integers(0, 8)
        if kind == 0:
            rows[i] = 0
        elif kind in (1, 2):
            top = (127.0 if kind == 1 else 448.0) * 2.0 ** int(r.integers(-6, 4))
            rows[i] *= 0.9 * top / rows[i].abs().max()
            rows[i, int(r.integers(0, shape[-1]))] = top * (1 + int(r.integers(-1, 2)) * 2.0 ** -8)
        elif kind == 3:
            rows[i] = torch.from_numpy(r.integers(-8, 9, shape[-1]) / 2.0).float()      # many ties
        else:
            rows[i] *= 2.0 ** int(r.integers(-12, 9))
    return x


class Cache:
    """A cache of 8 bits in memory of the test's own, filled with a pattern."""

    def __init__(self, amd, dev, dtype, layers, kv, d, page, pages, fill=0x5a):
        self.amd, self.dev, self.dtype, self.shape = amd, dev, dtype, (pages, layers, 2, kv, page * (d + 1))
        self.page, self.d = page, d
        self.size = int(np.prod(self.shape))
        self.mem = dev.put(np.full(self.size, fill, np.uint8))
        self.cache = amd.PagedCache(dev, layers, kv, d, page, pages, dtype, mem=self.mem.ptr)
        assert self.cache.nbytes == self.size

    def raw(self):
        self.dev.sync()
        return self.mem.download(np.uint8, self.size).reshape(self.shape)

    def rows(self, raw, seq, layer, part):
        """Codes [n, kv, d] and scale bytes [n, kv] of a sequence."""
        n = self.cache.length(seq)
        b = raw[self.cache.table(seq), layer, part]                          # [page, kv, bytes]
        c = b[..., :self.page * self.d].reshape(len(b), -1, self.page, self.d).transpose(0, 2, 1, 3)
        s = b[..., self.page * self.d:].transpose(0, 2, 1)
        return c.reshape(-1, *c.shape[2:])[:n], s.reshape(-1, s.shape[2])[:n]

    def close(self):
        self.cache.close()
        self.mem.free()


def strided(x, stride):
    """Rows [n, ...] with a stride of elements, what is between them 9."""
    n, w = x.shape[0], x[0].numel()
    y = torch.full((n, stride or w), 9.0, dtype=x.dtype)
    y[:, :w] = x.reshape(n, w)
    return y


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kv,d,page,stride", [(2, 64, 16, 0), (5, 128, 64, 0), (3, 80, 32, 264), (1, 16, 16, 0), (2, 96, 16, 320), (2, 48, 16, 0)])
def test_what_is_written_and_read_back(amd, dev, dtype, act, kv, d, page, stride):
    """Every byte of the cache, the untouched ones among them, and the rows read back."""
    T = ora.TYPES[act]
    c = Cache(amd, dev, dtype, 2, kv, d, page, 24)
    seqs = [c.cache.new() for _ in range(4)]
    held = {s: [np.zeros((0, kv, d))] * 2 for s in seqs}
    want = c.raw().copy()
    for step, n_new in enumerate(([page + 3, 1, 0, 2 * page], [1, 5, 0, 1], [7, page, 1, 0])):
        b = c.cache.batch(seqs, n_new, 2 * kv, act)
        n = sum(n_new)
        rows = [spread(100 * step + i + d, n, kv, d).to(T) for i in range(2)]
        bufs = [dev.put(ora.bits(strided(x, stride))) for x in rows]
        b.store(1, bufs[0].ptr, bufs[1].ptr, stride, stride)
        at = 0
        for s, k in zip(seqs, n_new):
            for part in range(2):
                x = rows[part][at:at + k].double().numpy()
                codes, scales = h8.codes_of(x, dtype)
                n0 = c.cache.length(s) - k
                for i in range(k):
                    pos = n0 + i
                    block = want[c.cache.table(s)[pos // page], 1, part]
                    block[:, (pos % page) * d:(pos % page + 1) * d] = codes[i]
                    block[:, page * d + pos % page] = scales[i]
                held[s][part] = np.concatenate([held[s][part], h8.values_of(codes, scales, dtype)])
            at += k
        assert np.array_equal(c.raw(), want), step
        total = sum(c.cache.length(s) for s in seqs)
        assert b.positions == total
        out = [dev.put(ora.bits(torch.full((total, stride or kv * d), 7.0, dtype=T))) for _ in range(2)]
        b.read(1, out[0].ptr, out[1].ptr, stride, stride)
        dev.sync()
        for part in range(2):
            got = ora.from_bits(out[part].download(ora.store_type(act), total * (stride or kv * d)), act).view(total, -1)
            full = np.concatenate([held[s][part] for s in seqs]).reshape(total, -1)
            assert torch.equal(got[:, :kv * d], torch.from_numpy(full).to(T)), (step, part)
            assert (got[:, kv * d:] == 7).all()
        b.close()
        for x in bufs + out:
            x.free()
    c.close()


@pytest.mark.parametrize("dtype", h8.HELD)
def test_every_code_under_every_scale(amd, dev, dtype):
    d, page = 128, 1024
    c = Cache(amd, dev, dtype, 1, 1, d, page, 1)
    raw = np.zeros(c.shape, np.uint8)
    low, high = (1, 247) if dtype == "int8" else (10, 246)
    scales = np.arange(page) // 2 % (high - low + 1) + low
    codes = (np.arange(page)[:, None] % 2 * 128 + np.arange(d)).astype(np.uint8)
    if dtype == "int8":
        codes[codes == 0x80] = 0                                             # (-128 is none)
    raw[0, 0, :, 0, :page * d] = codes.reshape(-1)
    raw[0, 0, :, 0, page * d:] = scales
    c.mem.upload(raw)
    s = c.cache.new()
    b = c.cache.batch([s], [page], 1, "float32")
    out = [dev.alloc(4 * page * d) for _ in range(2)]
    b.read(0, out[0].ptr, out[1].ptr)
    dev.sync()
    want = h8.values_of(codes, scales.astype(np.uint8), dtype).astype(np.float32)
    for x in out:
        np.testing.assert_array_equal(x.download(np.float32, page * d).reshape(page, d), want)
        x.free()
    b.close()
    c.close()


@pytest.mark.parametrize("dtype", h8.HELD)
def test_rows_at_the_ends_of_the_range(amd, dev, dtype):
    """Zeros, subnormal values, the largest that a row may hold and the first that it may
    not, infinities and NaN: each row by itself."""
    d = 64
    tops = [0.0, 1e-45, 2.0 ** -133, 2.0 ** -126, 2.0 ** -120, 127 * 2.0 ** -126, 448 * 2.0 ** -117, 1e38, h8.LARGEST,
            np.nextafter(np.float32(h8.LARGEST), np.float32(np.inf)), 3.4e38, np.inf, -np.inf, np.nan]
    x = np.zeros((len(tops), 1, d), np.float32)
    r = np.random.default_rng(5)
    for i, t in enumerate(tops):
        if np.isfinite(t):
            x[i, 0] = (r.uniform(-1, 1, d) * t).astype(np.float32)
        x[i, 0, 17] = t
    c = Cache(amd, dev, dtype, 1, 1, d, 16, 2)
    s = c.cache.new()
    b = c.cache.batch([s], [len(tops)], 1, "float32")
    bx, out = dev.put(x), [dev.alloc(x.nbytes) for _ in range(2)]
    b.store(0, bx.ptr, bx.ptr)
    codes, scales = h8.codes_of(x.astype(np.float64), dtype)
    got = c.rows(c.raw(), s, 0, 0)
    np.testing.assert_array_equal(got[1], scales)
    np.testing.assert_array_equal(got[0], codes)
    b.read(0, out[0].ptr, out[1].ptr)
    dev.sync()
    want = h8.values_of(codes, scales, dtype).astype(np.float32)
    for y in out:
        np.testing.assert_array_equal(y.download(np.float32, x.size).reshape(x.shape), want)
    assert np.isnan(want[9:]).all() and np.isfinite(want[:9]).all()
    b.close()
    c.close()
    for y in out + [bx]:
        y.free()


def step(amd, dev, act, dtype, heads, kv, d, page, lens, n_new, prefix=0, seed=0, scale=None, edit=None, check=True):
    """A step of sequences of lens[i] positions, the last n_new[i] of them new, behind `prefix`
    shared ones: rows out against 64 bits. Returns (rows, what was held)."""
    T = ora.TYPES[act]
    pages = -(-prefix // page) + sum(-(-n // page) + 1 for n in lens) + 2
    c = amd.PagedCache(dev, 2, kv, d, page, pages, dtype)
    scale = d ** -0.5 if scale is None else scale

    def rows(n, s):
        k, v = (normal(seed + 10 * s + i, n, kv, d).to(T) for i in range(2))
        if edit:
            edit(s, k, v)
        return k, v

    def store(ids, new, what):
        b = c.batch(ids, new, heads, act)
        if b.rows:
            bufs = [dev.put(ora.bits(torch.cat([w[i] for w in what]).contiguous())) for i in range(2)]
            b.store(1, *(x.ptr for x in bufs))
            dev.sync()
            for x in bufs:
                x.free()
        return b

    base, shared = c.new(), rows(prefix, 900)
    store([base], [prefix], [shared]).close()
    ids = c.fork(base, prefix, len(lens))
    own = [rows(n, i) for i, n in enumerate(lens)]
    store(ids, [n - m for n, m in zip(lens, n_new)], [tuple(x[:n - m] for x in o) for o, n, m in zip(own, lens, n_new)]).close()
    b = store(ids, n_new, [tuple(x[n - m:] for x in o) for o, n, m in zip(own, lens, n_new)])
    n = b.rows
    q = normal(seed + 7, n, heads, d).to(T)
    bq, bo = dev.put(ora.bits(q)), dev.put(ora.bits(torch.full((n, heads, d), 7.0, dtype=T)))
    b.attend(1, bq.ptr, bo.ptr, scale)
    dev.sync()
    got = ora.from_bits(bo.download(ora.store_type(act), n * heads * d), act).view(n, heads, d)
    at, all_held = 0, []
    for i, m in enumerate(n_new):
        held = [h8.held(torch.cat([s, o]).double().numpy(), dtype) for s, o in zip(shared, own[i])]
        all_held.append(held)
        if check:
            total = len(held[0])
            want, tol = h8.attend(q[at:at + m].double().numpy(), *held, total - m + 1 + np.arange(m), scale, act)
            ora.check(got[at:at + m], want, tol, f"sequence {i}")
        at += m
    b.attend(1, bq.ptr, bo.ptr, scale)                                       # the same call, the same bits
    dev.sync()
    again = ora.from_bits(bo.download(ora.store_type(act), n * heads * d), act).view(n, heads, d)
    assert torch.equal(ora.from_bits(ora.bits(got), act).view(torch.int32 if act == "float32" else torch.int16),
                       again.view(torch.int32 if act == "float32" else torch.int16))
    b.close()
    c.close()
    bq.free(), bo.free()
    return got, all_held


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 64), (20, 5, 128), (6, 3, 80), (8, 1, 96), (2, 2, 16)])
def test_attend_one_position_each(amd, dev, act, dtype, heads, kv, d):
    step(amd, dev, act, dtype, heads, kv, d, 16, [1, 2, 15, 16, 17, 33, 64, 130, 257], [1] * 9, seed=11)


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("page", [16, 64])
def test_attend_long_in_splits(amd, dev, act, dtype, page):
    step(amd, dev, act, dtype, 4, 1, 128, page, [2051, 700], [1, 3], seed=12)


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 64), (20, 5, 128), (6, 2, 80)])
@pytest.mark.parametrize("n_new", [5, 16, 33, 65])
def test_attend_many_new_positions(amd, dev, act, dtype, heads, kv, d, n_new):
    """64 and 128 rows a workgroup: prompts behind earlier positions, causal within."""
    step(amd, dev, act, dtype, heads, kv, d, 16, [n_new, n_new + 40, 300], [n_new] * 3, seed=13)


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("prefix", [256, 1000])
def test_attend_behind_a_shared_prefix(amd, dev, act, dtype, prefix):
    step(amd, dev, act, dtype, 8, 2, 64, 16, [1, 9, 30, 64, 1, 2, 3, 77, 5, 20], [1, 2, 1, 1, 1, 2, 3, 4, 1, 1], prefix=prefix, seed=14)


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
def test_attend_sequences_without_new_positions(amd, dev, act, dtype):
    step(amd, dev, act, dtype, 4, 2, 64, 16, [20, 0, 40, 33], [1, 0, 0, 2], seed=15)


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n_new", [1, 40])
def test_attend_rows_many_powers_of_two_apart(amd, dev, act, dtype, n_new):
    """Scales of keys and values far apart, a later row's too: each row by what it sees. (f16 rows hold less.)"""
    far = 60 if act != "float16" else 6

    def edit(s, k, v):
        r = np.random.default_rng(s)
        for i in range(k.shape[0]):
            v[i] = (v[i].float() * 2.0 ** int(r.integers(-far, far))).to(v.dtype)
            k[i] = (k[i].float() * 2.0 ** int(r.integers(-8, 3))).to(k.dtype)

    step(amd, dev, act, dtype, 4, 2, 64, 16, [150, 90], [n_new, n_new], seed=16, edit=edit)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("scale", [1e-30, 30.0])
def test_attend_other_scales(amd, dev, act, dtype, scale):
    step(amd, dev, act, dtype, 4, 2, 64, 16, [100, 70], [1, 20], seed=17, scale=scale)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("n_new", [1, 3, 40, 80])
@pytest.mark.parametrize("part", [0, 1])
def test_what_is_not_finite_reaches_those_who_see_it(amd, dev, act, dtype, n_new, part):
    """A row of NaN among the new positions: rows in front of it, and the other sequence, are as they were."""
    heads, kv, d, lens = 8, 2, 64, [120, 130]
    clean, _ = step(amd, dev, act, dtype, heads, kv, d, 16, lens, [n_new] * 2, seed=18)
    at = lens[0] - 1 - n_new // 2

    def edit(s, k, v):
        if s == 0:
            (k, v)[part][at, 1, 5] = math.inf if n_new % 2 else math.nan

    got, _ = step(amd, dev, act, dtype, heads, kv, d, 16, lens, [n_new] * 2, seed=18, edit=edit, check=False)
    seen = torch.zeros(2 * n_new, heads, dtype=torch.bool)
    seen[at - (lens[0] - n_new):n_new, 4:] = True
    assert torch.isnan(got[seen].float()).all()
    assert torch.equal(got[~seen], clean[~seen])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", h8.HELD)
def test_values_that_are_alike_come_back_as_they_are(amd, dev, act, dtype):
    def edit(s, k, v):
        v[:] = torch.linspace(-1.5, 1.0, v.shape[-1]).to(v.dtype)

    got, held = step(amd, dev, act, dtype, 4, 2, 64, 16, [300, 77], [1, 30], seed=19, edit=edit)
    at = 0
    for (_, v), n in zip(held, [1, 30]):
        want = torch.from_numpy(v[0]).repeat_interleave(2, 0).expand(n, -1, -1)
        tol = want.abs() * (2.0 ** -24 * 700 if act == "float32" else 2.0 ** -10 if act == "float16" else 2.0 ** -7)
        assert ((got[at:at + n].double() - want).abs() <= tol).all()
        at += n


@pytest.mark.parametrize("dtype", h8.HELD)
def test_pages_that_are_shared_copied_and_moved(amd, dev, dtype):
    """fork, copy, truncate, a write into what others hold, reorder and compact: rows and
    scales of every sequence, and of a partly copied page nothing else."""
    kv, d, page, layers = 2, 64, 16, 2
    c = Cache(amd, dev, dtype, layers, kv, d, page, 60)
    rows = {}

    def grow(ids, n_new, seed):
        b = c.cache.batch(ids, n_new, kv, "float32")
        for layer in range(layers):
            x = [spread(seed + 2 * layer + i, max(b.rows, 1), kv, d) for i in range(2)]
            bufs = [dev.put(y.numpy()) for y in x]
            b.store(layer, bufs[0].ptr, bufs[1].ptr)
            dev.sync()
            at = 0
            for s, n in zip(ids, n_new):
                for i in range(2):
                    new = h8.codes_of(x[i][at:at + n].double().numpy(), dtype)
                    old = rows.setdefault((s, layer, i), tuple(z[:0] for z in new))
                    rows[s, layer, i] = tuple(np.concatenate([o, z]) for o, z in zip(old, new))
                at += n
            for y in bufs:
                y.free()
        b.close()

    def like(s, src, n):
        for layer in range(layers):
            for i in range(2):
                rows[s, layer, i] = tuple(z[:n] for z in rows[src, layer, i])

    def check(ids):
        raw = c.raw()
        for s in ids:
            for layer in range(layers):
                for i in range(2):
                    got = c.rows(raw, s, layer, i)
                    for x, y in zip(got, rows[s, layer, i]):
                        assert np.array_equal(x, y), (s, layer, i)
        return raw

    a, b = c.cache.new(), c.cache.new()
    grow([a, b], [45, 16], 1)
    check([a, b])
    before = c.raw()
    f = c.cache.fork(a, 39, 2)
    for s in f:
        like(s, a, 39)
    raw = check([a, b] + f)
    for s in f:                                                              # 7 rows of the page; the rest keeps its bytes
        last = c.cache.table(s)[-1]
        assert np.array_equal(raw[last][..., 7 * d:page * d], before[last][..., 7 * d:page * d])
        assert np.array_equal(raw[last][..., page * d + 7:], before[last][..., page * d + 7:])
    grow([f[0], a], [20, 3], 20)
    k, = c.cache.copy([f[0]])
    like(k, f[0], 59)
    check([a, b, k] + f)
    c.cache.truncate(f[1], 20)
    like(f[1], f[1], 20)
    grow([f[1], b], [30, 1], 40)                                             # writes into a page that f[0] and a hold
    check([a, b, k] + f)
    ids, parents = [a, b] + f + [k], [3, 3, 1, 3, 0]
    old = {(s, layer, i): rows[s, layer, i] for s in ids for layer in range(layers) for i in range(2)}
    c.cache.reorder(ids, parents)
    for s, p in zip(ids, parents):
        for layer in range(layers):
            for i in range(2):
                rows[s, layer, i] = old[ids[p], layer, i]
    check(ids)
    grow(ids, [1, 2, 3, 4, 5], 60)
    check(ids)
    c.cache.free([b])
    c.cache.compact()
    check([a, k] + f)
    assert c.cache.in_use() == len({int(p) for s in [a, k] + f for p in c.cache.table(s)})
    c.close()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_reading_back_what_is_not_8_bits(amd, dev, dtype):
    kv, d, page = 3, 40, 16
    for act in ["float32", dtype] if dtype == "float16" else [dtype]:
        c = amd.PagedCache(dev, 2, kv, d, page, 100, dtype)
        seqs = [c.new() for _ in range(70)]
        lens = [1 + 3 * (i % 9) if i % 5 else 0 for i in range(70)]
        lens[33] = 150
        b = c.batch(seqs, lens, kv, act)
        n = sum(lens)
        T = ora.TYPES[act]
        x = [normal(31 + i, n, kv, d).to(T) for i in range(2)]
        bufs = [dev.put(ora.bits(y)) for y in x]
        out = [dev.alloc(n * kv * d * x[0].element_size()) for _ in range(2)]
        b.store(1, bufs[0].ptr, bufs[1].ptr)
        b.read(1, out[0].ptr, out[1].ptr)
        dev.sync()
        for y, o in zip(x, out):
            got = ora.from_bits(o.download(ora.store_type(act), n * kv * d), act).view(n, kv, d)
            assert torch.equal(got, y.to(ora.TYPES[dtype]).to(T))
        b.close()
        c.close()
        for y in bufs + out:
            y.free()


def test_offsets_past_32_bits(amd, dev):
    """A cache of more than 4 GiB of codes, a sequence at its end."""
    kv, d, page, heads, n = 8, 128, 64, 16, 150
    pages = (5 << 30) // (2 * kv * page * (d + 1))
    c = amd.PagedCache(dev, 1, kv, d, page, pages, "int8")
    first, s = c.new(), c.new()
    for at in range(0, (pages - 4) * page, 1 << 20):                         # (a batch has at most 2^24 rows)
        c.batch([first], [min(1 << 20, (pages - 4) * page - at)], kv, "float32").close()
    b = c.batch([s], [n], heads, "bfloat16")
    assert int(c.table(s).min()) * 2 * kv * page * (d + 1) > 1 << 32
    q, k, v = (normal(61 + i, n, h, d).bfloat16() for i, h in enumerate((heads, kv, kv)))
    bq, bk, bv = (dev.put(ora.bits(x)) for x in (q, k, v))
    bo, bb = dev.alloc(q.numel() * 2), [dev.alloc(k.numel() * 2) for _ in range(2)]
    b.store(0, bk.ptr, bv.ptr)
    b.attend(0, bq.ptr, bo.ptr, 0.1)
    b.read(0, bb[0].ptr, bb[1].ptr)
    dev.sync()
    got = ora.from_bits(bo.download(np.int16, q.numel()), "bfloat16").view(n, heads, d)
    held = [h8.held(x.double().numpy(), "int8") for x in (k, v)]
    want, tol = h8.attend(q.double().numpy(), *held, np.arange(n) + 1, 0.1, "bfloat16")
    ora.check(got, want, tol)
    for x, o in zip(held, bb):
        assert torch.equal(ora.from_bits(o.download(np.int16, k.numel()), "bfloat16").view(n, kv, d), torch.from_numpy(x).bfloat16())
    b.close()
    c.close()
    for x in [bq, bk, bv, bo] + bb:
        x.free()


@pytest.mark.parametrize("dtype", h8.HELD + ["float16"])
def test_a_cache_s_life(amd, dev, dtype):
    """Random steps, forks, copies, reorders, truncations and moves: what every sequence then
    reads back, against the rows that it was given."""
    r = np.random.default_rng(77)
    kv, d, page, pages, layers = 2, 48, 16, 90, 2
    c = amd.PagedCache(dev, layers, kv, d, page, pages, dtype)
    hold = (lambda x: x.half().float()) if dtype == "float16" else (lambda x: torch.from_numpy(h8.held(x.double().numpy(), dtype)).float())
    rows = {c.new(): [torch.zeros(0, kv, d) for _ in range(2 * layers)] for _ in range(4)}

    def check():
        ids = list(rows)
        b = c.batch(ids, [0] * len(ids), kv, "float32")
        n = b.positions
        assert n == sum(len(x[0]) for x in rows.values())
        out = [dev.alloc(max(n, 1) * kv * d * 4) for _ in range(2)]
        for layer in range(layers):
            b.read(layer, out[0].ptr, out[1].ptr)
            dev.sync()
            for i in range(2):
                want = torch.cat([rows[s][2 * layer + i] for s in ids])
                got = torch.from_numpy(out[i].download(np.float32, n * kv * d)).view(n, kv, d)
                assert torch.equal(got, want), (layer, i)
        b.close()
        for x in out:
            x.free()

    for step in range(120):
        ids, op = list(rows), r.integers(0, 8)
        room = pages - c.in_use()
        if op <= 2:                                                          # a step
            pick = [s for s in ids if r.random() < 0.7]
            new = [int(r.integers(0, 20)) for _ in pick]
            if sum(n // page + 2 for n in new) > room:
                continue
            b = c.batch(pick, new, kv, "float32")
            for layer in range(layers):
                x = [spread(1000 * step + 10 * layer + i, max(sum(new), 1), kv, d) / 64 for i in range(2)]
                bufs = [dev.put(y.numpy()) for y in x]
                b.store(layer, bufs[0].ptr, bufs[1].ptr)
                dev.sync()
                at = 0
                for s, n in zip(pick, new):
                    for i in range(2):
                        rows[s][2 * layer + i] = torch.cat([rows[s][2 * layer + i], hold(x[i][at:at + n])])
                    at += n
                for y in bufs:
                    y.free()
            b.close()
        elif op <= 4 and len(ids) > 1:                                       # beams
            some = [ids[i] for i in r.permutation(len(ids))[:r.integers(1, len(ids) + 1)]]
            if len(some) > room:
                continue
            parents = [int(r.integers(0, len(some))) for _ in some]
            old = [rows[s] for s in some]
            c.reorder(some, parents)
            for s, p in zip(some, parents):
                rows[s] = list(old[p])
        elif op == 5 and len(ids) < 9:
            s = ids[r.integers(0, len(ids))]
            n = int(r.integers(0, len(rows[s][0]) + 1))
            if room > 3:
                for f in c.fork(s, n, 2):
                    rows[f] = [x[:n] for x in rows[s]]
        elif op == 6:
            s = ids[r.integers(0, len(ids))]
            n = int(r.integers(0, len(rows[s][0]) + 1))
            c.truncate(s, n)
            rows[s] = [x[:n] for x in rows[s]]
            if len(ids) > 3:
                c.free([ids[0]])
                del rows[ids[0]]
        else:
            c.compact()
            assert all((c.table(s) < c.in_use()).all() for s in rows)
        if step % 6 == 5:
            check()
    check()
    c.close()
