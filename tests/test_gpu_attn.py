"""Attention over packed prompts and over a paged cache (sllm_gfx950_attn.h) on
the GPU, against attention in 64 bits (attn_oracle.py has the tolerances)."""
import ctypes
import math
from ctypes import c_void_p

import numpy as np
import pytest
import torch

import attn_oracle as ora

pytestmark = pytest.mark.gpu

PAIRS = [("float32", "float32"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")]


def normal(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


def prompt(amd, dev, dtype, heads, kv, d, q_len, k_len=None, seed=0, edit=None, scale=None, oracle=ora.attend):
    """Run and check one prompt plan on packed tensors; returns the output."""
    k_len = q_len if k_len is None else k_len
    T = ora.TYPES[dtype]
    q, k, v = (normal(seed + i, n, h, d).to(T) for i, (n, h) in enumerate([(sum(q_len), heads), (sum(k_len), kv), (sum(k_len), kv)]))
    if edit:
        edit(q, k, v)
    scale = d ** -0.5 if scale is None else scale
    bufs = [dev.put(ora.bits(x)) for x in (q, k, v)]
    filler = torch.full((max(sum(q_len), 1), heads, d), 7.0, dtype=T)
    out = dev.put(ora.bits(filler))
    plan = amd.PromptAttention(dev, dtype, heads, kv, d, q_len, k_len)
    plan.run(bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, out.ptr, scale)
    dev.sync()
    got = ora.from_bits(out.download(ora.store_type(dtype), sum(q_len) * heads * d), dtype).view(-1, heads, d)
    a = b = 0
    for i, (nq, nk) in enumerate(zip(q_len, k_len)):
        want, tol = oracle(q[a:a + nq].double().numpy(), k[b:b + nk].double().numpy(), v[b:b + nk].double().numpy(),
                           np.arange(nq) + nk - nq + 1, scale, dtype, dtype)
        ora.check(got[a:a + nq], want, tol, f"sequence {i}")
        a, b = a + nq, b + nk
    plan.close()
    for x in bufs + [out]:
        x.free()
    return got


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 64), (5, 1, 128), (3, 3, 80), (8, 2, 96), (2, 2, 8)])
@pytest.mark.parametrize("q_len", [[1], [37], [64, 65], [3, 0, 130, 1]])
def test_prompt(amd, dev, dtype, heads, kv, d, q_len):
    prompt(amd, dev, dtype, heads, kv, d, q_len, seed=11)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_longer(amd, dev, dtype, d):
    prompt(amd, dev, dtype, 2, 1, d, [300, 517], seed=12)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("heads,kv,d", [(8, 4, 64), (15, 5, 128), (12, 6, 80)])
def test_prompt_several_of_one_length(amd, dev, dtype, heads, kv, d):
    prompt(amd, dev, dtype, heads, kv, d, [130] * 16 + [65, 1], seed=19, oracle=ora.attend_rows)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
def test_prompt_several_of_one_length_and_what_is_not_finite(amd, dev, dtype):
    heads, kv, d, lens = 8, 4, 64, [130] * 16
    clean = prompt(amd, dev, dtype, heads, kv, d, lens, seed=21, oracle=ora.attend_rows)
    T = ora.TYPES[dtype]
    q, k, v = (normal(21 + i, sum(lens), h, d).to(T) for i, h in enumerate((heads, kv, kv)))
    k[130 + 60, 1, 3] = math.nan
    v[130 + 20, 2, 5] = math.inf
    v[130 + 129, :, 7] = -math.inf
    bufs = [dev.put(ora.bits(x)) for x in (q, k, v)]
    out = dev.alloc(clean.numel() * clean.element_size())
    plan = amd.PromptAttention(dev, dtype, heads, kv, d, lens)
    plan.run(bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, out.ptr, d ** -0.5)
    dev.sync()
    got = ora.from_bits(out.download(ora.store_type(dtype), clean.numel()), dtype).view_as(clean)
    seen = torch.zeros_like(clean, dtype=torch.bool)
    seen[130 + 60:260, 2:4] = True
    seen[130 + 20:260, 4:6, 5] = True
    seen[130 + 129, :, 7] = True
    assert torch.equal(got[~seen], clean[~seen])
    assert not torch.isfinite(got[130 + 60:260, 2:4].float()).any() and not torch.isfinite(got[130 + 20:260, 4:6, 5].float()).any()
    assert not torch.isfinite(got[130 + 129, :, 7].float()).any()
    plan.close()
    for x in bufs + [out]:
        x.free()


@pytest.mark.parametrize("dtype", list(ora.TYPES))
def test_prompt_few_rows_over_many_keys(amd, dev, dtype):
    prompt(amd, dev, dtype, 4, 2, 128, [1, 5, 8, 9, 1], [700, 333, 1, 90, 1500], seed=20)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
def test_prompt_behind_earlier_keys_and_rows_that_see_none(amd, dev, dtype):
    """Keys in front of the prompt's own; more rows than keys: the first see none
    and are 0, keys or no keys at all."""
    got = prompt(amd, dev, dtype, 4, 2, 64, [5, 70, 40, 9, 0], [200, 71, 8, 0, 6], seed=13)
    assert (got[75:75 + 32] == 0).all() and (got[115:124] == 0).all()


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prompt_what_a_row_does_not_see_does_not_reach_it(amd, dev, dtype, bad):
    """Keys and values that are not finite leave the rows in front of them, and
    the other sequences, as they are; the rows that see them are not finite."""
    heads, kv, d, lens = 4, 2, 64, [50, 90, 30]
    clean = prompt(amd, dev, dtype, heads, kv, d, lens, seed=14)
    T = ora.TYPES[dtype]
    q, k, v = (normal(14 + i, sum(lens), h, d).to(T) for i, h in enumerate((heads, kv, kv)))
    k[50 + 40, 0, 3] = bad                          # sequence 1, position 40
    v[50 + 20, 1, 5] = bad                          # position 20
    v[50 + 89, :, 7] = bad                          # its last position
    bufs = [dev.put(ora.bits(x)) for x in (q, k, v)]
    out = dev.alloc(clean.numel() * clean.element_size())
    plan = amd.PromptAttention(dev, dtype, heads, kv, d, lens)
    plan.run(bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, out.ptr, d ** -0.5)
    dev.sync()
    got = ora.from_bits(out.download(ora.store_type(dtype), clean.numel()), dtype).view_as(clean)
    seen = torch.zeros_like(clean, dtype=torch.bool)       # values that may differ
    seen[50 + 40:140, 0:2] = True
    seen[50 + 20:140, 2:4, 5] = True
    seen[50 + 89, :, 7] = True
    # (a row may take other roundings where its tile is gone through again: none here, sums are in the same order)
    assert torch.equal(got[~seen], clean[~seen])
    assert not torch.isfinite(got[50 + 89, :, 7].float()).any()
    assert not torch.isfinite(got[50 + 20:140, 2:4, 5].float()).any()
    for x in bufs + [out]:
        x.free()


def test_prompt_rows_that_are_all_lowest(amd, dev):
    """Scores of the type's lowest values still make a softmax."""
    def edit(q, k, v):
        q[:] = 0
        q[..., 0] = -65504.0
        k[..., 0] = 1.0
    prompt(amd, dev, "float16", 2, 1, 64, [40], seed=15, edit=edit, scale=1.0)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
def test_prompt_strides(amd, dev, dtype):
    """q, k and v side by side in one row with gaps, heads of out apart; what lies
    between is left alone. Then [head][token] tensors."""
    heads, kv, d, lens = 4, 2, 72, [33, 100]
    n, T = sum(lens), ora.TYPES[dtype]
    row = (heads + 2 * kv) * d + 24
    x = normal(16, n, row).to(T)
    q, k, v = x[:, :heads * d], x[:, heads * d + 8:(heads + kv) * d + 8], x[:, (heads + kv) * d + 16:(heads + 2 * kv) * d + 16]
    size = x.element_size()
    want, tol, at = [], [], 0
    for m in lens:
        w, t = ora.attend(*(y[at:at + m].reshape(m, h, d).double().numpy() for y, h in ((q, heads), (k, kv), (v, kv))),
                          np.arange(m) + 1, 0.1, dtype, dtype)
        want.append(w), tol.append(t)
        at += m
    want, tol = np.concatenate(want), np.concatenate(tol)
    bx = dev.put(ora.bits(x))
    o_head, o_tok = d + 8, heads * (d + 8) + 16
    bo = dev.put(ora.bits(torch.full((n, o_tok), 7.0, dtype=T)))
    plan = amd.PromptAttention(dev, dtype, heads, kv, d, lens)
    plan.run(bx.ptr, bx.ptr + (heads * d + 8) * size, bx.ptr + ((heads + kv) * d + 16) * size, bo.ptr, 0.1, (row, d), (row, d),
             (row, d), (o_tok, o_head))
    dev.sync()
    got = ora.from_bits(bo.download(ora.store_type(dtype), n * o_tok), dtype).view(n, o_tok)
    rows = got[:, :heads * o_head].reshape(n, heads, o_head)
    ora.check(rows[:, :, :d], want, tol)
    assert (rows[:, :, d:] == 7).all() and (got[:, heads * o_head:] == 7).all()
    # the same as [head][token][d]
    turned = [y.reshape(n, h, d).transpose(0, 1).contiguous() for y, h in ((q, heads), (k, kv), (v, kv))]
    bufs = [dev.put(ora.bits(y)) for y in turned]
    plan.run(*(b.ptr for b in bufs), bo.ptr, 0.1, (d, n * d), (d, n * d), (d, n * d), (d, n * d))
    dev.sync()
    again = ora.from_bits(bo.download(ora.store_type(dtype), n * heads * d), dtype).view(heads, n, d).transpose(0, 1)
    assert torch.equal(again, rows[:, :, :d])
    for b in bufs + [bx, bo]:
        b.free()


# A plan's workgroups have 16, 64 or 128 rows, by how much work there is beside its longest rows: one short prompt,
# a few of one length, many of one length.

@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("heads,kv,d,q_len,k_len", [(512, 512, 64, [129, 130], None), (768, 256, 64, [100, 45, 7], [100, 145, 4]),
                                                    (256, 256, 128, [300, 129], None), (512, 256, 80, [70, 131, 1], [75, 131, 260])])
def test_prompt_many_tiles(amd, dev, dtype, heads, kv, d, q_len, k_len):
    assert sum(-(-n * (heads // kv) // 128) for n in q_len) * kv >= 1024
    prompt(amd, dev, dtype, heads, kv, d, q_len, k_len, seed=17, oracle=ora.attend_rows)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
def test_prompt_many_tiles_with_strides_and_what_is_not_finite(amd, dev, dtype):
    """As packed, from rows with gaps and as [head][token]; then a key and values
    that are not finite, which reach the rows that see them alone."""
    heads, kv, d, lens = 512, 512, 64, [129, 130]
    clean = prompt(amd, dev, dtype, heads, kv, d, lens, seed=18, oracle=ora.attend_rows)
    T, n = ora.TYPES[dtype], sum(lens)
    q, k, v = (normal(18 + i, n, heads, d).to(T) for i in range(3))
    row, size = 3 * heads * d + 24, q.element_size()
    x = torch.zeros(n, row, dtype=T)
    for i, y in enumerate((q, k, v)):
        x[:, i * (heads * d + 8):][:, :heads * d] = y.view(n, -1)
    plan = amd.PromptAttention(dev, dtype, heads, kv, d, lens)
    bo, bx = dev.alloc(clean.numel() * size), dev.put(ora.bits(x))

    def out():
        dev.sync()
        return ora.from_bits(bo.download(ora.store_type(dtype), clean.numel()), dtype)

    plan.run(bx.ptr, bx.ptr + (heads * d + 8) * size, bx.ptr + 2 * (heads * d + 8) * size, bo.ptr, d ** -0.5, (row, d), (row, d),
             (row, d))
    assert torch.equal(out().view_as(clean), clean)
    bufs = [dev.put(ora.bits(y.transpose(0, 1).contiguous())) for y in (q, k, v)]
    plan.run(*(b.ptr for b in bufs), bo.ptr, d ** -0.5, (d, n * d), (d, n * d), (d, n * d), (d, n * d))
    assert torch.equal(out().view(heads, n, d).transpose(0, 1), clean)
    k[129 + 60, 5, 3] = math.nan
    v[129 + 20, 6, 5] = math.inf
    v[129 + 129, :, 7] = -math.inf
    more = [dev.put(ora.bits(y)) for y in (q, k, v)]
    plan.run(*(b.ptr for b in more), bo.ptr, d ** -0.5)
    got = out().view_as(clean)
    seen = torch.zeros_like(clean, dtype=torch.bool)
    seen[129 + 60:, 5] = True
    seen[129 + 20:, 6, 5] = True
    seen[129 + 129, :, 7] = True
    assert torch.equal(got[~seen], clean[~seen])
    assert not torch.isfinite(got[129 + 60:, 5].float()).any() and not torch.isfinite(got[129 + 20:, 6, 5].float()).any()
    assert not torch.isfinite(got[129 + 129, :, 7].float()).any()
    plan.close()
    for b in bufs + more + [bo, bx]:
        b.free()


# ---------------------------------------------------------------------------
# a paged cache
# ---------------------------------------------------------------------------

class Model:
    """A PagedCache and what each of its sequences holds, as float64 rows."""

    def __init__(self, amd, dev, act, dtype, layers, kv, d, page, n_pages, seed=0, garbage=math.nan):
        self.amd, self.dev, self.act, self.dtype, self.shape = amd, dev, act, dtype, (layers, kv, d, page, n_pages)
        self.cache = amd.PagedCache(dev, layers, kv, d, page, n_pages, dtype)
        fill = torch.full((n_pages * layers * 2 * kv * page * d,), garbage, dtype=ora.TYPES[dtype])
        raw = ora.bits(fill)
        amd.check(amd.lib().sllm_gfx950_h2d(c_void_p(self.cache.mem), amd.ptr(raw), raw.nbytes))
        self.rows, self.seed = {}, seed

    def memory(self):
        layers, kv, d, page, n = self.shape
        t = ora.store_type(self.dtype)
        out = np.empty(n * layers * 2 * kv * page * d, t)
        self.amd.check(self.amd.lib().sllm_gfx950_d2h(self.amd.ptr(out), c_void_p(self.cache.mem), out.nbytes))
        return ora.from_bits(out, self.dtype).view(n, layers, 2, kv, page, d)

    def new(self):
        s = self.cache.new()
        self.rows[s] = torch.zeros(self.shape[0], 2, 0, *self.shape[1:3], dtype=ora.TYPES[self.dtype])
        return s

    def step(self, seqs, n_new, heads, attend=True, scale=None, keep=False):
        """New random positions stored in every layer; each layer's attention checked."""
        layers, kv, d, page, _ = self.shape
        b = self.cache.batch(seqs, n_new, heads, self.act)
        assert b.rows == sum(n_new)
        A, T = ora.TYPES[self.act], ora.TYPES[self.dtype]
        scale = d ** -0.5 if scale is None else scale
        results = []
        for layer in range(layers):
            self.seed += 3
            q, k, v = (normal(self.seed + i, sum(n_new), h, d).to(A) for i, h in enumerate((heads, kv, kv)))
            bq, bk, bv = (self.dev.put(ora.bits(x)) for x in (q, k, v))
            bo = self.dev.alloc(max(q.numel(), 1) * q.element_size())
            b.store(layer, bk.ptr, bv.ptr)
            if attend:
                b.attend(layer, bq.ptr, bo.ptr, scale)
            self.dev.sync()
            at = 0
            for s, n in zip(seqs, n_new):
                if layer == 0:
                    r = self.rows[s]
                    self.rows[s] = torch.cat([r, torch.zeros(layers, 2, n, kv, d, dtype=T)], 2)
                r = self.rows[s]
                total = r.shape[2]
                r[layer, 0, total - n:] = k[at:at + n].to(T)
                r[layer, 1, total - n:] = v[at:at + n].to(T)
                at += n
            if attend:
                got = ora.from_bits(bo.download(ora.store_type(self.act), q.numel()), self.act).view(-1, heads, d)
                at = 0
                for s, n in zip(seqs, n_new):
                    r = self.rows[s][layer].double().numpy()
                    want, tol = ora.attend(q[at:at + n].double().numpy(), r[0], r[1], r.shape[1] - n + 1 + np.arange(n), scale,
                                           self.act, self.dtype)
                    ora.check(got[at:at + n], want, tol, f"layer {layer}, sequence {s}")
                    at += n
                results.append(got)
            for x in (bq, bk, bv, bo):
                x.free()
        if keep:
            return b, results
        b.close()
        return results

    def check_memory(self):
        """Every sequence's positions lie in its pages, bit for bit."""
        mem, page = self.memory(), self.shape[3]
        for s, r in self.rows.items():
            n = r.shape[2]
            assert self.cache.length(s) == n
            table = torch.from_numpy(self.cache.table(s)).long()
            assert len(table) == -(-n // page)
            if n:
                held = mem[table].permute(1, 2, 0, 4, 3, 5).reshape(self.shape[0], 2, -1, *self.shape[1:3])[:, :, :n]
                assert torch.equal(held, r), f"sequence {s}"

    def fork(self, s, n_tokens, n):
        out = self.cache.fork(s, n_tokens, n)
        for f in out:
            self.rows[f] = self.rows[s][:, :, :n_tokens].clone()
        return out

    def copy(self, seqs):
        out = self.cache.copy(seqs)
        for s, f in zip(seqs, out):
            self.rows[f] = self.rows[s].clone()
        return out

    def truncate(self, s, n):
        self.cache.truncate(s, n)
        self.rows[s] = self.rows[s][:, :, :n].clone()

    def free(self, seqs):
        self.cache.free(seqs)
        for s in seqs:
            del self.rows[s]

    def close(self):
        self.cache.close()


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("heads,kv,d,page", [(4, 1, 64, 16), (20, 5, 128, 64), (3, 3, 80, 32), (8, 1, 96, 16)])
def test_attend(amd, dev, act, dtype, heads, kv, d, page):
    """Sequences of nothing, one, some and many positions; no, one and several new
    ones; slots that nothing was stored to hold NaN."""
    m = Model(amd, dev, act, dtype, 2, kv, d, page, 60 if page == 16 else 30)
    s = [m.new() for _ in range(5)]
    m.step(s, [0, 1, 17, page * 3, 150], heads, attend=False)
    m.step(s, [1, 1, 1, 1, 1], heads)
    m.step(s, [0, 5, 2, 0, 9], heads)
    m.step([s[4], s[0]], [1, 3], heads)
    m.check_memory()
    m.close()


@pytest.mark.parametrize("act,dtype", PAIRS)
def test_attend_a_long_sequence_in_parts(amd, dev, act, dtype):
    m = Model(amd, dev, act, dtype, 1, 2, 128, 64, 40)
    a, b = m.new(), m.new()
    m.step([a, b], [2100, 3], 8, attend=False)
    m.step([a, b], [1, 1], 8)
    m.step([a], [7], 8)
    m.close()


@pytest.mark.parametrize("act,dtype", PAIRS)
def test_attend_a_prompt_behind_a_prefix(amd, dev, act, dtype):
    """Many new positions at once: rows in several tiles, some of them in parts."""
    m = Model(amd, dev, act, dtype, 1, 1, 64, 16, 120)
    a, b = m.new(), m.new()
    m.step([a, b], [900, 130], 4)
    m.step([a, b], [33, 200], 4)
    m.close()


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("prefix", [128, 200, 640])
def test_attend_shared_prefix(amd, dev, act, dtype, prefix):
    """Sequences that share a prefix, some of them a longer one, beside one that
    shares nothing; the prefix's pages are shared, what differs is not."""
    m = Model(amd, dev, act, dtype, 1, 2, 64, 32, 200)
    base, other = m.new(), m.new()
    m.step([base, other], [prefix, 90], 8, attend=False)
    kids = m.fork(base, prefix, 9)
    m.step([kids[0]], [300], 8, attend=False)
    grand = m.fork(kids[0], prefix + 290, 4)
    seqs = [grand[1], kids[3], other, kids[0], grand[0], kids[1], grand[3], kids[8], base]
    m.step(seqs, [1] * 9, 8)
    m.step(seqs, [1, 6, 2, 1, 40, 1, 0, 3, 1], 8)
    assert (m.cache.table(kids[3])[:prefix // 32] == m.cache.table(base)[:prefix // 32]).all()
    m.check_memory()
    m.close()


def test_attend_shared_prefix_of_many(amd, dev):
    """More rows over the prefix than one workgroup takes."""
    m = Model(amd, dev, "bfloat16", "bfloat16", 1, 1, 128, 64, 64)
    base = m.new()
    m.step([base], [700], 8, attend=False)
    kids = m.fork(base, 700, 40)
    m.step(kids, [1] * 40, 8)
    m.close()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("act,dtype", PAIRS)
def test_attend_later_drafts_do_not_reach_earlier_rows(amd, dev, act, dtype, bad):
    """A value that is not finite at the last of five new positions: the rows
    before it are as without it."""
    heads, kv, d = 4, 2, 64
    got = []
    for edit in (False, True):
        c = amd.PagedCache(dev, 1, kv, d, 16, 20, dtype)
        s = c.new()
        A = ora.TYPES[act]
        for n, last in ((70, False), (5, True)):
            b = c.batch([s], [n], heads, act)
            q, k, v = (normal(31 + i + n, n, h, d).to(A) for i, h in enumerate((heads, kv, kv)))
            if edit and last:
                k[4, 0, 0] = bad
                v[4, 1, 9] = bad
            bq, bk, bv = (dev.put(ora.bits(x)) for x in (q, k, v))
            bo = dev.alloc(q.numel() * q.element_size())
            b.store(0, bk.ptr, bv.ptr)
            b.attend(0, bq.ptr, bo.ptr, 0.125)
            dev.sync()
            out = ora.from_bits(bo.download(ora.store_type(act), q.numel()), act).view(n, heads, d)
            b.close()
            for x in (bq, bk, bv, bo):
                x.free()
        got.append(out)
        c.close()
    assert torch.isfinite(got[1][:4].float()).all() and torch.equal(got[0][:4], got[1][:4])
    assert not torch.isfinite(got[1][4, 2:, 9].float()).any()


def test_attend_f32_rows_of_any_size_over_an_f16_cache(amd, dev):
    """Queries far outside f16's range."""
    m = Model(amd, dev, "float32", "float16", 1, 2, 64, 16, 20)
    s = m.new()
    m.step([s], [60], 4, attend=False)
    for scale in (1e-6, 1e6):
        b = m.cache.batch([s], [1], 4, "float32")
        q = normal(5, 1, 4, 64) / scale * 3
        k, v = normal(6, 1, 2, 64), normal(7, 1, 2, 64)
        bufs = [dev.put(x.numpy()) for x in (q, k, v)]
        bo = dev.alloc(4 * 256)
        b.store(0, bufs[1].ptr, bufs[2].ptr)
        b.attend(0, bufs[0].ptr, bo.ptr, 0.125 * scale)
        dev.sync()
        r = torch.cat([m.rows[s][0], torch.stack([k, v]).half()], 1).double().numpy()
        want, tol = ora.attend(q.double().numpy(), r[0], r[1], [r.shape[1]], 0.125 * scale, "float32", "float16")
        ora.check(torch.from_numpy(bo.download(np.float32, 256)), want, tol)
        b.close()
        m.cache.truncate(s, 60)
    m.close()


def test_attend_strides_and_memory_around(amd, dev):
    """Rows apart in q, k, v and out; a cache in the caller's memory, with what
    lies around it left alone."""
    heads, kv, d, page, pages = 6, 2, 64, 16, 12
    desc = amd.PagesDesc(1, kv, d, page, pages, 1, None)
    size = amd.lib().sllm_gfx950_pages_bytes(ctypes.byref(desc))
    assert size == pages * 2 * kv * page * d * 2
    mem = dev.put(np.full(size // 2 + 256, 0x7e00, np.uint16))       # NaN
    c = amd.PagedCache(dev, 1, kv, d, page, pages, "float16", mem=mem.ptr + 256)
    s = [c.new(), c.new()]
    n_new = [40, 25]
    b = c.batch(s, n_new, heads)
    n, row = sum(n_new), (heads + 2 * kv) * d + 8
    x = normal(41, n, row).half()
    bx, bo = dev.put(ora.bits(x)), dev.put(np.full(n * (heads * d + 16), 0x4700, np.uint16))
    b.store(0, bx.ptr + heads * d * 2, bx.ptr + (heads + kv) * d * 2, row, row)
    b.attend(0, bx.ptr, bo.ptr, 0.125, row, heads * d + 16)
    dev.sync()
    got = ora.from_bits(bo.download(np.int16, n * (heads * d + 16)), "float16").view(n, -1)
    assert (got[:, heads * d:] == 7).all()
    at = 0
    for m in n_new:
        part = x[at:at + m].double()
        q, k, v = (part[:, a * d:(a + h) * d].reshape(m, h, d).numpy() for a, h in ((0, heads), (heads, kv), (heads + kv, kv)))
        want, tol = ora.attend(q, k, v, np.arange(m) + 1, 0.125, "float16", "float16")
        ora.check(got[at:at + m, :heads * d], want, tol)
        at += m
    raw = mem.download(np.uint16, size // 2 + 256)
    assert (raw[:128] == 0x7e00).all() and (raw[-128:] == 0x7e00).all()
    held = raw[128:-128].reshape(pages, 2, kv, page, d)
    table = list(c.table(s[0])) + list(c.table(s[1]))
    left = np.ones((pages, page), bool)
    for t, m in ((c.table(s[0]), 40), (c.table(s[1]), 25)):
        for j in range(m):
            left[t[j // page], j % page] = False
    assert sorted(table) == list(range(5))
    assert (held.transpose(0, 3, 1, 2, 4)[left] == 0x7e00).all()
    b.close()
    c.close()
    for y in (mem, bx, bo):
        y.free()


def test_store_rounds_to_nearest(amd, dev):
    """f32 rows into an f16 cache: ties to even, what is too large to infinity."""
    x = np.array([1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 65519.9, 65520.0, -1e30, 2.0 ** -25, 2.0 ** -25 * 1.01, np.nan], np.float32)
    c = amd.PagedCache(dev, 1, 1, 8, 16, 1, "float16")
    b = c.batch([c.new()], [1], 1, "float32")
    k, v = dev.put(x), dev.put(-x)
    b.store(0, k.ptr, v.ptr)
    dev.sync()
    out = np.empty(2 * 16 * 8, np.uint16)
    amd.check(amd.lib().sllm_gfx950_d2h(amd.ptr(out), c_void_p(c.mem), out.nbytes))
    out = out.view(np.float16).reshape(2, 16, 8)
    with np.errstate(over="ignore"):
        assert np.array_equal(out[0, 0], x.astype(np.float16), equal_nan=True)
        assert np.array_equal(out[1, 0], (-x).astype(np.float16), equal_nan=True)
    b.close()
    c.close()
    k.free(), v.free()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_pages_life(amd, dev, dtype):
    """Random forks, copies, truncations, steps, ends and compactions: every
    sequence keeps its own positions, bit for bit, and no page is lost."""
    m = Model(amd, dev, dtype, dtype, 2, 2, 64, 16, 150, garbage=5.0)
    r = np.random.RandomState(3)
    live = [m.new()]
    for i in range(120):
        what = r.randint(7)
        pick = live[r.randint(len(live))] if live else None
        room = m.shape[4] - m.cache.in_use()
        if (what <= 2 or pick is None) and room > 30:
            if not live or r.randint(3) == 0:
                live.append(m.new())
            some = list(r.permutation(live)[:4])
            m.step([int(s) for s in some], [int(r.randint(0, 40)) for _ in some], 4, attend=i % 10 == 0)
        elif what == 3 and pick is not None and room > 10 and len(live) < 12:
            live += m.fork(pick, int(r.randint(0, m.rows[pick].shape[2] + 1)), int(r.randint(1, 4)))
        elif what == 4 and pick is not None and room > 40 and len(live) < 12:
            live += m.copy([pick])
        elif what == 5 and pick is not None:
            m.truncate(pick, int(r.randint(0, m.rows[pick].shape[2] + 1)))
        elif live:
            m.free([pick])
            live.remove(pick)
        if i % 15 == 14:
            used = m.cache.in_use()
            before = [m.cache.table(s) for s in live]
            moved = m.cache.compact()
            assert moved == len({int(p) for t in before for p in t if p >= used})
            assert m.cache.in_use() == used and all((m.cache.table(s) < used).all() for s in live)
        if i % 8 == 7:
            m.check_memory()
            assert m.cache.in_use() == len({int(p) for s in live for p in m.cache.table(s)})
    m.check_memory()
    m.close()


def test_a_step_of_a_layer(amd, dev):
    """The operators as a layer uses them: projections of a batch's tokens, the new
    rows stored, attention, the output quantised for the next projection."""
    e, heads, kv, d = 512, 8, 2, 64
    m = Model(amd, dev, "float32", "float32", 1, kv, d, 16, 60)
    seqs = [m.new() for _ in range(3)]
    m.step(seqs, [33, 1, 100], heads, attend=False)
    n_new = [1, 2, 1]
    n = sum(n_new)
    w = {name: dev.put(amd.synth_i2s(amd.synth_seed(7, 0, 0, i), rows, e))
         for i, (name, rows) in enumerate((("q", e), ("k", kv * d), ("v", kv * d)))}
    x = normal(51, n, e)
    bx, bq8, bact = dev.put(x.numpy()), dev.alloc(n * e), dev.alloc(8 * n)
    out = {name: dev.alloc(4 * n * (e if name == "q" else kv * d)) for name in w}
    dev.linear_batch(w["q"].vp, e, e, bx.vp, n, bq8.vp, bact.vp, out["q"].vp)
    dev.gemm(w["k"].vp, kv * d, e, bq8.vp, bact.vp, n, out["k"].vp)
    dev.gemm(w["v"].vp, kv * d, e, bq8.vp, bact.vp, n, out["v"].vp)
    b = m.cache.batch(seqs, n_new, heads)
    att = dev.alloc(4 * n * e)
    b.store(0, out["k"].ptr, out["v"].ptr)
    b.attend(0, out["q"].ptr, att.ptr, 1e-4)
    q8, act = dev.alloc(n * e), dev.alloc(8 * n)
    dev.quant_act(att.vp, e, n, q8.vp, act.vp)
    dev.sync()
    got = {name: torch.from_numpy(o.download(np.float32, o.nbytes // 4)).view(n, -1, d) for name, o in out.items()}
    a = torch.from_numpy(att.download(np.float32, n * e)).view(n, heads, d)
    at = 0
    for s, k in zip(seqs, n_new):
        keys, values = (torch.cat([m.rows[s][0, i], got[c][at:at + k]]).double().numpy() for i, c in enumerate("kv"))
        want, tol = ora.attend(got["q"][at:at + k].double().numpy(), keys, values, len(keys) - k + 1 + np.arange(k), 1e-4,
                               "float32", "float32")
        ora.check(a[at:at + k], want, tol)
        at += k
    # the quantiser's rows are those of what attention wrote
    scale = np.frombuffer(act.download(np.uint8, 8 * n).tobytes(), [("s", "<f4"), ("n", "<i4")])["s"]
    assert np.array_equal(scale, np.float32(127) / np.abs(a.view(n, -1).numpy()).max(1))
    b.close()
    m.close()
    for y in [bx, bq8, bact, att, q8, act] + list(w.values()) + list(out.values()):
        y.free()


def test_offsets_past_32_bits(amd, dev):
    """A cache of more than 4 GiB, a sequence at its end."""
    kv, d, page = 8, 128, 64
    pages = (5 << 30) // (2 * kv * page * d * 2)
    c = amd.PagedCache(dev, 1, kv, d, page, pages, "float16")
    first, s = c.new(), c.new()
    c.batch([first], [(pages - 4) * page], kv).close()
    heads, n = 16, 150
    b = c.batch([s], [n], heads)
    assert int(c.table(s).min()) * 2 * kv * page * d * 2 > 1 << 32
    q, k, v = (normal(61 + i, n, h, d).half() for i, h in enumerate((heads, kv, kv)))
    bq, bk, bv = (dev.put(ora.bits(x)) for x in (q, k, v))
    bo = dev.alloc(q.numel() * 2)
    b.store(0, bk.ptr, bv.ptr)
    b.attend(0, bq.ptr, bo.ptr, 0.1)
    copy = None
    dev.sync()
    got = ora.from_bits(bo.download(np.int16, q.numel()), "float16").view(n, heads, d)
    want, tol = ora.attend(*(x.double().numpy() for x in (q, k, v)), np.arange(n) + 1, 0.1, "float16", "float16")
    ora.check(got, want, tol)
    b.close()
    c.free([first])
    assert c.compact() == 3 and c.table(s).max() == 2
    b = c.batch([s], [1], heads)
    copy = c.fork(s, n, 1)
    b.attend(0, bq.ptr, bo.ptr, 0.1)                # (position n was never stored: only that it runs within its pages)
    dev.sync()
    assert c.length(copy[0]) == n
    b.close()
    c.close()
    for x in (bq, bk, bv, bo):
        x.free()


def test_batch_in_a_graph(amd, dev):
    """Store and attend captured once and replayed, eager work in between: every
    replay gives what the eager calls give; two graphs of two batches share the
    cache's memory."""
    torch.cuda.init()
    stream = torch.cuda.ExternalStream(amd.lib().sllm_gfx950_stream())
    c = amd.PagedCache(dev, 1, 2, 64, 16, 80, "float16")
    heads, kv, d = 8, 2, 64
    base = c.new()
    x = normal(71, 400, kv, d).half()
    bx = dev.put(ora.bits(x))
    b0 = c.batch([base], [400], heads)
    b0.store(0, bx.ptr, bx.ptr)
    b0.close()
    jobs = []
    for j in range(2):
        seqs = c.fork(base, 390 - 7 * j, 3 + j)
        b = c.batch(seqs, [2] * len(seqs), heads)
        n = b.rows
        q, k, v = (normal(80 + 10 * j + i, n, h, d).half() for i, h in enumerate((heads, kv, kv)))
        bufs = [dev.put(ora.bits(y)) for y in (q, k, v)] + [dev.alloc(q.numel() * 2)]

        def call(b=b, bufs=bufs):
            b.store(0, bufs[1].ptr, bufs[2].ptr)
            b.attend(0, bufs[0].ptr, bufs[3].ptr, 0.125)

        call()
        dev.sync()
        want = bufs[3].download(np.int16, q.numel())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
            call()
        jobs.append((call, g, want, bufs, b))
    for turn in range(3):
        for call, g, want, bufs, _ in jobs:
            zero = np.zeros(want.size, np.int16)
            bufs[3].upload(zero)
            with torch.cuda.stream(stream):
                g.replay()
            dev.sync()
            assert np.array_equal(bufs[3].download(np.int16, want.size), want), turn
        jobs[turn % 2][0]()                          # eager, between the replays
        dev.sync()
    for _, _, _, bufs, b in jobs:
        b.close()
        for y in bufs:
            y.free()
    c.close()
    bx.free()


def test_what_takes_pages_is_refused_in_a_capture(amd, dev):
    torch.cuda.init()
    stream = torch.cuda.ExternalStream(amd.lib().sllm_gfx950_stream())
    m = Model(amd, dev, "float16", "float16", 1, 2, 64, 16, 40)
    s = m.new()
    b, first = m.step([s], [50], 4, keep=True)
    q = normal(m.seed, 50, 4, 64).half()
    bq, bo = dev.put(ora.bits(q)), dev.alloc(q.numel() * 2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
        for call in (lambda: m.cache.batch([s], [1], 4, "float16"), lambda: m.cache.fork(s, 37, 1), lambda: m.cache.copy([s]),
                     m.cache.compact, lambda: amd.PromptAttention(dev, "float16", 4, 2, 64, [9])):
            with pytest.raises(amd.GFX950Error, match="captured"):
                call()
        b.attend(0, bq.ptr, bo.ptr, 0.125)
    assert m.cache.length(s) == 50 and m.cache.in_use() == 4
    for _ in range(3):
        bo.upload(np.zeros(q.numel(), np.int16))
        with torch.cuda.stream(stream):
            g.replay()
        dev.sync()
        assert torch.equal(ora.from_bits(bo.download(np.int16, q.numel()), "float16").view_as(first[0]), first[0])
        m.check_memory()
    b.close()
    m.close()
    bq.free(), bo.free()


def test_the_same_call_gives_the_same_bits(amd, dev):
    m = Model(amd, dev, "float16", "float16", 1, 2, 128, 32, 120)
    base = m.new()
    m.step([base], [1500], 8, attend=False)
    kids = m.fork(base, 1490, 20)
    b, first = m.step(kids, [1] * 20, 8, keep=True)
    m.seed -= 3
    q = normal(m.seed + 3, 20, 8, 128).half()
    bq, bo = dev.put(ora.bits(q)), dev.alloc(q.numel() * 2)
    for _ in range(3):
        b.attend(0, bq.ptr, bo.ptr, 128 ** -0.5)
        dev.sync()
        assert torch.equal(ora.from_bits(bo.download(np.int16, q.numel()), "float16").view_as(first[0]), first[0])
    b.close()
    m.close()
    bq.free(), bo.free()
