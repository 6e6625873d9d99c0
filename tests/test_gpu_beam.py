"""The best continuations of beams (sllm_gfx950_attn.h) on the GPU, against 64 bits."""
import math

import numpy as np
import pytest
import torch

import attn_oracle as ora

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


def oracle(x, scores, ended, picks):
    """(scores, beams, tokens, tolerance) [groups][picks] of logits x [groups, beams, vocab] (float64).

    Tolerance: an exponential's argument is off by half a step of x - max and of its product,
    2^-23 |x - max| in all, the exponential by 2^-22 (two steps), sixteen values are summed
    in f32, the rest in f64: the log of the sum is off by the weighted mean of these and 2^-20.
    The result is rounded to f32."""
    groups, beams, vocab = x.shape
    out = []
    for g in range(groups):
        rows = []
        for b in range(beams):
            v, s, tol = np.where(np.isnan(x[g, b]), -np.inf, x[g, b]), scores[g, b], 0.0
            order = np.argsort(-v, kind="stable")
            n = min(picks, vocab)
            if ended is not None and ended[g, b] >= 0:
                t = np.concatenate([[ended[g, b]], [i for i in range(n) if i != ended[g, b]]])[:n]
                w = np.full(n, -np.inf)
                w[0] = s if np.isfinite(s) else -np.inf
                if not np.isfinite(s):
                    t = np.arange(n)
            elif not np.isfinite(s) or not np.isfinite(v.max()):
                t, w = np.arange(n), np.full(n, -np.inf)
            else:
                d = v - v.max()
                p = np.exp(d)
                t = order[:n]
                w = s + d[t] - math.log(p.sum())
                fine = p > 0
                tol = (p[fine] * (2.0 ** -22 - d[fine] * 2.0 ** -23)).sum() / p.sum() + 2.0 ** -20
            rows += [(-w[i], b, i, int(t[i]), tol) for i in range(n)]
        rows.sort(key=lambda r: r[:3])
        out.append(rows[:picks])
    get = lambda i: np.array([[r[i] for r in g] for g in out])      # noqa: E731
    return -get(0), get(1), get(3), get(4)


class Select:
    def __init__(self, amd, dev, x, scores, ended, picks, dtype, stride=0):
        self.dev, (g, b, v) = dev, x.shape
        self.shape, self.stride = (g, picks), stride
        t = torch.full((g * b, stride or v), 9.0, dtype=ora.TYPES[dtype])
        t[:, :v] = x.reshape(g * b, v)
        self.bufs = [dev.put(ora.bits(t)), dev.put(np.asarray(scores, np.float32))] + ([dev.put(np.asarray(ended, np.int32))] if ended is not None else [])
        self.out = [dev.put(np.full(g * picks + 8, 77, np.int32)) for _ in range(3)]
        self.plan = amd.BeamSelect(dev, g, b, v, picks, dtype)
        self.ptrs = [self.bufs[0].ptr, self.bufs[1].ptr, self.bufs[2].ptr if ended is not None else None] + [o.ptr for o in self.out]

    def run(self):
        self.plan.run(*self.ptrs, stride=self.stride)

    def read(self):
        self.dev.sync()
        n, got = self.shape[0] * self.shape[1], []
        for i, o in enumerate(self.out):
            y = o.download(np.int32, n + 8)
            assert (y[n:] == 77).all()
            got.append((y[:n].view(np.float32) if i == 0 else y[:n]).reshape(self.shape))
        return got

    def close(self):
        self.plan.close()
        for b in self.bufs + self.out:
            b.free()


def check(amd, dev, x, scores, picks, dtype="float32", ended=None, stride=0):
    x = x.to(ora.TYPES[dtype])
    s = Select(amd, dev, x, scores, ended, picks, dtype, stride)
    s.run()
    got = s.read()
    want, beam, token, tol = oracle(x.double().numpy(), np.asarray(scores, np.float32).astype(np.float64), ended, picks)
    assert np.array_equal(got[2], token), (got[2], token)
    assert np.array_equal(got[1], beam)
    live = np.isfinite(want)
    assert np.array_equal(np.isneginf(got[0]), ~live)
    assert (np.abs(got[0][live] - want[live]) <= tol[live] + 2.0 ** -23 * (np.abs(want[live]) + 1)).all()
    s.run()                                                          # the same call, the same bits
    again = s.read()
    assert all(np.array_equal(p.view(np.int32), q.view(np.int32)) for p, q in zip(got, again))
    s.close()
    return got


def scores_of(seed, groups, beams):
    return -4 - 3 * np.random.default_rng(seed).random((groups, beams)).astype(np.float32)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("groups,beams,vocab,picks", [(1, 1, 1, 1), (1, 4, 7, 8), (2, 3, 255, 64), (3, 5, 1009, 10), (2, 4, 4096, 8), (2, 2, 4097, 3),
                                                      (1, 4, 128256, 8), (3, 8, 32003, 16), (2, 32, 5000, 64), (1, 64, 999, 32), (40, 1, 20001, 5),
                                                      (1, 1, 300001, 64)])
def test_select(amd, dev, dtype, groups, beams, vocab, picks):
    x = normal(vocab + picks, groups, beams, vocab) * 2.5
    check(amd, dev, x, scores_of(1, groups, beams), picks, dtype)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("vocab,stride", [(1001, 1003), (1000, 1001), (999, 1024), (4099, 4101)])
def test_strides(amd, dev, dtype, vocab, stride):
    check(amd, dev, normal(5, 3, 3, vocab) * 2, scores_of(2, 3, 3), 7, dtype, stride=stride)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("order", ["rising", "falling", "alike", "steps", "two"])
@pytest.mark.parametrize("vocab", [300, 20000])
def test_orders_that_keep_the_list_moving(amd, dev, dtype, order, vocab):
    """Values that rise with the token (each is the best so far), fall, or are alike: ties to the lower token."""
    i = torch.arange(vocab).float()
    x = {"rising": i / 64 % 4096 / 256 + i / vocab, "falling": -i / vocab * 8, "alike": torch.full((vocab,), 0.25), "steps": (i / 7).floor() % 5,
         "two": (i % 2 == 0).float()}[order]
    check(amd, dev, x.expand(2, 3, vocab).contiguous(), [[-1.0, -2.5, -4.0]] * 2, 20, dtype)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("picks", [1, 7, 33, 64])
@pytest.mark.parametrize("seed", range(6))
def test_few_values_many_ties(amd, dev, dtype, picks, seed):
    """Values from a handful, in runs of every length: which of those that are alike are
    among the picks is the token's alone, however a wave comes by them."""
    r = np.random.default_rng(seed)
    x = torch.zeros(2, 2, 6000)
    for g in range(2):
        for b in range(2):
            at = 0
            while at < 6000:
                n = int(r.choice([1, 4, 8, 31, 64, 128, 300]))
                x[g, b, at:at + n] = float(r.choice([0.0, 0.0, 1.0, 1.0, 2.0] if seed % 2 else [0.0, 0.0, 0.0, 0.0, 3.0]))
                at += n
    x[0, 0, :] = 0
    x[0, 0, 256:320], x[0, 0, 64:128] = 5.0, 5.0
    check(amd, dev, x, [[-1.0, -30.0], [-1.0, -1.5]], picks, dtype)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("vocab", [1001, 9000])
def test_beams_that_are_alike(amd, dev, dtype, vocab):
    """The same logits and scores: the lower beam first, wherever its row lies in memory."""
    x = (normal(6, 1, 1, vocab) * 2).expand(2, 4, vocab).contiguous()
    got = check(amd, dev, x, np.full((2, 4), -2.0), 12, dtype)
    assert np.array_equal(got[1], np.tile(np.arange(12) % 4, (2, 1)))


def test_ended_and_dead_beams(amd, dev):
    vocab = 5003
    x = normal(7, 3, 4, vocab) * 2
    ended = np.full((3, 4), -1, np.int32)
    ended[0, 1], ended[1, :], ended[2, 3] = 2, [0, 5, 1, 5002], 7
    scores = scores_of(3, 3, 4)
    scores[0, 3], scores[2, 0], scores[2, 3] = -np.inf, np.nan, -np.inf
    check(amd, dev, x, scores, 9, ended=ended)
    first = np.full((3, 4), -np.inf, np.float32)                 # a first step: one beam, and more picks than it has tokens
    first[:, 0] = 0
    check(amd, dev, x[:, :, :5].contiguous(), first, 9)
    check(amd, dev, x[:, :, :3].contiguous(), scores, 12, ended=np.where(ended > 2, 1, ended))
    check(amd, dev, x, np.full((3, 4), -np.inf), 20)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
def test_masked_logits(amd, dev, dtype):
    """-infinity, the type's lowest value, NaN and +infinity among the logits; a row of nothing else."""
    vocab, low = 4500, torch.finfo(ora.TYPES[dtype]).min
    x = normal(8, 2, 6, vocab) * 2
    x[0, 0, 3:] = -math.inf
    x[0, 1, 1:] = low
    x[0, 2] = -math.inf
    x[0, 3] = low
    x[0, 4, ::3] = math.nan
    x[0, 5] = math.nan
    x[1, 0, 77] = math.inf
    x[1, 1, 4400:] = -math.inf
    x[1, 2, :4400] = -math.inf
    x[1, 3, 4499] = 60.0 if dtype != "float16" else 40.0
    x[1, 4] = 1000.0 + x[1, 4]
    check(amd, dev, x, scores_of(4, 2, 6), 30, dtype)


def test_large_logits(amd, dev):
    x = normal(9, 1, 3, 5000) * 1e30
    x[0, 1] = x[0, 1] * 1e-36
    check(amd, dev, x, scores_of(5, 1, 3), 10)


def test_in_graphs(amd, dev):
    """Two plans captured, replayed with eager calls between, and new logits between replays."""
    torch.cuda.init()
    stream = torch.cuda.ExternalStream(amd.lib().sllm_gfx950_stream())
    jobs = []
    for j, (g, b, v, k, dtype) in enumerate([(2, 4, 20001, 8, "bfloat16"), (1, 3, 500, 12, "float32")]):
        x, y = (normal(20 + 2 * j + i, g, b, v).to(ora.TYPES[dtype]) for i in range(2))
        s = Select(amd, dev, x, scores_of(j, g, b), None, k, dtype)
        s.run()
        dev.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            s.run()
            with pytest.raises(amd.GFX950Error, match="captured"):
                amd.BeamSelect(dev, 1, 1, 100, 1)
        jobs.append((s, graph, [x, y]))
    for turn in range(4):
        for s, graph, data in jobs:
            s.bufs[0].upload(ora.bits(data[turn % 2]))
            s.run()
            want = s.read()
            for o in s.out:
                o.upload(np.full(s.shape[0] * s.shape[1] + 8, 77, np.int32))
            with torch.cuda.stream(stream):
                graph.replay()
            assert all(np.array_equal(p.view(np.int32), q.view(np.int32)) for p, q in zip(s.read(), want)), turn
    for s, _, _ in jobs:
        s.close()


def test_beam_search_over_a_cache(amd, dev):
    """Two requests of three beams, four steps over a cache of 8 bits: each step's picks reorder the
    sequences, and the rows that they then hold are those of the tokens that were picked."""
    groups, beams, vocab, kv, d = 2, 3, 400, 1, 64
    table = normal(30, vocab, kv, d).to(torch.bfloat16)          # a token's keys and values
    c = amd.PagedCache(dev, 1, kv, d, 16, 40, "int8")
    plan = amd.BeamSelect(dev, groups, beams, vocab, beams)
    ids = [c.new() for _ in range(groups * beams)]
    history = [[] for _ in ids]
    scores = np.full((groups, beams), -np.inf, np.float32)
    scores[:, 0] = 0
    out = [dev.alloc(4 * groups * beams) for _ in range(3)]
    for step in range(20):
        x = normal(40 + step, groups, beams, vocab) * 2
        bx, bs = dev.put(x.numpy()), dev.put(scores)
        plan.run(bx.ptr, bs.ptr, None, *(o.ptr for o in out))
        dev.sync()
        scores, parent, token = (o.download(t, groups * beams).reshape(groups, beams) for o, t in zip(out, (np.float32, np.int32, np.int32)))
        at = (parent + beams * np.arange(groups)[:, None]).ravel().tolist()
        c.reorder(ids, at)
        history = [history[p] + [int(t)] for p, t in zip(at, token.ravel())]
        b = c.batch(ids, [1] * len(ids), 2, "bfloat16")
        rows = dev.put(ora.bits(table[torch.from_numpy(token.ravel()).long()].contiguous()))
        b.store(0, rows.ptr, rows.ptr)
        back = [dev.alloc(b.positions * kv * d * 2) for _ in range(2)]
        b.read(0, back[0].ptr, back[1].ptr)
        dev.sync()
        if step % 5 == 4 or step < 3:
            import held8_oracle as h8
            held = torch.from_numpy(h8.held(table.double().numpy(), "int8")).bfloat16()
            want = torch.cat([held[torch.tensor(h)] for h in history])
            for y in back:
                assert torch.equal(ora.from_bits(y.download(np.int16, want.numel()), "bfloat16").view_as(want), want), step
        b.close()
        for y in [bx, bs, rows] + back:
            y.free()
    assert np.isfinite(scores).all()
    plan.close()
    c.close()
    for o in out:
        o.free()
