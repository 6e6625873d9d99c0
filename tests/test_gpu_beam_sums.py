"""How exact the selection's logarithms of sums are (sllm_gfx950_attn.h) on the GPU, and the
order of beams whose sums are nearer to each other than that."""
import math

import numpy as np
import pytest
import torch

import attn_oracle as ora
from test_gpu_beam import Select, normal, scores_of

pytestmark = pytest.mark.gpu

STEP = 2048                          # logits that the four waves of a part take in a turn


def totals(x, scores):
    """score + logit - log sum of every continuation of x [beams, vocab] (float64), and what each beam's may be off by.

    u = 2^-24, d how far a logit lies below its beam's largest. An exponential's argument D is
    a difference rounded to f32, times log2(e) rounded to f32, rounded: 2.25 u D; the exponential
    itself 2 u (a step). A logit is taken relative to a reference at most 1 below the
    largest so far; what was summed is scaled by another exponential where the reference rises, by
    1 or more each time, and once at the end: at most d + 3 exponentials of together d + 2. Eight
    terms are summed in f32 (7 u), the rest in f64. So a term is off by u (4.25 d + 17.5) relative
    to itself, and the logarithm by the mean of that over the terms by their weight; then it is rounded to f32."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max(-1, keepdims=True)
    p = np.exp(x - top)
    s = p.sum(-1, keepdims=True)
    d = np.where(p > 0, top - x, 0.0)
    tol = (p * (17.5 + 4.25 * d)).sum(-1, keepdims=True) / s * 2.0 ** -24
    return scores[:, None] + (x - top) - np.log(s), tol[:, 0]


def check(amd, dev, x, scores, picks, dtype):
    """Every pick is worth what is said, none is named twice, they are in order, and what was
    left out is no better than the last by more than the two may be off."""
    x, scores = x.to(ora.TYPES[dtype]), np.asarray(scores, np.float32)
    s = Select(amd, dev, x, scores, None, picks, dtype)
    s.run()
    got, beam, token = s.read()
    s.close()
    for g in range(len(x)):
        want, tol = totals(x[g].double().numpy(), scores[g].astype(np.float64))
        mine = want[beam[g], token[g]]
        off = tol[beam[g]] + 2.0 ** -23 * (np.abs(mine) + 1)
        assert (np.abs(got[g] - mine) <= off).all(), (g, np.abs(got[g] - mine).max(), off)
        assert (np.diff(got[g]) <= 0).all()
        assert len(set(zip(beam[g].tolist(), token[g].tolist()))) == picks
        rest = (want - 2 * tol.max()).copy()
        rest[beam[g], token[g]] = -np.inf
        assert rest.max() <= mine.min()
    return got, beam, token


RISES = [(1 + k / 512) * 2.0 ** e for k, e in ((246, -10), (1, -12), (373, -12), (14, -10), (268, -8), (0, -9), (256, -13), (300, -5), (9, -1), (11, 0), (0, 5))]


@pytest.mark.parametrize("dtype,by", [("float32", b) for b in RISES] + [("bfloat16", 1.0), ("float16", 0.25)])
def test_logits_that_rise_all_along(amd, dev, dtype, by):
    """The same step up every 2048 logits: what a rise's rescaling leaves does not add up. (A
    step's exponential is off by the same part of itself each time: over 120 of them the sum was off by
    2^-19 with a reference that rose with every step.)"""
    vocab = STEP * 64 * (120 if dtype == "float32" else 3) + 37
    x = ((torch.arange(vocab) // STEP).double() * by).float()
    score = math.log(torch.exp(x.double() - x.max()).sum())      # so that the best is worth about 0, where f32 is fine
    check(amd, dev, x.expand(1, 1, -1), [[score]], 5, dtype)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("vocab", [1009, 32003, 128256])
def test_sums_of_logits_in_other_orders(amd, dev, dtype, vocab):
    """Beams with the same logits in another order, whose sums are the same: in any order
    among themselves, but worth what is said."""
    x = normal(3, vocab) * 2.5
    g = torch.Generator()
    g.manual_seed(4)
    x = torch.stack([x[torch.randperm(vocab, generator=g)] for _ in range(6)])[None]
    check(amd, dev, x, np.full((1, 6), -2.0), 20, dtype)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
def test_scores_a_step_apart(amd, dev, dtype):
    """The same logits and scores one step of f32 apart: that alone decides, in 64 bits."""
    vocab, beams = 20001, 8
    x = (normal(5, vocab) * 2).to(ora.TYPES[dtype]).float()
    x[777] = 20.0                                                # one token for each beam
    order = np.array([3, 0, 7, 1, 6, 2, 5, 4])
    scores = np.float32(-2.0) - order.astype(np.float32) * np.float32(2.0 ** -22)
    got, beam, token = check(amd, dev, x.expand(1, beams, vocab).contiguous(), scores[None], beams, dtype)
    assert np.array_equal(beam[0], np.argsort(order)) and (token == 777).all()


@pytest.mark.parametrize("dtype", list(ora.TYPES))
def test_many_beams_of_random_logits(amd, dev, dtype):
    check(amd, dev, normal(6, 8, 8, 32000) * 2.5, scores_of(7, 8, 8), 32, dtype)
    check(amd, dev, normal(8, 1, 4, 50001) / 64, scores_of(9, 1, 4), 16, dtype)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("groups,beams,vocab,picks", [(1 << 20, 1, 9, 3), (1 << 14, 64, 5, 32)])
def test_as_many_rows_as_a_plan_takes(amd, dev, dtype, groups, beams, vocab, picks):
    x = (normal(11, groups, beams, vocab) * 2).to(ora.TYPES[dtype])
    scores = -torch.rand(groups, beams, generator=torch.Generator().manual_seed(12))
    s = Select(amd, dev, x, scores.numpy(), None, picks, dtype)
    s.run()
    got, beam, token = (torch.from_numpy(y) for y in s.read())
    s.close()
    want = (scores.double()[..., None] + torch.log_softmax(x.double(), -1)).view(groups, -1)
    mine = want.gather(1, beam.long() * vocab + token.long())
    assert ((got.double() - mine).abs() <= 2.0 ** -17 + 2.0 ** -23 * (mine.abs() + 1)).all()
    assert (got[:, 1:] <= got[:, :-1]).all()
    best = want.topk(picks, 1).values                            # (in order, up to what logarithms are off by)
    assert ((mine - best).abs() <= 2.0 ** -16).all()
    at = (beam.long() * vocab + token.long()).sort(1).values
    assert (at[:, 1:] != at[:, :-1]).all()
