"""Queries of any size and shape over a paged cache (sllm_gfx950_attn.h) on the GPU,
f32 rows over an f16 cache above all: a row whose elements are many powers of two
apart, rows at the ends of f32's range, rows of zeros, keys with infinite elements.
Tolerances: attn_bounds.py."""
import math

import numpy as np
import pytest
import torch

import attn_bounds as bounds
import attn_oracle as ora

pytestmark = pytest.mark.gpu

PAIRS = [("float32", "float32"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")]
# new positions of two rows each: 16, 64 and 128 rows a workgroup
N_NEW = [1, 25, 70]


def normal(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("n_new", N_NEW)
@pytest.mark.parametrize("d,outlier", [(8, 3e4), (64, 300.0)])
def test_small_elements_beside_a_large_one_meet_a_large_key(amd, dev, act, dtype, n_new, d, outlier):
    """One element of the query is 3, the others are small, and so is the product of
    one of them with a key's outlier: what it adds to a score is all there is between
    the keys."""
    n, T = 300, ora.TYPES[act]
    q = normal(1, n_new, 2, d) * (3.0 / outlier)
    q[:, :, 0] = 3.0
    k, v = normal(2, n, 1, d) * 1e-3, normal(3, n, 1, d)
    k[:, :, 5] = outlier * normal(4, n, 1).sign()
    bounds.check_step(amd, dev, act, dtype, 2, [(k.to(T), v.to(T))], q.to(T), [n_new], 1.0, page=32)


@pytest.mark.parametrize("exponent", [-149, -140, -126, -113, -101, -100, -60, 60, 99, 100, 112, 113, 116, 127])
def test_f32_rows_at_the_ends_of_the_range(amd, dev, exponent):
    """Rows of up to 2^exponent, with the scale that makes their scores ordinary (as far as
    there is one: less than 2^-126 or over 2^126 it is not)."""
    n, n_new, d = 90, 3, 64
    q = torch.from_numpy(np.ldexp(np.random.RandomState(7).uniform(-1, 1, (n_new, 4, d)), exponent).astype(np.float32))
    scale = 2.0 ** max(min(-exponent - 1, 126), -126)
    seqs = [(normal(8, n, 2, d), normal(9, n, 2, d))]
    got = bounds.check_step(amd, dev, "float32", "float16", 4, seqs, q, [n_new], scale)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("n_new", N_NEW)
@pytest.mark.parametrize("scale", [1.0, 1e-20, 1e-37, 1e-44])
def test_rows_of_zeros(amd, dev, act, dtype, n_new, scale):
    """Every key a row sees weighs the same, and none that it does not see, whatever the
    scale; rows beside them that are not zero stay right."""
    n, d, T = 100, 64, ora.TYPES[act]
    q = normal(11, n_new, 2, d)
    q[:, 0] = 0.0
    seqs = [(normal(12, n, 1, d).to(T), normal(13, n, 1, d).to(T))]
    got = bounds.check_step(amd, dev, act, dtype, 2, seqs, q.to(T), [n_new], scale)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("n_new", N_NEW)
def test_keys_at_minus_infinity_weigh_nothing(amd, dev, act, dtype, n_new):
    """An infinite element of a key that takes a row's score to -inf: the row is that of
    the other keys. Queries of few bits, whose rest is 0; one of any; a tiny element
    beside a large one. The other KV head's rows, which see none, are untouched."""
    n, d, T = 200, 64, ora.TYPES[act]
    q = normal(21, n_new, 4, d)
    q[:, 0] = q[:, 0].half().float().mul(4).round().div(4)
    q[:, :2, 5] = q[:, :2, 5].abs() + 0.25
    q[:, :2, 9] = -q[:, :2, 9].abs() - 0.25
    if act != "float16":                                   # (it would be 0 there, which times infinity is NaN)
        q[0, 0, 9] = -2.0 ** -60                           # beside elements of about 1
    q = q.to(T)
    k, v = normal(22, n, 2, d).to(T), normal(23, n, 2, d).to(T)
    bad = [0, 40, n - n_new]
    k[bad, 0, 5] = -math.inf
    k[[77], 0, 9] = math.inf
    got = bounds.step(amd, dev, act, dtype, 4, [(k, v)], q, [n_new], 0.125)
    left = [i for i in range(n) if i not in bad + [77]]
    kc, vc = (x.to(ora.TYPES[dtype]).double().numpy() for x in (k, v))
    sees = n - n_new + 1 + np.arange(n_new)
    want, tol = bounds.attend(q[:, :2].double().numpy(), kc[left][:, :1], vc[left][:, :1], [sum(x < s for x in left) for s in sees],
                              0.125, act, dtype)
    ora.check(got[:, :2], want, tol)
    want, tol = bounds.attend(q[:, 2:].double().numpy(), kc[:, 1:], vc[:, 1:], sees, 0.125, act, dtype)
    ora.check(got[:, 2:], want, tol)
    # at +inf the row is not finite, from the key's position on
    k[bad, 0, 5] = math.inf
    got = bounds.step(amd, dev, act, dtype, 4, [(k, v)], q, [n_new], 0.125)
    assert not torch.isfinite(got[:, :2].float()).any() and torch.isfinite(got[:, 2:].float()).all()
