"""The softmax weights of attention on the GPU, as the products with the values
take them (sllm_gfx950_attn.h): those far below a row's largest keep their share,
and what they are divided by is the sum of just these. Tolerances: attn_bounds.py."""
import numpy as np
import pytest
import torch

import attn_bounds as bounds
import attn_oracle as ora

pytestmark = pytest.mark.gpu

PAIRS = [("float32", "float32"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")]
# new positions of two rows each: 16, 64 and 128 rows a workgroup
N_NEW = [1, 25, 70]


def sinks(n, at, d, T, seed):
    """Keys whose scores, by the first dimension, are 15 to 19 below those at `at`,
    whose values are 0, so that only the others' share is in the result."""
    r = np.random.RandomState(seed)
    k, v = np.zeros((n, 1, d)), r.uniform(32, 96, (n, 1, d))
    k[:, 0, 0] = -r.uniform(15.0, 19.0, n)
    k[at, 0, 0], v[at] = 0.0, 0.0
    return torch.tensor(k).to(T), torch.tensor(v).to(T)


def sink_queries(n, heads, d, T):
    q = torch.zeros(n, heads, d)
    q[:, :, 0] = 4.0
    return q.to(T)


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("n_new", N_NEW)
@pytest.mark.parametrize("where", ["first", "last"])
def test_many_keys_far_below_a_few(amd, dev, act, dtype, n_new, where):
    """Enough sequences and heads that a wave has hundreds of keys in a row; each finds
    one of the large ones, in its first tiles or in its last."""
    n, d, kv, T = 2000, 64, 32, ora.TYPES[act]
    at = [i for i in range(0, n, 32) if (i % 512 < 128) == (where == "first")]
    k, v = sinks(n, at, d, T, 5)
    seq = tuple(x.expand(n, kv, d).contiguous() for x in (k, v))
    q = sink_queries(8 * n_new, 2 * kv, d, T)
    got = bounds.step(amd, dev, act, dtype, 2 * kv, [seq] * 8, q, [n_new] * 8, 0.25, page=64).view(8, n_new, 2 * kv, d)
    assert torch.equal(got, got[:1, :, :1].expand_as(got))
    some = sorted({0, n_new // 2, n_new - 1})
    cached = (x.to(ora.TYPES[dtype]).double().numpy() for x in (k, v))
    want, tol = bounds.attend(q[some][:, :1].double().numpy(), *cached, np.array(some) + n - n_new + 1, 0.25, act, dtype)
    ora.check(got[0, some][:, :1], want, tol)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("n_q", [1, 40, 300])
def test_many_keys_of_a_prompt_far_below_one(amd, dev, dtype, n_q):
    n, d, T = 4000, 128, ora.TYPES[dtype]
    k, v = sinks(n, [0], d, T, 6)
    q = sink_queries(n_q, 2, d, T)
    got = bounds.prompt(amd, dev, dtype, q, k, v, [n_q], [n], 0.25)
    some = sorted({0, n_q // 2, n_q - 1})
    want, tol = bounds.attend(q[some].double().numpy(), k.double().numpy(), v.double().numpy(), np.array(some) + n - n_q + 1, 0.25,
                              dtype, dtype)
    ora.check(got[some], want, tol)


def uneven(n, d, dtype):
    """(keys, scale): with queries of 1 in the first dimension, one key in 16 has the
    largest score, and the others' weights are 0.9 half steps of the type over a half,
    so that all round down."""
    k = torch.zeros(n, 1, d)
    k[:, 0, 0] = -1.0
    k[::16] = 0.0
    return k.to(ora.TYPES[dtype]), float(np.log(2.0) - np.log1p(0.9 * bounds.HALF[dtype]))


def alike(n, d, T):
    v = torch.ones(n, 1, d)
    v[..., 1::2] = -2.0 ** 6
    v[..., 2::3] = 2.0 ** -6
    return v.to(T)


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("n_new", N_NEW)
def test_values_that_are_all_alike(amd, dev, act, dtype, n_new):
    """They come back as they are. Sums of weights and of weights times a power of two
    differ by the roundings of sums alone, (n + 8) 2^-24 each and a division, which
    rounding to 16 bits does not see."""
    n, d, heads, T = 1000, 64, 2, ora.TYPES[act]
    k, scale = uneven(n, d, dtype if dtype != "float32" else "bfloat16")
    v = alike(n, d, T)
    q = torch.zeros(n_new, heads, d)
    q[:, :, 0] = 1.0
    got = bounds.step(amd, dev, act, dtype, heads, [(k.to(T), v)], q.to(T), [n_new], scale, page=64)
    want = v[:1].expand(n_new, heads, d)
    if act == "float32":
        assert ((got - want).abs() <= (2 * (n + 8) + 3) * 2.0 ** -24 * want.abs()).all()
    else:
        assert (2 * (n + 8) + 3) * 2.0 ** -24 < bounds.HALF[act] / 2
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n_q", [1, 40, 300])
def test_values_of_a_prompt_that_are_all_alike(amd, dev, dtype, n_q):
    n, d, T = 1000, 128, ora.TYPES[dtype]
    k, scale = uneven(n, d, dtype)
    v = alike(n, d, T)
    q = torch.zeros(n_q, 2, d, dtype=T)
    q[:, :, 0] = 1.0
    assert torch.equal(bounds.prompt(amd, dev, dtype, q, k, v, [n_q], [n], scale), v[:1].expand(n_q, 2, d))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n_q", [20, 300, 2000])
def test_f32_results_are_divided_with_one_rounding_each(amd, dev, d, n_q):
    """Scores of 0 and values of 1: the sums are whole numbers n, and a prompt's result is n
    times the reciprocal of n, both correctly rounded; a step's, joined from parts or
    not, is n / n."""
    q, k, v = torch.ones(n_q, 2, d), torch.zeros(n_q, 1, d), torch.ones(n_q, 1, d)
    n = np.arange(1, n_q + 1, dtype=np.float32)
    want = torch.from_numpy(n * (np.float32(1) / n))[:, None, None].expand(n_q, 2, d)
    assert torch.equal(bounds.prompt(amd, dev, "float32", q, k, v, [n_q], [n_q], 1.0), want)
    got = bounds.step(amd, dev, "float32", "float32", 2, [(k, v)], q[:1], [1], 1.0, page=64)
    assert ((got == 1) | (got == want[-1:])).all()


def ramp(n, d, T, value):
    """Keys whose scores rise by 2^5 (as weights) over every 500, with large values: the
    running maximum need not move, and a sum of 2^5 times the values would overflow."""
    k = torch.zeros(n, 1, d)
    k[:, 0, 0] = torch.arange(n) % 500 * (5 * np.log(2.0) / 500)
    return k.to(T), torch.full((n, 1, d), value).to(T)


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("n_new", N_NEW)
def test_sums_of_large_values(amd, dev, act, dtype, n_new):
    """2000 values of 2^117 (f16: 2^15) and weights that sum up to 560 of the largest: within
    f32's range where no weight is over 1, and not where they may be 2^5."""
    n, d, kv, T = 2000, 64, 32, ora.TYPES[act]
    value = 2.0 ** (15 if dtype == "float16" else 117)
    k, v = ramp(n, d, T, value)
    seq = tuple(x.expand(n, kv, d).contiguous() for x in (k, v))
    q = sink_queries(8 * n_new, 2 * kv, d, T)
    got = bounds.step(amd, dev, act, dtype, 2 * kv, [seq] * 8, q, [n_new] * 8, 0.25, page=64)
    want = torch.full_like(got, value)
    assert ((got.double() - value).abs() <= (2 * (n + 8) + 3) * 2.0 ** -24 * value).all() if act == "float32" else torch.equal(got, want)


@pytest.mark.parametrize("dtype", list(ora.TYPES))
@pytest.mark.parametrize("n_q", [1, 40, 300])
def test_sums_of_large_values_of_a_prompt(amd, dev, dtype, n_q):
    n, d, T = 2000, 128, ora.TYPES[dtype]
    value = 2.0 ** (15 if dtype == "float16" else 117)
    k, v = ramp(n, d, T, value)
    got = bounds.prompt(amd, dev, dtype, sink_queries(n_q, 2, d, T), k, v, [n_q], [n], 0.25)
    want = torch.full_like(got, value)
    assert ((got.double() - value).abs() <= (2 * (n + 8) + 3) * 2.0 ** -24 * value).all() if dtype == "float32" else torch.equal(got, want)
