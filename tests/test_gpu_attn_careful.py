"""Keys and values that are not finite among many new positions over a paged cache
(sllm_gfx950_attn.h) on the GPU: workgroups of 16, 64 and 128 rows, their keys in
parts, with and without a shared prefix. Rows that do not see them keep every bit.
And such steps without them, against 64 bits (attn_bounds.py)."""
import math

import pytest
import torch

import attn_bounds as bounds
import attn_oracle as ora

pytestmark = pytest.mark.gpu

PAIRS = [("float32", "float32"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")]


def normal(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("d", [64, 128, 72])
@pytest.mark.parametrize("n_new", [3, 25, 70])
@pytest.mark.parametrize("prefix", [0, 400])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see(amd, dev, act, dtype, d, n_new, prefix, bad):
    heads, kv, n, T = 4, 2, 700 + n_new, ora.TYPES[act]
    shared = [normal(1 + i, prefix, kv, d).to(T) for i in range(2)]
    seqs = [tuple(torch.cat([s, normal(10 * j + i + 3, n - prefix, kv, d).to(T)]) for i, s in enumerate(shared)) for j in range(3)]
    q = normal(50, 3 * n_new, heads, d).to(T)

    def run():
        return bounds.step(amd, dev, act, dtype, heads, seqs, q, [n_new] * 3, d ** -0.5, prefix=prefix).view(3, n_new, heads, d)

    clean = run()
    assert torch.isfinite(clean.float()).all()
    k, v = seqs[1]
    at = n_new // 2                                     # of the new positions
    k[700 + at, 0, 3] = bad
    v[700 + at - 1, 1, 5] = bad
    v[700 + n_new - 1, :, 7] = bad
    got = run()
    may = torch.zeros_like(clean, dtype=torch.bool)     # values that may differ
    may[1, at:, :2] = True
    may[1, at - 1:, 2:, 5] = True
    may[1, n_new - 1, :, 7] = True
    assert torch.equal(got[~may], clean[~may])
    assert not torch.isfinite(got[1, at - 1:, 2:, 5].float()).any() and not torch.isfinite(got[1, n_new - 1, :, 7].float()).any()
    if math.isnan(bad):
        assert torch.isnan(got[1, at:, :2].float()).all()


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 128), (6, 2, 72), (5, 5, 96), (8, 1, 64)])
@pytest.mark.parametrize("n_new,prefix", [([3, 25, 70], 0), ([90, 1, 200], 400), ([1, 1, 150], 0)])
def test_many_new_positions(amd, dev, act, dtype, heads, kv, d, n_new, prefix):
    """Chunks of prompts and single positions in one step, against 64 bits."""
    T = ora.TYPES[act]
    shared = [normal(1 + i, prefix, kv, d).to(T) for i in range(2)]
    seqs = [tuple(torch.cat([s, normal(10 * j + i + 3, 300 + 77 * j + n, kv, d).to(T)]) for i, s in enumerate(shared))
            for j, n in enumerate(n_new)]
    q = normal(50, sum(n_new), heads, d).to(T)
    bounds.check_step(amd, dev, act, dtype, heads, seqs, q, n_new, d ** -0.5, page=32, prefix=prefix)


@pytest.mark.parametrize("act,dtype", PAIRS)
@pytest.mark.parametrize("n_new", [1, 25, 70])
def test_a_value_in_a_shared_prefix(amd, dev, act, dtype, n_new):
    """What all rows see reaches all of them in its dimension, and nothing else."""
    heads, kv, d, n, T = 4, 2, 64, 500 + n_new, ora.TYPES[act]
    shared = [normal(1 + i, 320, kv, d).to(T) for i in range(2)]
    seqs = [tuple(torch.cat([s, normal(10 * j + i + 3, n - 320, kv, d).to(T)]) for i, s in enumerate(shared)) for j in range(3)]
    q = normal(50, 3 * n_new, heads, d).to(T)
    clean = bounds.step(amd, dev, act, dtype, heads, seqs, q, [n_new] * 3, 0.125, prefix=320)
    seqs[0][1][150, 1, 9] = math.inf                    # (the prefix is the first sequence's)
    got = bounds.step(amd, dev, act, dtype, heads, seqs, q, [n_new] * 3, 0.125, prefix=320)
    may = torch.zeros_like(clean, dtype=torch.bool)
    may[:, 2:, 9] = True
    assert torch.equal(got[~may], clean[~may]) and not torch.isfinite(got[may].float()).any()
