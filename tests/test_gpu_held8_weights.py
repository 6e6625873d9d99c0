"""What weights of attention over a cache of 8 bits keep (sllm_gfx950_attn.h): 16 bits of
rows of f16 and bf16 where up to 64 rows share a workgroup, so that a result is off by its own
rounding and hardly more."""
import numpy as np
import pytest
import torch

import attn_oracle as ora
import held8_oracle as h8
import held8_rows as rows8
from test_gpu_held8 import step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", h8.HELD)
@pytest.mark.parametrize("act", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,kv,d,lens,n_new,prefix", [
    (20, 5, 128, [1000, 257, 33], [1, 1, 1], 0),                 # few rows: a sequence's own
    (8, 2, 64, [700, 300], [1, 3], 0),
    (6, 3, 80, [2000], [2], 0),
    (8, 2, 64, [300, 410], [16, 9], 0),                          # up to 64 rows: several positions
    (20, 5, 128, [500], [12], 0),
    (4, 2, 96, [350], [70], 0),                                  # (140 rows, too little work for more a workgroup)
    (8, 2, 128, [1, 9, 30, 64, 2, 77], [1, 1, 1, 2, 1, 1], 700)])       # a shared prefix
def test_weights_keep_16_bits(amd, dev, act, dtype, heads, kv, d, lens, n_new, prefix):
    def edit(s, k, v):                                           # keys that differ little: many weights count
        k[:] = (k.float() / 4).to(k.dtype)

    got, held = step(amd, dev, act, dtype, heads, kv, d, 16, lens, n_new, prefix=prefix, seed=51, edit=edit, check=False)
    g = torch.Generator()
    g.manual_seed(51 + 7)
    q = torch.randn(sum(n_new), heads, d, generator=g).to(ora.TYPES[act])
    at = 0
    for (k, v), m in zip(held, n_new):
        sees = len(k) - m + 1 + np.arange(m)
        want, tol = rows8.attend(q[at:at + m].double().numpy(), k, v, sees, d ** -0.5, act, 2.0 ** -16)
        ora.check(got[at:at + m], want, tol, f"{m} of {len(k)}")
        at += m
