"""Sine and cosine of rotary positions (sllm_gfx950_attn.h) on the GPU: rows of (1, 0) turn
into them."""
import numpy as np
import pytest
import torch

import held8_oracle as h8
from test_gpu_rope import rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("base", [1.5, 10000.0, 5e5])
def test_sine_and_cosine(amd, dev, layout, base):
    """2^-22, and 2 pi 2^-30 of the angle, whatever the position. (What is left of an angle, at
    most pi / 4, is rounded to f32 and multiplied by a constant: 2 times 2^-24 of it and the constant's
    own 2^-24, 2.4 times 2^-24; the series' operations leave 1.5 times 2^-24 more, its rest 2^-32.)"""
    d, n = 128, 4000
    r = np.random.default_rng(1)
    pos = np.concatenate([np.arange(64), -np.arange(64), [2 ** 31 - 1, -2 ** 31], r.integers(-2 ** 31, 2 ** 31, n),
                          (2.0 ** r.uniform(0, 31, n)).astype(np.int64)]).astype(np.int32)
    rope = amd.Rope(dev, d, base=base, layout=layout)
    q = torch.zeros(len(pos), 1, d)
    a, b = (slice(0, d // 2), slice(d // 2, d)) if layout == "half" else (slice(0, d, 2), slice(1, d, 2))
    q[..., a] = 1
    got = rows(amd, dev, rope, "float32", pos, q)[0][:, 0].double().numpy()
    rope.close()
    angle = pos.astype(np.longdouble)[:, None] * h8.frequencies(d, base)
    tol = 2.0 ** -22 + 2 * np.pi * 2.0 ** -30
    assert np.abs(got[:, a] - np.cos(angle).astype(np.float64)).max() <= tol
    assert np.abs(got[:, b] - np.sin(angle).astype(np.float64)).max() <= tol
