"""Attention in 64 bits for the tests of sllm_gfx950_attn.h, with the error that
the kernels' arithmetic may leave, and rows as the bits that the device holds."""
import numpy as np
import torch

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def bits(t):
    """A CPU tensor's bytes as a numpy array that can be uploaded."""
    t = t.contiguous()
    return t.numpy() if t.dtype == torch.float32 else t.view(torch.int16).numpy()


def from_bits(a, dtype):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return t if dtype == "float32" else t.view(TYPES[dtype])


def store_type(dtype):
    return np.float32 if dtype == "float32" else np.int16


def attend(q, k, v, sees, scale, act, cache):
    """Rows q [rows, heads, d] over k, v [keys, kv, d] (float64), row i over the
    first sees[i] keys: (out, tolerance), both [rows, heads, d].

    Tolerance. With u the half step of a type (2^-24 f32, 2^-11 f16, 2^-8 bf16),
    t = scale log2(e) s the exponents, A = sum p |v| / sum p:
    a score's sum of d products is off by at most (d + 4) 2^-24 sum |q k| (f32 over
    f16: q held to 2^-22, the 4); c, its product with s, and the subtraction of the
    maximum are off by 2^-24 |t| each, 2^x by 2^-23: e in all, relative to p. It
    enters numerator and denominator: 2 e A. The sums over n keys and over parts:
    (n + 8) 2^-24 A. p is rounded to the cache's type before the products with the
    values: u A, 2^-22 A as the sum of two f16; f16 values under 2^-14 lose up to
    2^-25 absolutely, and the largest p is at least 1: 2^-25 sum |v|. The result is
    rounded to the rows' type: u |out|."""
    rows, heads, d = q.shape
    keys, kv = k.shape[:2]
    half = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
    up = 0.0 if cache == "float32" else 2.0 ** -22 if act == "float32" else half[cache]
    sub = 2.0 ** -25 if cache == "float16" else 0.0
    out, tol = np.zeros((rows, heads, d)), np.zeros((rows, heads, d))
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        for i in range(rows):
            n = int(min(max(sees[i], 0), keys))
            if n == 0:
                continue
            s = scale * (kh[:n] @ q[i, h])
            p = np.exp(s - s.max())
            total = p.sum()
            out[i, h] = p @ vh[:n] / total
            a = p @ np.abs(vh[:n]) / total
            b = scale * (np.abs(kh[:n]) @ np.abs(q[i, h])).max()
            t = np.abs(s).max() * 1.4427 * 2
            e = (d + 4) * 2.0 ** -24 * b + 3 * 2.0 ** -24 * t + 2.0 ** -23
            tol[i, h] = a * (2 * e + (n + 8) * 2.0 ** -24 + up) + sub * np.abs(vh[:n]).sum(0) + half[act] * np.abs(out[i, h]) + 1e-37
    return out, tol


def attend_rows(q, k, v, sees, scale, act, cache):
    """attend() with a head's rows at once, for many of them."""
    rows, heads, d = q.shape
    keys, kv = k.shape[:2]
    half = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
    up = 0.0 if cache == "float32" else 2.0 ** -22 if act == "float32" else half[cache]
    sub = 2.0 ** -25 if cache == "float16" else 0.0
    out, tol = np.zeros((rows, heads, d)), np.zeros((rows, heads, d))
    n = np.clip(np.asarray(sees), 0, keys)
    some = n > 0
    seen = np.arange(keys)[None] < n[some, None]
    for h in range(heads if some.any() else 0):
        kh, vh, qh = k[:, h // (heads // kv)], v[:, h // (heads // kv)], q[some, h]
        s = scale * (qh @ kh.T)
        p = np.where(seen, np.exp(s - np.where(seen, s, -np.inf).max(1, keepdims=True)), 0.0)
        total = p.sum(1, keepdims=True)
        out[some, h] = p @ vh / total
        a = p @ np.abs(vh) / total
        b = (scale * np.where(seen, np.abs(qh) @ np.abs(kh).T, 0.0)).max(1)
        t = np.where(seen, np.abs(s), 0.0).max(1) * 1.4427 * 2
        e = ((d + 4) * 2.0 ** -24 * b + 3 * 2.0 ** -24 * t + 2.0 ** -23)[:, None]
        tol[some, h] = (a * (2 * e + (n[some, None] + 8) * 2.0 ** -24 + up) + sub * (seen.astype(float) @ np.abs(vh)) +
                        half[act] * np.abs(out[some, h]) + 1e-37)
    return out, tol


def check(got, want, tol, what=""):
    got = got.double().numpy().reshape(want.shape)
    bad = ~(np.abs(got - want) <= tol)
    if bad.any():
        i = np.argwhere(bad)[0]
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} values off, first at {tuple(i)}: got {got[tuple(i)]}, "
                             f"want {want[tuple(i)]} +- {tol[tuple(i)]}")
