"""Attention over keys and values held in 8 bits in 64 bits, a head's rows at once: as
held8_oracle.attend, for many rows, with the bits that weights are held to by the caller."""
import numpy as np

from held8_oracle import HALF


def attend(q, k, v, sees, scale, act, up):
    """Rows q [rows, heads, d] over k, v [keys, kv, d] as they are held (float64), row i over the
    first sees[i] keys: (out, tolerance).

    The tolerance is held8_oracle.attend's, with `up` what a weight is off by relative to itself
    as the products take it: 2^-8 where it is rounded to bf16 (half a step); 2^-16 as the sum of
    two bf16 values (cut off behind 8 bits it lacks under a step of them, 2^-7 of its power of
    two, and what it lacks is rounded to 8 bits: half of 2^-15 of that power of two); 2^-24 as
    the sum of three."""
    rows, heads, d = q.shape
    keys, kv = k.shape[:2]
    out, tol = np.zeros((rows, heads, d)), np.zeros((rows, heads, d))
    n = np.clip(np.asarray(sees), 0, keys)
    some = n > 0
    seen = np.arange(keys)[None] < n[some, None]
    for h in range(heads if some.any() else 0):
        kh, vh, x = k[:, h // (heads // kv)], v[:, h // (heads // kv)], q[some, h]
        s = scale * (x @ kh.T)
        p = np.where(seen, np.exp(s - np.where(seen, s, -np.inf).max(1, keepdims=True)), 0.0)
        total = p.sum(1, keepdims=True)
        o = p @ vh / total
        b = scale * (np.abs(x) @ np.abs(kh).T) * ((3 * d + 5) * 2.0 ** -24)
        t = 2 * np.where(seen, np.abs(s), 0.0).max(1, keepdims=True) / np.log(2)
        e = b + 4 * 2.0 ** -24 * t + (t / 8 + 3) * 2.0 ** -23
        lost = p * (e + up + (3 * n[some, None] + 8) * 2.0 ** -24)
        out[some, h] = o
        tol[some, h] = (lost @ np.abs(vh) + lost.sum(1, keepdims=True) * np.abs(o)) / total + (HALF[act] + 2.0 ** -23) * np.abs(o) + \
            (2.0 ** -25 if act == "float16" else 1e-37)
    return out, tol
