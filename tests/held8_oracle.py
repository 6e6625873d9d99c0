"""What a cache of 8 bits holds (sllm_gfx950_attn.h), rotary positions and attention
over such a cache in 64 bits, with the error that the kernels' arithmetic may leave."""
import numpy as np
import torch

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
HELD = ["int8", "float8_e4m3"]
LARGEST = 127 * 2.0 ** 120


def codes_of(x, dtype):
    """Rows x [..., d] (float64) as (codes, scale bytes): the smallest 2^e with room for the
    row's largest magnitude, and the row over it rounded to nearest, ties to even."""
    x = np.asarray(x, np.float64)
    room, low = (127.0, -126) if dtype == "int8" else (448.0, -117)
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(-1)
        bad = ~(top <= LARGEST)
    m, e = np.frexp(np.where(bad | (top == 0), room, top) / room)
    # (a quotient is rounded, so both neighbours of a power of two are tried)
    e = e - 1
    while True:
        short = np.ldexp(room, e) < np.where(bad, 0, top)
        if not short.any():
            break
        e = e + short
    e = np.maximum(np.where(top == 0, low, e), low)
    e = np.where(bad, 0, e)
    y = np.ldexp(np.where(bad[..., None], 0, x), -e[..., None])
    if dtype == "int8":
        codes = np.where(bad[..., None], 0, np.rint(y)).astype(np.int8).view(np.uint8)
    else:
        t = torch.from_numpy(np.ascontiguousarray(y)).to(torch.float32)      # (exact: 24 bits or fewer, or half of 2^-9 and less)
        codes = np.where(bad[..., None], 0x7f, e4m3_of(t.numpy().astype(np.float64)))
    return codes.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def e4m3_values():
    """The value of each of 256 codes: sign, 4 bits of exponent with bias 7, 3 of mantissa; 0x7f and 0xff NaN."""
    c = np.arange(256)
    s, e, m = np.where(c & 128, -1.0, 1.0), c >> 3 & 15, c & 7
    v = s * np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0))
    return np.where((c & 127) == 127, np.nan, v)


def e4m3_of(y):
    """The nearest code of values of at most 448, ties to the even one."""
    v = e4m3_values()[:127]
    a = np.abs(y)
    i = np.clip(np.searchsorted(v, a, side="right") - 1, 0, 125)
    up, down = v[i + 1] - a, a - v[i]
    i = i + ((up < down) | ((up == down) & (i % 2 == 1)))
    return i + np.where(np.signbit(y), 128, 0)


def values_of(codes, scales, dtype):
    """What codes [..., d] (uint8) and scale bytes [...] stand for, in 64 bits."""
    v = codes.view(np.int8).astype(np.float64) if dtype == "int8" else e4m3_values()[codes]
    with np.errstate(invalid="ignore"):
        return np.where(scales[..., None] == 255, np.nan, np.ldexp(v, scales[..., None].astype(int) - 127))


def held(x, dtype):
    """Rows as they are read back, in 64 bits."""
    return values_of(*codes_of(x, dtype), dtype)


def frequencies(n_rot, base, scaling="none", factor=1.0, original=0.0, fast=0.0, slow=0.0, freq=None):
    b = np.longdouble(base)
    if scaling == "ntk":
        b = b * np.longdouble(factor) ** (np.longdouble(n_rot) / (n_rot - 2))
    f = b ** (-2 * np.arange(n_rot // 2, dtype=np.longdouble) / n_rot) if freq is None else np.asarray(freq, np.longdouble)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        keep = np.clip((original * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f


def turn(x, pos, f, layout="half", magnitude=1.0, back=False):
    """(rows, tolerance without the last rounding): x [n, heads, d] float64 turned by pos [n].

    Tolerance of a value a cos - b sin, with u = 2^-24: an angle is off by at most 2^-30 of a
    turn, 2 pi 2^-30 < 2^-27 rad; the argument of the series and its terms leave at most 2 u
    of a sine or cosine absolutely, the magnitude's product u, the two products and the sum
    u each of |a| and |b|: 6 u magnitude (|a| + |b|) in all."""
    n_rot = 2 * len(f)
    angle = np.asarray(pos, np.longdouble)[:, None] * f * (-1 if back else 1)
    c, s = (magnitude * g(angle).astype(np.float64)[:, None] for g in (np.cos, np.sin))
    out, tol = x.copy(), np.zeros_like(x)
    a, b = (slice(0, n_rot // 2), slice(n_rot // 2, n_rot)) if layout == "half" else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    t = 6 * 2.0 ** -24 * magnitude * (np.abs(x[..., a]) + np.abs(x[..., b]))
    tol[..., a], tol[..., b] = t, t
    return out, tol


def attend(q, k, v, sees, scale, act):
    """Rows q [rows, heads, d] over k, v [keys, kv, d] as they are held (float64), row i over
    the first sees[i] keys: (out, tolerance).

    Queries and keys are exact as the products take them (queries of f32 as three bf16
    values: to 2^-24). A score's products and their partial sums: 3 d + 4 roundings of at most
    sum |q k| (three products for f32, fewer else). With t = s log2(e): c, its product
    and the maximum's subtraction 2^-24 |t| each, t at most T = 2 max |s| log2(e); the
    maximum moves at most T / 8 + 1 times, each an exponential; an exponential is off by
    2^-23: e in all, relative to p. p as the products take it: 2^-8 (bf16), 2^-16 (f16: cut
    off behind 8 bits, and the rest rounded to 8), 2^-24 (f32), and the sum that divides them is
    of p or of p so rounded. These enter numerator and denominator; so do sums of n terms, (n + 8)
    2^-24 three times for f32's three products; the division's rounding, and the result's."""
    rows, heads, d = q.shape
    keys, kv = k.shape[:2]
    up = {"float32": 2.0 ** -24, "float16": 2.0 ** -16, "bfloat16": 2.0 ** -8}[act]
    out, tol = np.zeros((rows, heads, d)), np.zeros((rows, heads, d))
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        for i in range(rows):
            n = int(min(max(sees[i], 0), keys))
            if n == 0:
                continue
            x, kn, av = q[i, h], kh[:n], np.abs(vh[:n])
            s = scale * (kn @ x)
            p = np.exp(s - s.max())
            o = p @ vh[:n] / p.sum()
            b = scale * (np.abs(kn) @ np.abs(x)) * ((3 * d + 5) * 2.0 ** -24)
            t = 2 * np.abs(s).max() / np.log(2)
            e = b + 4 * 2.0 ** -24 * t + (t / 8 + 3) * 2.0 ** -23
            lost = p * (e + up + (3 * n + 8) * 2.0 ** -24)
            out[i, h] = o
            tol[i, h] = (lost @ av + lost.sum() * np.abs(o)) / p.sum() + (HALF[act] + 2.0 ** -23) * np.abs(o) + \
                (2.0 ** -25 if act == "float16" else 1e-37)
    return out, tol
