"""Attention in 64 bits with the error of each step of the kernels' arithmetic
(sllm_gfx950_attn.h) bounded for itself: closer than attn_oracle.py where weights,
queries or values lie many powers of two apart. And whole steps over a paged cache
and prompts of given rows, for the tests that want such rows."""
import numpy as np
import torch

import attn_oracle as ora

HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def attend(q, k, v, sees, scale, act, cache):
    """Rows q [rows, heads, d] over k, v [keys, kv, d] (float64), row i over the
    first sees[i] keys: (out, tolerance), both [rows, heads, d].

    u: half a step, 2^-24 (f32), 2^-11 (f16), 2^-8 (bf16). For one row, Q its
    query's largest magnitude, s the scores in natural units, p = exp(s - max):

    * f32 queries over f16 keys are sums of two f16 values of a row scaled to
      2^14 <= Q < 2^15: the second is off by half a step of its own, which is 2^-22 of
      the element or, where it is subnormal, 2^-25 of a row of at least 2^14:
      max(2^-22 |q_i|, 2^-39 Q).
    * a score's sum of products: d roundings of partial sums of at most sum |q k| and
      4 of the powers of two and c (2 d with two products).
    * the exponent t = s log2(e): c, its product and the maximum's subtraction, 2^-24
      |t| each, t at most T = 2 max |s| log2(e); the maximum moves by 8 or more at a
      time, so at most T / 8 + 1 times, each an exponential; an exponential is
      off by 2^-23. e: all of it, relative to p.
    * p as the products take it: u of the cache's type, 2^-22 as two f16 values. f16
      weights are held 2^7 up: the largest is at least 2^7 and half the smallest
      step 2^-25, so 2^-32 of the largest is lost of any.
    * these enter numerator and denominator, |v| and |out|; so do the roundings of
      sums of n terms and of parts, (n + 8) 2^-24; the division's, and the result's u."""
    rows, heads, d = q.shape
    keys, kv = k.shape[:2]
    split = act == "float32" and cache == "float16"
    up = 0.0 if cache == "float32" else 2.0 ** -22 if split else HALF[cache]
    sub = 2.0 ** -32 if cache == "float16" else 0.0
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
            dq = np.maximum(2.0 ** -22 * np.abs(x), 2.0 ** -39 * np.abs(x).max()) if split else 0 * x
            b = scale * (np.abs(kn) @ ((d * (1 + split) + 4) * 2.0 ** -24 * np.abs(x) + dq))
            t = 2 * np.abs(s).max() / np.log(2)
            e = b + 4 * 2.0 ** -24 * t + (t / 8 + 3) * 2.0 ** -23
            lost = p * (e + up + (n + 8) * 2.0 ** -24) + sub * p.max()
            out[i, h] = o
            tol[i, h] = (lost @ av + lost.sum() * np.abs(o)) / p.sum() + (HALF[act] + 2.0 ** -23) * np.abs(o) + \
                (2.0 ** -25 if act == "float16" else 1e-37)
    return out, tol


def step(amd, dev, act, dtype, heads, seqs, q, n_new, scale, page=16, prefix=0):
    """One step over sequences of the given keys and values, (k, v) of
    [positions, kv, d] each in the rows' type, the last n_new[i] of them new; the first
    `prefix` positions of all are those of the first, shared. Rows out, sequence by sequence."""
    kv, d = seqs[0][0].shape[1:]
    pages = -(-prefix // page) + sum(-(-(len(k) - prefix) // page) + 1 for k, _ in seqs)
    c = amd.PagedCache(dev, 1, kv, d, page, pages, dtype)

    def store(ids, rows, b):
        k, v = (torch.cat([x[i] for x in rows]).contiguous() for i in (0, 1))
        bufs = [dev.put(ora.bits(x)) for x in (k, v)]
        b.store(0, *(x.ptr for x in bufs))
        dev.sync()
        for x in bufs:
            x.free()

    base = c.new()
    if prefix:
        b = c.batch([base], [prefix], heads, act)
        store([base], [tuple(x[:prefix] for x in seqs[0])], b)
        b.close()
    ids = c.fork(base, prefix, len(seqs))
    old = [len(k) - prefix - n for (k, _), n in zip(seqs, n_new)]
    if sum(old):
        b = c.batch(ids, old, heads, act)
        store(ids, [tuple(x[prefix:prefix + n] for x in s) for s, n in zip(seqs, old)], b)
        b.close()
    b = c.batch(ids, n_new, heads, act)
    store(ids, [tuple(x[len(x) - n:] for x in s) for s, n in zip(seqs, n_new)], b)
    bq, bo = dev.put(ora.bits(q)), dev.alloc(q.numel() * q.element_size())
    b.attend(0, bq.ptr, bo.ptr, scale)
    dev.sync()
    out = ora.from_bits(bo.download(ora.store_type(act), q.numel()), act).view(-1, heads, d)
    b.close()
    c.close()
    bq.free(), bo.free()
    return out


def check_step(amd, dev, act, dtype, heads, seqs, q, n_new, scale, **how):
    """step() against attend()."""
    got = step(amd, dev, act, dtype, heads, seqs, q, n_new, scale, **how)
    T, at = ora.TYPES[dtype], 0
    for i, ((k, v), n) in enumerate(zip(seqs, n_new)):
        kc, vc = (x.to(T).double().numpy() for x in (k, v))
        want, tol = attend(q[at:at + n].double().numpy(), kc, vc, len(kc) - n + 1 + np.arange(n), scale, act, dtype)
        ora.check(got[at:at + n], want, tol, f"sequence {i}")
        at += n
    return got


def prompt(amd, dev, dtype, q, k, v, q_len, k_len, scale):
    """A prompt plan on packed rows."""
    heads, kv, d = q.shape[1], k.shape[1], q.shape[2]
    bufs = [dev.put(ora.bits(x)) for x in (q, k, v)]
    out = dev.alloc(q.numel() * q.element_size())
    plan = amd.PromptAttention(dev, dtype, heads, kv, d, q_len, k_len)
    plan.run(*(b.ptr for b in bufs), out.ptr, scale)
    dev.sync()
    got = ora.from_bits(out.download(ora.store_type(dtype), q.numel()), dtype).view(q.shape)
    plan.close()
    for b in bufs + [out]:
        b.free()
    return got
