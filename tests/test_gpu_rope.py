"""Rotary positions (sllm_gfx950_attn.h) on the GPU, against 64 bits: rows by themselves and
on their way into a cache; and a step of a layer over a cache of 8 bits, captured and replayed."""
import numpy as np
import pytest
import torch

import attn_oracle as ora
import held8_oracle as h8

pytestmark = pytest.mark.gpu

SCALINGS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
            dict(scaling="parts", factor=16.0, original=8192.0, slow=1.0, fast=32.0, magnitude=1.25)]


def normal(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


def frequencies(n_rot, base=10000.0, magnitude=1.0, **how):
    return h8.frequencies(n_rot, base, **how)


def near(got, want, tol, act, what):
    """To the tolerance of the arithmetic and half a step of the rows' type."""
    least = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}[act]
    ora.check(got, want, tol + h8.HALF[act] * (np.abs(want) + tol) + least, what)


def rows(amd, dev, rope, act, pos, q, k=None, back=False, strides=(0, 0, 0, 0), in_place=False):
    """Rope.rows on CPU tensors; the outputs with what their strides leave between rows."""
    def put(x, stride):
        n, w = x.shape[0], x[0].numel()
        y = torch.full((n, stride or w), 9.0, dtype=x.dtype)
        y[:, :w] = x.reshape(n, w)
        return dev.put(ora.bits(y))

    n = q.shape[0]
    bp = dev.put(np.asarray(pos, np.int32))
    tensors = [q] if k is None else [q, k]
    ins = [put(x, strides[2 * i]) for i, x in enumerate(tensors)]
    outs = ins if in_place else [put(torch.full_like(x, 7.0), strides[2 * i + 1]) for i, x in enumerate(tensors)]
    rope.rows(act, bp.ptr, n, ins[0].ptr, q.shape[1], outs[0].ptr, *((ins[1].ptr, k.shape[1], outs[1].ptr) if k is not None else ()),
              strides=strides, back=back)
    dev.sync()
    got = []
    for i, x in enumerate(tensors):
        w, s = x[0].numel(), strides[2 * i + (not in_place)] or x[0].numel()
        y = ora.from_bits(outs[i].download(ora.store_type(act), n * s), act).view(n, s)
        assert (y[:, w:] == 9).all()
        got.append(y[:, :w].reshape(x.shape))
    for b in {id(b): b for b in ins + outs + [bp]}.values():
        b.free()
    return got


@pytest.mark.parametrize("act", list(ora.TYPES))
@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("how", SCALINGS, ids=lambda h: h.get("scaling", "none"))
@pytest.mark.parametrize("heads,kv,d,n_rot", [(20, 5, 128, 128), (4, 2, 64, 32), (3, 1, 80, 80), (8, 8, 96, 48), (1, 1, 8, 8), (5, 3, 120, 24)])
def test_rows(amd, dev, act, layout, how, heads, kv, d, n_rot):
    T, n = ora.TYPES[act], 37
    r = np.random.default_rng(d + n_rot)
    pos = np.concatenate([[0, 1, 2, 2047, 131071, (1 << 20) + 7, -1, -4096], r.integers(0, 1 << 17, n - 8)])
    q, k = normal(1, n, heads, d).to(T), normal(2, n, kv, d).to(T)
    rope = amd.Rope(dev, d, n_rot, layout=layout, **how)
    f, mag = frequencies(n_rot, **how), how.get("magnitude", 1.0)
    for back in (False, True):
        got = rows(amd, dev, rope, act, pos, q, k, back=back)
        for x, y in zip((q, k), got):
            want, tol = h8.turn(x.double().numpy(), pos, f, layout, mag, back)
            near(y, want, tol, act, f"back {back}")
            assert torch.equal(y[..., n_rot:], x[..., n_rot:])
    only, = rows(amd, dev, rope, act, pos, q)
    again, _ = rows(amd, dev, rope, act, pos, q, k)
    place = rows(amd, dev, rope, act, pos, q, k, in_place=True)
    assert torch.equal(only, again) and torch.equal(place[0], again)
    rope.close()


@pytest.mark.parametrize("act", list(ora.TYPES))
@pytest.mark.parametrize("n", [0, 1, 2, 3, 129, 5000])
def test_numbers_of_rows(amd, dev, act, n):
    T = ora.TYPES[act]
    pos = np.arange(n) * 3
    q, k = normal(3, n, 6, 64).to(T), normal(4, n, 2, 64).to(T)
    rope = amd.Rope(dev, 64, base=500000.0)
    if n == 0:
        rope.rows(act, 0, 0, 0, 6, 0)
    else:
        for x, y in zip((q, k), rows(amd, dev, rope, act, pos, q, k, strides=(400, 392, 136, 160))):
            near(y, *h8.turn(x.double().numpy(), pos, frequencies(64, 500000.0)), act, n)
    rope.close()


def test_frequencies_of_the_users_own_at_the_farthest_positions(amd, dev):
    """Angles at every position of 32 bits, a frequency of a turn and more among them."""
    f = [1.0, 3.0, 7.0, 2 * np.pi, -0.5, 1e-6, 1e-12, 0.0]
    pos = np.array([0, 1, 2 ** 31 - 1, -2 ** 31, 2 ** 30 + 12345, 2 ** 28, 999999937], np.int64)
    q = normal(5, len(pos), 3, 16)
    for layout in ("half", "pairs"):
        rope = amd.Rope(dev, 16, layout=layout, freq=f)
        got, = rows(amd, dev, rope, "float32", pos, q)
        # the angle in units of a turn, exactly: the frequency's float64 value times the position, in integers
        from fractions import Fraction
        turn = Fraction("6.28318530717958647692528676655900576839433879875021164194988918461563281257241799725606965")
        angle = np.array([[float((Fraction(float(x)) * int(p) / turn) % 1) for x in f] for p in pos]) * 2 * np.pi
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        x = q.double().numpy()
        a, b = (slice(0, 8), slice(8, 16)) if layout == "half" else (slice(0, 16, 2), slice(1, 16, 2))
        want, tol = x.copy(), np.zeros_like(x)
        want[..., a], want[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        tol[..., a] = tol[..., b] = 6 * 2.0 ** -24 * (np.abs(x[..., a]) + np.abs(x[..., b]))
        near(got, want, tol, "float32", layout)
        rope.close()


@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_back_is_the_gradient(amd, dev, layout):
    """Of sum(g * turned(x)): by the transposed formula (back, above) and by differences. The
    call is linear, so a difference over a whole step has no error but rounding: 2 n roundings of
    sums of up to sum |g y|."""
    n, heads, d, rot = 5, 2, 64, 48
    pos = np.array([0, 3, 1000, 77777, 5])
    rope = amd.Rope(dev, d, rot, layout=layout, magnitude=1.5)
    x, g, step = (normal(6 + i, n, heads, d) for i in range(3))
    y0, = rows(amd, dev, rope, "float32", pos, x)
    y1, = rows(amd, dev, rope, "float32", pos, x + step)
    grad, = rows(amd, dev, rope, "float32", pos, g, back=True)
    moved = ((x + step).double() - x.double())
    want = (g.double() * (y1.double() - y0.double())).sum()
    got = (grad.double() * moved).sum()
    size = (g.double().abs() * (y1.abs() + y0.abs()).double()).sum() + (grad.abs().double() * moved.abs()).sum()
    assert abs(got - want) <= 24 * 2.0 ** -24 * size
    rope.close()


@pytest.mark.parametrize("act,dtype", [("float32", "float32"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")] +
                         [(a, t) for a in ora.TYPES for t in h8.HELD])
@pytest.mark.parametrize("layout,d,rot", [("half", 128, 128), ("pairs", 64, 32), ("half", 80, 48)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_on_their_way_into_a_cache(amd, dev, act, dtype, layout, d, rot, in_place):
    """Queries turned, turned keys and values held: at their sequences' own positions."""
    T, heads, kv, page = ora.TYPES[act], 6, 2, 16
    c = amd.PagedCache(dev, 2, kv, d, page, 40, dtype)
    seqs, have, n_new = [c.new() for _ in range(4)], [0, 20, 15, 100], [3, 1, 40, 2]
    c.batch(seqs, have, heads, act).close()
    b = c.batch(seqs, n_new, heads, act)
    n = sum(n_new)
    q, k, v = (normal(10 + i, n, h, d).to(T) for i, h in enumerate((heads, kv, kv)))
    bufs = [dev.put(ora.bits(x)) for x in (q, k, v)]
    qo = bufs[0] if in_place else dev.alloc(bufs[0].nbytes)
    rope = amd.Rope(dev, d, rot, layout=layout, magnitude=0.75)
    b.rope_store(1, rope, bufs[0].ptr, qo.ptr, bufs[1].ptr, bufs[2].ptr)
    total = b.positions
    out = [dev.alloc(total * kv * d * q.element_size()) for _ in range(2)]
    b.read(1, out[0].ptr, out[1].ptr)
    dev.sync()
    pos = np.concatenate([h + np.arange(m) for h, m in zip(have, n_new)])
    new = np.concatenate([sum(have[:i + 1]) + sum(n_new[:i]) + np.arange(m) for i, m in enumerate(n_new)])
    f = frequencies(rot)
    near(ora.from_bits(qo.download(ora.store_type(act), q.numel()), act).view(q.shape), *h8.turn(q.double().numpy(), pos, f, layout, 0.75), act, "q")
    gk, gv = (ora.from_bits(o.download(ora.store_type(act), total * kv * d), act).view(total, kv, d)[torch.from_numpy(new)] for o in out)
    want, tol = h8.turn(k.double().numpy(), pos, f, layout, 0.75)
    if dtype in h8.HELD:
        # Half a step of the codes, whichever neighbour of a border a value or a row's largest
        # falls to. int8: 2^e is less than twice the largest over 127. e4m3: 2^-3 of the value, or where
        # it is subnormal 2^-9 2^e, 2^e less than twice the largest over 448.
        top = np.abs(want).max(-1, keepdims=True)
        held = h8.held(want, dtype)
        grid = top * 2 / 127 if dtype == "int8" else np.abs(want) * 2.0 ** -3 + top * 2.0 ** -8 / 448
        off = np.abs(gk.double().numpy() - want)
        assert (off <= grid / 2 * (1 + 2.0 ** -20) + tol + h8.HALF[act] * np.abs(want) + 2.0 ** -24).all()
        share = (np.abs(gk.double().numpy() - torch.from_numpy(held).to(T).double().numpy()) > tol).mean()
        assert share <= 1e-3                       # (a border within 2^-21 of a value or a largest: rare)
        assert torch.equal(gv, torch.from_numpy(h8.held(v.double().numpy(), dtype)).to(T))
    else:
        near(gk, want, tol + (0 if dtype == act else 2.0 ** -11 * np.abs(want) + 2.0 ** -25), act, "k")
        assert torch.equal(gv, v.to(ora.TYPES[dtype]).to(T))
    b.close()
    c.close()
    rope.close()
    for x in bufs + out + ([] if in_place else [qo]):
        x.free()


@pytest.mark.parametrize("dtype", h8.HELD)
def test_a_step_of_beams(amd, dev, dtype):
    """What a step of beam search calls, twice: queries, keys and values out of one
    projection's rows, turned and held; attention; the beams reordered. Eager, and captured and
    replayed with eager work between."""
    torch.cuda.init()
    stream = torch.cuda.ExternalStream(amd.lib().sllm_gfx950_stream())
    act, heads, kv, d, page, beams = "bfloat16", 8, 2, 64, 16, 4
    c = amd.PagedCache(dev, 1, kv, d, page, 60, dtype)
    rope = amd.Rope(dev, d, base=500000.0)
    width, f = (heads + 2 * kv) * d, frequencies(d, 500000.0)
    base = c.new()

    def step(ids, n_new, seed, graph=False):
        b = c.batch(ids, n_new, heads, act)
        n = b.rows
        qkv = normal(seed, n, heads + 2 * kv, d).bfloat16()
        bx, out, turned = dev.put(ora.bits(qkv)), dev.alloc(max(n, 1) * heads * d * 2), dev.alloc(max(n, 1) * heads * d * 2)
        q, k, v = bx.ptr, bx.ptr + heads * d * 2, bx.ptr + (heads + kv) * d * 2

        def call():
            b.rope_store(0, rope, q, turned.ptr, k, v, q_stride=width, k_stride=width, v_stride=width)
            b.attend(0, turned.ptr, out.ptr, d ** -0.5)

        call()
        dev.sync()
        got = out.download(np.int16, n * heads * d)
        if graph:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
                call()
            for turn in range(3):
                out.upload(np.zeros(got.size, np.int16))
                turned.upload(np.zeros(got.size, np.int16))
                with torch.cuda.stream(stream):
                    g.replay()
                dev.sync()
                assert np.array_equal(out.download(np.int16, got.size), got), turn
                call()
                dev.sync()
                assert np.array_equal(out.download(np.int16, got.size), got), turn
        tq = ora.from_bits(turned.download(np.int16, got.size), act).view(n, heads, d)
        total = b.positions
        back = [dev.alloc(total * kv * d * 4) for _ in range(2)]
        whole = c.batch(ids, [0] * len(ids), heads, "float32")
        whole.read(0, back[0].ptr, back[1].ptr)
        dev.sync()
        held = [x.download(np.float32, total * kv * d).reshape(total, kv, d).astype(np.float64) for x in back]
        rows, at, row = ora.from_bits(got, act).view(n, heads, d), 0, 0
        for s, m in zip(ids, n_new):
            size = c.length(s)
            want, tol = h8.attend(tq[row:row + m].double().numpy(), *(x[at:at + size] for x in held), size - m + 1 + np.arange(m), d ** -0.5, act)
            ora.check(rows[row:row + m], want, tol, f"sequence {s}")
            at, row = at + size, row + m
        whole.close()
        b.close()
        for x in [bx, out, turned] + back:
            x.free()
        return held

    step([base], [37], 1)
    ids = [base] + c.fork(base, 37, beams - 1)
    step(ids, [1] * beams, 2, graph=True)
    before = {s: step([s], [0], 3) for s in ids}
    c.reorder(ids, [2, 2, 0, 2])
    for s, p in zip(ids, [2, 2, 0, 2]):
        for x, y in zip(step([s], [0], 4), before[ids[p]]):
            assert np.array_equal(x, y)
    step(ids, [1] * beams, 5, graph=True)
    c.close()
    rope.close()
