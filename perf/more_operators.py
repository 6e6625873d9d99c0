"""The operators of a generation step over a cache held in 8 bits, as timed cases.

Kinds of case and their ranges:

rope      rotary positions of a step's or of whole prompts' queries and keys: 1..32768
          rows at positions up to 2^20, f32, f16 and bf16, pairs of neighbours or of
          halves, all or part of a head, plain or scaled frequencies, forward and back
keep      new keys and values written to a cache of 8 bits (rotated on the way or as
          they are) and the sequences read back: 1..64 sequences of 1..2048 new
          positions, int8 and e4m3 under f32, f16 and bf16 rows
attend    one step's attention of a batch over such a cache: 1..64 sequences of up to
          65536 positions, 1..8 new tokens each, with or without a shared prefix
select    the best continuations over beams and vocabulary: 1..32 groups of 1..8 beams,
          vocabularies of 500..128256, 1..32 picks, f32, f16 and bf16 logits
reorder   beams that go on from other beams' positions: 2..32 of 1..2000 positions

In its plain form (own is False) a case is elementary torch operations in 32 bits
(angles and log-probabilities in 64), over sequences padded to the longest.
"""
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_device = []


def _package():
    name = "saphira_llm_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, "saphira-llm_amd", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def device():
    """The library, opened on the first GPU (once per process)."""
    if not _device:
        torch.cuda.init()
        _device.append(_package().Device(0))
    return _device[0]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one user's next token at the 2B shape and the framework's activation type: latency
        {"name": "rope_step_f32", "kind": "rope", "dtype": "float32", "heads": 20, "kv": 5, "dim": 128, "rot": 128,
         "layout": "half", "scaling": "none", "factor": 1.0, "rows": 1, "far": 1101, "back": False, "mix": 1},
        # the prompts of a server's queue, frequencies scaled by parts for long contexts
        {"name": "rope_prompts_bf16", "kind": "rope", "dtype": "bfloat16", "heads": 20, "kv": 5, "dim": 128, "rot": 128,
         "layout": "half", "scaling": "parts", "factor": 16.0, "rows": 18355, "far": 131072, "back": False, "mix": 2},
        # gradients of a part of each head, neighbours paired
        {"name": "rope_back_f16", "kind": "rope", "dtype": "float16", "heads": 32, "kv": 8, "dim": 96, "rot": 48,
         "layout": "pairs", "scaling": "linear", "factor": 4.0, "rows": 4099, "far": 32768, "back": True, "mix": 3},
        # the first tokens of 64 chats, rotated as they are written
        {"name": "keep_step_e4m3", "kind": "keep", "act": "bfloat16", "dtype": "float8_e4m3", "heads": 20, "kv": 5,
         "dim": 128, "page": 64, "n": 64, "longest": 1, "have": 3, "rope": True, "mix": 4},
        # many prompts into the cache and out again for what comes after
        {"name": "keep_prompts_int8", "kind": "keep", "act": "float32", "dtype": "int8", "heads": 20, "kv": 5,
         "dim": 128, "page": 64, "n": 24, "longest": 2048, "have": 50, "rope": False, "mix": 5},
        # one user's next token, f32 activations: latency
        {"name": "attend_one_int8", "kind": "attend", "act": "float32", "dtype": "int8", "heads": 20, "kv": 5,
         "dim": 128, "page": 64, "n": 1, "prefix": 0, "longest": 1101, "new": 1, "mix": 6},
        # a step of 64 chats behind one long system prompt
        {"name": "attend_shared_int8", "kind": "attend", "act": "bfloat16", "dtype": "int8", "heads": 20, "kv": 5,
         "dim": 128, "page": 64, "n": 64, "prefix": 4096, "longest": 1024, "new": 1, "mix": 7},
        # long documents, one token each: what the memory gives
        {"name": "attend_long_e4m3", "kind": "attend", "act": "bfloat16", "dtype": "float8_e4m3", "heads": 20, "kv": 5,
         "dim": 128, "page": 128, "n": 8, "prefix": 0, "longest": 65536, "new": 1, "mix": 8},
        # one request's beams: latency
        {"name": "select_one_f32", "kind": "select", "dtype": "float32", "groups": 1, "beams": 4, "vocab": 128256,
         "picks": 8, "ended": 0, "mix": 9},
        # a server's requests, some beams at their end
        {"name": "select_many_bf16", "kind": "select", "dtype": "bfloat16", "groups": 32, "beams": 8, "vocab": 128256,
         "picks": 16, "ended": 2, "mix": 10},
        # a small vocabulary of an odd size
        {"name": "select_small_f16", "kind": "select", "dtype": "float16", "groups": 16, "beams": 5, "vocab": 1009,
         "picks": 10, "ended": 1, "mix": 11},
        # eight beams go on from four of them, all 30 layers of the 2B shape
        {"name": "reorder_8_bf16", "kind": "reorder", "dtype": "bfloat16", "layers": 30, "kv": 5, "dim": 128, "page": 64,
         "tokens": 1001, "n": 8, "mix": 12},
    ]


# (query heads, KV heads, head dimension): the 2B shape, the repository's small models, and other common splits
HEADS = [(20, 5, 128), (20, 5, 128), (8, 2, 64), (6, 2, 64), (4, 2, 64), (32, 8, 128), (8, 8, 96), (8, 1, 80)]
TYPES = ["float32", "float16", "bfloat16"]
HELD = ["int8", "float8_e4m3"]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "keep", "keep", "attend", "attend", "attend", "select", "select", "reorder"])
    heads, kv, dim = rng.choice(HEADS)
    mix, page = rng.randrange(1 << 20), rng.choice([16, 32, 64, 128])
    act, dtype = rng.choice(TYPES), rng.choice(HELD)
    while kind == "rope":
        c = {"kind": kind, "dtype": act, "heads": heads, "kv": kv, "dim": dim, "rot": rng.choice([dim, dim, dim // 2]),
             "layout": rng.choice(["half", "pairs"]), "scaling": rng.choice(["none", "linear", "ntk", "parts"]),
             "factor": rng.choice([2.0, 4.0, 8.0, 40.0]), "rows": _log(rng, 1, 32768), "far": _log(rng, 16, 1 << 20),
             "back": rng.random() < 0.3, "mix": mix}
        if c["scaling"] == "none":
            c["factor"] = 1.0
        if c["rows"] * (heads + kv) * dim <= 18355 * 25 * 128:
            return c
    while kind == "keep":
        rope = rng.random() < 0.5
        c = {"kind": kind, "act": rng.choice(TYPES[1:]) if rope else act, "dtype": dtype, "heads": heads, "kv": kv, "dim": dim,
             "page": page, "n": _log(rng, 1, 64), "longest": _log(rng, 1, 2048), "have": _log(rng, 1, 1000), "rope": rope, "mix": mix}
        if c["n"] * (c["longest"] + c["have"]) <= 24000 and (c["n"] * c["longest"] * heads * dim <= 1 << 26 or not rope):
            return c
    while kind == "attend":
        c = {"kind": kind, "act": act, "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "page": page,
             "n": _log(rng, 1, 64), "prefix": rng.choice([0, _log(rng, 1, 16000)]), "longest": _log(rng, 1, 65536),
             "new": rng.choice([1, 1, 1, rng.randint(2, 8)]), "mix": mix}
        if c["n"] * (c["prefix"] + c["longest"]) * kv * dim <= 8 * 65536 * 640:
            return c
    while kind == "select":
        c = {"kind": kind, "dtype": act, "groups": _log(rng, 1, 32), "beams": rng.randint(1, 8), "vocab": _log(rng, 500, 128256),
             "picks": rng.randint(1, 32), "ended": rng.randint(0, 2), "mix": mix}
        if c["ended"] < c["beams"]:
            return c
    return {"kind": kind, "dtype": act, "layers": _log(rng, 1, 30), "kv": kv, "dim": dim, "page": page,
            "tokens": _log(rng, 1, 2000), "n": _log(rng, 2, 32), "mix": mix}


def _lengths(n, longest, mix):
    """n lengths of 1..longest, spread over their logarithm, the first the longest."""
    r = random.Random(mix)
    return [longest] + [_log(r, max(1, longest // 16), longest) for _ in range(n - 1)]


class _Tables:
    """The pages of each sequence, handed out in order."""

    def __init__(self, page):
        self.page, self.used, self.seqs, self.lens = page, 0, [], []

    def _take(self):
        self.used += 1
        return self.used - 1

    def new(self):
        self.seqs.append([])
        self.lens.append(0)
        return len(self.seqs) - 1

    def extend(self, s, n):
        self.lens[s] += n
        while len(self.seqs[s]) * self.page < self.lens[s]:
            self.seqs[s].append(self._take())

    def fork(self, s, n):
        """n sequences that share s's whole pages; the copies of the page it ends in."""
        whole, out, copies = self.lens[s] // self.page, [], []
        for _ in range(n):
            f = self.new()
            self.seqs[f], self.lens[f] = self.seqs[s][:whole], self.lens[s]
            if self.lens[s] % self.page:
                copies.append(self._take())
                self.seqs[f].append(copies[-1])
            out.append(f)
        return out, copies


def _attend_plan(case):
    t, own_len = _Tables(case["page"]), _lengths(case["n"], case["longest"], case["mix"])
    copies, base = [], None
    if case["prefix"]:
        base = t.new()
        t.extend(base, case["prefix"])
        seqs, copies = t.fork(base, case["n"])
    else:
        seqs = [t.new() for _ in range(case["n"])]
    for s, n in zip(seqs, own_len):
        t.extend(s, n)
    for s in seqs:
        t.extend(s, case["new"])
    return t, base, seqs, own_len, copies


def _keep_plan(case):
    t, r = _Tables(case["page"]), random.Random(case["mix"] + 1)
    new = _lengths(case["n"], case["longest"], case["mix"])
    have = [r.randint(0, case["have"]) for _ in new]
    seqs = [t.new() for _ in new]
    for s, n in zip(seqs, have):
        t.extend(s, n)
    for s, n in zip(seqs, new):
        t.extend(s, n)
    return t, seqs, have, new


def _reorder_plan(case):
    """Which beam each beam goes on from (about half go on from themselves), its page numbers
    before and after, and the page copies (from, to)."""
    r, n, p = random.Random(case["mix"]), case["n"], case["page"]
    stay = sorted(r.sample(range(n), max(1, n // 2)))
    parents = [i if i in stay else r.choice(stay) for i in range(n)]
    per, whole = -(-case["tokens"] // p), case["tokens"] // p
    before = [list(range(i * per, (i + 1) * per)) for i in range(n)]
    free = sorted(x for i in range(n) if i not in stay for x in before[i])
    after, pairs = [], []
    for i in range(n):
        after.append(before[i] if i in stay else before[parents[i]][:whole])
        if i not in stay and case["tokens"] % p:
            to = free.pop(0)
            pairs.append((before[parents[i]][-1], to))
            after[-1] = after[-1] + [to]
    return parents, before, after, pairs


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _type(name):
    return getattr(torch, name)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(seed, *shapes):
    """Seeded N(0, 1) tensors on the GPU, one for each (type, shape...)."""
    g = _gen(seed)
    return [torch.randn(*s[1:], device="cuda", generator=g).to(_type(s[0])) for s in shapes]


BASE = 500000.0                      # the 2B model's


def _positions(case, seed):
    return torch.randint(0, case["far"], (case["rows"],), dtype=torch.int32, device="cuda", generator=_gen(seed + 1))


def _rope_inputs(case, seed):
    rows, t, d = case["rows"], case["dtype"], case["dim"]
    return _normal(seed, (t, rows, case["heads"], d), (t, rows, case["kv"], d)) + [_positions(case, seed)]


LAYERS, LAYER = 2, 1                 # keep and attend work on one layer of a cache of two


def _pool(case, seed, pages):
    """An 8-bit cache's memory as a user's earlier steps left it: for each page, layer, K or V
    and head, page rows of codes, then a scale byte for each row (2^(byte - 127))."""
    g, p, d = _gen(seed), case["page"], case["dim"]
    shape = (pages, LAYERS, 2, case["kv"], p)
    pool = torch.empty(*shape[:4], p * (d + 1), dtype=torch.uint8, device="cuda")
    codes = torch.randn(*shape, d, device="cuda", generator=g, dtype=torch.bfloat16)
    if case["dtype"] == "int8":
        codes = codes.mul_(32).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        codes = codes.mul_(128).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    pool[..., :p * d] = codes.view(*shape[:4], p * d)
    low = 127 - (5 if case["dtype"] == "int8" else 7)
    pool[..., p * d:] = torch.randint(low - 1, low + 2, shape, dtype=torch.uint8, device="cuda", generator=g)
    return pool


def _attend_inputs(case, seed):
    t, base, seqs, own_len, copies = _attend_plan(case)
    q, = _normal(seed + 7919, (case["act"], case["n"] * case["new"], case["heads"], case["dim"]))
    return t, base, seqs, own_len, copies, _pool(case, seed, t.used), q


def _keep_inputs(case, seed):
    t, seqs, have, new = _keep_plan(case)
    rows, d = sum(new), case["dim"]
    k, v, q = _normal(seed + 7919, *[(case["act"], rows, case["kv"], d)] * 2,
                      (case["act"], rows if case["rope"] else 1, case["heads"], d))
    return t, seqs, have, new, _pool(case, seed, t.used), q, k, v


def _select_inputs(case, seed):
    """Logits as wide as a model's, the beams' scores so far, and the tokens that some beams ended with (-1: none)."""
    g, n, b = _gen(seed), case["groups"], case["beams"]
    logits = torch.randn(n * b, case["vocab"], device="cuda", generator=g).mul_(2.5).to(_type(case["dtype"]))
    scores = -4 - 3 * torch.rand(n, b, device="cuda", generator=g)
    ended = torch.full((n, b), -1, dtype=torch.int32, device="cuda")
    ended[:, :case["ended"]] = 2
    return logits, scores, ended


def _reorder_inputs(case, seed):
    parents, before, after, pairs = _reorder_plan(case)
    pool = torch.empty(case["n"] * len(before[0]), case["layers"], 2, case["kv"], case["page"], case["dim"],
                       dtype=_type(case["dtype"]), device="cuda")
    pool.normal_(generator=_gen(seed))
    return pool, parents, before, after, pairs


def _cache(case, pool, layers):
    return _package().PagedCache(device(), layers, case["kv"], case["dim"], case["page"], pool.shape[0], case["dtype"],
                                 mem=pool.data_ptr())


def _long(v):
    return torch.tensor(v, dtype=torch.long, device="cuda")


def _padded(rows, fill=0):
    """Lists of different lengths as one tensor."""
    longest = max(len(r) for r in rows)
    return _long([list(r) + [fill] * (longest - len(r)) for r in rows])


def _frequencies(case):
    """Angles a position, in 64 bits, and what cos and sin are multiplied by."""
    rot, i = case["rot"], torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
    base = BASE * (case["factor"] ** (rot / (rot - 2)) if case["scaling"] == "ntk" else 1.0)
    f = base ** (-2 * i / rot)
    if case["scaling"] == "linear":
        f = f / case["factor"]
    if case["scaling"] == "parts":
        turns = 8192 * f / (2 * math.pi)                         # over the original length
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)        # fast ones stay, slow ones are divided
        f = f * keep + f / case["factor"] * (1 - keep)
    return f, 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "parts" else 1.0


def _rope(case):
    parts = dict(original=8192, fast=32.0, slow=1.0, magnitude=0.1 * math.log(case["factor"]) + 1.0) if case["scaling"] == "parts" else {}
    return _package().Rope(device(), case["dim"], case["rot"], BASE, layout=case["layout"], scaling=case["scaling"],
                           factor=case["factor"], **parts)


KEEP_ROPE = {"layout": "half", "scaling": "none", "factor": 1.0}


def prepare(case, seed):
    s = {"case": case}
    kind = case["kind"]
    if kind == "rope":
        s["q"], s["k"], s["pos"] = _rope_inputs(case, seed)
        s["qo"], s["ko"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        if own:
            s["rope"] = _rope(case)
            s["ptrs"] = [s[n].data_ptr() for n in ("pos", "q", "qo", "k", "ko")]
        else:
            s["f"], s["mag"] = _frequencies(case)
    elif kind == "keep":
        t, seqs, have, new, s["pool"], s["q"], s["k"], s["v"] = _keep_inputs(case, seed)
        total = sum(t.lens)
        s["qo"] = torch.empty_like(s["q"])
        s["ko"], s["vo"] = (torch.empty(total, case["kv"], case["dim"], dtype=_type(case["act"]), device="cuda") for _ in range(2))
        rot = dict(case, rot=case["dim"], **KEEP_ROPE)
        if own:
            c = s["cache"] = _cache(case, s["pool"], LAYERS)
            ids = [c.new() for _ in seqs]
            c.batch(ids, have, case["heads"], case["act"]).close()
            s["batch"] = c.batch(ids, new, case["heads"], case["act"])
            s["ptrs"] = [s[n].data_ptr() for n in ("q", "qo", "k", "v")]
            s["back"] = [s[n].data_ptr() for n in ("ko", "vo")]
            s["rope"] = _rope(rot)
        else:
            p = case["page"]
            every = [(t.seqs[i][j // p], j % p) for i in seqs for j in range(t.lens[i])]
            s["every"] = _long([a for a, _ in every]), _long([b for _, b in every])
            fresh = [i for i, (a, n) in enumerate((a, n) for a, n in zip(have, new)) for _ in range(n)]
            pos = [j for a, n in zip(have, new) for j in range(a, a + n)]
            s["at"] = _long([t.seqs[seqs[i]][j // p] for i, j in zip(fresh, pos)]), _long([j % p for j in pos])
            s["pos"] = _long(pos)
            s["f"], s["mag"] = _frequencies(rot)
    elif kind == "attend":
        t, base, seqs, own_len, copies, s["pool"], s["q"] = _attend_inputs(case, seed)
        s["out"] = torch.empty_like(s["q"])
        if own:
            torch.cuda.synchronize()
            c = s["cache"] = _cache(case, s["pool"], LAYERS)
            if case["prefix"]:
                b = c.new()
                c.batch([b], [case["prefix"]], case["heads"], case["act"]).close()
                ids = c.fork(b, case["prefix"], case["n"])
            else:
                ids = [c.new() for _ in seqs]
            c.batch(ids, own_len, case["heads"], case["act"]).close()
            s["batch"] = c.batch(ids, [case["new"]] * case["n"], case["heads"], case["act"])
            s["ptrs"] = [s["q"].data_ptr(), s["out"].data_ptr()]
        else:
            _copy_rows(case, s["pool"], t, base, copies)
            s["tables"], s["len"] = _padded([t.seqs[i] for i in seqs]), _long([t.lens[i] for i in seqs])
    elif kind == "select":
        s["logits"], s["scores"], s["ended"] = _select_inputs(case, seed)
        shape = case["groups"], case["picks"]
        s["out"] = torch.empty(shape, device="cuda")
        s["beam"], s["token"] = (torch.empty(shape, dtype=torch.int32, device="cuda") for _ in range(2))
        if own:
            s["plan"] = _package().BeamSelect(device(), case["groups"], case["beams"], case["vocab"], case["picks"], case["dtype"])
            s["ptrs"] = [s[n].data_ptr() for n in ("logits", "scores", "ended", "out", "beam", "token")]
    else:
        s["pool"], s["parents"], before, after, pairs = _reorder_inputs(case, seed)
        if own:
            c = s["cache"] = _cache(case, s["pool"], case["layers"])
            s["ids"] = [c.new() for _ in before]
            c.batch(s["ids"], [case["tokens"]] * case["n"], case["kv"], case["dtype"]).close()
        else:
            s["from"], s["to"] = _long([a for a, _ in pairs]), _long([b for _, b in pairs])
            s["tables"] = np.array(after, np.int32)
    torch.cuda.synchronize()
    return s


def _copy_rows(case, pool, t, base, copies):
    """What a fork copies of the page that its source ends in: rows of codes, and their scales."""
    r, d, p = case["prefix"] % case["page"], case["dim"], case["page"]
    for i in copies:
        for a, b in ((0, r * d), (p * d, p * d + r)):
            pool[i, ..., a:b] = pool[t.seqs[base][-1], ..., a:b]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _turn(x, pos, f, mag, rot, layout, back):
    """Rows [n, heads, d] in 32 bits, the first rot dimensions turned by pos * f (angles in 64)."""
    angle = pos.double()[:, None] * f
    cos, sin = ((g(angle) * mag).float()[:, None] for g in (torch.cos, torch.sin))
    sin = -sin if back else sin
    x = x.float()
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_rope(s):
    c = s["case"]
    s["qo"].copy_(_turn(s["q"], s["pos"], s["f"], s["mag"], c["rot"], c["layout"], c["back"]))
    s["ko"].copy_(_turn(s["k"], s["pos"], s["f"], s["mag"], c["rot"], c["layout"], c["back"]))


def _write(case, pool, at, part, x):
    """Rows x [n, kv, d] in 32 bits to 8 bits: the smallest power of two that leaves room for the row's largest."""
    p, d = case["page"], case["dim"]
    top, low = (127.0, -126) if case["dtype"] == "int8" else (448.0, -117)
    m, e = torch.frexp(x.abs().amax(-1).double() / top)
    e = torch.where(m > 0.5, e, e - 1).clamp_min(low)
    e = torch.where(m == 0, low, e)
    y = torch.ldexp(x.double(), -e[..., None])
    codes = y.round().to(torch.int8) if case["dtype"] == "int8" else y.float().to(torch.float8_e4m3fn)
    page, slot = at
    blocks = pool[:, LAYER, part]                                    # [page, kv, bytes]
    blocks[..., :p * d].unflatten(-1, (p, d))[page, :, slot] = codes.view(torch.uint8)
    blocks[..., p * d:][page, :, slot] = (e + 127).to(torch.uint8)


def _values(case, blocks):
    """The values of blocks [..., page * (d + 1)] of codes and scales, [..., page, d] in 32 bits."""
    p, d = case["page"], case["dim"]
    codes = blocks[..., :p * d].unflatten(-1, (p, d))
    codes = codes.view(torch.int8) if case["dtype"] == "int8" else codes.view(torch.float8_e4m3fn)
    return codes.float() * torch.exp2(blocks[..., p * d:].float() - 127)[..., None]


def _plain_keep(s):
    c, k, v = s["case"], s["k"].float(), s["v"].float()
    if c["rope"]:
        s["qo"].copy_(_turn(s["q"], s["pos"], s["f"], s["mag"], c["dim"], "half", False))
        k = _turn(k, s["pos"], s["f"], s["mag"], c["dim"], "half", False)
    _write(c, s["pool"], s["at"], 0, k)
    _write(c, s["pool"], s["at"], 1, v)
    page, slot = s["every"]
    values = _values(c, s["pool"][:, LAYER])                         # [page, 2, kv, slot, d]
    s["ko"].copy_(values[page, 0, :, slot])
    s["vo"].copy_(values[page, 1, :, slot])


def _plain_attend(s):
    c = s["case"]
    b, new, kv, g, d = c["n"], c["new"], c["kv"], c["heads"] // c["kv"], c["dim"]
    pages = _values(c, s["pool"][:, LAYER][s["tables"]])             # [b, page, 2, kv, slot, d]
    k, v = (pages[:, :, i].transpose(1, 2).reshape(b, kv, -1, d) for i in (0, 1))
    q = s["q"].view(b, new, kv, g, d).float().permute(0, 2, 1, 3, 4).reshape(b, kv, new * g, d)
    j, row = torch.arange(k.shape[2], device="cuda"), torch.arange(new, device="cuda").repeat_interleave(g)
    seen = j <= s["len"][:, None, None] - new + row[:, None]
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(d ** -0.5).masked_fill_(~seen[:, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    s["out"].copy_(out.view(b, kv, new, g, d).transpose(1, 2).reshape(b * new, kv * g, d))


def _plain_select(s):
    c = s["case"]
    n, b, vocab, k = c["groups"], c["beams"], c["vocab"], c["picks"]
    x = s["logits"].double()
    m = x.amax(-1, keepdim=True)
    x = x - (m + (x - m).exp().sum(-1, keepdim=True).log())
    token = torch.arange(vocab, device="cuda")
    end = s["ended"].view(-1, 1)
    x = torch.where(end >= 0, torch.where(token == end, 0.0, -math.inf).double(), x) + s["scores"].double().view(-1, 1)
    best, at = torch.sort(x.view(n, b * vocab), dim=-1, descending=True, stable=True)
    s["out"].copy_(best[:, :k])
    s["beam"].copy_(at[:, :k] // vocab)
    s["token"].copy_(at[:, :k] % vocab)


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if kind == "rope":
        if own:
            pos, q, qo, k, ko = s["ptrs"]
            s["rope"].rows(case["dtype"], pos, case["rows"], q, case["heads"], qo, k, case["kv"], ko, back=case["back"])
        else:
            _plain_rope(s)
        return s["qo"], s["ko"]
    if kind == "keep":
        if own:
            q, qo, k, v = s["ptrs"]
            if case["rope"]:
                s["batch"].rope_store(LAYER, s["rope"], q, qo, k, v)
            else:
                s["batch"].store(LAYER, k, v)
            s["batch"].read(LAYER, *s["back"])
        else:
            _plain_keep(s)
        return (s["ko"], s["vo"], s["qo"]) if case["rope"] else (s["ko"], s["vo"])
    if kind == "attend":
        if own:
            s["batch"].attend(LAYER, *s["ptrs"], case["dim"] ** -0.5)
        else:
            _plain_attend(s)
        return s["out"]
    if kind == "select":
        if own:
            s["plan"].run(*s["ptrs"])
        else:
            _plain_select(s)
        return s["out"], s["beam"], s["token"]
    if own:
        s["cache"].reorder(s["ids"], s["parents"])
        tables = s["cache"].tables(s["ids"])
    else:
        s["pool"][s["to"], :, :, :, :case["tokens"] % case["page"]] = s["pool"][s["from"], :, :, :, :case["tokens"] % case["page"]]
        tables = s["tables"]
    return {"pool": s["pool"], "tables": tables}


# ---------------------------------------------------------------------------
# the work of a pass, and its result in 64 bits
# ---------------------------------------------------------------------------

def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    kind = case["kind"]
    if kind == "select":
        live = case["groups"] * (case["beams"] - case["ended"])
        return {"bytes": float(live * case["vocab"] * _size(case["dtype"]) + case["groups"] * (8 * case["beams"] + 12 * case["picks"])),
                "flops": float(3 * live * case["vocab"])}
    d, kv = case["dim"], case["kv"]
    if kind == "rope":
        values = case["rows"] * (case["heads"] + kv) * d
        return {"bytes": float(2 * values * _size(case["dtype"]) + 4 * case["rows"]), "flops": 3.0 * values * case["rot"] / d}
    if kind == "keep":
        t, _, _, new = _keep_plan(case)
        size, rows, total = _size(case["act"]), sum(new), sum(t.lens)
        held = 2 * kv * (d + 1)                                       # a position of a layer
        return {"bytes": float(rows * (2 * kv * d * size + held) + total * (held + 2 * kv * d * size) +
                               (2 * rows * case["heads"] * d * size if case["rope"] else 0)),
                "flops": float(3 * rows * (case["heads"] + kv) * d if case["rope"] else 0)}
    if kind == "attend":
        t, _, seqs, _, _ = _attend_plan(case)
        new, lens = case["new"], [t.lens[s] for s in seqs]
        whole = case["prefix"] // case["page"] * case["page"]        # read once for all
        keys = whole + sum(n - whole for n in lens)
        pairs = sum(new * (n - new) + new * (new + 1) / 2 for n in lens)
        return {"bytes": float(2 * keys * kv * (d + 1) + 2 * case["n"] * new * case["heads"] * d * _size(case["act"])),
                "flops": float(4 * d * case["heads"] * pairs)}
    pairs = _reorder_plan(case)[3]
    row = 2 * case["layers"] * kv * d * _size(case["dtype"])
    return {"bytes": float((len({a for a, _ in pairs}) + len(pairs)) * (case["tokens"] % case["page"]) * row), "flops": 0.0}


def _exact_turn(x, pos, case, back):
    """Each pair as a complex number times magnitude * exp(i angle)."""
    rot = case["rot"]
    f, mag = _frequencies(case)
    angle = pos.double()[:, None, None] * f * (-1 if back else 1)
    x = x.double()
    half = case["layout"] == "half"
    z = torch.complex(*(x[..., :rot].unflatten(-1, (2, rot // 2)).unbind(-2) if half else x[..., :rot].unflatten(-1, (rot // 2, 2)).unbind(-1)))
    z = z * torch.polar(torch.full_like(angle, mag), angle)
    x[..., :rot] = torch.cat([z.real, z.imag], -1) if half else torch.view_as_real(z).flatten(-2)
    return x


def _exact_held(x, dtype):
    """What rows [n, kv, d] in 64 bits are held as, in 64 bits."""
    out = torch.empty_like(x)
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** (-126 if dtype == "int8" else -117))
    room = 127 if dtype == "int8" else 448
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / room))         # (a step too far at a border, then put right)
    for step in (-1, 0, 1):
        fits = torch.exp2(e + step) * room >= top
        scale = torch.where(fits & ((torch.exp2(e + step - 1) * room < top) | (step == -1)), torch.exp2(e + step).maximum(scale), scale)
    y = x / scale
    if dtype == "int8":
        out = torch.round(y) * scale
    else:
        ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)   # 3 bits behind the first; 2^-9 the least
        out = torch.round(y / ulp) * ulp * scale
    return out


def _one_exact(q, k, v, scale):
    """q [rows, heads, d] whose last row sees all of k, v [keys, kv, d], in 64 bits."""
    rows, heads, d = q.shape
    keys, kv = k.shape[:2]
    out = torch.zeros(rows, heads, d, dtype=torch.float64, device="cuda")
    i = torch.arange(rows, device="cuda")[:, None] + keys - rows
    for h in range(heads):
        kh, vh = (x[:, h // (heads // kv)].double() for x in (k, v))
        x = q[:, h].double() @ kh.t().contiguous() * scale
        x = torch.softmax(torch.where(torch.arange(keys, device="cuda") <= i, x, -math.inf), -1)
        out[:, h] = x @ vh
    return out


def _held_rows(case, pool, pages, n):
    """The first n positions of a sequence's pages, K and V: [2][n, kv, d] in 64 bits."""
    p, d = case["page"], case["dim"]
    raw = pool[_long(pages), LAYER]                                  # [page, 2, kv, bytes]
    codes = raw[..., :p * d].reshape(-1, 2, case["kv"], p, d)
    codes = codes.view(torch.int8 if case["dtype"] == "int8" else torch.float8_e4m3fn).to(torch.float64)
    x = codes * torch.pow(2.0, raw[..., p * d:].double() - 127)[..., None]
    return [x[:, i].permute(0, 2, 1, 3).reshape(-1, case["kv"], d)[:n] for i in (0, 1)]


def exact(case, seed):
    kind = case["kind"]
    if kind == "rope":
        q, k, pos = _rope_inputs(case, seed)
        return _exact_turn(q, pos, case, case["back"]), _exact_turn(k, pos, case, case["back"])
    if kind == "keep":
        t, seqs, have, new, pool, q, k, v = _keep_inputs(case, seed)
        pos = _long([j for a, n in zip(have, new) for j in range(a, a + n)])
        k, v = k.double(), v.double()
        rot = dict(case, rot=case["dim"], **KEEP_ROPE)
        if case["rope"]:
            q, k = _exact_turn(q, pos, rot, False), _exact_turn(k, pos, rot, False)
        parts, at = [], 0
        for s, a, n in zip(seqs, have, new):
            old = _held_rows(case, pool, t.seqs[s], a)
            parts.append([torch.cat([o, _exact_held(x[at:at + n], case["dtype"])]) for o, x in zip(old, (k, v))])
            at += n
        out = tuple(torch.cat([p[i] for p in parts]) for i in (0, 1))
        return out + (q,) if case["rope"] else out
    if kind == "attend":
        t, base, seqs, _, copies, pool, q = _attend_inputs(case, seed)
        _copy_rows(case, pool, t, base, copies)
        parts, new = [], case["new"]
        for i, s in enumerate(seqs):
            k, v = _held_rows(case, pool, t.seqs[s], t.lens[s])
            parts.append(_one_exact(q[i * new:(i + 1) * new], k, v, 1 / math.sqrt(case["dim"])))
        return torch.cat(parts)
    if kind == "select":
        logits, scores, ended = _select_inputs(case, seed)
        n, b, k = case["groups"], case["beams"], case["picks"]
        out, beams, tokens = [], [], []
        for g in range(n):
            found = []
            for i in range(b):
                x, s = logits[g * b + i].double().cpu().numpy(), float(scores[g, i])
                if ended[g, i] >= 0:
                    found.append((s, i, int(ended[g, i])))
                    continue
                m = x.max()
                lse = m + math.log(np.exp(x - m).sum())
                least = np.partition(x, -min(k, x.size))[-min(k, x.size)]
                found += [(s + x[j] - lse, i, int(j)) for j in np.nonzero(x >= least)[0]]
            found.sort(key=lambda f: (-f[0], f[1], f[2]))
            out.append([f[0] for f in found[:k]])
            beams.append([f[1] for f in found[:k]])
            tokens.append([f[2] for f in found[:k]])
        return tuple(torch.tensor(x, dtype=t) for x, t in ((out, torch.float64), (beams, torch.int32), (tokens, torch.int32)))
    pool, _, _, _, pairs = _reorder_inputs(case, seed)
    want, r = pool.double(), case["tokens"] % case["page"]
    for a, b in pairs:
        want[b, :, :, :, :r] = want[a, :, :, :, :r]
    return {"pool": want, "tables": None}
