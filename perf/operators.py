"""The operators for many sequences over a paged cache, as timed cases.

Kinds of case and their ranges:

prompt    causal attention over packed prompts of different lengths, grouped
          heads: 1..48 prompts of 1..16384 tokens, f32, f16 and bf16, with
          keys of earlier tokens in front of a prompt's own where it has some
attend    one step's attention of a batch over the pages of its sequences:
          1..64 sequences of up to 65536 positions, 1..8 new tokens each, with
          or without a prefix that all of them share, f32 cache, f16 cache
          under f32 activations, f16 and bf16
store     a step's or a prompt's new keys and values into those pages
fork      sequences that go on from one sequence's middle: its whole pages
          shared, the page that it ends in copied for each
turnover  a cache in use: the older half of the sequences freed, the pages of
          the others moved to the front, each of them copied whole

In its plain form (own is False) a case is elementary torch operations in 32
bits, over sequences padded to the longest.
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
        # a short chat turn of a small model, f32 activations: latency
        {"name": "prompt_short_f32", "kind": "prompt", "dtype": "float32", "heads": 8, "kv": 2, "dim": 64,
         "n": 1, "longest": 37, "before": 0, "mix": 1},
        # a few prompts of the 2B shape at the framework's own activation type
        {"name": "prompt_2b_f32", "kind": "prompt", "dtype": "float32", "heads": 20, "kv": 5, "dim": 128,
         "n": 4, "longest": 2048, "before": 0, "mix": 2},
        # the prompts that wait in a server's queue, all at once
        {"name": "prompt_ragged_bf16", "kind": "prompt", "dtype": "bfloat16", "heads": 20, "kv": 5, "dim": 128,
         "n": 24, "longest": 2048, "before": 0, "mix": 3},
        # one long document
        {"name": "prompt_long_f16", "kind": "prompt", "dtype": "float16", "heads": 20, "kv": 5, "dim": 128,
         "n": 1, "longest": 16384, "before": 0, "mix": 4},
        # one user's next token at the 2B shape, f32 cache: latency
        {"name": "attend_one_f32", "kind": "attend", "act": "float32", "dtype": "float32", "heads": 20, "kv": 5,
         "dim": 128, "page": 64, "n": 1, "prefix": 0, "longest": 1101, "new": 1, "mix": 5},
        # a step of 64 chats behind one long system prompt, f16 cache under f32 activations
        {"name": "attend_shared_f16", "kind": "attend", "act": "float32", "dtype": "float16", "heads": 20, "kv": 5,
         "dim": 128, "page": 64, "n": 64, "prefix": 4096, "longest": 1024, "new": 1, "mix": 6},
        # long documents, one token each: what the memory gives
        {"name": "attend_long_bf16", "kind": "attend", "act": "bfloat16", "dtype": "bfloat16", "heads": 20, "kv": 5,
         "dim": 128, "page": 128, "n": 8, "prefix": 0, "longest": 65536, "new": 1, "mix": 7},
        # drafted tokens to be verified: five rows a sequence, a prefix that ends inside a page
        {"name": "attend_draft_bf16", "kind": "attend", "act": "bfloat16", "dtype": "bfloat16", "heads": 32, "kv": 8,
         "dim": 128, "page": 16, "n": 32, "prefix": 1000, "longest": 700, "new": 5, "mix": 8},
        # the new rows of a step of 64 chats
        {"name": "store_step_f32", "kind": "store", "act": "float32", "dtype": "float32", "kv": 5, "dim": 128,
         "page": 64, "n": 64, "longest": 1, "have": 700, "mix": 9},
        # the rows of many prompts, rounded to an f16 cache
        {"name": "store_prompts_f16", "kind": "store", "act": "float32", "dtype": "float16", "kv": 5, "dim": 128,
         "page": 64, "n": 24, "longest": 2048, "have": 50, "mix": 10},
        # sixteen answers to one question, all 30 layers of the 2B shape
        {"name": "fork_16_f16", "kind": "fork", "dtype": "float16", "layers": 30, "kv": 5, "dim": 128, "page": 64,
         "tokens": 1001, "n": 16},
        # a server's cache turned over once
        {"name": "turnover_bf16", "kind": "turnover", "dtype": "bfloat16", "layers": 8, "kv": 5, "dim": 128,
         "page": 32, "n": 12, "longest": 1500, "mix": 12},
    ]


# (query heads, KV heads, head dimension): the 2B shape, the repository's small models, and other common splits
HEADS = [(20, 5, 128), (20, 5, 128), (8, 2, 64), (6, 2, 64), (4, 2, 64), (32, 8, 128), (8, 8, 96), (8, 1, 80)]
TYPES = ["float32", "float16", "bfloat16"]
PAIRS = [("float32", "float32"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "attend", "attend", "attend", "store", "fork", "turnover"])
    heads, kv, dim = rng.choice(HEADS)
    mix, page = rng.randrange(1 << 20), rng.choice([16, 32, 64, 128])
    act, dtype = rng.choice(PAIRS)
    while kind == "prompt":
        c = {"kind": kind, "dtype": rng.choice(TYPES), "heads": heads, "kv": kv, "dim": dim, "n": _log(rng, 1, 48),
             "longest": _log(rng, 1, 16384), "before": rng.choice([0, 0, _log(rng, 1, 2000)]), "mix": mix}
        if c["heads"] * c["n"] * c["longest"] * (c["longest"] + c["before"]) <= 2e9:
            return c
    while kind == "attend":
        c = {"kind": kind, "act": act, "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "page": page,
             "n": _log(rng, 1, 64), "prefix": rng.choice([0, _log(rng, 1, 16000)]), "longest": _log(rng, 1, 65536),
             "new": rng.choice([1, 1, 1, rng.randint(2, 8)]), "mix": mix}
        if c["n"] * (c["prefix"] + c["longest"]) * kv * dim <= 8 * 65536 * 640:
            return c
    while kind == "store":
        c = {"kind": kind, "act": act, "dtype": dtype, "kv": kv, "dim": dim, "page": page, "n": _log(rng, 1, 64),
             "longest": _log(rng, 1, 4096), "have": _log(rng, 1, 3000), "mix": mix}
        if c["n"] * (c["longest"] + c["have"]) <= 80000:
            return c
    if kind == "fork":
        return {"kind": kind, "dtype": rng.choice(TYPES), "layers": _log(rng, 1, 30), "kv": kv, "dim": dim, "page": page,
                "tokens": page * rng.randint(0, 20) + rng.randint(1, page - 1), "n": _log(rng, 1, 24)}
    return {"kind": kind, "dtype": rng.choice(TYPES), "layers": _log(rng, 1, 12), "kv": kv, "dim": dim, "page": page,
            "n": _log(rng, 1, 16), "longest": _log(rng, 1, 1500), "mix": mix}


def _lengths(n, longest, mix):
    """n lengths of 1..longest, spread over their logarithm, the first the longest."""
    r = random.Random(mix)
    return [longest] + [_log(r, max(1, longest // 16), longest) for _ in range(n - 1)]


def _prompt_lengths(case):
    q = _lengths(case["n"], case["longest"], case["mix"])
    r = random.Random(case["mix"] + 1)
    return q, [n + r.randint(0, case["before"]) for n in q]


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
        """n sequences that share s's whole pages; (source, copies) of the page it ends in."""
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
    """The batch's tables as they stand with the new tokens in: (tables, sequences, lengths, the fork's page copies)."""
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


def _store_plan(case):
    t, r = _Tables(case["page"]), random.Random(case["mix"] + 1)
    new = _lengths(case["n"], case["longest"], case["mix"])
    have = [r.randint(0, case["have"]) for _ in new]
    seqs = [t.new() for _ in new]
    for s, n in zip(seqs, have):
        t.extend(s, n)
    for s, n in zip(seqs, new):
        t.extend(s, n)
    return t, seqs, have, new


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _type(name):
    return getattr(torch, name)


def _normal(seed, *shapes):
    """Seeded N(0, 1) tensors on the GPU, one for each (type, shape...)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn(*s[1:], device="cuda", generator=g).to(_type(s[0])) for s in shapes]


def _prompt_inputs(case, seed):
    q_len, k_len = _prompt_lengths(case)
    t, h, kv, d = case["dtype"], case["heads"], case["kv"], case["dim"]
    return _normal(seed, (t, sum(q_len), h, d), (t, sum(k_len), kv, d), (t, sum(k_len), kv, d))


def _pool(case, seed, pages, layers):
    """A cache's memory, [page][layer][K, V][head][slot][dim], every slot holding something."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    pool = torch.empty(pages, layers, 2, case["kv"], case["page"], case["dim"], dtype=_type(case["dtype"]), device="cuda")
    pool.normal_(generator=g)
    return pool


LAYERS, LAYER = 2, 1                 # attend and store work on one layer of a cache of two


def _attend_inputs(case, seed):
    t, base, seqs, own_len, copies = _attend_plan(case)
    pool = _pool(case, seed, t.used, LAYERS)
    q, = _normal(seed + 7919, (case["act"], case["n"] * case["new"], case["heads"], case["dim"]))
    return t, base, seqs, own_len, copies, pool, q


def _store_inputs(case, seed):
    t, seqs, have, new = _store_plan(case)
    pool = _pool(case, seed, t.used, LAYERS)
    k, v = _normal(seed + 7919, *[(case["act"], sum(new), case["kv"], case["dim"])] * 2)
    return t, seqs, have, new, pool, k, v


def _fork_inputs(case, seed):
    t = _Tables(case["page"])
    s = t.new()
    t.extend(s, case["tokens"])
    seqs, copies = t.fork(s, case["n"])
    return _pool(case, seed, t.used, case["layers"]), t, s, seqs, copies


def _turnover_inputs(case, seed):
    lens = _lengths(case["n"], case["longest"], case["mix"])
    pages = sum(-(-n // case["page"]) for n in lens)
    return _pool(case, seed, 2 * pages, case["layers"]), lens, pages


def _cache(case, pool, layers):
    return _package().PagedCache(device(), layers, case["kv"], case["dim"], case["page"], pool.shape[0], case["dtype"],
                                 mem=pool.data_ptr())


def _long(v):
    return torch.tensor(v, dtype=torch.long, device="cuda")


def _padded(rows, fill=0):
    """Lists of different lengths as one tensor, and which of its places hold something."""
    longest = max(len(r) for r in rows)
    return _long([list(r) + [fill] * (longest - len(r)) for r in rows])


def prepare(case, seed):
    s = {"case": case}
    kind = case["kind"]
    if kind == "prompt":
        q_len, k_len = _prompt_lengths(case)
        s["q"], s["k"], s["v"] = _prompt_inputs(case, seed)
        s["out"] = torch.empty_like(s["q"])
        if own:
            s["plan"] = _package().PromptAttention(device(), case["dtype"], case["heads"], case["kv"], case["dim"], q_len, k_len)
            s["ptrs"] = [s[n].data_ptr() for n in ("q", "k", "v", "out")]
        else:
            q0, k0 = np.cumsum([0] + q_len), np.cumsum([0] + k_len)
            s["qi"] = _padded([range(a, a + n) for a, n in zip(q0, q_len)])
            s["ki"] = _padded([range(a, a + n) for a, n in zip(k0, k_len)])
            s["k_len"], s["shift"] = _long(k_len), _long([b - a for a, b in zip(q_len, k_len)])
            s["back"] = (_long(np.repeat(np.arange(len(q_len)), q_len)), _long(np.concatenate([np.arange(n) for n in q_len])))
    elif kind == "attend":
        t, base, seqs, own_len, copies, pool, s["q"] = _attend_inputs(case, seed)
        s["out"] = torch.empty_like(s["q"])
        s["pool"] = pool
        if own:
            torch.cuda.synchronize()
            c = s["cache"] = _cache(case, pool, LAYERS)
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
            if copies:
                pool[_long(copies), :, :, :, :case["prefix"] % case["page"]] = \
                    pool[t.seqs[base][-1], :, :, :, :case["prefix"] % case["page"]].clone()
            s["tables"], s["len"] = _padded([t.seqs[i] for i in seqs]), _long([t.lens[i] for i in seqs])
    elif kind == "store":
        t, seqs, have, new, s["pool"], s["k"], s["v"] = _store_inputs(case, seed)
        if own:
            c = s["cache"] = _cache(case, s["pool"], LAYERS)
            ids = [c.new() for _ in seqs]
            c.batch(ids, have, case["kv"], case["act"]).close()
            s["batch"] = c.batch(ids, new, case["kv"], case["act"])
            s["ptrs"] = [s["k"].data_ptr(), s["v"].data_ptr()]
        else:
            p = case["page"]
            at = [(t.seqs[i][j // p], j % p) for i, a, n in zip(seqs, have, new) for j in range(a, a + n)]
            s["at"] = _long([a for a, _ in at]), _long([b for _, b in at])
    elif kind == "fork":
        s["pool"], t, src, seqs, copies = _fork_inputs(case, seed)
        if own:
            c = s["cache"] = _cache(case, s["pool"], case["layers"])
            s["src"] = c.new()
            c.batch([s["src"]], [case["tokens"]], case["kv"], case["dtype"]).close()
            s["ids"] = []
        else:
            s["from"], s["to"] = t.seqs[src][-1], _long(copies)
            s["tables"] = np.array([t.seqs[i] for i in seqs], np.int32)
    else:
        s["pool"], lens, pages = _turnover_inputs(case, seed)
        if own:
            c = s["cache"] = _cache(case, s["pool"], case["layers"])
            s["older"] = [c.new() for _ in lens]
            c.batch(s["older"], lens, case["kv"], case["dtype"]).close()
            s["younger"] = [c.new() for _ in lens]
            c.batch(s["younger"], lens, case["kv"], case["dtype"]).close()
        else:
            s["half"] = pages
            p = case["page"]
            ends = np.cumsum([-(-n // p) for n in lens])
            rows = np.full(pages, p)
            rows[ends - 1] = [(n - 1) % p + 1 for n in lens]
            s["held"] = (torch.arange(p, device="cuda")[None] < _long(rows)[:, None]).view(pages, 1, 1, 1, p, 1)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _softmax_products(q, k, v, seen, scale):
    """softmax(scale q k^T over the seen) v in 32 bits: q [b, kv, rows, d], k and v [b, kv, keys, d], seen [b, 1, rows, keys].
    Rows that see nothing are 0."""
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    return torch.matmul(s, v) / total.masked_fill(total == 0, 1)


def _plain_prompt(s):
    c = s["case"]
    b, rows = s["qi"].shape
    keys, kv, g, d = s["ki"].shape[1], c["kv"], c["heads"] // c["kv"], c["dim"]
    q = s["q"][s["qi"]].float().view(b, rows, kv, g, d).permute(0, 2, 3, 1, 4).reshape(b, kv, g * rows, d)
    k, v = (s[n][s["ki"]].float().transpose(1, 2).contiguous() for n in ("k", "v"))
    i, j = torch.arange(rows, device="cuda"), torch.arange(keys, device="cuda")
    seen = (j <= i[:, None] + s["shift"][:, None, None]) & (j < s["k_len"][:, None, None])
    out = _softmax_products(q, k, v, seen.repeat(1, g, 1)[:, None], d ** -0.5)
    out = out.view(b, kv, g, rows, d).permute(0, 3, 1, 2, 4).reshape(b, rows, kv * g, d)
    s["out"].copy_(out[s["back"]])
    return s["out"]


def _plain_attend(s):
    c = s["case"]
    b, new, kv, g, d = c["n"], c["new"], c["kv"], c["heads"] // c["kv"], c["dim"]
    pages = s["pool"][:, LAYER][s["tables"]]                         # [b, page, 2, kv, slot, d]
    k, v = (pages[:, :, i].transpose(1, 2).reshape(b, kv, -1, d).float() for i in (0, 1))
    q = s["q"].view(b, new, kv, g, d).float().permute(0, 2, 1, 3, 4).reshape(b, kv, new * g, d)
    j, row = torch.arange(k.shape[2], device="cuda"), torch.arange(new, device="cuda").repeat_interleave(g)
    seen = j <= s["len"][:, None, None] - new + row[:, None]
    out = _softmax_products(q, k, v, seen[:, None], d ** -0.5)
    s["out"].copy_(out.view(b, kv, new, g, d).transpose(1, 2).reshape(b * new, kv * g, d))
    return s["out"]


def run(state):
    s, case = state, state["case"]
    kind, scale = case["kind"], case["dim"] ** -0.5
    if kind == "prompt":
        if not own:
            return _plain_prompt(s)
        s["plan"].run(*s["ptrs"], scale)
        return s["out"]
    if kind == "attend":
        if not own:
            return _plain_attend(s)
        s["batch"].attend(LAYER, *s["ptrs"], scale)
        return s["out"]
    if kind == "store":
        if own:
            s["batch"].store(LAYER, *s["ptrs"])
        else:
            page, slot = s["at"]
            s["pool"][page, LAYER, 0, :, slot] = s["k"].to(s["pool"].dtype)
            s["pool"][page, LAYER, 1, :, slot] = s["v"].to(s["pool"].dtype)
        return s["pool"]
    if kind == "fork":
        if own:
            s["cache"].free(s["ids"])
            s["ids"] = s["cache"].fork(s["src"], case["tokens"], case["n"])
            tables = s["cache"].tables(s["ids"])
        else:
            r, tables = case["tokens"] % case["page"], s["tables"]
            s["pool"][s["to"], :, :, :, :r] = s["pool"][s["from"], :, :, :, :r]
        return {"pool": s["pool"], "tables": tables}
    if own:
        c = s["cache"]
        c.free(s["older"])
        c.compact()
        s["older"], s["younger"] = s["younger"], c.copy(s["younger"])
    else:
        n, pool = s["half"], s["pool"]
        pool[:n] = pool[n:]
        pool[n:] = torch.where(s["held"], pool[:n], pool[n:])
    return s["pool"]


# ---------------------------------------------------------------------------
# the work of a pass, and its result in 64 bits
# ---------------------------------------------------------------------------

def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    kind = case["kind"]
    d, kv = case["dim"], case["kv"]
    if kind == "prompt":
        q_len, k_len = _prompt_lengths(case)
        rows = 2 * sum(q_len) * case["heads"] + 2 * sum(k_len) * kv
        pairs = sum(a * (b - a) + a * (a + 1) / 2 for a, b in zip(q_len, k_len))
        return {"bytes": float(rows * d * _size(case["dtype"])), "flops": float(4 * d * case["heads"] * pairs)}
    if kind == "attend":
        t, _, seqs, _, _ = _attend_plan(case)
        new, lens = case["new"], [t.lens[s] for s in seqs]
        whole = case["prefix"] // case["page"] * case["page"]        # read once for all
        keys = whole + sum(n - whole for n in lens)
        pairs = sum(new * (n - new) + new * (new + 1) / 2 for n in lens)
        return {"bytes": float(2 * keys * kv * d * _size(case["dtype"]) + 2 * case["n"] * new * case["heads"] * d * _size(case["act"])),
                "flops": float(4 * d * case["heads"] * pairs)}
    if kind == "store":
        rows = 2 * sum(_lengths(case["n"], case["longest"], case["mix"])) * kv
        return {"bytes": float(rows * d * (_size(case["act"]) + _size(case["dtype"]))), "flops": 0.0}
    row = 2 * case["layers"] * kv * d * _size(case["dtype"])         # one position in every layer
    if kind == "fork":
        return {"bytes": float((1 + case["n"]) * (case["tokens"] % case["page"]) * row), "flops": 0.0}
    # what is moved is read and written, and so is each copy
    return {"bytes": float(4 * sum(_lengths(case["n"], case["longest"], case["mix"])) * row), "flops": 0.0}


def _one_exact(q, k, v, scale):
    """q [rows, heads, d] whose last row sees all of k, v [keys, kv, d], in 64 bits."""
    rows, heads, d = q.shape
    keys, kv = k.shape[:2]
    out = torch.zeros(rows, heads, d, dtype=torch.float64, device="cuda")
    for h in range(heads):
        kh, vh = (x[:, h // (heads // kv)].double() for x in (k, v))
        for a in range(0, rows, 4096):
            b = min(rows, a + 4096)
            n = max(0, keys - rows + b)                                # no row of these sees more
            x = q[a:b, h].double() @ kh[:n].t() * scale
            i = torch.arange(a, b, device="cuda")[:, None] + keys - rows
            x = torch.softmax(torch.where(torch.arange(n, device="cuda") <= i, x, -math.inf), -1)
            out[a:b, h] = torch.where(i >= 0, x @ vh[:n], torch.zeros((), dtype=torch.float64, device="cuda"))
    return out


def exact(case, seed):
    kind, scale = case["kind"], 1 / math.sqrt(case["dim"])
    if kind == "prompt":
        q, k, v = _prompt_inputs(case, seed)
        parts, a, b = [], 0, 0
        for nq, nk in zip(*_prompt_lengths(case)):
            parts.append(_one_exact(q[a:a + nq], k[b:b + nk], v[b:b + nk], scale))
            a, b = a + nq, b + nk
        return torch.cat(parts)
    if kind == "attend":
        t, base, seqs, _, copies, pool, q = _attend_inputs(case, seed)
        r = case["prefix"] % case["page"]
        for i in copies:
            pool[i, :, :, :, :r] = pool[t.seqs[base][-1], :, :, :, :r]
        parts, new = [], case["new"]
        for i, s in enumerate(seqs):
            own_pages = pool[_long(t.seqs[s]), LAYER]                 # [page, 2, kv, slot, d]
            k, v = (own_pages[:, x].permute(0, 2, 1, 3).reshape(-1, case["kv"], case["dim"])[:t.lens[s]] for x in (0, 1))
            parts.append(_one_exact(q[i * new:(i + 1) * new], k, v, scale))
        return torch.cat(parts)
    if kind == "store":
        t, seqs, have, new, pool, k, v = _store_inputs(case, seed)
        want, row, p = pool.double(), 0, case["page"]
        for s, a, n in zip(seqs, have, new):
            at = torch.arange(a, a + n, device="cuda")
            page = _long(t.seqs[s])[at // p]
            for i, x in enumerate((k, v)):
                want[page, LAYER, i, :, at % p] = x[row:row + n].double()
            row += n
        return want
    if kind == "fork":
        pool, t, src, _, copies = _fork_inputs(case, seed)
        want, r = pool.double(), case["tokens"] % case["page"]
        for i in copies:
            want[i, :, :, :, :r] = want[t.seqs[src][-1], :, :, :, :r]
        return {"pool": want, "tables": None}
    pool, lens, n = _turnover_inputs(case, seed)
    want, at, p = pool.double(), 0, case["page"]
    want[:n] = want[n:].clone()
    for length in lens:
        whole, r = divmod(length, p)
        want[n + at:n + at + whole] = want[at:at + whole]
        if r:
            want[n + at + whole, :, :, :, :r] = want[at + whole, :, :, :, :r]
        at += -(-length // p)
    return want
