"""Performance cases of the paged key-value cache and the operators on it.

A cache holds keys and values of several sequences in pages: k and v are
[layers, pages, kv heads, tokens of a page, head size], `table` says which page
holds tokens p * page .. of a sequence (-1: none), `lengths` how many tokens it
has, `refs` how many sequences use a page.  Five kinds of call:

  rope     rotary positions of new queries and keys, and the write of the new
           keys and values into their pages
  decode   attention of one new token per sequence
  prompt   attention of several new tokens per sequence (prompts, their chunks,
           drafted tokens), with a sliding window and first tokens that stay visible
  fork     sequences that continue others: whole pages shared, the last one copied
  compact  sequences that keep some tokens of others, in fresh pages

New tokens are the last ones of their sequence, as they are after the cache has
been extended for them.
"""
import math
import os
import sys

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_IDS = {"f32": 0, "f16": 1, "bf16": 30}


def listed():
    return [
        # one decode step of 32 sequences: the smallest call of a layer, where latency counts
        {"name": "rope_decode32", "kind": "rope", "type": "bf16", "heads": 16, "kv": 8, "hs": 256, "page": 16, "n": 32,
         "lo": 300, "hi": 30000, "rows_lo": 1, "rows_hi": 1, "rot": 256, "pairs": False, "scaling": "none"},
        # prompts of three sequences far behind the trained length: part of the head, pairs side by side, scaled
        {"name": "rope_prompt", "kind": "rope", "type": "f16", "heads": 32, "kv": 4, "hs": 128, "page": 32, "n": 3,
         "lo": 9000, "hi": 120000, "rows_lo": 1500, "rows_hi": 4001, "rot": 64, "pairs": True, "scaling": "ramp"},
        # one sequence at the configured length: what a chat waits for
        {"name": "decode_one_8k", "kind": "decode", "type": "bf16", "heads": 16, "kv": 8, "hs": 256, "page": 16, "n": 1,
         "lo": 8192, "hi": 8192, "window": 0, "sinks": 0},
        # a served batch of unequal lengths, eight query heads to a key head
        {"name": "decode_batch64", "kind": "decode", "type": "f16", "heads": 32, "kv": 4, "hs": 128, "page": 32, "n": 64,
         "lo": 200, "hi": 16384, "window": 0, "sinks": 0},
        # a sliding-window layer of long streams, the pages between the first tokens and the window freed
        {"name": "decode_window_sinks", "kind": "decode", "type": "bf16", "heads": 8, "kv": 1, "hs": 512, "page": 16,
         "n": 24, "lo": 700, "hi": 60001, "window": 1024, "sinks": 4},
        # a few long documents with the reference's 32-bit cache
        {"name": "decode_long_f32", "kind": "decode", "type": "f32", "heads": 8, "kv": 2, "hs": 256, "page": 64, "n": 4,
         "lo": 20001, "hi": 65536, "window": 0, "sinks": 0},
        # five drafted tokens of each of eight sequences, checked at once
        {"name": "prompt_draft5", "kind": "prompt", "type": "bf16", "heads": 16, "kv": 8, "hs": 256, "page": 16, "n": 8,
         "lo": 1000, "hi": 16384, "rows_lo": 5, "rows_hi": 5, "window": 0, "sinks": 0},
        # a prompt of a thousand tokens in a sliding-window layer
        {"name": "prompt_window", "kind": "prompt", "type": "f16", "heads": 8, "kv": 2, "hs": 256, "page": 16, "n": 1,
         "lo": 1001, "hi": 1001, "rows_lo": 1001, "rows_hi": 1001, "window": 512, "sinks": 0},
        # chunks of several prompts behind what is cached already, window and first tokens, no round sizes
        {"name": "prompt_chunks_sinks", "kind": "prompt", "type": "f16", "heads": 16, "kv": 4, "hs": 128, "page": 32,
         "n": 4, "lo": 1201, "hi": 12001, "rows_lo": 301, "rows_hi": 1100, "window": 4096, "sinks": 16},
        # a whole prompt at the configured length, causal: the most work
        {"name": "prompt_8k", "kind": "prompt", "type": "bf16", "heads": 16, "kv": 8, "hs": 256, "page": 16, "n": 1,
         "lo": 8192, "hi": 8192, "rows_lo": 8192, "rows_hi": 8192, "window": 0, "sinks": 0},
        # sixteen prompts, each continued four ways
        {"name": "fork_64", "kind": "fork", "type": "bf16", "kv": 8, "hs": 256, "page": 32, "layers": 6, "n": 64, "from": 16,
         "lo": 500, "hi": 4001},
        # sixteen sequences that keep their first page and a quarter of the rest
        {"name": "compact_16", "kind": "compact", "type": "f16", "kv": 4, "hs": 128, "page": 16, "layers": 6, "n": 16,
         "from": 16, "lo": 1000, "hi": 8001, "keep": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["rope", "decode", "decode", "decode", "prompt", "prompt", "prompt", "fork", "compact"])
    c = {"kind": kind, "type": rng.choice(["f16", "bf16", "bf16", "f32"]), "page": rng.choice([16, 32, 64, 128, 256])}
    c["kv"] = rng.choice([1, 2, 3, 4, 8])
    c["hs"] = rng.choice([64, 80, 96, 128, 192, 256, 512])
    if kind in ("rope", "decode", "prompt"):
        c["heads"] = c["kv"] * rng.choice([1, 2, 3, 4, 8] if c["kv"] < 8 else [1, 2, 4])
        c["n"] = 1 if rng.random() < 0.3 else _log(rng, 1, 64)
        c["lo"] = _log(rng, 1, 20000)
        c["hi"] = max(c["lo"], _log(rng, 100, 50000))
    if kind in ("decode", "prompt"):
        c["window"] = rng.choice([0, 0, 128, 512, 1000, 1024, 4096])
        c["sinks"] = rng.choice([0, 1, 4, 16, 100]) if c["window"] else 0
    if kind == "rope":
        c |= {"rot": rng.choice([c["hs"], c["hs"], c["hs"] // 2, c["hs"] // 4]), "pairs": rng.random() < 0.5,
              "scaling": rng.choice(["none", "linear", "base", "ramp"])}
    if kind in ("rope", "prompt"):
        c["rows_lo"] = _log(rng, 1, 2000)
        c["rows_hi"] = max(c["rows_lo"], _log(rng, 1, 8000))
        c["lo"] = max(c["lo"], c["rows_lo"])
        c["hi"] = max(c["hi"], c["rows_hi"])
    if kind in ("fork", "compact"):
        c |= {"layers": rng.randint(1, 8), "n": _log(rng, 1, 96), "lo": _log(rng, 1, 2000)}
        c["from"] = rng.randint(1, c["n"])
        c["hi"] = max(c["lo"], _log(rng, 100, 8000))
        if kind == "compact":
            c["from"] = c["n"]
            c["keep"] = rng.choice([0.05, 0.25, 0.7])
    return c


def draw(rng):
    while True:
        c = _draw(rng)
        w, n = work(c), c["n"]
        if w["bytes"] > 1.0e9 or w["flops"] > 5.0e11:
            continue
        pages = (n + c.get("from", 0)) * c["hi"] * c["kv"] * c["hs"] * c.get("layers", 1)  # before sharing
        if pages > 6e8 or (c["kind"] == "prompt" and n * c["heads"] * c["rows_hi"] * c["hi"] > 1.2e9):
            continue  # the plain form's padded copies and scores
        return c


# ------------------------------------------------------------------- sizes ---

def _spread(lo, hi, n):
    """n whole numbers from hi down to lo, evenly over their logarithm."""
    if n == 1:
        return [hi]
    return [int(round(hi * (lo / hi) ** (i / (n - 1)))) for i in range(n)]


def _rows(c):
    if "rows_lo" not in c:
        return [1] * c["n"]
    return [min(r, l) for r, l in zip(_spread(c["rows_lo"], c["rows_hi"], c["n"]), _lengths(c))]


def _lengths(c):
    return _spread(c["lo"], c["hi"], c.get("from", c["n"]))


def _kept(c, length):
    """Tokens that compact keeps behind the first page."""
    return max(0, int((length - c["page"]) * c["keep"]))


def _visible(p, window, sinks):
    """Tokens that position p sees."""
    return p + 1 if not window else min(p + 1, window) + max(0, min(sinks, p + 1 - window))


def _seen(c, length, rows):
    """Cached tokens that the last `rows` positions of a sequence see together."""
    if not c.get("window"):
        return length
    first = max(0, length - rows - c["window"] + 1)
    return length - first + min(c["sinks"], first)


def work(case):
    c = case
    es = 4 if c["type"] == "f32" else 2
    lengths, kind = _lengths(c), c["kind"]
    if kind in ("fork", "compact"):
        row = 2 * c["kv"] * c["hs"] * es * c["layers"]
        src = [lengths[i % c["from"]] for i in range(c["n"])]
        moved = sum(l % c["page"] if kind == "fork" else _kept(c, l) for l in src)
        return {"bytes": 2.0 * row * moved + 8 * sum(-(-l // c["page"]) for l in src), "flops": 0}
    rows = _rows(c)
    q = sum(rows) * c["heads"] * c["hs"]
    if kind == "rope":
        kv = sum(rows) * c["kv"] * c["hs"]
        return {"bytes": 8.0 * q + 2 * kv * (4 + es), "flops": 0}
    seen = sum(_seen(c, l, r) for l, r in zip(lengths, rows))
    pairs = sum(_visible(p, c["window"], c["sinks"]) for l, r in zip(lengths, rows) for p in range(l - r, l))
    return {"bytes": 8.0 * q + 2.0 * seen * c["kv"] * c["hs"] * es, "flops": 4.0 * pairs * c["heads"] * c["hs"]}


# ------------------------------------------------------------------ inputs ---

def _freqs(c):
    """Angle per position of each pair, and what cosines and sines are multiplied by."""
    rot, base, factor, trained = c["rot"], 10000.0, 8.0, 16384.0
    if c["scaling"] == "base":
        base *= factor ** (rot / (rot - 2))
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if c["scaling"] == "linear":
        f = [v / factor for v in f]
    if c["scaling"] != "ramp":
        return f, 1.0
    at = [rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
    lo, hi = max(0.0, math.floor(at[0])), min(rot - 1.0, math.ceil(at[1]))
    out = []
    for i, v in enumerate(f):
        keep = 1.0 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))
        out.append(v * keep + v / factor * (1.0 - keep))
    return out, 1.0 + 0.1 * math.log(factor)


def _dev(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _inputs(case, seed):
    """A cache in use, its pages in no order, and the tensors of the call: from the seed alone."""
    c, kind = case, case["kind"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    typ, page, kv, hs, n, layers = _TYPES[c["type"]], c["page"], c["kv"], c["hs"], c["n"], c.get("layers", 1)
    lengths, rows = _lengths(c), _rows(c)
    paged = kind in ("fork", "compact")
    seqs = len(lengths) + (n if paged else 0)
    per_seq = -(-max(lengths) // page) + 3
    # the tokens that sequences still hold: with a window the pages that nothing sees again are freed, and a
    # call that only writes needs the last ones alone
    held = []
    for l, r in zip(lengths, rows if not paged else lengths):
        last = l - r if kind == "rope" else max(0, l - r - c["window"] + 1) if c.get("window") else 0
        first = c.get("sinks", 0) if c.get("window") else 0
        held.append([p for p in range(-(-l // page)) if (p + 1) * page > last or p * page < first])
    count = sum(len(h) for h in held)
    old = [1 + i % 3 for i in range(n)] if paged else []  # pages of the sequences that are replaced
    fresh = 0
    if kind == "fork":
        fresh = n
    elif kind == "compact":
        fresh = sum(-(-_kept(c, l) // page) + 1 for l in lengths)
    pages = count + sum(old) + 2 * fresh + 5
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    at = [(s, p) for s, h in enumerate(held) for p in h]
    at += [(len(lengths) + i, p) for i, m in enumerate(old) for p in range(m)]
    at_s, at_p = _dev([a[0] for a in at], torch.int64), _dev([a[1] for a in at], torch.int64)
    table = torch.full((seqs, per_seq), -1, dtype=torch.int32, device="cuda")
    table[at_s, at_p] = order[:len(at)]
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:len(at)].long()] = 1
    shape = (layers, pages, kv, page, hs)
    d = {"table": table, "refs": refs, "lengths": _dev(lengths + [m * page - 1 for m in old]),
         "status": torch.zeros(1, dtype=torch.int32, device="cuda")}

    def normal(*size, scale=1.0):
        return torch.randn(*size, device="cuda", generator=gen) * scale

    if paged:
        d["k"], d["v"] = (torch.empty(shape, dtype=typ, device="cuda").normal_(generator=gen) for _ in range(2))
        perm = torch.randperm(c["from"], generator=gen, device="cuda").int()
        d["src"] = perm[torch.arange(n, device="cuda") % c["from"]].contiguous()
        d["dst"] = (torch.randperm(n, generator=gen, device="cuda") + c["from"]).int()
        if kind == "compact":
            lens = d["lengths"][d["src"].long()].tolist()
            kept = [_kept(c, l) for l in lens]
            lists = [torch.randperm(max(0, l - page), generator=gen, device="cuda")[:m].sort().values + page
                     for l, m in zip(lens, kept)]
            d["keep"] = torch.cat(lists).int()
            d["prefix"] = _dev([min(page, l) for l in lens])
            d["begin"] = _dev([sum(kept[:i]) for i in range(n + 1)])
        return d
    order_s = torch.randperm(n, generator=gen, device="cuda")
    host_order = order_s.tolist()
    counts = [rows[i] for i in host_order]
    total = sum(rows)
    d["seqs"] = order_s.int()
    d["begin"] = _dev([sum(counts[:i]) for i in range(n + 1)])
    d["total"], d["most_rows"], d["most"] = total, max(rows), max(lengths)
    if kind == "rope":
        freqs, d["gain"] = _freqs(c)
        d["freqs"] = _dev(freqs, torch.float64)
        d["q"], d["kn"], d["vn"] = normal(total, c["heads"], hs), normal(total, kv, hs), normal(total, kv, hs)
        d["k"], d["v"] = torch.zeros(shape, dtype=typ, device="cuda"), torch.zeros(shape, dtype=typ, device="cuda")
        return d
    # keys with a common part and values that are not centred, as trained layers have them; queries large
    # enough that a softmax over many positions is neither flat nor one position
    d["k"] = (normal(*shape) + normal(1, 1, kv, 1, hs, scale=0.5)).to(typ)
    d["v"] = (normal(*shape) + normal(1, 1, kv, 1, hs, scale=0.3)).to(typ)
    d["q"] = normal(total, c["heads"], hs, scale=2.0)
    d["scale"] = 1.0 / math.sqrt(hs)
    return d


_ctx = None


def _context():
    """The program's one context, on torch's current stream: inputs, calls and what reads their results are in
    order.  Torch's default stream has no handle that a context takes, so the program leaves it for another."""
    global _ctx
    if _ctx is None:
        package = os.path.join(_ROOT, "gemma4.kt_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import g4hip
        _ctx = g4hip.Context(0)
    before = torch.cuda.current_stream()
    if before.cuda_stream == 0:
        torch.cuda.set_stream(torch.cuda.Stream())
        torch.cuda.current_stream().wait_stream(before)
    _ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return _ctx


def prepare(case, seed):
    ctx = _context() if own else None
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] in ("rope", "decode", "prompt"):
        s["out"] = torch.empty_like(s["q"])
    if own:
        import g4hip
        s["ctx"] = ctx
        s["cache"] = g4hip.KvCache(s["k"], s["v"], s["table"], s["lengths"], s["refs"], s["status"])
        if case["kind"] == "rope":
            s["rope"] = g4hip.Rope(s["freqs"], g4hip.ROPE_PAIRS if case["pairs"] else g4hip.ROPE_HALF, s["gain"])
    return s


# --------------------------------------------------------------------- run ---

def _own(s):
    import g4hip
    c, kind, ctx, cache = s["case"], s["case"]["kind"], s["ctx"], s["cache"]
    if kind == "rope":
        g4hip.kv_rope_write_dev(ctx, cache, 0, s["q"], s["out"], s["kn"], s["vn"], c["heads"], s["rope"], s["seqs"],
                                s["begin"], s["total"])
        return [s["out"], s["k"], s["v"]]
    if kind == "decode":
        g4hip.paged_attention_dev(ctx, cache, 0, s["q"], s["out"], c["heads"], s["seqs"], s["scale"], c["window"],
                                  c["sinks"])
        return s["out"]
    if kind == "prompt":
        g4hip.paged_prompt_dev(ctx, cache, 0, s["q"], s["out"], c["heads"], s["seqs"], s["begin"], s["total"],
                               s["scale"], c["window"], c["sinks"])
        return s["out"]
    if kind == "fork":
        g4hip.kv_fork_dev(ctx, cache, s["src"], s["dst"])
    else:
        g4hip.kv_compact_dev(ctx, cache, s["src"], s["dst"], s["prefix"], s["keep"], s["begin"])
    return [s["table"], s["lengths"], s["refs"], s["k"], s["v"]]


def _row_places(s):
    """For each new row: its entry in the list of sequences, and its position."""
    row = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    entry = (row[:, None] >= s["begin"][None, 1:]).sum(1)
    length = s["lengths"][s["seqs"].long()]
    return entry, (length - s["begin"][1:])[entry] + row


def _turn(x, cos, sin, rot, pairs):
    head, rest = x[..., :rot], x[..., rot:]
    if pairs:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).reshape(head.shape)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([head, rest], -1)


def _plain_rope(s):
    c = s["case"]
    entry, pos = _row_places(s)
    angle = pos.double()[:, None] * s["freqs"][None]
    cos, sin = ((f(angle) * s["gain"]).float()[:, None] for f in (torch.cos, torch.sin))
    out = _turn(s["q"], cos, sin, c["rot"], c["pairs"])
    at = s["table"][s["seqs"].long()[entry], (pos // c["page"]).long()].long()
    inside = (pos % c["page"]).long()
    s["k"][0, at, :, inside] = _turn(s["kn"], cos, sin, c["rot"], c["pairs"]).to(s["k"].dtype)
    s["v"][0, at, :, inside] = s["vn"].to(s["v"].dtype)
    return [out, s["k"], s["v"]]


def _gathered(s, pool):
    """The cached rows of each sequence of the list, [n, kv heads, tokens, head size]."""
    c = s["case"]
    pages = -(-s["most"] // c["page"])
    at = s["table"][s["seqs"].long(), :pages].long()
    x = pool[0][at.clamp(min=0)].float()  # n, pages, kv heads, page, head size
    return x.transpose(1, 2).reshape(c["n"], c["kv"], pages * c["page"], c["hs"])


def _softmax_av(scores, seen, v):
    scores = scores.masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return torch.matmul(e, v) / e.sum(-1, keepdim=True)


def _plain_attention(s):
    """Queries padded to the most rows of a sequence; the padding is not returned."""
    c = s["case"]
    n, kv, group, hs, most = c["n"], c["kv"], c["heads"] // c["kv"], c["hs"], s["most_rows"]
    entry, pos = _row_places(s)
    row = torch.arange(s["total"], device="cuda") - s["begin"].long()[entry]
    q = torch.zeros(n, most, c["heads"], hs, device="cuda")
    q[entry, row] = s["q"]
    q = q.reshape(n, most, kv, group, hs).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, hs)
    k, v = _gathered(s, s["k"]), _gathered(s, s["v"])
    scores = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    scores = scores.reshape(n, kv, group, most, -1)
    at = torch.zeros(n, most, dtype=torch.int32, device="cuda")
    at[entry, row] = pos
    t = torch.arange(scores.shape[-1], device="cuda", dtype=torch.int32)
    seen = t <= at[:, :, None]
    if c["window"]:
        seen &= (t > at[:, :, None] - c["window"]) | (t < c["sinks"])
    out = _softmax_av(scores, seen[:, None, None], v[:, :, None])
    return out.permute(0, 3, 1, 2, 4).reshape(n, most, c["heads"], hs)[entry, row]


def _plain_move(s):
    """fork and compact: the first pages shared, the rest copied token by token into the lowest free pages."""
    c, page = s["case"], s["case"]["page"]
    src, dst, table, refs = s["src"].long(), s["dst"].long(), s["table"], s["refs"]
    old = table[src]
    if c["kind"] == "fork":
        prefix = s["lengths"][src].long()
        length, most = prefix, page
    else:
        prefix = s["prefix"].long()
        length = prefix + (s["begin"][1:] - s["begin"][:-1]).long()
        most = page + int(c["hi"] * c["keep"])
    shared = prefix // page
    used = -(-length // page)
    need = used - shared
    free = torch.argsort((refs != 0).int(), stable=True)  # the free pages, the lowest first
    column = torch.arange(table.shape[1], device="cuda")
    is_shared = column < shared[:, None]
    is_fresh = ~is_shared & (column < used[:, None])
    first = torch.cumsum(need, 0) - need
    fresh = free[(first[:, None] + column - shared[:, None]).clamp(0, refs.numel() - 1)].int()
    new = torch.where(is_shared, old, torch.where(is_fresh, fresh, -1))
    # the tokens behind the shared pages
    to = shared[:, None] * page + torch.arange(most, device="cuda")
    wanted = to < length[:, None]
    frm = to
    if c["kind"] == "compact":
        i = (s["begin"][:-1].long()[:, None] + to - prefix[:, None]).clamp(0, max(0, s["keep"].numel() - 1))
        listed = s["keep"].long()[i] if s["keep"].numel() else i
        frm = torch.where(to < prefix[:, None], to, listed)
    frm, to = frm.clamp(0, old.shape[1] * page - 1), to.clamp(0, old.shape[1] * page - 1)
    e = torch.arange(c["n"], device="cuda")[:, None].expand_as(to)
    e, frm, to = e[wanted], frm[wanted], to[wanted]
    p, r = old[e, frm // page].long(), new[e, to // page].long()
    for pool in (s["k"], s["v"]):
        pool[:, r, :, to % page] = pool[:, p, :, frm % page]
    gone = table[dst]
    refs.index_add_(0, gone.clamp(min=0).reshape(-1), -(gone >= 0).int().reshape(-1))
    refs.index_add_(0, new.clamp(min=0).reshape(-1), (new >= 0).int().reshape(-1))
    table[dst] = new
    s["lengths"][dst] = length.int()
    return [table, s["lengths"], refs, s["k"], s["v"]]


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "rope":
        return _plain_rope(state)
    return _plain_attention(state) if kind in ("decode", "prompt") else _plain_move(state)


# ------------------------------------------------------------------- exact ---

def _exact_rope(c, s):
    out, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    begin, seqs, lengths, table = (s[x].tolist() for x in ("begin", "seqs", "lengths", "table"))
    half = c["rot"] // 2

    def turned(x, pos):
        z = torch.polar(torch.full((1, 1, 1), s["gain"], dtype=torch.float64, device="cuda"),
                        pos.double()[:, None, None] * s["freqs"])
        x = x.double()
        i = torch.arange(half, device="cuda")
        i, j = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + half)
        w = torch.complex(x[..., i], x[..., j]) * z
        x[..., i], x[..., j] = w.real, w.imag
        return x

    for e, q in enumerate(seqs):
        a, b = begin[e], begin[e + 1]
        pos = torch.arange(lengths[q] - (b - a), lengths[q], device="cuda")
        out[a:b] = turned(s["q"][a:b], pos)
        at = torch.tensor(table[q], device="cuda")[pos // c["page"]]
        k[0, at, :, pos % c["page"]] = turned(s["kn"][a:b], pos)
        v[0, at, :, pos % c["page"]] = s["vn"][a:b].double()
    return [out, k, v]


def _exact_attention(c, s):
    out = torch.empty_like(s["q"], dtype=torch.float64)
    begin, seqs, lengths = (s[x].tolist() for x in ("begin", "seqs", "lengths"))
    group = c["heads"] // c["kv"]
    for e, q in enumerate(seqs):
        a, b, length = begin[e], begin[e + 1], lengths[q]
        t = torch.arange(length, device="cuda")
        at = s["table"][q].long()[t // c["page"]]
        t, at = t[at >= 0], at[at >= 0]
        pos = torch.arange(length - (b - a), length, device="cuda")[:, None]
        hidden = t > pos
        if c["window"]:
            hidden |= (t <= pos - c["window"]) & (t >= c["sinks"])
        for h in range(c["heads"]):
            k, v = (s[x][0, at, h // group, t % c["page"]].double() for x in ("k", "v"))
            w = (s["q"][a:b, h].double() @ k.T) * s["scale"]
            out[a:b, h] = torch.softmax(w.masked_fill(hidden, -math.inf), 1) @ v
    return out


def _exact_move(c, s):
    page = c["page"]
    src, dst, table, lengths, refs = (s[x].tolist() for x in ("src", "dst", "table", "lengths", "refs"))
    k, v = s["k"].double(), s["v"].double()
    free = iter([p for p, r in enumerate(refs) if r == 0])
    before = [list(r) for r in table]
    moves = []
    for i, (a, b) in enumerate(zip(src, dst)):
        if c["kind"] == "fork":
            prefix, keep = lengths[a], []
        else:
            prefix, keep = int(s["prefix"][i]), s["keep"][int(s["begin"][i]):int(s["begin"][i + 1])].tolist()
        tokens = list(range(prefix // page * page, prefix)) + keep
        row = before[a][:prefix // page]
        for p in row:
            refs[p] += 1
        for x in range(0, len(tokens), page):
            p = next(free)
            refs[p] = 1
            row.append(p)
            moves += [(before[a][t // page], t % page, p, y) for y, t in enumerate(tokens[x:x + page])]
        for p in before[b]:
            if p >= 0:
                refs[p] -= 1
        table[b] = row + [-1] * (len(before[b]) - len(row))
        lengths[b] = prefix + len(keep)
    if moves:
        m = torch.tensor(moves, device="cuda").T
        for pool in (k, v):
            pool[:, m[2], :, m[3]] = pool[:, m[0], :, m[1]]
    return [_dev(table), _dev(lengths), _dev(refs), k, v]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, s)
    return _exact_attention(case, s) if case["kind"] in ("decode", "prompt") else _exact_move(case, s)
