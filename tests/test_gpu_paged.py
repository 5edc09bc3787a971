"""GPU tests of the paged key-value cache and the operators on it against plain forms in
64 bits (tests/paged_ref.py).

Bars.
 - Bookkeeping (tables, lengths, counts) and copied rows: exact.
 - Attention: |out - exact| <= 1e-5 * bound (paged_ref.attend).  A score is a sum of at
   most 512 products in at most 48 sequential additions of the matrix cores (three
   parts, 32 elements at a time, each rounded down by at most 2^-23) or 14 of the vector
   unit: 48 * 2^-23 = 5.8e-6 of its sum |q k|.  A weighted sum of up to 8192 tokens is at
   most 128 additions (64 tokens at a time): 128 * 2^-24 = 7.7e-6 of its sum w |v|, the
   exponential's 2^-22 and a product's rounding on top.
 - Rotations: the angle is within 2^-25 turns (1.9e-7), sine and cosine within 2^-22, two
   products and a sum round by 2^-24 each: below 6e-7 (|x| + |y|) gain.  The cache's type
   adds half a step (eps / 2), and for F16 2^-25 where it is subnormal."""
import itertools

import numpy as np
import pytest
import torch

from conftest import announce
from paged_ref import Model, attend

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *size, scale=1.0):
    return torch.randn(*size, generator=g) * scale


@pytest.fixture()
def run(g4, ctx):
    """The context on torch's stream of the test."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ctx.set_stream(stream.cuda_stream)
        yield ctx
        stream.synchronize()
    ctx.set_stream(None)


def filled(g4, ctx, seed, typ, layers, kv, hs, page, lengths, spare=4, slots=None, garbage=float("nan")):
    """A cache whose sequence s has lengths[s] random tokens in pages of no order; rows of
    no token hold `garbage`."""
    g = gen(seed)
    need = sum(-(-n // page) for n in lengths)
    pages, slots = need + spare, slots or len(lengths)
    per = max(1, max(-(-n // page) for n in lengths)) + 2
    cache = g4.KvCache.create(ctx, layers, kv, hs, page, pages, slots, per, DT[typ])
    k, v = (torch.full((layers, pages, kv, page, hs), garbage).to(DT[typ]) for _ in range(2))
    order = torch.randperm(pages, generator=g).tolist()
    table = np.full((slots, per), -1, np.int32)
    refs = np.zeros(pages, np.int32)
    for s, n in enumerate(lengths):
        for j in range(-(-n // page)):
            p = order.pop()
            table[s, j], refs[p] = p, 1
            m = min(page, n - j * page)
            for pool, mean in ((k, 0.3), (v, 0.2)):
                pool[:, p, :, :m] = (normal(g, layers, kv, m, hs) + mean).to(DT[typ])
    cache.k.copy_(k)
    cache.v.copy_(v)
    cache.table.copy_(torch.from_numpy(table))
    cache.refs.copy_(torch.from_numpy(refs))
    cache.lengths[:len(lengths)] = i32(lengths)
    return cache


def check_rows(out, places, model, layer, q, scale, window, sinks):
    """out[r] against the exact row for every (r, sequence, position); other rows are the caller's."""
    for r, seq, pos in places:
        o, b = attend(model, layer, q[r].cpu(), seq, pos, scale, window, sinks)
        err = (out[r].cpu().double() - o).abs()
        assert bool((err <= 1e-5 * b).all()), "row %d (sequence %d at %d): %g over %g" % (
            r, seq, pos, float(err.max()), float((1e-5 * b).min()))


# ------------------------------------------------------------------ decode ---

DECODE = [
    # type, heads, kv, head size, page, lengths, window, sinks
    ("bf16", 16, 8, 256, 16, [1000, 1, 17, 333], 0, 0),
    ("f16", 8, 1, 128, 32, [2049, 31, 32, 33], 0, 0),
    ("f32", 4, 2, 64, 16, [5, 700, 16], 0, 0),
    ("bf16", 8, 1, 512, 16, [900, 2], 100, 4),
    ("f16", 6, 2, 80, 64, [300, 65, 64], 0, 0),
    ("bf16", 3, 3, 96, 128, [129, 400], 50, 0),
    ("f32", 12, 4, 192, 256, [1025], 256, 300),
    ("bf16", 10, 2, 8, 16, [47], 0, 0),
    ("f16", 32, 2, 256, 16, [777, 20], 512, 17),
    ("f32", 24, 1, 512, 32, [100], 0, 0),
    ("bf16", 16, 8, 256, 16, [8192], 0, 0),
]


@pytest.mark.parametrize("typ,heads,kv,hs,page,lengths,window,sinks", DECODE, ids=[str(c) for c in DECODE])
def test_decode_attention(g4, run, typ, heads, kv, hs, page, lengths, window, sinks):
    announce("decode %s %d/%d/%d page %d %s window %d+%d" % (typ, heads, kv, hs, page, lengths, window, sinks))
    cache = filled(g4, run, 7 + hs, typ, 2, kv, hs, page, lengths)
    seqs = list(range(len(lengths)))[::-1] + [0]  # in another order, one of them twice
    g = gen(3)
    q = normal(g, len(seqs), heads, hs, scale=2.0).cuda()
    out = torch.full_like(q, float("nan"))
    g4.paged_attention_dev(run, cache, 1, q, out, heads, i32(seqs), hs ** -0.5, window, sinks)
    torch.cuda.synchronize()
    check_rows(out, [(r, s, lengths[s] - 1) for r, s in enumerate(seqs)], Model(cache), 1, q, hs ** -0.5, window, sinks)


def test_decode_one_token_is_its_value(g4, run):
    announce("decode, one token")
    cache = filled(g4, run, 5, "f16", 1, 2, 128, 16, [1, 1])
    q = torch.randn(2, 8, 128, device="cuda")
    out = torch.empty_like(q)
    g4.paged_attention_dev(run, cache, 0, q, out, 8, i32([1, 0]), 1.0)
    m = Model(cache)
    for r, s in ((0, 1), (1, 0)):
        v = m.rows(0, s, 1)[1][0].float()
        assert torch.equal(out[r].cpu(), v.repeat_interleave(4, 0))


def test_decode_of_what_is_not_there(g4, run):
    """Empty sequences, sequences out of range, holes and pages out of range: zeros, or
    what the tokens that are there give."""
    announce("decode, empty rows and missing pages")
    lengths = [0, 100, 100, 40]
    cache = filled(g4, run, 6, "bf16", 1, 2, 64, 16, lengths)
    cache.table[1, 2] = -1
    cache.table[1, 3] = cache.n_pages  # one behind the last
    cache.table[1, 4] = 0x7FFFFFFF
    cache.table[2, :] = -1
    model = Model(cache)
    q = torch.randn(6, 4, 64, device="cuda")
    for window, sinks in ((0, 0), (20, 3), (1, 0), (0x7FFFFFFF, 0x7FFFFFFF)):
        out = torch.full_like(q, float("nan"))
        g4.paged_attention_dev(run, cache, 0, q, out, 4, i32([0, 1, 2, 3, -1, 4]), 0.5, window, sinks)
        torch.cuda.synchronize()
        for r in (0, 2, 4, 5):
            assert bool((out[r] == 0).all()), r
        check_rows(out, [(1, 1, 99), (3, 3, 39)], model, 0, q, 0.5, window, sinks)


def test_decode_infinite_and_nan_values(g4, run):
    """What is not finite behaves as in the formula: a score of -infinity weighs nothing,
    one of NaN makes the row NaN, an infinite value stays infinite."""
    announce("decode, infinities and NaN among the seen")
    cache = filled(g4, run, 8, "bf16", 1, 1, 64, 16, [40, 40, 40])
    q = torch.ones(3, 2, 64, device="cuda")
    t = cache.table.cpu()
    cache.k[0, int(t[0, 0]), 0, 3, 5] = -float("inf")
    cache.k[0, int(t[1, 1]), 0, 2, 5] = float("nan")
    cache.v[0, int(t[2, 1]), 0, 7, 9] = float("inf")
    out = torch.zeros_like(q)
    g4.paged_attention_dev(run, cache, 0, q, out, 2, i32([0, 1, 2]), 0.1)
    torch.cuda.synchronize()
    m = Model(cache)
    k, v, _ = m.rows(0, 0, 40)
    w = torch.softmax(k[:, 0] @ torch.ones(64, dtype=torch.float64) * 0.1, 0)
    # the bar above: sum |q k| is about 64 * 0.9 * 0.1, so 1e-5 (1 + 2 * 5.8) sum w |v|
    assert torch.allclose(out[0, 0].cpu().double(), w @ v[:, 0], rtol=0, atol=1.3e-4)
    assert bool(torch.isnan(out[1]).all())
    assert bool((out[2, :, 9] == float("inf")).all()) and bool(torch.isfinite(out[2, :, :9]).all())


def test_decode_large_and_far_scores(g4, run):
    """Scores thousands apart: the weight is one token's, wherever it stands."""
    announce("decode, far scores")
    n = 500
    cache = filled(g4, run, 9, "f32", 1, 1, 128, 32, [n])
    model = Model(cache)
    k, v, _ = model.rows(0, 0, n)
    for at in (0, 250, 499):
        q = (k[at, 0] * 60.0).float().reshape(1, 1, 128).cuda()
        out = torch.empty_like(q)
        g4.paged_attention_dev(run, cache, 0, q, out, 1, i32([0]), 1.0)
        best = int((k[:, 0] @ k[at, 0]).argmax())
        assert torch.equal(out.cpu().reshape(-1), v[best, 0].float())


# ------------------------------------------------------------------ prompt ---

PROMPT = [
    # type, heads, kv, head size, page, lengths, rows, window, sinks
    ("bf16", 16, 8, 256, 16, [300], [300], 0, 0),
    ("f16", 8, 2, 256, 16, [257], [257], 100, 0),
    ("bf16", 4, 2, 128, 32, [500, 64, 1, 130], [77, 64, 1, 129], 0, 0),
    ("f16", 16, 4, 128, 16, [700, 333], [65, 200], 128, 16),
    ("f32", 4, 2, 64, 16, [150, 20], [150, 3], 0, 0),
    ("bf16", 8, 1, 512, 64, [200], [130], 0, 0),
    ("f16", 6, 2, 80, 16, [100, 90, 33], [33, 0, 33], 20, 2),
    ("f32", 3, 1, 192, 256, [600], [64], 300, 1),
    ("bf16", 10, 2, 8, 16, [70], [70], 0, 0),
    ("bf16", 16, 8, 256, 16, [2000, 1500, 40], [5, 5, 5], 0, 0),
    ("f32", 8, 1, 512, 32, [140], [33], 64, 8),
    ("f16", 4, 4, 512, 128, [300], [300], 1, 3),
    ("bf16", 24, 1, 96, 16, [100, 61], [50, 61], 0, 0),
]


@pytest.mark.parametrize("typ,heads,kv,hs,page,lengths,rows,window,sinks", PROMPT, ids=[str(c) for c in PROMPT])
def test_prompt_attention(g4, run, typ, heads, kv, hs, page, lengths, rows, window, sinks):
    announce("prompt %s %d/%d/%d page %d %s rows %s window %d+%d" % (typ, heads, kv, hs, page, lengths, rows, window,
                                                                     sinks))
    cache = filled(g4, run, 11 + hs, typ, 2, kv, hs, page, lengths)
    seqs = list(range(len(lengths)))[::-1]
    begin = np.concatenate([[2], 2 + np.cumsum([rows[s] for s in seqs])])  # two rows before, three behind
    total = int(begin[-1]) + 3
    q = normal(gen(4), total, heads, hs, scale=2.0).cuda()
    out = torch.full_like(q, -7.0)
    g4.paged_prompt_dev(run, cache, 1, q, out, heads, i32(seqs), i32(begin), total, hs ** -0.5, window, sinks)
    torch.cuda.synchronize()
    assert bool((out[:2] == -7).all()) and bool((out[total - 3:] == -7).all())
    places = [(int(begin[i]) + j, s, lengths[s] - rows[s] + j) for i, s in enumerate(seqs) for j in range(rows[s])]
    check_rows(out, places, Model(cache), 1, q, hs ** -0.5, window, sinks)


def test_prompt_rows_that_see_nothing(g4, run):
    """More rows than the sequence has tokens, sequences out of range, missing pages."""
    announce("prompt, rows that see nothing")
    lengths = [40, 90, 70]
    cache = filled(g4, run, 12, "bf16", 1, 2, 128, 16, lengths)
    cache.table[1, :3] = -1
    cache.table[2, 4] = cache.n_pages + 5
    model = Model(cache)
    begin = [0, 50, 140, 210, 215]
    q = torch.randn(215, 4, 128, device="cuda")
    out = torch.full_like(q, float("nan"))
    g4.paged_prompt_dev(run, cache, 0, q, out, 4, i32([0, 1, 2, 77]), i32(begin), 215, 0.3)
    torch.cuda.synchronize()
    assert bool((out[:10] == 0).all())          # positions before the first token
    assert bool((out[50:50 + 48] == 0).all())   # only tokens whose pages are gone
    assert bool((out[210:] == 0).all())
    places = [(10 + j, 0, j) for j in range(0, 40, 3)] + [(50 + p, 1, p) for p in range(48, 90, 5)]
    check_rows(out, places + [(140 + p, 2, p) for p in range(0, 70, 7)], model, 0, q, 0.3, 0, 0)


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
def test_prompt_infinite_and_nan_values(g4, run, typ):
    """A key of -infinity, a NaN key, an infinite value and a NaN query each reach the rows
    that see them, and no others."""
    announce("prompt, infinities and NaN among the seen, " + typ)
    n = 100
    cache = filled(g4, run, 13, typ, 1, 1, 128, 16, [n, n, n, n])
    t = cache.table.cpu()
    cache.k[0, int(t[0, 0]), 0, 3, 5] = -float("inf")
    cache.k[0, int(t[1, 2]), 0, 2, 5] = float("nan")    # token 34
    cache.v[0, int(t[2, 3]), 0, 7, 9] = float("inf")    # token 55
    q = (torch.rand(4 * n, 2, 128, generator=gen(1)) + 0.1).cuda()
    q[3 * n + 41, 1, 7] = float("nan")
    out = torch.zeros_like(q)
    begin = [i * n for i in range(5)]
    g4.paged_prompt_dev(run, cache, 0, q, out, 2, i32(range(4)), i32(begin), 4 * n, 0.1)
    torch.cuda.synchronize()
    k, v, _ = Model(cache).rows(0, 0, n)
    for pos in (3, 50, 99):  # the row at 3 sees it among four tokens
        for h in range(2):
            w = torch.softmax(k[:pos + 1, 0] @ q[pos, h].cpu().double() * 0.1, 0)
            # the bar above: sum |q k| is about 128 * 0.6 * 0.9 * 0.1, so 1e-5 (1 + 2 * 6.9) sum w |v|
            assert torch.allclose(out[pos, h].cpu().double(), w @ v[:pos + 1, 0], rtol=0, atol=1.5e-4)
    assert bool(torch.isfinite(out[:n]).all())
    assert bool(torch.isfinite(out[n:n + 34]).all()) and bool(torch.isnan(out[n + 34:2 * n]).all())
    o = out[2 * n:3 * n]
    assert bool(torch.isfinite(o[:55]).all()) and bool((o[55:, :, 9] == float("inf")).all())
    assert bool(torch.isfinite(o[55:, :, :9]).all()) and bool(torch.isfinite(o[55:, :, 10:]).all())
    bad = torch.isnan(out[3 * n:]).all(-1)
    assert bad.sum() == 1 and bool(bad[41, 1])


def test_prompt_of_single_rows_is_decode(g4, run):
    announce("prompt of single rows against decode")
    lengths = [400, 33, 1000]
    cache = filled(g4, run, 14, "bf16", 1, 2, 128, 16, lengths)
    q = torch.randn(3, 8, 128, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(q)
    g4.paged_attention_dev(run, cache, 0, q, a, 8, i32([0, 1, 2]), 0.2, 300, 5)
    g4.paged_prompt_dev(run, cache, 0, q, b, 8, i32([0, 1, 2]), i32([0, 1, 2, 3]), 3, 0.2, 300, 5)
    torch.cuda.synchronize()
    m = Model(cache)
    for out in (a, b):
        check_rows(out, [(r, r, lengths[r] - 1) for r in range(3)], m, 0, q, 0.2, 300, 5)


# ------------------------------------------------------------------ rotary ---

def turned(x, pos, freqs, gain, pairs):
    """x [..., heads, hs] at positions pos [...] in 64 bits, and what bounds its error."""
    x = x.double()
    half = freqs.numel()
    i = torch.arange(half)
    i, j = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    ang = pos.double()[:, None, None] * freqs
    a, b = x[..., i], x[..., j]
    out, size = x.clone(), x.abs() * 0
    out[..., i], out[..., j] = gain * (a * ang.cos() - b * ang.sin()), gain * (b * ang.cos() + a * ang.sin())
    size[..., i] = size[..., j] = gain * (a.abs() + b.abs())
    return out, 6e-7 * size


ROPE = [
    # heads, head size, rot, pairs, positions up to, rows
    (16, 256, 256, False, 30000, 5),
    (4, 128, 64, True, 1 << 20, 33),
    (3, 80, 20, False, 5000, 7),
    (1, 96, 96, True, 100, 1),
    (2, 64, 2, False, 1000, 3),
    (5, 512, 128, True, 1 << 27, 2),
    (2, 1026, 1024, False, 4000, 3),
    (1, 10, 6, True, 50, 4),
    (2, 40, 0, False, 50, 2),
]


@pytest.mark.parametrize("heads,hs,rot,pairs,far,rows", ROPE, ids=[str(c) for c in ROPE])
def test_rope(g4, run, heads, hs, rot, pairs, far, rows):
    announce("rope %d x %d rot %d pairs %s far %d rows %d" % (heads, hs, rot, pairs, far, rows))
    g = gen(20 + rot)
    x = normal(g, rows, heads, hs)
    pos = torch.randint(0, far, (rows,), generator=g, dtype=torch.int32)
    pos[0] = far - 1
    freqs = torch.tensor([10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
    rope = g4.Rope(freqs.cuda(), g4.ROPE_PAIRS if pairs else g4.ROPE_HALF, 1.25)
    exact, tol = turned(x, pos, freqs, 1.25, pairs)
    d = x.cuda()
    out = torch.full_like(d, float("nan"))
    g4.rope_dev(run, rope, d, out, rows, heads, hs, pos.cuda())
    shifted = torch.zeros(x.numel() + 1, device="cuda")[1:].view_as(x)  # not 16-byte aligned
    shifted.copy_(d)
    g4.rope_dev(run, rope, shifted, shifted, rows, heads, hs, pos.cuda())
    g4.rope_dev(run, rope, d, d, rows, heads, hs, pos.cuda())  # in place
    torch.cuda.synchronize()
    assert torch.equal(d, out)
    for o in (out, shifted):
        err = (o.cpu().double() - exact).abs()
        assert bool((err <= tol).all()), float((err - tol).max())


WRITE = [
    # type, heads, kv, head size, rot, pairs, page, lengths, rows
    ("bf16", 16, 8, 256, 256, False, 16, [300, 17, 16], [1, 1, 1]),
    ("f16", 8, 2, 128, 64, True, 32, [100, 65, 900], [40, 0, 33]),
    ("f32", 4, 4, 64, 32, False, 16, [20], [20]),
    ("bf16", 6, 3, 80, 20, False, 16, [50, 33], [3, 33]),
    ("f16", 4, 1, 8, 8, True, 16, [70], [70]),
    ("f16", 0, 2, 512, 0, False, 256, [257], [257]),  # no queries, nothing turned
]


@pytest.mark.parametrize("typ,heads,kv,hs,rot,pairs,page,lengths,rows", WRITE, ids=[str(c) for c in WRITE])
def test_rope_write(g4, run, typ, heads, kv, hs, rot, pairs, page, lengths, rows):
    announce("write %s %d/%d/%d rot %d pairs %s page %d %s rows %s" % (typ, heads, kv, hs, rot, pairs, page, lengths,
                                                                       rows))
    cache = filled(g4, run, 30 + hs, typ, 3, kv, hs, page, lengths, garbage=-3.0)
    model = Model(cache)
    seqs = list(range(len(lengths)))[::-1]
    single = all(r == 1 for r in rows)
    begin = np.concatenate([[0], np.cumsum([rows[s] for s in seqs])]) + (0 if single else 1)
    total = int(begin[-1]) + (0 if single else 2)
    g = gen(31)
    q, k, v = normal(g, total, max(1, heads), hs), normal(g, total, kv, hs), normal(g, total, kv, hs)
    k[0] = 1e-7  # subnormal in F16
    freqs = torch.tensor([10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
    rope = g4.Rope(freqs.cuda(), g4.ROPE_PAIRS if pairs else g4.ROPE_HALF, 1.1) if rot else None
    qd = q.cuda() if heads else None
    out = torch.full_like(qd, -7.0) if heads else None
    g4.kv_rope_write_dev(run, cache, 1, qd, out, k.cuda(), v.cuda(), heads, rope, i32(seqs),
                         None if single else i32(begin), total)
    torch.cuda.synchronize()
    assert int(cache.status_word.cpu()) == 0
    places = [(int(begin[i]) + j, s, lengths[s] - rows[s] + j) for i, s in enumerate(seqs) for j in range(rows[s])]
    at = torch.tensor([p[0] for p in places])
    pos = torch.tensor([p[2] for p in places])
    if heads:
        exact, tol = turned(q[at], pos, freqs, 1.1, pairs)
        assert bool(((out[at.cuda()].cpu().double() - exact).abs() <= tol).all())
        rest = [r for r in range(total) if r not in set(at.tolist())]
        assert bool((out[rest] == -7).all())
    exact, tol = turned(k[at], pos, freqs, 1.1, pairs)
    new_k = cache.k.cpu()
    for i, (r, s, p) in enumerate(places):
        page_at = model.table[s, p // page]
        got = new_k[1, page_at, :, p % page].double()
        step = 0.0 if typ == "f32" else torch.finfo(DT[typ]).eps / 2
        err = (got - exact[i]).abs()
        assert bool((err <= tol[i] + step * exact[i].abs() * (1 + 1e-6) + (2.0 ** -25 if typ == "f16" else 0)).all())
        model.write(1, s, p, got.to(DT[typ]), v[r])  # V is rounded to nearest, exactly
    model.same_contents(cache)
    model.same_books(cache)


def test_write_refuses_shared_and_missing_pages(g4, run):
    announce("write to shared and missing pages")
    cache = filled(g4, run, 33, "bf16", 1, 1, 64, 16, [40, 40, 40], garbage=0.0)
    cache.refs[int(cache.table[0, 2])] = 2
    cache.table[1, 2] = -1
    before = Model(cache)
    k = torch.ones(1, 1, 64, device="cuda")
    for s in (0, 1, 3, -1):
        g4.kv_rope_write_dev(run, cache, 0, None, None, k, k, 0, None, i32([s]), None, 1)
        with pytest.raises(g4.IndexOutOfBoundsException):
            g4.kv_status(run, cache)
        g4.kv_status(run, cache)  # cleared
        before.same_contents(cache)
    # more rows than tokens: those before the first token are not written
    k = torch.ones(45, 1, 64, device="cuda")
    g4.kv_rope_write_dev(run, cache, 0, None, None, k, k, 0, None, i32([2]), i32([0, 45]), 45)
    with pytest.raises(g4.IndexOutOfBoundsException):
        g4.kv_status(run, cache)


# ------------------------------------------------------------------- pages ---

def test_extend(g4, run):
    announce("extend")
    cache = filled(g4, run, 40, "bf16", 1, 1, 64, 16, [0, 15, 16, 33, 0], spare=40)
    model = Model(cache)
    for seqs, counts in (([1, 0, 3], [1, 40, 0]), ([2, 4, 1, 0], [1, 0, 1, 30]), ([4], [1])):
        g4.kv_extend_dev(run, cache, i32(seqs), i32(counts))
        model.extend(seqs, counts)
        torch.cuda.synchronize()
        model.same_books(cache)


def test_fork(g4, run):
    """Whole sequences, shorter ones, on themselves, in a circle, onto used ones."""
    announce("fork")
    cache = filled(g4, run, 41, "f16", 3, 2, 80, 16, [50, 16, 33, 1, 7], spare=12, slots=9)
    model = Model(cache)
    for src, dst, lengths in (([0, 0, 2], [5, 6, 7], None), ([5, 6], [6, 5], None), ([0, 1], [0, 1], [20, 16]),
                              ([0, 1, 2, 3], [1, 2, 3, 0], [17, 3, 32, 0]), ([7], [7], None), ([2, 2], [2, 8], None),
                              ([6], [3], [48])):
        g4.kv_fork_dev(run, cache, i32(src), i32(dst), None if lengths is None else i32(lengths))
        model.move(src, dst, lengths, None)
        torch.cuda.synchronize()
        model.same_books(cache)
        model.same_contents(cache)


@pytest.mark.parametrize("typ,hs,page", [("bf16", 64, 16), ("f32", 72, 32), ("f16", 512, 64)])
def test_compact(g4, run, typ, hs, page):
    announce("compact %s %d page %d" % (typ, hs, page))
    cache = filled(g4, run, 42, typ, 2, 3, hs, page, [200, 70, 16, 130, 0], spare=30, slots=8)
    model = Model(cache)
    rng = np.random.default_rng(1)
    calls = [([0, 1], [5, 6], None, [range(0, 200, 3), [69, 0, 0, 5]]),
             ([0, 3], [3, 0], [page, 0], [range(60, 180, 2), []]),
             ([1, 2, 4], [1, 7, 4], [70, 5, 0], [[], [15, 3], []]),
             ([5], [5], [33], [sorted(rng.choice(60, 20, replace=False))])]
    for src, dst, prefix, keep in calls:
        begin = np.concatenate([[0], np.cumsum([len(x) for x in keep])])
        flat = i32(itertools.chain(*keep))
        g4.kv_compact_dev(run, cache, i32(src), i32(dst), None if prefix is None else i32(prefix), flat, i32(begin))
        model.move(src, dst, prefix, keep)
        torch.cuda.synchronize()
        model.same_books(cache)
        model.same_contents(cache)


def test_free_and_trim(g4, run):
    announce("free and trim")
    cache = filled(g4, run, 43, "bf16", 1, 1, 64, 16, [200, 64, 65, 5, 0], spare=4, slots=6)
    model = Model(cache)
    g4.kv_fork_dev(run, cache, i32([0]), i32([5]))
    model.move([0], [5], None, None)
    for seqs, window, sinks in (([0, 1, 2, 3, 4], 30, 20), ([0], 1, 0), ([5, 2], 100000, 0), ([5], 5, 100000)):
        g4.kv_trim_dev(run, cache, i32(seqs), window, sinks)
        model.release(seqs, -(-sinks // 16) * 16, window)
        torch.cuda.synchronize()
        model.same_books(cache)
    for seqs in ([5, 4], [0, 1, 2, 3]):
        g4.kv_free_dev(run, cache, i32(seqs))
        model.release(seqs)
        torch.cuda.synchronize()
        model.same_books(cache)
    assert bool((cache.refs == 0).all()) and bool((cache.table == -1).all())
    g4.kv_extend_dev(run, cache, i32([3]), i32([70]))
    model.extend([3], [70])
    torch.cuda.synchronize()
    model.same_books(cache)
    g4.kv_init_dev(run, cache)
    torch.cuda.synchronize()
    assert bool((cache.refs == 0).all()) and bool((cache.table == -1).all()) and bool((cache.lengths == 0).all())


def test_calls_that_cannot_be_done_change_nothing(g4, run):
    announce("bookkeeping calls that cannot be done")
    cache = filled(g4, run, 44, "bf16", 1, 1, 64, 16, [40, 33, 16], spare=2, slots=4)
    cache.table[1, 0] = -1  # a hole
    model = Model(cache)
    e, nothing = i32([]), g4.IndexOutOfBoundsException
    calls = [
        (g4.OutOfMemoryError, lambda: g4.kv_extend_dev(run, cache, i32([0, 1]), i32([30, 16]))),
        (nothing, lambda: g4.kv_extend_dev(run, cache, i32([0, 4]), i32([1, 1]))),
        (nothing, lambda: g4.kv_extend_dev(run, cache, i32([-1]), i32([1]))),
        (nothing, lambda: g4.kv_extend_dev(run, cache, i32([0, 0]), i32([1, 1]))),
        (nothing, lambda: g4.kv_extend_dev(run, cache, i32([0]), i32([-1]))),
        (nothing, lambda: g4.kv_extend_dev(run, cache, i32([0]), i32([0x7FFFFFFF]))),
        (g4.OutOfMemoryError, lambda: g4.kv_fork_dev(run, cache, i32([0, 0, 0]), i32([1, 2, 3]))),
        (nothing, lambda: g4.kv_fork_dev(run, cache, i32([0, 0]), i32([3, 3]))),
        (nothing, lambda: g4.kv_fork_dev(run, cache, i32([9]), i32([3]))),
        (nothing, lambda: g4.kv_fork_dev(run, cache, i32([0]), i32([-5]))),
        (nothing, lambda: g4.kv_fork_dev(run, cache, i32([0]), i32([3]), i32([41]))),
        (nothing, lambda: g4.kv_fork_dev(run, cache, i32([0]), i32([3]), i32([-1]))),
        (nothing, lambda: g4.kv_fork_dev(run, cache, i32([1]), i32([3]), i32([10]))),  # ends in the hole
        (nothing, lambda: g4.kv_compact_dev(run, cache, i32([0]), i32([3]), None, i32([40]), i32([0, 1]))),
        (nothing, lambda: g4.kv_compact_dev(run, cache, i32([0]), i32([3]), None, i32([-1]), i32([0, 1]))),
        (nothing, lambda: g4.kv_compact_dev(run, cache, i32([1]), i32([3]), None, i32([20, 2]), i32([0, 2]))),
        (nothing, lambda: g4.kv_compact_dev(run, cache, i32([0]), i32([3]), None, i32([1, 2]), i32([0, 3]))),
        (nothing, lambda: g4.kv_compact_dev(run, cache, i32([0, 2]), i32([3, 2]), None, i32([1, 2]), i32([0, 2, 1]))),
        (nothing, lambda: g4.kv_compact_dev(run, cache, i32([0]), i32([3]), None, i32([1, 2]), i32([1, 2]))),
        (g4.OutOfMemoryError,
         lambda: g4.kv_compact_dev(run, cache, i32([0]), i32([3]), None, i32([1] * 33), i32([0, 33]))),
        (nothing, lambda: g4.kv_free_dev(run, cache, i32([0, 0]))),
        (nothing, lambda: g4.kv_trim_dev(run, cache, i32([0, 7]), 1)),
    ]
    q = torch.ones(1, 1, 64, device="cuda")
    for kind, call in calls:
        call()
        # while the status is set nothing runs
        g4.kv_extend_dev(run, cache, i32([0]), i32([1]))
        g4.kv_free_dev(run, cache, i32([0]))
        g4.kv_fork_dev(run, cache, i32([0]), i32([0]), i32([1]))
        g4.kv_rope_write_dev(run, cache, 0, None, None, q, q, 0, None, i32([0]), None, 1)
        out = torch.full_like(q, -7.0)
        g4.paged_attention_dev(run, cache, 0, q, out, 1, i32([0]), 1.0)
        g4.paged_prompt_dev(run, cache, 0, q, out, 1, i32([0]), i32([0, 1]), 1, 1.0)
        torch.cuda.synchronize()
        assert bool((out == -7).all())
        with pytest.raises(kind):
            g4.kv_status(run, cache)
        model.same_books(cache)
        model.same_contents(cache)
    # empty lists are nothing to do
    g4.kv_extend_dev(run, cache, e, e)
    g4.kv_fork_dev(run, cache, e, e)
    g4.kv_compact_dev(run, cache, e, e, None, e, i32([0]))
    g4.kv_free_dev(run, cache, e)
    g4.kv_trim_dev(run, cache, e, 1)
    g4.paged_attention_dev(run, cache, 0, q, q.clone(), 1, e)
    g4.kv_status(run, cache)
    model.same_books(cache)


def test_many_sequences_and_pages(g4, run):
    """The largest list, pages that a workgroup counts in several rounds."""
    announce("1024 sequences, 20000 pages")
    cache = g4.KvCache.create(run, 1, 1, 8, 16, 20000, 1024, 24, torch.float16)
    model = Model(cache)
    rng = np.random.default_rng(3)
    every = list(range(1024))
    counts = rng.integers(0, 200, 1024).tolist()
    g4.kv_extend_dev(run, cache, i32(every), i32(counts))
    model.extend(every, counts)
    order = rng.permutation(1024).tolist()
    g4.kv_free_dev(run, cache, i32(order[:400]))
    model.release(order[:400])
    src, dst = rng.choice(order[400:], 1024).tolist(), rng.permutation(1024).tolist()
    g4.kv_fork_dev(run, cache, i32(src), i32(dst))
    model.move(src, dst, None, None)
    g4.kv_extend_dev(run, cache, i32(order), i32([100] * 1024))
    model.extend(order, [100] * 1024)
    torch.cuda.synchronize()
    model.same_books(cache)


# ---------------------------------------------------------- as they are used ---

def test_a_session(g4, run):
    """Prompts in chunks, beams forked from them, steps with reordered beams under a
    sliding window with trimmed pages, a compacted sequence, the end: every attention
    against 64 bits over what the model of the cache holds."""
    announce("a session")
    heads, kv, hs, page, layers, window, sinks = 8, 2, 128, 16, 2, 48, 5
    cache = g4.KvCache.create(run, layers, kv, hs, page, 60, 6, 12, torch.bfloat16)
    model = Model(cache)
    rope = g4.Rope.create(run, hs, layout=g4.ROPE_HALF, scaling=g4.ROPE_SCALE_RAMP, factor=4.0, trained=64.0)
    freqs = rope.freqs.cpu()
    gain = float(g4.rope_freqs(hs, scaling=g4.ROPE_SCALE_RAMP, factor=4.0, trained=64.0)[1])
    g = gen(50)

    def step(seqs, counts, prompt):
        g4.kv_extend_dev(run, cache, i32(seqs), i32(counts))
        model.extend(seqs, counts)
        begin = np.concatenate([[0], np.cumsum(counts)])
        total = int(begin[-1])
        for layer in range(layers):
            q, k, v = normal(g, total, heads, hs), normal(g, total, kv, hs), normal(g, total, kv, hs)
            qo = torch.empty(total, heads, hs, device="cuda")
            g4.kv_rope_write_dev(run, cache, layer, q.cuda(), qo, k.cuda(), v.cuda(), heads, rope, i32(seqs),
                                 i32(begin), total)
            out = torch.empty_like(qo)
            w, f = (window, sinks) if layer else (0, 0)
            if prompt:
                g4.paged_prompt_dev(run, cache, layer, qo, out, heads, i32(seqs), i32(begin), total, hs ** -0.5, w, f)
            else:
                g4.paged_attention_dev(run, cache, layer, qo, out, heads, i32(seqs), hs ** -0.5, w, f)
            torch.cuda.synchronize()
            places = [(int(begin[i]) + j, s, int(model.lengths[s]) - c + j) for i, (s, c) in enumerate(zip(seqs, counts))
                      for j in range(c)]
            exact, tol = turned(q, torch.tensor([p[2] for p in places]), freqs, gain, False)
            assert bool(((qo.cpu().double() - exact).abs() <= tol).all())
            dev_k = cache.k.cpu()
            for r, s, p in places:
                at = model.table[s, p // page]
                model.write(layer, s, p, dev_k[layer, at, :, p % page], v[r])
            check_rows(out, places, model, layer, qo, hs ** -0.5, w, f)
        model.same_books(cache)
        model.same_contents(cache)

    step([0, 1], [37, 20], True)
    step([0, 1], [30, 3], True)
    g4.kv_fork_dev(run, cache, i32([0, 0, 1]), i32([2, 3, 4]))
    model.move([0, 0, 1], [2, 3, 4], None, None)
    step([0, 2, 3, 4], [1] * 4, False)
    g4.kv_fork_dev(run, cache, i32([2, 2, 4]), i32([0, 2, 3]))
    model.move([2, 2, 4], [0, 2, 3], None, None)
    step([3, 2, 0, 4], [1] * 4, False)
    step([3, 1], [4, 9], True)
    g4.kv_compact_dev(run, cache, i32([2]), i32([5]), i32([33]), i32(range(40, 69, 2)), i32([0, 15]))
    model.move([2], [5], [33], [range(40, 69, 2)])
    step([5, 0], [1, 1], False)
    g4.kv_free_dev(run, cache, i32([0, 1, 2, 3, 4]))
    model.release([0, 1, 2, 3, 4])
    step([5, 1], [1, 40], True)
    model.same_books(cache)
    g4.kv_status(run, cache)


def test_a_trimmed_window(g4, run):
    """A stream under a sliding window whose pages are given back as it goes: outputs as
    with all of them, in a pool far smaller than the stream."""
    announce("a trimmed window")
    heads, kv, hs, page, window, sinks = 4, 1, 64, 16, 40, 3
    cache = g4.KvCache.create(run, 1, kv, hs, page, 6, 1, 40, torch.float16)
    g = gen(51)
    ks, vs = [], []
    one = i32([0])
    for n in [20] + [7] * 30 + [1] * 40:
        g4.kv_extend_dev(run, cache, one, i32([n]))
        k, v, q = normal(g, n, kv, hs), normal(g, n, kv, hs), normal(g, n, heads, hs).cuda()
        g4.kv_rope_write_dev(run, cache, 0, None, None, k.cuda(), v.cuda(), 0, None, one, i32([0, n]), n)
        out = torch.empty_like(q)
        g4.paged_prompt_dev(run, cache, 0, q, out, heads, one, i32([0, n]), n, 0.2, window, sinks)
        g4.kv_trim_dev(run, cache, one, window, sinks)
        g4.kv_status(run, cache)
        ks.append(k.half().double())
        vs.append(v.half().double())
        kk, vv = torch.cat(ks), torch.cat(vs)
        for r in (0, n - 1):
            pos = len(kk) - n + r
            t = torch.arange(len(kk))
            see = (t <= pos) & ((t > pos - window) | (t < sinks))
            for h in range(heads):
                x = q[r, h].cpu().double() * 0.2
                w = torch.softmax(kk[see, 0] @ x, 0)
                bound = w @ vv[see, 0].abs() * (1 + 2 * float((kk[see, 0].abs() @ x.abs()).max()))
                assert bool(((out[r, h].cpu().double() - w @ vv[see, 0]).abs() <= 1e-5 * bound).all())
    assert int((cache.refs > 0).sum()) <= 5


def test_a_captured_step_advances(g4, ctx):
    """Extend, write and attend recorded once and replayed: each replay is the next token;
    eager work and synchronisations between them."""
    announce("a captured step")
    heads, kv, hs, page, n = 8, 2, 128, 16, 3
    c2 = g4.Context(0)
    try:
        c2.reserve(64 << 20)
        cache = g4.KvCache.create(c2, 1, kv, hs, page, 40, 4, 16, torch.bfloat16)
        rope = g4.Rope.create(c2, 64, layout=g4.ROPE_PAIRS)
        seqs, ones = i32([2, 0, 1]), i32([1, 1, 1])
        q, k, v = (torch.zeros(n, m, hs, device="cuda") for m in (heads, kv, kv))
        qo, out = torch.empty_like(q), torch.empty_like(q)

        def body():
            g4.kv_extend_dev(c2, cache, seqs, ones)
            g4.kv_rope_write_dev(c2, cache, 0, q, qo, k, v, heads, rope, seqs, None, n)
            g4.paged_attention_dev(c2, cache, 0, qo, out, heads, seqs, 0.1, 30, 2)
            g4.kv_trim_dev(c2, cache, seqs, 31, 2)  # one more, so that the check below finds what the step saw
            g4.kv_fork_dev(c2, cache, seqs[:1], i32_three)

        i32_three = i32([3])
        torch.cuda.synchronize()
        g4.kv_extend_dev(c2, cache, seqs, i32([14, 3, 20]))
        g4.kv_rope_write_dev(c2, cache, 0, None, None, torch.randn(37, kv, hs, device="cuda"),
                             torch.randn(37, kv, hs, device="cuda"), 0, None, seqs, i32([0, 14, 17, 37]), 37)
        c2.sync()
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c2.set_stream(stream.cuda_stream)
            body()
        c2.set_stream(None)
        lengths = {2: 14, 0: 3, 1: 20}
        g = gen(60)
        for i in range(40):
            for t in (q, k, v):
                t.copy_(normal(g, *t.shape))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            model = Model(cache)
            for s in lengths:
                lengths[s] += 1
                assert model.lengths[s] == lengths[s]
            assert model.lengths[3] == lengths[2] and int(cache.status_word.cpu()) == 0
            check_rows(out, [(r, s, lengths[s] - 1) for r, s in enumerate([2, 0, 1])], model, 0, qo, 0.1, 30, 2)
            if i % 5 == 0:  # the same, eagerly
                again = torch.empty_like(out)
                torch.cuda.synchronize()
                g4.paged_attention_dev(c2, cache, 0, qo, again, heads, seqs, 0.1, 30, 2)
                c2.sync()
                assert torch.equal(again, out)
    finally:
        torch.cuda.synchronize()
        c2.close()


def test_results_do_not_depend_on_what_ran_before(g4, run):
    """The same bits on a second run, after other calls used the context's scratch."""
    announce("the same bits twice")
    cache = filled(g4, run, 61, "bf16", 1, 2, 256, 16, [5000, 3, 800])
    q = torch.randn(3, 16, 256, device="cuda")
    p = torch.randn(700, 16, 256, device="cuda")
    seqs, begin = i32([0, 1, 2]), i32([0, 500, 501, 700])
    outs = []
    for i in range(3):
        a, b = torch.empty_like(q), torch.empty_like(p)
        g4.paged_attention_dev(run, cache, 0, q, a, 16, seqs, 0.06)
        g4.paged_prompt_dev(run, cache, 0, p, b, 16, seqs, begin, 700, 0.06)
        other = torch.randn(4000, 16, 256, device="cuda")
        g4.paged_prompt_dev(run, cache, 0, other, torch.empty_like(other), 16, i32([0]), i32([0, 4000]), 4000, 0.06)
        torch.cuda.synchronize()
        outs.append((a, b))
    for a, b in outs[1:]:
        assert torch.equal(a, outs[0][0]) and torch.equal(b, outs[0][1])


# ----------------------------------------------------- calls at their edges ---

def test_write_refuses_a_sequence_named_twice(g4, run):
    """Two rows for one place: neither is written; the other sequences' rows are."""
    announce("a sequence twice")
    cache = filled(g4, run, 70, "f16", 1, 2, 64, 16, [20, 9, 33], garbage=0.0)
    before = Model(cache)
    k = torch.ones(3, 2, 64, device="cuda")
    g4.kv_rope_write_dev(run, cache, 0, None, None, k, k, 0, None, i32([2, 1, 2]), None, 3)
    with pytest.raises(g4.IndexOutOfBoundsException):
        g4.kv_status(run, cache)
    page = int(before.table[2, 2])
    for mine, theirs in ((before.k, cache.k.cpu()), (before.v, cache.v.cpu())):
        assert torch.equal(mine[0, page].view(torch.int16), theirs[0, page].view(torch.int16))
    g4.kv_rope_write_dev(run, cache, 0, None, None, k, k, 0, None, i32([0, 0]), i32([0, 1, 3]), 3)
    with pytest.raises(g4.IndexOutOfBoundsException):
        g4.kv_status(run, cache)


@pytest.mark.parametrize("begin,rows", [([0, 5, 3, 9], 9), ([-1, 2, 4, 9], 9), ([0, 4, 8, 12], 9)], ids=str)
def test_rows_that_do_not_rise(g4, run, begin, rows):
    """Refused on the device: nothing is written, the cache says so."""
    announce("row_begin %s" % begin)
    cache = filled(g4, run, 71, "bf16", 1, 2, 64, 16, [20, 9, 33], garbage=0.0)
    before = Model(cache)
    q = torch.randn(rows, 4, 64, device="cuda")
    out = torch.full_like(q, 7.0)
    k = torch.ones(rows, 2, 64, device="cuda")
    for call in (lambda: g4.paged_prompt_dev(run, cache, 0, q, out, 4, i32([0, 1, 2]), i32(begin), rows, 0.1),
                 lambda: g4.kv_rope_write_dev(run, cache, 0, None, None, k, k, 0, None, i32([0, 1, 2]), i32(begin), rows)):
        call()
        with pytest.raises(g4.IndexOutOfBoundsException):
            g4.kv_status(run, cache)
    assert bool((out == 7.0).all())
    before.same_contents(cache)


@pytest.mark.parametrize("typ,heads,hs", [("f16", 16, 512), ("f32", 8, 512), ("bf16", 3, 64)], ids=str)
def test_the_longest_list(g4, run, typ, heads, hs):
    """1024 entries, sequences named many times, decode and prompt; the prompt's single
    rows against decode of the same."""
    announce("1024 entries, %s, %d heads of %d" % (typ, heads, hs))
    cache = filled(g4, run, 72, typ, 1, 1, hs, 16, [70, 1, 0, 16, 33, 200])
    model = Model(cache)
    order = [int(x) for x in torch.randint(0, 6, (1024,), generator=gen(73))]
    q = normal(gen(74), 1024, heads, hs).cuda()
    out, again = torch.empty_like(q), torch.empty_like(q)
    scale = hs ** -0.5
    g4.paged_attention_dev(run, cache, 0, q, out, heads, i32(order), scale, 40, 3)
    g4.paged_prompt_dev(run, cache, 0, q, again, heads, i32(order), i32(range(1025)), 1024, scale, 40, 3)
    torch.cuda.synchronize()
    rows = list(range(0, 1024, 61)) + [1022, 1023]
    for o in (out, again):
        check_rows(o, [(r, order[r], int(model.lengths[order[r]]) - 1) for r in rows], model, 0, q, scale, 40, 3)
    # the largest bound of a value is 1 sigma * 5 and the mean: rows of both differ by less than twice 1e-5 of it
    assert float((out - again).abs().max()) <= 2e-5 * 10


def test_offsets_beyond_32_bits(g4, run):
    """A cache of 9.7 GB a side: pages behind 4 GB and behind 2^31 elements give the bits of
    the same pages in a small cache."""
    announce("a large cache")
    kv, hs, page, pages, heads = 8, 512, 256, 1160, 16
    big = g4.KvCache.create(run, 2, kv, hs, page, pages, 2, 8, torch.float32)
    small = g4.KvCache.create(run, 2, kv, hs, page, 6, 2, 8, torch.float32)
    assert big.k[0].numel() > 1 << 30 and big.k.numel() > 1 << 31
    g = gen(75)
    far = [pages - 1, pages - 7, pages - 400, pages - 2, 700, pages - 3]
    length = 2 * page + 37
    for i, p in enumerate(far[:3]):
        for a, b in ((small.k, big.k), (small.v, big.v)):
            rows = normal(g, 2, kv, page, hs).cuda()
            a[:, i] = rows
            b[:, p] = rows
    big.refs.fill_(9)  # none is free but the ones below
    for c, ids in ((small, range(6)), (big, far)):
        ids = list(ids)
        c.table[0, :3] = i32(ids[:3])
        c.refs[i32(ids[:3]).long()] = 1
        c.refs[i32(ids[3:]).long()] = 0
        c.lengths[0] = length
    q1, qn = normal(g, 1, heads, hs).cuda(), normal(g, 300, heads, hs).cuda()
    k, v = normal(g, 5, kv, hs).cuda(), normal(g, 5, kv, hs).cuda()
    outs = []
    for c in (small, big):
        o1, on = torch.empty_like(q1), torch.empty_like(qn)
        g4.kv_extend_dev(run, c, i32([0]), i32([5]))
        g4.kv_rope_write_dev(run, c, 1, None, None, k, v, 0, None, i32([0]), i32([0, 5]), 5)
        g4.kv_fork_dev(run, c, i32([0]), i32([1]))
        g4.paged_attention_dev(run, c, 1, q1, o1, heads, i32([1]), 0.04)
        g4.paged_prompt_dev(run, c, 1, qn, on, heads, i32([1]), i32([0, 300]), 300, 0.04)
        assert g4.kv_status(run, c) is None
        outs.append((o1, on))
    assert int(big.table[1, 2]) == min(700, pages - 3) and big.table[1, :2].tolist() == far[:2]
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert torch.equal(big.k[:, 700, :, :42], big.k[:, far[2], :, :42])


def test_two_graphs_share_a_context(g4, ctx):
    """Decode and prompt recorded into two graphs over one workspace, replayed in turn with
    eager calls between, each replay against the eager result."""
    announce("two graphs")
    c2 = g4.Context(0)
    try:
        c2.reserve(128 << 20)
        one = filled(g4, c2, 76, "bf16", 1, 2, 128, 16, [1500, 40, 700])
        two = filled(g4, c2, 77, "f16", 1, 4, 64, 32, [900, 333])
        q, p = normal(gen(78), 3, 8, 128).cuda(), normal(gen(79), 500, 8, 64).cuda()
        a, b = torch.empty_like(q), torch.empty_like(p)
        s1, s2, begin = i32([2, 0, 1]), i32([1, 0]), i32([0, 100, 500])

        def decode(out):
            g4.paged_attention_dev(c2, one, 0, q, out, 8, s1, 0.1, 900, 4)

        def prompt(out):
            g4.paged_prompt_dev(c2, two, 0, p, out, 8, s2, begin, 500, 0.1)

        torch.cuda.synchronize()
        graphs, stream = [], torch.cuda.Stream()
        for body, out in ((decode, a), (prompt, b)):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                c2.set_stream(stream.cuda_stream)
                body(out)
            c2.set_stream(None)
            graphs.append(graph)
        g = gen(80)
        for i in range(6):
            for t in (q, p):
                t.copy_(normal(g, *t.shape))
            a.fill_(float("nan"))
            b.fill_(float("nan"))
            torch.cuda.synchronize()
            for j in (0, 1) if i % 2 else (1, 0, 1):
                graphs[j].replay()
            torch.cuda.synchronize()
            ea, eb = torch.empty_like(a), torch.empty_like(b)
            torch.cuda.synchronize()
            prompt(eb)
            decode(ea)
            c2.sync()
            assert torch.equal(a, ea) and torch.equal(b, eb)
    finally:
        torch.cuda.synchronize()
        c2.close()


@pytest.mark.parametrize("typ,window,sinks", [("f16", 0, 0), ("bf16", 150, 5), ("f32", 0, 0)], ids=str)
def test_more_heads_than_workgroups(g4, run, typ, window, sinks):
    """Decode and prompts with more heads, or query tiles, than the chip takes at once: their
    stretches cross from one to the next, and heads lie in up to three of them."""
    announce("more heads than workgroups, %s" % typ)
    kv, hs = 8, 64
    g = gen(81)
    lengths = [int(x) for x in torch.randint(1, 260, (75,), generator=g)] + [2500, 0, 1]
    cache = filled(g4, run, 82, typ, 1, kv, hs, 16, lengths)
    model = Model(cache)
    order = [int(x) for x in torch.randperm(len(lengths), generator=g)]
    q = normal(g, len(order), 16, hs).cuda()
    out = torch.empty_like(q)
    g4.paged_attention_dev(run, cache, 0, q, out, 16, i32(order), 0.12, window, sinks)
    torch.cuda.synchronize()
    rows = list(range(0, 78, 5)) + [order.index(75), order.index(76), order.index(77)]
    check_rows(out, [(r, order[r], lengths[order[r]] - 1) for r in rows], model, 0, q, 0.12, window, sinks)
    # 64 heads: 24 tokens to a query tile, 8 * (105 + 1 + 9) of them
    p = normal(g, 2720, 64, hs).cuda()
    out = torch.full_like(p, 7.0)
    begin = [0, 2500, 2501, 2709]
    seqs = [75, 77, 0]
    g4.paged_prompt_dev(run, cache, 0, p, out, 64, i32(seqs), i32(begin), 2720, 0.12, window, sinks)
    torch.cuda.synchronize()
    places = [(r, seqs[i], lengths[seqs[i]] - (begin[i + 1] - begin[i]) + r - begin[i]) for i in range(3)
              for r in range(begin[i], begin[i + 1]) if r % 173 == 0 or r in (1, 2499, 2500, 2501, 2708)]
    check_rows(out, [x for x in places if x[2] >= 0], model, 0, p, 0.12, window, sinks)
    for r, _, pos in places:
        assert pos >= 0 or bool((out[r] == 0).all())
    assert bool((out[2709:] == 7.0).all())
