"""GPU tests of how exact attention over a paged cache is, against the formula in 64 bits.

Bars.
 - A relative error e of every product of a score moves the result by at most
   2 e A w|v|, A the largest sum of |scale q k| of a token, w|v| the weighted sum of |v|.
   A score passes n matrix instructions one after the other (of 32 elements of 16 bits a
   part, or of 4 of 32 bits), each of which rounds the sum by at most 2^-23; the
   query's scaling, its parts (2^-22 where there are two) and the exponential make less than
   eight more such steps, and so do the weights, their parts and the sums over the few
   tokens here: e = (n + 8) 2^-23 in bar(), once for the scores and once for the values.
 - What is lost of a query's small elements beside its largest: F16 parts stand on steps of 2^-24
   where the largest is at least 2^14, so an element is off by at most 2^-25 / 2^14 of it."""
import pytest
import torch

from conftest import announce
from paged_ref import Model
from test_gpu_paged import filled, gen, i32, normal, run  # noqa: F401  (run is a fixture)

pytestmark = pytest.mark.gpu


def exact(q, k, v, scale):
    """One row of one head over k, v [tokens, head size] in 64 bits: (result, w|v|, A)."""
    q = q.double()
    w = torch.softmax(k @ q * scale, 0)
    return w @ v, w @ v.abs(), float((k.abs() @ q.abs()).max()) * abs(scale)


def bar(typ, hs, size, a):
    n = hs // 4 if typ == "f32" else -(-hs // 32) * {"f16": 2, "bf16": 3}[typ]
    return (n + 8) * 2.0 ** -23 * (1 + 2 * a) * size


def both(g4, ctx, cache, q, heads, seqs, lengths, scale):
    """Decode's row of every sequence, and the prompt of its last rows ([(sequence, position, out row)])."""
    out = torch.empty_like(q)
    n = len(seqs)
    g4.paged_attention_dev(ctx, cache, 0, q[:n], out[:n], heads, i32(seqs), scale)
    places = [(s, lengths[s] - 1, r) for r, s in enumerate(seqs)]
    rows = (q.shape[0] - n) // n
    g4.paged_prompt_dev(ctx, cache, 0, q[n:], out[n:], heads, i32(seqs), i32(range(0, rows * n + 1, rows)), rows * n, scale)
    places += [(s, lengths[s] - rows + j, n + i * rows + j) for i, s in enumerate(seqs) for j in range(rows)]
    torch.cuda.synchronize()
    return out.cpu().double(), places


@pytest.mark.parametrize("large", [1e2, 1e3, 3e4, 1e6], ids=str)
@pytest.mark.parametrize("typ,hs", [("f16", 128), ("f16", 256), ("f16", 64), ("bf16", 128), ("f32", 128)])
def test_small_elements_beside_a_large_one(g4, run, typ, hs, large):  # noqa: F811
    """One element of a query is far larger than the others and meets keys that are zero: the
    scores are the others'."""
    announce("one query element of %g, %s, heads of %d" % (large, typ, hs))
    lengths, heads, kv = [70, 33, 5], 4, 2
    cache = filled(g4, run, 110, typ, 1, kv, hs, 16, lengths)
    cache.k[..., hs // 2 + 3] = 0
    q = normal(gen(111), 3 + 3 * 4, heads, hs, scale=2.0)
    q[..., hs // 2 + 3] = large
    out, places = both(g4, run, cache, q.cuda(), heads, [2, 0, 1], lengths, hs ** -0.5)
    m = Model(cache)
    worst = 0.0
    for s, pos, r in places:
        k, v, _ = m.rows(0, s, pos + 1)
        for h in range(heads):
            kh = k[:, h // 2]
            o, size, a = exact(q[r, h], kh, v[:, h // 2], hs ** -0.5)
            lost = 2.0 ** -39 * large * float(kh.abs().sum(1).max()) * hs ** -0.5 if typ == "f16" else 0.0
            tol = bar(typ, hs, size, a) + 2 * lost * size
            worst = max(worst, float(((out[r, h] - o).abs() / tol).max()))
    assert worst <= 1, "%g of what is allowed" % worst


@pytest.mark.parametrize("size", [2.0 ** -115, 1e-30, 1e-3, 1e4, 1e30], ids=str)
def test_queries_of_any_size(g4, run, size):  # noqa: F811
    """The scale takes back what the queries have too much or too little."""
    announce("F16, queries of %g" % size)
    hs, heads, lengths = 80, 2, [40, 17]
    cache = filled(g4, run, 112, "f16", 1, 1, hs, 16, lengths)
    q = (normal(gen(113), 2 + 2 * 3, heads, hs).double() * size).float()
    scale = float(torch.tensor(hs ** -0.5 / size, dtype=torch.float64).float())
    out, places = both(g4, run, cache, q.cuda(), heads, [0, 1], lengths, scale)
    m = Model(cache)
    for s, pos, r in places:
        k, v, _ = m.rows(0, s, pos + 1)
        for h in range(heads):
            o, width, a = exact(q[r, h], k[:, 0], v[:, 0], scale)
            assert bool(((out[r, h] - o).abs() <= bar("f16", 96, width, a)).all())


@pytest.mark.parametrize("hs", [64, 256])
def test_subnormal_keys_and_values(g4, run, hs):  # noqa: F811
    """F16 keys and values below 2^-14 are what they say."""
    announce("F16 subnormal keys and values, heads of %d" % hs)
    lengths, heads, kv = [50, 90], 4, 1
    cache = filled(g4, run, 114, "f16", 1, kv, hs, 16, lengths, garbage=0.0)
    for t in (cache.k, cache.v):
        t.copy_((t.float() * 2.0 ** -18).half())
    q = normal(gen(115), 2 + 2 * 5, heads, hs, scale=2.0 ** 18)
    out, places = both(g4, run, cache, q.cuda(), heads, [1, 0], lengths, hs ** -0.5)
    m = Model(cache)
    for s, pos, r in places:
        k, v, _ = m.rows(0, s, pos + 1)
        for h in range(heads):
            o, size, a = exact(q[r, h], k[:, 0], v[:, 0], hs ** -0.5)
            assert bool(((out[r, h] - o).abs() <= bar("f16", hs, size, a)).all())


def causal(q, k, v, first, scale):
    """Rows of one head at positions first, first + 1 .. over k, v [tokens, head size] in 64 bits."""
    s = (q.double() @ k.T) * scale
    t = torch.arange(len(k), device=k.device)
    s = s.masked_fill(t > first + torch.arange(len(q), device=k.device)[:, None], -float("inf"))
    return torch.softmax(s, 1) @ v


def cut(x, bits):
    """fp32 values without all but their highest `bits` bits."""
    return (x.view(torch.int32) & -(1 << (24 - bits))).view(torch.float32)


@pytest.mark.parametrize("length", [150, 2500])
@pytest.mark.parametrize("typ,parts", [("bf16", 16), ("f16", 11), ("f32", 16)])
def test_errors_beside_the_largest_value(g4, run, typ, parts, length):  # noqa: F811
    """|out - exact| <= 3e-6 max |v| for queries and keys of ordinary size.  A score of up to
    8 (in powers of two) passes 12 matrix instructions of BF16 for 128 elements, 8 of F16 or 32
    of F32, of which each leaves out 2^-24 of it on average: 32 * 2^-24 * 8 ln 2 = 1.1e-5 of a
    weight at most.  A result is a mean of values with those weights, and what is common to
    them cancels: below 1.1e-5 of a mean |v| of 0.8, where the largest |v| is above 4.
    Queries with only `parts` bits, one 16-bit part fewer, err by more: that is checked here too, with
    the formula."""
    announce("errors of %s over %d tokens" % (typ, length))
    hs, heads, kv = 128, 4, 2
    cache = filled(g4, run, 116, typ, 1, kv, hs, 32, [length, length])
    q = normal(gen(117), length, heads, hs, scale=2.0).cuda()
    one = normal(gen(118), 2, heads, hs, scale=2.0).cuda()
    out, last = torch.empty_like(q), torch.empty_like(one)
    scale = hs ** -0.5
    g4.paged_prompt_dev(run, cache, 0, q, out, heads, i32([1]), i32([0, length]), length, scale)
    g4.paged_attention_dev(run, cache, 0, one, last, heads, i32([0, 1]), scale)
    torch.cuda.synchronize()
    m = Model(cache)
    worst = less = 0.0
    for s in (0, 1):
        k, v, _ = (t.cuda() if isinstance(t, torch.Tensor) else t for t in m.rows(0, s, length))
        for h in range(heads):
            kh, vh = k[:, h // 2].contiguous(), v[:, h // 2].contiguous()
            bound = 3e-6 * float(vh.abs().max())
            o = causal(one[s:s + 1, h], kh, vh, length - 1, scale)
            worst = max(worst, float((last[s:s + 1, h].double() - o).abs().max()) / bound)
            if s == 1:
                o = causal(q[:, h], kh, vh, 0, scale)
                worst = max(worst, float((out[:, h].double() - o).abs().max()) / bound)
                fewer = causal(cut(q[:, h].contiguous(), parts), kh, vh, 0, scale)
                less = max(less, float((fewer - o).abs().max()) / bound)
    print("[error] %s %d: %.2f of the bar, %.2f with a part fewer" % (typ, length, worst, less))
    assert worst <= 1 and less > 1
