"""GPU tests of allowed calls at the edges of attention over a paged cache: more query heads
to a kv head than a tile holds, the most heads, more query tiles than the plan's workgroup
has threads, two contexts at once.  Against plain forms in 64 bits, with the bars of
test_gpu_paged.py."""
import numpy as np
import pytest
import torch

from conftest import announce
from paged_ref import Model
from test_gpu_paged import check_rows, filled, gen, i32, normal, run  # noqa: F401  (run is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ,heads,kv,hs,window,sinks", [
    ("f16", 200, 1, 64, 0, 0),      # 192 rows a tile: 192 heads and 8
    ("bf16", 150, 1, 256, 30, 2),   # 128
    ("f32", 100, 1, 512, 0, 0),     # 64
    ("bf16", 1024, 1, 8, 0, 0),
    ("f16", 1024, 1024, 8, 20, 1),
    ("f32", 1024, 512, 16, 0, 0),
], ids=str)
def test_many_heads(g4, run, typ, heads, kv, hs, window, sinks):  # noqa: F811
    announce("%s, %d/%d heads of %d" % (typ, heads, kv, hs))
    lengths = [70, 1, 33]
    cache = filled(g4, run, 130, typ, 1, kv, hs, 16, lengths)
    model = Model(cache)
    q = normal(gen(131), 3 + 19, heads, hs).cuda()
    out = torch.full_like(q, float("nan"))
    scale = hs ** -0.5
    g4.paged_attention_dev(run, cache, 0, q[:3], out[:3], heads, i32([2, 0, 1]), scale, window, sinks)
    g4.paged_prompt_dev(run, cache, 0, q[3:], out[3:], heads, i32([0, 1, 2]), i32([0, 11, 12, 19]), 19, scale, window, sinks)
    torch.cuda.synchronize()
    places = [(0, 2, 32), (1, 0, 69), (2, 1, 0), (3, 0, 59), (8, 0, 64), (13, 0, 69), (14, 1, 0), (15, 2, 26), (21, 2, 32)]
    check_rows(out, places, model, 0, q, scale, window, sinks)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 7)], ids=str)
def test_more_query_tiles_than_threads(g4, run, window, sinks):  # noqa: F811
    """Four tokens to a query tile: 1250 of them, with sequences of no rows among the list."""
    announce("1250 query tiles, window %d" % window)
    heads, hs = 16, 512
    lengths = [3500, 1500, 9, 20]
    cache = filled(g4, run, 132, "bf16", 1, 1, hs, 64, lengths)
    model = Model(cache)
    seqs, rows = [1, 3, 0, 2], [1490, 0, 3500, 9]
    begin = [int(x) for x in np.concatenate([[0], np.cumsum(rows)])]
    total = begin[-1]
    q = normal(gen(133), total, heads, hs).cuda()
    out = torch.full_like(q, float("nan"))
    g4.paged_prompt_dev(run, cache, 0, q, out, heads, i32(seqs), i32(begin), total, hs ** -0.5, window, sinks)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all())
    places = [(begin[i] + j, s, lengths[s] - rows[i] + j) for i, s in enumerate(seqs) for j in range(rows[i])
              if j % 307 == 0 or j in (1, 3, 4, rows[i] - 1)]
    check_rows(out, places, model, 0, q, hs ** -0.5, window, sinks)


def test_two_contexts_at_once(g4, run):  # noqa: F811
    """Decode and prompts over one cache from two contexts, each on a stream of its own."""
    announce("two contexts at once")
    cache = filled(g4, run, 134, "f16", 1, 2, 128, 16, [2500, 700, 33])
    q, p = normal(gen(135), 3, 8, 128).cuda(), normal(gen(136), 600, 8, 128).cuda()
    seqs, begin = i32([0, 1, 2]), i32([0, 400, 590, 600])

    def calls(c, q, p):
        a, b = torch.empty_like(q), torch.empty_like(p)
        torch.cuda.synchronize()
        for _ in range(8):
            g4.paged_attention_dev(c, cache, 0, q, a, 8, seqs, 0.1, 600, 3)
            g4.paged_prompt_dev(c, cache, 0, p, b, 8, seqs, begin, 600, 0.1)
        return a, b

    want = calls(run, q, p)
    torch.cuda.synchronize()
    others = [g4.Context(0), g4.Context(0)]
    try:
        outs = [(torch.empty_like(q), torch.empty_like(p)) for _ in others]
        torch.cuda.synchronize()
        for _ in range(8):  # issued in turn: the contexts' streams run beside each other
            for c, (a, b) in zip(others, outs):
                g4.paged_attention_dev(c, cache, 0, q, a, 8, seqs, 0.1, 600, 3)
                g4.paged_prompt_dev(c, cache, 0, p, b, 8, seqs, begin, 600, 0.1)
        for c in others:
            c.sync()
        for a, b in outs:
            assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    finally:
        torch.cuda.synchronize()
        for c in others:
            c.close()
