"""GPU tests that a write of new rows is all or nothing: one row without a place, and neither
the cache nor the queries, turned in place, have changed; with the place restored the same
call gives the bits of a call that met no such row."""
import numpy as np
import pytest
import torch

from conftest import announce
from paged_ref import Model
from test_gpu_paged import filled, gen, i32, normal, run  # noqa: F401  (run is a fixture)

pytestmark = pytest.mark.gpu

CALLS = [
    # type, heads, kv, head size, page, sequences, rows of each (None: one, without row_begin)
    ("bf16", 8, 2, 64, 16, 1, None),
    ("f16", 4, 1, 64, 16, 1024, None),
    ("f32", 4, 2, 128, 32, 7, 3),
    ("bf16", 4, 2, 64, 16, 128, 16),       # 2048 rows: looked at by every workgroup
    ("f16", 2, 1, 64, 16, 3, 2000),        # 6000: by one before them
    ("bf16", 1, 1, 8, 64, 700, 9),
]

FAULTS = ["shared", "missing", "out of range", "short", "twice", "no sequence"]


def spoil(cache, seqs, at, rows, fault, other):
    """Takes the place of a row of entry `at` away; returns the list to use and how to restore."""
    lists = list(seqs)
    s, n = seqs[at], int(cache.lengths[seqs[at]])
    column = (n - 1 - (rows // 2)) // cache.page_tokens  # a page in the middle of the entry's rows
    page = int(cache.table[s, column])
    undo = []
    if fault == "shared":
        cache.refs[page] = 2
        undo.append(lambda: cache.refs.__setitem__(page, 1))
    elif fault in ("missing", "out of range"):
        cache.table[s, column] = -1 if fault == "missing" else cache.n_pages
        undo.append(lambda: cache.table.__setitem__((s, column), page))
    elif fault == "short":
        cache.lengths[s] = rows - 1
        undo.append(lambda: cache.lengths.__setitem__(s, n))
    elif fault == "twice":
        lists[at] = seqs[other]
    else:
        lists[at] = cache.lengths.numel()
    return lists, undo


@pytest.mark.parametrize("typ,heads,kv,hs,page,n,rows", CALLS, ids=[str(c) for c in CALLS])
def test_a_row_without_a_place_stops_the_write(g4, run, typ, heads, kv, hs, page, n, rows):  # noqa: F811
    announce("write of %d x %s rows, %s" % (n, rows, typ))
    count, g = rows or 1, gen(120)
    lengths = [count + int(x) for x in torch.randint(0, 40, (n,), generator=g)]
    cache = filled(g4, run, 121, typ, 1, kv, hs, page, lengths, garbage=0.0)
    start = [t.clone() for t in (cache.k, cache.v)]
    total = n * count
    q0, k, v = (normal(g, total, m, hs).cuda() for m in (heads, kv, kv))
    q = q0.clone()
    seqs = torch.randperm(n, generator=g).tolist()
    begin = None if rows is None else i32(range(0, total + 1, rows))
    rope = g4.Rope.create(run, hs // 2 // 2 * 2)

    def write(order):
        g4.kv_rope_write_dev(run, cache, 0, q, q, k, v, heads, rope, i32(order), begin, total)

    write(seqs)
    g4.kv_status(run, cache)
    good = [t.clone() for t in (q, cache.k, cache.v)]
    assert not torch.equal(q, q0)
    q.copy_(q0)
    for pool, was in zip((cache.k, cache.v), start):
        pool.copy_(was)
    before = Model(cache)
    for i, fault in enumerate(FAULTS):
        if fault == "twice" and n == 1:
            continue
        for at in sorted({0, n // 2, n - 1}):
            order, undo = spoil(cache, seqs, at, count, fault, (at + 1) % n)
            for _ in range(2):  # the status cleared, the same again
                write(order)
                with pytest.raises(g4.IndexOutOfBoundsException):
                    g4.kv_status(run, cache)
            for u in undo:
                u()
            torch.cuda.synchronize()
            assert torch.equal(q, q0), fault
            before.same_contents(cache)
    write(seqs)
    g4.kv_status(run, cache)
    for mine, theirs in zip((q, cache.k, cache.v), good):
        assert torch.equal(mine, theirs)


def test_entries_without_rows(g4, run):  # noqa: F811
    """They need no place: sequences out of range, empty, shared, or named by others; rows before
    and behind the entries are left as they are."""
    announce("write, entries without rows")
    cache = filled(g4, run, 122, "bf16", 1, 1, 64, 16, [40, 33, 0, 20], garbage=0.0)
    cache.refs[int(cache.table[1, 0])] = 2
    model = Model(cache)
    q, k, v = (normal(gen(123), 9, m, 64).cuda() for m in (2, 1, 1))
    out = torch.full_like(q, -7.0)
    rope = g4.Rope.create(run, 64)
    g4.kv_rope_write_dev(run, cache, 0, q, out, k, v, 2, rope, i32([99, 0, 2, 1, -1, 3, 99, 2]),
                         i32([1, 1, 4, 4, 4, 4, 7, 7, 7]), 9)
    g4.kv_status(run, cache)
    assert bool((out[0] == -7).all()) and bool((out[7:] == -7).all()) and not bool((out[1:7] == -7).any())
    for r, s, p in [(1 + j, 0, 37 + j) for j in range(3)] + [(4 + j, 3, 17 + j) for j in range(3)]:
        at = model.table[s, p // 16]
        model.write(0, s, p, cache.k[0, int(at), :, p % 16].cpu(), v[r].cpu())
    model.same_contents(cache)


def test_pages_in_the_middle_of_many_rows(g4, run):  # noqa: F811
    """Every page of a long entry is looked at, wherever the entry's rows begin."""
    announce("write, a shared page anywhere")
    for first, rows in ((0, 200), (5, 200), (1, 3000)):
        cache = filled(g4, run, 124, "f16", 1, 1, 8, 16, [rows + 21], garbage=0.0)
        before = Model(cache)
        k = torch.ones(first + rows, 1, 8, device="cuda")
        used = range(21 // 16, -(-(rows + 21) // 16))
        for column in list(used)[:14] + list(used)[-3:] + [used[len(used) // 2]]:
            page = int(before.table[0, column])
            cache.refs[page] = 2
            g4.kv_rope_write_dev(run, cache, 0, None, None, k, k, 0, None, i32([0]), i32([first, first + rows]), first + rows)
            with pytest.raises(g4.IndexOutOfBoundsException):
                g4.kv_status(run, cache)
            cache.refs[page] = 1
            before.same_contents(cache)
        cache.refs[int(before.table[0, 0])] = 2  # holds none of the rows
        g4.kv_rope_write_dev(run, cache, 0, None, None, k, k, 0, None, i32([0]), i32([first, first + rows]), first + rows)
        g4.kv_status(run, cache)
        assert int((cache.k == 1).sum()) == rows * 8 and np.array_equal(Model(cache).table, before.table)


@pytest.mark.parametrize("rows", [40, 1500])
def test_a_captured_write_meets_a_row_without_a_place(g4, rows):
    """Recorded once and replayed, with eager calls between: replays write while every row has a
    place, nothing at all while one has none, and go on after the status is cleared."""
    announce("a captured write of 2 x %d rows" % rows)
    c2 = g4.Context(0)
    try:
        cache = g4.KvCache.create(c2, 1, 1, 64, 16, 400, 2, 200, torch.float32)
        seqs, begin = i32([1, 0]), i32([0, rows, 2 * rows])
        rope = g4.Rope.create(c2, 64)
        q, k, v = (torch.zeros(2 * rows, m, 64, device="cuda") for m in (2, 1, 1))
        out = torch.empty_like(q)
        g4.kv_extend_dev(c2, cache, seqs, i32([rows + 7, rows]))
        g4.kv_status(c2, cache)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            c2.set_stream(stream.cuda_stream)
            g4.kv_rope_write_dev(c2, cache, 0, q, out, k, v, 2, rope, seqs, begin, 2 * rows)
        c2.set_stream(None)
        g, page = gen(125), int(cache.table[0, rows // 32])
        for i in range(6):
            for t in (q, k, v):
                t.copy_(normal(g, *t.shape))
            out.fill_(float("nan"))
            bad = i % 3 == 1
            cache.refs[page] = 3 if bad else 1
            before = Model(cache)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            if bad:
                assert int(cache.status_word.cpu()) == 2 and bool(torch.isnan(out).all())
                before.same_contents(cache)
                with pytest.raises(g4.IndexOutOfBoundsException):
                    g4.kv_status(c2, cache)
                continue
            wrote, mine = [t.clone() for t in (out, cache.k, cache.v)], torch.empty_like(out)
            torch.cuda.synchronize()
            g4.kv_rope_write_dev(c2, cache, 0, q, mine, k, v, 2, rope, seqs, begin, 2 * rows)
            g4.kv_status(c2, cache)
            assert not bool(torch.isnan(mine).any()) and torch.equal(mine, wrote[0])
            assert torch.equal(cache.k, wrote[1]) and torch.equal(cache.v, wrote[2])
            assert not torch.equal(before.v, cache.v.cpu())
    finally:
        torch.cuda.synchronize()
        c2.close()
