"""GPU tests of what forks and compactions leave: whose pages are whose, and every
sequence's tokens, read back through the table.  Nothing here repeats the library's
choice of pages: a call is checked by what it promises.  All comparisons are exact."""
import numpy as np
import pytest
import torch

from conftest import announce
from paged_ref import Model
from test_gpu_paged import DT, filled, i32, run  # noqa: F401  (run is a fixture)

pytestmark = pytest.mark.gpu


def contents(model, seq):
    """Keys and values of a sequence, [layers, tokens, kv heads, head size] as they are stored."""
    t = np.arange(int(model.lengths[seq]))
    p = torch.from_numpy(model.table[seq, t // model.page].astype(np.int64))
    assert bool((p >= 0).all())
    y = torch.from_numpy(t % model.page)
    return [pool[:, p, :, y].transpose(0, 1) for pool in (model.k, model.v)]


def check_owners(model):
    """refs counts the sequences of a page, and a page with room has one."""
    held = model.table[model.table >= 0]
    assert np.array_equal(np.bincount(held, minlength=model.pages), model.refs)
    for s, n in enumerate(model.lengths):
        assert (model.table[s, -(-int(n) // model.page):] == -1).all()
        if n % model.page:
            assert model.refs[model.table[s, n // model.page]] == 1, "the last page of sequence %d is shared" % s


def check_move(before, after, src, dst, prefix, keep):
    check_owners(after)
    for s in range(len(before.lengths)):
        i = dst.index(s) if s in dst else None
        if i is None:
            want = contents(before, s)
            assert np.array_equal(before.table[s], after.table[s])
        else:
            rows = list(range(prefix[i])) + list(keep[i])
            want = [x[:, rows] for x in contents(before, src[i])]
            whole = prefix[i] // before.page
            assert np.array_equal(before.table[src[i], :whole], after.table[s, :whole])  # shared, not copied
        for a, b in zip(want, contents(after, s)):
            assert a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def call(g4, ctx, cache, src, dst, prefix, keep):
    if keep is None:
        g4.kv_fork_dev(ctx, cache, i32(src), i32(dst), i32(prefix))
    else:
        begin = np.concatenate([[0], np.cumsum([len(x) for x in keep])])
        g4.kv_compact_dev(ctx, cache, i32(src), i32(dst), i32(prefix), i32([t for x in keep for t in x]), i32(begin))
    g4.kv_status(ctx, cache)


SHORTENED = [
    # lengths, src, dst, prefix: a sequence is shortened while others continue it
    ([32], [0, 0], [0, 1], [20, 32]),                # the page it would keep is full in its continuation
    ([64], [0, 0], [0, 1], [20, 64]),
    ([64], [0, 0], [1, 0], [64, 20]),                # in the other order
    ([64], [0, 0, 0], [0, 1, 2], [20, 33, 31]),      # taken over by the second, copied by the third
    ([70], [0, 0, 0], [0, 1, 2], [17, 16, 30]),      # nobody else shares it: kept
    ([70, 40], [0, 1, 0, 1], [0, 1, 2, 3], [65, 39, 70, 33]),  # both kept
    ([70, 40], [0, 1, 0, 1], [1, 0, 2, 3], [50, 20, 64, 32]),
]


@pytest.mark.parametrize("compact", [False, True], ids=["fork", "compact"])
@pytest.mark.parametrize("lengths,src,dst,prefix", SHORTENED, ids=[str(c) for c in SHORTENED])
def test_a_shortened_sequence_owns_its_last_page(g4, run, lengths, src, dst, prefix, compact):  # noqa: F811
    announce("shortened beside its continuations: %s from %s to %s, %s" % (lengths, src, dst, prefix))
    cache = filled(g4, run, 90, "bf16", 2, 2, 64, 16, lengths, spare=12, slots=4)
    before = Model(cache)
    keep = [[]] * len(src) if compact else None
    call(g4, run, cache, src, dst, prefix, keep)
    after = Model(cache)
    check_move(before, after, src, dst, prefix, [[]] * len(src))
    for i, (s, d) in enumerate(zip(src, dst)):  # nothing is copied where nothing has to be
        if s == d and prefix[i] % 16 and max(p // 16 for a, p in zip(src, prefix) if a == s) <= prefix[i] // 16:
            assert after.table[d, prefix[i] // 16] == before.table[d, prefix[i] // 16]
    # every one of them goes on by itself
    n = len(dst)
    g4.kv_extend_dev(run, cache, i32(dst), i32([3] * n))
    k = torch.randn(3 * n, 2, 64, device="cuda")
    g4.kv_rope_write_dev(run, cache, 1, None, None, k, -k, 0, None, i32(dst), i32(range(0, 3 * n + 1, 3)), 3 * n)
    g4.kv_status(run, cache)
    model = Model(cache)
    check_owners(model)
    for i, d in enumerate(dst):
        keys, values = contents(model, d)
        old = contents(after, d)
        assert torch.equal(keys[1, -3:], k[3 * i:3 * i + 3].cpu().bfloat16())
        assert torch.equal(values[1, -3:], -k[3 * i:3 * i + 3].cpu().bfloat16())
        assert torch.equal(keys[:, :-3], old[0]) and torch.equal(values[:, :-3], old[1])


@pytest.mark.parametrize("typ,page", [("f16", 16), ("f32", 64)])
def test_many_moves(g4, run, typ, page):  # noqa: F811
    """Forks and compactions in a row, sequences often their own source, lengths often at a
    page's border."""
    announce("many moves, %s, pages of %d" % (typ, page))
    rng = np.random.default_rng(page)
    slots, most = 7, 6 * page
    cache = filled(g4, run, 91, typ, 1, 1, 8, page, [most, 3 * page, page + 1, 5, 0], spare=120, slots=slots)
    for step in range(40):
        before = Model(cache)
        n = int(rng.integers(1, slots + 1))
        dst = rng.permutation(slots)[:n].tolist()
        src = [d if rng.random() < 0.5 else int(rng.integers(slots)) for d in dst]
        if rng.random() < 0.5:
            src = [src[0]] * n
        prefix = []
        for s in src:
            length = int(before.lengths[s])
            prefix.append(min(length, int(rng.integers(length // page + 1)) * page) if rng.random() < 0.4
                          else int(rng.integers(length + 1)))
        keep = [[int(rng.integers(before.lengths[s])) for _ in range(int(rng.integers(3 * page)))]
                if rng.random() < 0.4 and before.lengths[s] and p + 3 * page <= most else [] for s, p in zip(src, prefix)]
        if step % 2:
            keep = [[]] * n
        call(g4, run, cache, src, dst, prefix, None if step % 2 else keep)
        check_move(before, Model(cache), src, dst, prefix, keep)
        seqs = [s for s in range(slots) if int(cache.lengths[s]) + page + 3 <= most]
        if seqs:  # rows of what is new
            g4.kv_extend_dev(run, cache, i32(seqs), i32([page + 3] * len(seqs)))
            k = torch.randn(len(seqs) * (page + 3), 1, 8, device="cuda")
            g4.kv_rope_write_dev(run, cache, 0, None, None, k, k, 0, None, i32(seqs),
                                 i32(range(0, len(seqs) * (page + 3) + 1, page + 3)), len(k))
            g4.kv_status(run, cache)
            check_owners(Model(cache))
