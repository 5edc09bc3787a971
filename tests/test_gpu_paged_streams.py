"""GPU tests of what is ordered between torch's stream and a context's own."""
import pytest
import torch

from conftest import announce
from paged_ref import Model
from test_gpu_paged import i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("side", [False, True], ids=["default stream", "side stream"])
def test_a_new_cache_is_ready_for_the_contexts_own_stream(g4, side):
    """A cache made behind 100 ms of torch's work, extended and written at once on the
    context's own stream: nothing of it is cleared afterwards."""
    announce("a new cache behind torch's work")
    c2 = g4.Context(0)
    try:
        seqs, counts, begin = i32([1, 0]), i32([20, 3]), i32([0, 20, 23])
        k = torch.randn(23, 2, 64, device="cuda")
        x = torch.randn(8192, 8192, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.current_stream()):
            for _ in range(15):
                torch.mm(x, x, out=torch.empty_like(x))
            cache = g4.KvCache.create(c2, 3, 2, 64, 16, 300, 2, 4, torch.float32)
        g4.kv_extend_dev(c2, cache, seqs, counts)
        g4.kv_rope_write_dev(c2, cache, 2, None, None, k, -k, 0, None, seqs, begin, 23)
        g4.kv_status(c2, cache)
        torch.cuda.synchronize()
        model = Model(cache)
        assert model.lengths.tolist() == [3, 20] and model.table[:, :3].tolist() == [[2, -1, -1], [0, 1, -1]]
        assert model.refs.tolist() == [1, 1, 1] + [0] * 297
        for s, rows in ((1, k[:20]), (0, k[20:])):
            keys, values, there = model.rows(2, s, len(rows))
            assert there.all() and torch.equal(keys.float(), rows.cpu()) and torch.equal(values.float(), -rows.cpu())
        assert not bool(cache.k[:2].any()) and not bool(cache.v[:2].any())
    finally:
        torch.cuda.synchronize()
        c2.close()


def test_a_cache_made_in_a_capture(g4):
    """The fills are the graph's: each replay empties the cache again."""
    announce("a cache made in a capture")
    c2 = g4.Context(0)
    try:
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        one, count = i32([0]), i32([5])
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            c2.set_stream(stream.cuda_stream)
            cache = g4.KvCache.create(c2, 1, 1, 64, 16, 4, 2, 4)
        c2.set_stream(None)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert cache.lengths.tolist() == [0, 0] and bool((cache.table == -1).all())
            g4.kv_extend_dev(c2, cache, one, count)
            g4.kv_status(c2, cache)
            assert cache.lengths.tolist() == [5, 0] and cache.refs.tolist() == [1, 0, 0, 0]
    finally:
        torch.cuda.synchronize()
        c2.close()
