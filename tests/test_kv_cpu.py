"""CPU tests of the paged cache's host side: descriptions and arguments that are refused,
the rotary frequencies, what a call launches (over the stand-in runtime of
test_host_calls.py), and the Python wrappers' checks."""
import ctypes
import math

import numpy as np
import pytest
import torch

import g4hip
from test_host_calls import Program, hip  # noqa: F401  (the fixture)

INVALID, UNSUPPORTED, OUT_OF_RANGE = -1, -2, -3


def struct(**change):
    f = dict(type=30, n_layers=2, n_kv_heads=4, head_size=128, page_tokens=16, n_pages=100, max_seqs=8, max_pages=64,
             k=4096, v=8192, table=4096, lengths=4096, refs=4096, status=4096)
    f.update(change)
    return g4hip._KvStruct(**f)


def checked(**change):
    s = struct(**change)
    return g4hip.lib().g4_kv_check(ctypes.addressof(s))


def test_descriptions():
    assert checked() == 0
    assert checked(type=0) == 0 and checked(type=1) == 0
    assert checked(type=8) == UNSUPPORTED and checked(type=-1) == UNSUPPORTED
    assert g4hip.lib().g4_kv_check(None) == INVALID
    for hs in (8, 80, 96, 512):
        assert checked(head_size=hs) == 0
    for bad in (dict(head_size=0), dict(head_size=4), dict(head_size=100), dict(head_size=520), dict(head_size=-8),
                dict(page_tokens=8), dict(page_tokens=24), dict(page_tokens=512), dict(page_tokens=0),
                dict(n_layers=0), dict(n_kv_heads=0), dict(n_kv_heads=2000), dict(n_pages=0), dict(max_seqs=0),
                dict(max_seqs=1025), dict(max_pages=0), dict(n_pages=1 << 27), dict(max_pages=(1 << 26) + 1),
                dict(k=None), dict(v=None), dict(table=None), dict(lengths=None), dict(refs=None), dict(status=None),
                dict(k=4100), dict(v=8200), dict(table=4098), dict(status=4097)):
        assert checked(**bad) == INVALID, bad
        assert g4hip.last_error()
    assert checked(n_pages=(1 << 27) - 1, max_pages=1 << 26, max_seqs=1024) == 0


def test_null_contexts():
    L, s = g4hip.lib(), struct()
    at = ctypes.addressof(s)
    assert L.g4_kv_init_dev(None, at) == INVALID and L.g4_kv_status(None, at) == INVALID
    assert L.g4_kv_extend_dev(None, at, 1, 4096, 4096) == INVALID
    assert L.g4_kv_fork_dev(None, at, 1, 4096, 4096, None) == INVALID
    assert L.g4_kv_compact_dev(None, at, 1, 4096, 4096, None, 4096, 4096, 1) == INVALID
    assert L.g4_kv_free_dev(None, at, 1, 4096) == INVALID and L.g4_kv_trim_dev(None, at, 1, 4096, 1, 0) == INVALID
    assert L.g4_rope_dev(None, None, 4096, 4096, 1, 1, 8, 4096) == INVALID
    assert L.g4_kv_rope_write_dev(None, at, 0, None, None, None, 4096, 4096, 0, 1, 4096, None, 1) == INVALID
    assert L.g4_paged_attention_dev(None, at, 0, 4096, 8192, 4, 1, 4096, 1.0, 0, 0) == INVALID
    assert L.g4_paged_prompt_dev(None, at, 0, 4096, 8192, 4, 1, 4096, 4096, 1, 1.0, 0, 0) == INVALID


# ------------------------------------------------------------- frequencies ---

def test_frequencies():
    plain = np.array([10000.0 ** (-2 * i / 64) for i in range(32)])
    f, gain = g4hip.rope_freqs(64)
    assert np.allclose(f, plain, rtol=1e-14) and gain == 1.0
    f, gain = g4hip.rope_freqs(64, scaling=g4hip.ROPE_SCALE_LINEAR, factor=8.0)
    assert np.allclose(f, plain / 8, rtol=1e-14) and gain == 1.0
    f, _ = g4hip.rope_freqs(64, scaling=g4hip.ROPE_SCALE_BASE, factor=8.0)
    assert np.allclose(f, [(10000.0 * 8 ** (64 / 62)) ** (-2 * i / 64) for i in range(32)], rtol=1e-13)
    assert np.isclose(f[31], plain[31] / 8, rtol=1e-12)  # the slowest pair is divided by the factor, the first stays
    d = np.linspace(1, 4, 32, dtype=np.float32)
    f, _ = g4hip.rope_freqs(64, 500000.0, divisors=d)
    assert np.allclose(f, 500000.0 ** (-np.arange(32) / 32) / d, rtol=1e-14)


def test_ramped_frequencies():
    trained, factor = 4096.0, 16.0
    f, gain = g4hip.rope_freqs(128, scaling=g4hip.ROPE_SCALE_RAMP, factor=factor, trained=trained)
    plain = 10000.0 ** (-np.arange(64) / 64)
    turns = trained * plain / (2 * math.pi)
    assert abs(gain - (1 + 0.1 * math.log(factor))) < 1e-6
    ratio = plain / f
    # a pair next to where the ramp begins or ends belongs to it
    assert np.allclose(ratio[np.r_[turns[1:] > 32, False]], 1.0) and np.allclose(ratio[np.r_[False, turns[:-1] < 1]], factor)
    assert bool((np.diff(ratio) >= -1e-9).all()) and 1 < ratio[len(ratio) // 2 - 2] < factor
    share = 1 - (factor / ratio - 1) / (factor - 1)  # how far down the ramp: linear over the pairs
    inner = (share > 1e-9) & (share < 1 - 1e-9)
    assert inner.sum() > 5 and np.allclose(np.diff(share[inner]), np.diff(share[inner])[0])


def test_frequencies_that_are_refused():
    for args in (dict(rot=7), dict(rot=0), dict(rot=-2), dict(rot=8, base=1.0), dict(rot=8, base=float("nan")),
                 dict(rot=8, scaling=4), dict(rot=8, scaling=-1), dict(rot=8, scaling=1, factor=0.5),
                 dict(rot=8, scaling=1, factor=float("inf")), dict(rot=2, scaling=2, factor=2.0),
                 dict(rot=8, scaling=3, factor=2.0), dict(rot=8, scaling=3, factor=2.0, trained=100.0, fast=1.0),
                 dict(rot=8, divisors=np.zeros(4, np.float32))):
        with pytest.raises(g4hip.IllegalArgumentException):
            g4hip.rope_freqs(**args)
    with pytest.raises(g4hip.IndexOutOfBoundsException):
        g4hip.rope_freqs(8, divisors=np.ones(3, np.float32))
    assert g4hip.lib().g4_rope_freqs(8, 1e4, 0, 1.0, 0.0, 0.0, 0.0, None, None, None) == INVALID


# ------------------------------------------------------- calls and launches ---

KV_KERNELS = ["k_kv_init", "k_kv_extend", "k_kv_release", "k_kv_resolve", "k_kv_plan", "k_kv_move", "k_kv_write",
              "k_rope", "k_prompt_plan", "k_paged_prompt_join", "k_paged_prompt", "k_paged_split", "k_paged_join"]


def launched(p, call):
    before = len(p.log())
    rc = call()
    return rc, [next((k for k in KV_KERNELS if k in l[1]), l[1]) for l in p.log()[before:] if l[0] == "launch"]


def test_what_calls_launch(hip):
    with Program(hip) as p:
        s = struct()
        at, c = ctypes.addressof(s), p.ctx
        rope = g4hip._RopeStruct(4096, 64, 0, 1.0)
        r = ctypes.addressof(rope)
        assert launched(p, lambda: hip.g4_kv_init_dev(c, at)) == (0, ["k_kv_init"])
        assert launched(p, lambda: hip.g4_kv_extend_dev(c, at, 3, 4096, 4096)) == (0, ["k_kv_extend"])
        assert launched(p, lambda: hip.g4_kv_fork_dev(c, at, 3, 4096, 4096, None)) == (0, ["k_kv_plan", "k_kv_move"])
        assert launched(p, lambda: hip.g4_kv_compact_dev(c, at, 3, 4096, 4096, None, 4096, 4096, 9)) == (
            0, ["k_kv_resolve", "k_kv_plan", "k_kv_move"])
        assert launched(p, lambda: hip.g4_kv_free_dev(c, at, 3, 4096)) == (0, ["k_kv_release"])
        assert launched(p, lambda: hip.g4_kv_trim_dev(c, at, 3, 4096, 5, 0)) == (0, ["k_kv_release"])
        assert launched(p, lambda: hip.g4_rope_dev(c, r, 4096, 4096, 2, 4, 128, 4096)) == (0, ["k_rope"])
        assert launched(p, lambda: hip.g4_kv_rope_write_dev(c, at, 1, r, 4096, 4096, 4096, 4096, 8, 3, 4096, None, 3)) \
            == (0, ["k_kv_write"])
        assert launched(p, lambda: hip.g4_paged_attention_dev(c, at, 1, 1 << 20, 1 << 21, 8, 3, 4096, 1.0, 0, 0)) == (
            0, ["k_paged_split", "k_paged_join"])
        assert launched(p, lambda: hip.g4_paged_prompt_dev(c, at, 1, 1 << 20, 1 << 21, 8, 3, 4096, 4096, 9, 1.0, 0, 0)) \
            == (0, ["k_prompt_plan", "k_paged_prompt", "k_paged_prompt_join"])
        # nothing to do
        for call in (lambda: hip.g4_kv_extend_dev(c, at, 0, None, None), lambda: hip.g4_kv_free_dev(c, at, 0, None),
                     lambda: hip.g4_kv_fork_dev(c, at, 0, None, None, None),
                     lambda: hip.g4_kv_compact_dev(c, at, 0, None, None, None, None, None, 0),
                     lambda: hip.g4_rope_dev(c, r, None, None, 0, 4, 128, None),
                     lambda: hip.g4_kv_rope_write_dev(c, at, 1, r, None, None, None, None, 8, 0, None, None, 0),
                     lambda: hip.g4_paged_attention_dev(c, at, 1, None, None, 8, 0, None, 1.0, 0, 0),
                     lambda: hip.g4_paged_prompt_dev(c, at, 1, None, None, 8, 3, 4096, 4096, 0, 1.0, 0, 0)):
            assert launched(p, call) == (0, [])


def test_calls_that_are_refused(hip):
    with Program(hip) as p:
        s = struct()
        at, c = ctypes.addressof(s), p.ctx

        def att(layer=0, q=1 << 20, out=1 << 21, heads=8, n=3, seqs=4096, scale=1.0, window=0, sinks=0, kv=at):
            return hip.g4_paged_attention_dev(c, kv, layer, q, out, heads, n, seqs, scale, window, sinks)

        def prompt(begin=4096, rows=9, **k):
            a = dict(layer=0, q=1 << 20, out=1 << 21, heads=8, n=3, seqs=4096, scale=1.0, window=0, sinks=0, kv=at)
            a.update(k)
            return hip.g4_paged_prompt_dev(c, a["kv"], a["layer"], a["q"], a["out"], a["heads"], a["n"], a["seqs"],
                                           begin, rows, a["scale"], a["window"], a["sinks"])

        def write(layer=0, rope=(64, 0), q=4096, q_out=4096, k=4096, v=4096, heads=8, n=3, seqs=4096, begin=None,
                  rows=3):
            r = g4hip._RopeStruct(4096, rope[0], rope[1], 1.0) if rope else None
            return hip.g4_kv_rope_write_dev(c, at, layer, ctypes.addressof(r) if r else None, q, q_out, k, v, heads, n,
                                            seqs, begin, rows)

        def turn(rot=64, layout=0, freqs=4096, x=4096, out=4096, rows=2, heads=4, hs=128, pos=4096):
            r = g4hip._RopeStruct(freqs, rot, layout, 1.0)
            return hip.g4_rope_dev(c, ctypes.addressof(r), x, out, rows, heads, hs, pos)

        bad = struct(head_size=100)
        before = len(p.log())
        for f in (att, prompt):
            assert f(layer=2) == OUT_OF_RANGE and f(layer=-1) == OUT_OF_RANGE
            for k in (dict(heads=6), dict(heads=0), dict(heads=2048), dict(n=-1), dict(n=1025), dict(seqs=None),
                      dict(q=None), dict(out=None), dict(q=(1 << 20) + 4), dict(out=(1 << 21) + 8),
                      dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(sinks=-1),
                      dict(out=1 << 20), dict(out=(1 << 20) + 4096), dict(kv=None), dict(kv=ctypes.addressof(bad))):
                assert f(**k) == INVALID, k
        assert prompt(begin=None) == INVALID and prompt(rows=-1) == INVALID and prompt(rows=0x10000000) == INVALID
        for k in (dict(rope=(130, 0)), dict(rope=(63, 0)), dict(rope=(64, 2)), dict(rope=(-2, 0)), dict(q=None),
                  dict(q_out=None), dict(rope=None), dict(k=None), dict(v=None), dict(heads=0), dict(heads=1025),
                  dict(n=-1), dict(n=1025), dict(seqs=None), dict(rows=4), dict(rows=-1)):
            assert write(**k) == INVALID, k
        assert write(layer=2) == OUT_OF_RANGE
        for k in (dict(rot=130), dict(rot=5), dict(layout=-1), dict(freqs=None), dict(x=None), dict(out=None),
                  dict(rows=-1), dict(heads=0), dict(hs=0), dict(hs=127), dict(pos=None)):
            assert turn(**k) == INVALID, k
        for n, a, b in ((-1, 4096, 4096), (1025, 4096, 4096), (1, None, 4096), (1, 4096, None)):
            assert hip.g4_kv_extend_dev(c, at, n, a, b) == INVALID
            assert hip.g4_kv_fork_dev(c, at, n, a, b, None) == INVALID
            assert hip.g4_kv_compact_dev(c, at, n, a, b, None, 4096, 4096, 1) == INVALID
        assert hip.g4_kv_compact_dev(c, at, 1, 4096, 4096, None, 4096, None, 1) == INVALID
        assert hip.g4_kv_compact_dev(c, at, 1, 4096, 4096, None, None, 4096, 1) == INVALID
        assert hip.g4_kv_compact_dev(c, at, 1, 4096, 4096, None, 4096, 4096, -1) == INVALID
        assert hip.g4_kv_compact_dev(c, at, 1, 4096, 4096, None, 4096, 4096, 0x7FFFFFFF) == INVALID
        assert hip.g4_kv_free_dev(c, at, 1, None) == INVALID
        for w, k in ((0, 0), (-1, 0), (5, -1)):
            assert hip.g4_kv_trim_dev(c, at, 1, 4096, w, k) == INVALID
        assert [l for l in p.log()[before:] if l[0] == "launch"] == []


def test_capture_needs_reserved_scratch(hip):
    """Calls with a workspace are refused under capture until it is there; the others are recorded."""
    with Program(hip) as p:
        s = struct()
        at, c, stream = ctypes.addressof(s), p.ctx, p.stream()
        p.use(stream)
        hip.stub_capture(stream, 1)
        assert hip.g4_kv_fork_dev(c, at, 3, 4096, 4096, None) == INVALID
        assert hip.g4_kv_status(c, at) == INVALID
        assert hip.g4_kv_extend_dev(c, at, 3, 4096, 4096) == 0
        assert hip.g4_kv_free_dev(c, at, 3, 4096) == 0
        hip.stub_capture(stream, 0)
        assert hip.g4_ctx_reserve(c, 96 << 20) == 0
        hip.stub_capture(stream, 1)
        assert hip.g4_kv_fork_dev(c, at, 3, 4096, 4096, None) == 0
        assert hip.g4_paged_attention_dev(c, at, 0, 1 << 20, 1 << 21, 8, 3, 4096, 1.0, 0, 0) == 0
        assert hip.g4_paged_prompt_dev(c, at, 0, 1 << 20, 1 << 21, 8, 3, 4096, 4096, 9, 1.0, 0, 0) == 0
        assert not [l for l in p.log() if l[0] == "malloc" and int(l[1]) > (128 << 20)]
        hip.stub_capture(stream, 0)
        p.use(None)


# ------------------------------------------------------------------- Python ---

def test_wrappers_refuse_what_is_not_on_the_device():
    ctx = type("C", (), {"handle": None, "ordinal": 0})()
    i, f = torch.zeros(4, dtype=torch.int32), torch.zeros(4096)
    with pytest.raises(g4hip.IllegalArgumentException):
        g4hip.KvCache(torch.zeros(1, 4, 2, 16, 64), torch.zeros(1, 4, 2, 16, 64), i.reshape(2, 2), i[:2], i, i[:1])
    with pytest.raises(g4hip.IllegalArgumentException):
        g4hip.Rope(torch.zeros(4, dtype=torch.float64))
    cache = type("K", (), {"on": lambda self, c: 0, "head_size": 64, "n_kv_heads": 2})()
    for call in (lambda: g4hip.kv_extend_dev(ctx, cache, i, i), lambda: g4hip.kv_fork_dev(ctx, cache, i, i),
                 lambda: g4hip.kv_compact_dev(ctx, cache, i, i, None, i, i), lambda: g4hip.kv_free_dev(ctx, cache, 4096),
                 lambda: g4hip.kv_trim_dev(ctx, cache, i.numpy(), 4), lambda: g4hip.rope_dev(ctx, cache, f, f, 1, 1, 64, i),
                 lambda: g4hip.kv_rope_write_dev(ctx, cache, 0, f, f, f, f, 2, None, i, None, 4),
                 lambda: g4hip.paged_attention_dev(ctx, cache, 0, f, f, 2, i),
                 lambda: g4hip.paged_prompt_dev(ctx, cache, 0, f, f, 2, i, i, 4)):
        with pytest.raises(g4hip.IllegalArgumentException):
            call()


def test_overlapping_rotations_are_refused(hip):
    """In place or apart: a result that begins inside its operand would be read half turned."""
    with Program(hip) as p:
        s = struct()
        r = g4hip._RopeStruct(4096, 64, 0, 1.0)
        at, rope, c = ctypes.addressof(s), ctypes.addressof(r), p.ctx
        size = 2 * 4 * 128 * 4  # 2 rows of 4 heads of 128 floats
        for off, want in ((0, 0), (16, INVALID), (-16, INVALID), (size - 16, INVALID), (size, 0), (-size, 0)):
            assert hip.g4_rope_dev(c, rope, 1 << 20, (1 << 20) + off, 2, 4, 128, 4096) == want
        size = 3 * 8 * s.head_size * 4
        for off, want in ((0, 0), (16, INVALID), (-16, INVALID), (size - 16, INVALID), (size, 0)):
            assert hip.g4_kv_rope_write_dev(c, at, 0, rope, 1 << 20, (1 << 20) + off, 4096, 4096, 8, 3, 4096, None,
                                            3) == want
