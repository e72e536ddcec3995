"""Steps of a paged batch in which the sequences differ in what they receive, on a GPU, against 64-bit references."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as pr  # noqa: E402

pytestmark = pytest.mark.gpu
D = 128
SCALE = 1 / math.sqrt(D)


class _Half:
    """A cache half seen by the 64-bit reference."""

    def __init__(self, cache, desc, q):
        self.bits, self.dim, self.page = (q.bits if q else 0), cache.dim, cache.sequences.page_size
        if q is None:
            self.data = desc["data"]
        else:
            self.packed, self.norms, self.quant = desc["packed"], desc["norms"], q

    rotated, rows = pr.Pool.rotated, pr.Pool.rows


def _check(tq, cache, q, out, lens):
    """A single-token step's attention against 64 bits; its weights are 16-bit."""
    s = cache.sequences
    ref, tol = pr.decode_ref(tq, q[:, :, 0], _Half(cache, cache.k, cache._k_q), _Half(cache, cache.v, cache._v_q), s.table,
                             lens, SCALE, s.window, s.sinks, torch.finfo(torch.float16).eps / 2, q.dtype)
    pr.check(out[:, :, 0], ref, tol)


def _rows(B, H, T, dev, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((B, H, T, D), generator=g).half().to(dev) for _ in range(2)]


def _query(B, n_q, dev, seed):
    return torch.randn((B, n_q, 1, D), generator=torch.Generator().manual_seed(seed)).half().to(dev)


@pytest.mark.parametrize("k_bits", [0, 3])
@pytest.mark.parametrize("n,window,sinks", [(95, 64, 0), (163, 100, 4), (195, 100, 4), (96, 64, 0)])
def test_a_waiting_sequence_keeps_its_window(tq, dev, k_bits, n, window, sinks):
    """At these lengths the window of a sequence that receives nothing begins at the end of a page (and, last, behind it)."""
    cache, = tq.make_paged_caches(1, 20, 2, k_bits=k_bits, page_size=32, window=window, sinks=sinks)
    seqs = cache.sequences
    ids = [seqs.add(), seqs.add()]
    seqs.begin(ids, n)
    cache.update_and_fetch(*_rows(2, 2, n, dev, n))
    seqs.begin(ids, [1, 0])
    cache.update_and_fetch(*_rows(2, 2, 1, dev, n + 1))
    q = _query(2, 8, dev, n)
    out = cache.attention(q, SCALE)
    assert tq.paged_status(dev) == 0
    _check(tq, cache, q, out, [n + 1, n])


def test_a_waiting_sequence_in_a_replayed_step(tq, dev):
    """A captured step with a sequence that receives nothing, replayed over the end of its page: it neither grows nor
    changes, and the one that receives grows as in eager steps."""
    cache, = tq.make_paged_caches(1, 12, 2, page_size=32)
    seqs = cache.sequences
    ids = [seqs.add(), seqs.add()]
    seqs.begin(ids, 31)
    cache.update_and_fetch(*_rows(2, 2, 31, dev, 0))
    keys, values = _rows(2, 2, 1, dev, 1)
    q = _query(2, 8, dev, 2)
    seqs.begin(ids, [1, 0], reserve=4)

    def step():
        cache.update_and_fetch(keys, values)
        out = cache.attention(q, SCALE)
        seqs.advance_device()
        return out

    first = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(33, 37):
        graph.replay()
        assert seqs.lens.tolist() == [n + 1, 31]                # of the step to come
        _check(tq, cache, q, out, [n, 31])
        assert torch.equal(out[1], first[1])
    seqs.advance(4)
    assert [seqs.length(s) for s in ids] == [36, 31] and tq.paged_status(dev) == 0


def _three_layers(tq, dev, n=700):
    """Caches of three layers with different rows, one query each, and what attention gives one after the other."""
    caches = tq.make_paged_caches(3, 60, 2, page_size=32)
    seqs = caches[0].sequences
    ids = [seqs.add(), seqs.add()]
    seqs.begin(ids, [n, 3])
    for i, c in enumerate(caches):
        c.update_and_fetch(*_rows(2, 2, n, dev, i))
    seqs.begin(ids, 1)
    for i, c in enumerate(caches):
        c.update_and_fetch(*_rows(2, 2, 1, dev, 10 + i))
    qs = [_query(2, 8, dev, 20 + i) for i in range(3)]
    want = [c.attention(q, SCALE) for c, q in zip(caches, qs)]
    for c, q, w in zip(caches, qs, want):
        _check(tq, c, q, w, [n + 1, 4])
    return caches, qs, want


def test_layers_of_a_step_on_two_streams(tq, dev):
    """Two layers of a step attended at the same time on two streams, many times over: each stream has its own scratch."""
    caches, qs, want = _three_layers(tq, dev)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    outs = [[], []]
    for _ in range(40):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(caches[i].attention(qs[i], SCALE))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_layers_of_a_captured_step(tq, dev):
    """One graph with all layers, one with its layers on two branches: right in every replay, also side by side with each
    other and with eager calls."""
    caches, qs, want = _three_layers(tq, dev)
    torch.cuda.synchronize()
    main, side = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    chain, fork = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(chain, stream=main):
        a = [c.attention(q, SCALE) for c, q in zip(caches, qs)]
    with torch.cuda.graph(fork, stream=main):
        b = [caches[0].attention(qs[0], SCALE)]
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b.append(caches[1].attention(qs[1], SCALE))
        b.append(caches[2].attention(qs[2], SCALE))
        main.wait_stream(side)
    for t in a + b:
        t.zero_()
    torch.cuda.synchronize()
    eager = []
    for _ in range(20):
        with torch.cuda.stream(main):
            chain.replay()
        with torch.cuda.stream(side):
            fork.replay()
        eager.append(caches[0].attention(qs[0], SCALE))
    torch.cuda.synchronize()
    for got in (a, b):
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert all(torch.equal(e, want[0]) for e in eager) and tq.paged_status(dev) == 0
