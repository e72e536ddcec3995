"""Steps of a batch in which the sequences differ in what they receive (no GPU: a PagedSequences without layers moves no
data): what the step's attention reads is held, and what its replays write is the sequence's own."""
import random

import pytest


def _seqs(tq, n_pages=40, **kw):
    return tq.PagedSequences(n_pages, device="cpu", page_size=32, **kw)


def _assert_visible_held(seqs, seq, first):
    """Every position that a token at `first` or behind it sees has a page."""
    pages, n = seqs._pages[seq], seqs.length(seq)
    for p in range(n):
        if not seqs.window or p < seqs.sinks or p > first - seqs.window:
            assert pages[p // 32] >= 0, (n, p, pages)


@pytest.mark.parametrize("window,sinks", [(1, 0), (32, 0), (64, 0), (100, 4), (33, 40)])
def test_a_waiting_sequence_keeps_its_window(tq, window, sinks):
    """A sequence that receives nothing in a step attends from its last token (position length - 1), whatever its length
    relative to the pages; one that receives a token attends from that."""
    for n in range(1, 200):
        seqs = _seqs(tq, window=window, sinks=sinks)
        a, b = seqs.add(), seqs.add()
        seqs.begin([a, b], n)
        seqs.begin([a, b], [1, 0])
        _assert_visible_held(seqs, a, n)
        _assert_visible_held(seqs, b, n - 1)
        seqs.begin([b], 1)
        _assert_visible_held(seqs, b, n)


def test_replays_advance_only_what_receives(tq):
    """A captured one-token step replayed: a sequence that began it with 0 tokens stays where it is, on the device and on
    the host; steps of several tokens cannot be replayed as one-token steps."""
    seqs = _seqs(tq)
    a, b, c = seqs.add(), seqs.add(), seqs.add()
    seqs.begin([a, b, c], [31, 10, 0], reserve=7)
    with pytest.raises(ValueError, match="one new token"):
        seqs.advance_device()
    with pytest.raises(ValueError, match="one new token"):
        seqs.advance(1)
    assert [seqs.length(s) for s in (a, b, c)] == [31, 10, 0] and seqs.starts.tolist() == [0, 0, 0]
    seqs.begin([a, b, c], [1, 0, 0], reserve=5)
    for k in range(3):
        assert seqs.starts.tolist() == [31 + k, 10, 0] and seqs.lens.tolist() == [32 + k, 10, 0]
        seqs.advance_device()
    seqs.advance(2)
    assert [seqs.length(s) for s in (a, b, c)] == [34, 10, 0]
    assert seqs._host_starts == [33, 10, 0] and seqs._host_lens == [34, 10, 0]
    with pytest.raises(ValueError, match="no pages"):
        seqs.advance(100)
    with pytest.raises(ValueError):
        seqs.advance(-1)
    assert [seqs.length(s) for s in (a, b, c)] == [34, 10, 0]
