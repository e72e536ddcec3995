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


def test_replays_after_a_fork_write_to_pages_of_their_own(tq):
    """Pages reserved by an earlier step belong to the sequence they were taken for, not to its forks: whatever `advance`
    accepts ends in pages that nobody else holds."""
    seqs = _seqs(tq, n_pages=12)
    a = seqs.add()
    seqs.begin([a], 1, reserve=90)
    b = seqs.fork(a)
    assert seqs.used_pages == 3 and len(seqs._pages[b]) == 1
    seqs.begin([a, b], 1)
    for s in (a, b):
        for p in seqs._pages[s][seqs._host_starts[0] // 32:]:
            assert seqs._refs[p] == 1
    with pytest.raises(ValueError, match=f"sequence {b} has no pages"):
        seqs.advance(60)                                   # nothing is reserved for b
    seqs.begin([a, b], 1, reserve=60)
    seqs.advance(60)
    assert not set(seqs._pages[a]) & set(seqs._pages[b])
    assert seqs.length(a) == seqs.length(b) == 63


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_places_written_by_replays_are_private(tq, monkeypatch, window, sinks):
    """Random histories with forks, reserves and replays: every place a replay writes lies in a page of one sequence, what
    a step sees is held, and contents stay those of the sequence."""
    import turboquant_mlx_b200.paged_cache as pc
    for seed in range(30):
        rng = random.Random(seed)
        seqs = _seqs(tq, rng.choice([12, 30, 80]), window=window, sinks=sinks)
        place, text, token = {}, {}, 0

        def copy(_pools, src, dst):
            assert len(set(dst)) == len(dst) and not set(src) & set(dst)
            for s, d in zip(src, dst):
                for r in range(32):
                    place[d, r] = place.get((s, r))
        monkeypatch.setattr(pc, "copy_pages", copy)
        seqs.layers.append(type("L", (), {"pools": lambda self: [], "_resize": lambda self, n: None})())

        def write(s, pos):
            nonlocal token
            page = seqs._pages[s][pos // 32]
            assert page >= 0 and seqs._refs[page] == 1
            place[page, pos % 32] = token
            text[s].append(token)
            token += 1

        for _ in range(200):
            op = rng.choice(["step", "step", "step", "add", "fork", "free", "trim", "compact"])
            if op == "add":
                text[seqs.add()] = []
            elif op == "fork" and text:
                s = rng.choice(list(text))
                text[seqs.fork(s)] = list(text[s])
            elif op == "free" and text:
                s = rng.choice(list(text))
                seqs.free(s)
                del text[s]
            elif op == "trim" and text:
                s = rng.choice(list(text))
                try:
                    n = seqs.trim(s, rng.randint(1, 50))
                except ValueError:
                    assert window
                    continue
                text[s] = text[s][:len(text[s]) - n]
            elif op == "compact":
                seqs.compact()
            elif op == "step" and text:
                ids = rng.sample(list(text), rng.randint(1, len(text)))
                counts = [rng.choice([0, 1, 1, 1] if rng.random() < 0.6 else [0, 1, 40]) for _ in ids]
                if max(counts) == 0:
                    continue
                try:
                    seqs.begin(ids, counts, reserve=rng.choice([0, 0, 70]))
                except MemoryError:
                    continue
                for s, c in zip(ids, counts):
                    _assert_visible_held(seqs, s, len(text[s]) + min(c, 1) - 1)
                    for pos in range(len(text[s]), len(text[s]) + c):
                        write(s, pos)
                if rng.random() < 0.3:
                    s = rng.choice(ids)
                    text[seqs.fork(s)] = list(text[s])
                if max(counts) == 1:
                    n = rng.randint(0, 40)
                    try:
                        seqs.advance(n)
                    except ValueError:
                        n = 0
                    for _ in range(n):
                        for s, c in zip(ids, counts):
                            if c:
                                page = seqs._pages[s][len(text[s]) // 32]
                                # a fork made inside the step may share the page in hand, but not what is written now
                                assert page >= 0 and all(o == s or seqs.length(o) <= len(text[s]) or
                                                         page not in seqs._pages[o] for o in text)
                                place[page, len(text[s]) % 32] = token
                                text[s].append(token)
                                token += 1
            for s, want in text.items():
                assert seqs.length(s) == len(want)
                for i, t in enumerate(want):
                    page = seqs._pages[s][i // 32]
                    assert page < 0 and window or place[page, i % 32] == t


def test_forks_that_write_together_need_one_page_less(tq, monkeypatch):
    """The last of the sequences that share a page keeps it: a pool with room for the others' copies is enough, and one
    page less is refused with nothing changed."""
    import turboquant_mlx_b200.paged_cache as pc
    copied = []
    monkeypatch.setattr(pc, "copy_pages", lambda pools, src, dst: copied.append((src, dst)))
    for n_forks, idle in ((1, 0), (3, 0), (3, 2)):
        for spare in (0, -1):
            copies = n_forks + (idle > 0)                  # an idle fork keeps the page, so every writer copies
            n_pages = 1 + copies + spare
            seqs = _seqs(tq, n_pages)
            seqs.layers.append(type("L", (), {"pools": lambda self: []})())
            a = seqs.add()
            seqs.begin([a], 10)
            ids = [a] + [seqs.fork(a) for _ in range(n_forks)]
            for _ in range(idle):
                seqs.fork(a)
            copied.clear()
            if spare:
                with pytest.raises(MemoryError):
                    seqs.begin(ids, 1)
                assert [seqs.length(s) for s in ids] == [10] * len(ids) and not copied
            else:
                seqs.begin(ids, 1)
                assert seqs.free_pages == 0 and len({seqs._pages[s][0] for s in ids}) == len(ids)
                assert sum(len(src) for src, _ in copied) == copies


def test_a_page_that_slides_out_of_one_fork_is_kept_by_the_other(tq, monkeypatch):
    """A page that one active sequence frees behind its window while the other writes to it needs no copy."""
    import turboquant_mlx_b200.paged_cache as pc
    monkeypatch.setattr(pc, "copy_pages", lambda pools, src, dst: pytest.fail("copied"))
    seqs = _seqs(tq, 3, window=32)
    seqs.layers.append(type("L", (), {"pools": lambda self: []})())
    a = seqs.add()
    seqs.begin([a], 64)
    b = seqs.fork(a)
    seqs.trim(b, 44)
    first = seqs._pages[a][0]
    assert seqs._pages[b] == [first] and seqs.free_pages == 1
    seqs.begin([a, b], 1)
    assert seqs._pages[a][0] == -1 and seqs._pages[b] == [first] and seqs.free_pages == 0


def test_step_scratch_belongs_to_a_stream(tq, monkeypatch):
    """Attention calls of a step on two streams may run at the same time, so they do not share decode scratch; within a
    capture the call brings its own."""
    import types
    import torch
    import turboquant_mlx_b200.paged_cache as pc
    now = types.SimpleNamespace(stream=11, capturing=False)
    monkeypatch.setattr(pc, "paged_workspace_bytes", lambda device, dim: 64)
    monkeypatch.setattr(pc, "stream_handle", lambda device: now.stream, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now.capturing)
    seqs = _seqs(tq)
    a = seqs.add()
    seqs.begin([a], 1)
    first = seqs._workspace(128)
    assert first is seqs._workspace(128) and first is not seqs._workspace(64)
    now.stream = 12
    second = seqs._workspace(128)
    assert second is not first and second.data_ptr() != first.data_ptr() and not second.any()
    now.stream = 11
    assert seqs._workspace(128) is first
    now.capturing = True
    assert seqs._workspace(128) is None                    # a graph's scratch is the graph's
    now.capturing = False
    seqs.begin([a], 1)
    assert seqs._workspace(128) is not first
