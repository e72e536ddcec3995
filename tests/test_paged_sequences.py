"""Bookkeeping of the paged caches (no GPU: a PagedSequences without layers moves no data): every position of every
sequence stays in a page of its own or in one it rightly shares, through forks, trims, windows and compaction."""
import random

import pytest
import torch


@pytest.fixture()
def make(tq):
    def build(n_pages=40, **kw):
        return tq.PagedSequences(n_pages, device="cpu", page_size=32, **kw)
    return build


def _check(seqs):
    refs = [0] * seqs.n_pages
    for seq, pages in seqs._pages.items():
        assert len(pages) >= -(-seqs._lens[seq] // seqs.page_size)
        for p in pages:
            if p >= 0:
                refs[p] += 1
    assert refs == seqs._refs
    assert sorted(seqs._free) == [p for p in range(seqs.n_pages) if refs[p] == 0]
    assert seqs.free_pages + seqs.used_pages == seqs.n_pages


def test_random_histories(make, monkeypatch, tq):
    """A model of the contents (which token each place holds) follows every operation."""
    import turboquant_mlx_b200.paged_cache as pc
    for seed in range(30):
        rng = random.Random(seed)
        seqs = make(n_pages=rng.choice([6, 20, 60]))
        place = {}                                       # (page, row) -> token
        text = {}                                        # sequence -> its tokens

        def copy(_pools, src, dst):
            assert len(set(dst)) == len(dst) and not set(src) & set(dst)
            for s, d in zip(src, dst):
                for r in range(32):
                    place[d, r] = place.get((s, r))
        monkeypatch.setattr(pc, "copy_pages", copy)
        seqs.layers.append(type("L", (), {"pools": lambda self: [], "_resize": lambda self, n: None})())
        token = 0
        for _ in range(120):
            op = rng.choice(["begin", "begin", "begin", "add", "fork", "free", "trim", "compact"])
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
                n = rng.randint(0, 70)
                assert seqs.trim(s, n) == min(n, len(text[s]))
                text[s] = text[s][:max(0, len(text[s]) - n)]
            elif op == "compact":
                used = seqs.used_pages
                seqs.compact()
                assert all(p < used for pages in seqs._pages.values() for p in pages) and seqs.used_pages == used
            elif op == "begin" and text:
                ids = rng.sample(list(text), rng.randint(1, len(text)))
                counts = [rng.choice([0, 1, 1, 5, 32, 50]) for _ in ids]
                if max(counts) == 0:
                    continue
                before = (dict(seqs._lens), [list(p) for p in seqs._pages.values()], list(seqs._refs))
                try:
                    seqs.begin(ids, counts, reserve=rng.choice([0, 0, 40]))
                except MemoryError:
                    assert before == (dict(seqs._lens), [list(p) for p in seqs._pages.values()], list(seqs._refs))
                    continue
                assert seqs.lens.tolist() == [len(text[s]) + c for s, c in zip(ids, counts)]
                assert seqs.starts.tolist() == [len(text[s]) for s in ids]
                for b, (s, c) in enumerate(zip(ids, counts)):          # what an insert would do with the device table
                    for pos in range(len(text[s]), len(text[s]) + c):
                        place[int(seqs.table[b, pos // 32]), pos % 32] = token
                        text[s].append(token)
                        token += 1
            _check(seqs)
            for s, want in text.items():
                assert seqs.length(s) == len(want)
                assert [place[seqs._pages[s][i // 32], i % 32] for i in range(len(want))] == want


def test_window_frees_pages(make):
    seqs = make(n_pages=12, window=64, sinks=3)
    s = seqs.add()
    for step in range(40):
        seqs.begin([s], 10)
        n = seqs.length(s)
        first = n - 10                                    # the step's first token sees > first - 64
        pages = seqs._pages[s]
        for p in range(n):
            seen = p < 3 or p > first - 64
            if seen:
                assert pages[p // 32] >= 0, (n, p)
        assert sum(p >= 0 for p in pages) <= 1 + -(-(64 + 10) // 32) + 1
        _check(seqs)
    assert pages[0] >= 0 and pages[1] == -1               # the sinks' page stays
    with pytest.raises(ValueError, match="window have been freed"):
        seqs.trim(s, 200)
    seqs.free(s)
    assert seqs.free_pages == 12


def test_window_pages_shared_with_a_fork_stay(make):
    seqs = make(n_pages=12, window=32)
    a = seqs.add()
    seqs.begin([a], 100)
    b = seqs.fork(a)
    kept = list(seqs._pages[b])
    for _ in range(5):
        seqs.begin([a], 32)
    assert seqs._pages[b] == kept and all(seqs._refs[p] >= 1 for p in kept)
    _check(seqs)


def test_resize(make):
    seqs = make(n_pages=8)
    a, b = seqs.add(), seqs.add()
    seqs.begin([a, b], 64)
    seqs.free(a)
    with pytest.raises(ValueError, match="in use"):
        seqs.resize(2)
    assert seqs.compact() == 2 and seqs.used_pages == 2
    seqs.resize(2)
    assert seqs.free_pages == 0 and sorted(seqs._pages[b]) == [0, 1]
    seqs.resize(5)
    assert seqs.free_pages == 3
    _check(seqs)


def test_refusals(make, tq):
    for bad in (dict(page_size=48), dict(page_size=16), dict(window=-1), dict(sinks=2), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            tq.PagedSequences(4, device="cpu", **bad)
    with pytest.raises(ValueError):
        tq.PagedSequences(0, device="cpu")
    seqs = make(n_pages=4)
    s = seqs.add()
    for ids, n in (([], 1), ([s, s], 1), ([s], 0), ([s], [1, 2]), ([s], -1)):
        with pytest.raises(ValueError):
            seqs.begin(ids, n)
    with pytest.raises(KeyError):
        seqs.begin([s + 1], 1)
    with pytest.raises(MemoryError):
        seqs.begin([s], 129)
    assert seqs.length(s) == 0 and seqs.table is None
    seqs.begin([s], 1, reserve=20)
    with pytest.raises(ValueError, match="no pages"):
        seqs.advance(100)
    seqs.advance(20)
    assert seqs.length(s) == 21
    assert seqs.trim(s, 0) == 0 and seqs.trim(s, 1000) == 21 and seqs.length(s) == 0


def test_steps_end_with_what_invalidates_them(make):
    """After a trim, a free or a compaction of active sequences the device table is gone, not stale."""
    seqs = make()
    a, b = seqs.add(), seqs.add()
    for what in (lambda: seqs.trim(a, 1), lambda: seqs.free(b)):
        seqs.begin([a] if b not in seqs._pages else [a, b], 40)
        what()
        assert seqs.table is None and not seqs.active
    c = seqs.add()
    seqs.begin([c], 40)
    seqs.free(a)
    assert seqs.table is not None                         # another sequence: the step stands
    seqs.compact()
    assert seqs.table is None or torch.equal(seqs.table[0].cpu(), torch.tensor(seqs._pages[c], dtype=torch.int32))
