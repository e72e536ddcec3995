"""Paged TurboQuant caches: many sequences of different lengths over shared pools of pages, one pool per layer.
No counterpart in the reference (one growing array per layer and one length for the whole batch,
turboquant_mlx/cache.py:88-150); the words, norms and attention are those of `TurboQuantKVCache`.

`PagedSequences` is the bookkeeping all layers share: which page holds which positions of which sequence, and how
often a page is shared.  It moves no data except where a page must be copied (a shared page that is about to be
written, a compaction), which is one `copy_pages` launch for all layers.  `PagedTurboQuantCache` is one layer's pools
with the interface a model expects of a cache.  A step:

    seqs.begin([a, b], 1)                  # the active batch, and how many new tokens each sequence gets
    for every layer: cache.update_and_fetch(keys, values); attention through the hook (or cache.attention)

A sliding window (with sink tokens) belongs to the sequences: attention sees it, and pages that slid out are freed."""

from __future__ import annotations

import torch

from ._lib import stream_handle
from .cache import _Quantizer, _zero
from .packing import packed_dim
from .paged import copy_pages, paged_append, paged_decode, paged_dequantize, paged_workspace_bytes


class PagedSequences:
    """Pages, tables and lengths of the sequences of a batch server.

    n_pages pages of page_size positions (a power of two, 32 at least) in every layer's pools.  window > 0: a token
    sees the last `window` positions (itself included) and the first `sinks`."""

    def __init__(self, n_pages: int, page_size: int = 64, window: int = 0, sinks: int = 0, device=None):
        if page_size < 32 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of 2, at least 32, got {page_size}")
        if n_pages < 1:
            raise ValueError(f"n_pages must be positive, got {n_pages}")
        if window < 0 or sinks < 0 or (sinks and not window):
            raise ValueError(f"window ({window}) and sinks ({sinks}) must not be negative, and sinks need a window")
        self.n_pages, self.page_size, self.window, self.sinks = n_pages, page_size, window, sinks
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.layers: list = []
        self._free = list(range(n_pages - 1, -1, -1))       # taken from the end: low pages first
        self._refs = [0] * n_pages
        self._pages: dict = {}                              # sequence -> pages by position (-1: freed behind the window)
        self._lens: dict = {}
        self._next = 0
        self._drop_step()

    def _drop_step(self):
        """Forget the active step: its table may name pages that have moved or gone."""
        self.active: list = []
        self.table = self.starts = self.lens = self.counts = None
        self._host_starts: list = []
        self._host_lens: list = []
        self._host_counts: list = []
        self._most = 0
        self._scratch: dict = {}                            # (head_dim, stream) -> decode workspace, shared by the step's layers

    # ---- sequences --------------------------------------------------------------------------------------
    def add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lens[seq] = [], 0
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence with the contents of `seq`, sharing the pages that hold them until one of the two writes to them.
        Pages reserved for further tokens stay with `seq` alone: its replays write to them without another `begin`."""
        pages = self._pages[seq][:-(-self._lens[seq] // self.page_size)]
        new = self.add()
        for p in pages:
            if p >= 0:
                self._refs[p] += 1
        self._pages[new], self._lens[new] = pages, self._lens[seq]
        return new

    def free(self, seq: int) -> None:
        """Drop a sequence; pages nobody else shares become free."""
        self._release(self._pages.pop(seq))
        del self._lens[seq]
        if seq in self.active:
            self._drop_step()

    def trim(self, seq: int, n: int) -> int:
        """Remove the last n positions (at most all); returns how many."""
        n = min(n, self._lens[seq])
        if n <= 0:
            return 0
        keep = self._lens[seq] - n
        pages = self._pages[seq]
        if self.window and keep > 0 and any(p < 0 for p in pages[max(0, keep - self.window) // self.page_size:-(-keep // self.page_size)]):
            raise ValueError(f"cannot trim to {keep} positions: pages of their window have been freed")
        cut = -(-keep // self.page_size)
        self._release(pages[cut:])
        del pages[cut:]
        self._lens[seq] = keep
        if seq in self.active:
            self._drop_step()
        return n

    def length(self, seq: int) -> int:
        return self._lens[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def used_pages(self) -> int:
        return self.n_pages - len(self._free)

    # ---- pages ------------------------------------------------------------------------------------------
    def _release(self, pages) -> None:
        for p in pages:
            if p >= 0:
                self._refs[p] -= 1
                if self._refs[p] == 0:
                    self._free.append(p)

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def _pools(self) -> list:
        return [t for layer in self.layers for t in layer.pools()]

    def begin(self, ids, new_tokens=1, reserve: int = 0) -> None:
        """Start a step: `ids` are the active sequences, in batch order, each about to receive new_tokens positions (one
        number, or one per sequence).  Pages for them, and for `reserve` further tokens, are taken; pages behind the
        window are freed; shared pages that will be written are copied.  Raises MemoryError, with nothing changed, when
        the pool has too few free pages.  Work of the step before on other streams must have been joined to the current
        stream (its tables go back to the allocator, and its freed pages to other sequences)."""
        ids = list(ids)
        if len(set(ids)) != len(ids) or not ids:
            raise ValueError("a step needs at least one sequence, each named once")
        counts = [int(new_tokens)] * len(ids) if not hasattr(new_tokens, "__len__") else [int(c) for c in new_tokens]
        if len(counts) != len(ids) or min(counts) < 0 or max(counts) < 1 or reserve < 0:
            raise ValueError(f"{len(ids)} sequences, new tokens {counts}, reserve {reserve}")
        size = self.page_size
        todo, need, gone, writers = [], 0, [], {}            # writers: shared page -> active sequences that write to it
        for seq, c in zip(ids, counts):
            pages, start = self._pages[seq], self._lens[seq]
            want = -(-(start + c + (reserve if c else 0)) // size)
            first = start // size                            # page of the first new position
            shared = [i for i in range(first, min(want, len(pages))) if pages[i] >= 0 and self._refs[pages[i]] > 1] if c else []
            hidden = []
            if self.window:
                # the step attends from position `start`, a sequence that receives nothing from its last one
                hidden = [i for i in range(min(first, len(pages))) if pages[i] >= 0 and i * size >= self.sinks
                          and (i + 1) * size <= start + min(c, 1) - self.window]
                gone += [pages[i] for i in hidden]
            need += max(0, want - len(pages))
            for i in shared:
                writers[pages[i]] = writers.get(pages[i], 0) + 1
            todo.append((seq, start, c, want, shared, hidden))
        drops: dict = {}
        for p in gone:
            drops[p] = drops.get(p, 0) + 1
        freed = sum(1 for p, n in drops.items() if self._refs[p] == n)
        # each writer of a shared page copies it, except the last when nobody else is left
        need += sum(min(n, self._refs[p] - drops.get(p, 0) - 1) for p, n in writers.items())
        if need > len(self._free) + freed:
            raise MemoryError(f"the step needs {need} pages, {len(self._free) + freed} of {self.n_pages} are free")
        src, dst = [], []
        for seq, start, c, want, shared, hidden in todo:
            pages = self._pages[seq]
            self._release([pages[i] for i in hidden])
            for i in hidden:
                pages[i] = -1
        for seq, start, c, want, shared, hidden in todo:
            pages = self._pages[seq]
            for i in shared:
                if self._refs[pages[i]] == 1:                # the other owner has let go of it meanwhile
                    continue
                new = self._take()
                if i * size < start:                         # it holds positions of this sequence
                    src.append(pages[i])
                    dst.append(new)
                self._refs[pages[i]] -= 1
                pages[i] = new
            while len(pages) < want:
                pages.append(self._take())
            self._lens[seq] = start + c
        if src:
            copy_pages(self._pools(), src, dst)
        self.active = ids
        self._host_starts = [t[1] for t in todo]
        self._host_lens = [t[1] + t[2] for t in todo]
        self._host_counts = counts
        self._most = max(counts)
        self._scratch = {}
        width = max(1, max(len(self._pages[s]) for s in ids))
        rows = [self._pages[s] + [-1] * (width - len(self._pages[s])) for s in ids]
        # one upload: [starts | lens | counts | table]
        n = len(ids)
        flat = torch.tensor(self._host_starts + self._host_lens + counts + [p for r in rows for p in r], dtype=torch.int32)
        flat = flat.to(self.device)
        self.starts, self.lens, self.counts = flat[:n], flat[n:2 * n], flat[2 * n:3 * n]
        self.table = flat[3 * n:].view(n, width)

    def _workspace(self, dim: int):
        """Decode scratch of the step on the current stream: calls on different streams may run at the same time.  None in
        a capture, where the call takes scratch of the graph's own."""
        if torch.cuda.is_current_stream_capturing():
            return None
        key = dim, stream_handle(self.device)
        if key not in self._scratch:
            self._scratch[key] = torch.zeros((paged_workspace_bytes(self.device, dim),), dtype=torch.uint8, device=self.device)
        return self._scratch[key]

    def _one_token_step(self):
        if self._most > 1:
            raise ValueError(f"the step began with up to {self._most} tokens per sequence: only steps of at most one new token "
                             "per sequence are replayed")

    def advance_device(self) -> None:
        """One more token per active sequence that receives one, on the device only: the body of a captured decode step ends
        with it.  Sequences that began the step with 0 tokens stay where they are.  The pages must have been reserved
        (`begin(..., reserve=n)`); `advance` tells the host afterwards.  A captured step belongs to the `begin` in front of
        it: it reads that step's tables, and the next `begin` ends its use."""
        self._one_token_step()
        self.starts += self.counts
        self.lens += self.counts

    def advance(self, n: int) -> None:
        """Host lengths after n replays of a captured one-token step."""
        self._one_token_step()
        if n < 0:
            raise ValueError(f"{n} replays")
        grow = [n * c for c in self._host_counts]
        for seq, g in zip(self.active, grow):
            if self._lens[seq] + g > len(self._pages[seq]) * self.page_size:
                raise ValueError(f"sequence {seq} has no pages for {g} more tokens")
        for k, (seq, g) in enumerate(zip(self.active, grow)):
            self._lens[seq] += g
            self._host_starts[k] += g
            self._host_lens[k] += g

    def compact(self) -> int:
        """Move the used pages to the front of the pools, in one launch; returns how many moved.  The pages behind
        `used_pages` are free afterwards (`resize` can then give them back)."""
        used = [p for p in range(self.n_pages) if self._refs[p]]
        holes = [p for p in range(len(used)) if not self._refs[p]]
        moved = used[len(used) - len(holes):]
        if moved:
            if self.layers:
                copy_pages(self._pools(), moved, holes)
            to = dict(zip(moved, holes))
            for pages in self._pages.values():
                pages[:] = [to.get(p, p) for p in pages]
            for old, new in to.items():
                self._refs[new], self._refs[old] = self._refs[old], 0
            self._drop_step()
        self._free = list(range(self.n_pages - 1, len(used) - 1, -1))
        return len(moved)

    def resize(self, n_pages: int) -> None:
        """Grow or shrink every layer's pools to n_pages; pages that would be cut off must be free.  The pools are new
        tensors, so the active step ends here (a graph captured in it would go on with the old ones)."""
        if n_pages < 1 or any(self._refs[p] for p in range(n_pages, self.n_pages)):
            raise ValueError(f"pages behind {n_pages} are in use")
        self._drop_step()
        for layer in self.layers:
            layer._resize(n_pages)
        self._refs = (self._refs + [0] * n_pages)[:n_pages]
        self.n_pages = n_pages
        self._free = [p for p in range(n_pages - 1, -1, -1) if not self._refs[p]]


class PagedTurboQuantCache:
    """One layer's pages: packed keys and values (or, with k_bits = 0, keys kept in `dtype` as in the V-only cache).

    Same seeds, widths and words as `TurboQuantKVCache` (keys `seed`, values `seed + 1`)."""

    fused = True

    def __init__(self, sequences: PagedSequences, n_kv_heads: int, dim: int = 128, bits: int = 3, seed: int = 42,
                 k_bits: int | None = None, v_bits: int | None = None, dtype=torch.float16):
        self.sequences = sequences
        self.n_kv_heads, self.dim, self.seed = n_kv_heads, dim, seed
        self.k_bits = bits if k_bits is None else k_bits
        self.v_bits = bits if v_bits is None else v_bits
        self.dtype = dtype
        dev = sequences.device
        self._v_q = _Quantizer(dim, self.v_bits, seed + 1, dev)
        self._k_q = _Quantizer(dim, self.k_bits, seed, dev) if self.k_bits else None
        self.k, self.v = self._pool(self._k_q), self._pool(self._v_q)
        sequences.layers.append(self)

    def _pool(self, q):
        s = self.sequences
        shape = (s.n_pages, self.n_kv_heads, s.page_size)
        if q is None:
            return dict(format="dense", data=torch.zeros((*shape, self.dim), dtype=self.dtype, device=s.device))
        return dict(format="polar", packed=torch.zeros((*shape, packed_dim(self.dim, q.bits)), dtype=torch.uint32, device=s.device),
                    norms=torch.zeros(shape, dtype=torch.float32, device=s.device), bits=q.bits, signs=q.signs,
                    centroids=q.centroids, boundaries=q.boundaries)

    def pools(self) -> list:
        """The tensors that hold this layer's pages."""
        return [d[name] for d in (self.k, self.v) for name in ("data", "packed", "norms") if name in d]

    def _resize(self, n_pages):
        for d in (self.k, self.v):
            for name in ("data", "packed", "norms"):
                if name in d:
                    old = d[name]
                    new = torch.zeros((n_pages, *old.shape[1:]), dtype=old.dtype, device=old.device)
                    keep = min(n_pages, old.shape[0])
                    new[:keep] = old[:keep]
                    d[name] = new

    def _step(self):
        s = self.sequences
        if s.table is None:
            raise RuntimeError("no step is active: call begin() on the sequences first")
        return s

    # ---- the interface of a cache ----------------------------------------------------------------------
    @property
    def offset(self) -> int:
        """Position of the step's first new token (equal for all active sequences; pass positions explicitly, as
        `decode_step` takes them, where they differ)."""
        starts = set(self._step()._host_starts)
        if len(starts) != 1:
            raise ValueError("the active sequences differ in length")
        return starts.pop()

    def update_and_fetch(self, keys, values):
        """Store the step's new rows (B, H, T, dim), B = the active sequences; tokens behind a sequence's own count are
        padding.  Returns shape-only placeholders: attention reads the pages."""
        s = self._step()
        if keys.shape[0] != len(s.active) or keys.shape[1] != self.n_kv_heads:
            raise ValueError(f"keys are {tuple(keys.shape)}, the step has {len(s.active)} sequences and {self.n_kv_heads} heads")
        if keys.shape[2] < s._most:
            raise ValueError(f"{keys.shape[2]} tokens given, the step has up to {s._most} per sequence")
        paged_append(keys, values, k=self.k, v=self.v, page_table=s.table, starts=s.starts, counts=s.counts)
        B, H, _, D = keys.shape
        n = max(s._host_lens)
        return _zero(keys.dtype, keys.device).expand(B, H, n, D), _zero(values.dtype, values.device).expand(B, H, n, D)

    def make_mask(self, N, return_array: bool = False, window_size=None):
        """None for single tokens, "causal" otherwise (the window is the cache's own, not the mask's)."""
        if return_array or window_size is not None:
            raise ValueError("a paged cache keeps its window itself; array masks are not supported")
        return None if N == 1 else "causal"

    def attention(self, queries, scale: float, mask=None):
        """queries (B, n_q, T, dim) of the step's new tokens -> (B, n_q, T, dim) in their dtype.

        One token per sequence: `paged_decode`; a sequence that received none in this step is attended from its last
        position, as if the query were that token's (an empty one gives zeros).  Several: the sequences' rows are read
        back and the prompt kernel attends, causally and within the window; rows of padding tokens are zero."""
        s = self._step()
        B, n_q, T, D = queries.shape
        if not (mask is None or (isinstance(mask, str) and mask == "causal")):
            raise ValueError("paged attention takes no array masks")
        if B != len(s.active):
            raise ValueError(f"{B} queries, {len(s.active)} active sequences")
        if T == 1:
            out = paged_decode(queries[:, :, 0], k=self.k, v=self.v, page_table=s.table, seq_lens=s.lens, attn_scale=scale,
                               window=s.window, sinks=s.sinks, workspace=s._workspace(D))
            return out.unsqueeze(2)
        k, v = self.dequantized(queries.dtype)
        out = torch.zeros_like(queries)
        for b, (start, end) in enumerate(zip(s._host_starts, s._host_lens)):
            n = end - start
            if n:
                out[b:b + 1, :, :n] = _windowed_prompt(queries[b:b + 1, :, :n], k[b:b + 1, :, :end], v[b:b + 1, :, :end],
                                                       scale, s.window, s.sinks)
        return out

    def dequantized(self, dtype=None):
        """(K, V) (B, H, longest, dim) of the active sequences, zeros behind each and where pages were freed."""
        s = self._step()
        n = max(s._host_lens)
        return tuple(paged_dequantize(d, page_table=s.table, seq_lens=s.lens, length=n, dtype=dtype or self.dtype)
                     for d in (self.k, self.v))

    @property
    def nbytes(self) -> int:
        """Bytes of the pages in use."""
        s = self.sequences
        return sum(t.nbytes for t in self.pools()) // s.n_pages * s.used_pages

    def empty(self) -> bool:
        return self.sequences.used_pages == 0

    def is_trimmable(self) -> bool:
        return False           # per sequence: PagedSequences.trim


def _windowed_prompt(q, k, v, scale, window, sinks):
    """Causal prompt attention within a window: the tensor-core kernel where it covers the call, else the library's
    attention with the mask written out."""
    from .kernels import prefill_attention, prefill_supported
    if prefill_supported(q, k, v, "causal"):
        return prefill_attention(q, k, v, scale, causal=True, window=window, sinks=sinks)
    from .base import _dense_sdpa, create_causal_mask
    L, S = q.shape[2], k.shape[2]
    mask = create_causal_mask(L, offset=S - L, window_size=window or None, device=q.device)
    if sinks:
        rows = torch.arange(S - L, S, device=q.device)[:, None]
        at = torch.arange(S, device=q.device)
        mask = mask | ((at < sinks) & (at <= rows))
    return _dense_sdpa(q, k, v, scale, mask)


def make_paged_caches(num_layers: int, n_pages: int, n_kv_heads: int, dim: int = 128, bits: int = 3, page_size: int = 64,
                      window: int = 0, sinks: int = 0, k_bits: int | None = None, v_bits: int | None = None, seed: int = 42,
                      dtype=torch.float16, device=None) -> list:
    """One paged cache per layer over one `PagedSequences` (`caches[0].sequences`)."""
    seqs = PagedSequences(n_pages, page_size, window, sinks, device)
    return [PagedTurboQuantCache(seqs, n_kv_heads, dim, bits, seed, k_bits, v_bits, dtype) for _ in range(num_layers)]
