"""Kernel-level API of the paged caches: insert, decode attention, read-back and page copies on pools whose pages
belong to many sequences.  No counterpart in the reference, whose caches are one array per layer and whose batches
share one length (turboquant_mlx/cache.py:42-150).

Vocabulary (all tensors CUDA, on one device):
  pool        k / v dicts like those of `flash_decode`, with the pages in front:
                polar: dict(format="polar", packed (P, H, page, words) uint32, norms (P, H, page) float32, bits, signs,
                            centroids (to read), boundaries (to insert))
                dense: dict(format="dense", data (P, H, page, dim))       [keys of the V-only configuration]
              page is a power of two, 32 at least; the page and head strides are free, rows are contiguous.
  page_table  (B, width) int32: pool page of positions [i * page, (i + 1) * page) of sequence b.  Entries behind a
              sequence, or wholly outside its window, are never read (-1, by convention).
  seq_lens    (B,) int32, read when the kernel runs: a captured step can be replayed while they advance.
A page id outside the pool is never followed: inserts skip the row, results become NaN, and `paged_status` says so.
`paged_cache` keeps tables and pools for a model; these are the calls it makes."""

from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["paged_append", "paged_decode", "paged_dequantize", "copy_pages", "paged_status"]


def paged_append(keys: torch.Tensor, values: torch.Tensor, *, k: dict, v: dict, page_table: torch.Tensor,
                 starts: torch.Tensor, counts: torch.Tensor | None = None) -> None:
    """Store the new tokens of a ragged batch in their pages, keys and values in one launch.

    keys / values (B, H, T, dim), float32, float16 or bfloat16, rows contiguous, other strides free: token t of
    sequence b goes to position starts[b] + t of its page table, for t < counts[b] (every t without `counts`); padded
    tokens behind counts[b] are not read.  Packed halves get the words and norms `fused_quantize` gives; dense halves
    are copied and need the pages' own type.  Two tokens of one call must not share a place (sequences that share a
    page must not both write it)."""
    (_lib.native or _lib.load_native()).append(keys, values, k, v, page_table, starts, counts)


def paged_decode(q: torch.Tensor, *, k: dict, v: dict, page_table: torch.Tensor, seq_lens: torch.Tensor, attn_scale: float,
                 window: int = 0, sinks: int = 0, out: torch.Tensor | None = None, out_dtype=None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its pages: q (B, n_q, dim) -> (B, n_q, dim) in `out_dtype`
    (default q.dtype), the token being the last of seq_lens[b] positions.

    window > 0: the token sees positions >= seq_lens[b] - window and the first `sinks` ones (it counts itself, as
    `create_causal_mask` does); pages outside both may have been freed.  A sequence of length 0 gives zeros.
    Lengths beyond the table are cut to it.  `out` optionally names the tensor to write (rows contiguous).
    `workspace`: a zero-filled uint8 tensor of `paged_workspace_bytes` used by no other call that may be in flight
    together with this one; every call leaves it ready for the next.  Without it the calls of a stream share one, and the
    calls captured in a CUDA graph one per stream of the capture, from the graph's pool, zeroed by every replay.

    The weights are 16-bit in the tensor-core kernel (head_dim 128, 3 / 4-bit values, 16-bit or 3 / 4-bit keys, 16-bit
    queries); float32 queries and every other shape take the 32-bit kernel."""
    return (_lib.native or _lib.load_native()).decode(q, k, v, page_table, seq_lens, attn_scale, window, sinks, out, out_dtype, workspace)


def paged_workspace_bytes(device, dim: int) -> int:
    """Bytes of scratch one `paged_decode` call uses on this device (whatever its batch and lengths)."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    with torch.cuda.device(index):
        return _lib.lib().tq_paged_decode_workspace_bytes(dim)


def paged_dequantize(pool: dict, *, page_table: torch.Tensor, seq_lens: torch.Tensor, length: int, dtype=torch.float16,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Positions [0, length) of every sequence as dense rows: (B, H, length, dim) in `dtype`, the bits `dequant_fp16`
    and `packed_dequantize` give; rows at and behind seq_lens[b], and of pages that the sequence no longer holds
    (table entry -1), are zero.  Dense pools are gathered as they are.
    `out` optionally names the contiguous tensor to write."""
    return (_lib.native or _lib.load_native()).dequantize(pool, page_table, seq_lens, length, dtype, out)


def copy_pages(pools, src, dst) -> None:
    """Copy page src[i] to page dst[i] in every tensor of `pools` (contiguous, the page dimension in front, e.g. the
    packed words and norms of all layers) in one launch (per 128 tensors): a fork's last page, a compaction.

    src / dst: lists or CPU tensors, which are checked here, or int32 CUDA tensors, of which the kernel only checks
    that they lie inside the pools.  No page may be written twice, or both read and written, by one call."""
    (_lib.native or _lib.load_native()).copy_pages(pools, src, dst)


def paged_status(device) -> int:
    """What the paged kernels found wrong on this device since the last call (synchronises the current stream): 0
    nothing, 1 a page id outside the pool, 2 a position behind the page table, 3 a bounded wait that gave up, 4 a
    decode kernel that found its shared memory elsewhere than it counts on (3 and 4 are faults of the library)."""
    device = torch.device(device)
    word = ctypes.c_int(0)
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("paged_status cannot be captured in a CUDA graph")
        _lib.check(_lib.lib().tq_paged_status(ctypes.byref(word), torch.cuda.current_stream(device).cuda_stream))
    return word.value
