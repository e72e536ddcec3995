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
import struct

import torch

from . import _lib
from .packing import VALS_PER_WORD, packed_dim

__all__ = ["paged_append", "paged_decode", "paged_dequantize", "copy_pages", "paged_status"]

_workspaces: dict = {}           # (device index, stream, dim) -> scratch of the calls made on it outside of captures
_workspace_bytes: dict = {}      # (device index, dim) -> bytes: fixed by the SM count
_PACK = _lib.PAGED_PARAMS.pack   # tq_paged_params in one call: a launch's host time counts when its kernel takes 10 us
_SIZE = _lib.PAGED_PARAMS.size
_FORMATS = {torch.float32: _lib.TQ_F32, torch.float16: _lib.TQ_F16, torch.bfloat16: _lib.TQ_BF16}
_addressof = ctypes.addressof
_get_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_capturing = (torch._C._cuda_isCurrentStreamCapturing if hasattr(torch._C, "_cuda_isCurrentStreamCapturing")
              else torch.cuda.is_current_stream_capturing)
_raw_stream = _lib._raw_stream


def _call(fn, params: bytes, index: int) -> None:
    """One C call with device `index` current."""
    if index == _get_device():
        rc = fn(params)
    else:
        with torch.cuda.device(index):
            rc = fn(params)
    if rc:
        _lib.check(rc)


def _dtype(t: torch.Tensor) -> int:
    code = _FORMATS.get(t.dtype)
    return _lib.dtype_code(t.dtype) if code is None else code        # raises for anything else


def _table(x, count: int, what: str, keep: list) -> int:
    arr = _lib.host_floats(x)
    if arr is None or len(arr) != count:
        raise ValueError(f"{what}: {0 if arr is None else len(arr)} entries, {count} expected")
    keep.append(arr)
    return _addressof(arr)


def _half(desc: dict, what: str, dim: int | None, index: int, encode: bool, keep: list):
    """((pages, heads, page, dim), the tq_paged_half fields in front of `rows`) of a pool dict."""
    fmt = desc["format"]
    if fmt == "polar":
        packed, norms, bits = desc["packed"], desc["norms"], desc["bits"]
        if bits not in VALS_PER_WORD:
            raise ValueError(f"Unsupported bit width: {bits}. Use 1-4.")
        if dim is None:
            dim = desc["signs"].numel()
        shape, st, ns = packed.shape, packed.stride(), norms.stride()
        words = packed_dim(dim, bits)
        if packed.dtype is not torch.uint32 or len(shape) != 4 or st[3] != 1 or st[2] != words or shape[3] != words:
            raise ValueError(f"{what}: packed must be (pages, heads, page, {words}) uint32 with contiguous rows")
        if norms.dtype is not torch.float32 or norms.shape != shape[:3] or ns[2] != 1:
            raise ValueError(f"{what}: norms must be float32 {tuple(shape[:3])}, contiguous along the page")
        if packed.get_device() != index or norms.get_device() != index:
            raise ValueError(f"{what}: all tensors must be on cuda:{index}")
        signs = _table(desc["signs"], dim, what + ": signs", keep)
        levels = 1 << bits
        cents = 0 if encode else _table(desc["centroids"], levels, what + ": centroids", keep)
        bounds = _table(desc["boundaries"], levels - 1, what + ": boundaries", keep) if encode else 0
        return (shape[0], shape[1], shape[2], dim), (_lib.TQ_KV_POLAR, bits, 0), (
            packed.data_ptr(), norms.data_ptr(), st[0], st[1], ns[0], ns[1], cents, bounds, signs)
    if fmt == "dense":
        data = desc["data"]
        shape, st = data.shape, data.stride()
        if len(shape) != 4 or st[3] != 1 or st[2] != shape[3] or (dim is not None and shape[3] != dim):
            raise ValueError(f"{what}: dense pages must be (pages, heads, page, dim) with contiguous rows")
        if data.get_device() != index:
            raise ValueError(f"{what}: all tensors must be on cuda:{index}")
        return tuple(shape), (_lib.TQ_KV_DENSE, 0, _dtype(data)), (data.data_ptr(), 0, st[0], st[1], 0, 0, 0, 0, 0)
    raise ValueError(f"{what}: unknown page format {fmt!r}")


_NO_ROWS = (0, 0, 0, 0)
_NO_HALF = (0,) * 17


def _lens(t, what: str, batch: int, index: int) -> int:
    if t.dtype is not torch.int32 or t.shape != (batch,) or (batch > 1 and t.stride(0) != 1) or t.get_device() != index:
        raise ValueError(f"{what} must be a contiguous int32 ({batch},) tensor on cuda:{index}")
    return t.data_ptr()


def _pages(page_table, seq_lens, what: str, index: int):
    """(batch, table address, its row stride, its width, address of the lengths)."""
    if not page_table.is_cuda or not seq_lens.is_cuda:
        raise RuntimeError("libtqb200 operates on CUDA tensors only (no CPU path)")
    if page_table.dtype is not torch.int32 or page_table.ndim != 2 or page_table.get_device() != index:
        raise ValueError(f"page_table must be an int32 (batch, width) tensor on cuda:{index}")
    batch, width = page_table.shape
    row, step = page_table.stride()
    if batch < 1 or width < 1 or (step != 1 and width > 1):
        raise ValueError("page_table must have at least one sequence and one page, and contiguous rows")
    return batch, page_table.data_ptr(), row, width, _lens(seq_lens, what, batch, index)


def paged_append(keys: torch.Tensor, values: torch.Tensor, *, k: dict, v: dict, page_table: torch.Tensor,
                 starts: torch.Tensor, counts: torch.Tensor | None = None) -> None:
    """Store the new tokens of a ragged batch in their pages, keys and values in one launch.

    keys / values (B, H, T, dim), float32, float16 or bfloat16, rows contiguous, other strides free: token t of
    sequence b goes to position starts[b] + t of its page table, for t < counts[b] (every t without `counts`); padded
    tokens behind counts[b] are not read.  Packed halves get the words and norms `fused_quantize` gives; dense halves
    are copied and need the pages' own type.  Two tokens of one call must not share a place (sequences that share a
    page must not both write it)."""
    _lib.require_cuda(keys, values)
    index = keys.get_device()
    if keys.ndim != 4 or keys.shape != values.shape:
        raise ValueError(f"keys and values must be (batch, heads, tokens, dim) alike, got {tuple(keys.shape)} and {tuple(values.shape)}")
    if values.get_device() != index:
        raise ValueError(f"values must be on cuda:{index}")
    B, H, T, dim = keys.shape
    batch, table, row, width, lens = _pages(page_table, starts, "starts", index)
    if batch != B:
        raise ValueError(f"page_table has {batch} sequences, keys have {B}")
    keep: list = []
    geo, k0, k1 = _half(k, "keys", dim, index, True, keep)
    vgeo, v0, v1 = _half(v, "values", dim, index, True, keep)
    if vgeo != geo:
        raise ValueError("the pools of keys and values must agree in pages, heads, page size and dim")
    if geo[1] != H:
        raise ValueError(f"the pool has {geo[1]} heads, the new rows {H}")
    if keys.stride(3) != 1:
        keys = keys.contiguous()
    if values.stride(3) != 1:
        values = values.contiguous()
    kt, vt = _dtype(keys), _dtype(values)
    if k0[0] == _lib.TQ_KV_DENSE and kt != k0[2] or v0[0] == _lib.TQ_KV_DENSE and vt != v0[2]:
        raise ValueError("rows stored in dense pages must have the pages' dtype")
    n = 0
    if counts is not None:
        _lib.require_cuda(counts)
        n = _lens(counts, "counts", B, index)
    ks, vs = keys.stride(), values.stride()
    _call(_lib.lib().tq_paged_append, _PACK(
        _SIZE, B, 0, H, dim, geo[2], geo[0], table, row, lens, n, T, width, 0, 0, 0.0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
        _raw_stream(index), *k0, kt, *k1, keys.data_ptr(), ks[0], ks[1], ks[2], *v0, vt, *v1, values.data_ptr(), vs[0], vs[1], vs[2]),
        index)


def paged_decode(q: torch.Tensor, *, k: dict, v: dict, page_table: torch.Tensor, seq_lens: torch.Tensor, attn_scale: float,
                 window: int = 0, sinks: int = 0, out: torch.Tensor | None = None, out_dtype=None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its pages: q (B, n_q, dim) -> (B, n_q, dim) in `out_dtype`
    (default q.dtype), the token being the last of seq_lens[b] positions.

    window > 0: the token sees positions >= seq_lens[b] - window and the first `sinks` ones (it counts itself, as
    `create_causal_mask` does); pages outside both may have been freed.  A sequence of length 0 gives zeros.
    Lengths beyond the table are cut to it.  `out` optionally names the tensor to write (rows contiguous).
    `workspace`: a zero-filled uint8 tensor of `paged_workspace_bytes` used by no other call that may be in flight
    together with this one; every call leaves it ready for the next.  Without it the calls of a stream share one, and a
    call captured in a CUDA graph gets one of its own from the graph's pool.

    The weights are 16-bit in the tensor-core kernel (head_dim 128, 3 / 4-bit values, 16-bit or 3 / 4-bit keys, 16-bit
    queries); float32 queries and every other shape take the 32-bit kernel."""
    if not q.is_cuda:
        _lib.require_cuda(q)
    index = q.get_device()
    if q.ndim != 3:
        raise ValueError(f"q must be (batch, heads, dim), got {tuple(q.shape)}")
    if q.stride(2) != 1:
        q = q.contiguous()
    B, n_q, dim = shape = q.shape
    batch, table, row, width, lens = _pages(page_table, seq_lens, "seq_lens", index)
    if batch != B:
        raise ValueError(f"page_table has {batch} sequences, q has {B}")
    keep: list = []
    geo, k0, k1 = _half(k, "keys", dim, index, False, keep)
    vgeo, v0, v1 = _half(v, "values", dim, index, False, keep)
    if vgeo != geo:
        raise ValueError("the pools of keys and values must agree in pages, heads, page size and dim")
    if n_q == 0 or n_q % geo[1]:
        raise ValueError(f"n_q_heads ({n_q}) must equal n_kv_heads ({geo[1]}) * n_rep")
    if window < 0 or sinks < 0 or (sinks and not window):
        raise ValueError(f"window ({window}) and sinks ({sinks}) must not be negative, and sinks need a window")
    if out is None:
        out = torch.empty(shape, dtype=out_dtype or q.dtype, device=q.device)
    elif out.shape != shape or out.stride(2) != 1 or out.get_device() != index or (out_dtype or out.dtype) != out.dtype:
        raise ValueError(f"out must be {tuple(shape)} on cuda:{index}, with a contiguous last dimension and of out_dtype")
    stream = _raw_stream(index)
    if workspace is not None:
        need = paged_workspace_bytes(index, dim)
        if workspace.dtype is not torch.uint8 or not workspace.is_contiguous() or workspace.get_device() != index or workspace.numel() < need:
            raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes on cuda:{index}")
        scratch = (workspace.data_ptr(), workspace.numel())
    elif _capturing():                                      # the graph's own, zeroed by every replay
        workspace = torch.zeros((paged_workspace_bytes(index, dim),), dtype=torch.uint8, device=q.device)
        scratch = (workspace.data_ptr(), workspace.numel())
    else:
        kept = _workspaces.get((index, stream, dim))
        if kept is None:
            need = paged_workspace_bytes(index, dim)
            workspace = torch.zeros((need,), dtype=torch.uint8, device=q.device)
            kept = _workspaces[(index, stream, dim)] = (workspace, (workspace.data_ptr(), need))
        scratch = kept[1]
    qs, os = q.stride(), out.stride()
    _call(_lib.lib().tq_paged_decode, _PACK(
        _SIZE, B, n_q, geo[1], dim, geo[2], geo[0], table, row, lens, 0, 0, width, _dtype(q), _dtype(out), attn_scale,
        min(window, 0x7fffffff), min(sinks, 0x7fffffff), q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1],
        *scratch, stream, *k0, 0, *k1, *_NO_ROWS, *v0, 0, *v1, *_NO_ROWS), index)
    return out


def paged_workspace_bytes(device, dim: int) -> int:
    """Bytes of scratch one `paged_decode` call uses on this device (whatever its batch and lengths)."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    need = _workspace_bytes.get((index, dim))
    if need is None:
        with torch.cuda.device(index):
            need = _workspace_bytes[(index, dim)] = _lib.lib().tq_paged_decode_workspace_bytes(dim)
    return need


def paged_dequantize(pool: dict, *, page_table: torch.Tensor, seq_lens: torch.Tensor, length: int, dtype=torch.float16,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Positions [0, length) of every sequence as dense rows: (B, H, length, dim) in `dtype`, the bits `dequant_fp16`
    and `packed_dequantize` give; rows at and behind seq_lens[b], and of pages that the sequence no longer holds
    (table entry -1), are zero.  Dense pools are gathered as they are.
    `out` optionally names the contiguous tensor to write."""
    _lib.require_cuda(page_table)
    index = page_table.get_device()
    B, table, row, width, lens = _pages(page_table, seq_lens, "seq_lens", index)
    keep: list = []
    (n_pages, H, page, dim), v0, v1 = _half(pool, "pages", None, index, False, keep)
    if length < 0:
        raise ValueError(f"length must not be negative, got {length}")
    if out is None:
        out = torch.empty((B, H, length, dim), dtype=dtype, device=page_table.device)
    elif out.shape != (B, H, length, dim) or not out.is_contiguous() or out.get_device() != index:
        raise ValueError(f"out must be a contiguous ({B}, {H}, {length}, {dim}) tensor on cuda:{index}")
    _call(_lib.lib().tq_paged_dequantize, _PACK(
        _SIZE, B, 0, H, dim, page, n_pages, table, row, lens, 0, length, width, 0, _dtype(out), 0.0, 0, 0, 0, 0, 0,
        out.data_ptr(), 0, 0, 0, 0, _raw_stream(index), *_NO_HALF, *v0, 0, *v1, *_NO_ROWS), index)
    return out


def _page_ids(ids, n_pages: int, what: str, index: int):
    """int32 ids on the device, from a list or a CPU tensor (checked here) or a CUDA tensor (checked by the kernel)."""
    if isinstance(ids, torch.Tensor) and ids.is_cuda:
        if ids.dtype is not torch.int32 or ids.ndim != 1 or not ids.is_contiguous() or ids.get_device() != index:
            raise ValueError(f"{what} must be a contiguous one-dimensional int32 tensor on cuda:{index}")
        return ids, None
    if _capturing():
        raise RuntimeError(f"copy_pages in a captured graph needs {what} as a CUDA tensor")
    host = [int(i) for i in ids]
    bad = [i for i in host if not 0 <= i < n_pages]
    if bad:
        raise ValueError(f"{what}: page {bad[0]} is outside the pool of {n_pages}")
    return torch.tensor(host, dtype=torch.int32, device=torch.device("cuda", index)), host


def copy_pages(pools, src, dst) -> None:
    """Copy page src[i] to page dst[i] in every tensor of `pools` (contiguous, the page dimension in front, e.g. the
    packed words and norms of all layers) in one launch (per 128 tensors): a fork's last page, a compaction.

    src / dst: lists or CPU tensors, which are checked here, or int32 CUDA tensors, of which the kernel only checks
    that they lie inside the pools.  No page may be written twice, or both read and written, by one call."""
    pools = list(pools)
    if not pools:
        return
    T = torch.Tensor                                        # method descriptors in map: one call per tensor, nothing else
    _lib.require_cuda(pools[0])
    index, n_pages = pools[0].get_device(), pools[0].shape[0]
    ptrs = list(map(T.data_ptr, pools))
    if (set(map(T.get_device, pools)) != {index} or any([t.size(0) != n_pages for t in pools])
            or not all(map(T.is_contiguous, pools)) or any([p & 15 for p in ptrs])):
        raise ValueError("pools must be contiguous CUDA tensors, 16-byte aligned, of one device and one number of pages")
    sizes = [t.nbytes for t in pools]
    (src, hs), (dst, hd) = _page_ids(src, n_pages, "src", index), _page_ids(dst, n_pages, "dst", index)
    n_pairs = src.numel()
    if n_pairs != dst.numel():
        raise ValueError(f"{n_pairs} source and {dst.numel()} target pages")
    if hd is not None and len(set(hd)) != len(hd):
        raise ValueError("a target page is named twice")
    if hs is not None and hd is not None and set(hs) & set(hd):
        raise ValueError("a page is both read and written")
    if n_pages == 0 or n_pairs == 0:
        return
    sizes = [s // n_pages for s in sizes]
    if any(s == 0 or s % 16 for s in sizes):
        raise ValueError("pages must be multiples of 16 bytes")
    n = len(ptrs)
    args = struct.pack(f"={n}Q{n}q", *ptrs, *sizes)
    base = ctypes.cast(ctypes.c_char_p(args), ctypes.c_void_p).value
    fn = _lib.lib().tq_copy_pages
    _call(lambda _p: fn(base, base + 8 * n, n, n_pages, src.data_ptr(), dst.data_ptr(), n_pairs, _raw_stream(index)), args, index)


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
