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
from .packing import VALS_PER_WORD, packed_dim

__all__ = ["paged_append", "paged_decode", "paged_dequantize", "copy_pages", "paged_status"]

_workspace_bytes: dict = {}      # (device index, dim) -> bytes: fixed by the SM count
_ERR_CPU = "libtqb200 operates on CUDA tensors only (no CPU path)"


class _on:
    """The current device is `dev` inside the block (free when it already is)."""

    def __init__(self, dev):
        self.guard = None if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _half(H, desc: dict, what: str, dim: int | None, dev, encode: bool):
    """Fill a tq_paged_half from a pool dict; returns (pages, heads, page, dim)."""
    fmt = desc["format"]
    if fmt == "polar":
        packed, norms, bits = desc["packed"], desc["norms"], desc["bits"]
        if bits not in VALS_PER_WORD:
            raise ValueError(f"Unsupported bit width: {bits}. Use 1-4.")
        signs = _lib.host_floats(desc["signs"])
        if dim is None:
            dim = len(signs)
        shape, st, ns = packed.shape, packed.stride(), norms.stride()
        if (packed.dtype is not torch.uint32 or len(shape) != 4 or st[3] != 1 or st[2] != shape[3]
                or shape[3] != packed_dim(dim, bits)):
            raise ValueError(f"{what}: packed must be (pages, heads, page, {packed_dim(dim, bits)}) uint32 with contiguous rows")
        if norms.dtype is not torch.float32 or norms.shape != shape[:3] or ns[2] != 1:
            raise ValueError(f"{what}: norms must be float32 {tuple(shape[:3])}, contiguous along the page")
        if len(signs) != dim:
            raise ValueError(f"{what}: {len(signs)} signs for dim {dim}")
        if packed.device != dev or norms.device != dev:
            raise ValueError(f"{what}: all tensors must be on {dev}")
        H.format, H.bits = _lib.TQ_KV_POLAR, bits
        H.data, H.norms = packed.data_ptr(), norms.data_ptr()
        H.page_stride, H.head_stride = st[0], st[1]
        H.norm_page_stride, H.norm_head_stride = ns[0], ns[1]
        H.signs_host = signs
        levels = 1 << bits
        if encode:
            table = _lib.host_floats(desc["boundaries"])
            if len(table) != levels - 1:
                raise ValueError(f"{what}: {len(table)} boundaries for {bits} bits")
            H.boundaries_host = table
        else:
            table = _lib.host_floats(desc["centroids"])
            if len(table) != levels:
                raise ValueError(f"{what}: {len(table)} centroids for {bits} bits")
            H.centroids_host = table
        return shape[0], shape[1], shape[2], dim
    if fmt == "dense":
        data = desc["data"]
        shape, st = data.shape, data.stride()
        if len(shape) != 4 or st[3] != 1 or st[2] != shape[3] or (dim is not None and shape[3] != dim):
            raise ValueError(f"{what}: dense pages must be (pages, heads, page, dim) with contiguous rows")
        if data.device != dev:
            raise ValueError(f"{what}: all tensors must be on {dev}")
        H.format, H.dtype, H.data = _lib.TQ_KV_DENSE, _lib.dtype_code(data.dtype), data.data_ptr()
        H.page_stride, H.head_stride = st[0], st[1]
        return shape[0], shape[1], shape[2], shape[3]
    raise ValueError(f"{what}: unknown page format {fmt!r}")


def _lens(t, what: str, batch: int, dev):
    if t.dtype is not torch.int32 or t.shape != (batch,) or (batch > 1 and t.stride(0) != 1) or t.device != dev:
        raise ValueError(f"{what} must be a contiguous int32 ({batch},) tensor on {dev}")
    return t.data_ptr()


def _common(P, page_table, seq_lens, what: str, dev):
    """Table and lengths; returns the batch size."""
    if not page_table.is_cuda or not seq_lens.is_cuda:
        raise RuntimeError(_ERR_CPU)
    if page_table.dtype is not torch.int32 or page_table.ndim != 2 or page_table.stride(1) != 1 and page_table.shape[1] > 1:
        raise ValueError("page_table must be an int32 (batch, width) tensor with contiguous rows")
    if page_table.device != dev:
        raise ValueError(f"page_table must be on {dev}")
    batch, width = page_table.shape
    if batch < 1 or width < 1:
        raise ValueError("page_table must have at least one sequence and one page")
    P.struct_bytes = _PARAM_BYTES
    P.batch, P.page_table, P.table_stride, P.table_width = batch, page_table.data_ptr(), page_table.stride(0), width
    P.seq_lens = _lens(seq_lens, what, batch, dev)
    return batch


_PARAM_BYTES = ctypes.sizeof(_lib.PagedParams)


def paged_append(keys: torch.Tensor, values: torch.Tensor, *, k: dict, v: dict, page_table: torch.Tensor,
                 starts: torch.Tensor, counts: torch.Tensor | None = None) -> None:
    """Store the new tokens of a ragged batch in their pages, keys and values in one launch.

    keys / values (B, H, T, dim), float32, float16 or bfloat16, rows contiguous, other strides free: token t of
    sequence b goes to position starts[b] + t of its page table, for t < counts[b] (every t without `counts`); padded
    tokens behind counts[b] are not read.  Packed halves get the words and norms `fused_quantize` gives; dense halves
    are copied and need the pages' own type.  Two tokens of one call must not share a place (sequences that share a
    page must not both write it)."""
    _lib.require_cuda(keys, values)
    dev = keys.device
    if keys.ndim != 4 or keys.shape != values.shape:
        raise ValueError(f"keys and values must be (batch, heads, tokens, dim) alike, got {tuple(keys.shape)} and {tuple(values.shape)}")
    if values.device != dev:
        raise ValueError(f"values must be on {dev}")
    B, H, T, dim = keys.shape
    P = _lib.PagedParams()
    if _common(P, page_table, starts, "starts", dev) != B:
        raise ValueError(f"page_table has {page_table.shape[0]} sequences, keys have {B}")
    geo = _half(P.k, k, "keys", dim, dev, True)
    if _half(P.v, v, "values", dim, dev, True) != geo:
        raise ValueError("the pools of keys and values must agree in pages, heads, page size and dim")
    if geo[1] != H:
        raise ValueError(f"the pool has {geo[1]} heads, the new rows {H}")
    if keys.stride(3) != 1:
        keys = keys.contiguous()
    if values.stride(3) != 1:
        values = values.contiguous()
    for half, x in ((P.k, keys), (P.v, values)):
        st = x.stride()
        half.rows, half.rows_dtype = x.data_ptr(), _lib.dtype_code(x.dtype)
        half.rows_batch_stride, half.rows_head_stride, half.rows_token_stride = st[0], st[1], st[2]
    if P.k.format == _lib.TQ_KV_DENSE and P.k.rows_dtype != P.k.dtype or P.v.format == _lib.TQ_KV_DENSE and P.v.rows_dtype != P.v.dtype:
        raise ValueError("rows stored in dense pages must have the pages' dtype")
    if counts is not None:
        _lib.require_cuda(counts)
        P.counts = _lens(counts, "counts", B, dev)
    P.n_kv_heads, P.dim, P.page_size, P.n_pages, P.tokens = H, dim, geo[2], geo[0], T
    P.stream = torch.cuda.current_stream(dev).cuda_stream
    with _on(dev):
        _lib.check(_lib.lib().tq_paged_append(ctypes.byref(P)))


def paged_decode(q: torch.Tensor, *, k: dict, v: dict, page_table: torch.Tensor, seq_lens: torch.Tensor, attn_scale: float,
                 window: int = 0, sinks: int = 0, out: torch.Tensor | None = None, out_dtype=None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its pages: q (B, n_q, dim) -> (B, n_q, dim) in `out_dtype`
    (default q.dtype), the token being the last of seq_lens[b] positions.

    window > 0: the token sees positions >= seq_lens[b] - window and the first `sinks` ones (it counts itself, as
    `create_causal_mask` does); pages outside both may have been freed.  A sequence of length 0 gives zeros.
    Lengths beyond the table are cut to it.  `out` optionally names the tensor to write (rows contiguous).
    `workspace`: a uint8 tensor of `paged_workspace_bytes` on the device; without it each call allocates its own from
    torch's caching allocator (inside a captured graph: from the graph's pool), so overlapping calls and captured
    graphs never share one.

    The weights are 16-bit in the tensor-core kernel (head_dim 128, 3 / 4-bit values, 16-bit or 3 / 4-bit keys, 16-bit
    queries); float32 queries and every other shape take the 32-bit kernel."""
    _lib.require_cuda(q)
    dev = q.device
    if q.ndim != 3:
        raise ValueError(f"q must be (batch, heads, dim), got {tuple(q.shape)}")
    if q.stride(2) != 1:
        q = q.contiguous()
    B, n_q, dim = q.shape
    P = _lib.PagedParams()
    if _common(P, page_table, seq_lens, "seq_lens", dev) != B:
        raise ValueError(f"page_table has {page_table.shape[0]} sequences, q has {B}")
    geo = _half(P.k, k, "keys", dim, dev, False)
    if _half(P.v, v, "values", dim, dev, False) != geo:
        raise ValueError("the pools of keys and values must agree in pages, heads, page size and dim")
    if n_q == 0 or n_q % geo[1]:
        raise ValueError(f"n_q_heads ({n_q}) must equal n_kv_heads ({geo[1]}) * n_rep")
    if window < 0 or sinks < 0 or (sinks and not window):
        raise ValueError(f"window ({window}) and sinks ({sinks}) must not be negative, and sinks need a window")
    if out is None:
        out = torch.empty((B, n_q, dim), dtype=out_dtype or q.dtype, device=dev)
    elif out.shape != (B, n_q, dim) or out.stride(2) != 1 or out.device != dev or (out_dtype or out.dtype) != out.dtype:
        raise ValueError(f"out must be ({B}, {n_q}, {dim}) on {dev}, with a contiguous last dimension and of out_dtype")
    need = paged_workspace_bytes(dev, dim)
    if workspace is None:
        workspace = torch.empty((need,), dtype=torch.uint8, device=dev)
    elif workspace.dtype is not torch.uint8 or not workspace.is_contiguous() or workspace.device != dev or workspace.numel() < need:
        raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes on {dev}")
    st, so = q.stride(), out.stride()
    P.n_q_heads, P.n_kv_heads, P.dim, P.page_size, P.n_pages = n_q, geo[1], dim, geo[2], geo[0]
    P.q, P.q_dtype, P.q_batch_stride, P.q_head_stride = q.data_ptr(), _lib.dtype_code(q.dtype), st[0], st[1]
    P.out, P.out_dtype, P.out_batch_stride, P.out_head_stride = out.data_ptr(), _lib.dtype_code(out.dtype), so[0], so[1]
    P.attn_scale, P.window, P.sinks = attn_scale, min(window, 0x7fffffff), min(sinks, 0x7fffffff)
    P.workspace, P.workspace_bytes = workspace.data_ptr(), workspace.numel()
    P.stream = torch.cuda.current_stream(dev).cuda_stream
    with _on(dev):
        _lib.check(_lib.lib().tq_paged_decode(ctypes.byref(P)))
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
    and `packed_dequantize` give; rows at and behind seq_lens[b] are zero.  Dense pools are gathered as they are.
    `out` optionally names the contiguous tensor to write."""
    _lib.require_cuda(page_table)
    dev = page_table.device
    P = _lib.PagedParams()
    B = _common(P, page_table, seq_lens, "seq_lens", dev)
    n_pages, H, page, dim = _half(P.v, pool, "pages", None, dev, False)
    if length < 0:
        raise ValueError(f"length must not be negative, got {length}")
    if out is None:
        out = torch.empty((B, H, length, dim), dtype=dtype, device=dev)
    elif out.shape != (B, H, length, dim) or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out must be a contiguous ({B}, {H}, {length}, {dim}) tensor on {dev}")
    P.n_kv_heads, P.dim, P.page_size, P.n_pages, P.tokens = H, dim, page, n_pages, length
    P.out, P.out_dtype = out.data_ptr(), _lib.dtype_code(out.dtype)
    P.stream = torch.cuda.current_stream(dev).cuda_stream
    with _on(dev):
        _lib.check(_lib.lib().tq_paged_dequantize(ctypes.byref(P)))
    return out


def _page_ids(ids, n_pages: int, what: str):
    """int32 ids from a list or a CPU tensor (checked) or a CUDA tensor (its values are checked by the kernel)."""
    if isinstance(ids, torch.Tensor) and ids.is_cuda:
        if ids.dtype is not torch.int32 or ids.ndim != 1 or not ids.is_contiguous():
            raise ValueError(f"{what} must be a contiguous one-dimensional int32 tensor")
        return ids, None
    host = [int(i) for i in ids]
    bad = [i for i in host if not 0 <= i < n_pages]
    if bad:
        raise ValueError(f"{what}: page {bad[0]} is outside the pool of {n_pages}")
    return torch.tensor(host, dtype=torch.int32), host


def copy_pages(pools, src, dst) -> None:
    """Copy page src[i] to page dst[i] in every tensor of `pools` (contiguous, the page dimension in front, e.g. the
    packed words and norms of all layers) in one launch (per 128 tensors): a fork's last page, a compaction.

    src / dst: lists or CPU tensors, which are checked here, or int32 CUDA tensors, of which the kernel only checks
    that they lie inside the pools.  No page may be written twice, or both read and written, by one call."""
    pools = list(pools)
    if not pools:
        return
    _lib.require_cuda(*pools)
    dev, n_pages = pools[0].device, pools[0].shape[0]
    for t in pools:
        if t.device != dev or t.shape[0] != n_pages or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError("pools must be contiguous, 16-byte aligned, of one device and one number of pages")
    (src, hs), (dst, hd) = _page_ids(src, n_pages, "src"), _page_ids(dst, n_pages, "dst")
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} source and {dst.numel()} target pages")
    if hd is not None and len(set(hd)) != len(hd):
        raise ValueError("a target page is named twice")
    if hs is not None and hd is not None and set(hs) & set(hd):
        raise ValueError("a page is both read and written")
    if n_pages == 0 or src.numel() == 0:
        return
    sizes = [t.numel() // n_pages * t.element_size() for t in pools]
    if any(s == 0 or s % 16 for s in sizes):
        raise ValueError("pages must be multiples of 16 bytes")
    if src.device != dev:
        src = src.to(dev)
    if dst.device != dev:
        dst = dst.to(dev)
    n = len(pools)
    ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in pools])
    with _on(dev):
        _lib.check(_lib.lib().tq_copy_pages(ptrs, (ctypes.c_int64 * n)(*sizes), n, n_pages, src.data_ptr(), dst.data_ptr(),
                                            src.numel(), torch.cuda.current_stream(dev).cuda_stream))


def paged_status(device) -> int:
    """What the paged kernels found wrong on this device since the last call (synchronises the current stream): 0
    nothing, 1 a page id outside the pool, 2 a position behind the page table, 3 a bounded wait that gave up."""
    device = torch.device(device)
    word = ctypes.c_int(0)
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("paged_status cannot be captured in a CUDA graph")
        _lib.check(_lib.lib().tq_paged_status(ctypes.byref(word), torch.cuda.current_stream(device).cuda_stream))
    return word.value
