"""What the paged operators refuse, and with which status: validation happens before any CUDA call, so no GPU is
needed (the C entry points get made-up pointers, which a refused call never follows)."""
import ctypes

import pytest
import torch


@pytest.fixture()
def params(tq):
    """A valid argument block for a decode over 3-bit pages; returns (lib, block, things kept alive)."""
    lib = tq._lib
    signs = (ctypes.c_float * 128)(*([1.0] * 128))
    cents = (ctypes.c_float * 8)(*range(8))
    bounds = (ctypes.c_float * 7)(*range(7))
    P = lib.PagedParams()
    P.struct_bytes = ctypes.sizeof(P)
    P.batch, P.n_q_heads, P.n_kv_heads, P.dim, P.page_size, P.n_pages = 2, 8, 2, 128, 64, 10
    P.page_table, P.table_stride, P.table_width, P.seq_lens = 16, 4, 4, 16
    P.q, P.q_dtype, P.out, P.out_dtype, P.attn_scale = 16, 1, 16, 1, 0.1
    P.workspace, P.workspace_bytes, P.tokens = 16, 1 << 30, 5
    for H in (P.k, P.v):
        H.format, H.bits, H.data, H.norms = 0, 3, 16, 16
        H.page_stride, H.head_stride, H.norm_page_stride, H.norm_head_stride = 2 * 64 * 13, 64 * 13, 2 * 64, 64
        H.centroids_host, H.boundaries_host, H.signs_host = cents, bounds, signs
        H.rows, H.rows_dtype = 16, 1
    return lib.lib(), P, (signs, cents, bounds)


def _set(P, path, value):
    *head, last = path.split(".")
    for part in head:
        P = getattr(P, part)
    setattr(P, last, value)


@pytest.mark.parametrize("path,value,code", [
    ("struct_bytes", 8, -7), ("dim", 100, -1), ("dim", 16, -1), ("dim", 512, -1), ("page_size", 16, -7), ("page_size", 48, -7),
    ("page_size", 0, -7), ("batch", 0, -7), ("n_kv_heads", 0, -7), ("n_pages", 0, -7), ("n_pages", 1 << 31, -7),
    ("page_table", None, -7), ("seq_lens", None, -7), ("table_width", 0, -7), ("n_q_heads", 7, -3), ("n_q_heads", 0, -3),
    ("q", None, -7), ("out", None, -7), ("q_dtype", 3, -7), ("out_dtype", -1, -7), ("window", -1, -7), ("sinks", -1, -7),
    ("sinks", 4, -7), ("attn_scale", float("nan"), -7), ("attn_scale", float("inf"), -7), ("workspace", None, -5),
    ("workspace_bytes", 100, -5), ("workspace", 24, -4), ("k.data", None, -7), ("k.format", 2, -8), ("k.bits", 5, -2),
    ("v.bits", 0, -2), ("v.format", 1, -8), ("v.norms", None, -7), ("k.page_stride", -1, -7),
])
def test_decode_refusals(params, path, value, code):
    lib, P, _keep = params
    _set(P, path, value)
    assert lib.tq_paged_decode(ctypes.byref(P)) == code
    assert lib.tq_last_error_string()


def test_missing_tables_are_refused(params):
    lib, P, (signs, cents, bounds) = params
    P.v.centroids_host = None
    assert lib.tq_paged_decode(ctypes.byref(P)) == -7
    P.v.centroids_host = cents
    P.v.boundaries_host = None
    assert lib.tq_paged_append(ctypes.byref(P)) == -7
    P.v.boundaries_host = bounds
    bad = (ctypes.c_float * 128)(*([0.5] * 128))
    P.v.signs_host = bad
    assert lib.tq_paged_append(ctypes.byref(P)) == -7 and lib.tq_paged_dequantize(ctypes.byref(P)) == -7
    P.v.signs_host = None
    assert lib.tq_paged_decode(ctypes.byref(P)) == -7


@pytest.mark.parametrize("path,value,code", [
    ("k.rows", None, -7), ("v.rows_dtype", 9, -7), ("tokens", -1, -7), ("tokens", 1 << 31, -7), ("k.bits", 7, -2), ("dim", 96, -1),
])
def test_append_refusals(params, path, value, code):
    lib, P, _keep = params
    _set(P, path, value)
    assert lib.tq_paged_append(ctypes.byref(P)) == code


def test_append_dense_rows_need_the_pages_type(params):
    lib, P, _keep = params
    P.k.format, P.k.dtype, P.k.rows_dtype = 1, 2, 1
    assert lib.tq_paged_append(ctypes.byref(P)) == -7
    assert b"type" in lib.tq_last_error_string()


@pytest.mark.parametrize("path,value,code", [("tokens", -1, -7), ("out", None, -7), ("out_dtype", 5, -7), ("v.data", None, -7)])
def test_dequantize_refusals(params, path, value, code):
    lib, P, _keep = params
    _set(P, path, value)
    assert lib.tq_paged_dequantize(ctypes.byref(P)) == code


def test_empty_calls_do_nothing(params):
    lib, P, _keep = params
    P.tokens = 0
    assert lib.tq_paged_append(ctypes.byref(P)) == 0 and lib.tq_paged_dequantize(ctypes.byref(P)) == 0
    assert lib.tq_copy_pages(None, None, 0, 4, None, None, 3, None) == 0
    assert lib.tq_copy_pages((ctypes.c_void_p * 1)(16), (ctypes.c_int64 * 1)(16), 1, 4, None, None, 0, None) == 0


def test_null_block(tq):
    L = tq._lib.lib()
    assert L.tq_paged_decode(None) == -7 and L.tq_paged_append(None) == -7 and L.tq_paged_dequantize(None) == -7
    assert L.tq_paged_status(None, None) == -7


@pytest.mark.parametrize("ptr,nbytes,pages,pairs,code", [
    (8, 16, 4, 1, -4), (16, 24, 4, 1, -4), (16, 0, 4, 1, -4), (None, 16, 4, 1, -4), (16, 16, 0, 1, -7), (16, 16, 4, -1, -7)])
def test_copy_refusals(tq, ptr, nbytes, pages, pairs, code):
    L = tq._lib.lib()
    got = L.tq_copy_pages((ctypes.c_void_p * 1)(ptr), (ctypes.c_int64 * 1)(nbytes), 1, pages, 16, 16, pairs, None)
    assert got == code


def test_prompt_window_refusals(tq):
    L = tq._lib.lib()

    def call(causal, window, sinks, scale=0.1, size=None):
        P = tq._lib.PrefillParams()
        P.struct_bytes = ctypes.sizeof(P) if size is None else size
        P.dtype, P.batch, P.n_q_heads, P.n_kv_heads, P.dim, P.seq_q, P.seq_k = 1, 1, 2, 1, 128, 4, 4
        P.q = P.k = P.v = P.out = P.status = 16
        for name in ("q_strides", "k_strides", "v_strides", "o_strides"):
            setattr(P, name, (ctypes.c_int64 * 3)(1024, 1024, 1024))
        P.window, P.sinks, P.attn_scale, P.causal = window, sinks, scale, causal
        return L.tq_prefill_sdpa_window(ctypes.byref(P))

    assert call(1, -1, 0) == -7 and call(1, 4, -1) == -7 and call(1, 0, 3) == -7 and call(0, 4, 0) == -8
    assert call(1, 4, 0, scale=0.0) == -7 and call(1, 4, 0, size=8) == -7 and L.tq_prefill_sdpa_window(None) == -7


def test_wrappers_refuse_cpu_tensors(tq):
    x = torch.zeros((1, 2, 3, 128))
    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tq.paged_append(x, x, k={}, v={}, page_table=table, starts=lens)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tq.paged_decode(x[:, :, 0], k={}, v={}, page_table=table, seq_lens=lens, attn_scale=1.0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tq.paged_dequantize({}, page_table=table, seq_lens=lens, length=4)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tq.copy_pages([x], [0], [0])
    assert tq.copy_pages([], [0], [1]) is None


def test_native_calls_report_their_errors(tq):
    """Errors raised in the extension module arrive as Python exceptions, numbers in their texts included."""
    calls = tq._lib.load_native()
    for name, n in (("decode", 11), ("append", 7), ("dequantize", 6), ("copy_pages", 3), ("prefill", 9)):
        with pytest.raises(TypeError, match=f"{n} arguments expected, got 1"):
            getattr(calls, name)(None)
    with pytest.raises(TypeError, match="must be a tensor"):
        tq.copy_pages([3], [0], [1])
    with pytest.raises(TypeError, match="sequence of tensors"):
        tq.copy_pages(3, [0], [1])
    assert not tq.copy_pages([], [0], [1])
