"""Paged caches on a GPU: decode attention over pages, insert, read-back and page copies against 64-bit references."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as pr  # noqa: E402

pytestmark = pytest.mark.gpu

HALF_F16 = torch.finfo(torch.float16).eps / 2       # half a step of a 16-bit weight, relative


def _decode(tq, dev, *, lens, n_q, n_kv, dim=128, kbits=3, vbits=3, page=64, window=0, sinks=0, q_dtype=torch.float16,
            k_dtype=torch.float16, out_dtype=None, head_major=False, seed=0, scale=None, q_gain=1.0):
    table, pages = pr.make_table(lens, page, seed, window=window, sinks=sinks, dev=dev)
    k = pr.Pool(tq, seed + 10, pages, n_kv, page, dim, kbits, dev, dtype=k_dtype, head_major=head_major)
    v = pr.Pool(tq, seed + 20, pages, n_kv, page, dim, vbits, dev, head_major=head_major)
    q = (torch.randn((len(lens), n_q, dim), generator=torch.Generator().manual_seed(seed)) * q_gain).to(q_dtype).to(dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    got = tq.paged_decode(q, k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=scale, window=window,
                          sinks=sinks, out_dtype=out_dtype)
    assert got.dtype == (out_dtype or q_dtype) and got.shape == q.shape
    weight_eps = 0.0 if q_dtype == torch.float32 else HALF_F16
    ref, tol = pr.decode_ref(tq, q, k, v, table, lens, scale, window, sinks, weight_eps, got.dtype)
    pr.check(got, ref, tol, f"lens {lens}")
    assert tq.paged_status(dev) == 0
    return got, (q, k, v, table, seq, scale)


@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 500, 1000, 2049])
def test_decode_lengths(tq, dev, n):
    _decode(tq, dev, lens=[n], n_q=28, n_kv=4)


@pytest.mark.parametrize("kbits,vbits", [(0, 3), (0, 4), (3, 3), (3, 4), (4, 3), (4, 4), (1, 2), (2, 1)])
@pytest.mark.parametrize("q_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_decode_formats(tq, dev, kbits, vbits, q_dtype):
    _decode(tq, dev, lens=[333, 0, 1, 700], n_q=8, n_kv=2, kbits=kbits, vbits=vbits, q_dtype=q_dtype,
            k_dtype=torch.bfloat16 if q_dtype == torch.bfloat16 else torch.float16)


@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (3, 1), (8, 1), (9, 1), (32, 2), (6, 6), (28, 4), (17, 1)])
def test_decode_head_layouts(tq, dev, n_q, n_kv):
    _decode(tq, dev, lens=[450, 77], n_q=n_q, n_kv=n_kv)


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("kbits", [0, 3])
def test_decode_dims(tq, dev, dim, kbits):
    _decode(tq, dev, lens=[100, 300], n_q=4, n_kv=2, dim=dim, kbits=kbits, vbits=4)


@pytest.mark.parametrize("page", [32, 64, 128, 1024])
def test_decode_page_sizes(tq, dev, page):
    _decode(tq, dev, lens=[page, page + 1, 5 * page // 2, 3], n_q=7, n_kv=1, page=page, kbits=4)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 0), (100, 33), (100, 77), (257, 4), (5000, 4),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("kbits", [0, 3])
def test_decode_window(tq, dev, window, sinks, kbits):
    _decode(tq, dev, lens=[1000, 64, 1, 0, 333, 101, 100], n_q=8, n_kv=2, window=window, sinks=sinks, kbits=kbits)


def test_decode_many_sequences(tq, dev):
    """More sequences than a plan has entries, lengths 0 to 40."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 41, (2100,), generator=g).tolist()
    _decode(tq, dev, lens=lens, n_q=2, n_kv=1, page=32)


def test_decode_ragged_split(tq, dev):
    """One long sequence among short ones: its groups are split over many CTAs and joined."""
    _decode(tq, dev, lens=[9000, 1, 40, 0, 777], n_q=16, n_kv=2, kbits=4, vbits=3, page=128)


def test_decode_strides(tq, dev):
    _decode(tq, dev, lens=[333, 70], n_q=8, n_kv=2, head_major=True)
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=[200, 90], n_q=8, n_kv=2)
    wide = torch.zeros((2, 16, 160), dtype=q.dtype, device=dev)
    wide[:, ::2, 16:144] = q
    out = torch.full((2, 8, 3, 128), 7.0, dtype=q.dtype, device=dev)
    res = tq.paged_decode(wide[:, ::2, 16:144], k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=scale,
                          out=out[:, :, 1])
    assert torch.equal(res, got) and bool((out[:, :, 0] == 7).all()) and bool((out[:, :, 2] == 7).all())
    odd = torch.zeros((2 * 8 * 128 + 1,), dtype=q.dtype, device=dev)[1:].view(2, 8, 128)
    odd.copy_(q)
    assert torch.equal(tq.paged_decode(odd, k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=scale), got)


@pytest.mark.parametrize("kbits", [0, 3, 4])
def test_decode_ignores_hidden_places(tq, dev, kbits):
    """NaN and infinities behind a sequence, in front of its window and in foreign pages change nothing."""
    lens, window, sinks, page = [500, 130, 0], 100, 5, 64
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=lens, n_q=8, n_kv=2, kbits=kbits, window=window, sinks=sinks, page=page)
    seen = torch.zeros(v.norms.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in pr.visible(n, window, sinks):
            seen[table[b, p // page].item(), p % page] = True
    hidden = (~seen).to(dev)[:, None].expand(v.norms.shape)
    for bad in (float("nan"), float("inf"), -float("inf")):
        v.norms[hidden] = bad
        if kbits:
            k.norms[hidden] = bad
        else:
            k.data[hidden] = bad
        again = tq.paged_decode(q, k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=scale, window=window, sinks=sinks)
        assert torch.equal(again, got)


@pytest.mark.parametrize("q_dtype", [torch.float16, torch.float32])
def test_decode_page_outside_pool(tq, dev, q_dtype):
    """A bad page id is reported and turns its sequence into NaN; the others keep their results."""
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=[300, 200, 100], n_q=8, n_kv=2, q_dtype=q_dtype)
    for bad in (-1, v.norms.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 2] = bad
        out = tq.paged_decode(q, k=k.desc, v=v.desc, page_table=t, seq_lens=seq, attn_scale=scale)
        assert bool(out[1].isnan().all()) and torch.equal(out[0], got[0]) and torch.equal(out[2], got[2])
        assert tq.paged_status(dev) == 1 and tq.paged_status(dev) == 0


def test_decode_lengths_out_of_range(tq, dev):
    """Lengths beyond the table are cut to it, negative ones count as empty."""
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=[128, 128], n_q=4, n_kv=2)
    far = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=dev)
    out = tq.paged_decode(q, k=k.desc, v=v.desc, page_table=table, seq_lens=far, attn_scale=scale)
    assert torch.equal(out[0], got[0]) and bool((out[1] == 0).all())


@pytest.mark.parametrize("gain", [1e-3, 30.0, 3000.0])
def test_decode_query_magnitudes(tq, dev, gain):
    """Tiny and huge queries (rotation multiplies them by up to dim) stay within their bound."""
    _decode(tq, dev, lens=[200], n_q=8, n_kv=2, q_gain=gain, scale=1.0 / (gain * 10), q_dtype=torch.bfloat16)


def test_decode_shared_pages(tq, dev):
    """Two sequences over the same prefix pages see what one sequence sees."""
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=[192], n_q=8, n_kv=2)
    out = tq.paged_decode(q.expand(2, -1, -1), k=k.desc, v=v.desc, page_table=table.expand(2, -1).contiguous(),
                          seq_lens=seq.expand(2).contiguous(), attn_scale=scale)
    pr.check(out[1:], got.cpu().double(), (got.cpu().double().abs() + 1) * torch.finfo(got.dtype).eps)


def test_decode_graph_replay_and_streams(tq, dev):
    """Captured once, replayed with other lengths and tables; two graphs replayed side by side on two streams."""
    lens = [700, 300]
    made = [_decode(tq, dev, lens=lens, n_q=8, n_kv=2, kbits=b, seed=b) for b in (3, 4)]
    graphs = []
    for got, (q, k, v, table, seq, scale) in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = tq.paged_decode(q, k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=scale)
        graphs.append((g, out))
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (g, _out) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (got, _), (_, out) in zip(made, graphs):
        assert torch.equal(out, got)
    (got, (q, k, v, table, seq, scale)), (g, out) = made[0], graphs[0]
    seq.copy_(torch.tensor([33, 299], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    ref, tol = pr.decode_ref(tq, q, k, v, table, [33, 299], scale, weight_eps=HALF_F16, out_dtype=out.dtype)
    pr.check(out, ref, tol)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_decode_output_types(tq, dev, out_dtype):
    _decode(tq, dev, lens=[300, 40], n_q=8, n_kv=2, out_dtype=out_dtype)


@pytest.mark.parametrize("kbits", [0, 3])
def test_decode_one_bad_head_stays_alone(tq, dev, kbits):
    """A query head of NaN or infinity spoils its own row and no other."""
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=[200, 77], n_q=8, n_kv=2, kbits=kbits)
    for bad in (float("nan"), float("inf")):
        q2 = q.clone()
        q2[0, 3, 5] = bad
        out = tq.paged_decode(q2, k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=scale)
        keep = torch.ones((2, 8), dtype=torch.bool, device=dev)
        keep[0, 3] = False
        assert torch.equal(out[keep], got[keep]) and not bool(out[0, 3].isfinite().all())


@pytest.mark.parametrize("scale", [0.0, -0.05, 3.0])
def test_decode_scales(tq, dev, scale):
    _decode(tq, dev, lens=[300], n_q=8, n_kv=2, scale=scale, q_gain=0.3)


@pytest.mark.parametrize("what", ["norms", "words", "strides"])
def test_decode_unaligned_pools(tq, dev, what):
    """Pools whose rows are not 16-byte aligned take the general kernel: same values."""
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=[300, 77], n_q=8, n_kv=2)
    desc = dict(v.desc)
    P, H, page, words = v.packed.shape

    def shifted(t, pad):
        if what == "strides":
            wide = torch.zeros((P, H * t[0, 0].numel() + 1), dtype=torch.int32, device=dev)
            out = wide[:, :-1].view(P, H, *t.shape[2:]) if wide[:, :-1].is_contiguous() else wide.as_strided(
                t.shape, (wide.stride(0), *t.stride()[1:]))
        else:
            out = torch.zeros((t.numel() + 1,), dtype=torch.int32, device=dev)[1:].view(t.shape)
        out.copy_(t.view(torch.int32))
        return out.view(t.dtype)
    if what in ("words", "strides"):
        desc["packed"] = shifted(v.packed, 1)
    if what in ("norms", "strides"):
        desc["norms"] = shifted(v.norms, 1)
    out = tq.paged_decode(q, k=k.desc, v=desc, page_table=table, seq_lens=seq, attn_scale=scale)
    ref, tol = pr.decode_ref(tq, q, k, v, table, [300, 77], scale, weight_eps=HALF_F16, out_dtype=out.dtype)
    pr.check(out, ref, tol)


@pytest.mark.parametrize("kind", ["uneven", "huge", "tiny"])
def test_decode_other_codebooks(tq, dev, kind):
    """Codebooks that have no good 16-bit scale take the 32-bit kernel."""
    lens = [200]
    table, pages = pr.make_table(lens, 64, 0, dev=dev)
    k, v = pr.Pool(tq, 1, pages, 2, 64, 128, 3, dev), pr.Pool(tq, 2, pages, 2, 64, 128, 4, dev)
    for p in (k, v):
        n = 1 << p.bits
        base = torch.linspace(-2.1, 2.3, n) + 0.013 * torch.arange(n) ** 2
        p.quant.centroids = (base * {"uneven": 1.0, "huge": 1e6, "tiny": 1e-7}[kind]).float().to(dev)
        p.desc["centroids"] = p.quant.centroids
    q = torch.randn((1, 4, 128), generator=torch.Generator().manual_seed(0)).half().to(dev)
    scale = {"uneven": 0.05, "huge": 5e-8, "tiny": 5e5}[kind]
    out = tq.paged_decode(q, k=k.desc, v=v.desc, page_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                          attn_scale=scale, out_dtype=torch.float32)
    # "uneven" may take either kernel: a 16-bit codebook is off by at most 2^-13 there
    ref, tol = pr.decode_ref(tq, q, k, v, table, lens, scale, weight_eps=HALF_F16 + 4 * 2.0 ** -13, out_dtype=torch.float32)
    pr.check(out, ref, tol)


@pytest.mark.parametrize("stride", [(1 << 30) - 4096, 1 << 30])
def test_decode_offsets_beyond_32_bits(tq, dev, stride):
    """Pages whose byte offsets pass 2^32 (and element offsets 2^31): tensor-core and general kernel, insert, read-back and
    page copies."""
    H, page, words, P = 2, 64, 13, 3
    lens = [150]
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    small = [pr.Pool(tq, s, P, H, page, 128, 3, dev) for s in (1, 2)]
    q = torch.randn((1, 8, 128), generator=torch.Generator().manual_seed(0)).half().to(dev)
    seq = torch.tensor(lens, dtype=torch.int32, device=dev)
    want = tq.paged_decode(q, k=small[0].desc, v=small[1].desc, page_table=table, seq_lens=seq, attn_scale=0.1)
    buf = torch.empty((2 * stride + H * page * words,), dtype=torch.int32, device=dev)
    far = buf.as_strided((P, H, page, words), (stride, page * words, words, 1))
    far.copy_(small[1].packed.view(torch.int32))
    v = dict(small[1].desc, packed=far.view(torch.uint32))
    got = tq.paged_decode(q, k=small[0].desc, v=v, page_table=table, seq_lens=seq, attn_scale=0.1)
    ref, tol = pr.decode_ref(tq, q, small[0], small[1], table, lens, 0.1, weight_eps=HALF_F16, out_dtype=got.dtype)
    pr.check(got, ref, tol)
    assert stride >= 1 << 30 or torch.equal(got, want)
    assert torch.equal(tq.paged_dequantize(v, page_table=table, seq_lens=seq, length=150),
                       tq.paged_dequantize(small[1].desc, page_table=table, seq_lens=seq, length=150))
    x = torch.randn((1, H, 30, 128), device=dev, dtype=torch.float16)
    for desc in (v, small[1].desc):
        tq.paged_append(x, x, k=small[0].desc, v=desc, page_table=table, starts=torch.tensor([120], dtype=torch.int32, device=dev))
    assert torch.equal(far, small[1].packed.view(torch.int32))
    del buf, far, v
    big = torch.zeros((5, 1 << 28), dtype=torch.int32, device=dev)      # 1 GiB pages
    big[4, -7:] = 5
    tq.copy_pages([big], [4], [2])
    assert torch.equal(big[2], big[4]) and not bool(big[:2].any())


def test_decode_sliced_table(tq, dev):
    """Rows of a wider table, and one row seen by every sequence."""
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=[300, 77, 150], n_q=8, n_kv=2)
    wide = torch.full((3, table.shape[1] + 5), 1 << 30, dtype=torch.int32, device=dev)
    wide[:, 3:3 + table.shape[1]] = table
    part = wide[:, 3:3 + table.shape[1]]
    assert torch.equal(tq.paged_decode(q, k=k.desc, v=v.desc, page_table=part, seq_lens=seq, attn_scale=scale), got)
    same = table[:1].expand(3, -1)
    n = torch.tensor([300, 300, 300], dtype=torch.int32, device=dev)
    out = tq.paged_decode(q, k=k.desc, v=v.desc, page_table=same, seq_lens=n, attn_scale=scale)
    assert torch.equal(out, tq.paged_decode(q, k=k.desc, v=v.desc, page_table=same.contiguous(), seq_lens=n, attn_scale=scale))
    assert tq.paged_status(dev) == 0


def test_decode_two_streams_at_once(tq, dev):
    """Split groups of two eager streams in flight together: each stream has its own scratch."""
    a = _decode(tq, dev, lens=[9000], n_q=8, n_kv=1)
    b = _decode(tq, dev, lens=[7000, 40], n_q=28, n_kv=4, kbits=0, seed=5)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (s, (_, (q, k, v, table, seq, scale))) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                outs[i].append(tq.paged_decode(q, k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=scale))
    torch.cuda.synchronize()
    assert all(torch.equal(o, a[0]) for o in outs[0]) and all(torch.equal(o, b[0]) for o in outs[1])


def test_copy_pages_in_a_capture(tq, dev):
    pool = torch.zeros((4, 64), dtype=torch.int32, device=dev)
    src, dst = (torch.tensor([i], dtype=torch.int32, device=dev) for i in (1, 3))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            tq.copy_pages([pool], [1], [3])
        tq.copy_pages([pool], src, dst)
    pool[1] = 7
    graph.replay()
    assert torch.equal(pool[3], pool[1]) and not bool(pool[2].any())


def test_first_call_inside_a_capture(tq, dev):
    """A process whose first paged call is captured: works or raises, and the next eager call is right (child process)."""
    code = """
import torch, sys
sys.path.insert(0, %r); sys.path.insert(0, %r)
import __graft_entry__ as e, paged_ref as pr
tq = e.load_package(); dev = torch.device("cuda", 0)
table, pages = pr.make_table([100], 64, 0, dev=dev)
k, v = pr.Pool(tq, 1, pages, 2, 64, 128, 3, dev), pr.Pool(tq, 2, pages, 2, 64, 128, 3, dev)
q = torch.randn((1, 8, 128), device=dev, dtype=torch.float16)
seq = torch.tensor([100], dtype=torch.int32, device=dev)
call = lambda: tq.paged_decode(q, k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=0.1)
torch.cuda.synchronize()
g, out = torch.cuda.CUDAGraph(), None
try:
    with torch.cuda.graph(g):
        out = call()
except Exception as ex:
    print("raised", type(ex).__name__)
    out = None
want = call()
if out is not None:
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
ref, tol = pr.decode_ref(tq, q, k, v, table, [100], 0.1, weight_eps=2.0 ** -11, out_dtype=want.dtype)
pr.check(want, ref, tol)
print("fine")
""" % (os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__)))
    import subprocess
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_decode_repeats_exactly(tq, dev):
    got, (q, k, v, table, seq, scale) = _decode(tq, dev, lens=[5000, 3], n_q=28, n_kv=4)
    for _ in range(3):
        assert torch.equal(tq.paged_decode(q, k=k.desc, v=v.desc, page_table=table, seq_lens=seq, attn_scale=scale), got)


# ---- insert ---------------------------------------------------------------------------------------------------
def _append(tq, dev, *, starts, counts, tokens, n_kv=2, dim=128, kbits=3, vbits=4, page=64, dtype=torch.float16, seed=0,
            token_major=True, pass_counts=True):
    total = [s + c for s, c in zip(starts, counts)]
    table, pages = pr.make_table(total, page, seed, dev=dev)
    k = pr.Pool(tq, seed + 1, pages, n_kv, page, dim, kbits, dev, dtype=dtype)
    v = pr.Pool(tq, seed + 2, pages, n_kv, page, dim, vbits, dev)
    g = torch.Generator().manual_seed(seed)
    shape = (len(starts), tokens, n_kv, dim) if token_major else (len(starts), n_kv, tokens, dim)
    keys, values = [(torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[:3], generator=g))[..., None]).to(dtype).to(dev)
                    for _ in range(2)]
    if token_major:
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    for b, c in enumerate(counts):       # padded tokens may hold anything
        keys[b, :, c:] = float("nan")
        values[b, :, c:] = float("inf")
    want = []
    for x, pool in ((keys, k), (values, v)):
        if pool.bits == 0:
            data = pool.data.clone()
            for b, (s, c) in enumerate(zip(starts, counts)):
                for t in range(c):
                    data[table[b, (s + t) // page].item(), :, (s + t) % page] = x[b, :, t]
            want.append([data])
            continue
        packed, norms = pool.packed.clone().view(torch.int32), pool.norms.clone()
        for b, (s, c) in enumerate(zip(starts, counts)):
            if c == 0:
                continue
            w, nn = tq.fused_quantize(x[b, :, :c].reshape(-1, dim), pool.quant.signs, pool.quant.boundaries, dim, pool.bits)
            w, nn = w.view(torch.int32).view(n_kv, c, -1), nn.view(n_kv, c)
            pos = torch.arange(s, s + c, device=dev)
            pg = table[b].long()[pos // page]
            packed[pg, :, pos % page] = w.transpose(0, 1)
            norms[pg, :, pos % page] = nn.t()
        want.append([packed, norms])
    tq.paged_append(keys, values, k=k.desc, v=v.desc, page_table=table,
                    starts=torch.tensor(starts, dtype=torch.int32, device=dev),
                    counts=torch.tensor(counts, dtype=torch.int32, device=dev) if pass_counts else None)
    for pool, w in ((k, want[0]), (v, want[1])):
        have = [pool.data] if pool.bits == 0 else [pool.packed.view(torch.int32), pool.norms]
        for a, b in zip(have, w):
            assert torch.equal(a, b)
    assert tq.paged_status(dev) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kbits,vbits", [(0, 3), (3, 3), (4, 3), (3, 4), (1, 2), (2, 4)])
def test_append_words_and_neighbours(tq, dev, dtype, kbits, vbits):
    """The contiguous quantizer's words and norms at the right places, and nothing else touched."""
    _append(tq, dev, starts=[0, 61, 130, 5], counts=[70, 67, 0, 1], tokens=70, kbits=kbits, vbits=vbits, dtype=dtype)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 300])
@pytest.mark.parametrize("token_major", [True, False])
def test_append_lengths(tq, dev, tokens, token_major):
    _append(tq, dev, starts=[63, 0, 1000], counts=[tokens, max(1, tokens // 2), tokens], tokens=tokens, token_major=token_major)


@pytest.mark.parametrize("dim", [32, 64, 256])
def test_append_dims(tq, dev, dim):
    _append(tq, dev, starts=[40, 3], counts=[50, 9], tokens=50, dim=dim)


def test_append_without_counts(tq, dev):
    _append(tq, dev, starts=[40, 3], counts=[5, 5], tokens=5, pass_counts=False)


def test_append_extreme_rows(tq, dev):
    """Zero rows, subnormal and huge rows, rows at an odd element offset."""
    dim, page = 128, 32
    table = torch.tensor([[1]], dtype=torch.int32, device=dev)
    k, v = pr.Pool(tq, 1, 2, 1, page, dim, 3, dev), pr.Pool(tq, 2, 2, 1, page, dim, 4, dev)
    x = torch.randn((6, dim), generator=torch.Generator().manual_seed(4)).to(dev)
    x[0], x[1], x[2], x[3] = 0, x[1] * 1e-38, x[2] * 1e18, x[3] * 1e-8
    buf = torch.zeros((6 * dim + 1,), device=dev)[1:].view(1, 1, 6, dim)
    buf.copy_(x[None, None])
    tq.paged_append(buf, buf, k=k.desc, v=v.desc, page_table=table, starts=torch.zeros(1, dtype=torch.int32, device=dev))
    for pool in (k, v):
        w, n = tq.fused_quantize(x, pool.quant.signs, pool.quant.boundaries, dim, pool.bits)
        assert torch.equal(pool.packed[1, 0, :6].view(torch.int32), w.view(torch.int32)) and torch.equal(pool.norms[1, 0, :6], n)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_extreme_rows_of_a_prompt(tq, dev, dtype):
    """A prompt's worth of zero, subnormal, huge, infinite, NaN and border rows: the words of the contiguous quantizer."""
    dim, page, n = 128, 64, 100
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=dev)
    k, v = pr.Pool(tq, 1, 4, 2, page, dim, 3, dev), pr.Pool(tq, 2, 4, 2, page, dim, 4, dev)
    x = torch.randn((2, n, dim), generator=torch.Generator().manual_seed(4))
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = 0, x[:, 1] * 1e-6, x[:, 2] * 1e4, x[:, 3] * 1e-3
    x[:, 4, 7], x[:, 5, 9], x[:, 6, 127] = float("inf"), float("nan"), -float("inf")
    x[:, 7] = k.quant.signs.cpu()                       # rotates onto one axis
    x[:, 8] = 0
    x[:, 8, 64] = 1                                      # rotates to equal magnitudes
    if dtype == torch.bfloat16:
        x[:, 9], x[:, 10], x[:, 11] = x[:, 9] * 1e-38, x[:, 10] * 1e18, x[:, 11] * 1e30
    x = x.to(dtype).to(dev)
    tq.paged_append(x[None], x[None], k=k.desc, v=v.desc, page_table=table, starts=torch.zeros(1, dtype=torch.int32, device=dev))
    for pool in (k, v):
        w, nn = tq.fused_quantize(x.reshape(-1, dim), pool.quant.signs, pool.quant.boundaries, dim, pool.bits)
        w, nn = w.view(torch.int32).view(2, n, -1), nn.view(2, n)
        got = pool.packed.view(torch.int32)[[3, 1]].transpose(0, 1).flatten(1, 2)[:, :n]
        assert torch.equal(got, w)
        assert torch.equal(pool.norms[[3, 1]].transpose(0, 1).flatten(1, 2)[:, :n].nan_to_num(7.0), nn.nan_to_num(7.0))


@pytest.mark.parametrize("bits", [3, 4])
def test_append_other_codebooks(tq, dev, bits):
    """Borders that are uneven, nearly equal or all alike: the count of borders below, whatever the kernel."""
    dim, page, n, levels = 128, 32, 40, 1 << bits
    x = torch.randn((1, 1, n, dim), generator=torch.Generator().manual_seed(5)).half().to(dev)
    for seed, borders in enumerate((torch.linspace(-3, 3, levels - 1) ** 3, torch.linspace(-1e-4, 1e-4, levels - 1),
                                    torch.zeros(levels - 1), torch.linspace(0.1, 0.11, levels - 1))):
        k, v = pr.Pool(tq, 1, 3, 1, page, dim, bits, dev), pr.Pool(tq, 2, 3, 1, page, dim, bits, dev)
        borders = borders.to(dev)
        k.desc["boundaries"] = v.desc["boundaries"] = borders
        tq.paged_append(x, x, k=k.desc, v=v.desc, page_table=torch.tensor([[2, 0]], dtype=torch.int32, device=dev),
                        starts=torch.zeros(1, dtype=torch.int32, device=dev))
        for pool in (k, v):
            w, _ = tq.fused_quantize(x[0, 0], pool.quant.signs, borders, dim, bits)
            got = pool.packed.view(torch.int32)[[2, 0], 0].flatten(0, 1)[:n]
            assert torch.equal(got, w.view(torch.int32)), seed


def test_append_bad_places_in_a_prompt(tq, dev):
    """One page of a prompt outside the pool: its tokens are skipped, the others stored, neighbours untouched."""
    page, dim, n = 32, 128, 90
    k, v = pr.Pool(tq, 1, 4, 1, page, dim, 3, dev), pr.Pool(tq, 2, 4, 1, page, dim, 4, dev)
    x = torch.randn((1, 1, n, dim), device=dev, dtype=torch.float16)
    before = [(p.packed.view(torch.int32).clone(), p.norms.clone()) for p in (k, v)]
    tq.paged_append(x, x, k=k.desc, v=v.desc, page_table=torch.tensor([[2, 9, 0]], dtype=torch.int32, device=dev),
                    starts=torch.tensor([5], dtype=torch.int32, device=dev))
    assert tq.paged_status(dev) in (1, 2)
    pos = torch.arange(5, 5 + n, device=dev)
    keep = (pos // page) != 1
    for pool, (words, norms) in zip((k, v), before):
        w, nn = tq.fused_quantize(x[0, 0], pool.quant.signs, pool.quant.boundaries, dim, pool.bits)
        pg = torch.tensor([2, 9, 0], device=dev)[pos[keep] // page]
        words[pg, 0, pos[keep] % page] = w.view(torch.int32)[keep]
        norms[pg, 0, pos[keep] % page] = nn[keep]
        assert torch.equal(pool.packed.view(torch.int32), words) and torch.equal(pool.norms, norms)


def test_append_bad_places_are_skipped(tq, dev):
    """Pages outside the pool and positions behind the table are reported and not followed."""
    page, dim = 32, 128
    k, v = pr.Pool(tq, 1, 3, 1, page, dim, 3, dev), pr.Pool(tq, 2, 3, 1, page, dim, 3, dev)
    before = [t.clone() for t in (k.packed.view(torch.int32), k.norms, v.packed.view(torch.int32), v.norms)]
    x = torch.randn((1, 1, 4, dim), device=dev)
    for table, start, code in (([[3, 0]], 0, 1), ([[-1, 0]], 10, 1), ([[0, 1]], 64, 2), ([[0, 1]], -9, 2), ([[0, 1]], 2 ** 31 - 1, 2)):
        tq.paged_append(x, x, k=k.desc, v=v.desc, page_table=torch.tensor(table, dtype=torch.int32, device=dev),
                        starts=torch.tensor([start], dtype=torch.int32, device=dev))
        assert tq.paged_status(dev) == code
        for a, b in zip(before, (k.packed.view(torch.int32), k.norms, v.packed.view(torch.int32), v.norms)):
            assert torch.equal(a, b)


# ---- read back --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits,dim", [(3, 128), (4, 128), (1, 128), (2, 64), (3, 32), (4, 256), (0, 128)])
def test_read_back(tq, dev, dtype, bits, dim):
    """The contiguous decoder's bits, zeros behind each sequence."""
    lens, page, length, H = [100, 0, 1, 333], 64, 300, 2
    table, pages = pr.make_table(lens, page, 5, dev=dev)
    pool = pr.Pool(tq, 6, pages, H, page, dim, bits, dev, dtype=torch.float16)
    got = tq.paged_dequantize(pool.desc, page_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                              length=length, dtype=dtype)
    assert got.shape == (4, H, length, dim) and got.dtype == dtype
    for b, n in enumerate(lens):
        n = min(n, length)
        assert bool((got[b, :, n:] == 0).all())
        if n == 0:
            continue
        pg = table[b].long()[:-(-n // page)]
        if bits == 0:
            want = pool.data[pg].transpose(0, 1).flatten(1, 2)[:, :n].to(dtype)
        else:
            w = pool.packed.view(torch.int32)[pg].transpose(0, 1).flatten(1, 2)[:, :n].contiguous().view(torch.uint32)
            nn = pool.norms[pg].transpose(0, 1).flatten(1, 2)[:, :n].contiguous()
            f = tq.kernels._dequant(w.view(H * n, -1), nn.view(-1), pool.quant.centroids, pool.quant.signs, dim, bits, dtype)
            want = f.view(H, n, dim)
        assert torch.equal(got[b, :, :n], want)
    if bits:
        ref = pool.rows(tq, table[0].cpu().long()[:2], 100)
        # log2(dim) + 4 roundings of 32 bits, relative to the largest term sum of the butterfly, and one of the output
        reach = pool.rotated(tq, table[0].cpu().long()[:2], 100).abs().sum(-1, keepdim=True)
        tol = (math.log2(dim) + 4) * 2.0 ** -24 * reach + torch.finfo(dtype).eps / 2 * ref.abs() + 1e-12
        pr.check(got[0, :, :100], ref, tol)


def test_read_back_page_outside_pool(tq, dev):
    pool = pr.Pool(tq, 6, 4, 2, 32, 128, 3, dev)
    table = torch.tensor([[0, 9, 1]], dtype=torch.int32, device=dev)
    got = tq.paged_dequantize(pool.desc, page_table=table, seq_lens=torch.tensor([70], dtype=torch.int32, device=dev), length=80)
    assert bool(got[:, :, 32:64].isnan().all()) and bool(got[:, :, :32].isfinite().all()) and bool((got[:, :, 70:] == 0).all())
    assert tq.paged_status(dev) == 1


# ---- page copies ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n_pools", [1, 4, 130])
def test_copy_pages(tq, dev, n_pools):
    g = torch.Generator().manual_seed(1)
    pools = [torch.randint(0, 99, (10, 2, 32, 4 if i % 3 else 13), generator=g, dtype=torch.int32).to(dev) for i in range(n_pools)]
    want = [p.clone() for p in pools]
    src, dst = [1, 1, 7], [0, 9, 4]
    for p in want:
        p[dst] = p[src]
    tq.copy_pages(pools, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    tq.copy_pages(pools, torch.tensor([4], dtype=torch.int32, device=dev), torch.tensor([5], dtype=torch.int32, device=dev))
    for p in want:
        p[5] = p[4]
    tq.copy_pages(pools, [], [])
    assert all(torch.equal(a, b) for a, b in zip(pools, want)) and tq.paged_status(dev) == 0
    tq.copy_pages(pools, torch.tensor([4, 10], dtype=torch.int32, device=dev), torch.tensor([-1, 3], dtype=torch.int32, device=dev))
    assert all(torch.equal(a, b) for a, b in zip(pools, want)) and tq.paged_status(dev) == 1


# ---- prompt attention with a window --------------------------------------------------------------------------------
@pytest.mark.parametrize("L,S", [(1, 1), (5, 5), (127, 127), (128, 128), (129, 400), (300, 300), (700, 1000), (1, 500)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 4), (128, 0), (129, 130), (200, 300), (10 ** 6, 3)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_window(tq, dev, L, S, window, sinks, dtype):
    B, n_q, n_kv, D = 2, 4, 2, 128
    g = torch.Generator().manual_seed(L * 7 + S)
    q, k, v = [torch.randn((B, m, h, D), generator=g).to(dtype).to(dev).transpose(1, 2)
               for m, h in ((L, n_q), (S, n_kv), (S, n_kv))]
    scale = 1 / math.sqrt(D)
    got = tq.prefill_attention(q, k, v, scale, causal=True, window=window, sinks=sinks)
    assert tq.kernels.prefill_status(dev) == 0
    qd, kd, vd = [t.cpu().double() for t in (q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1))]
    s = qd @ kd.transpose(-1, -2) * scale
    mag = qd.abs() @ kd.abs().transpose(-1, -2) * scale
    i, j = torch.arange(L)[:, None] + S - L, torch.arange(S)
    seen = (j <= i) & ((j > i - window) | (j < sinks))
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    ref = p @ vd
    # scores: 128 products in 32 bits, 4 roundings of the scaled score, 2^-22 of the exponential; weights of the 16-bit
    # type; S terms summed in 32 bits; one rounding of the output
    d = ((D + 8) * 2.0 ** -24 * mag).masked_fill(~seen, 0).amax(-1, keepdim=True) + \
        4 * 2.0 ** -24 * s.abs().masked_fill(~seen, 0).amax(-1, keepdim=True) + 2.0 ** -22
    half = torch.finfo(dtype).eps / 2
    reach = p @ vd.abs()
    rel = 2 * d + half + S * 2.0 ** -24
    pr.check(got, ref, rel * reach + half * (ref.abs() + rel * reach) + 1e-12)


def test_prompt_window_equals_full_form_when_wide(tq, dev):
    q, k, v = [torch.randn((1, h, 300, 128), device=dev, dtype=torch.float16) for h in (4, 2, 2)]
    full = tq.prefill_attention(q, k, v, 0.1)
    assert torch.equal(tq.prefill_attention(q, k, v, 0.1, window=300, sinks=2), full)


@pytest.mark.parametrize("L,S,causal,window,sinks", [
    (64, 64, True, 0, 0), (64, 64, True, 20, 3), (130, 130, True, 0, 0), (130, 300, True, 100, 5), (200, 700, True, 300, 1),
    (513, 513, True, 0, 0), (513, 513, True, 140, 200), (90, 100, False, 0, 0), (150, 260, False, 0, 0)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_many_items(tq, dev, L, S, causal, window, sinks, dtype):
    """Several work items per SM, of one key tile and more, with scores large enough for the accumulators to be rescaled."""
    B, n_q, n_kv, D, gain = 11, 32, 8, 128, 4.0
    g = torch.Generator(device="cuda").manual_seed(L + S)
    q, k, v = [torch.randn((B, h, n, D), generator=g, device=dev).to(dtype) for h, n in ((n_q, L), (n_kv, S), (n_kv, S))]
    q = q * gain
    scale = 1 / math.sqrt(D)
    got = tq.prefill_attention(q, k, v, scale, causal=causal, window=window, sinks=sinks)
    again = tq.prefill_attention(q, k, v, scale, causal=causal, window=window, sinks=sinks)
    assert tq.kernels.prefill_status(dev) == 0 and torch.equal(got, again)
    half = torch.finfo(dtype).eps / 2
    i, j = torch.arange(L, device=dev)[:, None] + S - L, torch.arange(S, device=dev)
    seen = torch.ones((L, S), dtype=torch.bool, device=dev) if not causal else j <= i
    if window:
        seen &= (j > i - window) | (j < sinks)
    for b in range(B):                 # the tolerance of test_prompt_window
        qd, kd, vd = [t[b].double() for t in (q, k.repeat_interleave(n_q // n_kv, 1), v.repeat_interleave(n_q // n_kv, 1))]
        s = qd @ kd.transpose(-1, -2) * scale
        mag = qd.abs() @ kd.abs().transpose(-1, -2) * scale
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        ref = p @ vd
        d = ((D + 8) * 2.0 ** -24 * mag).masked_fill(~seen, 0).amax(-1, keepdim=True) + \
            4 * 2.0 ** -24 * s.abs().masked_fill(~seen, 0).amax(-1, keepdim=True) + 2.0 ** -22
        reach = p @ vd.abs()
        rel = 2 * d + half + S * 2.0 ** -24
        pr.check(got[b], ref.cpu(), (rel * reach + half * (ref.abs() + rel * reach) + 1e-12).cpu(), f"batch {b}")


def test_prompt_out_is_checked(tq, dev):
    q, k, v = [torch.randn((1, h, 40, 128), device=dev, dtype=torch.float16) for h in (4, 2, 2)]
    want = tq.prefill_attention(q, k, v, 0.1, window=16)
    out = torch.empty((1, 40, 4, 128), device=dev, dtype=torch.float16).transpose(1, 2)
    assert tq.prefill_attention(q, k, v, 0.1, window=16, out=out) is not None and torch.equal(out, want)
    for bad in (out.float(), out[:, :3], out.cpu(), torch.empty((1, 4, 40, 129), device=dev, dtype=torch.float16)[..., :128]):
        with pytest.raises(ValueError):
            tq.prefill_attention(q, k, v, 0.1, window=16, out=bad)
    with pytest.raises(ValueError):
        tq.prefill_attention(q, k, v[:, :, :39], 0.1)
    with pytest.raises(RuntimeError, match="CUDA"):
        tq.prefill_attention(q, k.cpu(), v, 0.1)
    odd = torch.randn((1 * 2 * 40 * 128 + 1,), device=dev).half()[1:].view(1, 2, 40, 128)        # not 16-byte aligned
    assert torch.equal(tq.prefill_attention(q, odd, v, 0.1, window=16), tq.prefill_attention(q, odd.clone(), v, 0.1, window=16))
