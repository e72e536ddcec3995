"""The paged cache as a model uses it: ragged batches through the hook, forks, windows, compaction, a decode loop."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as pr  # noqa: E402

pytestmark = pytest.mark.gpu
D = 128


class _Half:
    """A cache half seen by the 64-bit reference."""

    def __init__(self, cache, desc, q):
        self.bits, self.dim, self.page = (q.bits if q else 0), cache.dim, cache.sequences.page_size
        if q is None:
            self.data = desc["data"]
        else:
            self.packed, self.norms, self.quant = desc["packed"], desc["norms"], q

    rotated, rows = pr.Pool.rotated, pr.Pool.rows


def _reference(tq, cache, q, scale):
    s = cache.sequences
    return pr.decode_ref(tq, q, _Half(cache, cache.k, cache._k_q), _Half(cache, cache.v, cache._v_q), s.table,
                         s._host_lens, scale, s.window, s.sinks, torch.finfo(torch.float16).eps / 2, q.dtype)


@pytest.fixture()
def hook(tq):
    tq.apply_patch()
    yield tq.base
    tq.remove_patch()


def _tokens(B, H, T, dtype, dev, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((B, T, H, D), generator=g).to(dtype).to(dev).transpose(1, 2) for _ in range(2)]


@pytest.mark.parametrize("k_bits", [0, 3, 4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_ragged_batch_through_the_hook(tq, dev, hook, k_bits, window, sinks):
    """Prompts one by one, a fork, ragged decode steps: every step's attention against the 64-bit reference over the
    pages, and the pages against the contiguous cache that was fed the same rows."""
    dtype, n_kv, n_q, scale = torch.float16, 2, 8, 1 / math.sqrt(D)
    caches = tq.make_paged_caches(2, 30, n_kv, bits=3, k_bits=k_bits, page_size=32, window=window, sinks=sinks, dtype=dtype)
    seqs = caches[0].sequences
    plain = {}

    def feed(ids, T, seed, counts=None):
        seqs.begin(ids, T if counts is None else counts)
        keys, values = _tokens(len(ids), n_kv, T, dtype, dev, seed)
        q = torch.randn((len(ids), n_q, T, D), generator=torch.Generator().manual_seed(seed + 1)).to(dtype).to(dev)
        outs = []
        for c in caches:
            k, v = c.update_and_fetch(keys, values)
            outs.append(hook.scaled_dot_product_attention(q, k, v, c, scale, c.make_mask(T)))
        assert torch.equal(outs[0], outs[1])             # the layers hold the same
        for b, s in enumerate(ids):
            n = T if counts is None else counts[b]
            if n:
                plain[s].update_and_fetch(keys[b:b + 1, :, :n], values[b:b + 1, :, :n])
        return q, outs[0]

    def check_step(q, out):
        if q.shape[2] == 1:
            ref, tol = _reference(tq, caches[0], q[:, :, 0], scale)
            pr.check(out[:, :, 0], ref, tol)

    ids = []
    for i, n in enumerate((70, 1, 200)):
        s = seqs.add()
        plain[s] = tq.TurboQuantKVCache(bits=3, v_only=k_bits == 0, k_bits=k_bits or None)
        q, out = feed([s], n, 10 * i)
        check_step(q, out)
        ids.append(s)
    forked = seqs.fork(ids[2])
    plain[forked] = tq.TurboQuantKVCache(bits=3, v_only=k_bits == 0, k_bits=k_bits or None)
    state = [t.clone() for t in plain[ids[2]].state]
    plain[forked] = tq.TurboQuantKVCache.from_state(state, plain[ids[2]].meta_state)
    for step in range(3):
        check_step(*feed(ids + [forked], 1, 100 + step))
    check_step(*feed([ids[1], forked], 1, 150, counts=[0, 1]))
    q, out = feed([ids[0], ids[2]], 9, 160, counts=[9, 4])                 # a ragged continuation, several tokens
    assert bool((out[1, :, 4:] == 0).all()) and bool(out.isfinite().all())
    for s in ids + [forked]:
        pages = torch.tensor(seqs._pages[s], device=dev)
        n = seqs.length(s)
        for desc, name in ((caches[1].v, "v"),) + (((caches[1].k, "k"),) if k_bits else ()):
            words = desc["packed"].view(torch.int32)[pages.clamp(min=0)].transpose(0, 1).flatten(1, 2)[:, :n]
            norms = desc["norms"][pages.clamp(min=0)].transpose(0, 1).flatten(1, 2)[:, :n]
            held = (pages >= 0).repeat_interleave(32)[:n]
            want_w = getattr(plain[s], name + "_packed")[0, :, :n].contiguous().view(torch.int32)
            assert torch.equal(words[:, held], want_w[:, held])
            assert torch.equal(norms[:, held], getattr(plain[s], name + "_norms")[0, :, :n][:, held])
    seqs.free(ids[0])
    seqs.compact()
    check_step(*feed([forked, ids[1]], 1, 170))
    seqs.resize(seqs.used_pages + 4)
    check_step(*feed([ids[2], forked], 1, 180))
    for s in (ids[1], ids[2], forked):
        seqs.free(s)
    assert seqs.used_pages == 0 and tq.paged_status(dev) == 0


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_steps_attend_over_the_pages(tq, dev, hook, window, sinks, dim):
    """Several tokens behind a cached prefix, against 64 bits over the values the pages stand for."""
    n_kv, n_q, scale = 2, 4, 1 / math.sqrt(dim)
    cache = tq.make_paged_caches(1, 20, n_kv, dim=dim, page_size=32, window=window, sinks=sinks)[0]
    seqs = cache.sequences
    s = seqs.add()
    for T in (50, 33, 130):
        seqs.begin([s], T)
        g = torch.Generator().manual_seed(T)
        keys, values = [torch.randn((1, n_kv, T, dim), generator=g).half().to(dev) for _ in range(2)]
        q = torch.randn((1, n_q, T, dim), generator=g).half().to(dev)
        k, v = cache.update_and_fetch(keys, values)
        out = hook.scaled_dot_product_attention(q, k, v, cache, scale, "causal")
        n = seqs.length(s)
        kd, vd = [t.cpu().double().repeat_interleave(2, 1) for t in cache.dequantized(torch.float16)]
        sc = q.cpu().double() @ kd.transpose(-1, -2) * scale
        i, j = torch.arange(T)[:, None] + n - T, torch.arange(n)
        seen = (j <= i) & ((j > i - window) | (j < sinks)) if window else j <= i
        mag = (q.cpu().double().abs() @ kd.abs().transpose(-1, -2) * scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
        p = torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
        ref, reach = p @ vd, p @ vd.abs()
        half = torch.finfo(torch.float16).eps / 2
        # 32-bit scores (dim terms, 4 roundings), 16-bit weights, a 16-bit result; the library's attention may round its
        # scores to 16 bits too (dim 64 takes it): half a step of the largest score
        rel = 2 * ((dim + 12) * 2.0 ** -24 * mag + (half * mag if dim != 128 else 0)) + 2 * half + n * 2.0 ** -24
        pr.check(out, ref, rel * reach + half * (ref.abs() + rel * reach) + 1e-12)


def test_refusals(tq, dev, hook):
    cache = tq.make_paged_caches(1, 4, 2)[0]
    x = torch.zeros((1, 2, 1, D), dtype=torch.float16, device=dev)
    with pytest.raises(RuntimeError, match="begin"):
        cache.update_and_fetch(x, x)
    s = cache.sequences.add()
    cache.sequences.begin([s], 2)
    with pytest.raises(ValueError, match="2 per sequence"):
        cache.update_and_fetch(x, x)
    with pytest.raises(ValueError, match="sequences and"):
        cache.update_and_fetch(x[:, :1], x[:, :1])
    with pytest.raises(ValueError, match="array masks"):
        cache.attention(torch.zeros((1, 4, 2, D), device=dev), 1.0, torch.zeros((2, 2), device=dev))
    with pytest.raises(ValueError):
        cache.make_mask(3, return_array=True)
    # wrappers: shapes, types, devices of the arguments
    k, v, t, n = cache.k, cache.v, cache.sequences.table, cache.sequences.lens
    q = torch.zeros((1, 4, D), dtype=torch.float16, device=dev)
    ok = dict(k=k, v=v, page_table=t, seq_lens=n, attn_scale=1.0)
    tq.paged_decode(q, **ok)
    for bad in (dict(page_table=t.long()), dict(page_table=t[0]), dict(seq_lens=n.long()), dict(seq_lens=n.expand(2)),
                dict(k=dict(k, bits=4)), dict(k=dict(k, bits=5)), dict(k=dict(k, norms=k["norms"][:, :, :32])),
                dict(v=dict(v, packed=v["packed"].view(torch.int32))), dict(k=dict(format="affine")), dict(window=-1),
                dict(sinks=3), dict(out=q[:, :2]), dict(out=q.float(), out_dtype=torch.float16), dict(out_dtype=torch.int32),
                dict(workspace=torch.zeros(10, dtype=torch.uint8, device=dev)), dict(v=dict(format="dense", data=torch.zeros((4, 2, 64, D), device=dev))),
                dict(k=dict(k, centroids=v["boundaries"])), dict(attn_scale=float("nan"))):
        with pytest.raises(ValueError):
            tq.paged_decode(q, **{**ok, **bad})
    with pytest.raises(ValueError):
        tq.paged_decode(q[:, :3], **ok)
    with pytest.raises(ValueError):
        tq.paged_decode(q.double(), **ok)
    with pytest.raises(RuntimeError, match="CUDA"):
        tq.paged_decode(q, **{**ok, "page_table": t.cpu()})
    y = torch.zeros((1, 2, 2, D), dtype=torch.bfloat16, device=dev)
    args = dict(v=v, page_table=t, starts=n)
    dense = dict(format="dense", data=torch.zeros((4, 2, 64, D), dtype=torch.float16, device=dev))
    for bad in (dict(k=dense), dict(k=k, counts=n.long()), dict(k=k, starts=n.float())):
        with pytest.raises(ValueError):
            tq.paged_append(y, y, **{**args, **bad})
    with pytest.raises(ValueError):
        tq.paged_append(y, y[:, :, :1], k=k, **args)
    with pytest.raises(ValueError):
        tq.paged_dequantize(v, page_table=t, seq_lens=n, length=-1)
    pools = cache.pools()
    for src, dst in (([0], [0, 1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([4], [0]), ([0], [-1])):
        with pytest.raises(ValueError):
            tq.copy_pages(pools, src, dst)
    with pytest.raises(ValueError):
        tq.copy_pages([pools[0].transpose(0, 1)], [0], [1])
    with pytest.raises(ValueError):
        tq.copy_pages([torch.zeros((4, 3), device=dev)], [0], [1])
    for bad in (dict(window=-1), dict(sinks=2), dict(window=4, causal=False)):
        z = torch.zeros((1, 2, 4, D), dtype=torch.float16, device=dev)
        with pytest.raises(ValueError):
            tq.prefill_attention(z, z, z, 1.0, **bad)


def test_model_ragged_decode(tq, dev, hook):
    """A small model: prompts of three lengths, then all together; logits against the same model over contiguous caches,
    captured steps against eager ones, a fork that continues like its parent."""
    q2 = sys.modules["turboquant_mlx_b200.qwen2"] if "turboquant_mlx_b200.qwen2" in sys.modules else __import__(
        "importlib").import_module("turboquant_mlx_b200.qwen2")
    cfg = q2.Qwen2Config(n_layers=3, hidden=256, n_q_heads=8, n_kv_heads=2, ffn=512, vocab=500)
    model = q2.Qwen2Model(cfg, dev, dtype=torch.float16)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).to(dev) for n in (37, 90, 5)]

    def run(use_graph):
        caches = tq.make_paged_caches(cfg.n_layers, 40, cfg.n_kv_heads, page_size=32)
        dec = q2.PagedDecoder(model, caches)
        ids, firsts = zip(*[dec.prefill(p) for p in prompts])
        first = torch.cat(firsts)
        return dec, list(ids), first, dec.generate(list(ids), first, 40, use_graph=use_graph)

    dec, ids, first, toks = run(False)
    _, _, first2, toks2 = run(True)
    assert torch.equal(first, first2) and torch.equal(toks, toks2)
    assert [dec.seqs.length(s) for s in ids] == [37 + 40, 90 + 40, 5 + 40]
    # teacher-forced: the contiguous caches' logits at every step of each sequence
    for b, p in enumerate(prompts):
        flat = [tq.TurboQuantKVCache(bits=3, fused=True) for _ in range(cfg.n_layers)]
        logits = model.forward(p[None], flat)
        step = first[b:b + 1]
        paged = tq.make_paged_caches(cfg.n_layers, 40, cfg.n_kv_heads, page_size=32)
        seqs = paged[0].sequences
        s = seqs.add()
        seqs.begin([s], p.shape[0])
        mine = model.forward(p[None], paged)
        # both attend over the same rows with 16-bit weights (relative 2^-11 each) in 16-bit models: a few 16-bit steps of
        # the logits' scale per layer
        bound = 16 * cfg.n_layers * torch.finfo(torch.float16).eps * float(logits.float().abs().max())
        assert float((mine.float() - logits.float()).abs().max()) <= bound
        for k in range(6):
            seqs.begin([s], 1)
            a = model.decode_step(step, paged, seqs.starts)
            c = model.forward(step, flat)[:, -1]
            assert float((a.float() - c.float()).abs().max()) <= bound, (b, k)
            step = toks[b:b + 1, k:k + 1]
    # a fork continues exactly like its parent, in one batch with it
    twin = dec.seqs.fork(ids[1])
    last = toks[1:2, -1:]
    both = dec.generate([ids[1], twin], last.expand(2, 1).contiguous(), 10)
    assert torch.equal(both[0], both[1])
    assert dec.prefill(prompts[2], ids[2])[0] == ids[2] and dec.seqs.length(ids[2]) == 50
    with pytest.raises(RuntimeError, match="apply_patch"):
        tq.remove_patch()
        q2.PagedDecoder(model, dec.caches)


def test_decode_loop_with_window_in_a_graph(tq, dev, hook):
    """A windowed stream decoded far past its window, the pages of the run reserved before it: captured equals eager."""
    q2 = __import__("importlib").import_module("turboquant_mlx_b200.qwen2")
    cfg = q2.Qwen2Config(n_layers=2, hidden=256, n_q_heads=4, n_kv_heads=2, ffn=256, vocab=200)
    model = q2.Qwen2Model(cfg, dev, dtype=torch.bfloat16)
    prompt = torch.arange(50, device=dev) % 200
    got = []
    for use_graph in (False, True):
        caches = tq.make_paged_caches(2, 12, 2, bits=4, page_size=32, window=48, sinks=2, dtype=torch.bfloat16)
        dec = q2.PagedDecoder(model, caches)
        s, tok = dec.prefill(prompt)
        out = []
        for _ in range(4):
            out.append(dec.generate([s], tok, 60, use_graph=use_graph))
            tok = out[-1][:, -1:]
        got.append(torch.cat(out, 1))
        held = sum(p >= 0 for p in dec.seqs._pages[s])
        assert held <= 6 and dec.seqs.length(s) == 290
    assert torch.equal(got[0], got[1]) and tq.paged_status(dev) == 0


def test_step_scratch(tq, dev, hook):
    """A capture without an eager call in front brings its own scratch; steps do not share theirs; resize ends a step."""
    scale = 1 / math.sqrt(D)
    cache, = tq.make_paged_caches(1, 12, 1, page_size=32)
    seqs = cache.sequences
    ids = [seqs.add()]
    seqs.begin(ids, 300)
    cache.update_and_fetch(*_tokens(1, 1, 300, torch.float16, dev, 0))
    seqs.begin(ids, 1)
    keys, values = _tokens(1, 1, 1, torch.float16, dev, 1)
    q = torch.randn((1, 8, 1, D), generator=torch.Generator().manual_seed(2)).half().to(dev)
    cache.update_and_fetch(keys, values)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hook.scaled_dot_product_attention(q, keys, values, cache, scale, None)
    for _ in range(3):
        graph.replay()
        eager = hook.scaled_dot_product_attention(q, keys, values, cache, scale, None)
        assert torch.equal(out, eager)
    ref, tol = _reference(tq, cache, q[:, :, 0], scale)
    pr.check(out[:, :, 0], ref, tol)
    first = seqs._workspace(D)
    del graph
    seqs.begin(ids, 1)
    assert seqs._workspace(D) is not first
    with pytest.raises(ValueError, match="sink"):
        hook.scaled_dot_product_attention(q, keys, values, cache, scale, None, sinks=torch.zeros(8, device=dev))
    seqs.resize(16)
    with pytest.raises(RuntimeError, match="begin"):
        cache.update_and_fetch(keys, values)
