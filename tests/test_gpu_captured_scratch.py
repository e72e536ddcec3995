"""Decode and prompt calls captured in graphs: whose scratch they use."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


def _halves(tq, dev, seed, n=3000, n_kv=2):
    x = torch.randn((2, 1, n_kv, n, 128), generator=torch.Generator().manual_seed(seed)).half().to(dev)
    out = []
    for i in range(2):
        pq = tq.PolarQuantizer(128, 3, seed=seed + i, device=dev)
        w, norms = tq.fused_quantize(x[i].reshape(-1, 128), pq.signs, pq.boundaries, 128, 3)
        out.append(dict(format="polar", packed=w.view(1, n_kv, n, -1), norms=norms.view(1, n_kv, n), bits=3, signs=pq.signs,
                        centroids=pq.centroids))
    q = torch.randn((1, 8, 128), generator=torch.Generator().manual_seed(seed + 9)).half().to(dev)
    return lambda **kw: tq.flash_decode(q, k=out[0], v=out[1], attn_scale=0.09, **kw)


def test_two_graphs_side_by_side(tq, dev):
    """Captured one after the other on the capture stream of torch, replayed at the same time on two streams, with eager
    calls beside them; both were captured before any of them ran."""
    calls = [_halves(tq, dev, s) for s in (1, 50)]
    want = [c() for c in calls]
    p = [torch.randn((1, h, 300, 128), device=dev, dtype=torch.float16) for h in (4, 2, 2)]
    prompt = tq.prefill_attention(*p, 0.1)
    torch.cuda.synchronize()
    graphs = []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = [c() for _ in range(5)] + [tq.prefill_attention(*p, 0.1)]
        graphs.append((g, outs))
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    eager = []
    for _ in range(30):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager.append(calls[0]())
    torch.cuda.synchronize()
    for (_, outs), w in zip(graphs, want):
        assert all(torch.equal(o, w) for o in outs[:5]) and torch.equal(outs[5], prompt)
    assert all(torch.equal(e, want[0]) for e in eager)
    assert tq.kernels.flash_status(dev, 2) == 0 and tq.kernels.prefill_status(dev) == 0


def test_an_owner_first_seen_in_a_capture(tq, dev):
    """The zero fill of a capture runs with the graph only, so what an eager call would use is not made there."""
    # calls that overlap: each has an owner, and the geometry that overlapping calls take
    call = _halves(tq, dev, 7)
    stable = lambda owner: call(workspace_owner=owner, kv_stable=True, q_stable=True)
    want = stable(types.SimpleNamespace(_decode_ws=None))
    owners = [types.SimpleNamespace(_decode_ws=None) for _ in range(3)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [stable(o) for o in owners]
    assert all(o._decode_ws is None for o in owners)
    assert torch.equal(stable(owners[0]), want)
    first = owners[0]._decode_ws
    assert first is not None
    for _ in range(3):
        g.replay()
        assert torch.equal(stable(owners[0]), want) and owners[0]._decode_ws is first
    assert all(torch.equal(o, want) for o in outs)
    assert tq.kernels.workspace_status(first) == 0
