"""Caches made and used under torch.inference_mode, whose tensors have no version counter."""
import math

import pytest
import torch


def test_caches_are_made_in_inference_mode(tq):
    with torch.inference_mode():
        cache, = tq.make_paged_caches(1, 4, 2, device=torch.device("cpu"))
        book = cache.v["centroids"]
        assert list(tq._lib.host_floats(book)) == book.tolist()
        assert list(tq._lib.host_floats(cache.v["signs"])) == cache.v["signs"].tolist()
    book.mul_(2.0)                                          # seen: these tensors have a version
    assert list(tq._lib.host_floats(book)) == book.tolist()


def test_a_codebook_without_a_version_is_read_every_time(tq):
    with torch.inference_mode():
        t = torch.tensor([1.0, 2.0])
        assert list(tq._lib.host_floats(t)) == [1.0, 2.0]
        t.add_(1.0)
        assert list(tq._lib.host_floats(t)) == [2.0, 3.0]
        tq._lib.register_host_values(t, [2.0, 3.0])
        t.add_(1.0)
        assert list(tq._lib.host_floats(t)) == [3.0, 4.0]


@pytest.mark.gpu
def test_paged_steps_in_inference_mode(tq, dev):
    """The same bits as outside; a codebook of the caller's changed in place is the changed one."""
    def run():
        cache, = tq.make_paged_caches(1, 8, 2, page_size=32)
        seqs = cache.sequences
        ids = [seqs.add()]
        outs = []
        for n in (70, 1):
            g = torch.Generator().manual_seed(n)
            keys, values, q = [torch.randn((1, h, n, 128), generator=g).half().to(dev) for h in (2, 2, 8)]
            seqs.begin(ids, n)
            cache.update_and_fetch(keys, values)
            outs.append(cache.attention(q, 1 / math.sqrt(128)))
        own = dict(cache.v, centroids=cache.v["centroids"].clone())
        call = lambda: tq.paged_decode(q[:, :, 0], k=cache.k, v=own, page_table=seqs.table, seq_lens=seqs.lens, attn_scale=0.1)
        outs.append(call())
        own["centroids"].mul_(2.0)
        outs.append(call())
        return outs

    want = run()
    with torch.inference_mode():
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not torch.equal(want[2], want[3])
    assert tq.paged_status(dev) == 0
