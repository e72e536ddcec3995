"""Decode with more codebooks than one model has: results, and what a call costs once its codebook is known."""
import math
import os
import sys
import time

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as pr  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("paged", [True, False])
def test_many_codebooks(tq, dev, paged):
    """40 value codebooks in turn, one per call: every result is the codebook's own, and a second round of calls does not
    repeat the search for 16-bit factors (0.5 to 3 ms of host time each; a call takes 10 to 50 us)."""
    n, n_kv, n_q, D, books = 64, 1, 4, 128, 40
    scale = 1 / math.sqrt(D)
    v = pr.Pool(tq, 1, 1, n_kv, n, D, 4, dev)
    k = pr.Pool(tq, 2, 1, n_kv, n, D, 0, dev, dtype=torch.float16)
    q = torch.randn((1, n_q, D), generator=torch.Generator().manual_seed(3)).half().to(dev)
    table, lens = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([n], dtype=torch.int32, device=dev)
    base = v.quant.centroids
    descs = []
    for i in range(books):
        cent = base * (1 + i / 64) * (0.9 if paged else 1.1)           # no factor shared with another test
        tq._lib.host_floats(cent)
        descs.append(dict(v.desc, centroids=cent))

    def call(desc):
        if paged:
            return tq.paged_decode(q, k=k.desc, v=desc, page_table=table, seq_lens=lens, attn_scale=scale)
        return tq.flash_decode(q, k=k.desc, v=desc, attn_scale=scale)      # one page is one sequence's rows

    def round_of_calls():
        t = time.perf_counter()
        outs = [call(d) for d in descs]
        took = time.perf_counter() - t
        torch.cuda.synchronize()
        return took, outs

    call(v.desc)
    torch.cuda.synchronize()
    first, outs = round_of_calls()
    second = first
    for _ in range(3):
        took, again = round_of_calls()
        second = min(second, took)
        assert all(torch.equal(a, b) for a, b in zip(outs, again))
    assert second < first / 4, (first, second)
    # 16-bit weights, and centroids that a factor brings within 2^-13 of 16-bit values (relative, each)
    eps = torch.finfo(torch.float16).eps / 2 + 2.0 ** -13
    for i, desc in enumerate(descs):
        book = pr.Pool.__new__(pr.Pool)
        book.__dict__ = dict(v.__dict__)
        book.quant = type("Q", (), dict(centroids=desc["centroids"], signs=v.quant.signs))
        ref, tol = pr.decode_ref(tq, q, k, book, table, [n], scale, 0, 0, eps, outs[i].dtype)
        pr.check(outs[i], ref, tol, f"codebook {i}")
