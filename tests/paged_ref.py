"""64-bit reference of the paged operators, and pools to run them on (test infrastructure).

`Pool` holds random pages of one half (K or V); `decode_ref` evaluates the definition in float64 and returns, beside
the result, an error bound for a kernel that keeps sums and softmax statistics in 32 bits:

  scores   a dot product of dim terms in 32 bits is off by at most (dim + 8) 2^-24 sum|q k| (any order), the scaling,
           the subtraction of the maximum and the exponential by 4 more roundings of |s| and 2^-22 of the weight
  weights  exp turns an absolute score error d into a relative one of d; numerator and denominator: 2 d
  sums     n terms in 32 bits: n 2^-24 relative to the sum of magnitudes at most; splitting only shortens the chains
  rounding 16-bit weights (tensor cores): half a step, eps / 2, relative, of each term; scaled 16-bit codebooks: the
           searched factor leaves less than 2^-15 per centroid
  output   the accumulator lives in the rotated domain: out = butterfly(acc) / dim, so an error of acc_j reaches every
           element with weight 1 / dim: mean_j |error_j|;  plus half a step of the output type
"""
import math

import numpy as np
import torch


def hadamard(dim):
    h = np.ones((1, 1))
    while h.shape[0] < dim:
        h = np.block([[h, h], [h, -h]])
    return torch.from_numpy(h)


class Pool:
    """Random pages: `packed` (pages, heads, page, words), `norms`, sign vector and codebook; or dense rows."""

    def __init__(self, tq, seed, pages, heads, page, dim, bits, dev, dtype=None, head_major=False):
        g = torch.Generator().manual_seed(seed)
        self.bits, self.dim, self.page = bits, dim, page
        lead = (heads, pages) if head_major else (pages, heads)       # head_major: another order of the strides
        fix = (lambda t: t.to(dev).transpose(0, 1)) if head_major else (lambda t: t.to(dev))
        if bits == 0:
            self.data = fix(torch.randn((*lead, page, dim), generator=g).to(dtype))
            self.desc = dict(format="dense", data=self.data)
            return
        self.quant = tq.PolarQuantizer(dim, bits, seed=seed, device=dev)
        codes = torch.randint(0, 1 << bits, (*lead, page, dim), generator=g, dtype=torch.uint8)
        self.packed = fix(tq.pack_indices(codes, bits))
        self.norms = fix(torch.exp(torch.randn((*lead, page), generator=g) * 0.4) * math.sqrt(dim))
        self.desc = dict(format="polar", packed=self.packed, norms=self.norms, bits=bits, signs=self.quant.signs,
                         centroids=self.quant.centroids, boundaries=self.quant.boundaries)

    def rotated(self, tq, pages, n):
        """float64 rows norm * centroid / dim (before signs * butterfly) of the first n positions of these pages:
        (heads, n, dim) on the CPU."""
        packed = self.packed.cpu()[pages]
        codes = tq.unpack_indices(packed, self.bits, self.dim).long()
        rows = self.quant.centroids.cpu().double()[codes] * self.norms.cpu()[pages].double()[..., None] / self.dim
        return rows.transpose(0, 1).flatten(1, 2)[:, :n]

    def rows(self, tq, pages, n):
        """The values the pages stand for, float64."""
        if self.bits == 0:
            return self.data.cpu()[pages].double().transpose(0, 1).flatten(1, 2)[:, :n]
        return self.rotated(tq, pages, n) @ hadamard(self.dim) * self.quant.signs.cpu().double()


def make_table(lens, page, seed, spare=2, window=0, sinks=0, dev="cuda", width=None):
    """Shuffled pages; -1 behind a sequence and where its window has passed.  Returns (table, pages of the pool)."""
    need = [[i for i in range(-(-n // page)) if not (window and i * page >= sinks and (i + 1) * page <= n - window)]
            for n in lens]
    total = sum(map(len, need)) + spare
    order = iter(np.random.default_rng(seed).permutation(total).tolist())
    width = width or max(1, max(-(-n // page) for n in lens))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, pages in enumerate(need):
        for i in pages:
            table[b, i] = next(order)
    return table.to(dev), total


def visible(n, window, sinks):
    return [p for p in range(n) if not window or p >= n - window or p < sinks]


def decode_ref(tq, q, k, v, table, lens, scale, window=0, sinks=0, weight_eps=0.0, out_dtype=torch.float32):
    """(result, bound), float64 CPU (B, n_q, dim)."""
    B, n_q, dim = q.shape
    H = hadamard(dim)
    out = torch.zeros((B, n_q, dim), dtype=torch.float64)
    tol = torch.zeros_like(out)
    q = q.detach().cpu().double()
    book = 2.0 ** -15 if weight_eps else 0.0
    for b, n in enumerate(lens):
        at = visible(n, window, sinks)
        if not at:
            continue
        pages = table[b].cpu().long()[:-(-n // v.page)].clamp(min=0)
        vr = v.rotated(tq, pages, n)[:, at]
        kr = k.rows(tq, pages, n)[:, at] if k.bits == 0 else k.rotated(tq, pages, n)[:, at]
        rep = n_q // vr.shape[0]
        for h in range(n_q):
            x = q[b, h] if k.bits == 0 else (q[b, h] * k.quant.signs.cpu().double()) @ H
            kk, vv = kr[h // rep], vr[h // rep]
            s = kk @ x * scale
            mag = kk.abs() @ x.abs() * abs(scale)
            # 16-bit operands: the query as a pair of 16-bit values (2^-17 at worst), codebooks 2^-15
            d = float(((dim + 8) * 2.0 ** -24 * mag + 4 * 2.0 ** -24 * s.abs()).max()) + 2.0 ** -22
            if weight_eps:
                d += float(mag.max()) * (2.0 ** -17 + book)
            p = torch.softmax(s, 0)
            out[b, h] = (p @ vv) @ H * v.quant.signs.cpu().double()
            rel = 2 * d + len(at) * 2.0 ** -24 + weight_eps + book + (dim + 8) * 2.0 ** -24
            reach = float((p @ vv.abs()).sum())            # sum_j |acc_j|, each with weight 1 (vv carries 1 / dim)
            tol[b, h] = rel * reach + torch.finfo(out_dtype).eps / 2 * (out[b, h].abs() + rel * reach) + 1e-30
    return out, tol


def check(got, ref, tol, what=""):
    got = got.detach().cpu().double()
    worst = float(((got - ref).abs() / tol.clamp(min=1e-300)).max())
    assert torch.isfinite(got).all() and worst <= 1.0, f"{what}: error is {worst:.3f} of its bound"
