"""64-bit restatements of the bounded-cache operators (window and sink attention, attention weights,
eviction), written from their definitions, and the paged inputs their tests share.  CPU float64.

Tolerances (elementwise, from the arithmetic; u16 = 2^-8 is half a bf16 step, relative):
* an output row is sum_j p_j v_j / sum_j p_j with p_j rounded to bf16 before the product and the result
  rounded once more: |error| <= u16 |out| + u16 A, A = sum_j softmax_j |v_j|.  What is in 32 bits (scores,
  exponentials, sums) adds at most 2^-12 A: a score of 128 products of size <= 8 in sum of magnitudes carries
  at most 128 x 2^-23 x 8 x log2(e) x 2 < 2^-12 of relative weight.
* an attention weight is one 32-bit exponential of such a score: |error| <= 2^-12 added + 2^-22 |w| (the
  accumulator's own additions, at most a few at half a step 2^-24 each).
"""
import numpy as np
import torch

U16 = 2.0 ** -8
U32 = 2.0 ** -12


def visible(pos, n, window, sinks):
    """[len(pos), n] truth values: the row at position p sees j <= p, and under a window (0 = none) only
    j > p - window or j < sinks."""
    j = torch.arange(n)
    p = torch.as_tensor(pos)[:, None]
    vis = j <= p
    if window:
        vis = vis & ((j > p - window) | (j < sinks))
    return vis


def attend(q, K, V, vis, scale):
    """q [m, G, D], K/V [n, D], vis [m, n] -> out [m, G, D], A [m, G, D], lse [m, G], p [m, G, n] (64 bits);
    a row that sees nothing gives zeros and lse -inf."""
    q, K, V = q.double(), K.double(), V.double()
    x = torch.einsum("mgd,nd->mgn", q, K) * scale
    x = x.masked_fill(~vis[:, None], float("-inf"))
    lse = torch.logsumexp(x, -1)
    p = torch.where(vis[:, None], torch.exp(x - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None]),
                    torch.zeros_like(x))
    V = torch.where(vis.any(0)[:, None], V, torch.zeros_like(V))
    return torch.einsum("mgn,nd->mgd", p, V), torch.einsum("mgn,nd->mgd", p, V.abs()), lse, p


class Paged:
    """A paged cache of sequences `lens` with shuffled pages; layout 0 [nb, 2, page, Hkv, D], 1 [2, nb, page,
    Hkv, D].  Rows past each length (and page 0, the null block) hold NaN."""

    def __init__(self, lens, Hkv, D, page, layout=0, seed=0, extra_pages=1, dtype=torch.bfloat16):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.layout, self.Hkv, self.D = list(lens), page, layout, Hkv, D
        counts = [(n + page - 1) // page for n in lens]
        self.width = max([1] + counts)
        ids = torch.randperm(sum(counts) + extra_pages - 1, generator=g) + 1 if sum(counts) + extra_pages > 1 \
            else torch.zeros(0, dtype=torch.long)
        self.nb = sum(counts) + extra_pages
        self.table = torch.zeros((len(lens), self.width), dtype=torch.int32)
        self.K = [torch.randn((n, Hkv, D), generator=g).to(dtype) for n in lens]
        self.V = [torch.randn((n, Hkv, D), generator=g).to(dtype) for n in lens]
        kv = torch.full((self.nb, 2, page, Hkv, D), float("nan"), dtype=dtype)
        at = 0
        for b, n in enumerate(lens):
            self.table[b, :counts[b]] = ids[at:at + counts[b]].int()
            at += counts[b]
            for r in range(n):
                pg = int(self.table[b, r // page])
                kv[pg, 0, r % page] = self.K[b][r]
                kv[pg, 1, r % page] = self.V[b][r]
        self.kv = kv if layout == 0 else kv.transpose(0, 1).contiguous()
        self.seq = torch.tensor(lens, dtype=torch.int32)

    def rows(self, kv, table, b, n):
        """The first n rows (K, V) [n, Hkv, D] of table row b of a cache tensor."""
        if self.layout == 1:
            kv = kv.transpose(0, 1)
        idx = torch.arange(n)
        pg = table[b, idx // self.page].long()
        return kv[pg, 0, idx % self.page], kv[pg, 1, idx % self.page]


def check_out(got, ref, A, tag=""):
    got, ref = got.double().cpu(), ref.double()
    assert not torch.isnan(got).any(), tag
    bound = U16 * ref.abs() + (U16 + U32) * A + 1e-30
    worst = ((got - ref).abs() / bound).max() if got.numel() else torch.tensor(0.0)
    assert worst <= 1, (tag, float(worst))


def check_weights(got, before, added, tag=""):
    got, ref = got.double().cpu(), before.double() + added
    bound = U32 * added + 2.0 ** -22 * ref.abs()
    bad = (got - ref).abs() > bound
    assert not torch.isnan(got).any() and not bad.any(), (tag, float((got - ref).abs().max()))


def evict_rows(w, n, budget, sinks, recent):
    """Rows kept of n under accumulated weights w[>=n] (numpy float): the first `sinks`, the last `recent`, and
    the heaviest others up to `budget`, ties to the lowest row, NaN below everything; ascending."""
    if n <= budget:
        return np.arange(n)
    key = np.where(np.isnan(w[:n]), -np.inf, w[:n].astype(np.float64))
    mid = np.arange(sinks, n - recent)
    order = mid[np.lexsort((mid, -key[mid]))][:budget - sinks - recent]
    return np.sort(np.concatenate([np.arange(sinks), order, np.arange(n - recent, n)])).astype(np.int64)
