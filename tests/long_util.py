"""Helpers of the tests for windowed and weighed attention: requests over shuffled pages, and
the same attention in 64 bits from its definition."""

from __future__ import annotations

import math

import torch

from hayate_amd import PagedKVCacheManager

D = 128
DEV = "cuda"


def normal(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(torch.bfloat16)


class Requests:
    """A pool of N(0, 1) whose requests hold `cached` tokens on pages in shuffled order, with
    room for `fresh` more. The pool's first `skip` pages are neither used nor written."""

    def __init__(self, cached, fresh, hq=32, hkv=8, page=128, seed=0, layers=1, spare=3, skip=0):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.cached, self.fresh, self.hq, self.hkv = list(cached), list(fresh), hq, hkv
        need = [-(-(c + n) // page) for c, n in zip(cached, fresh)]
        pages = skip + sum(need) + spare
        self.m = PagedKVCacheManager(layers, hkv, D, pages * page, page, len(need) + 2,
                                     torch.bfloat16, DEV, num_q_heads=hq)
        for pool in (self.m.k_cache, self.m.v_cache):
            used = pool[..., skip * page :, :]
            used.copy_(normal(self.g, *used.shape))
        order = (skip + torch.randperm(pages - skip, generator=torch.Generator().manual_seed(
            seed + 1))).tolist()
        self.handles = []
        for c, n in zip(self.cached, need):
            h = self.m.allocate()
            self.m.claim_pages(h, order[:n])
            order = order[n:]
            h.length = c
            self.handles.append(h)
        self.q = normal(self.g, sum(self.fresh), hq, D)

    def rows(self, b):
        """Pool rows of request b's slots, its new tokens' included."""
        page = self.m.page_size
        t = torch.arange(self.cached[b] + self.fresh[b], device=DEV)
        return torch.tensor(self.handles[b].pages, device=DEV)[t // page] * page + t % page

    def expected(self, window=None, sinks=0, q=None, scale=None, layer=0):
        """(out, bound on |out| errors, weights per request) in 64 bits. The kernels round the
        probabilities to bf16 for the second product and the output to bf16, half a step (2^-8
        of the value) each; 1e-4 of the absolute sum covers the fp32 scores and sums: 128
        products of N(0, 1) values, 2^-24 * 128 * sum |q k| * scale = 6e-5 at most."""
        q = self.q if q is None else q
        scale = 1 / math.sqrt(D) if scale is None else scale
        k, v = self.m.k_cache[layer, 0], self.m.v_cache[layer, 0]
        out = torch.empty(sum(self.fresh), self.hq, D, dtype=torch.float64, device=DEV)
        bound, weights, at = torch.empty_like(out), [], 0
        for b, (c, n) in enumerate(zip(self.cached, self.fresh)):
            where = self.rows(b)
            i = torch.arange(c, c + n, device=DEV)[:, None]
            j = torch.arange(c + n, device=DEV)[None]
            hidden = j > i
            if window is not None:
                hidden = hidden | ((i - j >= window) & (j >= sinks))
            total = torch.zeros(c + n, dtype=torch.float64, device=DEV)
            for h in range(self.hq):
                keys = k[h // (self.hq // self.hkv), where].double()
                values = v[h // (self.hq // self.hkv), where].double()
                score = (q[at : at + n, h].double() @ keys.T * scale).masked_fill(hidden, -math.inf)
                p = torch.softmax(score, 1)
                # keys that no row sees have no part in it, whatever they hold
                p, values = p[:, ~hidden.all(0)], values[~hidden.all(0)]
                o, size = p @ values, p @ values.abs()
                out[at : at + n, h] = o
                bound[at : at + n, h] = (size + o.abs()) * 2**-8 + 1e-4 * size
                total[~hidden.all(0)] += p.sum(0)
            weights.append(total)
            at += n
        return out, bound, weights


def assert_close(out, expected, bound, what=""):
    off = (out.double() - expected).abs() / bound
    print(f"  {what} worst error / bound {float(off.max()):.3f}", flush=True)
    assert bool((off <= 1).all()), (what, float(off.max()))
