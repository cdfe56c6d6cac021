"""Drafted trees for the tests: random trees, caches in a pool whose every other
slot holds NaN, and the operators' definitions in 64 bits."""

from __future__ import annotations

import random

import torch

from hayate_amd import PagedKVCacheManager

D = 128


def wide_tree(rng: random.Random, n: int) -> list[int]:
    """Parents before children, early nodes with more of them, a few roots."""
    return [-1] + [rng.choice([-1, *range(max(0, i // 3), i), *range(i)]) for i in range(1, n)]


def chain(n: int) -> list[int]:
    return list(range(-1, n - 1))


def line(tree: list[int], i: int) -> list[int]:
    """Node i's ancestors and itself, from the root on."""
    nodes = []
    while i >= 0:
        nodes.append(i)
        i = tree[i]
    return nodes[::-1]


def depth(tree: list[int], i: int) -> int:
    return len(line(tree, i)) - 1


def seen(cached: int, tree: list[int]) -> torch.Tensor:
    """(nodes, cached + nodes): what each node sees."""
    m = torch.zeros(len(tree), cached + len(tree), dtype=torch.bool)
    m[:, :cached] = True
    for i in range(len(tree)):
        m[i, [cached + j for j in line(tree, i)]] = True
    return m


def make_pool(cached, spans, *, q_heads=32, kv_heads=8, page=128, layers=1, seed=0, spare=3,
              device="cuda", slots=None):
    """A pool of NaN in which handle b holds cached[b] tokens of N(0, 1) on pages in drawn
    order, with room for spans[b] more."""
    rng = random.Random(seed)
    need = [-(-(c + n) // page) for c, n in zip(cached, spans)]
    total = sum(need) + spare
    m = PagedKVCacheManager(layers, kv_heads, D, total * page, page, slots or len(cached) + 2,
                            torch.bfloat16, device, num_q_heads=q_heads)
    m.k_cache.fill_(float("nan"))
    m.v_cache.fill_(float("nan"))
    order = list(range(total))
    rng.shuffle(order)
    g = torch.Generator(device=device).manual_seed(seed)
    handles, at = [], 0
    for c, n in zip(cached, need):
        h = m.allocate()
        m.claim_pages(h, order[at : at + n])
        at += n
        h.length = c
        rows = physical(m, h, c)
        for pool in (m.k_cache, m.v_cache):
            pool[:, :, :, rows] = torch.randn((layers, 1, kv_heads, c, D), generator=g,
                                              device=device).to(torch.bfloat16)
        handles.append(h)
    return m, handles


def physical(m, h, length: int) -> torch.Tensor:
    t = torch.arange(length, device=m.device)
    pages = torch.tensor(h.pages or [0], device=m.device)
    return pages[t // m.page_size] * m.page_size + t % m.page_size


def attention64(q, k, v, mask, scale=None):
    """q (n, Hq, D), k and v (Hkv, keys, D), mask (n, keys): the attention in 64 bits, and
    sum_j p_j |v_j| (what a relative error of the probabilities can move). Masked keys
    and values do not enter, whatever they hold."""
    q, k, v, mask = q.double().cpu(), k.double().cpu(), v.double().cpu(), mask.cpu()
    n, hq, _ = q.shape
    group = hq // k.shape[0]
    scale = D**-0.5 if scale is None else scale
    out, size = torch.empty_like(q), torch.empty_like(q)
    for i in range(n):
        keys = mask[i].nonzero()[:, 0]
        for h in range(k.shape[0]):
            rows = slice(h * group, (h + 1) * group)
            p = torch.softmax(q[i, rows] @ k[h, keys].T * scale, -1)
            out[i, rows] = p @ v[h, keys]
            size[i, rows] = p @ v[h, keys].abs()
    return out, size


# The probabilities are rounded to bf16 (half a step: 2^-8 of each) before they meet
# V, and the result once (2^-8 of it). Scores, sums and products are fp32: a score is off by at
# most 128 * 2^-24 of the sum of its 128 products' sizes, which stays under 200 for N(0, 1)
# rows; at scale 128^-0.5 that is 1.4e-4 of a probability, and the sums over the keys (at most
# 4,096 here, 2^-24 a step, 2.5e-4) bring it below 2^-11 in all.
P_STEP = 2.0**-8 + 2.0**-11


def assert_attention(out, ref, size, what=""):
    off = (out.double().cpu() - ref).abs()
    allowed = P_STEP * size + 2.0**-8 * ref.abs() * (1 + P_STEP) + 2.0**-8 * P_STEP * size
    assert torch.isfinite(out).all(), what
    worst = (off - allowed).max().item()
    assert worst <= 0, (what, worst, off.max().item())
