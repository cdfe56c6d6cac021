"""Operators for drafted tokens and for moving a cache's pages, as cases that can
be timed and whose results can be compared.

Four operators, on a paged K/V pool of (layers, 1, kv heads, tokens, 128) bf16:

  attend  attention for trees of drafted tokens over their requests' caches:
          ``PagedTreeBatch.attend_layer``
  append  what comes before it: q/k RMSNorm and rope of the drafted tokens at
          their depths, K and V written to their slots:
          ``PagedTreeBatch.norm_rope_write_layer``
  move    tokens of a request moved forward in its cache, in every layer, after
          a verified draft or an eviction: ``PagedKVCacheManager.move_tokens``
  copy    pages copied to others in every layer, when requests are forked:
          ``PagedKVCacheManager.copy_pages``

A drafted token i of a request with c cached tokens sits in slot c + i, is
rotated at position c + depth(i), and attends to the c cached tokens, its
ancestors and itself. With `own` the framework's calls run, else their plain
forms in torch. Lengths, trees and paths belong to the case (``lens`` seeds them),
page placement and values to the seed.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 128  # head size
EPS = 1e-6
THETA = 1_000_000
POSITIONS = 40_960
LAYERS = 36
DEV = "cuda"


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one user, a small tree on a short chat: the smallest call, latency counts
        _attend("attend 1x8 on 500", batch=1, nodes=8, lo=500, hi=500),
        # a served batch with short linear drafts (a prompt lookup's) and spread contexts
        _attend("attend 32 chains of 5", batch=32, nodes=5, lo=256, hi=4096, tree="chain"),
        # the default batch limit with ordinary trees of odd sizes
        _attend("attend 20x26 ragged", batch=20, nodes=26, nodes_lo=11, lo=200, hi=4000),
        # long documents under large trees: the largest reads and products
        _attend("attend 8x64 on 32k", batch=8, nodes=64, lo=30_000, hi=32_700),
        # very wide trees, more rows than one tile takes
        _attend("attend 4x200 on 3k", batch=4, nodes=200, nodes_lo=150, lo=2500, hi=3500),
        # the norm, rope and append before the smallest and before a full batch
        _attend("append 1x8", kind="append", batch=1, nodes=8, lo=500, hi=500),
        _attend("append 32x60", kind="append", batch=32, nodes=60, nodes_lo=30, lo=256, hi=4096),
        # one user's accepted path, all layers
        _move("move 1 path of 5", batch=1, nodes=26, path=5, lo=700, hi=700, lens=24),
        # the accepted paths of a served batch
        _move("move 32 paths", batch=32, nodes=60, path=9, lo=256, hi=2000),
        # a long conversation that drops its middle: first tokens and recent ones stay
        {"name": "move evict 5999", "kind": "move", "layers": LAYERS, "page": 128, "kv_heads": 8,
         "evict": True, "batch": 1, "first": 16, "recent": 5999, "dropped": 6100, "lens": 3},
        # samples of one prompt: each gets its own copy of the partly filled last page
        _copy("copy 15 tails", pairs=15, tokens=77, last=77),
        # a fork that shares nothing, of a long prompt
        _copy("copy 32 pages", pairs=32, tokens=128, last=50),
    ]


def _attend(name, kind="attend", batch=1, nodes=8, nodes_lo=None, lo=1, hi=1, tree="wide",
            page=128, q_heads=32, kv_heads=8, lens=7):
    case = {"kind": kind, "batch": batch, "nodes": nodes,
            "nodes_lo": nodes if nodes_lo is None else nodes_lo, "ctx_lo": lo, "ctx_hi": hi,
            "tree": tree, "page": page, "q_heads": q_heads, "kv_heads": kv_heads, "lens": lens}
    return dict(case, name=name) if name else case


def _move(name, batch, nodes, path, lo, hi, layers=LAYERS, page=128, kv_heads=8, lens=7):
    case = {"kind": "move", "evict": False, "layers": layers, "page": page, "kv_heads": kv_heads,
            "batch": batch, "nodes": nodes, "path": path, "ctx_lo": lo, "ctx_hi": hi, "lens": lens}
    return dict(case, name=name) if name else case


def _copy(name, pairs, tokens, last, layers=LAYERS, page=128, kv_heads=8):
    """`pairs` pages of `tokens` filled tokens, the last one of `last`."""
    case = {"kind": "copy", "layers": layers, "page": page, "kv_heads": kv_heads, "pairs": pairs,
            "tokens": tokens, "last": last}
    return dict(case, name=name) if name else case


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "move", "move", "copy"])
    page = rng.choice([128, 128, 256])
    if kind in ("attend", "append"):
        q_heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 8), (16, 8), (64, 8), (32, 2),
                                        (8, 8)])
        nodes = _log(rng, 1, 256)
        batch = _log(rng, 1, max(1, min(48, 1500 // nodes)))
        # keys read in all, and products of queries with keys, below the largest listed case's
        most = min(32_000, 200_000 // batch, 400_000_000 // (batch * nodes * q_heads))
        hi = _log(rng, 1, max(2, most))
        return _attend(None, kind=kind, batch=batch, nodes=nodes,
                       nodes_lo=max(1, int(nodes * rng.choice([1.0, 0.6, 0.1]))),
                       lo=int(hi * rng.choice([1.0, 0.4, 0.05])), hi=hi,
                       tree=rng.choice(["wide", "wide", "chain"]), page=page,
                       q_heads=q_heads, kv_heads=kv_heads, lens=rng.randrange(1 << 20))
    layers = rng.choice([LAYERS, LAYERS, _log(rng, 1, LAYERS)])
    if kind == "copy":
        pairs = _log(rng, 1, 4096 // page)
        return _copy(None, pairs=pairs, tokens=rng.choice([page, rng.randint(1, page)]),
                     last=rng.randint(1, page), layers=layers, page=page,
                     kv_heads=rng.choice([8, 8, 2]))
    if rng.random() < 0.4:
        recent = _log(rng, 1, 5900)
        return {"kind": "move", "layers": layers, "page": page, "kv_heads": 8, "evict": True,
                "batch": 1, "first": rng.randint(0, 40), "recent": recent,
                "dropped": recent + _log(rng, 1, 6000 - recent), "lens": rng.randrange(1 << 20)}
    nodes = _log(rng, 2, 256)
    return _move(None, batch=_log(rng, 1, 40), nodes=nodes,
                 path=rng.randint(1, max(1, min(12, nodes // 2))), lo=1, hi=_log(rng, 1, 1500),
                 layers=layers, page=page, lens=rng.randrange(1 << 20))


def _lengths(case):
    """(cached tokens, drafted tokens) of every request."""
    r = random.Random(case["lens"])
    cached = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    return cached, [r.randint(case["nodes_lo"], case["nodes"]) for _ in cached]


def _parents(case):
    """The tree of every request: each node's parent among the nodes before it,
    -1 for a child of the cached context."""
    r = random.Random(case["lens"] + 1)
    trees = []
    for n in _lengths(case)[1]:
        if case["tree"] == "chain":
            trees.append(list(range(-1, n - 1)))
        else:  # nodes in the order of their likelihood: early ones get more children
            trees.append([-1] + [max(-1, int(i * r.random() ** 2) - (r.random() < 0.15))
                                 for i in range(1, n)])
    return trees


def _moves(case):
    """Per request: the first position that is filled, and the positions that its
    tokens come from, ascending. A pass is repeated on the same cache, so no
    filled position is read by a later token."""
    r = random.Random(case["lens"])
    if case["evict"]:
        first, gap = case["first"], case["dropped"]
        return [first], [[first + gap + i for i in range(case["recent"])]], [
            first + gap + case["recent"]]
    starts, sources, sizes = [], [], []
    for _ in range(case["batch"]):
        c, m = r.randint(case["ctx_lo"], case["ctx_hi"]), r.randint(1, case["path"])
        stay = r.randint(0, m)  # the path begins with the likeliest nodes
        starts.append(c)
        sources.append([c + i for i in range(stay)]
                       + [c + i for i in sorted(r.sample(range(m, case["nodes"]), m - stay))])
        sizes.append(c + case["nodes"])
    return starts, sources, sizes


# --------------------------------------------------------------- the inputs
class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.host = random.Random(seed)

    def normal(self, *shape, std=1.0, mean=0.0):
        x = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
        flat, step = x.view(-1), 1 << 27
        for i in range(0, flat.numel(), step):
            n = min(step, flat.numel() - i)
            flat[i : i + n] = torch.randn(n, generator=self.g, device=DEV) * std + mean
        return x


def _pools(case, gen, sizes):
    """Pools of N(0, 1) and the pages of every request, in drawn order."""
    page = case["page"]
    need = [-(-n // page) for n in sizes]
    order = list(range(sum(need) + 3))
    gen.host.shuffle(order)
    lists, at = [], 0
    for n in need:
        lists.append(order[at : at + n])
        at += n
    shape = (case.get("layers", 1), 1, case["kv_heads"], len(order) * page, D)
    return lists, gen.normal(*shape), gen.normal(*shape)


def _inputs(case, seed):
    """Everything a pass reads, as plain tensors and lists."""
    gen = _Gen(seed)
    if case["kind"] == "copy":
        n = case["pairs"]
        lists, k, v = _pools(case, gen, [n * case["page"]] * 2)
        return {"lists": lists, "cached": [n * case["page"]] * 2, "k_pool": k, "v_pool": v,
                "src": lists[0], "dst": lists[1],
                "tokens": [case["tokens"]] * (n - 1) + [case["last"]]}
    if case["kind"] == "move":
        starts, sources, sizes = _moves(case)
        lists, k, v = _pools(case, gen, sizes)
        return {"lists": lists, "cached": sizes, "k_pool": k, "v_pool": v, "starts": starts,
                "sources": [np.array(s, dtype=np.int64) for s in sources]}
    cached, drafted = _lengths(case)
    lists, k, v = _pools(case, gen, [c + n for c, n in zip(cached, drafted)])
    heads, total = case["q_heads"] + 2 * case["kv_heads"], sum(drafted)
    got = {"lists": lists, "cached": cached, "drafted": drafted, "parents": _parents(case),
           "k_pool": k, "v_pool": v, "qkv": gen.normal(total, heads, D)}
    if case["kind"] == "append":
        freq = 1.0 / THETA ** (torch.arange(0, D, 2, dtype=torch.float32, device=DEV) / D)
        angle = torch.arange(POSITIONS, dtype=torch.float32, device=DEV)[:, None] * freq[None]
        angle = torch.cat([angle, angle], dim=1)
        got.update(cos=torch.cos(angle), sin=torch.sin(angle),
                   q_norm=gen.normal(D, std=0.1, mean=1.0), k_norm=gen.normal(D, std=0.1, mean=1.0))
    return got


def _table(lists):
    """(requests, most pages) page ids, 0 past a request's own."""
    table = torch.zeros(len(lists), max(1, max(len(p) for p in lists)), dtype=torch.long)
    for row, pages in enumerate(lists):
        table[row, : len(pages)] = torch.tensor(pages, dtype=torch.long)
    return table.to(DEV)


def _ancestry(parents):
    """Per request a (nodes, nodes) table of which node each one sees, and the
    depth of each node."""
    sees, depths = [], []
    for tree in parents:
        m, depth = np.zeros((len(tree), len(tree)), dtype=bool), []
        for i, p in enumerate(tree):
            if p >= 0:
                m[i] = m[p]
            m[i, i] = True
            depth.append(depth[p] + 1 if p >= 0 else 0)
        sees.append(m)
        depths.append(depth)
    return sees, depths


def prepare(case, seed):
    inp = _inputs(case, seed)
    state = {"case": case, **inp}
    kind = case["kind"]
    if kind in ("attend", "append"):
        hq, hkv, qkv = case["q_heads"], case["kv_heads"], inp["qkv"]
        # as a program has them: views of one projection, and for the attention
        # the rotated q that the append returned, contiguous
        state.update(q=qkv[:, :hq].contiguous() if kind == "attend" else qkv[:, :hq],
                     k=qkv[:, hq : hq + hkv], v=qkv[:, hq + hkv :])
    if own:
        return _own_state(state)
    state["table"] = _table(inp["lists"])
    if kind in ("attend", "append"):
        sees, depths = _ancestry(inp["parents"])
        most = max(inp["drafted"])
        mask = np.zeros((len(sees), most, most), dtype=bool)
        for b, m in enumerate(sees):
            mask[b, : len(m), : len(m)] = m
        state.update(
            mask=torch.from_numpy(mask).to(DEV),
            cached_t=torch.tensor(inp["cached"], device=DEV),
            drafted_t=torch.tensor(inp["drafted"], device=DEV),
            depth=torch.tensor([d for tree in depths for d in tree], device=DEV))
    return state


def _own_state(state):
    """The pool with its requests in place, and the tick's batch. The manager's
    tensors become the inputs' own (a pool holds what earlier ticks wrote)."""
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "hayate-exp_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from hayate_amd import PagedKVCacheManager

    case, k = state["case"], state.pop("k_pool")
    m = PagedKVCacheManager(k.shape[0], case["kv_heads"], D, k.shape[3], case["page"],
                            len(state["lists"]), torch.bfloat16, DEV,
                            num_q_heads=case.get("q_heads"))
    m.k_cache.copy_(k)
    m.v_cache.copy_(state.pop("v_pool"))
    handles = []
    for c, pages in zip(state["cached"], state["lists"]):
        h = m.allocate()
        m.claim_pages(h, pages)
        h.length = c
        handles.append(h)
    state.update(m=m, handles=handles)
    if case["kind"] in ("attend", "append"):
        state["batch"] = m.begin_tree(handles, state["parents"])
    return state


# ---------------------------------------------------------------- the passes
def run(state):
    with torch.inference_mode():
        return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    kind = s["case"]["kind"]
    if kind == "attend":
        return {"out": s["batch"].attend_layer(s["q"], 0)}
    m = s["m"]
    if kind == "append":
        q = s["batch"].norm_rope_write_layer(0, s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"],
                                             EPS, s["cos"], s["sin"])
        return {"q": q, "k_pool": m.k_cache, "v_pool": m.v_cache}
    if kind == "move":
        m.move_tokens(s["handles"], s["sources"], s["starts"])
    else:
        m.copy_pages(s["src"], s["dst"], s["tokens"])
    return {"k_pool": m.k_cache, "v_pool": m.v_cache}


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "attend":
        return {"out": _plain_attend(s)}
    if kind == "append":
        q = _plain_append(s)
        return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    src, dst = _plain_rows(s)
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, :, :, dst] = pool[:, :, :, src]
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_attend(s):
    case = s["case"]
    page, hq, hkv = case["page"], case["q_heads"], case["kv_heads"]
    cached, drafted, mask = s["cached_t"], s["drafted_t"], s["mask"]
    batch, most = mask.shape[:2]
    keys = torch.arange(s["table"].shape[1] * page, device=DEV)
    where = s["table"][:, keys // page] * page + keys % page
    k = s["k_pool"][0, 0][:, where].transpose(0, 1).float()  # (batch, kv heads, keys, D)
    v = s["v_pool"][0, 0][:, where].transpose(0, 1).float()
    # rows of a request beyond its nodes repeat a row of the batch and are dropped
    node = torch.arange(most, device=DEV)
    live = node[None] < drafted[:, None]
    row = (torch.cumsum(drafted, 0) - drafted)[:, None] + node[None]
    q = s["q"][row.clamp(max=s["q"].shape[0] - 1)].float()
    q = q.view(batch, most, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, D)
    score = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D)
    slot = keys[None] - cached[:, None]  # (batch, keys): the drafted token in it, if >= 0
    at = slot.clamp(0, most - 1)[:, None].expand(batch, most, -1)
    seen = (slot < 0)[:, None] | ((slot < drafted[:, None])[:, None] & mask.gather(2, at))
    score = score.view(batch, hkv, hq // hkv, most, -1)
    score.masked_fill_(~(seen | ~live[:, :, None])[:, None, None], -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True))
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(batch, hkv, -1, score.shape[-1]), v).view(*total.shape[:4], D)
    out = (out / total).permute(0, 3, 1, 2, 4).reshape(batch, most, hq, D)
    request, node = _plain_packed(s)
    return out[request, node].to(torch.bfloat16)


def _plain_packed(s):
    """Request and node of every packed row."""
    n = s["q"].shape[0]
    request = torch.repeat_interleave(s["drafted_t"], output_size=n)
    first = torch.cumsum(s["drafted_t"], 0) - s["drafted_t"]
    return request, torch.arange(n, device=DEV) - first[request]


def _plain_append(s):
    page, (request, node) = s["case"]["page"], _plain_packed(s)
    slot = s["cached_t"][request] + node
    position = s["cached_t"][request] + s["depth"]
    cos, sin = s["cos"][position][:, None], s["sin"][position][:, None]
    q = _plain_rotate(s["q"].float(), s["q_norm"].float(), cos, sin)
    k = _plain_rotate(s["k"].float(), s["k_norm"].float(), cos, sin)
    where = s["table"][request, slot // page] * page + slot % page
    s["k_pool"][0, 0][:, where] = k.transpose(0, 1).to(torch.bfloat16)
    s["v_pool"][0, 0][:, where] = s["v"].transpose(0, 1)
    return q.to(torch.bfloat16)


def _plain_rotate(x, weight, cos, sin):
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    return x * cos + torch.cat([-x[..., D // 2 :], x[..., : D // 2]], dim=-1) * sin


def _plain_rows(s):
    """Physical tokens that are read and written."""
    page = s["case"]["page"]
    if s["case"]["kind"] == "copy":
        src, dst, tokens = (np.array(s[x]) for x in ("src", "dst", "tokens"))
        offset = np.arange(page)[None]
        filled = offset < tokens[:, None]
        return tuple(torch.from_numpy((x[:, None] * page + offset)[filled]).to(DEV)
                     for x in (src, dst))
    sizes = np.array([len(x) for x in s["sources"]])
    request = np.repeat(np.arange(len(sizes)), sizes)
    to = np.arange(sizes.sum()) - (np.cumsum(sizes) - sizes - s["starts"])[request]
    request, src, dst = (torch.from_numpy(x).to(DEV)
                         for x in (request, np.concatenate(s["sources"]), to))
    return tuple(s["table"][request, x // page] * page + x % page for x in (src, dst))


# ------------------------------------------------------------ bytes and flops
def work(case):
    """Each K and V row read once and each row in or out moved once."""
    row = 2 * D
    if case["kind"] in ("attend", "append"):
        cached, drafted = _lengths(case)
        hq, hkv, n = case["q_heads"], case["kv_heads"], sum(drafted)
        if case["kind"] == "append":
            # rows in and out, and a cos and a sin row for each token
            return {"bytes": n * ((2 * hq + 4 * hkv) * row + 8 * D), "flops": 0}
        pairs = sum(c * t for c, t in zip(cached, drafted))
        pairs += sum(int(m.sum()) for m in _ancestry(_parents(case))[0])
        kv = sum(cached) + n
        return {"bytes": kv * 2 * hkv * row + 2 * n * hq * row, "flops": 4 * hq * D * pairs}
    if case["kind"] == "copy":
        tokens = (case["pairs"] - 1) * case["tokens"] + case["last"]
    else:
        starts, sources, _ = _moves(case)
        tokens = sum(int(x != c + i) for c, xs in zip(starts, sources) for i, x in enumerate(xs))
    return {"bytes": max(1, tokens) * 4 * case["layers"] * case["kv_heads"] * row, "flops": 0}


# ------------------------------------------------------------ 64-bit results
def exact(case, seed):
    inp = _inputs(case, seed)
    page, kind = case["page"], case["kind"]
    k, v = inp.pop("k_pool").double(), inp.pop("v_pool").double()
    pools = {"k_pool": k, "v_pool": v}
    if kind == "copy":
        for a, b, n in zip(inp["src"], inp["dst"], inp["tokens"]):
            for pool in (k, v):
                pool[:, :, :, b * page : b * page + n] = pool[:, :, :, a * page : a * page + n]
        return pools
    if kind == "move":
        for pages, start, sources in zip(inp["lists"], inp["starts"], inp["sources"]):
            where = [p * page + o for p in pages for o in range(page)]
            src = torch.tensor([where[i] for i in sources], dtype=torch.long, device=DEV)
            dst = torch.tensor(where[start : start + len(sources)], dtype=torch.long, device=DEV)
            for pool in (k, v):
                pool.index_copy_(3, dst, pool.index_select(3, src))
        return pools
    hq, hkv = case["q_heads"], case["kv_heads"]
    group, qkv, outs, at = hq // hkv, inp["qkv"].double(), [], 0
    for pages, c, tree in zip(inp["lists"], inp["cached"], inp["parents"]):
        n = len(tree)
        rows = qkv[at : at + n]
        at += n
        lines = []  # of every node: itself and its ancestors
        for i, p in enumerate(tree):
            lines.append(lines[p] + [i] if p >= 0 else [i])
        where = torch.tensor(pages, device=DEV).repeat_interleave(page) * page
        where = (where + torch.arange(page, device=DEV).repeat(len(pages)))[: c + n]
        if kind == "append":
            pos = torch.tensor([c + len(x) - 1 for x in lines], device=DEV)
            turned = []
            for part, w in ((rows[:, :hq], inp["q_norm"]), (rows[:, hq : hq + hkv], inp["k_norm"])):
                x = part / torch.sqrt((part * part).sum(-1, keepdim=True) / D + EPS) * w.double()
                a, b = x[..., : D // 2], x[..., D // 2 :]
                co, si = (inp[t][pos, : D // 2].double()[:, None] for t in ("cos", "sin"))
                turned.append(torch.cat([a * co - b * si, b * co + a * si], -1))
            outs.append(turned[0])
            k[0, 0][:, where[c:]] = turned[1].transpose(0, 1)
            v[0, 0][:, where[c:]] = rows[:, hq + hkv :].transpose(0, 1)
            continue
        hidden = torch.ones(n, n, dtype=torch.bool)
        for i, line in enumerate(lines):
            hidden[i, line] = False
        hidden = hidden.to(DEV)
        out = torch.empty(n, hq, D, dtype=torch.float64, device=DEV)
        for h in range(hq):
            keys, values = k[0, 0, h // group, where], v[0, 0, h // group, where]
            score = rows[:, h] @ keys.T * D**-0.5
            score[:, c:] = score[:, c:].masked_fill(hidden, -math.inf)
            out[:, h] = torch.softmax(score, -1) @ values
        outs.append(out)
    return {"q": torch.cat(outs), **pools} if kind == "append" else {"out": torch.cat(outs)}
