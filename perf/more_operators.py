"""Operators for long generations over a paged cache, as cases that can be timed and
whose results can be compared.

Four operators; K and V in pools of (layers, 1, kv heads, tokens, 128) bf16:

  window  attention in which a token sees the last `window` tokens, itself among
          them, and the first `sinks` ones: ``attend_layer`` of a batch begun with
          ``begin_tick(handles, query_lens, window=..., sinks=...)``
  weigh   attention over the whole cache that also adds up what weight every cached
          token got from this tick's queries, all heads together: ``attend_layer``
          of a batch begun with ``begin_tick(handles, query_lens, weights=...)``
  keep    the tokens that stay when caches are cut to a budget: the first ones, the
          last ones, and the heaviest of the others:
          ``PagedKVCacheManager.keep_positions``
  verify  the drafted tokens of a tree tick against the target's probabilities, from
          given uniform numbers: ``hayate_amd.sampler.verify_tree``

With `own` the framework's calls run, else their plain forms in torch. Lengths, trees
and windows belong to the case (``lens`` seeds them), page placement, values and the
drafted tokens to the seed.
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
VOCAB = 151_936
DEV = "cuda"


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one user drafts from a small part of a long document: the smallest call
        _attend("window 1 on 30k", batch=1, lo=30_000, hi=30_000, window=500, sinks=4),
        # a served batch with spread contexts, some shorter than the window
        _attend("window 32 on 4k", batch=32, lo=256, hi=4096, window=1000, sinks=4),
        # wide windows on long contexts: the largest reads
        _attend("window 20 on 32k", batch=20, lo=8000, hi=32_000, window=4096, sinks=64),
        # prompt chunks, some at their prompt's start
        _attend("window chunks 4x512", batch=4, q=512, lo=0, hi=5000, window=1024, sinks=4),
        # one user's decode with the weights kept
        _attend("weigh 1 on 2k", kind="weigh", batch=1, lo=2000, hi=2000),
        # a served batch's
        _attend("weigh 32 on 4k", kind="weigh", batch=32, lo=256, hi=8000),
        # prompt chunks: every row of theirs weighs every token before it
        _attend("weigh chunks 2x512", kind="weigh", batch=2, q=512, lo=1000, hi=3584),
        # one conversation is cut to a quarter
        _keep("keep 1024 of 4001", batch=1, lo=4001, hi=4001, budget=1024, sinks=4, recent=64),
        # the default batch limit on long documents
        _keep("keep 2047 of 32k", batch=20, lo=3000, hi=32_700, budget=2047, sinks=16, recent=500),
        # one user's short draft, sampled
        _verify("verify chain of 8", batch=1, nodes=8, tree="chain", temps=[0.7]),
        # trees of a small model's likeliest tokens, requests with their own settings
        _verify("verify 16x26 mixed", batch=16, nodes=26, nodes_lo=9,
                temps=[0.0, 0.7, 1.0, 1.3], top_k=[0, 50], top_p=[1.0, 0.9, 1.0]),
        # drafts that were sampled, with the probabilities they came from
        _verify("verify 32 chains of 5", batch=32, nodes=5, nodes_lo=3, tree="chain",
                temps=[1.0, 0.8], drafts=True),
    ]


def _attend(name, kind="window", batch=1, q=1, q_lo=None, decodes=0, lo=0, hi=0, window=0, sinks=0,
            page=128, q_heads=32, kv_heads=8, lens=7):
    """`decodes` of the batch's requests bring one token, the others q_lo to q."""
    case = {"kind": kind, "batch": batch, "q": q, "q_lo": q if q_lo is None else q_lo,
            "decodes": decodes, "ctx_lo": lo, "ctx_hi": hi, "window": window, "sinks": sinks,
            "page": page, "q_heads": q_heads, "kv_heads": kv_heads, "lens": lens}
    return dict(case, name=name) if name else case


def _keep(name, batch, lo, hi, budget, sinks, recent, lens=7):
    case = {"kind": "keep", "batch": batch, "ctx_lo": lo, "ctx_hi": hi, "budget": budget,
            "sinks": sinks, "recent": recent, "lens": lens}
    return dict(case, name=name) if name else case


def _verify(name, batch, nodes, nodes_lo=None, tree="wide", temps=(1.0,), top_k=(0,), top_p=(1.0,),
            drafts=False, vocab=VOCAB, dtype="bfloat16", lens=7):
    """Requests take the temperatures, top_k (0: none) and top_p in turn."""
    case = {"kind": "verify", "batch": batch, "nodes": nodes,
            "nodes_lo": nodes if nodes_lo is None else nodes_lo, "tree": tree,
            "temps": ",".join(map(str, temps)), "top_k": ",".join(map(str, top_k)),
            "top_p": ",".join(map(str, top_p)), "drafts": drafts, "vocab": vocab, "dtype": dtype,
            "lens": lens}
    return dict(case, name=name) if name else case


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["window"] * 4 + ["weigh"] * 3 + ["keep", "verify", "verify"])
    lens = rng.randrange(1 << 20)
    if kind == "keep":
        hi = _log(rng, 2, 32_700)
        budget = _log(rng, 1, min(hi, 8000))
        sinks = rng.randint(0, min(64, budget))
        return _keep(None, batch=_log(rng, 1, 20), lo=int(hi * rng.choice([1.0, 0.4, 0.05])), hi=hi,
                     budget=budget, sinks=sinks,
                     recent=rng.choice([0, 1, rng.randint(0, budget - sinks)]) if budget > sinks
                     else 0, lens=lens)
    if kind == "verify":
        drafts = rng.random() < 0.4
        chain = drafts or rng.random() < 0.2
        nodes = _log(rng, 1, 12 if chain else 128)
        batch = _log(rng, 1, max(1, min(32, (200 if drafts else 400) // nodes)))
        return _verify(None, batch=batch, nodes=nodes,
                       nodes_lo=max(1, int(nodes * rng.choice([1.0, 0.3]))),
                       tree="chain" if chain else "wide",
                       temps=rng.choice([[0.0], [0.7], [1.0, 0.0], [1.0, 0.6, 1.5]]),
                       top_k=rng.choice([[0], [0], [20], [0, 50]]),
                       top_p=rng.choice([[1.0], [1.0], [0.9], [1.0, 0.8]]), drafts=drafts,
                       vocab=rng.choice([VOCAB, VOCAB, 32_000, _log(rng, 2, 131_072)]),
                       dtype=rng.choice(["bfloat16", "bfloat16", "float16"]), lens=lens)
    q_heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 8), (16, 8), (64, 8), (32, 2), (8, 8)])
    q = rng.choice([1, 1, _log(rng, 2, 512)])
    batch = _log(rng, 1, 32 if q == 1 else max(1, min(12, 1500 // q)))
    window, sinks = 0, 0
    # keys read in all, and products of queries with keys, below the largest listed cases'
    most = min(32_000, 100_000 // batch, 80_000_000 // (batch * q * q_heads))
    if kind == "window":
        window, sinks = _log(rng, 1, min(8192, most)), rng.choice([0, 4, _log(rng, 1, 300)])
        most = 32_000 if q == 1 else 12_000
    hi = _log(rng, 1, max(2, most))
    return _attend(None, kind=kind, batch=batch, q=q, q_lo=max(1, int(q * rng.choice([1, 0.3]))),
                   decodes=0 if q == 1 else rng.choice([0, 0, batch // 2]),
                   lo=int(hi * rng.choice([1.0, 0.4, 0.0])), hi=hi, window=window, sinks=sinks,
                   page=rng.choice([128, 128, 256]), q_heads=q_heads, kv_heads=kv_heads, lens=lens)


def _lengths(case):
    """(cached tokens, this tick's tokens) of every request."""
    r = random.Random(case["lens"])
    cached = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    return cached, [1 if i < case["decodes"] else r.randint(case["q_lo"], case["q"])
                    for i in range(case["batch"])]


def _parents(case):
    """The tree of every request: node 0 is its last token, whose successors are drafted."""
    r = random.Random(case["lens"] + 1)
    trees = []
    for _ in range(case["batch"]):
        n = r.randint(case["nodes_lo"], case["nodes"])
        if case["tree"] == "chain":
            trees.append(list(range(-1, n - 1)))
        else:  # nodes in the order of their likelihood: early ones get more children
            trees.append([-1] + [min(i - 1, int(i * r.random() ** 2)) for i in range(1, n)])
    return trees


def _settings(case):
    """Temperature, top_k (0: none) and top_p of every request."""
    given = [[float(x) for x in case[name].split(",")] for name in ("temps", "top_k", "top_p")]
    return [[values[b % len(values)] for values in given] for b in range(case["batch"])]


# --------------------------------------------------------------- the inputs
class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.host = random.Random(seed)

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        x = torch.empty(shape, dtype=dtype, device=DEV)
        flat, step = x.view(-1), 1 << 27
        for i in range(0, flat.numel(), step):
            n = min(step, flat.numel() - i)
            flat[i : i + n] = torch.randn(n, generator=self.g, device=DEV) * std
        return x

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device=DEV)


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
    shape = (1, 1, case["kv_heads"], len(order) * page, D)
    return lists, gen.normal(*shape), gen.normal(*shape)


def _inputs(case, seed):
    """Everything a pass reads, as plain tensors and lists."""
    gen = _Gen(seed)
    if case["kind"] == "keep":
        r = random.Random(case["lens"])
        lens = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
        # heavy-tailed, and equal where the sums are those of a few bf16 numbers
        weights = (-torch.log(gen.uniform(case["batch"] + 2, max(lens) + 5))) ** 3
        return {"lens": lens, "weights": weights.to(torch.bfloat16).float()}
    if case["kind"] == "verify":
        return _verify_inputs(case, gen)
    cached, fresh = _lengths(case)
    sizes = [c + n for c, n in zip(cached, fresh)]
    lists, k, v = _pools(case, gen, sizes)
    got = {"lists": lists, "cached": cached, "fresh": fresh, "k_pool": k, "v_pool": v,
           "q": gen.normal(sum(fresh), case["q_heads"], D)}
    if case["kind"] == "weigh":  # what earlier ticks and layers added up
        got["weights"] = gen.uniform(case["batch"] + 1, max(sizes) + 3)
    return got


def _verify_inputs(case, gen):
    """Logits with a few likely tokens a row, and drafted tokens that are mostly the likelier
    ones of their parent's row."""
    parents, vocab = _parents(case), case["vocab"]
    sizes = [len(t) for t in parents]
    n, few = sum(sizes), min(6, vocab)
    first = np.repeat(np.cumsum(sizes) - sizes, sizes)
    packed = np.concatenate([np.asarray(t) for t in parents])
    parent = torch.from_numpy(np.where(packed < 0, 0, packed) + first).to(DEV)
    logits = gen.normal(n, vocab, std=2.0, dtype=torch.float32)
    likely = (gen.uniform(n, few) * vocab).long().clamp(max=vocab - 1)
    rank = torch.arange(few, device=DEV)
    logits.scatter_(1, likely, 16.0 - 2.0 * rank + gen.uniform(n, few))
    logits = logits.to(getattr(torch, case["dtype"]))
    own_token = (gen.uniform(n) * vocab).long().clamp(max=vocab - 1)
    pick = (gen.uniform(n) ** 3 * few).long().clamp(max=few - 1)
    tokens = torch.where(gen.uniform(n) < 0.85, likely[parent, pick], own_token)
    got = {"parents": parents, "logits": logits, "tokens": tokens,
           "uniforms": gen.uniform(n + len(sizes))}
    if case["drafts"]:  # a draft model's probabilities, near the target's
        near = logits[parent].float() + gen.normal(n, vocab, std=0.7, dtype=torch.float32)
        got["drafts"] = torch.softmax(near, -1)
    return got


def _table(lists):
    """(requests, most pages) page ids, 0 past a request's own."""
    table = torch.zeros(len(lists), max(1, max(len(p) for p in lists)), dtype=torch.long)
    for row, pages in enumerate(lists):
        table[row, : len(pages)] = torch.tensor(pages, dtype=torch.long)
    return table.to(DEV)


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        return _own_state(state)
    kind = case["kind"]
    if kind == "keep":
        state["lens"] = torch.tensor(state["lens"], device=DEV)
    elif kind == "verify":
        _plain_trees(state)
    else:
        state["table"] = _table(state["lists"])
        # single tokens and chunks apart, so that one does not pad the other
        fresh = np.array(state["fresh"])
        first = np.cumsum(fresh) - fresh
        state["groups"] = []
        for which in (fresh == 1, fresh > 1):
            if which.any():
                (b,) = np.nonzero(which)
                state["groups"].append((int(fresh[b].max()), *(
                    torch.from_numpy(np.asarray(x)).to(DEV)
                    for x in (b, np.array(state["cached"])[b], fresh[b], first[b]))))
    return state


def _plain_trees(s):
    """Packed trees as tables: every node's request and parent, its earlier siblings, and its
    ancestors and itself."""
    case, parents = s["case"], s["parents"]
    n, at = sum(len(t) for t in parents), 0
    request, parent, root = np.zeros(n, int), np.zeros(n, int), np.zeros(n, bool)
    line = np.zeros((n, n), bool)
    for b, tree in enumerate(parents):
        for i, p in enumerate(tree):
            request[at + i], root[at + i], parent[at + i] = b, p < 0, at + max(p, 0)
            if p >= 0:
                line[at + i] = line[at + p]
            line[at + i, at + i] = True
        at += len(tree)
    earlier = (parent[:, None] == parent[None]) & (np.arange(n)[:, None] > np.arange(n)[None])
    earlier &= ~root[:, None] & ~root[None]
    first = np.searchsorted(request, np.arange(len(parents)))
    temp, top_k, top_p = np.array(_settings(case)).T
    s.update({name: torch.from_numpy(x).to(DEV) for name, x in (
        ("request", request), ("parent", parent), ("root", root), ("line", line),
        ("earlier", earlier), ("first", first),
        ("temp", temp.astype(np.float32)), ("top_k", top_k.astype(np.int64)),
        ("top_p", top_p.astype(np.float32)))})
    s["levels"] = int(line.sum(1).max())
    s["cuts"] = bool((top_k > 0).any() or (top_p < 1).any())


def _own_state(s):
    """What a program has at hand: the pool with its requests in place, and the tick's batch."""
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "hayate-exp_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from hayate_amd import PagedKVCacheManager

    case = s["case"]
    if case["kind"] in ("keep", "verify"):
        # (the pool holds lengths and trees only: its rows are not read)
        sizes = s["lens"] if case["kind"] == "keep" else [len(t) for t in s["parents"]]
        m = PagedKVCacheManager(1, 1, D, sum(n + 128 for n in sizes), 128, len(sizes),
                                torch.bfloat16, DEV)
        handles = [m.allocate() for _ in sizes]
        if case["kind"] == "keep":
            for h, n in zip(handles, sizes):
                m.reserve(h, n)
                h.length = n
        else:
            s["batch"] = m.begin_tree(handles, s["parents"])
            s["settings"] = [[x[0] for x in _settings(case)],
                             [int(x[1]) or None for x in _settings(case)],
                             [x[2] for x in _settings(case)]]
        return dict(s, m=m, handles=handles)
    k = s.pop("k_pool")
    m = PagedKVCacheManager(1, case["kv_heads"], D, k.shape[3], case["page"], len(s["lists"]),
                            torch.bfloat16, DEV, num_q_heads=case["q_heads"])
    m.k_cache.copy_(k)
    m.v_cache.copy_(s.pop("v_pool"))
    handles = []
    for c, pages in zip(s["cached"], s["lists"]):
        h = m.allocate()
        m.claim_pages(h, pages)
        h.length = c
        handles.append(h)
    how = ({"window": case["window"], "sinks": case["sinks"]} if case["kind"] == "window"
           else {"weights": s["weights"]})
    return dict(s, m=m, handles=handles, batch=m.begin_tick(handles, s["fresh"], **how))


# ---------------------------------------------------------------- the passes
def run(state):
    with torch.inference_mode():
        return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    case = s["case"]
    if case["kind"] == "window":
        return {"out": s["batch"].attend_layer(s["q"], 0)}
    if case["kind"] == "weigh":
        return {"out": s["batch"].attend_layer(s["q"], 0), "weights": s["weights"]}
    if case["kind"] == "keep":
        return {"positions": s["m"].keep_positions(s["handles"], s["weights"], case["budget"],
                                                   sinks=case["sinks"], recent=case["recent"])}
    from hayate_amd.sampler import verify_tree

    paths, lengths, tokens = verify_tree(s["batch"], s["logits"], s["tokens"], *s["settings"],
                                         s["uniforms"], s.get("drafts"))
    return {"paths": paths, "lengths": lengths, "tokens": tokens}


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "keep":
        return {"positions": _plain_keep(s)}
    if kind == "verify":
        return _plain_verify(s)
    out = torch.empty_like(s["q"])
    for group in s["groups"]:
        _plain_attend(s, out, *group)
    return {"out": out} if kind == "window" else {"out": out, "weights": s["weights"]}


def _plain_attend(s, out, most, b, cached, fresh, first):
    """Requests b with `cached` tokens and `fresh` new ones, at most `most`, whose packed rows
    begin at `first`."""
    case = s["case"]
    page, hq, hkv, window, sinks = (case[x] for x in ("page", "q_heads", "kv_heads", "window",
                                                      "sinks"))
    width = s["table"].shape[1] * page
    keys = torch.arange(width, device=DEV).expand(len(b), width)
    if window and sinks + window + most - 1 < width:  # the keys that some row may see
        span = torch.arange(window + most - 1, device=DEV)
        keys = torch.cat([keys[:, :sinks], (cached - window + 1).clamp(min=sinks)[:, None] + span], 1)
    at = keys.clamp(max=width - 1)
    where = s["table"][b[:, None], at // page] * page + at % page
    k = s["k_pool"][0, 0][:, where].transpose(0, 1).float()  # (requests, kv heads, keys, D)
    v = s["v_pool"][0, 0][:, where].transpose(0, 1).float()
    node = torch.arange(most, device=DEV)
    live = node < fresh[:, None]
    row = (first[:, None] + node).clamp(max=len(out) - 1)
    q = s["q"][row].float()
    q = q.view(len(b), most, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(len(b), hkv, -1, D)
    score = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D)
    place = (cached[:, None] + node)[:, :, None]  # of every row
    seen = keys[:, None] <= place
    if window:
        seen &= (keys[:, None] < sinks) | (place - keys[:, None] < window)
    # (a request's rows beyond its own see the keys of a row of it, and are dropped)
    score = score.view(len(b), hkv, hq // hkv, most, -1)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score = torch.exp(score - score.amax(-1, keepdim=True))
    score /= score.sum(-1, keepdim=True)
    got = torch.matmul(score.view(len(b), hkv, -1, score.shape[-1]), v)
    got = got.view(len(b), hkv, hq // hkv, most, D).permute(0, 3, 1, 2, 4)
    out[row[live]] = got.reshape(len(b), most, hq, D)[live].to(torch.bfloat16)
    if not window:
        score *= live[:, None, None, :, None]
        n = min(width, s["weights"].shape[1])
        s["weights"][b, :n] += score.sum((1, 2, 3))[:, :n]


def _plain_keep(s):
    case, lens = s["case"], s["lens"][:, None]
    weights = s["weights"][: len(lens)]
    at = torch.arange(weights.shape[1], device=DEV)[None]
    always = ((at < case["sinks"]) | (at >= lens - case["recent"])) & (at < lens)
    rank = torch.where(always, math.inf, weights).masked_fill(at >= lens, -math.inf)
    order = torch.argsort(rank, dim=1, descending=True, stable=True)[:, : case["budget"]]
    kept = torch.where(order < lens, order, weights.shape[1])
    if kept.shape[1] < case["budget"]:
        more = kept.new_full((len(kept), case["budget"] - kept.shape[1]), weights.shape[1])
        kept = torch.cat([kept, more], 1)
    kept = torch.sort(kept, dim=1).values
    return torch.where(kept < weights.shape[1], kept, -1).to(torch.int32)


def _plain_verify(s):
    n, vocab = s["logits"].shape
    request, parent, earlier = s["request"], s["parent"], s["earlier"]
    greedy = s["temp"] == 0
    best = torch.argmax(s["logits"], -1)
    # 64 bits: a draw's border is one of many thousand
    score = s["logits"].double() / torch.where(greedy, 1, s["temp"]).double()[request, None]
    if s["cuts"]:
        ordered, index = torch.sort(score, dim=-1, descending=True, stable=True)
        k = torch.where(s["top_k"] > 0, s["top_k"].clamp(max=vocab), vocab)[request, None]
        ordered.masked_fill_(ordered < ordered.gather(1, k - 1), -math.inf)
        before = torch.cumsum(torch.softmax(ordered, -1), -1)
        before = torch.cat([torch.zeros_like(before[:, :1]), before[:, :-1]], 1)
        p = s["top_p"].double()[request, None]
        ordered.masked_fill_((before > p) & (p < 1), -math.inf)
        score.scatter_(1, index, ordered)
        del ordered, index, before
    p = torch.softmax(score, -1)
    del score
    x, u = s["tokens"], s["uniforms"].double()
    of_x = p[parent, x]
    if "drafts" in s:
        took = u[:n] * s["drafts"][torch.arange(n, device=DEV), x].double() < of_x
    else:
        twice = (earlier & (x[:, None] == x[None])).any(1)
        of_x = torch.where(twice, 0, of_x)
        took = u[:n] * (1 - torch.where(earlier, of_x, 0).sum(1)) < of_x
    took = torch.where(greedy[request], x == best[parent], took)
    took &= ~(earlier & took).any(1)
    took |= s["root"]
    path = ~(s["line"] & ~took).any(1)  # nodes whose line was taken throughout
    node = torch.arange(n, device=DEV)
    requests = torch.arange(len(greedy), device=DEV)
    of = path & (request == requests[:, None])  # (requests, nodes)
    last = torch.where(of, node, -1).amax(1)
    left = p[last]
    if "drafts" in s:
        child = (parent == last[:, None]) & ~s["root"]
        refused = child.any(1, keepdim=True)
        less = (left - s["drafts"][child.int().argmax(1)].double()).clamp(min=0)
        less = torch.where(refused, less, left)
    else:
        less = left.clone()
        child = ((parent == last[:, None]) & ~s["root"]).nonzero()
        less[child[:, 0], x[child[:, 1]]] = 0
    mass = torch.cumsum(torch.where(less.sum(1, keepdim=True) > 0, less, left), 1)
    drawn = (mass <= u[n:, None] * mass[:, -1:]).sum(1)
    tokens = torch.where(greedy, best[last], drawn)
    nodes = torch.where(of, node - s["first"][:, None], n).sort(1).values[:, : s["levels"]]
    return {"paths": torch.where(nodes < n, nodes, -1).to(torch.int32),
            "lengths": of.sum(1).to(torch.int32), "tokens": tokens[:, None]}


# ------------------------------------------------------------ bytes and flops
def work(case):
    """Each K and V row that some token sees, each logit and each row in or out moved once."""
    row = 2 * D
    if case["kind"] == "keep":
        r = random.Random(case["lens"])
        lens = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
        return {"bytes": 4 * sum(lens) + 4 * case["budget"] * len(lens), "flops": 0}
    if case["kind"] == "verify":
        n = sum(len(t) for t in _parents(case))
        logits = n * case["vocab"] * 2
        # of the draft's probabilities one row for a refused request
        drafts = case["batch"] * case["vocab"] * 4 if case["drafts"] else 0
        return {"bytes": logits + drafts, "flops": 0}
    cached, fresh = _lengths(case)
    hq, hkv, window, sinks = (case[x] for x in ("q_heads", "kv_heads", "window", "sinks"))
    keys = pairs = 0
    for c, n in zip(cached, fresh):
        if not window:
            keys += c + n
            pairs += n * c + n * (n + 1) // 2
            continue
        low = max(0, c - window + 1)
        keys += c + n - max(0, low - sinks)
        pairs += sum(t + 1 - max(0, t - window + 1 - sinks) for t in range(c, c + n))
    moved = keys * 2 * hkv * row + 2 * sum(fresh) * hq * row
    if not window:
        moved += 8 * keys
    return {"bytes": moved, "flops": 4 * hq * D * pairs}


# ------------------------------------------------------------ 64-bit results
def exact(case, seed):
    inp = _inputs(case, seed)
    if case["kind"] == "keep":
        rows = []
        for b, n in enumerate(inp["lens"]):
            w = inp["weights"][b, :n].cpu().numpy()
            kept = list(range(n))
            if n > case["budget"]:
                a, z = case["sinks"], n - case["recent"]
                others = sorted(range(a, z), key=lambda i: (-w[i], i))
                others = others[: case["budget"] - a - case["recent"]]
                kept = sorted(kept[:a] + others + kept[z:])
            rows.append(kept + [-1] * (case["budget"] - len(kept)))
        return {"positions": torch.tensor(rows, dtype=torch.int32)}
    if case["kind"] == "verify":
        return _exact_verify(case, inp)
    page, hq, hkv = case["page"], case["q_heads"], case["kv_heads"]
    k, v, outs, at = inp["k_pool"].double(), inp["v_pool"].double(), [], 0
    weights = inp["weights"].double() if "weights" in inp else None
    for b, (pages, c, n) in enumerate(zip(inp["lists"], inp["cached"], inp["fresh"])):
        rows = inp["q"][at : at + n].double()
        at += n
        where = torch.tensor(pages, device=DEV).repeat_interleave(page) * page
        where = (where + torch.arange(page, device=DEV).repeat(len(pages)))[: c + n]
        i = torch.arange(c, c + n, device=DEV)[:, None]
        j = torch.arange(c + n, device=DEV)[None]
        hidden = j > i
        if case["window"]:
            hidden |= (j >= case["sinks"]) & (j <= i - case["window"])
        out = torch.empty(n, hq, D, dtype=torch.float64, device=DEV)
        for h in range(hq):
            keys, values = k[0, 0, h // (hq // hkv), where], v[0, 0, h // (hq // hkv), where]
            weight = torch.softmax((rows[:, h] @ keys.T * D**-0.5).masked_fill(hidden, -math.inf), 1)
            out[:, h] = weight @ values
            if weights is not None:
                weights[b, : c + n] += weight.sum(0)
        outs.append(out)
    got = {"out": torch.cat(outs)}
    return got if weights is None else {**got, "weights": weights}


def _exact_verify(case, inp):
    """The walk down each tree, node by node."""
    x, u, at = inp["tokens"].tolist(), inp["uniforms"].tolist(), 0
    paths, tokens, levels = [], [], 1
    n_all = len(x)

    def distribution(row, t, k, p):
        score = row.double() / float(np.float32(t))
        if k:
            score[score < torch.topk(score, min(int(k), len(score))).values[-1]] = -math.inf
        prob = torch.softmax(score, 0)
        if p < 1:
            value, index = torch.sort(prob, descending=True, stable=True)
            over = (torch.cumsum(value, 0) > float(np.float32(p))).nonzero()
            if len(over):
                prob[index[int(over[0]) + 1 :]] = 0
                prob /= prob.sum()
        return prob

    for b, (tree, (t, k, p)) in enumerate(zip(inp["parents"], _settings(case))):
        rows, depth = inp["logits"][at : at + len(tree)], []
        for parent in tree:
            depth.append(depth[parent] + 1 if parent >= 0 else 1)
        levels, path, node = max(levels, max(depth)), [0], 0
        while True:
            children = [i for i, parent in enumerate(tree) if parent == node and i != 0]
            left, found = None, None
            if t > 0:
                prob = distribution(rows[node], t, k, p)
                left = prob.clone()
            for i in children:
                token = x[at + i]
                if t == 0:
                    taken = token == int(torch.argmax(rows[node]))
                elif case["drafts"]:
                    q = inp["drafts"][at + i].double()
                    taken = u[at + i] * float(q[token]) < float(prob[token])
                    less = torch.clamp(prob - q, min=0)
                else:
                    taken = u[at + i] * float(left.sum()) < float(left[token])
                    less = left.clone()
                    less[token] = 0
                if taken:
                    found = i
                    break
                left = less if t > 0 else None
            if found is None:
                break
            path.append(found)
            node = found
        if t == 0:
            tokens.append(int(torch.argmax(rows[node])))
        else:
            mass = torch.cumsum(left if float(left.sum()) > 0 else prob, 0)
            tokens.append(int((mass > u[n_all + b] * mass[-1]).nonzero()[0]))
        paths.append(path)
        at += len(tree)
    return {"paths": torch.tensor([path + [-1] * (levels - len(path)) for path in paths],
                                  dtype=torch.int32),
            "lengths": torch.tensor([len(path) for path in paths], dtype=torch.int32),
            "tokens": torch.tensor(tokens, dtype=torch.int64)[:, None]}
