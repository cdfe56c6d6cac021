"""Windowed drafts, their verification, weights and eviction in one loop, as a program uses them:
the model drafts for itself with a window over a fork of its cache, a tree tick checks the drafts
on the whole cache, and the cache is cut by the weights that its tokens got."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from hayate_amd import PagedKVCacheManager
    from hayate_amd.model import Qwen3Config, Qwen3Model, init_synthetic_weights
    from hayate_amd.sampler import Sampler

DEV = "cuda"
LAYERS = 2


def make_model():
    with torch.device(DEV):
        model = Qwen3Model(Qwen3Config(num_layers=LAYERS, vocab_size=512, hidden_size=512,
                                       num_heads=8, num_kv_groups=2, intermediate_size=1024,
                                       max_position_embeddings=4096))
    init_synthetic_weights(model, 3)
    return model.eval()


class Request:
    def __init__(self, temperature=0.0, top_k=None, top_p=None):
        self.temperature, self.top_k, self.top_p = temperature, top_k, top_p


def manager(requests=4):
    return PagedKVCacheManager(LAYERS, 2, 128, 16_384, 128, 2 * requests, torch.bfloat16, DEV,
                               num_q_heads=8)


def tick(model, m, handles, tokens, **how):
    """One tick of packed tokens; (requests, vocab) logits of each one's last."""
    batch = m.begin_tick(handles, [len(t) for t in tokens], **how)
    logits, _, _ = model(torch.tensor([[x for t in tokens for x in t]], device=DEV),
                         paged_cache=batch)
    m.commit_tick(handles, [len(t) for t in tokens])
    return logits[:, -1]


def draft(model, m, handles, last, steps, window, sinks):
    """Greedy drafts of `steps` tokens a request, on forks that see a window of the cache."""
    forks = [m.fork(h) for h in handles]
    chains, at = [[] for _ in handles], [[x] for x in last]
    for _ in range(steps):
        at = [[x] for x in torch.argmax(tick(model, m, forks, at, window=window, sinks=sinks),
                                        -1).tolist()]
        for chain, x in zip(chains, at):
            chain += x
    for f in forks:
        m.release(f)
    return chains


def round_of(model, m, handles, requests, last, sampler, steps=4, window=96, sinks=4):
    """Drafts, one tree tick, and the commit; the new tokens of each request."""
    chains = draft(model, m, handles, last, steps, window, sinks)
    trees = [list(range(-1, steps)) for _ in handles]
    tokens = torch.tensor([x for n, chain in zip(last, chains) for x in [n, *chain]], device=DEV)
    batch = m.begin_tree(handles, trees)
    logits, _, _ = model(tokens[None], paged_cache=batch)
    paths, drawn = sampler.verify(logits, tokens, batch, requests)
    m.commit_tree(handles, batch, paths)
    return [[chain[i - 1] for i in path[1:]] + [n]
            for chain, path, n in zip(chains, paths, drawn)], paths


def test_drafted_tokens_are_the_models_own():
    """Greedy: every token that the loop emits is the largest logit (within bf16 rounding) of a
    plain pass over the whole sequence, and drafts were taken."""
    with torch.inference_mode():
        model, m = make_model(), manager()
        g = torch.Generator().manual_seed(1)
        prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (300, 150, 40)]
        handles = [m.allocate() for _ in prompts]
        last = torch.argmax(tick(model, m, handles, prompts), -1).tolist()
        texts = [[x] for x in last]
        taken = 0
        for _ in range(6):
            fresh, paths = round_of(model, m, handles, [Request()] * 3, last, Sampler())
            taken += sum(len(p) - 1 for p in paths)
            for text, new in zip(texts, fresh):
                text += new
            last = [text[-1] for text in texts]
            for h, prompt, text in zip(handles, prompts, texts):
                assert h.length == len(prompt) + len(text) - 1
        assert taken > 0
        for prompt, text in zip(prompts, texts):
            whole = prompt + text
            one = manager(1)
            h = one.allocate()
            done = len(prompt) - 1
            if done:
                tick(model, one, [h], [whole[:done]])
            rows = whole[done:-1]
            batch = one.begin_tree([h], [list(range(-1, len(rows) - 1))])
            logits = model(torch.tensor([rows], device=DEV), paged_cache=batch)[0][:, 0].float()
            chosen = logits[torch.arange(len(rows)), torch.tensor(whole[done + 1 :])]
            # the same logits from other kernels: bf16 states through two layers
            assert (logits.amax(-1) - chosen <= 0.05 * logits.std(-1)).all()


def test_sampled_requests_end_where_they_should():
    with torch.inference_mode():
        model, m = make_model(), manager()
        g = torch.Generator().manual_seed(2)
        prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (200, 100)]
        handles = [m.allocate() for _ in prompts]
        last = torch.argmax(tick(model, m, handles, prompts), -1).tolist()
        requests = [Request(0.8, 40, 0.95), Request(0.0)]
        sampler = Sampler(generator=torch.Generator(device=DEV).manual_seed(5))
        lengths = [h.length for h in handles]
        for _ in range(4):
            fresh, paths = round_of(model, m, handles, requests, last, sampler)
            lengths = [n + len(p) for n, p in zip(lengths, paths)]
            assert [h.length for h in handles] == lengths
            assert all(len(new) == len(p) for new, p in zip(fresh, paths))
            assert all(0 <= x < 512 for new in fresh for x in new)
            last = [new[-1] for new in fresh]


def test_a_bounded_cache():
    """Decode with weights and cut to a budget again and again: lengths, pages and rope positions
    go on, and the weights are those of the tokens that stay."""
    with torch.inference_mode():
        model, m = make_model(), manager()
        g = torch.Generator().manual_seed(4)
        prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (400, 90)]
        handles = [m.allocate() for _ in prompts]
        weights = torch.zeros(m.max_requests, 1024, device=DEV)
        logits = tick(model, m, handles, prompts, weights=weights)
        # each row of attention adds up to one: layers x heads x rows
        assert torch.allclose(weights.sum(1)[[h.slot for h in handles]],
                              torch.tensor([LAYERS * 8.0 * len(p) for p in prompts], device=DEV),
                              rtol=1e-3)
        seen = [len(p) for p in prompts]
        for step in range(60):
            last = torch.argmax(logits, -1).tolist()
            logits = tick(model, m, handles, [[x] for x in last], weights=weights)
            seen = [n + 1 for n in seen]
            if step % 20 == 19:
                before = weights.clone()
                kept = m.evict(handles, weights, 128, sinks=4, recent=30)
                for h, at in zip(handles, kept):
                    assert h.length == len(at) <= 128 and at[:4] == [0, 1, 2, 3]
                    assert torch.equal(weights[h.slot, : len(at)],
                                       before[h.slot, torch.tensor(at, device=DEV)])
                    assert len(h.pages) == 1 or h.length > 128
            assert [h.next_position for h in handles] == seen
        assert logits.isfinite().all()
        # the cut caches draft and verify like any other
        last = torch.argmax(logits, -1).tolist()
        fresh, paths = round_of(model, m, handles, [Request()] * 2, last, Sampler(), window=40)
        assert [h.next_position for h in handles] == [n + len(p) for n, p in zip(seen, paths)]
