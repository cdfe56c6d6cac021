"""Verification of drafted trees (csrc/verify.hip) against the walk in 64 bits, node by node,
and against what it is for: paths and draws distributed as the target's own samples.

The kernel's probabilities come from 32-bit sums (relative error below 1e-6) and a draw's masses
are exact to 64 bits, so a test or a draw of a given number differs from the walk's with a
chance below 1e-6 a node: the seeds below have none."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from hayate_amd import PagedKVCacheManager
    from hayate_amd.sampler import Sampler, verify_tree

DEV = "cuda"


def batch_of(trees):
    m = PagedKVCacheManager(1, 1, 128, sum(len(t) + 128 for t in trees), 128, len(trees),
                            torch.bfloat16, DEV)
    return m.begin_tree([m.allocate() for _ in trees], trees)


def target(row, t, k, p):
    """The target's distribution of one row of logits."""
    score = row.double() / float(np.float32(t))
    if k is not None:
        score[score < torch.topk(score, min(k, len(score))).values[-1]] = -math.inf
    # (torch's softmax of float64 is off by up to 2e-6 of a probability on the GPU)
    prob = torch.exp(score - score.max())
    prob /= prob.sum()
    if p is not None and p < 1:
        value, index = torch.sort(prob, descending=True, stable=True)
        over = (torch.cumsum(value, 0) > float(np.float32(p))).nonzero()
        if len(over):
            prob[index[int(over[0]) + 1 :]] = 0
            prob /= prob.sum()
    return prob


def walk(trees, logits, tokens, temps, ks, ps, uniforms, drafts):
    x, u, n, at, out = tokens.tolist(), uniforms.tolist(), len(tokens), 0, []
    for b, (tree, t, k, p) in enumerate(zip(trees, temps, ks, ps)):
        path, node = [0], 0
        while True:
            row, found = logits[at + node], None
            if t:
                prob = target(row, t, k, p)
                left = prob.clone()
            for i in (i for i, parent in enumerate(tree) if parent == node and i):
                token = x[at + i]
                if not t:
                    took = token == int(torch.argmax(row))
                elif drafts is not None:
                    q = drafts[at + i].double()
                    took = u[at + i] * float(q[token]) < float(prob[token])
                    left = left if took else torch.clamp(prob - q, min=0)
                else:
                    took = u[at + i] * float(left.sum()) < float(left[token])
                    if not took:
                        left[token] = 0
                if took:
                    found = i
                    break
            if found is None:
                break
            path.append(found)
            node = found
        if not t:
            drawn = int(torch.argmax(row))
        else:
            mass = torch.cumsum(left if float(left.sum()) > 0 else prob, 0)
            drawn = int((mass > u[n + b] * mass[-1]).nonzero()[0])
        out.append((path, drawn))
        at += len(tree)
    return out


def inputs(trees, vocab, seed, dtype=torch.bfloat16, peak=8.0, drafts=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = sum(len(t) for t in trees)
    rand = lambda *s: torch.rand(s, generator=g, device=DEV)  # noqa: E731
    logits = torch.randn((n, vocab), generator=g, device=DEV) * 2
    few = min(4, vocab)
    likely = (rand(n, few) * vocab).long()
    logits.scatter_add_(1, likely, peak * rand(n, few))
    wide = torch.empty((n, vocab + 5), dtype=dtype, device=DEV)
    wide[:, 3 : 3 + vocab] = logits
    logits = wide[:, 3 : 3 + vocab]  # rows at any alignment
    first = np.cumsum([0] + [len(t) for t in trees[:-1]])
    parent = torch.tensor([f + max(p, 0) for f, t in zip(first, trees) for p in t], device=DEV)
    tokens = likely[parent, (rand(n) * few).long()]
    tokens = torch.where(rand(n) < 0.8, tokens, (rand(n) * vocab).long())
    q = torch.softmax(logits[parent].float() + torch.randn(
        (n, vocab), generator=g, device=DEV), -1) if drafts else None
    return logits, tokens, rand(n + len(trees)), q


def check(trees, vocab, seed, temps, ks, ps, **kw):
    logits, tokens, uniforms, q = inputs(trees, vocab, seed, **kw)
    paths, lengths, drawn = verify_tree(batch_of(trees), logits, tokens, temps, ks, ps, uniforms, q)
    want = walk(trees, logits, tokens, temps, ks, ps, uniforms, q)
    assert paths.dtype == lengths.dtype == torch.int32 and drawn.dtype == torch.int64
    levels = max(len(p) for p in (line for t in trees for line in lines(t)))
    assert paths.shape == (len(trees), levels) and drawn.shape == (len(trees), 1)
    for b, (path, token) in enumerate(want):
        got = paths[b].tolist()
        assert got == path + [-1] * (levels - len(path)), (b, got, path)
        assert int(lengths[b]) == len(path) and int(drawn[b]) == token, (b, token)
    return sum(len(p) for p, _ in want) / len(want)


def lines(tree):
    out = []
    for i, p in enumerate(tree):
        out.append(out[p] + [i] if p >= 0 else [i])
    return out


def random_tree(g, n):
    return [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, n)]


SETTINGS = [(0.0, None, None), (1.0, None, None), (0.7, 20, None), (1.3, None, 0.9),
            (0.6, 50, 0.8), (1.0, 1, None), (2.0, 10**7, 1.0), (1.0, None, 0.01)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 1000, 8191, 8192, 8193, 40_000])
def test_trees_with_settings_of_their_own(vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    trees = [random_tree(g, n) for n in (1, 2, 3, 9, 33, 64, 65, 130)]
    for shift in range(3):
        settings = (SETTINGS[shift:] + SETTINGS[:shift])[: len(trees)]
        length = check(trees, vocab, vocab + shift, *map(list, zip(*settings)), dtype=dtype)
    # some drafts stand (over 40,000 tokens the mass of N(0, 2) logits, e^12.6, leaves a likely
    # one at 8 above them a percent)
    assert not 1000 <= vocab < 10_000 or length > 1


def test_the_largest_trees_and_vocabulary():
    g = torch.Generator().manual_seed(5)
    trees = [random_tree(g, 256), [-1] + [0] * 255, list(range(-1, 255)), [-1]]
    check(trees, 151_936, 5, [1.0, 0.9, 0.5, 1.0], [None, 40, None, None], [None] * 4, peak=16.0)


@pytest.mark.parametrize("vocab", [5, 3000, 151_936])
def test_chains_with_draft_probabilities(vocab):
    trees = [list(range(-1, n - 1)) for n in (1, 2, 5, 8, 3, 6, 4, 9, 2, 2, 7)]
    settings = (SETTINGS + SETTINGS)[: len(trees)]
    for seed in range(3):
        check(trees, vocab, seed, *map(list, zip(*settings)), drafts=True)


def test_more_requests_than_one_launch_takes():
    g = torch.Generator().manual_seed(6)
    trees = [random_tree(g, 1 + i % 7) for i in range(150)]
    settings = [SETTINGS[i % len(SETTINGS)] for i in range(150)]
    check(trees, 2000, 6, *map(list, zip(*settings)))
    chains = [list(range(-1, i % 6)) for i in range(150)]
    check(chains, 2000, 7, *map(list, zip(*settings)), drafts=True)


@pytest.mark.parametrize("cut", [{70}, {0}, {63, 64}, set(range(80)) - {5, 66}])
def test_cut_requests_among_others(cut):
    """Which rows are cut differs by launch of 64 requests: in none, one, or nearly all of them."""
    g = torch.Generator().manual_seed(len(cut))
    trees = [random_tree(g, int(torch.randint(1, 6, (1,), generator=g))) for _ in range(80)]
    temps = [0.0 if b % 5 == 1 and b not in cut else 0.9 for b in range(80)]
    ks = [11 if b in cut and b % 2 else None for b in range(80)]
    ps = [0.7 if b in cut and not b % 2 else None for b in range(80)]
    check(trees, 9000, 17, temps, ks, ps)


def test_more_parts_than_workgroups_that_pick():
    g = torch.Generator().manual_seed(12)
    trees = [random_tree(g, 1 + i % 5) for i in range(30)]
    settings = [SETTINGS[i % len(SETTINGS)] for i in range(30)]
    check(trees, 40_000, 8, *map(list, zip(*settings)))
    chains = [list(range(-1, i % 4)) for i in range(30)]
    check(chains, 40_000, 9, *map(list, zip(*settings)), drafts=True)


@pytest.mark.parametrize("requests,vocab", [(1, 151_936), (3, 151_936), (6, 151_936), (40, 20_000)])
def test_draws_from_new_rows_time_after_time(requests, vocab):
    """The masses of a row's parts, told from workgroup to workgroup, are those of this call and of
    none before: rows of one peak each, at a place of its own, many draws in a row."""
    g = torch.Generator(device=DEV).manual_seed(requests)
    batch = batch_of([[-1]] * requests)
    settings = [0.9] * requests, [None] * requests, [None] * requests
    tokens = torch.zeros(requests, dtype=torch.int64, device=DEV)
    base = torch.randn((requests, vocab), generator=g, device=DEV).to(torch.bfloat16)
    got, want = [], []
    for _ in range(150):
        at = torch.randint(0, vocab, (requests, 1), generator=g, device=DEV)
        logits = base.scatter(1, at, 9.0)  # half of the mass, about
        uniforms = torch.rand(2 * requests, generator=g, device=DEV)
        got.append(verify_tree(batch, logits, tokens, *settings, uniforms)[2][:, 0])
        score = logits.double() / float(np.float32(0.9))
        mass = torch.cumsum(torch.exp(score - score.amax(1, keepdim=True)), 1)
        over = mass > uniforms[requests:, None].double() * mass[:, -1:]
        want.append(over.byte().argmax(1))
    assert torch.equal(torch.stack(got), torch.stack(want))


def test_equal_tokens_and_certain_ones():
    """Siblings with one token: refused once, refused for good. A token that has all the mass
    stands whatever the number; where everything is refused the draw is from p."""
    trees = [[-1, 0, 0, 0, 0]] * 4
    logits = torch.zeros((20, 50), dtype=torch.bfloat16, device=DEV)
    logits[:, 7] = 3.0
    tokens = torch.tensor([1, 7, 7, 7, 9] * 4, device=DEV)
    uniforms = torch.full((24,), 0.999, device=DEV)
    uniforms[20:] = torch.tensor([0.0, 0.3, 0.6, 0.99999], device=DEV)
    settings = [1.0] * 4, [None] * 4, [None] * 4
    paths, lengths, drawn = verify_tree(batch_of(trees), logits, tokens, *settings, uniforms)
    assert lengths.tolist() == [1] * 4
    assert drawn.flatten().tolist() == [p[1] for p in walk(trees, logits, tokens, *settings,
                                                            uniforms, None)]
    assert 7 not in drawn and 9 not in drawn
    logits[:, 7] = 200.0
    paths, lengths, drawn = verify_tree(batch_of(trees), logits, tokens, *settings, uniforms)
    # (u = 0 takes the first token with any mass, here e^-200 of it)
    assert paths.tolist() == [[0, 1]] * 4 and drawn.flatten().tolist() == [0, 7, 7, 7]
    # (rows that are no distribution, so that the test fails) what is left is e^-200 a token
    # of the others, or nothing: then the draw is from p
    chain = [[-1, 0]]
    numbers = torch.tensor([0.0, 0.5, 0.2], device=DEV)
    q = torch.zeros((2, 50), device=DEV)
    q[:, 7] = 4.0
    for rest, want in ((0.0, 10), (4.0, 7)):
        q[:, :7] = q[:, 8:] = rest
        _, lengths, drawn = verify_tree(batch_of(chain), logits[:2], tokens[:2], [1.0], [None],
                                        [None], numbers, q)
        assert lengths.tolist() == [1] and drawn.tolist() == [[want]]
        assert walk(chain, logits[:2], tokens[:2], [1.0], [None], [None], numbers, q) == [([0], want)]


@pytest.mark.parametrize("value", [-1.0, 2.5, 0.0])
def test_more_equal_logits_than_16_bits_count(value):
    """70,000 to 100,000 of a row are equal (of the zeros, half are negative): cut within,
    above and below them."""
    vocab, tree = 140_000, [-1, 0, 0, 2, 2, 2]
    settings = [(1.0, None, 0.97), (0.8, 100, None), (1.0, 120_000, 0.6), (1.5, 80_000, None),
                (0.7, None, 0.2)]
    trees = [tree] * len(settings)
    g = torch.Generator(device=DEV).manual_seed(5)
    logits = torch.randn((30, vocab), generator=g, device=DEV)
    for i in range(30):
        same = torch.randperm(vocab, generator=g, device=DEV)[: 70_000 + 1000 * i]
        logits[i, same] = value
        logits[i, same[::2]] *= -1 if value == 0 else 1
    peaks = torch.randint(0, vocab, (30, 3), generator=g, device=DEV)
    for j in range(3):
        logits[torch.arange(30), peaks[:, j]] = 11.0 + j / 4
    logits = logits.to(torch.bfloat16)
    parent = torch.tensor([6 * b + max(p, 0) for b in range(5) for p in tree], device=DEV)
    tokens = peaks[parent, torch.randint(0, 3, (30,), generator=g, device=DEV)]
    for _ in range(3):
        uniforms = torch.rand(35, generator=g, device=DEV)
        t, k, p = map(list, zip(*settings))
        paths, lengths, drawn = verify_tree(batch_of(trees), logits, tokens, t, k, p, uniforms)
        want = walk(trees, logits, tokens, t, k, p, uniforms, None)
        for b, (path, token) in enumerate(want):
            assert paths[b, : len(path)].tolist() == path and int(lengths[b]) == len(path)
            assert int(drawn[b]) == token


def test_tokens_outside_the_vocabulary_are_refused():
    logits = torch.randn(6, 30, device=DEV).to(torch.bfloat16)
    tokens = torch.tensor([0, -1, 30, 2**40, -(2**40), 31], device=DEV)
    for t in (0.0, 1.0):
        for tree, q in (([-1, 0, 0, 0, 0, 0], None),
                        (list(range(-1, 5)), torch.full((6, 30), 1 / 30, device=DEV))):
            _, lengths, drawn = verify_tree(batch_of([tree]), logits, tokens, [t], [None], [None],
                                            torch.full((7,), 0.5, device=DEV), q)
            assert lengths.tolist() == [1] and 0 <= int(drawn) < 30


def test_greedy_rows_take_the_first_largest_logit_and_nan():
    logits = torch.zeros((4, 9000), dtype=torch.bfloat16, device=DEV)
    logits[0, [8500, 40]] = 5.0
    logits[1] = -0.0
    logits[1, 3] = 0.0
    logits[2, 8999] = float("nan")
    logits[3] = float("-inf")
    trees = [[-1], [-1], [-1], [-1]]
    _, _, drawn = verify_tree(batch_of(trees), logits, torch.zeros(4, dtype=torch.long, device=DEV),
                              [0.0] * 4, [None] * 4, [None] * 4, torch.zeros(8, device=DEV))
    assert drawn.flatten().tolist() == torch.argmax(logits, -1).tolist() == [40, 0, 8999, 0]


def test_infinite_logits_off_the_path_do_not_count():
    """A row that no path reaches may hold anything; -inf is no mass."""
    trees = [[-1, 0, 0]]
    logits = torch.zeros((3, 100), dtype=torch.bfloat16, device=DEV)
    logits[0, 5] = 50.0
    logits[2] = float("nan")
    logits[1, :50] = float("-inf")
    paths, _, drawn = verify_tree(batch_of(trees), logits, torch.tensor([0, 5, 6], device=DEV),
                                  [1.0], [None], [None], torch.tensor([0.0, 0.5, 0.5, 0.5], device=DEV))
    assert paths.tolist() == [[0, 1]] and int(drawn) == 75


def test_paths_and_draws_are_distributed_as_the_target():
    """The first token that a request gets, drafted or drawn, over many requests with the same
    logits: its frequency is p within 5 standard deviations, in trees and in chains with drafts
    drawn from q."""
    g = torch.Generator(device=DEV).manual_seed(1)
    vocab, n = 6, 20_000
    row = torch.randn(vocab, generator=g, device=DEV).to(torch.bfloat16)
    p = torch.softmax(row.double() / float(np.float32(0.8)), 0)
    for tree in ([-1, 0, 0, 0], [-1, 0]):
        trees, size = [tree] * n, len(tree)
        logits = row.expand(n * size, vocab).contiguous()
        uniforms = torch.rand(n * size + n, generator=g, device=DEV)
        tokens, q = torch.tensor([0, 3, 1, 4][:size], device=DEV).repeat(n), None
        if size == 2:
            one = torch.softmax(torch.randn(vocab, generator=g, device=DEV), 0)
            q = one.expand(n * size, vocab).contiguous()
            tokens = torch.multinomial(one, n * size, replacement=True, generator=g)
        paths, lengths, drawn = verify_tree(batch_of(trees), logits, tokens, [0.8] * n, [None] * n,
                                            [None] * n, uniforms, q)
        child = paths[:, 1].clamp(min=0).long() + size * torch.arange(n, device=DEV)
        got = torch.where(lengths > 1, tokens[child], drawn[:, 0])
        share = torch.bincount(got, minlength=vocab).double() / n
        assert ((share - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all(), (share, p)
        assert 0 < int((lengths > 1).sum()) < n


def test_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(3)
    trees = [random_tree(g, n) for n in (5, 20, 1)]
    settings = [1.0, 0.7, 0.0], [None, 30, None], [0.9, None, None]
    logits, tokens, uniforms, _ = inputs(trees, 9000, 3)
    batch = batch_of(trees)
    eager = verify_tree(batch, logits, tokens, *settings, uniforms)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = verify_tree(batch, logits, tokens, *settings, uniforms)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify_tree(batch, logits, tokens, *settings, uniforms)
    for step in range(4):
        new = inputs(trees, 9000, 50 + step)
        logits.copy_(new[0]), tokens.copy_(new[1]), uniforms.copy_(new[2])
        graph.replay()
        torch.cuda.synchronize()
        eager = verify_tree(batch, logits, tokens, *settings, uniforms)
        assert all(torch.equal(a, b) for a, b in zip(eager, out)), step


def test_strided_inputs():
    trees = [[-1, 0, 0, 1], [-1, 0]]
    logits, tokens, uniforms, _ = inputs(trees, 500, 9)
    settings = [1.0, 0.9], [None, 5], [None, 0.9]
    want = verify_tree(batch_of(trees), logits, tokens, *settings, uniforms)
    got = verify_tree(batch_of(trees), logits.T.contiguous().T, tokens.repeat_interleave(2)[::2],
                      *settings, uniforms.repeat_interleave(3)[::3])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = verify_tree(batch_of(trees), logits[:, None], tokens, *settings, uniforms)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_parameter_types():
    trees = [[-1, 0, 0, 1], [-1, 0], [-1]]
    logits, tokens, uniforms, _ = inputs(trees, 500, 9)
    want = verify_tree(batch_of(trees), logits, tokens, [1.0, 0.5, 0.0], [7, None, 3],
                       [1.0, 0.75, None], uniforms)
    got = verify_tree(batch_of(trees), logits, tokens, [1, np.float32(0.5), np.int64(0)],
                      [np.int64(7), None, np.int32(3)], [1, np.float64(0.75), None], uniforms)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_the_samplers_form():
    class Request:
        def __init__(self, temperature, top_k=None, top_p=None):
            self.temperature, self.top_k, self.top_p = temperature, top_k, top_p

    trees = [[-1, 0, 0, 1], [-1, 0], [-1]]
    logits, tokens, _, _ = inputs(trees, 500, 9)
    requests = [Request(0.0), Request(0.8, 20, 0.9), Request(1.0)]
    gens = [torch.Generator(device=DEV).manual_seed(4) for _ in range(2)]
    batch = batch_of(trees)
    paths, drawn = Sampler(generator=gens[0]).verify(logits, tokens, batch, requests)
    want = verify_tree(batch, logits, tokens, [0.0, 0.8, 1.0], [None, 20, None], [None, 0.9, None],
                       torch.rand(10, generator=gens[1], device=DEV))
    assert paths == [row[:n] for row, n in zip(want[0].tolist(), want[1].tolist())]
    assert drawn == want[2].flatten().tolist()
    assert [batch.check_path(b, path) for b, path in enumerate(paths)] == paths
    with pytest.raises(ValueError):
        Sampler().verify(logits, tokens, batch, requests[:2])
