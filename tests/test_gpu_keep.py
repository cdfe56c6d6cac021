"""The tokens that stay when caches are cut to a budget (csrc/keep.hip) against a sort, and the
eviction that moves them: pages, K, V, weights and positions."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from hayate_amd import PagedKVCacheManager
    from long_util import D, DEV, Requests, normal

INF, NAN = float("inf"), float("nan")


def expected(w, n, budget, sinks, recent):
    """Positions by a stable sort in 64 bits; NaN sorts first."""
    if n <= budget:
        return list(range(n)) + [-1] * (budget - n)
    w = w[:n].double().cpu().numpy()
    between = range(sinks, n - recent)
    order = sorted(between, key=lambda i: (0 if np.isnan(w[i]) else 1,
                                           0.0 if np.isnan(w[i]) else -w[i], i))
    return sorted([*range(sinks), *order[: budget - sinks - recent], *range(n - recent, n)])


def choose(lens, weights, budget, sinks, recent):
    m = PagedKVCacheManager(1, 1, D, sum(lens) + 128 * len(lens) + 128, 128, len(lens),
                            torch.bfloat16, DEV)
    handles = [m.allocate() for _ in lens]
    for h, n in zip(handles, lens):
        m.reserve(h, n)
        h.length = n
    got = m.keep_positions(handles, weights, budget, sinks=sinks, recent=recent)
    assert got.dtype == torch.int32 and got.shape == (len(lens), budget)
    for b, (h, n) in enumerate(zip(handles, lens)):
        assert got[b].tolist() == expected(weights[h.slot], n, budget, sinks, recent), (b, n)


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (7, 2, 5),
                                                 (64, 4, 16), (65, 0, 0), (1000, 4, 32),
                                                 (2047, 100, 1900)])
def test_lengths_around_the_budget_and_the_waves(budget, sinks, recent):
    g = torch.Generator(device=DEV).manual_seed(budget)
    lens = [0, 1, budget - 1, budget, budget + 1, budget + 63, budget + 64, budget + 1024,
            1023 + budget, 4001, 5 * budget]
    weights = torch.rand(len(lens), max(lens) + 3, generator=g, device=DEV) ** 8
    choose(lens, weights, budget, sinks, recent)


@pytest.mark.parametrize("n", [32_768 + 10, 32_768 + 11, 70_000])
def test_long_rows_are_read_again(n):
    g = torch.Generator(device=DEV).manual_seed(n)
    weights = torch.rand(2, n, generator=g, device=DEV).to(torch.bfloat16).float()  # many ties
    choose([n, n - 5], weights, 3000, 4, 6)


def test_equal_weights_go_by_position():
    for value in (0.0, -0.0, 1.5, -2.0, INF, -INF, NAN, 1e-45):
        choose([3000], torch.full((1, 3000), value, device=DEV), 500, 3, 9)
    g = torch.Generator(device=DEV).manual_seed(3)
    few = torch.tensor([0.0, -0.0, 1.0, -1.0, INF, -INF, NAN, 1e-45, -1e-45, 3e38], device=DEV)
    weights = few[torch.randint(0, len(few), (6, 2500), generator=g, device=DEV)]
    for budget in (1, 100, 600, 1300, 2000, 2499):
        choose([2500] * 6, weights, budget, 0, 0)


def test_more_requests_than_one_launch_takes():
    g = torch.Generator(device=DEV).manual_seed(8)
    weights = torch.rand(150, 400, generator=g, device=DEV)[:, 3:390]
    choose([int(x) for x in torch.randint(0, 387, (150,))], weights, 90, 2, 5)


def test_values_that_differ_in_their_last_bit():
    """Keys that share their first 22 bits."""
    g = torch.Generator(device=DEV).manual_seed(4)
    bits = 0x3F800000 + torch.randint(0, 700, (1, 9000), generator=g, device=DEV, dtype=torch.int32)
    choose([9000], bits.view(torch.float32), 4000, 10, 10)


def test_a_length_of_another_whole_type():
    m = PagedKVCacheManager(1, 1, D, 256, 128, 1, torch.bfloat16, DEV)
    h = m.allocate()
    m.commit_tick([h], np.array([m.reserve_tick([h], np.array([9]))[0]]))
    weights = torch.arange(9.0, device=DEV)[None]
    assert m.keep_positions([h], weights, 3, sinks=1, recent=0).tolist() == [[0, 7, 8]]


def test_captured_and_on_another_stream():
    r = Requests([900, 50], [0, 0], seed=1)
    weights = torch.rand(r.m.max_requests, 900, generator=r.g, device=DEV)
    eager = r.m.keep_positions(r.handles, weights, 200)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = r.m.keep_positions(r.handles, weights, 200)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = r.m.keep_positions(r.handles, weights, 200)
    for step in range(3):
        weights.copy_(torch.rand(weights.shape, generator=r.g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, r.m.keep_positions(r.handles, weights, 200)), step


def test_evict_moves_tokens_weights_and_positions():
    r = Requests([900, 100, 2000, 301], [0] * 4, seed=2, layers=3)
    weights = torch.rand(r.m.max_requests, 2050, generator=r.g, device=DEV)
    before = weights.clone()
    snaps = [r.m.snapshot(h) for h in r.handles]
    free = r.m.free_page_count
    chosen = r.m.keep_positions(r.handles, weights, 300, sinks=4, recent=20).tolist()
    kept = r.m.evict(r.handles, weights, 300, sinks=4, recent=20)
    assert [h.length for h in r.handles] == [300, 100, 300, 300]
    assert r.m.free_page_count == free + (8 - 3) + 0 + (16 - 3) + 0
    for h, snap, row, at in zip(r.handles, snaps, chosen, kept):
        assert at == [x for x in row if x >= 0]
        now = r.m.snapshot(h)
        index = torch.tensor(at, device=DEV)
        assert torch.equal(now.k, snap.k[:, :, index]) and torch.equal(now.v, snap.v[:, :, index])
        if len(at) < snap.length:
            assert torch.equal(weights[h.slot, : len(at)], before[h.slot, index])
            assert (weights[h.slot, len(at) :] == 0).all()
            assert h.positions.tolist() == at and h.next_position == snap.length
        else:
            assert torch.equal(weights[h.slot], before[h.slot]) and h.positions is None
    assert torch.equal(weights[4:], before[4:])
    # and again, of what is left
    kept = r.m.evict(r.handles, weights, 90, sinks=0, recent=1)
    assert [len(x) for x in kept] == [90] * 4
    assert r.handles[1].next_position == 100 and r.handles[0].next_position == 900


def test_evict_of_shared_pages_leaves_the_sharer_alone():
    r = Requests([700], [0], seed=5)
    child = r.m.fork(r.handles[0])
    snap = r.m.snapshot(child)
    weights = torch.rand(r.m.max_requests, 700, generator=r.g, device=DEV)
    r.m.evict(r.handles, weights, 200)
    now = r.m.snapshot(child)
    assert torch.equal(now.k, snap.k) and torch.equal(now.v, snap.v) and child.length == 700


def test_evict_without_room_for_copies_changes_nothing():
    r = Requests([700], [0], seed=5, spare=0)
    r.m.fork(r.handles[0])
    weights = torch.rand(r.m.max_requests, 700, generator=r.g, device=DEV)
    before, pages = weights.clone(), list(r.handles[0].pages)
    with pytest.raises(MemoryError):
        r.m.evict(r.handles, weights, 500)
    assert torch.equal(weights, before) and r.handles[0].pages == pages
    assert r.handles[0].length == 700 and r.handles[0].positions is None


def test_a_table_made_under_inference_mode():
    r = Requests([400], [0], seed=6)
    with torch.inference_mode():
        weights = torch.rand(r.m.max_requests, 400, generator=r.g, device=DEV)
    r.m.evict(r.handles, weights, 100)
    assert (weights[0, 100:] == 0).all() and r.handles[0].length == 100


def test_attention_after_an_eviction():
    """A tick on the cut cache attends to what stayed, and its weights add to the moved ones."""
    r = Requests([500], [1], seed=7)
    weights = torch.rand(r.m.max_requests, 600, generator=r.g, device=DEV)
    r.m.evict(r.handles, weights, 130, sinks=4, recent=16)
    r.cached = [130]
    before = weights.clone()
    k, v = normal(r.g, 1, r.hkv, D), normal(r.g, 1, r.hkv, D)
    batch = r.m.begin_tick(r.handles, [1], weights=weights)
    batch.write_layer(0, k, v)
    out = batch.attend_layer(r.q, 0)
    r.m.commit_tick(r.handles, [1])
    want, bound, total = r.expected()
    assert ((out.double() - want).abs() <= bound).all()
    assert torch.allclose(weights[0, :131].double(), before[0, :131].double() + total[0], rtol=2e-4)
    assert r.handles[0].length == 131 and r.handles[0].next_position == 501
