"""Rope positions of caches that dropped tokens: kept keys keep their rotation, so what is
appended afterwards goes on behind the last kept token's position. Bookkeeping, without a GPU."""

import numpy as np
import pytest
import torch

import hayate_amd.paged_cache as pc
from hayate_amd import Cache, PagedKVCacheManager, PrefixCache
from tree_util import chain


@pytest.fixture
def m(monkeypatch):
    """A pool in host memory whose rows stay where they are."""
    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    monkeypatch.setattr(PagedKVCacheManager, "move_tokens", lambda self, *args: None)
    return PagedKVCacheManager(1, 8, 128, 16 * 128, 128, 6, torch.bfloat16, "cpu", num_q_heads=32)


def handle(m, length):
    h = m.allocate()
    m.reserve(h, length)
    h.length = length
    return h


def test_appends_follow_the_last_kept_token(m):
    h, plain = handle(m, 500), handle(m, 70)
    assert h.next_position == 500 and m.begin_tick([h], [1]).positions is None
    m.compact(h, [*range(16), *range(300, 490)])  # ten tokens at the end go, too
    assert h.length == 206 and h.next_position == 490
    batch = m.begin_tree([h, plain], [[-1, 0, 0, 1], [-1]])
    assert batch.positions.tolist() == [490, 491, 491, 492, 70]
    tick = m.begin_tick([plain, h], [2, 3])
    assert tick.positions.tolist() == [70, 71, 490, 491, 492]
    assert tick.cache_lens.tolist() == [70, 206]
    uniform = m.begin_batch([h, plain], 2)
    assert uniform.positions.tolist() == [490, 491, 70, 71]
    assert m.begin_tick([plain], [1]).positions is None
    m.commit_tick([h], [3])
    assert h.length == 209 and h.next_position == 493


def test_prefixes_have_no_gaps(m):
    h = handle(m, 500)
    m.compact(h, range(300))
    assert h.positions is None and h.next_position == 300
    m.compact(h, [*range(100), 200])
    assert h.next_position == 201
    m.truncate(h, 100)
    assert h.positions is None and h.next_position == 100
    m.compact(h, [5, 6])
    assert h.next_position == 7
    m.compact(h, [])
    assert h.positions is None and h.next_position == 0


def test_compact_again_truncate_and_commit(m):
    h = handle(m, 300)
    m.compact(h, [0, 1, *range(100, 300)])
    m.reserve(h, 204)
    m.commit_tick([h], [2])  # positions 300 and 301
    m.compact(h, [1, 2, 201, 202, 203])
    assert list(h.positions) == [1, 100, 299, 300, 301] and h.next_position == 302
    batch = m.begin_tree([h], [chain(4)])
    assert batch.positions.tolist() == [302, 303, 304, 305]
    m.commit_tree([h], batch, [[0, 1]])
    assert h.length == 7 and h.next_position == 304
    m.truncate(h, 6)
    assert h.next_position == 303
    m.truncate(h, 2)
    assert h.next_position == 101 and list(h.positions) == [1, 100]
    assert m.begin_tick([h], [1]).positions.tolist() == [101]
    m.release(h)
    assert m.allocate().positions is None


def test_forks_and_prefixes_carry_them(m):
    h = handle(m, 300)
    m.compact(h, [*range(10), *range(200, 300)])
    assert m.fork(h).next_position == 300
    assert m.fork(h, 50).next_position == 240
    assert m.fork(h, 10).positions is None
    copied = m.fork(h, 60, copy=True)
    assert copied.next_position == 250
    m.release(copied)
    prefix = m.share(h, 100)
    assert m.allocate_for_request(prefix).next_position == 290
    short = prefix.slice(8)
    g = m.allocate_for_request(short)
    assert g.positions is None and g.next_position == 8
    prefix.reset()
    assert prefix.positions is None
    m.truncate(h, 20)  # the fork's own positions stay
    assert h.next_position == 210


def test_copies_out_of_the_pool_carry_them(m, monkeypatch):
    taken = []
    monkeypatch.setattr(m, "_gather", lambda pages, n: Cache.from_tensors(
        *[torch.zeros(1, 8, n, 128, dtype=torch.bfloat16)] * 2))
    h = handle(m, 300)
    m.compact(h, [*range(10), *range(200, 300)])
    for cache in (m.snapshot(h), m.share(h).to_cache()):
        assert list(cache.positions) == [*range(10), *range(200, 300)]
        assert list(cache.slice(12).positions) == [*range(10), 200, 201]
        assert cache.slice(9, clone=True).positions is None
        cache.reset()
        assert cache.positions is None
    assert m.snapshot(h, 10).positions is None
    # and back into a pool

    class Lib:
        def hy_page_scatter(self, *args):
            taken.append(args)
            return 0

    monkeypatch.setattr(pc._native, "lib", lambda: Lib())
    cache = m.snapshot(h, 12)
    g = m.allocate_for_request(cache)
    assert taken and g.length == 12 and g.next_position == 202
    m.import_cache(g, cache.slice(4))
    assert g.positions is None and g.next_position == 4


def test_a_prompt_with_gaps_is_no_prefix(m):
    """What was computed behind dropped tokens is not the cache of the tokens that stayed."""
    h = handle(m, 300)
    m.compact(h, [*range(150), *range(200, 300)])
    cache = PrefixCache(1000)
    shared = m.share(h)
    refs = [m.page_refcount(p) for p in h.pages]
    with pytest.raises(ValueError):
        cache.put(list(range(250)), shared)
    assert len(cache) == 0 and [m.page_refcount(p) for p in h.pages] == refs
    cache.put(list(range(150)), shared)  # none dropped in front of these
    assert cache.get(list(range(200))).length == 150


def test_handles_still_compare():
    a, b = pc.PagedCacheHandle(0, [1], 2), pc.PagedCacheHandle(0, [1], 2)
    a.positions = np.arange(3)
    b.positions = np.arange(3)
    assert a == b
