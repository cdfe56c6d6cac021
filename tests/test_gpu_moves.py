"""Token moves and page copies on the GPU, bit for bit."""

import random

import numpy as np
import pytest
import torch

from hayate_amd import _native
from tree_util import D, chain, make_pool, physical, wide_tree, line

pytestmark = pytest.mark.gpu


def bits(x):
    return x.view(torch.int16)


def logical(m, h, n):
    rows = physical(m, h, n)
    return [bits(p)[:, 0][:, :, rows].clone() for p in (m.k_cache, m.v_cache)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def scramble(m):
    """Every slot of the pool its own bits (NaN among them)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for p in (m.k_cache, m.v_cache):
        bits(p).copy_(torch.randint(-(1 << 15), 1 << 15, p.shape, generator=g, device="cuda",
                                    dtype=torch.int16))


def moved(before, sources, start):
    out = [x.clone() for x in before]
    for x, old in zip(out, before):
        x[:, :, start : start + len(sources)] = old[:, :, list(sources)]
    return out


SOURCES = {
    "one": (100, [103]),
    "itself": (5, [5, 6, 7]),
    "over itself": (0, list(range(1, 400))),
    "by a page": (0, list(range(128, 700))),
    "far over itself": (16, list(range(40, 900))),
    "every other": (0, list(range(0, 900, 2))),
    "every third from 1": (0, list(range(1, 900, 3))),
    "a path": (517, [517, 519, 520, 560, 571]),
    "all but one": (0, [i for i in range(900) if i != 300]),
}


@pytest.mark.parametrize("name", SOURCES)
@pytest.mark.parametrize("layers,kv_heads,page", [(1, 8, 128), (5, 2, 128), (3, 1, 256)])
def test_moves(name, layers, kv_heads, page):
    start, sources = SOURCES[name]
    m, (h, other) = make_pool([900, 300], [0, 0], layers=layers, kv_heads=kv_heads, page=page)
    scramble(m)
    whole = [bits(p).clone() for p in (m.k_cache, m.v_cache)]
    before = logical(m, h, 900)
    m.move_tokens([h], [np.array(sources)], [start])
    assert same(logical(m, h, 900), moved(before, sources, start))
    assert h.length == 900
    # nothing else changed
    rows = physical(m, h, 900)[start : start + len(sources)]
    for p, old in zip((m.k_cache, m.v_cache), whole):
        old[:, :, :, rows] = bits(p)[:, :, :, rows]
        assert torch.equal(bits(p), old)


def test_moves_of_many_runs_take_several_launches():
    """Over 320 runs in one call, each launch reading what no earlier one wrote."""
    m, (h,) = make_pool([4000], [0], layers=2, kv_heads=2)
    scramble(m)
    before = logical(m, h, 4000)
    sources = sorted(random.Random(1).sample(range(4000), 1500))
    m.move_tokens([h], [sources], [0])
    assert same(logical(m, h, 4000), moved(before, sources, 0))


def test_moves_of_several_requests():
    rng = random.Random(2)
    cached = [rng.randint(1, 400) for _ in range(40)]
    m, handles = make_pool(cached, [30] * 40, layers=2)
    scramble(m)
    before = [logical(m, h, c + 30) for h, c in zip(handles, cached)]
    paths = [sorted(rng.sample(range(30), rng.randint(0, 8))) for _ in cached]
    m.move_tokens(handles, [[c + i for i in p] for c, p in zip(cached, paths)], cached)
    for h, c, old, p in zip(handles, cached, before, paths):
        assert same(logical(m, h, c + 30), moved(old, [c + i for i in p], c))


def test_moves_into_shared_pages_leave_the_other_owner_alone():
    m, (h,) = make_pool([500], [0], layers=2, spare=6)
    scramble(m)
    before = logical(m, h, 500)
    prefix, child = m.share(h, 400), m.fork(h)
    m.move_tokens([h], [list(range(200, 500))], [100])
    assert same(logical(m, h, 500), moved(before, range(200, 500), 100))
    assert same(logical(m, child, 500), before)
    assert torch.equal(bits(prefix.to_cache().k), before[0][:, :, :400])
    assert h.pages[0] != child.pages[0]  # position 100 lies in page 0
    m.release(child)
    prefix.reset()
    m.release(h)
    assert m.free_page_count == m.num_pages


def test_compact_frees_the_emptied_pages():
    m, (h,) = make_pool([1000], [100], layers=2)
    scramble(m)
    before = logical(m, h, 1000)
    free = m.free_page_count
    keep = list(range(4)) + list(range(700, 1000))
    m.compact(h, keep)
    assert h.length == 304 and len(h.pages) == 3
    assert m.free_page_count == free + 6
    assert same(logical(m, h, 304), [x[:, :, keep] for x in before])
    m.compact(h, range(304))
    assert h.length == 304
    m.compact(h, torch.tensor([0, 303]))
    assert same(logical(m, h, 2), [x[:, :, [0, 999]] for x in before])
    m.compact(h, [])
    assert h.length == 0 and not h.pages


def test_commit_tree_moves_every_layer_and_frees_the_rest():
    rng = random.Random(4)
    cached, sizes = [127, 0, 300, 64], [60, 5, 200, 1]
    m, handles = make_pool(cached, sizes, layers=3)
    trees = [wide_tree(rng, n) for n in sizes]
    batch = m.begin_tree(handles, trees)
    scramble(m)
    before = [logical(m, h, c + n) for h, c, n in zip(handles, cached, sizes)]
    paths = [line(trees[0], 59), [], line(trees[2], 180), [0]]
    m.commit_tree(handles, batch, paths)
    for h, c, old, path in zip(handles, cached, before, paths):
        n = c + len(path)
        assert h.length == n and len(h.pages) == -(-n // 128)
        assert same(logical(m, h, n), [x[:, :, list(range(c)) + [c + i for i in path]] for x in old])


def test_moves_captured_and_replayed():
    m, (h,) = make_pool([600], [0], layers=4)
    m.move_tokens([h], [[10]], [5])  # loads the kernel before the capture
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        m.move_tokens([h], [range(100, 500)], [50])
    for seed in range(3):
        scramble(m)
        before = logical(m, h, 600)
        for _ in range(seed + 1):
            want = moved(before, range(100, 500), 50)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            before = logical(m, h, 600)
            assert same(before, want)


# ------------------------------------------------------------------- copies
@pytest.mark.parametrize("layers,kv_heads,page", [(1, 8, 128), (4, 2, 128), (3, 1, 256), (2, 3, 32)])
@pytest.mark.parametrize("n", [1, 5])
def test_copies(layers, kv_heads, page, n):
    m, (a, b) = make_pool([n * page, n * page], [0, 0], layers=layers, kv_heads=kv_heads, page=page)
    scramble(m)
    want = [bits(p).clone() for p in (m.k_cache, m.v_cache)]
    tokens = [page, 0, 1, page - 1, 17][:n]
    for x in want:
        for s, d, t in zip(a.pages, b.pages, tokens):
            x[:, :, :, d * page : d * page + t] = x[:, :, :, s * page : s * page + t]
    m.copy_pages(a.pages, b.pages, tokens)
    assert same([bits(m.k_cache), bits(m.v_cache)], want)
    m.copy_pages(a.pages, b.pages)
    assert same(logical(m, a, n * page), logical(m, b, n * page))


def test_copies_of_more_pages_than_a_launch_takes():
    n = 700
    m, (a, b) = make_pool([n * 32, n * 32], [0, 0], kv_heads=1, page=32)
    scramble(m)
    m.copy_pages(a.pages, b.pages)
    assert same(logical(m, a, n * 32), logical(m, b, n * 32))


def test_one_page_to_several():
    m, (a, b) = make_pool([128, 640], [0, 0], layers=2)
    scramble(m)
    m.copy_pages([a.pages[0]] * 5, b.pages)
    one = logical(m, a, 128)
    many = logical(m, b, 640)
    for i in range(5):
        assert same(one, [x[:, :, 128 * i : 128 * i + 128] for x in many])


def test_fork_with_copies_shares_nothing():
    m, (h,) = make_pool([300], [0], layers=3, spare=8)
    scramble(m)
    before = logical(m, h, 300)
    child = m.fork(h, 290, copy=True)
    assert not set(child.pages) & set(h.pages) and child.length == 290
    assert same(logical(m, child, 290), [x[:, :, :290] for x in before])
    empty = m.fork(h, 0, copy=True)
    assert empty.length == 0 and not empty.pages
    m.release(child)
    m.release(empty)
    free = m.free_page_count
    hold = m.allocate()
    m.reserve(hold, (free - 2) * 128)  # two pages left, three wanted
    slots = len(m._free_slots)
    with pytest.raises(MemoryError):
        m.fork(h, 300, copy=True)
    assert m.free_page_count == 2 and len(m._free_slots) == slots


def test_copy_on_write_of_many_forks_in_one_tick():
    """Twelve samples of one prompt append in one tick: each gets its own copy of the
    partly filled page, the last sharer keeps the original."""
    m, (h,) = make_pool([200], [0], layers=3, spare=20, slots=20)
    scramble(m)
    before = logical(m, h, 200)
    forks = [m.fork(h) for _ in range(12)]
    m.release(h)
    m.begin_tick(forks, [1] * 12)
    assert len({f.pages[1] for f in forks}) == 12 and len({f.pages[0] for f in forks}) == 1
    assert all(m.page_refcount(f.pages[1]) == 1 for f in forks)
    for f in forks:
        assert same(logical(m, f, 200), before)


def test_move_and_copy_past_2_31_elements():
    from hayate_amd import PagedKVCacheManager

    page, pages = 256, (1 << 31) // (256 * D) + 64
    m = PagedKVCacheManager(1, 1, D, pages * page, page, 2, torch.bfloat16, "cuda")
    h = m.allocate()
    m.claim_pages(h, [pages - 1, 0, pages - 2])
    h.length = 600
    rows = physical(m, h, 600)
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in (m.k_cache, m.v_cache):
        p[:, :, :, rows] = torch.randn(1, 1, 1, 600, D, generator=g, device="cuda").to(torch.bfloat16)
    before = logical(m, h, 600)
    child = m.fork(h, copy=True)
    m.move_tokens([h], [range(37, 600)], [0])
    assert same(logical(m, h, 600), moved(before, range(37, 600), 0))
    assert same(logical(m, child, 600), before)


def test_a_refused_call_enqueues_nothing():
    m, (h,) = make_pool([300], [0], layers=2)
    scramble(m)
    before = [bits(p).clone() for p in (m.k_cache, m.v_cache)]
    lib = _native.lib()

    def move(src, first):
        a = [np.array(x, dtype=np.int32) for x in
             (h.pages, [0, len(h.pages)], [0], src, [0, len(src)], [first])]
        return lib.hy_kv_move(m.k_cache.data_ptr(), m.v_cache.data_ptr(), m.k_cache.stride(0),
                              m.k_cache.stride(2), m.num_pages, *(x.ctypes.data for x in a), 1, 2,
                              8, D, m.page_size, None)

    for src, first in (([5, 384], 4), ([5, 4], 0), ([7, 9, 9], 1), ([3, 4], 4)):
        assert move(src, first) == _native.HY_EINVAL
    torch.cuda.synchronize()
    assert same([bits(m.k_cache), bits(m.v_cache)], before)


def test_two_moves_of_drafted_tokens_out_of_a_shared_page():
    """The second move reads a drafted token behind the first one's, in the copy that the first
    one made of the shared page."""
    m, (h,) = make_pool([100], [28], layers=2, spare=6)
    scramble(m)
    before = logical(m, h, 128)
    child = m.fork(h)
    m.move_tokens([h], [[105]], [100])
    m.move_tokens([h], [[110, 120]], [101])
    want = [x.clone() for x in before]
    for x, old in zip(want, before):
        x[:, :, 100:103] = old[:, :, [105, 110, 120]]
    assert h.pages[0] != child.pages[0] and same(logical(m, h, 128), want)
    assert same(logical(m, child, 128), before)


def test_one_sequence_keeps_what_another_reads():
    """Two sequences over one shared page, in C: tokens that stay for one may be read for the
    other's moves, and both may read a token."""
    m, (h, g) = make_pool([128, 128], [0, 0], layers=2, kv_heads=3)
    scramble(m)
    a, b = logical(m, h, 128), logical(m, g, 128)
    arrays = [np.array(x, dtype=np.int32) for x in (
        [h.pages[0], g.pages[0], h.pages[0]], [0, 1, 3], [0, 0],
        [5, 6, 90, 129, 133, 134, 218], [0, 3, 7], [5, 10])]
    rc = _native.lib().hy_kv_move(
        m.k_cache.data_ptr(), m.v_cache.data_ptr(), m.k_cache.stride(0), m.k_cache.stride(2),
        m.num_pages, *(x.ctypes.data for x in arrays), 2, 2, 3, D, m.page_size, None)
    assert rc == _native.HY_OK, _native.last_error()
    torch.cuda.synchronize()
    # the first sequence: 5 and 6 stay, 90 goes to 7; the second, whose positions from 128 on
    # are the first one's page: its 1, 5, 6 and 90 to 10 .. 13
    want = [x.clone() for x in a], [x.clone() for x in b]
    for x, y, old in zip(*want, a):
        x[:, :, 7] = old[:, :, 90]
        y[:, :, 10:14] = old[:, :, [1, 5, 6, 90]]
    assert same(logical(m, h, 128), want[0]) and same(logical(m, g, 128), want[1])


def test_a_page_past_2_31_elements():
    """Pages of 2^25 tokens: a row's offset inside one passes 32 bits."""
    from hayate_amd import PagedKVCacheManager

    page = 1 << 25
    m = PagedKVCacheManager(1, 1, D, 2 * page, page, 2, torch.bfloat16, "cuda")
    h = m.allocate()
    m.claim_pages(h, [1])
    h.length = page
    rows = torch.tensor([0, 1, (1 << 24) - 1, 1 << 24, (1 << 24) + 5, page - 1], device="cuda")
    for p in (m.k_cache, m.v_cache):
        bits(p)[:, :, :, rows] = -1
        bits(p)[:, :, :, page + rows] = torch.arange(6 * D, device="cuda",
                                                     dtype=torch.int16).view(1, 1, 1, 6, D)
    child = m.fork(h, copy=True)
    assert child.pages == [0]
    for p in (m.k_cache, m.v_cache):
        assert torch.equal(bits(p)[:, :, :, rows], bits(p)[:, :, :, page + rows])
