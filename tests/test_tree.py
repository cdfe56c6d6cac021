"""Drafted trees, token moves and page copies without a GPU: the planner, the
metadata, the bookkeeping, and what is refused before any device work."""

import ctypes
import random

import numpy as np
import pytest
import torch

from hayate_amd import PagedKVCacheManager, PagedTreeBatch, _native
from tree_util import chain, depth, line, wide_tree


def pool(pages=12, page=128, layers=1, slots=6):
    return PagedKVCacheManager(layers, 8, 128, pages * page, page, slots, torch.bfloat16, "cpu",
                               num_q_heads=32)


def handle(m, length):
    h = m.allocate()
    m.reserve(h, length)
    h.length = length
    return h


# ----------------------------------------------------------------- planner
def check_plan(q_lens, kv_lens, hq=32, hkv=8, cus=256):
    """Every (tile, key step) of every request is in one piece of one chunk, pieces keep to the
    page table's range, and partials do not overlap."""
    q, kv = np.asarray(q_lens), np.asarray(kv_lens)
    p = _native.plan_tree(q, kv, hq, hkv, cus)
    group = hq // hkv
    chunks = p.items[: 2 * p.n_chunks].reshape(-1, 16)
    pieces = p.items[2 * p.n_chunks :]
    assert 1 <= p.n_chunks <= -(-cus // hkv)
    assert chunks[0, 0] == 0 and chunks[-1, 1] == len(pieces)
    assert (chunks[1:, 0] == chunks[:-1, 1]).all() and (chunks[:, 1] > chunks[:, 0]).all()
    steps = -(-(pieces[:, 4] - pieces[:, 3]) // 64)
    assert (steps > 0).all()
    for ch in chunks:
        assert ch[2] == steps[ch[0] : ch[1]].sum()
        assert (ch[8:] == pieces[ch[0]]).all()
        mine = pieces[ch[0] : ch[1]]
        assert ch[3] == (mine[:, 2] - mine[:, 1] == q[mine[:, 0]]).all()
    starts = np.concatenate([[0], np.cumsum(q)])
    at, used, merged, rows = 0, [], {}, 0
    for m in p.merge:
        merged[int(m[0]), int(m[1])] = m
    for b in range(len(q)):
        node = 0
        while node < q[b]:
            seq, q0, q1 = pieces[at, :3]
            assert seq == b and q0 == node and node < q1 <= q[b]
            assert (q1 - q0) * group <= 256
            rows = max(rows, (q1 - q0) * group)
            blocks = -(-int(q1 - q0) * group // 32)
            end, key, first = kv[b] - q[b] + q1, 0, at
            while key < end:
                r = pieces[at]
                assert tuple(r[:3]) == (seq, q0, q1) and r[3] == key and key < r[4] <= end
                assert r[3] % 64 == 0 and (r[4] % 64 == 0 or r[4] == end)
                assert r[6] == starts[b] and r[7] == kv[b] - q[b]
                key = r[4]
                at += 1
            if at == first + 1:
                assert pieces[first, 5] == -1 and (seq, q0) not in merged
            else:
                m = merged.pop((int(seq), int(q0)))
                assert m[2] == q1 and m[4] == at - first and m[5] == starts[b] and m[6] == blocks
                for i in range(first, at):
                    assert pieces[i, 5] == m[3] + (i - first) * blocks
                    used += range(pieces[i, 5], pieces[i, 5] + blocks)
            node = q1
    assert at == len(pieces) and not merged
    assert sorted(used) == list(range(p.n_slots)) and p.max_rows == rows
    # in key steps: the planner counts a piece after the chunk's first as 4, 3 in launches of
    # more than 128 rows
    cost = chunks[:, 2] + (4 if p.max_rows <= 128 else 3) * (chunks[:, 1] - chunks[:, 0] - 1)
    return p, cost


@pytest.mark.parametrize("seed", range(12))
def test_plan_covers_everything_once(seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 60))
    q = rng.integers(1, int(rng.choice([2, 30, 257])), size=n)
    kv = q + rng.integers(0, int(rng.choice([2, 500, 20000])), size=n)
    for hq, hkv in ((32, 8), (8, 8), (16, 1), (64, 4)):
        check_plan(q, kv, hq, hkv)


def test_plan_shares_the_steps_evenly():
    rng = np.random.default_rng(3)
    q = rng.integers(4, 20, size=20)
    _, cost = check_plan(q, q + rng.integers(200, 4000, size=20))
    assert len(cost) == 32 and cost.max() <= cost.mean() + 2
    _, cost = check_plan([64] * 8, [32064] * 8)
    # a chunk is closed when another piece would not pay: at most a piece's cost short
    assert len(cost) == 32 and cost.max() - cost.min() <= 3


def test_plan_of_small_work_and_few_units():
    p, _ = check_plan([1], [1])
    assert p.n_chunks == 1 and not len(p.merge) and p.n_slots == 0
    check_plan([256] * 3, [256] * 3, 128, 8)
    check_plan([5] * 300, [6] * 300)
    check_plan([5, 9], [500, 700], cus=1)
    check_plan([5, 9], [500, 700], 64, 64, cus=8)


def test_plan_refusals():
    def call(q, kv, hq=32, hkv=8, items=1000, merges=1000):
        q, kv = np.asarray(q, dtype=np.int32), np.asarray(kv, dtype=np.int32)
        a, b = np.zeros((items, 8), np.int32), np.zeros((merges, 8), np.int32)
        c = np.zeros(5, np.int32)
        return _native.lib().hy_plan_tree(q.ctypes.data, kv.ctypes.data, len(q), hq, hkv, 256,
                                          a.ctypes.data, items, b.ctypes.data, merges, c.ctypes.data)

    assert call([3], [10]) == _native.HY_OK
    assert call([0], [10]) == _native.HY_EINVAL
    assert call([11], [10]) == _native.HY_EINVAL
    assert call([257], [300]) == _native.HY_EUNSUPPORTED
    assert call([3], [10], hq=24) == _native.HY_EUNSUPPORTED
    assert call([3], [10], hq=30) == _native.HY_EINVAL
    assert call([3], [10000], items=4) == _native.HY_ENOSPACE
    assert call([3], [10000], merges=0) == _native.HY_ENOSPACE
    assert call([3], [2**31 - 128]) == _native.HY_EUNSUPPORTED


def test_lines_refusals():
    def call(parents, q_lens, words=4):
        p, q = np.array(parents, np.int32), np.array(q_lens, np.int32)
        lines, depths = np.zeros((len(p), 8), np.uint32), np.zeros(len(p), np.int32)
        return _native.lib().hy_tree_lines(p.ctypes.data, q.ctypes.data, len(q), words,
                                           lines.ctypes.data, depths.ctypes.data)

    assert call([-1, 0, 0], [3]) == _native.HY_OK
    assert call([-1, 0, -1, 0], [2, 2]) == _native.HY_OK
    for parents, q, words in (([-1, 1], [2], 4), ([0], [1], 4), ([-1, -2], [2], 4),
                              ([-1, 0, 1], [2, 1], 4), (chain(129), [129], 4), ([], [0], 4),
                              ([-1], [1], 3), ([-1], [1], 12)):
        assert call(parents, q, words) == _native.HY_EINVAL
    assert call(chain(256), [256], 8) == _native.HY_OK


# ---------------------------------------------------------------- metadata
@pytest.mark.parametrize("sizes", [[1], [3, 40], [256, 1, 33]])
def test_batch_metadata(sizes):
    rng = random.Random(sum(sizes))
    trees = [wide_tree(rng, n) for n in sizes]
    m = pool(pages=22)
    handles = [handle(m, rng.randint(1, 300)) for _ in sizes]
    batch = m.begin_tree(handles, trees)
    assert isinstance(batch, PagedTreeBatch) and batch.varlen and not batch.decode_only
    assert batch.every_logit and not m.begin_tick([handle(m, 5)], [1]).every_logit
    words = batch.line_words
    assert words == 4 * -(-max(sizes) // 128) and batch._lines_ptr % 16 == 0
    lines = batch.lines.numpy().view(np.uint32).reshape(-1, words)
    row = 0
    for h, tree in zip(handles, trees):
        assert len(h.pages) == -(-(h.length + len(tree)) // 128)
        for i in range(len(tree)):
            assert batch.positions[row] == h.length + depth(tree, i)
            got = [j for j in range(32 * words) if lines[row, j >> 5] >> (j & 31) & 1]
            assert got == line(tree, i)
            row += 1


def test_begin_tree_refusals_change_nothing():
    m = pool()
    a, b = handle(m, 100), handle(m, 20)
    free = m.free_page_count
    for trees in ([[-1]], [[-1], []], [[-1], [0]], [[-1], [-1, 1]], [[-1], [-1, -2]],
                  [[-1], chain(257)]):
        with pytest.raises(ValueError):
            m.begin_tree([a, b], trees)
    for trees in ([[-1], [-1.0]], [[-1], [None]], [[-1], [[-1]]], [[-1], "ab"], [[-1], [True]]):
        with pytest.raises(TypeError):
            m.begin_tree([a, b], trees)
    with pytest.raises(ValueError):
        m.begin_tree([a, a], [[-1], [-1]])
    with pytest.raises(ValueError):
        m.begin_tree([], [])
    m.release(b)
    with pytest.raises(RuntimeError):
        m.begin_tree([a, b], [[-1], [-1]])
    big = handle(m, m.free_page_count * 128)
    with pytest.raises(MemoryError):
        m.begin_tree([a, big], [chain(10), chain(10)])
    m.release(big)
    assert m.free_page_count == free + 1 and len(a.pages) == 1


def test_paths():
    m = pool()
    tree = [-1, 0, 0, 1, -1, 4]
    batch = m.begin_tree([handle(m, 5)], [tree])
    assert batch.check_path(0, []) == []
    assert batch.check_path(0, np.array([0, 1, 3])) == [0, 1, 3]
    assert batch.check_path(0, [4, 5]) == [4, 5]
    for bad in ([1], [0, 3], [0, 1, 2], [6], [-1], [0, 0]):
        with pytest.raises(ValueError):
            batch.check_path(0, bad)
    with pytest.raises(TypeError):
        batch.check_path(0, [0.0])


def test_commit_tree_without_moves_is_bookkeeping(monkeypatch):
    import hayate_amd.paged_cache as pc

    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    m = pool()
    a, b = handle(m, 100), handle(m, 250)
    batch = m.begin_tree([a, b], [chain(40), chain(10)])
    assert [len(h.pages) for h in (a, b)] == [2, 3]
    free = m.free_page_count
    with pytest.raises(ValueError):
        m.commit_tree([a], batch, [[0]])
    with pytest.raises(ValueError):
        m.commit_tree([a, b], batch, [[0], [1]])
    with pytest.raises(ValueError):
        m.commit_tree([b, a], batch, [[0], [0]])
    with pytest.raises(ValueError):
        pool().commit_tree([a, b], batch, [[0], [0]])
    assert (a.length, b.length) == (100, 250)
    m.commit_tree([a, b], batch, [[0, 1, 2], range(8)])
    assert (a.length, b.length) == (103, 258)
    assert [len(h.pages) for h in (a, b)] == [1, 3] and m.free_page_count == free + 1
    with pytest.raises(ValueError):  # committed already
        m.commit_tree([a, b], batch, [[0], [0]])


def test_commit_tree_takes_the_batch_s_handles(monkeypatch):
    """Handles of the same length in another order, or another handle of that length, would
    commit one request's path to another."""
    import hayate_amd.paged_cache as pc

    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    m = pool()
    a, b, other = (handle(m, 100) for _ in range(3))
    batch = m.begin_tree([a, b], [chain(3), chain(3)])
    for handles in ([b, a], [a, other], [a, a]):
        with pytest.raises(ValueError):
            m.commit_tree(handles, batch, [[0], [0]])
    m.commit_tree([a, b], batch, [[0], [0, 1]])
    assert (a.length, b.length) == (101, 102)


def test_a_tree_that_cannot_be_planned_reserves_nothing(monkeypatch):
    import hayate_amd.paged_cache as pc

    def refuse(self, *args):
        raise NotImplementedError

    m = pool()
    h = handle(m, 100)
    free, pages = m.free_page_count, list(h.pages)
    monkeypatch.setattr(pc.PagedTreeBatch, "__init__", refuse)
    with pytest.raises(NotImplementedError):
        m.begin_tree([h], [chain(200)])
    assert m.free_page_count == free and h.pages == pages


# ------------------------------------------------------------ moves, copies
def test_data_operations_need_a_gpu():
    m = pool()
    h = handle(m, 300)
    with pytest.raises(RuntimeError):
        m.move_tokens([h], [[5]], [1])
    with pytest.raises(RuntimeError):
        m.copy_pages([h.pages[0]], [h.pages[1]])
    with pytest.raises(RuntimeError):
        m.fork(h, copy=True)
    with pytest.raises(RuntimeError):
        m.compact(h, [3])
    assert h.length == 300 and len(h.pages) == 3 and m.free_page_count == 9


def test_move_and_copy_refusals(monkeypatch):
    import hayate_amd.paged_cache as pc

    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    m = pool()
    h, g = handle(m, 300), handle(m, 128)
    for src, start in (([5, 5], 0), ([5, 4], 0), ([5], 6), ([384], 0), ([-1], 0), ([3], -1),
                       ([2, 3], 3)):
        with pytest.raises(ValueError):
            m.move_tokens([h], [src], [start])
    for src, start in (([5.0], 0), ([[5]], 0), (["a"], 0), ([5], 0.5), ([5], True)):
        with pytest.raises(TypeError):
            m.move_tokens([h], [src], [start])
    with pytest.raises(ValueError):
        m.move_tokens([h, h], [[5], [6]], [0, 0])
    with pytest.raises(ValueError):
        m.move_tokens([h], [[5], [6]], [0])
    m.move_tokens([], [], [])
    m.move_tokens([h], [[]], [0])
    m.move_tokens([h], [[7, 8]], [7])
    for src, dst, n in (([0], [0, 1], None), ([99], [g.pages[0]], None), ([-1], [g.pages[0]], None),
                        ([h.pages[0]], [12], None), (h.pages[:1], g.pages, [129]),
                        (h.pages[:1], g.pages, [-1]), (h.pages[:1], g.pages, [1, 2]),
                        (h.pages[:1], [m._free_pages[-1]], None), ([m._free_pages[-1]], g.pages, None)):
        with pytest.raises(ValueError):
            m.copy_pages(src, dst, n)
    child = m.fork(h)
    with pytest.raises(ValueError):  # a shared page is not written
        m.copy_pages(g.pages, h.pages[:1])
    for keep in ([300], [-1], [4, 4], [5, 4]):
        with pytest.raises(ValueError):
            m.compact(h, keep)
    m.release(child)
    m.compact(h, range(130))
    assert h.length == 130 and len(h.pages) == 2
    m.release(g)
    for call in (lambda: m.move_tokens([g], [[1]], [0]), lambda: m.compact(g, []),
                 lambda: m.fork(g, copy=True)):
        with pytest.raises(RuntimeError):
            call()


def test_pools_of_other_rows(monkeypatch):
    """The copy-on-write of a pool whose rows the kernels do not move copies as before; moving
    tokens in one is refused."""
    import hayate_amd.paged_cache as pc

    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    for dtype, dim in ((torch.float32, 128), (torch.bfloat16, 64)):
        m = PagedKVCacheManager(2, 3, dim, 6 * 128, 128, 4, dtype, "cpu")
        m.k_cache.normal_()
        m.v_cache.normal_()
        h = handle(m, 200)
        child = m.fork(h)
        want = [p[:, :, :, 128 * h.pages[1] : 128 * h.pages[1] + 72].clone() for p in (m.k_cache, m.v_cache)]
        m.begin_batch([child], 1)
        assert child.pages[1] != h.pages[1]
        for p, x in zip((m.k_cache, m.v_cache), want):
            assert torch.equal(p[:, :, :, 128 * child.pages[1] : 128 * child.pages[1] + 72], x)
        with pytest.raises(NotImplementedError):
            m.move_tokens([h], [[5]], [3])


def c_arrays(*lists):
    return [(ctypes.c_int32 * max(1, len(x)))(*x) for x in lists]


def c_move(pages, src, first, page_start=None, src_start=None, first_page=None, **kw):
    """hy_kv_move on a pool of 8 pages of 128 that is never touched."""
    n = len(first)
    args = c_arrays(pages, page_start or [0, len(pages)], first_page or [0] * n, src,
                    src_start or [0, len(src)], first)
    args = {**dict(k=4096, v=4096, ls=8 * 1024 * 128, hs=1024 * 128, num_pages=8),
            **dict(zip(("p_pages", "p_start", "p_first", "p_src", "p_ss", "p_to"), args)),
            **dict(n=n, layers=2, heads=8, dim=128, page=128, stream=None), **kw}
    return _native.lib().hy_kv_move(*args.values())


def test_c_moves_are_checked_before_any_launch():
    bad = [
        ([0, 1], [5, 5], [0]), ([0, 1], [6, 5], [0]), ([0, 1], [3], [4]), ([0, 1], [256], [0]),
        ([0, 1], [-1], [-2]), ([0, 8], [200], [0]), ([0, -1], [200], [0]), ([], [1], [0]),
    ]
    for pages, src, first in bad:
        assert c_move(pages, src, first) == _native.HY_EINVAL, (pages, src, first)
        assert _native.last_error()
    # one page twice: position 128 is position 0, which the first of these moves wrote
    assert c_move([0, 0], [2, 128], [0]) == _native.HY_EINVAL
    # two sequences that write one page, or one that reads what the other wrote
    two = dict(page_start=[0, 1, 2], src_start=[0, 1, 2])
    assert c_move([3, 3], [5, 5], [1, 1], **two) == _native.HY_EINVAL
    assert c_move([3, 3], [5, 1], [1, 0], **two) == _native.HY_EINVAL
    assert c_move([3, 4], [5, 5], [1, 1], page_start=[0, 1, 0], src_start=[0, 1, 2]) == _native.HY_EINVAL
    assert c_move([3, 4], [5, 5], [1, 1], page_start=[0, 1, 2], src_start=[0, 2, 1]) == _native.HY_EINVAL
    # positions count from the first page given
    assert c_move([3], [5], [1], first_page=[1]) == _native.HY_EINVAL
    assert c_move([3], [5], [1], first_page=[-1]) == _native.HY_EINVAL
    # tokens that stay need no launch
    assert c_move([0, 1], [7, 8, 130][:2], [7]) == _native.HY_OK
    assert c_move([3], [130, 131], [130], first_page=[1]) == _native.HY_OK
    assert c_move([], [], []) == _native.HY_OK


def test_c_pools_are_checked():
    for kw in (dict(k=None), dict(v=None), dict(k=4098), dict(ls=1024 * 128), dict(hs=128),
               dict(hs=1024 * 128 + 4), dict(num_pages=0), dict(num_pages=1 << 24), dict(p_pages=None),
               dict(p_start=None), dict(p_first=None), dict(p_src=None), dict(p_ss=None), dict(p_to=None),
               dict(n=-1), dict(layers=0), dict(heads=0), dict(page=0), dict(layers=1 << 23)):
        assert c_move([0, 1], [5], [3], **kw) == _native.HY_EINVAL, kw
    assert c_move([0, 1], [5], [3], dim=64) == _native.HY_EUNSUPPORTED


@pytest.mark.parametrize("src,dst,tokens", [([0, 1], [2, 2], None), ([0, 1], [1, 2], None),
                                            ([3], [3], None), ([-1], [0], None), ([0], [8], None),
                                            ([0], [1], [129]), ([0], [1], [-1])])
def test_c_copies_are_checked_before_any_launch(src, dst, tokens):
    lib = _native.lib()
    a, b, t = c_arrays(src, dst, tokens or [])
    assert lib.hy_page_copy(4096, 4096, 8 * 1024 * 128, 1024 * 128, 8, a, b, t if tokens else None,
                            len(src), 2, 8, 128, 128, None) == _native.HY_EINVAL
    assert _native.last_error()


def test_c_tree_attention_is_checked():
    lib = _native.lib()
    good = dict(q=4096, qs=0, qt=4096, qh=128, out=4096, os=0, ot=4096, oh=128, k=4096, v=4096,
                hs=128 * 1000, pt=4096, pts=4, lines=4096, words=4, items=4096, chunks=1, rows=32,
                merge=None, merges=0, slots=0, ws=None, wsb=0, hq=32, hkv=8, dim=128, page=128,
                scale=0.1, stream=None)

    def call(**kw):
        args = {**good, **kw}
        return lib.hy_paged_tree(*args.values())

    for kw in (dict(scale=0.0), dict(scale=float("nan")), dict(hq=30), dict(chunks=-1),
               dict(chunks=65536), dict(rows=0), dict(rows=257), dict(words=0), dict(words=5), dict(words=12),
               dict(q=None), dict(out=None), dict(k=None), dict(v=None), dict(pt=None),
               dict(lines=None), dict(items=None), dict(merges=1, slots=2, ws=4096, wsb=1 << 30),
               dict(merge=4096, merges=1),
               dict(q=4098), dict(lines=4100), dict(qh=100), dict(ot=4), dict(hs=1001)):
        assert call(**kw) == _native.HY_EINVAL, kw
    for kw in (dict(dim=64), dict(page=96), dict(page=16), dict(hq=24), dict(hq=256)):
        assert call(**kw) == _native.HY_EUNSUPPORTED, kw
    assert call(slots=2) == _native.HY_ENOSPACE
    assert call(chunks=0) == _native.HY_OK
    assert lib.hy_tree_workspace_bytes(0, 8, 128) == 0
    assert lib.hy_tree_workspace_bytes(3, 8, 128) == 3 * 8 * 32 * (128 + 2) * 4

def test_moves_into_a_shared_page_keep_what_is_reserved_in_it(monkeypatch):
    """Drafted tokens sit past the handle's length. A move that gives the handle its own copy of
    a page takes all of them over: a later move may still read them."""
    import hayate_amd.paged_cache as pc

    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    m = pool()
    h = handle(m, 100)
    m.begin_tree([h], [chain(20)])
    m.fork(h)
    copied = []
    monkeypatch.setattr(m, "_copy_pages", lambda src, dst, tokens: copied.append(list(tokens)))
    monkeypatch.setattr(pc._native, "lib", lambda: type("", (), {"hy_kv_move": lambda *a: 0}))
    m.move_tokens([h], [[105]], [100])
    assert copied == [[128]]

@pytest.mark.parametrize("make", [lambda x: np.array(x, dtype=np.int64), torch.tensor,
                                  lambda x: np.array(x, dtype=np.int32)])
def test_a_batch_keeps_its_own_trees(make):
    """A caller may write the next tick's parents into the same arrays."""
    m = pool()
    h = handle(m, 5)
    tree = make([-1, 0, 1, 0])
    batch = m.begin_tree([h], [tree])
    tree[:] = -1
    assert batch.check_path(0, [0, 1, 2]) == [0, 1, 2]
    with pytest.raises(ValueError):
        batch.check_path(0, [2])
    tree = make([-1, 0, 1, 0])
    batch = PagedTreeBatch(m, [tree], [5], [list(h.pages)], None)
    tree[:] = -1
    assert batch.check_path(0, [0, 1, 2]) == [0, 1, 2]


def test_c_moves_of_sequences_that_share_a_page():
    """A position that a sequence fills, by a move or by a token that stays, is written for no
    other one, and a written token is read for no other one, in whichever order they come."""
    two = dict(page_start=[0, 1, 2], src_start=[0, 1, 2])
    for moves in (((5, 1), (9, 5)),    # the second writes what the first read
                  ((9, 5), (5, 1)),    # the first writes what the second reads
                  ((5, 5), (9, 5)),    # ... or what stays for the first
                  ((9, 5), (5, 5)),
                  ((9, 5), (9, 5))):   # both write it
        src, first = [m[0] for m in moves], [m[1] for m in moves]
        assert c_move([3, 3], src, first, **two) == _native.HY_EINVAL, moves
        assert "share" in _native.last_error()
    # read for two others, then written for itself
    assert c_move([3, 3, 3], [5, 5, 9], [1, 2, 5], page_start=[0, 1, 2, 3],
                  src_start=[0, 1, 2, 3]) == _native.HY_EINVAL
    # both read it, and the second, which reads it in front of the token that it fills it with
    assert c_move([3, 3], [5, 5, 6, 7, 8], [1, 2], page_start=[0, 1, 2],
                  src_start=[0, 1, 5]) == _native.HY_EINVAL
    # one page twice in a sequence: position 130 is position 2, which stays
    assert c_move([0, 0], [*range(2, 130), 140], [2]) == _native.HY_EINVAL
    # a shared page whose tokens stay for both
    assert c_move([3, 3], [5, 6, 5, 6, 7], [5, 5], page_start=[0, 1, 2],
                  src_start=[0, 2, 5]) == _native.HY_OK


def test_c_moves_begin_inside_their_arrays():
    for kw in (dict(page_start=[-1, 1]), dict(src_start=[-2, 1])):
        assert c_move([3], [5], [1], **kw) == _native.HY_EINVAL
        assert "negative" in _native.last_error()


def test_a_tree_on_small_pages_reserves_nothing():
    """Pages below what ticks take are refused before any is reserved."""
    m = PagedKVCacheManager(1, 8, 128, 12 * 64, 64, 2, torch.bfloat16, "cpu", num_q_heads=32)
    h = m.allocate()
    m.reserve(h, 60)
    h.length = 60
    free = list(m._free_pages)
    with pytest.raises(ValueError):
        m.begin_tree([h], [chain(100)])
    assert m._free_pages == free and len(h.pages) == 1


def test_pages_of_a_refused_tree_return_in_their_order(monkeypatch):
    import hayate_amd.paged_cache as pc

    m = pool()
    handles = [handle(m, 100), handle(m, 100)]
    free = list(m._free_pages)
    monkeypatch.setattr(pc.PagedTreeBatch, "__init__", lambda *args: 1 // 0)
    with pytest.raises(ZeroDivisionError):
        m.begin_tree(handles, [chain(200), chain(200)])
    assert m._free_pages == free


def test_a_batch_is_committed_once(monkeypatch):
    """Also where nothing was accepted: the slots may hold the next tick's tokens by then."""
    import hayate_amd.paged_cache as pc

    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    m = pool()
    h = handle(m, 100)
    batch = m.begin_tree([h], [chain(3)])
    with pytest.raises(ValueError):
        m.commit_tree([h], batch, [[1]])
    m.commit_tree([h], batch, [[]])
    other = m.begin_tree([h], [chain(3)])
    with pytest.raises(ValueError):
        m.commit_tree([h], batch, [[0]])
    m.commit_tree([h], other, [[0]])
    assert h.length == 101
