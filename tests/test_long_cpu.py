"""Host side of windowed and weighed attention, without a GPU: the planners' lists against the
definition, token by token, and the refusals of the entry points."""

import numpy as np
import pytest
import torch

from hayate_amd import PagedKVCacheManager, _native


def keys_of(first_pos, window, sinks, unit):
    """(ns, gap) of a range of rows from first_pos on, from the definition."""
    low = max(0, first_pos - window + 1)
    ns = -(-sinks // unit) * unit
    gap = max(0, low // unit * unit - ns)
    return ns, gap


def in_sight(pos, window, sinks):
    return {j for j in range(pos + 1) if pos - j < window or j < sinks}


CASES = [(1, 0), (1, 5), (33, 1), (64, 64), (100, 31), (500, 4), (10_000, 0), (2**31 - 1, 3),
         (7, 2**30)]


@pytest.mark.parametrize("window,sinks", CASES)
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8), (16, 1)])
def test_every_key_in_sight_is_planned_once(window, sinks, hq, hkv):
    rng = np.random.default_rng(window % 1000 + sinks % 1000)
    q = np.array([1, 1, 1, 1, 2, 70, 130, 1, 33, 1], dtype=np.int32)
    kv = q + np.concatenate([[0, 30, 31, 1500], rng.integers(0, 900, 6)]).astype(np.int32)
    plan = _native.plan_tick(q, kv, hq, hkv, 128, 256, 0, window, sinks)
    pieces = plan.decode[plan.n_chunks :]
    for b in np.flatnonzero(q == 1):
        ns, gap = keys_of(kv[b] - 1, window, sinks, 32)
        of = pieces[pieces[:, 0] == b]
        numbers = [x for p in of for x in range(p[1], p[2])]
        assert numbers == list(range(kv[b] - gap))  # in order, without a hole
        keys = [x if x < ns else x + gap for x in numbers]
        sight = in_sight(kv[b] - 1, window, sinks)
        assert sight <= set(keys)
        assert max(keys) == kv[b] - 1 and len(set(keys)) == len(keys)
        # a slice of 32 without a key in sight would leave a wave without a maximum
        for p in of:
            for x in range(p[1], p[2], 32):
                assert sight & {y if y < ns else y + gap for y in range(x, min(x + 32, p[2]))}
        assert of[-1][7] == 1 and not of[:-1, 7].any() and (of[:, 6] == kv[b] - 1).all()
    for b in np.flatnonzero(q > 1):
        cache = kv[b] - q[b]
        of = plan.prefill[plan.prefill[:, 0] == b]
        for q0, q1 in {(x[1], x[2]) for x in of.tolist()}:
            ns, gap = keys_of(cache + q0, window, sinks, 32)
            ranges = sorted((x[3], x[4]) for x in of.tolist() if x[1] == q0)
            assert ranges[0][0] == 0 and ranges[-1][1] == cache + q1 - gap
            assert all(a[1] == z[0] and z[0] % 64 == 0 for a, z in zip(ranges, ranges[1:]))
            sight = set().union(*(in_sight(cache + t, window, sinks) for t in range(q0, q1)))
            keys = {x if x < ns else x + gap for x in range(cache + q1 - gap)}
            assert sight <= keys and max(keys) == cache + q1 - 1
        tokens = sorted({t for x in of for t in range(x[1], x[2])})
        assert tokens == list(range(q[b]))


def test_a_plan_without_a_window_is_the_plan_of_a_wide_one():
    q, kv = np.array([1, 40, 1, 300]), np.array([700, 900, 1, 300])
    a = _native.plan_tick(q, kv, 32, 8, 128, 256)
    b = _native.plan_tick(q, kv, 32, 8, 128, 256, 0, 1000, 0)
    for name in ("decode", "merge", "prefill", "prefill_merge"):
        assert np.array_equal(getattr(a, name), getattr(b, name))


@pytest.mark.parametrize("window,sinks", [(0, 0), (-1, 0), (1, -1), (1, 2**30 + 1)])
def test_the_planner_refuses(window, sinks):
    with pytest.raises(ValueError):
        _native.plan_tick(np.array([1]), np.array([5]), 32, 8, 128, 256, 0, window, sinks)


@pytest.mark.parametrize("hq,hkv,cus", [(32, 8, 256), (8, 8, 4), (16, 1, 256), (1, 1, 1)])
def test_weigh_lists_cover_every_pair_once(hq, hkv, cus):
    rng = np.random.default_rng(hq + cus)
    q = np.array([1, 2, 300, 1, 512, 17, 1], dtype=np.int32)
    kv = q + rng.integers(0, 900, len(q)).astype(np.int32)
    rows = np.array([4, 0, 2, 9, 1, 3, 7], dtype=np.int32)
    merge = _native.plan_tick(q, kv, hq, hkv, 128, cus).merge
    p = _native.plan_weigh(q, kv, rows, hq, hkv, cus, merge)
    start = np.cumsum(q) - q
    taken = np.zeros(p.scores, dtype=bool)
    for b in range(len(q)):
        adds = p.adds[p.adds[:, 0] == rows[b]]
        assert [t for a in adds for t in range(a[1], a[2])] == list(range(kv[b]))
        assert (adds[:, 2] - adds[:, 1] <= 256).all() and (adds[:, 1] % 256 == 0).all()
        if q[b] == 1:
            slots = merge[merge[:, 0] == b][0]
            assert (adds[:, 3] == slots[2]).all() and (adds[:, 4] == slots[1]).all()
            assert (adds[:, 5] == 1).all() and (adds[:, 6] == p.score_start[b]).all()
            assert p.score_start[b] % 4 == 0
            # whole slices of 32 scores, none of another sequence's
            room = slice(p.score_start[b], p.score_start[b] + -(-kv[b] // 32) * 32)
            assert room.stop <= p.scores and not taken[room].any()
            taken[room] = True
            continue
        cache = kv[b] - q[b]
        items = p.items[p.items[:, 0] == b]
        assert (items[:, 5] == start[b]).all() and (items[:, 6] == cache).all()
        assert len({x for x in items[:, 7]}) == 1 and (adds[:, 6] == items[0, 7]).all()
        for a in adds:
            of = items[items[:, 1] == a[1]]
            of = of[np.argsort(of[:, 4])]
            # the parts that the addition reads, and each of them written
            assert a[4] == of[0, 4] * hkv and a[3] == len(of) * hkv and a[5] == 0
            assert [x for x in of[:, 4]] == list(range(of[0, 4], of[0, 4] + len(of)))
            assert of[-1, 4] < p.parts and of[0, 7] + a[1] + 256 <= p.partials
            tokens = [t for x in of for t in range(x[2], x[3])]
            assert tokens == list(range(tokens[0], q[b]))
            # tokens before them see none of the block's keys
            assert tokens[0] == 0 or cache + tokens[0] - 1 < a[1]


def manager(**kw):
    return PagedKVCacheManager(2, 8, 128, 1024, 128, 4, torch.bfloat16, "cpu", num_q_heads=32, **kw)


def test_refusals_of_a_tick():
    m = manager()
    h = m.allocate()
    good = torch.zeros(4, 200)
    for kw, error in [
        ({"window": 0}, ValueError), ({"window": -3}, ValueError), ({"window": 2.0}, TypeError),
        ({"window": True}, TypeError), ({"window": 5, "sinks": -1}, ValueError),
        ({"window": 5, "sinks": 1.5}, TypeError), ({"sinks": 4}, ValueError),
        ({"window": 5, "weights": good}, NotImplementedError),
        ({"weights": good.double()}, TypeError), ({"weights": [[0.0]]}, TypeError),
        ({"weights": torch.zeros(200)}, ValueError), ({"weights": torch.zeros(0, 200)}, ValueError),
        ({"weights": torch.zeros(4, 2)}, ValueError),
        ({"weights": torch.zeros(200, 4).T}, ValueError),
        ({"weights": torch.zeros(1, 200).expand(4, 200)}, ValueError),
        ({"weights": torch.zeros(4, 200, requires_grad=True)}, ValueError),
    ]:
        for begin in (lambda: m.begin_tick([h], [3], **kw), lambda: m.begin_batch([h], 3, **kw)):
            with pytest.raises(error):
                begin()
        assert not h.pages, kw  # nothing is reserved for a refused tick
    for _ in range(2):
        other = m.allocate()
    with pytest.raises(ValueError, match="slot"):
        m.begin_tick([other], [1], weights=torch.zeros(2, 200))
    m16 = PagedKVCacheManager(1, 8, 128, 256, 128, 1, torch.float16, "cpu", num_q_heads=32)
    with pytest.raises(TypeError):
        m16.begin_tick([m16.allocate()], [1], weights=good)
    m16 = PagedKVCacheManager(1, 8, 128, 256, 128, 1, torch.float16, "cpu", num_q_heads=32)
    with pytest.raises(TypeError, match="window"):
        m16.begin_tick([m16.allocate()], [1], window=9)


def test_a_tick_with_a_form_of_its_own():
    m = manager()
    h = m.allocate()
    batch = m.begin_tick([h], [3], window=7, sinks=2)
    assert (batch.window, batch.sinks, batch.weights) == (7, 2, None)
    batch = m.begin_batch([h], 3, window=10**12)
    assert batch.window == m.capacity_tokens
    weights = torch.zeros(4, 200)
    assert m.begin_tick([h], [1], weights=weights).weights is weights
    batch = m.begin_tick([h], [1])
    assert batch.window is None and batch.weights is None
    with pytest.raises(NotImplementedError):
        m.begin_tick([h], [1], window=3).decode_layer(0, *[None] * 8, no_alloc=True)


# Pointers that no entry may follow: every call below is refused before anything is enqueued.
AT = 1 << 20


def _tick_args(**kw):
    a = dict(q=AT, q_seq=0, q_tok=4096, q_head=128, out=AT, o_seq=0, o_tok=4096, o_head=128, k=AT, v=AT,
             pool_head=128 * 256, table=AT, table_stride=2, q_start=AT, kv_lens=AT, decode=AT,
             n_decode=1, merge=AT, n_merge=1, n_slots=2, ws=AT, ws_bytes=1 << 30, prefill=AT,
             n_prefill=1, prefill_merge=AT, n_prefill_merge=0, n_prefill_slots=0, prefill_ws=AT,
             prefill_ws_bytes=1 << 30, num_seqs=2, hq=32, hkv=8, head_dim=128, page=128)
    assert not set(kw) - set(a)
    return list({**a, **kw}.values())


EINVAL, EUNSUPPORTED, ENOSPACE = -1, -3, -4


@pytest.mark.parametrize("kw,tail,code", [
    ({}, (0, 0, 0.1), EINVAL), ({}, (5, -1, 0.1), EINVAL), ({}, (5, 2**30 + 1, 0.1), EINVAL),
    ({}, (5, 0, 0.0), EINVAL), ({"n_merge": 0}, (5, 0, 0.1), EINVAL),
    ({"n_decode": 0}, (5, 0, 0.1), EINVAL), ({"n_decode": -1}, (5, 0, 0.1), EINVAL),
    ({"n_decode": 0, "n_merge": 0, "n_prefill": 0, "n_prefill_merge": 1}, (5, 0, 0.1), EINVAL),
    ({"q": None}, (5, 0, 0.1), EINVAL), ({"hq": 30}, (5, 0, 0.1), EINVAL),
    ({"head_dim": 64}, (5, 0, 0.1), EUNSUPPORTED), ({"hq": 24}, (5, 0, 0.1), EUNSUPPORTED),
    ({"ws_bytes": 100}, (5, 0, 0.1), ENOSPACE),
])
def test_the_windowed_entry_refuses(kw, tail, code):
    assert _native.lib().hy_paged_window(*_tick_args(**kw), *tail, None) == code
    assert _native.lib().hy_last_error()


@pytest.mark.parametrize("kw,weigh,code", [
    ({}, {"n_weigh": -1}, EINVAL), ({}, {"n_weigh": 65536}, EINVAL), ({}, {"n_add": -1}, EINVAL),
    ({}, {"scores": None}, EINVAL), ({}, {"score_start": None}, EINVAL),
    ({}, {"scores": AT + 4}, EINVAL), ({}, {"score_stride": 30}, EINVAL),
    ({}, {"partials": None}, EINVAL), ({}, {"partials": AT + 8}, EINVAL),
    ({}, {"partial_stride": 30}, EINVAL), ({}, {"row_ml": None}, EINVAL), ({}, {"row_ml": AT + 4}, EINVAL),
    ({}, {"weights": None}, EINVAL), ({}, {"adds": None}, EINVAL), ({}, {"items": None}, EINVAL),
    ({"q": AT + 2}, {}, EINVAL), ({"q_tok": 4095}, {}, EINVAL), ({"n_merge": 0}, {}, EINVAL),
    ({"hq": 2048, "hkv": 128}, {}, EUNSUPPORTED), ({"head_dim": 64}, {}, EUNSUPPORTED),
])
def test_the_weighing_entry_refuses(kw, weigh, code):
    tail = dict(items=AT, n_weigh=1, adds=AT, n_add=1, score_start=AT, scores=AT, score_stride=64,
                partials=AT, partial_stride=256, row_ml=AT, weights=AT, weights_stride=100, scale=0.1)
    assert not set(weigh) - set(tail)
    tail = {**tail, **weigh}.values()
    assert _native.lib().hy_paged_weigh(*_tick_args(**kw), *tail, None) == code
    assert _native.lib().hy_last_error()


@pytest.mark.parametrize("kw", [
    {"n": -1}, {"budget": 0}, {"sinks": -1}, {"recent": -1}, {"sinks": 8}, {"sinks": 4, "recent": 4},
    {"weights": None}, {"out": None}, {"rows": None}, {"lens": None}, {"row": -1}, {"len": -1},
    {"len": 2**30 + 1},
])
def test_the_keeping_entry_refuses(kw):
    a = dict(weights=AT, n=2, budget=7, sinks=1, recent=2, out=AT, row=0, len=9, rows=0, lens=0)
    a = {**a, **kw}
    rows, lens = np.array([0, a["row"]], dtype=np.int32), np.array([3, a["len"]], dtype=np.int32)
    rc = _native.lib().hy_keep_positions(
        a["weights"], 100, None if a["rows"] is None else rows.ctypes.data,
        None if a["lens"] is None else lens.ctypes.data, a["n"], a["budget"], a["sinks"], a["recent"],
        a["out"], None)
    assert rc == EINVAL and _native.lib().hy_last_error()


@pytest.mark.parametrize("kw,code", [
    ({"dtype": 2}, EINVAL), ({"vocab": 0}, EINVAL), ({"levels": 0}, EINVAL), ({"n": -1}, EINVAL),
    ({"vocab": 2**23}, EUNSUPPORTED), ({"logits": None}, EINVAL), ({"valid": None}, EINVAL),
    ({"q_len": 0}, EINVAL), ({"q_len": 257}, EINVAL), ({"temperature": -1.0}, EUNSUPPORTED),
    ({"temperature": float("nan")}, EUNSUPPORTED), ({"temperature": 1e31}, EUNSUPPORTED),
    ({"top_k": 0}, EINVAL), ({"top_p": 0.0}, EINVAL), ({"ws_bytes": -1}, ENOSPACE),
])
def test_the_verifying_entry_refuses(kw, code):
    lib = _native.lib()
    a = dict(logits=AT, dtype=0, vocab=1000, levels=3, n=2, valid=AT, q_len=4, temperature=1.0,
             top_k=5, top_p=0.5, ws_bytes=0)
    a = {**a, **kw}
    need = lib.hy_verify_workspace_bytes(3 + a["q_len"], 2, a["vocab"])
    ints = lambda x: np.array([3, x], dtype=np.int32)  # noqa: E731
    q_lens, top_k = ints(a["q_len"]), ints(a["top_k"])
    temperature, top_p = (np.array([1, a[x]], dtype=np.float32) for x in ("temperature", "top_p"))
    rc = lib.hy_verify_tree(
        a["logits"], 1000, a["dtype"], a["vocab"], AT, AT, q_lens.ctypes.data, a["n"],
        temperature.ctypes.data, top_k.ctypes.data, top_p.ctypes.data, AT, None, 0, AT, a["levels"], AT,
        AT, a["valid"], AT, need + a["ws_bytes"], None)
    assert rc == code and lib.hy_last_error()
