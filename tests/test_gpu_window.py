"""Attention with a sliding window and sinks (csrc/decode.hip, csrc/prefill.hip with kWindow)
against its definition in 64 bits, and its own rules: what a row does not see never reaches
it, and the calls agree with each other."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from long_util import D, DEV, Requests, assert_close, normal


def check(r, window, sinks, scale=None, what=""):
    batch = r.m.begin_tick(r.handles, r.fresh, window=window, sinks=sinks)
    out = batch.attend_layer(r.q, 0, scale)
    expected, bound, _ = r.expected(window, sinks, scale=scale)
    assert_close(out, expected, bound, what)
    return out


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (31, 0), (32, 4), (33, 33),
                                          (64, 64), (100, 5), (128, 1), (1000, 96), (5000, 4),
                                          (200, 100_000), (2**31 - 1, 0)])
def test_decode_lengths_around_the_window_and_slices(window, sinks):
    edge = min(window, 1500)
    cached = [0, 1, 30, 31, 32, 63, 64, 127, 128, 129, edge - 1, edge, edge + 1, edge + 31,
              edge + 32, edge + 64 + min(sinks, 100), 2 * edge + 200, 3001]
    r = Requests(cached, [1] * len(cached), seed=window % 97 + sinks % 89)
    check(r, window, sinks, what=f"decode {window}/{sinks}")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (40, 0), (63, 4), (64, 64), (65, 65),
                                          (130, 3), (257, 200), (900, 4), (10_000, 4)])
def test_chunks_around_the_window_and_tiles(window, sinks):
    cached = [0, 0, 1, 63, 64, 200, 511, 1500, 2111]
    fresh = [2, 300, 64, 65, 129, 7, 512, 33, 200]
    r = Requests(cached, fresh, seed=window + sinks)
    check(r, window, sinks, what=f"chunks {window}/{sinks}")


@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 8), (64, 8), (32, 2), (1, 1), (4, 4)])
@pytest.mark.parametrize("page", [128, 256])
def test_head_groups_and_pages(hq, hkv, page):
    r = Requests([700, 0, 1234, 40, 3000], [1, 150, 77, 1, 513], hq=hq, hkv=hkv, page=page, seed=hq)
    check(r, 301, 5, what=f"{hq}/{hkv} page {page}")


def test_split_tiles_join():
    """Few rows over a wide window: the planner cuts the keys, and rows of a part may see none
    of it."""
    r = Requests([12_000, 9000], [100, 3], seed=5)
    check(r, 6000, 70, what="wide window")
    r = Requests([9000], [64], seed=6)
    check(r, 6, 4000, what="many sinks, narrow window")


@pytest.mark.parametrize("seed", range(6))
def test_random_mixed_ticks(seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    n = pick(1, 24)
    fresh = [1 if pick(0, 2) else pick(2, 200) for _ in range(n)]
    r = Requests([pick(0, 2500) for _ in range(n)], fresh, seed=seed)
    check(r, pick(1, 1200), pick(0, 150), what=f"seed {seed}")


def test_scale_and_tokens_per_split():
    r = Requests([900, 2000, 10], [1, 1, 1], seed=2)
    r.m.tokens_per_split = 96
    check(r, 500, 10, scale=0.3, what="scale")


@pytest.mark.parametrize("fresh", [1, 70])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), 3e38])
def test_unseen_keys_do_not_reach_a_row(fresh, value):
    """K and V of slots that a row does not see, in its slices and tiles or not, may hold
    anything: the rows are those of a cache that holds zeros there, bit for bit."""
    cached, window, sinks = [700, 333, 1500], 150, 5
    r = Requests(cached, [fresh] * 3, seed=4)
    outs = []
    for fill in (0.0, value):
        for b, c in enumerate(cached):
            rows = r.rows(b)[sinks : c - window + 1]  # seen by no row of this tick
            r.m.k_cache[0, 0][:, rows] = fill
            r.m.v_cache[0, 0][:, rows] = fill
        batch = r.m.begin_tick(r.handles, r.fresh, window=window, sinks=sinks)
        outs.append(batch.attend_layer(r.q, 0))
    assert torch.equal(*outs)
    assert outs[0].isfinite().all()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("hq", [32, 8])
def test_values_that_some_rows_of_a_chunk_see(value, hq):
    """An infinite or NaN V reaches the rows whose window holds it (on the window's lower edge,
    among the chunk's own tokens, or next to the sinks) and no other."""
    c, n, window, sinks = 400, 140, 130, 7
    r = Requests([c], [n], hq=hq, seed=9)
    slots = {3: 17, 6: 3, 7: 5, c - 100: 40, c - 1: 0, c + 60: 127, c + n - 1: 64}
    rows = r.rows(0)
    clean, bound, _ = r.expected(window, sinks)
    for slot, dim in slots.items():
        r.m.v_cache[0, 0][:, rows[slot], dim] = value
    out = r.m.begin_tick(r.handles, r.fresh, window=window, sinks=sinks).attend_layer(r.q, 0).double()
    i = torch.arange(c, c + n, device=DEV)
    hit = torch.zeros(n, D, dtype=torch.bool, device=DEV)
    for slot, dim in slots.items():
        hit[:, dim] |= (i >= slot) & ((slot < sinks) | (i - slot < window))
    hit = hit[:, None].expand(n, hq, D)
    assert torch.equal(hit, ~out.isfinite())
    if value == value:
        assert (out[hit] == value).all()
    else:
        assert out[hit].isnan().all()
    assert_close(out[~hit], clean[~hit], bound[~hit], "others")


def test_both_infinities_make_nan():
    r = Requests([100], [40], seed=3)
    rows = r.rows(0)
    r.m.v_cache[0, 0][:, rows[90], 8] = float("inf")
    r.m.v_cache[0, 0][:, rows[95], 8] = float("-inf")
    out = r.m.begin_tick(r.handles, r.fresh, window=20, sinks=0).attend_layer(r.q, 0)
    # (token i sits in slot 100 + i and sees slots 81 + i .. 100 + i)
    assert out[:10, :, 8].isnan().all()
    assert (out[10:15, :, 8] == float("-inf")).all()
    assert out[15:].isfinite().all()


def test_uniform_batches_and_strided_rows():
    r = Requests([600, 90, 1400], [5, 5, 5], seed=8)
    batch = r.m.begin_batch(r.handles, 5, window=200, sinks=4)
    wide = normal(r.g, 3, 5, r.hq + 16, D)
    q = wide[:, :, 8 : 8 + r.hq]  # (B, T, H, D) rows inside a projection
    out = batch.attend_layer(q.transpose(1, 2), 0).transpose(1, 2).reshape(15, r.hq, D)
    expected, bound, _ = r.expected(200, 4, q=q.reshape(15, r.hq, D))
    assert_close(out, expected, bound, "uniform")
    one = Requests([600, 90, 1400], [1, 1, 1], seed=8)
    batch = one.m.begin_batch(one.handles, 1, window=200, sinks=4)
    out = batch.attend_layer(one.q.view(3, 1, -1, D).transpose(1, 2), 0)
    expected, bound, _ = one.expected(200, 4)
    assert_close(out.reshape(3, -1, D), expected, bound, "uniform decode")


def _tables(n):
    freq = 1e6 ** (-torch.arange(0, D, 2, device=DEV) / D)
    angle = torch.arange(n, device=DEV)[:, None] * freq
    angle = torch.cat([angle, angle], 1)
    return torch.cos(angle), torch.sin(angle)


@pytest.mark.parametrize("varlen", [True, False])
def test_fused_decode_equals_the_two_calls(varlen):
    """decode_layer with a window: the same bits as norm_rope_write_layer then attend_layer, the
    pool's included."""
    cached = [0, 5, 31, 32, 500, 511, 512, 1500, 2047]
    cos, sin = _tables(4096)
    results = []
    for fused in (True, False):
        r = Requests(cached, [1] * len(cached), seed=12)
        qkv = normal(r.g, len(cached), r.hq + 2 * r.hkv, D)
        qw, kw = normal(r.g, D), normal(r.g, D)
        if varlen:
            batch = r.m.begin_tick(r.handles, r.fresh, window=300, sinks=40)
        else:
            batch = r.m.begin_batch(r.handles, 1, window=300, sinks=40)
            qkv = qkv[:, None]
        q, k, v = qkv.split([r.hq, r.hkv, r.hkv], -2)
        if fused:
            rot, out = batch.decode_layer(0, q, k, v, qw, kw, 1e-6, cos, sin)
        else:
            rot = batch.norm_rope_write_layer(0, q, k, v, qw, kw, 1e-6, cos, sin)
            out = batch.attend_layer(rot if varlen else rot.transpose(1, 2), 0)
        results.append((rot, out, r.m.k_cache, r.m.v_cache))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_a_window_over_the_whole_cache_changes_nothing():
    r = Requests([900, 3000, 17], [1, 1, 1], seed=21)
    whole = r.m.begin_tick(r.handles, r.fresh).attend_layer(r.q, 0)
    assert torch.equal(whole, check(r, 5000, 0))
    assert torch.equal(whole, check(r, 10, 5000))


def test_replayed_graph_and_other_stream():
    r = Requests([700, 2500, 0, 90], [1, 130, 64, 1], seed=31)
    batch = r.m.begin_tick(r.handles, r.fresh, window=256, sinks=4)
    q = r.q.clone()
    eager = batch.attend_layer(q, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = batch.attend_layer(q, 0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = batch.attend_layer(q, 0)
    for step in range(3):
        q.copy_(normal(r.g, *q.shape))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, batch.attend_layer(q, 0)), step


def test_positions_of_a_compacted_cache_do_not_move_the_window():
    """The window counts slots, also where the cache dropped tokens before them."""
    r = Requests([500], [1], seed=14)
    r.m.compact(r.handles[0], [*range(10), *range(200, 500)])
    r.cached = [310]
    check(r, 100, 4)

