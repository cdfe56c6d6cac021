"""Attention that adds up the cached tokens' weights (csrc/weigh.hip and the calls before it)
against its definition in 64 bits.

The bound on a weight: a probability's relative error is that of its score, 128 products of
N(0, 1) values added in fp32 (2^-24 * 128 * sum |q k| * scale = 6e-5 at most), of the exponent's
two roundings (|argument| < 64: 8e-6) and of the row's sum; adding n of them in fp32, at most 128
in a row before they are joined pairwise or by wave, 128 * 2^-24 = 8e-6 more. 2e-4 holds them;
what was in the table before adds half a step of the result, 2^-24."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from long_util import D, DEV, Requests, assert_close, normal
    from test_gpu_window import _tables


def table(r, width=None, fill=0.0):
    rows = r.m.max_requests
    width = max(c + n for c, n in zip(r.cached, r.fresh)) if width is None else width
    return torch.full((rows, width), fill, device=DEV)


def check(r, weights=None, scale=None, what=""):
    weights = table(r, fill=0.5) if weights is None else weights
    before = weights.clone()
    batch = r.m.begin_tick(r.handles, r.fresh, weights=weights)
    out = batch.attend_layer(r.q, 0, scale)
    expected, bound, total = r.expected(scale=scale)
    assert_close(out, expected, bound, what)
    plain = r.m.begin_tick(r.handles, r.fresh).attend_layer(r.q, 0, scale)
    assert torch.equal(out, plain)  # the weights are an addition
    for h, t in zip(r.handles, total):
        n = len(t)
        want = before[h.slot, :n].double() + t
        off = (weights[h.slot, :n].double() - want).abs()
        assert (off <= 2e-4 * t + 2**-23 * want).all(), (what, float((off / want).max()))
        before[h.slot, :n] = weights[h.slot, :n]
    assert torch.equal(weights, before)  # and nothing else in the table moved
    return weights


@pytest.mark.parametrize("batch", [1, 5, 24])
def test_decode(batch):
    cached = ([0, 1, 3, 31, 32, 33, 63, 255, 256, 257, 511, 512, 700, 1023, 1500, 2047, 2048,
               3000, 64, 127, 128, 129, 5, 900])[:batch]
    check(Requests(cached, [1] * batch, seed=batch), what=f"decode {batch}")
    check(Requests([20_000], [1], seed=1), what="long decode")


def test_chunks():
    cached = [0, 0, 0, 1, 255, 256, 257, 1000, 2500]
    fresh = [2, 257, 64, 31, 200, 512, 3, 65, 130]
    check(Requests(cached, fresh, seed=3), what="chunks")


@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 8), (64, 8), (32, 2), (1, 1), (4, 4)])
def test_head_groups(hq, hkv):
    check(Requests([700, 0, 1234, 40, 3000], [1, 150, 77, 1, 513], hq=hq, hkv=hkv, page=256,
                   seed=hq), what=f"{hq}/{hkv}")


@pytest.mark.parametrize("split", [32, 96, 1000, 100_000])
def test_many_partials_and_long_chunks(split):
    """Hundreds of partials, of which 64 are joined at a time, and chunks of more slices than
    a wave holds the scores of (104 with four heads to a kv head, 52 with eight)."""
    r = Requests([9000, 2048, 700, 63], [1, 1, 1, 1], seed=split)
    r.m.tokens_per_split = split
    check(r, what=f"split {split}")
    one = Requests([9000], [1], hq=64, hkv=8, seed=split)
    one.m.tokens_per_split = split
    check(one, what=f"split {split}, one")
    if split == 100_000:
        chunks = one.m.begin_tick(one.handles, one.fresh).plan(64).host.decode[:, 2]
        assert int(chunks[0]) > 4 * 52


@pytest.mark.parametrize("hq,hkv", [(128, 8), (2, 1), (80, 5)])
def test_more_and_fewer_heads_than_a_waves_lanes(hq, hkv):
    """(partials of 64 heads are read at a time, outputs of eight joined)"""
    check(Requests([2500, 0, 40], [1, 1, 33], hq=hq, hkv=hkv, seed=hq), what=f"{hq}/{hkv}")


@pytest.mark.parametrize("seed", range(6))
def test_random_mixed_ticks(seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    n = pick(1, 24)
    fresh = [1 if pick(0, 2) else pick(2, 200) for _ in range(n)]
    r = Requests([pick(0, 2500) for _ in range(n)], fresh, seed=seed)
    check(r, scale=0.05 if seed == 3 else None, what=f"seed {seed}")


def test_keys_behind_32_bit_offsets():
    """Pools whose last pages lie 2^31 elements and more into each head: 9 GB."""
    r = Requests([700, 90, 0], [1, 150, 70], hq=8, hkv=1, seed=2, skip=(2**31 // 128) // 128 + 1)
    assert min(min(h.pages) for h in r.handles) * 128 * 128 >= 2**31
    check(r, what="far")
    out = r.m.begin_tick(r.handles, r.fresh, window=100, sinks=3).attend_layer(r.q, 0)
    expected, bound, _ = r.expected(100, 3)
    assert_close(out, expected, bound, "far, window")


def test_rows_of_the_table():
    """Rows by slot, not by place in the batch; a wider table, rows apart and off 16 bytes."""
    r = Requests([100, 900, 300], [1, 40, 1], seed=2)
    r.handles = [r.handles[2], r.handles[0], r.handles[1]]
    r.cached = [300, 100, 900]
    r.fresh = [1, 1, 40]
    wide = torch.full((9, 2003), 0.25, device=DEV)
    weights = wide[:, 1:1501]
    check(r, weights, what="rows")
    assert (wide[:, 0] == 0.25).all() and (wide[:, 1501:] == 0.25).all()


def test_layers_and_ticks_add_up():
    r = Requests([200, 90], [1, 5], seed=6, layers=3)
    weights = table(r)
    batch = r.m.begin_tick(r.handles, r.fresh, weights=weights)
    want = [0, 0]
    for layer in range(3):
        batch.attend_layer(r.q, layer)
        want = [a + t for a, t in zip(want, r.expected(layer=layer)[2])]
    for h, t in zip(r.handles, want):
        assert ((weights[h.slot, : len(t)].double() - t).abs() <= 2e-4 * t).all()
    # every row's probabilities sum to one: 3 layers x heads x tokens
    sums = [weights[h.slot].sum().item() for h in r.handles]
    assert sums == pytest.approx([3 * 32 * 1, 3 * 32 * 5], rel=2e-4)


def test_uniform_batches_and_strided_rows():
    r = Requests([600, 90, 1400], [5, 5, 5], seed=8)
    weights = table(r)
    batch = r.m.begin_batch(r.handles, 5, weights=weights)
    wide = normal(r.g, 3, 5, r.hq + 16, D)
    q = wide[:, :, 8 : 8 + r.hq]
    out = batch.attend_layer(q.transpose(1, 2), 0).transpose(1, 2).reshape(15, r.hq, D)
    expected, bound, total = r.expected(q=q.reshape(15, r.hq, D))
    assert_close(out, expected, bound, "uniform")
    for h, t in zip(r.handles, total):
        assert ((weights[h.slot, : len(t)].double() - t).abs() <= 2e-4 * t).all()


def test_decode_layer_makes_the_two_calls():
    cos, sin = _tables(4096)
    results = []
    for fused in (True, False):
        r = Requests([0, 31, 500, 1500], [1] * 4, seed=12)
        weights = table(r)
        qkv = normal(r.g, 4, r.hq + 2 * r.hkv, D)
        qw, kw = normal(r.g, D), normal(r.g, D)
        batch = r.m.begin_tick(r.handles, r.fresh, weights=weights)
        q, k, v = qkv.split([r.hq, r.hkv, r.hkv], -2)
        if fused:
            rot, out = batch.decode_layer(0, q, k, v, qw, kw, 1e-6, cos, sin)
        else:
            rot = batch.norm_rope_write_layer(0, q, k, v, qw, kw, 1e-6, cos, sin)
            out = batch.attend_layer(rot, 0)
        results.append((rot, out, weights))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert results[0][2].sum().item() == pytest.approx(4 * 32, rel=2e-4)


def test_stale_slots_behind_a_cache_weigh_nothing():
    """Slots past a request's last token may hold anything."""
    r = Requests([100, 300, 20], [1, 70, 1], seed=4)
    clean = check(r)
    live = torch.cat([r.rows(b) for b in range(3)])
    stale = torch.ones(r.m.capacity_tokens, dtype=torch.bool, device=DEV)
    stale[live] = False
    for value in (float("nan"), float("inf")):
        r.m.k_cache[0, 0][:, stale] = value
        r.m.v_cache[0, 0][:, stale] = value
        assert torch.equal(check(r), clean)


def test_same_sums_every_time_and_replayed():
    r = Requests([700, 2500, 0, 90], [1, 130, 64, 1], seed=31)
    weights = table(r)
    batch = r.m.begin_tick(r.handles, r.fresh, weights=weights)
    q = r.q.clone()
    batch.attend_layer(q, 0)
    first = weights.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        weights.zero_()
        batch.attend_layer(q, 0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(weights, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = batch.attend_layer(q, 0)
    for step in range(3):
        q.copy_(normal(r.g, *q.shape))
        weights.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = weights.clone()
        weights.zero_()
        assert torch.equal(out, batch.attend_layer(q, 0)), step
        assert torch.equal(got, weights), step
