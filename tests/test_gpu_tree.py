"""Attention and append for trees of drafted tokens, on the GPU, against their
definitions in 64 bits; and the tick they make up, from draft to commit."""

import random

import numpy as np
import pytest
import torch

from hayate_amd import PagedTreeBatch, compute_rope_params
from tree_util import (
    D,
    assert_attention,
    attention64,
    chain,
    depth,
    line,
    make_pool,
    physical,
    seen,
    wide_tree,
)

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def check(m, handles, trees, cached, q, out, layer=0, scale=None, nodes=None):
    at = 0
    for b, (h, tree, c) in enumerate(zip(handles, trees, cached)):
        rows = physical(m, h, c + len(tree))
        pick = range(len(tree)) if nodes is None else [i for i in nodes if i < len(tree)]
        pick = torch.tensor(list(pick), dtype=torch.long)
        ref, size = attention64(q[at + pick.to(q.device)], m.k_cache[layer, 0][:, rows],
                                m.v_cache[layer, 0][:, rows], seen(c, tree)[pick], scale)
        assert_attention(out[at + pick.to(out.device)], ref, size, f"request {b}")
        at += len(tree)


def attend(cached, trees, q_heads=32, kv_heads=8, page=128, seed=1, direct=False, nodes=None, **kw):
    sizes = [len(t) for t in trees]
    m, handles = make_pool(cached, sizes, q_heads=q_heads, kv_heads=kv_heads, page=page, seed=seed)
    if direct:  # page sizes below the manager's own limit
        for h, n in zip(handles, sizes):
            m.reserve(h, h.length + n)
        batch = PagedTreeBatch(m, trees, cached, [list(h.pages) for h in handles], q_heads)
    else:
        batch = m.begin_tree(handles, trees)
    n = sum(sizes)
    q = normal(n, q_heads, D, seed=seed)
    batch.write_layer(0, normal(n, kv_heads, D, seed=seed + 1), normal(n, kv_heads, D, seed=seed + 2))
    out = batch.attend_layer(q, 0, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype
    check(m, handles, trees, cached, q, out, nodes=nodes, **kw)
    return batch, q, out


@pytest.mark.parametrize("cached", [0, 1, 31, 32, 63, 64, 65, 127, 128, 500])
@pytest.mark.parametrize("n", [1, 2, 7, 16, 33])
def test_one_request(cached, n):
    attend([cached], [wide_tree(random.Random(cached + n), n)])


@pytest.mark.parametrize("q_heads,kv_heads", [(8, 8), (16, 8), (32, 8), (64, 8), (32, 2), (4, 4),
                                              (16, 1), (24, 3)])
@pytest.mark.parametrize("n", [1, 5, 17, 64])
def test_head_groups(q_heads, kv_heads, n):
    rng = random.Random(n)
    attend([200, 33], [wide_tree(rng, n), wide_tree(rng, max(1, n // 2))], q_heads, kv_heads)


@pytest.mark.parametrize("n", [63, 65, 100, 129, 255, 256])
@pytest.mark.parametrize("q_heads", [32, 128])
def test_wide_trees_take_several_tiles(n, q_heads):
    attend([90], [wide_tree(random.Random(n), n)], q_heads=q_heads,
           nodes=sorted({0, 1, n // 3, n // 2, n - 2, n - 1}))


def test_ragged_batch_of_every_size():
    rng = random.Random(5)
    cached = [0, 3, 4000, 64, 127, 1000, 31, 640, 2, 2500]
    sizes = [1, 64, 9, 33, 1, 16, 40, 2, 128, 5]
    attend(cached, [wide_tree(rng, n) for n in sizes], nodes=[0, 1, 8, 31, 32, 63, 127])


def test_many_small_requests():
    """More requests than chunks: chunks of many pieces, written without a merge."""
    rng = random.Random(6)
    cached = [rng.randint(0, 90) for _ in range(150)]
    attend(cached, [wide_tree(rng, rng.randint(1, 6)) for _ in cached])


@pytest.mark.parametrize("page", [32, 64, 256, 512])
def test_page_sizes(page):
    rng = random.Random(page)
    attend([0, 77, 300], [wide_tree(rng, n) for n in (3, 40, 12)], page=page, direct=page < 128)


def test_scale():
    attend([100], [wide_tree(random.Random(1), 12)], scale=0.031)


def test_a_chain_is_a_prompt_chunk():
    """A chain of drafted tokens sees what a prompt chunk's tokens see: both paths are
    within the bound of the same 64-bit result."""
    m, handles = make_pool([300], [40], seed=3)
    q, k, v = normal(40, 32, D, seed=1), normal(40, 8, D, seed=2), normal(40, 8, D, seed=3)
    tick = m.begin_tick(handles, [40])
    tick.write_layer(0, k, v)
    chunk = tick.attend_layer(q, 0)
    out = m.begin_tree(handles, [chain(40)]).attend_layer(q, 0)
    rows = physical(m, handles[0], 340)
    ref, size = attention64(q, m.k_cache[0, 0][:, rows], m.v_cache[0, 0][:, rows],
                            seen(300, chain(40)))
    assert_attention(chunk, ref, size)
    assert_attention(out, ref, size)


def test_large_scores_keep_their_maximum():
    """Scores of several hundred: the exponent base moves, nothing overflows."""
    m, handles = make_pool([700], [20], seed=8)
    tree = wide_tree(random.Random(8), 20)
    batch = m.begin_tree(handles, [tree])
    q = normal(20, 32, D, seed=1, std=8.0)
    batch.write_layer(0, normal(20, 8, D, seed=2, std=8.0), normal(20, 8, D, seed=3))
    out = batch.attend_layer(q, 0)
    rows = physical(m, handles[0], 720)
    ref, size = attention64(q, m.k_cache[0, 0][:, rows], m.v_cache[0, 0][:, rows], seen(700, tree))
    off = (out.double().cpu() - ref).abs()
    # a score's 128 products sum to under 128 * 64 in size (rows of N(0, 8): 0.64 * 64 each in
    # the mean), so its fp32 sum is off by at most 128 * 2^-24 * 8192 * 128^-0.5 = 5.6e-3: as
    # much of a probability, and of the sum that divides it
    assert (off <= (2.0**-8 + 2.0**-11 + 2 * 5.6e-3) * size + 2.0**-7 * ref.abs()).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["k", "v"])
def test_other_branches_may_hold_anything(bad, where):
    """Non-finite K or V of one branch reaches its own nodes and no other's."""
    m, handles = make_pool([70, 64], [30, 7], seed=4)
    trees = [[-1, 0, 0, 1, 2, 3, 4, 5, 6, 7] + [8 + (i % 2) for i in range(20)], wide_tree(random.Random(2), 7)]
    batch = m.begin_tree(handles, trees)
    q, k, v = normal(37, 32, D, seed=1), normal(37, 8, D, seed=2), normal(37, 8, D, seed=3)
    sick = 4  # seen by nodes 4, 6, 8, ...
    (k if where == "k" else v)[sick, 3, 40:45] = bad
    batch.write_layer(0, k, v)
    out = batch.attend_layer(q, 0)
    at = 0
    for h, tree, c in zip(handles, trees, [70, 64]):
        rows = physical(m, h, c + len(tree))
        mask = seen(c, tree)
        ref, size = attention64(q[at : at + len(tree)], m.k_cache[0, 0][:, rows],
                                m.v_cache[0, 0][:, rows], mask)
        for i in range(len(tree)):
            got = out[at + i].double().cpu()
            if at == 0 and sick in line(tree, i):
                heads = slice(12, 16)
                if where == "v":
                    assert not torch.isfinite(got[heads, 40:45]).any()
                    if bad == bad:
                        assert (got[heads, 40:45] == bad).all()
                    got[heads, 40:45] = ref[i, heads, 40:45] = size[i, heads, 40:45] = 0
                else:
                    continue
            assert_attention(got, ref[i], size[i], (at, i))
        at += len(tree)


@pytest.mark.parametrize("q_heads,kv_heads", [(8, 8), (32, 8), (64, 8)])
def test_a_row_that_sees_one_bad_key_in_a_part(q_heads, kv_heads):
    """Forty roots: each sees, of the drafted slots, its own only. With no cached tokens an
    infinite value there is the row's result; a key that is NaN makes the row NaN also where the
    last part of a split request holds no other key that it sees."""
    n = 40
    tree = [-1] * n
    m, handles = make_pool([0], [n], q_heads=q_heads, kv_heads=kv_heads, seed=4)
    batch = m.begin_tree(handles, [tree])
    q, k, v = normal(n, q_heads, D, seed=1), normal(n, kv_heads, D, seed=2), normal(n, kv_heads, D, seed=3)
    v[35, :, 7] = float("inf")
    v[3, :, 9] = -float("inf")
    batch.write_layer(0, k, v)
    out = batch.attend_layer(q, 0)
    # a row that sees one key takes its value as it is
    assert torch.equal(out, v.repeat_interleave(q_heads // kv_heads, dim=1))

    from hayate_amd import _native

    # a request before another one, cut where its drafted slots begin
    def cut_there(cached, other):
        plan = _native.plan_tree(np.array([n, 1]), np.array([cached + n, other + 1]), q_heads, kv_heads,
                                 m.num_cus)
        pieces = plan.items[2 * plan.n_chunks :]
        return any(r[0] == 0 and r[3] == cached for r in pieces.tolist())

    cached, other = next((c, x) for c in range(64, 1 << 16, 64) for x in range(0, 4096, 64)
                         if cut_there(c, x))
    m, handles = make_pool([cached, other], [n, 1], q_heads=q_heads, kv_heads=kv_heads, seed=4)
    batch = m.begin_tree(handles, [tree, [-1]])
    k[11] = float("nan")
    v = v.nan_to_num(0, 0, 0)
    last = normal(1, q_heads, D, seed=5)
    batch.write_layer(0, torch.cat([k, last[:, :kv_heads]]), torch.cat([v, last[:, :kv_heads]]))
    out = batch.attend_layer(torch.cat([q, last]), 0)[:n]
    assert torch.isnan(out[11]).all()
    rows = physical(m, handles[0], cached + n)
    others = [i for i in range(n) if i != 11]
    ref, size = attention64(q[others], m.k_cache[0, 0][:, rows], m.v_cache[0, 0][:, rows],
                            seen(cached, tree)[others])
    assert_attention(out[others], ref, size)


def test_pools_of_other_types_are_refused():
    from hayate_amd import PagedKVCacheManager

    m = PagedKVCacheManager(1, 8, D, 512, 128, 2, torch.float16, "cuda")
    batch = m.begin_tree([m.allocate()], [[-1]])
    with pytest.raises(TypeError):
        batch.attend_layer(torch.zeros(1, 32, D, dtype=torch.float16, device="cuda"), 0)


def test_strided_rows():
    """q, k and v as views of one projection, as the model has them."""
    m, handles = make_pool([150, 20], [12, 5], seed=4)
    trees = [wide_tree(random.Random(3), 12), chain(5)]
    batch = m.begin_tree(handles, trees)
    qkv = normal(17, 48, D, seed=1)
    batch.write_layer(0, qkv[:, 32:40], qkv[:, 40:])
    out = batch.attend_layer(qkv[:, :32], 0)
    assert torch.equal(out, batch.attend_layer(qkv[:, :32].contiguous(), 0))
    check(m, handles, trees, [150, 20], qkv[:, :32], out)
    # rows that are not 16-byte aligned are copied
    loose = torch.empty(17 * 32 * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(17, 32, D)
    loose.copy_(qkv[:, :32])
    assert torch.equal(out, batch.attend_layer(loose, 0))


def test_same_bits_every_time_and_neighbours_do_not_matter():
    cached = [900, 10, 333]
    trees = [wide_tree(random.Random(i), n) for i, n in enumerate((20, 3, 50))]
    batch, q, out = attend(cached, trees)
    for _ in range(3):
        assert torch.equal(out, batch.attend_layer(q, 0))


def test_another_stream_and_another_layer():
    m, handles = make_pool([400], [9], layers=3, seed=2)
    tree = wide_tree(random.Random(4), 9)
    batch = m.begin_tree(handles, [tree])
    q, k, v = normal(9, 32, D, seed=1), normal(9, 8, D, seed=2), normal(9, 8, D, seed=3)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        batch.write_layer(2, k, v)
        out = batch.attend_layer(q, 2)
    s.synchronize()
    check(m, handles, [tree], [400], q, out, layer=2)
    assert torch.isnan(m.k_cache[0, 0][:, physical(m, handles[0], 409)[400:]]).all()


def test_captured_and_replayed():
    """Append and attention captured once and replayed on new inputs, with eager work
    between, equal the eager calls bit for bit."""
    m, handles = make_pool([700, 45], [24, 6], seed=2)
    trees = [wide_tree(random.Random(4), 24), chain(6)]
    batch = m.begin_tree(handles, trees)
    cos, sin = compute_rope_params(D, 1_000_000, 1024, device="cuda")
    qw, kw = normal(D, seed=8), normal(D, seed=9)
    q, k, v = normal(30, 32, D, seed=1), normal(30, 8, D, seed=2), normal(30, 8, D, seed=3)

    def step():
        rot = batch.norm_rope_write_layer(0, q, k, v, qw, kw, 1e-6, cos, sin)
        return rot, batch.attend_layer(rot, 0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(10, 14):
        for t, x in zip((q, k, v), (32, 8, 8)):
            t.copy_(normal(30, x, D, seed=seed * x))
        want = step()
        pools = m.k_cache.clone(), m.v_cache.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # bits, since the pool's free slots hold NaN
        assert torch.equal(m.k_cache.view(torch.int16), pools[0].view(torch.int16))
        assert torch.equal(m.v_cache.view(torch.int16), pools[1].view(torch.int16))


def test_an_unplanned_batch_is_refused_in_a_capture():
    m, handles = make_pool([100], [8], q_heads=None)
    batch = m.begin_tree(handles, [chain(8)])
    q, k = normal(8, 32, D), normal(8, 8, D)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.write_layer(0, k, k)
        with pytest.raises(RuntimeError):
            batch.attend_layer(q, 0)
    graph.replay()
    assert batch.attend_layer(q, 0).isfinite().all()


@pytest.mark.parametrize("q_heads,kv_heads", [(32, 8), (16, 1), (4, 4)])
@pytest.mark.parametrize("sizes,cached", [([200], [130]), ([200] * 8, [3000] * 8),
                                          ([256, 3, 70], [900, 40, 2000])])
def test_tiles_of_128_and_of_256_rows(sizes, cached, q_heads, kv_heads):
    """Trees of more rows than a tile holds, in tiles of both sizes."""
    trees = [wide_tree(random.Random(i), n) for i, n in enumerate(sizes)]
    attend(cached, trees, q_heads, kv_heads, nodes=[0, 31, 32, 63, 64, 65, 127, 150, 199, 255])


def test_pages_past_2_31_elements():
    """A head of over 2^31 elements, its last pages in use."""
    from hayate_amd import PagedKVCacheManager

    page, pages = 256, (1 << 31) // (256 * D) + 64
    m = PagedKVCacheManager(1, 1, D, pages * page, page, 2, torch.bfloat16, "cuda", num_q_heads=4)
    h = m.allocate()
    m.claim_pages(h, [pages - 1, 0, pages - 2])
    h.length = 600
    rows = physical(m, h, 620)
    m.k_cache[:, :, :, rows] = normal(1, 1, 1, 620, D, seed=1)
    m.v_cache[:, :, :, rows] = normal(1, 1, 1, 620, D, seed=2)
    tree = wide_tree(random.Random(1), 20)
    q = normal(20, 4, D, seed=3)
    out = m.begin_tree([h], [tree]).attend_layer(q, 0)
    check(m, [h], [tree], [600], q, out)


# ---------------------------------------------------------------- the append
def append_case(cached, trees, q_heads=32, kv_heads=8, norm=True, rope=True):
    sizes = [len(t) for t in trees]
    n = sum(sizes)
    # planned on the first attend_layer only: the append takes any number of query heads
    m, handles = make_pool(cached, sizes, q_heads=None, kv_heads=kv_heads, seed=3)
    batch = m.begin_tree(handles, trees)
    qkv = normal(n, q_heads + 2 * kv_heads, D, seed=1)
    q, k, v = qkv[:, :q_heads], qkv[:, q_heads : q_heads + kv_heads], qkv[:, q_heads + kv_heads :]
    w = [1 + normal(D, seed=s, std=0.1) if norm else None for s in (5, 6)]
    tables = compute_rope_params(D, 1_000_000, 4096, device="cuda") if rope else (None, None)
    before = m.k_cache.clone(), m.v_cache.clone()
    rot = batch.norm_rope_write_layer(0, q, k, v, *w, 1e-6, *tables, k_eps=1e-5)
    return m, handles, batch, (q, k, v), w, tables, before, rot


@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (True, False)])
def test_append_rotates_at_the_depth(norm, rope):
    """Every row has the bits that the plain append gives it at position c + depth, K and V
    land in slot c + i, and no other slot changes."""
    cached, trees = [0, 130, 640], [wide_tree(random.Random(i), n) for i, n in enumerate((3, 40, 9))]
    m, handles, batch, (q, k, v), w, tables, before, rot = append_case(cached, trees, norm=norm,
                                                                       rope=rope)
    at = 0
    for h, tree, c in zip(handles, trees, cached):
        for i in range(len(tree)):
            assert batch.positions[at + i].item() == c + depth(tree, i)
        rows = physical(m, h, c + len(tree))[c:]
        for d in sorted({depth(tree, i) for i in range(len(tree))}):
            nodes = [at + i for i in range(len(tree)) if depth(tree, i) == d]
            # a request of its own with c + d cached tokens decodes each of these tokens
            for row in nodes:
                one, (oh,) = make_pool([c + d], [1])
                tick = one.begin_tick([oh], [1])
                want = tick.norm_rope_write_layer(0, q[row : row + 1], k[row : row + 1],
                                                  v[row : row + 1], *w, 1e-6, *tables, k_eps=1e-5)
                assert torch.equal(rot[row], want[0])
                slot = physical(one, oh, c + d + 1)[-1]
                assert torch.equal(m.k_cache[0, 0][:, rows[row - at]], one.k_cache[0, 0][:, slot])
        assert torch.equal(m.v_cache[0, 0][:, rows], v[at : at + len(tree)].transpose(0, 1))
        for pool, old in zip((m.k_cache, m.v_cache), before):
            old[:, :, :, rows] = pool[:, :, :, rows]
        at += len(tree)
    for pool, old in zip((m.k_cache, m.v_cache), before):
        assert torch.equal(pool.view(torch.int16), old.view(torch.int16))


@pytest.mark.parametrize("q_heads,kv_heads", [(32, 8), (8, 8), (64, 4), (40, 8), (12, 12)])
def test_append_against_64_bits(q_heads, kv_heads):
    """Two roundings to bf16 (the norm's output and the result): each coordinate of a
    pair is off by at most 2^-8 of the normed coordinates it is made of, and of itself."""
    cached, trees = [100, 7], [wide_tree(random.Random(1), 21), chain(4)]
    m, handles, batch, (q, k, v), w, (cos, sin), _, rot = append_case(cached, trees, q_heads, kv_heads)
    pos = [c + depth(t, i) for c, t in zip(cached, trees) for i in range(len(t))]
    slots = torch.cat([physical(m, h, c + len(t))[c:] for h, c, t in zip(handles, cached, trees)])
    got_k = m.k_cache[0, 0][:, slots].transpose(0, 1)
    for x, weight, eps, got in ((q, w[0], 1e-6, rot), (k, w[1], 1e-5, got_k)):
        x = x.double()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
        co, si = (t[torch.tensor(pos, device="cuda"), : D // 2].double()[:, None] for t in (cos, sin))
        a, b = x[..., : D // 2], x[..., D // 2 :]
        ref = torch.cat([a * co - b * si, b * co + a * si], -1)
        size = torch.cat([(a * co).abs() + (b * si).abs(), (b * co).abs() + (a * si).abs()], -1)
        # fp32 steps (norm: 4 roundings, rotation: 3) are under 2^-20
        allowed = (2.0**-8 + 2.0**-20) * size + 2.0**-8 * (ref.abs() + 2.0**-7 * size)
        assert ((got.double() - ref).abs() <= allowed).all()


def test_positions_past_the_rope_tables_are_refused():
    m, handles = make_pool([100], [8])
    batch = m.begin_tree(handles, [chain(8)])
    q, k = normal(8, 32, D), normal(8, 8, D)
    cos, sin = compute_rope_params(D, 10_000, 104, device="cuda")
    with pytest.raises(ValueError):
        batch.norm_rope_write_layer(0, q, k, k, None, None, 1e-6, cos, sin)


def test_a_wide_tree_needs_its_depths_positions_only():
    """Slots 100 .. 139, positions 100 and 101: tables of 102 positions are enough."""
    m, handles = make_pool([100], [40])
    tree = [-1] * 20 + list(range(20))
    batch = m.begin_tree(handles, [tree])
    q, k = normal(40, 32, D), normal(40, 8, D)
    full = compute_rope_params(D, 10_000, 200, device="cuda")
    want = batch.norm_rope_write_layer(0, q, k, k, None, None, 1e-6, *full)
    got = batch.norm_rope_write_layer(0, q, k, k, None, None, 1e-6,
                                      *(t[:102].contiguous() for t in full))
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        batch.norm_rope_write_layer(0, q, k, k, None, None, 1e-6,
                                    *(t[:101].contiguous() for t in full))


def test_refusals():
    m, handles = make_pool([10], [4])
    batch = m.begin_tree(handles, [chain(4)])
    q = normal(4, 32, D)
    for bad, error in ((q[:3], ValueError), (q.float(), TypeError), (q.cpu(), RuntimeError),
                       (q[:, :30], ValueError), (q[:, :0], ValueError),
                       (q[:, :, :64], ValueError), (q[None], ValueError)):
        with pytest.raises(error):
            batch.attend_layer(bad, 0)
    with pytest.raises(NotImplementedError):  # groups of 3
        batch.attend_layer(q[:, :24], 0)
    with pytest.raises(IndexError):
        batch.attend_layer(q, 1)
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            batch.attend_layer(q, 0, scale=scale)
    with pytest.raises(ValueError):  # a tree tick is not a decode tick
        batch.decode_layer(0, q, q[:, :8], q[:, :8], None, None, 1e-6, None, None)


# ------------------------------------------------------------- the whole tick
def small_model(layers=3):
    from hayate_amd.model import Qwen3Config, Qwen3Model, init_synthetic_weights

    with torch.device("cuda"):
        model = Qwen3Model(Qwen3Config(num_layers=layers, vocab_size=512, hidden_size=512,
                                       intermediate_size=1024, num_heads=8, num_kv_groups=2,
                                       max_position_embeddings=2048))
    init_synthetic_weights(model, 3)
    model.eval().initialize_rope("cuda")
    return model


def cosine(a, b):
    return torch.nn.functional.cosine_similarity(a.double(), b.double(), dim=-1)


@pytest.mark.parametrize("nodes", [(6, 9), (30, 22)])
@torch.inference_mode()
def test_draft_check_commit_and_go_on(nodes):
    """Two requests' prompts, a tree tick, the commit of a path of each and one more decode
    tick, against the same tokens decoded one by one. The logits of both pass through the same
    model in bf16; they are compared by direction."""
    model = small_model()
    rng = random.Random(9)
    prompts = [[rng.randrange(512) for _ in range(n)] for n in (150, 37)]
    trees = [wide_tree(rng, n) for n in nodes]
    tokens = [[rng.randrange(512) for _ in t] for t in trees]
    paths = [line(t, max(range(len(t)), key=lambda i: (depth(t, i), i))) for t in trees]
    assert all(p != list(range(len(p))) for p in paths)

    def start():
        from hayate_amd import PagedKVCacheManager

        m = PagedKVCacheManager(3, 2, D, 2048, 128, 4, torch.bfloat16, "cuda", num_q_heads=8)
        m.k_cache.fill_(float("nan"))
        m.v_cache.fill_(float("nan"))
        handles = [m.allocate() for _ in prompts]
        batch = m.begin_tick(handles, [len(p) for p in prompts])
        model(torch.tensor([sum(prompts, [])], device="cuda"), paged_cache=batch)
        m.commit_tick(handles, [len(p) for p in prompts])
        return m, handles

    def decode(m, handles, toks):
        batch = m.begin_tick(handles, [1] * len(handles))
        logits, _, _ = model(torch.tensor([toks], device="cuda"), paged_cache=batch)
        m.commit_tick(handles, [1] * len(handles))
        return logits[:, 0]

    m, handles = start()
    free = m.free_page_count
    batch = m.begin_tree(handles, trees)
    logits, _, _ = model(torch.tensor([sum(tokens, [])], device="cuda"), paged_cache=batch)
    assert logits.shape == (sum(nodes), 1, 512)
    m.commit_tree(handles, batch, paths)
    assert [h.length for h in handles] == [len(p) + len(x) for p, x in zip(prompts, paths)]
    assert free - m.free_page_count == sum(len(h.pages) for h in handles) - 3
    after = decode(m, handles, [7, 8])

    for b, (tree, toks, path) in enumerate(zip(trees, tokens, paths)):
        one, hs = start()
        at = sum(nodes[:b])
        for i in path:
            want = decode(one, [hs[b]], [toks[i]])
            assert cosine(logits[at + i], want).item() > 0.999
        want = decode(one, [hs[b]], [7 + b])
        assert cosine(after[b : b + 1], want).item() > 0.999
        rows = physical(m, handles[b], handles[b].length)
        other = physical(one, hs[b], hs[b].length)
        # layer 0's cache comes from the same embeddings: its bits differ only where the
        # projections' rows were summed in another order
        for pool, alone in ((m.k_cache, one.k_cache), (m.v_cache, one.v_cache)):
            assert cosine(pool[0, 0][:, rows], alone[0, 0][:, other]).min().item() > 0.9999


@pytest.mark.parametrize("n,cached", [(20, 900), (1, 40), (70, 3000), (200, 500)])
def test_a_request_alone_and_among_sick_neighbours(n, cached):
    """The plan cuts a request by the whole batch, so its bits may differ; what its neighbours
    hold, NaN in every key and value, reaches none of them."""
    tree = wide_tree(random.Random(n), n)
    q, k, v = normal(n, 32, D, seed=1), normal(n, 8, D, seed=2), normal(n, 8, D, seed=3)
    m, (h,) = make_pool([cached], [n], seed=7)
    rows = physical(m, h, cached)
    own = [p[0, 0][:, rows].clone() for p in (m.k_cache, m.v_cache)]
    batch = m.begin_tree([h], [tree])
    batch.write_layer(0, k, v)
    rows = physical(m, h, cached + n)
    ref, size = attention64(q, m.k_cache[0, 0][:, rows], m.v_cache[0, 0][:, rows], seen(cached, tree))
    assert_attention(batch.attend_layer(q, 0), ref, size, "alone")
    for before, after in (([700, 64], [33]), ([5], [2000, 1, 130]), ([3] * 40, [90] * 40)):
        rng = random.Random(len(before))
        others = [wide_tree(rng, rng.randint(1, 60)) for _ in before + after]
        trees = others[: len(before)] + [tree] + others[len(before) :]
        m, handles = make_pool([*before, cached, *after], [len(t) for t in trees], seed=7)
        mine = len(before)
        m.k_cache.fill_(float("nan"))
        m.v_cache.fill_(float("nan"))
        rows = physical(m, handles[mine], cached)
        for p, x in zip((m.k_cache, m.v_cache), own):
            p[0, 0][:, rows] = x
        batch = m.begin_tree(handles, trees)
        at = sum(len(t) for t in trees[:mine])
        every = [torch.full((sum(len(t) for t in trees), x.shape[1], D), float("nan"),
                            dtype=torch.bfloat16, device="cuda") for x in (q, k, v)]
        for x, y in zip(every, (q, k, v)):
            x[at : at + n] = y
        batch.write_layer(0, *every[1:])
        out = batch.attend_layer(every[0], 0)
        assert_attention(out[at : at + n], ref, size, (before, after))


@pytest.mark.parametrize("sizes,cached", [([9], [500]), ([20, 5, 33], [900, 10, 3000]),
                                          ([200, 60], [2500, 800])])
def test_lists_padded_with_empty_records(sizes, cached):
    """A caller with a fixed launch size pads the chunk and the merge records: the same bits."""
    from hayate_amd import _native

    m, handles = make_pool(cached, sizes, seed=3)
    batch = m.begin_tree(handles, [wide_tree(random.Random(i), n) for i, n in enumerate(sizes)])
    n = sum(sizes)
    q, k, v = normal(n, 32, D, seed=1), normal(n, 8, D, seed=2), normal(n, 8, D, seed=3)
    batch.write_layer(0, k, v)
    want = batch.attend_layer(q, 0)
    plan = batch.plan(32).host
    chunks, merges = plan.n_chunks + 7, len(plan.merge) + 5
    items = np.zeros((2 * chunks + len(plan.items) - 2 * plan.n_chunks, 8), dtype=np.int32)
    items[: 2 * plan.n_chunks] = plan.items[: 2 * plan.n_chunks]
    items[2 * chunks :] = plan.items[2 * plan.n_chunks :]
    merge = np.zeros((merges, 8), dtype=np.int32)
    merge[: len(plan.merge)] = plan.merge
    slots = max(1, plan.n_slots)
    size = _native.tree_workspace_bytes(slots, 8, D)
    items, merge = torch.from_numpy(items).cuda(), torch.from_numpy(merge).cuda()
    space, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.full_like(q, float("nan"))
    rc = _native.lib().hy_paged_tree(
        q.data_ptr(), 0, 32 * D, D, out.data_ptr(), 0, 32 * D, D, m.k_cache.data_ptr(),
        m.v_cache.data_ptr(), m.k_cache.stride(2), batch.page_table.data_ptr(),
        batch.page_table.stride(0), batch.lines.data_ptr(), batch.line_words, items.data_ptr(),
        chunks, plan.max_rows, merge.data_ptr(), merges, slots, space.data_ptr(), size, 32, 8, D,
        m.page_size, D**-0.5, torch.cuda.current_stream().cuda_stream)
    assert rc == _native.HY_OK, _native.last_error()
    assert torch.equal(out, want)
