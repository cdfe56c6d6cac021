"""Ticks after an eviction, on the GPU: what is appended to a cache that dropped tokens is
rotated behind the last kept token's position. Against attention in 64 bits over keys rotated
at the positions that they were written for."""

import pytest
import torch

from hayate_amd import compute_rope_params
from tree_util import D, assert_attention, attention64, chain, depth, make_pool, physical, seen

pytestmark = pytest.mark.gpu

HQ, HKV = 32, 8


def normal(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def rotated(x, positions, tables):
    """The bits that a plain append gives rows x (n, heads, D) at these positions, each through
    a pool of its own with that many cached tokens."""
    out = []
    for row, at in zip(x, positions):
        one, (h,) = make_pool([0], [1], q_heads=None, kv_heads=HKV)
        h.length = 0
        cos, sin = (t[at : at + 1].contiguous() for t in tables)
        q = one.begin_tick([h], [1]).norm_rope_write_layer(
            0, row[None], normal(1, HKV, D), normal(1, HKV, D), None, None, 1e-6, cos, sin)
        out.append(q[0])
    return torch.stack(out)


KEEP = [*range(16), *range(300, 420), *range(505, 700)]
NEXT = 700


def evicted(extra=0):
    m, handles = make_pool([700, 130], [40, 40], q_heads=HQ, kv_heads=HKV, seed=5, spare=8)
    kept = [p[0, 0][:, physical(m, handles[0], 700)[KEEP]].clone() for p in (m.k_cache, m.v_cache)]
    m.compact(handles[0], KEEP)
    assert handles[0].next_position == NEXT
    return m, handles, kept


def check(m, h, kept, q, k, v, positions, tables, rot, out, tree=None):
    """Rows of h in a tick: q, k, v its own projections, out packed."""
    n, c = len(positions), len(KEEP)
    want_q, want_k = rotated(q, positions, tables), rotated(k, positions, tables)
    assert torch.equal(rot, want_q)
    rows = physical(m, h, c + n)
    assert torch.equal(m.k_cache[0, 0][:, rows[c:]], want_k.transpose(0, 1))
    assert torch.equal(m.v_cache[0, 0][:, rows[c:]], v.transpose(0, 1))
    for pool, x in zip((m.k_cache, m.v_cache), kept):
        assert torch.equal(pool[0, 0][:, rows[:c]], x)
    ref, size = attention64(want_q, torch.cat([kept[0], want_k.transpose(0, 1)], 1),
                            torch.cat([kept[1], v.transpose(0, 1)], 1), seen(c, tree or chain(n)))
    assert_attention(out, ref, size)


@pytest.mark.parametrize("lens", [(1, 1), (1, 9), (9, 1), (33, 4)])
def test_ticks(lens):
    m, handles, kept = evicted()
    tables = compute_rope_params(D, 1_000_000, 1024, device="cuda")
    batch = m.begin_tick(handles, list(lens))
    n = sum(lens)
    q, k, v = normal(n, HQ, D, seed=1), normal(n, HKV, D, seed=2), normal(n, HKV, D, seed=3)
    rot = batch.norm_rope_write_layer(0, q, k, v, None, None, 1e-6, *tables)
    out = batch.attend_layer(rot, 0)
    a = lens[0]
    check(m, handles[0], kept, q[:a], k[:a], v[:a], range(NEXT, NEXT + a), tables, rot[:a], out[:a])
    # the other request's positions are its slots
    assert torch.equal(rot[a:], rotated(q[a:], range(130, 130 + lens[1]), tables))


@pytest.mark.parametrize("n", [1, 5])
def test_uniform_batches(n):
    m, (h, other), kept = evicted()
    tables = compute_rope_params(D, 1_000_000, 1024, device="cuda")
    batch = m.begin_batch([other, h], n)
    q, k, v = normal(2, n, HQ, D, seed=1), normal(2, n, HKV, D, seed=2), normal(2, n, HKV, D, seed=3)
    rot = batch.norm_rope_write_layer(0, q, k, v, None, None, 1e-6, *tables)
    out = batch.attend_layer(rot.transpose(1, 2), 0).transpose(1, 2)
    check(m, h, kept, q[1], k[1], v[1], range(NEXT, NEXT + n), tables, rot[1], out[1])
    assert torch.equal(rot[0], rotated(q[0], range(130, 130 + n), tables))


@pytest.mark.parametrize("uniform", [False, True])
def test_the_fused_decode_call(uniform):
    """decode_layer gives what its two calls give."""
    m, handles, kept = evicted()
    tables = compute_rope_params(D, 1_000_000, 1024, device="cuda")
    batch = m.begin_batch(handles, 1) if uniform else m.begin_tick(handles, [1, 1])
    q, k, v = normal(2, HQ, D, seed=1), normal(2, HKV, D, seed=2), normal(2, HKV, D, seed=3)
    args = [x[:, None] if uniform else x for x in (q, k, v)]
    rot, out = batch.decode_layer(0, *args, None, None, 1e-6, *tables)
    assert rot.shape == args[0].shape and out.shape == ((2, HQ, 1, D) if uniform else (2, HQ, D))
    rot, out = rot.reshape(2, HQ, D), out.reshape(2, HQ, D)
    check(m, handles[0], kept, q[:1], k[:1], v[:1], [NEXT], tables, rot[:1], out[:1])
    assert torch.equal(rot[1:], rotated(q[1:], [130], tables))
    with pytest.raises(NotImplementedError):
        batch.decode_layer(0, *args, None, None, 1e-6, *tables, no_alloc=True)


def test_trees():
    m, handles, kept = evicted()
    tables = compute_rope_params(D, 1_000_000, 1024, device="cuda")
    tree = [-1, 0, 0, 1, -1, 4, 2]
    batch = m.begin_tree(handles, [tree, [-1]])
    q, k, v = normal(8, HQ, D, seed=1), normal(8, HKV, D, seed=2), normal(8, HKV, D, seed=3)
    rot = batch.norm_rope_write_layer(0, q, k, v, None, None, 1e-6, *tables)
    out = batch.attend_layer(rot, 0)
    at = [NEXT + depth(tree, i) for i in range(7)]
    check(m, handles[0], kept, q[:7], k[:7], v[:7], at, tables, rot[:7], out[:7], tree=tree)
    m.commit_tree(handles, batch, [[0, 2, 6], [0]])
    assert [h.next_position for h in handles] == [NEXT + 3, 131]
    # and a decode token behind the accepted path
    batch = m.begin_tick(handles, [1, 1])
    assert batch.positions.tolist() == [NEXT + 3, 131]


def test_the_rope_tables_have_to_reach_the_positions():
    m, handles, _ = evicted()
    batch = m.begin_tick(handles, [1, 1])
    q, k = normal(2, HQ, D), normal(2, HKV, D)
    for rows, ok in ((NEXT + 1, True), (NEXT, False)):
        tables = compute_rope_params(D, 10_000, rows, device="cuda")
        if ok:
            batch.norm_rope_write_layer(0, q, k, k, None, None, 1e-6, *tables)
        else:
            with pytest.raises(ValueError):
                batch.norm_rope_write_layer(0, q, k, k, None, None, 1e-6, *tables)


@torch.inference_mode()
def test_the_model_and_its_graphs():
    """A decode tick of the model after an eviction: the graph runner leaves it to the eager
    path, whose tick equals the same tick in a pool that was filled with the kept rows."""
    from hayate_amd import PagedKVCacheManager
    from hayate_amd.model import Qwen3Config, Qwen3Model, init_synthetic_weights
    from hayate_amd.tick_graph import StaticTickBatch, TickGraphRunner

    with torch.device("cuda"):
        model = Qwen3Model(Qwen3Config(num_layers=2, vocab_size=512, hidden_size=512,
                                       intermediate_size=1024, num_heads=8, num_kv_groups=2,
                                       max_position_embeddings=2048))
    init_synthetic_weights(model, 3)
    model.eval().initialize_rope("cuda")
    m = PagedKVCacheManager(2, 2, D, 2048, 128, 4, torch.bfloat16, "cuda", num_q_heads=8)
    h = m.allocate()
    batch = m.begin_tick([h], [300])
    model(torch.arange(300, device="cuda")[None] % 512, paged_cache=batch)
    m.commit_tick([h], [300])
    m.compact(h, [*range(4), *range(200, 300)])
    other = m.allocate_for_request(m.snapshot(h))
    assert other.next_position == 300
    m.reserve_tick([h], [1])
    assert TickGraphRunner(model, m, 2048).run([h], [1], [7]) is None
    assert not StaticTickBatch(m, [1], 8, 2048).refresh([h])
    got = []
    for x in (h, other):
        batch = m.begin_tick([x], [1])
        got.append(model(torch.tensor([[7]], device="cuda"), paged_cache=batch)[0])
        rows = physical(m, x, 105)
        got.append(m.k_cache[:, 0, :, rows])
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
    assert got[0].isfinite().all()
