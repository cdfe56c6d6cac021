"""A batch's device memory (page table, lengths, lines, positions, work lists, partials) is
freed to the stream it was made on. Calls on another stream have to name it to the allocator
first, or a batch dropped behind them leaves its memory to others while they still read it.
Without a GPU: streams are numbers, the kernels a stand-in that launches nothing."""

import pytest
import torch

import hayate_amd.paged_cache as pc
from hayate_amd import PagedKVCacheManager, _native
from tree_util import chain

LAUNCHES = {"hy_kv_append", "hy_qknorm_rope_append", "hy_qknorm_rope_append_at", "hy_paged_tree",
            "hy_paged_decode", "hy_paged_decode_merge", "hy_paged_prefill",
            "hy_paged_prefill_merge", "hy_paged_decode_append", "hy_paged_decode_append_noalloc"}


class NoLaunch:
    def __init__(self, lib):
        self.lib = lib

    def __getattr__(self, name):
        return (lambda *args: 0) if name in LAUNCHES else getattr(self.lib, name)


@pytest.fixture
def streams(monkeypatch):
    """`now[0]` is the current stream; `recorded` holds (address, stream) of every tensor named
    to the allocator."""
    now, recorded, lib = ["A"], set(), NoLaunch(_native.lib())
    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    monkeypatch.setattr(pc, "_stream_handle", lambda device: now[0])
    monkeypatch.setattr(_native, "lib", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(torch.Tensor, "record_stream",
                        lambda self, s: recorded.add((self.data_ptr(), s)), raising=False)
    return now, recorded


def rows(n, heads):
    return torch.zeros(n, heads, 128, dtype=torch.bfloat16)


def call(batch, name, n, heads=(32, 8)):
    q, k = rows(n, heads[0]), rows(n, heads[1])
    if not batch.varlen:
        q, k = q.view(batch.num_seqs, -1, heads[0], 128), k.view(batch.num_seqs, -1, heads[1], 128)
    if name == "write":
        batch.write_layer(0, *[k if batch.varlen else k.transpose(1, 2)] * 2)
    elif name == "append":
        batch.norm_rope_write_layer(0, q, k, k, None, None, 1e-6, None, None)
    elif name == "attend":
        batch.attend_layer(q if batch.varlen else q.transpose(1, 2), 0)
    else:
        batch.decode_layer(0, q, k, k, None, None, 1e-6, None, None)


def begin(kind):
    m = PagedKVCacheManager(1, 8, 128, 16 * 128, 128, 2, torch.bfloat16, "cpu")
    h = m.allocate()
    m.reserve(h, 1500)
    h.length = 1500
    if kind == "tree":
        return m.begin_tree([h], [chain(40)]), 40
    if kind == "tick":
        return m.begin_tick([h], [40]), 40
    return m.begin_batch([h], 1), 1


@pytest.mark.parametrize("kind,name", [
    ("tree", "write"), ("tree", "append"), ("tree", "attend"),
    ("tick", "write"), ("tick", "append"), ("tick", "attend"),
    ("decode", "write"), ("decode", "append"), ("decode", "attend"), ("decode", "fused")])
def test_metadata_is_recorded_on_the_stream_that_reads_it(streams, kind, name):
    now, recorded = streams
    batch, n = begin(kind)
    meta = batch._meta.data_ptr()
    call(batch, name, n)
    assert not recorded  # on its own stream nothing is to be said
    now[0] = "B"
    call(batch, name, n)
    assert (meta, "B") in recorded


@pytest.mark.parametrize("kind", ["tree", "tick", "decode"])
def test_lists_made_on_a_second_stream(streams, kind):
    """Planned by the first attend_layer, on another stream than the metadata was made on: that
    stream reads foreign metadata, and a third one foreign lists as well."""
    now, recorded = streams
    batch, n = begin(kind)
    meta = batch._meta.data_ptr()
    now[0] = "B"
    call(batch, "attend", n)
    assert recorded == {(meta, "B")}
    plan = batch.plan(32)
    lists = plan.lists if kind == "tree" else plan.decode if kind == "decode" else plan.prefill
    now[0] = "C"
    call(batch, "attend", n)
    assert {(meta, "C"), (lists.data_ptr(), "C")} <= recorded
    # the partials, too
    space = plan.prefill_workspace if kind == "tick" else plan.workspace
    assert space is not None and (space.data_ptr(), "C") in recorded
    now[0] = "A"
    recorded.clear()
    call(batch, "write", n)
    assert (meta, "A") not in recorded
