"""What verification and eviction refuse, without a GPU."""

import pytest
import torch

from hayate_amd import PagedKVCacheManager
from hayate_amd.sampler import verify_tree

TREES = [[-1, 0, 0], [-1, 0]]


def manager(requests=2):
    return PagedKVCacheManager(1, 1, 128, 1024, 128, requests, torch.bfloat16, "cpu")


def call(trees=TREES, **kw):
    m = manager(len(trees))
    batch = m.begin_tree([m.allocate() for _ in trees], trees)
    n, b = batch.total_tokens, batch.num_seqs
    args = {"logits": torch.zeros(n, 50, dtype=torch.bfloat16), "tokens": torch.zeros(n, dtype=torch.long),
            "temperature": [1.0] * b, "top_k": [None] * b, "top_p": [None] * b,
            "uniforms": torch.zeros(n + b), "draft_probs": None, **kw}
    return verify_tree(kw.pop("batch", batch), *[args[x] for x in (
        "logits", "tokens", "temperature", "top_k", "top_p", "uniforms", "draft_probs")])


@pytest.mark.parametrize("kw,error", [
    ({"logits": torch.zeros(5, 50)}, TypeError),
    ({"logits": torch.zeros(4, 50, dtype=torch.bfloat16)}, ValueError),
    ({"logits": torch.zeros(5, 2, 50, dtype=torch.bfloat16)}, ValueError),
    ({"logits": torch.zeros(5, 0, dtype=torch.bfloat16)}, ValueError),
    ({"tokens": torch.zeros(5, dtype=torch.int32)}, TypeError),
    ({"tokens": torch.zeros(4, dtype=torch.long)}, ValueError),
    ({"uniforms": torch.zeros(7, dtype=torch.float64)}, TypeError),
    ({"uniforms": torch.zeros(5)}, ValueError),
    ({"temperature": [1.0]}, ValueError), ({"temperature": [1.0, -1.0]}, ValueError),
    ({"temperature": [1.0, 1e-40]}, ValueError), ({"temperature": [1.0, float("nan")]}, ValueError),
    ({"top_k": [0, None]}, ValueError), ({"top_k": [2.5, None]}, ValueError),
    ({"top_p": [0.0, None]}, ValueError), ({"top_p": [1.5, None]}, ValueError),
    ({"top_p": [None]}, ValueError),
    ({"trees": [[-1, -1, 0], [-1, 0]]}, ValueError),
    ({"draft_probs": torch.zeros(5, 50)}, NotImplementedError),
    ({"trees": [[-1, 0, 1], [-1, 0]], "draft_probs": torch.zeros(5, 50).double()}, TypeError),
    ({"trees": [[-1, 0, 1], [-1, 0]], "draft_probs": torch.zeros(5, 49)}, ValueError),
    ({"batch": "a batch"}, TypeError),
    ({}, RuntimeError),  # no GPU
])
def test_verification_refuses(kw, error):
    with pytest.raises(error):
        call(**kw)


def test_the_batch_has_its_parents_on_the_device():
    m = manager()
    batch = m.begin_tree([m.allocate(), m.allocate()], TREES)
    assert batch.packed_parents.tolist() == [-1, 0, 0, -1, 0] and batch.levels == 2
    assert batch.positions.tolist() == [0, 1, 1, 0, 1]


@pytest.mark.parametrize("kw,error", [
    ({"budget": 0}, ValueError), ({"budget": 2.0}, TypeError), ({"budget": True}, TypeError),
    ({"budget": 10, "sinks": 6, "recent": 5}, ValueError), ({"budget": 10, "sinks": -1}, ValueError),
    ({"budget": 10, "recent": -1}, ValueError), ({"budget": 40}, RuntimeError),
])
def test_eviction_refuses(kw, error):
    m = manager()
    h = m.allocate()
    m.reserve(h, 100)
    h.length = 100
    budget = kw.pop("budget")
    for f in (m.keep_positions, m.evict):
        with pytest.raises(error):
            f([h], torch.zeros(2, 200), budget, **{"sinks": 0, "recent": 0, **kw})
    assert h.length == 100


def test_eviction_refuses_handles():
    m = manager()
    h = m.allocate()
    with pytest.raises(ValueError, match="twice"):
        m.evict([h, h], torch.zeros(2, 200), 10)
    m.release(h)
    for f in (m.keep_positions, m.evict):
        with pytest.raises(RuntimeError, match="released"):
            f([h], torch.zeros(2, 200), 40)
