"""Rows, tables and weights that the kernels would read past, refused before any launch. Without
a GPU: the kernels are a stand-in that launches nothing, and `meta` is the other device."""

import pytest
import torch

import hayate_amd.paged_cache as pc
from hayate_amd import PagedKVCacheManager, _native
from tree_util import chain

BF16 = torch.bfloat16


class NoLaunch:
    def __getattr__(self, name):
        if name.startswith(("hy_kv_append", "hy_qknorm", "hy_paged")):
            return lambda *args: 0
        return getattr(LIB, name)


LIB = _native.lib()


@pytest.fixture
def m(monkeypatch):
    monkeypatch.setattr(pc, "_require_hip", lambda t, what: None)
    monkeypatch.setattr(_native, "lib", NoLaunch)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    return PagedKVCacheManager(1, 8, 128, 16 * 128, 128, 2, BF16, "cpu")


def batches(m):
    h = m.allocate()
    yield m.begin_tree([h], [chain(6)]), lambda n, heads, dim=128, **kw: torch.zeros(n, heads, dim, **kw)
    yield m.begin_tick([h], [6]), lambda n, heads, dim=128, **kw: torch.zeros(n, heads, dim, **kw)
    yield m.begin_batch([h], 6), lambda n, heads, dim=128, **kw: torch.zeros(1, n, heads, dim, **kw)
    yield m.begin_batch([h], 1), lambda n, heads, dim=128, **kw: torch.zeros(1, n, heads, dim, **kw)


def test_rows_of_another_shape(m):
    for batch, rows in batches(m):
        n = batch.total_tokens
        q, k = rows(n, 32, dtype=BF16), rows(n, 8, dtype=BF16)

        def append(q=q, k=k, v=None):
            return batch.norm_rope_write_layer(0, q, k, k if v is None else v, None, None, 1e-6,
                                               None, None)

        append()
        # a head of the wrong size, too few and too many tokens, for q and for k and v
        bad_q = [rows(n, 32, 64, dtype=BF16), rows(n, 32, 256, dtype=BF16), rows(n + 1, 32, dtype=BF16),
                 rows(n - 1, 32, dtype=BF16)]
        bad_k = [rows(n, 8, 64, dtype=BF16), rows(n + 1, 8, dtype=BF16), rows(n - 1, 8, dtype=BF16)]
        if not batch.varlen:
            bad_q.append(q.expand(2, -1, -1, -1).contiguous())
            bad_k.append(k.expand(2, -1, -1, -1).contiguous())
        for x in bad_q:
            with pytest.raises(ValueError):
                append(q=x)
            with pytest.raises(ValueError):
                batch.attend_layer(x if batch.varlen else x.transpose(1, 2), 0)
            if batch.decode_only:
                with pytest.raises(ValueError):
                    batch.decode_layer(0, x, k, k, None, None, 1e-6, None, None)
        for x in bad_k:
            with pytest.raises(ValueError):
                append(k=x)
            with pytest.raises(ValueError):
                y = x if batch.varlen else x.transpose(1, 2)
                batch.write_layer(0, y, y)


def test_rows_tables_and_weights_elsewhere(m):
    for batch, rows in batches(m):
        n = batch.total_tokens
        q, k = rows(n, 32, dtype=BF16), rows(n, 8, dtype=BF16)
        w, table = torch.zeros(128, dtype=BF16), torch.zeros(2048, 128)
        good = dict(q=q, k=k, v=k, qw=w, kw=w, cos=table, sin=table)

        def append(**kw):
            x = {**good, **kw}
            return batch.norm_rope_write_layer(0, x["q"], x["k"], x["v"], x["qw"], x["kw"], 1e-6,
                                               x["cos"], x["sin"])

        append()
        for name, t in good.items():
            with pytest.raises(ValueError):
                append(**{name: t.to("meta")})
        with pytest.raises(ValueError):
            batch.write_layer(0, *[(k if batch.varlen else k.transpose(1, 2)).to("meta")] * 2)
        with pytest.raises(ValueError):
            batch.attend_layer((q if batch.varlen else q.transpose(1, 2)).to("meta"), 0)


def test_tables_of_another_shape(m):
    for batch, rows in batches(m):
        n = batch.total_tokens
        q, k = rows(n, 32, dtype=BF16), rows(n, 8, dtype=BF16)
        full = torch.zeros(2048, 128)
        for cos, sin in ((full[:, :64], full[:, :64]), (full, full[:100]), (full, full[:, :64]),
                         (full.view(-1), full.view(-1))):
            with pytest.raises(ValueError):
                batch.norm_rope_write_layer(0, q, k, k, None, None, 1e-6, cos, sin)
