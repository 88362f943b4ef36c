"""The index tables of packed documents: what a captured graph reads lives on, whatever the caches drop.  On the CPU, with the native
call, the tables' device and the capture replaced."""
import contextlib
import gc
import weakref
from functools import lru_cache

import pytest
import torch

from openkimi_b200 import _lib, gated_delta, ops


class _Rows:
    """What the Python side looks at of a tensor on a device."""

    is_cuda, device = True, torch.device("cuda", 0)

    def __init__(self, *shape):
        self.shape = torch.Size(shape)

    def dim(self):
        return len(self.shape)


class _Native:
    def __init__(self):
        self.seen = []

    def env_flags(self):
        return 0

    def chunk_gdr(self, *args):
        self.seen.append([weakref.ref(t) for t in args if isinstance(t, torch.Tensor)])

    chunk_kda = chunk_gdr


@pytest.fixture
def native(monkeypatch):
    table = lambda cu, device: torch.tensor(cu)  # noqa: E731
    monkeypatch.setattr(ops, "_chunk_tables_cached", lru_cache(maxsize=64)(lambda cu, device: (table(cu, device), table(cu, device), 7, table(cu, device), 3)))
    monkeypatch.setattr(gated_delta, "_offsets", lru_cache(maxsize=64)(table))
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    native = _Native()
    monkeypatch.setattr(_lib, "host", lambda: native)
    monkeypatch.setattr(ops, "_in_graphs", {})
    return native


def _call(kind, cu):
    q = _Rows(1, 4096, 1, 64)
    if kind == "gdr":
        gated_delta.chunk_gated_delta_rule(q, q, q, q, q, cu_seqlens_cpu=cu)
    else:
        ops.chunk_kda(q, q, q, q, q, cu_seqlens=_Offsets(), cu_seqlens_cpu=cu)


class _Offsets:
    """The caller's offsets on the device."""

    def to(self, **kw):
        return self

    def contiguous(self):
        return self


@pytest.mark.parametrize("kind", ["gdr", "kda"])
def test_a_layout_captured_twice_with_evictions_between(native, monkeypatch, kind):
    capturing = False
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    cu = torch.tensor([0, 70, 300])
    graphs = []
    for _ in range(3):
        _call(kind, cu)  # (warm-up: the tables are made outside a capture)
        capturing = True
        _call(kind, cu)
        graphs.append(native.seen[-1])
        capturing = False
        for i in range(70):
            _call(kind, torch.tensor([0, 1 + i, 301]))
        gc.collect()
        for tables in graphs:
            assert len(tables) >= 3 and all(t() is not None for t in tables)


def test_tables_of_other_layouts_go(native, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for i in range(70):
        _call("gdr", torch.tensor([0, 1 + i, 301]))
    gc.collect()
    assert all(t() is None for t in native.seen[0]) and all(t() is not None for t in native.seen[-1])
