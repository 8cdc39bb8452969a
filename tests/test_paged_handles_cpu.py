"""Objects of a closed context: their calls are refused, whatever context they
are made with (a new one may lie where the closed one lay)."""
from __future__ import annotations

import ctypes
import types

import pytest

import qasr_attn as Q


class _Lib:
    """Destroys nothing: there is nothing behind the numbers."""

    def __init__(self):
        self.gone = []

    def __getattr__(self, name):
        return lambda h: self.gone.append((name, h.value))


@pytest.fixture
def lib(monkeypatch):
    x = _Lib()
    monkeypatch.setattr(Q, "load", lambda: x)
    return x


def _made(cls, n, **members):
    x = object.__new__(cls)
    x.__dict__.update(members, _handle=ctypes.c_void_p(n))
    return x


def _objects():
    ctx = types.SimpleNamespace(handle=ctypes.c_void_p(1))
    pool = _made(Q.PagePool, 2, ctx=ctx)
    mem = types.SimpleNamespace(handle=ctypes.c_void_p(3), close=lambda: None)
    return ctx, pool, [pool, _made(Q.BeamSelect, 4, ctx=ctx)] + [
        _made(c, 0, ctx=ctx, pool=pool, _mem=mem) for c in (Q.PagedPlan, Q.PagedFork)]


def test_no_handle_without_the_context(lib):
    ctx, pool, objects = _objects()
    assert [x.handle.value for x in objects] == [2, 4, 3, 3]
    ctx.handle = None
    assert [x.handle for x in objects] == [None] * 4
    pool.close()
    objects[1].close()
    assert lib.gone == [("qasr_pages_destroy", 2), ("qasr_beam_destroy", 4)], "and still closed"
    pool.close()
    assert len(lib.gone) == 2


def test_no_handle_without_the_pool(lib):
    _, pool, objects = _objects()
    pool.close()
    assert [x.handle for x in objects[2:]] == [None] * 2
    assert objects[1].handle.value == 4
    objects[1].close()
    assert objects[1].handle is None
