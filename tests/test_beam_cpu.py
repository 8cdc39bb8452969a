"""Beam selection and forks without a GPU: refusals of the C ABI and the
binding, and the plain implementations themselves."""
from __future__ import annotations

import ctypes
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import beam_model as B  # noqa: E402
import paged8_model as M8  # noqa: E402
import qasr_attn as Q  # noqa: E402
from test_paged_cpu import _ctx, _i, _passed_size_checks, _refused  # noqa: E402


def _f(*shape):
    return torch.zeros(shape)


def test_abi_null_arguments():
    lib = Q.load()
    h = ctypes.c_void_p()
    E = Q.QASR_EINVAL
    assert lib.qasr_pages_create_e4m3(None, 4, 16, ctypes.byref(h)) == E
    assert lib.qasr_pages_get_scales(None, None) == E
    assert lib.qasr_paged_fork_create(None, None, 1, 1, ctypes.byref(h)) == E
    assert lib.qasr_paged_fork_get_info(None, None) == E
    assert lib.qasr_paged_fork(None, None, 1, None, None, None, 1, None, None, None, None) == E
    assert lib.qasr_beam_create(None, 1, 1, 1, 1, ctypes.byref(h)) == E
    assert lib.qasr_beam_select(None, None, 1, None, 1, None, None, -1, None, None, None, None, None) == E
    assert lib.qasr_last_error()
    lib.qasr_paged_fork_destroy(None)
    lib.qasr_beam_destroy(None)


def test_fork_refuses_short_tensors():
    c = _ctx()
    f = types.SimpleNamespace(handle=None, pool=types.SimpleNamespace(pages=10))
    good = dict(lens=_i(3), parent=_i(3), table=_i(3, 4), shared=_i(10), ring=_i(10), cursor=_i(2))
    call = lambda **k: Q.paged_fork(c, f, *{**good, **k}.values())  # noqa: E731
    for bad in (dict(lens=_i(2)), dict(table=_i(2, 4)), dict(table=_i(12)), dict(shared=_i(9)), dict(ring=_i(11)),
                dict(cursor=_i(1))):
        _refused(lambda: call(**bad))
    _passed_size_checks(call)


def test_select_refuses_short_tensors():
    c, s = _ctx(), types.SimpleNamespace(handle=None, width=3, vocab=50, k=4)
    good = dict(logits=_f(6, 50), scores=_f(6), parent=_i(8), token=_i(8), out_scores=_f(8), done=None, eos=-1,
                out_done=None)
    call = lambda **k: Q.beam_select(c, s, *{**good, **k}.values())  # noqa: E731
    for bad in (dict(logits=_f(6, 49)), dict(logits=_f(300)), dict(logits=_f(7, 50)), dict(logits=_f(0, 50)),
                dict(scores=_f(5)), dict(parent=_i(7)), dict(token=_i(7)), dict(out_scores=_f(7)),
                dict(done=_i(5)), dict(out_done=_i(7)), dict(logits=_f(1, 50).expand(6, 50))):
        _refused(lambda: call(**bad))
    with pytest.raises(ValueError):
        call(logits=_f(50, 6).t())
    _passed_size_checks(call)


def test_plain_select():
    x = np.log(np.array([[0.5, 0.3, 0.2], [0.1, 0.1, 0.8]]))
    got = B.select(x, [-1.0, -1.5], 2, 3)
    assert [g[:2] for g in got] == [(0, 0), (1, 2), (0, 1)]
    assert np.allclose([g[2] for g in got], [-1 + np.log(0.5), -1.5 + np.log(0.8), -1 + np.log(0.3)])
    # an ended beam, a dead one, ties, fewer candidates than places
    got = B.select(x, [-1.0, -1.2], 2, 3, done=[0, 1], eos=2)
    assert [g[:2] for g in got] == [(1, 2), (0, 0), (0, 1)] and [g[3] for g in got] == [1, 0, 0]
    got = B.select(np.zeros((2, 2)), [0.0, 0.0], 2, 5)
    assert [g[:2] for g in got] == [(0, 0), (0, 1), (1, 0), (1, 1), (-1, -1)]
    assert [g[:2] for g in B.select(x, [-np.inf, 0.0], 2, 2)] == [(1, 2), (1, 0)]


def test_plain_fork():
    # Two requests share page 9 and have an unfinished page each.
    lens, table = [20, 24, 0], [[9, 1], [9, 2], [-1, -1]]
    shared, ring, cursor = [0] * 10, [3, 4, 5, 6, 7, 8, 0, -1, -1, -1], [0, 7]
    shared[9] = 1
    status, copies = B.fork(lens, [1, 1, 1], table, shared, ring, cursor, 10, 16)
    assert status == [0, 0, 0] and lens == [24, 24, 24]
    assert table == [[9, 3], [9, 2], [9, 4]] and copies == [(2, 3, 8), (2, 4, 8)]
    assert shared[9] == 2 and cursor == [2, 6] and ring[7] == 1
    status, _ = B.fork(lens, [-1, -1, -1], table, shared, ring, cursor, 10, 16)
    assert lens == [0, 0, 0] and shared == [0] * 10 and cursor == [2, 10]
    assert [ring[(8 + k) % 10] for k in range(4)] == [9, 3, 2, 4]


def test_plain_e4m3():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(M8.value(np.arange(256)), t, equal_nan=True)
    x = torch.randn(4000, dtype=torch.float64) * 10 ** torch.empty(4000, dtype=torch.float64).uniform_(-4, 2)
    x = x.float().clamp(-448, 448)
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(M8.nearest(x.double().numpy()), want)
    for top, k in ((0.0, -15), (448.0, 0), (448.5, 1), (224.0, -1), (65504.0, 8), (2.0 ** -24, -15)):
        assert M8.unit(top) == k
