"""The paged KV cache without a GPU: refusals of the C ABI and the binding, and
the capacities that the plan's workspaces are allocated for."""
from __future__ import annotations

import ctypes
import types

import pytest

torch = pytest.importorskip("torch")

import qasr_attn as Q  # noqa: E402

NQH, NKVH, HD = 16, 8, 128
TOT, QD = (NQH + 2 * NKVH) * HD, NQH * HD


def _ctx():
    cfg = types.SimpleNamespace(head_dim=HD, num_attention_heads=NQH, num_key_value_heads=NKVH)
    return types.SimpleNamespace(cfg=cfg, nqh=NQH, nkvh=NKVH, handle=None, device=0)


def _plan(nreq=2):
    return types.SimpleNamespace(handle=None, nreq=nreq, pool=types.SimpleNamespace(pages=10))


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _h(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def _refused(fn):
    with pytest.raises(Q.QasrError) as e:
        fn()
    assert e.value.code == Q.QASR_EINVAL


def _passed_size_checks(fn):
    with pytest.raises(ValueError, match="GPU"):
        fn()


def test_abi_null_arguments():
    lib = Q.load()
    h = ctypes.c_void_p()
    E = Q.QASR_EINVAL
    assert lib.qasr_pages_create(None, 4, 16, ctypes.byref(h)) == E
    assert lib.qasr_pages_get_info(None, None) == E
    assert lib.qasr_paged_plan_create(None, None, 1, 1, ctypes.byref(h)) == E
    assert lib.qasr_paged_plan_get_info(None, None) == E
    assert lib.qasr_paged_plan_build(None, None, 1, None, None, None, 1, None, None, None) == E
    assert lib.qasr_paged_append(None, None, 0, 1, None, None, None, None, None) == E
    assert lib.qasr_paged_attn(None, None, 0, 1, None, 1, None, None, None) == E
    assert lib.qasr_last_error()
    lib.qasr_pages_destroy(None)
    lib.qasr_paged_plan_destroy(None)


def test_plan_refuses_short_tensors():
    c, p = _ctx(), _plan()
    call = lambda *a: Q.paged_plan(c, p, *a)  # noqa: E731
    _refused(lambda: call(_i(1), _i(2), _i(2, 4)))                       # lens
    _refused(lambda: call(_i(2), _i(2), _i(1, 4)))                       # table
    _refused(lambda: call(_i(2), _i(2), _i(8)))                          # table of one dimension
    _refused(lambda: call(_i(2), _i(2), _i(2, 4), _i(9), _i(2)))         # ring
    _refused(lambda: call(_i(2), _i(2), _i(2, 4), _i(10), _i(1)))        # cursor
    _refused(lambda: call(_i(2), _i(2), _i(2, 4), _i(10)))               # ring alone
    _refused(lambda: call(_i(2), _i(2), _i(2, 4), None, _i(2)))
    _passed_size_checks(lambda: call(_i(2), _i(2), _i(2, 4), _i(10), _i(2)))


def test_append_and_attn_refuse_short_tensors():
    c, p, g = _ctx(), _plan(), _h(HD)
    _refused(lambda: Q.paged_append(c, p, 0, _h(3, TOT - 1), g, g, _h(3, QD)))
    _refused(lambda: Q.paged_append(c, p, 0, _h(3 * TOT), g, g, _h(3, QD)))
    _refused(lambda: Q.paged_append(c, p, 0, _h(3, TOT), g, g, _h(2, QD)))
    _refused(lambda: Q.paged_append(c, p, 0, _h(3, TOT), _h(64), g, _h(3, QD)))
    _passed_size_checks(lambda: Q.paged_append(c, p, 0, _h(3, TOT), g, g, _h(3, QD)))
    _refused(lambda: Q.paged_attn(c, p, 0, _i(1, 4), _h(3, QD), _h(3, QD)))
    _refused(lambda: Q.paged_attn(c, p, 0, _i(2, 4), _h(3, TOT), _h(3, QD)))
    _refused(lambda: Q.paged_attn(c, p, 0, _i(2, 4), _h(3, QD), _h(2, QD)))
    _passed_size_checks(lambda: Q.paged_attn(c, p, 0, _i(2, 4), _h(3, QD), _h(3, QD)))


def test_shapes_fit_the_workspaces():
    """Every (length, rows) stays within what a plan allocates: 32 records a
    row and 2048 a request, 64 items (32 with up to 16 row blocks or with row
    blocks of 64 rows) or one a row block."""
    seen = set()
    for rows in list(range(1, 140)) + [255, 256, 257, 511, 512, 1000, 2048, 4097, 16384, 65536]:
        for length in (0, 1, 100, 496, 511, 512, 513, 1024, 5000, 8192, 16383, 1 << 20, 1 << 24):
            block, n, splits = Q.plan_paged(length, rows)
            assert n == -(-rows // block) and 1 <= splits <= 32
            assert n * splits <= max(64 if block == 16 and n > 16 else 32, n)
            if splits > 1:
                assert rows * splits <= min(32 * rows, 2048)
                # no range is empty: a row block has at least as many tiles
                assert -(-(length + min(rows, block)) // 128) >= splits
            seen.add((block, min(splits, 2)))
    assert seen == {(16, 1), (16, 2), (64, 1), (64, 2)}


def test_plan_paged_refuses():
    for length, rows in ((-1, 1), (0, 0), (0, -3), ((1 << 24) + 1, 1), (0, 65537)):
        _refused(lambda: Q.plan_paged(length, rows))


def test_ranges_of_a_short_context():
    """A plan's split state counts on it: no request of a context of max_seq
    positions has more than ceil(max_seq / 512) ranges."""
    for max_seq in (1, 511, 512, 513, 1024, 1025, 2048, 5000, 16384):
        for rows in {1, 2, 15, 16, 17, 64, 65, 255, 256, 257, 300, 513, 1000, 4000, max_seq}:
            for length in {0, 1, 500, max_seq // 2, max_seq - rows - 1, max_seq - rows}:
                if length >= 0 and length + rows <= max_seq:
                    assert Q.plan_paged(length, rows)[2] <= -(-max_seq // 512)
