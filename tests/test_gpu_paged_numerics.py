"""The paged attention's arithmetic at its edges, for items of up to 8 rows, of
up to 16 and of 64, split and not."""
from __future__ import annotations

import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_model as M  # noqa: E402
import qasr_attn as Q  # noqa: E402
from test_gpu_paged import Paged, i32, randn, run_attn, shuffled_table  # noqa: E402
from test_gpu_paged_work import needed, some_rows  # noqa: E402
from workloads import HD, NQH, QDIM  # noqa: E402

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def kind(c, r):
    """(rows of an item: 8, 16 or 64; split or not) of r rows after c keys."""
    block, _, splits = Q.plan_paged(c, r)
    return (8 if r <= 8 else block), splits > 1


def one(c, r, ps, spare=2, seed=4, mate=0):
    """A pool with one request of r rows after c keys, keys and queries
    normal.  `mate` further pages are a second request's, which has page 0."""
    need = -(-(c + r) // ps)
    table, _ = shuffled_table(random.Random(seed), [need], need + spare, need)
    if 0 in table[0]:  # page 0 stays with others
        table[0][table[0].index(0)] = next(x for x in range(1, need + spare) if x not in table[0])
    p = Paged(need + spare, ps, 1 + bool(mate), r + mate, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    return p, pool, table


def at(table, ps, key):
    """A key's page and row, for indexing the pool: a number or a range."""
    t = np.asarray(table[0])
    return torch.tensor(t[np.asarray(key) // ps]).cuda(), torch.tensor(np.asarray(key) % ps).cuda()


def set_keys(pool, table, ps, keys, kv, value):
    pages, rows = at(table, ps, np.asarray(list(keys)))
    pool[0, pages, kv, :, rows] = value


def check_rows(p, table, q, out, c, rows, hidden=(), heads=(0, 15)):
    """Rows `rows` against the definition in 64 bits over the keys that are
    in the pool and not in `hidden` (their scores are -inf: they weigh
    nothing)."""
    ps, pool = p.pool.page_rows, p.pool.tensor()[0]
    n = c + max(rows) + 1
    ids = np.asarray(table[0][:-(-n // ps)])
    ok = (ids >= 0) & (ids < p.pool.pages)
    seen = np.repeat(ok, ps)[:n]
    seen[[k for k in hidden if k < n]] = False
    kv = pool[torch.tensor(np.where(ok, ids, 0)).cuda()]
    for h in heads:
        x = kv[:, :, h // 2].double().cpu().numpy()
        k, v = (np.where(seen[:, None], x[:, s].reshape(-1, HD)[:n], 0) for s in (0, 1))
        cols = slice(h * HD, (h + 1) * HD)
        want, bound = M.attend(q[rows][:, cols].double().cpu().numpy(), k, v, [c + r for r in rows], seen)
        d = np.abs(out[rows][:, cols].double().cpu().numpy() - want)
        assert (d <= bound).all(), (h, float(np.nanmax(d / bound)), np.argwhere(~(d <= bound))[:4])


# ---- a key range whose scores are all -inf ----------------------------------

SPLIT = [(1500, 1, (512, 1024)), (1500, 6, (512, 1024)), (1500, 12, (500, 1030)), (10500, 200, (2000, 6000))]


@pytest.mark.parametrize("c,r,gone", SPLIT)
def test_a_range_of_minus_infinity_behind_an_evicted_page(gpu, c, r, gone):
    """A whole range scores -inf but for an evicted page's keys; what page 0
    holds, infinities, is nobody's here."""
    assert kind(c, r)[1]
    ps = 16
    p, pool, table = one(c, r, ps)
    q = randn(6, r, QDIM).abs()  # so that a key of -inf scores -inf
    set_keys(pool, table, ps, range(*gone), 0, -INF)
    table[0][(gone[0] + gone[1]) // 2 // ps] = -1
    pool[0, 0, 1] = INF
    out = run_attn(p, [(c, r)], i32(table), q)
    check_rows(p, table, q, out, c, some_rows(r, random.Random(1)), range(*gone))
    p.close()


@pytest.mark.parametrize("c,r,first", [(1500, 6, 1024), (1500, 12, 1000), (10500, 200, 9000)])
@pytest.mark.parametrize("bad", [INF, NAN])
def test_a_range_of_minus_infinity_before_a_later_rows_value(gpu, c, r, first, bad):
    """The last range scores -inf throughout, and a later row's value in it is
    not finite: the rows that do not see it are the definition, those that do
    have a weight of 0 times it, NaN, in that dim alone."""
    assert kind(c, r)[1]
    ps, row = 16, r * 3 // 4
    p, pool, table = one(c, r, ps)
    q = randn(6, r, QDIM).abs()
    set_keys(pool, table, ps, range(first, c + r), 0, -INF)
    page, off = at(table, ps, c + row)
    pool[0, page, 1, :, off, 5] = bad
    out = run_attn(p, [(c, r)], i32(table), q)
    seers = out[row:].view(-1, NQH, HD).clone()
    pool[0, page, 1, :, off, 5] = 0.0
    check_rows(p, table, q, out, c, [x for x in some_rows(r, random.Random(1)) if x < row], range(first, c + r))
    assert bool(torch.isnan(seers[:, :, 5]).all())
    seers[:, :, 5] = 0
    assert bool(torch.isfinite(seers).all())
    p.close()


@pytest.mark.parametrize("c,r", [(20, 1), (20, 12), (1500, 1), (1500, 6), (1500, 12), (0, 2100), (10500, 200)])
@pytest.mark.parametrize("bad", [INF, NAN])
def test_only_scores_of_minus_infinity_give_zeros(gpu, c, r, bad):
    """Whatever the values are."""
    ps = 16
    p, pool, table = one(c, r, ps)
    q = randn(6, r, QDIM).abs()
    set_keys(pool, table, ps, range(c + r), 0, -INF)
    page, off = at(table, ps, (c + r) // 2)
    pool[0, page, 1, :, off, 5] = bad
    out = run_attn(p, [(c, r)], i32(table), q)
    assert bool((out == 0).all())
    p.close()
