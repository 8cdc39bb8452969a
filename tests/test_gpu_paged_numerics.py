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
from test_gpu_paged_work import some_rows  # noqa: E402
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


# ---- columns computed again -------------------------------------------------

def half_weight(lo=0.5, hi=0.51):
    """f16 numbers (a, b) whose product as a score, a b / sqrt(128), has a
    weight p = exp(score) in [lo, hi] that lies as far from an f16 number as
    can be found, above it; and p."""
    a = np.arange(1.0, 2.0, 2.0 ** -10)
    b = -np.arange(6.0, 8.0, 2.0 ** -8)
    assert np.array_equal(a.astype(np.float16), a) and np.array_equal(b.astype(np.float16), b)
    p = np.exp(a[:, None] * b[None] * HD ** -0.5)
    off = np.where((p >= lo) & (p <= hi), (p - p.astype(np.float16).astype(float)) / p, 0)
    i, j = np.unravel_index(off.argmax(), off.shape)
    assert off[i, j] > 4.5e-4
    return float(a[i]), float(b[j]), float(p[i, j])


def two_weights(pool, table, ps, n, every=8):
    """Keys of one dim: every 8th has weight 1, the others half_weight()'s p.
    Returns the query and p."""
    a, b, w = half_weight()
    set_keys(pool, table, ps, range(n), 0, 0.0)
    keys = [k for k in range(n) if k % every]
    pages, rows = at(table, ps, np.asarray(keys))
    pool[0, pages, 0, :, rows, 0] = b
    return a, w


AGAIN = [(20, 5), (20, 12), (1500, 6), (1500, 12), (0, 2100), (10500, 200)]


@pytest.mark.parametrize("c,r", AGAIN)
def test_columns_computed_again_keep_a_constant_value(gpu, c, r):
    """Every value is 2 - 2^-10, but one of the last row's is not finite: the
    32 dims of it are computed again for all rows of the last row block.  A
    weighted mean of a constant is the constant, however the weights are
    rounded, as long as the mean divides by the sum of the same weights: the
    longest f32 sum has 2100 terms (its divisor's 2100 / 64 a lane), which moves
    the result by less than 2 * (2100 + 33 + 40) * 2^-24 = 2.6e-4, and half a step
    of f16 below 2 is 4.9e-4."""
    ps, value = 16, 2.0 - 2.0 ** -10
    p, pool, table = one(c, r, ps)
    a, _ = two_weights(pool, table, ps, c + r)
    q = torch.zeros((r, QDIM), dtype=torch.float16, device="cuda")
    q.view(r, NQH, HD)[:, :, 0] = a
    set_keys(pool, table, ps, range(c + r), 1, value)
    page, off = at(table, ps, c + r - 1)
    pool[0, page, 1, :, off, 5] = INF
    out = run_attn(p, [(c, r)], i32(table), q).view(r, NQH, HD)
    assert bool(torch.isinf(out[-1, :, 5]).all())
    out[-1, :, 5] = value
    assert bool((out == value).all()), out[out != value][:4]
    p.close()


@pytest.mark.parametrize("c,r", [(30, 7), (900, 8), (2000, 5), (900, 14), (2500, 13), (300, 90)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_columns_computed_again_against_64_bits(gpu, c, r, what):
    """A bad key in the middle of the new rows: the rows before it, and where
    its value is bad the other dims of the rows after it, are within the bound
    of the definition."""
    ps, row = 32, r // 2
    p, pool, table = one(c, r, ps)
    page, off = at(table, ps, c + row)
    kept = pool[0, page, :, :, off].clone()
    if what == "k":
        pool[0, page, 0, :, off, 3] = NAN
    else:
        pool[0, page, 1, :, off, 5] = INF
    q = randn(6, r, QDIM)
    out = run_attn(p, [(c, r)], i32(table), q)
    pool[0, page, :, :, off] = kept
    check_rows(p, table, q, out, c, list(range(row)), heads=range(0, NQH, 3))
    seers = out[row:].view(-1, NQH, HD)
    if what == "k":
        assert bool(torch.isnan(seers).all())
    else:
        assert bool(torch.isinf(seers[:, :, 5]).all())
        pool[0, page, 1, :, off, 5] = 0.0  # a dim of its own: set alike on both sides
        seers[:, :, 5] = 0
        rows = list(range(row, r))
        keep = pool.clone()
        pool[:, :, 1, :, :, 5] = 0
        check_rows(p, table, q, out, c, rows, heads=range(0, NQH, 3))
        pool.copy_(keep)
    p.close()


# ---- what others hold -------------------------------------------------------

@pytest.mark.parametrize("c,r,evicted", [(1000, 1, (4, 40)), (1000, 6, (0, 60)), (700, 12, (1, 30)),
                                         (300, 100, (0, 18)), (5200, 400, (10, 300)), (0, 2100, (0, 0))])
def test_bits_do_not_depend_on_the_pages_of_others(gpu, c, r, evicted):
    """A request with evicted pages, beside one that holds page 0: whatever
    page 0 holds, the first one's bits are the same."""
    ps = 16
    p, pool, table = one(c, r, ps, mate=1)
    table[0][evicted[0]:evicted[1]] = [(-1, p.pool.pages, 2 ** 31 - 1)[i % 3] for i in range(*evicted)]
    both = i32([table[0], [0] + [-1] * (len(table[0]) - 1)])
    q = randn(6, r + 1, QDIM)
    outs = []
    for value in (0.5, NAN, INF, -INF, 65504.0):
        pool[0, 0] = value
        outs.append(run_attn(p, [(c, r), (7, 1)], both, q)[:r].clone())
    for out in outs:
        assert torch.equal(out, outs[0])
    check_rows(p, table, q, outs[0], c, some_rows(r, random.Random(1)))
    p.close()


# ---- the weights' bits --------------------------------------------------------

@pytest.mark.parametrize("c,r", [(300, 1), (250, 8), (767, 1), (760, 3), (2000, 2), (40, 24)])
def test_few_rows_hold_their_weights_to_22_bits(gpu, c, r):
    """Items of up to 8 rows, a lone row's among them, weigh keys as the slot
    pool's decode step does: not rounded to f16.  Every 8th key has weight 1
    and value 1, the others weight p, just above an f16 number by 4.8e-4 of
    it, and value -1/4: the mean of n1 keys and n2 others is (n1 - n2 p / 4) /
    (n1 + n2 p), and f16 weights move it by about 1e-4, while it is about 0.03
    and its own f16 rounding 1.5e-5.
    Scores are single products: 3 roundings of an exponent near 1, exp2's error
    and the split of a weight (2^-22) are below 2^-20 of it together.  A wave
    adds the two products of each key of its quarter of the keys (n / 2 f32
    sums), then the waves and up to 32 ranges join; the weights' own sum has n /
    16 terms a lane: (0.6 n + 80) 2^-24 of the mean |v|."""
    ps = 16
    p, pool, table = one(c, r, ps)
    a, w = two_weights(pool, table, ps, c + r)
    q = torch.zeros((r, QDIM), dtype=torch.float16, device="cuda")
    q.view(r, NQH, HD)[:, :, 0] = a
    ones = range(0, c + r, 8)
    set_keys(pool, table, ps, range(c + r), 1, -0.25)
    set_keys(pool, table, ps, ones, 1, 1.0)
    out = run_attn(p, [(c, r)], i32(table), q).double().cpu().numpy()
    rows = range(r) if r <= 8 else range(16, r)  # the last row block of a chunk
    for row in rows:
        n = c + row + 1
        n1 = len(range(0, n, 8))
        n2 = n - n1
        want = (n1 - 0.25 * n2 * w) / (n1 + n2 * w)
        f16 = float(np.float16(w))
        moved = abs((n1 - 0.25 * n2 * f16) / (n1 + n2 * f16) - want)
        mean = (n1 + 0.25 * n2 * w) / (n1 + n2 * w)
        allow = (2.0 ** -20 + (0.6 * n + 80) * 2.0 ** -24) * mean + 2.0 ** -11 * abs(want) + 2.0 ** -25
        assert moved > 2 * allow, "f16 weights would pass"
        assert np.abs(out[row] - want).max() <= allow, (row, np.abs(out[row] - want).max(), allow, moved)
    p.close()


@pytest.mark.parametrize("c,r", [(500, 1), (500, 8), (1500, 2)])
def test_few_rows_keep_small_weights(gpu, c, r):
    """Weights of about 2^-16 of the largest, which f16 holds to 9 bits, and
    values of 1000 on them: one key of weight 1 and value 1 a slice, the others
    b.  The result's f16 rounding is 2^-11 of it, the exponent of 16 is off by
    2^-20 and exp2 by less (2^-19), a weight below 2^-21 is held to 2^-32 of the
    largest, and the f32 sums move it by (0.6 n + 80) 2^-24."""
    ps = 16
    a = 1.0
    b = float(np.float16(-16.56 * np.log(2.0) * HD ** 0.5))
    w = float(np.exp(a * b * HD ** -0.5))
    near = float(np.float16(w))
    assert abs(near - w) / w > 2.5e-3
    p, pool, table = one(c, r, ps)
    set_keys(pool, table, ps, range(c + r), 0, 0.0)
    small = [k for k in range(c + r) if k % 16]
    pages, rows = at(table, ps, np.asarray(small))
    pool[0, pages, 0, :, rows, 0] = b
    set_keys(pool, table, ps, range(c + r), 1, 0.0)
    set_keys(pool, table, ps, small, 1, 1000.0)
    q = torch.zeros((r, QDIM), dtype=torch.float16, device="cuda")
    q.view(r, NQH, HD)[:, :, 0] = a
    out = run_attn(p, [(c, r)], i32(table), q).double().cpu().numpy()
    for row in range(r):
        n = c + row + 1
        n1 = len(range(0, n, 16))
        n2 = n - n1
        want = 1000 * n2 * w / (n1 + n2 * w)
        allow = want * (2.0 ** -11 + 2.0 ** -19 + 2.0 ** -32 / w + (0.6 * n + 80) * 2.0 ** -24)
        assert np.abs(out[row] - want).max() <= allow, (row, out[row][:2], want, allow)
    p.close()


# ---- scores past 2^24 -------------------------------------------------------

MILLIONS = [(20, 1), (20, 7), (20, 12), (1500, 1), (1500, 6), (1500, 12), (0, 2100), (10500, 200)]


@pytest.mark.parametrize("c,r,again", [(*x, False) for x in MILLIONS] + [(*x, True) for x in MILLIONS if x[1] > 1])
def test_scores_of_millions_pick_their_key(gpu, c, r, again):
    """Scores of 10^8, where a step of f32 is 8 to 64: a row's largest score
    leads by more than any rounding (128 products of f32: 2^-17 sum |q k|, 10^4
    here), so its key's value is the result, to the bit.  `again`: and the last
    row's value is not finite, so that the columns of its block are computed
    again."""
    ps = 16
    p, pool, table = one(c, r, ps)
    pool[:, :, 0] = randn(8, *pool[:, :, 0].shape, std=1e4)
    q = randn(6, r, QDIM, std=1e4)
    if again:
        page, off = at(table, ps, c + r - 1)
        pool[0, page, 1, :, off, 5] = INF
    out = run_attn(p, [(c, r)], i32(table), q).view(r, NQH, HD)
    rows = [x for x in some_rows(r, random.Random(1)) if x < r - 1 or not again]
    kv = pool[0, torch.tensor(table[0]).cuda()]
    checked = 0
    for h in (0, 15):
        k, v = (kv[:, s, h // 2].reshape(-1, HD)[:c + r] for s in (0, 1))
        s = (q.view(r, NQH, HD)[rows, h].double().cpu() @ k.double().cpu().T) * HD ** -0.5
        s[torch.arange(c + r)[None] > torch.tensor([c + x for x in rows])[:, None]] = -INF
        top = s.topk(2, dim=1)
        lead = (top.values[:, 0] - top.values[:, 1]) > 2e4
        checked += int(lead.sum())
        want = v[top.indices[:, 0].cuda()][lead.cuda()]
        assert torch.equal(out[rows, h][lead.cuda()], want), (h, (out[rows, h][lead.cuda()] != want).sum())
    assert checked >= len(rows)
    p.close()
