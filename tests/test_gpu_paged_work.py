"""The paged attention where there is much of it: wide row blocks, more items
than workgroups, long splits, with what a masked place may hold; and the
refusals of the paged entry points through a real context."""
from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_model as M  # noqa: E402
import qasr_attn as Q  # noqa: E402
from gpu_helpers import rope_tables, say  # noqa: E402
from test_gpu_paged import Paged, i32, randn, run_attn, shuffled_table  # noqa: E402
from workloads import HD, NKVH, NQH, QDIM, TOT  # noqa: E402

pytestmark = pytest.mark.gpu


def needed(batch, ps):
    return [-(-(c + r) // ps) for c, r in batch]


def some_rows(r, rnd, n=24):
    """The rows where a row block of 16 or 64 begins or ends, and others."""
    edges = {0, r - 1, 15, 16, 63, 64, 65, r // 64 * 64, r // 64 * 64 - 1, r // 16 * 16}
    return sorted({x for x in edges if 0 <= x < r} | {rnd.randrange(r) for _ in range(n)})


def check_rows(p, batch, table, q, out, layer=0, heads=(0,), seed=1):
    """Some rows of every request against the definition in 64 bits."""
    ps, pages = p.pool.page_rows, p.pool.pages
    pool = p.pool.tensor()[layer]
    rnd = random.Random(seed)
    r0 = 0
    for i, (c, r) in enumerate(batch):
        if r <= 0:
            continue
        rows = some_rows(r, rnd)
        ids = torch.tensor(table[i][:-(-(c + r) // ps)])
        ok = (ids >= 0) & (ids < pages)
        at = torch.where(ok, ids, 0).long().cuda()
        seen = np.repeat(ok.numpy(), ps)[:c + r]
        for h in heads:
            cols = slice(h * HD, (h + 1) * HD)
            kv = pool[at][:, :, h // 2].double().cpu().numpy()
            k = np.where(seen[:, None], kv[:, 0].reshape(-1, HD)[:c + r], 0)
            v = np.where(seen[:, None], kv[:, 1].reshape(-1, HD)[:c + r], 0)
            qs = q[r0:r0 + r][rows][:, cols].double().cpu().numpy()
            got = out[r0:r0 + r][rows][:, cols].double().cpu().numpy()
            want, bound = M.attend(qs, k, v, [c + x for x in rows], seen)
            d = np.abs(got - want)
            assert (d <= bound).all(), (i, h, float((d / bound).max()),
                                        [(rows[a], b) for a, b in np.argwhere(d > bound)[:4]])
        r0 += r


def assert_wide(batch):
    assert any(Q.plan_paged(c, r)[0] == 64 for c, r in batch if r > 0)


WIDE = [
    [(4000, 512)], [(1500, 1100)], [(0, 2048)], [(7000, 300)], [(3600, 575)], [(0, 2051)],
    [(16000, 135)],
    [(900, 1), (4000, 512), (40, 20), (0, 0), (1600, 1090), (3000, 1)],
]


@pytest.mark.parametrize("ps", [16, 64, 256])
@pytest.mark.parametrize("batch", WIDE, ids=lambda b: "+".join(f"{r}@{c}" for c, r in b))
def test_wide_row_blocks_against_64_bits(gpu, ps, batch):
    assert_wide(batch)
    need = needed(batch, ps)
    pages = sum(need) + 2
    table, _ = shuffled_table(random.Random(7), need, pages, max(need) + 1)
    rows = sum(r for _, r in batch)
    p = Paged(pages, ps, len(batch), rows + 2, layers=2, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(11, *pool.shape))
    q = randn(12, rows + 2, QDIM, std=1.5)
    say(f"wide ps={ps} {batch}")
    out = run_attn(p, batch, i32(table), q, layer=1)
    assert bool((out[rows:] == 7).all()), "rows behind the last one are left as they were"
    check_rows(p, batch, table, q, out, layer=1, heads=(0, 13))
    p.close()


@pytest.mark.parametrize("batch", [[(5000, 300)], [(4200, 272)], [(6000, 257), (3, 1), (4100, 400)]],
                         ids=lambda b: "+".join(f"{r}@{c}" for c, r in b))
def test_many_narrow_row_blocks_in_ranges(gpu, batch):
    """More than 16 row blocks of 16 rows, each in two or three ranges."""
    for c, r in batch:
        block, blocks, splits = Q.plan_paged(c, r)
        assert block == 16 and (r == 1 or (blocks > 16 and splits > 1))
    ps, need = 32, needed(batch, 32)
    table, _ = shuffled_table(random.Random(1), need, sum(need) + 1, max(need))
    rows = sum(r for _, r in batch)
    p = Paged(sum(need) + 1, ps, len(batch), rows, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, rows, QDIM)
    out = run_attn(p, batch, i32(table), q).clone()
    check_rows(p, batch, table, q, out, heads=(2, 15))
    assert torch.equal(run_attn(p, batch, i32(table), q), out)
    p.close()


@pytest.mark.parametrize("nkvh", [1, 3, 16])
def test_wide_other_head_counts(gpu, nkvh):
    batch, ps = [(5200, 401), (100, 30), (700, 1)], 32
    assert_wide(batch)
    need = needed(batch, ps)
    table, _ = shuffled_table(random.Random(1), need, sum(need) + 1, max(need))
    rows = sum(r for _, r in batch)
    p = Paged(sum(need) + 1, ps, 3, rows, nkvh=nkvh, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, rows, 2 * nkvh * HD)
    out = run_attn(p, batch, i32(table), q)
    check_rows(p, batch, table, q, out, heads=range(2 * nkvh) if nkvh < 4 else (0, 9, 31))
    p.close()


def test_wide_peaked_scores(gpu):
    """Scores of hundreds, and the running maximum moving late."""
    batch, ps = [(3300, 600)], 64
    assert_wide(batch)
    need = needed(batch, ps)
    table, _ = shuffled_table(random.Random(1), need, sum(need), max(need))
    p = Paged(sum(need), ps, 1, 600, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, 600, QDIM, std=30.0)
    check_rows(p, batch, table, q, run_attn(p, batch, i32(table), q), heads=(2, 9))
    p.close()


@pytest.mark.parametrize("bad", [float("nan"), float("-inf"), -65504.0])
def test_wide_ignores_what_lies_behind_the_keys(gpu, bad):
    batch, ps = [(4000, 513), (12, 2100), (30, 1)], 128
    assert_wide(batch)
    need = needed(batch, ps)
    pages = sum(need) + 3
    table, _ = shuffled_table(random.Random(2), need, pages, max(need) + 2)
    rows = sum(r for _, r in batch)
    p = Paged(pages, ps, 3, rows, rope=False)
    pool = p.pool.tensor()
    x = randn(5, *pool.shape)
    y = torch.full_like(x, bad)
    for i, (c, r) in enumerate(batch):
        for j in range(need[i]):
            keep = min(ps, c + r - j * ps)
            y[:, table[i][j], :, :, :keep] = x[:, table[i][j], :, :, :keep]
    pool.copy_(y)
    q = randn(6, rows, QDIM)
    check_rows(p, batch, table, q, run_attn(p, batch, i32(table), q), heads=(0, 7))
    p.close()


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("batch,at", [([(4000, 520)], 4277), ([(0, 2100)], 901), ([(10500, 200)], 10563)])
def test_wide_infinities_reach_only_the_rows_that_see_them(gpu, batch, at, what):
    """A bad key of the new rows: the rows before it keep their values (within
    both runs' bounds), those that see it take what the definition gives."""
    assert_wide(batch)
    ps, (c, r) = 32, batch[0]
    need = needed(batch, ps)
    table, _ = shuffled_table(random.Random(4), need, need[0] + 2, need[0])
    p = Paged(need[0] + 2, ps, 1, r, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    page, off = table[0][at // ps], at % ps
    kept = pool[0, page, :, :, off].clone()
    if what == "k":
        pool[0, page, 0, :, off, 3] = float("nan")
    else:
        pool[0, page, 1, :, off, 5] = float("inf")
    q = randn(6, r, QDIM)
    out = run_attn(p, batch, i32(table), q)
    pool[0, page, :, :, off] = kept  # the rows before it: the definition without it
    first = at - c
    assert bool(torch.isfinite(out[:first]).all())
    rows = [x for x in some_rows(r, random.Random(3)) if x < first] + [first - 1]
    ids = torch.tensor(table[0]).cuda()
    for h in (0, 15):
        kv = pool[0][ids][:, :, h // 2].double().cpu().numpy()
        k, v = (kv[:, s].reshape(-1, HD)[:c + r] for s in (0, 1))
        cols = slice(h * HD, (h + 1) * HD)
        want, bound = M.attend(q[rows][:, cols].double().cpu().numpy(), k, v, [c + x for x in rows],
                               np.ones(c + r, bool))
        d = np.abs(out[rows][:, cols].double().cpu().numpy() - want)
        assert (d <= bound).all(), (h, float((d / bound).max()))
    seers = out[first:].view(-1, NQH, HD)
    if what == "v":
        assert bool(torch.isinf(seers[:, :, 5]).all())
        assert bool(torch.isfinite(seers[:, :, 6:]).all())
    else:
        assert bool(torch.isnan(seers).all())
    p.close()


def test_wide_leaves_evicted_pages_out(gpu):
    """Entries outside the pool, whole ranges of them and at a range's end."""
    batch, ps = [(5200, 400), (0, 2100)], 16
    assert_wide(batch)
    need = needed(batch, ps)
    pages = sum(need)
    table, _ = shuffled_table(random.Random(2), need, pages, max(need))
    gone = [x for t in (table[0][4:200], table[1][0:9]) for x in t]
    table[0][4:200] = [-1] * 196
    table[1][0:9] = [pages, 2 ** 31 - 1, -2 ** 31] * 3
    p = Paged(pages, ps, 2, 2500, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    pool[:, gone] = float("nan")
    q = randn(6, 2500, QDIM)
    d_table = i32(table)
    # The second request's own new rows lie on entries outside the pool: with
    # a given table such a request is refused, so it is planned on whole ones.
    whole = [list(t) for t in table]
    whole[1][0:9] = gone[-9:]
    Q.paged_plan(p.ctx, p.plan, i32([c for c, _ in batch]), i32([r for _, r in batch]), d_table)
    assert p.plan.status[:2].tolist() == [M.OK, M.EINVAL]
    out = torch.full_like(q, 7.0)
    Q.paged_attn(p.ctx, p.plan, 0, d_table, q, out)
    assert bool((out[400:] == 7).all())
    check_rows(p, batch[:1], table[:1], q, out, heads=(0, 11))
    pool[:, gone] = randn(8, 1, len(gone), *pool.shape[2:])
    out = run_attn(p, batch, i32([table[0], whole[1]]), q)
    check_rows(p, batch, [table[0], whole[1]], q, out, heads=(5,))
    p.close()


def test_wide_bits_do_not_depend_on_the_batch_or_the_pages(gpu):
    batch, ps = [(4000, 512), (900, 1), (7000, 300), (1500, 1100)], 64
    assert_wide(batch)
    need = needed(batch, ps)
    pages = 2 * sum(need)
    rows = sum(r for _, r in batch)
    p = Paged(pages, ps, len(batch), rows, rope=False)
    pool = p.pool.tensor()
    t1, other = shuffled_table(random.Random(2), need, pages, max(need))
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, rows, QDIM)
    whole = run_attn(p, batch, i32(t1), q).clone()
    r0 = 0
    for i, (c, r) in enumerate(batch):
        ids = other[:need[i]]
        pool[:, i32(ids).long()] = pool[:, i32(t1[i][:need[i]]).long()]
        out = run_attn(p, [(c, r)], i32([ids]), q[r0:r0 + r].contiguous())
        assert torch.equal(out, whole[r0:r0 + r]), i
        r0 += r
    for _ in range(3):
        assert torch.equal(run_attn(p, batch, i32(t1), q), whole)
    p.close()


@pytest.mark.parametrize("batch", [[(300, 5)], [(300, 14)], [(1800, 8)], [(4000, 530)]])
def test_a_broken_query_reaches_only_its_own_row_and_head(gpu, batch):
    """NaN in one (row, q head): the other columns of its block are finite and
    right."""
    ps, (c, r) = 32, batch[0]
    need = needed(batch, ps)
    table, _ = shuffled_table(random.Random(4), need, need[0], need[0])
    p = Paged(need[0], ps, 1, r, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, r, QDIM)
    row, head = r // 2, 4
    good = q.clone()
    q[row, head * HD + 17] = float("nan")
    out = run_attn(p, batch, i32(table), q)
    v = out.view(r, NQH, HD)
    assert bool(torch.isnan(v[row, head]).all())
    v[row, head] = 0
    assert bool(torch.isfinite(v).all())
    clean = run_attn(p, batch, i32(table), good)
    v[row, head] = clean.view(r, NQH, HD)[row, head]
    check_rows(p, batch, table, good, out, heads=(head, head + 1, 0))
    p.close()


def test_scores_of_minus_infinity(gpu):
    """Keys whose scores are -inf weigh nothing; a row with no other is zero."""
    batch, ps = [(40, 1), (40, 3), (700, 12)], 16
    need = needed(batch, ps)
    table, _ = shuffled_table(random.Random(4), need, sum(need), max(need))
    p = Paged(sum(need), ps, 3, 16, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, 16, QDIM).abs()  # so that a key of -inf scores -inf
    pool[:, table[0][:need[0]], 0] = float("-inf")        # every key of request 0
    pool[:, table[1][0], 0, :, 3:9] = float("-inf")       # some of request 1
    pool[:, table[2][:20], 0] = float("-inf")             # whole tiles of request 2
    out = run_attn(p, batch, i32(table), q)
    assert bool((out[0] == 0).all())
    # the definition over the keys that weigh something
    r0 = 1
    for i in (1, 2):
        c, r = batch[i]
        ids = torch.tensor(table[i][:need[i]]).cuda()
        for h in (0, 9):
            kv = pool[0][ids][:, :, h // 2].double().cpu().numpy()
            k, v = (kv[:, s].reshape(-1, HD)[:c + r] for s in (0, 1))
            seen = np.isfinite(k).all(axis=1)
            cols = slice(h * HD, (h + 1) * HD)
            want, bound = M.attend(q[r0:r0 + r, cols].double().cpu().numpy(), np.where(seen[:, None], k, 0), v,
                                   range(c, c + r), seen)
            d = np.abs(out[r0:r0 + r, cols].double().cpu().numpy() - want)
            assert (d <= bound).all(), (i, h, float((d / bound).max()))
        r0 += r
    p.close()


# ---- more items than workgroups --------------------------------------------

@pytest.mark.parametrize("nkvh", [1, 8])
def test_more_items_than_workgroups(gpu, nkvh):
    """Hundreds of single rows and some chunks, twice: the drawing of items
    begins anew with every call."""
    rnd = random.Random(5)
    batch = [(rnd.randint(0, 1500), 1) for _ in range(600)] + [(300, 200), (0, 33), (2600, 17)]
    rnd.shuffle(batch)
    ps = 32
    need = needed(batch, ps)
    pages = sum(need)
    table, _ = shuffled_table(rnd, need, pages, max(need))
    rows = sum(r for _, r in batch)
    p = Paged(pages, ps, len(batch), rows, nkvh=nkvh, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, rows, 2 * nkvh * HD)
    out = run_attn(p, batch, i32(table), q).clone()
    check_rows(p, batch, table, q, out, heads=(2 * nkvh - 1,))
    for _ in range(3):
        assert torch.equal(run_attn(p, batch, i32(table), q), out)
    # a step of one row right behind
    one = run_attn(p, batch[:1], i32(table[:1]), q[:batch[0][1]].contiguous())
    assert torch.equal(one, out[:batch[0][1]])
    p.close()


def test_most_requests(gpu):
    """1024 requests, lengths from zero on, every fourth idle or ended."""
    rnd = random.Random(6)
    batch = [(i % 130, (1, 1, 1, 0)[i % 4]) for i in range(1024)]
    ps = 16
    need = needed(batch, ps)
    table, _ = shuffled_table(rnd, need, sum(need), max(need))
    rows = sum(r for _, r in batch)
    p = Paged(sum(need), ps, 1024, rows, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, rows, QDIM)
    out = run_attn(p, batch, i32(table), q)
    check_rows(p, batch, table, q, out, heads=(4,))
    p.close()


def test_largest_step(gpu):
    """65536 rows of 1024 requests, some requests of one row, some large."""
    rnd = random.Random(9)
    rows = [1] * 300 + [700, 1500, 2100, 4000] + [rnd.randint(2, 130) for _ in range(719)]
    rows.append(65536 - sum(rows))
    rnd.shuffle(rows)
    assert len(rows) == 1024 and min(rows) > 0
    batch = [(rnd.choice([0, 1, rnd.randint(0, 700)]), r) for r in rows]
    ps = 64
    need = needed(batch, ps)
    table, _ = shuffled_table(rnd, need, sum(need), max(need))
    p = Paged(sum(need), ps, 1024, 65536, nkvh=1, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, 65536, 2 * HD)
    out = run_attn(p, batch, i32(table), q)
    assert p.plan.status.tolist() == [M.OK] * 1024
    starts = p.plan.row_start.tolist()
    assert starts[-1] == 65536
    big = sorted(range(1024), key=lambda i: -rows[i])[:4]
    for i in big + rnd.sample(range(1024), 24) + [0, 1023]:
        r0, r1 = starts[i], starts[i + 1]
        check_rows(p, batch[i:i + 1], table[i:i + 1], q[r0:r1], out[r0:r1], heads=(i % 2,))
    p.close()


@pytest.mark.parametrize("ps", [16, 64])
def test_long_contexts_find_their_keys(gpu, ps):
    """100000 keys on shuffled pages, ranges of many pages: a row whose query is
    a multiple of one key gives that key's value.  Its score is 4 |k|^2 /
    sqrt(128), 45 +- 6, the others' are normal with deviation s = 4 |k| /
    sqrt(128), about 4, whose exponentials average e^(s^2/2), about e^8: 20 below
    it and more, so all of them weigh less than 100000 e^-20."""
    n, nkvh = 100000, 2
    need = -(-(n + 1) // ps)
    at = [0, 5, 511, 1700, 1791, 1792, 3124, 3125, 30000, 77777, n - 3, n - 1]
    p = Paged(need, ps, len(at), len(at), nkvh=nkvh, max_seq=1 << 17, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    ids = random.Random(1).sample(range(need), need)
    q = torch.empty((len(at), 2 * nkvh, HD), dtype=torch.float16, device="cuda")
    want = torch.empty_like(q)
    for i, t in enumerate(at):
        kv = pool[0, ids[t // ps], :, :, t % ps]
        for h in range(2 * nkvh):
            q[i, h], want[i, h] = 4 * kv[0, h // 2], kv[1, h // 2]
    out = run_attn(p, [(n, 1)] * len(at), i32([ids] * len(at)), q.view(len(at), -1))
    # two f16 roundings (the weight's and the result's) of values below 8, and
    # the other keys
    d = (out.view_as(want).double() - want.double()).abs().max().item()
    assert d <= 2 * 2.0 ** -11 * 8 + 2 * 100000 * np.exp(-20.0) * 8, d
    # not so when its page is gone
    gone = list(ids)
    gone[77777 // ps] = -1
    out2 = run_attn(p, [(n, 1)], i32([gone]), q[9:10].view(1, -1))
    assert bool(torch.isfinite(out2).all())
    assert float((out2.view(-1).double() - want[9].view(-1).double()).abs().max()) > 0.5
    p.close()


def test_replayed_graph_of_changing_work(gpu):
    """One captured [plan, attention] over lengths and row counts that change
    between the replays: wide, split, single and no work at all, with eager
    calls of another plan in between."""
    ps, n = 64, 8
    p = Paged(400, ps, n, 1200, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    ids = random.Random(3).sample(range(400), 400)
    width = 50
    table = [ids[i * width:(i + 1) * width] for i in range(n)]
    d_table, lens, rows = i32(table), i32([0] * n), i32([0] * n)
    q = randn(6, 1200, QDIM)
    out = torch.full_like(q, 7.0)
    eager = Q.PagedPlan(p.ctx, p.pool, n, 1200)

    def step(plan, o):
        Q.paged_plan(p.ctx, plan, lens, rows, d_table)
        Q.paged_attn(p.ctx, plan, 0, d_table, q, o)

    step(p.plan, out)
    torch.cuda.synchronize()
    assert bool((out == 7).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(p.plan, out)
    for batch in ([(900, 1)] * 8, [(2000, 900), (1, 1), (3000, 1), (5, 0), (0, 16)], [(0, 0)],
                  [(2100, 1)] * 5, [(2450, 750), (40, 40)], [(2450, 750), (40, 40)], [(0, 1)]):
        batch = batch + [(0, 0)] * (n - len(batch))
        lens.copy_(i32([c for c, _ in batch]))
        rows.copy_(i32([r for _, r in batch]))
        out.fill_(7.0)
        graph.replay()
        want = torch.full_like(q, 7.0)
        step(eager, want)
        torch.cuda.synchronize()
        assert torch.equal(out, want), batch
        check_rows(p, batch, table, q, out, heads=(3,))
    eager.close()
    p.close()


def test_on_another_stream(gpu):
    """Torch's current stream is the one that the calls run on."""
    batch, ps = [(4000, 512), (900, 1)], 64
    need = needed(batch, ps)
    table, _ = shuffled_table(random.Random(2), need, sum(need), max(need))
    p = Paged(sum(need), ps, 2, 513, rope=False)
    pool = p.pool.tensor()
    q = torch.empty((513, QDIM), dtype=torch.float16, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        pool.copy_(randn(5, *pool.shape))  # ordered before the calls by the stream alone
        q.copy_(randn(6, 513, QDIM))
        d_table = i32(table)
        Q.paged_plan(p.ctx, p.plan, i32([4000, 900]), i32([512, 1]), d_table)
        out = torch.zeros_like(q)
        Q.paged_attn(p.ctx, p.plan, 0, d_table, q, out)
        out2 = out.clone()
    torch.cuda.synchronize()
    check_rows(p, batch, table, q, out2, heads=(1,))
    p.close()


# ---- refusals ---------------------------------------------------------------

def refused(code, fn):
    with pytest.raises(Q.QasrError) as e:
        fn()
    assert e.value.code == code, e.value


def test_creates_refuse(gpu):
    ctx, other = (Q.Context(NQH, NKVH, HD, 2, 1e-6, 512, 0) for _ in range(2))
    for ps in (0, 1, 8, 17, 48, 512, -16):
        refused(Q.QASR_EINVAL, lambda: Q.PagePool(ctx, 4, ps))
    for pages, ps in ((0, 16), (-1, 16), (1 << 27, 16), (1 << 23, 256), (2 ** 31 - 1, 16)):
        refused(Q.QASR_EINVAL, lambda: Q.PagePool(ctx, pages, ps))
    pool = Q.PagePool(ctx, 4, 16)
    for n, rows in ((0, 1), (1025, 1), (-1, 1), (1, 0), (1, -5), (1, 65537)):
        refused(Q.QASR_EINVAL, lambda: Q.PagedPlan(ctx, pool, n, rows))
    refused(Q.QASR_EINVAL, lambda: Q.PagedPlan(other, pool, 1, 1))
    pool.close()
    other.close()
    ctx.close()


def test_a_failed_allocation_is_not_the_next_calls_error(gpu):
    """A pool far larger than the card: refused, and what follows runs."""
    ctx = Q.Context(NQH, NKVH, HD, 28, 1e-6, 512, 0)
    refused(Q.QASR_ENOMEM, lambda: Q.PagePool(ctx, (1 << 27) - 1, 16))
    pool = Q.PagePool(ctx, 4, 16)
    plan = Q.PagedPlan(ctx, pool, 1, 1)
    table = i32([[2]])
    Q.paged_plan(ctx, plan, i32([3]), i32([1]), table)
    q = randn(3, 1, QDIM)
    out = torch.full_like(q, 7.0)
    Q.paged_attn(ctx, plan, 5, table, q, out)
    torch.cuda.synchronize()
    assert bool((out == 0).all())  # a zeroed pool
    plan.close()
    pool.close()
    ctx.close()


def test_a_shared_prefix_is_given_back_once(gpu):
    """Two requests over one prefix of whole pages; the first to end leaves the
    shared entries out, the last gives them back."""
    p = Paged(8, 16, 2, 4, rope=False)
    ring, cursor = i32([5, 6, 7, 0, 0, 0, 0, 0]), i32([0, 3])
    table = i32([[0, 1, -1, -1], [0, 1, -1, -1]])
    p.plan.lens.copy_(i32([32, 32]))
    p.plan.cursor.copy_(cursor)
    step = lambda rows: Q.paged_plan(p.ctx, p.plan, p.plan.lens, i32(rows), table, ring, p.plan.cursor)  # noqa: E731
    step([1, 2])
    assert table.tolist() == [[0, 1, 5, -1], [0, 1, 6, -1]] and p.plan.cursor.tolist() == [2, 1]
    table[0, :2] = -1
    step([-1, 1])
    assert p.plan.status.tolist() == [0, 0] and p.plan.lens.tolist() == [0, 35]
    assert p.plan.cursor.tolist() == [2, 2]
    step([0, -1])
    head, free = p.plan.cursor.tolist()
    assert sorted(ring[(head + k) % 8].item() for k in range(free)) == [0, 1, 5, 6, 7]
    p.close()


def test_calls_refuse(gpu):
    p = Paged(8, 16, 2, 5, layers=2, max_seq=512, rope=False)
    other = Paged(8, 16, 2, 5, layers=2, max_seq=512, rope=False)
    ctx, plan = p.ctx, p.plan
    one, table, wide = i32([1, 1, 1]), i32([[0], [1], [2]]), i32([[0, 3], [1, 4], [2, 5]])
    qkv, g = randn(1, 6, TOT), randn(2, HD)
    q, out = randn(3, 6, QDIM), torch.full((6, QDIM), 7.0, dtype=torch.float16, device="cuda")
    # before the first build
    refused(Q.QASR_ESTATE, lambda: Q.paged_append(ctx, plan, 0, qkv[:2], g, g, q))
    refused(Q.QASR_ESTATE, lambda: Q.paged_attn(ctx, plan, 0, table[:2], q[:2], out))
    # the plan's limits, other contexts' plans, halves of a ring
    refused(Q.QASR_ERANGE, lambda: Q.paged_plan(ctx, plan, one, one, table))
    refused(Q.QASR_EINVAL, lambda: Q.paged_plan(other.ctx, plan, one[:2], one[:2], table))
    refused(Q.QASR_EINVAL, lambda: Q.paged_plan(ctx, plan, one[:2], one[:2], table, i32(list(range(8)))))
    refused(Q.QASR_EINVAL, lambda: Q.paged_plan(ctx, plan, one[:0], one[:0], table))
    Q.paged_plan(ctx, plan, one[:2], one[:2], table)
    for layer in (-1, 2):
        refused(Q.QASR_EINVAL, lambda: Q.paged_append(ctx, plan, layer, qkv[:2], g, g, q))
        refused(Q.QASR_EINVAL, lambda: Q.paged_attn(ctx, plan, layer, table, q[:2], out))
    refused(Q.QASR_ESTATE, lambda: Q.paged_append(ctx, plan, 0, qkv[:2], g, g, q))  # no RoPE tables
    refused(Q.QASR_ERANGE, lambda: Q.paged_append(ctx, plan, 0, qkv, g, g, q))
    refused(Q.QASR_ERANGE, lambda: Q.paged_attn(ctx, plan, 0, table, q, out))
    refused(Q.QASR_EINVAL, lambda: Q.paged_attn(ctx, plan, 0, wide, q[:2], out))  # another stride
    refused(Q.QASR_EINVAL, lambda: Q.paged_attn(other.ctx, plan, 0, table, q[:2], out))
    # outputs over inputs, and rows that 16-byte accesses cannot take
    refused(Q.QASR_EINVAL, lambda: Q.paged_attn(ctx, plan, 0, table, q[:2], q[:2]))
    refused(Q.QASR_EINVAL, lambda: Q.paged_attn(ctx, plan, 0, table, q[:2], q[1:3]))
    refused(Q.QASR_EINVAL, lambda: Q.paged_append(ctx, plan, 0, qkv[:2], g, g, qkv.view(-1)[:2 * QDIM]))
    odd = q.view(-1)[1:1 + 2 * QDIM].view(2, QDIM)
    refused(Q.QASR_EINVAL, lambda: Q.paged_attn(ctx, plan, 0, table, odd, out))
    refused(Q.QASR_EINVAL, lambda: Q.paged_append(ctx, plan, 0, qkv[:2], randn(2, HD + 1)[1:], g, q))
    # tensors of other types, devices and layouts
    for bad in (one[:2].long(), one[:2].cpu(), i32([1, 0, 1, 0])[::2]):
        with pytest.raises((Q.QasrError, ValueError, TypeError)):
            Q.paged_plan(ctx, plan, bad, one[:2], table)
    for bad in (q[:2].float(), q[:2].cpu(), q.t().contiguous().t()[:2], q[:2].bfloat16()):
        with pytest.raises((Q.QasrError, ValueError, TypeError)):
            Q.paged_attn(ctx, plan, 0, table, bad, out)
    # the C entry's own: negative rows, null pointers
    lib, null = Q.load(), ctypes.c_void_p()
    assert lib.qasr_paged_attn(ctx.handle, plan.handle, 0, -1, null, 1, null, null, null) == Q.QASR_EINVAL
    assert lib.qasr_paged_attn(ctx.handle, plan.handle, 0, 1, null, 1, null, null, null) == Q.QASR_EINVAL
    assert lib.qasr_paged_attn(ctx.handle, plan.handle, 0, 0, null, 1, null, null, null) == Q.QASR_OK
    assert lib.qasr_paged_append(ctx.handle, plan.handle, 0, 1, null, null, null, null, null) == Q.QASR_EINVAL
    assert lib.qasr_paged_plan_build(ctx.handle, plan.handle, 1, null, null, null, 1, null, null,
                                     null) == Q.QASR_EINVAL
    assert bool((out == 7).all())
    # none of it did harm
    Q.paged_plan(ctx, plan, one[:2], one[:2], table)
    Q.paged_attn(ctx, plan, 0, table, q[:2], out)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all()) and bool((out[2:] == 7).all())
    other.close()
    p.close()


def test_positions_past_the_rope_tables_are_refused(gpu):
    """Tables shorter than max_seq: such rows are not placed."""
    p = Paged(8, 16, 3, 8, max_seq=512, rope=False)
    c, s = rope_tables()
    p.ctx.set_rope_tables(c[:40], s[:40])
    table = i32([[0, 1, 2], [3, 4, 5], [6, 7, -1]])
    Q.paged_plan(p.ctx, p.plan, i32([39, 38, 0]), i32([1, 3, 1]), table)
    assert p.plan.status.tolist() == [M.OK, M.ERANGE, M.OK]
    assert p.plan.row_pos.tolist() == [39, -1, -1, -1, 0, -1, -1, -1]
    p.close()
