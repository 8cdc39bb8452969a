"""Paged steps at their edges: pages that the pool does not have, arrays that
overlap, closed objects, the size of a plan, other head counts, fewer rows than
planned."""
from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

import qasr_attn as Q  # noqa: E402
from gpu_helpers import Gpu  # noqa: E402
from test_gpu_paged import Paged, check_attn, i32, randn, run_attn, shuffled_table  # noqa: E402
from workloads import HD, NKVH, NQH, QDIM, TOT  # noqa: E402

pytestmark = pytest.mark.gpu


# ---- append -----------------------------------------------------------------

@pytest.mark.parametrize("rows", [40, 830])
def test_rows_on_a_page_outside_the_pool_attend_what_is_before_them(gpu, rows):
    """The ring holds an id that the pool does not have: the rows that fall on
    it are stored nowhere and seen by none, but they have a position, so their
    queries are roped and attend the keys before them."""
    ps, start = 16, 16
    pages = (start + rows) // ps + 8
    p = Paged(pages, ps, 1, rows)
    pool = p.pool.tensor()
    pool.copy_(randn(1, *pool.shape))
    before = pool.clone()
    ids = random.Random(2).sample(range(pages), pages)
    bad = 1  # place of the id in the request's new pages
    ring = ids[1:] + ids[:1]
    ring[bad] = pages + 3
    table = i32([ids[:1] + [-1] * (rows // ps + 1)])
    qkv, g = randn(2, rows, TOT), randn(3, 2, HD) + 1
    q = torch.full((rows, QDIM), 7.0, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    Q.paged_plan(p.ctx, p.plan, i32([start]), i32([rows]), table, i32(ring), i32([0, pages - 1]))
    assert p.plan.status[0].item() == 0
    lost = range(bad * ps, (bad + 1) * ps)
    assert [r for r in range(rows) if p.plan.row_slot[r].item() < 0] == list(lost)
    Q.paged_append(p.ctx, p.plan, 0, qkv, g[0], g[1], q)
    Q.paged_attn(p.ctx, p.plan, 0, table, q, out)

    ref = Gpu(1, start + rows)
    q_ref = torch.empty_like(q)
    Q.qk_norm_rope_append(ref.ctx, ref.kv, 0, [(0, start, rows)], qkv, g[0], g[1], q_ref)
    assert torch.equal(q, q_ref)
    slots, want, t = ref.kv.tensor(), before.clone(), table[0].tolist()
    for pos in range(start, start + rows):
        if pos - start not in lost:
            want[0, t[pos // ps], :, :, pos % ps] = slots[0, 0, :, :, pos]
    assert torch.equal(pool, want)
    check_attn(p, [(start, rows)], table, q, out, heads=(0, 15))
    ref.close()
    p.close()


@pytest.mark.parametrize("nkvh", [1, 5, 9, 16])
@pytest.mark.parametrize("batch", [[(20, 1), (0, 37), (15, 2)], [(3, 300), (1000, 1), (0, 640)]])
def test_append_of_other_head_counts_has_the_bits_of_stage_a(gpu, nkvh, batch):
    """Up to 24 heads and more, few rows and many."""
    ps, tot, qd = 32, 4 * nkvh * HD, 2 * nkvh * HD
    lens, rows = [c for c, _ in batch], [r for _, r in batch]
    total = sum(rows)
    need = [-(-(c + r) // ps) for c, r in batch]
    table, _ = shuffled_table(random.Random(3), need, sum(need) + 2, max(need))
    p = Paged(sum(need) + 2, ps, len(batch), total + 3, nkvh=nkvh)
    pool = p.pool.tensor()
    pool.copy_(randn(1, *pool.shape))
    want = pool.clone()
    qkv, g = randn(2, total + 3, tot), randn(3, 2, HD) + 1
    q = torch.full((total + 3, qd), 7.0, dtype=torch.float16, device="cuda")
    Q.paged_plan(p.ctx, p.plan, i32(lens), i32(rows), i32(table))
    Q.paged_append(p.ctx, p.plan, 0, qkv, g[0], g[1], q)
    kv = Q.KVPool(p.ctx, len(batch), max(c + r for c, r in batch))
    q_ref = torch.empty((total, qd), dtype=torch.float16, device="cuda")
    Q.qk_norm_rope_append(p.ctx, kv, 0, [(i, c, r) for i, (c, r) in enumerate(batch)], qkv, g[0], g[1], q_ref)
    assert torch.equal(q[:total], q_ref) and bool((q[total:] == 7).all())
    slots = kv.tensor()
    for i, (c, r) in enumerate(batch):
        for pos in range(c, c + r):
            want[0, table[i][pos // ps], :, :, pos % ps] = slots[i, 0, :, :, pos]
    assert torch.equal(pool, want)
    kv.close()
    p.close()


# ---- attention --------------------------------------------------------------

@pytest.mark.parametrize("batch,cuts", [([(1500, 12)], (1, 5, 8, 9, 11)), ([(1500, 8)], (1, 3)),
                                        ([(5000, 300)], (17, 160, 289)), ([(10500, 200)], (1, 63, 64, 65, 190)),
                                        ([(0, 2100)], (1, 100, 2099)),
                                        ([(900, 1), (4000, 512), (40, 20)], (1, 2, 200, 513, 520))])
def test_fewer_rows_than_planned(gpu, batch, cuts):
    """Row blocks and key ranges cut short by the caller's rows, wide and
    split: the rows there are come out, those behind stay, and the plan serves
    the whole step afterwards."""
    ps = 16
    need = [-(-(c + r) // ps) for c, r in batch]
    table, _ = shuffled_table(random.Random(1), need, sum(need), max(need))
    rows = sum(r for _, r in batch)
    p = Paged(sum(need), ps, len(batch), rows, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, rows, QDIM)
    d_table = i32(table)
    whole = run_attn(p, batch, d_table, q).clone()
    check_attn(p, batch, d_table, q, whole, heads=(3,))
    for cut in cuts:
        out = torch.full_like(q, 7.0)
        Q.paged_attn(p.ctx, p.plan, 0, d_table, q[:cut], out)
        assert bool((out[cut:] == 7).all())
        left, part = cut, []
        for c, r in batch:
            part.append((c, min(r, left)))
            left -= part[-1][1]
        check_attn(p, part, d_table, q[:cut], out[:cut], heads=(3,))
        Q.paged_attn(p.ctx, p.plan, 0, d_table, q, out)
        assert torch.equal(out, whole)
    p.close()


# ---- what a build takes -----------------------------------------------------

def refused(fn):
    with pytest.raises(Q.QasrError) as e:
        fn()
    assert e.value.code == Q.QASR_EINVAL, e.value


def test_build_refuses_arrays_that_overlap(gpu):
    """What one workgroup of a build writes and another reads, save the plan's
    lens and cursor in their own places."""
    n, pages, width = 4, 16, 3
    p = Paged(pages, 16, n, 16, rope=False)
    c, plan = p.ctx, p.plan
    lens, rows, cursor = i32([3] * n), i32([1] * n), i32([0, pages])
    ring, table = i32(list(range(pages))), i32([[i, -1, -1] for i in range(n)])
    build = lambda *a: refused(lambda: Q.paged_plan(c, plan, *a))  # noqa: E731
    # in the plan's own memory
    build(plan.lens, plan.lens, table, ring, cursor)
    build(lens, plan.status, table, ring, cursor)
    build(plan.row_pos, rows, table, ring, cursor)
    build(plan.row_start[1:], rows, table, ring, cursor)
    build(lens, rows, plan.row_slot[:n * width].view(n, width), ring, cursor)
    build(lens, rows, plan.row_slot[:n * width].view(n, width))
    build(lens, rows, table, plan.row_pos, cursor)
    build(lens, rows, table, ring, plan.row_start[:2])
    # each other's
    a = i32([0] * 64)
    view = lambda at: a[at:at + n * width].view(n, width)  # noqa: E731
    build(lens, rows, view(0), a[n * width - 1:n * width - 1 + pages], cursor)
    build(a[n * width - 1:][:n], rows, view(0), ring, cursor)
    build(lens, a[:n], view(n - 1), ring, cursor)
    build(lens, rows, view(0), ring, a[1:3])
    build(a[pages - 1:pages - 1 + n], rows, table, a[:pages], cursor)
    build(lens, a[4:4 + n], table, a[:pages], cursor)
    build(lens, rows, table, a[:pages], a[pages - 1:pages + 1])
    lib = Q.load()
    assert lib.qasr_paged_plan_build(c.handle, plan.handle, n, lens.data_ptr() + 2, rows.data_ptr(), table.data_ptr(),
                                     width, None, None, None) == Q.QASR_EINVAL
    # side by side in one allocation, lens and rows the same array, and in place
    a[:n * width] = table.view(-1)
    a[12:28], a[28:30], a[30:34], a[34:38] = ring, i32([4, 12]), lens, rows
    Q.paged_plan(c, plan, a[30:34], a[34:38], view(0), a[12:28], a[28:30])
    assert plan.status.tolist() == [0] * n and plan.lens.tolist() == [4] * n
    Q.paged_plan(c, plan, rows, rows, table)
    assert plan.status.tolist() == [0] * n and plan.lens.tolist() == [2] * n
    plan.cursor.copy_(i32([4, 12]))
    Q.paged_plan(c, plan, plan.lens, rows, table, ring, plan.cursor)
    assert plan.status.tolist() == [0] * n and plan.lens.tolist() == [3] * n
    p.close()


def test_calls_on_a_closed_pool_are_refused(gpu):
    """A plan whose pool or context is closed: its calls are refused, and it can
    still be closed."""
    def make():
        ctx = Q.Context(NQH, NKVH, HD, 1, 1e-6, 128, 0)
        pool = Q.PagePool(ctx, 4, 16)
        plan = Q.PagedPlan(ctx, pool, 2, 4)
        table = i32([[0], [1]])
        Q.paged_plan(ctx, plan, i32([3, 3]), i32([1, 1]), table)
        torch.cuda.synchronize()
        q, out = randn(1, 2, QDIM), torch.zeros((2, QDIM), dtype=torch.float16, device="cuda")
        qkv, g = randn(2, 2, TOT), randn(3, HD)

        def calls():
            refused(lambda: Q.paged_plan(ctx, plan, i32([3, 3]), i32([1, 1]), table))
            refused(lambda: Q.paged_attn(ctx, plan, 0, table, q, out))
            refused(lambda: Q.paged_append(ctx, plan, 0, qkv, g, g, out))

        return ctx, pool, plan, calls

    ctx, pool, plan, calls = make()
    pool.close()
    calls()
    refused(lambda: pool.info())
    refused(lambda: Q.PagedPlan(ctx, pool, 1, 1))
    plan.close()
    ctx.close()
    ctx, pool, plan, calls = make()
    ctx.close()
    calls()
    with pytest.raises(Q.QasrError):
        pool.tensor()
    plan.close()
    calls()
    pool.close()


@pytest.mark.parametrize("max_seq,ranges", [(400, 0), (512, 0), (513, 2), (2048, 4), (5000, 10), (16384, 32), (1 << 20, 32)])
def test_a_plan_holds_no_more_split_state_than_its_context_needs(gpu, max_seq, ranges):
    """Records of 130 floats a q head: a key range of 512 keys or more a record
    for each row, at most 32 ranges a row and 2048 records a request.  Beside
    them a plan has items, counters and row maps, below 5 MB here."""
    ctx = Q.Context(NQH, NKVH, HD, 1, 1e-6, max_seq, 0)
    pool = Q.PagePool(ctx, 4, 16)
    for n, rows in ((1, 1), (64, 64), (3, 4096), (64, 2048)):
        plan = Q.PagedPlan(ctx, pool, n, rows)
        state = min(rows * ranges, n * 2048 if ranges else 0) * NQH * 130 * 4
        assert state <= plan.bytes <= state + 5e6, (n, rows, state, plan.bytes)
        plan.close()
    pool.close()
    ctx.close()


@pytest.mark.parametrize("max_seq,batch", [(513, [(512, 1), (0, 513), (505, 8)]), (1024, [(1023, 1), (1000, 24), (900, 124)]),
                                           (2048, [(2047, 1), (1800, 248), (0, 2048), (1500, 548)])])
def test_positions_up_to_the_last_of_a_short_context(gpu, max_seq, batch):
    """The split state of a plan for exactly these rows is as short as it gets."""
    ps = 16
    need = [-(-(c + r) // ps) for c, r in batch]
    table, _ = shuffled_table(random.Random(1), need, sum(need), max(need))
    rows = sum(r for _, r in batch)
    p = Paged(sum(need), ps, len(batch), rows, max_seq=max_seq, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, rows, QDIM)
    out = run_attn(p, batch, i32(table), q)
    assert p.plan.status.tolist() == [0] * len(batch)
    check_attn(p, batch, i32(table), q, out, heads=(0, 13))
    p.close()


def test_two_plans_take_turns_over_one_pool(gpu):
    """Single rows on a plan of their own, chunks on a larger one: each build
    goes on from the lens and the cursor of the other plan."""
    ps, pages, n = 16, 60, 4
    p = Paged(pages, ps, n, n)
    large = Q.PagedPlan(p.ctx, p.pool, n, 100)
    ring, cursor = p.pool.free_ring()
    table = torch.full((n, 14), -1, dtype=torch.int32, device="cuda")
    g = randn(3, 2, HD) + 1
    lens, at, cur = [0] * n, i32([0] * n), cursor
    for t, rows in enumerate([[20, 30, 15, 1], [1] * n, [1, 0, 1, 1], [40, 1, 1, 20], [1] * n, [0, 33, 0, 1], [1] * n]):
        plan = p.plan if max(rows) <= 1 else large
        total = sum(rows)
        qkv = randn(50 + t, total, TOT)
        q, out = (torch.empty((total, QDIM), dtype=torch.float16, device="cuda") for _ in range(2))
        Q.paged_plan(p.ctx, plan, at, i32(rows), table, ring, cur)
        Q.paged_append(p.ctx, plan, 0, qkv, g[0], g[1], q)
        Q.paged_attn(p.ctx, plan, 0, table, q, out)
        at, cur = plan.lens, plan.cursor
        assert plan.status.tolist() == [0] * n
        check_attn(p, list(zip(lens, rows)), table, q, out, heads=(0, 7))
        lens = [a + b for a, b in zip(lens, rows)]
        assert at.tolist() == lens
    held = [x for i in range(n) for x in table[i, :-(-lens[i] // ps)].tolist()]
    head, free = cur.tolist()
    assert sorted(held + [ring[(head + k) % pages].item() for k in range(free)]) == list(range(pages))
    large.close()
    p.close()
