"""The paged KV cache on the GPU: plan, append and attention against plain
implementations (paged_model.py) and against the slot pool's operators, and a
run of them together as a server uses them."""
from __future__ import annotations

import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_model as M  # noqa: E402
import qasr_attn as Q  # noqa: E402
from gpu_helpers import Gpu, rope_tables, say  # noqa: E402
from workloads import HD, NKVH, NQH, QDIM, TOT  # noqa: E402

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def randn(seed, *shape, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).half()


class Paged:
    """A context, a pool and a plan, closed in order."""

    def __init__(self, pages, ps, requests, rows, nkvh=NKVH, layers=1, max_seq=16384, rope=True):
        self.ctx = Q.Context(2 * nkvh, nkvh, HD, layers, 1e-6, max_seq, 0)
        if rope:
            c, s = rope_tables()
            self.ctx.set_rope_tables(c[:max_seq], s[:max_seq])
        self.pool = Q.PagePool(self.ctx, pages, ps)
        self.plan = Q.PagedPlan(self.ctx, self.pool, requests, rows)

    def close(self):
        torch.cuda.synchronize()
        self.plan.close()
        self.pool.close()
        self.ctx.close()


def shuffled_table(rnd, need, pages, width, spare=0):
    """A table whose rows list distinct random pages: need[i] each."""
    ids = rnd.sample(range(pages), sum(need))
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return table, [p for p in range(pages) if p not in set(ids)]


# ---- plan -----------------------------------------------------------------

def check_plan(p, lens, rows, table, ring, cursor, in_place=False):
    n, ps, pages = len(lens), p.pool.page_rows, p.pool.pages
    d_table, d_ring = i32(table), i32(ring) if ring is not None else None
    d_len, d_cur = i32(lens), i32(cursor) if ring is not None else None
    if in_place:
        p.plan.lens[:n].copy_(d_len)
        d_len = p.plan.lens
        if ring is not None:
            p.plan.cursor.copy_(d_cur)
            d_cur = p.plan.cursor
    Q.paged_plan(p.ctx, p.plan, d_len, i32(rows), d_table, d_ring, d_cur)
    torch.cuda.synchronize()
    want = M.plan(lens, rows, table, ring, cursor, pages, ps, p.ctx.cfg.max_seq, p.plan.max_rows)
    pl = p.plan
    got = {"status": pl.status[:n], "lens": pl.lens[:n], "row_start": pl.row_start[:n + 1],
           "row_pos": pl.row_pos, "row_slot": pl.row_slot}
    for name, t in got.items():
        assert t.tolist() == want[name], name
    assert d_table.tolist() == table
    if ring is not None:
        assert pl.cursor.tolist() == want["cursor"]
        assert d_ring.tolist() == ring
    return want


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,ps,max_rows,short", [
    (1, 16, 1, False), (5, 32, 40, False), (16, 16, 700, True), (64, 256, 1024, True),
    (65, 64, 3000, False), (300, 16, 9000, True), (1024, 128, 2100, False), (1024, 16, 1024, True)])
def test_plan_matches_plain(gpu, n, ps, max_rows, short, in_place):
    rnd = random.Random(n * 1000 + ps)
    lens, rows = [], []
    left = max_rows
    for _ in range(n):
        kind = rnd.random()
        lens.append(rnd.choice([0, 1, ps - 1, ps, ps + 1, rnd.randint(0, 3000)]))
        r = 0 if kind < 0.1 else -1 if kind < 0.2 else 1 if kind < 0.8 else rnd.randint(1, 400)
        r = min(r, left)
        left -= max(r, 0)
        rows.append(r)
    need = [-(-c // ps) for c in lens]
    full = [-(-(c + max(r, 0)) // ps) for c, r in zip(lens, rows)]
    width = max(full) + rnd.randint(0, 3)
    grow = sum(full) - sum(need)
    pages = sum(need) + grow + 9
    table, other = shuffled_table(rnd, need, pages, width)
    free = grow * 2 // 3 if short else grow
    rnd.shuffle(other)
    head = rnd.randint(0, pages - 1)
    ring = [rnd.choice([-1, 0, pages - 1]) for _ in range(pages)]  # what lies outside the free run
    for k in range(free):
        ring[(head + k) % pages] = other[k]
    p = Paged(pages, ps, n, max_rows, rope=False)
    say(f"plan n={n} ps={ps} rows={sum(max(r, 0) for r in rows)} pages={pages} free={free}")
    w = check_plan(p, lens, rows, table, ring, [head, free], in_place)
    assert short == (M.ENOMEM in w["status"]) or not short or grow < 3
    p.close()


def test_plan_refuses_requests_one_by_one(gpu):
    """Every reason of refusal beside requests that are placed."""
    ps, pages, width, max_rows = 16, 64, 6, 60
    p = Paged(pages, ps, 16, max_rows, max_seq=90, rope=False)
    lens = [5, -1, 3, 20, 95, 80, 33, 17, 16, 100, 40, 7, 8, 0, 2]
    rows = [1, 2, -2, 1, 0, 11, 3, 5, 1, -1, -1, 9, 1, 40, 1]
    need = [max(0, min(width, -(-c // ps))) for c in lens]
    rnd = random.Random(3)
    table, other = shuffled_table(rnd, need, pages, width)
    table[6][2] = -1           # the torn page of request 6 is not in the pool
    table[7][1] = pages        # nor is request 7's
    table[10][1] = -5          # an evicted page of an ended request is not given back
    ring = other + [0] * (pages - len(other))
    w = check_plan(p, lens, rows, table, ring, [0, len(other)])
    assert w["status"][:8] == [0, 1, 1, 0, 1, 2, 1, 1]
    assert w["status"][13] == 2  # rows past max_rows
    p.close()


@pytest.mark.parametrize("cursor", [[-1, 3], [64, 3], [0, -2], [0, 65]])
def test_plan_with_a_broken_cursor_has_no_free_page(gpu, cursor):
    p = Paged(64, 16, 4, 8, rope=False)
    table = i32([[-1] * 4] * 2)
    Q.paged_plan(p.ctx, p.plan, i32([0, 0]), i32([1, 0]), table, i32(list(range(64))), i32(cursor))
    assert p.plan.status[:2].tolist() == [M.ENOMEM, 0]
    assert p.plan.row_slot.tolist() == [-1] * 8 and p.plan.cursor.tolist() == [0, 0]
    assert table.tolist() == [[-1] * 4] * 2
    p.close()


def test_plan_with_a_given_table(gpu):
    p = Paged(40, 16, 3, 50, rope=False)
    table = [[4, 9, 2, 7], [1, 3, -1, -1], [0, 40, 5, 6]]
    w = check_plan(p, [30, 16, 10], [20, 30, 8], table, None, None)
    assert w["status"] == [0, 1, 1]
    p.close()


def test_views_keep_the_memory_alive(gpu):
    """A view of a plan's or pool's memory outlives the Python objects; the
    memory goes with the last of them."""
    import gc
    import weakref

    def make():
        ctx = Q.Context(NQH, NKVH, HD, 1, 1e-6, 128, 0)
        pool = Q.PagePool(ctx, 4, 16)
        plan = Q.PagedPlan(ctx, pool, 3, 5)
        Q.paged_plan(ctx, plan, i32([2, 0, 7]), i32([1, 1, 1]), i32([[0], [1], [2]]))
        pool.tensor()[0, 1] = 3
        return plan.row_slot[1:4], pool.tensor()[0, 1, 0], weakref.ref(plan._mem), weakref.ref(pool)

    slots, page, mem, pool = make()
    gc.collect()
    assert mem() is not None and pool() is not None
    junk = [torch.full((1 << 20,), 9, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert slots.tolist() == [16, 39, -1]
    assert bool((page == 3).all())
    del slots, junk
    gc.collect()
    assert mem() is None
    del page
    gc.collect()
    assert pool() is None


# ---- append ---------------------------------------------------------------

@pytest.mark.parametrize("ps", [16, 128])
@pytest.mark.parametrize("batch", [[(0, 1)], [(511, 1), (30, 5), (100, 0), (15, 18)],
                                   [(3, 300), (1000, 1), (0, 640)]])
def test_append_has_the_bits_of_stage_a(gpu, ps, batch):
    lens, rows = [c for c, _ in batch], [r for _, r in batch]
    total, pad = sum(rows), 3
    need = [-(-(c + r) // ps) for c, r in batch]
    pages = sum(need) + 4
    table, _ = shuffled_table(random.Random(ps), need, pages, max(need) + 1)
    p = Paged(pages, ps, len(batch), total + pad, layers=2)
    pool = p.pool.tensor()
    pool.copy_(randn(1, *pool.shape))
    before = pool.clone()
    qkv, g = randn(2, total + pad, TOT), randn(3, 2, HD) + 1
    q_out = torch.full((total + pad, QDIM), 7.0, dtype=torch.float16, device="cuda")
    Q.paged_plan(p.ctx, p.plan, i32(lens), i32(rows), i32(table))
    Q.paged_append(p.ctx, p.plan, 1, qkv, g[0], g[1], q_out)

    cap = max(c + r for c, r in batch)
    ref = Gpu(len(batch), cap)
    q_ref = torch.empty((total, QDIM), dtype=torch.float16, device="cuda")
    segs = [(i, c, r) for i, (c, r) in enumerate(batch) if r]
    Q.qk_norm_rope_append(ref.ctx, ref.kv, 0, segs, qkv, g[0], g[1], q_ref)
    assert torch.equal(q_out[:total], q_ref)
    assert bool((q_out[total:] == 7).all()), "rows behind the last one are left as they were"
    slots, want = ref.kv.tensor(), before.clone()
    for i, (c, r) in enumerate(batch):
        for pos in range(c, c + r):
            want[1, table[i][pos // ps], :, :, pos % ps] = slots[i, 0, :, :, pos]
    assert torch.equal(pool, want)
    ref.close()
    p.close()


# ---- attention ------------------------------------------------------------

def run_attn(p, batch, table, q, layer=0, out=None):
    Q.paged_plan(p.ctx, p.plan, i32([c for c, _ in batch]), i32([r for _, r in batch]), table)
    if out is None:
        out = torch.full_like(q, 7.0)
    Q.paged_attn(p.ctx, p.plan, layer, table, q, out)
    torch.cuda.synchronize()
    return out


def check_attn(p, batch, table, q, out, layer=0, heads=None):
    """Every row of every request against the definition in 64 bits."""
    ps, nkvh, pages = p.pool.page_rows, p.ctx.nkvh, p.pool.pages
    pool = p.pool.tensor()[layer]
    qf, of = q.double().cpu().numpy(), out.double().cpu().numpy()
    r0 = 0
    for i, (c, r) in enumerate(batch):
        if r <= 0:
            continue
        ids = table[i][:-(-(c + r) // ps)].cpu()
        ok = (ids >= 0) & (ids < pages)
        kv = pool[torch.where(ok, ids, 0).long().cuda()].double().cpu().numpy()
        seen = np.repeat(ok.numpy(), ps)[:c + r]
        for h in (range(2 * nkvh) if heads is None else heads):
            k = kv[:, 0, h // 2].reshape(-1, HD)[:c + r]
            v = kv[:, 1, h // 2].reshape(-1, HD)[:c + r]
            cols = slice(h * HD, (h + 1) * HD)
            want, bound = M.attend(qf[r0:r0 + r, cols], np.where(seen[:, None], k, 0),
                                   np.where(seen[:, None], v, 0), range(c, c + r), seen)
            d = np.abs(of[r0:r0 + r, cols] - want)
            assert (d <= bound).all(), (i, h, float((d / bound).max()), np.argwhere(d > bound)[:4])
        r0 += r


SHAPES = [
    # lengths of one, and around slices, tiles and ranges
    [(0, 1)], [(14, 1), (15, 1), (16, 1), (30, 1), (31, 1), (32, 1)],
    [(126, 1), (127, 1), (128, 1), (255, 1), (256, 1), (700, 1)],
    # a lone long one: every range count
    [(4095, 1)], [(8200, 1)], [(16383, 1)],
    # chunks: row blocks of 16 and of 64, their last ones short
    [(0, 2)], [(0, 15), (1, 16), (60, 17)], [(100, 31), (0, 32), (500, 33)],
    [(0, 64)], [(77, 65)], [(1000, 130)], [(0, 300)], [(2000, 16)], [(3000, 70)],
    # idle requests between the others
    [(5, 0), (40, 1), (7, 0), (9, 3), (300, 0)],
    [(900, 1), (0, 45), (33, 7), (1500, 2), (250, 90), (0, 1)],
]


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("batch", SHAPES, ids=lambda b: "+".join(f"{r}@{c}" for c, r in b))
def test_attn_against_64_bits(gpu, ps, batch):
    need = [-(-(c + r) // ps) for c, r in batch]
    pages = sum(need) + 2
    table, _ = shuffled_table(random.Random(7), need, pages, max(need) + 1)
    rows = sum(r for _, r in batch)
    p = Paged(pages, ps, len(batch), rows + 2, layers=2, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(11, *pool.shape))
    q = randn(12, rows + 2, QDIM, std=1.5)
    say(f"attn ps={ps} {batch}")
    out = run_attn(p, batch, i32(table), q, layer=1)
    assert bool((out[rows:] == 7).all()), "rows behind the last one are left as they were"
    check_attn(p, batch, i32(table), q, out, layer=1, heads=(0, 5, 15))
    p.close()


@pytest.mark.parametrize("nkvh", [1, 2, 5, 16])
def test_attn_other_head_counts(gpu, nkvh):
    batch, ps = [(700, 1), (40, 20), (300, 80)], 32
    need = [-(-(c + r) // ps) for c, r in batch]
    table, _ = shuffled_table(random.Random(1), need, sum(need) + 1, max(need))
    p = Paged(sum(need) + 1, ps, 3, 101, nkvh=nkvh, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, 101, 2 * nkvh * HD)
    out = run_attn(p, batch, i32(table), q)
    check_attn(p, batch, i32(table), q, out)
    p.close()


def test_attn_peaked_scores(gpu):
    """Scores of hundreds: weights of 1 and 0, and the running maximum moving
    late."""
    batch, ps = [(900, 1), (500, 40), (200, 100)], 16
    need = [-(-(c + r) // ps) for c, r in batch]
    table, _ = shuffled_table(random.Random(1), need, sum(need), max(need))
    p = Paged(sum(need), ps, 3, 141, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, 141, QDIM, std=30.0)
    out = run_attn(p, batch, i32(table), q)
    check_attn(p, batch, i32(table), q, out, heads=(2, 9))
    p.close()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -65504.0])
def test_attn_ignores_what_lies_behind_the_keys(gpu, bad):
    """Pages hold anything behind the last key, and so do other pages."""
    batch, ps = [(0, 1), (40, 1), (700, 1), (33, 9), (100, 70)], 64
    need = [-(-(c + r) // ps) for c, r in batch]
    pages = sum(need) + 3
    table, _ = shuffled_table(random.Random(2), need, pages, max(need) + 2)
    p = Paged(pages, ps, 5, 82, rope=False)
    pool = p.pool.tensor()
    x = randn(5, *pool.shape)
    y = torch.full_like(x, bad)
    for i, (c, r) in enumerate(batch):
        for j in range(need[i]):
            keep = min(ps, c + r - j * ps)
            y[:, table[i][j], :, :, :keep] = x[:, table[i][j], :, :, :keep]
    pool.copy_(y)
    q = randn(6, 82, QDIM)
    out = run_attn(p, batch, i32(table), q)
    check_attn(p, batch, i32(table), q, out, heads=(0, 7, 14))
    p.close()


@pytest.mark.parametrize("what", ["k", "v", "both"])
@pytest.mark.parametrize("batch,at", [([(20, 12)], 25), ([(900, 14)], 907), ([(300, 90)], 341),
                                      ([(2000, 80)], 2079)])
def test_attn_infinities_reach_only_the_rows_that_see_them(gpu, batch, at, what):
    ps, (c, r) = 16, batch[0]
    need = -(-(c + r) // ps)
    table = [random.Random(4).sample(range(need + 2), need)]
    p = Paged(need + 2, ps, 1, r, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, r, QDIM)
    clean = run_attn(p, batch, i32(table), q).clone()
    page, off = table[0][at // ps], at % ps
    if what != "v":
        pool[0, page, 0, :, off, 3] = float("nan")
    if what != "k":
        pool[0, page, 1, :, off, 5] = float("inf")
    out = run_attn(p, batch, i32(table), q)
    check_attn_rows = at - c  # rows before it do not see the key
    assert bool(torch.isfinite(out[:check_attn_rows]).all())
    d = (out[:check_attn_rows].double() - clean[:check_attn_rows].double()).abs()
    # Recomputed in f32 weights: each side is within its own bound of the
    # exact value, 2 * (2^-11 (|out| + 2 * 1.05 mean |v - out|)) + sums.
    assert float(d.max()) <= 2 * (2.0 ** -11 * (4.5 + 2.1 * 9) + 2 * (c + r) * 2.0 ** -24 * 5), float(d.max())
    seers = out[check_attn_rows:].view(-1, NQH, HD)
    if what == "v":
        assert bool(torch.isinf(seers[:, :, 5]).all())
        assert bool(torch.isfinite(seers[:, :, 6:]).all())
    else:
        assert bool(torch.isnan(seers).all())
    p.close()


def test_attn_leaves_evicted_pages_out(gpu):
    """Entries outside the pool: their keys are not attended; a row that sees
    none gives zeros."""
    batch, ps = [(1000, 1), (250, 20), (600, 100), (64, 1)], 16
    need = [-(-(c + r) // ps) for c, r in batch]
    pages = sum(need)
    table, _ = shuffled_table(random.Random(2), need, pages, max(need))
    table[0][4:50] = [-1] * 46
    table[1][0], table[1][3] = pages, 2 ** 31 - 1
    table[2][1:30] = [-7] * 29
    p = Paged(pages, ps, 4, 122, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    pool[:, 0] = float("nan") if 0 not in sum(table, []) else pool[:, 0]
    q = randn(6, 122, QDIM)
    out = run_attn(p, batch, i32(table), q)
    check_attn(p, batch, i32(table), q, out, heads=(0, 11))
    p.close()


def test_attn_of_a_row_without_keys_is_zero(gpu):
    """Every cached page evicted, and the new row's page an id that the ring
    should not hold: the row sees no key."""
    p = Paged(8, 16, 2, 2, rope=False)
    p.pool.tensor().copy_(randn(5, *p.pool.tensor().shape))
    table = i32([[-1, 9, -4, 8, -1], [3, -1, -1, -1, -1]])
    Q.paged_plan(p.ctx, p.plan, i32([64, 5]), i32([1, 1]), table, i32([-1, 1, 2, 4, 5, 6, 7, 0]), i32([0, 1]))
    assert p.plan.status.tolist() == [0, 0] and p.plan.row_slot.tolist() == [-1, 53]
    q = randn(6, 2, QDIM)
    out = torch.full_like(q, 7.0)
    Q.paged_attn(p.ctx, p.plan, 0, table, q, out)
    torch.cuda.synchronize()
    assert bool((out[0] == 0).all())
    check_attn(p, [(5, 1)], table[1:], q[1:], out[1:], heads=(0, 8))
    p.close()


def test_attn_bits_do_not_depend_on_the_batch_or_the_pages(gpu):
    batch, ps = [(900, 1), (2100, 20), (33, 7), (1500, 2), (250, 90), (5000, 1)], 16
    need = [-(-(c + r) // ps) for c, r in batch]
    pages = 2 * sum(need)
    rows = sum(r for _, r in batch)
    p = Paged(pages, ps, len(batch), rows, rope=False)
    pool = p.pool.tensor()
    t1, other = shuffled_table(random.Random(2), need, pages, max(need))
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, rows, QDIM)
    whole = run_attn(p, batch, i32(t1), q).clone()
    # Alone, on other pages.
    r0 = 0
    for i, (c, r) in enumerate(batch):
        ids = other[:need[i]]
        pool[:, i32(ids).long()] = pool[:, i32(t1[i][:need[i]]).long()]
        out = run_attn(p, [(c, r)], i32([ids]), q[r0:r0 + r].contiguous())
        assert torch.equal(out, whole[r0:r0 + r]), i
        r0 += r
    assert torch.equal(run_attn(p, batch, i32(t1), q), whole)
    p.close()


def test_attn_shared_prefix_pages(gpu):
    """One page listed by several requests."""
    batch, ps = [(100, 1), (100, 5), (100, 40)], 32
    table = [[3, 1, 0, 4, 5], [3, 1, 0, 2, 6], [3, 1, 0, 7, 8]]
    p = Paged(9, ps, 3, 46, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    q = randn(6, 46, QDIM)
    out = run_attn(p, batch, i32(table), q)
    check_attn(p, batch, i32(table), q, out, heads=(3,))
    p.close()


def test_attn_leaves_refused_requests_alone(gpu):
    p = Paged(8, 16, 3, 40, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    table = i32([[0, -1], [1, 2], [3, 4]])
    q = randn(6, 33, QDIM)
    out = run_attn(p, [(14, 10), (20, 3), (0, 20)], table, q)  # the first lacks its second page
    assert p.plan.status.tolist() == [M.EINVAL, 0, 0]
    assert bool((out[:10] == 7).all())
    assert not bool((out[10:] == 7).any())
    # fewer rows than planned: those behind are left out
    part = torch.full((20, QDIM), 7.0, dtype=torch.float16, device="cuda")
    Q.paged_attn(p.ctx, p.plan, 0, table, q[:20].contiguous(), part)
    assert torch.equal(part[:13], out[:13])
    check_attn(p, [(20, 3)], table[1:2], q[10:13], part[10:13], heads=(0,))
    check_attn(p, [(0, 7)], table[2:3], q[13:20], part[13:20], heads=(0, 9))
    p.close()


def test_attn_pages_past_32_bits(gpu):
    """A layer of more than 2^32 bytes, and the next layer behind it."""
    ps = 256  # 1 MB a page
    pages = 4200
    p = Paged(pages, ps, 2, 41, layers=2, rope=False)
    pool = p.pool.tensor()
    table = [[pages - 1, 2, pages - 2, 4099], [4101, 1, -1, -1]]
    batch = [(800, 1), (300, 40)]
    ids = i32([x for t in table for x in t if x >= 0]).long()
    for layer in (0, 1):
        pool[layer, ids] = randn(layer, len(ids), *pool.shape[2:])
    q = randn(6, 41, QDIM)
    for layer in (0, 1):
        out = run_attn(p, batch, i32(table), q, layer=layer)
        check_attn(p, batch, i32(table), q, out, layer=layer, heads=(0, 15))
    p.close()


# ---- together -------------------------------------------------------------

def test_two_plans_on_two_streams(gpu):
    """Two plans of one pool on streams of their own, each with split ranges."""
    ps = 16
    p = Paged(900, ps, 4, 64, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(5, *pool.shape))
    plan2 = Q.PagedPlan(p.ctx, p.pool, 4, 64)
    rnd = random.Random(8)
    work = []
    for plan, batch in ((p.plan, [(5000, 1), (700, 20)]), (plan2, [(3000, 4), (2500, 1)])):
        need = [-(-(c + r) // ps) for c, r in batch]
        table, _ = shuffled_table(rnd, need, 900, max(need))
        q = randn(len(work), sum(r for _, r in batch), QDIM)
        work.append((plan, batch, i32(table), q, torch.empty_like(q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for plan, batch, table, q, out, st in work:
            with torch.cuda.stream(st):
                Q.paged_plan(p.ctx, plan, i32([c for c, _ in batch]), i32([r for _, r in batch]), table)
                Q.paged_attn(p.ctx, plan, 0, table, q, out)
    torch.cuda.synchronize()
    for plan, batch, table, q, out, st in work:
        check_attn(p, batch, table, q, out, heads=(1,))
    plan2.close()
    p.close()


def test_replayed_graph_decodes_on(gpu):
    """A captured token step whose lengths, table and ring live on the GPU:
    every replay appends a row to each request, takes pages as they fill, and
    gives what the slot pool's step gives."""
    layers, n, ps, start = 2, 3, 16, [14, 0, 130]
    p = Paged(40, ps, n, n, layers=layers)
    ref = Gpu(n, 256, layers=layers)
    g = randn(3, layers, 2, HD) + 1
    ring, cursor = p.pool.free_ring()
    table = torch.full((n, 12), -1, dtype=torch.int32, device="cuda")
    # Prompts, eagerly.
    big = Q.PagedPlan(p.ctx, p.pool, n, 160)
    Q.paged_plan(p.ctx, big, i32([0] * n), i32(start), table, ring, cursor)
    qkv = randn(9, layers, sum(start), TOT)
    qo = torch.empty((sum(start), QDIM), dtype=torch.float16, device="cuda")
    for l in range(layers):
        Q.paged_append(p.ctx, big, l, qkv[l], g[l, 0], g[l, 1], qo)
        Q.qk_norm_rope_append(ref.ctx, ref.kv, l, [(i, 0, s) for i, s in enumerate(start) if s], qkv[l],
                              g[l, 0], g[l, 1], qo)
    p.plan.lens[:n].copy_(big.lens[:n])
    p.plan.cursor.copy_(big.cursor)
    x = torch.zeros((layers, n, TOT), dtype=torch.float16, device="cuda")
    ones = i32([1] * n)
    q = torch.empty((n, QDIM), dtype=torch.float16, device="cuda")
    out = torch.empty((layers, n, QDIM), dtype=torch.float16, device="cuda")

    def step():
        Q.paged_plan(p.ctx, p.plan, p.plan.lens, ones, table, ring, p.plan.cursor)
        for l in range(layers):
            Q.paged_append(p.ctx, p.plan, l, x[l], g[l, 0], g[l, 1], q)
            Q.paged_attn(p.ctx, p.plan, l, table, q, out[l])

    # An eager first step (code loading), then the capture.
    want = torch.empty((n, QDIM), dtype=torch.float16, device="cuda")
    graph = None
    for t in range(50):
        x.copy_(randn(100 + t, layers, n, TOT))
        if t == 1:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        if graph is None:
            step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert p.plan.status[:n].tolist() == [0] * n
        assert p.plan.lens[:n].tolist() == [s + t + 1 for s in start]
        for l in range(layers):
            Q.decode_step(ref.ctx, ref.kv, l, [s + t for s in start], x[l], g[l, 0], g[l, 1], want)
            d = (out[l].double() - want.double()).abs()
            # Both within 2^-11 (2.1 mean |v - out| + |out|) of the exact
            # value; the slot step keeps f32 weights.
            assert float(d.max()) <= 2.0 ** -11 * (2.1 * 9 + 2 * 5), (t, l, float(d.max()))
    held = table[table >= 0]
    assert held.unique().numel() == held.numel() == sum(-(-(s + 50) // ps) for s in start)
    kv, slots = p.pool.tensor(), ref.kv.tensor()
    for i, s in enumerate(start):
        for pos in range(s + 50):
            page = int(table[i, pos // ps])
            assert torch.equal(kv[:, page, :, :, pos % ps], slots[i, :, :, :, pos])
    big.close()
    ref.close()
    p.close()


def test_a_server_admits_grows_and_ends_requests(gpu):
    """Random steps over one pool: chunks and single rows, requests that end
    and others that take their pages.  Every row's output is the definition
    over the rows its request has stored, and no page is ever held twice."""
    rnd = random.Random(17)
    ps, pages, n, max_rows = 16, 16, 6, 120
    p = Paged(pages, ps, n, max_rows)
    ring, _ = p.pool.free_ring()
    p.plan.cursor.copy_(i32([0, pages]))
    p.plan.lens.zero_()
    table = torch.full((n, 40), -1, dtype=torch.int32, device="cuda")
    g = randn(3, 2, HD) + 1
    lens = [0] * n
    refused = 0
    for t in range(40):
        rows = []
        for i in range(n):
            if lens[i] and rnd.random() < 0.12:
                rows.append(-1)
            elif lens[i] == 0:
                rows.append(rnd.choice([0, rnd.randint(1, 70)]))
            else:
                rows.append(rnd.choice([1, 1, 1, 0, rnd.randint(2, 20)]))
        while sum(max(r, 0) for r in rows) > max_rows:
            rows[rows.index(max(rows))] = 0
        Q.paged_plan(p.ctx, p.plan, p.plan.lens, i32(rows), table, ring, p.plan.cursor)
        total = sum(max(r, 0) for r in rows)
        status = p.plan.status[:n].tolist()
        refused += sum(s != 0 for s in status)
        if total:
            qkv = randn(1000 + t, total, TOT)
            q = torch.zeros((total, QDIM), dtype=torch.float16, device="cuda")
            out = torch.full((total, QDIM), 7.0, dtype=torch.float16, device="cuda")
            Q.paged_append(p.ctx, p.plan, 0, qkv, g[0], g[1], q)
            Q.paged_attn(p.ctx, p.plan, 0, table, q, out)
            torch.cuda.synchronize()
            r0 = 0
            for i in range(n):
                m = max(rows[i], 0)
                if m and status[i] == 0:
                    check_attn(p, [(lens[i], m)], table[i:i + 1], q[r0:r0 + m], out[r0:r0 + m],
                               heads=(rnd.randrange(NQH),))
                elif m:
                    assert bool((out[r0:r0 + m] == 7).all())
                r0 += m
        lens = [0 if r == -1 else c + r if s == 0 else c for c, r, s in zip(lens, rows, status)]
        assert p.plan.lens[:n].tolist() == lens
        held = [x for i in range(n) for x in table[i, :-(-lens[i] // ps)].tolist()]
        head, free = p.plan.cursor.tolist()
        idle = [ring[(head + k) % pages].item() for k in range(free)]
        assert sorted(held + idle) == list(range(pages)), t
    assert refused, "the pool is small enough for refusals"
    p.close()
