"""8-bit pages on the GPU: what stage (a) stores against a plain
implementation, code by code, and attention over them against the definition
in 64 bits and against an f16 pool of the same values, bit by bit."""
from __future__ import annotations

import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged8_model as M8  # noqa: E402
import qasr_attn as Q  # noqa: E402
from gpu_helpers import rope_tables, say  # noqa: E402
from test_gpu_paged import SHAPES, Paged, check_attn, i32, randn, run_attn, shuffled_table  # noqa: E402
from test_gpu_paged_work import WIDE, assert_wide  # noqa: E402
from workloads import HD, NKVH, QDIM, TOT  # noqa: E402

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


class Paged8(Paged):
    """With e4m3 pages."""

    def __init__(self, pages, ps, requests, rows, nkvh=NKVH, layers=1, max_seq=16384, rope=True):
        self.ctx = Q.Context(2 * nkvh, nkvh, HD, layers, 1e-6, max_seq, 0)
        if rope:
            c, s = rope_tables()
            self.ctx.set_rope_tables(c[:max_seq], s[:max_seq])
        self.pool = Q.PagePool(self.ctx, pages, ps, "e4m3")
        self.plan = Q.PagedPlan(self.ctx, self.pool, requests, rows)


def bits(t):
    return t.view(torch.uint8)


def values(pool):
    """What an e4m3 pool stands for, in f16: exact for units of 2^-15 .. 2^8."""
    x = pool.tensor().float().view(*pool.scales().shape, 16, HD)
    return (x * pool.scales().float()[..., None, None]).flatten(-3, -2).half()


def fill(pool, seed, lo=-10, hi=-6, std=100.0):
    """Random values and units 2^lo .. 2^(hi-1)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t, s = pool.tensor(), pool.scales()
    t.copy_((torch.randn(t.shape, device="cuda", generator=g) * std).clamp_(-448, 448))
    bits(s).copy_(torch.randint(lo + 127, hi + 127, s.shape, device="cuda", generator=g))


def both(batch, ps, nkvh=NKVH, seed=1, spare=2, layers=1):
    """An e4m3 pool, an f16 pool and a table of the batch for both."""
    need = [-(-(c + r) // ps) for c, r in batch]
    pages, rows = sum(need) + spare, sum(max(r, 0) for _, r in batch)
    table, _ = shuffled_table(random.Random(seed), need, pages, max(need) + 1)
    a = Paged8(pages, ps, len(batch), rows + 2, nkvh=nkvh, layers=layers, rope=False)
    b = Paged(pages, ps, len(batch), rows + 2, nkvh=nkvh, layers=layers, rope=False)
    return a, b, table, rows


def same_bits(x, y):
    return bool(((x.view(torch.int16) == y.view(torch.int16)) | (x.isnan() & y.isnan())).all())


# ---- pool -------------------------------------------------------------------

def test_pool_is_zero_and_half_as_large(gpu):
    a, b, _, _ = both([(40, 1)], 32, layers=3)
    assert a.pool.info().bytes * 2 == b.pool.info().bytes
    assert a.pool.tensor().shape == b.pool.tensor().shape
    assert a.pool.scales().shape == (3, a.pool.pages, 2, NKVH, 2)
    assert bool((bits(a.pool.tensor()) == 0).all()) and bool((a.pool.scales().float() == 1).all())
    with pytest.raises(Q.QasrError) as e:
        b.pool.scales()
    assert e.value.code == Q.QASR_EINVAL
    with pytest.raises(Q.QasrError):
        Q.PagePool(a.ctx, 4, 16, "int8")
    for ps in (8, 48, 512):
        with pytest.raises(Q.QasrError):
            Q.PagePool(a.ctx, 4, ps, "e4m3")
    a.close()
    b.close()


# ---- append -----------------------------------------------------------------

def run_append(p8, p16, batch, table, qkv, gains, layer=0):
    """The step on both pools.  The f16 pool's stage (a) has its own tests: its
    K and V are what the codes are rounded from."""
    rows = sum(max(r, 0) for _, r in batch)
    out = []
    for p in (p8, p16):
        q = torch.full((rows, QDIM * p.ctx.nkvh // NKVH), 7.0, dtype=torch.float16, device="cuda")
        Q.paged_plan(p.ctx, p.plan, i32([c for c, _ in batch]), i32([r for _, r in batch]), i32(table))
        Q.paged_append(p.ctx, p.plan, layer, qkv, gains[0], gains[1], q)
        out.append(q)
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]), "roped queries"


def step_codes(codes, units, p16, batch, table, ps, layer=0):
    """The plain implementation of the same step: codes [layer][page][2][kvh]
    [ps][hd], units [..][ps / 16] exponents, changed in place."""
    x = p16.pool.tensor()[layer].double().cpu().numpy()
    pages, nkvh = x.shape[0], x.shape[2]
    for i, (c, r) in enumerate(batch):
        at = c
        while at < c + r:
            to = min(c + r, at // 16 * 16 + 16)
            page, row = table[i][at // ps], at % ps
            if 0 <= page < pages:
                b = row // 16
                z = slice(16 * b, 16 * b + 16)
                for kv in range(2):
                    for h in range(nkvh):
                        codes[layer, page, kv, h, z], units[layer, page, kv, h, b] = M8.store(
                            codes[layer, page, kv, h, z], int(units[layer, page, kv, h, b]), row % 16,
                            x[page, kv, h, row:row + to - at])
            at = to


def check_codes(p8, codes, units):
    got = M8.canon(bits(p8.pool.tensor()).cpu().numpy().astype(np.int64))
    want = M8.canon(codes)
    assert np.array_equal(bits(p8.pool.scales()).cpu().numpy().astype(np.int64) - 127, units)
    d = got != want
    assert not d.any(), (int(d.sum()), np.argwhere(d)[:4], got[d][:4], want[d][:4])


def new_rows(seed, rows, nkvh=NKVH, wild=False):
    """Raw rows; `wild`: V of every size down to nothing, up to the largest f16
    number, some of it not finite."""
    qkv = randn(seed, rows, 4 * nkvh * HD)
    if wild:
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + 1)
        v = qkv[:, 3 * nkvh * HD:].view(rows, nkvh, HD)
        e = torch.randint(-26, 15, (rows, nkvh, 1), device="cuda", generator=g)
        v.copy_(v.double() * 2.0 ** e)
        kind = torch.randint(0, 12, (rows, nkvh), device="cuda", generator=g)
        v[kind == 0] = 0.0
        v[kind == 1] = 65504.0
        at = torch.randint(0, HD, (rows, nkvh), device="cuda", generator=g)
        for k, bad in ((2, INF), (3, -INF), (4, NAN)):
            row, head = (kind == k).nonzero().unbind(1)
            v[row, head, at[row, head]] = bad
        row, head = (kind == 5).nonzero().unbind(1)
        v[row, head] = INF
    return qkv


@pytest.mark.parametrize("ps", [16, 32, 256])
@pytest.mark.parametrize("wild", [False, True])
def test_append_against_plain(gpu, ps, wild):
    """Steps one after the other: prompts, chunks that start inside a block,
    single rows, idle requests, a step that starts every request anew."""
    steps = [[(0, 5), (0, 40), (0, 1), (0, 16)], [(5, 1), (40, 30), (1, 14), (16, 0)],
             [(6, 1), (70, 1), (15, 1), (16, 1)], [(7, 25), (71, 9), (16, 17), (17, 15)],
             [(32, 1), (80, 0), (33, 1), (32, 1)], [(0, 3), (0, 1), (0, 64), (0, 2)]]
    need = [8 * 16 // ps + 1] * 4
    pages = sum(need) + 2
    table, _ = shuffled_table(random.Random(ps), need, pages, need[0])
    a, b = Paged8(pages, ps, 4, 128, layers=2), Paged(pages, ps, 4, 128, layers=2)
    fill(a.pool, 3)
    gains = randn(4, 2, HD) + 1
    codes = bits(a.pool.tensor()).cpu().numpy().astype(np.int64)
    units = bits(a.pool.scales()).cpu().numpy().astype(np.int64) - 127
    for n, batch in enumerate(steps):
        say(f"append8 ps={ps} wild={wild} step {n}")
        run_append(a, b, batch, table, new_rows(10 * n, sum(r for _, r in batch), wild=wild), gains, 1)
        step_codes(codes, units, b, batch, table, ps, 1)
        check_codes(a, codes, units)
    a.close()
    b.close()


@pytest.mark.parametrize("nkvh", [1, 3, 16])
def test_append_of_many_rows_and_other_head_counts(gpu, nkvh):
    batch, ps = [(3, 200), (20, 1), (0, 37), (31, 2), (9, 100)] + [(i, 1) for i in range(40)], 64
    need = [-(-(c + r) // ps) for c, r in batch]
    pages, rows = sum(need) + 1, sum(r for _, r in batch)
    table, _ = shuffled_table(random.Random(1), need, pages, max(need))
    a, b = (P(pages, ps, len(batch), rows, nkvh=nkvh) for P in (Paged8, Paged))
    fill(a.pool, 3)
    codes = bits(a.pool.tensor()).cpu().numpy().astype(np.int64)
    units = bits(a.pool.scales()).cpu().numpy().astype(np.int64) - 127
    run_append(a, b, batch, table, new_rows(1, rows, nkvh, True), randn(4, 2, HD) + 1)
    step_codes(codes, units, b, batch, table, ps)
    check_codes(a, codes, units)
    a.close()
    b.close()


def test_append_leaves_rows_without_a_slot_out(gpu):
    """A page outside the pool in the middle of a chunk, a refused request."""
    ps, pages = 16, 12
    a, b = Paged8(pages, ps, 3, 90), Paged(pages, ps, 3, 90)
    fill(a.pool, 3)
    codes = bits(a.pool.tensor()).cpu().numpy().astype(np.int64)
    units = bits(a.pool.scales()).cpu().numpy().astype(np.int64) - 127
    # With a ring the ids come as they are: the second fresh page is no page.
    lens, rows = [7, -1, 0], [50, 3, 20]
    table = [[4, -1, -1, -1, -1], [0, -1, -1, -1, -1], [-1] * 5]
    ring = [1, pages + 9, 2, 3, 5] + [-1] * (pages - 5)
    qkv, gains = new_rows(1, 73, wild=True), randn(4, 2, HD) + 1
    out = []
    for p in (a, b):
        q = torch.full((73, QDIM), 7.0, dtype=torch.float16, device="cuda")
        t = i32(table)
        Q.paged_plan(p.ctx, p.plan, i32(lens), i32(rows), t, i32(ring), i32([0, 5]))
        Q.paged_append(p.ctx, p.plan, 0, qkv, gains[0], gains[1], q)
        out.append(q)
    assert p.plan.status.tolist() == [0, 1, 0]
    assert torch.equal(out[0], out[1])
    t = t.tolist()
    step_codes(codes, units, b, [(7, 50), (0, 0), (0, 20)], [t[0], t[1], t[2]], ps)
    check_codes(a, codes, units)
    a.close()
    b.close()


# ---- attention --------------------------------------------------------------

@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("batch", SHAPES + WIDE[:3] + WIDE[-2:], ids=lambda b: "+".join(f"{r}@{c}" for c, r in b))
def test_attn_has_the_bits_of_f16_pages(gpu, ps, batch):
    a, b, table, rows = both(batch, ps, layers=2)
    fill(a.pool, 5)
    b.pool.tensor().copy_(values(a.pool))
    q = randn(6, rows + 2, QDIM, std=1.5)
    say(f"attn8 ps={ps} {batch}")
    x, y = run_attn(a, batch, i32(table), q, layer=1), run_attn(b, batch, i32(table), q, layer=1)
    assert same_bits(x, y)
    assert bool((x[rows:] == 7).all())
    a.close()
    b.close()


class Values:
    """An e4m3 pool's values in the place of an f16 pool, for check_attn."""

    def __init__(self, p):
        self.ctx, self.pool = p.ctx, self
        self.page_rows, self.pages, self.at = p.pool.page_rows, p.pool.pages, values(p.pool)

    def tensor(self):
        return self.at


@pytest.mark.parametrize("batch", [[(30, 1), (700, 8)], [(500, 12), (0, 33)], [(1500, 1)], [(60, 130)]])
def test_attn_against_64_bits(gpu, batch):
    a, b, table, rows = both(batch, 32)
    fill(a.pool, 5, -12, -5)
    q = randn(6, rows + 2, QDIM, std=1.5)
    out = run_attn(a, batch, i32(table), q)
    check_attn(Values(a), batch, i32(table), q, out, heads=(0, 7, 15))
    a.close()
    b.close()


@pytest.mark.parametrize("nkvh", [1, 2, 5, 16])
def test_attn_other_head_counts(gpu, nkvh):
    batch = [(700, 1), (40, 20), (300, 80), (4000, 512)]
    assert_wide(batch)
    a, b, table, rows = both(batch, 32, nkvh=nkvh)
    fill(a.pool, 5)
    b.pool.tensor().copy_(values(a.pool))
    q = randn(6, rows + 2, 2 * nkvh * HD)
    assert same_bits(run_attn(a, batch, i32(table), q), run_attn(b, batch, i32(table), q))
    a.close()
    b.close()


@pytest.mark.parametrize("lo,hi", [(-15, -14), (7, 9), (-15, 9)])
@pytest.mark.parametrize("batch", [[(40, 1), (600, 5)], [(300, 14)], [(4000, 530)]])
def test_attn_at_the_ends_of_the_units(gpu, lo, hi, batch):
    """f16's smallest numbers, and its largest: 240 times 2^8."""
    a, b, table, rows = both(batch, 16)
    fill(a.pool, 5, lo, hi)
    t = a.pool.tensor()
    t.copy_(t.float().clamp(-240, 240))
    b.pool.tensor().copy_(values(a.pool))
    q = randn(6, rows + 2, QDIM)
    assert same_bits(run_attn(a, batch, i32(table), q), run_attn(b, batch, i32(table), q))
    a.close()
    b.close()


@pytest.mark.parametrize("what", ["k", "v", "both"])
@pytest.mark.parametrize("batch,at", [([(20, 12)], 25), ([(1500, 6)], 1502), ([(900, 14)], 907), ([(300, 90)], 341),
                                      ([(4000, 520)], 4277)])
def test_attn_nan_reaches_only_the_rows_that_see_it(gpu, batch, at, what):
    ps = 16
    a, b, table, rows = both(batch, ps)
    fill(a.pool, 5)
    page, row = table[0][at // ps], at % ps
    for kv in (0, 1):
        if what in (("k", "both"), ("v", "both"))[kv]:
            bits(a.pool.tensor())[0, page, kv, :, row, 7] = 0x7F
    b.pool.tensor().copy_(values(a.pool))
    q = randn(6, rows + 2, QDIM)
    x, y = run_attn(a, batch, i32(table), q), run_attn(b, batch, i32(table), q)
    assert same_bits(x, y)
    seen = at - batch[0][0]
    assert bool(x[:seen].isfinite().all()) and bool(x[seen:rows].isnan().any(1).all())
    a.close()
    b.close()


@pytest.mark.parametrize("batch", [[(600, 1), (300, 9)], [(4000, 512)]])
def test_attn_ignores_what_lies_behind_the_keys(gpu, batch):
    """NaN codes and NaN scales behind the last key, and evicted pages."""
    ps = 64
    a, b, table, rows = both(batch, ps)
    fill(a.pool, 5)
    q = randn(6, rows + 2, QDIM)
    table[0][3] = -1
    want = run_attn(a, batch, i32(table), q)
    for i, (c, r) in enumerate(batch):
        n = c + r
        page = table[i][(n - 1) // ps]
        if n % ps:
            bits(a.pool.tensor())[0, page, :, :, n % ps:] = 0x7F
            bits(a.pool.scales())[0, page, :, :, -(-(n % ps) // 16):] = 0xFF
    used = {p for t in table for p in t}
    for p in set(range(a.pool.pages)) - used:
        bits(a.pool.tensor())[0, p] = 0xFF
    assert torch.equal(run_attn(a, batch, i32(table), q), want)
    check_attn(Values(a), batch, i32(table), q, want, heads=(3,))
    a.close()
    b.close()


# ---- together ---------------------------------------------------------------

def test_replayed_token_after_token(gpu):
    """A graph of a step (plan, stage (a), attention, two layers), captured on a
    stream of its own, that moves on by itself, with eager work between the
    replays: the same bits as the same steps without a graph."""
    ps, steps = 16, 20  # past the end of blocks and pages
    rnd = random.Random(3)
    lens = [5, 15, 16, 60]
    out = []
    for captured in (False, True):
        p = Paged8(40, ps, 4, 4, layers=2)
        fill(p.pool, 1)
        table, _ = shuffled_table(rnd if not captured else random.Random(3), [-(-(c + steps) // ps) for c in lens], 40, 8)
        table, cur, one = i32(table), i32(lens), i32([1] * 4)
        gains = randn(2, 2, 2, HD, std=0.1) + 1
        x = torch.zeros((2, 4, TOT), dtype=torch.float16, device="cuda")
        q, o = (torch.zeros((2, 4, QDIM), dtype=torch.float16, device="cuda") for _ in range(2))

        def step():
            Q.paged_plan(p.ctx, p.plan, p.plan.lens, one, table)
            for l in range(2):
                Q.paged_append(p.ctx, p.plan, l, x[l], gains[l, 0], gains[l, 1], q[l])
                Q.paged_attn(p.ctx, p.plan, l, table, q[l], o[l])

        if captured:
            p.plan.lens.copy_(cur)
            step()
            fill(p.pool, 1)
            torch.cuda.synchronize()
            graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(graph, stream=stream):
                step()
        p.plan.lens.copy_(cur)
        got = []
        for k in range(steps):
            x.copy_(randn(100 + k, 2, 4, TOT) * 2.0 ** (k % 5 - 2))
            graph.replay() if captured else step()
            assert p.plan.status.tolist() == [0] * 4
            got.append(o.clone())
        out.append((got, bits(p.pool.tensor()).clone(), bits(p.pool.scales()).clone()))
        torch.cuda.synchronize()
        if captured:
            del graph
        p.close()
    (a, pool_a, units_a), (b, pool_b, units_b) = out
    assert all(same_bits(s, t) for s, t in zip(a, b))
    assert torch.equal(pool_a, pool_b) and torch.equal(units_a, units_b)


def test_pages_past_32_bits(gpu):
    """Stage (a) into pages whose offsets pass 2^32 bytes, a prompt and single
    rows, and attention over them."""
    ps, pages = 256, 9000
    batch = [(0, 700), (0, 1), (0, 40)]
    p8, p16 = Paged8(pages, ps, 3, 800), Paged(pages, ps, 3, 800)
    table = [[pages - 1, pages - 300, pages - 7], [pages - 2, -1, -1], [pages - 400, -1, -1]]
    assert (pages - 400) * 2 * NKVH * ps * HD > 1 << 32
    qkv, gains = new_rows(5, 741), randn(6, 2, HD, std=0.1) + 1
    run_append(p8, p16, batch, table, qkv, gains)
    used = torch.tensor([x for t in table for x in t if x >= 0], device="cuda")
    x, u = p8.pool.tensor()[0, used], p8.pool.scales()[0, used]
    exact = (x.float().view(*u.shape, 16, HD) * u.float()[..., None, None]).flatten(-3, -2).half()
    near = p16.pool.tensor()[0, used]
    # Half a step of a value, or of the block's unit.
    bound = near.float().abs() * 2.0 ** -4 + (u.float() * 2.0 ** -10).repeat_interleave(16, -1)[..., None]
    assert bool(((exact.float() - near.float()).abs() <= bound).all())
    p16.pool.tensor()[0, used] = exact
    q = randn(7, 741, QDIM)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    for p, out in ((p8, a), (p16, b)):
        Q.paged_attn(p.ctx, p.plan, 0, i32(table), q, out)
    assert same_bits(a, b) and bool((a[700] != 0).any())
    p8.close()
    p16.close()


def test_steps_of_a_server(gpu):
    """Admission, chunks and decoding over both kinds of pool, with a ring: the
    outputs over 8 bits are the definition's over what the pages stand for,
    and near those over f16."""
    ps, n, pages = 16, 3, 64
    a, b = Paged8(pages, ps, n, 200, layers=2), Paged(pages, ps, n, 200, layers=2)
    state = []
    for p in (a, b):
        ring, cur = p.pool.free_ring()
        p.plan.cursor.copy_(cur)
        p.plan.lens.zero_()
        state.append((torch.full((n, 20), -1, dtype=torch.int32, device="cuda"), ring))
    gains = randn(4, 2, 2, HD, std=0.1) + 1
    lens = [0] * n
    for step, rows in enumerate([(37, 0, 64), (20, 50, 1), (1, 1, 1), (1, 30, 1), (1, 1, -1), (1, 1, 17)]):
        total = sum(max(r, 0) for r in rows)
        qkv = randn(100 + step, 2, total, TOT)
        outs = []
        for p, (table, ring) in zip((a, b), state):
            Q.paged_plan(p.ctx, p.plan, p.plan.lens, i32(rows), table, ring, p.plan.cursor)
            out = torch.empty((2, total, QDIM), dtype=torch.float16, device="cuda")
            q = torch.empty_like(out)
            for l in range(2):
                Q.paged_append(p.ctx, p.plan, l, qkv[l], gains[l, 0], gains[l, 1], q[l])
                Q.paged_attn(p.ctx, p.plan, l, table, q[l], out[l])
            outs.append((q, out))
        assert a.plan.status.tolist() == [0] * n
        assert torch.equal(outs[0][0], outs[1][0])
        batch = [(c, max(r, 0)) for c, r in zip(lens, rows)]
        for l in range(2):
            check_attn(Values(a), batch, state[0][0].cpu(), outs[0][0][l], outs[0][1][l], layer=l, heads=(0, 9))
        # A value is off by 2^-4 of itself at most, a score of mean square 1 by
        # as much of its terms: far below half of the outputs' size.
        x, y = outs[0][1].float(), outs[1][1].float()
        assert float((x - y).norm() / y.norm()) < 0.5
        lens = [0 if r == -1 else c + r for c, r in zip(lens, rows)]
    a.close()
    b.close()
