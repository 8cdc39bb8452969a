"""Forks of paged requests where their arrays are at their ends: cursors that
are none, parents without rows, the longest request, counts that are too low;
and a beam search whose every beam is compared with one that shares no page."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

import beam_model as B  # noqa: E402
import qasr_attn as Q  # noqa: E402
from gpu_helpers import say  # noqa: E402
from test_gpu_fork import State  # noqa: E402
from test_gpu_paged import Paged, i32, randn  # noqa: E402
from test_gpu_paged8 import Paged8, bits, same_bits  # noqa: E402
from workloads import HD, NKVH, QDIM, TOT  # noqa: E402

pytestmark = pytest.mark.gpu


def arrays(s, parent):
    return [i32(x) for x in (s.lens, parent, s.table, s.shared, s.ring, s.cursor)]


@pytest.mark.parametrize("cursor", [[-1, 3], [20, 3], [0, -1], [0, 21]])
def test_a_cursor_that_is_none_takes_no_pages_back(gpu, cursor):
    """Without copies too the call is refused: it cannot put pages into a ring
    whose place it does not know, nor lose the ring's own."""
    s = State(4, 20, 16, 4)
    for i, c in enumerate((20, 33, 16, 0)):
        s.grow(i, c)
    right, s.cursor = s.cursor, cursor
    pages = bits(s.p.pool.tensor()).clone()
    for parent in ([0, -1, 2, 3], [0, 1, 2, 3], [-1] * 4, [2] * 4):
        d = arrays(s, parent)
        before = [t.clone() for t in d]
        Q.paged_fork(s.p.ctx, s.fork, *d)
        assert s.fork.status.tolist() == [B.EINVAL] * 4, parent
        assert all(torch.equal(a, b) for a, b in zip(d, before)), parent
    assert torch.equal(bits(s.p.pool.tensor()), pages)
    s.cursor = right
    s.step([2, 2, 2, -1])
    s.step([-1] * 4)
    assert s.cursor[1] == 20
    s.close()


def test_an_empty_ring(gpu):
    """Parents without rows or with whole pages alone want no copy, others do."""
    s = State(4, 20, 16, 4)
    s.cursor = [7, 0]
    status, _ = s.step([0, 0, 0, 0])
    assert status == [0] * 4
    s.cursor = [0, 20]
    s.grow(0, 32)
    s.grow(1, 5)
    s.new_pages(s.cursor[1])
    status, copies = s.step([0, 1, 0, 0])
    assert status == [0] * 4 and not copies
    status, _ = s.step([0, 1, 1, 0])
    assert status == [0, 0, B.ENOMEM, 0]
    s.close()


def test_the_longest_request(gpu):
    """2^31 - 1 rows, all but a few pages of them evicted: the table's last column
    is shared out and given back as any other."""
    ps, width, pages, most = 256, 1 << 23, 8, (1 << 31) - 1
    p = Paged(pages, ps, 2, 4, nkvh=1, rope=False)
    pool = p.pool.tensor()
    pool.copy_(randn(1, *pool.shape))
    fork = Q.PagedFork(p.ctx, p.pool, 2, width)
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    table[0, 0], table[0, width - 1] = 3, 5
    lens, shared = i32([most, 0]), p.pool.share_counts()
    ring, cursor = i32([0, 1, 2, 4, 6, 7, -1, -1]), i32([0, 6])
    call = lambda *parent: Q.paged_fork(p.ctx, fork, lens, i32(parent), table, shared, ring, cursor)  # noqa: E731
    call(0, 0)
    assert fork.status.tolist() == [0, 0] and lens.tolist() == [most, most]
    assert table[:, 0].tolist() == [3, 3] and table[:, width - 1].tolist() == [5, 0]
    assert int((table != -1).sum()) == 4
    assert shared.tolist() == [0, 0, 0, 1, 0, 0, 0, 0] and cursor.tolist() == [1, 5]
    assert torch.equal(pool[:, 0, :, :, :255], pool[:, 5, :, :, :255])
    call(0, -1)
    assert lens.tolist() == [most, 0] and shared.tolist() == [0] * 8
    assert cursor.tolist() == [1, 6] and ring[6].item() == 0
    call(-1, -1)
    assert lens.tolist() == [0, 0] and cursor.tolist() == [1, 8]
    assert ring.tolist() == [5, 1, 2, 4, 6, 7, 0, 3]
    torch.cuda.synchronize()
    fork.close()
    p.close()


def test_pages_that_come_back_too_often_do_not_overfill_the_ring(gpu):
    """Counts below the truth: each of many holders gives the same pages back."""
    n, width, pages = 64, 300, 40
    p = Paged(pages, 16, n, n, nkvh=1, rope=False)
    fork = Q.PagedFork(p.ctx, p.pool, n, width)
    table = torch.arange(width, device="cuda").remainder(pages).int().repeat(n, 1)
    around = torch.full((3 * pages,), 77, dtype=torch.int32, device="cuda")
    ring = around[pages:2 * pages]
    for free in (0, 7, pages):
        around.fill_(77)
        lens, cursor = i32([16 * width] * n), i32([5, free])
        Q.paged_fork(p.ctx, fork, lens, i32([-1] * n), table.clone(), p.pool.share_counts(), ring, cursor)
        assert fork.status.tolist() == [0] * n and not bool(lens.any())
        assert cursor.tolist() == [5, pages]
        assert bool((around[:pages] == 77).all()) and bool((around[2 * pages:] == 77).all())
        got = ring.roll(-5).tolist()
        assert got[:free] == [77] * free and all(0 <= x < pages for x in got[free:])
    fork.close()
    p.close()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("ps", [16, 32])
def test_each_beam_keeps_its_history(gpu, ps, f8):
    """Steps of selection, fork, plan, stage (a) and attention, beside a pool in
    which every beam has pages of its own, copied whole from its parent's by
    torch: the same lengths, the same K and V at every position, the same bits of
    outputs.  And V is the raw V that was appended for it."""
    width, groups, vocab, layers, cols, steps = 3, 2, 500, 2, 6, 24
    n = width * groups
    make = Paged8 if f8 else Paged
    p, own = make(60, ps, n, 100, layers=layers), make(n * cols, ps, n, 100, layers=layers)
    sel, fork = Q.BeamSelect(p.ctx, groups, width, vocab), Q.PagedFork(p.ctx, p.pool, n, cols)
    ring, cur = p.pool.free_ring()
    shared, table = p.pool.share_counts(), torch.full((n, cols), -1, dtype=torch.int32, device="cuda")
    own_table = torch.arange(n * cols, dtype=torch.int32, device="cuda").view(n, cols)
    plan = p.plan
    plan.cursor.copy_(cur)
    plan.lens.zero_()
    gains = randn(4, layers, 2, HD, std=0.1) + 1
    scores = torch.full((n,), -float("inf"), device="cuda")
    scores[::width] = 0.0
    done, parent, token = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    values = [torch.zeros((layers, 0, NKVH, HD), dtype=torch.float16, device="cuda")] * n  # raw V

    def held(pool, ids, c):
        """[layers][2][kvh][c][hd] of a request's pages."""
        x = pool[:, ids[:-(-c // ps)].long()]
        return x.permute(0, 2, 3, 1, 4, 5).flatten(3, 4)[:, :, :, :c]

    def step(rows, seed):
        total = sum(rows)
        qkv = randn(seed, layers, total, TOT) * 2.0 ** (seed % 5 - 2)
        before = [v.shape[1] for v in values]
        Q.paged_plan(p.ctx, plan, plan.lens, i32(rows), table, ring, plan.cursor)
        Q.paged_plan(own.ctx, own.plan, i32(before), i32(rows), own_table)
        assert plan.status.tolist() == own.plan.status.tolist() == [0] * n
        outs = []
        for x, t in ((p, table), (own, own_table)):
            q, out = (torch.zeros((layers, total, QDIM), dtype=torch.float16, device="cuda") for _ in range(2))
            for l in range(layers):
                Q.paged_append(x.ctx, x.plan, l, qkv[l], gains[l, 0], gains[l, 1], q[l])
                Q.paged_attn(x.ctx, x.plan, l, t, q[l], out[l])
            outs.append((q, out))
        assert torch.equal(outs[0][0], outs[1][0]) and same_bits(outs[0][1], outs[1][1])
        at = 0
        for i, r in enumerate(rows):
            v = qkv[:, at:at + r, -NKVH * HD:].view(layers, r, NKVH, HD)
            values[i] = torch.cat([values[i], v], 1)
            at += r

    def compare():
        assert plan.lens[:n].tolist() == [v.shape[1] for v in values]
        for i, v in enumerate(values):
            c = v.shape[1]
            got = held(bits(p.pool.tensor()), table[i], c)
            assert torch.equal(got, held(bits(own.pool.tensor()), own_table[i], c))
            if f8:
                unit = p.pool.scales().float().repeat_interleave(16, -1)[..., None]
                unit = held(unit, table[i], c)[:, 1].transpose(1, 2)
                x = held(p.pool.tensor().float(), table[i], c)[:, 1].transpose(1, 2) * unit
                # Half a step of the value (e4m3: 2^-4 of it, or 2^-10 units); a
                # unit that grew rounded once more, values below 2^-6 units.
                bound = v.float().abs() * 2.0 ** -4 + unit * 2.0 ** -9
                assert bool(((x - v.float()).abs() <= bound).all())
            else:
                assert torch.equal(held(p.pool.tensor(), table[i], c)[:, 1].transpose(1, 2), v)

    step([30, 0, 0, 21, 0, 0], 100)
    shuffled = 0
    for k in range(steps):
        say(f"beams ps={ps} f8={f8} step {k}")
        g = torch.Generator(device="cuda")
        g.manual_seed(k)
        logits = torch.randn((n, vocab), device="cuda", generator=g) * 3
        Q.beam_select(p.ctx, sel, logits, scores, parent, token, scores, done, 7, done)
        Q.paged_fork(p.ctx, fork, plan.lens, parent, table, shared, ring, plan.cursor)
        assert fork.status.tolist() == [0] * n
        par = parent.tolist()
        shuffled += par != list(range(n))
        pool = bits(own.pool.tensor())
        pool.copy_(pool.view(layers, n, cols, *pool.shape[2:])[:, par].reshape(pool.shape))
        if f8:
            units = bits(own.pool.scales())
            units.copy_(units.view(layers, n, cols, *units.shape[2:])[:, par].reshape(units.shape))
        values[:] = [values[j] for j in par]
        compare()
        rows = [1 - d for d in done.tolist()]
        if not any(rows):
            break
        step(rows, 200 + k)
        compare()
    assert shuffled > steps // 2
    Q.paged_fork(p.ctx, fork, plan.lens, i32([-1] * n), table, shared, ring, plan.cursor)
    assert int(plan.cursor[1]) == 60 and not bool(shared.any())
    fork.close()
    sel.close()
    own.close()
    p.close()


def test_two_at_once_and_two_graphs_of_one_workspace(gpu):
    """Forks on two streams, each with its own workspace and pool; then two graphs
    of one workspace, of different requests, replayed in turn."""
    def model(s, parent):
        return B.fork(s.lens, parent, s.table, s.shared, s.ring, s.cursor, s.pages, s.ps)[1]

    def same(s, d):
        for got, want in zip(d, (s.lens, s.table, s.shared, s.ring, s.cursor)):
            assert got.tolist() == want

    states = [State(12, 300, 16, 20, True, 3, 2, seed=1), State(5, 90, 64, 9, False, 2, 8, seed=2)]
    streams, held, pages = (torch.cuda.Stream(), torch.cuda.Stream()), [], []
    for s in states:
        for i in range(s.n):
            s.grow(i, 37 + 11 * i)
        held.append([i32(x) for x in (s.lens, s.table, s.shared, s.ring, s.cursor)])
        pages.append(bits(s.p.pool.tensor()).clone())
    parents = [[[(7 * k + 3 * i) % s.n for i in range(s.n)] for k in range(4)] for s in states]
    dev = [[i32(p) for p in x] for x in parents]
    torch.cuda.synchronize()
    for k in range(4):
        for s, d, p, stream in zip(states, held, dev, streams):
            Q.paged_fork(s.p.ctx, s.fork, d[0], p[k], *d[1:], stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for s, d, p, want in zip(states, held, parents, pages):
        for x in p:
            for a, b, r in model(s, x):
                want[:, b, :, :, :r] = want[:, a, :, :, :r]
        same(s, d)
        assert torch.equal(bits(s.p.pool.tensor()), want)

    # Requests 0 .. 4 and all 12 of one pool: rows of one table.
    s, d = states[0], held[0]
    parent = [i32([0] * 5), i32(list(range(12)))]
    graphs = []
    for p in parent:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            Q.paged_fork(s.p.ctx, s.fork, d[0], p, *d[1:])
        graphs.append(g)
    for k in range(6):
        g, p = graphs[k % 2], parent[k % 2]
        n = p.numel()
        x = [(5 * k + i * (k + 1)) % n for i in range(n)]
        p.copy_(i32(x))
        g.replay()
        torch.cuda.synchronize()
        assert s.fork.status[:n].tolist() == [0] * n
        # (The requests that are not in the call hold what they held.)
        lens, table = s.lens[:n], s.table[:n]
        B.fork(lens, x, table, s.shared, s.ring, s.cursor, s.pages, s.ps)
        s.lens[:n], s.table[:n] = lens, table
        same(s, d)
        for i in range(s.n):
            s.grow(i, k)
        for t, v in zip(d, (s.lens, s.table, s.shared, s.ring, s.cursor)):
            t.copy_(i32(v))
    del g, graphs
    for s in states:
        s.close()
