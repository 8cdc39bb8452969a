"""Forks of paged requests on the GPU against a plain implementation in whole
numbers, page contents included, and a beam search on pages as a server runs
it."""
from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

import beam_model as B  # noqa: E402
import qasr_attn as Q  # noqa: E402
from gpu_helpers import say  # noqa: E402
from test_gpu_paged import Paged, check_attn, i32, randn  # noqa: E402
from test_gpu_paged8 import Paged8, Values, bits, fill  # noqa: E402
from workloads import HD, QDIM, TOT  # noqa: E402

pytestmark = pytest.mark.gpu


class State:
    """What a server holds, on the GPU and as lists, and the fork of both."""

    def __init__(self, n, pages, ps, width, f8=False, layers=1, nkvh=2, seed=1):
        P = Paged8 if f8 else Paged
        self.p = P(pages, ps, n, 4 * n, nkvh=nkvh, layers=layers, rope=False)
        self.f8, self.n, self.pages, self.ps, self.width = f8, n, pages, ps, width
        pool = self.p.pool
        if f8:
            fill(pool, seed)
        else:
            pool.tensor().copy_(randn(seed, *pool.tensor().shape))
        self.fork = Q.PagedFork(self.p.ctx, pool, n, width)
        self.lens, self.table = [0] * n, [[-1] * width for _ in range(n)]
        self.shared, self.ring, self.cursor = [0] * pages, list(range(pages)), [0, pages]

    def close(self):
        torch.cuda.synchronize()
        self.fork.close()
        self.p.close()

    def new_pages(self, k):
        head, free = self.cursor
        assert k <= free
        self.cursor = [(head + k) % self.pages, free - k]
        return [self.ring[(head + j) % self.pages] for j in range(k)]

    def grow(self, i, rows):
        have, full = -(-self.lens[i] // self.ps), -(-(self.lens[i] + rows) // self.ps)
        self.table[i][have:full] = self.new_pages(full - have)
        self.lens[i] += rows

    def shuffle(self, rnd):
        """The free ids in another order, from another place of the ring on."""
        head, free = self.cursor
        ids = [self.ring[(head + j) % self.pages] for j in range(free)]
        rnd.shuffle(ids)
        head = rnd.randrange(self.pages)
        self.ring = [rnd.choice([-1, 0, self.pages + 3]) for _ in range(self.pages)]
        for j, p in enumerate(ids):
            self.ring[(head + j) % self.pages] = p
        self.cursor = [head, free]

    def step(self, parent, stream=None):
        """Both forks; everything compared."""
        n, pool = len(parent), self.p.pool
        d = [i32(x) for x in (self.lens, parent, self.table, self.shared, self.ring, self.cursor)]
        before = bits(pool.tensor()).clone(), bits(pool.scales()).clone() if self.f8 else None
        Q.paged_fork(self.p.ctx, self.fork, *d, stream=stream)
        torch.cuda.synchronize()
        status, copies = B.fork(self.lens, parent, self.table, self.shared, self.ring, self.cursor, self.pages, self.ps)
        assert self.fork.status[:n].tolist() == status
        for name, got, want in zip(("lens", "parent", "table", "shared", "ring", "cursor"), d,
                                   (self.lens, parent, self.table, self.shared, self.ring, self.cursor)):
            assert got.tolist() == want, name
        want, scales = before
        for a, b, r in copies:
            want[:, b, :, :, :r] = want[:, a, :, :, :r]
            if self.f8:
                k = -(-r // 16)
                scales[:, b, :, :, :k] = scales[:, a, :, :, :k]
        assert torch.equal(bits(pool.tensor()), want)
        if self.f8:
            assert torch.equal(bits(pool.scales()), scales)
        return status, copies


@pytest.mark.parametrize("n,ps,width,f8,nkvh,layers", [
    (1, 16, 3, False, 1, 1), (5, 16, 40, False, 8, 3), (5, 16, 40, True, 8, 3), (12, 32, 17, True, 2, 2),
    (12, 64, 16, False, 3, 1), (40, 256, 5, True, 2, 2), (70, 128, 33, False, 1, 1), (300, 16, 20, True, 1, 1),
    (1024, 16, 18, False, 1, 1)])
def test_fork_against_plain(gpu, n, ps, width, f8, nkvh, layers):
    """A sequence of forks, growing and ending requests."""
    rnd = random.Random(n * ps)
    pages = n * width + 5 if n < 100 else n * 8
    s = State(n, pages, ps, width, f8, layers, nkvh)
    for turn in range(6):
        s.shuffle(rnd)
        for i in range(n):
            room = min(width * ps - s.lens[i], 6 * ps)
            want = rnd.choice([0, 1, rnd.randint(0, 2 * ps), ps - s.lens[i] % ps]) if turn else rnd.randint(0, 3 * ps)
            want = min(want, room)
            if -(-(s.lens[i] + want) // ps) - -(-s.lens[i] // ps) < s.cursor[1] // (n - i + 1):
                # A page that others hold is not written: forks leave none such.
                s.grow(i, want)
        kind = rnd.choice(["beams", "any", "one", "keep", "end some"])
        parent = list(range(n))
        if kind == "beams":
            parent = [i // 4 * 4 + rnd.randrange(min(4, n - i // 4 * 4)) for i in range(n)]
        elif kind == "any":
            parent = [rnd.randrange(n) for _ in range(n)]
        elif kind == "one":
            parent = [rnd.randrange(n)] * n
        elif kind == "end some":
            parent = [rnd.choice([-1, i, rnd.randrange(n)]) for i in range(n)]
        say(f"fork n={n} ps={ps} f8={f8} turn {turn} {kind}")
        s.step(parent)
    s.step([-1] * n)
    assert s.cursor[1] == pages and not any(s.shared)
    s.close()


def test_nothing_or_all(gpu):
    """Parents and lengths out of range, too few free pages: nothing changes."""
    s = State(4, 20, 16, 4)
    for i, c in enumerate((20, 33, 16, 0)):
        s.grow(i, c)
    for parent in ([0, 4, 2, 3], [0, 1, -2, 3], [1 << 30, 1, 2, -(1 << 30)]):
        status, _ = s.step(parent)
        assert B.EINVAL in status
    for bad in (-1, 65, (1 << 31) - 1):
        lens = list(s.lens)
        s.lens[3] = bad
        status, _ = s.step([0, 0, 0, 0])
        assert status == [0, 0, 0, B.EINVAL]
        s.lens = lens
    s.new_pages(s.cursor[1] - 2)
    status, _ = s.step([1, 1, 1, 1])
    assert status == [B.ENOMEM, 0, B.ENOMEM, B.ENOMEM]
    status, copies = s.step([1, 1, 1, -1])
    assert not any(status) and len(copies) == 2
    for cursor in ([-1, 3], [20, 3], [0, -1], [0, 21]):  # no free page
        s.cursor = cursor
        d = [i32(x) for x in (s.lens, [0, 0, 0, -1], s.table, s.shared, s.ring, s.cursor)]
        Q.paged_fork(s.p.ctx, s.fork, *d)
        assert s.fork.status.tolist() == [0, B.ENOMEM, B.ENOMEM, 0]
        assert d[5].tolist() == cursor and d[2].tolist() == s.table
    s.close()


def test_pages_outside_the_pool(gpu):
    """Evicted entries, an evicted unfinished page, an id of the ring that is no
    page, a page that another request outside the call holds."""
    s = State(6, 40, 16, 6, f8=True)
    for i, c in enumerate((70, 40, 20, 55, 0, 33)):
        s.grow(i, c)
    s.table[0][1] = -1
    s.table[1][2] = 99        # unfinished, of request 1
    s.shared[s.table[3][3]] = 1  # held elsewhere too
    head = s.cursor[0]
    s.ring[(head + 1) % 40] = 1 << 20
    status, copies = s.step([0, 0, 1, 1, 3, 2])
    assert not any(status) and len(copies) == 1 and s.table[4][3] == 1 << 20
    s.close()


def test_release_of_many_pages(gpu):
    """Tables of thousands of columns, wide enough for several turns of the
    ring's part, most of them free."""
    s = State(3, 9000, 16, 6000, nkvh=1)
    s.grow(0, 16 * 5000 + 3)
    s.step([0, 0, 0])
    s.grow(1, 700)
    s.step([1, 1, -1])
    s.step([-1, -1, -1])
    assert s.cursor[1] == 9000
    s.close()


def test_on_another_stream_and_replayed(gpu):
    s = State(6, 200, 16, 30)
    for i in range(6):
        s.grow(i, 37 + i)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    s.step([1, 1, 2, 2, 2, 5], stream=stream.cuda_stream)
    torch.cuda.synchronize()
    parent = i32([0, 0, 3, 3, 2, 1])
    d = [i32(x) for x in (s.lens, s.table, s.shared, s.ring, s.cursor)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Q.paged_fork(s.p.ctx, s.fork, d[0], parent, *d[1:])
    for turn in range(4):
        parents = parent.tolist()
        graph.replay()
        torch.cuda.synchronize()
        B.fork(s.lens, parents, s.table, s.shared, s.ring, s.cursor, s.pages, s.ps)
        for got, want in zip(d, (s.lens, s.table, s.shared, s.ring, s.cursor)):
            assert got.tolist() == want
        parent.copy_(i32([(turn * 3 + i) % 6 for i in range(6)]))
    del graph
    s.close()


def test_the_largest_fork(gpu):
    """1024 requests with tables of 700 pages: a prefix that all share, pages of
    their own, most of them given up at once; then all."""
    rnd = random.Random(5)
    n, ps, width, pages = 1024, 16, 700, 40000
    s = State(n, pages, ps, width, True, 1, 1)
    s.grow(0, 16 * 600 + 5)
    s.step([0] * n)
    s.shuffle(rnd)
    for i in range(n):
        s.grow(i, rnd.randint(0, 300))
    s.step([rnd.randrange(40) for _ in range(n)])
    assert s.cursor[1] > 20000
    s.step([-1] * n)
    assert s.cursor[1] == pages and not any(s.shared)
    s.close()


def test_copies_past_32_bits(gpu):
    """Pages whose offsets pass 2^32 bytes."""
    rnd = random.Random(11)
    s = State(4, 9000, 256, 4, True, 1, 8)
    for _ in range(3):
        s.shuffle(rnd)
        s.cursor[1] = 9000 - sum(-(-c // 256) for c in s.lens)
        far = sorted((s.ring[(s.cursor[0] + j) % 9000] for j in range(s.cursor[1])), reverse=True)
        for j, page in enumerate(far):
            s.ring[(s.cursor[0] + j) % 9000] = page
        for i in range(4):
            s.grow(i, rnd.randint(1, 200))
        status, copies = s.step([1, 1, 2, 2])
        assert not any(status) and copies and min(to for _, to, _ in copies) * 2 * 8 * 256 * HD > 1 << 32
        s.step([0, -1, 2, -1])
    s.close()


def test_replayed_with_copies(gpu):
    """A graph whose every replay shares, copies and gives back, of 8-bit pages,
    with eager work between the replays."""
    rnd = random.Random(9)
    s = State(6, 200, 32, 12, True, 2, 2)
    for i in range(6):
        s.grow(i, 40 + 11 * i)
    d = [i32(x) for x in (s.lens, s.table, s.shared, s.ring, s.cursor)]
    parent = i32(list(range(6)))
    pool = s.p.pool
    Q.paged_fork(s.p.ctx, s.fork, d[0], parent, *d[1:])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Q.paged_fork(s.p.ctx, s.fork, d[0], parent, *d[1:])
    for _ in range(5):
        parents = [rnd.randrange(6) for _ in range(6)]
        parent.copy_(i32(parents))
        want, units = bits(pool.tensor()).clone(), bits(pool.scales()).clone()
        graph.replay()
        torch.cuda.synchronize()
        _, copies = B.fork(s.lens, parents, s.table, s.shared, s.ring, s.cursor, s.pages, s.ps)
        for a, b, r in copies:
            want[:, b, :, :, :r] = want[:, a, :, :, :r]
            units[:, b, :, :, :-(-r // 16)] = units[:, a, :, :, :-(-r // 16)]
        for got, w in zip(d, (s.lens, s.table, s.shared, s.ring, s.cursor)):
            assert got.tolist() == w
        assert torch.equal(bits(pool.tensor()), want) and torch.equal(bits(pool.scales()), units)
        for i in range(6):  # the requests go on, each by its own rows
            s.grow(i, rnd.randint(0, 9))
        for t, v in zip(d, (s.lens, s.table, s.shared, s.ring, s.cursor)):
            t.copy_(i32(v))
    del graph
    s.close()


def test_fork_refuses(gpu):
    p = Paged(20, 16, 4, 8, rope=False)
    for bad in ((0, 4), (1025, 4), (4, 0), (4, (1 << 24) + 1)):
        with pytest.raises(Q.QasrError) as e:
            Q.PagedFork(p.ctx, p.pool, *bad)
        assert e.value.code == Q.QASR_EINVAL
    f = Q.PagedFork(p.ctx, p.pool, 4, 6)
    z = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(lens=z(4), parent=z(4), table=z(4, 6), shared=z(20), ring=z(20), cursor=z(2))

    def refused(code=Q.QASR_EINVAL, **k):
        with pytest.raises(Q.QasrError) as e:
            Q.paged_fork(p.ctx, f, *{**good, **k}.values())
        assert e.value.code == code

    refused(Q.QASR_ERANGE, lens=z(5), parent=z(5), table=z(5, 6))
    refused(Q.QASR_ERANGE, table=z(4, 7))
    same = z(40)
    refused(shared=same[:20], ring=same[10:30])
    refused(lens=same[:4], parent=same[3:7])
    refused(lens=f.status)
    refused(parent=good["lens"])
    for bad in (dict(lens=z(4).float()), dict(ring=z(20).cpu()), dict(table=z(6, 4).t())):
        with pytest.raises(ValueError):
            Q.paged_fork(p.ctx, f, *{**good, **bad}.values())
    other = Paged(20, 16, 4, 8, rope=False)
    with pytest.raises(Q.QasrError):
        Q.paged_fork(other.ctx, f, *good.values())
    other.close()
    Q.paged_fork(p.ctx, f, *good.values())
    torch.cuda.synchronize()
    status = f.status  # keeps the memory, not the handle
    p.pool.close()
    with pytest.raises(Q.QasrError):
        Q.paged_fork(p.ctx, f, *good.values())
    assert status.tolist() == [0, Q.QASR_ENOMEM, Q.QASR_ENOMEM, Q.QASR_ENOMEM] or status.tolist() == [0] * 4
    f.close()
    p.close()


@pytest.mark.parametrize("f8", [False, True])
def test_a_beam_search_on_pages(gpu, f8):
    """Two prompts of 3 beams each: prefill into one beam, fork, then steps of
    selection, fork, plan, append and attention.  Each beam's outputs are the
    definition's over its own history, which a second pool, without sharing,
    holds; and all pages come back."""
    width, groups, ps, vocab, pages = 3, 2, 16, 500, 80
    n = width * groups
    P = Paged8 if f8 else Paged
    p = P(pages, ps, n, 100, layers=2)
    sel = Q.BeamSelect(p.ctx, groups, width, vocab)
    fork = Q.PagedFork(p.ctx, p.pool, n, 12)
    ring, cur = p.pool.free_ring()
    shared, table = p.pool.share_counts(), torch.full((n, 12), -1, dtype=torch.int32, device="cuda")
    plan = p.plan
    plan.cursor.copy_(cur)
    plan.lens.zero_()
    gains = randn(4, 2, 2, HD, std=0.1) + 1
    scores = torch.full((n,), -float("inf"), device="cuda")
    scores[::width] = 0.0
    done, parent, token = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    history = [[] for _ in range(n)]  # (seed, row) of the raw rows that a beam's cache is made of

    def run(rows, seed):
        total = sum(rows)
        qkv = randn(seed, 2, total, TOT)
        Q.paged_plan(p.ctx, plan, plan.lens, i32(rows), table, ring, plan.cursor)
        assert plan.status.tolist() == [0] * n
        q, out = (torch.zeros((2, total, QDIM), dtype=torch.float16, device="cuda") for _ in range(2))
        for l in range(2):
            Q.paged_append(p.ctx, plan, l, qkv[l], gains[l, 0], gains[l, 1], q[l])
            Q.paged_attn(p.ctx, plan, l, table, q[l], out[l])
        r = 0
        for i in range(n):
            history[i] = history[i] + [(seed, r + k) for k in range(rows[i])]
            r += rows[i]
        return q, out

    def lens():
        return [len(h) for h in history]

    run([30, 0, 0, 21, 0, 0], 100)
    for step in range(14):
        g = torch.Generator(device="cuda")
        g.manual_seed(step)
        logits = torch.randn((n, vocab), device="cuda", generator=g) * 3
        Q.beam_select(p.ctx, sel, logits, scores, parent, token, scores, done, 7, done)
        Q.paged_fork(p.ctx, fork, plan.lens, parent, table, shared, ring, plan.cursor)
        assert fork.status.tolist() == [0] * n
        history[:] = [list(history[i]) if i >= 0 else [] for i in parent.tolist()]
        assert plan.lens[:n].tolist() == lens()
        rows = [0 if d or i < 0 else 1 for d, i in zip(done.tolist(), parent.tolist())]
        q, out = run(rows, 200 + step)
        batch = [(c - r, r) for c, r in zip(lens(), rows)]
        view = Values(p) if f8 else p
        check_attn(view, batch, table.cpu(), q[1], out[1], layer=1, heads=(0, 9))
    # What the pages hold is each beam's own history: the first rows' V.
    raw = {}
    pool = (Values(p) if f8 else p.pool).tensor()
    for i in range(n):
        for pos, (seed, row) in enumerate(history[i]):
            if seed not in raw:
                raw[seed] = randn(seed, 2, {100: 51}.get(seed, n), TOT) if seed == 100 else None
            if raw[seed] is None:
                continue
            v = raw[seed][1, row, -8 * HD:].view(8, HD)
            got = pool[1, table[i, pos // ps].item(), 1, :, pos % ps]
            if f8:
                assert float((got.float() - v.float()).norm() / v.float().norm()) < 0.05
            else:
                assert torch.equal(got, v)
    Q.paged_fork(p.ctx, fork, plan.lens, i32([-1] * n), table, shared, ring, plan.cursor)
    assert int(plan.cursor[1]) == pages and not bool(shared.any())
    fork.close()
    sel.close()
    p.close()
