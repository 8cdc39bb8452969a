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
