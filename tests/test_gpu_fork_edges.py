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
