"""Paged steps at their edges: pages that the pool does not have."""
from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

import qasr_attn as Q  # noqa: E402
from gpu_helpers import Gpu  # noqa: E402
from test_gpu_paged import Paged, check_attn, i32, randn  # noqa: E402
from workloads import HD, QDIM, TOT  # noqa: E402

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
