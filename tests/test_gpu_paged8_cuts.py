"""Steps over e4m3 pages of fewer rows than their plan has: row blocks, key
ranges and blocks of a unit cut short by the caller's rows."""
from __future__ import annotations

import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import qasr_attn as Q  # noqa: E402
from gpu_helpers import say  # noqa: E402
from test_gpu_paged import Paged, i32, randn, run_attn, shuffled_table  # noqa: E402
from test_gpu_paged8 import Paged8, bits, both, check_codes, fill, new_rows, same_bits, step_codes, values  # noqa: E402
from workloads import HD, QDIM  # noqa: E402

pytestmark = pytest.mark.gpu


def cut_batch(batch, cut):
    out = []
    for c, r in batch:
        out.append((c, min(r, cut)))
        cut -= out[-1][1]
    return out


@pytest.mark.parametrize("batch,cuts", [
    ([(10, 3), (700, 14), (120, 12), (40, 300)], (1, 2, 5, 17, 20, 29, 30, 328)),
    ([(4000, 600), (1500, 2)], (1, 63, 65, 130, 599, 601)),
    ([(2040, 12), (1020, 9), (505, 8), (250, 8)], (4, 11, 15, 24, 30))])
def test_attention_of_fewer_rows(gpu, batch, cuts):
    """Also where a whole range lies behind the last key that is left."""
    ps = 16
    a, b, table, rows = both(batch, ps)
    fill(a.pool, 5)
    b.pool.tensor().copy_(values(a.pool))
    q, table = randn(6, rows, QDIM), i32(table)
    whole = run_attn(a, batch, table, q).clone()
    assert same_bits(whole, run_attn(b, batch, table, q))
    for cut in cuts:
        say(f"attn8 {cut} of {rows} rows")
        outs = []
        for p in (a, b):
            out = torch.full_like(q, 7.0)
            Q.paged_attn(p.ctx, p.plan, 0, table, q[:cut], out)
            outs.append(out)
        assert same_bits(*outs) and bool((outs[0][cut:] == 7).all())
        Q.paged_attn(a.ctx, a.plan, 0, table, q, outs[0])
        assert torch.equal(outs[0], whole)
    a.close()
    b.close()


@pytest.mark.parametrize("ps", [16, 64])
def test_stage_a_of_fewer_rows(gpu, ps):
    """A step's first rows, then all of them, into blocks that hold some already."""
    batch, nkvh = [(5, 30), (16, 1), (31, 40), (0, 20), (9, 1)], 2
    need = [-(-(c + r) // ps) for c, r in batch]
    pages, rows = sum(need) + 1, sum(r for _, r in batch)
    table, _ = shuffled_table(random.Random(1), need, pages, max(need))
    a, b = (P(pages, ps, len(batch), rows, nkvh=nkvh) for P in (Paged8, Paged))
    fill(a.pool, 3)
    codes = bits(a.pool.tensor()).cpu().numpy().astype(np.int64)
    units = bits(a.pool.scales()).cpu().numpy().astype(np.int64) - 127
    qkv, gains = new_rows(1, rows, nkvh, True), randn(4, 2, HD) + 1
    for p in (a, b):
        Q.paged_plan(p.ctx, p.plan, i32([c for c, _ in batch]), i32([r for _, r in batch]), i32(table))
    for cut in (1, 12, 30, 33, 75, rows):
        say(f"append8 {cut} of {rows} rows")
        outs = []
        for p in (a, b):
            q = torch.full((rows, 2 * nkvh * HD), 7.0, dtype=torch.float16, device="cuda")
            Q.paged_append(p.ctx, p.plan, 0, qkv[:cut], gains[0], gains[1], q)
            outs.append(q)
        assert torch.equal(*outs) and bool((outs[0][cut:] == 7).all())
        step_codes(codes, units, b, cut_batch(batch, cut), table, ps)
        check_codes(a, codes, units)
    a.close()
    b.close()
