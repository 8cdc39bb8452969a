"""Attention over e4m3 pages in key ranges of more than 8 tiles, whose units
come in several loads of 64 groups: the bits of f16 pages that hold the same
values."""
from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

import qasr_attn as Q  # noqa: E402
from gpu_helpers import say  # noqa: E402
from test_gpu_paged import Paged, i32, randn, run_attn, shuffled_table  # noqa: E402
from test_gpu_paged8 import Paged8, Values, bits, fill, same_bits, values  # noqa: E402
from test_gpu_paged_work import check_rows  # noqa: E402
from workloads import QDIM  # noqa: E402

pytestmark = pytest.mark.gpu

TILE, LOAD = 128, 8  # keys of a tile, tiles of a load of units

# Of more than 8 and of more than 16 tiles a range: blocks of 16 rows, and of up
# to 8 in contexts past 32 ranges of 512 keys.
LONG = [[(1200, 300)], [(2500, 200), (17, 1)], [(4000, 256), (1100, 290)], [(40000, 1), (70000, 5)], [(100000, 1)],
        [(70000, 14)]]


def tiles_a_range(c, r):
    """Of a request's longest row block."""
    rows, _, splits = Q.plan_paged(c, r)
    assert rows == 16, "narrow"
    return -(-(-(-(c + r) // TILE)) // splits)


def both(batch, ps, nkvh=2, seed=1):
    need = [-(-(c + r) // ps) for c, r in batch]
    pages, rows = sum(need) + 2, sum(r for _, r in batch)
    table, _ = shuffled_table(random.Random(seed), need, pages, max(need) + 1)
    p = [P(pages, ps, len(batch), rows, nkvh=nkvh, max_seq=1 << 17, rope=False) for P in (Paged8, Paged)]
    fill(p[0].pool, 5, -12, -5)
    return p, table, rows


def compare(p, batch, table, q, note):
    p[1].pool.tensor().copy_(values(p[0].pool))
    say(f"attn8 ranges {note}")
    x, y = (run_attn(t, batch, i32(table), q) for t in p)
    assert same_bits(x, y)
    return x


@pytest.mark.parametrize("ps", [16, 64, 256])
@pytest.mark.parametrize("batch", LONG, ids=lambda b: "+".join(f"{r}@{c}" for c, r in b))
def test_units_of_long_ranges(gpu, ps, batch):
    assert max(tiles_a_range(c, r) for c, r in batch) > LOAD
    p, table, rows = both(batch, ps)
    q = randn(6, rows, 4 * 128)
    x = compare(p, batch, table, q, f"ps={ps} {batch}")
    check_rows(Values(p[0]), batch, table, q, x, heads=(0, 3))
    for t in p:
        t.close()


@pytest.mark.parametrize("batch", [LONG[0], LONG[4]], ids=lambda b: "+".join(f"{r}@{c}" for c, r in b))
def test_evicted_pages_and_nan_past_the_first_load(gpu, batch):
    """In the second load's tiles: a page outside the pool, then a NaN unit there,
    which nobody sees; then a NaN that all rows see."""
    ps = 16
    (c, r), = batch
    n = tiles_a_range(c, r)
    assert n > LOAD
    p, table, rows = both(batch, ps, seed=3)
    q = randn(6, rows, 4 * 128)
    at = (LOAD * TILE + 40) // ps  # in the first range
    page, table[0][at] = table[0][at], -1
    want = compare(p, batch, table, q, "evicted")
    assert bool(want.isfinite().all())
    check_rows(Values(p[0]), batch, table, q, want, heads=(0, 3))
    bits(p[0].pool.scales())[0, page] = 0xFF
    assert torch.equal(run_attn(p[0], batch, i32(table), q), want)
    bits(p[0].pool.scales())[0, page] = 120
    table[0][at] = page
    whole = compare(p, batch, table, q, "seen")
    assert not torch.equal(whole, want)
    bits(p[0].pool.tensor())[0, page, :, :, 3, 7] = 0x7F
    got = compare(p, batch, table, q, "nan")
    assert bool(got.isnan().any(1).all())
    for t in p:
        t.close()


def test_many_heads_of_a_long_range(gpu):
    batch = [(1200, 300), (40000, 3)]
    p, table, rows = both(batch, 32, nkvh=8)
    compare(p, batch, table, randn(6, rows, QDIM), "8 kv heads")
    for t in p:
        t.close()
