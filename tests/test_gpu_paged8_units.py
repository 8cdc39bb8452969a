"""Units that a caller has stored: every power of two that a scale byte can be,
also those that stage (a) does not choose."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_paged import i32, randn, run_attn  # noqa: E402
from test_gpu_paged8 import Paged8, bits, both, fill, same_bits, values  # noqa: E402
from workloads import HD, QDIM  # noqa: E402

pytestmark = pytest.mark.gpu


def test_every_unit(gpu):
    """Requests of one key each, whose output is its value: code times unit, rounded
    to f16 once, infinities among them."""
    n = 255
    p = Paged8(n, 16, n, n, nkvh=1, rope=False)
    t, u = bits(p.pool.tensor()), bits(p.pool.scales())
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    codes = torch.randint(0, 256, t.shape, device="cuda", generator=g, dtype=torch.uint8)
    codes[(codes & 127) == 127] = 0x30
    codes[:, :, 0] = 0
    t.copy_(codes)
    u[0, :, 0] = 127
    u[0, :, 1] = torch.arange(n, device="cuda", dtype=torch.uint8)[:, None, None]
    out = run_attn(p, [(0, 1)] * n, i32([[i] for i in range(n)]), randn(2, n, 2 * HD))
    two = torch.ldexp(torch.ones(n, dtype=torch.float64, device="cuda"), torch.arange(n, device="cuda") - 127)
    want = (p.pool.tensor()[0, :, 1, 0, 0].double() * two[:, None]).half()
    assert bool(want.isinf().any()) and bool((want.abs() < 2.0 ** -14).any())
    for h in (0, 1):
        assert torch.equal(out[:, h * HD:(h + 1) * HD], want)
    p.close()


@pytest.mark.parametrize("lo,hi", [(-40, -14), (-30, 6)])
@pytest.mark.parametrize("batch", [[(40, 1), (600, 5)], [(300, 14)], [(4000, 530)]])
def test_small_units_beside_others(gpu, lo, hi, batch):
    a, b, table, rows = both(batch, 16)
    fill(a.pool, 5, lo, hi)
    b.pool.tensor().copy_(values(a.pool))
    q = randn(6, rows + 2, QDIM)
    assert same_bits(run_attn(a, batch, i32(table), q), run_attn(b, batch, i32(table), q))
    a.close()
    b.close()
