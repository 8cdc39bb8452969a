"""Scores of the beam selection against a bound derived from its arithmetic,
and the order of candidates whose scores are equal or next to it."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from gpu_helpers import say  # noqa: E402
from test_gpu_beam import Sel, gen, peaked  # noqa: E402

pytestmark = pytest.mark.gpu


def bounds(x):
    """How far log sum exp of each row [rows][vocab] may be off.

    A term is e^(v - M) in its tile of 2048, M the tile's largest, and the tile
    weighs e^(M - top).  Both exponents are f32 differences times f32 log2(e):
    three roundings of 2^-24 (the constant's among them) of v - M and of M - top,
    together of top - v; for every 128 tiles more the sum so far moves to a new largest
    by another, and all of them add up to top - v all the same.  Each exponential is
    off by 2^-23 (the instruction's 1 ulp), five of them at 2^20 tokens.  f32 additions: 8 terms of
    each of 4 sums, 2 to join them, 6 across the lanes, 2^-24 each; the tile's
    product with its weight one more.  All relative to the term, so the logarithm is
    off by their mean over the terms' weights; f64 adds nothing that counts (2^-40)."""
    x = x.double()
    top = x.amax(-1, keepdim=True)
    p = torch.softmax(x, -1)
    mean = (p * torch.where(p > 0, top - x, torch.zeros_like(x))).sum(-1)
    return 3 * 2.0 ** -24 * mean + 5 * 2.0 ** -23 + (8 + 2 + 6 + 1) * 2.0 ** -24 + 2.0 ** -40


@pytest.mark.parametrize("groups,width,vocab,std", [
    (1, 5, 151936, 2.0), (4, 3, 500, 2.0), (2, 2, 2048, 8.0), (3, 4, 30001, 0.01), (2, 2, 151936, 20.0),
    (1, 2, 300000, 3.0), (1, 1, 1 << 20, 1.0)])
def test_scores_within_the_arithmetic(gpu, groups, width, vocab, std):
    k = 8
    s = Sel(groups, width, vocab, k)
    logits = peaked(1, groups * width, vocab, std)
    scores = -10 * torch.rand(groups * width, device="cuda", generator=gen(2))
    parent, token, got, _ = s.run(logits, scores)
    bound = bounds(logits).cpu()
    p = (torch.log_softmax(logits.double(), -1) + scores.double()[:, None]).cpu()
    row = parent.long()
    want = p[row, token.long()]
    off = (got.double() - want).abs()
    say(f"beam scores {groups}x{width} of {vocab}: off by {float(off.max()):.2g}, bound {float(bound.max()):.2g}")
    assert bool((off <= bound[row] + 2.0 ** -24 * want.abs()).all())
    # Whatever is better than a place by more than both bounds comes before it.
    for g in range(groups):
        at = slice(g * k, g * k + k)
        best = p[g * width:(g + 1) * width].flatten().topk(k)[0]
        slack = 2 * float(bound[g * width:(g + 1) * width].max())
        assert bool(((want[at] - best).abs() <= slack).all())
        assert len({(int(r), int(t)) for r, t in zip(parent[at], token[at])}) == k
    s.close()


def test_order_of_scores_next_to_each_other(gpu):
    """Within a beam the larger logit comes first also where the scores are equal
    in 64 bits, equal logits by token; between beams equal scores go to the lower
    beam, whose logits may be the smaller ones."""
    s = Sel(1, 2, 4, 8)
    run = lambda x, sc: [t.tolist() for t in s.run(torch.tensor(x, device="cuda"), torch.tensor(sc, device="cuda"))[:2]]  # noqa: E731
    tiny = [0.0, 1e-20, 2e-20, -0.0]
    top = max(tiny)
    lse = top + np.log(np.exp(np.array(tiny) - top).sum())
    assert len({-1.0 + (t - lse) for t in tiny}) == 1, "equal scores"
    assert run([tiny, tiny], [-1.0, -1.0]) == [[0] * 4 + [1] * 4, [2, 1, 0, 3] * 2]
    # Beam scores whose steps are larger than the logits' differences.
    near = [1.0, 1.0 + 2 ** -20, 1.0, 1.0 + 2 ** -19]
    assert run([near, near[::-1]], [-1e13, -1e13]) == [[0] * 4 + [1] * 4, [3, 1, 0, 2, 0, 2, 1, 3]]
    assert run([near, near], [-1e13, -1e12]) == [[1] * 4 + [0] * 4, [3, 1, 0, 2] * 2]
    s.close()
