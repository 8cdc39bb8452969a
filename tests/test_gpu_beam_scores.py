"""Scores of the beam selection against a bound derived from its arithmetic,
and the order of candidates whose scores are equal or next to it."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from gpu_helpers import say  # noqa: E402
from test_gpu_beam import Sel, gen, peaked  # noqa: E402

pytestmark = pytest.mark.gpu


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
