"""Rows before the head that fill their blocks, warps and strips badly, against 64 bits."""
import pytest
import torch

from mormot2_ai_b200.parts import embedding
from tests import score_oracle as oracle
from tests.test_scores_gpu import head_case, make_head

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [129, 143, 191, 255, 289, 385])
@pytest.mark.parametrize("top", [0, 20])
def test_warps_with_rows_missing(rows, top, monkeypatch):
    """A warp whose last rows are not there, beside whole ones, in strips that tell one another what they
    found: the first tile's look ahead, its note and the loads behind it."""
    monkeypatch.setattr(embedding, "scores_through_memory", lambda *sizes: False)
    h, w, tokens, dh, dw, dt = head_case(rows, 75000, 64, rows + top, torch.bfloat16)
    head = make_head(dw, torch.bfloat16)
    x = h @ w.T
    first = None
    for _ in range(3):
        got = head.score(dh, dt, top)
        head.linear.rt.check()
        if first is None:
            first = got
            oracle.check(got, x, tokens, top)
        for a, b in zip(got.tensors(), first.tensors()):
            assert torch.equal(a, b)
