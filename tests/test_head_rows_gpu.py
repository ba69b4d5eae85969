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


@pytest.mark.parametrize("rows,top", [(100, 0), (300, 5), (2048, 0), (64 * 256, 5)])
def test_nearly_certain_in_wide_strips(rows, top):
    """Rows whose likeliest token has all but some 1e-5, S - 1: a strip has up to 594 tiles (64 blocks of rows,
    one strip each), none of which may be lost beside that token's 1. With W = S - 1 (the sum over all other
    tokens) and D the greatest distance of a logit that counts, log p = -log1p(W) is off by
      W (2 + 1.173 D) 2^-23    the exponentials (their documented bound),
      W (30 + tiles) 2^-24     additions on a value's way: 10 in a piece of 32, 8 pieces, the tiles, 12 parts,
      W 2^-22                  log1pf (2 units),
      10 * 2^-24               the one piece in which the likeliest token itself is added up, 10 additions at most.
    The likeliest tokens stand at both ends of a strip, inside and beside others."""
    V, K, M = 151936, 16, 22.25
    gen = torch.Generator(device="cuda").manual_seed(rows)
    special = torch.tensor([0, 37, 255, 70001, V // 2, V - 1, V - 40, 8], device="cuda")
    w = torch.zeros((V, K), device="cuda")
    w[:, 8:] = torch.randint(-64, 65, (V, 8), generator=gen, device="cuda") * 2.0 ** -6
    w[special] = 0.0
    w[special, torch.arange(8, device="cuda")] = M
    h = torch.zeros((rows, K), device="cuda")
    which = torch.randint(0, 8, (rows,), generator=gen, device="cuda")
    h[torch.arange(rows, device="cuda"), which] = 1.0
    h[:, 8:] = torch.randint(-32, 33, (rows, 8), generator=gen, device="cuda") * 2.0 ** -6
    tokens = special[which].to(torch.int32)
    head = make_head(w.bfloat16(), torch.bfloat16)
    got = head.score(h.bfloat16(), tokens, top)
    head.linear.rt.check()
    wide, rest, far = w.double().t(), [], 0.0
    for a in range(0, rows, 512):
        d = h[a:a + 512].double() @ wide - M
        far = max(far, -float(d.min()))
        rest.append(torch.exp(d.scatter_(1, special[which[a:a + 512], None], -float("inf"))).sum(1))
    rest = torch.cat(rest)
    assert 1e-5 < float(rest.min()) and float(rest.max()) < 1e-4
    off = (got.logprobs.double() + torch.log1p(rest)).abs()
    tol = rest * ((2 + 1.173 * far) * 2.0 ** -23 + (30 + V // 256 + 1) * 2.0 ** -24 + 2.0 ** -22) + 10 * 2.0 ** -24
    assert float((off - tol).max()) <= 0.0
    if top:
        assert torch.equal(got.top_ids[:, 0], tokens) and torch.equal(got.top_logprobs[:, 0], got.logprobs)
