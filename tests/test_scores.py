"""Scores and a step's arrays without a GPU: refusals, the layout on the host, pages in bulk, the
generation loop that carries scores along, what a text's score says."""
import math
import random

import pytest
import torch

from mormot2_ai_b200 import CacheError, InferError, KernelError, PartSpec, token_scores
from mormot2_ai_b200 import kernels as K
from mormot2_ai_b200.cache.pages import CacheBook, FreeList, GroupPlan
from mormot2_ai_b200.client import TextScore
from mormot2_ai_b200.engine.generate import Request, generate
from mormot2_ai_b200.parts import HEADS
from mormot2_ai_b200.sampling import Scores
from mormot2_ai_b200.sampling.scores import TokenScore
from tests.test_generate_loop import ScriptedRun, ScriptedStepper

i32 = lambda *v: torch.tensor(v, dtype=torch.int32)


def test_token_scores_refusals():
    x, t = torch.zeros(3, 10), i32(1, 2, 3)
    bad = [(x.double(), t, 1, None), (x.bfloat16(), t, 1, None), (x[0], t, 1, None),
           (x[:, :0], t, 0, None), (x.t().contiguous().t(), t, 1, None), (x, t.long(), 1, None),
           (x, t[:2], 1, None), (x, t[:, None], 1, None), (x, t, -1, None), (x, t, 11, None),
           (x, t, 33, None), (x, t, True, None), (x, t, 1.0, None), (x, t, 1, 0), (x, t, 5, 4)]
    for args in bad:
        with pytest.raises(InferError):
            token_scores(*args)
    with pytest.raises(InferError):
        token_scores(x, t, 2, None, Scores.empty(3, 1, "cpu"))
    with pytest.raises(KernelError, match="not on the GPU"):
        token_scores(x, t, 1)


def test_head_score_refusals():
    head = HEADS.build(PartSpec("lm_head", {"name": "w", "tied": False, "vocab_size": 50,
                                            "hidden_size": 8}))
    h, t = torch.zeros(3, 8, dtype=torch.bfloat16), i32(1, 2, 3)
    for args in ((h[:, :7], t, 1), (h[0], t, 1), (h.t().contiguous().t(), t, 1), (h, t.long(), 1),
                 (h, t[:2], 1), (h, t, 33), (h, t, 3, 2), (h, t, 0, 0)):
        with pytest.raises(InferError):
            head.score(*args)


def test_step_index_refusals():
    a = lambda n: torch.zeros(n, dtype=torch.int32)
    good = [a(3), a(3), a(3), a(4), a(9), a(9), a(9)]
    for k in range(7):
        for wrong in (a(2), good[k].long(), good[k][:, None], torch.zeros(2 * len(good[k]), dtype=torch.int32)[::2]):
            with pytest.raises(KernelError):
                K.step_index(*good[:k], wrong, *good[k + 1:])
    with pytest.raises(KernelError, match="not on the GPU"):
        K.step_index(*good)


def test_map_pages_refusals():
    a = lambda *n: torch.zeros(*n, dtype=torch.int32)
    good = [a(4, 6), a(3), a(3), a(3), a(3), a(5)]
    for k in range(6):
        for wrong in (good[k].long(), good[k][None], good[k][:2] if 0 < k < 5 else good[k].float()):
            with pytest.raises(KernelError):
                K.map_pages(*good[:k], wrong, *good[k + 1:])
    with pytest.raises(KernelError):
        K.map_pages(a(6, 4).t(), *good[1:])
    with pytest.raises(KernelError):
        K.map_pages(*good, -1)
    with pytest.raises(KernelError, match="not on the GPU"):
        K.map_pages(*good)


def test_scores_in_a_buffer():
    buffer = torch.arange(3 * (2 + 2 * 4), dtype=torch.int32).view(torch.float32)
    s = Scores.in_buffer(buffer, 3, 4)
    s.logprobs.copy_(torch.tensor([-1.0, -2.0, -3.0]))
    s.entropy.copy_(torch.tensor([0.5, 1.5, 2.5]))
    s.top_logprobs.copy_(-torch.arange(12.0).view(3, 4))
    assert s.top_ids.tolist() == [[6, 7, 8, 9], [10, 11, 12, 13], [14, 15, 16, 17]]
    rows = s.on_host()
    assert rows[1] == TokenScore(-2.0, 1.5, [(10, -4.0), (11, -5.0), (12, -6.0), (13, -7.0)])
    copy = Scores.in_buffer(torch.zeros_like(buffer), 3, 4)
    copy.put(torch.tensor([2, 0, 1]), s)
    assert copy.logprobs.tolist() == [-2.0, -3.0, -1.0] and copy.top_ids[2].tolist() == [6, 7, 8, 9]
    copy.rows(1, 3).take(s.rows(0, 2))
    assert copy.on_host()[1:] == rows[:2]
    assert Scores.in_buffer(torch.zeros(6), 3, 0).on_host()[2] == TokenScore(0.0, 0.0, [])


def test_text_score():
    t = TextScore([TokenScore(math.log(0.5), 0.0, []), TokenScore(math.log(0.125), 0.0, [])])
    assert math.isclose(t.logprob, math.log(1 / 16)) and math.isclose(t.perplexity, 4.0)
    assert TextScore([]).perplexity == 1.0
    assert TextScore([TokenScore(-math.inf, 0.0, [])]).perplexity == math.inf
    assert math.isnan(TextScore([TokenScore(math.nan, 0.0, [])]).perplexity)


def test_take_many_hands_out_what_take_does():
    a, b = FreeList(9, "page"), FreeList(9, "page")
    for f in (a, b):
        f.take(), f.take(), f.take()
        f.give(1)
    assert a.take_many(4) == [b.take() for _ in range(4)]
    assert a.take_many(0) == [] and a.free == b.free == 3 and a._held == b._held
    with pytest.raises(CacheError):
        a.take_many(4)
    assert a.free == 3


def test_grow_maps_what_reserve_maps():
    plans = [GroupPlan(1, 16, 0, [0], 60, 20, 0), GroupPlan(1, 16, 70, [1], 24, 3, 3)]
    rng = random.Random(3)
    a, b = CacheBook(plans, 8, 1280), CacheBook(plans, 8, 1280)
    for book in (a, b):
        for _ in range(8):
            book.open()
    refused = 0
    for _ in range(200):
        slots = rng.sample(range(8), rng.randint(1, 8))
        requests = [(s, min(1280, a.length[s] + rng.randint(0, 150))) for s in slots]
        try:
            entries = a.reserve(requests)
        except CacheError:
            refused += 1
            with pytest.raises(CacheError):
                b.grow(requests)
            for book in (a, b):
                for s in slots[:3]:
                    book.truncate(s, 0)
            assert a.pages == b.pages
            continue
        for (held, pages), mine in zip(b.grow(requests), entries):
            assert [p for _, _, p in mine] == pages
            assert [(s, h + j) for (s, _), (h, n) in zip(requests, held) for j in range(n)] == [
                (s, e) for s, e, _ in mine]
        assert a.pages == b.pages and a.high == b.high
        for s, n in requests:
            a.commit(s, n)
            b.commit(s, n)
    assert refused > 3


class ScoredRun(ScriptedRun):
    def read(self):
        got = super().read()
        self.last_scores = [f"score of {t}" for t in got]
        return got


class ScoredStepper(ScriptedStepper):
    top = 3

    def prefill(self, entries):
        got = super().prefill(entries)
        self.last_scores = [f"score of {t}" for t in got]
        return got

    def decode(self, members):
        self.open_runs += 1
        return ScoredRun(self, members)


def test_the_loop_carries_scores():
    scripts = {1: [10, 11, 99, 12], 2: [20, 21, 22, 23, 24, 25], 3: [99], 4: [40, 41, 99]}
    reqs = [Request([1, 5, 5], 10, {99}), Request([2], 4, {99}), Request([3] * 7, 10, {99}),
            Request([4], 9, {99})]
    for o in generate(ScoredStepper(scripts, max_batch=2), reqs):
        assert o.scores == [f"score of {t}" for t in o.tokens]
    for o in generate(ScriptedStepper(scripts), reqs):
        assert o.scores is None
