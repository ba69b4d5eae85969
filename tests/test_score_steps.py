"""Steps that score, without a GPU: an engine whose model is a table of logits by token, on the host."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from mormot2_ai_b200 import Engine, Entry, InferError, LlmClient, PartSpec
from mormot2_ai_b200 import kernels as K
from mormot2_ai_b200.cache.pages import CacheBook, GroupPlan
from mormot2_ai_b200.parts import HEADS
from mormot2_ai_b200.sampling import Scores

VOCAB, SLOTS, CONTEXT = 50, 4, 1024


class TableModel:
    """The logits behind a token are a row of a table and do not depend on what stood before."""

    def __init__(self):
        self.logp = torch.randn((VOCAB, VOCAB), generator=torch.Generator().manual_seed(1)).log_softmax(1)

    def forward(self, ctx, cache, on_state=None, score=None):
        if not ctx.n_want:
            return None
        x = self.logp[ctx.wanted]
        if score is None:
            return x
        given, top, limit = score
        assert given.shape == (ctx.n_want,)
        values, ids = x.topk(top, dim=1)
        return Scores(x.gather(1, given.long()[:, None])[:, 0], -(x.exp() * x).sum(1), ids.to(torch.int32),
                      values)


class Buffers:
    copied_bytes = 0

    def fill(self, seqs, longest_first=False):
        wanted = [int(s[2][w]) for s in seqs for w in s[3]]
        return SimpleNamespace(T=sum(len(s[2]) for s in seqs), B=len(seqs), n_want=len(wanted),
                               wanted=wanted, entry_slots=None, decode=all(len(s[2]) == 1 for s in seqs))


def table_engine(prefill_chunk=64, max_step_tokens=100):
    eng = Engine.__new__(Engine)
    plans = [GroupPlan(1, 16, 0, [0], 64, CONTEXT // 64, 0)]
    eng.book = CacheBook(plans, SLOTS, CONTEXT)
    eng.cache = SimpleNamespace(map_grown=lambda *lists: None, reset_state=lambda slot: None)
    eng.rt = SimpleNamespace(device=torch.device("cpu"))
    eng.buffers, eng.model = Buffers(), TableModel()
    eng.vocab_size, eng.max_context, eng.max_slots = VOCAB, CONTEXT, SLOTS
    eng.prefill_chunk, eng.max_step_tokens = prefill_chunk, max_step_tokens
    eng.has_state, eng.state_ok, eng.ids = False, [True] * SLOTS, [[] for _ in range(SLOTS)]
    eng.run = eng.on_state = None
    eng.use_graphs, eng.sort_from, eng.passes = False, 1 << 30, 0
    return eng


def text(n, seed=0):
    return np.random.default_rng(seed).integers(0, VOCAB, n).tolist()


@pytest.mark.parametrize("places", [np.array([[0, 1, 2], [3, 4, 5]]), np.array(3), np.zeros((3, 0), int),
                                    np.zeros((1, 2, 2), int)])
def test_places_that_are_no_list_are_refused(places):
    """Before any page is reserved, and whether or not the count of rows is that of the given tokens."""
    eng = table_engine()
    slot = eng.open()
    for n in (8, 200):
        with pytest.raises(InferError, match="shape"):
            eng.step([Entry(slot, text(n), places)])
        for given in ([1, 2], [1] * 6, [1], []):
            with pytest.raises(InferError, match="shape"):
                eng.score([Entry(slot, text(n), places, given)], top=2)
    assert eng.length(slot) == 0 and eng.book.held_pages(0) == 0 and eng.passes == 0


def test_places_in_rows_of_one():
    """A column of places is as many rows as places."""
    eng = table_engine()
    slot, t = eng.open(), text(150)
    x = eng.step([Entry(slot, t, np.array([[7], [149]]))])
    assert torch.equal(x, eng.model.logp[[t[7], t[149]]])
    assert eng.step([Entry(slot, [1], np.zeros((0, 3), int))]) is None


@pytest.mark.parametrize("cut", [dict(), dict(max_step_tokens=64), dict(prefill_chunk=7, max_step_tokens=30),
                                 dict(prefill_chunk=1000, max_step_tokens=1000)])
@pytest.mark.parametrize("places", [[99, 70], [99, 70, 99], [70, 99], [30, 0, 7], list(range(99, 63, -1)),
                                    [5, 5, 2, 99, 0], [99], []])
def test_places_in_any_order(places, cut):
    """All wanted rows in one of a step's several passes, or spread over them, one text or several."""
    eng = table_engine(**cut)
    for others in ([], [[3, 1]], [[], [0]]):
        ids = [text(100)] + [text(5, seed=9 + i) for i in range(len(others))]
        wants = [places] + others
        given = [text(len(w), seed=31 + i) for i, w in enumerate(wants)]
        for kind in (list, np.array):
            slots = [eng.open() for _ in ids]
            got = eng.score([Entry(s, t, kind(w) if w else w, g)
                             for s, t, w, g in zip(slots, ids, wants, given)], top=4)
            rows = eng.model.logp[[t[w] for t, want in zip(ids, wants) for w in want]]
            tokens = torch.tensor([g for one in given for g in one], dtype=torch.long)
            assert torch.equal(got.logprobs, rows.gather(1, tokens[:, None])[:, 0])
            values, order = rows.topk(4, dim=1)
            assert torch.equal(got.top_ids, order.to(torch.int32)) and torch.equal(got.top_logprobs, values)
            for s in slots:
                eng.close(s)


def test_a_head_on_another_device(monkeypatch):
    """Rows beside a head whose weight another device holds: refused before anything is launched."""
    head = HEADS.build(PartSpec("lm_head", {"name": "w", "tied": False, "vocab_size": 50, "hidden_size": 8}))
    weight = SimpleNamespace(get_device=lambda: 1, device="cuda:1")
    head.linear = SimpleNamespace(weight=weight, rt=None)
    monkeypatch.setattr(K, "elsewhere", lambda device: False)       # the rows' device is the current one
    h, tokens = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(InferError, match="weight on cuda:1"):
        head.score(h, tokens, 2)


def table_client(max_batch=2, vocab_limit=None):
    client = LlmClient.__new__(LlmClient)
    client.engine = table_engine()
    client.engine.plans = client.engine.book.plans
    client.engine.rt.check = lambda: None
    client.max_batch, client.vocab_limit = max_batch, vocab_limit
    return client


def test_texts_in_batches():
    client = table_client()
    texts = [text(n, seed=n) for n in (3, 1, 150, 2, 90)]
    got = client.score(texts, top=2)
    for t, s in zip(texts, got):
        want = client.engine.model.logp[t[:-1]].gather(1, torch.tensor(t[1:]).long()[:, None])[:, 0]
        assert [x.logprob for x in s.tokens] == want.tolist()
        assert all(len(x.alternatives) == 2 for x in s.tokens)
    assert client.engine.book.slots.free == SLOTS


@pytest.mark.parametrize("texts,top,match", [
    ([[1, 2], [3, 4], [5, 6], [7, 40]], 1, "sequence 3: token 40"),      # to score, but no candidate
    ([[1, 2], [3, 4], [5, 6], [50, 4]], 1, "sequence 3: token 50"), ([[1, 2], [3, -1]], 1, "sequence 1: token -1"),
    ([[1, 2], []], 1, "sequence 1: empty"), ([[1], [2]], 33, "33 alternatives"), ([[1]], -1, "alternatives"),
    ([[1, 2]], 31, "31 alternatives"), ([[1, 2]], True, "alternatives")])
def test_texts_are_refused_before_any_runs(texts, top, match):
    client = table_client(vocab_limit=30)
    with pytest.raises(InferError, match=match):
        client.score(texts, top=top)
    assert client.engine.passes == 0 and client.engine.book.slots.free == SLOTS


def test_a_first_token_is_fed_and_not_scored():
    client = table_client(vocab_limit=30)
    assert [len(s.tokens) for s in client.score([[45, 3, 29], [45]], top=1)] == [2, 0]
