"""Scores through the engine, the client and the command line: given texts, and the tokens of answers."""
import importlib

import numpy as np
import pytest

from mormot2_ai_b200 import CacheError, Engine, Entry, InferError, LlmClient, Sampling
from mormot2_ai_b200.cli import main
from mormot2_ai_b200.parts import embedding
from mormot2_ai_b200.sampling import DeviceSampler
from tests import score_oracle as oracle

pytestmark = pytest.mark.gpu


def engine_of(tiny, dtype, **more):
    more.setdefault("max_tokens", 4096)
    more.setdefault("max_slots", 8)
    return Engine.from_folder(tiny.folder, dtype=dtype, **more)


def logits_off(eng):
    """How far two orders of summation may take a logit of the head apart: a rounding of 2^-23 for each
    of its K products, of rows whose root mean square is at most the norm's largest weight."""
    w = eng.model.head.linear.weight.double()
    K = w.shape[1]
    size = K ** 0.5 * float(eng.model.final_norm.weight.double().abs().max())
    return K * 2.0 ** -23 * size * float(w.norm(dim=1).max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cut", [{}, dict(prefill_chunk=16, max_step_tokens=40)])
def test_score_is_what_the_logits_say(tiny, dtype, cut):
    eng = engine_of(tiny, dtype, **cut)
    rng = np.random.default_rng(1)
    texts = [tiny.tokens(n, seed=n) for n in (50, 2, 31, 1, 64)]
    wants = [list(range(49)), [0], [30, 0, 7, 7], [], [63]]
    givens = [texts[0][1:], None, [5, 6, 7, 8], [], [int(rng.integers(0, tiny.config.vocab_size))]]
    logits = []
    for kind in ("step", "score"):
        slots = [eng.open() for _ in texts]
        if kind == "step":
            x = eng.step([Entry(s, t, w) for s, t, w in zip(slots, texts, wants)]).double().cpu()
        else:
            entries = [Entry(slots[0], texts[0]), Entry(slots[1], texts[1])]
            entries += [Entry(s, t, w, g) for s, t, w, g in
                        zip(slots[2:], texts[2:], wants[2:], givens[2:])]
            got = eng.score(entries, top=7)
        assert [eng.length(s) for s in slots] == [len(t) for t in texts]
        for s in slots:
            eng.close(s)
    givens[1] = texts[1][1:]
    tokens = [g for one in givens for g in one]
    eng.rt.check()
    oracle.check(got, x.numpy(), tokens, 7, 0.0 if dtype == "float32" else logits_off(eng))


@pytest.mark.parametrize("kind", [np.int8, np.uint8, np.int16, np.int64, np.float64])
def test_places_of_any_integer_type(tiny, kind):
    """Places behind rows whose number the array's own type does not hold, and in a step of single tokens."""
    eng = engine_of(tiny, "float32")
    texts = [tiny.tokens(n, seed=n) for n in (100, 110, 120)]
    slots = [eng.open() for _ in texts]
    places = [7, 99, 3]
    want = eng.step([Entry(s, t, places) for s, t in zip(slots, texts)]).clone()
    alone = eng.step([Entry(slots[0], [5], [0, 0])]).clone()
    for s in slots:
        eng.truncate(s, 0)
    got = eng.step([Entry(s, t, np.array(places, kind)) for s, t in zip(slots, texts)])
    eng.rt.check()
    assert (got == want).all()
    assert (eng.step([Entry(slots[0], [5], np.array([0, 0], kind))]) == alone).all()
    for bad in ([100, 0], [-1], [3, 300]):
        with pytest.raises(InferError):
            eng.step([Entry(slots[0], texts[0], np.array(bad, np.int16))])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_score_token_by_token(tiny, dtype):
    """Decode passes: eager, captured, replayed; then a score of nothing."""
    eng = engine_of(tiny, dtype)
    ids = [tiny.tokens(9, seed=k) for k in range(3)]
    slots = [eng.open() for _ in ids]
    twins = [eng.open() for _ in ids]
    for t in range(8):
        got = eng.score([Entry(s, [i[t]], given=[i[t + 1]]) for s, i in zip(slots, ids)], top=4)
        kept = [x.clone() for x in got.tensors()]
        x = eng.step([Entry(s, [i[t]]) for s, i in zip(twins, ids)])
        oracle.check(type(got)(*kept), x.double().cpu().numpy(), [i[t + 1] for i in ids], 4)
    got = eng.score([Entry(slots[0], [1]), Entry(slots[1], [2, 3], want=[], given=[])], top=2)
    assert got.logprobs.shape == (0,) and got.top_ids.shape == (0, 2)
    assert eng.length(slots[0]) == 9 and eng.length(slots[1]) == 10
    eng.rt.check()


FAMILIES = ["busavik", "fimudra", "sezopel", "laralix", "lotirax", "tenusun"]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("family", FAMILIES)
def test_every_family_scores(family, dtype, tmp_path, monkeypatch):
    """Heads with a factor or capped logits, states, several passes: the fused form and the stored one
    against the logits of a step of the same engine."""
    models = importlib.import_module(f"tests.{family}_models")
    for name in models.SMALL:
        small = models.SmallModel(name, str(tmp_path / name))
        eng = Engine.from_folder(small.folder, dtype=dtype, max_tokens=1024, max_slots=3, prefill_chunk=40)
        head, norms = eng.model.head, []
        forward = head.forward

        def watched(h):
            norms.append(float(h.double().norm(dim=1).max()))
            return forward(h)
        texts = [small.tokens(n, seed=n) for n in (70, 3, 41)]
        slots = [eng.open() for _ in texts]
        head.forward = watched
        x = eng.step([Entry(s, t, list(range(len(t) - 1))) for s, t in zip(slots, texts)])
        head.forward = forward
        x = x.double().cpu().numpy()
        w = head.linear.weight.double()
        # the products' order, the factor, the cap (a division, tanh and a product, each side its own)
        off = abs(head.scale) * w.shape[1] * 2.0 ** -23 * max(norms) * float(w.norm(dim=1).max())
        off += 2.0 ** -23 * np.abs(x).max() + 2.0 ** -23 * 8 * head.softcap
        for fused in (False, True):
            monkeypatch.setattr(embedding, "scores_through_memory", lambda *sizes: not fused)
            for s in slots:
                eng.truncate(s, 0)
            got = eng.score([Entry(s, t) for s, t in zip(slots, texts)], top=6)
            eng.rt.check()
            oracle.check(got, x, [t for one in texts for t in one[1:]], 6, off)


def test_score_refusals(tiny_a_model):
    eng = engine_of(tiny_a_model, "float32")
    slot = eng.open()
    V = eng.vocab_size
    for entry in (Entry(slot, [1, 2], want=[0]), Entry(slot, [1, 2], given=[3]),
                  Entry(slot, [1, 2], [0], [3, 4]), Entry(slot, [1, 2], [0], [V]),
                  Entry(slot, [1, 2], [2], [3]), Entry(slot, [1, 2], [-1], [3]),
                  Entry(slot, [1, V], [0], [3]), Entry(slot, [], [], [])):
        with pytest.raises(InferError):
            eng.score([entry], top=3)
        assert eng.length(slot) == 0
    with pytest.raises(InferError):
        eng.score([Entry(slot, [1, 200])], vocab_limit=100)
    for top in (-1, 33, 2.0, True):
        with pytest.raises(InferError):
            eng.score([Entry(slot, [1, 2])], top=top)
    with pytest.raises(InferError):
        eng.score([])
    with pytest.raises(CacheError):
        eng.score([Entry(slot + 1, [1, 2])])
    sampler = DeviceSampler(eng.rt.device, eng.max_slots, eng.vocab_size)
    eng.step([Entry(slot, [1])])
    with pytest.raises(InferError):
        eng.decode_run([slot], [2], [3], sampler, Sampling(), top=40)
    assert eng.run is None
    with pytest.raises(InferError):
        eng.decode_run([slot], [2], [3], sampler, Sampling(), history=True, top=4)
    assert eng.run is None


def test_client_scores_texts(tiny):
    """Against the plain implementation's logits, in batches of two (three texts at most fit)."""
    client = LlmClient(tiny.folder, dtype="float32", max_batch=2, cache_tokens=512)
    limit = client.max_context
    texts = [tiny.tokens(n, seed=40 + n) for n in (30, 1, 2, 70, min(limit, 200) + 1)]
    got = client.score(texts, top=5)
    assert [len(s.tokens) for s in got] == [len(t) - 1 for t in texts]
    for text, s in zip(texts, got):
        if len(text) == 1:
            assert s.perplexity == 1.0 and s.logprob == 0.0
            continue
        ref = np.asarray(tiny.reference(text[:-1]), dtype=np.float64)
        lp, h, ids, alt = oracle.scores(ref, text[1:], 5)
        # a logit is off by 1e-5 of the largest, a log probability by twice that and its own rounding
        tol = 2e-5 * max(1.0, np.abs(ref).max()) + 2e-5
        assert np.abs(np.array([t.logprob for t in s.tokens]) - lp).max() < tol
        assert np.abs(np.array([t.entropy for t in s.tokens]) - h).max() < 10 * tol
        for k, t in enumerate(s.tokens):
            assert len(t.alternatives) == 5
            for (i, p), q in zip(t.alternatives, alt[k]):
                assert abs(p - q) < tol and abs(ref[k][i] - ref[k][ids[k][0]] + alt[k][0] - p) < tol
        assert abs(np.log(s.perplexity) + lp.mean()) < tol
    assert all(client.engine.book.held_pages(g) == 0 for g in range(len(client.engine.plans)))
    for bad in ([[]], [[1, tiny.config.vocab_size]], [[1] * (limit + 2)]):
        with pytest.raises(InferError):
            client.score(bad)
    with pytest.raises(InferError):
        client.score([[1, 2, 3]], top=33)
    assert client.engine.stats()["slots_open"] == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("how", [dict(temperature=0.0), dict(temperature=0.9, top_k=20)])
def test_answers_with_their_scores(tiny, dtype, how):
    client = LlmClient(tiny.folder, dtype=dtype, max_batch=3, cache_tokens=1024)
    prompts = [tiny.tokens(n, seed=70 + n) for n in (4, 33, 17, 1, 9)]
    plain = client.generate(prompts, max_tokens=9, seed=5, stop=[], **how)
    got = client.generate(prompts, max_tokens=9, seed=5, stop=[], logprobs=6, **how)
    assert [o.tokens for o in got] == plain
    said = client.score([p + a for p, a in zip(prompts, plain)], top=6)
    tol = 1e-4 if dtype == "float32" else 0.15
    for p, o, s in zip(prompts, got, said):
        assert len(o.scores) == len(o.tokens) == 9
        for token, mine, ref in zip(o.tokens, o.scores, s.tokens[len(p) - 1:]):
            assert abs(mine.logprob - ref.logprob) < tol and abs(mine.entropy - ref.entropy) < 4 * tol
            assert len(mine.alternatives) == 6
            values = [q for _, q in mine.alternatives]
            assert values == sorted(values, reverse=True)
            if how["temperature"] == 0.0:
                assert mine.alternatives[0] == (token, mine.logprob)
    none = client.generate(prompts[:1], max_tokens=3, seed=5, stop=[], logprobs=0, **how)
    assert [len(t.alternatives) for t in none[0].scores] == [0, 0, 0]
    assert client.generate(prompts[:1], max_tokens=3, seed=5, stop=[], details=True, **how)[0].scores is None


def test_commands(tiny_b_model, capsys):
    folder = tiny_b_model.folder
    assert main(["llm-score", folder, "5,17,3,9;4", "f32", "--top", "2", "--max-context", "64"]) == 0
    lines = capsys.readouterr().out.splitlines()
    assert lines[0].startswith("3 tokens scored: log probability -") and len(lines) == 5
    assert [line.split()[0] for line in lines[1:4]] == ["17", "3", "9"]
    assert lines[4] == "0 tokens scored: log probability 0.0000, perplexity 1.0000"
    assert main(["llm-quickstart", folder, "5,17", "f32", "--max-tokens", "3", "--logprobs", "1",
                 "--temperature", "0", "--max-context", "64"]) == 0
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 4 and [int(line.split()[0]) for line in lines[1:]] == [
        int(t) for t in lines[0].split(",")]
