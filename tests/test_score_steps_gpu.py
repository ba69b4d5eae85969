"""Scores at places in any order, of texts that take several passes, against the logits of a step."""
import numpy as np
import pytest

from mormot2_ai_b200 import Entry, InferError
from tests import score_oracle as oracle
from tests.test_score_engine_gpu import engine_of, logits_off

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,places", [
    (100, [99, 70]), (100, [99, 70, 99]), (100, list(range(99, 63, -1))), (100, [30, 0, 7]),
    (100, [99, 3, 70, 3]), (65, [64, 64]), (65, [64, 5]), (120, [64])])
def test_places_in_any_order(tiny, dtype, n, places):
    """All wanted rows in the last of two passes, in the first, in both, in a pass of a single token (which
    is captured the second time and replayed the third); alone and beside another text."""
    eng = engine_of(tiny, dtype, prefill_chunk=64)
    rng = np.random.default_rng(n)
    off = 0.0 if dtype == "float32" else logits_off(eng)
    for others in ([], [(90, [80, 66]), (3, [2, 0])]):
        ids = [tiny.tokens(k, seed=k) for k in [n] + [k for k, _ in others]]
        wants = [places] + [w for _, w in others]
        given = [rng.integers(0, eng.vocab_size, len(w)).tolist() for w in wants]
        slots = [eng.open() for _ in ids]
        x = eng.step([Entry(s, t, w) for s, t, w in zip(slots, ids, wants)]).double().cpu().numpy()
        for kind in (list, np.array, list):
            for s in slots:
                eng.truncate(s, 0)
            got = eng.score([Entry(s, t, kind(w), g) for s, t, w, g in zip(slots, ids, wants, given)], top=9)
            eng.rt.check()
            oracle.check(got, x, [g for one in given for g in one], 9, off)
        for s in slots:
            eng.close(s)


def test_places_that_are_no_list(tiny):
    eng = engine_of(tiny, "float32", prefill_chunk=64)
    slot, t = eng.open(), tiny.tokens(100, seed=1)
    for places in (np.array([[0, 1, 2], [3, 4, 5]]), np.array(3)):
        with pytest.raises(InferError):
            eng.score([Entry(slot, t, places, [1, 2])])
        with pytest.raises(InferError):
            eng.step([Entry(slot, t, places)])
    assert eng.length(slot) == 0 and eng.faults() == []
