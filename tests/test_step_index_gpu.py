"""The arrays of a packed step and the page tables' rows, worked out on the device from lengths."""
import numpy as np
import pytest
import torch

from mormot2_ai_b200 import kernels as K
from mormot2_ai_b200.cache.pages import PAGE, CacheBook, GroupPlan, pages_for
from mormot2_ai_b200.cache.storage import CacheStorage
from mormot2_ai_b200.engine.batch import StepBuffers
from tests.gpu_helpers import DEV

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device=DEV)


def sequences(B, seed, most, zeros=0.2):
    rng = np.random.default_rng(seed)
    new = rng.integers(1, most + 1, B)
    new[rng.random(B) < zeros] = 0
    return rng.permutation(2 * B)[:B], rng.integers(0, 5000, B), new


@pytest.mark.parametrize("B,most,spare", [(1, 1, 0), (1, 5000, 3), (3, 40, 1), (64, 300, 0),
                                          (1023, 3, 5), (1024, 20, 0), (1025, 9, 2), (5000, 4, 100)])
def test_step_index(B, most, spare):
    slots, past, new = sequences(B, B + most, most, 0.2 if B > 1 else 0.0)
    T = int(new.sum())
    arrays = [torch.full((T + spare,), -7, dtype=torch.int32, device=DEV) for _ in range(3)]
    start = torch.full((B + 1,), -7, dtype=torch.int32, device=DEV)
    K.step_index(i32(slots), i32(past), i32(new), start, *arrays)
    seq = np.repeat(np.arange(B), new)
    starts = np.concatenate([[0], np.cumsum(new)])
    want = [seq, past[seq] + np.arange(T) - starts[seq], slots[seq]]
    assert start.tolist() == starts.tolist()
    for got, w in zip(arrays, want):
        assert got[:T].tolist() == w.tolist() and got[T:].tolist() == [-7] * spare


def test_step_index_of_nothing_and_of_too_much():
    start = torch.full((1,), 5, dtype=torch.int32, device=DEV)
    none = i32([])
    K.step_index(none, none, none, start, none, none, none)
    assert start.tolist() == [0]
    start = torch.zeros(4, dtype=torch.int32, device=DEV)
    empty = [torch.zeros(0, dtype=torch.int32, device=DEV) for _ in range(3)]
    K.step_index(i32([3, 1, 2]), i32([0, 9, 4]), i32([0, 0, -5]), start, *empty)
    assert start.tolist() == [0, 0, 0, 0]
    # arrays shorter than the step: what does not fit is not written
    guard = [torch.full((8,), -7, dtype=torch.int32, device=DEV) for _ in range(3)]
    K.step_index(i32([3, 1, 2]), i32([0, 9, 4]), i32([2, 3, 4]), start, *(g[:4] for g in guard))
    assert start.tolist() == [0, 2, 5, 9]
    assert guard[1].tolist() == [0, 1, 9, 10, -7, -7, -7, -7]


@pytest.mark.parametrize("B,ring", [(1, 0), (5, 0), (64, 0), (64, 9), (1024, 3), (1500, 0)])
def test_map_pages(B, ring):
    rng = np.random.default_rng(B + ring)
    slots, past, new = sequences(B, B, 700)
    max_pages = ring or 100
    up = lambda n: np.minimum(-(-n // PAGE), ring) if ring else -(-n // PAGE)
    # some hold more pages than their positions take (a run that was cut short)
    held = np.minimum(up(past) + (rng.random(B) < 0.3) * rng.integers(0, 4, B), max_pages)
    more = np.maximum(0, up(past + new) - held)
    pages = rng.permutation(int(more.sum()) + 50)[:int(more.sum())]
    table = torch.full((2 * B, max_pages), -3, dtype=torch.int32, device=DEV)
    want = np.full((2 * B, max_pages), -3)
    at = 0
    for s, h, m in zip(slots, held, more):
        want[s, h:h + m] = pages[at:at + m]
        at += m
    K.map_pages(table, i32(slots), i32(past), i32(new), i32(held), i32(pages), ring)
    assert np.array_equal(table.cpu().numpy(), want)


def test_map_pages_stays_inside():
    """Slots and entries outside the table, and more entries than pages, are left."""
    big = torch.full((8, 4), -3, dtype=torch.int32, device=DEV)
    table = big[2:6]
    K.map_pages(table, i32([-1, 4, 1, 3, 0]), i32([0] * 5), i32([64, 64, 6 * 64, 64, 64]),
                i32([0, 0, 1, 0, 0]), i32([10, 11, 12, 13, 14, 15, 16, 17]))
    assert big[:2].eq(-3).all() and big[6:].eq(-3).all()
    assert table[1].tolist() == [-3, 12, 13, 14] and table[3].tolist() == [17, -3, -3, -3]
    assert table[0].eq(-3).all() and table[2].eq(-3).all()


@pytest.mark.parametrize("B,lo,hi,wants", [(3, 30, 60, "last"), (40, 1, 90, "last"),
                                           (17, 5, 333, "all"), (9, 50, 70, "mixed")])
def test_fill(B, lo, hi, wants):
    """A step's context is what its sequences say, for many tokens as for few."""
    rng = np.random.default_rng(B)
    seqs = []
    for b in range(B):
        n = int(rng.integers(lo, hi + 1))
        want = {"last": [n - 1], "all": np.arange(n),
                "mixed": [[], [0], [n - 1, 0, 0], np.arange(n - 1)][b % 4]}[wants]
        tokens = rng.integers(0, 999, n)
        seqs.append((int(rng.permutation(64)[b]) if B <= 1 else b * 3 % 50, int(rng.integers(0, 3000)),
                     tokens if b % 2 else tokens.tolist(), want))
    buffers = StepBuffers(16384, 64, torch.device(DEV))
    for _ in range(2):
        c = buffers.fill(seqs)
        new = [len(s[2]) for s in seqs]
        starts = np.concatenate([[0], np.cumsum(new)])
        assert c.T == starts[-1] and c.B == B and c.host_new == new
        assert c.tok_ids.tolist() == [int(t) for s in seqs for t in s[2]]
        assert c.tok_seq.tolist() == [b for b, n in enumerate(new) for _ in range(n)]
        assert c.tok_pos.tolist() == [s[1] + i for s in seqs for i in range(len(s[2]))]
        assert c.tok_slot.tolist() == [s[0] for s in seqs for _ in s[2]]
        assert c.seq_slot.tolist() == c.entry_slots.tolist() == [s[0] for s in seqs]
        assert c.seq_start.tolist() == starts.tolist() and c.seq_past.tolist() == [s[1] for s in seqs]
        assert c.want_rows.tolist() == [int(starts[b]) + int(w) for b, s in enumerate(seqs) for w in s[3]]


@pytest.mark.parametrize("max_context", [256, 40960])
def test_tables_follow_the_book(max_context):
    """Growing, cutting and giving back: the tables on the device name the book's pages, whether rows
    are copied or a kernel writes the entries."""
    slots = 48
    plans = [GroupPlan(1, 16, 0, [0], 3000, pages_for(max_context), 0),
             GroupPlan(1, 16, 100, [1], 600, min(6, pages_for(max_context)), 6)]
    if max_context == 256:
        plans = plans[:1]
    book = CacheBook(plans, slots, max_context)
    cache = CacheStorage(plans, slots, torch.bfloat16, torch.device(DEV), {})
    rng = np.random.default_rng(max_context)
    held = {}
    for turn in range(30):
        for s in list(held):
            if rng.random() < 0.2:
                book.close(s)
                del held[s]
            elif rng.random() < 0.1:
                book.truncate(s, 0)
                held[s] = 0
        while len(held) < slots and rng.random() < 0.9:
            held[book.open()] = 0
        mine = [s for s in held if rng.random() < 0.7]
        new = [int(min(rng.integers(1, 900 if turn % 3 else 3), max_context - held[s])) for s in mine]
        mine, new = zip(*[(s, n) for s, n in zip(mine, new) if n > 0]) if any(new) else ((), ())
        past = [held[s] for s in mine]
        grown = book.grow([(s, p + n) for s, p, n in zip(mine, past, new)])
        cache.map_grown(list(mine), past, list(new), grown)
        for s, p, n in zip(mine, past, new):
            book.commit(s, p + n)
            held[s] = p + n
        assert cache.table_faults(book) == []
