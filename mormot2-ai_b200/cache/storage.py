"""The cache on the device: per group the pooled keys and values of its lines and the page
table, and per state line the fixed-size state of every slot.

Layout of a line's keys (values alike): ``[pages, kv_heads, 64, head_dim]`` — the 64
positions of a page for one KV head are contiguous, so attention streams whole tiles.
The element type is the activation type of the engine (bfloat16, or float32 on the 32-bit
path); the reference keeps half floats or floats (``model.qwen3.cuda.pas:907-937``).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Tuple

import torch

from .. import kernels as K
from .guards import Guards, alloc
from .pages import PAGE, CacheBook, GroupPlan


@dataclass
class CacheLine:
    """What a mixer gets of its line: pools, the page table of its group and the ring size."""
    k: torch.Tensor            # [pages, kv_heads, PAGE, head_dim]
    v: Optional[torch.Tensor]  # None in a group of one plane (rows that hold a latent)
    page_table: torch.Tensor   # int32 [slots, max_pages] on the device
    max_pages: int
    ring_pages: int
    window: int
    kv_heads: int
    head_dim: int
    v_dim: int = 0             # the size of a value row (0: head_dim)


class CacheStorage:
    def __init__(self, plans: List[GroupPlan], max_slots: int, dtype: torch.dtype,
                 device: torch.device, state_needs: Dict[int, "StateNeed"],
                 guards: Optional[Guards] = None):
        self.plans = plans
        self.pools: List[torch.Tensor] = []
        self.tables: List[torch.Tensor] = []
        self.lines: Dict[int, CacheLine] = {}
        self.value_pools: Dict[int, torch.Tensor] = {}   # of groups whose value rows differ in size
        for g, plan in enumerate(plans):
            v_dim = getattr(plan, "v_dim", 0)
            if v_dim and plan.planes == 2:
                # keys and values in pools of their own: [lines, 1, pages, kv_heads, PAGE, size]
                pool = alloc(guards, f"keys of group {g}",
                             (len(plan.lines), 1, plan.n_pages, plan.kv_heads, PAGE,
                              plan.head_dim), dtype, device)
                self.value_pools[g] = alloc(guards, f"values of group {g}",
                                            (len(plan.lines), plan.n_pages, plan.kv_heads, PAGE,
                                             v_dim), dtype, device)
            else:
                pool = alloc(guards, f"keys and values of group {g}",
                             (len(plan.lines), plan.planes, plan.n_pages, plan.kv_heads, PAGE,
                              plan.head_dim),
                             dtype, device)
            table = alloc(guards, f"page table of group {g}", (max_slots, plan.max_pages),
                          torch.int32, device)
            self.pools.append(pool)
            self.tables.append(table)
            for i, line in enumerate(plan.lines):
                if g in self.value_pools:
                    values = self.value_pools[g][i]
                else:
                    values = pool[i, 1] if plan.planes > 1 else None
                self.lines[line] = CacheLine(pool[i, 0], values, table, plan.max_pages,
                                             plan.ring_pages, plan.window, plan.kv_heads,
                                             plan.head_dim, v_dim)
        # what a step's new pages are written to the tables from: per group five lists at most
        room = sum(4 * max_slots + p.n_pages for p in plans)
        self.lists_host = torch.zeros(room, dtype=torch.int32).pin_memory() if room else None
        self.lists = alloc(guards, "lists of new pages", (room,), torch.int32, device)
        self.lists_copied = torch.cuda.Event()
        self.lists_busy = False
        # fixed-size state per slot, at its initial value when a sequence starts; beside it a
        # copy of the same size that a step saves the slots it touches into, so that a step
        # that fails half way leaves the state it found
        self.state_init: Dict[int, float] = {l: float(n.init) for l, n in state_needs.items()}
        self.states: Dict[int, torch.Tensor] = {
            line: alloc(guards, f"state of line {line}", (max_slots,) + tuple(n.shape),
                        getattr(torch, n.dtype), device, float(n.init))
            for line, n in state_needs.items()}
        self.saved: Dict[int, torch.Tensor] = {l: torch.empty_like(s)
                                               for l, s in self.states.items()}

    def bytes(self) -> int:
        return (sum(p.numel() * p.element_size() for p in self.pools)
                + sum(p.numel() * p.element_size() for p in self.value_pools.values())
                + sum(2 * s.numel() * s.element_size() for s in self.states.values()))

    def map_pages(self, new_entries: List[List[Tuple[int, int, int]]]) -> None:
        """Writes the new table entries of ``CacheBook.reserve`` to the device tables, in the order of
        the stream; whatever is launched next finds them there."""
        work = []
        for g, entries in enumerate(new_entries):
            first: Dict[int, int] = {}
            many: Dict[int, int] = {}
            for slot, entry, _ in entries:
                first.setdefault(slot, entry)
                many[slot] = many.get(slot, 0) + 1
            pages = {slot: [] for slot in first}
            for slot, _, page in entries:
                pages[slot].append(page)
            work.append((list(first), [0] * len(first),
                         [PAGE * (first[s] + many[s]) for s in first], list(first.values()),
                         [p for s in first for p in pages[s]]))
        if self._write_entries(work):
            # a kernel may read a table ahead of its wait for the kernel before it, which then must
            # not be the one that wrote it
            self.lists[:1].copy_(self.lists_host[:1], non_blocking=True)
            self.lists_copied.record()

    def map_grown(self, slots: List[int], past: List[int], new: List[int], grown) -> None:
        """``map_pages`` for what ``CacheBook.grow`` returned for distinct ``slots`` that held
        ``past`` positions and grow by ``new``. A copy has to follow on the stream before kernels that
        read tables ahead of their waits (the one of the step's index arrays does)."""
        work = []
        for held, pages in grown:
            if len(pages) <= 0:
                work.append(())
                continue
            some = [i for i, (_, n) in enumerate(held) if n]
            work.append(([slots[i] for i in some], [past[i] for i in some], [new[i] for i in some],
                         [held[i][0] for i in some], pages))
        self._write_entries(work)

    def _write_entries(self, work) -> bool:
        """Per group the slots, past and new positions, pages held, and new pages; whether there
        were any. The lists go to the device in one copy."""
        flat: List[int] = []
        for lists in work:
            for one in lists:
                flat += one
        if not flat:
            return False
        if self.lists_busy:
            self.lists_copied.synchronize()          # the last copy must have read the host's lists
        self.lists_host.numpy()[:len(flat)] = flat
        self.lists[:len(flat)].copy_(self.lists_host[:len(flat)], non_blocking=True)
        self.lists_copied.record()
        self.lists_busy = True
        at = 0
        for g, lists in enumerate(work):
            if lists and lists[0]:
                B, N = len(lists[0]), len(lists[4])
                K.map_pages_packed(self.tables[g], self.lists, at, B, N, self.plans[g].ring_pages)
                at += 4 * B + N
        return True

    def table_faults(self, book: CacheBook) -> List[str]:
        """Compares the page tables on the device with the bookkeeping: every entry that a
        sequence holds must name the page the book gave it, and no page may be held twice.
        Returns what is wrong (nothing, when all is well)."""
        out = []
        for g, table in enumerate(self.tables):
            dev = table.cpu()
            seen: Dict[int, int] = {}
            for slot in range(dev.shape[0]):
                for entry, page in enumerate(book.pages[g][slot]):
                    if int(dev[slot, entry]) != page:
                        out.append(f"group {g}, slot {slot}, entry {entry}: the device table "
                                   f"names page {int(dev[slot, entry])}, the book page {page}")
                    if page in seen:
                        out.append(f"group {g}: page {page} is held by slots {seen[page]} "
                                   f"and {slot}")
                    seen[page] = slot
        return out

    def reset_state(self, slot: int) -> None:
        for line, s in self.states.items():
            s[slot].fill_(self.state_init[line])

    def save_states(self, slots: torch.Tensor) -> None:
        """Keeps a copy of the state of ``slots`` (int64 indices on the device)."""
        for line, s in self.states.items():
            self.saved[line].index_copy_(0, slots, s.index_select(0, slots))

    def restore_states(self, slots: torch.Tensor) -> None:
        """Puts the copy of ``save_states`` back."""
        for line, s in self.states.items():
            s.index_copy_(0, slots, self.saved[line].index_select(0, slots))
