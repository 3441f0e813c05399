"""Forked requests, pages that move, pools that change their size: no page lost, nothing written by one request seen by another."""
import random

import numpy as np
import pytest
import torch

from pytriton_llama_b200.cache.manager import CacheManager, OutOfPages, OutOfSlots, PagePool
from pytriton_llama_b200.parts.base import CacheNeed

FULL = CacheNeed(kind="full", kv_heads=1, head_dim=16)
FULL8 = CacheNeed(kind="full", kv_heads=1, head_dim=16, bits=8)
WINDOW = CacheNeed(kind="window", kv_heads=1, head_dim=32, window=21, keep_first=3)
CHUNK = CacheNeed(kind="chunk", kv_heads=1, head_dim=32, window=40)
POOLED = CacheNeed(kind="full", kv_heads=1, head_dim=16, pool_block=5, states=(("s", (3,)),))
STATE = CacheNeed(kind="none", state_shape=(2,))


def copy(tensors, src, dst):
    assert len(src) == len(dst) and len(set(dst)) == len(dst) and not set(src) & set(dst)
    for t in tensors:
        t[list(dst)] = t[list(src)]


class Content:
    """Stores a number per token through the manager's slots and reads it back through its block tables."""

    def __init__(self, entries, page_size=16, pages=60, max_requests=8, max_seq_len=200):
        self.m = CacheManager(entries, page_size, pages, max_requests, max_seq_len, "cpu", torch.float32)
        self.said = {}
        self.next = 1

    def cell(self, gi, e, page, off):
        grp = self.m.groups[gi]
        if grp.need.bits == 8:
            return grp.kv[e][page, 0, 0, off], 0
        return grp.kv[e].view(grp.pool.num_pages, -1, grp.need.head_dim)[page, off], 0

    def append(self, req, n):
        if not self.m.has(req):
            self.m.admit(req)
            self.said[req] = []
        slots = self.m.append(req, n)
        start = len(self.said[req])
        ids = [self.next + i for i in range(n)]
        self.next += n
        self.said[req] += ids
        for gi, sl in slots.items():
            for e in self.m.groups[gi].entries:
                for i, s in enumerate(sl):
                    if s >= 0:
                        row, at = self.cell(gi, e, s // self.m.page_size, s % self.m.page_size)
                        row[at] = (ids[i] % 251) if self.m.groups[gi].need.bits == 8 else ids[i]
        for grp in self.m.groups:
            for t in grp.state_tensors():
                t[self.m.slot_of(req)] = ids[-1]
        assert len(self.said[req]) == start + n

    def fork(self, req, children):
        self.m.fork(req, children, copy)
        for c in children:
            self.said[c] = list(self.said[req])

    def release(self, req):
        self.m.release(req)
        del self.said[req]

    def check(self):
        self.m.check_invariants()
        for req, ids in self.said.items():
            assert self.m.tokens_of(req) == len(ids)
            for gi, grp in enumerate(self.m.groups):
                for t in grp.state_tensors() if ids else ():
                    assert (t[self.m.slot_of(req)] == ids[-1]).all()
                if not grp.paged:
                    continue
                table = self.m.block_table(req, gi)
                kind, ps = grp.need.kind, self.m.page_size
                if kind == "summary":
                    at = {i // grp.need.window: ids[i] for i in range(len(ids)) if (i + 1) % grp.need.window == 0}
                else:
                    first = 0
                    if kind == "window":
                        first = max(0, len(ids) - grp.need.window)
                    if kind == "chunk":
                        first = (len(ids) - 1) // grp.need.window * grp.need.window if ids else 0
                    at = {i: ids[i] for i in range(len(ids)) if i >= first or (kind == "window" and i < grp.need.keep_first)}
                for i, want in at.items():
                    for e in grp.entries:
                        row, o = self.cell(gi, e, table[i // ps], i % ps)
                        assert int(row[o]) == (want % 251 if grp.need.bits == 8 else want), (req, gi, i)


ENTRIES = {"full": {0: FULL, 1: FULL}, "bits8": {0: FULL8}, "window": {0: WINDOW, 1: FULL}, "chunk": {0: CHUNK, 3: STATE}, "pooled": {0: POOLED, -1: STATE}}


@pytest.mark.parametrize("kind", ENTRIES)
def test_random_lives(kind):
    rng = random.Random(kind)
    c = Content(ENTRIES[kind])
    names = iter(range(10 ** 6))
    for step in range(400):
        do = rng.choice(["append", "append", "append", "new", "fork", "release", "compact", "resize"])
        live = list(c.said)
        try:
            if do == "new" or not live:
                c.append(next(names), rng.randint(1, 50))
            elif do == "append":
                c.append(rng.choice(live), rng.choice([1, 1, 2, 16, 33]))
            elif do == "fork":
                c.fork(rng.choice(live), [next(names) for _ in range(rng.randint(1, 3))])
            elif do == "release":
                c.release(rng.choice(live))
            elif do == "compact":
                c.m.compact(copy)
                for grp in c.m.groups:
                    if grp.paged:
                        assert all(grp.pool.holders(p) == 0 for p in range(grp.pool.used_pages, grp.pool.num_pages))
            else:
                c.m.resize(rng.randint(20, 70), copy)
        except (OutOfPages, OutOfSlots, ValueError) as e:
            if isinstance(e, ValueError):
                assert "the limit is" in str(e)
            for r in list(c.m.live_requests()):
                if r not in c.said or (not c.said[r] and c.m.tokens_of(r) == 0):
                    c.m.release(r)
                    c.said.pop(r, None)
            if c.said and rng.random() < 0.5:
                c.release(rng.choice(list(c.said)))
        c.check()
    for r in list(c.said):
        c.release(r)
    c.check()
    assert all(not g.paged or g.pool.used_pages == 0 for g in c.m.groups)


def test_a_fork_shares_its_full_pages():
    c = Content({0: FULL, 1: FULL}, page_size=16)
    c.append("a", 35)
    c.fork("a", ["b", "c"])
    tables = [c.m.block_table(r, 0) for r in "abc"]
    assert tables[0][:2] == tables[1][:2] == tables[2][:2] and len({t[2] for t in tables}) == 3
    assert c.m.groups[0].pool.used_pages == 5
    c.append("b", 20)
    c.append("a", 1)
    c.release("a")
    c.check()
    c.append("d", 32)
    c.fork("d", ["e"])               # at a page's end there is nothing to copy
    assert c.m.block_table("e", 0) == c.m.block_table("d", 0)
    c.append("d", 3)
    c.append("e", 3)
    c.check()


def test_a_fork_that_does_not_fit_changes_nothing():
    c = Content({0: FULL}, pages=4, max_requests=3)
    c.append("a", 35)
    with pytest.raises(OutOfPages):
        c.fork("a", ["b", "c"])
    with pytest.raises(OutOfSlots):
        c.fork("a", ["b", "c", "d"])
    for bad in (["a"], ["b", "b"]):
        with pytest.raises(ValueError):
            c.fork("a", bad)
    with pytest.raises(KeyError):
        c.fork("x", ["b"])
    c.check()
    assert c.m.free_slots() == 2 and c.m.groups[0].pool.free_pages == 1
    c.fork("a", [])
    c.fork("a", ["b"])
    c.check()


def test_a_request_that_has_not_begun_is_forked():
    m = CacheManager({0: POOLED, 1: STATE}, 16, 8, 4, 64, "cpu", torch.float32)
    for grp in m.groups:
        for t in grp.state_tensors():
            t.fill_(7)
    m.admit("a")
    m.fork("a", ["b"], copy)
    assert (m.groups[m.entry_group[1]].state[1][m.slot_of("b")] == 0).all()
    m.append("b", 3)
    m.check_invariants()


def test_pages_that_a_sibling_holds_do_not_come_back():
    m = CacheManager({0: CacheNeed(kind="window", kv_heads=1, head_dim=16, window=16)}, 16, 4, 4, 200, "cpu", torch.float32)
    m.admit("a")
    m.append("a", 48)
    m.fork("a", ["b"], copy)
    assert m.pages_needed("a", 1)[0] == 1            # its first pages are the other's too
    m.append("a", 1)
    with pytest.raises(OutOfPages):
        m.append("b", 33)
    m.check_invariants()
    m.release("b")
    m.append("a", 40)
    m.check_invariants()


def test_pool_compacts_and_changes_its_size():
    p = PagePool(10)
    a = p.take(8)
    for x in (0, 2, 5):
        p.give_back(x)
    p.share(7)
    moves = p.compact()
    assert moves == {6: 0, 7: 2} or moves == {6: 0, 7: 2, 5: 5}
    assert p.holders(moves[7]) == 2 and p.used_pages == 5 and p.take(1) == [5]
    p.check()
    with pytest.raises(OutOfPages):
        p.resize(5)
    p.resize(6)
    assert p.free_pages == 0
    p.resize(20)
    assert p.take(14) == list(range(6, 20))
    p.check()
    assert len(a) == 8


def test_resize_refuses_less_than_is_held():
    c = Content({0: FULL8}, pages=10)
    c.append("a", 60)
    with pytest.raises(OutOfPages):
        c.m.resize(3, copy)
    c.m.resize(4, copy)
    assert c.m.groups[0].kv[0].shape[0] == c.m.groups[0].words[0].shape[0] == 4
    c.check()


class NoMemory(RuntimeError):
    pass


def no_memory(monkeypatch, good, after=10 ** 9):
    """Of the next allocations the first ``good`` succeed, those behind them do not, from ``after`` on they do again."""
    real, count = torch.zeros, [0]

    def zeros(*args, **kwargs):
        count[0] += 1
        if good < count[0] <= after:
            raise NoMemory(f"allocation {count[0]}")
        return real(*args, **kwargs)
    monkeypatch.setattr(torch, "zeros", zeros)


@pytest.mark.parametrize("recovers", [False, True])
@pytest.mark.parametrize("pages", [12, 90])
@pytest.mark.parametrize("good", range(6))
@pytest.mark.parametrize("kind", ["full", "bits8", "window", "pooled"])
def test_a_resize_without_memory_leaves_a_whole_cache(kind, good, pages, recovers):
    """Whichever tensor there is no memory for: pools and tensors agree, requests hold what they held and go on, and a later resize works.  Where
    there is memory to go back, the number of pages is the old one."""
    c = Content(ENTRIES[kind] | ({2: FULL8} if kind == "full" else {}))
    c.append("x", 20)
    c.append("a", 60)
    c.append("b", 33)
    c.release("x")
    before = {gi: grp.pool.num_pages for gi, grp in enumerate(c.m.groups) if grp.paged}
    want = c.m.pages_after_resize(pages)
    with pytest.MonkeyPatch.context() as patch:
        no_memory(patch, good, good + 1 if recovers else 10 ** 9)
        if good >= sum(len(g.page_tensors()) for gi, g in enumerate(c.m.groups) if g.paged and want[gi] != before[gi]):
            c.m.resize(pages, copy)
            before = want
        else:
            with pytest.raises(NoMemory):
                c.m.resize(pages, copy)
    for gi, n in before.items():
        grp = c.m.groups[gi]
        assert grp.pool.num_pages in ((n,) if recovers else (n, min(n, want[gi])))
        assert {t.shape[0] for t in grp.page_tensors()} == {grp.pool.num_pages} and all(t.is_contiguous() for t in grp.page_tensors())
    c.check()
    c.append("a", 40)
    c.fork("a", ["d"])
    c.append("d", 3)
    c.check()
    c.m.resize(40, copy)
    c.check()
    assert all(grp.pool.num_pages == t.shape[0] for grp in c.m.groups if grp.paged for t in grp.page_tensors())


def test_pages_that_a_window_has_passed_are_counted_without_a_look_at_each():
    """A long request's blocks below the window are nearly all given back; planning a step asks the pool about those that are still held."""
    m = CacheManager({0: CacheNeed(kind="window", kv_heads=1, head_dim=16, window=40)}, 16, 30, 3, 20000, "cpu", torch.float32, allocate=False)
    m.admit("a")
    for _ in range(19000 // 38):
        m.append("a", 38)
    looked_at = []

    class Blocks(np.ndarray):
        def tolist(self):
            looked_at.append(self.size)
            return super().tolist()
    have = m.tokens_of("a")
    first = max(0, have - 39) // 16
    alone = sum(p >= 0 for p in m.block_table("a", 0)[:first])
    table = m._requests["a"].tables[0]
    table.pages = table.pages.view(Blocks)
    assert m.pages_needed("a", 38)[0] == -(-(have + 38) // 16) - -(-have // 16) - alone
    assert sum(looked_at) == alone > 0 and first > 1000
    m.fork("a", ["b"], copy)
    assert m.pages_needed("a", 38)[0] == -(-(have + 38) // 16) - -(-have // 16)
    m.check_invariants()
