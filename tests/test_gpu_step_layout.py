"""Steps laid out on the device against the same by loops and against the host's cache manager."""
import random

import pytest
import torch

from draft_helpers import plain_layout, random_tree
from spite_b200.cache import CacheManager, Window
from spite_b200.cache.manager import GroupKey
from spite_b200.kernels.api import KernelError, PageTables, StepLayout

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def k():
    from spite_b200.kernels.cuda import CudaKernels
    return CudaKernels(torch.bfloat16, DEV)


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


class State:
    """Pages of R rows on the device and the same as lists."""

    def __init__(self, rows, width, page, window, n_pages, seed=0, pool=True):
        self.page, self.window, self.width = page, window, width
        self.tables, self.held = [[-1] * width for _ in range(rows)], [0] * rows
        self.free = list(range(n_pages))
        random.Random(seed).shuffle(self.free)
        self.n_free = n_pages
        self.pages = PageTables(tables=ints(self.tables), held=ints(self.held), page_size=page, window=window, free_pages=ints(self.free) if pool else None,
                                n_free=ints([n_pages]) if pool else None)

    def out(self, S, M, words=0, width=None):
        blank = lambda *shape, dtype=torch.int32: torch.full(shape, -9, dtype=dtype, device=DEV)
        return StepLayout(block_table=blank(S, width or self.width), cu_seqlens=blank(S + 1), positions=blank(M), seg_of_token=blank(M),
                          slot_map=blank(M, dtype=torch.int64), status=blank(1), ancestors=blank(M, words) if words else None)

    def same(self):
        assert self.pages.tables.tolist() == self.tables and self.pages.held.tolist() == self.held
        if self.pages.n_free is not None:
            assert int(self.pages.n_free) == self.n_free
            assert self.pages.free_pages.tolist()[:self.n_free] == self.free[:self.n_free]

    def step(self, k, slots, lengths, new, parents=None, room=0, words=0, width=None):
        total = sum(max(n, 0) for n, s in zip(new, slots) if s >= 0)
        out = self.out(len(slots), total + room, words, width)
        flat = None if parents is None else ints([v for t in parents for v in t] or [0])
        k.layout_step(self.pages, ints(slots), ints(lengths), ints(new), out, parents=flat)
        assert int(out.status) == 0
        n_free, block, cu, pos, seg, slot, sets = plain_layout(
            self.tables, self.held, self.page, self.window, self.free if self.pages.free_pages is not None else None, self.n_free, slots, lengths, new,
            None if parents is None else [v for t in parents for v in t], width or self.width, words)
        self.n_free = n_free
        self.same()
        assert out.block_table.tolist() == block and out.cu_seqlens.tolist() == cu
        for got, want in ((out.positions, pos), (out.seg_of_token, seg), (out.slot_map, slot)):
            assert got.tolist() == want + [-9] * room
        if words:
            assert out.ancestors.tolist() == sets + [[-9] * words] * room
        return out


WINDOWS = [Window("full"), Window("sliding", 1), Window("sliding", 37), Window("chunk", 48), Window("chunk", 7)]


@pytest.mark.parametrize("window", WINDOWS, ids=lambda w: f"{w.kind}{w.size}")
@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_many_steps(k, page, window):
    """Requests come, grow by trees, single tokens and portions, stand still, end: as the loops have it after every step."""
    r = random.Random(page + window.size)
    rows, most = 9, 400
    st = State(rows, -(-most // page), page, window, rows * -(-most // page), seed=page)
    lengths = [0] * rows
    ended = [False] * rows
    for step in range(25):
        slots = r.sample(range(rows), r.randint(1, rows))
        trees = step % 3 != 2
        new = []
        for s in slots:
            if r.random() < 0.12 and st.held[s]:
                new.append(-1)
            else:
                new.append(min(r.choice([0, 1, 1, 5, 40, 65]), most - lengths[s]))
        if r.random() < 0.4:
            slots, new = slots + [-1], new + [r.randint(0, 5)]
        parents = [random_tree(r, max(n, 0) if s >= 0 else 0, r.random() < 0.3) for s, n in zip(slots, new)] if trees else None
        words = 3 if trees or r.random() < 0.5 else 0
        st.step(k, slots, lengths, new, parents, room=r.randint(0, 3), words=words)
        st.step(k, slots, lengths, new, parents, words=words)              # once more: takes nothing further
        for s, n in zip(slots, new):
            if s >= 0:
                lengths[s] = 0 if n < 0 else lengths[s] + r.randint(min(1, n), n)


@pytest.mark.parametrize("window", WINDOWS, ids=lambda w: f"{w.kind}{w.size}")
def test_same_pages_as_the_cache_manager(k, window):
    """Driven in the same order, the device's stack hands out the pages that the host's pool does."""
    page, rows, n_pages = 16, 5, 90
    mgr = CacheManager([GroupKey(window, 1, 64)], page, n_pages, rows)
    st = State(rows, 40, page, window, n_pages)
    st.free = list(range(n_pages - 1, -1, -1))                # (as the pool stacks them)
    st.pages.free_pages.copy_(ints(st.free))
    lengths, r = [0] * rows, random.Random(3)
    for step in range(30):
        live = [s for s in range(rows) if s in mgr.requests]
        ends = [s for s in live if r.random() < 0.1]
        slots = sorted(set(ends + r.sample(range(rows), 3)))
        new = [-1 if s in ends else min(r.choice([1, 1, 17, 30]), 600 - lengths[s]) for s in slots]
        for s in ends:
            mgr.release(s)
        order = [s for s in slots if s in ends] + [s for s in slots if s not in ends]        # (the manager gives back before it takes)
        new = [new[slots.index(s)] for s in order]
        out = st.step(k, order, lengths, new)
        for s, n in zip(order, new):
            if n > 0:
                if s not in mgr.requests:
                    mgr.admit(s)
                mgr.reserve(s, n)
        for i, (s, n) in enumerate(zip(order, new)):
            if n > 0:
                table = mgr.block_table(s, 0)
                assert out.block_table[i].tolist()[:len(table)] == table
                lengths[s] += n
            elif n < 0:
                lengths[s] = 0
        # the manager frees what a window has passed when the step has run, the device when the next step of the request is laid out
        for s, n in zip(order, new):
            if n > 0:
                mgr.commit(s)
        st2 = State.out(st, 1, 1)
        for s in [x for x, n in zip(order, new) if n > 0]:
            k.layout_step(st.pages, ints([s]), ints(lengths), ints([0]), st2)
            st.n_free = plain_layout(st.tables, st.held, page, window, st.free, st.n_free, [s], lengths, [0], None, 40, 0)[0]
        st.same()
        assert st.n_free == mgr.free_pages()[0]


@pytest.mark.parametrize("S", [1, 31, 33, 1023, 1024, 1025, 4096])
def test_many_requests(k, S):
    r = random.Random(S)
    page = 16
    st = State(S + 3, 6, page, Window("sliding", 20), 6 * S + 20, seed=S)
    lengths = [0] * (S + 3)
    slots = r.sample(range(S + 3), S)
    for _ in range(3):
        new = [-1 if r.random() < 0.05 and st.held[s] else min(r.choice([0, 1, 3, 17]), 90 - lengths[s]) for s in slots]
        st.step(k, slots, lengths, new, words=1, room=2)
        for s, n in zip(slots, new):
            lengths[s] = 0 if n < 0 else lengths[s] + n


def test_long_requests_and_deep_trees(k):
    """A portion of thousands of tokens beside the deepest and the widest tree."""
    st = State(3, 2100, 64, Window("full"), 6400, seed=1)
    st.step(k, [0, 1, 2], [0, 0, 0], [60000, 5, 131])
    lengths = [60000, 3, 131]
    trees = [list(range(-1, 1023)), [-1] + [0] * 1023, [-1, -1, -1]]
    st.step(k, [2, 0, 1], lengths, [3, 1024, 1024], [trees[2], trees[0], trees[1]], words=32)
    st.step(k, [2, 0], [131000, 130000, 131], [1, -1], words=1)


def test_tables_without_a_stack(k):
    """Tables that the host keeps: nothing is given back or taken."""
    st = State(4, 8, 16, Window("sliding", 16), 1, pool=False)
    st.tables = [[5, 6, 7, -1, -1, -1, -1, -1], [-1, 1, 2, 3, -1, -1, -1, -1], [-1] * 8, [9, -1, -1, -1, -1, -1, -1, -1]]
    st.held = [3, 4, 0, 1]
    st.pages.tables.copy_(ints(st.tables))
    st.pages.held.copy_(ints(st.held))
    st.step(k, [1, 0, 3, 2, -1], [40, 60, 0, 16], [4, 8, 0, 0, 3], [random_tree(random.Random(1), n) for n in (4, 8, 0, 0, 0)], words=1, width=4)
    out = st.out(1, 20)
    k.layout_step(st.pages, ints([0]), ints([40, 60, 0, 16]), ints([9]), out)         # a page short
    assert int(out.status) == StepLayout.MALFORMED
    st.same()


def test_a_step_that_cannot_be_laid_out_changes_nothing(k):
    st = State(4, 8, 16, Window("sliding", 20), 10, seed=2)
    lengths = [50, 0, 20, 0]
    st.step(k, [0, 2], [0, 0, 0, 0], [50, 20])                # 4 + 2 of 10 pages
    bad, few = StepLayout.MALFORMED, StepLayout.OUT_OF_PAGES

    def refused(slots, new, status, *, lengths=lengths, parents=None, M=200, words=0, width=8):
        out = st.out(len(slots), M, words, width)
        k.layout_step(st.pages, ints(slots), ints(lengths), ints(new), out, parents=None if parents is None else ints(parents))
        assert int(out.status) == status
        st.same()
        assert out.cu_seqlens.tolist() == [0] * (len(slots) + 1) and (out.block_table == -1).all()
        assert (out.positions == -9).all() and (out.slot_map == -9).all()

    refused([1, 3], [60, 40], few)                            # 7 pages, 4 are free, and the window of nobody in the step has passed one
    refused([0, 1, 3], [1, 64, 30], few)                      # (row 0 gives one back: 5, but 6 are needed)
    refused([1, 1], [1, 1], bad)                              # a row twice
    refused([1, 4], [1, 1], bad)
    refused([-2], [1], bad)
    refused([1], [-2], bad)
    refused([0], [1], bad, lengths=[65, 0, 0, 0])             # longer than its pages
    refused([0], [1], bad, lengths=[-1, 0, 0, 0])
    refused([1], [129], bad)                                  # more pages than a row has
    refused([0], [20], bad, width=4)                          # more pages than the step's table has
    refused([0, 1], [1, 5], bad, M=5)                         # more tokens than room
    refused([1], [5], bad, parents=[-1, 0])                   # fewer parents than tokens
    refused([1], [33], bad, words=1)                          # more tokens than bits
    refused([1], [2147483647], bad)
    refused([0], [2147483647], bad)
    for n in (-1, 11):
        st.pages.n_free.fill_(n)
        out = st.out(1, 4)
        k.layout_step(st.pages, ints([1]), ints(lengths), ints([1]), out)
        assert int(out.status) == bad and int(st.pages.n_free) == n
    st.pages.n_free.fill_(st.n_free)
    st.step(k, [0, 1], lengths, [1, 64])                      # and goes on: 1 back, 4 taken


def test_parents_that_point_forward(k):
    """A parent that is not smaller is none."""
    st = State(1, 8, 16, Window("full"), 8)
    out = st.out(1, 5, 1)
    k.layout_step(st.pages, ints([0]), ints([0]), ints([5]), out, parents=ints([7, 0, 2, 1, -5]))
    assert out.positions.tolist() == [0, 1, 0, 2, 0] and out.ancestors[:, 0].tolist() == [1, 3, 4, 11, 0] and int(out.slot_map[4]) == -1


def test_in_a_graph(k):
    st = State(3, 20, 16, Window("full"), 60)
    slots, lengths, new, out = ints([2, 0]), ints([0, 0, 0]), ints([5, 3]), st.out(2, 40, 2)
    call = lambda: k.layout_step(st.pages, slots, lengths, new, out, parents=None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    st.n_free = plain_layout(st.tables, st.held, 16, st.window, st.free, st.n_free, [2, 0], [0] * 3, [5, 3], None, 20, 0)[0]
    have = [0, 0, 0]
    for n in ([30, 1], [4, 17], [-1, 2]):
        have = [have[0] + 3, 0, have[2] + 5]
        lengths.copy_(ints(have))
        new.copy_(ints(n))
        graph.replay()
        torch.cuda.synchronize()
        st.n_free = plain_layout(st.tables, st.held, 16, st.window, st.free, st.n_free, [2, 0], have, n, None, 20, 0)[0]
        st.same()
        assert int(out.status) == 0


def test_refusals(k):
    st = State(3, 4, 16, Window("full"), 12)
    slots, lengths, new = ints([0, 1]), ints([0, 0, 0]), ints([1, 1])
    good = lambda: st.out(2, 8, 1)
    for change in (dict(slots=slots.long()), dict(lengths=ints([0, 0])), dict(new=ints([1])), dict(slots=ints([[0, 1]])), dict(slots=ints([]), new=ints([]))):
        a = {**dict(slots=slots, lengths=lengths, new=new), **change}
        with pytest.raises(KernelError):
            k.layout_step(st.pages, a["slots"], a["lengths"], a["new"], good())
    for name, value in (("slot_map", ints([0] * 8)), ("positions", ints([0] * 7)), ("status", ints([0, 0])), ("cu_seqlens", ints([0] * 2)),
                        ("block_table", ints([[0]])), ("ancestors", ints([0] * 8)), ("ancestors", ints([[0]] * 4))):
        out = good()
        setattr(out, name, value)
        with pytest.raises(KernelError):
            k.layout_step(st.pages, slots, lengths, new, out)
    keep = st.pages.n_free
    for value in (None, ints([1, 2])):
        st.pages.n_free = value
        with pytest.raises(KernelError):
            k.layout_step(st.pages, slots, lengths, new, good())
    st.pages.n_free = keep
    with pytest.raises(KernelError):
        k.layout_step(st.pages, slots, lengths, new, st.out(2, 8, 33))
    st.same()
