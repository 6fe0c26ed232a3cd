"""The accepted path of drafted trees and its cache rows against the same by loops."""
import random

import pytest
import torch

from draft_helpers import ancestor_sets, plain_accept, random_tree
from spite_b200.kernels.api import KernelError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def kernels():
    from spite_b200.kernels.cuda import CudaKernels
    return {t: CudaKernels(t, DEV) for t in (torch.float32, torch.bfloat16)}


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def check(kernels, counts, *, dtype=torch.bfloat16, shapes=((2, 2, 2, 16, 64),), depth=None, seed=0, chain=False, vocab=3, holes=False, slots=True, alias=False,
          keep=0):
    """`shapes`: (caches, planes, kv heads, page size, head size) of every group; a small vocabulary makes paths long."""
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    S, M = len(counts), sum(counts)
    trees = [list(range(-1, n - 1)) if chain else random_tree(r, n, r.random() < 0.3) for n in counts]
    parents = [p for t in trees for p in t]
    tokens, targets = [r.randrange(vocab) for _ in range(M)], [r.randrange(vocab) for _ in range(M)]
    for t, a in zip(trees, [sum(counts[:s]) for s in range(S)]):          # the targets lead to some node, unless a sibling in front of the way takes over
        at = max((i for i, up in enumerate(ancestor_sets(t)) if 0 in up and r.random() < 0.7), default=0)
        while t and 0 <= t[at] < at:
            targets[a + t[at]] = tokens[a + at]
            at = t[at]
    depth = depth or max(counts + [1])
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    want = plain_accept(tokens, None if chain else parents, targets, cu, depth)
    caches, expect = [], []
    for n, planes, heads, page, size in shapes:
        pages = -(-M // page) + S + 1
        places = torch.randperm(pages * page, generator=g)[:M]
        kv = torch.randn(n, planes, pages, heads, page, size, generator=g).to(dtype)
        scales = torch.randn(n, pages, heads, page, generator=g) if planes == 1 else None
        if holes:
            places[torch.rand(M, generator=g) < 0.2] = -1
            places[torch.rand(M, generator=g) < 0.1] = pages * page + 5
        after, after_s = kv.clone(), None if scales is None else scales.clone()
        for s in range(S):
            for d in range(want[0][s]):
                a, b = int(places[cu[s] + want[1][s][d]]), int(places[cu[s] + d])
                if min(a, b) >= 0 and max(a, b) < pages * page and want[1][s][d] != d:
                    after[:, :, b // page, :, b % page] = kv[:, :, a // page, :, a % page]
                    if scales is not None:
                        after_s[:, b // page, :, b % page] = scales[:, a // page, :, a % page]
        caches.append((kv.to(DEV), places.to(DEV), None if scales is None else scales.to(DEV)))
        expect.append((after, after_s))
    rows = S + 2
    order = r.sample(range(rows), S) if slots else list(range(S))
    lengths = [r.randrange(1000) for _ in range(rows)]
    got_len = ints(lengths) if alias else torch.full((rows,), -5, dtype=torch.int32, device=DEV)
    out = dict(counts=ints([-3] * S), path=ints([[-3] * depth] * S), emitted=ints([[-3] * depth] * S))
    kernels[dtype].accept_drafts(ints(tokens), None if chain else ints(parents), ints(targets), ints(cu), caches, **out, slots=ints(order) if slots else None,
                                 lengths=got_len if alias else ints(lengths), lengths_out=got_len)
    assert out["counts"].tolist() == want[0] and out["path"].tolist() == want[1] and out["emitted"].tolist() == want[2]
    right = list(lengths) if alias else [-5] * rows
    for s, row in enumerate(order):
        right[row] = lengths[row] + want[0][s]
    assert got_len.tolist() == right
    for (kv, _, scales), (after, after_s) in zip(caches, expect):
        assert torch.equal(kv.cpu(), after)
        assert scales is None or torch.equal(scales.cpu(), after_s)
    return want


@pytest.mark.parametrize("counts", [[1], [2], [0, 3, 0], [8], [33, 1, 64, 7], [5] * 70, [1024], [300, 1000]])
def test_trees(kernels, counts):
    found = [max(check(kernels, counts, seed=s, vocab=v)[0]) for s, v in ((1, 2), (2, 3), (3, 50), (4, 100000), (5, 100000))]
    assert max(counts) < 8 or max(found) > 2                   # (of the plain form: that the cases follow paths at all)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shapes", [
    ((1, 2, 1, 1, 1),), ((3, 2, 5, 7, 3),), ((1, 1, 2, 16, 24),), ((48, 2, 8, 64, 128),), ((2, 2, 2, 64, 128), (5, 1, 1, 16, 64), (1, 2, 3, 32, 2)),
])
def test_caches(kernels, dtype, shapes):
    """Rows of a few bytes and of many, keys alone with their factors, several groups with slot maps of their own."""
    check(kernels, [20, 40, 13], dtype=dtype, shapes=shapes, seed=4, vocab=2)


def test_chains_and_limits(kernels):
    check(kernels, [40, 9, 70], chain=True, vocab=2, seed=3)
    check(kernels, [1024], chain=True, vocab=1, seed=3)        # everything is right: nothing moves
    check(kernels, [30, 60], vocab=1, depth=4, seed=5)
    check(kernels, [30, 60], vocab=1, depth=1, seed=5)
    check(kernels, [30, 60], vocab=2, slots=False, alias=True, seed=6)


def test_rows_without_a_place(kernels):
    for seed in range(4):
        check(kernels, [50, 60, 10], vocab=1, holes=True, seed=seed)


def test_without_caches_and_lengths(kernels):
    out = dict(counts=ints([0]), path=ints([[0, 0, 0]]), emitted=ints([[0, 0, 0]]))
    kernels[torch.float32].accept_drafts(ints([7, 8, 8]), ints([-1, 0, 0]), ints([8, 5, 6]), ints([0, 3]), [], **out)
    assert out["counts"].tolist() == [2] and out["path"].tolist() == [[0, 1, -1]] and out["emitted"].tolist() == [[8, 5, -1]]


def test_beyond_32_bits(kernels):
    """A cache of more than 2^32 bytes whose accepted rows lie at its far end."""
    kv = torch.zeros((1, 2, 150000, 1, 64, 128), dtype=torch.bfloat16, device=DEV)       # 2.4 GB a plane
    last = 150000 * 64 - 1
    kv[0, :, -1, 0, 63] = 3.0
    out = dict(counts=ints([0]), path=ints([[0, 0]]), emitted=ints([[0, 0]]))
    kernels[torch.bfloat16].accept_drafts(ints([7, 9, 8]), ints([-1, 0, 0]), ints([8, 5, 6]), ints([0, 3]), [(kv, ints([last - 2, last - 1, last], torch.int64), None)], **out)
    assert out["path"].tolist() == [[0, 2]]
    assert (kv[0, :, -1, 0, 62:] == 3.0).all() and int((kv != 0).sum()) == 2 * 2 * 128


def test_refusals(kernels):
    k = kernels[torch.bfloat16]
    kv = torch.zeros((1, 2, 2, 1, 16, 8), dtype=torch.bfloat16, device=DEV)
    base = dict(tokens=ints([1, 2]), parents=ints([-1, 0]), targets=ints([2, 3]), cu_seqlens=ints([0, 2]), caches=[(kv, ints([0, 1], torch.int64), None)],
                counts=ints([0]), path=ints([[0, 0]]), emitted=ints([[0, 0]]), slots=ints([0]), lengths=ints([0]), lengths_out=ints([0]))

    def call(**kw):
        a = {**base, **kw}
        first = [a.pop(n) for n in ("tokens", "parents", "targets", "cu_seqlens", "caches")]
        k.accept_drafts(*first, **a)
    for kw in (dict(tokens=ints([1, 2], torch.int64)), dict(targets=ints([1])), dict(parents=ints([-1])), dict(counts=ints([0, 0])), dict(path=ints([[0]])),
               dict(emitted=ints([[0, 0, 0]])), dict(lengths=None), dict(lengths_out=ints([0, 0])), dict(slots=ints([0, 1])), dict(cu_seqlens=ints([0])),
               dict(caches=[(kv.float(), ints([0, 1], torch.int64), None)]), dict(caches=[(kv[0], ints([0, 1], torch.int64), None)]),
               dict(caches=[(kv, ints([0, 1]), None)]), dict(caches=[(kv, ints([0], torch.int64), None)]), dict(caches=base["caches"] * 9),
               dict(caches=[(kv, ints([0, 1], torch.int64), torch.zeros(3, device=DEV))]), dict(tokens=torch.tensor([1, 2], dtype=torch.int32))):
        with pytest.raises(KernelError):
            call(**kw)
    call()
    assert base["counts"].tolist() == [2]
