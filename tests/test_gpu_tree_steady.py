"""Attention of drafted trees: a row's bits are its own, whatever lies beside it and how often it is asked for, and whatever other host threads call."""
import threading

import pytest
import torch

from draft_helpers import TreeCase
from spite_b200.cache import Window
from test_gpu_tree_attention import kernels, run  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
FULL = Window("full")


def call(k, case, out=None, **more):
    q, batch, cache = case.step(DEV)
    out = torch.zeros_like(q) if out is None else out
    k.tree_attention(q, out, batch, cache, num_heads=case.heads, window=FULL, softmax_scale=case.size ** -0.5, **more)
    return out


@pytest.mark.parametrize("dtype,heads,size", [(BF, 5, 128), (BF, 5, 64), (BF, 8, 64), (F32, 5, 64)])
@pytest.mark.parametrize("slopes", [False, True], ids=["cap", "cap and slopes"])
def test_a_capped_row_depends_on_itself_alone(kernels, dtype, heads, size, slopes):  # noqa: F811
    """Other rows of its warp (siblings, the next request's, rows that are no node's) and rows of the cache that it does not see change no bit of a row."""
    k = kernels[dtype]
    more = dict(score_softcap=4.0)
    if slopes:
        more["head_slopes"] = (torch.arange(heads, dtype=F32) / 16).to(DEV)
    case = TreeCase([200, 70], [9, 30], heads=heads, kv_heads=1, size=size, dtype=dtype, seed=2, padding=True, scale=0.5)
    case.kv = torch.nan_to_num(case.kv, nan=0.0)              # (padding rows and what lies behind: any numbers)
    first = call(k, case, **more).clone()
    assert torch.isfinite(first).all()
    for _ in range(3):                                       # other launches in between leave other numbers in shared memory
        call(k, TreeCase([300], [25], heads=heads, kv_heads=1, size=size, dtype=dtype, seed=3, scale=30.0))
        assert torch.equal(call(k, case, **more), first)
    keep = case.q.clone()
    for row in (1, 8, 9, 12):                                # one row louder: all others as before
        case.q[row] *= 100
        rest = [i for i in range(case.M) if i != row]
        assert torch.equal(call(k, case, **more)[rest], first[rest])
        case.q.copy_(keep)
    for s in range(2):
        for j in range(case.lens[s] + case.counts[s], len(case.table[s]) * 64):
            if int(case.table[s, j // 64]) >= 0:
                case.kv[:, int(case.table[s, j // 64]), :, j % 64] = 1000.0
        for i in range(case.counts[s]):
            if i not in case.sets[s][i]:
                j = case.lens[s] + i
                case.kv[:, int(case.table[s, j // 64]), :, j % 64] = -1000.0
    assert torch.equal(call(k, case, **more), first)


@pytest.mark.parametrize("dtype,size", [(BF, 128), (BF, 48), (F32, 64), (F32, 200)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_is_not_finite_changes_no_other_row(kernels, dtype, size, value):  # noqa: F811
    """A query, or a drafted node's key, that is not finite: rows that do not see it keep their bits."""
    k = kernels[dtype]
    case = TreeCase([300, 70], [9, 30], heads=4, kv_heads=2, size=size, dtype=dtype, seed=2, trees=[[-1, 0, 0, 1, 2, 3, 3, 4, 4], list(range(-1, 29))])
    first = call(k, case).clone()
    assert torch.isfinite(first).all()
    for row in (0, 5, 20):
        keep = case.q[row].clone()
        case.q[row, 7] = value
        rest = [i for i in range(case.M) if i != row]
        got = call(k, case)
        assert torch.equal(got[rest], first[rest]) and not torch.isfinite(got[row]).all()
        case.q[row] = keep
    j = 300 + 1                                              # node 1 of the first tree, seen by 1, 3, 5 and 6
    case.kv[0, int(case.table[0, j // 64]), :, j % 64, 5] = float("nan")
    got = call(k, case)
    rest = [i for i in range(case.M) if i not in (1, 3, 5, 6)]
    assert torch.equal(got[rest], first[rest]) and torch.isnan(got[[1, 3, 5, 6]]).all()


@pytest.mark.parametrize("dtype,heads,size", [(BF, 8, 128), (BF, 4, 64), (F32, 4, 64)])
def test_requests_of_several_launches_with_shared_items(kernels, dtype, heads, size):  # noqa: F811
    """1,500 requests (640 a launch), long ones in every launch, whose keys are shared among blocks: the launches use one scratch one after the other."""
    lens = [5000 if s in (3, 700, 1290) else 9000 if s in (639, 640, 1499) else s % 3 for s in range(1500)]
    counts = [20 if n > 100 else s % 2 for s, n in enumerate(lens)]
    case = TreeCase(lens, counts, heads=heads, kv_heads=1, size=size, dtype=dtype, seed=8)
    out = run(kernels, case)
    for _ in range(3):
        assert torch.equal(call(kernels[dtype], case), out)


def test_launches_are_counted(kernels):  # noqa: F811
    k = kernels[BF]

    def launches(case):
        before = k.launches_by_library["attention_tree_tc"]
        call(k, case)
        return k.launches_by_library["attention_tree_tc"] - before
    assert launches(TreeCase([100], [8], heads=4, kv_heads=1, size=64, dtype=BF)) == 1           # (two pages: nothing is shared)
    assert launches(TreeCase([1000], [8], heads=4, kv_heads=1, size=64, dtype=BF)) == 2
    assert launches(TreeCase([10] * 641, [1] * 641, heads=4, kv_heads=1, size=64, dtype=BF)) == 2
    assert launches(TreeCase([10] * 640 + [1000], [1] * 641, heads=4, kv_heads=1, size=64, dtype=BF)) == 4


def test_launches_are_counted(kernels):  # noqa: F811
    k = kernels[BF]

    def launches(lens, counts, width=None):
        before = k.launches_by_library["attention_tree_tc"]
        call(k, TreeCase(lens, counts, heads=4, kv_heads=1, size=64, dtype=BF, width=width))
        return k.launches_by_library["attention_tree_tc"] - before
    assert launches([100], [8]) == 1                          # (two pages: nothing is shared, nothing is joined)
    assert launches([1000], [8]) == 2
    assert launches([10] * 641, [1] * 641) == 2               # (640 requests a launch)
    assert launches([10] * 641, [1] * 641, width=20) == 4


@pytest.mark.parametrize("dtype,shapes", [(BF, [(600, 64, 64), (1, 64, 64)]), (F32, [(2, 200, 64), (2, 136, 64)]), (F32, [(2, 128, 64), (2, 16, 64)])],
                         ids=["requests", "large heads", "small heads"])
def test_two_host_threads(dtype, shapes):
    """Calls of different sizes from two threads, each with kernels and a stream of its own: a launch's shared memory is not limited by another's."""
    from spite_b200.kernels.cuda import CudaKernels
    errors, results = [], [None, None]
    cases = [TreeCase([9] * n, [2] * n, heads=2, kv_heads=1, size=size, page=page, dtype=dtype, seed=n + size) for n, size, page in shapes]
    ks = [CudaKernels(dtype, DEV) for _ in cases]
    want = [call(k, c).clone() for k, c in zip(ks, cases)]
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def work(i):
        try:
            q, batch, cache = cases[i].step(DEV)
            out = torch.zeros_like(q)
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            start.wait(timeout=60)
            with torch.cuda.stream(stream):
                for _ in range(3000):
                    ks[i].tree_attention(q, out, batch, cache, num_heads=2, window=FULL, softmax_scale=cases[i].size ** -0.5)
            stream.synchronize()
            results[i] = out
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for got, right in zip(results, want):
        assert torch.equal(got, right)
