"""NaN, infinities and the largest numbers in queries, keys and values of a step of drafted trees: what a row sees decides what it is, as the formula says.
The float32 kernel has that element by element; on the tensor cores a value that is not finite may reach rows of its request that do not see it."""
import math

import pytest
import torch

from draft_helpers import TreeCase, tolerance
from spite_b200.cache import Window

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
HEADS, KV_HEADS = 4, 2


@pytest.fixture(scope="module")
def kernels():
    from spite_b200.kernels.cuda import CudaKernels
    return {t: CudaKernels(t, DEV) for t in (F32, BF)}


def bits(dtype, value):
    """A number by its bits."""
    return torch.tensor(value, dtype=torch.int64).to(torch.int32).view(F32) if dtype == F32 else torch.tensor(value, dtype=torch.int64).to(torch.int16).view(BF)


# the NaN that the device's arithmetic makes, one with the sign, a quiet one; the largest number
NANS = {F32: (0x7FFFFFFF, 0xFFFFFFFF - (1 << 32), 0x7FC00000), BF: (0x7FFF, 0xFFFF - (1 << 16), 0x7FC0)}
LARGEST = {F32: 0x7F7FFFFF, BF: 0x7F7F}


def formula(case, window, scale, sink=None):
    """(outputs, the same of the values' sizes, the largest score of absolute products) in 64 bits, row by row over what the row sees alone."""
    out = torch.zeros((case.M, HEADS, case.size), dtype=torch.float64)
    size, biggest = torch.zeros_like(out), 0.0
    for s, (have, n) in enumerate(zip(case.lens, case.counts)):
        first = int(case.cu[s])
        for i in range(n):
            pos = [int(p) for p in case.positions[first:first + n]]
            low = window.lowest_visible(pos[i])
            seen = [j for j in range(low, have)] + [have + a for a in sorted(case.sets[s][i]) if pos[a] >= low]
            pages, offs = torch.tensor([int(case.table[s, j // case.page]) for j in seen]), torch.tensor([j % case.page for j in seen])
            for h in range(HEADS):
                k, v = (case.kv[x, pages, h // (HEADS // KV_HEADS), offs].double() for x in (0, -1))
                q = case.q[first + i].view(HEADS, -1)[h].double()
                x = k @ q * scale
                products = (k.abs() @ q.abs()) * scale
                biggest = max([biggest] + [float(p) for p in products if math.isfinite(p)])
                top = x.max()
                if sink is not None:
                    top = torch.maximum(top, torch.tensor(float(sink)).double())
                if top == -math.inf:
                    continue
                w = torch.exp(x - top)
                total = w.sum() + (0.0 if sink is None else math.exp(sink - float(top)))
                out[first + i, h] = (w[:, None] * v).sum(0) / total
                size[first + i, h] = (w[:, None] * v.abs()).sum(0) / total
    return out.view(case.M, -1), size.view(case.M, -1), biggest


def run(kernels, case, window=Window("full"), sink=None, rows=None):
    k, scale = kernels[case.q.dtype], case.size ** -0.5
    q, batch, cache = case.step(DEV)
    out = torch.zeros_like(q)
    k.tree_attention(q, out, batch, cache, num_heads=HEADS, window=window, softmax_scale=scale, sink_logit=sink)
    assert not k.errors()
    want, size, biggest = formula(case, window, scale, sink)
    got = out.double().cpu()
    rows = list(range(case.M)) if rows is None else rows
    got, want, size = got[rows], want[rows], size[rows]
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want)), f"{kind.__name__}: {int(kind(got).sum())} elements, {int(kind(want).sum())} in the formula"
    there = torch.isfinite(want)
    allowed = tolerance(case, want, size, biggest, rounded_weights=True)
    worst = float(((got - want).abs() / allowed)[there].max()) if there.any() else 0.0
    assert worst <= 1.0, f"{worst:.2f} times the allowed error"
    return got


def place(case, s, j):
    """(page, offset) of place j of request s."""
    return int(case.table[s, j // case.page]), j % case.page


def make(dtype, lens=(70, 30, 0), counts=(20, 7, 40), size=64, seed=1):
    return TreeCase(list(lens), list(counts), heads=HEADS, kv_heads=KV_HEADS, size=size, dtype=dtype, seed=seed)


# Of the float32 kernel: one share of the keys; several, of which the joining kernel makes the result; heads of more than 128 elements; of an odd number.
EXACT = [(F32, (70, 30, 0), (20, 7, 40), 64), (F32, (900, 2003, 5), (20, 7, 40), 64), (F32, (130, 61, 0), (9, 33, 2), 200), (F32, (40, 30, 9), (9, 7, 2), 33),
         (BF, (70, 30, 0), (20, 7, 40), 48), (BF, (900, 303, 5), (20, 7, 40), 200)]
# Of the tensor cores' kernel: one row tile a request, the same with its keys shared among blocks, pairs of row tiles.
OTHERS = [(BF, (70, 30, 0), (20, 7, 40), 64), (BF, (9000, 2003, 5), (20, 7, 40), 128), (BF, (900, 300, 5), (90, 140, 70), 64)]
ids = lambda cases: [f"{'fp32' if t == F32 else 'bf16'}-{a[0]}+{n[0]}-{hd}" for t, a, n, hd in cases]
BY_SHAPE = pytest.mark.parametrize("dtype,lens,counts,size", EXACT + OTHERS, ids=ids(EXACT + OTHERS))
BY_EXACT_SHAPE = pytest.mark.parametrize("dtype,lens,counts,size", EXACT, ids=ids(EXACT))


@BY_SHAPE
@pytest.mark.parametrize("which", range(3))
def test_nan_in_a_query(kernels, dtype, lens, counts, size, which):
    """A NaN in one element of a row's head: that head of that row is NaN, whatever it sees."""
    case = make(dtype, lens, counts, size)
    for row in (0, 3, counts[0] + 2, case.M - 1):
        case.q[row, (row % HEADS) * size + 5] = bits(dtype, NANS[dtype][which])
    run(kernels, case)
    run(kernels, case, sink=0.5)


@BY_SHAPE
@pytest.mark.parametrize("which", range(3))
def test_nan_in_a_settled_key(kernels, dtype, lens, counts, size, which):
    """Every row of the request is NaN in the heads of that kv head."""
    case = make(dtype, lens, counts, size)
    page, off = place(case, 0, lens[0] // 3)
    case.kv[0, page, 1, off, 7] = bits(dtype, NANS[dtype][which])
    run(kernels, case)
    if (dtype, lens, counts, size) in EXACT:
        run(kernels, case, Window("sliding", lens[0] - lens[0] // 3 + 2))       # deep nodes do not see it


@BY_SHAPE
@pytest.mark.parametrize("which", range(3))
def test_nan_in_a_settled_value(kernels, dtype, lens, counts, size, which):
    """That element is NaN."""
    case = make(dtype, lens, counts, size)
    page, off = place(case, 0, lens[0] // 2)
    case.kv[1, page, 0, off, 9] = bits(dtype, NANS[dtype][which])
    run(kernels, case)
    if (dtype, lens, counts, size) in EXACT:
        run(kernels, case, Window("sliding", lens[0] - lens[0] // 2 + 2))


@BY_EXACT_SHAPE
@pytest.mark.parametrize("plane", [0, 1])
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
def test_what_siblings_hold(kernels, dtype, lens, counts, size, plane, value):
    """A node's key or value that is not finite reaches the nodes that see it and no others."""
    case = make(dtype, lens, counts, size)
    for s, node in ((0, 1), (0, counts[0] // 2), (2, counts[2] - 1)):
        page, off = place(case, s, lens[s] + node)
        case.kv[plane, page, node % KV_HEADS, off, (5 * node) % size] = bits(dtype, NANS[dtype][0]) if value == "nan" else float(value)
    got = run(kernels, case)
    assert torch.isfinite(got).any() and not torch.isfinite(got).all()


@BY_EXACT_SHAPE
def test_infinite_settled_numbers(kernels, dtype, lens, counts, size):
    """Scores of minus infinity weigh nothing, of plus infinity make NaN; infinite values come out."""
    for plane in (0, 1):
        for sign in (1, -1):
            case = make(dtype, lens, counts, size)
            page, off = place(case, 0, 2)
            case.kv[plane, page, 0, off, 3] = sign * math.inf
            run(kernels, case)
            run(kernels, case, sink=-1.0)


@BY_SHAPE
def test_scores_of_minus_infinity(kernels, dtype, lens, counts, size):
    """A whole tile of keys, or every key, that scores minus infinity."""
    case = make(dtype, lens, counts, size)
    case.q.view(case.M, HEADS, size)[:, :, 0] = 1.0
    for j in range(min(64, lens[0])):
        page, off = place(case, 0, j)
        case.kv[0, page, :, off, 0] = -math.inf
    run(kernels, case)
    run(kernels, case, sink=0.0)
    for j in range(lens[1] + counts[1]):
        page, off = place(case, 1, j)
        case.kv[0, page, :, off, 0] = -math.inf
    got = run(kernels, case)
    assert (got[counts[0]:counts[0] + counts[1]] == 0).all()


@BY_SHAPE
def test_the_largest_numbers(kernels, dtype, lens, counts, size):
    """Keys of the largest number against queries that make ordinary scores of them; in float32 values of the largest number (the tensor cores' kernel's
    weights are up to 2^8 before the division)."""
    case = make(dtype, lens, counts, size)
    most = bits(dtype, LARGEST[dtype])
    case.q.view(case.M, HEADS, size)[:, :, 0] = 2.0 ** -126
    for s, j in ((0, 1), (1, 20), (0, lens[0])):
        page, off = place(case, s, j)
        case.kv[0, page, :, off, 0] = most
    run(kernels, case)
    if (dtype, lens, counts, size) in EXACT:
        page, off = place(case, 0, 40)
        case.kv[1, page, 1, off, 4] = most
        page, off = place(case, 1, 25)
        case.kv[1, page, 0, off, size - 1] = -most
        run(kernels, case)


@BY_SHAPE
def test_rows_of_nan_alone(kernels, dtype, lens, counts, size):
    """A query whose every score is NaN is NaN in every element; the rows beside it are what they are."""
    case = make(dtype, lens, counts, size)
    for row in (2, counts[0], case.M - 1):
        case.q[row] = bits(dtype, NANS[dtype][0])
    run(kernels, case)
    run(kernels, case, sink=1.0)
