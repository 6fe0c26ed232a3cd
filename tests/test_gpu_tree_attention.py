"""Attention of trees of drafted tokens against the formula in 64 bits, at the sizes and masks where it can go wrong."""
import pytest
import torch

from draft_helpers import TreeCase, tolerance
from spite_b200.cache import LayerCache, Window
from spite_b200.kernels.api import DistanceBias, KernelError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FULL = Window("full")


@pytest.fixture(scope="module")
def kernels():
    from spite_b200.kernels.cuda import CudaKernels
    return {t: CudaKernels(t, DEV) for t in (torch.float32, torch.bfloat16)}


def run(kernels, case, window=FULL, *, out=None, scale=None, distance_rows=None, out_by_head=False, **more):
    """The kernel's result against the formula's; returns the result."""
    k = kernels[case.q.dtype]
    scale = scale or case.size ** -0.5
    q, batch, cache = case.step(DEV)
    out = torch.full_like(q, float("nan")) if out is None else out
    dev = {n: v.to(DEV) if isinstance(v, torch.Tensor) else v for n, v in more.items()}
    if distance_rows is not None:
        dev["distance_bias"] = DistanceBias.from_rows(distance_rows.t().contiguous().to(DEV), list(range(distance_rows.shape[1])))
    k.tree_attention(q, out, batch, cache, num_heads=case.heads, window=window, softmax_scale=scale, out_by_head=out_by_head, **dev)
    assert not k.errors()
    want, size, biggest = case.plain(window, scale, distance_rows=distance_rows, **more)
    got = out.double().cpu()
    if out_by_head:
        got = got.view(case.heads, -1, case.size).transpose(0, 1).reshape(out.shape)
    allowed = tolerance(case, want, size, biggest, rounded_weights=True)
    off = (got[:case.M] - want).abs()
    assert torch.isfinite(got[:case.M]).all(), "not finite"
    worst = float((off / allowed).max()) if case.M else 0.0
    assert worst <= 1.0, f"{worst:.2f} times the allowed error"
    return out


BF, F32 = torch.bfloat16, torch.float32
SHAPES = [
    # heads, kv heads, head size, page size
    (8, 8, 128, 64), (40, 8, 128, 64), (32, 8, 64, 64), (7, 1, 128, 128), (6, 2, 64, 64), (24, 1, 64, 64), (130, 1, 64, 64), (128, 1, 128, 64),
    (6, 2, 16, 16), (5, 1, 24, 5), (4, 2, 96, 64), (4, 2, 128, 32), (2, 2, 200, 64), (3, 1, 33, 7), (40, 2, 256, 16),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads,kv_heads,size,page", SHAPES)
def test_head_layouts(kernels, dtype, heads, kv_heads, size, page):
    run(kernels, TreeCase([70, 0, 131], [5, 3, 17], heads=heads, kv_heads=kv_heads, size=size, page=page, dtype=dtype, seed=heads + size))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,counts", [
    ([0], [1]), ([1], [1]), ([63], [1]), ([64], [1]), ([63], [2]), ([62], [70]), ([0], [64]), ([5], [65]), ([1000], [33]), ([700, 3, 0, 64], [0, 9, 1, 130]),
    ([0, 0], [0, 4]), ([129, 250, 17, 64, 511, 8], [26, 27, 25, 51, 52, 1]),
])
def test_lengths(kernels, dtype, lens, counts):
    run(kernels, TreeCase(lens, counts, heads=10, kv_heads=2, size=128 if dtype == BF else 64, dtype=dtype, seed=sum(lens) + len(counts)))


@pytest.mark.parametrize("dtype,size", [(BF, 128), (BF, 64), (BF, 32), (F32, 64)])
@pytest.mark.parametrize("window", [Window("sliding", 1), Window("sliding", 2), Window("sliding", 7), Window("sliding", 64), Window("sliding", 150), Window("chunk", 32),
                                    Window("chunk", 100), Window("chunk", 1)], ids=lambda w: f"{w.kind}{w.size}")
def test_windows(kernels, dtype, size, window):
    """Windows that end in the settled tokens, inside the tree (deep nodes see some of their ancestors only) and in front of everything."""
    chain = list(range(-1, 39))
    case = TreeCase([300, 95, 0, 64], [20, 13, 5, 40], heads=6, kv_heads=2, size=size, dtype=dtype, seed=window.size)
    run(kernels, case, window)
    run(kernels, TreeCase([300, 96], [40, 40], heads=6, kv_heads=2, size=size, dtype=dtype, seed=7, trees=[chain, chain]), window)


@pytest.mark.parametrize("dtype,size", [(BF, 128), (BF, 96), (F32, 64)])
def test_padding_and_rows_that_see_nothing(kernels, dtype, size):
    """Padding nodes: their cache rows hold NaN, nobody sees them; without settled tokens they see nothing, and their result is zero."""
    case = TreeCase([0, 40, 200], [9, 30, 70], heads=4, kv_heads=1, size=size, dtype=dtype, seed=5, padding=True)
    out = run(kernels, case)
    empty = [i for i in range(9) if not case.sets[0][i]]
    assert empty and (out[empty] == 0).all()
    run(kernels, case, head_sinks=torch.tensor([0.0, 3.0, -2.0, float("-inf")]))
    run(kernels, case, Window("sliding", 16), sink_logit=0.5)


def test_rows_behind_the_last_request(kernels):
    for dtype, size in ((BF, 128), (F32, 64)):
        case = TreeCase([100, 7], [12, 3], heads=4, kv_heads=2, size=size, dtype=dtype, seed=3, extra_rows=20)
        out = torch.full((35, 4 * size), 7.5, dtype=dtype, device=DEV)
        run(kernels, case, out=out)
        assert (out[15:] == 7.5).all()


@pytest.mark.parametrize("dtype,size,planes", [(BF, 128, 2), (BF, 64, 2), (BF, 64, 1), (F32, 48, 2), (F32, 64, 1)])
def test_everything_on_a_score(kernels, dtype, size, planes):
    g = torch.Generator().manual_seed(11)
    case = TreeCase([200, 33], [20, 70], heads=8, kv_heads=2, size=size, dtype=dtype, seed=9, planes=planes, key_scales=planes == 1)
    M = case.M
    gates, slopes, sinks = torch.rand(M, 8, generator=g), torch.rand(8, generator=g) * 0.1, torch.randn(8, generator=g)
    run(kernels, case, head_gates=gates, head_sinks=sinks)
    run(kernels, case, head_slopes=slopes, sink_logit=1.0, out_by_head=True)
    run(kernels, case, Window("sliding", 50), score_softcap=2.5, head_slopes=slopes)
    run(kernels, case, score_softcap=30.0)
    run(kernels, case, distance_rows=torch.randn(8, 40, generator=g))


@pytest.mark.parametrize("dtype,size", [(BF, 128), (BF, 64), (F32, 64)])
def test_large_scores(kernels, dtype, size):
    """Scores of some hundreds: the running maximum moves, weights vanish."""
    run(kernels, TreeCase([400, 1], [30, 40], heads=4, kv_heads=2, size=size, dtype=dtype, seed=1, scale=4.0))


@pytest.mark.parametrize("dtype,size,nodes", [(BF, 128, 1024), (BF, 64, 700), (F32, 16, 1024)])
def test_largest_trees(kernels, dtype, size, nodes):
    run(kernels, TreeCase([100], [nodes], heads=2, kv_heads=1, size=size, dtype=dtype, seed=2))


@pytest.mark.parametrize("dtype,size", [(BF, 64), (F32, 16)])
def test_many_requests(kernels, dtype, size):
    run(kernels, TreeCase([(37 * s) % 150 for s in range(1000)], [s % 4 for s in range(1000)], heads=2, kv_heads=1, size=size, dtype=dtype, seed=8))


@pytest.mark.parametrize("dtype,heads,size", [(BF, 5, 128), (BF, 8, 64), (F32, 2, 64)])
def test_long_contexts_are_shared_among_blocks(kernels, dtype, heads, size):
    """Contexts that are cut along the keys, beside ones that are not."""
    n = 20001 if dtype == BF else 5003
    case = TreeCase([n, 10, 3000], [30, 30, 64], heads=heads, kv_heads=1, size=size, dtype=dtype, seed=6)
    run(kernels, case)
    run(kernels, case, Window("sliding", 2000), sink_logit=0.0)


def test_bits_that_mean_nothing(kernels):
    """Bits of later nodes and of nodes that the request does not have change nothing."""
    for dtype, size in ((BF, 128), (F32, 64)):
        case = TreeCase([90], [40], heads=4, kv_heads=2, size=size, dtype=dtype, seed=4, n_words=3)
        first = run(kernels, case)
        for i in range(40):
            for a in range(i + 1, 96):
                word = int(case.ancestors[i, a // 32]) | (1 << (a % 32))
                case.ancestors[i, a // 32] = word - (1 << 32) if word >= 1 << 31 and word > 0 else word
        assert torch.equal(run(kernels, case), first)


@pytest.mark.parametrize("dtype,size", [(BF, 128), (F32, 64)])
def test_graph_and_stream(kernels, dtype, size):
    """Captured on another stream and replayed with other contents: the launch does not depend on the lengths."""
    k = kernels[dtype]
    small = TreeCase([5, 0], [12, 7], heads=4, kv_heads=2, size=size, dtype=dtype, seed=1, width=40)
    large = TreeCase([900, 1700], [12, 7], heads=4, kv_heads=2, size=size, dtype=dtype, seed=2, width=40)
    want = [run(kernels, c) for c in (small, large)]
    q, batch, cache = large.step(DEV)
    out = torch.empty_like(q)
    call = lambda: k.tree_attention(q, out, batch, cache, num_heads=4, window=FULL, softmax_scale=size ** -0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    for case, right in ((small, want[0]), (large, want[1])):
        q.copy_(case.q)
        batch.positions.copy_(case.positions)
        batch.ancestors.copy_(case.ancestors)
        batch.block_tables[0].copy_(case.table)
        cache.kv.zero_()
        cache.kv[:, :case.kv.shape[1]].copy_(case.kv)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, right)


def test_two_calls_at_once(kernels):
    """Two streams, each call with scratch of its own."""
    k = kernels[BF]
    cases = [TreeCase([3000], [40], heads=8, kv_heads=1, size=128, dtype=BF, seed=s) for s in (1, 2)]
    want = [run(kernels, c) for c in cases]
    steps = [c.step(DEV) for c in cases]
    outs = [torch.empty_like(s[0]) for s in steps]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for (q, batch, cache), out, stream in zip(steps, outs, streams):
            with torch.cuda.stream(stream):
                k.tree_attention(q, out, batch, cache, num_heads=8, window=FULL, softmax_scale=128 ** -0.5)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("dtype,size", [(BF, 128), (F32, 128)])
def test_beyond_32_bits(kernels, dtype, size):
    """A cache of more than 2^31 elements whose pages in use lie at its far end."""
    k = kernels[dtype]
    case = TreeCase([200, 40], [20, 30], heads=4, kv_heads=1, size=size, dtype=dtype, seed=12)
    want = run(kernels, case)
    n, more = case.kv.shape[1], 150000
    big = torch.zeros((2, more, 1, 64, size), dtype=dtype, device=DEV)                  # 1.2 * 10^9 elements a plane
    big[:, more - n:] = case.kv.to(DEV)
    q, batch, _ = case.step(DEV)
    table = batch.block_tables[0]
    batch.block_tables[0] = torch.where(table >= 0, table + (more - n), table)
    out = torch.empty_like(q)
    k.tree_attention(q, out, batch, LayerCache(0, big, None, 64, False), num_heads=4, window=FULL, softmax_scale=size ** -0.5)
    assert torch.equal(out, want)


def test_pages_that_are_not_there(kernels):
    """A table's holes and page numbers outside the cache are not read: what they would hold is seen by nobody, or is another page's."""
    for dtype, size in ((BF, 64), (F32, 64)):
        case = TreeCase([70, 130], [5, 6], heads=2, kv_heads=1, size=size, dtype=dtype, seed=3)
        q, batch, cache = case.step(DEV)
        out = torch.zeros_like(q)
        for bad in (-1, -(1 << 31), 1 << 30, case.kv.shape[1]):
            batch.block_tables[0][:] = bad
            kernels[dtype].tree_attention(q, out, batch, cache, num_heads=2, window=FULL, softmax_scale=0.125)
        torch.cuda.synchronize()
        assert not kernels[dtype].errors()


def test_refusals(kernels):
    k = kernels[F32]
    case = TreeCase([9], [4], heads=4, kv_heads=2, size=16, seed=1)
    q, batch, cache = case.step(DEV)
    out = torch.empty_like(q)
    call = lambda **kw: k.tree_attention(kw.pop("q", q), kw.pop("out", out), batch, cache,
                                         **{**dict(num_heads=4, window=FULL, softmax_scale=0.25), **kw})
    for kw in (dict(num_heads=3), dict(num_heads=0), dict(softmax_scale=0.0), dict(score_softcap=-1.0), dict(out=out[:2]), dict(q=q[:3], out=out[:3]), dict(q=q.bfloat16()),
               dict(head_sinks=torch.zeros(3, device=DEV)), dict(q=q.t())):
        with pytest.raises(KernelError):
            call(**kw)
    keep = batch.ancestors
    for bad in (None, keep[:2], keep.long(), keep.view(-1), keep[:, :0]):
        batch.ancestors = bad
        with pytest.raises(KernelError):
            call()
    batch.ancestors = keep
    call()
