"""Keys and values written by a step's slot map: only rows that are a token of the step write, whatever lies behind them."""
import random

import pytest
import torch

from draft_helpers import plain_accept, random_tree
from spite_b200.cache import LayerCache, Window
from spite_b200.engine.batch import StepBatch
from spite_b200.kernels.api import KernelError, PageTables, StepLayout

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def kernels():
    from spite_b200.kernels.cuda import CudaKernels
    return {t: CudaKernels(t, DEV) for t in (F32, BF)}


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def step_of(n_rows, cu, table, positions, seg, slot_map):
    return StepBatch(n_tokens=n_rows, segments=[], token_ids=None, positions=positions, seg_of_token=seg, cu_seqlens=cu, slots=None, logit_rows=None,
                     block_tables=[table], slot_maps=[slot_map])


# (the kernel of 16-byte words, the general one; both types; keys that are the values, with a factor each)
@pytest.mark.parametrize("dtype,size,one_plane", [(BF, 128, False), (BF, 64, False), (BF, 48, False), (F32, 64, False), (BF, 64, True), (F32, 32, True)])
@pytest.mark.parametrize("tokens", [0, 1, 23, 40])
def test_rows_behind_the_last_token_write_nothing(kernels, dtype, size, one_plane, tokens):
    k, g = kernels[dtype], torch.Generator().manual_seed(tokens + size)
    heads, kv_heads, pages, page, rows = 4, 2, 6, 16, 40
    kv = torch.randn((1 if one_plane else 2, pages, kv_heads, page, size), generator=g).to(dtype).to(DEV)
    scale = torch.full((pages, kv_heads, page), 7.0, device=DEV) if one_plane else None
    slots = torch.randperm(pages * page, generator=g)[:rows]
    slots[5], slots[11] = -1, pages * page
    slots[18] = 1 << 40
    cu = [0, tokens // 2, tokens // 2, tokens]
    qkv = torch.randn((rows, (heads + (1 if one_plane else 2) * kv_heads) * size), generator=g).to(dtype).to(DEV)
    q = torch.zeros((rows, heads * size), dtype=dtype, device=DEV)
    positions = torch.randint(-100, 1 << 20, (rows,), generator=g).to(torch.int32)
    batch = step_of(rows, ints(cu), ints([[-1]] * 3), positions.to(DEV), ints([-7] * rows), slots.to(DEV))
    want, want_scale = kv.clone(), None if scale is None else scale.clone()
    for t in range(tokens):
        s = int(slots[t])
        if 0 <= s < pages * page:
            for plane in range(kv.shape[0]):
                at = (heads + plane * kv_heads) * size
                want[plane, s // page, :, s % page] = qkv[t, at:at + kv_heads * size].view(kv_heads, size)
            if one_plane:
                want_scale[s // page, :, s % page] = 1.0
    k.qk_prepare(qkv, q, batch, LayerCache(0, kv, None, page, True, scale), num_heads=heads, rotation=None, qk_norm=None, temperature=None,
                 values_are_keys=one_plane)
    assert torch.equal(kv, want) and (scale is None or torch.equal(scale, want_scale))
    assert torch.equal(q[:tokens], qkv[:tokens, :heads * size])
    if tokens == 40:
        for bad in (None, batch.cu_seqlens.long(), batch.cu_seqlens[:0]):
            batch.cu_seqlens = bad
            with pytest.raises(KernelError):
                k.qk_prepare(qkv, q, batch, LayerCache(0, kv, None, page, True, scale), num_heads=heads, rotation=None, qk_norm=None, temperature=None,
                             values_are_keys=one_plane)


@pytest.mark.parametrize("dtype,size", [(BF, 128), (BF, 48), (F32, 64)])
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_a_loop_over_buffers_of_fixed_size(kernels, dtype, size, captured):
    """Layout, keys and values, attention, acceptance over buffers with room for more than a step brings, which the host does not look into: steps get smaller,
    a request ends and another begins, nodes are padding, a step runs out of pages.  Every settled row of the cache stays bit for bit."""
    k, r, g = kernels[dtype], random.Random(size), torch.Generator(device=DEV).manual_seed(size)
    heads, kv_heads, page, rows, room, n_pages, S = 4, 2, 16, 4, 200, 14, 3
    blank = lambda *shape, dtype=torch.int32: torch.full(shape, 0, dtype=dtype, device=DEV)
    kv = torch.randn((1, 2, n_pages, kv_heads, page, size), generator=g, device=DEV).to(dtype)
    pages = PageTables(tables=ints([[-1] * 12] * rows), held=ints([0] * rows), page_size=page, window=Window("full"), free_pages=ints(list(range(n_pages))),
                       n_free=ints([n_pages]))
    lengths, slots, new, parents = ints([0] * rows), ints([0] * S), ints([0] * S), blank(room)
    tokens, targets = blank(room), blank(room)
    out = StepLayout(block_table=blank(S, 12), cu_seqlens=blank(S + 1), positions=blank(room), seg_of_token=blank(room), slot_map=blank(room, dtype=torch.int64),
                     status=blank(1), ancestors=blank(room, 2))
    qkv = blank(room, (heads + 2 * kv_heads) * size, dtype=dtype)
    q, o = blank(room, heads * size, dtype=dtype), blank(room, heads * size, dtype=dtype)
    counts, path, emitted = blank(S), blank(S, 64), blank(S, 64)
    batch = step_of(room, out.cu_seqlens, out.block_table, out.positions, out.seg_of_token, out.slot_map)
    batch.ancestors = out.ancestors

    def step():
        k.layout_step(pages, slots, lengths, new, out, parents=parents)
        k.qk_prepare(qkv, q, batch, LayerCache(0, kv[0], None, page, True), num_heads=heads, rotation=None, qk_norm=None, temperature=None)
        k.tree_attention(q, o, batch, LayerCache(0, kv[0], None, page, False), num_heads=heads, window=Window("full"), softmax_scale=size ** -0.5)
        k.accept_drafts(tokens, parents, targets, out.cu_seqlens, [(kv, out.slot_map, None)], counts=counts, path=path, emitted=emitted, slots=slots, lengths=lengths,
                        lengths_out=lengths)
    run = step
    if captured:
        slots.copy_(ints([-1] * S))                          # (a step without requests, outside the graph and in it)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
        run = graph.replay
    text = {}                                                # row -> settled keys and values [n, 2, kv heads, size]
    plan = [([0, 1, 2], [40, 30, 20]), ([0, 1, 2], [40, 20, 9]), ([0, 1, 2], [9, 0, 33]), ([0, 1, 2], [1, 1, 1]), ([2, 0, -1], [5, 2, 7]), ([0, 1, 2], [3, -1, 4]),
            ([3, 0, 2], [60, 1, 30]), ([3, 0, 2], [64, 64, 64]), ([2, 3, 0], [2, 1, 1]), ([-1, -1, -1], [5, 5, 5]), ([0, 2, 3], [1, 0, 2])]
    refused = 0
    for s_rows, s_new in plan:
        ns = [max(n, 0) if row >= 0 else 0 for row, n in zip(s_rows, s_new)]
        first = all(row < 0 or not len(text.get(row, [])) for row in s_rows)
        trees = [list(range(-1, n - 1)) if first else random_tree(r, n, r.random() < 0.4) for n in ns]
        flat, n_all = [p for t in trees for p in t], sum(ns)
        toks = [1 if first else r.randrange(2) for _ in range(n_all)]
        want_next = [1 if first else r.randrange(2) for _ in range(n_all)]
        fill = lambda t, v: t.copy_(ints(v + [r.randrange(-3, 3) for _ in range(t.numel() - len(v))]))
        fill(parents, flat); fill(tokens, toks); fill(targets, want_next)
        slots.copy_(ints(s_rows)); new.copy_(ints(s_new))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=DEV))
        run()
        torch.cuda.synchronize()
        status, made = int(out.status), qkv.view(room, heads + 2 * kv_heads, size)[:, heads:].reshape(room, 2, kv_heads, size)
        if status:
            assert status == StepLayout.OUT_OF_PAGES and counts.tolist() == [0] * S
            refused += 1
        else:
            cu = [0]
            for n in ns:
                cu.append(cu[-1] + n)
            n_kept, ways, _ = plain_accept(toks, flat, want_next, cu, 64)
            assert counts.tolist() == n_kept
            for s, row in enumerate(s_rows):
                if row >= 0 and s_new[s] < 0:
                    text.pop(row, None)
                    lengths[row] = 0
                elif row >= 0:
                    keep = made[[cu[s] + i for i in ways[s][:n_kept[s]]]].clone()
                    text[row] = torch.cat([text[row], keep]) if row in text else keep
        assert lengths.tolist() == [len(text.get(row, [])) for row in range(rows)]
        for row, kept in text.items():
            table = pages.tables[row].tolist()
            assert len(kept) <= 16 * sum(p >= 0 for p in table)
            at = [(table[j // page], j % page) for j in range(len(kept))]
            got = kv[0][:, [a for a, _ in at], :, [b for _, b in at]]                # [n, 2, kv heads, size]
            assert torch.equal(got, kept), f"row {row}: settled keys or values have changed"
    assert refused == 1 and len(text) == 3
