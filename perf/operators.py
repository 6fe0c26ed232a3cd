"""Operators of a step that verifies drafted tokens: attention of token trees over the paged cache, the step's block tables and
slot map from the requests' lengths, and the acceptance of a path with its cache rows moved into place.

A case names the operator (`kind`) and its sizes.  `prepare` makes what a serving program has in hand before the call (the cache,
its tables, the drafted trees), `run` is one call, `exact` the same in 64 bits or by plain loops.
"""
from __future__ import annotations

import math
import random

import torch

DEV = "cuda:0"
own = False


def listed():
    return [
        # one chat request early in its answer, eight drafted tokens: the smallest call, latency counts
        dict(name="tree_one_short", kind="tree", dtype="bf16", requests=1, nodes=8, ragged=False, context=100, heads=40, kv_heads=8, size=128, window=0, sinks=False),
        # a decode batch of Llama-4-Scout's heads at the context of the benchmark, 16 drafted tokens a request
        dict(name="tree_batch", kind="tree", dtype="bf16", requests=8, nodes=16, ragged=False, context=8192, heads=40, kv_heads=8, size=128, window=0, sinks=False),
        # one request far into a long document: few rows, the whole device has to share one context
        dict(name="tree_long", kind="tree", dtype="bf16", requests=1, nodes=64, ragged=False, context=131072, heads=40, kv_heads=8, size=128, window=0, sinks=False),
        # a full house of requests of all lengths with trees of all sizes, a sliding window and a learned sink per head
        dict(name="tree_ragged_window", kind="tree", dtype="bf16", requests=64, nodes=48, ragged=True, context=4096, heads=32, kv_heads=8, size=64, window=1024, sinks=True),
        # wide trees and many query heads a kv head: the one that is bound by the products
        dict(name="tree_wide", kind="tree", dtype="bf16", requests=16, nodes=64, ragged=False, context=8192, heads=64, kv_heads=8, size=128, window=0, sinks=False),
        # the float32 kernel set, odd sizes
        dict(name="tree_float32", kind="tree", dtype="fp32", requests=4, nodes=13, ragged=True, context=2047, heads=16, kv_heads=4, size=128, window=0, sinks=False),
        # the next step of one request with eight drafted tokens: the smallest layout
        dict(name="layout_one", kind="layout", requests=1, nodes=8, trees=True, context=100, width=64, page=64, window=0, ends=0),
        # a decode batch with trees, long contexts, two requests that have just ended
        dict(name="layout_trees", kind="layout", requests=64, nodes=32, trees=True, context=131072, width=2049, page=64, window=0, ends=2),
        # many requests without drafts: single tokens beside portions of prompts, a sliding window whose pages go back
        dict(name="layout_portions", kind="layout", requests=250, nodes=64, trees=False, context=16384, width=260, page=64, window=4096, ends=5),
        # one request's accepted tokens in the caches of four layers: the smallest call
        dict(name="accept_one", kind="accept", dtype="bf16", requests=1, nodes=8, depth=4, caches=4, kv_heads=8, size=128, page=64),
        # a decode batch in the caches of 48 layers of Scout's heads
        dict(name="accept_batch", kind="accept", dtype="bf16", requests=8, nodes=16, depth=5, caches=48, kv_heads=8, size=128, page=64),
        # a full house with large, deep trees, pages of 16 positions
        dict(name="accept_many", kind="accept", dtype="bf16", requests=61, nodes=50, depth=9, caches=24, kv_heads=8, size=64, page=16),
    ]


def draw(rng):
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))
    kind = rng.choice(["tree", "tree", "tree", "layout", "accept"])
    if kind == "tree":
        kv_heads, group, size = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([64, 128, 128])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        context = log(30, 60000) if dtype == "bf16" else log(30, 2500)
        requests = max(1, min(log(1, 64), (131072 if dtype == "bf16" else 8192) // context))
        return dict(kind=kind, dtype=dtype, requests=requests, nodes=log(1, 64 if dtype == "bf16" else 16), ragged=rng.random() < 0.7, context=context,
                    heads=kv_heads * group, kv_heads=kv_heads, size=size, window=rng.choice([0, 0, log(50, 8192)]), sinks=rng.random() < 0.3)
    if kind == "layout":
        trees, context, page = rng.random() < 0.6, log(60, 131072), rng.choice([16, 64, 64])
        nodes = log(1, 64) if trees else log(1, 200)
        requests = max(1, min(log(1, 250), 4_000_000 // context))
        return dict(kind=kind, requests=requests, nodes=nodes, trees=trees, context=context, width=(context + nodes) // page + rng.randint(1, 40), page=page,
                    window=rng.choice([0, 0, log(20, 8192)]), ends=rng.randint(0, min(4, requests - 1)))
    nodes = log(2, 64)
    return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp32"]), requests=log(1, 61), nodes=nodes, depth=rng.randint(1, max(1, min(9, nodes // 2))), caches=log(1, 24),
                kv_heads=rng.choice([1, 2, 4, 8]), size=rng.choice([64, 128]), page=rng.choice([16, 64]))


# ------------------------------------------------------------------ inputs
def _shares(case, of, least=1):
    """The requests' numbers of `of`, the same for every seed: equal, or from a few to all."""
    r = random.Random(case[of] * 31 + case["requests"])
    if not case.get("ragged", True):
        return [case[of]] * case["requests"]
    return [case[of]] + [r.randint(least, max(least, case[of])) for _ in range(case["requests"] - 1)]


def _contexts(case):
    r = random.Random(case["context"] * 17 + case["requests"])
    if not case.get("ragged", True):
        return [case["context"] - r.randint(0, min(63, case["context"] - 1)) for _ in range(case["requests"])]
    return [case["context"]] + [max(1, int(case["context"] * r.random() ** 1.5)) for _ in range(case["requests"] - 1)]


def _draws(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 29), random.Random(int(seed) * 7919 + 5)


def _tree(r, n, depth=None):
    """Parents of n drafted tokens: node 0 is the request's own next token; with `depth`, nodes spread over so many levels."""
    if depth is None:
        return [-1] + [r.randint(max(0, i // 2 - 2), i - 1) for i in range(1, n)]
    parents, level = [-1], [0]
    for i in range(1, n):
        want = min(depth, 1 + (i - 1) * depth // max(1, n - 1))
        above = [a for a in range(i) if level[a] == want - 1]
        parents.append(r.choice(above))
        level.append(want)
    return parents


def _cat(lists):
    return torch.tensor([v for x in lists for v in x], dtype=torch.int32)


def _bits(parents, n_words):
    """The ancestor sets (a node itself among them) of one tree as rows of 32-bit words."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    words = [[(v >> 32 * w) & 0xFFFFFFFF for w in range(n_words)] for v in rows]
    return [[w - (1 << 32) if w >= 1 << 31 else w for w in row] for row in words]


def _levels(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def prepare(case, seed):
    return {"tree": _prepare_tree, "layout": _prepare_layout, "accept": _prepare_accept}[case["kind"]](case, seed)


def _prepare_tree(case, seed):
    g, r = _draws(seed)
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32}[case["dtype"]]
    counts, lens = _shares(case, "nodes"), _contexts(case)
    S, M, page = case["requests"], sum(counts), 64
    trees = [_tree(r, n) for n in counts]
    n_words = -(-max(counts) // 32)
    need = [-(-(a + n) // page) for a, n in zip(lens, counts)]
    ids = torch.randperm(sum(need) + 3, generator=g, device=DEV).to(torch.int32)
    table = torch.full((S, max(need)), -1, dtype=torch.int32)
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    used, host_ids = 0, ids.cpu()
    for s, k in enumerate(need):
        table[s, :k] = host_ids[used:used + k]
        used += k
    normal = lambda *shape, dtype=dt: torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, 1.0, generator=g)
    return dict(case=case, q=normal(M, case["heads"] * case["size"]), kv=normal(2, sum(need) + 3, case["kv_heads"], page, case["size"]),
                block_table=table.to(DEV), cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV),
                positions=_cat([[a + d for d in _levels(t)] for a, t in zip(lens, trees)]).to(DEV),
                seg_of_token=_cat([[s] * n for s, n in enumerate(counts)]).to(DEV),
                ancestors=torch.tensor([row for t in trees for row in _bits(t, n_words)], dtype=torch.int32, device=DEV),
                sinks=normal(case["heads"], dtype=torch.float32) if case["sinks"] else None, lens=lens, counts=counts)


def _layout_sizes(case):
    """(tokens cached, tokens brought: -1 where the request has ended) of every request."""
    r = random.Random(case["context"] + 3 * case["requests"])
    lens = _contexts(case)
    new = _shares(case, "nodes") if case["trees"] else [1 if r.random() < 0.8 else r.randint(2, max(2, case["nodes"])) for _ in lens]
    new = [min(n, case["nodes"]) for n in new]
    for s in range(case["ends"]):
        new[-1 - 2 * s % len(new)] = -1
    return lens, new


def _prepare_layout(case, seed):
    g, r = _draws(seed)
    S, W, page = case["requests"], case["width"], case["page"]
    lens, new = _layout_sizes(case)
    rows = list(range(S + 5))
    r.shuffle(rows)
    slots = rows[:S]
    total = sum(max(n, 0) for n in new)
    held = [-(-a // page) for a in lens]
    first = [max(0, a - r.randint(0, 40) - case["window"]) // page if case["window"] else 0 for a in lens]     # (some pages have already gone back)
    pages = sum(held) + sum(max(n, 0) // page + 2 for n in new) + 7
    ids = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu()
    tables, used = torch.full((S + 5, W), -1, dtype=torch.int32), 0
    held_of, len_of = torch.zeros(S + 5, dtype=torch.int32), torch.zeros(S + 5, dtype=torch.int32)
    for s, row in enumerate(slots):
        k = held[s] - first[s]
        tables[row, first[s]:held[s]] = ids[used:used + k]
        used += k
        held_of[row], len_of[row] = held[s], lens[s]
    free = torch.zeros(pages, dtype=torch.int32)
    free[:pages - used] = ids[used:]
    parents, n_words = None, 0
    if case["trees"]:
        parents = _cat([_tree(r, n) for n in new if n > 0]).to(DEV)
        n_words = -(-max(new) // 32)
    blank = lambda *shape, dtype=torch.int32: torch.full(shape, -7, dtype=dtype, device=DEV)
    return dict(case=case, slots=torch.tensor(slots, dtype=torch.int32, device=DEV), lengths=len_of.to(DEV),
                new_tokens=torch.tensor(new, dtype=torch.int32, device=DEV), tables=tables.to(DEV), held=held_of.to(DEV), free_pages=free.to(DEV),
                n_free=torch.tensor([pages - used], dtype=torch.int32, device=DEV), parents=parents, block_table=blank(S, W), cu_seqlens=blank(S + 1),
                positions=blank(total + 3), seg_of_token=blank(total + 3), slot_map=blank(total + 3, dtype=torch.int64),
                ancestors=blank(total + 3, n_words) if n_words else None, status=blank(1))


def _accepted(case):
    """How many drafted tokens of every request are right, the same for every seed."""
    r = random.Random(case["nodes"] * 13 + case["requests"])
    return [r.randint(0, case["depth"]) for _ in range(case["requests"])]


def _prepare_accept(case, seed):
    g, r = _draws(seed)
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32}[case["dtype"]]
    S, n, page = case["requests"], case["nodes"], case["page"]
    parents, tokens, targets, slot_map, lens = [], [], [], [], []
    pages = S * (n // page + 2)
    ids = torch.randperm(pages, generator=g, device=DEV).tolist()
    for s, right in enumerate(_accepted(case)):
        tree = _tree(r, n, case["depth"])
        tok = [r.randint(0, 200000) for _ in tree]
        want = [r.randint(200001, 202047) for _ in tree]              # (matches no drafted token)
        at = r.choice([i for i, d in enumerate(_levels(tree)) if d == min(right, max(_levels(tree)))])
        while tree[at] >= 0:                                          # the target tokens lead to that node
            want[tree[at]] = tok[at]
            at = tree[at]
        first = r.randint(0, page - 1)
        own_pages = ids[s * (n // page + 2):(s + 1) * (n // page + 2)]
        slot_map += [own_pages[(first + i) // page] * page + (first + i) % page for i in range(n)]
        parents += tree
        tokens += tok
        targets += want
        lens.append(first + page * r.randint(0, 100))
    ints = lambda v, dtype=torch.int32: torch.tensor(v, dtype=dtype, device=DEV)
    blank = lambda *shape: torch.full(shape, -7, dtype=torch.int32, device=DEV)
    kv = torch.empty((case["caches"], 2, pages, case["kv_heads"], page, case["size"]), dtype=dt, device=DEV).normal_(0.0, 1.0, generator=g)
    return dict(case=case, kv=kv, tokens=ints(tokens), parents=ints(parents), targets=ints(targets), slot_map=ints(slot_map, torch.int64),
                cu_seqlens=ints([s * n for s in range(S + 1)]), slots=ints(list(range(S))[::-1]), lengths=ints(lens), lengths_out=blank(S),
                counts=blank(S), path=blank(S, case["depth"] + 1), emitted=blank(S, case["depth"] + 1))


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return {"tree": _own_tree, "layout": _own_layout, "accept": _own_accept}[state["case"]["kind"]](state)
    return {"tree": _plain_tree, "layout": _plain_layout, "accept": _plain_accept}[state["case"]["kind"]](state)


_KERNELS = {}


def _kernels(dtype):
    """The kernel set that a program keeps, by activation type."""
    if dtype not in _KERNELS:
        from spite_b200.kernels.cuda import CudaKernels
        _KERNELS[dtype] = CudaKernels(dtype, DEV)
    return _KERNELS[dtype]


def _own_tree(st):
    case, q = st["case"], st["q"]
    k = _kernels(q.dtype)
    if "batch" not in st:                                             # what a program keeps of the step and of the layer's cache
        from spite_b200.cache import LayerCache, Window
        from spite_b200.engine.batch import StepBatch
        st["batch"] = StepBatch(n_tokens=q.shape[0], segments=[], token_ids=None, positions=st["positions"], seg_of_token=st["seg_of_token"],
                                cu_seqlens=st["cu_seqlens"], slots=None, logit_rows=None, block_tables=[st["block_table"]], ancestors=st["ancestors"])
        st["cache"] = LayerCache(0, st["kv"], None, st["kv"].shape[3], False)
        st["window"] = Window("sliding", case["window"]) if case["window"] else Window("full")
    out = torch.empty_like(q)
    k.tree_attention(q, out, st["batch"], st["cache"], num_heads=case["heads"], window=st["window"], softmax_scale=case["size"] ** -0.5, head_sinks=st["sinks"])
    return out


def _own_layout(st):
    if "pages" not in st:
        from spite_b200.cache import Window
        from spite_b200.kernels.api import PageTables, StepLayout
        case = st["case"]
        st["pages"] = PageTables(tables=st["tables"], held=st["held"], page_size=case["page"],
                                 window=Window("sliding", case["window"]) if case["window"] else Window("full"), free_pages=st["free_pages"], n_free=st["n_free"])
        st["layout"] = StepLayout(**{n: st[n] for n in ("block_table", "cu_seqlens", "positions", "seg_of_token", "slot_map", "ancestors", "status")})
    _kernels(torch.bfloat16).layout_step(st["pages"], st["slots"], st["lengths"], st["new_tokens"], st["layout"], parents=st["parents"])
    return _layout_outputs(st)


def _own_accept(st):
    _kernels(st["kv"].dtype).accept_drafts(st["tokens"], st["parents"], st["targets"], st["cu_seqlens"], [(st["kv"], st["slot_map"], None)], counts=st["counts"],
                                           path=st["path"], emitted=st["emitted"], slots=st["slots"], lengths=st["lengths"], lengths_out=st["lengths_out"])
    return [st[n] for n in ("counts", "path", "emitted", "lengths_out", "kv")]


def _layout_outputs(st):
    return {n: st[n] for n in ("tables", "held", "free_pages", "n_free", "block_table", "cu_seqlens", "positions", "seg_of_token", "slot_map", "ancestors", "status")
            if st[n] is not None}


# ------------------------------------------------------------------ plain forms
def _plain_tree(st):
    case, q, kv, table, cu = st["case"], st["q"], st["kv"], st["block_table"].long(), st["cu_seqlens"].long()
    nq, nkv, hd, page = case["heads"], case["kv_heads"], case["size"], kv.shape[3]
    M, S = q.shape[0], table.shape[0]
    seg = st["seg_of_token"].long()
    pos = st["positions"].long()
    n = cu[1:] - cu[:-1]
    length = pos[cu[:-1]]                                              # [S] the first drafted token's position
    N, L = max(st["counts"]), max(a + b for a, b in zip(st["lens"], st["counts"]))
    node = torch.arange(M, device=DEV) - cu[seg]
    # every request's queries, positions and ancestor bits, padded to the largest tree
    qp = torch.zeros((S, N, nq, hd), device=DEV)
    qp[seg, node] = q.view(M, nq, hd).float()
    pp = torch.zeros((S, N), dtype=torch.long, device=DEV)
    pp[seg, node] = pos
    words = st["ancestors"].long()
    bits = (words[:, torch.arange(N, device=DEV) // 32] >> (torch.arange(N, device=DEV) % 32)) & 1
    anc = torch.zeros((S, N, N), dtype=torch.bool, device=DEV)
    anc[seg, node] = bits.bool()
    # the keys' places and positions, and who sees them
    place = torch.arange(L, device=DEV)
    held = place[None, :] < (length + n)[:, None]                     # [S, L]
    rel = place[None, :] - length[:, None]
    inside = (rel >= 0) & held
    at = rel.clamp(0, N - 1)
    key_pos = torch.where(inside, pp.gather(1, at), place[None, :])
    seen = torch.where(inside[:, None, :], anc.gather(2, at[:, None, :].expand(S, N, L)), held[:, None, :])
    if case["window"]:
        seen &= key_pos[:, None, :] > pp[:, :, None] - case["window"]
    pages = table[torch.arange(S, device=DEV)[:, None], (place // page).clamp(max=table.shape[1] - 1)[None, :]]
    rows = torch.where(held & (pages >= 0), pages, 0) * page + (place % page)[None, :]
    flat = kv.permute(0, 1, 3, 2, 4).reshape(2, -1, nkv, hd)          # [2, pages * page, nkv, hd]
    k, v = (flat[i][rows].float().permute(0, 2, 1, 3) for i in (0, 1))         # [S, nkv, L, hd]
    g = nq // nkv
    qs = qp.view(S, N, nkv, g, hd).permute(0, 2, 3, 1, 4).reshape(S, nkv, g * N, hd)
    s = (qs @ k.transpose(2, 3)) * hd ** -0.5                          # [S, nkv, g * N, L]
    s = s.view(S, nkv, g, N, L).masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    sink = None if st["sinks"] is None else st["sinks"].view(1, nkv, g, 1, 1)
    top = top if sink is None else torch.maximum(top, sink)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    o = (w.view(S, nkv, g * N, L) @ v).view(S, nkv, g, N, hd) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, N, nq * hd)
    return o[seg, node].to(q.dtype)


def _plain_layout(st):
    case = st["case"]
    page, W, slots = case["page"], case["width"], st["slots"].long()
    new, tables, held_of, free, n_free = st["new_tokens"].long(), st["tables"], st["held"], st["free_pages"], st["n_free"].long()
    length, held = st["lengths"].long()[slots], held_of.long()[slots]
    S, P, col = slots.numel(), free.numel(), torch.arange(W, device=DEV)[None, :]
    rows = tables[slots].long()
    ended = (new < 0)[:, None]
    # pages that no later token reads go back, in the requests' order and within one from the first
    first = (length - case["window"] + 1).clamp(min=0) // page if case["window"] else torch.zeros_like(length)
    goes = (rows >= 0) & (col < held[:, None]) & (ended | (col < first[:, None]))
    order = goes.reshape(-1).cumsum(0) - 1
    stack = torch.cat([free, free.new_zeros(1)])
    stack[torch.where(goes.reshape(-1), n_free + order, P)] = rows.reshape(-1).int()
    top = n_free + goes.sum()
    rows = torch.where(goes, -1, rows)
    held = torch.where(new < 0, 0, held)
    # pages that the step's tokens need, from the top of the stack
    need = torch.where(new < 0, 0, torch.maximum(held, -(-(length + new.clamp(min=0)) // page)))
    comes = (col >= held[:, None]) & (col < need[:, None])
    taken = (comes.reshape(-1).cumsum(0) - 1).view(S, W)
    rows = torch.where(comes, stack[(top - 1 - taken).clamp(0, P)].long(), rows)
    free.copy_(stack[:P])
    tables[slots] = rows.int()
    held_of[slots] = need.int()
    st["n_free"].copy_(top - comes.sum())
    st["block_table"].copy_(rows)
    # the tokens
    cu = torch.cat([new.new_zeros(1), new.clamp(min=0).cumsum(0)])
    st["cu_seqlens"].copy_(cu)
    cap = st["positions"].numel()
    t = torch.arange(cap, device=DEV)
    real = t < cu[-1]
    seg = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=S - 1)
    node = t - cu[seg]
    place = length[seg] + node
    position = place
    if st["parents"] is not None:
        words = st["ancestors"].shape[1]
        par = torch.cat([st["parents"].long(), t.new_full((cap - st["parents"].numel(),), -1)])
        up = torch.where(par >= 0, cu[seg] + par, cap)                # the parent's row, or one that stands for none
        up = torch.cat([up, up.new_full((1,), cap)])
        bit = torch.zeros((cap + 1, 32 * words), dtype=torch.bool, device=DEV)
        bit[t, node.clamp(0, 32 * words - 1)] = real
        for _ in range((32 * words).bit_length()):                    # ancestors of ancestors: twice as far each time
            bit = bit | bit[up]
            up = up[up]
        position = length[seg] + bit[:cap].sum(1) - 1
        packed = (bit[:cap].view(cap, words, 32).long() << torch.arange(32, device=DEV)).sum(-1)
        packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).int()
        st["ancestors"].copy_(torch.where(real[:, None], packed, st["ancestors"]))
    slot = rows[seg, (place // page).clamp(0, W - 1)] * page + place % page
    st["positions"].copy_(torch.where(real, position, st["positions"].long()))
    st["seg_of_token"].copy_(torch.where(real, seg, st["seg_of_token"].long()))
    st["slot_map"].copy_(torch.where(real, slot, st["slot_map"]))
    st["status"].zero_()
    return _layout_outputs(st)


def _plain_accept(st):
    case, cu = st["case"], st["cu_seqlens"].long()
    S, n, D = case["requests"], case["nodes"], case["depth"] + 1
    parents, tokens, targets = (st[x].view(S, n) for x in ("parents", "tokens", "targets"))
    child = torch.arange(n, device=DEV)
    fits = (parents[:, None, :] == child[None, :, None]) & (tokens[:, None, :] == targets[:, :, None])      # [S, node, its child]
    follow = torch.where(fits, child, n).amin(-1)                     # the first child that is the target token; n: none
    follow = torch.cat([follow, follow.new_full((S, 1), n)], 1)
    path = [follow.new_zeros((S, 1))]
    for _ in range(D - 1):
        path.append(follow.gather(1, path[-1]))
    path = torch.cat(path, 1)
    on = path < n
    count = on.sum(1)
    st["counts"].copy_(count)
    st["path"].copy_(torch.where(on, path, -1))
    st["emitted"].copy_(torch.where(on, targets.long().gather(1, path.clamp(max=n - 1)), -1))
    slots = st["slots"].long()
    st["lengths_out"][slots] = (st["lengths"].long()[slots] + count).int()
    # the rows of the accepted tokens move to the places that follow the cached ones (read before any is written)
    kv, page = st["kv"], case["page"]
    place = st["slot_map"].view(S, n)
    src, dst = place.gather(1, torch.where(on, path, 0)), place.gather(1, torch.where(on, torch.arange(D, device=DEV)[None, :].clamp(max=n - 1), 0))
    src, dst = src.reshape(-1), dst.reshape(-1)                       # (places of a path that has ended repeat the first row, which stays)
    kv[:, :, dst // page, :, dst % page] = kv[:, :, src // page, :, src % page]
    return [st[x] for x in ("counts", "path", "emitted", "lengths_out", "kv")]


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case["kind"] == "layout":
        return None                                                   # whole numbers only
    st = prepare(case, seed)
    return _exact_tree(st) if case["kind"] == "tree" else _exact_accept(st)


def _exact_tree(st):
    case = st["case"]
    nq, nkv, hd, page = case["heads"], case["kv_heads"], case["size"], 64
    cu, table, pos = st["cu_seqlens"].tolist(), st["block_table"].tolist(), st["positions"].tolist()
    anc = st["ancestors"].cpu().tolist()
    out = torch.zeros((st["q"].shape[0], nq, hd), dtype=torch.float64, device=DEV)
    for s in range(case["requests"]):
        a, b, have = cu[s], cu[s + 1], pos[cu[s]]
        ids = torch.tensor(table[s][:-(-(have + b - a) // page)], device=DEV)
        keys, values = (st["kv"][i, ids].transpose(1, 2).reshape(-1, nkv, hd)[:have + b - a].double() for i in (0, 1))
        mask = torch.ones((b - a, have + b - a), dtype=torch.bool)
        for i in range(b - a):
            for j in range(b - a):
                mask[i, have + j] = anc[a + i][j // 32] >> (j % 32) & 1
        at = torch.tensor(list(range(have)) + pos[a:b])
        if case["window"]:
            mask &= at[None, :] > torch.tensor(pos[a:b])[:, None] - case["window"]
        mask = mask.to(DEV)
        for h in range(nq):
            x = st["q"][a:b].view(b - a, nq, hd)[:, h].double() @ keys[:, h * nkv // nq].T / math.sqrt(hd)
            x = torch.where(mask, x, torch.full_like(x, -math.inf))
            if st["sinks"] is not None:
                x = torch.cat([x, st["sinks"][h].double().expand(b - a, 1)], 1)
            p = torch.softmax(x, 1)[:, :have + b - a]
            out[a:b, h] = p @ values[:, h * nkv // nq]
    return out.view(out.shape[0], -1)


def _exact_accept(st):
    case, kv = st["case"], st["kv"].clone()
    S, n, D, page = case["requests"], case["nodes"], case["depth"] + 1, case["page"]
    parents, tokens, targets, place = (st[x].tolist() for x in ("parents", "tokens", "targets", "slot_map"))
    counts, paths, emitted, lengths = [], [], [], st["lengths"].tolist()
    for s in range(S):
        at, path = 0, [0]
        while len(path) < D:
            nxt = [c for c in range(n) if parents[s * n + c] == at and tokens[s * n + c] == targets[s * n + at]]
            if not nxt:
                break
            at = nxt[0]
            path.append(at)
        for d, node in enumerate(path):
            a, b = place[s * n + node], place[s * n + d]
            kv[:, :, b // page, :, b % page] = st["kv"][:, :, a // page, :, a % page]
        counts.append(len(path))
        paths.append(path + [-1] * (D - len(path)))
        emitted.append([targets[s * n + i] for i in path] + [-1] * (D - len(path)))
        lengths[S - 1 - s] += len(path)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    return [ints(counts), ints(paths), ints(emitted), ints(lengths), kv]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "tree":
        counts, lens = _shares(case, "nodes"), _contexts(case)
        size = 2 if case["dtype"] == "bf16" else 4
        # (a window's rows reach over the last `window` positions; a tree is a few positions deep)
        seen = [min(a, case["window"]) if case["window"] else a for a in lens]
        keys = sum(a + n for a, n in zip(seen, counts))
        pairs = sum(a * n + n * max(1, n.bit_length()) for a, n in zip(seen, counts))
        return dict(bytes=keys * 2 * case["kv_heads"] * case["size"] * size + 2 * sum(counts) * case["heads"] * case["size"] * size,
                    flops=4.0 * pairs * case["heads"] * case["size"])
    if case["kind"] == "layout":
        lens, new = _layout_sizes(case)
        total = sum(max(n, 0) for n in new)
        words = -(-max(new) // 32) if case["trees"] else 0
        held = sum(-(-(a + max(n, 0)) // case["page"]) for a, n in zip(lens, new))
        return dict(bytes=4 * (held + case["requests"] * (case["width"] + 5) + total * (4 + words + (1 if case["trees"] else 0))), flops=total)
    size = 2 if case["dtype"] == "bf16" else 4
    moved = sum(_accepted(case))
    return dict(bytes=2 * moved * case["caches"] * 2 * case["kv_heads"] * case["size"] * size + 12 * case["requests"] * (case["nodes"] + case["depth"]), flops=case["requests"] * case["nodes"])
