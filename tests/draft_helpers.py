"""Plain forms of the operators of a step that verifies drafted tokens, in 64 bits and by loops, and random cases for them."""
from __future__ import annotations

import math
import random

import torch

from spite_b200.cache import LayerCache, Window
from spite_b200.engine.batch import StepBatch


def random_tree(r: random.Random, n: int, padding: bool = False) -> list:
    """Parents of n nodes; with `padding` some of the last ones are padding (-2)."""
    parents = [-1 if i == 0 or r.random() < 0.05 else r.randint(max(0, i - 6), i - 1) for i in range(n)]
    if padding and n > 1:
        for i in range(n - r.randint(1, max(1, n // 3)), n):
            parents[i] = -2
    return parents


def depths(parents: list) -> list:
    out = []
    for i, p in enumerate(parents):
        out.append(out[p] + 1 if 0 <= p < i else 0)
    return out


def ancestor_sets(parents: list) -> list:
    """{itself and its ancestors} of every node; empty for padding."""
    out = []
    for i, p in enumerate(parents):
        if p < -1:
            out.append(set())
        elif 0 <= p < i:
            out.append(out[p] | {i} | ({p} if parents[p] < -1 else set()))
        else:
            out.append({i})
    return out


def words_of(sets: list, n_words: int) -> list:
    rows = []
    for s in sets:
        v = sum(1 << a for a in s)
        row = [(v >> (32 * w)) & 0xFFFFFFFF for w in range(n_words)]
        rows.append([w - (1 << 32) if w >= 1 << 31 else w for w in row])
    return rows


class TreeCase:
    """A step of requests with trees over a paged cache.  Rows of the cache that hold no key of a request are NaN."""

    def __init__(self, lens, counts, *, heads, kv_heads, size, page=64, dtype=torch.float32, seed=0, planes=2, key_scales=False, extra_rows=0, padding=False,
                 width=None, n_words=None, trees=None, scale=1.0):
        r = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.lens, self.counts, self.heads, self.kv_heads, self.size, self.page = list(lens), list(counts), heads, kv_heads, size, page
        self.trees = trees or [random_tree(r, n, padding) for n in counts]
        self.sets = [ancestor_sets(t) for t in self.trees]
        S, M = len(lens), sum(counts)
        self.M = M
        need = [-(-(a + n) // page) for a, n in zip(lens, counts)]
        n_pages = sum(need) + 2
        ids = torch.randperm(n_pages, generator=g).tolist()
        W = width or max(need + [1])
        self.table = torch.full((S, W), -1, dtype=torch.int32)
        self.kv = torch.full((planes, n_pages, kv_heads, page, size), float("nan"), dtype=dtype)
        self.key_scale = torch.full((n_pages, kv_heads, page), float("nan")) if key_scales else None
        used = 0
        for s, k in enumerate(need):
            mine = ids[used:used + k]
            used += k
            self.table[s, :k] = torch.tensor(mine, dtype=torch.int32)
            for j in range(lens[s] + counts[s]):
                i = j - lens[s]
                if i >= 0 and i not in self.sets[s][i]:
                    continue                                    # padding: its row holds anything
                self.kv[:, mine[j // page], :, j % page] = (torch.randn(planes, kv_heads, size, generator=g) * scale).to(dtype)
                if key_scales:
                    self.key_scale[mine[j // page], :, j % page] = torch.rand(kv_heads, generator=g) + 0.5
        cap = M + extra_rows
        self.q = (torch.randn(cap, heads * size, generator=g) * scale).to(dtype)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32)
        self.positions = torch.tensor([a + d for a, t in zip(lens, self.trees) for d in depths(t)] + [-7] * extra_rows, dtype=torch.int32)
        self.seg = torch.tensor([s for s, n in enumerate(counts) for _ in range(n)] + [-7] * extra_rows, dtype=torch.int32)
        n_words = n_words or max(1, -(-max(counts + [1]) // 32))
        rows = [row for sets in self.sets for row in words_of(sets, n_words)]
        self.ancestors = torch.tensor(rows + [[-1] * n_words] * extra_rows, dtype=torch.int32).view(cap, n_words)

    def step(self, device):
        dev = lambda t: None if t is None else t.to(device)
        batch = StepBatch(n_tokens=self.q.shape[0], segments=[], token_ids=None, positions=dev(self.positions), seg_of_token=dev(self.seg),
                          cu_seqlens=dev(self.cu), slots=None, logit_rows=None, block_tables=[dev(self.table)], ancestors=dev(self.ancestors))
        return dev(self.q), batch, LayerCache(0, dev(self.kv), None, self.page, False, dev(self.key_scale))

    def plain(self, window: Window, softmax_scale, *, sink_logit=None, head_sinks=None, head_slopes=None, head_gates=None, score_softcap=None,
              distance_rows=None):
        """(outputs, the same with the values' absolute values, the largest sum |q k| softmax_scale) in 64 bits."""
        hd, G = self.size, self.heads // self.kv_heads
        out = torch.zeros((self.M, self.heads, hd), dtype=torch.float64)
        size = torch.zeros_like(out)
        biggest = 0.0
        for s, (have, n) in enumerate(zip(self.lens, self.counts)):
            if not n:
                continue
            first = int(self.cu[s])
            at = list(range(have)) + [have + d for d in depths(self.trees[s])]
            real = [True] * have + [i in self.sets[s][i] for i in range(n)]
            rows = [(int(self.table[s, j // self.page]), j % self.page) for j in range(have + n)]
            pages, offs = torch.tensor([a for a, _ in rows]), torch.tensor([b for _, b in rows])
            k = self.kv[0, pages, :, offs].double()             # [L, nkv, hd]
            v = self.kv[-1, pages, :, offs].double()
            f = torch.ones(have + n, self.kv_heads, dtype=torch.float64) if self.key_scale is None else self.key_scale[pages, :, offs].double()
            seen = torch.zeros((n, have + n), dtype=torch.bool)
            for i in range(n):
                low = window.lowest_visible(at[have + i])
                for j in range(have + n):
                    if not real[j] or at[j] < low:
                        continue
                    seen[i, j] = j < have or (j - have) in self.sets[s][i]
            dist = torch.tensor(at[have:])[:, None] - torch.tensor(at)[None, :]
            for h in range(self.heads):
                g = h // G
                q = self.q[first:first + n].view(n, self.heads, hd)[:, h].double()
                kk = torch.where(torch.tensor(real)[:, None], k[:, g], torch.zeros(()).double())
                vv = torch.where(torch.tensor(real)[:, None], v[:, g], torch.zeros(()).double())
                x = q @ kk.T * softmax_scale * torch.where(torch.tensor(real), f[:, g], torch.ones(()).double())
                biggest = max(biggest, float((q.abs() @ kk.abs().T).max()) * softmax_scale)
                if score_softcap:
                    x = score_softcap * torch.tanh(x / score_softcap)
                if head_slopes is not None:
                    x = x - float(head_slopes[h]) * dist
                if distance_rows is not None:
                    row = distance_rows[h].double()
                    x = x + row[dist.clamp(0, row.numel() - 1)]
                x = x.masked_fill(~seen, -math.inf)
                sink = head_sinks[h] if head_sinks is not None else sink_logit
                top = x.max(1, keepdim=True).values
                if sink is not None:
                    top = top.clamp(min=float(sink))
                top = torch.where(top == -math.inf, torch.zeros_like(top), top)
                w = torch.exp(x - top)
                total = w.sum(1, keepdim=True)
                if sink is not None:
                    total = total + torch.exp(float(sink) - top)
                w = w / total.clamp(min=1e-300)
                gate = 1.0 if head_gates is None else head_gates[first:first + n, h].double()[:, None]
                out[first:first + n, h] = w @ vv * gate
                size[first:first + n, h] = w @ vv.abs() * (gate if head_gates is None else gate.abs())
        return out.view(self.M, -1), size.view(self.M, -1), biggest


def tolerance(case: TreeCase, out, size, biggest, *, rounded_weights: bool):
    """How far an output element may be off, from the roundings that it takes: scores are sums of `size` products in float32 (and a few
    more operations), whose error, relative to the sum of the products' sizes, is below size / 2^24, and turns into a relative error
    of a weight twice (the weight and the maximum it is relative to); sums over n keys are added in tiles of at least 32; a weight
    may be rounded to bfloat16 (half a step, 2^-8), the result is."""
    keys = max([a + n for a, n in zip(case.lens, case.counts)] + [1])
    small = 2.0 ** -24 * (2 * (case.size + 8) * max(1.0, biggest) + keys / 8 + 64)
    if case.q.dtype == torch.bfloat16:
        return 2.0 ** -8 * out.abs() + (small + (2.0 ** -8 if rounded_weights else 0.0)) * size + 1e-30
    return small * size + 2.0 ** -24 * out.abs() + 1e-30


# ------------------------------------------------------------------ layout
def plain_layout(tables, held, page, window, free, n_free, slots, lengths, new, parents, width, n_words):
    """`layout_step` by loops over lists (changed in place: tables, held, free); returns (n_free, block_table, cu, positions, seg, slot_map, sets)."""
    for s, row in enumerate(slots):
        if row < 0 or free is None:
            continue
        low = held[row] if new[s] < 0 else min(held[row], window.first_needed(lengths[row]) // page)
        first = low
        while first > 0 and tables[row][first - 1] >= 0:
            first -= 1
        for j in range(first, low):
            free[n_free] = tables[row][j]
            n_free += 1
            tables[row][j] = -1
    for s, row in enumerate(slots):
        if row < 0 or free is None:
            continue
        need = 0 if new[s] < 0 else max(held[row], -(-(lengths[row] + new[s]) // page))
        have = 0 if new[s] < 0 else held[row]
        for j in range(have, need):
            n_free -= 1
            tables[row][j] = free[n_free]
        held[row] = need
    block, cu, pos, seg, slot, sets = [], [0], [], [], [], []
    for s, row in enumerate(slots):
        n = max(new[s], 0) if row >= 0 else 0
        block.append([-1] * width if row < 0 or new[s] < 0 else (tables[row] + [-1] * width)[:width])
        tree = list(range(-1, n - 1)) if parents is None else parents[cu[-1]:cu[-1] + n]
        mine = ancestor_sets(tree)
        sets += mine
        for i, d in enumerate(depths(tree)):
            place = lengths[row] + i
            pg = tables[row][place // page]
            pos.append(lengths[row] + d)
            seg.append(s)
            slot.append(pg * page + place % page if pg >= 0 and tree[i] >= -1 else -1)
        cu.append(cu[-1] + n)
    return n_free, block, cu, pos, seg, slot, words_of(sets, n_words) if n_words else None


# ------------------------------------------------------------------ acceptance
def plain_accept(tokens, parents, targets, cu, depth):
    """(counts, path, emitted) by loops."""
    counts, paths, emitted = [], [], []
    for s in range(len(cu) - 1):
        a, n = cu[s], cu[s + 1] - cu[s]
        par = list(range(-1, n - 1)) if parents is None else parents[a:a + n]
        path, at = [], 0 if n else None
        while at is not None and len(path) < depth:
            path.append(at)
            at = next((c for c in range(at + 1, n) if par[c] == at and tokens[a + c] == targets[a + at]), None)
        counts.append(len(path))
        paths.append(path + [-1] * (depth - len(path)))
        emitted.append([targets[a + i] for i in path] + [-1] * (depth - len(path)))
    return counts, paths, emitted
