"""The stand-in kernel set of `reference_kernels.py` with the operators of a step that verifies drafted tokens, for the engine's host logic
on a machine without a GPU."""
from __future__ import annotations

import dataclasses

import torch

from draft_helpers import plain_accept, plain_layout
from reference_kernels import TorchReferenceKernels
from spite_b200.cache import LayerCache


class TreeReferenceKernels(TorchReferenceKernels):
    def layout_step(self, pages, slots, lengths, new_tokens, out, *, parents=None):
        tables, held = pages.tables.tolist(), pages.held.tolist()
        free = None if pages.free_pages is None else pages.free_pages.tolist()
        words = 0 if out.ancestors is None else out.ancestors.shape[1]
        _, block, cu, pos, seg, slot, sets = plain_layout(
            tables, held, pages.page_size, pages.window, free, 0 if free is None else int(pages.n_free), slots.tolist(), lengths.tolist(),
            new_tokens.tolist(), None if parents is None else parents.tolist(), out.block_table.shape[1], words)
        assert free is None
        out.status.zero_()
        out.block_table.copy_(torch.tensor(block, dtype=torch.int32))
        out.cu_seqlens.copy_(torch.tensor(cu, dtype=torch.int32))
        for t, v in ((out.positions, pos), (out.seg_of_token, seg), (out.slot_map, slot)):
            t[:len(v)] = torch.tensor(v, dtype=t.dtype)
        if words:
            out.ancestors[:len(sets)] = torch.tensor(sets, dtype=torch.int32)

    def qk_prepare(self, qkv, q_out, batch, cache, **kw):
        if batch.slot_maps is None or not cache.write:
            return super().qk_prepare(qkv, q_out, batch, cache, **kw)
        # into a page of its own for every token, and from there to the row that the slot map names
        M, kv = qkv.shape[0], cache.kv
        P = kv.shape[3]
        tmp = torch.zeros((kv.shape[0], M) + tuple(kv.shape[2:]), dtype=kv.dtype)
        scales = None if cache.key_scale is None else torch.zeros((M,) + tuple(cache.key_scale.shape[1:]))
        own = torch.arange(M, dtype=torch.int32)
        width = int(batch.positions.max()) // P + 1
        proxy = dataclasses.replace(batch, seg_of_token=own, block_tables=[own[:, None].expand(M, width)] * len(batch.block_tables), slot_maps=None)
        super().qk_prepare(qkv, q_out, proxy, LayerCache(cache.group, tmp, cache.state, P, True, scales), **kw)
        for t in range(M):
            slot, at = int(batch.slot_maps[cache.group][t]), int(batch.positions[t]) % P
            kv[:, slot // P, :, slot % P] = tmp[:, t, :, at]
            if scales is not None:
                cache.key_scale[slot // P, :, slot % P] = scales[t, :, at]

    def tree_attention(self, q, out, batch, cache, *, num_heads, window, softmax_scale, sink_logit=None, head_sinks=None, head_slopes=None, head_gates=None,
                       out_by_head=False, score_softcap=None, distance_bias=None):
        assert not out_by_head
        kv, P, hd = cache.kv, cache.kv.shape[3], cache.kv.shape[4]
        group = num_heads // kv.shape[2]
        pos, seg, cu, table = batch.positions.tolist(), batch.seg_of_token.tolist(), batch.cu_seqlens.tolist(), batch.block_tables[cache.group].tolist()
        for t in range(cu[-1]):
            first = cu[seg[t]]
            have, low = pos[first], window.lowest_visible(pos[t])
            nodes = [a for a in range(t - first + 1) if int(batch.ancestors[t, a // 32]) >> (a % 32) & 1]
            places = [(j, j) for j in range(low, have)] + [(have + a, pos[first + a]) for a in nodes if pos[first + a] >= low]
            rows = torch.tensor([(table[seg[t]][j // P], j % P) for j, _ in places])
            assert bool((rows[:, 0] >= 0).all()), "read from a page that was given back"
            dist = pos[t] - torch.tensor([p for _, p in places])
            K, V = kv[0, rows[:, 0], :, rows[:, 1]].to(self.acc), kv[-1, rows[:, 0], :, rows[:, 1]].to(self.acc)
            for h in range(num_heads):
                s = K[:, h // group] @ q[t].view(num_heads, hd)[h].to(self.acc) * softmax_scale
                if cache.key_scale is not None:
                    s = s * cache.key_scale[rows[:, 0], h // group, rows[:, 1]]
                if score_softcap:
                    s = score_softcap * torch.tanh(s / score_softcap)
                if head_slopes is not None:
                    s = s - float(head_slopes[h]) * dist
                if distance_bias is not None:
                    s = s + distance_bias.padded[h, distance_bias.PAD + dist.clamp(max=distance_bias.length - 1)]
                sink = sink_logit if head_sinks is None else float(head_sinks[h])
                w = torch.softmax(s if sink is None else torch.cat([s, s.new_tensor([sink])]), 0)[:len(places)]
                o = w @ V[:, h // group]
                out[t, h * hd:(h + 1) * hd] = (o if head_gates is None else o * head_gates[t, h]).to(out.dtype)

    def accept_drafts(self, tokens, parents, targets, cu_seqlens, caches, *, counts, path, emitted, slots=None, lengths=None, lengths_out=None):
        cu = cu_seqlens.tolist()
        n, paths, out = plain_accept(tokens.tolist(), None if parents is None else parents.tolist(), targets.tolist(), cu, path.shape[1])
        for t, v in ((counts, n), (path, paths), (emitted, out)):
            t.copy_(torch.tensor(v, dtype=torch.int32))
        for kv, slot_map, scales in caches:
            P, places = kv.shape[4], slot_map.tolist()
            for s in range(len(n)):
                for d in range(n[s]):
                    a, b = places[cu[s] + paths[s][d]], places[cu[s] + d]
                    kv[:, :, b // P, :, b % P] = kv[:, :, a // P, :, a % P].clone()
                    if scales is not None:
                        scales[:, b // P, :, b % P] = scales[:, a // P, :, a % P].clone()


def drive(engine, prompts: dict, n: int, draft, seed=0) -> dict:
    """`n` next tokens of every request by verified steps; `draft(request, text so far)` gives a tree over its next token.  Some requests sit a step out."""
    import random
    r = random.Random(seed)
    out, accepted = {}, 0
    for req, p in prompts.items():
        if len(p) > 1:
            engine.step([(req, p[:-1], [])])
    text = {q: list(p) for q, p in prompts.items()}
    out = {q: [] for q in prompts}
    while any(len(v) < n for v in out.values()):
        live = [q for q in prompts if len(out[q]) < n and (r.random() < 0.8 or len(prompts) == 1)]
        if not live:
            continue
        trees = []
        for q in live:
            tokens, parents = draft(q, text[q])
            trees.append((q, tokens, parents))
        for q, got in zip(live, engine.verify(trees)):
            assert got
            accepted += len(got) - 1
            out[q] += got
            text[q] += got
            assert engine.cached_tokens(q) == len(text[q]) - 1
        engine.cache.check_invariants()
    for q in prompts:
        engine.finish(q)
    engine.cache.check_invariants()
    return {q: v[:n] for q, v in out.items()}, accepted


def drafts_from(truth: dict, vocab: int, seed=0, most=12):
    """Trees that often hold the right continuation (`truth`[request], the greedy tokens) among wrong ones."""
    import random
    r = random.Random(seed)

    def draft(q, text):
        rest = truth[q][len(text):] if len(truth[q]) > len(text) else []
        tokens, parents = [text[-1]], [-1]
        right = 0                                            # the last node of the right way
        for i in range(r.randint(0, most)):
            if rest and r.random() < 0.5:
                tokens.append(rest.pop(0))
                parents.append(right)
                right = len(tokens) - 1
            else:
                tokens.append(r.randrange(vocab))
                parents.append(r.randrange(len(tokens) - 1))
        return tokens, parents
    return draft
