"""Steps that verify drafted trees on the GPU: the operators together, as a program uses them."""
import pytest
import torch

import helpers as H
import plain_llama4 as plain
import sezazen_helpers as S
from spite_b200.kernels.api import PageTables, StepLayout
from tree_kernels import drafts_from, drive

pytestmark = pytest.mark.gpu
# Of the logit scale.  The engine's tests hold every step's logits to 2e-5 (float32) and 2e-2 (bfloat16) of the plain implementation's; two steps that
# are both within that of it are within twice that of one another.
TOL = {"float32": 2 * 2e-5, "bfloat16": 2 * 2e-2}


def engine_of(folder, dtype, **kw):
    from spite_b200.engine import Engine, Model
    return Engine(Model.from_folder(folder, dtype=dtype, device="cuda:0"), **{**dict(cache_tokens=2048, page_size=64, max_requests=4), **kw})


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
@pytest.mark.parametrize("page_size", [16, 64])
def test_the_tokens_of_single_steps(tmp_path, name, page_size):
    """float32: whatever is drafted, the tokens are the plain implementation's greedy ones."""
    folder = H.write_model(tmp_path, name)
    cfg, tensors = plain.read_model_folder(folder)
    prompts = {q: H.random_tokens(cfg["vocab_size"], n, 30 + n) for q, n in (("a", 29), ("b", 1), ("c", 130), ("d", 63))}
    truth = {q: list(p) + plain.generate_greedy(cfg, tensors, p, 40) for q, p in prompts.items()}
    got, accepted = drive(engine_of(folder, "float32", page_size=page_size), prompts, 30, drafts_from(truth, cfg["vocab_size"], page_size, most=40), page_size)
    for q, p in prompts.items():
        assert got[q] == truth[q][len(p):len(p) + 30]
    assert accepted > 20


MODELS = [("A", H.write_model), ("C", H.write_model), ("D", H.write_model)] + [(n, S.write_model) for n in S.CONFIGS]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,write", MODELS, ids=[n for n, _ in MODELS])
def test_the_logits_of_single_steps(tmp_path, name, write, dtype):
    """The logits of every node on a way are those of decode steps along it; siblings and later drafts change nothing, also once they are cached."""
    import random
    folder = write(tmp_path, name)
    engine = engine_of(folder, dtype)
    vocab = engine.model.plan.vocab_size
    r = random.Random(5)
    text = [r.randrange(vocab) for _ in range(40 + 60)]
    for q in ("one", "tree"):
        engine.step([(q, text[:40], [])])
    singles = torch.stack([engine.step([("one", [t], [0])])[0].clone() for t in text[40:]])
    scale, at, worst = float(singles.abs().max()), 40, 0.0
    while at < len(text):
        n = min(r.randint(1, 24), len(text) - at)
        tokens, parents, way = [text[at]], [-1], [0]
        for t in text[at + 1:at + n]:
            for _ in range(r.randint(0, 2)):                 # wrong drafts beside the way and below it
                tokens.append((t + 1 + r.randrange(vocab - 1)) % vocab)
                parents.append(r.randrange(len(tokens) - 1))
            tokens.append(t)
            parents.append(way[-1])
            way.append(len(tokens) - 1)
        kept = []

        def targets(logits):
            kept.append(logits.clone())
            want = torch.full((len(tokens),), vocab, dtype=torch.int32)          # (no drafted token is that)
            for node, t in zip(way, text[at + 1:at + n]):
                want[node] = t
            want[way[-1]] = text[at + n] if at + n < len(text) else 0
            return want.to(logits.device)
        assert engine.verify([("tree", tokens, parents)], targets)[0] == (text[at + 1:at + n + 1] + [0])[:n]
        worst = max(worst, float((kept[0][way] - singles[at - 40:at - 40 + n]).abs().max()) / scale)
        at += n
    assert worst <= TOL[dtype], f"{worst:.2e} of the logit scale"


def test_a_loop_that_the_host_does_not_look_into():
    """Layout, attention, acceptance and layout again on a device-side stack of pages: lengths and pages come out as the drafts were accepted, and the
    attention of the second step finds the accepted rows where the first step's nodes were moved from."""
    from draft_helpers import TreeCase, tolerance
    from spite_b200.cache import LayerCache, Window
    from spite_b200.engine.batch import StepBatch
    from spite_b200.kernels.cuda import CudaKernels
    dev, dtype, heads, kv_heads, size, page = "cuda:0", torch.bfloat16, 8, 2, 128, 64
    k = CudaKernels(dtype, dev)
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=dev)
    g = torch.Generator(device=dev).manual_seed(3)
    kv = torch.randn((1, 2, 20, kv_heads, page, size), generator=g, device=dev).to(dtype)
    pages = PageTables(tables=ints([[-1] * 6] * 3), held=ints([0, 0, 0]), page_size=page, window=Window("full"), free_pages=ints(list(range(20))), n_free=ints([20]))
    lengths, slots = ints([0, 0, 0]), ints([2, 0])
    blank = lambda *shape, t=torch.int32: torch.zeros(shape, dtype=t, device=dev)
    out = StepLayout(block_table=blank(2, 6), cu_seqlens=blank(3), positions=blank(300), seg_of_token=blank(300), slot_map=blank(300, t=torch.int64), status=blank(1),
                     ancestors=blank(300, 1))
    # a prompt each, written by the slot map
    k.layout_step(pages, slots, lengths, ints([100, 63]), StepLayout(**{**out.__dict__, "ancestors": None}))
    prompt = torch.randn((163, 2, kv_heads, size), generator=g, device=dev).to(dtype)
    kv[0][:, out.slot_map[:163] // page, :, out.slot_map[:163] % page] = prompt
    lengths.copy_(ints([63, 0, 100]))
    text = [[prompt[:100]], [prompt[100:]]]
    for step in range(6):
        new = ints([5, 3])
        parents = ints([-1, 0, 0, 2, 3, -1, 0, 1])
        k.layout_step(pages, slots, lengths, new, out, parents=parents)
        rows = torch.randn((8, 2, kv_heads, size), generator=g, device=dev).to(dtype)
        kv[0][:, out.slot_map[:8] // page, :, out.slot_map[:8] % page] = rows
        q = torch.randn((300, heads * size), generator=g, device=dev).to(dtype)
        o = torch.zeros_like(q)
        batch = StepBatch(n_tokens=300, segments=[], token_ids=None, positions=out.positions, seg_of_token=out.seg_of_token, cu_seqlens=out.cu_seqlens, slots=None,
                          logit_rows=None, block_tables=[out.block_table], ancestors=out.ancestors)
        k.tree_attention(q, o, batch, LayerCache(0, kv[0], None, page, False), num_heads=heads, window=Window("full"), softmax_scale=size ** -0.5)
        counts, path, emitted = blank(2), blank(2, 5), blank(2, 5)
        k.accept_drafts(ints([9, 1, 2, 3, 4, 9, 5, 6]), parents, ints([2, 0, 3, 4, 7, 5, 8, 8]), out.cu_seqlens, [(kv, out.slot_map, None)], counts=counts, path=path,
                        emitted=emitted, slots=slots, lengths=lengths, lengths_out=lengths)
        assert int(out.status) == 0 and counts.tolist() == [4, 2] and path.tolist() == [[0, 2, 3, 4, -1], [0, 1, -1, -1, -1]]
        assert emitted.tolist() == [[2, 3, 4, 7, -1], [5, 8, -1, -1, -1]]
        # the attention's result from the rows themselves
        have = [sum(t.shape[0] for t in x) for x in text]
        case = TreeCase(have, [5, 3], heads=heads, kv_heads=kv_heads, size=size, dtype=dtype, trees=[[-1, 0, 0, 2, 3], [-1, 0, 1]])
        case.q = q[:8].cpu()
        for s, (a, b) in enumerate(((0, 5), (5, 8))):
            for j, row in enumerate(torch.cat(text[s] + [rows[a:b]]).cpu()):
                case.kv[:, int(case.table[s, j // page]), :, j % page] = row
        want, weight, biggest = case.plain(Window("full"), size ** -0.5)
        assert ((o[:8].double().cpu() - want).abs() <= tolerance(case, want, weight, biggest, rounded_weights=True)).all() and (o[8:] == 0).all()
        text[0].append(rows[[0, 2, 3, 4]])
        text[1].append(rows[[5, 6]])
    assert lengths.tolist() == [63 + 12, 0, 100 + 24] and pages.held.tolist() == [2, 0, 2]
