"""Steps that verify drafted trees, on the host: the kernels are replaced by their plain restatements, everything else is the product code.  Greedy
tokens have to be those that the plain implementation produces one by one, whatever was drafted."""
import pytest
import torch

import helpers as H
import plain_llama4 as plain
from spite_b200.cache import CacheError, CacheManager, OutOfPages, Window
from spite_b200.cache.manager import GroupKey
from spite_b200.engine import ContextOverflow, DraftTree, Engine, Model, StepError
from tree_kernels import TreeReferenceKernels, drafts_from, drive


@pytest.fixture(scope="module", params=["A", "B"])
def setup(request, tmp_path_factory):
    folder = H.write_model(tmp_path_factory.mktemp(f"model{request.param}"), request.param)
    model = Model.from_folder(folder, dtype="float32", device="cpu", kernels=TreeReferenceKernels(torch.float32, "cpu"))
    cfg, tensors = plain.read_model_folder(folder)
    prompts = {q: H.random_tokens(cfg["vocab_size"], n, 30 + n) for q, n in (("a", 29), ("b", 1), ("c", 40))}
    truth = {q: list(p) + plain.generate_greedy(cfg, tensors, p, 24) for q, p in prompts.items()}
    return model, prompts, truth


@pytest.mark.parametrize("page_size,seed", [(16, 0), (5, 1), (64, 2)])
def test_the_tokens_of_single_steps(setup, page_size, seed):
    """Trees cross pages and chunks of the attention; requests come and go; the accepted rows are where later steps expect them."""
    model, prompts, truth = setup
    engine = Engine(model, cache_tokens=512, page_size=page_size, max_requests=4)
    got, accepted = drive(engine, prompts, 20, drafts_from(truth, model.plan.vocab_size, seed), seed)
    for q, p in prompts.items():
        assert got[q] == truth[q][len(p):len(p) + 20]
    assert accepted > 10


def test_other_targets(setup):
    """The way follows whatever `targets` says."""
    model, prompts, _ = setup
    engine = Engine(model, cache_tokens=256, page_size=16, max_requests=2)
    engine.step([("a", prompts["a"][:9], [])])
    seen = []

    def targets(logits):
        seen.append(tuple(logits.shape))
        return torch.tensor([5, 7, 9, 11, 3], dtype=torch.int32)
    assert engine.verify([DraftTree("a", [1, 5, 5, 9, 11], [-1, 0, 0, 2, 3])], targets) == [[5, 7]]       # the first of two equal children
    assert seen == [(5, model.plan.vocab_size)] and engine.cached_tokens("a") == 11
    assert engine.verify([DraftTree("a", [7, 5, 7, 11, 3], [-1, 0, 1, 2, 3])], targets) == [[5, 7, 9]]


def test_a_step_that_cannot_run_changes_nothing(setup):
    model, prompts, _ = setup
    engine = Engine(model, cache_tokens=64, page_size=16, max_requests=2, max_positions=50)
    engine.step([("a", prompts["a"][:20], [])])
    before = (engine.cached_tokens("a"), engine.cache.free_pages())
    vocab = model.plan.vocab_size
    for trees, error in (([("a", [1, 2], [-1, 1])], StepError), ([("a", [1, 2], [0, 0])], StepError), ([("a", [1, 2], [-1])], StepError), ([("a", [], [])], StepError),
                         ([("a", [1], [-1]), ("a", [1], [-1])], StepError), ([("a", [vocab], [-1])], StepError), ([("a", [1] * 31, [-1] + [0] * 30)], ContextOverflow),
                         ([("a", [1], [-1]), ("b", [1] * 50, [-1] + [0] * 49)], OutOfPages)):
        with pytest.raises(error):
            engine.verify(trees)
        engine.cache.check_invariants()
        assert (engine.cached_tokens("a"), engine.cache.free_pages()) == before and not engine.is_live("b")
    assert engine.verify([]) == []

    def broken(logits):
        raise RuntimeError("no targets")
    with pytest.raises(RuntimeError):
        engine.verify([("a", [1, 2], [-1, 0])], broken)
    assert (engine.cached_tokens("a"), engine.cache.free_pages()) == before


def test_models_with_a_state_are_refused(tmp_path):
    import paposun_helpers as P
    name = next(iter(P.CONFIGS))
    folder = P.write_model(tmp_path, name)
    model = Model.from_folder(folder, dtype="float32", device="cpu", kernels=TreeReferenceKernels(torch.float32, "cpu"))
    engine = Engine(model, cache_tokens=64, page_size=16, max_requests=2)
    with pytest.raises(StepError):
        engine.verify([("a", [1], [-1])])
    assert not engine.is_live("a")


@pytest.mark.parametrize("window", [Window("full"), Window("sliding", 20), Window("chunk", 24)], ids=lambda w: w.kind)
def test_commit_of_a_part(window):
    """Only the kept tokens are cached, the pages behind them go back, and the next reserve takes up from there."""
    m = CacheManager([GroupKey(window, 1, 8)], 8, 40, 2)
    m.admit("r")
    n = 0
    for new, kept in ((30, 30), (17, 1), (9, 9), (25, 3), (1, 1), (40, 0), (12, 11)):
        m.reserve("r", new)
        m.commit("r", kept)
        n += kept
        m.check_invariants()
        rc = m.get("r")
        assert rc.n_tokens == n and len(rc.tables[0]) == -(-n // 8)
        low = window.first_needed(n) // 8
        assert all(p < 0 for p in rc.tables[0][:low]) and all(p >= 0 for p in rc.tables[0][low:])
    m.reserve("r", 3)
    for bad in (-1, 4):
        with pytest.raises(CacheError):
            m.commit("r", bad)
    m.rollback("r")
