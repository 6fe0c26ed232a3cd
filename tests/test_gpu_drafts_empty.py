"""Steps of drafted tokens with nothing in them, and trees beyond what a request may bring."""
import pytest
import torch

from spite_b200.cache import Window
from spite_b200.kernels.api import KernelError, StepLayout
from test_gpu_step_layout import State, ints, k  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_no_parents_are_not_chains(k):  # noqa: F811
    """`parents` without elements are fewer than the step's tokens, and enough where it has none."""
    st = State(2, 8, 16, Window("full"), 10)
    none = ints([])
    out = st.out(2, 20, 1)
    k.layout_step(st.pages, ints([0, 1]), ints([0, 0]), ints([3, 0]), out, parents=none)
    assert int(out.status) == StepLayout.MALFORMED and out.cu_seqlens.tolist() == [0, 0, 0]
    st.same()
    out = st.out(2, 20, 1)
    k.layout_step(st.pages, ints([0, -1]), ints([0, 0]), ints([0, 3]), out, parents=none)
    assert int(out.status) == 0 and out.cu_seqlens.tolist() == [0, 0, 0]
    st.same()


@pytest.mark.parametrize("chain", [False, True])
def test_a_step_without_tokens(k, chain):  # noqa: F811
    """No request has accepted anything, lengths stay as they are, nothing moves."""
    kv = torch.ones((1, 2, 2, 1, 16, 8), dtype=torch.bfloat16, device=DEV)
    none = ints([])
    out = dict(counts=ints([9, 9]), path=ints([[9, 9]] * 2), emitted=ints([[9, 9]] * 2))
    lengths, lengths_out = ints([5, 6, 7]), ints([0, 0, 0])
    k.accept_drafts(none, None if chain else none, none, ints([0, 0, 0]), [(kv, ints([], torch.int64), None)], **out, slots=ints([2, 0]), lengths=lengths,
                    lengths_out=lengths_out)
    assert out["counts"].tolist() == [0, 0] and out["path"].tolist() == [[-1, -1]] * 2 and out["emitted"].tolist() == [[-1, -1]] * 2
    assert lengths_out.tolist() == [5, 0, 7] and (kv == 1).all()
    st = State(3, 8, 16, Window("full"), 10)
    out = st.out(2, 0)
    k.layout_step(st.pages, ints([2, -1]), lengths, ints([-1, 4]), out)
    assert int(out.status) == 0 and out.cu_seqlens.tolist() == [0, 0, 0]
    with pytest.raises(KernelError):
        k.accept_drafts(none, ints([1]), none, ints([0, 0]), [], counts=ints([0]), path=ints([[0]]), emitted=ints([[0]]))


def test_a_way_ends_in_front_of_node_1024(k):  # noqa: F811
    """Nodes from 1,024 on are not looked at: what is returned is the beginning of the way."""
    n = 1100
    parents = [-1] + list(range(1099))
    out = dict(counts=ints([9]), path=torch.full((1, 1024), -9, dtype=torch.int32, device=DEV), emitted=torch.full((1, 1024), -9, dtype=torch.int32, device=DEV))
    k.accept_drafts(ints([1] * n), ints(parents), ints([1] * n), ints([0, n]), [], **out)
    assert out["counts"].tolist() == [1024] and out["path"].tolist() == [list(range(1024))]
    parents = [-1, 0] + [1] * 1096 + [1, 1098]                # the only child that fits is node 1,098
    tokens = [1, 1] + [2] * 1096 + [1, 1]
    k.accept_drafts(ints(tokens), ints(parents), ints([1] * n), ints([0, n]), [], **out)
    assert out["counts"].tolist() == [2] and out["path"].tolist() == [[0, 1] + [-1] * 1022]
