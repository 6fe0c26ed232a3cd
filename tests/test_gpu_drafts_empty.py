"""Steps of drafted tokens with nothing in them."""
import pytest

from spite_b200.cache import Window
from spite_b200.kernels.api import StepLayout
from test_gpu_step_layout import State, ints, k  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


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
