"""Layouts that are refused for requests which hold pages: a slot twice, an ended row whose count of pages cannot be right.  Nothing changes, and the step is
empty.  (What is left of such a request on the way: tests/test_layout_refused.py.)"""
import pytest
import torch

from spite_b200.cache import Window
from spite_b200.kernels.api import StepLayout
from test_gpu_step_layout import State, ints, k  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests", [2, 40, 700])
def test_refused_requests_that_hold_pages(k, requests):  # noqa: F811
    rows = requests + 3
    st = State(rows, 8, 16, Window("sliding", 20), 8 * rows, seed=2)
    lengths = [50] * rows
    st.step(k, list(range(requests)), [0] * rows, [50] * requests)          # four pages each, of which the window has passed one

    def refused(slots, new, held=None):
        out = st.out(len(slots), 200)
        if held is not None:
            st.pages.held[slots[0]] = held
        k.layout_step(st.pages, ints(slots), ints(lengths), ints(new), out)
        if held is not None:
            assert int(st.pages.held[slots[0]]) == held
            st.pages.held[slots[0]] = 4
        assert int(out.status) == StepLayout.MALFORMED
        st.same()
        assert out.cu_seqlens.tolist() == [0] * (len(slots) + 1) and (out.block_table == -1).all()
        assert (out.positions == -9).all() and (out.slot_map == -9).all()

    others = list(range(2, requests))
    refused([0, 0] + others, [-1, -1] + [0] * len(others))    # twice, both ended
    refused([0, 0] + others, [-1, 1] + [0] * len(others))
    refused([1, 1] + others, [1, 1] + [0] * len(others))      # twice behind the window
    refused(others + [1, 1], [0] * len(others) + [0, -1])
    for held in (9, 4096, -1):                                # ended, with more pages than a row has, or fewer than none
        refused([0] + others, [-1] + [0] * len(others), held)
    st.step(k, [1, 0], lengths, [1, -1])                      # and goes on
