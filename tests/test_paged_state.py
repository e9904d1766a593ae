"""The host side of a paged batch (no GPU is reached): what a step that fails
leaves behind."""

from types import SimpleNamespace

import pytest
import torch

from persona.mistral import MistralLoRAModel, PagedState


class _Fails:
    def index_select(self, *_):
        raise RuntimeError("a failed call")


def _state():
    return PagedState(slots=torch.zeros(3, dtype=torch.int32), page_size=4, page_table=torch.zeros(3, 4, dtype=torch.int32),
                      k_cache=[None], v_cache=[None], k_scale=[None], v_scale=[None], lengths=[0, 0, 0],
                      pages=[[], [], []], free=list(range(7)))


def test_a_step_that_fails_leaves_the_sequences_as_they_were():
    st = _state()
    st._grow([5, 0, 3])
    kept = (list(st.lengths), [list(p) for p in st.pages], list(st.free))
    model = SimpleNamespace(cfg=SimpleNamespace(vocab=50), device=torch.device("cpu"), embed=_Fails())
    model._extend_rows = lambda *a: MistralLoRAModel._extend_rows(model, *a)
    for chunks in ([[1], [2] * 9, [3] * 2], [[1] * 4, [], []], [[], [7], []]):
        with pytest.raises(RuntimeError, match="a failed call"):
            MistralLoRAModel.extend(model, st, chunks)
        assert (st.lengths, st.pages, st.free) == kept
    with pytest.raises(ValueError, match="no free pages"):
        MistralLoRAModel.extend(model, st, [[1] * 11, [1] * 16, [1] * 13])
    assert (st.lengths, st.pages, st.free) == kept
    # the next step that is carried out has its pages in the table
    st._grow([4, 1, 6])
    assert st.lengths == [9, 1, 9] and sorted(sum(st.pages, st.free)) == list(range(7))
    for b, p in enumerate(st.pages):
        assert st.page_table[b, :len(p)].tolist() == p
