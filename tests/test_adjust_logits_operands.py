"""What `ops.adjust_logits` takes for numbers of the rows, with a stand-in for the library; no GPU."""
import pytest
import torch

from tests.test_serving_operands import library                               # noqa: F401 (a fixture)

NAMES = ["repetition_penalty", "frequency_penalty", "presence_penalty", "temperature"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("lead, given", [((2, 3), (3, 2)), ((4,), (2, 2)), ((2, 3, 2), (3, 2, 2)), ((2, 3), (2, 1)), ((2, 3), (3,)), ((2, 3, 2), (2, 6)),
                                         ((2, 3, 2), (6, 2)), ((2, 6), (3, 4)), ((2, 1, 3), (3, 2)), ((2, 1, 3), (3, 1, 2))])
def test_numbers_of_other_rows_are_refused(library, lead, given, name):  # noqa: F811
    """As many values as rows are not enough: in another shape they may be in another order."""
    from native_sparse_attention_pytorch_amd import ops
    with pytest.raises(RuntimeError, match=f"adjust_logits: {name}"):
        ops.adjust_logits(torch.zeros(*lead, 5), **{name: torch.ones(given)})
    assert not library.calls


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("lead, given", [((2, 3), (2, 3)), ((2, 3), (6,)), ((2, 3), (1, 1)), ((2, 3), ()), ((2, 3), (1,)), ((4,), (4,)), ((), ()), ((), (1,)), ((1, 1), (1,)), ((4, 1), (4, 1)),
                                         ((1, 3), (3,)), ((2, 3), (1, 6)), ((2, 3), (6, 1)), ((4, 1), (1, 4)), ((1, 3), (3, 1)), ((2, 1, 3), (2, 3)), ((2, 1, 3), (1, 2, 3))])
def test_numbers_of_the_rows_are_taken(library, lead, given, name):  # noqa: F811
    """In the rows' shape, or all along one axis, or one for all; axes of one value may be anywhere."""
    from native_sparse_attention_pytorch_amd import ops
    ops.adjust_logits(torch.zeros(*lead, 5), **{name: torch.ones(given)})
    assert [call for call, _ in library.calls] == ["nsa_adjust_logits"]
