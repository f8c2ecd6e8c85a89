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


@pytest.mark.parametrize("kind", [torch.int64, torch.int32])
@pytest.mark.parametrize("lead", [(3,), (1,), (2, 3), ()])
def test_a_history_that_grows_is_looked_up(library, lead, kind):  # noqa: F811
    """A sequence is one token longer at each step: the checks and the descriptor of the first serve the others, with the length of each."""
    from native_sparse_attention_pytorch_amd import ops
    logits = torch.zeros(*lead, 40)
    for t in range(0, 300):
        ops.adjust_logits(logits, torch.zeros(*lead, t, dtype=kind), repetition_penalty=1.2)
        name, args = library.calls[-1]
        desc = ops._LOGITS_DESC.unpack(args[0])
        assert name == "nsa_adjust_logits" and desc[:6] == (logits.numel() // 40, 40, 40, 2, t, kind == torch.int64)
    assert ops._logits_plan.cache_info().misses == 1
    wide = torch.zeros(*lead, 80, dtype=kind)[..., ::2]                          # not contiguous: copied, and a plan of its own
    ops.adjust_logits(logits, wide, repetition_penalty=1.2)
    assert library.calls[-1][1][2] != wide.data_ptr() and ops._LOGITS_DESC.unpack(library.calls[-1][1][0])[4] == 40
    with pytest.raises(RuntimeError, match="adjust_logits: history"):
        ops.adjust_logits(logits, torch.zeros((), dtype=kind))


def test_sampling_looks_up_what_it_does_to_logits(library, monkeypatch):  # noqa: F811
    """`Transformer.sample` hands in the tokens so far; the prompt's logits lie further apart than a token's."""
    from native_sparse_attention_pytorch_amd import ops
    from native_sparse_attention_pytorch_amd.transformer import Transformer
    model = Transformer(num_tokens=40, dim=64, depth=1, dim_head=64, heads=1, kv_heads=1)
    monkeypatch.setattr(Transformer, "forward", lambda self, ids, cache=None, return_cache=False: (torch.zeros(2, ids.shape[1] if cache is None else 1, 40), []))
    model.sample(torch.zeros(2, 5, dtype=torch.long), 30, temperature=0., presence_penalty=0.5, use_cache_kv=True)
    assert [ops._LOGITS_DESC.unpack(args[0])[4] for _, args in library.calls] == list(range(5, 30))
    assert ops._logits_plan.cache_info().misses == 2
