"""Which memory ops.newton_schulz and training.Muon name to the library, without a GPU: every address is that of a matrix that is alive at the launch."""
import pytest
import torch

from tests.stand_in import stand_in  # noqa: F401


def _turned(m, n, seed):
    """'m n' with the strides of its transpose."""
    return torch.randn(n, m, generator=torch.Generator().manual_seed(seed)).t()


@pytest.mark.parametrize("sizes", [[(200, 300)] * 3, [(300, 200), (40, 50), (300, 200), (41, 50), (24, 512)], [(8, 16)] * 60])
def test_copies_live_until_the_launch(stand_in, sizes):
    """A list of matrices whose rows are not contiguous: each copy has memory of its own."""
    from native_sparse_attention_pytorch_amd import ops
    given = [_turned(m, n, i) for i, (m, n) in enumerate(sizes)]
    got = ops.newton_schulz(given)
    (_, addresses, _), = stand_in.calls
    assert len(set(addresses)) == len(given)
    for o, g in zip(got, given):
        assert torch.equal(o, 2 * g)


def test_batches_and_views_among_them(stand_in):
    from native_sparse_attention_pytorch_amd import ops
    wide = torch.randn(3, 20, 90)
    given = [_turned(30, 40, 0), wide[:, :, 3:70], wide.transpose(1, 2), _turned(30, 40, 1), torch.randn(5, 6)[None].expand(3, 5, 6), wide[0, ::2, 1:]]
    for o, g in zip(ops.newton_schulz(given), given):
        assert o.shape == g.shape and o.is_contiguous() and torch.equal(o, 2 * g)


def test_muon_of_transposed_parameters(stand_in):
    """Parameters stored transposed: their momenta and updates have their strides."""
    from native_sparse_attention_pytorch_amd.training import Muon
    params = [torch.nn.Parameter(_turned(30, 20, i)) for i in range(3)]
    before, grads = [p.detach().clone() for p in params], [_turned(30, 20, 10 + i) for i in range(3)]
    for p, g in zip(params, grads):
        p.grad = g
    Muon(params, lr=0.1, momentum=0.5, nesterov=False).step()
    for p, b, g in zip(params, before, grads):
        torch.testing.assert_close(p.detach(), b - 0.1 * 1.5 ** 0.5 * 2 * g)


@pytest.mark.parametrize("make", [lambda: torch.randn(8, 1).t(), lambda: torch.randn(3, 8, 1).mT, lambda: torch.randn(8, 1), lambda: torch.randn(1)[None].expand(1, 1),
                                  lambda: torch.randn(5, 1, 8)[:, :, :1], lambda: torch.randn(8).as_strided((1, 8), (0, 1)), lambda: torch.randn(2, 8, 1).mT.unsqueeze(0)])
def test_matrices_of_one_row_or_column(stand_in, make):
    """Where a matrix has one row, torch calls it contiguous whatever that row's stride."""
    from native_sparse_attention_pytorch_amd import ops
    given = make()
    for o in (ops.newton_schulz(given), ops.newton_schulz([given, given])[1]):
        assert torch.equal(o, 2 * given)
