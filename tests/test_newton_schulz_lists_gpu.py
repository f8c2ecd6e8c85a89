"""Lists of matrices that ops.newton_schulz copies before it launches: the bits of contiguous ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _turned(m, n, seed, dtype=torch.float32):
    return torch.randn(n, m, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype).t()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sizes", [[(200, 300)] * 3, [(300, 200), (24, 512), (300, 200), (41, 50), (24, 512), (700, 130)], [(8, 16)] * 60])
def test_transposed_matrices_of_a_list(sizes, dtype):
    from native_sparse_attention_pytorch_amd import ops
    given = [_turned(m, n, i, dtype) for i, (m, n) in enumerate(sizes)]
    want = ops.newton_schulz([g.contiguous() for g in given])
    for o, w in zip(ops.newton_schulz(given), want):
        assert torch.equal(o, w)


def test_transposed_batches_among_them():
    from native_sparse_attention_pytorch_amd import ops
    wide = torch.randn(3, 120, 90, device=DEV)
    given = [_turned(130, 140, 0), wide[:, :, 3:70], wide.transpose(1, 2), _turned(130, 140, 1), wide[0, ::2, 1:]]
    want = ops.newton_schulz([g.contiguous() for g in given])
    for o, w in zip(ops.newton_schulz(given), want):
        assert torch.equal(o, w)


def test_muon_of_transposed_parameters():
    """A step of parameters stored transposed is that of contiguous ones."""
    from native_sparse_attention_pytorch_amd.training import Muon
    sizes = [(130, 70), (130, 70), (24, 100)]
    moved = []
    for make in (lambda t: t, lambda t: t.contiguous()):
        params = [torch.nn.Parameter(make(_turned(m, n, i))) for i, (m, n) in enumerate(sizes)]
        opt = Muon(params, lr=0.1)
        for step in range(2):
            for i, p in enumerate(params):
                p.grad = make(_turned(*p.shape, 10 * step + i + 3))
            opt.step()
        moved.append([p.detach() for p in params])
    for a, b in zip(*moved):
        assert torch.equal(a, b)


def test_matrices_of_one_row():
    """(8, 1).t() has one row and a row stride of 1."""
    from native_sparse_attention_pytorch_amd import ops
    for given in (torch.randn(8, 1, device=DEV).t(), torch.randn(3, 500, 1, device=DEV).mT, torch.randn(70000, 1, device=DEV).t()):
        for o, w in zip(ops.newton_schulz([given, given]), ops.newton_schulz([given.clone(memory_format=torch.contiguous_format)] * 2)):
            assert torch.equal(o, w) and o.isfinite().all()
