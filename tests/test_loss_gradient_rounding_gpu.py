"""How far gradients of ops.linear_cross_entropy are off beside the rounding of their own type, at sizes of every tile."""
import pytest
import torch

from tests.test_linear_cross_entropy_gpu import BF16, F16, _inputs, _exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,times", [(F16, 1.1), (BF16, 1.05)])
@pytest.mark.parametrize("n,d,v", [(20, 130, 400), (257, 768, 50000), (2047, 768, 6000), (4100, 256, 9000)])
def test_gradients_are_off_by_their_rounding(n, d, v, dtype, times):
    """fp16: G's two halves hold 22 bits, so what is left are fp32 sums: a tenth of the rounding with room.  bf16: G's 11 bits are off by an eighth of
    what a bf16 result is, where a result hangs on one entry of G, as a label's row of dw does: sqrt(1 + 1/64) = 1.008, and 1.05 with room."""
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(n, d, v, dtype, seed=11)
    if dtype == F16:
        weights = weights * 64      # (out of fp16's subnormals)
    x.requires_grad_(), w.requires_grad_()
    got = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels, reduction="none"), (x, w), weights)
    _, (dx, _), (dw, _) = _exact(x.detach(), w.detach(), labels, "none", weights)
    for g, e in zip(got, (dx, dw)):
        assert float((g.double() - e).norm()) <= times * float((e.to(dtype).double() - e).norm())
