"""ops.linear_cross_entropy where rows of one call weigh very differently: each row's dx against float64 within a bound of its own row.

A row's G, each entry off by two logits' dL, 2^-16 and 2^-22 of the distance in front of an exponential (rel), is held in 11 bits (bf16) or 22 down to
2^-38 of the row's largest entry; the rest as in tests/test_linear_cross_entropy_gpu.py.  For dw a row of x is multiplied by what the row's G weighs
beside the largest row's, so a term G x is off by 2^-38 of the largest of all, and once more for G itself."""
import pytest
import torch

from tests.test_linear_cross_entropy_gpu import BF16, F16, F32, DEV, _inputs, _within

pytestmark = pytest.mark.gpu


def _bounds(x, w, labels, weights):
    """float64 (dx, tolerance), (dw, tolerance) of the losses' sum weighted with `weights`; no row is ignored."""
    h, u = (2 ** -22, 2 ** -24) if x.dtype == F32 else (0., torch.finfo(x.dtype).eps / 2)
    n, d, v = *x.shape, len(w)
    x6, w6, g, at = x.double(), w.double(), weights.double()[:, None], labels[:, None]
    logits, size = x6 @ w6.t().contiguous(), x6.abs() @ w6.abs().t().contiguous()
    far = logits - logits.gather(1, at)
    others = torch.exp(far).scatter(1, at, 0.)
    r = others.sum(-1, keepdim=True)
    rel = 2 * (((d / 4 + 8) * 2 ** -24 + 2 * h) * size).amax(-1, keepdim=True) + 2 ** -16 + 2 ** -22 * far.abs().amax(-1, keepdim=True)
    G = g * (others / (1 + r)).scatter(1, at, -r / (1 + r))
    dG = G.abs() * (2 * rel + (2 ** -11 if x.dtype == BF16 else 2 ** -22)) + 2 ** -38 * G.abs().amax(-1, keepdim=True)
    floor = 2. ** -25 if x.dtype == F16 else torch.finfo(x.dtype).tiny
    dx, Gt = G @ w6, G.t().contiguous()
    tx = dG @ w6.abs() + G.abs() @ ((h + (v / 4 + 16) * 2 ** -24) * w6.abs() + 2 ** -38 * float(w6.abs().max()))
    dw = Gt @ x6
    tw = dG.t().contiguous() @ x6.abs() + Gt.abs() @ ((h + (n / 4 + 16) * 2 ** -24) * x6.abs()) + n * 2 ** -37 * float(G.abs().max() * x6.abs().max())
    return (dx, 1.01 * tx + u * dx.abs() + floor), (dw, 1.01 * tw + u * dw.abs() + floor)


def _check(x, w, labels, weights):
    from native_sparse_attention_pytorch_amd import ops
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
    got = torch.autograd.grad(loss, (x, w), weights)
    want = _bounds(x.detach(), w.detach(), labels, weights)
    for g, e, what in zip(got, want, ("dx", "dw")):
        _within(g, e, what)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,d,v", [(20, 96, 300), (100, 96, 2000), (600, 64, 9000), (33, 130, 32000)])
def test_likely_labels_beside_unlikely_ones(n, d, v, dtype):
    """Labels that lead by 5, 18 and 30, and any, in turn: r from 10^3 down to 1e-10."""
    x, w, labels, weights = _inputs(n, d, v, dtype, seed=4, ignored=0.)
    w32 = w.float()[labels]
    gap = torch.tensor([5., 18., 30.], device=DEV)[torch.arange(n, device=DEV) % 3, None]
    led = (w32 * gap / w32.square().sum(-1, keepdim=True)).to(dtype)
    x = torch.where((torch.arange(n, device=DEV) % 4 == 0)[:, None], x, led)
    _check(x, w, labels, weights * (1e3 if dtype == F16 else 1.))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,d,v", [(20, 96, 300), (100, 96, 2000), (600, 64, 9000), (64, 130, 32000)])
def test_weights_of_eight_magnitudes(n, d, v, dtype):
    x, w, labels, _ = _inputs(n, d, v, dtype, seed=6, ignored=0.)
    weights = 10. ** -(torch.arange(n, device=DEV) % 9).float() * torch.where(torch.arange(n, device=DEV) % 2 == 0, 1., -1.) * (1e3 if dtype == F16 else 1.)
    _check(x, w, labels, weights)


def test_rows_that_are_not_finite_leave_the_others():
    """A row without a number has no dx and makes none of dw; the other rows' dx are what they were."""
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(70, 64, 300, F32, ignored=0.)
    grads = []
    for bad in (False, True):
        x2 = x.clone()
        if bad:
            x2[5, 3] = float("nan")
        x2.requires_grad_()
        grads.append(torch.autograd.grad(ops.linear_cross_entropy(x2, w, labels, reduction="none"), x2, weights)[0])
    keep = torch.arange(70, device=DEV) != 5
    assert torch.equal(grads[0][keep], grads[1][keep]) and grads[1][5].isnan().all()
