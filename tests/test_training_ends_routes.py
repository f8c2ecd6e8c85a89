"""Tracers, transforms and forward mode around ops.linear_cross_entropy and ops.newton_schulz, without a GPU (tests/stand_in.py computes in the
library's place): a traced call computes on the inputs that it is run on, and what the operators have no rule for is refused."""
import pytest
import torch
from torch.autograd import forward_ad

from tests.stand_in import stand_in  # noqa: F401

TRACES = ["make_fx", "make_fx fake", "make_fx pre_dispatch", "jit.trace"]


def _traced(how, fn, args):
    from torch.fx.experimental.proxy_tensor import make_fx
    if how == "jit.trace":
        return torch.jit.trace(fn, args, check_trace=False)
    return make_fx(fn, tracing_mode="fake" if "fake" in how else "real", pre_dispatch="pre" in how)(*args)


def _loss_args(seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(6, 8, generator=g), torch.randn(5, 8, generator=g), torch.randint(0, 5, (6,), generator=g)


@torch.no_grad()
@pytest.mark.parametrize("how", TRACES)
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_a_traced_loss_computes(stand_in, how, reduction):
    from native_sparse_attention_pytorch_amd import ops
    fn = lambda x, w, labels: ops.linear_cross_entropy(x, w, labels, reduction=reduction)
    run = _traced(how, fn, _loss_args(0))
    x, w, labels = _loss_args(1)
    want = (x * w[labels]).sum(-1)
    torch.testing.assert_close(run(x, w, labels), want if reduction == "none" else want.mean())


@torch.no_grad()
@pytest.mark.parametrize("how", TRACES)
def test_a_traced_update_computes(stand_in, how):
    from native_sparse_attention_pytorch_amd import ops
    run = _traced(how, lambda a, b: tuple(ops.newton_schulz([a, b])), (torch.randn(4, 6), torch.randn(7, 3)))
    a, b = torch.randn(4, 6), torch.randn(7, 3)
    for got, want in zip(run(a, b), (2 * a, 2 * b)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("how", ["make_fx", "make_fx fake"])
def test_traced_gradients_compute(stand_in, how):
    """The backward pass is recorded as well."""
    from native_sparse_attention_pytorch_amd import ops

    def fn(x, w, labels, weights):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        return torch.autograd.grad(ops.linear_cross_entropy(x, w, labels, reduction="none"), (x, w), weights)
    run = _traced(how, fn, (*_loss_args(0), torch.rand(6)))
    stand_in.calls.clear()
    weights = torch.rand(6) + 2
    for got in run(*_loss_args(1), weights):
        torch.testing.assert_close(got, torch.full_like(got, float(1 + weights.sum())))
    assert ("nsa_loss_bwd",) in stand_in.calls


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(stand_in, grad):
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels = _loss_args(0)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual_x, dual_w = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w))
        for args in ((dual_x, w, labels), (x, dual_w, labels), (dual_x[None], w, labels[None])):
            with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                ops.linear_cross_entropy(*args)
        for updates in (dual_w, [x, dual_w]):
            with pytest.raises(RuntimeError, match="forward"):
                ops.newton_schulz(updates)
        # what has no tangent is served
        assert ops.linear_cross_entropy(x, w, labels).shape == () and torch.equal(ops.newton_schulz(w), 2 * w)
    for fn in (lambda t: ops.linear_cross_entropy(t, w, labels), lambda t: ops.newton_schulz(t)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(fn, (x,), (torch.ones_like(x),))


@torch.no_grad()
def test_batched_calls(stand_in):
    """vmap calls the operator once for each of the batch; it has no such way for a list of matrices."""
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels = _loss_args(0)
    got = torch.vmap(lambda t: ops.linear_cross_entropy(t, w, labels))(torch.stack((x, 2 * x)))
    want = (x * w[labels]).sum(-1).mean()
    torch.testing.assert_close(got, torch.stack((want, 2 * want)))
    stand_in.calls.clear()
    try:
        got = torch.vmap(lambda t: ops.newton_schulz(t))(torch.stack((x, x + 1)))
    except RuntimeError:
        assert not stand_in.calls
    else:
        assert torch.equal(got, 2 * torch.stack((x, x + 1)))


def test_functional_gradients_are_refused(stand_in):
    """(torch's transforms take no registered rule of this form)"""
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels = _loss_args(0)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: ops.linear_cross_entropy(t, w, labels))(x)
    assert not stand_in.calls


def test_a_dispatch_mode_sees_the_operator(stand_in):
    from torch.utils._python_dispatch import TorchDispatchMode
    from native_sparse_attention_pytorch_amd import ops
    seen = []

    class Look(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    x, w, labels = _loss_args(0)
    with Look(), torch.no_grad():
        ops.linear_cross_entropy(x, w, labels)
        ops.newton_schulz([x, w])
    assert sum("linear_cross_entropy_fwd" in s for s in seen) == 1 and sum("newton_schulz" in s for s in seen) == 1
