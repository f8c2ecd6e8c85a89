"""The routes of tests/test_training_ends_routes.py with the library itself, and those of the attention operators, which share them."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
DEV = "cuda"
TRACES = ["make_fx", "make_fx fake", "make_fx pre_dispatch", "jit.trace"]


def _traced(how, fn, args):
    from torch.fx.experimental.proxy_tensor import make_fx
    if how == "jit.trace":
        return torch.jit.trace(fn, args, check_trace=False)
    return make_fx(fn, tracing_mode="fake" if "fake" in how else "real", pre_dispatch="pre" in how)(*args)


def _loss_args(seed, n=40):
    g = torch.Generator().manual_seed(seed)
    return [t.to(DEV) for t in (torch.randn(n, 64, generator=g), torch.randn(130, 64, generator=g), torch.randint(0, 130, (n,), generator=g))]


@torch.no_grad()
@pytest.mark.parametrize("how", TRACES)
@pytest.mark.parametrize("n", [20, 40])
def test_a_traced_loss_computes(how, n):
    from native_sparse_attention_pytorch_amd import ops
    fn = lambda x, w, labels: ops.linear_cross_entropy(x, w, labels, reduction="none")
    run = _traced(how, fn, _loss_args(0, n))
    args = _loss_args(1, n)
    assert torch.equal(run(*args), fn(*args))


@pytest.mark.parametrize("how", ["make_fx", "make_fx fake"])
def test_traced_gradients_compute(how):
    from native_sparse_attention_pytorch_amd import ops

    def fn(x, w, labels, weights):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        return torch.autograd.grad(ops.linear_cross_entropy(x, w, labels, reduction="none"), (x, w), weights)
    run = _traced(how, fn, (*_loss_args(0), torch.rand(40, device=DEV)))
    args = *_loss_args(1), torch.rand(40, device=DEV)
    for got, want in zip(run(*args), fn(*args)):
        assert torch.equal(got, want)


@torch.no_grad()
@pytest.mark.parametrize("how", TRACES)
def test_a_traced_update_computes(how):
    from native_sparse_attention_pytorch_amd import ops
    make = lambda: (torch.randn(70, 130, device=DEV), torch.randn(24, 100, device=DEV))
    fn = lambda a, b: tuple(ops.newton_schulz([a, b]))
    run, args = _traced(how, fn, make()), make()
    for got, want in zip(run(*args), fn(*args)):
        assert torch.equal(got, want)


def test_tangents_are_refused():
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels = _loss_args(0)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(w, torch.ones_like(w))
        with pytest.raises(NotImplementedError, match="forward mode"):
            ops.linear_cross_entropy(x, dual, labels)
        with pytest.raises(NotImplementedError, match="forward mode"):
            ops.newton_schulz([x, dual])
        assert ops.linear_cross_entropy(x, w, labels).isfinite()


def _attention(seed):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(1, h, 96, 64, generator=g).bfloat16().to(DEV) for h in (4, 2, 2))
    idx = torch.randint(0, 6, (1, 2, 96, 3), generator=g).to(DEV)
    return q, k, v, idx, (idx * 16 < torch.arange(96, device=DEV)[None, None, :, None] // 16 * 16)


@torch.no_grad()
@pytest.mark.parametrize("how", TRACES)
def test_traced_attention_computes(how):
    """Block selection and a sliding window."""
    from native_sparse_attention_pytorch_amd import ops
    fn = lambda q, k, v, idx, mask: (ops._select_fwd(q, k, v, idx, mask, None, 16, True, 0.125)[0],
                                     ops._dense_fwd(q, k, v, 0, True, 32, 1, 0, 0, 1, True, 0.125)[0])
    run, args = _traced(how, fn, _attention(0)), _attention(1)
    for got, want in zip(run(*args), fn(*args)):
        assert torch.equal(got, want)


def test_tangents_of_attention_are_refused():
    from native_sparse_attention_pytorch_amd import ops
    q, k, v, idx, mask = _attention(0)
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        ops._select_fwd(forward_ad.make_dual(q, q), k, v, idx, mask, None, 16, True, 0.125)
