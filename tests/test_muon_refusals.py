"""What training.Muon refuses, before a step has changed anything, and parameters on several devices: no GPU."""
import pytest
import torch

from native_sparse_attention_pytorch_amd import ops
from native_sparse_attention_pytorch_amd.training import Muon
from tests.stand_in import stand_in  # noqa: F401


def _params(count=2):
    params = [torch.nn.Parameter(torch.randn(4, 6)) for _ in range(count)]
    for p in params:
        p.grad = torch.ones_like(p)
    return params


def _unchanged(opt, params, error, match):
    before = [p.detach().clone() for p in params]
    with pytest.raises(error, match=match):
        opt.step()
    assert not opt.state and all(torch.equal(p.detach(), b) for p, b in zip(params, before))


@pytest.mark.parametrize("bad", [dict(steps=0), dict(steps=101), dict(eps=-1.), dict(eps=float("nan")), dict(coefficients=(5., 0., 0.)), dict(coefficients=(1., 2.)),
                                 dict(lr=-1.), dict(lr=float("nan")), dict(momentum=1.), dict(weight_decay=-1.)])
def test_numbers_out_of_range(bad):
    """At once, for a group of its own too; and where a group is changed afterwards, by the step."""
    params = _params()
    with pytest.raises(ValueError):
        Muon(params, **bad)
    with pytest.raises(ValueError):
        Muon([dict(params=params[:1]), dict(params=params[1:], **bad)])
    opt = Muon(params[:1])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=params[1:], **bad))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=params[1:]))
    opt.param_groups[1].update(bad)
    torch.Tensor.is_cuda = True
    try:
        _unchanged(opt, params, ValueError, "Muon|newton_schulz")
    finally:
        del torch.Tensor.is_cuda


def test_parameters_that_are_not_on_a_gpu():
    params = _params()
    _unchanged(Muon(params), params, RuntimeError, "needs a GPU")


def test_sparse_gradients(stand_in):
    params = _params()
    params[1].grad = torch.ones(4, 6).to_sparse()
    _unchanged(Muon([dict(params=params[:1]), dict(params=params[1:])]), params, RuntimeError, "sparse")


def test_each_device_has_its_own_call(monkeypatch, stand_in):
    params = [torch.nn.Parameter(torch.randn(4, 6, device=d)) for d in ("cpu", "meta", "cpu")]
    for p in params:
        p.grad = torch.ones_like(p)
    seen = []

    def update(updates, **kw):
        seen.append({u.device.type for u in updates})
        return [torch.zeros_like(u) for u in updates]
    monkeypatch.setattr(ops, "newton_schulz", lambda updates, **kw: update(updates, **kw) if updates else [])
    before = params[0].detach().clone()
    Muon(params).step()
    assert seen == [{"cpu"}, {"meta"}] and torch.equal(params[0].detach(), before)


def test_a_learning_rate_in_a_tensor(stand_in):
    params = _params(1)
    before = params[0].detach().clone()
    Muon(params, lr=torch.tensor(0.5), momentum=0., nesterov=False).step()
    torch.testing.assert_close(params[0].detach(), before - 0.5 * 2)
