"""What ops.linear_cross_entropy, ops.newton_schulz and training.Muon refuse, and their C entries' checks of arguments: no GPU."""
import ctypes as C

import pytest
import torch

from native_sparse_attention_pytorch_amd import _lib, ops
from native_sparse_attention_pytorch_amd.training import Muon


def test_host_tensors_are_refused():
    x, w, labels = torch.randn(4, 64), torch.randn(10, 64), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.linear_cross_entropy(x, w, labels)
    with pytest.raises(ValueError, match="reduction"):
        ops.linear_cross_entropy(x, w, labels, reduction="max")
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.newton_schulz(w)
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.newton_schulz([w, w])
    assert ops.newton_schulz([]) == [] and ops.newton_schulz(()) == ()


@pytest.mark.parametrize("arguments", [dict(steps=0), dict(steps=101), dict(eps=-1.), dict(eps=float("nan")), dict(coefficients=(1., 2.)),
                                       dict(coefficients=(5., 0., 0.)), dict(coefficients=(float("nan"), 0., 0.)), dict(coefficients=(3.4445, -4.775, 8.))])
def test_newton_schulz_arguments(arguments):
    with pytest.raises(ValueError, match="newton_schulz"):
        ops.newton_schulz(torch.randn(4, 4), **arguments)


def test_muon_arguments():
    p = torch.nn.Parameter(torch.randn(4, 4))
    for bad in (dict(lr=-1.), dict(momentum=1.), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            Muon([p], **bad)
    with pytest.raises(ValueError, match="matrices"):
        Muon([p, torch.nn.Parameter(torch.randn(4))])
    with pytest.raises(ValueError, match="float64"):
        Muon([p, torch.nn.Parameter(torch.randn(4, 4).double())])
    assert Muon([p]).step(lambda: 3.) == 3.      # no gradients: nothing to do


def _sizes(d, weight=0):
    got = [C.c_size_t() for _ in range(3)]
    return _lib.lib().nsa_loss_workspace_bytes(C.byref(d), weight, *map(C.byref, got)), [g.value for g in got]


def _desc(**kw):
    base = dict(rows=100, dim=64, vocab=300, dtype=0, reduction=1, labels_int64=1, ignore_index=-100, x_stride=64, w_stride=64)
    return _lib.LossDesc(**{**base, **kw})


def test_loss_entry_checks_its_descriptor():
    assert _sizes(_desc())[0] == 0
    for bad in (dict(rows=-1), dict(dim=0), dict(vocab=0), dict(dtype=3), dict(dtype=-1), dict(reduction=3), dict(x_stride=63), dict(w_stride=63)):
        assert _sizes(_desc(**bad))[0] == -1, bad
    for bad in (dict(rows=(1 << 24) + 1), dict(dim=(1 << 16) + 1, x_stride=1 << 17, w_stride=1 << 17), dict(vocab=(1 << 24) + 1)):
        assert _sizes(_desc(**bad))[0] == -2, bad


@pytest.mark.parametrize("rows", [0, 1, 32, 33, 64, 65, 1000])
@pytest.mark.parametrize("dtype", [0, 2])
def test_traced_shapes_are_the_real_ones(rows, dtype):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = (torch.empty(n, 64, dtype=(torch.bfloat16, None, torch.float32)[dtype]) for n in (rows, 300))
        labels = torch.empty(rows, dtype=torch.int64)
        for reduction in (0, 1):
            loss, state = ops.linear_cross_entropy_fwd(x, w, labels, -100, reduction)
            assert loss.shape == ((rows,) if reduction == 0 else ()) and state.numel() == _sizes(_desc(rows=rows, dtype=dtype))[1][0]
        for wanted in ((True, True), (True, False), (False, True)):
            dx, dw = ops.linear_cross_entropy_bwd(loss, x, w, state, -100, 1, *wanted)
            assert dx.shape == (rows if wanted[0] else 0, 64) and dw.shape == (300 if wanted[1] else 0, 64) and dw.dtype == w.dtype


def test_loss_workspaces_hold_pieces_not_logits():
    for rows, dim, vocab, dtype in ((16384, 4096, 131072, 0), (16384, 4096, 131072, 2), (1 << 20, 512, 50021, 0), (8, 512, 256, 1)):
        rc, (state, fwd, bwd) = _sizes(_desc(rows=rows, dim=dim, vocab=vocab, dtype=dtype, x_stride=dim, w_stride=dim))
        each = 4 if dtype == 2 else 2
        assert rc == 0 and state <= 24 * (rows + 64) + 4096      # six numbers a row
        # what is kept of the forward, beside a piece of the weight: a pair of numbers for 32 to 128 logits
        assert fwd <= rows * vocab / 4 + rows * dim * each + (300 << 20)
        # a piece of G and of the weight, x again, and the slices of dx
        assert bwd <= (320 << 20) + 1024 * rows * each + 9 * (rows + 64) * dim * 4 + 4 * (64 << 20) * 4, (bwd, rows, dim, vocab)


def test_entries_check_pointers_and_workspaces():
    L, d, one = _lib.lib(), _desc(), C.c_void_p(256)
    rc, (state, fwd, bwd) = _sizes(d, 256)
    assert L.nsa_loss_fwd(C.byref(d), 256, 0, 256, 256, state, 256, fwd, 256, 0) == -1
    assert L.nsa_loss_fwd(C.byref(d), 256, 256, 256, 256, state - 1, 256, fwd, 256, 0) == -3
    assert L.nsa_loss_fwd(C.byref(d), 256, 256, 256, 256, state, 256, fwd - 1, 256, 0) == -3
    assert L.nsa_loss_bwd(C.byref(d), 256, 256, 256, state, 256, 256, bwd - 1, 256, 256, 0) == -3
    assert L.nsa_loss_bwd(C.byref(d), 256, 256, 256, state, 256, 256, bwd, 0, 0, 0) == -1
    assert L.nsa_loss_bwd(C.byref(d), 0, 256, 256, state, 256, 256, bwd, 256, 256, 0) == -1
    ints, longs, ptrs = C.c_int32 * 1, C.c_int64 * 1, C.c_void_p * 1
    need = C.c_size_t()
    assert L.nsa_newton_workspace_bytes(1, ints(40), ints(50), C.byref(need)) == 0
    call = lambda rows=40, cols=50, stride=50, at=256, to=256, dtype=2, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, ws=need.value: L.nsa_newton_schulz(
        1, ints(rows), ints(cols), ptrs(at), longs(stride), ptrs(to), dtype, steps, a, b, c, eps, one, ws, 0)
    assert call(rows=0) == -1 and call(stride=49) == -1 and call(at=0) == -1 and call(to=0) == -1 and call(dtype=3) == -1
    assert call(steps=0) == -1 and call(steps=101) == -1 and call(eps=-1.) == -1 and call(at=258) == -1
    assert call(to=258) == -1 and call(dtype=0, at=257) == -1
    assert call(a=5., b=0., c=0.) == -2 and call(ws=need.value - 1) == -3
    assert L.nsa_newton_workspace_bytes(1, ints((1 << 20) + 1), ints(4), C.byref(need)) == -2
    assert L.nsa_newton_workspace_bytes(1, ints(1 << 16), ints(1 << 16), C.byref(need)) == -2
    assert L.nsa_newton_schulz(0, None, None, None, None, None, 0, 5, 1., 0., 0., 0., None, 0, 0) == 0


def test_entries_check_alignment():
    L, d = _lib.lib(), _desc(dtype=2)
    _, (state, fwd, bwd) = _sizes(d, 256)
    good = dict(x=256, w=256, labels=256, state=256, ws=256, loss=256)
    for bad in (dict(x=258), dict(w=257), dict(labels=260), dict(state=272), dict(ws=384), dict(loss=258)):
        p = {**good, **bad}
        assert L.nsa_loss_fwd(C.byref(d), p["x"], p["w"], p["labels"], p["state"], state, p["ws"], fwd, p["loss"], 0) == -1, bad
    good = dict(x=256, w=256, state=256, dloss=256, ws=256, dx=256, dw=256)
    for bad in (dict(x=258), dict(w=257), dict(state=272), dict(dloss=258), dict(ws=384), dict(dx=258), dict(dw=257)):
        p = {**good, **bad}
        assert L.nsa_loss_bwd(C.byref(d), p["x"], p["w"], p["state"], state, p["dloss"], p["ws"], bwd, p["dx"], p["dw"], 0) == -1, bad
    ints, longs, ptrs, need = C.c_int32 * 1, C.c_int64 * 1, C.c_void_p * 1, C.c_size_t()
    assert L.nsa_newton_workspace_bytes(1, ints(40), ints(50), C.byref(need)) == 0
    assert L.nsa_newton_schulz(1, ints(40), ints(50), ptrs(256), longs(50), ptrs(256), 2, 5, 1.5, -0.5, 0., 1e-7, 272, need.value, 0) == -1


def test_a_model_made_before_the_option_has_it_off():
    from native_sparse_attention_pytorch_amd.transformer import Transformer
    model = Transformer(num_tokens=11, dim=64, depth=1, heads=1, fused_loss=True)
    assert model.fused_loss
    del model.__dict__["fused_loss"]
    assert model.fused_loss is False
