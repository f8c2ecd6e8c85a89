"""The registered operators behind ops.linear_cross_entropy and ops.newton_schulz check what they are given: a traced graph calls them with whatever it
is run on.  Nothing refused here reaches the library; no GPU."""
import pytest
import torch

from tests.stand_in import stand_in  # noqa: F401

X, W, LABELS = torch.randn(6, 8), torch.randn(5, 8), torch.zeros(6, dtype=torch.int64)
BAD = {
    "x of another type": (X.bfloat16(), W, LABELS), "weight of another type": (X, W.half(), LABELS), "both of another": (X.double(), W.double(), LABELS),
    "x of 3 axes": (X[None], W, LABELS[None]), "x of 1": (X[0], W, LABELS[0]), "a weight of 1": (X, W[0], LABELS), "fewer features": (X[:, :7], W, LABELS),
    "fewer labels": (X, W, LABELS[:5]), "labels of 2 axes": (X, W, LABELS[:, None]), "real labels": (X, W, LABELS.float()), "short labels": (X, W, LABELS.short()),
    "no entries": (X, W[:0], LABELS), "labels elsewhere": (X, W, LABELS.to("meta")), "a weight elsewhere": (X, W.to("meta"), LABELS),
}


@pytest.mark.parametrize("what", BAD)
def test_loss(stand_in, what):
    from native_sparse_attention_pytorch_amd import ops
    if "elsewhere" not in what:                    # (tensors without memory: the operator makes others of the results' shapes)
        with pytest.raises(RuntimeError, match="linear_cross_entropy"):
            ops.linear_cross_entropy_fwd(*BAD[what], -100, 1)
    if what not in ("x of 3 axes", "x of 1"):      # (these are taken row by row)
        with pytest.raises(RuntimeError, match="linear_cross_entropy"):
            ops.linear_cross_entropy(*BAD[what])
    assert not stand_in.calls


@pytest.mark.parametrize("bad", [dict(dloss=torch.ones(6)), dict(dloss=torch.ones(()), reduction=0), dict(dloss=torch.ones(5), reduction=0), dict(x=X.half()),
                                 dict(x=X[None]), dict(weight=W[:, :7]), dict(state=torch.zeros(3000)), dict(state=torch.zeros(6000, dtype=torch.uint8)[::2])])
def test_loss_gradients(stand_in, bad):
    from native_sparse_attention_pytorch_amd import ops
    good = dict(dloss=torch.ones(()), x=X, weight=W, state=torch.zeros(2816, dtype=torch.uint8), ignore_index=-100, reduction=1, want_dx=True, want_dw=True)
    ops.linear_cross_entropy_bwd(**good)
    stand_in.calls.clear()
    with pytest.raises(RuntimeError, match="linear_cross_entropy"):
        ops.linear_cross_entropy_bwd(**{**good, **bad})
    assert not stand_in.calls


@pytest.mark.parametrize("matrices", [[X, X.half()], [X.double()], [X[0]], [X[None, None]], [X, X[:0]], []])
def test_updates(stand_in, matrices):
    from native_sparse_attention_pytorch_amd import ops
    with pytest.raises(RuntimeError):
        ops.newton_schulz_op(matrices, 5, 1.5, -0.5, 0., 1e-7)
    assert not stand_in.calls


def test_host_tensors():
    from native_sparse_attention_pytorch_amd import ops
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.linear_cross_entropy_fwd(X, W, LABELS, -100, 1)
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.linear_cross_entropy_bwd(torch.ones(()), X, W, torch.zeros(2816, dtype=torch.uint8), -100, 1, True, True)
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.newton_schulz_op([X], 5, 1.5, -0.5, 0., 1e-7)


def test_a_state_that_is_too_short():
    """The entry is told how long the state is, not how long it should be."""
    import ctypes as C
    from native_sparse_attention_pytorch_amd import _lib
    d = _lib.LossDesc(rows=6, dim=8, vocab=5, dtype=2, reduction=1, labels_int64=1, ignore_index=-100, x_stride=8, w_stride=8)
    state, fwd, bwd = C.c_size_t(), C.c_size_t(), C.c_size_t()
    assert _lib.lib().nsa_loss_workspace_bytes(C.byref(d), 256, C.byref(state), C.byref(fwd), C.byref(bwd)) == 0
    assert _lib.lib().nsa_loss_bwd(C.byref(d), 256, 256, 256, state.value - 1, 256, 256, bwd.value, 256, 256, 0) == -3
