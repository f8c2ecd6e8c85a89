"""The library's loss and update entries without a GPU: a stand-in that reads and writes host tensors through the addresses it is given, so that
tests see which memory a call names and what lies there at the time of the launch."""
import contextlib
import ctypes as C

import numpy as np
import pytest
import torch


def _rows(address, rows, cols, stride, each=4):
    return [np.frombuffer((C.c_char * (cols * each)).from_address(address + r * stride * each), dtype={4: np.float32, 8: np.int64}[each]) for r in range(rows)]


class StandIn:
    """fp32 only.  The update of a matrix is twice the matrix; a row's loss is x . w[label] (0 where ignored), dx and dw 1 + its gradients' size."""

    def __init__(self):
        self.calls = []

    def nsa_newton_workspace_bytes(self, many, rows, cols, out):
        out._obj.value = 256
        return 0

    def nsa_newton_schulz(self, many, rows, cols, ins, strides, outs, dtype, *rest):
        self.calls.append(("nsa_newton_schulz", list(ins), list(strides)))
        if any(strides[k] < cols[k] for k in range(many)):
            return -1
        for k in range(many):
            got = _rows(outs[k], rows[k], cols[k], cols[k])
            for to, row in zip(got, _rows(ins[k], rows[k], cols[k], strides[k])):
                to[:] = 2 * row
        return 0

    def nsa_loss_workspace_bytes(self, d, weight, *sizes):
        for size, value in zip(sizes, (1280 + 24 * 64 * max(1, (d._obj.rows + 63) // 64), 256, 256)):
            size._obj.value = value
        return 0

    def nsa_loss_fwd(self, d, x, weight, labels, state, state_bytes, ws, ws_bytes, loss, stream):
        self.calls.append(("nsa_loss_fwd",))
        d = d._obj
        at = _rows(labels, 1, d.rows, d.rows, 8)[0] if d.rows else []
        xs, ws = _rows(x, d.rows, d.dim, d.x_stride), _rows(weight, d.vocab, d.dim, d.w_stride)
        each = np.array([0. if t == d.ignore_index else float(row @ ws[t]) for row, t in zip(xs, at)], dtype=np.float32)
        if d.reduction == 0:
            _rows(loss, 1, d.rows, d.rows)[0][:] = each
        else:
            _rows(loss, 1, 1, 1)[0][:] = each.sum() / (max(1, int((at != d.ignore_index).sum())) if d.reduction == 1 else 1)
        return 0

    def nsa_loss_bwd(self, d, x, weight, state, state_bytes, dloss, ws, ws_bytes, dx, dw, stream):
        self.calls.append(("nsa_loss_bwd",))
        d = d._obj
        g = _rows(dloss, 1, d.rows if d.reduction == 0 else 1, d.rows)[0].sum()
        for to, rows in ((dx, d.rows), (dw, d.vocab)):
            if to:
                for row in _rows(to, rows, d.dim, d.dim):
                    row[:] = 1 + g
        return 0


@pytest.fixture
def stand_in(monkeypatch):
    from native_sparse_attention_pytorch_amd import _lib, ops
    made = StandIn()
    monkeypatch.setattr(_lib, "lib", lambda: made)
    monkeypatch.setattr(ops, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    ops._loss_sizes.cache_clear()
    yield made
    ops._loss_sizes.cache_clear()
