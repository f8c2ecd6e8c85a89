"""Sizes that nsa_loss_* takes and refuses, by the launches that they would need: no GPU."""
import ctypes as C

import pytest

from native_sparse_attention_pytorch_amd import _lib


def _sizes(rows, dim, vocab, dtype, weight=0):
    d = _lib.LossDesc(rows=rows, dim=dim, vocab=vocab, dtype=dtype, reduction=1, labels_int64=1, ignore_index=-100, x_stride=dim, w_stride=dim)
    got = [C.c_size_t() for _ in range(3)]
    return _lib.lib().nsa_loss_workspace_bytes(C.byref(d), weight, *map(C.byref, got)), [g.value for g in got]


@pytest.mark.parametrize("rows,dim,vocab,dtype,tile", [
    (1 << 20, 64, 1 << 19, 0, 256), (1 << 22, 512, 1 << 17, 1, 256), (1 << 23, 64, 1 << 16, 0, 256), (1 << 16, 64, 1 << 23, 0, 256),   # the weight in place
    (1 << 23, 64, 1 << 20, 2, 256), (1 << 22, 1088, 1 << 20, 2, 128),      # pieces of 2^20 and of 61440 entries
])
def test_launches_of_more_threads_than_there_are(rows, dim, vocab, dtype, tile):
    """One launch makes the tiles of all rows with all entries, or those of a piece: 512 threads for each 256 x 256 (128 x 128), 2^32 at most."""
    assert _sizes(rows, dim, vocab, dtype)[0] == -2
    entries = vocab if dtype != 2 else min(vocab, (256 << 20) // (-(-dim // 64) * 64 * 4) // 256 * 256)
    most = ((1 << 32) - 1) // 512 // -(-entries // tile) * tile            # rows that a launch still holds
    assert _sizes(most, dim, vocab, dtype)[0] == 0 and _sizes(most + 1, dim, vocab, dtype)[0] == -2


def test_sizes_in_use_are_taken():
    for rows, dim, vocab in ((16384, 4096, 131072), (1 << 20, 1024, 131072), (1 << 24, 64, 256), (32, 64, 1 << 24), (64, 64, 1 << 24), (1 << 24, 64, 64)):
        for dtype in (0, 1, 2):
            assert _sizes(rows, dim, vocab, dtype)[0] == 0, (rows, dim, vocab, dtype)
