"""Attention over long ranges of the 8-bit cache, whose tiles work-groups share, against the definition in 64 bits: both head sizes, all types, windows that begin inside a tile."""
import pytest
import torch

from tests import serving_reference as R
from tests.test_cache8_attend_gpu import DEV, TYPES, close, made, on_device, spoil

pytestmark = pytest.mark.gpu


# (a unit of more than 50 tiles of 32 keys is shared, or of more than 96 where there are 256 units)
@pytest.mark.parametrize("window", [None, 1700, 2345, 4100])
@pytest.mark.parametrize("hk, g", [(1, 4), (2, 1), (1, 20)])
@pytest.mark.parametrize("d, block", [(64, 32), (128, 16), (128, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_ragged_lengths(dtype, d, block, hk, g, window):
    from native_sparse_attention_pytorch_amd import ops
    lengths = [6016, 0, 1, 1699, 1701, 4113, 2350, 6001]
    q, cache = made(len(lengths), hk, g, 6016, d, block, dtype, seed=g + hk)
    cache = spoil(cache, lengths)
    got = ops.cache8_attend(q.to(DEV), on_device(cache), torch.tensor(lengths, dtype=torch.int32, device=DEV), window=window)
    close(got, *R.attend(q, cache, lengths, window or 0), keys=6016)
    assert not got[1].any()


@pytest.mark.parametrize("window", [None, 2003])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b, hk, g, n", [(1, 2, 8, 20000), (3, 2, 2, 5003)])
def test_one_length(dtype, b, hk, g, n, window):
    from native_sparse_attention_pytorch_amd import ops
    q, cache = made(b, hk, g, -(-n // 32) * 32, 128, 32, dtype, seed=n)
    cache = spoil(cache, [n] * b)
    got = ops.cache8_attend(q.to(DEV), on_device(cache), n, window=window)
    close(got, *R.attend(q, cache, [n] * b, window or 0), keys=n)


@pytest.mark.parametrize("d", [64, 128])
def test_many_units(d):
    """256 units of up to 125 tiles."""
    from native_sparse_attention_pytorch_amd import ops
    lengths = [(i * 997) % 4001 for i in range(64)]
    q, cache = made(64, 4, 1, 4000, d, 16, "bf16", seed=d)
    got = ops.cache8_attend(q.to(DEV), on_device(spoil(cache, lengths)), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    close(got, *R.attend(q, cache, lengths), keys=4000)
