"""ops.linear_cross_entropy of many rows: those that count are found by counts of 1024 rows each past 32768 of them, the largest |G| in a launch of its own
past 65536."""
import pytest
import torch

from tests.test_linear_cross_entropy_gpu import BF16, F16, F32, DEV, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,dtype", [(32768, BF16), (32769, F32), (33793, F16), (65536, BF16), (65537, F32), (100001, F16), (300007, BF16)])
def test_many_rows(n, dtype):
    x, w, labels, weights = _inputs(n, 24, 40, dtype, seed=n, ignored=0.3)
    labels[:5000] = -100                       # whole counts of none, and of all
    labels[9000:12000] = 3
    weights = 10. ** -(torch.arange(n, device=DEV) % 5).float()
    _check(x, w, labels.int() if n % 2 else labels, "none", weights)


@pytest.mark.parametrize("counted", [[], [0], [69999], [1023, 1024, 40000]])
def test_few_of_many_rows(counted):
    x, w, labels, weights = _inputs(70000, 24, 40, BF16, ignored=0.)
    kept = labels[counted].clone()
    labels.fill_(-100)
    labels[counted] = kept
    if counted:
        _check(x, w, labels, "mean", weights)
    else:
        from native_sparse_attention_pytorch_amd import ops
        assert ops.linear_cross_entropy(x, w, labels).isnan() and not ops.linear_cross_entropy(x, w, labels, reduction="none").any()
