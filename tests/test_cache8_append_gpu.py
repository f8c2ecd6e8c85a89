"""Rows into the 8-bit cache against a definition in 64 bits: codes and scales are equal, and nothing else of the cache changes."""
import math

import pytest
import torch

from tests import serving_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def garbage(batch, heads, rows, d, block, seed):
    """A cache of any bytes (no NaN: they would compare unequal to themselves) and any powers of two."""
    g = torch.Generator().manual_seed(seed)
    codes = lambda: torch.randint(0, 255, (batch, heads, rows, d), generator=g, dtype=torch.uint8)
    clean = lambda c: torch.where((c & 0x7f) == 0x7f, torch.zeros_like(c), c).view(R.FP8)
    scales = lambda: 2. ** torch.randint(-9, 3, (batch, heads, rows // block), generator=g).float()
    return clean(codes()), clean(codes()), scales(), scales()


def check(cache, host, k, v, starts, counts, block, call):
    from native_sparse_attention_pytorch_amd import ops
    wanted = []
    for codes, scales, x in ((host[0], host[2], k), (host[1], host[3], v)):
        codes, scales = codes.double(), scales.double()
        full = torch.nn.functional.pad(x.double().cpu(), (0, codes.shape[3] - x.shape[3]))
        R.append(codes, scales, full, starts, counts, block)
        wanted.append((codes, scales))
    call(ops)
    for name, got, want in (("keys", cache.keys, wanted[0][0]), ("values", cache.values, wanted[1][0]), ("key scales", cache.key_scales, wanted[0][1]),
                            ("value scales", cache.value_scales, wanted[1][1])):
        got = got.double().cpu()
        same = (got == want) | (got.isnan() & want.isnan())
        assert same.all(), f"{name}: {int((~same).sum())} differ, first at {torch.nonzero(~same)[0].tolist()}"


CASES = [
    # rows, capacity, starts, counts
    (1, 256, [0, 5, 127, 255], None),
    (1, 256, [16, 64, 128, 200], [1, 0, 1, 1]),
    (3, 256, [14, 126, 250, 255], None),                 # two blocks at once; past the capacity
    (130, 384, [0, 1, 250, 383], [130, 129, 7, 130]),
    (300, 384, [0, 100, 31, 84], [300, 1, 500, -3]),
]


@pytest.mark.parametrize("rows, capacity, starts, counts", CASES)
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_each_sequence(dtype, d, block, rows, capacity, starts, counts):
    from native_sparse_attention_pytorch_amd.ops import Cache8
    g = torch.Generator().manual_seed(rows + block)
    k, v = ((torch.randn(4, 2, rows, d, generator=g) * 2. ** torch.randint(-6, 9, (4, 2, 1, 1), generator=g)).to(TYPES[dtype]) for _ in range(2))
    host = garbage(4, 2, capacity, d, block, 3)
    cache = Cache8(*(t.to(DEV) for t in host))
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
    check(cache, host, k, v, starts, [rows] * 4 if counts is None else counts, block, lambda ops: ops.cache8_append(cache, k.to(DEV), v.to(DEV), at, n))


@pytest.mark.parametrize("d", [1, 48, 80, 100])
def test_other_head_sizes_are_padded(d):
    from native_sparse_attention_pytorch_amd import ops
    cache = ops.make_cache8(2, 3, 50, d, block=16)
    assert cache.keys.shape == (2, 3, 64, 64 if d <= 64 else 128) and cache.block == 16
    host = tuple(t.cpu() for t in cache)
    k, v = torch.randn(2, 3, 21, d), torch.randn(2, 3, 21, d)
    check(cache, host, k, v, [20, 20], [21, 21], 16, lambda ops: ops.cache8_append(cache, k.to(DEV), v.to(DEV), 20))
    for got, x in zip(cache.rows(20, 21, torch.float32), (k, v)):
        # (a code is off by half a step: 2^-4 of a value, or 2^-10 of the scale, which is below 2^-7 of the block's largest value)
        assert got.shape == (2, 3, 21, cache.keys.shape[3]) and ((got[..., :d].cpu() - x).abs() <= x.abs() * 2 ** -4 + x.abs().max() * 2 ** -17).all()


def test_what_is_no_number_and_ends_of_the_range():
    from native_sparse_attention_pytorch_amd.ops import Cache8
    x = torch.randn(1, 5, 32, 64)
    x[0, 0, 3, 7], x[0, 0, 4, 8], x[0, 0, 5, 9] = math.inf, -math.inf, math.nan       # does not count for the scale
    x[0, 1] *= 2. ** -130                                                                # below the smallest scale, denormal ones too
    x[0, 2] = torch.randn(32, 64).sign() * 3e38                                          # above the largest
    x[0, 3] = 0.
    x[0, 4, :16] = 448. * 2. ** -3                                                       # exactly at, and one rounding above
    x[0, 4, 16:] = torch.nextafter(torch.tensor(448. * 2. ** 5), torch.tensor(1e9))
    x[0, 0, 20:] = math.nan                                                              # a block of nothing
    host = garbage(1, 5, 32, 64, 16, 5)
    cache = Cache8(*(t.to(DEV) for t in host))
    check(cache, host, x, x.flip(3), [0], [32], 16, lambda ops: ops.cache8_append(cache, x.to(DEV), x.flip(3).to(DEV)))
    assert cache.key_scales[0, 1].eq(2. ** -110).all() and cache.key_scales[0, 2].eq(2. ** 119).all() and cache.key_scales[0, 3].eq(2. ** -110).all()
    assert cache.key_scales[0, 4].tolist() == [2. ** -3, 2. ** 6]


def test_a_scale_that_grows_and_one_that_stays():
    """Token by token: held rows change where the scale grows, and are the same bytes where it does not."""
    from native_sparse_attention_pytorch_amd import ops
    cache = ops.make_cache8(1, 1, 32, 64, block=32)
    host = [t.cpu().double() for t in cache]
    x = torch.randn(1, 1, 32, 64, generator=torch.Generator().manual_seed(2)) * torch.logspace(-2, 2, 32, base=2.)[torch.randperm(32, generator=torch.Generator().manual_seed(4))][:, None]
    for i in range(32):
        ops.cache8_append(cache, x[:, :, i:i + 1].to(DEV), -x[:, :, i:i + 1].to(DEV), i)
        R.append(host[0], host[2], x[:, :, i:i + 1].double(), [i], [1], 32)
        R.append(host[1], host[3], -x[:, :, i:i + 1].double(), [i], [1], 32)
        assert all(torch.equal(got.cpu().double(), want) for got, want in zip(cache, host))


def test_views():
    """k and v as a projection leaves them, a cache that is part of another, starts that are part of a table."""
    from native_sparse_attention_pytorch_amd import ops
    b, hq, hk, n, d = 2, 4, 2, 37, 64
    qkv = torch.randn(b, n, (hq + 2 * hk) * d, device=DEV, dtype=torch.bfloat16)
    _, k, v = (t.view(b, n, -1, d).transpose(1, 2) for t in qkv.split((hq * d, hk * d, hk * d), dim=-1))
    whole = ops.make_cache8(5, 2 * hk, 128, d, block=32)
    for t in whole:
        t.view(torch.uint8)[:] = 7
    part = ops.Cache8(*(t[1:5:2, 1:1 + hk] for t in whole))
    before = [t.clone() for t in whole]
    host = tuple(t.cpu() for t in part)
    table = torch.tensor([[9, 1], [60, 2]], dtype=torch.int32, device=DEV)
    check(part, host, k, v, [9, 60], [n, n], 32, lambda ops: ops.cache8_append(part, k, v, table[:, 0]))
    for t, old in zip(whole, before):
        t, old = t.view(torch.uint8), old.view(torch.uint8)
        rest = torch.ones(t.shape[:2], dtype=torch.bool, device=DEV)
        rest[1:5:2, 1:1 + hk] = False
        assert torch.equal(t[rest], old[rest])
    odd = torch.randn(b, hk, n, d + 1, device=DEV)[..., 1:]                  # rows that begin nowhere in particular
    host = tuple(t.cpu() for t in part)
    check(part, host, odd, odd * 3, [3, 3], [n, n], 32, lambda ops: ops.cache8_append(part, odd, odd * 3, torch.tensor([3], device=DEV)))
    same = k[:, :1].expand(b, hk, n, d)                                      # one head for all
    host = tuple(t.cpu() for t in part)
    check(part, host, same, same, [0, 0], [n, n], 32, lambda ops: ops.cache8_append(part, same, same))


def test_no_rows():
    from native_sparse_attention_pytorch_amd import ops
    cache = ops.make_cache8(1, 1, 16, 64, block=16)
    before = [t.clone() for t in cache]
    none = torch.zeros(1, 1, 0, 64, device=DEV)
    ops.cache8_append(cache, none, none, 16)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))


def test_a_cache_beyond_32_bits():
    """Rows whose offset in the cache is above 2^32."""
    from native_sparse_attention_pytorch_amd import ops
    rows = (1 << 25) + 4096
    cache = ops.make_cache8(1, 1, rows, 128, block=64)
    k = torch.randn(1, 1, 70, 128, device=DEV, dtype=torch.bfloat16)
    ops.cache8_append(cache, k, -k, rows - 100)
    got_k, got_v = cache.rows(rows - 100, 70, torch.float32)
    assert ((got_k - k.float()).abs() <= k.float().abs() * 2 ** -4 + 2 ** -10).all() and torch.equal(got_k, -got_v)
    assert not cache.keys.view(torch.uint8)[0, 0, :1 << 20].any() and not cache.keys.view(torch.uint8)[0, 0, rows - 30:].any()
