"""Attention of one token over the 8-bit cache against a definition in 64 bits, which says how far results may be off."""
import math

import pytest
import torch

from tests import serving_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def made(b, hk, g, n, d, block, dtype, seed=0, d0=None):
    gen = torch.Generator().manual_seed(seed)
    d0 = d0 or d
    k = torch.randn(b, hk, n, d, generator=gen) * (1 + 3 * (torch.arange(d) % 13 == 2)) * 2. ** torch.randint(-3, 2, (b, hk, n // block, 1, 1), generator=gen).expand(
        b, hk, n // block, block, 1).reshape(b, hk, n, 1)
    v = torch.randn(b, hk, n, d, generator=gen) * 2. ** torch.randint(-3, 2, (b, hk, n // block), generator=gen).repeat_interleave(block, 2)[..., None]
    k[..., d0:], v[..., d0:] = 0, 0
    (keys, key_scales), (values, value_scales) = R.quantized(k, block), R.quantized(v, block)
    q = (torch.randn(b, hk * g, 1, d0, generator=gen) * 1.5).to(TYPES[dtype])
    return q, (keys, values, key_scales, value_scales)


def spoil(cache, lengths):
    """Behind its last token a sequence has NaN codes, and NaN scales of the blocks that begin there."""
    keys, values, key_scales, value_scales = (t.clone() for t in cache)
    block = keys.shape[2] // key_scales.shape[2]
    for i, n in enumerate(lengths):
        keys.view(torch.uint8)[i, :, n:], values.view(torch.uint8)[i, :, n:] = 0x7f, 0xff
        key_scales[i, :, -(-n // block):] = math.nan
        value_scales[i, :, -(-n // block):] = math.inf
    return keys, values, key_scales, value_scales


def on_device(cache):
    from native_sparse_attention_pytorch_amd.ops import Cache8
    return Cache8(*(t.to(DEV) for t in cache))


def close(got, want, largest, off, keys):
    assert got.shape == want.shape
    bound = R.attend_bound(want, largest, off, got.dtype, keys)
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} out of bounds, worst {(err / bound).max().item():.3g} times, first at {torch.nonzero(bad)[0].tolist()}"


@pytest.mark.parametrize("window", [None, 1, 16, 40, 333])
@pytest.mark.parametrize("g", [1, 2, 5, 16, 20, 32])
@pytest.mark.parametrize("d, block", [(64, 16), (64, 128), (128, 32), (128, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_newest_keys(dtype, d, block, g, window):
    from native_sparse_attention_pytorch_amd import ops
    lengths = [0, 1, 15, 17, 64, 255, 641, 768]
    q, cache = made(8, 2, g, 768, d, block, dtype, seed=g)
    cache = spoil(cache, lengths)
    got = ops.cache8_attend(q.to(DEV), on_device(cache), torch.tensor(lengths, dtype=torch.int32, device=DEV), window=window)
    assert got.dtype == TYPES[dtype] and got.is_contiguous()
    close(got, *R.attend(q, cache, lengths, window or 0), keys=768)
    assert not got[0].any()


@pytest.mark.parametrize("b, hk, n", [(1, 1, 20000), (3, 2, 4999), (70, 3, 130)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_long_and_many(dtype, b, hk, n):
    from native_sparse_attention_pytorch_amd import ops
    q, cache = made(b, hk, 4, -(-n // 32) * 32, 64, 32, dtype, seed=b)
    got = ops.cache8_attend(q.to(DEV), on_device(cache), n)
    close(got, *R.attend(q, cache, [n] * b), keys=n)


SELECTIONS = [(1, 3), (4, 4), (16, 7), (48, 5), (64, 16), (80, 2), (200, 1), (64, 0), (5, 40)]


@pytest.mark.parametrize("size, chosen", SELECTIONS)
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dtype, d, block, g", [("bf16", 64, 32, 4), ("bf16", 128, 16, 20), ("fp16", 128, 64, 3), ("fp32", 64, 128, 8)])
def test_selected_blocks(dtype, d, block, g, per_head, size, chosen):
    from native_sparse_attention_pytorch_amd import ops
    lengths = [1, 63, 64, 65, 500, 768, 0]
    b, hk = len(lengths), 2
    q, cache = made(b, hk, g, 768, d, block, dtype, seed=size)
    cache = spoil(cache, lengths)
    gen = torch.Generator().manual_seed(chosen)
    units = hk * g if per_head else hk
    idx = torch.randint(-1, 768 // size + 2, (b, units, 1, chosen), generator=gen)
    fmask = torch.rand(b, units, 1, chosen, generator=gen) < 0.8
    at = torch.tensor(lengths, device=DEV)                                  # int64
    # a block that begins behind the sequence, or is no block, has no key; one that ends behind it has those before
    got = ops.cache8_select_attend(q.to(DEV), on_device(cache), at, size, idx.to(DEV), fmask.to(DEV))
    want = R.attend(q, cache, lengths, size=size, idx=idx, fmask=fmask)
    close(got, *want, keys=size * (chosen + 1))
    again = ops.cache8_select_attend(q.to(DEV), on_device(cache), at.to(torch.int32), size, idx.to(DEV, torch.int32), fmask.to(DEV).to(torch.uint8))
    assert torch.equal(got, again)


def test_block_numbers_beyond_the_cache():
    from native_sparse_attention_pytorch_amd import ops
    q, cache = made(1, 1, 2, 128, 64, 32, "bf16")
    fmask = torch.ones(1, 1, 1, 4, dtype=torch.bool)
    far = torch.tensor([[[[1, 1 << 40, -(1 << 60), (1 << 63) - 1]]]])
    got = ops.cache8_select_attend(q.to(DEV), on_device(cache), 100, 16, far.to(DEV), fmask.to(DEV))
    close(got, *R.attend(q, cache, [100], size=16, idx=far, fmask=fmask), keys=128)
    twice = torch.tensor([[[[2, 2, 6, 3]]]], dtype=torch.int32)            # (6: the newest token's own)
    got = ops.cache8_select_attend(q.to(DEV), on_device(cache), 100, 16, twice.to(DEV), fmask.to(DEV))
    close(got, *R.attend(q, cache, [100], size=16, idx=twice, fmask=fmask), keys=128)


def test_lengths_beyond_the_cache_and_below_zero():
    from native_sparse_attention_pytorch_amd import ops
    q, cache = made(3, 1, 2, 96, 64, 32, "fp32")
    for dtype in (torch.int32, torch.int64):
        got = ops.cache8_attend(q.to(DEV), on_device(cache), torch.tensor([97, 2 ** 31 - 1, -5], dtype=dtype, device=DEV))
        close(got, *R.attend(q, cache, [96, 96, 0]), keys=96)


@pytest.mark.parametrize("d0, scale", [(1, None), (40, 0.3), (100, None), (128, 0.)])
def test_other_head_sizes_and_scales(d0, scale):
    from native_sparse_attention_pytorch_amd import ops
    d = 64 if d0 <= 64 else 128
    q, cache = made(2, 2, 3, 96, d, 32, "bf16", d0=d0)
    got = ops.cache8_attend(q.to(DEV), on_device(cache), 90, scale=scale)
    close(got, *R.attend(q, cache, [90, 90], scale=scale), keys=96)


@pytest.mark.parametrize("dtype", TYPES)
def test_views(dtype):
    """Queries as a projection leaves them, a cache that is part of another, lengths that are part of a table or one for all."""
    from native_sparse_attention_pytorch_amd import ops
    q, cache = made(4, 4, 2, 128, 64, 32, dtype, seed=9)
    whole = on_device(cache)
    part = ops.Cache8(*(t[1:4:2, :2] for t in whole))
    host = tuple(t.cpu() for t in part)
    wide = torch.randn(2, 1, 3 * 4 * 64, device=DEV).to(TYPES[dtype])
    views = wide[..., 256:512].view(2, 1, 4, 64).transpose(1, 2), wide[..., 3:259].view(2, 1, 4, 64).transpose(1, 2), wide[:1, :, :64].view(1, 1, 1, 64).expand(2, 4, 1, 64)
    table = torch.tensor([[100, 0], [33, 0]], dtype=torch.int32, device=DEV)
    for view in views:
        close(ops.cache8_attend(view, part, table[:, 0]), *R.attend(view.cpu(), host, [100, 33]), keys=128)
        close(ops.cache8_attend(view, part, table[1, 0]), *R.attend(view.cpu(), host, [33, 33]), keys=128)


def test_infinities_and_nan_of_the_keys_it_attends():
    """A NaN key or value is seen by the heads that attend it, and by no other sequence or kv head."""
    from native_sparse_attention_pytorch_amd import ops
    q, cache = made(2, 2, 2, 96, 64, 32, "bf16")
    clean = ops.cache8_attend(q.to(DEV), on_device(cache), 96)
    cache[0].view(torch.uint8)[0, 1, 50, 3] = 0x7f
    cache[1].view(torch.uint8)[1, 0, 7, 5] = 0xff
    got = ops.cache8_attend(q.to(DEV), on_device(cache), 96)
    assert got[0, 2:].isnan().all() and got[1, :2, 0, 5].isnan().all()
    assert torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[1, 2:], clean[1, 2:])
    rest = torch.arange(64, device=DEV) != 5
    assert torch.equal(got[1, :2][..., rest], clean[1, :2][..., rest])


def test_a_cache_beyond_32_bits():
    from native_sparse_attention_pytorch_amd import ops
    rows = (1 << 25) + 4096
    cache = ops.make_cache8(1, 1, rows, 128, block=64)
    k, v = (torch.randn(1, 1, 200, 128, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    ops.cache8_append(cache, k, v, rows - 300)
    first = (rows - 300) // 64 * 64
    near = ops.Cache8(cache.keys[:, :, first:].contiguous(), cache.values[:, :, first:].contiguous(), cache.key_scales[:, :, first // 64:].contiguous(),
                      cache.value_scales[:, :, first // 64:].contiguous())
    q = torch.randn(1, 4, 1, 128, device=DEV, dtype=torch.bfloat16)
    length = rows - 100
    want = R.attend(q.cpu(), tuple(t.cpu() for t in near), [length - first], window=150)
    close(ops.cache8_attend(q, cache, length, window=150), *want, keys=150)
    idx = torch.tensor([[[[(length - 1) // 64 - 1]]]], device=DEV)
    one = torch.ones_like(idx, dtype=torch.bool)
    near_idx = idx.cpu() - first // 64
    want = R.attend(q.cpu(), tuple(t.cpu() for t in near), [length - first], size=64, idx=near_idx, fmask=one.cpu())
    close(ops.cache8_select_attend(q, cache, length, 64, idx, one), *want, keys=192)


def test_calls_on_streams_in_graphs_and_again():
    """The same bits from every call: on another stream, captured and replayed with other work between, two graphs one after the other."""
    from native_sparse_attention_pytorch_amd import ops
    q, cache = made(3, 2, 4, 2048, 128, 32, "bf16")
    q, cache, at = q.to(DEV), on_device(cache), torch.tensor([2048, 77, 1000], dtype=torch.int32, device=DEV)
    idx = torch.randint(0, 12, (3, 2, 1, 6), device=DEV)
    fmask = torch.rand(3, 2, 1, 6, device=DEV) < 0.7
    calls = [lambda: ops.cache8_attend(q, cache, at), lambda: ops.cache8_select_attend(q, cache, at, 64, idx, fmask)]
    first = [c() for c in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c, want in zip(calls, first):
            assert torch.equal(c(), want)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c())
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=DEV))
        at.copy_(torch.randint(1, 2049, (3,), device=DEV))
        for g in graphs:
            g.replay()
        for c, got in zip(calls, outs):
            assert torch.equal(got, c())
        torch.cuda.synchronize()


@pytest.mark.parametrize("what", ["all", "window", "blocks", "packed blocks"])
def test_more_sequences_than_a_launch_takes(what):
    """2050 sequences over one cache (expanded, as a prompt that all share): a launch takes 2048."""
    from native_sparse_attention_pytorch_amd import ops
    b, n, at = 2050, 3264, [0, 1, 1024, 2046, 2047, 2048, 2049]
    _, cache = made(1, 1, 1, n, 64, 64, "bf16")
    gen = torch.Generator().manual_seed(5)
    q = torch.randn(b, 2, 1, 64, generator=gen).bfloat16()
    lengths = torch.randint(0, n + 1, (b,), generator=gen, dtype=torch.int32)
    lengths[2048] = n
    many = ops.Cache8(*(t.to(DEV).expand(b, *t.shape[1:]) for t in cache))
    few = tuple(t.expand(len(at), *t.shape[1:]) for t in cache)
    args = {"all": {}, "window": {"window": 40}, "blocks": {"size": 32}, "packed blocks": {"size": 24}}[what]
    if "size" in args:
        args["idx"] = torch.randint(0, n // args["size"], (b, 1, 1, 4), generator=gen)
        args["fmask"] = torch.rand(b, 1, 1, 4, generator=gen) < 0.8
        got = ops.cache8_select_attend(q.to(DEV), many, lengths.to(DEV), args["size"], args["idx"].to(DEV), args["fmask"].to(DEV))
        args["idx"], args["fmask"] = args["idx"][at], args["fmask"][at]
    else:
        got = ops.cache8_attend(q.to(DEV), many, lengths.to(DEV), **args)
    close(got[at], *R.attend(q[at], few, lengths[at].tolist(), **args), keys=n)


def test_rows_far_apart():
    """Rows of the largest distance that is taken, where 32 bits just hold the offsets of sixteen; beyond it the call is refused."""
    from native_sparse_attention_pytorch_amd import ops
    step = (1 << 28) - 16
    far = [torch.empty(31 * step + 64, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).as_strided((1, 1, 32, 64), (64, 64, step, 1)) for _ in range(2)]
    near = ops.make_cache8(1, 1, 32, 64, block=16)
    cache = ops.Cache8(*far, near.key_scales.clone(), near.value_scales.clone())
    k, v = (torch.randn(1, 1, 29, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    q = torch.randn(1, 4, 1, 64, device=DEV, dtype=torch.bfloat16)
    idx, one = torch.zeros(1, 1, 1, 1, dtype=torch.int64, device=DEV), torch.ones(1, 1, 1, 1, dtype=torch.bool, device=DEV)
    for c in (cache, near):
        ops.cache8_append(c, k, v)
    assert torch.equal(cache.keys[:, :, :29].view(torch.uint8), near.keys[:, :, :29].view(torch.uint8))
    for n in (29, 16, 5):
        for window in (None, 7):
            assert torch.equal(ops.cache8_attend(q, cache, n, window=window), ops.cache8_attend(q, near, n, window=window))
        for size in (16, 8):
            assert torch.equal(ops.cache8_select_attend(q, cache, n, size, idx, one), ops.cache8_select_attend(q, near, n, size, idx, one))
    beyond = [t.as_strided((1, 1, 16, 64), (64, 64, step + 16, 1)) for t in far]
    with pytest.raises(RuntimeError, match="nsa_cache8_workspace_bytes"):
        ops.cache8_attend(q, ops.Cache8(*beyond, near.key_scales[:, :, :1], near.value_scales[:, :, :1]), 5)


@pytest.mark.parametrize("size, chosen", [(64, 40), (16, 150), (40, 60), (7, 300)])
@pytest.mark.parametrize("dtype, d, block, g, per_head", [("bf16", 64, 32, 4, False), ("bf16", 128, 16, 20, False), ("fp16", 128, 64, 3, True), ("fp32", 64, 128, 8, False), ("fp32", 128, 32, 2, True)])
def test_many_selected_blocks(dtype, d, block, g, per_head, size, chosen):
    """So many that work-groups share them."""
    from native_sparse_attention_pytorch_amd import ops
    lengths = [2, 700, 2816, 0]
    b, hk = len(lengths), 2
    q, cache = made(b, hk, g, 2816, d, block, dtype, seed=chosen)
    cache = spoil(cache, lengths)
    gen = torch.Generator().manual_seed(size)
    units = hk * g if per_head else hk
    idx = torch.randint(-1, 2816 // size + 2, (b, units, 1, chosen), generator=gen, dtype=torch.int32)
    fmask = torch.rand(b, units, 1, chosen, generator=gen) < 0.8
    got = ops.cache8_select_attend(q.to(DEV), on_device(cache), torch.tensor(lengths, device=DEV, dtype=torch.int32), size, idx.to(DEV), fmask.to(DEV))
    close(got, *R.attend(q, cache, lengths, size=size, idx=idx, fmask=fmask), keys=size * (chosen + 1))
    assert not got[3].any()


@pytest.mark.parametrize("lengths", [[40000], [40000, 3, 0, 39999]])
@pytest.mark.parametrize("dtype, g", [("bf16", 4), ("fp32", 1), ("bf16", 20)])
def test_few_units_of_many_tiles(dtype, g, lengths):
    from native_sparse_attention_pytorch_amd import ops
    q, cache = made(len(lengths), 1, g, 40000, 64, 64, dtype, seed=g)
    got = ops.cache8_attend(q.to(DEV), on_device(spoil(cache, lengths)), torch.tensor(lengths, device=DEV, dtype=torch.int32))
    close(got, *R.attend(q, cache, lengths), keys=40000)
