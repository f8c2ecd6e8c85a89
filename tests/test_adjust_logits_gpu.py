"""What is done to logits against a definition in 64 bits.  At most six fp32 roundings, each relative to what it is of: the bound counts them."""
import math

import pytest
import torch

from tests import serving_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def check(x, got, each):
    """`each`: the arguments of R.adjust for every row."""
    assert got.dtype == torch.float32 and got.shape == x.shape
    for r in range(x.shape[0]):
        a = each(r)
        want, got_r, u = R.adjust(x[r].cpu(), **a), got[r].double().cpu(), 2. ** -24
        rest = {k: v for k, v in a.items() if k != "allowed"}
        free = R.adjust(x[r].cpu().abs() * max(1., a.get("repetition", 1.), 1 / a.get("repetition", 1.)), **{
            **rest, "repetition": 1., "frequency": -abs(a.get("frequency", 0.)), "presence": -abs(a.get("presence", 0.)),
            "bias": None if a.get("bias") is None else a["bias"].abs()})
        ok = (got_r == want) | ((got_r - want).abs() <= 6 * u * free.abs() + 1e-45) | (got_r.isnan() & want.isnan())
        assert ok.all(), f"row {r}: {int((~ok).sum())} entries, first {torch.nonzero(~ok)[0].item()}: {got_r[~ok][0].item()}, {want[~ok][0].item()}"


def tokens(rows, t, vocab, gen):
    """Some tokens often, and padding of several kinds."""
    h = (torch.rand(rows, t, generator=gen) ** 3 * vocab).long()
    return torch.where(torch.rand(rows, t, generator=gen) < 0.1, torch.tensor([-1, vocab, 1 << 40])[torch.randint(0, 3, (rows, t), generator=gen)], h)


@pytest.mark.parametrize("rows, vocab, t", [(1, 1, 1), (1, 7, 30), (3, 31, 0), (2, 33, 5), (5, 1000, 999), (4, 1025, 300), (2, 50021, 4000), (1, 131072, 77), (300, 257, 64)])
@pytest.mark.parametrize("mask", ["none", "bool", "words"])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_their_own(dtype, mask, rows, vocab, t):
    from native_sparse_attention_pytorch_amd import ops
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g) * 4).to(TYPES[dtype])
    history = tokens(rows, t, vocab, g)
    lengths = torch.randint(-2, t + 3, (rows,), generator=g)
    numbers = {n: torch.rand(rows, generator=g) * s + lo for n, s, lo in (("repetition", 1., 0.6), ("frequency", 1., -0.3), ("presence", 1., -0.3), ("temperature", 2., 0.1))}
    bias = torch.randn(rows, vocab, generator=g)
    allowed = {"none": None, "bool": torch.rand(rows, vocab, generator=g) < 0.5,
               "words": torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g).to(torch.int32)}[mask]
    if allowed is not None:
        allowed[0] = 0                                            # nothing is allowed
    to = lambda v: None if v is None else v.to(DEV)
    got = ops.adjust_logits(to(x), to(history), to(lengths), repetition_penalty=to(numbers["repetition"]), frequency_penalty=to(numbers["frequency"]),
                            presence_penalty=to(numbers["presence"]), bias=to(bias), temperature=to(numbers["temperature"]), allowed=to(allowed))
    check(x, got, lambda r: dict(history=history[r], lengths=min(int(lengths[r]), t), bias=bias[r], allowed=None if allowed is None else allowed[r],
                                 **{n: v[r].item() for n, v in numbers.items()}))
    if allowed is not None:
        assert (got[0] == -math.inf).all()


@pytest.mark.parametrize("what", ["nothing", "temperature", "repetition", "frequency and presence", "bias", "words for all", "bool for all", "one number on the device"])
def test_parts(what):
    from native_sparse_attention_pytorch_amd import ops
    g = torch.Generator().manual_seed(1)
    x, history = torch.randn(3, 130, generator=g) * 4, torch.randint(0, 130, (3, 50), generator=g, dtype=torch.int32)
    vector, bits, words = torch.randn(130, generator=g), torch.rand(130, generator=g) < 0.5, torch.tensor([1, -1, 1 << 31, 0, 2], dtype=torch.int64).to(torch.int32)
    one = torch.tensor(1.25)
    host = {"nothing": {}, "temperature": dict(temperature=0.7), "repetition": dict(history=history, repetition=1.3), "frequency and presence": dict(
        history=history, frequency=0.25, presence=-0.5), "bias": dict(bias=vector), "words for all": dict(allowed=words), "bool for all": dict(allowed=bits),
        "one number on the device": dict(history=history, repetition=one)}[what]
    rename = {"repetition": "repetition_penalty", "frequency": "frequency_penalty", "presence": "presence_penalty"}
    got = ops.adjust_logits(x.to(DEV), **{rename.get(k, k): v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in host.items()})
    check(x, got, lambda r: {k: v[r] if k == "history" else v.item() if k == "repetition" and isinstance(v, torch.Tensor) else v for k, v in host.items()})
    if what == "nothing":
        assert torch.equal(got.cpu(), x)


def test_what_is_no_number():
    from native_sparse_attention_pytorch_amd import ops
    x = torch.tensor([[math.inf, -math.inf, math.nan, math.nan, 1., -0., 0.]])
    allowed = torch.tensor([True, True, True, False, False, True, True])
    got = ops.adjust_logits(x.to(DEV), torch.arange(7, device=DEV)[None], repetition_penalty=2., presence_penalty=0.5, allowed=allowed.to(DEV)).cpu()
    assert got[0, :2].tolist() == [math.inf, -math.inf] and got[0, 2].isnan() and got[0, 3:].tolist() == [-math.inf, -math.inf, -0.5, -0.5]


def test_views_and_shapes():
    from native_sparse_attention_pytorch_amd import ops
    g = torch.Generator().manual_seed(1)
    whole = torch.randn(2, 3, 5, 200, generator=g).bfloat16()
    history = torch.randint(0, 100, (2, 3, 11), generator=g)
    bias, allowed = torch.randn(2, 3, 100, generator=g), torch.rand(2, 3, 200, generator=g) < 0.6
    for x in (whole[:, :, 2, 50:150], whole[:, :, 4, 1:200:2], whole[0, 0, 0, 7:107].expand(2, 3, 100)):
        allow = allowed[..., ::2]
        got = ops.adjust_logits(x.to(DEV) if x.is_contiguous() else torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=DEV).copy_(x) if 0 not in x.stride()
                                else x[0, 0].to(DEV).expand(2, 3, 100), history.to(DEV), frequency_penalty=0.1, bias=bias.to(DEV).bfloat16(), allowed=allowed.to(DEV)[..., ::2])
        assert got.shape == (2, 3, 100) and got.is_contiguous()
        check(x.reshape(6, 100), got.view(6, 100), lambda r: dict(history=history.view(6, 11)[r], frequency=0.1, bias=bias.bfloat16().view(6, 100)[r],
                                                                   allowed=allow.reshape(6, 100)[r]))
    one = torch.randn(40, generator=g)
    check(one[None], ops.adjust_logits(one.to(DEV), torch.tensor([3, 3, 4], device=DEV), frequency_penalty=1.)[None], lambda r: dict(history=torch.tensor([3, 3, 4]), frequency=1.))
    assert ops.adjust_logits(torch.zeros(0, 5, device=DEV)).shape == (0, 5)
    # a row of its own length: rows may be anywhere in a larger tensor, the last of it included
    far = torch.randn(4, 333, device=DEV)
    assert torch.equal(ops.adjust_logits(far[1:, 5:]), far[1:, 5:])


def test_two_graphs_and_other_streams():
    from native_sparse_attention_pytorch_amd import ops
    x, history = torch.randn(4, 5000, device=DEV), torch.randint(0, 5000, (4, 200), device=DEV)
    call = lambda: ops.adjust_logits(x, history, repetition_penalty=1.2, frequency_penalty=0.1, temperature=0.9)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    side = torch.cuda.Stream()
    for _ in range(4):
        x.normal_()
        history.random_(0, 5000)
        for g in graphs:
            g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call()
        torch.cuda.current_stream().wait_stream(side)
        want = call()
        assert all(torch.equal(o, want) for o in (*outs, other))
        torch.cuda.synchronize()
