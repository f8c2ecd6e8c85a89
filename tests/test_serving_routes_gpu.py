"""The 8-bit cache's operators and ops.adjust_logits as traces record them, compiled, and together as a step of a program uses them."""
import pytest
import torch

from tests import serving_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
TRACES = ["make_fx", "make_fx fake", "make_fx pre_dispatch", "jit.trace"]


def _traced(how, fn, args):
    from torch.fx.experimental.proxy_tensor import make_fx
    if how == "jit.trace":
        return torch.jit.trace(fn, args, check_trace=False)
    return make_fx(fn, tracing_mode="fake" if "fake" in how else "real", pre_dispatch="pre" in how)(*args)


def _args(seed, b=2, hk=2, g=3, n=96, d=64):
    from native_sparse_attention_pytorch_amd import ops
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    cache = ops.make_cache8(b, hk, n, d, block=16)
    with torch.no_grad():
        ops.cache8_append(cache, randn(b, hk, 50, d), randn(b, hk, 50, d))
    at = torch.tensor([50, 31], dtype=torch.int32, device=DEV)
    idx = torch.randint(0, 3, (b, hk, 1, 2), device=DEV, generator=gen)
    return (*cache, randn(b, hk * g, 1, d).bfloat16(), randn(b, hk, 1, d).bfloat16(), randn(b, hk, 1, d).bfloat16(), at, idx, torch.rand(b, hk, 1, 2, device=DEV, generator=gen) < 0.7,
            randn(b, 100), torch.randint(0, 100, (b, 9), device=DEV, generator=gen))


def _step(keys, values, key_scales, value_scales, q, k, v, at, idx, fmask, logits, history):
    from native_sparse_attention_pytorch_amd import ops
    cache = ops.Cache8(keys, values, key_scales, value_scales)
    ops.cache8_append(cache, k, v, at)
    return (ops.cache8_attend(q, cache, at + 1, window=20), ops.cache8_select_attend(q, cache, at + 1, 16, idx, fmask),
            ops.adjust_logits(logits, history, repetition_penalty=1.3, allowed=logits > -1))


@torch.no_grad()
@pytest.mark.parametrize("how", TRACES)
def test_a_traced_step_computes(how):
    run, given, same = _traced(how, _step, _args(0)), _args(1), _args(1)
    for got, want in zip(run(*given), _step(*same)):
        assert torch.equal(got, want)
    for a, b in zip(given[:4], same[:4]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))           # the cache was written


@torch.no_grad()
def test_a_compiled_step_computes():
    run, given, same = torch.compile(_step, backend="aot_eager"), _args(1), _args(1)
    for got, want in zip(run(*given), _step(*same)):
        assert torch.equal(got, want)
    for a, b in zip(given[:4], same[:4]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@torch.no_grad()
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_conversation(dtype):
    """A prompt, then tokens: every one goes into the cache and attends it, in sequences of their own lengths, a step captured and replayed; against the
    definition in 64 bits of the cache as it is."""
    from native_sparse_attention_pytorch_amd import ops
    b, hk, g, d, block = 3, 2, 4, 64, 32
    cache = ops.make_cache8(b, hk, 200, d, block=block)
    gen = torch.Generator(device=DEV).manual_seed(0)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen).to(dtype)
    counts = torch.tensor([100, 37, 64], dtype=torch.int32, device=DEV)
    ops.cache8_append(cache, randn(b, hk, 100, d), randn(b, hk, 100, d), 0, counts)
    lengths = counts.clone()
    q, k, v = randn(b, hk * g, 1, d), randn(b, hk, 1, d), randn(b, hk, 1, d)
    idx, fmask = torch.tensor([0, 1], device=DEV).expand(b, hk, 1, 2).contiguous(), torch.ones(b, hk, 1, 2, dtype=torch.bool, device=DEV)

    def step():
        ops.cache8_append(cache, k, v, lengths)
        lengths.add_(1)
        return ops.cache8_attend(q, cache, lengths), ops.cache8_attend(q, cache, lengths, window=33), ops.cache8_select_attend(q, cache, lengths, 16, idx, fmask)
    graph = torch.cuda.CUDAGraph()
    kept, at = [t.clone() for t in cache], lengths.clone()
    step()                                                            # (warm-up, taken back)
    for t, old in zip(cache, kept):
        t.copy_(old)
    lengths.copy_(at)
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(70):
        for t in (q, k, v):
            t.copy_(randn(*t.shape))
        graph.replay()
        if i % 23 == 0 or i == 69:
            host, n = tuple(t.cpu() for t in cache), lengths.tolist()
            assert n == [101 + i, 38 + i, 65 + i]
            for got, want in zip(outs, (R.attend(q.cpu(), host, n), R.attend(q.cpu(), host, n, window=33), R.attend(q.cpu(), host, n, size=16, idx=idx.cpu(), fmask=fmask.cpu()))):
                err = (got.double().cpu() - want[0]).abs()
                assert (err <= R.attend_bound(*want, dtype, 200)).all()
            rows_k, rows_v = cache.rows(n[0] - 1, 1, torch.float32)
            # half a step of a value, or of the scale's smallest code: the scale is below 2^-7 of the largest of 32 rows of these
            for rows, x in ((rows_k, k), (rows_v, v)):
                assert ((rows[0] - x[0].float()).abs() <= x[0].float().abs() * 2 ** -4 + 2 ** -10 * 2 ** -4).all()


def test_calls_at_once_on_two_streams():
    """Each call has its own workspace: what runs beside it changes nothing."""
    from native_sparse_attention_pytorch_amd import ops
    gen = torch.Generator(device=DEV).manual_seed(3)
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=gen).bfloat16()
    work = []
    for rows in (9000, 12000):
        cache = ops.make_cache8(3, 4, rows, 128, block=64)
        ops.cache8_append(cache, rand(3, 4, rows, 128), rand(3, 4, rows, 128))
        lengths = torch.tensor([rows, rows // 3, 1], dtype=torch.int32, device=DEV)
        history = torch.randint(0, 50000, (40, 700), device=DEV, generator=gen)
        work.append((rand(3, 16, 1, 128), cache, lengths, rand(40, 50000), history))

    def step(q, cache, lengths, logits, history):
        return ops.cache8_attend(q, cache, lengths), ops.cache8_attend(q, cache, lengths, window=3000), ops.adjust_logits(logits, history, repetition_penalty=1.3)
    want = [step(*w) for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, w, to in zip(streams, work, got):
            with torch.cuda.stream(s):
                to.append(step(*w))
    torch.cuda.synchronize()
    for to, here in zip(got, want):
        for results in to:
            for a, b in zip(results, here):
                assert torch.equal(a, b)
