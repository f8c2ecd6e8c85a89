"""What the 8-bit cache's operators and ops.adjust_logits are given is checked before anything of it is read by address.  A stand-in for the library counts
what reaches it and reads nothing; no GPU."""
import contextlib

import pytest
import torch

FP8 = torch.float8_e4m3fn


class Counted:
    def __init__(self):
        self.calls = []

    def nsa_cache8_workspace_bytes(self, desc, out):
        out._obj.value = 256
        return 0

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    from native_sparse_attention_pytorch_amd import _lib, ops
    made = Counted()
    monkeypatch.setattr(_lib, "lib", lambda: made)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: {"cpu": 0, "meta": 1}[t.device.type], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    for plan in (ops._append_plan, ops._attend8_plan, ops._logits_plan):
        plan.cache_clear()
    yield made
    for plan in (ops._append_plan, ops._attend8_plan, ops._logits_plan):
        plan.cache_clear()


def codes(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(FP8)


def cache(b=2, hk=2, n=64, d=64, block=16):
    from native_sparse_attention_pytorch_amd.ops import Cache8
    return Cache8(codes(b, hk, n, d), codes(b, hk, n, d), torch.ones(b, hk, n // block), torch.ones(b, hk, n // block))


GOOD = cache()
BAD_CACHES = {
    "bytes": GOOD._replace(keys=GOOD.keys.view(torch.uint8)), "values of another type": GOOD._replace(values=torch.zeros(2, 2, 64, 64)),
    "e5m2": GOOD._replace(keys=GOOD.keys.view(torch.float8_e5m2)), "scales of another type": GOOD._replace(key_scales=GOOD.key_scales.bfloat16()),
    "fewer values": GOOD._replace(values=GOOD.values[:, :, :48]), "fewer scales": GOOD._replace(value_scales=GOOD.value_scales[:, :, :3]),
    "scales of other heads": GOOD._replace(key_scales=torch.ones(2, 3, 4), value_scales=torch.ones(2, 3, 4)),
    "three axes": cache()._replace(keys=codes(2, 64, 64), values=codes(2, 64, 64)), "80 features": cache(d=80), "blocks of 8": cache(block=8), "blocks of 48": cache(n=96, block=48),
    "an uneven last block": GOOD._replace(key_scales=torch.ones(2, 2, 3), value_scales=torch.ones(2, 2, 3)), "no rows": cache(n=0), "no sequences": cache(b=0),
    "keys and values laid out apart": GOOD._replace(values=codes(2, 64, 2, 64).transpose(1, 2)), "scales laid out apart": GOOD._replace(value_scales=torch.ones(2, 4, 2).transpose(1, 2)),
    "features apart": GOOD._replace(keys=codes(2, 2, 64, 128)[..., ::2], values=codes(2, 2, 64, 128)[..., ::2]),
    "rows off 16 bytes": GOOD._replace(keys=codes(2, 2, 64, 72)[..., :64], values=codes(2, 2, 64, 72)[..., :64]),
    "off a boundary": GOOD._replace(keys=codes(2, 2, 64, 80)[..., 8:72], values=codes(2, 2, 64, 80)[..., 8:72]),
    "rows that overlap": GOOD._replace(keys=codes(2, 2, 32, 64).as_strided((2, 2, 64, 64), (2048, 1024, 16, 1)), values=codes(2, 2, 32, 64).as_strided((2, 2, 64, 64), (2048, 1024, 16, 1))),
    "elsewhere": GOOD._replace(values=GOOD.values.to("meta")), "scales elsewhere": GOOD._replace(key_scales=GOOD.key_scales.to("meta")),
}
Q, K = torch.randn(2, 6, 1, 64), torch.randn(2, 2, 5, 64)
IDX, MASK = torch.zeros(2, 2, 1, 3, dtype=torch.int32), torch.ones(2, 2, 1, 3, dtype=torch.bool)
AT = torch.tensor([3, 4], dtype=torch.int32)


@pytest.mark.parametrize("what", BAD_CACHES)
def test_caches(library, what):
    from native_sparse_attention_pytorch_amd import ops
    c = BAD_CACHES[what]
    for call in (lambda: ops.cache8_append(c, K, K), lambda: ops.cache8_attend(Q, c, 5), lambda: ops.cache8_select_attend(Q, c, 5, 16, IDX, MASK),
                 lambda: ops.cache8_append_op(*c, K, K, None, 0, None), lambda: ops.cache8_attend_op(Q, *c, None, 5, 0, 0, None, None, 0.1))[:3 if "elsewhere" in what else 5]:
        with pytest.raises((RuntimeError, NotImplementedError), match="cache8|meta"):
            call()
    assert not library.calls


BAD_ROWS = {
    "doubles": (K.double(), K.double()), "two types": (K, K.bfloat16()), "fewer values": (K, K[:, :, :4]), "other heads": (torch.randn(2, 4, 5, 64),) * 2,
    "other sequences": (K[:1], K[:1]), "three axes": (K[0], K[0]), "too wide": (torch.randn(2, 2, 5, 65),) * 2, "no features": (K[..., :0], K[..., :0]),
    "past the end": (K, K, 60), "before the start": (K, K, -1), "real starts": (K, K, AT.float()), "three starts": (K, K, torch.zeros(3, dtype=torch.int32)),
    "a table of starts": (K, K, AT[:, None]), "short starts": (K, K, AT.short()), "starts elsewhere": (K, K, AT.to("meta")), "real counts": (K, K, 0, AT.float()),
    "one count": (K, K, 0, AT[:1]), "counts elsewhere": (K, K, 0, AT.to("meta")), "values elsewhere": (K, K.to("meta")),
}


@pytest.mark.parametrize("what", BAD_ROWS)
def test_rows(library, what):
    from native_sparse_attention_pytorch_amd import ops
    with pytest.raises((RuntimeError, NotImplementedError), match="cache8_append|meta"):
        ops.cache8_append(cache(), *BAD_ROWS[what])
    assert not library.calls


@pytest.mark.parametrize("shared", [GOOD._replace(keys=codes(1, 2, 64, 64).expand(2, 2, 64, 64), values=codes(1, 2, 64, 64).expand(2, 2, 64, 64)),
                                    GOOD._replace(key_scales=torch.ones(2, 1, 4).expand(2, 2, 4), value_scales=torch.ones(2, 1, 4).expand(2, 2, 4))])
def test_a_cache_whose_sequences_share_memory_is_read_only(library, shared):
    from native_sparse_attention_pytorch_amd import ops
    ops.cache8_attend(Q, shared, 5)
    assert len(library.calls) == 1
    with pytest.raises(RuntimeError, match="share memory"):
        ops.cache8_append(shared, K, K)
    rows_first = GOOD._replace(keys=codes(2, 64, 2, 64).transpose(1, 2), values=codes(2, 64, 2, 64).transpose(1, 2))
    ops.cache8_append(rows_first, K, K)
    assert len(library.calls) == 2


BAD_QUERIES = {
    "doubles": dict(q=Q.double()), "two tokens": dict(q=torch.randn(2, 6, 2, 64)), "three axes": dict(q=Q[:, :, 0]), "other sequences": dict(q=Q[:1]),
    "uneven heads": dict(q=Q[:, :5]), "too many heads": dict(q=torch.randn(2, 66, 1, 64)), "no heads": dict(q=Q[:, :0]), "too wide": dict(q=torch.randn(2, 6, 1, 100)),
    "elsewhere": dict(q=Q.to("meta")), "more keys than there are": dict(lengths=65), "fewer than none": dict(lengths=-1), "real lengths": dict(lengths=AT.float()),
    "three lengths": dict(lengths=torch.zeros(3, dtype=torch.int64)), "a table": dict(lengths=AT[None]), "lengths elsewhere": dict(lengths=AT.to("meta")),
}
BAD_SELECTIONS = {
    "no block": dict(block=0), "a negative block": dict(block=-16), "a block too large": dict(block=1 << 40), "real blocks": dict(idx=IDX.float()), "short blocks": dict(idx=IDX.short()),
    "a real mask": dict(fmask=MASK.float()), "a mask of others": dict(fmask=MASK[..., :2]), "three axes": dict(idx=IDX[:, :, 0], fmask=MASK[:, :, 0]),
    "of other heads": dict(idx=IDX[:, :1], fmask=MASK[:, :1]), "of two tokens": dict(idx=IDX.expand(2, 2, 2, 3), fmask=MASK.expand(2, 2, 2, 3)), "elsewhere": dict(idx=IDX.to("meta")),
}


@pytest.mark.parametrize("what", BAD_QUERIES)
def test_queries(library, what):
    from native_sparse_attention_pytorch_amd import ops
    given = {"q": Q, "lengths": 5, **BAD_QUERIES[what]}
    for call in (lambda: ops.cache8_attend(given["q"], cache(), given["lengths"]), lambda: ops.cache8_select_attend(given["q"], cache(), given["lengths"], 16, IDX, MASK)):
        with pytest.raises((RuntimeError, NotImplementedError), match="cache8|meta"):
            call()
    assert not library.calls


def test_windows(library):
    from native_sparse_attention_pytorch_amd import ops
    for window in (0, -3):
        with pytest.raises(RuntimeError, match="window"):
            ops.cache8_attend(Q, cache(), 5, window=window)
    ops.cache8_attend(Q, cache(), 5, window=1 << 40)           # (more than there can be: all)
    assert len(library.calls) == 1


@pytest.mark.parametrize("what", BAD_SELECTIONS)
def test_selections(library, what):
    from native_sparse_attention_pytorch_amd import ops
    given = {"block": 16, "idx": IDX, "fmask": MASK, **BAD_SELECTIONS[what]}
    with pytest.raises((RuntimeError, NotImplementedError), match="cache8_select_attend|meta"):
        ops.cache8_select_attend(Q, cache(), 5, given["block"], given["idx"], given["fmask"])
    assert not library.calls


X, H = torch.randn(3, 40), torch.zeros(3, 7, dtype=torch.int64)
BAD_LOGITS = {
    "doubles": dict(logits=X.double()), "whole logits": dict(logits=H), "no entries": dict(logits=X[:, :0]), "one number": dict(logits=X[0, 0]),
    "real history": dict(history=H.float()), "history of others": dict(history=H[:2]), "history of one": dict(history=H[0]), "bytes of history": dict(history=H.byte()),
    "lengths without history": dict(history_lengths=torch.zeros(3, dtype=torch.int32)), "lengths of others": dict(history=H, history_lengths=torch.zeros(2, dtype=torch.int32)),
    "real lengths": dict(history=H, history_lengths=torch.zeros(3)), "a short bias": dict(bias=torch.zeros(39)), "a bias of others": dict(bias=torch.zeros(2, 40)),
    "a whole bias": dict(bias=torch.zeros(40, dtype=torch.int64)), "a short mask": dict(allowed=torch.ones(39, dtype=torch.bool)), "bytes of a mask": dict(allowed=torch.ones(40, dtype=torch.uint8)),
    "words too few": dict(allowed=torch.ones(1, dtype=torch.int32)), "words of others": dict(allowed=torch.ones(2, 2, dtype=torch.int32)), "long words": dict(allowed=torch.ones(2, dtype=torch.int64)),
    "penalties of others": dict(repetition_penalty=torch.ones(2)), "whole penalties": dict(frequency_penalty=torch.ones(3, dtype=torch.int64)),
    "a table of temperatures": dict(temperature=torch.ones(1, 3)), "history elsewhere": dict(history=H.to("meta")), "a bias elsewhere": dict(bias=torch.zeros(40, device="meta")),
    "a temperature elsewhere": dict(temperature=torch.ones(3, device="meta")),
}


@pytest.mark.parametrize("what", BAD_LOGITS)
def test_logits(library, what):
    from native_sparse_attention_pytorch_amd import ops
    given = dict(BAD_LOGITS[what])
    with pytest.raises((RuntimeError, NotImplementedError), match="adjust_logits|meta"):
        ops.adjust_logits(given.pop("logits", X), **given)
    assert not library.calls


@pytest.mark.parametrize("bad", [dict(repetition_penalty=0.), dict(repetition_penalty=-1), dict(repetition_penalty=float("inf")), dict(temperature=0), dict(temperature=float("nan")),
                                 dict(frequency_penalty=float("nan")), dict(presence_penalty=float("inf"))])
def test_numbers(library, bad):
    from native_sparse_attention_pytorch_amd import ops
    with pytest.raises(ValueError, match="adjust_logits"):
        ops.adjust_logits(X, H, **bad)
    assert not library.calls


def test_gradients_and_tangents(library):
    from torch.autograd import forward_ad

    from native_sparse_attention_pytorch_amd import ops
    for call in (lambda t: ops.cache8_attend(t(Q), cache(), 5), lambda t: ops.cache8_append(cache(), t(K), K), lambda t: ops.cache8_append(cache(), K, t(K)),
                 lambda t: ops.cache8_select_attend(t(Q), cache(), 5, 16, IDX, MASK), lambda t: ops.adjust_logits(t(X)), lambda t: ops.adjust_logits(X, bias=t(X[0])),
                 lambda t: ops.adjust_logits(X, temperature=t(X[:, 0]))):
        needs = lambda x: x.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            call(needs)
        with pytest.raises(NotImplementedError, match="forward mode"), torch.no_grad(), forward_ad.dual_level():
            call(lambda x: forward_ad.make_dual(x, torch.ones_like(x)))
        assert not library.calls
        with torch.no_grad():
            call(needs)
        assert library.calls.pop()


def test_a_call_goes_to_the_device_of_its_tensors(library, monkeypatch):
    from native_sparse_attention_pytorch_amd import ops
    current, seen = [3], []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        seen.append(index)
        yield
        current[0] = before
    monkeypatch.setattr(torch.cuda, "device", device)
    ops.cache8_append(cache(), K, K)
    ops.cache8_attend(Q, cache(), 5)
    ops.adjust_logits(X)
    assert seen == [0, 0, 0] and current[0] == 3 and len(library.calls) == 3


def test_host_tensors():
    from native_sparse_attention_pytorch_amd import ops
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.cache8_append(cache(), K, K)
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.cache8_attend(Q, cache(), 5)
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.adjust_logits(X)


@pytest.mark.parametrize("bad", [dict(block=24), dict(rows=0), dict(batch=0), dict(kv_heads=0), dict(dim_head=0)])
def test_making_a_cache(bad):
    from native_sparse_attention_pytorch_amd import ops
    given = {**dict(batch=1, kv_heads=2, rows=20, dim_head=48, block=32), **bad}
    with pytest.raises(ValueError, match="make_cache8"):
        ops.make_cache8(**given, device="cpu")
    with pytest.raises(RuntimeError, match="128 features"):
        ops.make_cache8(1, 1, 16, 129, device="cpu")
    made = ops.make_cache8(1, 2, 20, 48, device="cpu")
    assert made.keys.shape == (1, 2, 32, 64) and made.key_scales.shape == (1, 2, 1) and made.block == 32


def test_entries_refuse_what_they_cannot_run():
    """The library's own checks, before any launch."""
    import ctypes as C

    from native_sparse_attention_pytorch_amd import _lib
    from native_sparse_attention_pytorch_amd.ops import _CACHE8_DESC, _LOGITS_DESC
    L, n = _lib.lib(), C.c_size_t()
    names = "batch hk group dim block cap dtype length lstride window size chosen per_head idx64 scale reserved s0 s1 s2 z0 z1 q0 q1".split()
    good = dict(zip(names, (2, 2, 4, 64, 16, 64, 0, 0, 0, 0, 0, 0, 0, 0, 0.1, 0, 8192, 4096, 64, 8, 4, 512, 64)))
    ask = lambda **bad: L.nsa_cache8_workspace_bytes(_CACHE8_DESC.pack(*{**good, **bad}.values()), C.byref(n))
    assert ask() == 0
    for bad in (dict(batch=0), dict(hk=0), dict(group=0), dict(cap=0), dict(cap=63), dict(block=0), dict(dtype=3), dict(dtype=-1), dict(window=-1), dict(size=-1), dict(chosen=-1),
                dict(s0=8), dict(s1=8), dict(s2=72), dict(s2=48), dict(reserved=1)):
        assert ask(**bad) == -1, bad
    for bad in (dict(dim=96, s2=96), dict(block=8), dict(block=48, cap=96), dict(group=33), dict(cap=1 << 30, block=64, batch=1 << 22), dict(size=1 << 29, chosen=2),
                dict(chosen=(1 << 20) + 1, size=1), dict(s2=1 << 31)):
        assert ask(**bad) == -2, bad
    assert L.nsa_cache8_workspace_bytes(None, C.byref(n)) == -1 and L.nsa_cache8_workspace_bytes(_CACHE8_DESC.pack(*good.values()), None) == -1
    three = C.c_int64 * 3
    at = 1 << 20
    append = lambda rows=1, k=at, v=at, keys=at, values=at, ks=at, vs=at, stride=(512, 256, 64), **bad: L.nsa_cache8_append(
        _CACHE8_DESC.pack(*{**good, **bad}.values()), rows, k, three(*stride), v, three(*stride), None, None, keys, values, ks, vs, 0)
    assert append(rows=0) == 0
    for bad in (dict(rows=-1), dict(k=0), dict(v=0), dict(keys=0), dict(values=0), dict(ks=0), dict(vs=0), dict(k=at + 8), dict(keys=at + 8), dict(stride=(512, 256, 60)), dict(batch=0)):
        assert append(**bad) == -1, bad
    assert append(dim=96, s2=96) == -2 and append(batch=1 << 25) == -2
    attend = lambda q=at, keys=at, values=at, ks=at, vs=at, idx=at, mask=at, ws=at, bytes_=1 << 30, out=at, **bad: L.nsa_cache8_attend(
        _CACHE8_DESC.pack(*{**good, **bad}.values()), q, keys, values, ks, vs, None, idx, mask, ws, bytes_, out, 0)
    for bad in (dict(q=0), dict(q=at + 2), dict(keys=0), dict(keys=at + 4), dict(values=0), dict(ks=0), dict(vs=0), dict(out=0), dict(q0=4), dict(q1=4), dict(size=16, chosen=2, idx=0),
                dict(size=16, chosen=2, mask=0), dict(cap=4096, ws=0), dict(cap=4096, ws=at + 4)):
        assert attend(**bad) == -1, bad
    assert attend(cap=4096, bytes_=16) == -3
    names = "rows stride vocab dtype history h64 kind bstride astride r f p t rep freq pres temp".split()
    row = dict(zip(names, (2, 40, 40, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1., 0., 0., 1.)))
    adjust = lambda x=at, history=None, allowed=None, out=at, **bad: L.nsa_adjust_logits(_LOGITS_DESC.pack(*{**row, **bad}.values()), x, history, None, None, None, None, None,
                                                                                        allowed, None, out, 0)
    assert adjust(rows=0) == 0
    for bad in (dict(rows=-1), dict(vocab=0), dict(dtype=3), dict(history=None, h64=0, kind=3), dict(kind=1), dict(kind=2), dict(x=0), dict(out=0)):
        assert adjust(**bad) == -1, bad
    assert L.nsa_adjust_logits(None, at, None, None, None, None, None, None, None, None, at, 0) == -1
    assert adjust(rows=(1 << 30) + 1) == -2 and adjust(rows=1 << 25) == -2
