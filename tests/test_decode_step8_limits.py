"""Which decode steps over an 8-bit cache the library takes, as its workspace query answers on the host; no GPU."""
import ctypes as C

import pytest


def _ask(capacity=(), cache=()):
    from native_sparse_attention_pytorch_amd import _lib
    from native_sparse_attention_pytorch_amd.ops import _CACHE8_DESC
    d = _lib.DecodeStepDesc()
    good = dict(batch=2, heads=4, kv_heads=2, dim_head=64, pos=95, num_compressed=16, per_block=2, block=16, num_sel=2, share=1, window=16, scale=0.125, num_mem=1)
    for name, value in {**good, **dict(capacity)}.items():
        setattr(d, name, value)
    d.kc_stride[:] = d.vc_stride[:] = (2 * 96 * 64, 96 * 64, 64)
    d.ck_stride[:] = d.cv_stride[:] = (2 * 17 * 64, 17 * 64, 64)
    d.krun_stride[:] = d.vrun_stride[:] = (2 * 32 * 64, 32 * 64)
    d.q_stride[:] = d.k_stride[:] = d.v_stride[:] = (528, 64)
    names = "batch kv_heads group dim block cap dtype length step window size chosen per_head idx64 scale reserved s0 s1 s2 z0 z1 q0 q1".split()
    of = dict(zip(names, (2, 2, 2, 64, 32, 96, 0, 0, 0, 0, 0, 0, 0, 0, 0.125, 0, 2 * 96 * 64, 96 * 64, 64, 6, 3, 0, 0)))
    n = C.c_size_t()
    rc = _lib.lib().nsa_decode_step8_workspace_bytes(C.byref(d), _CACHE8_DESC.pack(*{**of, **dict(cache)}.values()), C.byref(n))
    return rc, n.value


def test_steps_that_are_taken():
    for capacity in ({}, dict(num_compressed=1), dict(num_sel=0), dict(per_block=3, block=24), dict(share=0), dict(window=0)):
        rc, n = _ask(capacity)
        assert rc == 0 and n > 0, capacity


@pytest.mark.parametrize("capacity, cache", [(dict(num_compressed=0), {}), (dict(num_compressed=0, num_sel=0, num_mem=0), {}), (dict(heads=128), dict(group=64)),
                                             (dict(per_block=1, num_compressed=2049), {}), (dict(num_sel=65, num_compressed=200), {}), ({}, dict(s2=1 << 28))])
def test_steps_that_are_refused(capacity, cache):
    """Layers without compressed keys, groups of more than 32 heads, more blocks than a wave chooses from, rows too far apart."""
    assert _ask(capacity, cache)[0] == -2


@pytest.mark.parametrize("cache", [dict(group=4), dict(batch=3), dict(dtype=1), dict(cap=64), dict(dim=128, s2=128), dict(reserved=1), dict(kv_heads=1)])
def test_caches_of_another_step(cache):
    assert _ask(cache=cache)[0] == -1
