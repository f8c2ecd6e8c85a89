"""ops.newton_schulz and training.Muon against float64.

Bound.  With the default coefficients singular values stay below 1.21, where the slope of s -> a s + b s^3 + c s^5, and with it what a step
makes of an error (its divided differences lie within the slopes), is at most 4.  Beginning with norm 1, five steps make at most 4^5 = 2^10 of the first
rounding; a later one is relative to X, which grows by at most 3.45 a step, and met by the fewer steps left: together 4 times as much for each
unit.  A step rounds X, A, B (22 bits and more: 2^-23 at most) and sums; |a| + |b| |A| + |c| |A|^2 of it reach X: 8 units.  So the error's norm is at
most 2^10 * 4 * 8 * 2^-23 = 2^-8, beside a rounding of the result.  That holds for the worst case; errors of different elements are independent, and the
test that the result is no less exact than with fp32 products is the sharper one."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ABC = (3.4445, -4.7750, 2.0315)


def _exact(g, steps=5, abc=ABC, eps=1e-7, dtype=torch.float64):
    a, b, c = abc
    x = g.to(dtype)
    x = x / (torch.linalg.matrix_norm(x.double(), keepdim=True).to(dtype) + eps)
    turned = x.shape[-2] > x.shape[-1]
    x = (x.mT if turned else x).contiguous()
    for _ in range(steps):
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if turned else x


def _check(got, g, **kw):
    want = _exact(g, **kw)
    assert got.shape == g.shape and got.dtype == g.dtype and got.is_contiguous()
    off = torch.linalg.matrix_norm(got.double() - want)
    assert (off <= 2 ** -8 + torch.finfo(g.dtype).eps / 2 * torch.linalg.matrix_norm(want) + torch.finfo(g.dtype).tiny).all(), float(off.max())


def _g(*size, dtype=F32, seed=0, scale=1.):
    return (torch.randn(*size, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 500), (500, 1), (3, 2), (24, 512), (31, 33), (64, 64), (65, 63), (63, 129), (129, 64), (200, 1000),
                                 (1000, 200), (257, 255), (520, 516)])
def test_sizes_and_types(m, n, dtype):
    from native_sparse_attention_pytorch_amd import ops
    g = _g(m, n, dtype=dtype)
    _check(ops.newton_schulz(g), g)


@pytest.mark.parametrize("m,n", [(2049, 2050), (4100, 1100), (1030, 8200)])
def test_large_tiles(m, n):
    from native_sparse_attention_pytorch_amd import ops
    g = _g(m, n)
    got = ops.newton_schulz(g)
    _check(got, g)
    off = lambda x: float((x.double() - _exact(g)).norm())
    assert off(got) <= 1.5 * off(_exact(g, dtype=F32)) + 1e-6 * min(m, n) ** 0.5


@pytest.mark.parametrize("m,n", [(1, 1), (9, 40), (17, 33), (40, 40), (24, 512), (64, 300), (48, 48), (70, 130), (130, 3000), (512, 512), (1000, 300)])
def test_no_less_exact_than_fp32_products(m, n):
    """Of what the result is (its norm is about the root of the smaller side), or 1e-6 of it."""
    from native_sparse_attention_pytorch_amd import ops
    for seed in range(3):
        g = _g(m, n, seed=seed)
        want = _exact(g)
        off = lambda x: float((x.double() - want).norm() / want.norm())
        assert off(ops.newton_schulz(g)) <= max(1e-6, 1.5 * off(_exact(g, dtype=F32))), seed


@pytest.mark.parametrize("m,n", [(40, 60), (200, 130)])
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-9, 3e-8, 1e-6, 1e30])
def test_norms_beside_eps_and_far_from_it(m, n, scale):
    """Where the norm is small beside eps, X starts at norm / eps and stays near linear: a few units of 2^-22 of it a step."""
    from native_sparse_attention_pytorch_amd import ops
    g = _g(m, n, scale=scale)
    got, want = ops.newton_schulz(g), _exact(g)
    assert float((got.double() - want).norm()) <= 2 ** -14 * float(want.norm())
    _check(got, g)


def test_zeros_and_what_is_not_finite():
    from native_sparse_attention_pytorch_amd import ops
    for m, n in ((5, 9), (70, 300)):
        assert not ops.newton_schulz(torch.zeros(m, n, device=DEV)).any()
        assert ops.newton_schulz(torch.zeros(m, n, device=DEV), eps=0.).isnan().all()
        g = _g(m, n)
        clean = ops.newton_schulz(g)
        g2 = g.clone()
        g2[2, 3] = math.nan
        bad, good = ops.newton_schulz([g2, g])
        assert bad.isnan().all() and torch.equal(good, clean)
        g2[2, 3] = math.inf
        assert not ops.newton_schulz(g2).isfinite().all()


def test_few_directions():
    """Rank one and rank two: the directions that are there come out near 1, the others stay what rounding makes of zero."""
    from native_sparse_attention_pytorch_amd import ops
    for m, n in ((30, 50), (300, 200)):
        g = _g(m, 1) @ _g(1, n, seed=1)
        _check(ops.newton_schulz(g), g)
        s = torch.linalg.svdvals(ops.newton_schulz(g).double())
        assert 0.6 < s[0] < 1.25 and s[1] < 2 ** -8


def test_lists_batches_and_layouts():
    from native_sparse_attention_pytorch_amd import ops
    gs = [_g(24, 512), _g(3, 100, 70, seed=1), _g(70, 100, dtype=BF16, seed=2), _g(2, 2, 40, 30, seed=3), _g(0, 5), _g(2, 0, 4, seed=4)]
    out = ops.newton_schulz(tuple(gs))
    assert isinstance(out, tuple) and [o.shape for o in out] == [g.shape for g in gs]
    for o, g in zip(out, gs):
        assert o.dtype == g.dtype
        if g.numel():
            _check(o, g)
    # the same matrices alone and in other layouts, each next to others of the same sizes: the same bits
    wide = _g(100, 90, seed=5)
    view = wide[3:73, 7:87]
    alone = ops.newton_schulz([view.contiguous()])[0]
    padded = torch.zeros(70, 81, device=DEV)[:, 1:]
    padded.copy_(view)
    for other in (view, padded, view.t().contiguous().t(), view.clone()[None][0]):
        assert torch.equal(ops.newton_schulz(other), alone)
    assert torch.equal(ops.newton_schulz(torch.stack((view, view)))[1], ops.newton_schulz([view, view.contiguous()])[0])
    _check(ops.newton_schulz(view[:1].expand(70, 80)), view[:1].expand(70, 80).contiguous())


def test_more_matrices_than_one_launch_takes():
    from native_sparse_attention_pytorch_amd import ops
    gs = [_g(8 + i, 70 - i % 9, seed=i) for i in range(130)]
    for o, g in zip(ops.newton_schulz(gs), gs):
        _check(o, g)
    many = _g(200, 12, 20, seed=7)
    _check(ops.newton_schulz(many), many)


@pytest.mark.parametrize("steps,abc", [(1, ABC), (2, ABC), (10, ABC), (12, (1.5, -0.5, 0.)), (6, (1.875, -1.25, 0.375)), (3, (0.5, 0., 0.))])
@pytest.mark.parametrize("m,n", [(30, 45), (150, 90)])
def test_steps_and_coefficients(m, n, steps, abc):
    """(slopes of at most 4 for all of these; with more steps the first rounding has grown no further: values near 1 are where slopes are below 1.7)"""
    from native_sparse_attention_pytorch_amd import ops
    g = _g(m, n)
    _check(ops.newton_schulz(g, steps=steps, coefficients=abc), g, steps=steps, abc=abc)


def test_refusals():
    from native_sparse_attention_pytorch_amd import ops
    g = _g(4, 4)
    with pytest.raises(RuntimeError, match="expected bf16, fp16 or fp32 matrices"):
        ops.newton_schulz(g.double())
    with pytest.raises(RuntimeError, match="expected bf16, fp16 or fp32 matrices"):
        ops.newton_schulz(g[0])
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.newton_schulz(g.requires_grad_())
    with pytest.raises(RuntimeError, match="on one GPU"):
        ops.newton_schulz([g.detach(), torch.zeros(2, 2)])


def test_captured_replay_and_another_stream():
    from native_sparse_attention_pytorch_amd import ops
    held = [_g(130, 70), _g(24, 100, seed=1)]
    ops.newton_schulz(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.newton_schulz(held)
    for seed in range(4):
        new = [_g(130, 70, seed=seed, scale=10. ** -seed), _g(24, 100, seed=seed + 9)]
        for h, g in zip(held, new):
            h.copy_(g)
        graph.replay()
        want = ops.newton_schulz(new)
        torch.cuda.synchronize()
        for o, w in zip(out, want):
            assert torch.equal(o, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.newton_schulz(new)
    side.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(other, want))


@pytest.mark.parametrize("nesterov,decay", [(True, 0.1), (False, 0.)])
def test_muon_steps(nesterov, decay):
    """Three steps against the same formulas in float64; a parameter without a gradient stays, one of three axes is a matrix of its first."""
    from native_sparse_attention_pytorch_amd.training import Muon
    shapes = [(40, 24), (24, 40), (65, 130), (6, 5, 4), (10, 10)]
    params = [torch.nn.Parameter(_g(*s, seed=i)) for i, s in enumerate(shapes)]
    exact = [p.detach().double() for p in params]
    buffers = [torch.zeros_like(e) for e in exact]
    lr = 0.05
    opt = Muon(params, lr=lr, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    tol = 0.
    for step in range(3):
        for i, p in enumerate(params[:-1]):
            p.grad = _g(*p.shape, seed=100 + 10 * step + i)
        opt.step()
        for i in range(4):
            g = params[i].grad.double()
            buffers[i] = 0.9 * buffers[i] + g
            u = (g + 0.9 * buffers[i] if nesterov else buffers[i]).flatten(1)
            exact[i] = (1 - lr * decay) * exact[i] - lr * max(1, u.shape[0] / u.shape[1]) ** 0.5 * _exact(u).view(exact[i].shape)
        # an update within 2^-8 (see above; its own rounding of the momentum in fp32 is among the 8 units), fp32 elsewhere
        tol += lr * 2 ** 0.5 * 2 ** -8 + 1e-5
        for p, e in zip(params, exact):
            assert float((p.detach().double() - e).norm()) <= tol
    assert "momentum_buffer" not in opt.state[params[-1]]
    again = Muon(params, lr=lr)
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[params[0]]["momentum_buffer"], opt.state[params[0]]["momentum_buffer"])


@pytest.mark.parametrize("m,n", [(70, 80), (130, 70), (128, 1000), (512, 512), (1024, 600)])
def test_bf16_results_are_off_by_their_rounding(m, n):
    """The last two steps of a bf16 result are made of fp16 values, 2^-12 off each: together at most half of what rounding the result to bf16
    adds (2^-9 on average over a binade's values 2^-9.2), so at most sqrt(1 + 1/4) of it."""
    from native_sparse_attention_pytorch_amd import ops
    for seed in range(3):
        g = _g(m, n, dtype=BF16, seed=seed)
        want = _exact(g)
        off = lambda x: float((x.double() - want).norm())
        assert off(ops.newton_schulz(g)) <= 1.25 ** 0.5 * off(want.to(BF16)), seed


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n", [(70, 130), (300, 200)])
@pytest.mark.parametrize("eps", [1e-7, 1., 30., 1e3])
def test_16_bit_matrices_begin_exactly(m, n, dtype, eps):
    """They are held as they are, times a power of two, whatever the norm: fp16 results are fp32's and a rounding (2^-14: a few units of 2^-22 a
    step, as for fp32); bf16's last two steps add at most half of the rounding."""
    from native_sparse_attention_pytorch_amd import ops
    for scale in (1., 3.7, 2 ** -9):
        g = _g(m, n, dtype=dtype, scale=scale)
        got, want = ops.newton_schulz(g, eps=eps), _exact(g, eps=eps)
        off = lambda x: float((x.double() - want).norm())
        assert off(got) <= (1.25 ** 0.5 if dtype == BF16 else 1.) * off(want.to(dtype)) + 2 ** -14 * float(want.norm()), scale


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("steps", [1, 2, 3, 4])
def test_few_steps_of_16_bits(dtype, steps):
    """One and two steps of a bf16 result are made of fp16 values from the beginning: 8 roundings of 2^-12 a step, each growing at most 4 times in a
    step that follows or makes it."""
    from native_sparse_attention_pytorch_amd import ops
    for m, n in ((130, 70), (90, 3000)):
        g = _g(m, n, dtype=dtype)
        got, want = ops.newton_schulz(g, steps=steps), _exact(g, steps=steps)
        off = float((got.double() - want).norm())
        tol = 8 * 2 ** -12 * (4, 20)[steps - 1] if dtype == BF16 and steps < 3 else 2 ** -8
        assert off <= tol + torch.finfo(dtype).eps / 2 * float(want.norm())


def test_a_parameter_without_elements_is_left_alone():
    from native_sparse_attention_pytorch_amd.training import Muon
    params = [torch.nn.Parameter(torch.zeros(5, 0, device=DEV)), torch.nn.Parameter(_g(6, 4))]
    for p in params:
        p.grad = torch.ones_like(p)
    before = params[1].detach().clone()
    Muon(params).step()
    assert not torch.equal(params[1], before) and params[0].shape == (5, 0)


@pytest.mark.parametrize("m,n,dtype", [(24, 512, F32), (130, 70, F16), (70, 130, BF16)])
def test_in_place(m, n, dtype):
    """The C entry writes a contiguous matrix over itself; the operator never writes its arguments."""
    import ctypes as C

    from native_sparse_attention_pytorch_amd import _lib, ops
    g = _g(m, n, dtype=dtype)
    kept = g.clone()
    want = ops.newton_schulz(g)
    assert torch.equal(g, kept)
    ints, longs, ptrs, need = C.c_int32 * 1, C.c_int64 * 1, C.c_void_p * 1, C.c_size_t()
    _lib.check(_lib.lib().nsa_newton_workspace_bytes(1, ints(m), ints(n), C.byref(need)), "nsa_newton_workspace_bytes")
    ws = torch.empty(need.value, dtype=torch.uint8, device=DEV)
    code = {BF16: 0, F16: 1, F32: 2}[dtype]
    _lib.check(_lib.lib().nsa_newton_schulz(1, ints(m), ints(n), ptrs(g.data_ptr()), longs(n), ptrs(g.data_ptr()), code, 5, *ABC, 1e-7, ws.data_ptr(),
                                            need.value, torch.cuda.current_stream().cuda_stream), "nsa_newton_schulz")
    assert torch.equal(g, want)


def test_two_graphs_and_launches_between_them():
    """Two captured calls keep their own workspaces: replayed in turn, with launched calls between them, each gives its own result."""
    from native_sparse_attention_pytorch_amd import ops
    held = [[_g(130, 70, seed=1), _g(40, 600, seed=2)], [_g(90, 300, seed=3)]]
    for h in held:
        ops.newton_schulz(h)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.newton_schulz(h))
        graphs.append(graph)
    for seed in range(3):
        for h in held:
            for i, t in enumerate(h):
                t.copy_(_g(*t.shape, seed=10 * seed + i))
        for graph in graphs:
            graph.replay()
        want = [ops.newton_schulz(h) for h in held]
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for out, ws in zip(outs, want) for o, w in zip(out, ws))


def test_traced():
    from native_sparse_attention_pytorch_amd import ops
    gs = [_g(70, 130), _g(24, 100, seed=1)]
    want = ops.newton_schulz(gs)
    got = torch.compile(lambda a, b: ops.newton_schulz([a, b]), backend="aot_eager", fullgraph=True)(*gs)
    assert all(torch.equal(o, w) for o, w in zip(got, want))
    with pytest.raises(RuntimeError, match="nsa_newton_schulz"):
        torch.compile(lambda a, b: ops.newton_schulz([a, b], coefficients=(5., 0., 0.)), backend="aot_eager", fullgraph=True)(*gs)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_muon_of_16_bit_parameters(dtype):
    """The momentum is held in fp32, through a saved state too; the parameter is rounded at each of a step's two operations on it."""
    from native_sparse_attention_pytorch_amd.training import Muon
    p = torch.nn.Parameter(_g(70, 40, dtype=dtype))
    opt = Muon([p], lr=0.05, momentum=0.9, weight_decay=0.1)
    buffer = torch.zeros(70, 40, dtype=torch.float64, device=DEV)
    for step in range(3):
        p.grad = _g(70, 40, dtype=dtype, seed=20 + step, scale=2. ** -12 if step else 1.)      # (2^-12 of the buffer: gone in 16 bits)
        buffer = 0.9 * buffer + p.grad.double()
        want = (1 - 0.05 * 0.1) * p.detach().double() - 0.05 * (70 / 40) ** 0.5 * _exact(p.grad.double() + 0.9 * buffer)
        opt.step()
        u = torch.finfo(dtype).eps / 2
        assert float((p.detach().double() - want).norm()) <= 2 * 1.01 * u * float(want.norm()) + 0.05 * (70 / 40) ** 0.5 * 2 ** -8
        kept = opt.state[p]["momentum_buffer"]
        assert kept.dtype == F32 and float((kept.double() - buffer).abs().max()) <= 2 ** -22 * float(buffer.abs().max())
    again = Muon([p], lr=0.05)
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[p]["momentum_buffer"], kept) and again.state[p]["momentum_buffer"].dtype == F32
    assert again.state[p]["momentum_buffer"].data_ptr() != kept.data_ptr() and again.param_groups[0]["momentum"] == 0.9
