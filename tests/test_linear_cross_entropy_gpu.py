"""ops.linear_cross_entropy against float64, forward and gradients.

Bounds, from the arithmetic (u = torch.finfo(type).eps / 2; fp32 operands are held in 22 bits and more, H = 2^-22, the others exactly, H = 0):
  a logit     d products in fp32 sums of 16 (three of them for fp32 operands): dL = ((d / 4 + 8) 2^-24 + 2 H) |x| |w|^T
  lse         moves by at most the largest dL of its row; exponentials and their sum are off by 2^-16 of themselves (chains of at most 250
              additions), the logarithm by two steps of the result
  G           fp16, 2^-11 of itself (fp32: H) and 2^-38 of the largest weight, beside p (dL + d lse + 2^-18)
  gradients   the operands' own H and 2^-38 of their largest value, fp32 sums, and one rounding u
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(n, d, v, dtype, seed=0, ignored=0.2, scale=1.):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, d, generator=g) * scale).to(dtype)
    w = (torch.randn(v, d, generator=g) * d ** -0.5).to(dtype)
    labels = torch.randint(0, v, (n,), generator=g)
    labels[torch.rand(n, generator=g) < ignored] = -100
    return x.to(DEV), w.to(DEV), labels.to(DEV), torch.rand(n, generator=g).to(DEV) + 0.1


def _exact(x, w, labels, reduction, weights, ignore=-100):
    """float64: (loss, tolerance), (dx, tolerance), (dw, tolerance); `weights`: one per row, or the one of the loss."""
    h = 2 ** -22 if x.dtype == F32 else 0.
    u = torch.finfo(x.dtype).eps / 2
    n, d, v = *x.shape, len(w)
    live = labels != ignore
    x6, w6 = x.double()[live], w.double()
    lab, count = labels[live].long(), int(live.sum())
    logits, size = x6 @ w6.t().contiguous(), x6.abs() @ w6.abs().t().contiguous()
    dl = ((d / 4 + 8) * 2 ** -24 + 2 * h) * size
    lse = torch.logsumexp(logits, -1)
    own = logits.gather(1, lab[:, None])[:, 0]
    dlse = dl.amax(-1) + 2 ** -16 + 2 ** -22 * lse.abs()
    each = torch.zeros(n, dtype=torch.float64, device=DEV)
    off = torch.zeros_like(each)
    each[live] = lse - own
    off[live] = dlse + dl.gather(1, lab[:, None])[:, 0] + 2 ** -22 * (lse.abs() + own.abs())
    if reduction == "none":
        loss, dloss = each, off
        g = weights.double()[live]
    else:
        by = count if reduction == "mean" else 1
        loss = each.sum() / by if by else each.sum() * math.nan
        dloss = off.sum() / max(by, 1) + 2 ** -23 * loss.abs()
        g = (weights.double() / max(by, 1)).expand(count)
    p = torch.exp(logits - lse[:, None])
    G = p.clone()
    G[torch.arange(count, device=DEV), lab] -= 1
    G *= g[:, None]
    top = float(g.abs().max()) if count else 0.
    dG = g.abs()[:, None] * p * (dl + dlse[:, None] + 2 ** -18) + (2 ** -11 if x.dtype != F32 else h) * G.abs() + 2 ** -38 * top
    grads = []
    for a, da, b, k in ((G, dG, w6, v), (G.t().contiguous(), dG.t().contiguous(), x6, count)):
        most = float(b.abs().max()) if b.numel() else 0.
        want = a @ b
        tol = da @ b.abs() + a.abs() @ (h * b.abs() + 2 ** -38 * most) + (k / 4 + 16) * 2 ** -24 * (a.abs() @ b.abs())
        grads.append((want, 1.01 * tol + u * want.abs() + torch.finfo(x.dtype).tiny * 2 * u))
    dx, tx = torch.zeros(n, d, dtype=torch.float64, device=DEV), torch.zeros(n, d, dtype=torch.float64, device=DEV)
    dx[live], tx[live] = grads[0]
    return (loss, dloss), (dx, tx), grads[1]


def _within(got, want, what):
    want, tol = want
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got.double() - want).abs() <= tol) & ~(got.isnan() & want.isnan())
    assert not bad.any(), (what, int(bad.sum()), bad.numel(), bad.nonzero()[:3].tolist(), float((got.double() - want).abs().nan_to_num().max()))


def _check(x, w, labels, reduction, weights, ignore=-100):
    from native_sparse_attention_pytorch_amd import ops
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    weights = weights if reduction == "none" else weights[0]
    loss = ops.linear_cross_entropy(x, w, labels, ignore_index=ignore, reduction=reduction)
    assert loss.dtype == F32
    dx, dw = torch.autograd.grad(loss, (x, w), weights)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    want = _exact(x.detach(), w.detach(), labels, reduction, weights, ignore)
    for got, exact, what in zip((loss.detach(), dx, dw), want, ("loss", "dx", "dw")):
        _within(got, exact, what)
    return loss.detach(), dx, dw


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,d,v,reduction", [
    (1, 1, 1, "mean"),             # one logit: loss and gradients zero
    (1, 64, 2, "sum"),
    (3, 7, 63, "none"),            # features that are no multiple of anything
    (31, 64, 257, "mean"),         # up to 32 rows: tiles of 32 tokens
    (33, 100, 65, "none"),         # one row past them
    (64, 129, 129, "mean"),
    (127, 192, 1000, "sum"),
    (129, 72, 255, "none"),
    (300, 512, 256, "mean"),       # the byte-level model's vocabulary
])
def test_small_and_odd_sizes(n, d, v, reduction, dtype):
    _check(*_inputs(n, d, v, dtype)[:3], reduction, _inputs(n, d, v, dtype)[3])


@pytest.mark.parametrize("n,d,v,dtype", [
    (2050, 64, 16391, BF16),       # tiles of 256 x 256, cut on every side
    (2050, 72, 16391, F32),
    (16390, 64, 9001, BF16),       # gradients in two pieces of the vocabulary
    (16390, 64, 9001, F32),        # three pieces
    (40, 4100, 17001, F32),        # the forward's planes in two pieces
    (24, 256, 40003, BF16),        # few rows, a slice of the vocabulary for each part of dx
])
def test_large_tiles_and_pieces(n, d, v, dtype):
    x, w, labels, weights = _inputs(n, d, v, dtype, seed=3)
    _check(x, w, labels, "none", weights)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,d,v", [
    (1, 8, 129),                   # features short of one copy of 128 bytes
    (2, 63, 128),
    (4, 65, 300),
    (16, 128, 31),
    (17, 256, 500),                # whole sums of 256
    (31, 264, 127),                # and one step more
    (32, 1000, 385),
    (32, 520, 1),
    (3, 7, 16383),                 # the last vocabulary of narrow tiles
    (17, 65, 16400),               # and wide ones
    (31, 264, 20001),
    (5, 1000, 16385),
])
def test_few_rows(n, d, v, dtype):
    """Up to 32 rows, from rows at multiples of 16 bytes and from others: the same sums in the same order."""
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(n, d, v, dtype, seed=d, ignored=0.3 if n > 2 else 0.)
    _check(x, w, labels, "none", weights)
    wide = max(8, (d + 7) // 8 * 8) + 8
    at = [torch.randn(r, wide, device=DEV).to(dtype) for r in (n, v, n, v)]
    at[0][:, :d], at[1][:, :d], at[2][:, 1:d + 1], at[3][:, 3:d + 3] = x, w, x, w
    want = ops.linear_cross_entropy(at[0][:, :d], at[1][:, :d], labels, reduction="none")
    got = ops.linear_cross_entropy(at[2][:, 1:d + 1], at[3][:, 3:d + 3], labels.int(), reduction="none")
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,d,v", [
    (70, 72, 700),                 # rows in place, their last 64 features read with what is left of them
    (200, 200, 2500),
    (1500, 120, 5000),
    (600, 1096, 1100),
    (1100, 520, 40001),            # tiles of 256
    (33, 2056, 1500),              # tiles of 64, long sums
])
def test_features_short_of_whole_steps(n, d, v, dtype):
    x, w, labels, weights = _inputs(n, d, v, dtype, seed=5)
    _check(x, w, labels, "none", weights)
    wide = torch.randn(v, d + 24, device=DEV).to(dtype)
    wide[:, 8:d + 8] = w
    _check(x, wide[:, 8:d + 8], labels, "mean", weights)


@pytest.mark.parametrize("n", [20, 100])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_likely_labels(n, dtype):
    """Losses down to 1e-12.  Where the label has the row's largest logit by far, its own logit's error drops out: the loss, and its G but for the
    weight, are a sum of the others' exponentials, each off by two logits' dL and 2^-16 of itself, beside the label's own 1.  That 1 goes
    through at most 16 additions in its lane, one of the wave's halves, 4 of waves and 7 of parts, each off by 2^-24 (sums below 2): 28 2^-24."""
    from native_sparse_attention_pytorch_amd import ops
    d, v = 96, 300
    _, w, labels, weights = _inputs(n, d, v, dtype, seed=7, ignored=0.)
    x = (w.float()[labels] * torch.linspace(8, 40, n, device=DEV)[:, None]).to(dtype)
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
    dx, = torch.autograd.grad(loss, x, weights)
    x6, w6, at = x.detach().double(), w.detach().double(), labels[:, None]
    logits, size = x6 @ w6.t().contiguous(), x6.abs() @ w6.abs().t().contiguous()
    h, u = (2 ** -22, 2 ** -24) if dtype == F32 else (0., torch.finfo(dtype).eps / 2)
    dl = 2 * (((d / 4 + 8) * 2 ** -24 + 2 * h) * size).amax(-1, keepdim=True) + 2 ** -16
    assert (logits.argmax(-1) == labels).all()
    others = torch.exp(logits - logits.gather(1, at)).scatter(1, at, 0.)
    want = torch.log1p(others.sum(-1, keepdim=True))
    assert want.min() < 1e-10
    _within(loss.detach(), (want[:, 0], (dl * want)[:, 0] + 28 * 2 ** -24), "loss")
    G = weights.double()[:, None] * (others / (1 + others.sum(-1, keepdim=True))).scatter(1, at, torch.expm1(-want))
    dG = G.abs() * (2 * dl + (2 ** -11 if dtype != F32 else h)) + 2 ** -38 * float(weights.max())
    dG.scatter_add_(1, at, weights.double()[:, None] * 28 * 2 ** -24)
    tol = dG @ w6.abs() + G.abs() @ ((h + v / 4 * 2 ** -24) * w6.abs() + 2 ** -38 * float(w6.abs().max()))
    _within(dx, (G @ w6, 1.01 * tol + u * (G @ w6).abs() + torch.finfo(dtype).tiny * 2 * u), "dx")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_do_not_count_are_not_read(dtype):
    """Whole runs of ignored rows, NaN and infinities in them; their gradients are zeros."""
    x, w, labels, weights = _inputs(200, 96, 300, dtype, ignored=0.)
    labels[:70] = -100
    labels[130:133] = -100
    labels[199] = -100
    clean = _check(x, w, labels, "mean", weights)
    dirty = x.clone()
    dirty[:70], dirty[131], dirty[199] = math.nan, math.inf, -math.inf
    from native_sparse_attention_pytorch_amd import ops
    dirty.requires_grad_()
    w2 = w.clone().requires_grad_()
    loss = ops.linear_cross_entropy(dirty, w2, labels)
    dx, dw = torch.autograd.grad(loss, (dirty, w2), weights[0])
    for got, want in zip((loss, dx, dw), clean):
        assert torch.equal(got, want)
    assert not dx[labels == -100].any()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n", [5, 100])
def test_no_row_counts(n, reduction):
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(n, 64, 300, BF16)
    labels.fill_(-100)
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, labels, reduction=reduction)
    assert loss.isnan() if reduction == "mean" else not loss.any()
    dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
    assert not dx.any() and not dw.any()


def test_no_rows_at_all():
    from native_sparse_attention_pytorch_amd import ops
    w = torch.randn(70, 64, device=DEV, dtype=BF16, requires_grad=True)
    x, labels = torch.empty(2, 0, 64, device=DEV, dtype=BF16, requires_grad=True), torch.empty(2, 0, device=DEV, dtype=torch.int64)
    assert ops.linear_cross_entropy(x, w, labels).isnan() and ops.linear_cross_entropy(x, w, labels, reduction="sum") == 0
    loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
    assert loss.shape == (2, 0)
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    assert dx.shape == x.shape and not dw.any()


def test_labels_outside_the_vocabulary_say_so():
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, _ = _inputs(40, 64, 100, BF16, ignored=0.)
    labels[3], labels[17], labels[20] = 100, -1, 1 << 40
    loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
    assert loss.isnan().nonzero()[:, 0].tolist() == [3, 17, 20]
    x.requires_grad_()
    dx, = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), x)
    assert dx[3].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_that_are_not_finite_stay_in_their_row(dtype):
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(140, 64, 300, dtype, ignored=0.)
    want = ops.linear_cross_entropy(x, w, labels, reduction="none")
    x[5, 3], x[90, 0] = math.nan, math.inf
    loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
    keep = torch.ones(140, dtype=torch.bool, device=DEV)
    keep[5] = keep[90] = False
    assert torch.equal(loss[keep], want[keep]) and not loss[~keep].isfinite().any()


def test_logits_of_any_size():
    """Logits of +-3e4: no overflow, the loss is the distance from the largest."""
    x, w, labels, weights = _inputs(70, 128, 500, BF16, scale=1e4)
    _check(x, w, labels, "none", weights)
    # weights of the losses that are small, of either sign, or zero
    x, w, labels, weights = _inputs(70, 128, 500, BF16)
    _check(x, w, labels, "none", weights * 1e-20 * torch.where(torch.arange(70, device=DEV) % 2 == 0, 1, -1))
    _check(x, w, labels, "none", weights * 0)
    # weights as small as 1e-30, rows that are zero, a row 2^20 times another
    x, w, labels, weights = _inputs(70, 128, 500, F32)
    w[::3] = 0
    w *= 1e-30
    _check(x * 1e28, w, labels, "none", weights)
    w = _inputs(70, 128, 500, BF16)[1]
    w[7] *= 2 ** 10
    w[8] *= 2 ** -10
    _check(x.to(BF16), w, labels, "none", weights)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_layouts(dtype):
    """Row strides, odd addresses, overlapping rows, transposed weights, int32 and strided labels, more axes."""
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(90, 64, 200, dtype)
    want = _check(x, w, labels, "none", weights)

    def same(x2, w2, labels2, shape=(90,)):
        x2, w2 = x2.detach().requires_grad_(), w2.detach().requires_grad_()
        loss = ops.linear_cross_entropy(x2, w2, labels2, reduction="none")
        assert loss.shape == shape
        dx, dw = torch.autograd.grad(loss, (x2, w2), weights.view(shape))
        for got, exact in zip((loss.reshape(90), dx.reshape(90, 64), dw), want):
            assert torch.equal(got, exact)
    wide = torch.randn(90, 77, device=DEV).to(dtype)
    wide[:, 5:69] = x
    same(wide[:, 5:69], w, labels)
    tall = torch.randn(201, 67, device=DEV).to(dtype)
    tall[1:, 3:] = w
    same(x, tall[1:, 3:], labels.int())
    same(x, w.t().contiguous().t(), torch.stack((labels, labels), 1)[:, 1])
    same(x.view(3, 30, 64), w, labels.view(3, 30), (3, 30))
    same(x.view(30, 3, 64).transpose(0, 1).contiguous().transpose(0, 1), w, labels.view(30, 3), (30, 3))
    one = x[:1].expand(90, 64)
    got = ops.linear_cross_entropy(one, w, labels, reduction="none")
    assert torch.equal(got, ops.linear_cross_entropy(one.contiguous(), w, labels, reduction="none"))


def test_other_ignore_index_and_single_gradients():
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(70, 64, 150, BF16, ignored=0.)
    labels[::4] = 7
    _, dx, dw = _check(x, w, labels, "sum", weights, ignore=7)
    for wanted in (0, 1):
        pair = [x.clone(), w.clone()]
        pair[wanted].requires_grad_()
        got, = torch.autograd.grad(ops.linear_cross_entropy(*pair, labels, ignore_index=7, reduction="sum"), pair[wanted], weights[0])
        assert torch.equal(got, (dx, dw)[wanted])
    assert not ops.linear_cross_entropy(x, w, labels).requires_grad


def test_the_same_bits_again_and_twice_backward():
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(500, 192, 3001, BF16)
    first = _check(x, w, labels, "none", weights)
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
    for _ in range(2):
        dx, dw = torch.autograd.grad(loss, (x, w), weights, retain_graph=True)
        assert torch.equal(loss, first[0]) and torch.equal(dx, first[1]) and torch.equal(dw, first[2])
    # another weighting of the same forward, then the first again
    torch.autograd.grad(loss, (x, w), weights * 3, retain_graph=True)
    assert torch.equal(torch.autograd.grad(loss, x, weights)[0], first[1])


def test_gradient_against_differences():
    """Along a direction of logits that changes them by t per row at most, the third derivative of a loss is at most t^3, so differences of
    +-h are off by h^2 t^3 / 6, and by the losses' own error over h."""
    from native_sparse_attention_pytorch_amd import ops
    n, d, v, h = 40, 48, 130, 2 ** -5
    x, w, labels, weights = _inputs(n, d, v, F32, seed=9)
    g = torch.Generator().manual_seed(10)
    ux, uw = torch.randn(n, d, generator=g).to(DEV) * 0.2, torch.randn(v, d, generator=g).to(DEV) * 0.02
    live = labels != -100
    for du, dv in ((ux, torch.zeros_like(uw)), (torch.zeros_like(ux), uw)):
        t = 2 * (du.double() @ w.double().t() + x.double() @ dv.double().t()).abs().amax(-1)
        a, b = ((ops.linear_cross_entropy(x + s * h * du, w + s * h * dv, labels, reduction="none").double() * weights).sum() for s in (1, -1))
        (_, off), (dx, _), (dw, _) = _exact(x, w, labels, "none", weights)
        x2, w2 = x.clone().requires_grad_(), w.clone().requires_grad_()
        gx, gw = torch.autograd.grad(ops.linear_cross_entropy(x2, w2, labels, reduction="none"), (x2, w2), weights)
        slope = (gx.double() * du).sum() + (gw.double() * dv).sum()
        tol = (weights * live * (h * h * t ** 3 / 6)).sum() + 2 * (weights * off).sum() / h + 2 ** -18 * ((dx * du).abs().sum() + (dw * dv).abs().sum())
        assert abs((a - b) / (2 * h) - slope) <= tol, (float((a - b) / (2 * h)), float(slope), float(tol))


def test_second_derivatives_are_refused():
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, _ = _inputs(20, 64, 100, BF16)
    x.requires_grad_()
    dx, = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        dx.float().sum().backward()


def test_under_autocast_and_on_another_stream():
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, _ = _inputs(100, 128, 300, F32)
    want = ops.linear_cross_entropy(x.bfloat16(), w.bfloat16(), labels)
    w.requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        loss = ops.linear_cross_entropy(x, w, labels)
    dw, = torch.autograd.grad(loss, w)
    assert torch.equal(loss, want) and dw.dtype == F32
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.linear_cross_entropy(x.bfloat16(), w.bfloat16(), labels)
    side.synchronize()
    assert torch.equal(other, want)


def test_captured_forward_and_backward_replay():
    """One graph of forward and backward, new inputs each replay (their number of counting rows too), eager calls between the replays."""
    from native_sparse_attention_pytorch_amd import ops

    def both(x, w, labels, weights):
        loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), weights))
    sets = [_inputs(300, 128, 700, BF16, seed=s, ignored=0.1 * s) for s in range(4)]
    held = [t.clone() for t in sets[0]]
    held[0].requires_grad_(), held[1].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(*held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*held)
    for inputs in sets + sets[:1]:
        with torch.no_grad():
            for a, b in zip(held, inputs):
                a.copy_(b)
        graph.replay()
        fresh = [t.clone() for t in inputs]
        fresh[0].requires_grad_(), fresh[1].requires_grad_()
        want = both(*fresh)
        torch.cuda.synchronize()
        for got, w in zip(out, want):
            assert torch.equal(got, w)


def test_traced():
    """The traced call and its gradients are the launched ones."""
    from native_sparse_attention_pytorch_amd import ops
    run = torch.compile(lambda x, w, labels: ops.linear_cross_entropy(x, w, labels, reduction="none"), backend="aot_eager", fullgraph=True)
    for n in (20, 100):
        x, w, labels, weights = _inputs(n, 64, 300, BF16)
        want = _check(x, w, labels, "none", weights)
        x.requires_grad_(), w.requires_grad_()
        loss = run(x, w, labels)
        for got, exact in zip((loss, *torch.autograd.grad(loss, (x, w), weights)), want):
            assert torch.equal(got, exact)


def test_few_rows_replay():
    """A captured forward of up to 32 rows takes other labels, and other numbers of rows that count, at each replay."""
    from native_sparse_attention_pytorch_amd import ops
    sets = [_inputs(24, 200, 900, F16, seed=s, ignored=i) for s, i in enumerate((0., 0.5, 1.1, 0.2))]
    held = [t.clone() for t in sets[0][:3]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear_cross_entropy(*held, reduction="none")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        each, mean = ops.linear_cross_entropy(*held, reduction="none"), ops.linear_cross_entropy(*held)
    for inputs in sets + sets[:1]:
        for a, b in zip(held, inputs):
            a.copy_(b)
        graph.replay()
        want = ops.linear_cross_entropy(*inputs[:3], reduction="none"), ops.linear_cross_entropy(*inputs[:3])
        torch.cuda.synchronize()
        assert torch.equal(each, want[0]) and torch.equal(mean.nan_to_num(nan=-1.), want[1].nan_to_num(nan=-1.))


@pytest.mark.parametrize("n", [20, 40])
def test_weights_past_4_gigabytes(n):
    """Offsets of weights and gradients past 32 bits: the last entries' logits and gradients (in float64, piece by piece of the vocabulary)."""
    from native_sparse_attention_pytorch_amd import ops
    d, v = 4096, 600011
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(n, d, device=DEV, dtype=BF16, generator=g)
    w = torch.randn(v, d, device=DEV, dtype=BF16, generator=g) * d ** -0.5
    labels = torch.randint(v - 1000, v, (n,), device=DEV, generator=g)
    weights = torch.rand(n, device=DEV, generator=g) + 0.1
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
    dx, dw = torch.autograd.grad(loss, (x, w), weights)
    x6, size = x.detach().double(), x.detach().double().abs()
    pieces = [w.detach()[i:i + 60000].double() for i in range(0, v, 60000)]
    lse = torch.logsumexp(torch.cat([x6 @ p.t().contiguous() for p in pieces], 1), 1)
    # logits as in _exact, where |x| |w| is at most 4096 times a product's mean of 0.64 d^-1/2, twice that with room
    dl = (d / 4 + 8) * 2 ** -24 * 2 * 0.64 * d ** 0.5
    own = (x6 * w.detach()[labels].double()).sum(1)
    _within(loss.detach(), (lse - own, torch.full_like(own, 2 * dl + 2 ** -16 + 2 ** -20)), "loss")
    want, tol = torch.zeros_like(x6), torch.zeros_like(x6)
    for i, p in enumerate(pieces):
        G = torch.exp(x6 @ p.t().contiguous() - lse[:, None])
        off = G * (2 * dl + 2 ** -15 + 2 ** -11) + 2 ** -38
        at = (labels - 60000 * i)
        here = (at >= 0) & (at < len(p))
        rows = here.nonzero()[:, 0]
        off[rows, at[here]] += 2 ** -11 + 2 * dl + 2 ** -15
        G[rows, at[here]] -= 1
        G, off = G * weights.double()[:, None], off * weights.double()[:, None]
        want += G @ p
        tol += off @ p.abs() + 2 ** -14 * (G.abs() @ p.abs())
        if i in (0, len(pieces) - 1):
            exact = G.t().contiguous() @ x6
            _within(dw[60000 * i:60000 * i + len(p)], (exact, off.t().contiguous() @ size + 2 ** -20 * (G.t().contiguous().abs() @ size) + 2 ** -8 * exact.abs()), "dw")
    _within(dx, (want, tol + 2 ** -8 * want.abs()), "dx")


@pytest.mark.parametrize("n,d,v", [(20, 130, 400), (90, 200, 1000), (257, 64, 2000)])
def test_fp16_gradients_are_off_by_their_rounding(n, d, v):
    """G's two halves hold 22 bits, so what is left beside the rounding of the result are fp32 sums: a tenth of it with room."""
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, weights = _inputs(n, d, v, F16, seed=11)
    x.requires_grad_(), w.requires_grad_()
    got = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels, reduction="none"), (x, w), weights)
    _, (dx, _), (dw, _) = _exact(x.detach(), w.detach(), labels, "none", weights)
    for g, e in zip(got, (dx, dw)):
        assert float((g.double() - e).norm()) <= 1.1 * float((e.to(F16).double() - e).norm())


@pytest.mark.parametrize("n,dtype", [(20, BF16), (100, BF16), (100, F16), (20, F32), (100, F32)])
def test_the_operators_are_what_they_are_registered_as(n, dtype):
    """Arguments are left as they are, traced results are shaped like the real ones."""
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels, _ = _inputs(n, 64, 300, dtype)
    loss, state = ops.linear_cross_entropy_fwd(x, w, labels, -100, 1)
    for op, args in ((torch.ops.nsa_amd.linear_cross_entropy_fwd, (x.clone().requires_grad_(), w.clone().requires_grad_(), labels, -100, 1)),
                     (torch.ops.nsa_amd.linear_cross_entropy_bwd, (torch.ones((), device=DEV), x, w, state, -100, 1, True, True))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("n", [1, 33])
@pytest.mark.parametrize("gap", [5., 20., 45.])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_losses_far_below_a_rounding_of_one(n, gap, dtype):
    """log(1 + r) with r down to 2^-53 (below, nothing) and its gradients, to the relative error of the others' exponentials: two logits' dL, 2^-16 for the sums, and for
    the exponents' own rounding 2^-22 of the distance in front of it."""
    from native_sparse_attention_pytorch_amd import ops
    d, v = 96, 300
    _, w, labels, weights = _inputs(n, d, v, dtype, seed=8, ignored=0.)
    x = (w.float()[labels] * gap / w.float()[labels].square().sum(-1, keepdim=True)).to(dtype)
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, labels, reduction="none")
    dx, dw = torch.autograd.grad(loss, (x, w), weights)
    x6, w6, at = x.detach().double(), w.detach().double(), labels[:, None]
    logits, size = x6 @ w6.t().contiguous(), x6.abs() @ w6.abs().t().contiguous()
    h, u = (2 ** -22, 2 ** -24) if dtype == F32 else (0., torch.finfo(dtype).eps / 2)
    far = logits - logits.gather(1, at)
    rel = 2 * (((d / 4 + 8) * 2 ** -24 + 2 * h) * size).amax(-1, keepdim=True) + 2 ** -16 + 2 ** -22 * far.abs().amax(-1, keepdim=True)
    others = torch.exp(far).scatter(1, at, 0.)
    r = others.sum(-1, keepdim=True)
    assert gap < 45 or r.max() < 1e-9
    seen = torch.where(r < 2 ** -53, 0., r)
    _within(loss.detach(), (torch.log1p(seen)[:, 0], (rel * torch.log1p(r))[:, 0]), "loss")
    G = weights.double()[:, None] * (others / (1 + r)).scatter(1, at, -seen / (1 + r))
    dG = G.abs() * (2 * rel + (2 ** -11 if dtype != F32 else h)) + 2 ** -38 * float(G.abs().max())
    for got, left, off, right, k in ((dx, G, dG, w6, v), (dw, G.t().contiguous(), dG.t().contiguous(), x6, n)):
        want = left @ right
        tol = off @ right.abs() + left.abs() @ ((h + (k / 4 + 16) * 2 ** -24) * right.abs() + 2 ** -38 * float(right.abs().max()))
        # (fp16 results below 2^-24 are multiples of it)
        _within(got, (want, 1.01 * tol + u * want.abs() + (2. ** -25 if dtype == F16 else torch.finfo(dtype).tiny)), gap)
