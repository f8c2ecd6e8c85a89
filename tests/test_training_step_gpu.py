"""Loss, gradients and update together, as a training step uses them: `Transformer(fused_loss=True)`, `training.Fp32Masters`, `training.Muon`,
launched and replayed from a graph."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _model(fused, vocab=300, **kw):
    from native_sparse_attention_pytorch_amd.transformer import Transformer
    torch.manual_seed(5)
    return Transformer(num_tokens=vocab, dim=256, depth=2, dim_head=64, heads=4, kv_heads=2, fused_loss=fused,
                       sparse_attn_kwargs=dict(sliding_window_size=32, compress_block_size=16, compress_block_sliding_stride=8,
                                               selection_block_size=16, num_selected_blocks=4), **kw).to(DEV)


def _ids(seed, vocab=300):
    return torch.randint(0, vocab, (3, 258), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_model_takes_the_fused_loss(dtype):
    """The same state dict; the loss is that of the model's logits before they are rounded: with logits of at most L a bf16 rounding (2^-9 of
    them) moves a loss by 2^-8 L, fp32 ones by the sums' 2^-18 L."""
    plain, fused = _model(False).to(dtype), _model(True).to(dtype)
    fused.load_state_dict(plain.state_dict())
    ids = _ids(1)
    losses = [m(ids, return_loss=True) for m in (plain, fused)]
    logits = plain(ids[:, :-1])
    assert torch.equal(logits, fused(ids[:, :-1]))
    tol = (2 ** -8 if dtype == torch.bfloat16 else 2 ** -18) * float(logits.detach().abs().max())
    assert abs(losses[0] - losses[1]) <= tol
    names = [n for n, p in plain.named_parameters() if p.requires_grad]
    grads = [torch.autograd.grad(l, [p for p in m.parameters() if p.requires_grad], allow_unused=True) for l, m in zip(losses, (plain, fused))]
    for name, a, b in zip(names, *grads):
        assert (a is None) == (b is None), name
    # of the projection: (p - target) x, p off by tol of itself, bf16 logits' gradients rounded as well (2^-8)
    at = names.index("to_logits.weight")
    a, b = grads[0][at].double(), grads[1][at].double()
    assert float((a - b).norm() / b.norm()) <= 2 * tol + 2 ** -7


def test_ids_that_are_ignored():
    """Labels of -100 are left out, as the mean of F.cross_entropy leaves them out."""
    from native_sparse_attention_pytorch_amd import ops
    model = _model(True).bfloat16()
    ids = _ids(2)
    with torch.no_grad():
        hidden = torch.randn(3, 257, 256, device=DEV).bfloat16()
        labels = ids[:, 1:].clone()
        labels[:, :100] = -100
        got = ops.linear_cross_entropy(hidden, model.to_logits.weight, labels)
        want = F.cross_entropy((hidden.double() @ model.to_logits.weight.double().t()).flatten(0, 1), labels.flatten())
    assert abs(got - want) < 1e-4


def test_a_hooked_or_other_projection_keeps_the_logits():
    model = _model(True).bfloat16()
    ids, seen = _ids(3), []
    with torch.no_grad():
        model(ids, return_loss=True)
        handle = model.to_logits.register_forward_hook(lambda m, i, o: seen.append(o.shape))
        hooked = model(ids, return_loss=True)
        handle.remove()
        assert seen == [(3, 257, 300)]
        model.to_logits = torch.nn.Linear(256, 300).to(DEV).bfloat16()
        assert model(ids, return_loss=True).isfinite() and hooked.isfinite()


def _matrices(masters, model):
    named = [n for n, _ in model.named_parameters()]
    own = [m for m, n in zip(masters.masters, named) if m.dim() == 2 and "token_emb" not in n and "to_logits" not in n]
    mine = set(map(id, own))
    return own, [m for m in masters.masters if id(m) not in mine and m.is_floating_point()]


def test_training_steps_launched_and_replayed():
    """A step launched and the same step replayed from a graph agree in loss and gradients for every batch; the masters move by Muon's and Adam's
    updates, the model's parameters are their roundings, and orthogonalised updates have the size that their formula gives."""
    from native_sparse_attention_pytorch_amd.training import Fp32Masters, GraphedStep, Muon
    model = _model(True)
    masters = Fp32Masters(model)
    own, rest = _matrices(masters, model)
    assert len(own) >= 8
    muon, adam = Muon(own, lr=0.01), torch.optim.Adam(rest, lr=1e-3)

    class Both:
        def step(self):
            muon.step()
            adam.step()
    step = GraphedStep(model, _ids(0))
    for seed in range(4):
        ids = _ids(seed)
        for p in model.parameters():
            p.grad = None
        want = model(ids, return_loss=True)
        want.backward()
        grads = [None if p.grad is None else p.grad.clone() for p in model.parameters()]
        torch.cuda.synchronize()
        loss = step(ids)
        torch.cuda.synchronize()
        assert abs(loss - want) < 1e-5
        for (n, p), g in zip(model.named_parameters(), grads):
            if g is not None and not n.endswith("bias"):       # (those are sums in another order while recording)
                assert torch.equal(p.grad, g), n
        before = [m.detach().clone() for m in own]
        masters.step(Both())
        for m, b in zip(own, before):
            moved = (m.detach() - b).double()
            rows, cols = m.shape
            # singular values of an orthogonalised update are at most 1.21, and not all of them small
            size = float(torch.linalg.matrix_norm(moved, 2)) / (0.01 * max(1, rows / cols) ** 0.5)
            assert size < 1.25, (rows, cols, size)
        for m, p in zip(masters.masters, model.parameters()):
            assert torch.equal(p.detach(), m.detach().bfloat16())


def test_refusals():
    from native_sparse_attention_pytorch_amd import ops
    x, w, labels = torch.randn(4, 64, device=DEV).bfloat16(), torch.randn(10, 64, device=DEV).bfloat16(), torch.zeros(4, device=DEV, dtype=torch.int64)
    for bad in ((x.float(), w, labels), (x.double(), w.double(), labels), (x, w[:, :60], labels), (x, w, labels[:3]), (x, w[0], labels),
                (x, w[:0], labels), (x, w, labels.float()), (x, w.cpu(), labels), (x, w, labels.cpu())):
        with pytest.raises(RuntimeError, match="linear_cross_entropy"):
            ops.linear_cross_entropy(*bad)
