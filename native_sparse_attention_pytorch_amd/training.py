"""Mixed-precision training of a bf16 model against fp32 master weights.

Under `torch.autocast` every projection of every layer casts its fp32 weight, bias and input to bf16 on the way in and
its gradients back on the way out: at the size of the reference's training script (train.py:22-50: dim 512, depth 6,
1024 tokens) that is ~270 of a step's ~940 kernel launches, and the step is bound by its launches, not by the GPU.
Here the model itself is bf16 (no casts inside the step) and the optimizer works on fp32 copies of its parameters:
one multi-tensor copy takes the bf16 gradients to the masters, one takes the updated masters back.  The arithmetic is
the same as under autocast - bf16 operands rounded from fp32 masters, fp32 accumulation, fp32 update - and the loss
curve agrees with the fp32 oracle as closely.

`GraphedStep` goes one further for fixed shapes: the forward and backward of the bf16 model are recorded once into a HIP
graph and replayed per step (one launch instead of ~700); the optimizer stays outside the graph.

`Muon` is an optimizer for the matrices among the parameters (the masters, or a model's own): momentum whose update is orthogonalised, all
matrices of a step together (ops.newton_schulz).
"""
from __future__ import annotations

import torch
from torch import nn


class Fp32Masters:
    """`model` (its parameters still fp32, freshly initialised or loaded) is cast to bf16 in place; `self.masters` are the
    fp32 originals, to be handed to any torch optimizer.  Per step: `loss.backward()`, then `step(optimizer)`."""

    def __init__(self, model: nn.Module):
        self.masters = [p.detach().clone().float() for p in model.parameters()]
        model.bfloat16()
        self.params = list(model.parameters())
        for m in self.masters:
            m.requires_grad_(True)

    @torch.no_grad()
    def step(self, optimizer: torch.optim.Optimizer) -> None:
        live = [(m, p) for m, p in zip(self.masters, self.params) if p.grad is not None]
        for m, p in zip(self.masters, self.params):
            if p.grad is None:
                m.grad = None               # no gradient this step: the optimizer skips it
            elif m.grad is None:
                m.grad = torch.empty_like(m)
        torch._foreach_copy_([m.grad for m, _ in live], [p.grad for _, p in live])
        optimizer.step()
        torch._foreach_copy_(self.params, self.masters)
        for p in self.params:
            p.grad = None


class GraphedStep:
    """Forward + backward of `model(ids, return_loss=True)` (or of `loss_fn(model, ids)`) as one replayed HIP graph, for a
    bf16 model (e.g. under `Fp32Masters`) and inputs of one fixed shape.

        step = GraphedStep(model, example_ids)
        loss = step(ids)            # gradients are in p.grad of the model's parameters afterwards
        masters.step(optimizer)     # or optimizer.step() on the model's own parameters

    The graph holds no memset node of a library reduction (their replays gave wrong bias gradients on this platform):
    while it is recorded every bias gradient is a column sum by this library's kernel (ops.colsum_supported) and the
    feed-forward projections go through ops.linear (Transformer._feed_forward).  The gradient tensors are the graph's own:
    every call re-attaches them to the parameters (an optimizer helper may have set `p.grad = None`) and every replay
    overwrites them, so gradients do not accumulate across calls.  `loss` is a tensor that the next call overwrites.
    Create it before the model's first normally launched training step (a `Transformer` that has been stepped is refused:
    recording one ended the process here); replays and launched steps may be mixed freely afterwards."""

    def __init__(self, model: nn.Module, example_ids: torch.Tensor, warmup: int = 3, loss_fn=None):
        # loss_fn(model, ids) -> scalar loss; default: the Transformer's own `model(ids, return_loss=True)`
        self.loss_fn = loss_fn if loss_fn is not None else (lambda m, ids: m(ids, return_loss=True))
        if not example_ids.is_cuda:
            raise RuntimeError("GraphedStep needs device tensors")
        if torch.is_autocast_enabled() or any(p.requires_grad and p.is_floating_point() and p.dtype != torch.bfloat16 for p in model.parameters()):
            # under autocast / with fp32 parameters the projections run through the library's own autograd, whose bias
            # gradients are the sums that replay wrongly
            raise RuntimeError("GraphedStep records a bf16 model outside autocast (cast it with Fp32Masters or .bfloat16())")
        if getattr(model, "_launched_grad_steps", False):
            # recording after normally launched training steps of the same model ended the process (segmentation fault inside
            # the recording) on this platform, with backward() and with autograd.grad() alike; a model that has not been
            # stepped yet records and replays correctly, also next to other models trained in the same process
            raise RuntimeError("GraphedStep must be created before the model's first normally launched training step "
                               "(build the model, then GraphedStep, then train through it)")
        self.model = model
        self.params = [p for p in model.parameters()]
        self.ids = example_ids.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        # torch.autograd.grad, not backward(): the gradients come back as the recording's own tensors instead of passing
        # through the parameters' gradient accumulator nodes (which belong to the stream that created them)
        wanted = [p for p in self.params if p.requires_grad]
        model._recording_warmup = True
        try:
            with torch.cuda.stream(side):                # allocator and library warm-up outside the recording
                for _ in range(max(1, warmup)):
                    torch.autograd.grad(self.loss_fn(model, self.ids), wanted, allow_unused=True)
        finally:
            model._recording_warmup = False
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            loss = self.loss_fn(model, self.ids)
            grads = torch.autograd.grad(loss, wanted, allow_unused=True)
            self.loss = loss.detach()
        by_param = dict(zip(map(id, wanted), grads))
        self.grads = [by_param.get(id(p)) for p in self.params]

    def __call__(self, ids: torch.Tensor) -> torch.Tensor:
        if ids.shape != self.ids.shape or ids.dtype != self.ids.dtype:
            raise RuntimeError(f"GraphedStep was recorded for ids of shape {tuple(self.ids.shape)}, got {tuple(ids.shape)}")
        for p, g in zip(self.params, self.grads):
            p.grad = g
        self.ids.copy_(ids)
        self.graph.replay()
        return self.loss


class Muon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates, for matrices (parameters of more axes are taken as first axis by the rest):

        buffer <- momentum buffer + gradient;  update = gradient + momentum buffer (nesterov) or the buffer
        p <- (1 - lr weight_decay) p - lr sqrt(max(1, rows / columns)) newton_schulz(update)

    Embeddings, norm weights and biases belong to another optimizer; vectors are refused.  The momentum buffer and the update are fp32, of 16-bit
    parameters too: gradients below 2^-8 of the buffer would be lost in bf16.

        masters = Fp32Masters(model)
        matrices = [m for m, (name, p) in zip(masters.masters, model.named_parameters())
                    if p.dim() == 2 and "token_emb" not in name and "to_logits" not in name]
        muon = Muon(matrices, lr=0.02)

    A step that cannot be taken (a parameter that is not on a GPU, a sparse gradient, a group's number out of range) is refused before anything of it
    is done.  Parameters may lie on several devices.
    """

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0., steps: int = 5,
                 coefficients=(3.4445, -4.7750, 2.0315), eps: float = 1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            self._check_numbers(self.param_groups[-1])
            for p in self.param_groups[-1]["params"]:
                if p.dim() < 2:
                    raise ValueError(f"Muon takes matrices, got a parameter of shape {tuple(p.shape)}")
                if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                    raise ValueError(f"Muon takes fp32, bf16 or fp16 parameters, got {p.dtype}")
        except ValueError:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_numbers(group) -> None:
        from . import ops
        if not (group["lr"] >= 0 and group["weight_decay"] >= 0 and 0 <= group["momentum"] < 1):
            raise ValueError(f"Muon: lr {group['lr']}, momentum {group['momentum']}, weight_decay {group['weight_decay']}")
        ops.newton_schulz([], steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"])

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # (the base class rounds a state to its parameter's type)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(ids, (p for group in self.param_groups for p in group["params"])):
            kept = state_dict["state"].get(i, {}).get("momentum_buffer")
            if kept is not None:
                self.state[p]["momentum_buffer"] = kept.to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        from . import ops
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        todo = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None and p.numel()]
            if params:
                self._check_numbers(group)
            for p in params:
                if not p.is_cuda:
                    raise RuntimeError(f"Muon: a parameter on {p.device}: needs a GPU (HIP kernels, no CPU fallback)")
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
            for device in dict.fromkeys(p.device for p in params):
                todo.append((group, float(group["lr"]), [p for p in params if p.device == device]))
        for group, lr, params in todo:
            grads = [p.grad for p in params]
            for p in params:
                if "momentum_buffer" not in self.state[p]:
                    self.state[p]["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
            buffers = [self.state[p]["momentum_buffer"] for p in params]
            torch._foreach_mul_(buffers, group["momentum"])
            torch._foreach_add_(buffers, grads)
            updates = torch._foreach_add(grads, buffers, alpha=group["momentum"]) if group["nesterov"] else buffers
            updates = ops.newton_schulz([u.flatten(1) for u in updates], steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"])
            if group["weight_decay"]:
                torch._foreach_mul_(params, 1 - lr * group["weight_decay"])
            torch._foreach_mul_(updates, [-lr * max(1., u.shape[0] / u.shape[1]) ** 0.5 for u in updates])
            torch._foreach_add_(params, [u.view(p.shape) for u, p in zip(updates, params)])
        return loss
