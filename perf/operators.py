"""The two ends of a training step as they are measured: the loss of a projection onto a vocabulary, with its gradients
(`ops.linear_cross_entropy`), and the orthogonalised updates of an optimizer (`ops.newton_schulz`).

`listed()` are the cases by name, `draw(rng)` gives others of the same ranges; `prepare` makes what a program holds before the call, `run` is
one pass - in the operators' plain form, or, where `own` is true, as a program calls this package -, `work` what a pass cannot do without,
`exact` the definition in 64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


def loss(name, dtype, rows, dim, vocab, train, reduction="mean", ignored=0.0):
    return dict(name=name, kind="loss", dtype=dtype, rows=rows, dim=dim, vocab=vocab, train=train, reduction=reduction, ignored=ignored)


def update(name, dtype, matrices):
    """`matrices`: sizes as 'rows x columns x how many', several of them separated by commas."""
    return dict(name=name, kind="update", dtype=dtype, matrices=matrices)


def listed():
    return [
        # the smallest call: log-probabilities of the next token of 8 sequences under the byte-level model
        loss("score_bytes_8", "bf16", 8, 512, 256, False, "none"),
        # rescoring a few candidates under a large model: one pass over a weight of a gigabyte
        loss("score_131k_24", "bf16", 24, 4096, 131072, False, "none"),
        # evaluation of a prompt left in the default type, nothing of a round size
        loss("score_fp32_odd", "fp32", 1021, 1000, 32003, False, "mean"),
        # a training step of the byte-level model: 8 sequences of 1024 tokens, the last of each without a label of its own
        loss("train_bytes_8k", "bf16", 8184, 512, 256, True),
        # fine-tuning a medium model: prompts are masked, 40 % of the rows have no label
        loss("train_50k_masked", "bf16", 8192, 1024, 50021, True, "mean", 0.4),
        # pretraining a large model: 8192 tokens, a vocabulary of 128000
        loss("train_128k", "bf16", 8192, 4096, 128000, True),
        # a small model in half precision, losses weighted row by row
        loss("train_fp16_weighted", "fp16", 2047, 768, 32000, True, "none", 0.1),
        # a model trained in the default type
        loss("train_fp32", "fp32", 4095, 1024, 32000, True),
        # the smallest update: one matrix of a gate projection, fp32 masters
        update("update_gate", "fp32", "24x512x1"),
        # all matrices of the byte-level model: 6 layers (qkv, output, feed-forward up and down; gates)
        update("update_bytes", "fp32", "1024x512x6,512x512x6,2048x512x6,512x2048x6,24x512x6"),
        # odd sizes, a tall and a wide one in bf16
        update("update_odd", "bf16", "1021x2741x2,2741x1021x1"),
        # a large layer's projections
        update("update_large", "bf16", "6144x4096x1,4096x16384x1"),
    ]


def draw(rng):
    def spread(lo, hi):                      # whole numbers, even over their logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def size(lo, hi):                        # a multiple of 64, of 8, or any
        n = spread(lo, hi)
        return max(lo, n // 64 * 64, 1) if rng.random() < 0.4 else max(lo, n // 8 * 8, 1) if rng.random() < 0.5 else n

    if rng.random() < 0.6:
        dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32"))
        train = rng.random() < 0.6
        while True:
            case = loss("", dtype, spread(1, 16384), size(64, 4096), size(256, 131072), train, rng.choice(("mean", "mean", "sum", "none")),
                        rng.choice((0.0, 0.0, 0.1, 0.5)))
            n, d, v = case["rows"], case["dim"], case["vocab"]
            if n * d * v <= 4 * 10 ** 12 // (4 if dtype == "fp32" else 1) and n * v <= 1 << 30:
                break
    else:
        dtype, left, parts = rng.choice(("bf16", "fp16", "fp32", "fp32")), 4 * 10 ** 11, []
        for _ in range(rng.choice((1, 1, 2, 3))):
            m, n, count = size(8, 4096), size(8, 8192), rng.choice((1, 1, 2, 6))
            a, b = min(m, n), max(m, n)
            if count * a * a * b > left:
                a = b = m = n = min(a, 1024)
                count = 1
            left -= count * a * a * b
            parts.append(f"{m}x{n}x{count}")
        case = update("", dtype, ",".join(parts))
    del case["name"]
    return case


def sizes(case):
    return [(int(m), int(n)) for m, n, count in (part.split("x") for part in case["matrices"].split(",")) for _ in range(int(count))]


def work(case):
    each = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "update":
        flops = sum(STEPS * (3 * min(s) ** 2 * max(s) + min(s) ** 3) for s in sizes(case))         # symmetric products: one half
        return dict(bytes=sum(2 * m * n * each for m, n in sizes(case)), flops=flops)
    n, d, v = case["rows"], case["dim"], case["vocab"]
    live = n * (1 - case["ignored"])
    losses = n * 4 if case["reduction"] == "none" else 4
    if not case["train"]:
        return dict(bytes=(live * d + v * d) * each + n * 8 + losses, flops=2 * live * v * d)
    return dict(bytes=(live * d + n * d + 2 * v * d) * each + n * 8 + 2 * losses, flops=6 * live * v * d)


def inputs_of_loss(case, seed):
    """Hidden states behind a norm (some features larger than others), a weight whose rows have a common part, labels that the logits favour,
    and what the losses are weighted with."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    n, d, v = case["rows"], case["dim"], case["vocab"]
    dtype = DTYPES[case["dtype"]]
    randn = lambda *size: torch.randn(*size, device=DEVICE, generator=g)
    labels = torch.randint(0, v, (n,), device=DEVICE, generator=g)
    w = torch.empty(v, d, dtype=dtype, device=DEVICE)
    common = 0.2 * randn(d)
    for at in range(0, v, 16384):            # (in pieces: the largest would take 2 GB at once in fp32)
        w[at:at + 16384] = ((randn(min(v, at + 16384) - at, d) + common) * d ** -0.5).to(dtype)
    x = randn(n, d) * (1 + randn(d).abs()) + 0.1 * d ** 0.5 * w[labels].float() * randn(n, 1).abs() * 8
    x = (x * x.square().mean(-1, keepdim=True).rsqrt() * 2).to(dtype)
    if case["ignored"]:
        first = torch.rand(n, device=DEVICE, generator=g) < case["ignored"]
        runs = torch.arange(n, device=DEVICE) // 61          # prompts: whole runs of rows
        labels = labels.masked_fill(first[(runs * 61).clamp(max=n - 1)], IGNORE)
    weights = torch.rand(n, device=DEVICE, generator=g) / n if case["reduction"] == "none" else torch.rand((), device=DEVICE, generator=g) + 0.5
    return x, w, labels, weights


def inputs_of_update(case, seed):
    """Momenta: a few strong directions over noise, as the gradients of a layer have them."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    randn = lambda *size: torch.randn(*size, device=DEVICE, generator=g)
    made = []
    for m, n in sizes(case):
        r = max(1, min(m, n) // 16)
        strong = (randn(m, r) * torch.logspace(0, -1, r, device=DEVICE)) @ randn(r, n)
        made.append(((0.2 * strong + randn(m, n)) * 1e-3).to(DTYPES[case["dtype"]]))
    return made


def prepare(case, seed):
    if case["kind"] == "update":
        return dict(case=case, updates=inputs_of_update(case, seed))
    x, w, labels, weights = inputs_of_loss(case, seed)
    if case["train"]:
        x.requires_grad_()
        w.requires_grad_()
    return dict(case=case, x=x, w=w, labels=labels, weights=weights)


def plain_loss(x, w, labels, reduction, weights):
    """Losses and, where `weights` is given, the gradients of their sum weighted with it."""
    x32, w32, live = x.float(), w.float(), labels != IGNORE
    logits = x32 @ w32.t()
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(-1, keepdim=True)
    at = labels.clamp(min=0)[:, None]
    each = torch.where(live, (torch.log(total) + top - logits.gather(1, at))[:, 0], 0.0)
    count = live.sum()
    value = each if reduction == "none" else each.sum() if reduction == "sum" else each.sum() / count
    if weights is None:
        return value
    g = weights if reduction == "none" else weights.expand(len(labels)) if reduction == "sum" else (weights / count).expand(len(labels))
    p /= total
    p.scatter_add_(1, at, torch.full_like(top, -1.0))
    p *= torch.where(live, g, 0.0)[:, None]
    return value, (p @ w32).to(x.dtype), (p.t() @ x32).to(w.dtype)


def plain_update(g):
    a, b, c = COEFFICIENTS
    x = g.float()
    x = x / (x.square().sum().sqrt() + EPS)
    x = x if x.shape[0] <= x.shape[1] else x.t()
    for _ in range(STEPS):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x if g.shape[0] <= g.shape[1] else x.t()).to(g.dtype).contiguous()


def run(state):
    case = state["case"]
    if own:
        from native_sparse_attention_pytorch_amd import ops
        if case["kind"] == "update":
            return ops.newton_schulz(state["updates"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        x, w, labels, weights = (state[k] for k in ("x", "w", "labels", "weights"))
        value = ops.linear_cross_entropy(x, w, labels, ignore_index=IGNORE, reduction=case["reduction"])
        if not case["train"]:
            return value
        return (value.detach(), *torch.autograd.grad(value, (x, w), weights))
    if case["kind"] == "update":
        return [plain_update(g) for g in state["updates"]]
    with torch.no_grad():
        return plain_loss(state["x"], state["w"], state["labels"], case["reduction"], state["weights"] if case["train"] else None)


def exact(case, seed):
    if case["kind"] == "update":
        if sum(STEPS * 2 * (2 * min(s) ** 2 * max(s) + min(s) ** 3) for s in sizes(case)) > 2e13:
            return None
        found = []
        for g in inputs_of_update(case, seed):
            q = g.double()
            q = q / (torch.linalg.vector_norm(q) + EPS)
            wide = q.shape[0] <= q.shape[1]
            for _ in range(STEPS):
                # a q + b (q q') q + c (q q')^2 q, from the shorter side
                s = q @ q.mT if wide else q.mT @ q
                poly = COEFFICIENTS[1] * s + COEFFICIENTS[2] * (s @ s)
                q = COEFFICIENTS[0] * q + (poly @ q if wide else q @ poly)
            found.append(q)
        return found
    n, d, v = case["rows"], case["dim"], case["vocab"]
    if n * d * v * (6 if case["train"] else 2) > 2e13:
        return None
    x, w, labels, weights = inputs_of_loss(case, seed)
    live = (labels != IGNORE).nonzero()[:, 0]
    count = len(live)
    w64 = w.double()
    each = torch.zeros(n, dtype=torch.float64, device=DEVICE)
    dx = torch.zeros(n, d, dtype=torch.float64, device=DEVICE)
    dw = torch.zeros(v, d, dtype=torch.float64, device=DEVICE)
    g = weights.double()
    g = (g if case["reduction"] == "none" else g.expand(n) / (count if case["reduction"] == "mean" else 1))
    rows = max(1, (1 << 27) // v)
    for at in live.split(rows):
        x64 = x[at].double()
        logp = torch.log_softmax(x64 @ w64.mT, dim=-1)
        each[at] = -logp[torch.arange(len(at), device=DEVICE), labels[at]]
        if case["train"]:
            dl = logp.exp_()
            dl[torch.arange(len(at), device=DEVICE), labels[at]] -= 1
            dl *= g[at, None]
            dx[at] = dl @ w64
            dw += dl.mT @ x64
    value = each if case["reduction"] == "none" else each.sum() / (count if case["reduction"] == "mean" else 1)
    return (value, dx, dw) if case["train"] else value
