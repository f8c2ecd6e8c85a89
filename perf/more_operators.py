"""A serving step's operators as they are measured: a key / value cache held in 8 bits with a scale for each block of tokens and head
(`ops.cache8_append`), the attention of one token per sequence over it - over all keys or the newest ones (`ops.cache8_attend`) and over
selected blocks (`ops.cache8_select_attend`) - and what is done to the logits before a token is drawn (`ops.adjust_logits`).

`listed()` are the cases by name, `draw(rng)` gives others of the same ranges; `prepare` makes what a program holds before the call, `run` is
one pass - in the operators' plain form, or, where `own` is true, as a program calls this package -, `work` what a pass cannot do without,
`exact` the definition in 64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = torch.float8_e4m3fn
TOP = 448.0                                  # the largest value of e4m3
LEAST, MOST = -110, 119                      # exponents of a block's scale


def append(name, dtype, batch, kv_heads, dim, block, held, rows):
    """`rows` more keys and values for each sequence; sequences hold up to `held` tokens; of a chunk of several rows some sequences take fewer."""
    return dict(name=name, kind="append", dtype=dtype, batch=batch, kv_heads=kv_heads, dim=dim, block=block, held=held, rows=rows)


def attend(name, dtype, batch, heads, kv_heads, dim, block, longest, shortest, window=0):
    return dict(name=name, kind="attend", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, block=block, longest=longest,
                shortest=shortest, window=window)


def select(name, dtype, batch, heads, kv_heads, dim, block, longest, shortest, chosen, size, per_head=False):
    """`chosen` blocks of `size` keys for each kv head, or for each head."""
    return dict(name=name, kind="select", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, block=block, longest=longest,
                shortest=shortest, chosen=chosen, size=size, per_head=per_head)


def logits(name, dtype, batch, vocab, history, mask, bias):
    """`history`: tokens so far in the longest sequence; `mask`: none, packed (32 tokens a word) or bool."""
    return dict(name=name, kind="logits", dtype=dtype, batch=batch, vocab=vocab, history=history, mask=mask, bias=bias)


def listed():
    return [
        # a serving step of 64 sequences: one token of each goes into its cache
        append("append_token_64", "bf16", 64, 8, 128, 32, 1000, 1),
        # a prompt of nothing round, as a whole
        append("append_prompt_30011", "bf16", 1, 4, 64, 64, 0, 30011),
        # prompts that come in chunks, behind what their sequences hold, of a model in the default type
        append("append_chunks_fp32", "fp32", 6, 5, 128, 16, 2003, 1021),
        # the window of the newest tokens of a layer, a head of its own for each, in the default type
        attend("window_fp32", "fp32", 8, 8, 8, 64, 32, 6011, 100, 513),
        # one long conversation, as the selection benchmark has its heads
        attend("attend_32k", "bf16", 1, 32, 8, 128, 32, 32768, 32768),
        # 48 sequences of all lengths
        attend("attend_ragged_48", "bf16", 48, 32, 8, 128, 32, 16384, 1),
        # half a million tokens, few heads
        attend("attend_500k", "fp16", 1, 16, 2, 128, 64, 524287, 524287),
        # the selected blocks of one long sequence: 16 of 64 keys and the newest
        select("select_32k", "bf16", 1, 32, 8, 128, 64, 32768, 32768, 16, 64),
        # 32 sequences of up to 64k tokens
        select("select_batch_32", "bf16", 32, 16, 4, 64, 64, 65536, 500, 16, 64),
        # the byte-level model: 8 sequences that may not repeat themselves
        logits("logits_bytes_8", "bf16", 8, 256, 512, "none", False),
        # 64 sequences of a large model, each under a grammar of its own
        logits("logits_128k_64", "bf16", 64, 128000, 4096, "packed", False),
        # a vocabulary of no round size in the default type: which tokens are allowed, one truth value each, and a bias for all
        logits("logits_50021_300", "fp32", 300, 50021, 777, "bool", True),
    ]


def draw(rng):
    def spread(lo, hi):                      # whole numbers, even over their logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind, dtype = rng.choice(("append", "attend", "attend", "select", "logits")), rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "logits":
        while True:
            batch, vocab = spread(1, 512), spread(100, 131072)
            if batch * vocab <= 15 * 10 ** 6:
                break
        case = logits("", dtype, batch, vocab, rng.choice((0, spread(1, 8192), spread(1, 8192))), rng.choice(("none", "packed", "bool")), rng.random() < 0.4)
    else:
        dim, block, kv_heads, group = rng.choice((64, 128)), rng.choice((16, 32, 32, 64, 128)), rng.choice((1, 2, 3, 4, 8, 8, 16)), rng.choice((1, 2, 4, 4, 5, 8, 16, 32))
        if kind == "append":
            while True:
                batch, held, rows = spread(1, 64), rng.choice((0, spread(1, 4096))), rng.choice((1, spread(1, 4096), spread(64, 32768)))
                if batch * kv_heads * dim * (held + rows + 2 * block) <= 1 << 27:
                    break
            case = append("", dtype, batch, kv_heads, dim, block, held, rows)
        else:
            while True:
                batch, longest = spread(1, 64), spread(1, 262144)
                if batch * kv_heads * dim * (longest + block) <= 1 << 29:
                    break
            shortest = longest if rng.random() < 0.4 else spread(1, longest)
            if kind == "attend":
                case = attend("", dtype, batch, group * kv_heads, kv_heads, dim, block, longest, shortest, rng.choice((0, 0, spread(1, 2048))))
            else:
                case = select("", dtype, batch, group * kv_heads, kv_heads, dim, block, longest, shortest, rng.choice((1, 4, 7, 16, 32)),
                              rng.choice((4, 16, 32, 64, 64, 80)), rng.random() < 0.25)
    del case["name"]
    return case


def lengths_of(case):
    """How many tokens each sequence holds: from the shortest to the longest, evenly over their logarithm, in no order."""
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
    order = sorted(range(b), key=lambda i: i * 7919 % b + i / b)
    made = [hi] * b
    for at, i in enumerate(order[1:]):
        made[i] = max(lo, min(hi, round(lo * (hi / lo) ** ((at + 0.5) / b))))
    return made


def starts_of(case):
    """How many rows each sequence held, and how many it takes."""
    b, held, rows = case["batch"], case["held"], case["rows"]
    return [held - i * 37 % (held + 1) if held else 0 for i in range(b)], [rows if i % 3 == 0 else max(1, rows - i * 101 % rows) for i in range(b)]


def capacity(case):
    block = case["block"]
    most = case["held"] + case["rows"] + block if case["kind"] == "append" else case["longest"]
    return (most + block - 1) // block * block


def seen(case, length):
    """Keys that a sequence's token attends."""
    if case["kind"] == "attend":
        return min(length, case["window"]) if case["window"] else length
    size = case["size"]
    earlier = (length - 1) // size
    return min(case["chosen"], earlier) * size + length - earlier * size


def work(case):
    each = 4 if case["dtype"] == "fp32" else 2
    b = case["batch"]
    if case["kind"] == "logits":
        n, v = b * case["vocab"], case["vocab"]
        mask = {"none": 0, "packed": b * ((v + 31) // 32) * 4, "bool": n}[case["mask"]]
        return dict(bytes=n * (each + 4) + b * case["history"] * 8 + mask + 4 * v * case["bias"] + 16 * b, flops=4 * n)
    hk, d = case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        rows = sum(starts_of(case)[1])
        return dict(bytes=2 * rows * hk * d * (each + 1) + 8 * hk * (rows // case["block"] + b) + 8 * b, flops=4 * rows * hk * d)
    keys = sum(seen(case, n) for n in lengths_of(case))
    units = case["heads"] if case.get("per_head") else hk
    moved = keys * units * 2 * (d + 4 / case["block"]) + 2 * b * case["heads"] * d * each
    return dict(bytes=moved + (9 * b * units * case["chosen"] if case["kind"] == "select" else 0), flops=4 * keys * case["heads"] * d)


def powers(amax):
    """The smallest power of two that takes amax into the range of e4m3."""
    m, e = torch.frexp(amax.float())
    k = torch.where(m > 0.875, e - 8, e - 9).clamp(LEAST, MOST)
    return torch.where(amax > 0, k, torch.full_like(k, LEAST))


def power(k):
    """2^k in fp32 to the last bit, of k from -126 on."""
    return ((k + 127) << 23).view(torch.float32)


def rounded(x, k):
    return (x.float() * power(-k)).clamp(-TOP, TOP).to(FP8)


def quantized(x, block):
    """'b h n d' -> e4m3 of the same shape and fp32 scales 'b h n/block'."""
    b, h, n, d = x.shape
    x = x.view(b, h, n // block, block, d)
    k = powers(x.abs().amax((-1, -2)))
    return rounded(x, k[..., None, None]).view(b, h, n, d), power(k)


def keys_and_values(case, n, randn):
    """Keys with a few features larger than the others and a part that all tokens share, values without."""
    b, hk, d = case["batch"], case["kv_heads"], case["dim"]
    k = randn(b, hk, n, d)
    k *= 1 + 3 * (torch.arange(d, device=DEVICE) % 29 == 3)
    k += randn(1, hk, 1, d)
    return k, randn(b, hk, n, d) * 0.7


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    randn = lambda *size: torch.randn(*size, device=DEVICE, generator=g)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=DEVICE)
    dtype, b = DTYPES[case["dtype"]], case["batch"]
    if case["kind"] == "logits":
        v, t = case["vocab"], case["history"]
        x = (randn(b, v) * 2.5 + 1).to(dtype)
        # a text repeats some tokens often
        history = (v * torch.rand(b, t, device=DEVICE, generator=g).pow(4)).long().clamp(max=v - 1) if t else None
        counts = ints([t - i * 53 % (t // 2 + 1) for i in range(b)]) if t else None
        rand = lambda: torch.rand(b, device=DEVICE, generator=g)
        state = dict(case=case, x=x, history=history, counts=counts, repetition=1 + 0.3 * rand(), frequency=0.2 * rand(), presence=0.5 * rand(),
                     temperature=0.5 + rand(), bias=randn(v) if case["bias"] else None, allowed=None)
        if case["mask"] == "packed":
            words = torch.randint(-2 ** 31, 2 ** 31 - 1, (b, (v + 31) // 32), device=DEVICE, generator=g, dtype=torch.int64)
            state["allowed"] = words.to(torch.int32)
        elif case["mask"] == "bool":
            state["allowed"] = torch.rand(b, v, device=DEVICE, generator=g) < 0.3
        return state
    n, block = capacity(case), case["block"]
    k, v = keys_and_values(case, n, randn)
    (keys, key_scales), (values, value_scales) = quantized(k, block), quantized(v, block)
    state = dict(case=case, cache=(keys, values, key_scales, value_scales))
    if case["kind"] == "append":
        k, v = keys_and_values(case, case["rows"], randn)
        starts, counts = starts_of(case)
        return dict(state, k=(k * 1.5).to(dtype), v=(v * 1.5).to(dtype), starts=ints(starts), counts=ints(counts))
    hq, d = case["heads"], case["dim"]
    lengths = lengths_of(case)
    state.update(q=(randn(b, hq, 1, d) * 1.2).to(dtype), lengths=ints(lengths))
    if case["kind"] == "select":
        size, s, units = case["size"], case["chosen"], hq if case["per_head"] else case["kv_heads"]
        blocks = (n + size - 1) // size
        earlier = (state["lengths"].long() - 1) // size
        score = torch.rand(b, units, 1, max(blocks, s), device=DEVICE, generator=g)
        score = score.masked_fill(torch.arange(max(blocks, s), device=DEVICE) >= earlier[:, None, None, None], -1.0)
        best, idx = score.topk(s, dim=-1)
        state.update(idx=idx.to(torch.int32), fmask=best >= 0)
    return state


def plain_append(codes, scales, x, starts, counts, block):
    """The blocks that take rows: those they hold keep their values, in units of a scale that holds the new ones too."""
    b, h, n, d = x.shape
    touched = (n + block - 1) // block + 1
    first, end = starts.long(), (starts + counts).long()
    ids = (first // block)[:, None] + torch.arange(touched, device=DEVICE)
    ids = torch.minimum(ids, torch.tensor(scales.shape[2] - 1, device=DEVICE))
    at = torch.arange(b, device=DEVICE)[:, None]
    pos = ids[..., None] * block + torch.arange(block, device=DEVICE)                                   # 'b blocks block'
    held, new = pos < first[:, None, None], (pos >= first[:, None, None]) & (pos < end[:, None, None])
    rows = x.permute(0, 2, 1, 3)[at[..., None], (pos - first[:, None, None]).clamp(0, n - 1)]            # 'b blocks block h d'
    rows = torch.where(new[..., None, None], rows.float(), 0.0).permute(0, 1, 3, 2, 4)                   # 'b blocks h block d'
    raw = codes.view(torch.uint8).view(b, h, -1, block, d)
    before = raw[at, :, ids]                                                                             # 'b blocks h block d'
    s0 = scales[at, :, ids]                                                                              # 'b blocks h'
    k0 = torch.frexp(s0)[1] - 1
    k = powers(rows.abs().amax((-1, -2)))
    k = torch.where(held.any(-1)[..., None], torch.maximum(k, k0), k)
    moved = (before.view(FP8).float() * power((k0 - k).clamp(min=-126))[..., None, None]).clamp(-TOP, TOP).to(FP8)
    made = rounded(rows, k[..., None, None])
    pick = lambda m: m[:, :, None, :, None]
    after = torch.where(pick(new), made.view(torch.uint8), torch.where(pick(held), moved.view(torch.uint8), before))
    any_new = new.any(-1)
    after = torch.where(any_new[..., None, None, None], after, before)
    raw[at, :, ids] = after
    scales[at, :, ids] = torch.where(any_new[..., None], power(k), s0)


def softmax_products(q, k, v, live):
    """q 'u g d', k and v 'u n d', live 'u n' -> 'u g d'; nothing live: zeros."""
    s = (q * q.shape[-1] ** -0.5) @ k.transpose(1, 2)
    s = s.masked_fill(~live[:, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > float("-inf"), top, 0.0))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, (p @ v) / total, 0.0)


def plain_attend(state):
    case, (keys, values, key_scales, value_scales), q = state["case"], state["cache"], state["q"]
    b, hk, n, d = keys.shape
    block, g = case["block"], q.shape[1] // hk
    k = (keys.float().view(b, hk, -1, block, d) * key_scales[..., None, None]).view(b * hk, n, d)
    v = (values.float().view(b, hk, -1, block, d) * value_scales[..., None, None]).view(b * hk, n, d)
    at, length = torch.arange(n, device=DEVICE), state["lengths"].long()[:, None]
    live = at < length
    if case["window"]:
        live &= at >= length - case["window"]
    out = softmax_products(q.float().view(b * hk, g, d), k, v, live[:, None].expand(b, hk, n).reshape(b * hk, n))
    return out.view(q.shape).to(q.dtype)


def plain_select(state):
    case, (keys, values, key_scales, value_scales), q = state["case"], state["cache"], state["q"]
    b, hk, n, d = keys.shape
    block, size, g = case["block"], case["size"], q.shape[1] // hk
    idx, fmask, length = state["idx"][:, :, 0].long(), state["fmask"][:, :, 0], state["lengths"].long()
    units = idx.shape[1]
    latest = ((length - 1) // size)[:, None, None].expand(b, units, 1)
    blocks = torch.cat((idx, latest), -1)
    pos = blocks[..., None] * size + torch.arange(size, device=DEVICE)
    live = torch.cat((fmask, torch.ones_like(latest, dtype=torch.bool)), -1)[..., None] & (pos < length[:, None, None, None])
    pos, live = pos.reshape(b, units, -1).clamp(max=n - 1), live.reshape(b * units, -1)
    at, head = torch.arange(b, device=DEVICE)[:, None, None], (torch.arange(units, device=DEVICE) // (units // hk))[:, None]
    rows = lambda codes, scales: (codes.view(torch.uint8)[at, head, pos].view(FP8).float() * scales[at, head, pos // block][..., None]).view(b * units, -1, d)
    out = softmax_products(q.float().view(b * units, g * hk // units, d), rows(keys, key_scales), rows(values, value_scales), live)
    return out.view(q.shape).to(q.dtype)


def plain_logits(state):
    x, history, allowed = state["x"].float(), state["history"], state["allowed"]
    b, v = x.shape
    if history is not None:
        t = history.shape[1]
        live = torch.arange(t, device=DEVICE) < state["counts"][:, None]
        count = torch.zeros(b, v, device=DEVICE).scatter_add_(1, history, live.float())
        said = count > 0
        penalised = torch.where(x > 0, x / state["repetition"][:, None], x * state["repetition"][:, None])
        penalised = penalised - state["frequency"][:, None] * count - state["presence"][:, None]
        x = torch.where(said, penalised, x)
    if state["bias"] is not None:
        x = x + state["bias"]
    x = x / state["temperature"][:, None]
    if allowed is not None:
        if allowed.dtype == torch.int32:
            allowed = ((allowed[..., None] >> torch.arange(32, device=DEVICE)) & 1).bool().view(b, -1)[:, :v]
        x = x.masked_fill(~allowed, float("-inf"))
    return x


def run(state):
    case = state["case"]
    if own:
        from native_sparse_attention_pytorch_amd import ops
        if case["kind"] == "logits":
            return ops.adjust_logits(state["x"], state["history"], state["counts"], repetition_penalty=state["repetition"],
                                     frequency_penalty=state["frequency"], presence_penalty=state["presence"], bias=state["bias"],
                                     temperature=state["temperature"], allowed=state["allowed"])
        cache = ops.Cache8(*state["cache"])
        if case["kind"] == "append":
            ops.cache8_append(cache, state["k"], state["v"], state["starts"], state["counts"])
            return tuple(cache)
        if case["kind"] == "attend":
            return ops.cache8_attend(state["q"], cache, state["lengths"], window=case["window"] or None)
        return ops.cache8_select_attend(state["q"], cache, state["lengths"], case["size"], state["idx"], state["fmask"])
    if case["kind"] == "logits":
        return plain_logits(state)
    if case["kind"] == "append":
        keys, values, key_scales, value_scales = state["cache"]
        plain_append(keys, key_scales, state["k"], state["starts"], state["counts"], case["block"])
        plain_append(values, value_scales, state["v"], state["starts"], state["counts"], case["block"])
        return state["cache"]
    return plain_attend(state) if case["kind"] == "attend" else plain_select(state)


def nearest_e4m3(y):
    """The e4m3 value next to y, halves to even, in 64 bits: steps of 2^-9 below 2^-6, of an eighth of the power of two above."""
    a = y.abs().clamp(max=TOP)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.round(a / step) * step, y)


def exact_append(state):
    case = state["case"]
    block, (starts, counts) = case["block"], starts_of(case)
    out = []
    for codes, scales, x in zip(state["cache"][:2], state["cache"][2:], (state["k"], state["v"])):
        codes, scales, x = codes.double(), scales.double(), x.double()
        for i, (start, count) in enumerate(zip(starts, counts)):
            for at in range(start // block, (start + count - 1) // block + 1):
                lo, hi = max(start, at * block), min(start + count, (at + 1) * block)
                rows = x[i, :, lo - start:hi - start]
                top = rows.abs().amax((-1, -2)) / TOP
                # (the logarithm may be off by one rounding next to a power of two)
                k = torch.ceil(torch.log2(top.clamp(min=2.0 ** -200)) - 0.25)
                k = torch.where(torch.exp2(k) < top, k + 1, k).clamp(LEAST, MOST)
                unit = torch.exp2(k)
                if lo > at * block:
                    unit = torch.maximum(unit, scales[i, :, at])
                    codes[i, :, at * block:lo] = nearest_e4m3(codes[i, :, at * block:lo] * (scales[i, :, at] / unit)[:, None, None])
                codes[i, :, lo:hi] = nearest_e4m3(rows / unit[:, None, None])
                scales[i, :, at] = unit
        out.append((codes, scales))
    (keys, key_scales), (values, value_scales) = out
    return keys, values, key_scales, value_scales


def exact_attention(state):
    case, (keys, values, key_scales, value_scales), q = state["case"], state["cache"], state["q"].double()
    hk, d = keys.shape[1], keys.shape[3]
    g, block = q.shape[1] // hk, case["block"]
    out = torch.zeros_like(q)
    for i, length in enumerate(lengths_of(case)):
        def rows(codes, scales, j, at):
            return codes[i, j].view(torch.uint8)[at].view(FP8).double() * scales[i, j].double()[at // block][:, None]
        for h in range(q.shape[1]) if case.get("per_head") else range(hk):
            per_head = case.get("per_head")
            j, cols = (h // g, slice(h, h + 1)) if per_head else (h, slice(h * g, h * g + g))
            if case["kind"] == "attend":
                at = torch.arange(max(0, length - case["window"]) if case["window"] else 0, length, device=DEVICE)
            else:
                size, own_block = case["size"], (length - 1) // case["size"]
                chosen = state["idx"][i, h, 0][state["fmask"][i, h, 0]].long()
                at = (chosen[:, None] * size + torch.arange(size, device=DEVICE)).reshape(-1)
                at = torch.cat((at, torch.arange(own_block * size, length, device=DEVICE)))
            w = torch.softmax(q[i, cols, 0] @ rows(keys, key_scales, j, at).mT / math.sqrt(d), -1)
            out[i, cols, 0] = w @ rows(values, value_scales, j, at)
    return out


def exact_logits(state):
    x, v = state["x"].double(), state["case"]["vocab"]
    each = lambda name: state[name].double()[:, None]
    if state["history"] is not None:
        said = torch.stack([torch.bincount(row[:int(n)], minlength=v) for row, n in zip(state["history"], state["counts"])])
        lower = x * each("repetition") ** (1 - 2 * (x > 0).double()) - each("presence") - said * each("frequency")
        x = torch.where(said > 0, lower, x)
    if state["bias"] is not None:
        x = x + state["bias"].double()
    x = x / each("temperature")
    allowed = state["allowed"]
    if allowed is not None:
        if allowed.dtype == torch.int32:
            at = torch.arange(v, device=DEVICE)
            allowed = (allowed.long()[:, at // 32] // 2 ** (at % 32)) % 2 == 1
        x = torch.where(allowed, x, -math.inf)
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "append":
        blocks = sum((s + c - 1) // case["block"] - s // case["block"] + 1 for s, c in zip(*starts_of(case)))
        return exact_append(state) if blocks <= 20000 else None
    return exact_logits(state) if case["kind"] == "logits" else exact_attention(state)
