"""The 8-bit cache, the attention over it and what is done to logits, in 64 bits on the host, one row and one head after the other."""
import math

import torch

FP8 = torch.float8_e4m3fn


def e4m3(y):
    """Nearest e4m3 value, halves to even: steps of 2^-9 below 2^-6, of an eighth of the power of two above; beyond 448: 448."""
    a = y.abs().clamp(max=448.)
    _, e = torch.frexp(a.clamp(min=2. ** -6))
    step = torch.ldexp(torch.ones_like(a), e - 4)
    return torch.copysign(torch.round(a / step) * step, y)


def scale_of(rows):
    """Of a block's new rows: the smallest power of two that takes the largest finite value to 448."""
    finite = rows[rows.isfinite()]
    top = finite.abs().max().item() if finite.numel() else 0.
    k = -110
    while top > 448. * 2. ** k and k < 119:
        k += 1
    return 2. ** k


def append(codes, scales, x, starts, counts, block):
    """codes 'b h n d' and scales 'b h n/block' in 64 bits, changed in place."""
    b, h, rows, _ = x.shape
    for i in range(b):
        start, end = starts[i], min(starts[i] + max(0, min(counts[i], rows)), codes.shape[2])
        for j in range(h):
            for blk in range(start // block, (end - 1) // block + 1 if end > start else 0):
                lo, hi = max(start, blk * block), min(end, (blk + 1) * block)
                new = x[i, j, lo - start:hi - start]
                s = scale_of(new)
                if lo > blk * block:
                    old = scales[i, j, blk].item()
                    s = max(s, old)
                    if s != old:
                        codes[i, j, blk * block:lo] = e4m3(codes[i, j, blk * block:lo] * (old / s))
                codes[i, j, lo:hi] = torch.where(new.isfinite(), e4m3(new / s), math.nan)
                scales[i, j, blk] = s


def quantized(x, block):
    """Codes and scales of 'b h n d' as the cache would hold them, quickly."""
    b, h, n, d = x.shape
    x = x.double().view(b, h, n // block, block, d)
    _, e = torch.frexp(x.abs().amax((-1, -2)) / 448.)
    unit = torch.ldexp(torch.ones(e.shape, dtype=torch.float64, device=x.device), e)
    unit = torch.where(unit / 2 >= x.abs().amax((-1, -2)) / 448., unit / 2, unit).clamp(2. ** -110, 2. ** 119)
    return e4m3(x / unit[..., None, None]).to(FP8).view(b, h, n, d), unit.float()


def rows_of(codes, scales, block, at):
    """Rows `at` of one head, in 64 bits."""
    return codes.view(torch.uint8)[at].view(FP8).double() * scales.double()[at // block][:, None]


def attend(q, cache, lengths, window=0, size=0, idx=None, fmask=None, scale=None):
    """(outputs 'b hq 1 d' in 64 bits, the largest |v| that each attends, how far fp32 scores of its keys may be off)."""
    keys, values, key_scales, value_scales = cache
    b, hq, _, d0 = q.shape
    hk, n, d = keys.shape[1:]
    block = n // key_scales.shape[2]
    scale = d0 ** -0.5 if scale is None else scale
    out = torch.zeros(b, hq, 1, d0, dtype=torch.float64)
    largest, off = torch.zeros(b, hq, 1, 1, dtype=torch.float64), torch.zeros(b, hq, 1, 1, dtype=torch.float64)
    for i in range(b):
        length = lengths[i]
        if length == 0:
            continue
        per_head = idx is not None and idx.shape[1] == hq
        each = 1 if per_head else hq // hk
        for u in range(hq // each):
            h, j = slice(u * each, u * each + each), u * each // (hq // hk)
            if size:
                at = [k for blk, ok in zip(idx[i, u, 0].tolist(), fmask[i, u, 0].tolist()) if ok and 0 <= blk <= n
                      for k in range(blk * size, min(blk * size + size, length))]
                at += range((length - 1) // size * size, length)
            else:
                at = range(max(0, length - window) if window else 0, length)
            at = torch.tensor(list(at))
            k = rows_of(keys[i, j], key_scales[i, j], block, at)[:, :d0]
            v = rows_of(values[i, j], value_scales[i, j], block, at)[:, :d0]
            x = q[i, h, 0].double() * scale
            out[i, h, 0] = torch.softmax(x @ k.T, -1) @ v
            largest[i, h] = v.abs().max()
            off[i, h] = (d0 + 16) * 2. ** -24 * (x.abs() @ k.abs().T).amax()
    return out, largest, off


def attend_bound(want, largest, off, dtype, keys):
    """How far the kernels may be off: the result's rounding; probabilities of `keys` keys whose sum is in fp32 and that are kept to 16 bits (24 of fp32 queries):
    2^-17 or 2^-24 of the largest value each way; what the scores are off changes a probability by as much, relative to itself, and their sum too."""
    kept = 2. ** -24 if dtype == torch.float32 else 2. ** -17
    return torch.finfo(dtype).eps / 2 * want.abs() + largest * (2 * kept + 2 * keys * 2. ** -24 + 2 * off) + torch.finfo(dtype).tiny


def adjust(x, history=None, lengths=None, repetition=1., frequency=0., presence=0., bias=None, temperature=1., allowed=None):
    """One row in 64 bits."""
    x = x.double().clone()
    if history is not None:
        tokens = history.tolist()[:len(history) if lengths is None else max(0, lengths)]
        for t in {t for t in tokens if 0 <= t < len(x)}:
            x[t] = (x[t] / repetition if x[t] > 0 else x[t] * repetition) - frequency * tokens.count(t) - presence
    if bias is not None:
        x = x + bias.double()
    x = x / temperature
    if allowed is not None:
        if allowed.dtype == torch.int32:
            words = [w & 0xffffffff for w in allowed.tolist()]
            allowed = torch.tensor([bool(words[i // 32] >> (i % 32) & 1) for i in range(len(x))])
        x = x.masked_fill(~allowed, -math.inf)
    return x
