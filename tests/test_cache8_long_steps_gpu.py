"""Decode steps over an 8-bit cache whose window or blocks are shared by several work-groups, and from prompts that have no compressed key yet, against their parts in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF16, FP8 = "cuda", torch.bfloat16, torch.float8_e4m3fn

# A work-group has 256 keys of a branch.
#                        dim, heads, kv_heads, dim_head, window, compress block, stride, selection block, selected, share, prompt, max_len
LAYERS = {
    "a window of three": (64, 4, 2, 64, 700, 16, 16, 16, 2, True, 805, 900),
    "a window not yet full": (64, 8, 1, 128, 1500, 16, 16, 32, 1, True, 300, 2000),
    "blocks of three": (128, 8, 2, 128, 40, 32, 16, 64, 8, True, 1001, 1100),
    "blocks of three for each head": (64, 6, 2, 64, 16, 16, 16, 64, 8, False, 990, 1100),
    "small blocks of two": (64, 4, 2, 64, 20, 8, 8, 8, 40, True, 650, 700),
    "small blocks of two for each head": (64, 4, 1, 128, 300, 8, 8, 8, 33, False, 650, 700),
    "blocks of six keys": (64, 4, 4, 64, 20, 8, 8, 48, 9, True, 901, 1000),
    "both": (64, 20, 1, 128, 513, 16, 16, 64, 16, True, 1500, 1700),
    "nothing compressed": (64, 4, 2, 64, 16, 16, 16, 16, 2, True, 3, 90),
    "nothing compressed, blocks of six keys": (64, 4, 2, 64, 16, 32, 8, 48, 2, True, 5, 90),
    "one token, nothing compressed": (64, 5, 1, 48, 300, 16, 8, 16, 4, True, 1, 700),
}


def _layer(name):
    from native_sparse_attention_pytorch_amd import SparseAttention
    dim, heads, kv_heads, d, window, cbs, st, block, chosen, share, prompt, max_len = LAYERS[name]
    torch.manual_seed(heads + prompt)
    m = SparseAttention(dim=dim, dim_head=d, heads=heads, kv_heads=kv_heads, causal=True, sliding_window_size=window, compress_block_size=cbs,
                        compress_block_sliding_stride=st, selection_block_size=block, num_selected_blocks=chosen, query_heads_share_selected_kv=share).to(DEV, BF16)
    with torch.no_grad():
        for p in (m.k_intrablock_positions, m.v_intrablock_positions, m.compress_mem_kv, m.to_strategy_combine[0].weight):
            p.normal_(0, 0.1)
        _, cache = m(torch.randn(2, prompt, dim, device=DEV, dtype=BF16), return_cache=True)
    return m, cache, max_len


@torch.no_grad()
@pytest.mark.parametrize("name", LAYERS)
def test_a_step_is_its_parts(name):
    """The cache as `cache8_append` leaves it, bit for bit; the output from the cache and the projections: a branch is off by its probabilities (kept to 8 bits at least, 2^-9 of the
    largest value), by what the fp32 scores of its keys are off, and by its rounding to bf16 (2^-9), the branches' sum by 2^-9, the output by 2^-8."""
    from native_sparse_attention_pytorch_amd import ops
    from native_sparse_attention_pytorch_amd.decode_session import DecodeSession
    m, cache, max_len = _layer(name)
    session = DecodeSession(m, cache, max_len=max_len, cache_dtype=FP8)
    b, hk, hq, d0, d = 2, m.kv_heads, m.heads, m.dim_head, session.d
    each, block, npf, scale = hq // hk, m.selection_block_size, m.selection_block_size // m.compress_block_sliding_stride, d0 ** -0.5
    assert "nothing" not in name or session.nc == 0
    for _ in range(20):
        x = torch.randn(b, 1, m.to_qkv.in_features, device=DEV, dtype=BF16)
        pos, nc = session.pos, session.nc
        before = ops.Cache8(*(t.clone() for t in session.cache8))
        out = session.step(x)
        qkvg = (ops.skinny_linear(x, session.w_cat, None, m.norm.weight, session._eps()) if session.own_in and session.own_norm
                else torch.nn.functional.linear(m.norm(x), session.w_cat))            # (as the step makes them)
        heads = lambda at, n: qkvg[..., at:at + n * d].view(b, 1, n, d).transpose(1, 2)
        q, k, v = heads(0, hq), heads(hq * d, hk), heads((hq + hk) * d, hk)
        rq, rk = ops.rotary(q, session.freqs, pos), ops.rotary(k, session.freqs, pos)
        ops.cache8_append(before, rk, v, pos)
        for got, want in zip(session.cache8, before):
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))

        keys, vals = (t.double()[..., :d0] for t in session.cache8.rows(0, pos + 1, torch.float32))
        ck, cv = session.CK[:, :, :nc], session.CV[:, :, :nc]
        gates = torch.sigmoid(qkvg[..., (hq + 2 * hk) * d:][..., :3 * hq].double() + m.to_strategy_combine[0].bias.double()).view(b, hq, 3)
        merged, size = torch.zeros(b, hq, d0, dtype=torch.float64, device=DEV), torch.zeros(b, hq, dtype=torch.float64, device=DEV)
        chosen = min(m.num_selected_blocks, nc // npf)
        if chosen:
            logits = ops.decode_range_attend(q, ck, cv, 0, nc, session.mem_k, session.mem_v, return_logits=True)[1] * (d / d0) ** 0.5
            _, idx, fmask = ops.decode_importance_topk(logits, hk, npf, m.query_heads_share_selected_kv, chosen)
        for i in range(b):
            for h in range(hq):
                j = h // each
                row = h if chosen and idx.shape[1] == hq else j
                blocks = [blk for blk, ok in zip(idx[i, row, 0].tolist(), fmask[i, row, 0].tolist()) if ok] if chosen else []
                at = [p for blk in blocks for p in range(blk * block, blk * block + block)] + list(range(pos // block * block, pos + 1))
                first = max(0, pos - m.sliding_window_size)
                parts = [(rq, keys[i, j, at], vals[i, j, at], 1), (rq, keys[i, j, first:pos + 1], vals[i, j, first:pos + 1], 2)]
                if nc:
                    parts.append((q, torch.cat((session.mem_k[j], ck[i, j]))[:, :d0].double(), torch.cat((session.mem_v[j], cv[i, j]))[:, :d0].double(), 0))
                for query, kk, vv, s in parts:
                    y = query[i, h, 0, :d0].double() * scale
                    off = (d + 16) * 2. ** -24 * (kk.abs() @ y.abs()).max()
                    merged[i, h] += gates[i, h, s] * (torch.softmax(kk @ y, -1) @ vv)
                    size[i, h] += gates[i, h, s] * vv.abs().max() * (2 ** -8 + 2 ** -9 + 2 * off)
        w = m.combine_heads.weight.double()
        want = merged.view(b, -1) @ w.T
        bound = size.repeat_interleave(d0, 1) @ w.abs().T + 2 ** -8 * want.abs()
        far = (out[:, 0].double() - want).abs()
        assert (far <= bound).all(), f"token {pos}: {(far / bound).max().item():.3g} times the bound"
