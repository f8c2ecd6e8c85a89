"""Decode sessions over an 8-bit cache: a step against its parts in 64 bits and against the operators by themselves, replayed and launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF16, FP8 = "cuda", torch.bfloat16, torch.float8_e4m3fn

#         dim, heads, kv_heads, dim_head, window, compress block, stride, selection block, selected, share
LAYERS = {
    "byte model": (128, 4, 2, 64, 16, 16, 8, 16, 2, True),
    "small blocks": (64, 4, 4, 64, 32, 4, 4, 4, 4, True),
    "wide heads": (128, 8, 2, 128, 40, 16, 16, 32, 3, True),
    "heads that select": (96, 4, 2, 64, 7, 8, 4, 8, 2, False),
    "odd heads": (64, 5, 1, 48, 21, 16, 8, 48, 2, True),
    "no blocks": (64, 2, 2, 64, 300, 16, 16, 16, 0, True),
    "many heads": (64, 20, 1, 64, 100, 8, 8, 16, 5, True),
}


def _layer(name, b=3, prompt=37, scale=1.):
    from native_sparse_attention_pytorch_amd import SparseAttention
    dim, heads, kv_heads, d, window, cbs, st, block, chosen, share = LAYERS[name]
    torch.manual_seed(b + heads)
    m = SparseAttention(dim=dim, dim_head=d, heads=heads, kv_heads=kv_heads, causal=True, sliding_window_size=window, compress_block_size=cbs,
                        compress_block_sliding_stride=st, selection_block_size=block, num_selected_blocks=chosen, query_heads_share_selected_kv=share).to(DEV, BF16)
    with torch.no_grad():
        for p in (m.k_intrablock_positions, m.v_intrablock_positions, m.compress_mem_kv, m.to_strategy_combine[0].weight):
            p.normal_(0, 0.1)
        _, cache = m(torch.randn(b, prompt, dim, device=DEV, dtype=BF16) * scale, return_cache=True)
    return m, cache


def _softmax(q, k, v):
    return torch.softmax(q @ k.T * q.shape[-1] ** -0.5, -1) @ v


@torch.no_grad()
@pytest.mark.parametrize("name", LAYERS)
def test_a_step_is_its_parts(name):
    """What goes into the cache, bit for bit; the layer's output, from the projections that the step made and the cache that it left.  A branch is off by its
    rounding to bf16 and its probabilities' (2^-9 each of the largest value), their sum by 2^-9, the output by 2^-8."""
    from native_sparse_attention_pytorch_amd import ops
    from native_sparse_attention_pytorch_amd.decode_session import DecodeSession
    m, cache = _layer(name)
    session, plain = DecodeSession(m, cache, max_len=90, cache_dtype=FP8), DecodeSession(m, cache, max_len=90)
    assert session.cache8 is not None
    b, hk, hq, d0, d = 3, m.kv_heads, m.heads, m.dim_head, session.d
    for _ in range(40):
        x = torch.randn(b, 1, m.to_qkv.in_features, device=DEV, dtype=BF16)
        pos, nc = session.pos, session.nc
        before = ops.Cache8(*(t.clone() for t in session.cache8))
        out = session.step(x)
        plain.step(x)
        qkvg = (ops.skinny_linear(x, session.w_cat, None, m.norm.weight, session._eps()) if session.own_in and session.own_norm
                else torch.nn.functional.linear(m.norm(x), session.w_cat))            # (as the step makes them)
        heads = lambda at, n: qkvg[..., at:at + n * d].view(b, 1, n, d).transpose(1, 2)
        q, k, v = heads(0, hq), heads(hq * d, hk), heads((hq + hk) * d, hk)
        rq, rk = ops.rotary(q, session.freqs, pos), ops.rotary(k, session.freqs, pos)
        ops.cache8_append(before, rk, v, pos)
        for got, want in zip(session.cache8, before):
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
        for got, want in zip(session.cache()[1][1], plain.cache()[1][1]):
            assert torch.equal(got, want)                                    # the open window is what it was
        assert torch.equal(session.CK, plain.CK) and torch.equal(session.CV, plain.CV)

        keys, vals = (t.double() for t in session.cache8.rows(0, pos + 1, torch.float32))
        ck, cv = session.CK[:, :, :nc], session.CV[:, :, :nc]
        gates = torch.sigmoid(qkvg[..., (hq + 2 * hk) * d:][..., :3 * hq].double() + m.to_strategy_combine[0].bias.double()).view(b, hq, 3)
        merged, size = torch.zeros(b, hq, d0, dtype=torch.float64, device=DEV), torch.zeros(b, hq, dtype=torch.float64, device=DEV)
        npf, block = m.selection_block_size // m.compress_block_sliding_stride, m.selection_block_size
        chosen = min(m.num_selected_blocks, nc // npf)
        if nc:
            logits = ops.decode_range_attend(q, ck, cv, 0, nc, session.mem_k, session.mem_v, return_logits=True)[1] * (d / d0) ** 0.5
        if chosen:
            _, idx, fmask = ops.decode_importance_topk(logits, hk, npf, m.query_heads_share_selected_kv, chosen)
        for i in range(b):
            for h in range(hq):
                j = h // (hq // hk)
                row = h if chosen and idx.shape[1] == hq else j
                blocks = [blk for blk, ok in zip(idx[i, row, 0].tolist(), fmask[i, row, 0].tolist()) if ok] if chosen else []
                at = [p for blk in blocks for p in range(blk * block, blk * block + block)] + list(range(pos // block * block, pos + 1))
                window = list(range(max(0, pos - m.sliding_window_size), pos + 1))
                parts = [(rq, keys[i, j, at], vals[i, j, at], 1), (rq, keys[i, j, window], vals[i, j, window], 2)]
                if nc:
                    parts.append((q, torch.cat((session.mem_k[j], ck[i, j])).double(), torch.cat((session.mem_v[j], cv[i, j])).double(), 0))
                for query, kk, vv, s in parts:
                    merged[i, h] += gates[i, h, s] * _softmax(query[i, h, :, :d0].double(), kk[:, :d0], vv[:, :d0])[0]
                    size[i, h] += gates[i, h, s] * vv.abs().max()
        w = m.combine_heads.weight.double()
        want = merged.view(b, -1) @ w.T
        bound = (2 ** -8 + 2 ** -9) * size.repeat_interleave(d0, 1) @ w.abs().T + 2 ** -8 * want.abs()
        assert ((out[:, 0].double() - want).abs() <= bound).all(), f"token {pos}: {((out[:, 0].double() - want).abs() / bound).max().item():.3g} times the bound"


@torch.no_grad()
@pytest.mark.parametrize("name", ["byte model", "small blocks", "odd heads"])
def test_replayed_steps_are_the_launched_ones(name):
    """A recorded step replayed between other work, against launches of the same session's parts; past the capacity nothing is written."""
    from native_sparse_attention_pytorch_amd.decode_session import DecodeSession
    m, cache = _layer(name)
    session, other = (DecodeSession(m, cache, max_len=71, cache_dtype=FP8) for _ in range(2))
    graphs = session.graphs
    for i in range(34):
        x = torch.randn(3, 1, m.to_qkv.in_features, device=DEV, dtype=BF16)
        event = session.completes_window()
        session.x_buf.copy_(x)
        step = not session.direct and event                  # (of a session that launches its steps the second graph is the window's alone)
        graphs[step].replay()
        got = session.outs[step].clone()
        if event and not step:
            graphs[True].replay()
        session.advance_host(event)
        assert torch.equal(got, other.step(x))
        if i % 5 == 0:
            torch.cuda.synchronize()
    assert session.pos == 71
    for a, c in zip(session.cache8, other.cache8):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    graphs[False].replay()
    torch.cuda.synchronize()
    for a, c in zip(session.cache8, other.cache8):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    with pytest.raises(RuntimeError, match="capacity"):
        session.step(x)


@torch.no_grad()
def test_a_session_goes_back_to_the_module_s_caches():
    """What the codes stand for is exact in bf16: a session made from another's caches, and the module's own step from them, read the same keys."""
    from native_sparse_attention_pytorch_amd.decode_session import DecodeSession
    m, cache = _layer("byte model", prompt=64)
    session = DecodeSession(m, cache, max_len=128, cache_dtype=FP8)
    for _ in range(5):
        session.step(torch.randn(3, 1, 128, device=DEV, dtype=BF16))
    back = session.cache()
    for t, rows in zip(back[0], session.cache8.rows(0, 69, torch.float32)):
        assert t.dtype == BF16 and torch.equal(t.float(), rows[..., :t.shape[-1]])
    again = DecodeSession(m, back, max_len=128, cache_dtype=FP8)
    for a, c in zip(again.cache8.rows(0, 69, torch.float32), session.cache8.rows(0, 69, torch.float32)):
        assert torch.equal(a, c)
    x = torch.randn(3, 1, 128, device=DEV, dtype=BF16)
    out, _ = m(x, cache=back, return_cache=True)
    # one key of 70 in 8 bits or 16, the output of three gated branches: within an eighth of e4m3's half step
    assert (out.float() - session.step(x).float()).abs().max() <= 2 ** -4 * out.float().abs().max()


def _model():
    from native_sparse_attention_pytorch_amd.transformer import Transformer
    torch.manual_seed(0)
    return Transformer(num_tokens=256, dim=128, depth=2, dim_head=64, heads=4, kv_heads=2, sparse_attn_kwargs=dict(
        sliding_window_size=16, compress_block_size=16, compress_block_sliding_stride=8, selection_block_size=16, num_selected_blocks=2)).to(DEV, BF16)


@torch.no_grad()
def test_a_model_s_session():
    from native_sparse_attention_pytorch_amd.decode_session import TransformerDecodeSession
    model, ids = _model(), torch.randint(0, 256, (2, 50), device=DEV)
    _, caches = model(ids, return_cache=True)
    session, other = (TransformerDecodeSession(model, caches, max_len=90, cache_dtype=FP8) for _ in range(2))
    for _ in range(40):
        token = torch.randint(0, 256, (2, 1), device=DEV)
        first = other.layers[0]
        event = first.completes_window()
        other.tok.copy_(token)
        want = other._body(advance=1, event=event, count=True)
        for s in other.layers:
            s.advance_host(event)
        assert torch.equal(session.step(token), want)


@torch.no_grad()
@pytest.mark.parametrize("how", ["parallel", "cached", "session", "8 bits"])
def test_sampling_with_penalties_biases_and_masks(how):
    model, prompt = _model(), torch.randint(0, 256, (3, 20), device=DEV)
    more = dict(parallel={}, cached=dict(use_cache_kv=True), session=dict(use_cache_kv=True, use_graph=True))
    more["8 bits"] = dict(more["session"], cache_dtype=FP8)
    run = lambda **args: model.sample(prompt, 60, **more[how], **args)
    assert run().shape == (3, 40)
    for temperature in (0., 1.):
        whole = torch.cat((prompt, run(temperature=temperature, presence_penalty=1e6)), 1)
        for old, row in zip(prompt.tolist(), whole.tolist()):
            assert len(set(row[20:])) == 40 and not set(row[20:]) & set(old)              # nothing twice, nothing of the prompt
    allowed = torch.zeros(256, dtype=torch.bool, device=DEV)
    allowed[65:70] = True
    assert set(run(allowed=allowed).flatten().tolist()) <= set(range(65, 70))
    bias = torch.full((256,), -1e9, device=DEV)
    bias[7] = 0
    assert (run(logit_bias=bias, repetition_penalty=torch.tensor([1.2, 1., 0.9], device=DEV)) == 7).all()

    def even_after_odd(tokens):
        ok = torch.zeros(3, 256, dtype=torch.bool, device=DEV)
        ok[:, :] = (torch.arange(256, device=DEV) + tokens[:, -1:]) % 2 == 1
        return ok
    whole = torch.cat((prompt[:, -1:], run(allowed=even_after_odd)), 1)
    assert ((whole[:, 1:] + whole[:, :-1]) % 2 == 1).all()


def test_what_a_session_refuses():
    from native_sparse_attention_pytorch_amd.decode_session import DecodeSession
    m, cache = _layer("byte model")
    with pytest.raises(ValueError, match="cache_dtype"):
        DecodeSession(m, cache, max_len=90, cache_dtype=torch.float16)
    with pytest.raises(ValueError, match="cache_dtype"):
        _model().sample(torch.zeros(1, 4, dtype=torch.long, device=DEV), 8, cache_dtype=FP8)
