"""A session over an 8-bit cache runs its step before the first token, for the libraries and for the recording: none of that is in the caches.  A bf16 row that
such a step writes is the next token's, who overwrites it; the scale of the block that it is in would stay, and with it what the block's other rows were rounded to."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF16, FP8 = "cuda", torch.bfloat16, torch.float8_e4m3fn
LAYER = dict(sliding_window_size=16, compress_block_size=16, compress_block_sliding_stride=8, selection_block_size=16, num_selected_blocks=2)


def _held(caches, rows):
    """The 8-bit cache that holds a prompt's keys and values, and nothing else."""
    from native_sparse_attention_pytorch_amd import ops
    (k, v), _ = caches
    made = ops.make_cache8(k.shape[0], k.shape[1], rows, k.shape[3])
    ops.cache8_append(made, k, v)
    return made


def _smaller(caches):
    """The same caches with keys and values of a 256th: a row of the usual size takes another scale by far."""
    (k, v), rest = caches
    return (k * 2. ** -8, v * 2. ** -8), rest


def _same(cache8, want):
    for got, expected in zip(cache8, want):
        places = (got.view(torch.uint8) != expected.view(torch.uint8)).sum().item()
        assert places == 0


@torch.no_grad()
@pytest.mark.parametrize("prompt", [1, 31, 32, 37, 63, 89])
def test_a_model_s_session_holds_the_prompt(prompt):
    from native_sparse_attention_pytorch_amd.decode_session import TransformerDecodeSession
    from native_sparse_attention_pytorch_amd.transformer import Transformer
    torch.manual_seed(prompt)
    model = Transformer(num_tokens=256, dim=128, depth=2, dim_head=64, heads=4, kv_heads=2, sparse_attn_kwargs=LAYER).to(DEV, BF16)
    _, caches = model(torch.randint(0, 256, (2, prompt), device=DEV), return_cache=True)
    caches = [_smaller(c) for c in caches]
    session = TransformerDecodeSession(model, caches, max_len=90, cache_dtype=FP8)
    for layer, cache in zip(session.layers, caches):
        assert layer.state.tolist() == [prompt, cache[1][0][0].shape[-2]] == [layer.pos, layer.nc]
        _same(layer.cache8, _held(cache, 90))
    # a step's row is the only one that a step adds
    token = torch.randint(0, 256, (2, 1), device=DEV)
    before = [[t.clone() for t in layer.cache8] for layer in session.layers]
    session.step(token)
    for layer, held in zip(session.layers, before):
        assert layer.state[0].item() == prompt + 1
        other = torch.arange(layer.cache8.keys.shape[2], device=DEV) // 32 != prompt // 32
        for got, want in zip(layer.cache8[:2], held[:2]):
            assert torch.equal(got.view(torch.uint8)[:, :, other], want.view(torch.uint8)[:, :, other])


@torch.no_grad()
@pytest.mark.parametrize("norm", ["its own", "one with a bias"])
@pytest.mark.parametrize("prompt", [37, 64])
def test_a_layer_s_session_holds_the_prompt(prompt, norm):
    """A norm of the caller's with a bias has rows that are not zero for the token of zeros that the session runs with."""
    from native_sparse_attention_pytorch_amd import SparseAttention
    from native_sparse_attention_pytorch_amd.decode_session import DecodeSession
    torch.manual_seed(prompt)
    m = SparseAttention(dim=128, dim_head=64, heads=4, kv_heads=2, causal=True, **LAYER).to(DEV, BF16)
    _, cache = m(torch.randn(3, prompt, 128, device=DEV, dtype=BF16), return_cache=True)
    if norm != "its own":
        m.norm = torch.nn.LayerNorm(128).to(DEV, BF16)
        m.norm.bias.normal_()
    cache = _smaller(cache)
    session = DecodeSession(m, cache, max_len=90, cache_dtype=FP8)
    _same(session.cache8, _held(cache, 90))
    assert session.state.tolist() == [prompt, session.nc]
    for t in range(3):
        session.step(torch.randn(3, 1, 128, device=DEV, dtype=BF16))
    assert session.state[0].item() == prompt + 3
