"""Sampling at a temperature draws from the model's distribution, over the share of the vocabulary that is kept."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("thres, kept", [(0., 64), (0.9, 7)])
def test_tokens_come_as_often_as_they_are_likely(thres, kept):
    from native_sparse_attention_pytorch_amd.transformer import Transformer
    torch.manual_seed(1)
    model = Transformer(num_tokens=64, dim=64, depth=1, dim_head=64, heads=1).to("cuda", torch.bfloat16)
    n, prompt = 4000, torch.randint(0, 64, (1, 9), device="cuda")
    logits = model(prompt.expand(n, 9).contiguous())[0, -1].float() / 0.7
    low = logits.topk(kept).values[-1]
    p = torch.softmax(logits.masked_fill(logits < low, -torch.inf), 0)
    drawn = model.sample(prompt.expand(n, 9).contiguous(), 10, temperature=0.7, filter_thres=thres)
    often = torch.bincount(drawn.flatten(), minlength=64).float()
    # six deviations of each count: 64 of them stray so far once in 10^7 times
    assert ((often - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt() + 1e-3).all()
    assert (often > 0).sum() > kept // 2
