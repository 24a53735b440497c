"""GPT and its blocks as their callers have them, on the CPU."""
import pytest
import torch
from torch import nn

KW = dict(n_layer=2, n_head=2, n_embd=128, vocab_size=33, block_size=32, lrid_rank=32)


def model(**kw):
    from attnres_b200.gpt import GPT, GPTConfig

    return GPT(GPTConfig(**{**KW, **kw}))


def test_generate_refuses_what_does_not_fit_before_it_works():
    from attnres_b200.gpt import GPTCache

    m = model().to(torch.bfloat16)
    calls = []
    m.transformer.wte.register_forward_hook(lambda *a: calls.append(1))
    cache = GPTCache(m.cfg, 1, 12, page_size=16, device="cpu")
    idx = torch.zeros(1, 8, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="do not fit"):
        m.generate(idx, 6, cache=cache)  # 8 and 5 more; the last choice is not written
    with pytest.raises(RuntimeError, match="positions"):
        m.generate(idx, 26)
    assert not calls and cache.used == 0


def test_blocks_call_their_attention_as_before():
    """An attention module that takes the hidden states alone, as the reference's does, still fits into a block."""
    from attnres_b200.gpt import Block, GPTConfig

    class Plain(nn.Module):
        def forward(self, x):
            return 2 * x, x[..., :32]

    block = Block(GPTConfig(**KW))
    block.attn = Plain()
    x = torch.randn(1, 3, 128)
    seen = []
    block.attn.register_forward_pre_hook(lambda module, args: seen.append(len(args)))
    out, key = block.forward_attention(x, x_is_normalized=True)
    assert out.shape == x.shape and key.shape == (1, 3, 32) and seen == [1]


def test_a_model_calls_its_blocks_as_before():
    m = model(fused=False)
    idx = torch.randint(0, 33, (2, 7))
    want = m(idx)
    for block in m.transformer.layers:
        of = type(block).forward_attention
        block.forward_attention = lambda x, x_is_normalized=False, block=block, of=of: of(block, x, x_is_normalized)
    assert torch.equal(m(idx), want)
