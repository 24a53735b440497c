"""The rotary tables that the fused layer and the cache take follow the module: its device, and the sin and cos buffers
of the state that it holds."""
import copy

import pytest
import torch

KW = dict(n_layer=2, n_head=2, n_embd=128, vocab_size=33, block_size=16, lrid_rank=32)


def model(**kw):
    from attnres_b200.gpt import GPT, GPTConfig

    return GPT(GPTConfig(**{**KW, **kw}))


def ropes(m):
    return [layer.attn.rope for layer in m.transformer.layers]


def same(tables, buffers):
    return all(torch.equal(t, b[0, 0].float()) for t, b in zip(tables, buffers))


@pytest.mark.parametrize("fused_layer", [False, True])
def test_a_model_built_on_meta_is_materialised(fused_layer):
    whole = model()
    with torch.device("meta"):
        m = model(fused_layer=fused_layer)
    m.to_empty(device="cpu")
    m.load_state_dict(whole.state_dict())
    for a, b in zip(ropes(m), ropes(whole)):
        assert all(t.device.type == "cpu" and t.dtype == torch.float32 for t in a.tables)
        assert same(a.tables, (a.cos, a.sin)) and torch.equal(a.tables[0], b.tables[0])


def test_a_model_built_on_meta_takes_a_state_by_assignment():
    whole = model()
    with torch.device("meta"):
        m = model()
    m.load_state_dict(whole.state_dict(), assign=True)
    for r in ropes(m):
        assert all(t.device.type == "cpu" for t in r.tables) and same(r.tables, (r.cos, r.sin))


def test_built_on_meta_in_16_bits():
    """The buffers of a 16-bit state are the config's tables rounded: the layer's stay in full precision."""
    whole = model().to(torch.bfloat16)
    with torch.device("meta"):
        m = model().to(torch.bfloat16)
    m.to_empty(device="cpu")
    m.load_state_dict(whole.state_dict())
    exact = ropes(model())[0]
    for r in ropes(m):
        assert r.cos.dtype == torch.bfloat16 and same(r.tables, (exact.cos, exact.sin))


