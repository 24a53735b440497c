"""A model whose cached tokens cannot be attended to (float32, or heads that kv4_attention is not built for) says so
before it does any of the work or writes anything."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def model(dtype, **kw):
    from attnres_b200.gpt import GPT, GPTConfig

    torch.manual_seed(2)
    base = dict(n_layer=2, n_head=4, n_embd=256, vocab_size=61, block_size=32, lrid_rank=32, attnres_num_blocks=2)
    return GPT(GPTConfig(**{**base, **kw})).cuda().to(dtype).eval()


@pytest.mark.parametrize("dtype,kw", [(torch.float32, {}), (torch.bfloat16, dict(n_head=8)), (torch.bfloat16, dict(n_head=2, n_embd=192))])
def test_generate_refuses_before_the_prompt(dtype, kw):
    from attnres_b200.gpt import GPTCache

    m = model(dtype, **kw)
    idx = torch.randint(0, 61, (2, 5), device="cuda")
    calls = []
    m.transformer.wte.register_forward_hook(lambda *a: calls.append(1))
    with pytest.raises(RuntimeError, match="kv4_attention"):
        m.generate(idx, 2)
    assert not calls
    with torch.no_grad():
        want = m(idx)[:, -1].argmax(-1)
    assert torch.equal(m.generate(idx, 1)[:, 5], want)  # one token needs no cached ones
    cache = GPTCache(m.cfg, 2, 16)
    with torch.no_grad():
        m(idx, cache=cache)
        before = [[t.clone() for t in p.tensors()] for p in cache.pools]
        with pytest.raises(RuntimeError, match="kv4_attention"):
            m(idx[:, :1], cache=cache)
        with pytest.raises(RuntimeError, match="kv4_attention"):
            m.generate(idx[:, :1], 1, cache=cache)
    assert cache.used == 5
    for p, old in zip(cache.pools, before):
        for t, o in zip(p.tensors(), old):
            assert torch.equal(t.view(torch.uint8), o.view(torch.uint8))
