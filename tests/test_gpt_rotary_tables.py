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


# ---------------------------------------------------------------------------
# the buffers' values
# ---------------------------------------------------------------------------
def other_state(dtype=torch.float32):
    """The state of a model with another rotary base."""
    return model(rope_theta=777.0).to(dtype).state_dict()


@pytest.mark.parametrize("assign", [False, True])
def test_tables_follow_a_loaded_state(assign):
    m = model()
    m.load_state_dict(other_state(), assign=assign)
    for r in ropes(m):
        assert same(r.tables, (r.cos, r.sin)) and torch.equal(r.tables[0], ropes(model(rope_theta=777.0))[0].cos[0, 0])


def test_tables_follow_a_loaded_state_in_16_bits():
    m = model().to(torch.bfloat16)
    m.load_state_dict(other_state(torch.bfloat16))
    for r in ropes(m):
        assert same(r.tables, (r.cos, r.sin))


def test_tables_follow_writes_casts_and_copies():
    m = model()
    r = ropes(m)[0]
    exact = [t.clone() for t in r.tables]
    r.cos.fill_(1.0)  # as a broadcast of buffers from another rank writes them
    assert bool((r.tables[0] == 1).all()) and torch.equal(r.tables[1], exact[1])
    c = copy.deepcopy(m)
    assert bool((ropes(c)[0].tables[0] == 1).all())
    c.to(torch.bfloat16)
    assert bool((ropes(c)[0].tables[0] == 1).all()) and torch.equal(ropes(c)[0].tables[1], exact[1])
    r.cos = torch.zeros_like(r.cos)
    assert bool((r.tables[0] == 0).all())


def test_a_cast_keeps_the_full_precision_and_a_saved_state_repeats():
    a = model()
    exact = [t.clone() for t in ropes(a)[0].tables]
    a.to(torch.bfloat16)
    b = model().to(torch.bfloat16)
    b.load_state_dict(a.state_dict())
    for m in (a, b):
        assert all(torch.equal(x, y) for x, y in zip(ropes(m)[0].tables, exact))


def test_tables_under_inference_mode():
    with torch.inference_mode():
        m = model()
        assert same(ropes(m)[0].tables, (ropes(m)[0].cos, ropes(m)[0].sin))


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [False, True])
def test_fused_layer_and_cache_turn_as_the_unfused_layer_does(compiled):
    """Logits after loading a state of another rotary base: as close to the fp32 model's as the unfused layer's are."""
    from attnres_b200.gpt import GPTCache

    kw = dict(n_embd=512, n_head=4, lrid_rank=64, block_size=64, rope_theta=100000.0)
    torch.manual_seed(3)
    state = model(**{**kw, "rope_theta": 50.0}).state_dict()

    def loaded(dtype, **more):
        m = model(**kw, **more).cuda().to(dtype)
        m.load_state_dict(state)
        return m.eval()

    idx = torch.randint(0, KW["vocab_size"], (2, 64), device="cuda")
    with torch.no_grad():
        want = loaded(torch.float32, fused=False)(idx)
        plain = (loaded(torch.bfloat16)(idx).float() - want).norm()
        m = loaded(torch.bfloat16, fused_layer=True)
        run = torch.compile(m, fullgraph=True) if compiled else m
        assert float((run(idx).float() - want).norm()) <= 1.5 * float(plain)
        if not compiled:  # the prompt of a cached call is attended to in full precision
            assert float((m(idx, cache=GPTCache(m.cfg, 2, 64)).float() - want).norm()) <= 1.5 * float(plain)
            stale = model(**kw, fused_layer=True).cuda().to(torch.bfloat16)
            stale.load_state_dict({k: v for k, v in state.items() if "rope" not in k}, strict=False)
            assert float((stale.eval()(idx).float() - want).norm()) > 3 * float(plain)  # the bases do differ


def test_a_model_of_fake_tensors_runs_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    torch.set_default_dtype(torch.bfloat16)
    try:
        with FakeTensorMode(), torch.device("cuda"):
            m = model(fused_layer=True)
            assert m(torch.zeros(1, 4, dtype=torch.int64)).shape == (1, 4, KW["vocab_size"])
    finally:
        torch.set_default_dtype(torch.float32)
