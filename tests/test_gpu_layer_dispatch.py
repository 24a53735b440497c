"""The layer operators under what watches or transforms PyTorch's operators: traces hold the calls rather than their
results, dispatch modes see them, and a derivative that does not exist is an error rather than a zero."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import attnres_b200 as A

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rope_inputs(seed=0):
    angle = torch.rand(9, 32, device="cuda", generator=gen(7)) * 6
    return torch.randn(2, 9, 4 * 64, device="cuda", generator=gen(seed)).to(torch.bfloat16), angle.cos(), angle.sin()


def kv_inputs(seed=0):
    cache = A.KV4Cache.empty(2, 16, 2, 64)
    for t in cache.tensors():
        t.zero_()
    table, n = torch.arange(2, device="cuda", dtype=torch.int32)[:, None], torch.full((2,), 5, device="cuda", dtype=torch.int32)
    k = torch.randn(2, 5, 2, 64, device="cuda", generator=gen(seed)).to(torch.bfloat16)
    A.kv4_append(cache, k, k, table, n - 5)
    return cache, table, n, k


def calls():
    """name -> (function of one tensor, that tensor for a seed)"""
    _, cos, sin = rope_inputs()
    w = (torch.randn(32, 64, device="cuda", generator=gen(3)) / 8).to(torch.bfloat16)
    cache, table, n, _ = kv_inputs()

    def append(k):
        A.kv4_append(cache, k, k, table, n - 5)
        return A.kv4_read(cache, table, n - 5, 5)[0]

    return {
        "qk_norm_rope": (lambda x: A.qk_norm_rope(x, 2, 1, cos, sin)[0], lambda s: rope_inputs(s)[0]),
        "swiglu_projection": (lambda x: A.swiglu_projection(x, w),
                              lambda s: torch.randn(6, 64, device="cuda", generator=gen(s)).to(torch.bfloat16)),
        "kv4_attention": (lambda x: A.kv4_attention(x, cache, table, n),
                          lambda s: torch.randn(2, 1, 4, 64, device="cuda", generator=gen(s)).to(torch.bfloat16)),
        "kv4_append": (append, lambda s: kv_inputs(s)[3]),
    }


NAMES = ["qk_norm_rope", "swiglu_projection", "kv4_attention", "kv4_append"]


@pytest.mark.parametrize("name", NAMES)
def test_symbolic_trace_holds_the_call(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    f, make = calls()[name]
    graph = make_fx(f)(make(1))
    assert any(name in str(node.target) for node in graph.graph.nodes)
    got = graph(make(2))
    assert torch.equal(got, f(make(2))) and not torch.equal(got, f(make(1)))


@pytest.mark.parametrize("name", NAMES)
def test_jit_trace_holds_the_call(name):
    f, make = calls()[name]
    traced = torch.jit.trace(f, (make(1),), check_trace=False)
    got = traced(make(2))
    assert torch.equal(got, f(make(2))) and not torch.equal(got, f(make(1)))


@pytest.mark.parametrize("name", NAMES)
def test_dispatch_modes_see_the_call(name):
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    f, make = calls()[name]
    x = make(1)
    with Watch():
        got = f(x)
    assert any(f"attnres.{name}" in s for s in seen) and torch.equal(got, f(x))


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    import torch.autograd.forward_ad as fwd

    f, make = calls()[name]
    x = make(1)
    with fwd.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(fwd.make_dual(x, torch.ones_like(x)))
        f(x)  # no tangent: fine
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("which", ["qk_norm_rope", "swiglu_projection"])
def test_checkpointed_gradients(which):
    """Recomputation under a policy runs below a dispatch mode and gives the same gradients."""
    from torch.utils.checkpoint import checkpoint

    f, make = calls()[which]
    x = make(1).requires_grad_(True)
    (want,) = torch.autograd.grad(f(x).float().square().sum(), [x])
    (got,) = torch.autograd.grad(checkpoint(f, x, use_reentrant=False).float().square().sum(), [x])
    assert torch.equal(got, want)
