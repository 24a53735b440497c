"""qk_norm_rope with norm weights of another type than the projection (a 16-bit projection under float32 weights is
what mixed-precision training has): the weights multiply as they are and their gradients come in their own type, not
by way of the projection's. Tolerances as in test_gpu_qk_rope, without the 16-bit rounding for the weights' gradients."""
import pytest
import torch

import attnres_b200 as A
from test_gpu_qk_rope import definition, inputs, near

pytestmark = pytest.mark.gpu

PAIRS = [(torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float32, torch.float32),
         (torch.bfloat16, torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16, torch.float16),
         (torch.float32, torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("dtype,tq,tk", PAIRS)
@pytest.mark.parametrize("shape", [(2, 37, 4, 4, 64), (1, 1, 6, 2, 128), (2, 9, 3, 1, 30), (3, 701, 6, 2, 64)])
@pytest.mark.parametrize("interleaved", [True, False])
def test_matches_definition(shape, dtype, tq, tk, interleaved):
    B, T, Hq, Hkv, D = shape
    qkv, _, grads, cos, sin, pos = inputs(*shape, dtype, weighted=False)
    g = torch.Generator(device="cuda").manual_seed(9)
    wq, wk = ((1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(t).requires_grad_(True) for t in (tq, tk))
    leaves = [qkv.requires_grad_(True), wq, wk]
    out = A.qk_norm_rope(qkv, Hq, Hkv, cos, sin, positions=pos, q_weight=wq, k_weight=wk, interleaved=interleaved)
    got = torch.autograd.grad(out, leaves, grads)
    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    want = definition(ref[0], Hq, Hkv, cos, sin, pos, ref[1], ref[2], interleaved=interleaved)
    wgrad = torch.autograd.grad(want, ref, [x.double() for x in grads])
    for name, a, b in zip(("q", "k", "v"), out, want):
        near(name, a.detach(), b, dtype)
    rows = (B, T, Hq + 2 * Hkv, D)
    near("dqkv", got[0].view(rows), wgrad[0].view(rows), dtype)
    for name, a, b, t, h in (("dwq", got[1], wgrad[1], tq, Hq), ("dwk", got[2], wgrad[2], tk, Hkv)):
        near(name, a, b, t, scale=float(B * T * h))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_step_too_small_for_16_bits_is_seen(dtype):
    """1 + 2^-11 has no 16-bit neighbour but 1 (bf16 and f16 both round it there)."""
    qkv, _, _, cos, sin, pos = inputs(1, 3, 2, 1, 64, torch.float32, weighted=False)
    w = torch.full((64,), 1 + 2.0 ** -11 / 1.5, device="cuda")
    x = qkv.to(dtype)
    # the plain 16-bit outputs differ in some elements once the weight is not rounded away
    q, _, _ = A.qk_norm_rope(x, 2, 1, cos, sin, positions=pos, q_weight=w)
    plain, _, _ = A.qk_norm_rope(x, 2, 1, cos, sin, positions=pos, q_weight=torch.ones_like(w))
    assert not torch.equal(q, plain)


def test_one_weight_only_and_no_tokens():
    qkv, _, grads, cos, sin, pos = inputs(2, 5, 4, 2, 64, torch.bfloat16, weighted=False)
    w = torch.rand(64, device="cuda").add_(0.5).requires_grad_(True)
    out = A.qk_norm_rope(qkv, 4, 2, cos, sin, positions=pos, k_weight=w)
    (got,) = torch.autograd.grad(out, [w], grads)
    ref = w.detach().double().requires_grad_(True)
    want = definition(qkv.double(), 4, 2, cos, sin, pos, None, ref)
    (wg,) = torch.autograd.grad(want[1], [ref], grads[1].double())
    near("dwk", got, wg, torch.float32, scale=float(2 * 5 * 2))
    out = A.qk_norm_rope(qkv[:, :0], 4, 2, cos, sin, k_weight=w)
    (got,) = torch.autograd.grad([o.sum() for o in out], [w], allow_unused=True)
    assert got.dtype == torch.float32 and bool((got == 0).all())


def test_traces_under_compile():
    qkv, _, grads, cos, sin, pos = inputs(2, 16, 4, 2, 64, torch.bfloat16, weighted=False)
    leaves = [qkv.requires_grad_(True), torch.rand(64, device="cuda").requires_grad_(True)]

    def f(x, a):
        return A.qk_norm_rope(x, 4, 2, cos, sin, positions=pos, q_weight=a)

    want, got = f(*leaves), torch.compile(f, fullgraph=True)(*leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(got, leaves, grads), torch.autograd.grad(want, leaves, grads)):
        assert a.dtype == b.dtype and torch.equal(a, b)
