"""swiglu_projection on the GPU against a float64 composition of its definition.

Tolerances, for sums of K products of rounded inputs held in fp32: h is rounded
once, so |error| <= r |h| plus fp32 rounding of the two sums, 2^-20 sqrt(K) of their
scale (the root mean square of a product times sqrt(K)) through factors of order
one. The gradients also see du and dg rounded once: every term of their sums is off
by at most r of itself, so |error| <= r |value| + r * sqrt(sum of the squares of the
terms) * 4 (four standard deviations and more of independent roundings). r is 2^-8
for bf16 and 2^-11 for f16, twice the unit roundoff.
"""
import pytest
import torch

import attnres_b200 as A

pytestmark = pytest.mark.gpu

ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.bfloat16, torch.float16]


def inputs(N, C, F, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, C, device="cuda", generator=g).to(dtype)
    w = (torch.randn(2 * F, C, device="cuda", generator=g) / C ** 0.5).to(dtype)
    dh = torch.randn(N, F, device="cuda", generator=g).to(dtype)
    return x, w, dh


def definition(x, w, dh):
    """h, dx, dW in float64, and for the gradients the root of the sum of their terms' squares."""
    x, w, dh = x.double(), w.double(), dh.double()
    F = w.shape[0] // 2
    y = x @ w.t()
    u, g = y[:, :F], y[:, F:]
    s = torch.sigmoid(g)
    d = torch.cat([dh * g * s, dh * u * s * (1 + g * (1 - s))], 1)
    return (u * g * s, d @ w, d.t() @ x, ((d ** 2) @ (w ** 2)).sqrt(), ((d ** 2).t() @ (x ** 2)).sqrt())


def within(name, got, want, bound):
    assert got.shape == want.shape, name
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"{name}: {float((err - bound).max()):.3e} over the bound"


def check(x, w, dh, dtype):
    r = ROUND[dtype]
    h = A.swiglu_projection(x, w)
    dx, dw = torch.autograd.grad(h, [x, w], dh)
    want_h, want_dx, want_dw, sx, sw = definition(x.detach(), w.detach(), dh)
    assert h.dtype == dx.dtype == dtype and dw.dtype == w.dtype
    scale = 2.0 ** -20 * x.shape[-1] ** 0.5 * (1 + want_h.abs())
    within("h", h.detach(), want_h, r * want_h.abs() + scale)
    within("dx", dx, want_dx, r * want_dx.abs() + 4 * r * sx + 1e-6)
    within("dw", dw, want_dw, r * want_dw.abs() + 4 * r * sw + 1e-6)
    with torch.no_grad():
        assert torch.equal(A.swiglu_projection(x, w), h.detach())


SHAPES = [(1, 8, 8), (1, 1024, 4096), (7, 64, 128), (8, 72, 136), (9, 520, 24), (17, 256, 264), (32, 1024, 512),
          (33, 64, 128), (100, 136, 72), (128, 64, 128), (129, 200, 264), (300, 1024, 1000), (515, 776, 392),
          (1000, 8, 8), (2100, 1024, 2048)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_definition(shape, dtype):
    x, w, dh = inputs(*shape, dtype)
    check(x.requires_grad_(True), w.requires_grad_(True), dh, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [5, 70])
def test_strided_and_unaligned(N, dtype):
    x, w, dh = inputs(N, 128, 64, dtype)
    for off in (8, 3):  # aligned rows, and rows that have to be copied
        wide = torch.zeros(N, 128 + 24, device="cuda", dtype=dtype)
        wide[:, off:off + 128] = x
        ww = torch.zeros(128, 128 + 16, device="cuda", dtype=dtype)
        ww[:, off:off + 128] = w
        dd = torch.zeros(N, 64 + 16, device="cuda", dtype=dtype)
        dd[:, off:off + 64] = dh
        check(wide[:, off:off + 128].detach().requires_grad_(True), ww[:, off:off + 128].detach().requires_grad_(True),
              dd[:, off:off + 64], dtype)
    check(x.t().contiguous().t().requires_grad_(True), w.requires_grad_(True), dh, dtype)


def test_leading_dimensions_and_wide_weights():
    x, w, dh = inputs(6, 64, 32, torch.bfloat16)
    w32 = w.float().requires_grad_(True)
    x3 = x.view(2, 3, 64).requires_grad_(True)
    h = A.swiglu_projection(x3, w32)
    assert h.shape == (2, 3, 32)
    dx, dw = torch.autograd.grad(h, [x3, w32], dh.view(2, 3, 32))
    assert dx.shape == x3.shape and dw.dtype == torch.float32
    want = torch.autograd.grad(A.swiglu_projection(x.requires_grad_(True), w.requires_grad_(True)), [x, w], dh)
    assert torch.equal(dx.view(6, 64), want[0]) and torch.equal(dw, want[1].float())


@pytest.mark.parametrize("want", ["x", "w"])
def test_one_gradient_only(want):
    x, w, dh = inputs(200, 128, 64, torch.bfloat16)
    both = torch.autograd.grad(A.swiglu_projection(x.requires_grad_(True), w.requires_grad_(True)), [x, w], dh)
    leaf = (x if want == "x" else w).detach().requires_grad_(True)
    args = (leaf, w.detach()) if want == "x" else (x.detach(), leaf)
    (got,) = torch.autograd.grad(A.swiglu_projection(*args), [leaf], dh)
    assert torch.equal(got, both[0 if want == "x" else 1])


def test_gradient_of_a_sum():
    """The gradient of sum() is one value seen through strides of zero."""
    x, w, _ = inputs(40, 64, 32, torch.bfloat16)
    x.requires_grad_(True)
    (got,) = torch.autograd.grad(A.swiglu_projection(x, w).sum(), [x])
    (want,) = torch.autograd.grad(A.swiglu_projection(x, w), [x], torch.ones(40, 32, device="cuda", dtype=x.dtype))
    assert torch.equal(got, want)


def test_gradient_against_differences():
    """Central differences in float64 of the definition at the kernel's inputs, h = 1e-4: their own error is below
    1e-6 of the gradient's scale, the kernel's is a rounding to f16 and its two roundings' sums: 2^-9 in all."""
    x, w, dh = inputs(64, 128, 64, torch.float16)
    got = torch.autograd.grad(A.swiglu_projection(x.requires_grad_(True), w.requires_grad_(True)), [x, w], dh)

    def loss(a, b):
        y = a @ b.t()
        return (y[:, :64] * torch.nn.functional.silu(y[:, 64:]) * dh.double()).sum()

    gen = torch.Generator(device="cuda").manual_seed(1)
    a, b = x.detach().double(), w.detach().double()
    for i in range(2):
        for _ in range(3):
            d = torch.randn(got[i].shape, device="cuda", generator=gen).double()
            up = loss(a + 1e-4 * d, b) if i == 0 else loss(a, b + 1e-4 * d)
            down = loss(a - 1e-4 * d, b) if i == 0 else loss(a, b - 1e-4 * d)
            diff, want = float(up - down) / 2e-4, float((got[i].double() * d).sum())
            assert abs(diff - want) <= 2.0 ** -9 * float(got[i].double().norm() * d.norm())


@pytest.mark.parametrize("N", [4, 200])
def test_saturated_gates(N):
    """silu at +-200 and +-inf: no NaN where the definition has none."""
    for gate in (200.0, -200.0, 0.0):
        x = torch.zeros(N, 8, device="cuda", dtype=torch.bfloat16)
        x[:, 0], x[:, 1] = 1.0, gate
        w = torch.zeros(16, 8, device="cuda", dtype=torch.bfloat16)
        w[:8, 0], w[8:, 1] = 3.0, 1.0
        x.requires_grad_(True)
        h = A.swiglu_projection(x, w)
        want = 3.0 * torch.nn.functional.silu(torch.tensor(gate, dtype=torch.float64))
        assert bool(((h.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-30).all())
        (dx,) = torch.autograd.grad(h, [x], torch.ones_like(h))
        assert bool(torch.isfinite(dx).all())


def test_no_tokens():
    w = torch.ones(16, 8, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x = torch.empty(3, 0, 8, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    h = A.swiglu_projection(x, w)
    assert h.shape == (3, 0, 8)
    dx, dw = torch.autograd.grad(h.sum(), [x, w])
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


def test_repeats_bitwise_and_on_another_stream():
    x, w, dh = inputs(700, 256, 264, torch.bfloat16)
    x, w = x.requires_grad_(True), w.requires_grad_(True)

    def once():
        h = A.swiglu_projection(x, w)
        return (h.detach(), *torch.autograd.grad(h, [x, w], dh))

    want = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = once()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_op_traces_under_compile():
    x, w, dh = inputs(64, 128, 64, torch.bfloat16)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    want = A.swiglu_projection(*leaves)
    got = torch.compile(lambda a, b: A.swiglu_projection(a, b), fullgraph=True)(*leaves)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, dh), torch.autograd.grad(want, leaves, dh)):
        assert torch.equal(a, b)


def test_refusals():
    x, w, _ = inputs(4, 64, 32, torch.bfloat16)
    for bad in ((x.cpu(), w), (x, w.cpu()), (x.float(), w), (x.double(), w), (x, w[:, :56]), (x, w[:-1]),
                (x[:, :60], w[:, :60]), (x, w[:24]), (x, w[0])):
        with pytest.raises(RuntimeError):
            A.swiglu_projection(*bad)
    h = A.swiglu_projection(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(h, [x], torch.ones_like(h), create_graph=True)


def test_status_word_stays_clear():
    from attnres_b200 import _native

    assert _native.device_status() == 0
