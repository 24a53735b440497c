"""Gates at the ends of their range in swiglu_projection: the definition's h = u g / (1 + e^-g) and its derivatives in 64
bits, infinities and NaN included. (silu(-inf) is -inf / inf, NaN; its derivative at either infinity is NaN too.)"""
import pytest
import torch

import attnres_b200 as A

pytestmark = pytest.mark.gpu

INF = float("inf")


def one_gate(N, value, gate, dtype):
    """u = value and g = gate in row 0 for every output; row 1 has u = 2, g = 1."""
    x = torch.zeros(N, 8, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = 2.0, 1.0
    x[0, 0], x[0, 1] = value, gate
    w = torch.zeros(16, 8, device="cuda", dtype=dtype)
    w[:8, 0], w[8:, 1] = 1.0, 1.0
    return x.requires_grad_(True), w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [4, 200])  # the streaming kernel, the tiles
@pytest.mark.parametrize("gate", [-INF, INF, float("nan"), -6e4, 6e4, -88.0, -87.5, 88.5, -20.0, 20.0])
def test_ends_of_the_range(gate, N, dtype):
    """An infinite or NaN x meets zero weights too (0 * inf is NaN), so u and h are NaN there in the definition as well;
    rows beside it are not touched. Finite gates: one rounding, and 2^-20 of fp32 arithmetic; results below 2^-126 may
    be zero."""
    x, w = one_gate(N, 3.0, gate, dtype)
    h = A.swiglu_projection(x, w)
    (dx,) = torch.autograd.grad(h, [x], torch.ones_like(h))
    u, g = (x.detach().double() @ w.double().t()).chunk(2, -1)
    s = torch.sigmoid(g)
    want, wx = u * g * s, torch.cat([g * s, u * s * (1 + g * (1 - s))], -1) @ w.double()
    r = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    finite = abs(gate) < INF
    for got, exact, terms in ((h.detach(), want, 1), (dx, wx, 8)):
        rows = slice(0 if finite else 1, None)
        a, b = got.double()[rows], exact[rows]
        beyond = b.abs() > torch.finfo(dtype).max  # float16 has no 3 * 6e4
        assert torch.equal(a[beyond], torch.copysign(torch.full_like(b[beyond], INF), b[beyond]))
        assert bool(((a - b).abs() <= 2 * terms * r * b.abs() + 2.0 ** -24 * terms)[~beyond].all())
        if not finite:
            assert bool(got[0, :1].isnan().all()) and bool(exact[0, :1].isnan().all())
    assert bool(h[1:].isfinite().all()) and bool(dx[1:].isfinite().all())


@pytest.mark.parametrize("N", [4, 200])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_gates_beside_finite_values(sign, N):
    """All weights non-zero, so that g = +-inf and u = +-inf alone: h is inf * inf, and NaN at -inf (inf * NaN)."""
    x = torch.ones(N, 8, device="cuda", dtype=torch.bfloat16)
    x[0, 3] = INF
    w = torch.full((16, 8), 0.5, device="cuda", dtype=torch.bfloat16)
    w[8:] *= sign
    h = A.swiglu_projection(x, w)
    u, g = (x.double() @ w.double().t()).chunk(2, -1)
    want = u * g / (1 + torch.exp(-g))
    assert torch.equal(h[0].isnan(), want[0].isnan()) and torch.equal(h[0].isinf(), want[0].isinf())
    assert bool(((h[1:].double() - want[1:]).abs() <= 2.0 ** -7 * want[1:].abs()).all())
