"""qk_norm_rope on the GPU against a float64 composition of its definition.

Tolerances. The kernel computes in fp32 (a norm's sum over D terms, two products
and a sum per output: relative error below about 1e-5 of the row's largest
element for D <= 512) and rounds once: 2^-9 (bf16) / 2^-12 (f16) relative for the
outputs, doubled. Weight gradients add over tokens x heads in fp32: 1e-5 times
the sum of the terms' magnitudes, plus the output's rounding.
"""
import pytest
import torch

import attnres_b200 as A

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -23
ROUND = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def tables(rows, half, seed=0):
    g = torch.Generator().manual_seed(seed)
    angle = torch.rand(rows, half, generator=g, dtype=torch.float64) * 6.283
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def definition(qkv, Hq, Hkv, cos, sin, positions, wq, wk, normalize=True, interleaved=True, eps=EPS):
    """float64, on whatever device; differentiable."""
    B, T, width = qkv.shape
    D = width // (Hq + 2 * Hkv)
    x = qkv.view(B, T, Hq + 2 * Hkv, D)
    c, s = cos.double()[positions][:, :, None], sin.double()[positions][:, :, None]
    rot = 2 * cos.shape[1]
    out = []
    for part, w in ((x[:, :, :Hq], wq), (x[:, :, Hq:Hq + Hkv], wk)):
        y = part * torch.rsqrt((part ** 2).mean(-1, keepdim=True) + eps) if normalize else part
        if w is not None:
            y = y * w
        r, rest = y[..., :rot], y[..., rot:]
        a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
        u, v = a * c - b * s, a * s + b * c
        r = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
        out.append(torch.cat([r, rest], -1))
    return out[0], out[1], x[:, :, Hq + Hkv:]


def near(name, got, want, dtype, scale=None):
    """|got - want| <= 2 * rounding * |want| + 1e-5 * (the scale of what was summed)."""
    want = want.detach()
    bound = 2 * ROUND[dtype] * want.abs() + 1e-5 * (want.abs().amax(-1, keepdim=True) if scale is None else scale) + 1e-7
    err = (got.double() - want).abs()
    assert got.shape == want.shape and got.dtype == dtype, name
    assert bool((err <= bound).all()), f"{name}: {float((err - bound).max()):.3e} over the bound"


def inputs(B, T, Hq, Hkv, D, dtype, seed=0, rot=None, weighted=True, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(B, T, (Hq + 2 * Hkv) * D, device="cuda", generator=g) * std).to(dtype)
    w = [(1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(dtype) if weighted else None for _ in range(2)]
    grads = [torch.randn(B, T, h, D, device="cuda", generator=g).to(dtype) for h in (Hq, Hkv, Hkv)]
    cos, sin = tables(T + 11, (D if rot is None else rot) // 2, seed)
    pos = torch.randint(0, T + 11, (B, T), device="cuda", generator=g)
    return qkv, w, grads, cos, sin, pos


def check(B, T, Hq, Hkv, D, dtype, rot=None, weighted=True, interleaved=True, normalize=True, narrow=False):
    qkv, (wq, wk), grads, cos, sin, pos = inputs(B, T, Hq, Hkv, D, dtype, rot=rot, weighted=weighted)
    leaves = [qkv] + ([wq, wk] if weighted else [])
    for t in leaves:
        t.requires_grad_(True)
    out = A.qk_norm_rope(qkv, Hq, Hkv, cos, sin, positions=pos.to(torch.int32) if narrow else pos, q_weight=wq,
                         k_weight=wk, normalize=normalize, interleaved=interleaved)
    got = torch.autograd.grad(out, leaves, grads)
    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    want = definition(ref[0], Hq, Hkv, cos, sin, pos, *(ref[1:] if weighted else (None, None)), normalize=normalize,
                      interleaved=interleaved)
    wgrad = torch.autograd.grad(want, ref, [g.double() for g in grads])
    for name, a, b in zip(("q", "k", "v"), out, want):
        near(name, a.detach(), b, dtype)
    H, shape = Hq + 2 * Hkv, (B, T, Hq + 2 * Hkv, D)
    near("dqkv", got[0].view(shape), wgrad[0].view(shape), dtype)
    if weighted:
        for name, a, b, h in (("dwq", got[1], wgrad[1], Hq), ("dwk", got[2], wgrad[2], Hkv)):
            near(name, a, b, dtype, scale=float(B * T * h))  # |g xhat| is about 1
    return H


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("shape", [(2, 37, 4, 4, 64), (1, 1, 16, 16, 64), (3, 33, 6, 2, 128), (1, 5, 2, 1, 80),
                                   (2, 9, 3, 1, 30), (1, 7, 8, 1, 256), (1, 3, 1, 1, 512), (1, 70, 5, 3, 32)])
def test_matches_definition(shape, dtype, interleaved):
    check(*shape, dtype, interleaved=interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rot", [0, 2, 16, 32, 48])
@pytest.mark.parametrize("interleaved", [True, False])
def test_partial_rotation(rot, interleaved, dtype):
    check(2, 11, 4, 2, 64, dtype, rot=rot, interleaved=interleaved, narrow=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_norm_or_weights(dtype):
    check(2, 19, 4, 2, 64, dtype, weighted=False, normalize=False)
    check(2, 19, 4, 2, 64, dtype, weighted=False)
    check(2, 19, 4, 2, 64, dtype, weighted=True, normalize=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens(dtype):
    """More rows than one round of blocks: the weight sums go through several rows a block."""
    check(3, 701, 6, 2, 64, dtype)


def test_default_positions_count_each_sequence():
    qkv, _, _, cos, sin, _ = inputs(3, 13, 4, 2, 64, torch.float32, weighted=False)
    got = A.qk_norm_rope(qkv, 4, 2, cos, sin)
    pos = torch.arange(13, device="cuda").expand(3, 13)
    for a, b in zip(got, definition(qkv.double(), 4, 2, cos, sin, pos, None, None)):
        near("default positions", a, b, torch.float32)


def test_strided_inputs_and_gradients():
    qkv, _, _, cos, sin, pos = inputs(2, 21, 4, 2, 64, torch.bfloat16, weighted=False)
    wide = torch.randn(2, 21, 8 * 64 + 24, device="cuda", dtype=torch.bfloat16)
    for off in (0, 8, 5):  # 16-byte aligned rows, and rows that are not
        wide[..., off:off + 512] = qkv
        view = wide[..., off:off + 512].detach().requires_grad_(True)
        grads = [torch.randn(2, h, 21, 64, device="cuda", dtype=torch.bfloat16).transpose(1, 2) for h in (4, 2, 2)]
        out = A.qk_norm_rope(view, 4, 2, cos, sin, positions=pos)
        (got,) = torch.autograd.grad(out, [view], grads)
        ref = qkv.detach().double().requires_grad_(True)
        want = definition(ref, 4, 2, cos, sin, pos, None, None)
        (wg,) = torch.autograd.grad(want, [ref], [g.double() for g in grads])
        for a, b in zip(out, want):
            near("strided", a.detach(), b, torch.bfloat16)
        near("strided grad", got.view(2, 21, 8, 64), wg.view(2, 21, 8, 64), torch.bfloat16)
    rows = qkv[:1].expand(2, 21, 512)  # a batch that is one row read twice
    want = definition(rows.double(), 4, 2, cos, sin, pos, None, None)
    for a, b in zip(A.qk_norm_rope(rows, 4, 2, cos, sin, positions=pos), want):
        near("expanded", a, b, torch.bfloat16)


def test_gradients_of_some_outputs_only():
    """An output that takes no part in the loss has no gradient (None) and counts as zero."""
    qkv, _, grads, cos, sin, pos = inputs(2, 6, 4, 2, 64, torch.float32, weighted=False)
    qkv.requires_grad_(True)
    q, k, v = A.qk_norm_rope(qkv, 4, 2, cos, sin, positions=pos)
    (got,) = torch.autograd.grad((k * grads[1]).sum(), [qkv])
    ref = qkv.detach().double().requires_grad_(True)
    want = definition(ref, 4, 2, cos, sin, pos, None, None)
    (wg,) = torch.autograd.grad((want[1] * grads[1].double()).sum(), [ref])
    near("dqkv", got.view(2, 6, 8, 64), wg.view(2, 6, 8, 64), torch.float32)


def test_gradient_against_differences():
    """Central differences of a scalar of the fp32 kernel, h = 2^-7: error h^2/6 times a third derivative of order
    one plus 2 * 1e-6 / h of rounding over sums of 8 * 64 terms: 5e-3 of the gradient's scale."""
    qkv, (wq, wk), grads, cos, sin, pos = inputs(1, 1, 4, 2, 64, torch.float32)
    qkv, wq, wk = (t.requires_grad_(True) for t in (qkv, wq, wk))

    def loss(a, b, c):
        return sum((o.double() * g.double()).sum() for o, g in zip(
            A.qk_norm_rope(a, 4, 2, cos, sin, positions=pos, q_weight=b, k_weight=c), grads))

    got = torch.autograd.grad(loss(qkv, wq, wk), [qkv, wq, wk])
    g = torch.Generator(device="cuda").manual_seed(3)
    for i in range(3):
        for _ in range(4):
            d = torch.randn(got[i].shape, device="cuda", generator=g)
            args = [t.detach() for t in (qkv, wq, wk)]
            h = 2.0 ** -7
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + h * d, args[i] - h * d
            diff = float(loss(*up) - loss(*down)) / (2 * h)
            want = float((got[i].double() * d.double()).sum())
            assert abs(diff - want) <= 5e-3 * float(got[i].double().norm() * d.double().norm()), (i, diff, want)


def test_rows_of_zeros_and_large_values():
    cos, sin = tables(4, 32)
    for dtype in DTYPES:
        big = 3e4 if dtype == torch.float16 else 1e18
        qkv = torch.zeros(1, 3, 3 * 64, device="cuda", dtype=dtype)
        qkv[0, 1] = big
        qkv[0, 2] = -big
        qkv.requires_grad_(True)
        out = A.qk_norm_rope(qkv, 1, 1, cos, sin)
        pos = torch.arange(3, device="cuda")[None]
        want = definition(qkv.detach().double(), 1, 1, cos, sin, pos, None, None)
        for a, b in zip(out, want):
            near("extreme", a.detach(), b, dtype)
        assert all(bool(torch.isfinite(t).all()) for t in torch.autograd.grad([o.sum() for o in out], [qkv]))


def test_position_outside_the_tables_is_nan_and_reads_nothing():
    qkv, _, grads, cos, sin, _ = inputs(1, 4, 2, 1, 64, torch.bfloat16, weighted=False)
    rows = cos.shape[0]
    pos = torch.tensor([[0, -1, rows, rows - 1]], device="cuda")
    qkv.requires_grad_(True)
    q, k, v = A.qk_norm_rope(qkv, 2, 1, cos, sin, positions=pos)
    bad = torch.tensor([False, True, True, False], device="cuda")
    for t in (q, k):
        assert torch.equal(t.isnan().all(-1).all(-1)[0], bad) and torch.equal(t.isnan().any(-1).any(-1)[0], bad)
    assert torch.equal(v.flatten(), qkv.detach()[..., 3 * 64:].flatten())
    (g,) = torch.autograd.grad([q, k, v], [qkv], grads)
    assert torch.equal(g.view(1, 4, 4, 64).isnan().any(-1)[0, :, :3].any(-1), bad)
    assert not bool(g.view(1, 4, 4, 64)[:, :, 3].isnan().any())


def test_no_tokens():
    cos, sin = tables(4, 32)
    for shape in ((0, 5, 256), (2, 0, 256)):
        qkv = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(64, device="cuda", requires_grad=True)
        out = A.qk_norm_rope(qkv, 2, 1, cos, sin, q_weight=w)
        assert out[0].shape == (*shape[:2], 2, 64)
        g = torch.autograd.grad([o.sum() for o in out], [qkv, w])
        assert g[0].shape == shape and torch.equal(g[1], torch.zeros_like(w))


def test_weight_gradients_repeat_bitwise():
    qkv, (wq, wk), grads, cos, sin, pos = inputs(3, 333, 6, 2, 128, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (qkv, wq, wk)]

    def once():
        out = A.qk_norm_rope(qkv, 6, 2, cos, sin, positions=pos, q_weight=wq, k_weight=wk)
        return torch.autograd.grad(out, leaves, grads)

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


def test_runs_on_the_current_stream():
    qkv, _, _, cos, sin, pos = inputs(2, 64, 4, 2, 64, torch.bfloat16, weighted=False)
    want = A.qk_norm_rope(qkv, 4, 2, cos, sin, positions=pos)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        late = qkv.clone()
        for _ in range(20):
            late = late + 0
        got = A.qk_norm_rope(late, 4, 2, cos, sin, positions=pos)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_op_traces_under_compile():
    qkv, (wq, wk), grads, cos, sin, pos = inputs(2, 16, 4, 2, 64, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (qkv, wq, wk)]

    def f(x, a, b):
        q, k, v = A.qk_norm_rope(x, 4, 2, cos, sin, positions=pos, q_weight=a, k_weight=b)
        return q, k, v

    want = f(*leaves)
    got = torch.compile(f, fullgraph=True)(*leaves)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(got, leaves, grads), torch.autograd.grad(want, leaves, grads)):
        assert torch.equal(a, b)


def test_second_derivative_is_refused():
    qkv, _, grads, cos, sin, pos = inputs(1, 4, 2, 1, 64, torch.float32, weighted=False)
    out = A.qk_norm_rope(qkv.requires_grad_(True), 2, 1, cos, sin, positions=pos)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(out, [qkv], grads, create_graph=True)


def test_refusals():
    cos, sin = tables(8, 32)
    qkv = torch.zeros(1, 4, 4 * 64, device="cuda")
    for bad in (dict(qkv=qkv.cpu()), dict(qkv=qkv[0]), dict(qkv=qkv[..., :-1]), dict(qkv=qkv.double()),
                dict(num_heads=0), dict(cos=cos[:, :-1]), dict(cos=cos.double(), sin=sin.double()),
                dict(cos=cos[:3], sin=sin[:3]), dict(positions=torch.zeros(1, 3, device="cuda", dtype=torch.int64)),
                dict(positions=torch.zeros(1, 4, device="cuda")), dict(q_weight=torch.ones(63, device="cuda")),
                dict(cos=torch.zeros(8, 33, device="cuda"), sin=torch.zeros(8, 33, device="cuda")),
                dict(qkv=torch.zeros(1, 4, 4 * 514, device="cuda"))):
        kw = dict(qkv=qkv, num_heads=2, num_kv_heads=1, cos=cos, sin=sin)
        kw.update(bad)
        with pytest.raises(RuntimeError):
            A.qk_norm_rope(**kw)
