"""The 4-bit cache on the GPU: kv4_append / kv4_read against the quantiser's definition,
kv4_attention against a float64 softmax over the values that the cache stands for.

Tolerances of the attention, with r = 2^-8 for bf16 and 2^-11 for f16 outputs. Weights and
values are rounded to f16 before they are multiplied, which leaves each term of the
output's sum within r of itself; the roundings are independent, so four times r times the
root of the sum of the terms' squares bounds their sum. The output is rounded once. The fp32
sums behind a score leave it off by less than 2^-13 at these sizes (sums of up to 128
products of |q| <= 5 with codes up to 15, times a step below 1 and the scale), which moves
the output by 2^-12 of the weighted sum of |v| at most.
"""
import pytest
import torch

import attnres_b200 as A
from attnres_b200 import _native

pytestmark = pytest.mark.gpu

ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def quantise(x):
    """(step, low, code) of groups of 32, in x's precision."""
    g = x.unflatten(-1, (-1, 32))
    step = ((g.amax(-1) - g.amin(-1)) * (1.0 / 15.0)).half().to(x.dtype)[..., None]
    low = g.amin(-1).half().to(x.dtype)[..., None]
    code = torch.where(step > 0, ((g - low) / step).round().clamp(0, 15), torch.zeros_like(g))
    return step, low, code


def values(x):
    step, low, code = quantise(x)
    return (low + step * code).flatten(-2)


def dirty(pages, page, heads, D):
    """A pool whose places hold what the worst owner before could have left: NaN, inf, any code."""
    cache = A.KV4Cache.empty(pages, page, heads, D)
    g = gen(9)
    for t in cache.tensors():
        if t.dtype == torch.uint8:
            t.random_(0, 256, generator=g)
        else:
            t.copy_(torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").repeat(t.numel() // 3 + 1)[
                :t.numel()].view(t.shape))
    return cache


def table_of(B, per, pages, seed=0):
    return torch.randperm(pages, generator=gen(seed), device="cuda")[:B * per].view(B, per).to(torch.int32)


def ints(*v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


# ---------------------------------------------------------------------------
# writing and reading
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 64, 16), (3, 37, 2, 128, 16), (2, 130, 5, 64, 64), (2, 5, 3, 32, 32),
                                   (1, 70, 1, 96, 16), (1, 3, 2, 512, 16), (5, 1, 16, 64, 128)])
def test_append_then_read(shape, dtype):
    B, T, H, D, page = shape
    start = ints(*[(7 * b) % 23 for b in range(B)])
    per = -(-(22 + T) // page)
    cache, table = dirty(B * per + 2, page, H, D), table_of(B, per, B * per + 2)
    g = gen(1)
    k = (torch.randn(B, T, H, D, device="cuda", generator=g) * 3 + 1).to(dtype)
    v = torch.randn(B, T, H, D, device="cuda", generator=g).to(dtype)
    before = [t.clone() for t in cache.tensors()]
    A.kv4_append(cache, k, v, table, start)
    for x, y in zip((k, v), A.kv4_read(cache, table, start, T, dtype=torch.float32)):
        assert torch.equal(y, values(x.float()))
        step, low, _ = quantise(x.double())
        off = (y.double() - x.double()).unflatten(-1, (-1, 32)).abs()
        assert bool((off <= 0.5 * step * (1 + 2.0 ** -10) + 2.0 ** -10 * (low.abs() + 15 * step)).all())
    for x, y in zip((k, v), A.kv4_read(cache, table, start, T, dtype=dtype)):
        assert y.dtype == dtype and torch.equal(y, values(x.float()).to(dtype))
    # nothing else was touched
    at = start.long()[:, None] + torch.arange(T, device="cuda")
    pg, place = torch.gather(table.long(), 1, at // page), at % page
    for t, old in zip(cache.tensors(), before):
        old[pg, :, place] = t[pg, :, place]
        assert torch.equal(t.view(torch.uint8), old.view(torch.uint8))


def test_ties_and_constant_groups():
    x = torch.zeros(1, 4, 1, 64, device="cuda")
    x[0, 0, 0, :32] = torch.arange(32, device="cuda") * 0.5            # every second value is a tie: 15.5 / 15 a step
    x[0, 1, 0, :32] = torch.linspace(0, 15, 31, device="cuda").repeat(2)[:32]  # steps of 1, ties at halves
    x[0, 2] = 2.5                                                         # constant
    x[0, 3, 0, 0] = 1e-9                                                  # a step that underflows
    cache, table = dirty(1, 16, 1, 64), ints(0)[None]
    A.kv4_append(cache, x, x, table, ints(0))
    for y in A.kv4_read(cache, table, ints(0), 4, dtype=torch.float32):
        assert torch.equal(y, values(x))


def test_near_ties_follow_the_division():
    """Many random quotients within 1e-5 of a tie: the codes are those of the IEEE division."""
    g = gen(5)
    n = torch.randint(0, 15, (1, 512, 1, 64), device="cuda", generator=g)
    near = (torch.rand(n.shape, device="cuda", generator=g) - 0.5) * 2e-5
    step = (torch.rand(1, 512, 1, 2, 1, device="cuda", generator=g) + 0.5).half().float()
    x = ((n + 0.5 + near).unflatten(-1, (2, 32)) * step)
    x[..., 0], x[..., 1] = 0.0, (15 * step)[..., 0]
    x = x.flatten(-2)
    cache, table = dirty(32, 16, 1, 64), torch.arange(32, device="cuda", dtype=torch.int32)[None]
    A.kv4_append(cache, x, -x, table, ints(0))
    for a, y in zip((x, -x), A.kv4_read(cache, table, ints(0), 512, dtype=torch.float32)):
        assert torch.equal(y, values(a))


def test_infinity_and_nan_stay_in_their_group():
    x = torch.randn(1, 3, 2, 64, device="cuda", generator=gen(2))
    for i, bad in enumerate((float("nan"), float("inf"), -float("inf"))):
        x[0, i, 1, 40] = bad
    cache, table = dirty(1, 16, 2, 64), ints(0)[None]
    A.kv4_append(cache, x, x, table, ints(0))
    for y in A.kv4_read(cache, table, ints(0), 3, dtype=torch.float32):
        assert bool(y[:, :, 1, 32:].isnan().all())
        clean = x.clone()
        clean[:, :, 1, 32:] = 0
        assert torch.equal(y[:, :, 1, :32], values(clean)[:, :, 1, :32]) and torch.equal(y[:, :, 0], values(clean)[:, :, 0])


def test_counts_and_missing_pages():
    B, T, H, D, page = 4, 20, 2, 64, 16
    cache, table = dirty(9, page, H, D), table_of(B, 2, 9)
    table[2, 1], table[3, 0] = -1, 9  # no page; a page the pool does not have
    k, v = (torch.randn(B, T, H, D, device="cuda", generator=gen(i)) for i in (1, 2))
    counts, start = ints(20, 0, 20, 3), ints(5, 3, 0, 0)
    before = [t.clone() for t in cache.tensors()]
    _native.device_status(reset=True)
    A.kv4_append(cache, k, v, table, start, counts)
    assert _native.device_status(reset=True) == 8
    got = A.kv4_read(cache, table, start, T, counts, dtype=torch.float32)
    assert _native.device_status(reset=True) == 8
    there = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    there[0], there[2, :16] = True, True
    for x, y in zip((k, v), got):
        want = torch.where(there[..., None, None], values(x), torch.zeros_like(x))
        assert torch.equal(y, want)
    at = start.long()[:, None] + torch.arange(T, device="cuda")
    pg, place = table.long().clamp(0, 8).gather(1, (at // page).clamp(max=1)), at % page
    for t, old in zip(cache.tensors(), before):
        old[pg[there], :, place[there]] = t[pg[there], :, place[there]]
        assert torch.equal(t.view(torch.uint8), old.view(torch.uint8))
    A.kv4_append(cache, k, v, table, ints(-1, 40, 32, 32), ints(1, 1, 1, 1))  # before the first and past the last place
    assert _native.device_status(reset=True) == 8
    for t, old in zip(cache.tensors(), before):
        assert torch.equal(t.view(torch.uint8), old.view(torch.uint8))


def test_strided_keys():
    B, T, H, D = 2, 9, 4, 64
    wide = torch.randn(B, H, T, D + 8, device="cuda", generator=gen(3)).to(torch.bfloat16)
    table, start = table_of(B, 1, 2), ints(0, 3)
    for off in (0, 8, 3):
        x = wide[..., off:off + D].transpose(1, 2)
        cache = dirty(2, 16, H, D)
        A.kv4_append(cache, x, x.contiguous(), table, start)
        k, v = A.kv4_read(cache, table, start, T, dtype=torch.float32)
        assert torch.equal(k, v) and torch.equal(k, values(x.float()))


def test_documented_layout():
    """One row, element by element, from the bytes as include/attnres_b200.h lays them out."""
    D, G = 128, 4
    x = torch.randn(1, 1, 1, D, device="cuda", generator=gen(4))
    cache = dirty(1, 16, 1, D)
    A.kv4_append(cache, x, x, ints(0)[None], ints(5))
    step, low, code = (t[0, 0, 0].cpu() for t in quantise(x))
    kc, vc = cache.k_codes[0, 0, 5].cpu(), cache.v_codes[0, 0, 5].cpu()
    for e in range(D):
        g, i = e // 32, e % 32
        byte = 4 * ((i // 8) * G + g) + (i % 8) // 2
        assert (int(kc[byte]) >> (4 * (i % 2))) & 15 == int(code[g, i])
        byte = 2 * ((i // 4) * G + g) + (i % 4) // 2
        assert (int(vc[byte]) >> (4 * (i % 2))) & 15 == int(code[g, i])
    for p in (cache.k_params, cache.v_params):
        assert torch.equal(p[0, 0, 5].float().cpu(), torch.cat([step, low], -1))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def filled(lengths, H, D, page, dtype, seed=0, std=1.0):
    """A pool in which each sequence's places hold random keys and values, the rest NaN; K, V as they read back."""
    B, longest = len(lengths), max(max(lengths), 1)
    per = -(-longest // page)
    cache, table = dirty(B * per + 1, page, H, D), table_of(B, per, B * per + 1, seed)
    g = gen(seed)
    k = (torch.randn(B, longest, H, D, device="cuda", generator=g) * std).to(dtype)
    v = torch.randn(B, longest, H, D, device="cuda", generator=g).to(dtype)
    n = ints(*lengths)
    A.kv4_append(cache, k, v, table, torch.zeros_like(n), n)
    return cache, table, n, values(k.float()).double(), values(v.float()).double()


def definition(q, K, V, lengths, counts, scale):
    """out, lse, and the two sums of the bound, in float64."""
    B, T, Hq, D = q.shape
    group = Hq // K.shape[2]
    K, V = (x.repeat_interleave(group, 2).transpose(1, 2) for x in (K, V))
    z = q.double().transpose(1, 2) @ K.transpose(-1, -2) * scale
    n, c = (torch.tensor(x, device="cuda")[:, None, None] for x in (lengths, counts))
    t, j = torch.arange(T, device="cuda")[None, :, None], torch.arange(K.shape[2], device="cuda")
    see = ((j <= n - c + t) & (t < c))[:, None].expand(B, Hq, T, -1)
    z = z.masked_fill(~see, -float("inf"))
    lse = z.logsumexp(-1)
    p = torch.where(see, torch.exp(z - torch.where(lse == -float("inf"), torch.zeros_like(lse), lse)[..., None]),
                    torch.zeros_like(z))
    V = torch.where(see.any(2)[..., None], V, torch.zeros_like(V))
    swap = lambda x: x.transpose(1, 2)  # noqa: E731
    return swap(p @ V), swap(lse), swap(((p ** 2) @ (V ** 2)).sqrt()), swap(p @ V.abs())


def check(lengths, T, Hq, H, D, page, dtype, counts=None, seed=0, std=1.0):
    cache, table, n, K, V = filled(lengths, H, D, page, dtype, seed, std)
    q = torch.randn(len(lengths), T, Hq, D, device="cuda", generator=gen(seed + 50)).to(dtype)
    _native.device_status(reset=True)
    out, lse = A.kv4_attention(q, cache, table, n, None if counts is None else ints(*counts), return_lse=True)
    assert _native.device_status() == 0
    compare(out, lse, definition(q, K, V, lengths, counts or [T] * len(lengths), D ** -0.5), dtype)
    return cache, table, n, q, out


def compare(out, lse, want, dtype):
    r = ROUND[dtype]
    o, z, square, weight = want
    assert out.shape == o.shape and out.dtype == dtype and lse.dtype == torch.float32
    empty = z == -float("inf")
    assert torch.equal(lse == -float("inf"), empty) and bool((out[empty] == 0).all())
    err = (out.double() - o).abs()
    bound = r * o.abs() + 4 * r * square + 2.0 ** -12 * weight + 1e-9
    assert bool((err <= bound).all()), f"out: {float((err - bound).max()):.3e} over the bound"
    assert bool(((lse.double() - z)[~empty].abs() <= 2.0 ** -12).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("shape", [((1,), 1, 1, 1), ((300,), 1, 16, 16), ((33, 1, 64, 129), 1, 8, 2),
                                   ((500, 17, 0, 4), 3, 6, 2), ((77, 40), 2, 12, 1), ((1000, 31, 32), 1, 24, 8),
                                   ((200, 5), 5, 8, 8), ((130, 260), 9, 4, 2)])
def test_attention_matches_definition(shape, page, D, dtype):
    lengths, T, Hq, H = shape
    check(list(lengths), T, Hq, H, D, page, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_many_lengths(dtype):
    check(list(range(0, 140)), 1, 2, 1, 64, 48, dtype)
    check(list(range(0, 70)), 4, 2, 2, 128, 16, dtype)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_long(D):
    """Several stretches, joined; 70 000 places."""
    check([70001, 9, 12345], 1, 4, 2, D, 64, torch.bfloat16)
    check([20000], 3, 8, 1, D, 128, torch.float16)


def test_attention_counts():
    check([40, 7, 9, 3], 6, 4, 2, 64, 16, torch.bfloat16, counts=[6, 0, 1, 5])
    check([300, 0, 260], 3, 16, 2, 128, 32, torch.float16, counts=[2, 3, 1])


def test_attention_large_scores():
    """Scores in the hundreds: one key takes the whole weight."""
    check([500, 33], 1, 4, 2, 64, 16, torch.bfloat16, std=0.0)  # and all scores equal
    cache, table, n, K, V = filled([500], 2, 64, 16, torch.bfloat16, std=30.0)
    q = (torch.randn(1, 1, 4, 64, device="cuda", generator=gen(3)) * 4).to(torch.bfloat16)
    out = A.kv4_attention(q, cache, table, n)
    z = torch.einsum("bthd,bjhd->bthj", q.double(), K.repeat_interleave(2, 2)) / 8
    top2 = z.topk(2, -1).values
    assert bool((top2[..., 0] > 100).all())
    sure = top2[..., 0] - top2[..., 1] > 30
    want = torch.gather(V.repeat_interleave(2, 2).transpose(1, 2), 2, z.argmax(-1).transpose(1, 2)[..., None].expand(1, 4, 1, 64))
    err = (out.transpose(1, 2).double() - want).abs()
    assert bool((err[sure.transpose(1, 2)] <= 2.0 ** -6 * (want.abs()[sure.transpose(1, 2)] + 1)).all())


def test_attention_ignores_what_it_may_not_see():
    """A later token's NaN key and value leave the earlier tokens' rows alone and reach its own."""
    B, T, H, D, page = 1, 3, 2, 64, 16
    lengths = [50]
    cache, table, n, K, V = filled(lengths, H, D, page, torch.bfloat16)
    bad = torch.full((1, 1, H, D), float("nan"), device="cuda")
    A.kv4_append(cache, bad, bad, table, ints(49))
    q = torch.randn(B, T, H, D, device="cuda", generator=gen(8)).to(torch.bfloat16)
    out = A.kv4_attention(q, cache, table, n)
    o, _, square, weight = definition(q[:, :2], K[:, :49], V[:, :49], [49], [2], D ** -0.5)
    err = (out[:, :2].double() - o).abs()
    assert bool((err <= 2.0 ** -8 * (o.abs() + 4 * square) + 2.0 ** -12 * weight).all())
    assert bool(out[:, 2].isnan().all())


def test_attention_missing_page_counts_as_empty():
    cache, table, n, K, V = filled([64, 40], 1, 64, 16, torch.bfloat16)
    table[0, 1] = -1
    table[1, 2] = 1 << 20
    q = torch.randn(2, 1, 2, 64, device="cuda", generator=gen(8)).to(torch.bfloat16)
    _native.device_status(reset=True)
    out, lse = A.kv4_attention(q, cache, table, n, return_lse=True)
    assert _native.device_status(reset=True) == 8
    keep = [torch.cat([x[:1, :16], x[:1, 32:64]], 1) for x in (K, V)]
    compare(out[:1], lse[:1], definition(q[:1], *keep, [48], [1], 0.125), torch.bfloat16)
    compare(out[1:], lse[1:], definition(q[1:], K[1:, :32], V[1:, :32], [32], [1], 0.125), torch.bfloat16)


def test_attention_lengths_beyond_the_table_are_clipped():
    cache, table, n, K, V = filled([64], 1, 64, 16, torch.bfloat16)
    q = torch.randn(1, 1, 2, 64, device="cuda", generator=gen(8)).to(torch.bfloat16)
    assert torch.equal(A.kv4_attention(q, cache, table, ints(1000)), A.kv4_attention(q, cache, table, n))
    assert bool((A.kv4_attention(q, cache, table, ints(-5)) == 0).all())
    assert bool((A.kv4_attention(q, cache, table[:, :0], n) == 0).all())


def test_attention_strided_queries_and_scale():
    cache, table, n, q, out = check([90, 20], 2, 4, 2, 64, 16, torch.bfloat16)
    wide = torch.zeros(2, 4, 2, 64 + 3, device="cuda", dtype=torch.bfloat16)
    for off in (0, 3):
        wide[..., off:off + 64] = q.transpose(1, 2)
        assert torch.equal(A.kv4_attention(wide[..., off:off + 64].transpose(1, 2), cache, table, n), out)
    flat = A.kv4_attention(q, cache, table, n, scale=0.0)
    _, v = A.kv4_read(cache, table, ints(0, 0), 90, n, dtype=torch.float32)
    want = v[0, :89].double().mean(0)
    assert bool(((flat[0, 0].double() - want.repeat_interleave(2, 0)).abs() <= 2.0 ** -8 * (want.abs().repeat_interleave(2, 0) + 0.5)).all())


def test_attention_repeats_bitwise_and_on_another_stream():
    cache, table, n, q, out = check([5000, 12, 700], 1, 8, 2, 128, 64, torch.bfloat16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = A.kv4_attention(q, cache, table, n)
    side.synchronize()
    assert torch.equal(again, out)


def test_pool_beyond_32_bit_offsets():
    """Pages whose byte offset in the pool passes 2^31 and 2^32."""
    page, H, D = 64, 8, 128
    per_page = page * H * D // 2
    pages = (1 << 32) // per_page + 40
    cache = A.KV4Cache.empty(pages, page, H, D)
    table = ints(pages - 1, (1 << 31) // per_page + 1, pages - 2)[None]
    k, v = (torch.randn(1, 150, H, D, device="cuda", generator=gen(i)).to(torch.bfloat16) for i in (1, 2))
    A.kv4_append(cache, k, v, table, ints(0))
    for x, y in zip((k, v), A.kv4_read(cache, table, ints(0), 150, dtype=torch.float32)):
        assert torch.equal(y, values(x.float()))
    q = torch.randn(1, 1, 16, D, device="cuda", generator=gen(3)).to(torch.bfloat16)
    out, lse = A.kv4_attention(q, cache, table, ints(150), return_lse=True)
    compare(out, lse, definition(q, values(k.float()).double(), values(v.float()).double(), [150], [1], D ** -0.5),
            torch.bfloat16)


def test_no_sequences_or_tokens():
    cache = A.KV4Cache.empty(2, 16, 2, 64)
    for B, T in ((0, 1), (2, 0)):
        table, n = torch.zeros(B, 1, device="cuda", dtype=torch.int32), torch.zeros(B, device="cuda", dtype=torch.int32)
        x = torch.zeros(B, T, 2, 64, device="cuda", dtype=torch.bfloat16)
        A.kv4_append(cache, x, x, table, n)
        assert A.kv4_read(cache, table, n, T)[0].shape == (B, T, 2, 64)
        assert A.kv4_attention(x, cache, table, n).shape == (B, T, 2, 64)


def test_ops_trace_under_compile():
    cache, table, n, q, _ = check([90, 20], 1, 4, 2, 64, 16, torch.bfloat16)
    k = torch.randn(2, 1, 2, 64, device="cuda", generator=gen(4)).to(torch.bfloat16)

    def step(k, q):
        A.kv4_append(cache, k, k, table, n - 1)
        return A.kv4_attention(q, cache, table, n), *A.kv4_read(cache, table, n - 1, 1)

    want = step(k, q)
    got = torch.compile(step, fullgraph=True)(k, q)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals():
    cache, table, n = A.KV4Cache.empty(2, 16, 2, 64), ints(0)[None], ints(4)
    k = torch.zeros(1, 1, 2, 64, device="cuda")
    q = torch.zeros(1, 1, 4, 64, device="cuda", dtype=torch.bfloat16)
    kc, kp, vc, vp = cache.tensors()
    for pool in ((kc.cpu(), kp, vc, vp), (kc.float(), kp, vc, vp), (kc, kp.float(), vc, vp), (kc, kp, vc[:, :1], vp),
                 (kc[:, :, :8], kp[:, :, :8], vc[:, :, :8], vp[:, :, :8]), (kc, kp[..., :1], vc, vp), (kc[0], kp, vc, vp)):
        bad = A.KV4Cache(*pool)
        for call in (lambda: A.kv4_append(bad, k, k, table, n), lambda: A.kv4_read(bad, table, n, 1),
                     lambda: A.kv4_attention(q, bad, table, n)):
            with pytest.raises(RuntimeError):
                call()
    for call in (lambda: A.kv4_append(cache, k, k[:, :, :1], table, n), lambda: A.kv4_append(cache, k, k.half(), table, n),
                 lambda: A.kv4_append(cache, k.double(), k.double(), table, n), lambda: A.kv4_append(cache, k.cpu(), k, table, n),
                 lambda: A.kv4_append(cache, k, k, table.long(), n), lambda: A.kv4_append(cache, k, k, table, n.long()),
                 lambda: A.kv4_append(cache, k, k, table, n, ints(1, 1)), lambda: A.kv4_append(cache, k, k, table[0], n),
                 lambda: A.kv4_append(cache, k.requires_grad_(True), k, table, n),
                 lambda: A.kv4_read(cache, table, n, -1), lambda: A.kv4_read(cache, table, n, 1, dtype=torch.float64),
                 lambda: A.kv4_attention(q.float(), cache, table, n), lambda: A.kv4_attention(q[:, :, :3], cache, table, n),
                 lambda: A.kv4_attention(q[..., :32], cache, table, n), lambda: A.kv4_attention(q[0], cache, table, n),
                 lambda: A.kv4_attention(q, cache, table, ints(1, 2)),
                 lambda: A.kv4_attention(q.requires_grad_(True), cache, table, n)):
        with pytest.raises(RuntimeError):
            call()
    small = A.KV4Cache.empty(2, 16, 2, 32)
    with pytest.raises(RuntimeError, match="64 and 128"):
        A.kv4_attention(torch.zeros(1, 1, 2, 32, device="cuda", dtype=torch.bfloat16), small, table, n)
    for bad in ((2, 8, 2, 64), (2, 24, 2, 64), (2, 16, 2, 48)):
        with pytest.raises(RuntimeError):
            A.KV4Cache.empty(*bad)


def test_status_word_is_clear():
    assert _native.device_status(reset=True) == 0
