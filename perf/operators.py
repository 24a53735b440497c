"""Cases for measuring the operators of a transformer layer around the depth read.

  qk_norm_rope       the fused q/k/v projection's output split into heads, q and k RMS-normed per head and
                     rotated by position; forward, and forward + backward
  swiglu_projection  silu(x Wg^T) * (x Wv^T) with both halves of one weight; forward, and forward + backward
  kv4_append,        keys and values quantised to 4 bits as they are written into a paged cache, and read
  kv4_read           back as the values they stand for
  kv4_attention      attention of new query tokens over such a cache

With `own` false, run() computes each in elementary torch operations in 32 bits; with `own` true it calls
attnres_b200. exact() is each operator's definition in 64 bits.

The cache's format (group = 32 elements of a head, G = head_dim / 32):
  k_codes, v_codes    uint8 [pages, kv heads, page size, head_dim / 2], two codes a byte, the lower first
  k_params, v_params  float16 [pages, kv heads, page size, G, 2]: a group's step and its lowest value
  element = low + step * code. A row's codes lie in the order in which a tensor-core lane takes them:
  keys   4 x G words of 8 codes: word (c, g) holds elements 32 g + 8 c + 0..7
  values 8 x G half words of 4 codes: half word (r, g) holds elements 32 g + 4 r + 0..3
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 32
F32_EPS = 2.0 ** -23  # eps of every norm of the model: float32's


def _package():
    path = os.path.join(os.getcwd(), "lr-attnres_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import attnres_b200

    return attnres_b200


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _rope(name, B, T, Hq, Hkv, D, dtype, train, interleaved, weighted):
    return dict(name=name, op="rope", B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, train=train,
                interleaved=interleaved, weighted=weighted)


def _mlp(name, N, C, F, dtype, train):
    return dict(name=name, op="mlp", N=N, C=C, F=F, dtype=dtype, train=train)


def _cache(name, B, T, Hkv, D, page, past, dtype):
    return dict(name=name, op="cache", B=B, T=T, Hkv=Hkv, D=D, page=page, past=past, dtype=dtype)


def _attend(name, B, T, Hq, Hkv, D, page, longest, ragged, dtype):
    return dict(name=name, op="attend", B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, longest=longest, ragged=ragged,
                dtype=dtype)


def listed():
    return [
        # one new token of four sequences through the 24-layer GPT's attention heads: latency
        _rope("rope decode", 4, 1, 16, 16, 64, "bf16", False, True, False),
        # the GPT's training step: 8 sequences of 2048 tokens, forward and backward
        _rope("rope train", 8, 2048, 16, 16, 64, "bf16", True, True, False),
        # a model with shared key heads, learned norm weights and half-split rotation, an odd length
        _rope("rope shared heads", 3, 1237, 20, 4, 128, "f16", True, False, True),
        # the GPT's MLP for a single token: the weights are read once
        _mlp("mlp one token", 1, 1024, 4096, "bf16", False),
        # a decoding batch of odd size
        _mlp("mlp decode batch", 27, 1024, 4096, "bf16", False),
        # a width and a token count that no tile divides, forward and backward
        _mlp("mlp ragged", 1531, 776, 2056, "f16", True),
        # the GPT's training step
        _mlp("mlp train", 16384, 1024, 4096, "bf16", True),
        # one new token of 32 sequences written behind what they hold
        _cache("cache decode", 32, 1, 16, 64, 64, 1000, "bf16"),
        # the prompts of 6 sequences, a length that ends inside a page
        _cache("cache prompt", 6, 4001, 8, 128, 64, 0, "bf16"),
        # one sequence's next token with a short past: latency
        _attend("attend short", 1, 1, 16, 16, 64, 64, 300, False, "bf16"),
        # a decoding batch of ragged lengths, 4 query heads to a key head
        _attend("attend batch", 24, 1, 32, 8, 128, 64, 6000, True, "f16"),
        # long documents, three tokens a sequence to check at once
        _attend("attend long", 8, 3, 16, 16, 64, 64, 50000, False, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    """An MLP width of 512 to 4096, a multiple of 8."""
    return 8 * rng.choice([n for n in range(64, 513) if n != 384])


def draw(rng):
    op = rng.choice(["rope", "mlp", "cache", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "rope":
        B = rng.randint(1, 8)
        D = rng.choice([64, 128, 80])
        Hkv = rng.choice([1, 2, 4, 8])
        c = _rope("", B, max(1, _log(rng, 1, 16384) // B), Hkv * rng.choice([1, 2, 3]), Hkv, D,
                  rng.choice(["bf16", "f16", "f32"]), rng.random() < 0.6, rng.random() < 0.5, rng.random() < 0.5)
    elif op == "mlp":
        c = _mlp("", _log(rng, 1, 16384), 8 * rng.randint(32, 128), _width(rng), dtype,
                 rng.random() < 0.5)
    elif op == "cache":
        B = rng.randint(1, 16)
        c = _cache("", B, max(1, _log(rng, 1, 24000) // B), rng.choice([1, 2, 4, 8]), rng.choice([64, 128]),
                   rng.choice([16, 64, 128]), _log(rng, 1, 3000), rng.choice(["bf16", "f16", "f32"]))
    else:
        B = rng.randint(1, 32)
        Hkv = rng.choice([1, 2, 4, 8])
        c = _attend("", B, rng.choice([1, 1, 1, 2, 5]), Hkv * rng.choice([1, 2, 4, 6]), Hkv, rng.choice([64, 128]),
                    rng.choice([16, 32, 64, 128]), max(1, _log(rng, 8, 200000) // B), rng.random() < 0.5, dtype)
    del c["name"]
    return c


def _lengths(case):
    """Keys of each sequence of an attention case, its query tokens among them: one in five of a ragged batch is
    short, and its second sequence has none."""
    B, n = case["B"], case["longest"]
    if not case["ragged"]:
        return [max(1, n - (b % 3)) for b in range(B)]
    got = [max(1, (n * (1 + (7 * b) % 16)) // 16) for b in range(B)]
    for b in range(4, B, 5):
        got[b] = min(n, 1 + b)
    if B > 1:
        got[1] = 0
    return got


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        tokens, heads, D = case["B"] * case["T"], case["Hq"] + 2 * case["Hkv"], case["D"]
        row = tokens * heads * D
        qk = tokens * (case["Hq"] + case["Hkv"]) * D
        by, fl = 2 * row * e + tokens * D * 4, 7 * qk
        if case["train"]:  # reads the three gradients and the q and k columns again, writes the projection's gradient
            by, fl = by + (2 * row + qk) * e + tokens * D * 4, fl + 14 * qk
        return {"bytes": by, "flops": fl}
    if case["op"] == "mlp":
        N, C, F = case["N"], case["C"], case["F"]
        by, fl = (N * C + 2 * F * C + N * F) * e, 4.0 * N * C * F
        if case["train"]:  # x, weight and the output's gradient in, the gradients of x and weight out
            by, fl = by + (2 * N * C + 4 * F * C + N * F) * e, 3 * fl
        return {"bytes": by, "flops": fl}
    code = case["D"] // 2 + case["D"] // GROUP * 4  # bytes of a row of a head in the cache
    if case["op"] == "cache":
        rows = 2 * case["B"] * case["T"] * case["Hkv"]
        return {"bytes": rows * (2 * case["D"] * e + 2 * code), "flops": rows * case["D"] * 6}
    keys = sum(_lengths(case))
    q = case["B"] * case["T"] * case["Hq"] * case["D"]
    return {"bytes": 2 * keys * case["Hkv"] * code + 2 * q * e,
            "flops": 4.0 * keys * case["T"] * case["Hq"] * case["D"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * std).to(dtype)


def _pack_k(n):
    """Codes [..., D] (0..15) -> uint8 [..., D / 2] in the order of the keys."""
    G = n.shape[-1] // GROUP
    n = n.reshape(*n.shape[:-1], G, 4, 4, 2).transpose(-4, -3)
    return (n[..., 0] + 16 * n[..., 1]).to(torch.uint8).flatten(-3)


def _pack_v(n):
    G = n.shape[-1] // GROUP
    n = n.reshape(*n.shape[:-1], G, 8, 2, 2).transpose(-4, -3)
    return (n[..., 0] + 16 * n[..., 1]).to(torch.uint8).flatten(-3)


def _unpack(codes, lanes):
    """uint8 [..., D / 2] -> codes [..., G, 32] as they stand in the head; `lanes` 4 (keys) or 8 (values)."""
    G = codes.shape[-1] * 2 // GROUP
    n = torch.stack([codes & 15, codes >> 4], dim=-1)
    return n.reshape(*codes.shape[:-1], lanes, G, GROUP // lanes).transpose(-3, -2).flatten(-2)


def _quantise(x):
    """x [..., D] -> (codes [..., D] as floats, params float16 [..., G, 2]), in x's type (32 or 64 bits)."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    top, low = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    step = ((top - low) * (1.0 / 15.0)).half()
    low = low.half()
    n = torch.where(step > 0, ((g - low.to(x.dtype)) / step.to(x.dtype)).round().clamp(0, 15), torch.zeros_like(g))
    return n.flatten(-2), torch.cat([step, low], dim=-1)


def _pages(case, tokens, g):
    """A page table whose pages lie in the pool in no order, and the pool's size."""
    per = -(-max(1, tokens) // case["page"])
    total = case["B"] * per + 3
    order = torch.randperm(total, generator=g, device=DEV)[: case["B"] * per]
    return order.reshape(case["B"], per).to(torch.int32), total


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "rope":
        B, T, Hq, Hkv, D = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
        start = [(5 + 37 * b) % 97 for b in range(B)]
        table = max(start) + T
        freq = torch.outer(torch.arange(table, device=DEV, dtype=torch.float64),
                           500000.0 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D))
        s["cos"], s["sin"] = freq.cos().float(), freq.sin().float()
        s["positions"] = (torch.tensor(start, device=DEV)[:, None] + torch.arange(T, device=DEV)).to(torch.int32)
        s["qkv"] = _randn(g, B, T, (Hq + 2 * Hkv) * D, dtype=dt, std=1.5).requires_grad_(case["train"])
        s["wq"] = s["wk"] = None
        if case["weighted"]:
            s["wq"] = (1 + _randn(g, D, std=0.2)).to(dt).requires_grad_(case["train"])
            s["wk"] = (1 + _randn(g, D, std=0.2)).to(dt).requires_grad_(case["train"])
        if case["train"]:
            s["grads"] = [_randn(g, B, T, h, D, dtype=dt) for h in (Hq, Hkv, Hkv)]
    elif case["op"] == "mlp":
        N, C, F = case["N"], case["C"], case["F"]
        s["x"] = _randn(g, N, C, dtype=dt).requires_grad_(case["train"])
        s["w"] = _randn(g, 2 * F, C, dtype=dt, std=1.0 / math.sqrt(C)).requires_grad_(case["train"])
        if case["train"]:
            s["dh"] = _randn(g, N, F, dtype=dt)
    else:
        B, T, Hkv, D, page = (case[k] for k in ("B", "T", "Hkv", "D", "page"))
        if case["op"] == "cache":
            start = [max(0, case["past"] - 13 * b) for b in range(B)]
            s["table"], total = _pages(case, max(start) + T, g)
            s["start"] = torch.tensor(start, device=DEV, dtype=torch.int32)
            # keys come with a few channels that stand out, values without
            loud = 1 + 4 * (torch.rand(Hkv, D, generator=g, device=DEV) > 0.95)
            s["k"] = (_randn(g, B, T, Hkv, D) * loud).to(dt)
            s["v"] = _randn(g, B, T, Hkv, D, dtype=dt)
        else:
            lengths = _lengths(case)
            s["table"], total = _pages(case, max(lengths), g)
            s["lengths"] = torch.tensor(lengths, device=DEV, dtype=torch.int32)
            s["q"] = _randn(g, B, T, case["Hq"], D, dtype=dt)
        s["cache"] = []
        for pack, loud in ((_pack_k, True), (_pack_v, False)):
            if case["op"] == "cache":  # what other tokens left there
                codes = torch.randint(0, 256, (total, Hkv, page, D // 2), generator=g, device=DEV, dtype=torch.uint8)
                params = _randn(g, total, Hkv, page, D // GROUP, 2, dtype=torch.float16)
            else:
                codes = torch.empty(total, Hkv, page, D // 2, device=DEV, dtype=torch.uint8)
                params = torch.empty(total, Hkv, page, D // GROUP, 2, device=DEV, dtype=torch.float16)
                chunk = max(1, (1 << 26) // (Hkv * page * D))
                for a in range(0, total, chunk):
                    x = _randn(g, min(chunk, total - a), Hkv, page, D)
                    if loud:
                        x = x * (1 + 2 * (torch.arange(D, device=DEV) % 29 == 0))
                    n, p = _quantise(x)
                    codes[a:a + chunk], params[a:a + chunk] = pack(n), p
            s["cache"] += [codes, params]
    return s


# ---------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits, rounded once
# ---------------------------------------------------------------------------
def _rotate(x, cos, sin, interleaved, inverse=False):
    """Rotates the pairs of x [B, T, H, D] by cos, sin [B, T, 1, D / 2]."""
    if inverse:
        sin = -sin
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    u, v = a * cos - b * sin, a * sin + b * cos
    return torch.stack([u, v], dim=-1).flatten(-2) if interleaved else torch.cat([u, v], dim=-1)


def _plain_rope(s):
    c = s["case"]
    B, T, Hq, Hkv, D = (c[k] for k in ("B", "T", "Hq", "Hkv", "D"))
    dt = s["qkv"].dtype
    cos, sin = (s[k][s["positions"].long()][:, :, None] for k in ("cos", "sin"))
    x = s["qkv"].float().view(B, T, Hq + 2 * Hkv, D)
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]

    def forward(x, w):
        inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + F32_EPS)
        y = x * inv
        return _rotate(y if w is None else y * w.float(), cos, sin, c["interleaved"]).to(dt)

    out = [forward(q, s["wq"]), forward(k, s["wk"]), v.to(dt)]
    if not c["train"]:
        return out

    def backward(x, w, dy):
        inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + F32_EPS)
        y = x * inv
        g = _rotate(dy.float(), cos, sin, c["interleaved"], inverse=True)
        dw = None if w is None else (g * y).sum((0, 1, 2)).to(dt)
        g = g if w is None else g * w.float()
        return inv * (g - y * (g * y).mean(-1, keepdim=True)), dw

    dq, dwq = backward(q, s["wq"], s["grads"][0])
    dk, dwk = backward(k, s["wk"], s["grads"][1])
    out.append(torch.cat([dq, dk, s["grads"][2].float()], dim=2).flatten(2).to(dt))
    return out + [dwq, dwk] if c["weighted"] else out


def _plain_mlp(s):
    x, w, dt = s["x"].float(), s["w"].float(), s["x"].dtype
    F = s["case"]["F"]
    u, g = x @ w[:F].t(), x @ w[F:].t()
    sig = torch.sigmoid(g)
    h = (u * g * sig).to(dt)
    if not s["case"]["train"]:
        return h
    dh = s["dh"].float()
    du = dh * g * sig
    dg = dh * u * sig * (1 + g * (1 - sig))
    dx = (du @ w[:F] + dg @ w[F:]).to(dt)
    return h, dx, torch.cat([du.t() @ x, dg.t() @ x]).to(dt)


def _slots(s, T):
    """(page, place in it) of tokens start .. start + T of each sequence: [B, T] each."""
    at = s["start"].long()[:, None] + torch.arange(T, device=DEV)
    page = s["case"]["page"]
    return torch.gather(s["table"].long(), 1, at // page), at % page


def _plain_cache(s):
    page, place = _slots(s, s["case"]["T"])
    kc, kp, vc, vp = s["cache"]
    out = []
    for x, codes, params, pack, lanes in ((s["k"], kc, kp, _pack_k, 4), (s["v"], vc, vp, _pack_v, 8)):
        n, p = _quantise(x.float())
        codes[page, :, place] = pack(n)
        params[page, :, place] = p
        p = params[page, :, place].float()
        out.append((p[..., 1:] + p[..., :1] * _unpack(codes[page, :, place], lanes)).flatten(-2).to(x.dtype))
    return out


def _gathered(s, codes, params, lanes):
    """The first `longest` rows of each sequence's cache: [B, Hkv, longest, D] in 32 bits."""
    t = s["table"].long()
    n = _unpack(codes[t], lanes)
    p = params[t].float()
    x = (p[..., 1:] + p[..., :1] * n).flatten(-2)  # [B, pages, Hkv, page, D]
    return x.transpose(1, 2).flatten(2, 3)[:, :, : max(1, int(s["case"]["longest"]))]


def _plain_attend(s):
    c = s["case"]
    B, T, Hq, Hkv, D = (c[k] for k in ("B", "T", "Hq", "Hkv", "D"))
    kc, kp, vc, vp = s["cache"]
    K = _gathered(s, kc, kp, 4)
    q = s["q"].float().view(B, T, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    z = (q @ K.transpose(-1, -2)).view(B, Hkv, T, Hq // Hkv, -1) * (1.0 / math.sqrt(D))
    at = s["lengths"].long()[:, None] - T + torch.arange(T, device=DEV)  # the query's own place
    see = torch.arange(K.shape[2], device=DEV) <= at[..., None]          # [B, T, longest]
    z = z.masked_fill(~see[:, None, :, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p)).reshape(B, Hkv, -1, K.shape[2])
    del z, K
    out = p @ _gathered(s, vc, vp, 8)
    return out.view(B, Hkv, T, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, T, Hq, D).to(s["q"].dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if not own:
        with torch.no_grad():
            return {"rope": _plain_rope, "mlp": _plain_mlp, "cache": _plain_cache, "attend": _plain_attend}[c["op"]](s)
    A = _package()
    if c["op"] == "rope":
        out = A.qk_norm_rope(s["qkv"], c["Hq"], c["Hkv"], s["cos"], s["sin"], positions=s["positions"],
                             q_weight=s["wq"], k_weight=s["wk"], interleaved=c["interleaved"])
        if not c["train"]:
            return list(out)
        leaves = [s["qkv"]] + ([s["wq"], s["wk"]] if c["weighted"] else [])
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, s["grads"]))
    if c["op"] == "mlp":
        h = A.swiglu_projection(s["x"], s["w"])
        if not c["train"]:
            return h
        return (h.detach(), *torch.autograd.grad(h, [s["x"], s["w"]], s["dh"]))
    cache = A.KV4Cache(*s["cache"])
    if c["op"] == "cache":
        A.kv4_append(cache, s["k"], s["v"], s["table"], s["start"])
        return list(A.kv4_read(cache, s["table"], s["start"], c["T"], dtype=s["k"].dtype))
    return A.kv4_attention(s["q"], cache, s["table"], s["lengths"])


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rope(s):
    c = s["case"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    cos, sin = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
    pair = torch.arange(D // 2, device=DEV)
    first, second = (2 * pair, 2 * pair + 1) if c["interleaved"] else (pair, pair + D // 2)
    with torch.enable_grad():
        qkv = s["qkv"].detach().double().requires_grad_(True)
        ws = [None if w is None else w.detach().double().requires_grad_(True) for w in (s["wq"], s["wk"])]
        x = qkv.unflatten(-1, (Hq + 2 * Hkv, D))
        out = []
        for part, w in ((x[:, :, :Hq], ws[0]), (x[:, :, Hq:Hq + Hkv], ws[1])):
            y = part / torch.sqrt((part * part).sum(-1, keepdim=True) / D + F32_EPS)
            y = y if w is None else y * w
            z = torch.zeros_like(y)
            a, b = y[..., first], y[..., second]
            z = z.index_add(-1, first, a * cos[:, :, None] - b * sin[:, :, None])
            out.append(z.index_add(-1, second, b * cos[:, :, None] + a * sin[:, :, None]))
        out.append(x[:, :, Hq + Hkv:].clone())
        if not c["train"]:
            return [t.detach() for t in out]
        grads = torch.autograd.grad(out, [qkv] + [w for w in ws if w is not None], [g.double() for g in s["grads"]])
    return [t.detach() for t in out] + list(grads)


def _exact_mlp(s):
    x, w, F = s["x"].detach().double(), s["w"].detach().double(), s["case"]["F"]
    y = torch.einsum("nc,fc->nf", x, w)
    u, g = y[:, :F], y[:, F:]
    if not s["case"]["train"]:
        return u * g / (1 + torch.exp(-g))
    # d silu(g) / dg from the quotient's rule
    e = torch.exp(-g)
    silu, slope = g / (1 + e), (1 + e + g * e) / (1 + e) ** 2
    d = torch.cat([s["dh"].double() * silu, s["dh"].double() * u * slope], dim=1)
    return u * silu, torch.einsum("nf,fc->nc", d, w), torch.einsum("nf,nc->fc", d, x)


def _exact_cache(s):
    out = []
    for x in (s["k"].double(), s["v"].double()):
        g = x.unflatten(-1, (-1, GROUP))
        low = g.min(-1).values.half().double()[..., None]
        step = ((g.max(-1).values - g.min(-1).values) / 15).half().double()[..., None]
        n = torch.floor((g - low) / torch.where(step > 0, step, torch.ones_like(step)))
        rest = (g - low) / torch.where(step > 0, step, torch.ones_like(step)) - n
        n = n + ((rest > 0.5) | ((rest == 0.5) & (n % 2 == 1)))
        out.append((low + step * n.clamp(0, 15)).flatten(-2))
    return out


def _exact_attend(s):
    c = s["case"]
    B, T, Hq, Hkv, D, page = (c[k] for k in ("B", "T", "Hq", "Hkv", "D", "page"))
    G = D // GROUP
    element = torch.arange(D, device=DEV)
    group, inside = element // GROUP, element % GROUP
    kc, kp, vc, vp = s["cache"]
    out = torch.zeros(B, T, Hq, D, device=DEV, dtype=torch.float64)

    def rows(codes, params, b, h, n, lanes):
        per = GROUP // lanes
        nibble = (inside // per * G + group) * per + inside % per
        pages = s["table"][b, : -(-n // page)].long()
        byte = codes[pages, h].flatten(0, 1)[:n][:, nibble // 2].double()
        n4 = torch.where(nibble % 2 == 0, byte % 16, torch.floor(byte / 16))
        p = params[pages, h].flatten(0, 1)[:n].double()
        return p[:, group, 1] + p[:, group, 0] * n4

    for b, n in enumerate(_lengths(c)):
        for h in range(Hkv if n else 0):
            K, V = rows(kc, kp, b, h, n, 4), rows(vc, vp, b, h, n, 8)
            for t in range(T):
                last = n - T + t
                if last < 0:
                    continue
                for r in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                    z = (K[:last + 1] @ s["q"][b, t, r].double()) / math.sqrt(D)
                    out[b, t, r] = torch.softmax(z, 0) @ V[:last + 1]
    return out


def exact(case, seed):
    if case["op"] == "attend" and case["B"] * case["T"] * case["Hq"] > 20000:
        return None
    s = prepare(case, seed)
    return {"rope": _exact_rope, "mlp": _exact_mlp, "cache": _exact_cache, "attend": _exact_attend}[case["op"]](s)
