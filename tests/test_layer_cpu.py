"""The layer operators without a GPU: the C ABI's answers to bad arguments, the binding's refusals, the fake (meta)
implementations that let graphs be traced, and the GPT's parameters with and without the fused layer."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import attnres_b200 as A
from attnres_b200 import _native as N

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4
P = ctypes.c_void_p(64)  # never read: the call is turned down first
ODD = ctypes.c_void_p(68)
STRIDES = (ctypes.c_int64 * 9)(*[0] * 9)


def rope(n=4, T=2, hq=2, hkv=1, D=64, rot=64, dtype=N.DTYPE_BF16, qkv=P, stride=256, cos=P, sin=P, rows=8, pos=None, wq=None,
         wk=None, q=P, k=P, v=P):
    return N.load().attnres_qk_norm_rope_forward(n, T, hq, hkv, D, rot, dtype, qkv, stride, cos, sin, rows, pos, 0, wq, wk, 1,
                                                 1e-6, 1, q, k, v, None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=5), INVALID), (dict(n=-2), INVALID), (dict(T=0), INVALID), (dict(hq=0), INVALID), (dict(hkv=5000), INVALID),
    (dict(D=0), INVALID), (dict(rot=63), INVALID), (dict(rot=66), INVALID), (dict(rot=-2), INVALID), (dict(dtype=9), INVALID),
    (dict(D=520, rot=64, stride=4 * 520), UNSUPPORTED), (dict(stride=255), INVALID), (dict(qkv=None), INVALID),
    (dict(cos=None), INVALID), (dict(sin=None), INVALID), (dict(rows=1), INVALID), (dict(q=None), INVALID),
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(n=1 << 40, T=1), UNSUPPORTED), (dict(n=0, qkv=None, q=None), 0)])
def test_qk_norm_rope_arguments(kw, status):
    assert rope(**kw) == status, N.load().attnres_last_error()


def test_qk_norm_rope_backward_arguments():
    def call(gq=P, gk=P, gv=P, strides=STRIDES, dqkv=P, wq=None, dwq=None, ws=None, size=0):
        return N.load().attnres_qk_norm_rope_backward(4, 2, 2, 1, 64, 64, N.DTYPE_BF16, P, 256, P, P, 8, None, 0, wq, None, 1,
                                                      1e-6, 1, gq, gk, gv, strides, dqkv, dwq, None, ws, size, None)

    for kw in (dict(gq=None), dict(gk=None), dict(gv=None), dict(strides=None), dict(dqkv=None), dict(dwq=P)):
        assert call(**kw) == INVALID
    assert call(wq=P, dwq=P) == WORKSPACE and call(wq=P, dwq=P, ws=P, size=16) == WORKSPACE
    assert N.load().attnres_qk_norm_rope_backward_workspace_bytes(0) == 0
    assert N.load().attnres_qk_norm_rope_backward_workspace_bytes(64) >= 2 * 64 * 4


def swiglu(n=4, C=64, F=32, dtype=N.DTYPE_BF16, x=P, xs=64, w=P, ws=64, h=P):
    return N.load().attnres_swiglu_forward(n, C, F, dtype, x, xs, w, ws, h, None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), INVALID), (dict(C=0), INVALID), (dict(F=0), INVALID), (dict(dtype=7), INVALID), (dict(xs=56), INVALID),
    (dict(ws=56), INVALID), (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(h=None), INVALID),
    (dict(dtype=N.DTYPE_F32), UNSUPPORTED), (dict(C=60, xs=64), UNSUPPORTED), (dict(F=36), UNSUPPORTED),
    (dict(xs=68), UNSUPPORTED), (dict(ws=65), UNSUPPORTED), (dict(x=ODD), UNSUPPORTED), (dict(w=ODD), UNSUPPORTED),
    (dict(h=ODD), UNSUPPORTED), (dict(n=1 << 31), UNSUPPORTED), (dict(n=0, x=None, h=None), 0)])
def test_swiglu_arguments(kw, status):
    assert swiglu(**kw) == status, N.load().attnres_last_error()


def test_swiglu_backward_arguments():
    L = N.load()
    size = L.attnres_swiglu_backward_workspace_bytes(4, 32)
    assert size == 4 * 2 * 32 * 2 and L.attnres_swiglu_backward_workspace_bytes(0, 32) == 0

    def call(gh=P, gs=32, dx=P, dw=P, ws=P, size=size):
        return L.attnres_swiglu_backward(4, 64, 32, N.DTYPE_BF16, P, 64, P, 64, gh, gs, dx, dw, ws, size, None)

    for kw, status in ((dict(gh=None), INVALID), (dict(gs=24), INVALID), (dict(gs=36), UNSUPPORTED), (dict(gh=ODD), UNSUPPORTED),
                       (dict(dx=ODD), UNSUPPORTED), (dict(dw=ODD), UNSUPPORTED), (dict(ws=ODD), UNSUPPORTED),
                       (dict(ws=None), WORKSPACE), (dict(size=size - 1), WORKSPACE), (dict(dx=None, dw=None), 0)):
        assert call(**kw) == status, (kw, L.attnres_last_error())


def pool(kc=P, kp=P, vc=P, vp=P, pages=4, heads=2, page=16, D=64, table=P, stride=2, max_pages=2):
    return [kc, kp, vc, vp, pages, heads, page, D, table, stride, max_pages]


def kv4(entry, start=P, batch=2, T=1, dtype=N.DTYPE_BF16, a=P, b=P, q_heads=4, strides=STRIDES, scale=1.0, lse=None, ws=P,
        size=1 << 30, **kw):
    L = N.load()
    if entry == "append":
        return L.attnres_kv4_append(*pool(**kw), start, None, batch, T, dtype, a, strides, b, strides, None)
    if entry == "read":
        return L.attnres_kv4_read(*pool(**kw), start, None, batch, T, dtype, a, b, None)
    return L.attnres_kv4_attention(*pool(**kw), start, None, batch, T, q_heads, dtype, a, strides, scale, b, lse, ws, size, None)


@pytest.mark.parametrize("entry", ["append", "read", "attention"])
@pytest.mark.parametrize("kw,status", [
    (dict(pages=-1), INVALID), (dict(heads=0), INVALID), (dict(page=0), INVALID), (dict(D=0), INVALID), (dict(max_pages=-1), INVALID),
    (dict(batch=-1), INVALID), (dict(T=-1), INVALID), (dict(dtype=5), INVALID), (dict(kc=None), INVALID), (dict(vp=None), INVALID),
    (dict(table=None), INVALID), (dict(start=None), INVALID), (dict(a=None), INVALID), (dict(b=None), INVALID),
    (dict(stride=1), INVALID), (dict(page=24), UNSUPPORTED), (dict(D=48), UNSUPPORTED), (dict(D=544), UNSUPPORTED),
    (dict(kc=ODD), UNSUPPORTED), (dict(vp=ODD), UNSUPPORTED), (dict(batch=70000), UNSUPPORTED),
    (dict(max_pages=1 << 27, stride=1 << 27), UNSUPPORTED), (dict(pages=1 << 31), UNSUPPORTED), (dict(batch=0), 0), (dict(T=0), 0)])
def test_kv4_arguments(entry, kw, status):
    assert kv4(entry, **kw) == status, N.load().attnres_last_error()


def test_kv4_attention_arguments():
    for kw, status in ((dict(dtype=N.DTYPE_F32), UNSUPPORTED), (dict(D=32), UNSUPPORTED), (dict(q_heads=3), INVALID),
                       (dict(q_heads=0), INVALID), (dict(strides=None), INVALID), (dict(b=ODD), UNSUPPORTED),
                       (dict(ws=ODD), UNSUPPORTED), (dict(max_pages=4096, stride=4096, ws=None), WORKSPACE),
                       (dict(max_pages=4096, stride=4096, size=64), WORKSPACE)):
        assert kv4("attention", **kw) == status, (kw, N.load().attnres_last_error())
    need = N.load().attnres_kv4_attention_workspace_bytes
    assert need(2, 16, 64, 4096, 2, 1, 4) > 0 and need(2, 16, 64, 1, 2, 1, 4) == 0 and need(0, 16, 64, 4096, 2, 1, 4) == 0


def test_cpu_tensors_are_refused():
    cos = torch.zeros(4, 32)
    cache, table, n = A.KV4Cache.empty(2, 16, 2, 64, device="cpu"), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: A.qk_norm_rope(torch.zeros(1, 2, 256), 2, 1, cos, cos),
                 lambda: A.swiglu_projection(torch.zeros(2, 64).half(), torch.zeros(64, 64).half()),
                 lambda: A.kv4_append(cache, x, x, table, n), lambda: A.kv4_read(cache, table, n, 1),
                 lambda: A.kv4_attention(x, cache, table, n)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_fake_shapes():
    mode = FakeTensorMode()
    with mode:
        def new(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        ops = torch.ops.attnres  # the backward ops by name: autograd's engine wants a real device
        qkv, cos, w = new(2, 5, 8 * 64), new(9, 16, dtype=torch.float32), new(64)
        out = A.qk_norm_rope(qkv, 4, 2, cos, cos, q_weight=w)
        assert [tuple(t.shape) for t in out] == [(2, 5, 4, 64), (2, 5, 2, 64), (2, 5, 2, 64)]
        g = ops.qk_norm_rope_backward(*out, qkv, cos, cos, None, w, None, 4, 2, True, 1e-6, True, True, False)
        assert g[0].shape == qkv.shape and g[1].shape == w.shape and g[2].shape == (0,)
        x, w1 = new(2, 5, 64), new(48, 64)
        h = A.swiglu_projection(x, w1)
        assert h.shape == (2, 5, 24)
        g = ops.swiglu_projection_backward(h, x, w1, True, True)
        assert g[0].shape == x.shape and g[1].shape == w1.shape
        cache = A.KV4Cache.empty(8, 16, 2, 64)
        table, n = new(3, 2, dtype=torch.int32), new(3, dtype=torch.int32)
        k = new(3, 1, 2, 64)
        assert A.kv4_append(cache, k, k, table, n) is None
        assert [tuple(t.shape) for t in A.kv4_read(cache, table, n, 7)] == [(3, 7, 2, 64)] * 2
        o, lse = A.kv4_attention(new(3, 1, 6, 64), cache, table, n, return_lse=True)
        assert o.shape == (3, 1, 6, 64) and lse.shape == (3, 1, 6) and lse.dtype == torch.float32


def test_gpt_keeps_its_parameters():
    from attnres_b200.gpt import GPT, GPTConfig

    kw = dict(n_layer=2, n_head=2, n_embd=128, vocab_size=33, block_size=16, lrid_rank=32)
    a, b = GPT(GPTConfig(**kw)), GPT(GPTConfig(**kw, fused_layer=True))
    assert {k: v.shape for k, v in a.state_dict().items()} == {k: v.shape for k, v in b.state_dict().items()}
    b.to(torch.bfloat16)
    rope = b.transformer.layers[0].attn.rope
    assert rope.sin.dtype == torch.bfloat16 and all(t.dtype == torch.float32 and t.shape == (16, 32) for t in rope.tables)
