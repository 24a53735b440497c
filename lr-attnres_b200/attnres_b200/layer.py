"""Operators of the transformer layer around the depth read, over libattnres_b200.

  qk_norm_rope(...)       q/k/v split of a fused projection, per-head RMS norm of q and k and the
                          rotation by position in one pass (the steps of the reference's attention
                          between its projection and scaled_dot_product_attention)

Every tensor argument must live on one CUDA device; the work is enqueued on that
device's current stream through the C ABI. There is no CPU fallback: a CPU tensor
is a RuntimeError.

Under torch.compile (and for fake tensors) a call is the attnres:: torch.library
op of the same name, which traces and carries its autograd formula. Eager calls go
to the same launchers directly, through an autograd Function when a gradient is
wanted: the op's dispatch costs tens of microseconds of host time, more than the
kernels take at a decoding step's sizes.
"""
import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _native as N
from .ops import F32_EPS, _dtype_code

_EAGER_TYPES = (Tensor, torch.nn.Parameter)


def _eager(*tensors):
    """Whether a call on these tensors may go straight to the launchers."""
    if torch.compiler.is_compiling():
        return False
    for t in tensors:
        if t is not None and type(t) not in _EAGER_TYPES:
            return False
    return True


def _wants_grad(*tensors):
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _same_device(what, first, *tensors):
    """All on `first`'s CUDA device."""
    if not first.is_cuda:
        raise RuntimeError(f"attnres_b200: {what} inputs must be CUDA tensors (there is no CPU path)")
    dev = first.device
    for t in tensors:
        if t is not None and t.device != dev:
            raise RuntimeError(f"attnres_b200: {what} inputs must be on one device, got {dev} and {t.device}")


def _call(what, device, fn, *args):
    """fn(*args, stream) on the device's current stream; a non-zero status raises."""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        N.check(rc, what)


def _p(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# q/k norm and rotation
# ---------------------------------------------------------------------------
def _rope_args(qkv, cos, sin, positions, q_weight, k_weight, num_heads, num_kv_heads, normalize, eps, interleaved):
    """The C entries' leading arguments, the tensors they point into, and (B, T, D)."""
    what = "qk_norm_rope"
    _same_device(what, qkv, cos, sin, positions, q_weight, k_weight)
    heads = num_heads + 2 * num_kv_heads
    if num_heads < 1 or num_kv_heads < 1:
        raise RuntimeError(f"attnres_b200: {what} needs at least one query and one key head")
    if qkv.dim() != 3 or qkv.size(2) % heads or qkv.size(2) == 0:
        raise RuntimeError(f"attnres_b200: {what} takes qkv [B, T, ({num_heads} + 2 * {num_kv_heads}) * head_dim], "
                           f"got {tuple(qkv.shape)}")
    B, T, width = qkv.shape
    D = width // heads
    code = _dtype_code(qkv.dtype)
    stride = qkv.stride(1) if T > 1 else (qkv.stride(0) if B > 1 else width)
    if qkv.stride(2) != 1 or stride < width or (T > 1 and B > 1 and qkv.stride(0) != T * stride):
        qkv, stride = qkv.contiguous(), width  # rows of one stride that do not overlap
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise RuntimeError(f"attnres_b200: {what} takes cos and sin [positions, rotary_dim / 2], got "
                           f"{tuple(cos.shape)} and {tuple(sin.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise RuntimeError(f"attnres_b200: {what} takes float32 cos and sin")
    cos, sin = cos.contiguous(), sin.contiguous()
    rows, half = cos.shape
    if 2 * half > D:
        raise RuntimeError(f"attnres_b200: {what} rotary_dim {2 * half} exceeds head_dim {D}")
    wide = 0
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (B, T):
            raise RuntimeError(f"attnres_b200: {what} takes positions [B, T] int32 or int64")
        positions, wide = positions.contiguous(), int(positions.dtype == torch.int64)
    elif B and T > rows and half:
        raise RuntimeError(f"attnres_b200: {what} has {T} tokens and tables of {rows} positions")
    weights = []
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (D,):
            raise RuntimeError(f"attnres_b200: {what} weights are [head_dim] = [{D}]")
        weights.append(None if w is None else w.to(qkv.dtype).contiguous())
    args = (B * T, max(T, 1), num_heads, num_kv_heads, D, 2 * half, code, _p(qkv), stride, _p(cos), _p(sin), rows,
            _p(positions), wide, _p(weights[0]), _p(weights[1]), int(normalize), eps, int(interleaved))
    return args, (qkv, cos, sin, positions, weights), (B, T, D)


def _rope_forward(qkv, cos, sin, positions, q_weight, k_weight, num_heads, num_kv_heads, normalize, eps, interleaved):
    args, keep, (B, T, D) = _rope_args(qkv, cos, sin, positions, q_weight, k_weight, num_heads, num_kv_heads,
                                       normalize, eps, interleaved)
    q = qkv.new_empty((B, T, num_heads, D))
    k = qkv.new_empty((B, T, num_kv_heads, D))
    v = qkv.new_empty((B, T, num_kv_heads, D))
    _call("attnres_qk_norm_rope_forward", qkv.device, N.load().attnres_qk_norm_rope_forward, *args, q.data_ptr(),
          k.data_ptr(), v.data_ptr())
    return q, k, v


def _rope_backward(grad_q, grad_k, grad_v, qkv, cos, sin, positions, q_weight, k_weight, num_heads, num_kv_heads,
                   normalize, eps, interleaved, want_q_weight, want_k_weight):
    """(d qkv, d q_weight or None, d k_weight or None)."""
    args, keep, (B, T, D) = _rope_args(qkv, cos, sin, positions, q_weight, k_weight, num_heads, num_kv_heads,
                                       normalize, eps, interleaved)
    grads, strides = [], []
    for g, heads in ((grad_q, num_heads), (grad_k, num_kv_heads), (grad_v, num_kv_heads)):
        if g is None:
            g = qkv.new_zeros(1).expand(B, T, heads, D)
        if g.dtype != qkv.dtype or g.stride(3) != 1:
            g = g.to(qkv.dtype).contiguous()
        grads.append(g)
        strides += g.stride()[:3]
    dqkv = qkv.new_empty((B, T, (num_heads + 2 * num_kv_heads) * D))
    dws, ws, size = [None, None], None, 0
    if want_q_weight or want_k_weight:
        size = N.load().attnres_qk_norm_rope_backward_workspace_bytes(D)
        ws = qkv.new_empty(size, dtype=torch.uint8)
        dws = [qkv.new_empty(D) if want else None for want in (want_q_weight, want_k_weight)]
    _call("attnres_qk_norm_rope_backward", qkv.device, N.load().attnres_qk_norm_rope_backward, *args, _p(grads[0]),
          _p(grads[1]), _p(grads[2]), (ctypes.c_int64 * 9)(*strides), dqkv.data_ptr(), _p(dws[0]), _p(dws[1]), _p(ws),
          size)
    dws = [None if dw is None else dw.to(w.dtype) for dw, w in zip(dws, (q_weight, k_weight))]
    return dqkv, dws[0], dws[1]


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, cos, sin, positions, q_weight, k_weight, *how):
        ctx.how = how
        ctx.save_for_backward(qkv, cos, sin, positions, q_weight, k_weight)
        return _rope_forward(qkv, cos, sin, positions, q_weight, k_weight, *how)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_q, grad_k, grad_v):
        need = ctx.needs_input_grad
        dqkv, dwq, dwk = _rope_backward(grad_q, grad_k, grad_v, *ctx.saved_tensors, *ctx.how, need[4], need[5])
        return (dqkv, None, None, None, dwq, dwk) + (None,) * len(ctx.how)


@torch.library.custom_op("attnres::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(qkv: Tensor, cos: Tensor, sin: Tensor, positions: Optional[Tensor], q_weight: Optional[Tensor],
                    k_weight: Optional[Tensor], num_heads: int, num_kv_heads: int, normalize: bool, eps: float,
                    interleaved: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _rope_forward(qkv, cos, sin, positions, q_weight, k_weight, num_heads, num_kv_heads, normalize, eps,
                         interleaved)


@qk_norm_rope_op.register_fake
def _(qkv, cos, sin, positions, q_weight, k_weight, num_heads, num_kv_heads, normalize, eps, interleaved):
    B, T, width = qkv.shape
    D = width // (num_heads + 2 * num_kv_heads)
    kv = (B, T, num_kv_heads, D)
    return qkv.new_empty((B, T, num_heads, D)), qkv.new_empty(kv), qkv.new_empty(kv)


@torch.library.custom_op("attnres::qk_norm_rope_backward", mutates_args=())
def qk_norm_rope_backward_op(grad_q: Tensor, grad_k: Tensor, grad_v: Tensor, qkv: Tensor, cos: Tensor, sin: Tensor,
                             positions: Optional[Tensor], q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                             num_heads: int, num_kv_heads: int, normalize: bool, eps: float, interleaved: bool,
                             want_q_weight: bool, want_k_weight: bool) -> tuple[Tensor, Tensor, Tensor]:
    """Empty tensors where a weight gradient is not wanted."""
    dqkv, dwq, dwk = _rope_backward(grad_q, grad_k, grad_v, qkv, cos, sin, positions, q_weight, k_weight, num_heads,
                                    num_kv_heads, normalize, eps, interleaved, want_q_weight, want_k_weight)
    return dqkv, qkv.new_empty(0) if dwq is None else dwq, qkv.new_empty(0) if dwk is None else dwk


@qk_norm_rope_backward_op.register_fake
def _(grad_q, grad_k, grad_v, qkv, cos, sin, positions, q_weight, k_weight, num_heads, num_kv_heads, normalize, eps,
      interleaved, want_q_weight, want_k_weight):
    return (qkv.new_empty(qkv.shape), torch.empty_like(q_weight) if want_q_weight else qkv.new_empty(0),
            torch.empty_like(k_weight) if want_k_weight else qkv.new_empty(0))


def _rope_setup(ctx, inputs, output):
    ctx.how = inputs[6:]
    ctx.save_for_backward(*inputs[:6])


def _rope_bwd(ctx, grad_q, grad_k, grad_v):
    need = ctx.needs_input_grad
    qkv, cos, sin, positions, q_weight, k_weight = ctx.saved_tensors
    grads = qk_norm_rope_backward_op(grad_q, grad_k, grad_v, qkv, cos, sin, positions, q_weight, k_weight, *ctx.how,
                                     need[4], need[5])
    return (grads[0], None, None, None, grads[1] if need[4] else None, grads[2] if need[5] else None) + (None,) * 5


qk_norm_rope_op.register_autograd(_rope_bwd, setup_context=_rope_setup)


def qk_norm_rope(qkv: Tensor, num_heads: int, num_kv_heads: int, cos: Tensor, sin: Tensor,
                 positions: Optional[Tensor] = None, q_weight: Optional[Tensor] = None,
                 k_weight: Optional[Tensor] = None, eps: Optional[float] = None, normalize: bool = True,
                 interleaved: bool = True):
    """Heads of a fused projection, q and k RMS-normed per head and rotated by position.

    qkv [B, T, (num_heads + 2 num_kv_heads) * head_dim] (query, key, then value heads) gives
    q [B, T, num_heads, head_dim] and k, v [B, T, num_kv_heads, head_dim], dense. cos, sin float32
    [positions, rotary_dim / 2], rotary_dim <= head_dim; the remaining elements pass unrotated.
    positions [B, T] int32 or int64 (default: the token's index in its sequence); a token whose
    position lies outside the tables gets NaN queries and keys. interleaved pairs elements
    (2i, 2i + 1), otherwise (i, i + rotary_dim / 2). q_weight, k_weight [head_dim] multiply the normed
    heads. normalize=False leaves the norm out; eps defaults to float32's, as the model's norms have it.
    Differentiable in qkv and the weights."""
    how = (int(num_heads), int(num_kv_heads), bool(normalize), F32_EPS if eps is None else float(eps), bool(interleaved))
    if not _eager(qkv, cos, sin, positions, q_weight, k_weight):
        return qk_norm_rope_op(qkv, cos, sin, positions, q_weight, k_weight, *how)
    if _wants_grad(qkv, q_weight, k_weight):
        return _QkNormRope.apply(qkv, cos, sin, positions, q_weight, k_weight, *how)
    return _rope_forward(qkv, cos, sin, positions, q_weight, k_weight, *how)
