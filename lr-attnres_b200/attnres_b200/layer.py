"""Operators of the transformer layer around the depth read, over libattnres_b200.

  qk_norm_rope(...)       q/k/v split of a fused projection, per-head RMS norm of q and k and the
                          rotation by position in one pass (the steps of the reference's attention
                          between its projection and scaled_dot_product_attention)
  swiglu_projection(...)  the gated half of the MLP: both projections, silu and the product in one kernel

Every tensor argument must live on one CUDA device; the work is enqueued on that
device's current stream through the C ABI. There is no CPU fallback: a CPU tensor
is a RuntimeError, as is any argument that a check turns down.

Eager calls go straight to the compiled binding (_layer.so, csrc/layer_binding.cpp),
which checks, allocates and carries autograd. Under torch.compile, and for fake
tensors, a call is the attnres:: torch.library op of the same name, which traces and
has the same autograd formula.
"""
from typing import Optional

import torch
from torch import Tensor

from . import _native as N
from .ops import F32_EPS

_EAGER_TYPES = (Tensor, torch.nn.Parameter)
_binding = None


def _load():
    """The compiled binding; it is built together with the library it calls."""
    global _binding
    if _binding is None:
        N.load()
        try:
            from . import _layer
        except ImportError as e:
            raise N.AttnResError(f"attnres_b200/_layer.so cannot be loaded ({e}); build it with "
                                 "`python lr-attnres_b200/build.py`") from e
        _binding = _layer
    return _binding


def _eager(*tensors):
    """Whether a call on these tensors may go straight to the binding."""
    if torch.compiler.is_compiling():
        return False
    for t in tensors:
        if t is not None and type(t) not in _EAGER_TYPES:
            return False
    return True


# ---------------------------------------------------------------------------
# q/k norm and rotation
# ---------------------------------------------------------------------------
@torch.library.custom_op("attnres::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(qkv: Tensor, cos: Tensor, sin: Tensor, positions: Optional[Tensor], q_weight: Optional[Tensor],
                    k_weight: Optional[Tensor], num_heads: int, num_kv_heads: int, normalize: bool, eps: float,
                    interleaved: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _load().qk_norm_rope(qkv, num_heads, num_kv_heads, cos, sin, positions, q_weight, k_weight, eps, normalize,
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
    dqkv, dwq, dwk = _load().qk_norm_rope_backward(grad_q, grad_k, grad_v, qkv, cos, sin, positions, q_weight, k_weight,
                                                   num_heads, num_kv_heads, normalize, eps, interleaved, want_q_weight,
                                                   want_k_weight)
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
    eps = F32_EPS if eps is None else eps
    if _eager(qkv, cos, sin, positions, q_weight, k_weight):
        return _load().qk_norm_rope(qkv, num_heads, num_kv_heads, cos, sin, positions, q_weight, k_weight, eps, normalize,
                                    interleaved)
    return qk_norm_rope_op(qkv, cos, sin, positions, q_weight, k_weight, int(num_heads), int(num_kv_heads),
                           bool(normalize), float(eps), bool(interleaved))


# ---------------------------------------------------------------------------
# gated projection
# ---------------------------------------------------------------------------
@torch.library.custom_op("attnres::swiglu_projection", mutates_args=())
def swiglu_projection_op(x: Tensor, weight: Tensor) -> Tensor:
    return _load().swiglu_projection(x, weight)


@swiglu_projection_op.register_fake
def _(x, weight):
    return x.new_empty((*x.shape[:-1], weight.shape[0] // 2))


@torch.library.custom_op("attnres::swiglu_projection_backward", mutates_args=())
def swiglu_projection_backward_op(grad_h: Tensor, x: Tensor, weight: Tensor, want_x: bool,
                                  want_weight: bool) -> tuple[Tensor, Tensor]:
    """Empty tensors where a gradient is not wanted."""
    dx, dw = _load().swiglu_projection_backward(grad_h, x, weight, want_x, want_weight)
    return x.new_empty(0) if dx is None else dx, weight.new_empty(0) if dw is None else dw


@swiglu_projection_backward_op.register_fake
def _(grad_h, x, weight, want_x, want_weight):
    return x.new_empty(x.shape if want_x else (0,)), weight.new_empty(weight.shape if want_weight else (0,))


def _swiglu_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _swiglu_bwd(ctx, grad_h):
    x, weight = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw = swiglu_projection_backward_op(grad_h, x, weight, need[0], need[1])
    return dx if need[0] else None, dw if need[1] else None


swiglu_projection_op.register_autograd(_swiglu_bwd, setup_context=_swiglu_setup)


def swiglu_projection(x: Tensor, weight: Tensor) -> Tensor:
    """h = v * silu(g) with [v, g] = x weight^T, the model's MLP up to its output projection.

    x [..., in] float16 or bfloat16; weight [2 * hidden, in] holds the value rows, then the gate rows
    (the layout of the model's fc1), and is cast to x's type. Both widths are multiples of 8. The
    products are summed and gated in fp32, h [..., hidden] is rounded once. Differentiable in both;
    the backward forms v and g again rather than keeping them."""
    if _eager(x, weight):
        return _load().swiglu_projection(x, weight)
    return swiglu_projection_op(x, weight)
