"""Operators of the transformer layer around the depth read, over libattnres_b200.

  qk_norm_rope(...)       q/k/v split of a fused projection, per-head RMS norm of q and k and the
                          rotation by position in one pass (the steps of the reference's attention
                          between its projection and scaled_dot_product_attention)
  swiglu_projection(...)  the gated half of the MLP: both projections, silu and the product in one kernel
  KV4Cache, kv4_append, kv4_read, kv4_attention
                          keys and values of past tokens in 4 bits, in pages: written, read back, and
                          attended to by new tokens

Every tensor argument must live on one CUDA device; the work is enqueued on that
device's current stream through the C ABI. There is no CPU fallback: a CPU tensor
is a RuntimeError, as is any argument that a check turns down.

Eager calls go straight to the compiled binding (_layer.so, csrc/layer_binding.cpp),
which checks, allocates and carries autograd. Under torch.compile and other tracers,
dispatch modes and function transforms, and for fake tensors, a call is the attnres::
torch.library op of the same name, which traces and has the same autograd formula.
There are no forward-mode derivatives: a tensor with a tangent is a RuntimeError.
"""
from typing import Optional

import torch
from torch import Tensor

from . import _native as N
from .ops import F32_EPS

_EAGER_TYPES = (Tensor, torch.nn.Parameter)
_dispatch_modes, _jit_tracing = torch._C._len_torch_dispatch_stack, torch._C._is_tracing
_transform, _transforms = torch._C._functorch.peek_interpreter_stack, torch._C._functorch.get_interpreter_stack
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
    """Whether a call on these tensors may go straight to the binding: nobody traces, transforms or watches PyTorch's
    operators, which the binding's calls are none of."""
    if torch.compiler.is_compiling():
        return False
    if _dispatch_modes() or _jit_tracing():
        return False
    if _transform() is not None:
        if any(t.key() == torch._C._functorch.TransformType.Jvp for t in _transforms()):
            raise RuntimeError("attnres_b200: the layer operators have no forward-mode derivative")
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
    position lies outside the tables gets NaN in the rotated elements of its queries and keys. interleaved pairs elements
    (2i, 2i + 1), otherwise (i, i + rotary_dim / 2). q_weight, k_weight [head_dim] multiply the normed
    heads in their own type (float32 weights beside a 16-bit qkv are not rounded to it, nor their
    gradients). normalize=False leaves the norm out; eps defaults to float32's, as the model's norms have it.
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


# ---------------------------------------------------------------------------
# 4-bit key/value cache
# ---------------------------------------------------------------------------
class KV4Cache:
    """A pool of pages of keys and values in 4 bits.

    Groups of 32 elements of a head: element = low + step * code. k_codes, v_codes uint8 [pages,
    kv_heads, page_size, head_dim / 2]; k_params, v_params float16 [pages, kv_heads, page_size,
    head_dim / 32, 2] hold each group's step and low. A row's codes lie in the order in which the
    attention's tensor-core lanes take them (include/attnres_b200.h). page_size is a multiple of 16,
    head_dim of 32; 5 bits an element in all.

    The sequences' pages are the caller's to hand out: place t of sequence b is in page
    page_table[b, t // page_size]. Calls touch the places they are given and nothing else; a place
    without a valid page is skipped (bit 8 of the device status word tells)."""

    __slots__ = ("k_codes", "k_params", "v_codes", "v_params")

    def __init__(self, k_codes: Tensor, k_params: Tensor, v_codes: Tensor, v_params: Tensor):
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params

    @classmethod
    def empty(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device="cuda"):
        """A pool whose places hold nothing yet."""
        if page_size < 16 or page_size % 16 or head_dim < 32 or head_dim % 32:
            raise RuntimeError(f"attnres_b200: KV4Cache takes a page_size that is a multiple of 16 and a head_dim that is "
                               f"a multiple of 32, got {page_size} and {head_dim}")
        codes = (num_pages, num_kv_heads, page_size, head_dim // 2)
        params = (num_pages, num_kv_heads, page_size, head_dim // 32, 2)
        make = [torch.empty(shape, device=device, dtype=dt)
                for _ in range(2) for shape, dt in ((codes, torch.uint8), (params, torch.float16))]
        return cls(*make)

    def tensors(self):
        return self.k_codes, self.k_params, self.v_codes, self.v_params


@torch.library.custom_op("attnres::kv4_append", mutates_args=("k_codes", "k_params", "v_codes", "v_params"))
def kv4_append_op(k_codes: Tensor, k_params: Tensor, v_codes: Tensor, v_params: Tensor, k: Tensor, v: Tensor,
                  page_table: Tensor, start: Tensor, counts: Optional[Tensor]) -> None:
    _load().kv4_append(k_codes, k_params, v_codes, v_params, k, v, page_table, start, counts)


@kv4_append_op.register_fake
def _(k_codes, k_params, v_codes, v_params, k, v, page_table, start, counts):
    return None


@torch.library.custom_op("attnres::kv4_read", mutates_args=())
def kv4_read_op(k_codes: Tensor, k_params: Tensor, v_codes: Tensor, v_params: Tensor, page_table: Tensor, start: Tensor,
                tokens: int, counts: Optional[Tensor], dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    return _load().kv4_read(k_codes, k_params, v_codes, v_params, page_table, start, tokens, counts, dtype)


@kv4_read_op.register_fake
def _(k_codes, k_params, v_codes, v_params, page_table, start, tokens, counts, dtype):
    shape = (page_table.shape[0], tokens, k_codes.shape[1], 2 * k_codes.shape[3])
    return k_codes.new_empty(shape, dtype=dtype), k_codes.new_empty(shape, dtype=dtype)


@torch.library.custom_op("attnres::kv4_attention", mutates_args=())
def kv4_attention_op(q: Tensor, k_codes: Tensor, k_params: Tensor, v_codes: Tensor, v_params: Tensor, page_table: Tensor,
                     lengths: Tensor, counts: Optional[Tensor], scale: float) -> tuple[Tensor, Tensor]:
    return _load().kv4_attention(q, k_codes, k_params, v_codes, v_params, page_table, lengths, counts, scale, True)


@kv4_attention_op.register_fake
def _(q, k_codes, k_params, v_codes, v_params, page_table, lengths, counts, scale):
    return q.new_empty(q.shape), q.new_empty(q.shape[:3], dtype=torch.float32)


def kv4_append(cache: KV4Cache, k: Tensor, v: Tensor, page_table: Tensor, start: Tensor,
               counts: Optional[Tensor] = None) -> None:
    """Quantises the new tokens' keys and values into places start[b] .. of the cache.

    k, v [B, T, kv_heads, head_dim] float32, float16 or bfloat16, any strides; page_table int32
    [B, max_pages]; start int32 [B] (how many keys the sequence holds already); counts int32 [B]
    (default T): how many of the T tokens sequence b really has. Step and low are rounded to float16
    and each code is the nearest value to what will be read back. Groups that hold an infinity or a NaN
    read back as NaN, and so do those whose step or low overflows float16 (a least value beyond +-65504, or
    a range beyond 15 times that). No gradient."""
    if _eager(k, v, page_table, start, counts):
        _load().kv4_append(cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, k, v, page_table, start, counts)
    else:
        kv4_append_op(*cache.tensors(), k, v, page_table, start, counts)


def kv4_read(cache: KV4Cache, page_table: Tensor, start: Tensor, tokens: int, counts: Optional[Tensor] = None,
             dtype: torch.dtype = torch.bfloat16):
    """The keys and values in places start[b] .. start[b] + tokens of each sequence: two tensors
    [B, tokens, kv_heads, head_dim], zeros from counts[b] on and where there is no page."""
    if _eager(cache.k_codes, page_table, start, counts):
        return _load().kv4_read(cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, page_table, start, tokens,
                                counts, dtype)
    return kv4_read_op(*cache.tensors(), page_table, start, int(tokens), counts, dtype)


def kv4_attention(q: Tensor, cache: KV4Cache, page_table: Tensor, lengths: Tensor, counts: Optional[Tensor] = None,
                  scale: Optional[float] = None, return_lse: bool = False):
    """Attention of new tokens over the cache, which holds their own keys and values already.

    q [B, T, heads, head_dim] float16 or bfloat16, head_dim 64 or 128; query head h reads key head
    h // (heads / kv_heads). lengths int32 [B] counts a sequence's keys, the new ones among them; its
    token t < counts[b] (int32, default T) stands at place lengths[b] - counts[b] + t and sees the
    places up to its own, as far as the table goes (bit 8 of the status word tells of lengths beyond it). scale defaults to head_dim ** -0.5. Returns out [B, T, heads, head_dim] in
    q's type, with return_lse also the log of the softmax's sum, float32 [B, T, heads]. A token that
    sees nothing gives zeros and -inf. Meant for one to a few new tokens: the cache is read once for
    every 16 query rows of a key head. No gradient."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if _eager(q, cache.k_codes, page_table, lengths, counts):
        out, lse = _load().kv4_attention(q, cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, page_table,
                                         lengths, counts, scale, return_lse)
    else:
        out, lse = kv4_attention_op(q, *cache.tensors(), page_table, lengths, counts, float(scale))
    return (out, lse) if return_lse else out
