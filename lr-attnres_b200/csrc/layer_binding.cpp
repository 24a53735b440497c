// PyTorch binding of the transformer-layer operators: argument checks, output
// allocation, autograd and the calls into the C ABI, in C++ because at a decoding
// step's sizes the same steps in Python and ctypes take several times the kernels'
// own time (split + norm + rotation of four tokens: 26 us in Python, 3 us on the
// GPU). Errors are C++ exceptions that pybind11 turns into RuntimeError.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include "attnres_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return ATTNRES_DTYPE_F32;
    case at::kHalf: return ATTNRES_DTYPE_F16;
    case at::kBFloat16: return ATTNRES_DTYPE_BF16;
    default:
      TORCH_CHECK(false, "attnres_b200: unsupported dtype ", t.scalar_type(), "; use float32, float16 or bfloat16");
  }
}

void check_status(int rc, const char* what) {
  static const char* const names[] = {"ok", "invalid argument", "unsupported", "CUDA error", "workspace too small"};
  TORCH_CHECK(rc == ATTNRES_OK, what, " failed (", rc >= 0 && rc <= 4 ? names[rc] : "?", "): ", attnres_last_error());
}

void check_cuda(const char* what, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "attnres_b200: ", what, " inputs must be CUDA tensors (there is no CPU path)");
}
void check_device(const char* what, const Tensor& first, const Tensor& t) {
  TORCH_CHECK(!t.defined() || t.device() == first.device(), "attnres_b200: ", what,
              " inputs must be on one device, got ", first.device(), " and ", t.device());
}

Tensor or_undefined(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mut(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// An uninitialised tensor on `like`'s device, without the trip through the dispatcher
// (half the cost of at::empty, and a call makes up to three).
Tensor fresh(const Tensor& like, at::IntArrayRef shape, at::ScalarType dtype) {
  return at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt);
}
Tensor fresh(const Tensor& like, at::IntArrayRef shape) { return fresh(like, shape, like.scalar_type()); }

// Makes the tensor's device current and hands out its current stream.
struct Launch {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Launch(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream().stream()) {}
};

// The backward kernels have no gradient of their own: better no second derivative
// than a silent zero.
void check_first_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "attnres_b200: ", what, " cannot be differentiated twice (create_graph)");
}

// Nor is there a forward-mode derivative.
void check_no_tangent(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "attnres_b200: ", what, " has no forward-mode derivative");
}

// ---------------------------------------------------------------------------
// qk_norm_rope
// ---------------------------------------------------------------------------
struct RopeHow {
  int64_t q_heads, kv_heads;
  bool normalize;
  double eps;
  bool interleaved;
};

// The checked arguments of one call, rows made uniform where they were not.
struct RopeCall {
  Tensor qkv, cos, sin, positions, wq, wk;
  int64_t B, T, D, stride;
  int code, wide;  // the ABI's dtype; 64-bit positions
  at::ScalarType wtype;
  RopeHow how;

  RopeCall(const Tensor& qkv_, const Tensor& cos_, const Tensor& sin_, const Tensor& positions_, const Tensor& wq_,
           const Tensor& wk_, const RopeHow& h)
      : qkv(qkv_), positions(positions_), wide(0), how(h) {
    const char* what = "qk_norm_rope";
    check_cuda(what, qkv);
    for (const Tensor* t : {&cos_, &sin_, &positions_, &wq_, &wk_}) check_device(what, qkv, *t);
    TORCH_CHECK(h.q_heads >= 1 && h.kv_heads >= 1 && h.q_heads <= 4096 && h.kv_heads <= 4096,
                "attnres_b200: qk_norm_rope needs 1 to 4096 query and key heads, got ", h.q_heads, " and ", h.kv_heads);
    const int64_t heads = h.q_heads + 2 * h.kv_heads;
    TORCH_CHECK(qkv.dim() == 3 && qkv.size(2) > 0 && qkv.size(2) % heads == 0, "attnres_b200: qk_norm_rope takes qkv [B, T, (",
                h.q_heads, " + 2 * ", h.kv_heads, ") * head_dim], got ", qkv.sizes());
    B = qkv.size(0);
    T = qkv.size(1);
    const int64_t width = qkv.size(2);
    D = width / heads;
    code = dtype_code(qkv);
    stride = T > 1 ? qkv.stride(1) : (B > 1 ? qkv.stride(0) : width);
    if (qkv.stride(2) != 1 || stride < width || (T > 1 && B > 1 && qkv.stride(0) != T * stride)) {
      qkv = qkv.contiguous();  // rows of one stride that do not overlap
      stride = width;
    }
    TORCH_CHECK(cos_.dim() == 2 && cos_.sizes() == sin_.sizes(),
                "attnres_b200: qk_norm_rope takes cos and sin [positions, rotary_dim / 2], got ", cos_.sizes(), " and ",
                sin_.sizes());
    TORCH_CHECK(cos_.scalar_type() == at::kFloat && sin_.scalar_type() == at::kFloat,
                "attnres_b200: qk_norm_rope takes float32 cos and sin");
    cos = cos_.contiguous();
    sin = sin_.contiguous();
    TORCH_CHECK(2 * cos.size(1) <= D, "attnres_b200: qk_norm_rope rotary_dim ", 2 * cos.size(1), " exceeds head_dim ", D);
    if (positions.defined()) {
      wide = positions.scalar_type() == at::kLong;
      TORCH_CHECK((wide || positions.scalar_type() == at::kInt) && positions.dim() == 2 && positions.size(0) == B &&
                      positions.size(1) == T,
                  "attnres_b200: qk_norm_rope takes positions [B, T] int32 or int64");
      positions = positions.contiguous();
    } else {
      TORCH_CHECK(B == 0 || cos.size(1) == 0 || T <= cos.size(0), "attnres_b200: qk_norm_rope has ", T,
                  " tokens and tables of ", cos.size(0), " positions");
    }
    for (const Tensor* w : {&wq_, &wk_})
      TORCH_CHECK(!w->defined() || (w->dim() == 1 && w->size(0) == D),
                  "attnres_b200: qk_norm_rope weights are [head_dim] = [", D, "]");
    // weights of the data's type go as they are, others in fp32
    wtype = qkv.scalar_type();
    for (const Tensor* w : {&wq_, &wk_})
      if (w->defined() && w->scalar_type() != qkv.scalar_type()) wtype = at::kFloat;
    if (wq_.defined()) wq = wq_.to(wtype).contiguous();
    if (wk_.defined()) wk = wk_.to(wtype).contiguous();
    if (wtype != qkv.scalar_type()) code |= ATTNRES_WEIGHTS_F32;
  }
  int64_t tokens() const { return B * T; }
  int64_t seq() const { return T > 0 ? T : 1; }
};

std::vector<Tensor> rope_forward(const Tensor& qkv, const Tensor& cos, const Tensor& sin, const Tensor& positions,
                                 const Tensor& wq, const Tensor& wk, const RopeHow& how) {
  const RopeCall c(qkv, cos, sin, positions, wq, wk, how);
  const Tensor q = fresh(qkv, {c.B, c.T, how.q_heads, c.D});
  const Tensor k = fresh(qkv, {c.B, c.T, how.kv_heads, c.D});
  const Tensor v = fresh(qkv, {c.B, c.T, how.kv_heads, c.D});
  const Launch on(c.qkv);
  check_status(attnres_qk_norm_rope_forward(
                   c.tokens(), c.seq(), how.q_heads, how.kv_heads, c.D, 2 * c.cos.size(1), c.code, ptr(c.qkv), c.stride,
                   static_cast<const float*>(ptr(c.cos)), static_cast<const float*>(ptr(c.sin)), c.cos.size(0),
                   ptr(c.positions), c.wide, ptr(c.wq), ptr(c.wk), how.normalize, how.eps, how.interleaved, mut(q),
                   mut(k), mut(v), on.stream),
               "attnres_qk_norm_rope_forward");
  return {q, k, v};
}

// {d qkv, d q weight, d k weight}, undefined where not wanted.
std::vector<Tensor> rope_backward(const std::array<Tensor, 3>& grads, const Tensor& qkv, const Tensor& cos,
                                  const Tensor& sin, const Tensor& positions, const Tensor& wq, const Tensor& wk,
                                  const RopeHow& how, bool want_wq, bool want_wk) {
  const RopeCall c(qkv, cos, sin, positions, wq, wk, how);
  Tensor g[3];
  int64_t strides[9];
  for (int i = 0; i < 3; ++i) {
    const int64_t heads = i == 0 ? how.q_heads : how.kv_heads;
    g[i] = grads[i];
    if (!g[i].defined()) {  // an output that took no part in the loss
      g[i] = at::zeros({1}, qkv.options()).expand({c.B, c.T, heads, c.D});
    }
    TORCH_CHECK(g[i].dim() == 4 && g[i].size(0) == c.B && g[i].size(1) == c.T && g[i].size(2) == heads &&
                    g[i].size(3) == c.D,
                "attnres_b200: qk_norm_rope backward takes gradients of its outputs' shapes");
    check_device("qk_norm_rope", qkv, g[i]);
    if (g[i].scalar_type() != qkv.scalar_type() || g[i].stride(3) != 1) g[i] = g[i].to(qkv.scalar_type()).contiguous();
    for (int j = 0; j < 3; ++j) strides[3 * i + j] = g[i].stride(j);
  }
  const Tensor dqkv = fresh(qkv, {c.B, c.T, (how.q_heads + 2 * how.kv_heads) * c.D});
  Tensor dwq, dwk, workspace;
  size_t bytes = 0;
  if (want_wq || want_wk) {
    const Launch on(c.qkv);
    bytes = attnres_qk_norm_rope_backward_workspace_bytes(c.D);
    workspace = fresh(qkv, {static_cast<int64_t>(bytes)}, at::kByte);
    if (want_wq) dwq = fresh(qkv, {c.D}, c.wtype);
    if (want_wk) dwk = fresh(qkv, {c.D}, c.wtype);
  }
  const Launch on(c.qkv);
  check_status(attnres_qk_norm_rope_backward(
                   c.tokens(), c.seq(), how.q_heads, how.kv_heads, c.D, 2 * c.cos.size(1), c.code, ptr(c.qkv), c.stride,
                   static_cast<const float*>(ptr(c.cos)), static_cast<const float*>(ptr(c.sin)), c.cos.size(0),
                   ptr(c.positions), c.wide, ptr(c.wq), ptr(c.wk), how.normalize, how.eps, how.interleaved, ptr(g[0]),
                   ptr(g[1]), ptr(g[2]), strides, mut(dqkv), mut(dwq), mut(dwk), mut(workspace), bytes, on.stream),
               "attnres_qk_norm_rope_backward");
  if (dwq.defined()) dwq = dwq.to(wq.scalar_type());
  if (dwk.defined()) dwk = dwk.to(wk.scalar_type());
  return {dqkv, dwq, dwk};
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& cos, const Tensor& sin,
                               const OptTensor& positions, const OptTensor& q_weight, const OptTensor& k_weight,
                               const RopeHow& how) {
    const Tensor pos = or_undefined(positions), wq = or_undefined(q_weight), wk = or_undefined(k_weight);
    ctx->save_for_backward({qkv, cos, sin, pos, wq, wk});
    ctx->saved_data["heads"] = std::vector<int64_t>{how.q_heads, how.kv_heads, how.normalize, how.interleaved};
    ctx->saved_data["eps"] = how.eps;
    ctx->set_materialize_grads(false);
    return rope_forward(qkv, cos, sin, pos, wq, wk, how);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    check_first_order("qk_norm_rope");
    const auto s = ctx->get_saved_variables();
    const auto h = ctx->saved_data["heads"].toIntVector();
    const RopeHow how{h[0], h[1], h[2] != 0, ctx->saved_data["eps"].toDouble(), h[3] != 0};
    // the context numbers the inputs that are there: qkv, cos, sin, positions, weights
    size_t at = s[3].defined() ? 4 : 3;
    const bool want_wq = s[4].defined() && ctx->needs_input_grad(at++);
    const bool want_wk = s[5].defined() && ctx->needs_input_grad(at);
    const auto d = rope_backward({g[0], g[1], g[2]}, s[0], s[1], s[2], s[3], s[4], s[5], how, want_wq, want_wk);
    return {d[0], Tensor(), Tensor(), Tensor(), d[1], d[2], Tensor()};
  }
};

py::tuple tuple3(const std::vector<Tensor>& t) { return py::make_tuple(t[0], t[1], t[2]); }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

py::tuple py_qk_norm_rope(const Tensor& qkv, int64_t q_heads, int64_t kv_heads, const Tensor& cos, const Tensor& sin,
                          const OptTensor& positions, const OptTensor& q_weight, const OptTensor& k_weight, double eps,
                          bool normalize, bool interleaved) {
  const RopeHow how{q_heads, kv_heads, normalize, eps, interleaved};
  const Tensor pos = or_undefined(positions), wq = or_undefined(q_weight), wk = or_undefined(k_weight);
  check_no_tangent("qk_norm_rope", {&qkv, &cos, &sin, &wq, &wk});
  if (wants_grad({&qkv, &wq, &wk}))
    return tuple3(QkNormRope::apply(qkv, cos, sin, positions, q_weight, k_weight, how));
  return tuple3(rope_forward(qkv, cos, sin, pos, wq, wk, how));
}

py::tuple py_qk_norm_rope_backward(const Tensor& gq, const Tensor& gk, const Tensor& gv, const Tensor& qkv,
                                   const Tensor& cos, const Tensor& sin, const OptTensor& positions,
                                   const OptTensor& q_weight, const OptTensor& k_weight, int64_t q_heads,
                                   int64_t kv_heads, bool normalize, double eps, bool interleaved, bool want_wq,
                                   bool want_wk) {
  const RopeHow how{q_heads, kv_heads, normalize, eps, interleaved};
  return tuple3(rope_backward({gq, gk, gv}, qkv, cos, sin, or_undefined(positions), or_undefined(q_weight),
                              or_undefined(k_weight), how, want_wq, want_wk));
}

// ---------------------------------------------------------------------------
// swiglu_projection
// ---------------------------------------------------------------------------
// t as `rows` rows of `width` elements, 16-byte aligned and one stride apart without
// overlap; a copy only where it does not lie like that.
struct Rows {
  Tensor t;
  int64_t stride;

  Rows() = default;
  Rows(const Tensor& from, int64_t rows, int64_t width) : t(from), stride(width) {
    if (!t.is_contiguous()) {
      if (t.dim() != 2) t = t.reshape({rows, width});
      if (rows > 1) stride = t.stride(0);
      if (t.stride(1) != 1 || stride < width || stride % 8 != 0) {
        t = t.contiguous();
        stride = width;
      }
    }
    if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0) {
      t = t.clone(at::MemoryFormat::Contiguous);
      stride = width;
    }
  }
};

struct SwigluCall {
  Rows x, w;
  int64_t N, C, F;
  int code;

  SwigluCall(const Tensor& x_, const Tensor& w_) {
    const char* what = "swiglu_projection";
    check_cuda(what, x_);
    check_device(what, x_, w_);
    TORCH_CHECK(x_.scalar_type() == at::kHalf || x_.scalar_type() == at::kBFloat16,
                "attnres_b200: swiglu_projection takes float16 or bfloat16, got ", x_.scalar_type());
    TORCH_CHECK(x_.dim() >= 1 && w_.dim() == 2 && w_.size(1) == x_.size(-1) && w_.size(0) % 2 == 0,
                "attnres_b200: swiglu_projection takes x [..., in] and weight [2 * hidden, in], got ", x_.sizes(), " and ",
                w_.sizes());
    C = x_.size(-1);
    F = w_.size(0) / 2;
    TORCH_CHECK(C > 0 && F > 0 && C % 8 == 0 && F % 8 == 0 && C < (1 << 28) && F < (1 << 28),
                "attnres_b200: swiglu_projection takes widths that are multiples of 8, got in ", C, " and hidden ", F);
    N = x_.numel() / C;
    code = dtype_code(x_);
    x = Rows(x_, N, C);
    w = Rows(w_.to(x_.scalar_type()), 2 * F, C);
  }
};

std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = last;
  return shape;
}

Tensor swiglu_forward(const Tensor& x, const Tensor& w) {
  const SwigluCall c(x, w);
  const Tensor h = fresh(x, with_last(x, c.F));
  const Launch on(c.x.t);
  check_status(attnres_swiglu_forward(c.N, c.C, c.F, c.code, ptr(c.x.t), c.x.stride, ptr(c.w.t), c.w.stride, mut(h),
                                      on.stream),
               "attnres_swiglu_forward");
  return h;
}

// {dx, dW}, undefined where not wanted.
std::vector<Tensor> swiglu_backward(const Tensor& grad_h, const Tensor& x, const Tensor& w, bool want_x, bool want_w) {
  const SwigluCall c(x, w);
  check_device("swiglu_projection", x, grad_h);
  TORCH_CHECK(grad_h.dim() == x.dim() && grad_h.numel() == c.N * c.F && (x.dim() == 0 || grad_h.size(-1) == c.F),
              "attnres_b200: swiglu_projection backward takes a gradient of its output's shape");
  const Rows g(grad_h.to(x.scalar_type()), c.N, c.F);
  Tensor dx, dw;
  if (want_x) dx = fresh(x, x.sizes());
  if (want_w) dw = fresh(x, {2 * c.F, c.C});
  const int64_t bytes = attnres_swiglu_backward_workspace_bytes(c.N, c.F);
  const Tensor workspace = fresh(x, {bytes}, at::kByte);
  const Launch on(c.x.t);
  check_status(attnres_swiglu_backward(c.N, c.C, c.F, c.code, ptr(c.x.t), c.x.stride, ptr(c.w.t), c.w.stride, ptr(g.t),
                                       g.stride, mut(dx), mut(dw), mut(workspace), bytes, on.stream),
               "attnres_swiglu_backward");
  if (want_w) dw = dw.to(w.scalar_type());
  return {dx, dw};
}

struct Swiglu : torch::autograd::Function<Swiglu> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w) {
    ctx->save_for_backward({x, w});
    return swiglu_forward(x, w);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    check_first_order("swiglu_projection");
    const auto s = ctx->get_saved_variables();
    return swiglu_backward(g[0], s[0], s[1], ctx->needs_input_grad(0), ctx->needs_input_grad(1));
  }
};

Tensor py_swiglu(const Tensor& x, const Tensor& w) {
  check_no_tangent("swiglu_projection", {&x, &w});
  if (wants_grad({&x, &w})) return Swiglu::apply(x, w);
  return swiglu_forward(x, w);
}

py::tuple py_swiglu_backward(const Tensor& grad_h, const Tensor& x, const Tensor& w, bool want_x, bool want_w) {
  const auto d = swiglu_backward(grad_h, x, w, want_x, want_w);
  return py::make_tuple(d[0], d[1]);
}

// ---------------------------------------------------------------------------
// 4-bit cache
// ---------------------------------------------------------------------------
struct PoolCall {
  Tensor kc, kp, vc, vp, table, per_sequence, counts;
  int64_t pages, heads, page, D, B, max_pages;

  PoolCall(const char* what, const Tensor& kc_, const Tensor& kp_, const Tensor& vc_, const Tensor& vp_,
           const Tensor& table_, const Tensor& per_, const OptTensor& counts_)
      : kc(kc_), kp(kp_), vc(vc_), vp(vp_), table(table_), per_sequence(per_), counts(or_undefined(counts_)) {
    check_cuda(what, kc);
    for (const Tensor* t : {&kp, &vc, &vp, &table, &per_sequence, &counts}) check_device(what, kc, *t);
    TORCH_CHECK(kc.dim() == 4 && kc.scalar_type() == at::kByte, "attnres_b200: ", what,
                " takes codes uint8 [pages, kv_heads, page_size, head_dim / 2]");
    pages = kc.size(0);
    heads = kc.size(1);
    page = kc.size(2);
    D = 2 * kc.size(3);
    TORCH_CHECK(page > 0 && page % 16 == 0 && D > 0 && D % 32 == 0 && D <= 512 && heads > 0, "attnres_b200: ", what,
                " takes a page_size that is a multiple of 16 and a head_dim that is a multiple of 32 up to 512, got ", page,
                " and ", D);
    TORCH_CHECK(vc.sizes() == kc.sizes() && vc.scalar_type() == at::kByte, "attnres_b200: ", what,
                " takes key and value codes of one shape");
    for (const Tensor* p : {&kp, &vp})
      TORCH_CHECK(p->scalar_type() == at::kHalf && p->dim() == 5 && p->size(0) == pages && p->size(1) == heads &&
                      p->size(2) == page && p->size(3) == D / 32 && p->size(4) == 2,
                  "attnres_b200: ", what, " takes params float16 [pages, kv_heads, page_size, head_dim / 32, 2]");
    for (const Tensor* p : {&kc, &kp, &vc, &vp})
      TORCH_CHECK(p->is_contiguous() && reinterpret_cast<uintptr_t>(p->const_data_ptr()) % 16 == 0, "attnres_b200: ", what,
                  " takes contiguous, 16-byte aligned pool tensors");
    TORCH_CHECK(table.dim() == 2 && table.scalar_type() == at::kInt, "attnres_b200: ", what,
                " takes page_table int32 [batch, max_pages]");
    B = table.size(0);
    max_pages = table.size(1);
    TORCH_CHECK(per_sequence.dim() == 1 && per_sequence.size(0) == B && per_sequence.scalar_type() == at::kInt,
                "attnres_b200: ", what, " takes start or lengths int32 [batch]");
    TORCH_CHECK(!counts.defined() || (counts.dim() == 1 && counts.size(0) == B && counts.scalar_type() == at::kInt),
                "attnres_b200: ", what, " takes counts int32 [batch]");
    if (!table.is_contiguous()) table = table.contiguous();
    if (!per_sequence.is_contiguous()) per_sequence = per_sequence.contiguous();
    if (counts.defined() && !counts.is_contiguous()) counts = counts.contiguous();
  }
  const int* ints(const Tensor& t) const { return static_cast<const int*>(ptr(t)); }
};

// A [B, T, heads, D] tensor with a dense last dim; its strides.
Tensor rows4(const char* what, const char* name, const Tensor& t, int64_t B, int64_t heads, int64_t D, int64_t (&strides)[3]) {
  TORCH_CHECK(t.dim() == 4 && t.size(0) == B && t.size(2) == heads && t.size(3) == D, "attnres_b200: ", what, " takes ",
              name, " [", B, ", tokens, ", heads, ", ", D, "], got ", t.sizes());
  const Tensor r = t.stride(3) == 1 ? t : t.contiguous();
  for (int i = 0; i < 3; ++i) strides[i] = r.stride(i);
  return r;
}

void no_gradient(const char* what, std::initializer_list<const Tensor*> ts) {
  check_no_tangent(what, ts);
  TORCH_CHECK(!wants_grad(ts), "attnres_b200: ", what, " has no gradient; call it under torch.no_grad() or detach its inputs");
}

void py_kv4_append(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp, const Tensor& k, const Tensor& v,
                   const Tensor& table, const Tensor& start, const OptTensor& counts) {
  const char* what = "kv4_append";
  const PoolCall c(what, kc, kp, vc, vp, table, start, counts);
  check_device(what, kc, k);
  check_device(what, kc, v);
  no_gradient(what, {&k, &v});
  int64_t ks[3], vs[3];
  const Tensor kr = rows4(what, "k", k, c.B, c.heads, c.D, ks), vr = rows4(what, "v", v, c.B, c.heads, c.D, vs);
  TORCH_CHECK(kr.size(1) == vr.size(1) && kr.scalar_type() == vr.scalar_type(),
              "attnres_b200: kv4_append takes k and v of one shape and type");
  const Launch on(kc);
  check_status(attnres_kv4_append(mut(kc), mut(kp), mut(vc), mut(vp), c.pages, c.heads, c.page, c.D, c.ints(c.table),
                                  c.max_pages, c.max_pages, c.ints(c.per_sequence), c.ints(c.counts), c.B, kr.size(1),
                                  dtype_code(kr), ptr(kr), ks, ptr(vr), vs, on.stream),
               "attnres_kv4_append");
}

py::tuple py_kv4_read(const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp, const Tensor& table,
                      const Tensor& start, int64_t tokens, const OptTensor& counts, at::ScalarType dtype) {
  const PoolCall c("kv4_read", kc, kp, vc, vp, table, start, counts);
  TORCH_CHECK(tokens >= 0 && tokens < (1 << 30), "attnres_b200: kv4_read takes a number of tokens, got ", tokens);
  const Tensor k = fresh(kc, {c.B, tokens, c.heads, c.D}, dtype);
  const Tensor v = fresh(kc, {c.B, tokens, c.heads, c.D}, dtype);
  const Launch on(kc);
  check_status(attnres_kv4_read(ptr(kc), ptr(kp), ptr(vc), ptr(vp), c.pages, c.heads, c.page, c.D, c.ints(c.table),
                                c.max_pages, c.max_pages, c.ints(c.per_sequence), c.ints(c.counts), c.B, tokens,
                                dtype_code(k), mut(k), mut(v), on.stream),
               "attnres_kv4_read");
  return py::make_tuple(k, v);
}

py::tuple py_kv4_attention(const Tensor& q, const Tensor& kc, const Tensor& kp, const Tensor& vc, const Tensor& vp,
                           const Tensor& table, const Tensor& lengths, const OptTensor& counts, double scale,
                           bool want_lse) {
  const char* what = "kv4_attention";
  const PoolCall c(what, kc, kp, vc, vp, table, lengths, counts);
  check_device(what, kc, q);
  no_gradient(what, {&q});
  TORCH_CHECK(q.dim() == 4 && q.size(2) > 0 && q.size(2) % c.heads == 0, "attnres_b200: kv4_attention takes q [", c.B,
              ", tokens, a multiple of ", c.heads, " heads, ", c.D, "], got ", q.sizes());
  TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
              "attnres_b200: kv4_attention takes float16 or bfloat16 queries, got ", q.scalar_type());
  TORCH_CHECK(c.D == 64 || c.D == 128, "attnres_b200: kv4_attention is built for head_dim 64 and 128, got ", c.D);
  const int64_t T = q.size(1), Hq = q.size(2);
  int64_t qs[3];
  const Tensor qr = rows4(what, "q", q, c.B, Hq, c.D, qs);
  const Tensor out = fresh(q, {c.B, T, Hq, c.D});
  Tensor lse, workspace;
  if (want_lse) lse = fresh(q, {c.B, T, Hq}, at::kFloat);
  const Launch on(kc);
  const int64_t bytes =
      c.B && T ? attnres_kv4_attention_workspace_bytes(c.heads, c.page, c.D, c.max_pages, c.B, T, Hq) : 0;
  if (bytes) workspace = fresh(kc, {bytes}, at::kByte);
  check_status(attnres_kv4_attention(ptr(kc), ptr(kp), ptr(vc), ptr(vp), c.pages, c.heads, c.page, c.D, c.ints(c.table),
                                     c.max_pages, c.max_pages, c.ints(c.per_sequence), c.ints(c.counts), c.B, T, Hq,
                                     dtype_code(qr), ptr(qr), qs, scale, mut(out), static_cast<float*>(mut(lse)),
                                     mut(workspace), bytes, on.stream),
               "attnres_kv4_attention");
  return py::make_tuple(out, lse);
}

}  // namespace

PYBIND11_MODULE(_layer, m) {
  m.def("kv4_append", &py_kv4_append);
  m.def("kv4_read", &py_kv4_read);
  m.def("kv4_attention", &py_kv4_attention);
  m.def("swiglu_projection", &py_swiglu);
  m.def("swiglu_projection_backward", &py_swiglu_backward);
  m.def("qk_norm_rope", &py_qk_norm_rope);
  m.def("qk_norm_rope_backward", &py_qk_norm_rope_backward);
}
