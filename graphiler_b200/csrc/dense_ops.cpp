// my_ops::* registrations of the dense operators of a transformer block on node rows: norm, 8-bit rows and product, gated
// feed-forward.  Thin shims over the C ABI (include/gphl.h) like torch_ops.cpp: validate, allocate on the inputs' device from PyTorch's
// caching allocator (a captured call's scratch is private to its graph), launch on the current stream.  `rms_norm` and
// `gated_linear` are differentiable; the others record no gradients.  No counterpart in the reference's registry.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>
#include <torch/script.h>

#include <tuple>

#include "gphl.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

constexpr int64_t BLOCK = 128;        // values of one 8-bit scale
// Rows of at most this width keep no projections for the backward pass of the gated feed-forward: making g and u again costs 4 k operations
// an element, storing and reading them 16 bytes.  A step in bf16, made again / kept: 300,000 x 256 -> 1024 1.40 / 1.74 ms, 100,000 x 1024 ->
// 1024 1.35 / 1.27 ms.
constexpr int64_t RECOMPUTE_K = 768;

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
void check_rc(int rc, const char *what) { TORCH_CHECK(rc == GPHL_OK, what, " failed (", rc, "): ", gphl_last_error()); }
void *stream_of(const Tensor &x) { return at::cuda::getCurrentCUDAStream(x.get_device()).stream(); }
const void *ptr(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
void *mut(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

int dtype_of(torch::ScalarType t, const char *what) {
  TORCH_CHECK(t == torch::kFloat32 || t == torch::kBFloat16 || t == torch::kFloat16, what, " must be float32, bfloat16 or float16");
  return t == torch::kFloat32 ? GPHL_F32 : t == torch::kBFloat16 ? GPHL_BF16 : GPHL_F16;
}
void on_device(std::initializer_list<const Tensor *> ts) {
  const Tensor *first = nullptr;
  for (const Tensor *t : ts) {
    if (!t || !t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), "operators need CUDA tensors (there is no CPU path)");
    if (!first) first = t;
    TORCH_CHECK(t->device() == first->device(), "all tensors must live on one device");
  }
}
void contiguous(std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts) TORCH_CHECK(!t || !t->defined() || t->is_contiguous(), "operators need contiguous tensors");
}
// New memory beside `t`, straight from the caching allocator: through the dispatcher each tensor and each view of it costs the host a microsecond.
Tensor plain(const Tensor &t, torch::ScalarType s, at::IntArrayRef shape) { return Tensor(at::detail::empty_cuda(shape, s, t.device(), c10::nullopt)); }
// A tensor made here and not yet handed out, seen with other sizes and strides.
Tensor as(Tensor t, at::IntArrayRef sizes, at::IntArrayRef strides) {
  t.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides);
  return t;
}
Tensor scratch(int64_t bytes, const Tensor &like) {
  return bytes > 0 ? plain(like, torch::kUInt8, {bytes}) : Tensor();
}

// ---- norm -------------------------------------------------------------------------------------------------------

int norm_args(const Tensor &x, const Tensor &w, double eps, const Tensor &res, const char *what) {
  on_device({&x, &w, &res});
  contiguous({&x, &w, &res});
  TORCH_CHECK(x.dim() == 2 && w.dim() == 1 && w.size(0) == x.size(1), what, " needs rows (m, n) and a weight of n values");
  TORCH_CHECK(!res.defined() || (res.sizes() == x.sizes() && res.scalar_type() == x.scalar_type()), what, ": the residual must have the rows' shape and type");
  TORCH_CHECK(w.scalar_type() == x.scalar_type() || w.scalar_type() == torch::kFloat32, what, ": the weight must have the rows' type or be float32");
  TORCH_CHECK(eps >= 0, what, ": eps must not be negative");
  return dtype_of(x.scalar_type(), "rows");
}

// (y, r, rstd); r is undefined without a residual, rstd unless wanted
std::tuple<Tensor, Tensor, Tensor> norm_run(const Tensor &x, const Tensor &w, double eps, const Tensor &res, bool want_rstd) {
  const int dt = norm_args(x, w, eps, res, "rms_norm");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = plain(x, x.scalar_type(), x.sizes()), r, rstd;
  if (res.defined()) r = plain(x, x.scalar_type(), x.sizes());
  if (want_rstd) rstd = plain(x, torch::kFloat32, {x.size(0)});
  check_rc(gphl_rms_norm(dt, x.size(0), x.size(1), ptr(x), ptr(res), ptr(w), dtype_of(w.scalar_type(), "weight"), (float)eps, mut(y), mut(r),
                         static_cast<float *>(mut(rstd)), stream_of(x)),
           "rms_norm");
  return {y, r, rstd};
}

std::tuple<Tensor, Tensor> rms_norm_grad(const Tensor &r, const Tensor &w, const Tensor &rstd, const Tensor &dy, const OptTensor &dr_) {
  const Tensor dr = dr_.value_or(Tensor());
  const int dt = norm_args(r, w, 0.0, Tensor(), "rms_norm_grad");
  on_device({&r, &rstd, &dy, &dr});
  contiguous({&rstd, &dy, &dr});
  TORCH_CHECK(dy.sizes() == r.sizes() && dy.scalar_type() == r.scalar_type() && (!dr.defined() || (dr.sizes() == r.sizes() && dr.scalar_type() == r.scalar_type())),
              "rms_norm_grad: gradients must have the rows' shape and type");
  TORCH_CHECK(rstd.scalar_type() == torch::kFloat32 && rstd.dim() == 1 && rstd.size(0) == r.size(0), "rms_norm_grad: rstd must hold one float32 per row");
  c10::cuda::CUDAGuard guard(r.device());
  Tensor dx = plain(r, r.scalar_type(), r.sizes()), dw = plain(w, w.scalar_type(), w.sizes());
  Tensor ws = scratch(gphl_rms_norm_grad_workspace_bytes(dt, r.size(0), r.size(1)), r);
  check_rc(gphl_rms_norm_grad(dt, r.size(0), r.size(1), ptr(r), ptr(w), dtype_of(w.scalar_type(), "weight"), static_cast<const float *>(ptr(rstd)), ptr(dy),
                              ptr(dr), mut(dx), mut(dw), mut(ws), stream_of(r)),
           "rms_norm_grad");
  return {dx, dw};
}

std::vector<Tensor> rms_norm_rows(const Tensor &x, const Tensor &w, double eps, const OptTensor &res, bool return_rstd) {
  auto [y, r, rstd] = norm_run(x, w, eps, res.value_or(Tensor()), return_rstd);
  std::vector<Tensor> out{y};
  if (r.defined()) out.push_back(r);
  if (return_rstd) out.push_back(rstd);
  return out;
}

// (..., n) as rows; an empty last dimension keeps the number of rows.
Tensor rows_of(const Tensor &t) {
  if (t.dim() == 2 && t.is_contiguous()) return t;
  int64_t m = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) m *= t.size(i);
  return t.reshape({m, t.size(-1)}).contiguous();
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, double eps, const OptTensor &res_) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor res = res_.value_or(Tensor());
    ctx->set_materialize_grads(false);
    const Tensor rows = rows_of(x);
    auto [y, r, rstd] = norm_run(rows, w, eps, res.defined() ? rows_of(res) : res, true);
    ctx->saved_data["shape"] = x.sizes().vec();
    // kept as the caller's own tensors, so that a change in place before the backward pass is noticed
    if (r.defined()) r = r.view(x.sizes());
    ctx->save_for_backward({r.defined() ? r : x.is_contiguous() ? x : rows, w, rstd});
    variable_list out{y.view(x.sizes())};
    if (r.defined()) out.push_back(r);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "rms_norm: first derivatives only (create_graph is not supported)");
    const Tensor dy = grads[0], dr = grads.size() > 1 ? grads[1] : Tensor();
    if (!dy.defined()) return {dr, Tensor(), Tensor(), dr};         // only the sum went on: its gradient passes through
    const auto saved = ctx->get_saved_variables();
    auto [dx, dw] = rms_norm_grad(rows_of(saved[0]), saved[1], saved[2], rows_of(dy), dr.defined() ? OptTensor(rows_of(dr)) : c10::nullopt);
    dx = dx.view(ctx->saved_data["shape"].toIntVector());
    return {dx, dw, Tensor(), grads.size() > 1 ? dx : Tensor()};    // two outputs: there was a residual
  }
};

// A tangent would be dropped without a word where nothing else wants gradients.
void no_tangents(std::initializer_list<const Tensor *> ts, const char *what) {
  for (const Tensor *t : ts) TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what, ": no derivatives in forward mode");
}

bool wants_grad(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A captured backward pass must not reach gradients that belong to the default stream: the engine would make that stream wait for the
// capture, which ends the process.  An input's gradient belongs to the stream of the graph that it is part of: for a leaf, of any living graph.
// (Other streams may join a capture: warm-up on a side stream, with its outputs kept, is fine.)
void capturable(std::initializer_list<const Tensor *> ts, const char *what) {
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return;
  for (const Tensor *t : ts) {
    if (!t->defined() || !t->requires_grad()) continue;
    const auto node = t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn();
    const auto stream = node ? node->stream() : std::nullopt;
    TORCH_CHECK(!stream || *stream != c10::cuda::getDefaultCUDAStream(t->get_device()).unwrap(), what,
                ": an input's gradients belong to a graph that was recorded on the default stream, which a capture cannot reach (drop that graph's outputs first)");
  }
}

std::vector<Tensor> rms_norm(const Tensor &x, const Tensor &w, double eps, const OptTensor &res_) {
  const Tensor res = res_.value_or(Tensor());
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 1 && x.size(-1) == w.size(0), "rms_norm needs rows (..., n) and a weight of n values");
  TORCH_CHECK(!res.defined() || res.sizes() == x.sizes(), "rms_norm: the residual must have the rows' shape and type");
  on_device({&x, &w, &res});
  no_tangents({&x, &w, &res}, "rms_norm");
  const Tensor wc = w.contiguous();
  if (wants_grad({&x, &w, &res})) {
    capturable({&x, &w, &res}, "rms_norm");
    return RmsNorm::apply(x, wc, eps, res_);
  }
  auto [y, r, rstd] = norm_run(rows_of(x), wc, eps, res.defined() ? rows_of(res) : res, false);
  std::vector<Tensor> out{y.view(x.sizes())};
  if (r.defined()) out.push_back(r.view(x.sizes()));
  return out;
}

// ---- 8-bit rows and weights ---------------------------------------------------------------------------------------

struct Codes {
  Tensor q, s;
};
// Empty codes as the quantisers lay them out: rows padded to 16 bytes, a block's scales of consecutive rows together.
Codes new_rows(int64_t m, int64_t n, const Tensor &like) {
  const int64_t row = up(n, 16), blocks = up(n, BLOCK) / BLOCK;
  return {as(plain(like, torch::kFloat8_e4m3fn, {m, row}), {m, n}, {row, 1}), as(plain(like, torch::kFloat32, {blocks, m}), {m, blocks}, {1, m})};
}

std::vector<Tensor> rms_norm_fp8(const Tensor &x, const Tensor &w, double eps, const OptTensor &res_) {
  const Tensor res = res_.value_or(Tensor());
  const int dt = norm_args(x, w, eps, res, "rms_norm_fp8");
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t m = x.size(0), n = x.size(1);
  Codes y = new_rows(m, n, x);
  Tensor r;
  if (res.defined()) r = plain(x, x.scalar_type(), x.sizes());
  check_rc(gphl_rms_norm_fp8(dt, m, n, ptr(x), ptr(res), ptr(w), dtype_of(w.scalar_type(), "weight"), (float)eps, mut(y.q), up(n, 16),
                             static_cast<float *>(mut(y.s)), m, mut(r), stream_of(x)),
           "rms_norm_fp8");
  std::vector<Tensor> out{y.q, y.s};
  if (r.defined()) out.push_back(r);
  return out;
}

std::tuple<Tensor, Tensor> quantize_fp8(const Tensor &x) {
  on_device({&x});
  contiguous({&x});
  const int dt = dtype_of(x.scalar_type(), "quantize_fp8: rows");
  TORCH_CHECK(x.dim() == 2, "quantize_fp8 needs rows (m, k)");
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t m = x.size(0), n = x.size(1);
  Codes y = new_rows(m, n, x);
  check_rc(gphl_quantize_fp8(dt, m, n, ptr(x), mut(y.q), up(n, 16), static_cast<float *>(mut(y.s)), m, stream_of(x)), "quantize_fp8");
  return {y.q, y.s};
}

std::tuple<Tensor, Tensor> quantize_fp8_weight(const Tensor &w) {
  on_device({&w});
  contiguous({&w});
  const int dt = dtype_of(w.scalar_type(), "quantize_fp8_weight: weights");
  TORCH_CHECK(w.dim() == 2 || w.dim() == 3, "quantize_fp8_weight needs (k, n) or (types, k, n)");
  c10::cuda::CUDAGuard guard(w.device());
  const int64_t t = w.dim() == 3 ? w.size(0) : 1, k = w.size(-2), n = w.size(-1);
  Tensor q = plain(w, torch::kFloat8_e4m3fn, {t, n, up(k, 16)}), s = plain(w, torch::kFloat32, {t, up(n, BLOCK) / BLOCK, up(k, BLOCK) / BLOCK});
  check_rc(gphl_quantize_fp8_weight(dt, t, k, n, ptr(w), mut(q), up(k, 16), static_cast<float *>(mut(s)), stream_of(w)), "quantize_fp8_weight");
  return {q.slice(2, 0, k), s};
}

// Checks codes and scales; returns the bytes from row to row.
int64_t code_rows(const Tensor &q, const Tensor &s, int64_t dim, const char *what) {
  on_device({&q, &s});
  TORCH_CHECK(q.scalar_type() == torch::kFloat8_e4m3fn && s.scalar_type() == torch::kFloat32 && q.dim() == dim && s.dim() == dim, what,
              " must be float8_e4m3fn values with float32 scales, both of ", dim, " dimensions");
  const int64_t k = q.size(-1), n = q.size(-2), kb = up(k, BLOCK) / BLOCK;
  TORCH_CHECK(dim != 2 || (s.size(0) == n && s.size(1) == kb), what, ": scales of shape ", s.sizes(), ", (", n, ", ", kb, ") are needed");
  TORCH_CHECK(dim != 3 || (s.size(0) == q.size(0) && s.size(1) == up(n, BLOCK) / BLOCK && s.size(2) == kb && s.is_contiguous()), what,
              ": scales must be contiguous, one per 128 x 128 values");
  if (q.numel() == 0) return up(std::max<int64_t>(k, 1), 16);
  // the strides of dimensions of one element say nothing
  const bool several = dim == 3 && q.size(0) > 1;
  const int64_t row = n > 1 ? q.stride(-2) : several ? q.stride(0) : up(k, 16);
  TORCH_CHECK((k == 1 || q.stride(-1) == 1) && row % 16 == 0 && row >= k && (!several || q.stride(0) == n * row) && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              what, ": rows of codes must be contiguous and start on 16-byte boundaries, equally far apart (as the quantisers lay them out)");
  // the last row's padding is read too (and counts for nothing)
  TORCH_CHECK((q.storage_offset() + (q.numel() / k - 1) * row + up(k, 16)) <= (int64_t)q.storage().nbytes(), what, ": the last row of codes must be padded to 16 bytes like the others");
  return row;
}

Tensor dequantize_fp8(const Tensor &q, const Tensor &s, torch::ScalarType type) {
  const int64_t row = code_rows(q, s, 2, "dequantize_fp8: rows");
  const int dt = dtype_of(type, "dequantize_fp8: the output");
  c10::cuda::CUDAGuard guard(q.device());
  Tensor y = plain(q, type, q.sizes());
  check_rc(gphl_dequantize_fp8(dt, q.size(0), q.size(1), ptr(q), row, static_cast<const float *>(ptr(s)), s.stride(0), s.stride(1), mut(y), stream_of(q)),
           "dequantize_fp8");
  return y;
}

Tensor segment_mm_fp8(const Tensor &q, const Tensor &s, const Tensor &wq, const Tensor &ws, const OptTensor &pointer_, torch::ScalarType type,
                      const OptTensor &out) {
  const Tensor pointer = pointer_.value_or(Tensor());
  const int64_t xrow = code_rows(q, s, 2, "segment_mm_fp8: rows"), wrow = code_rows(wq, ws, 3, "segment_mm_fp8: weights");
  const int64_t m = q.size(0), k = q.size(1), t = wq.size(0), n = wq.size(1);
  TORCH_CHECK(wq.size(2) == k, "inner dimensions differ");
  TORCH_CHECK(pointer.defined() || t == 1, "segment_mm_fp8: several types need a type pointer");
  on_device({&q, &wq, &pointer, out ? &*out : nullptr});
  contiguous({&pointer, out ? &*out : nullptr});
  TORCH_CHECK(!pointer.defined() || (pointer.scalar_type() == torch::kInt32 && pointer.numel() == t + 1),
              "segment_mm_fp8: the type pointer must hold types + 1 int32 values");
  if (out) {
    TORCH_CHECK(out->dim() == 2 && out->size(0) == m && out->size(1) == n, "segment_mm_fp8: out must be (m, n)");
    TORCH_CHECK(!at::GradMode::is_enabled() || !out->requires_grad(), "segment_mm_fp8: out wants gradients, and none are recorded");
    type = out->scalar_type();
  }
  const int dt = dtype_of(type, "segment_mm_fp8: the output");
  c10::cuda::CUDAGuard guard(q.device());
  Tensor y = out ? *out : plain(q, type, {m, n});
  if (out && !y.is_inference()) torch::autograd::impl::bump_version(y);      // what autograd kept of it is noticed to have changed
  Tensor work = scratch(gphl_segment_mm_fp8_workspace_bytes(t, pointer.defined(), m, k, n), q);
  check_rc(gphl_segment_mm_fp8(t, static_cast<const int32_t *>(ptr(pointer)), m, k, n, ptr(q), xrow, static_cast<const float *>(ptr(s)), s.stride(0),
                               s.stride(1), ptr(wq), wrow, static_cast<const float *>(ptr(ws)), dt, mut(y), mut(work), stream_of(q)),
           "segment_mm_fp8");
  return y;
}

// ---- gated feed-forward -------------------------------------------------------------------------------------------

int activation(const c10::string_view name, const char *what) {
  if (name == "silu") return GPHL_ACT_SILU;
  if (name == "gelu") return GPHL_ACT_GELU;
  if (name == "relu") return GPHL_ACT_RELU;
  TORCH_CHECK(false, what, ": unknown activation '", name, "' (silu, gelu, relu)");
}

struct Gated {
  int dt, act;
  int64_t m, k, f;
  bool transposed;          // the weights are views of contiguous (f, k) tensors
};
Gated gated_args(const Tensor &x, const Tensor &wg, const Tensor &wu, c10::string_view act, const char *what) {
  on_device({&x, &wg, &wu});
  Gated a{};
  a.act = activation(act, what);
  TORCH_CHECK(x.dim() == 2 && wg.dim() == 2 && wg.sizes() == wu.sizes() && wg.size(0) == x.size(1), what, " needs rows (m, k) and two weights (k, f)");
  TORCH_CHECK(x.scalar_type() == torch::kBFloat16 || x.scalar_type() == torch::kFloat16, what, ": rows must be bfloat16 or float16");
  TORCH_CHECK(wg.scalar_type() == x.scalar_type() && wu.scalar_type() == x.scalar_type(), what, ": rows and weights must have one type");
  a.dt = dtype_of(x.scalar_type(), what);
  a.m = x.size(0), a.k = x.size(1), a.f = wg.size(1);
  a.transposed = !(wg.is_contiguous() && wu.is_contiguous());
  contiguous({&x});
  TORCH_CHECK(!a.transposed || (wg.t().is_contiguous() && wu.t().is_contiguous()), "operators need contiguous tensors (the two weights, or their transposes)");
  return a;
}

// A 16-bit matrix in rows that start on 16-byte boundaries: the tensor itself, or a padded copy.
struct Rows16 {
  Tensor t;
  int64_t ld;
};
Rows16 rows16(const Tensor &x, bool transposed = false) {
  const int64_t m = x.size(transposed ? 1 : 0), n = x.size(transposed ? 0 : 1);
  if (n % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0) return {x, n};
  Tensor p = plain(x, x.scalar_type(), {m, up(n, 8)});
  check_rc(gphl_pad_rows_16(m, n, ptr(x), mut(p), stream_of(x)), "pad_rows");
  return {p, up(n, 8)};
}

// (h, g, u); the projections only if kept
std::tuple<Tensor, Tensor, Tensor> gated_run(const Tensor &x, const Tensor &wg, const Tensor &wu, c10::string_view act, bool keep) {
  const Gated a = gated_args(x, wg, wu, act, "gated_linear");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor h = plain(x, x.scalar_type(), {a.m, a.f}), g, u;
  const int64_t ld = up(a.f, 4);
  if (keep) g = plain(x, torch::kFloat32, {a.m, ld}), u = plain(x, torch::kFloat32, {a.m, ld});
  if (a.k == 0) {
    h.zero_();
    if (keep) g.zero_(), u.zero_();
    return {h, g, u};
  }
  const Rows16 xs = rows16(x), gs = rows16(wg, a.transposed), us = rows16(wu, a.transposed);
  Tensor work = scratch(gphl_gated_workspace_bytes(a.m, a.k, a.f), x);
  check_rc(gphl_gated(a.dt, a.act, a.m, a.k, a.f, ptr(xs.t), xs.ld, ptr(gs.t), ptr(us.t), gs.ld, a.transposed, mut(h), static_cast<float *>(mut(g)),
                      static_cast<float *>(mut(u)), ld, mut(work), stream_of(x)),
           "gated_linear");
  return {h, g, u};
}

// (dx, dWg, dWu); without g and u the projections are made again
std::tuple<Tensor, Tensor, Tensor> gated_grad_run(const Tensor &dh, const Tensor &g, const Tensor &u, const Tensor &x, const Tensor &wg, const Tensor &wu,
                                                  c10::string_view act, bool want_dx, bool want_dw) {
  const Gated a = gated_args(x, wg, wu, act, "gated_linear_grad");
  on_device({&x, &dh, &g, &u});
  contiguous({&dh, &g, &u});
  const int64_t ld = up(a.f, 4);
  TORCH_CHECK(dh.dim() == 2 && dh.size(0) == a.m && dh.size(1) == a.f && dh.scalar_type() == x.scalar_type(),
              "gated_linear_grad: dh must have the output's shape and type");
  for (const Tensor *t : {&g, &u})
    TORCH_CHECK(g.defined() == u.defined() && (!t->defined() || (t->dim() == 2 && t->size(0) == a.m && t->size(1) == ld && t->scalar_type() == torch::kFloat32)),
                "gated_linear_grad: g and u must be the projections that gated_linear returned");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor dx, dg, du;
  if (want_dx) dx = plain(x, x.scalar_type(), x.sizes());
  if (want_dw) {
    dg = plain(x, x.scalar_type(), {a.transposed ? a.f : a.k, a.transposed ? a.k : a.f});
    du = plain(x, x.scalar_type(), dg.sizes());
  }
  const Rows16 xs = rows16(x), gs = rows16(wg, a.transposed), us = rows16(wu, a.transposed);
  Tensor work = scratch(gphl_gated_grad_workspace_bytes(a.m, a.k, a.f), x);
  check_rc(gphl_gated_grad(a.dt, a.act, a.m, a.k, a.f, ptr(dh), static_cast<const float *>(ptr(g)), static_cast<const float *>(ptr(u)), ld, ptr(xs.t), xs.ld,
                           ptr(gs.t), ptr(us.t), gs.ld, a.transposed, mut(dx), mut(dg), mut(du), mut(work), stream_of(x)),
           "gated_linear_grad");
  if (a.transposed && want_dw) dg = dg.t(), du = du.t();
  return {dx, dg, du};
}

std::vector<Tensor> gated_rows(const Tensor &x, const Tensor &wg, const Tensor &wu, c10::string_view act, bool keep) {
  auto [h, g, u] = gated_run(x, wg, wu, act, keep);
  return keep ? std::vector<Tensor>{h, g, u} : std::vector<Tensor>{h};
}
std::vector<Tensor> gated_grad(const Tensor &dh, const OptTensor &g, const OptTensor &u, const Tensor &x, const Tensor &wg, const Tensor &wu,
                               c10::string_view act, bool want_dx, bool want_dw) {
  auto [dx, dg, du] = gated_grad_run(dh, g.value_or(Tensor()), u.value_or(Tensor()), x, wg, wu, act, want_dx, want_dw);
  std::vector<Tensor> out;
  if (want_dx) out.push_back(dx);
  if (want_dw) out.push_back(dg), out.push_back(du);
  return out;
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &wg, const Tensor &wu, std::string act) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor rows = rows_of(x);
    auto [h, g, u] = gated_run(rows, wg, wu, act, rows.size(1) > RECOMPUTE_K);
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["act"] = act;
    ctx->save_for_backward({x.is_contiguous() ? x : rows, wg, wu, g, u});
    auto shape = x.sizes().vec();
    shape.back() = wg.size(1);
    return h.view(shape);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "gated_linear: first derivatives only (create_graph is not supported)");
    const auto s = ctx->get_saved_variables();
    const bool need_x = ctx->needs_input_grad(0), need_g = ctx->needs_input_grad(1), need_u = ctx->needs_input_grad(2);
    auto [dx, dg, du] = gated_grad_run(rows_of(grads[0]), s[3], s[4], rows_of(s[0]), s[1], s[2], ctx->saved_data["act"].toStringRef(), need_x, need_g || need_u);
    return {need_x ? dx.view(ctx->saved_data["shape"].toIntVector()) : Tensor(), need_g ? dg : Tensor(), need_u ? du : Tensor(), Tensor()};
  }
};

Tensor gated_linear(const Tensor &x, const Tensor &wg, const Tensor &wu, c10::string_view act) {
  TORCH_CHECK(x.dim() >= 1 && wg.dim() == 2 && x.size(-1) == wg.size(0), "gated_linear needs rows (..., k) and two weights (k, f)");
  on_device({&x, &wg, &wu});
  no_tangents({&x, &wg, &wu}, "gated_linear");
  if (wants_grad({&x, &wg, &wu})) {
    capturable({&x, &wg, &wu}, "gated_linear");
    return GatedLinear::apply(x, wg, wu, std::string(act));
  }
  auto shape = x.sizes().vec();
  shape.back() = wg.size(1);
  return std::get<0>(gated_run(rows_of(x), wg, wu, act, false)).view(shape);
}

// [q, scales], or [h] in a type of 16 or 32 bits
std::vector<Tensor> gated_linear_fp8(const Tensor &q, const Tensor &s, const Tensor &gq, const Tensor &gs, const Tensor &uq, const Tensor &us,
                                     c10::string_view act_name, torch::ScalarType type) {
  const int act = activation(act_name, "gated_linear_fp8");
  const int64_t xrow = code_rows(q, s, 2, "gated_linear_fp8: rows"), wrow = code_rows(gq, gs, 3, "gated_linear_fp8: weights"),
                urow = code_rows(uq, us, 3, "gated_linear_fp8: weights");
  on_device({&q, &gq, &uq});
  const int64_t m = q.size(0), k = q.size(1), f = gq.size(1);
  TORCH_CHECK(gq.size(0) == 1 && uq.sizes() == gq.sizes() && gq.size(2) == k, "gated_linear_fp8 needs two weights (1, f, k) and rows (m, k)");
  TORCH_CHECK(urow == wrow, "gated_linear_fp8: the two weights must be laid out alike");
  const bool codes = type == torch::kFloat8_e4m3fn;
  const int dt = codes ? GPHL_F32 : dtype_of(type, "gated_linear_fp8: the output");
  c10::cuda::CUDAGuard guard(q.device());
  if (k == 0) {
    Tensor z = torch::zeros({m, f}, q.options().dtype(codes ? torch::kFloat32 : type));
    if (!codes) return {z};
    auto [a, b] = quantize_fp8(z);
    return {a, b};
  }
  Codes y;
  Tensor h;
  if (codes) y = new_rows(m, f, q);
  else h = plain(q, type, {m, f});
  Tensor work = scratch(gphl_gated_fp8_workspace_bytes(m, k, f, codes), q);
  check_rc(gphl_gated_fp8(act, m, k, f, ptr(q), xrow, static_cast<const float *>(ptr(s)), s.stride(0), s.stride(1), ptr(gq), static_cast<const float *>(ptr(gs)),
                          ptr(uq), static_cast<const float *>(ptr(us)), wrow, dt, mut(h), mut(y.q), up(f, 16), static_cast<float *>(mut(y.s)), m, mut(work),
                          stream_of(q)),
           "gated_linear_fp8");
  if (codes) return {y.q, y.s};
  return {h};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(my_ops, m) {
  m.def("rms_norm(Tensor x, Tensor weight, float eps, Tensor? residual) -> Tensor[]", &rms_norm);
  m.def("rms_norm_rows(Tensor x, Tensor weight, float eps, Tensor? residual, bool return_rstd) -> Tensor[]", &rms_norm_rows);
  m.def("rms_norm_grad(Tensor r, Tensor weight, Tensor rstd, Tensor dy, Tensor? dr) -> (Tensor, Tensor)", &rms_norm_grad);
  m.def("rms_norm_fp8(Tensor x, Tensor weight, float eps, Tensor? residual) -> Tensor[]", &rms_norm_fp8);
  m.def("quantize_fp8(Tensor x) -> (Tensor, Tensor)", &quantize_fp8);
  m.def("quantize_fp8_weight(Tensor w) -> (Tensor, Tensor)", &quantize_fp8_weight);
  m.def("dequantize_fp8(Tensor q, Tensor scales, ScalarType dtype) -> Tensor", &dequantize_fp8);
  m.def("segment_mm_fp8(Tensor q, Tensor scales, Tensor w, Tensor w_scales, Tensor? type_pointer, ScalarType dtype, Tensor(a!)? out) -> Tensor(a!)",
        &segment_mm_fp8);
  m.def("gated_linear(Tensor x, Tensor w_gate, Tensor w_up, str activation) -> Tensor", &gated_linear);
  m.def("gated_linear_rows(Tensor x, Tensor w_gate, Tensor w_up, str activation, bool return_projections) -> Tensor[]", &gated_rows);
  m.def("gated_linear_grad(Tensor dh, Tensor? g, Tensor? u, Tensor x, Tensor w_gate, Tensor w_up, str activation, bool want_dx, bool want_dw) -> Tensor[]",
        &gated_grad);
  m.def("gated_linear_fp8(Tensor q, Tensor scales, Tensor wg, Tensor wg_scales, Tensor wu, Tensor wu_scales, str activation, ScalarType dtype) -> Tensor[]",
        &gated_linear_fp8);
}
