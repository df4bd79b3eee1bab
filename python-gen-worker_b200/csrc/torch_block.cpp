// torch.ops.gwb200: layer norm with modulation, rotary positions and gated
// feed-forward projections over the C ABI (include/gwb200.h), with their gradients.
//
// The dispatcher's CUDA key holds the plain calls; the Autograd key records a
// node only when a gradient is wanted and otherwise goes straight below, so
// an inference call costs one dispatch. Outputs and workspaces come from
// torch's allocator on the input's device; work goes to that device's current
// stream, whatever device is current. Wrong arguments raise ValueError (the
// Python wrappers turn it into the package's error); a backward pass asked to
// build a graph of its own is refused.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <tuple>
#include <vector>

#include "../../include/gwb200.h"

namespace gwb200_block {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

int dtype_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return GWB_DTYPE_F32;
    case at::kBFloat16: return GWB_DTYPE_BF16;
    case at::kHalf: return GWB_DTYPE_F16;
    default: break;
  }
  NEED(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  return -1;
}

void check_status(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, ": ", gwb_status_string(rc), " (status ", rc, ")");
}

void need_on(const Tensor& t, const char* name, const Tensor& x) {
  NEED(t.is_cuda() && t.device() == x.device(), name, " must be on ", x.device(), ", got ",
       t.device());
}

void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
const void* ptr(const OptTensor& t) { return has(t) ? t->const_data_ptr() : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const OptTensor& t) { return has(t) && t->requires_grad(); }

// A backward pass under create_graph would need gradients of its own.
template <typename... Ts>
void refuse_second_order(const char* what, const Ts&... ts) {
  if (!at::GradMode::is_enabled()) return;
  const bool any = (wants(ts) || ...);
  TORCH_CHECK(!any, what, " has no second derivative (create_graph=True)");
}

// Below the Autograd key no tangent is looked at: a dual tensor of forward-mode
// differentiation would lose its own without a word.
bool tangent_of(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool tangent_of(const OptTensor& t) { return has(t) && tangent_of(*t); }
template <typename... Ts>
void refuse_tangents(const char* what, const Ts&... ts) {
  NEED(!(tangent_of(ts) || ...), what, " has no forward-mode derivative: use reverse mode");
}

// While a graph that used a leaf lives, torch keeps that leaf's gradient on the
// stream of that graph. A backward pass captured on another stream would have
// to wait for it across the capture, which breaks the capture in the middle of
// the engine's work. Refused here, where the forward call is captured.
void refuse_foreign_leaf(const char* what, const Tensor& t) {
  if (!wants(t) || !t.is_leaf() || !t.is_cuda()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return;
  const auto stream = node->stream();
  const c10::Stream now = c10::cuda::getCurrentCUDAStream(t.device().index()).unwrap();
  TORCH_CHECK(!stream.has_value() || *stream == now, what,
              " is captured while a graph of the same leaf lives on another stream: capture with"
              " leaves of its own (t.detach().requires_grad_()), or let that graph go first");
}
void refuse_foreign_leaf(const char* what, const OptTensor& t) {
  if (has(t)) refuse_foreign_leaf(what, *t);
}
// A tensor that stands for one while a call is traced or transformed: there may
// be no GPU, and nothing is captured.
bool traced(const Tensor& t) {
  return t.defined() &&
         t.key_set().has_any(c10::DispatchKeySet(
             {c10::DispatchKey::Python, c10::DispatchKey::Functionalize,
              c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched}));
}
bool traced(const OptTensor& t) { return has(t) && traced(*t); }
template <typename... Ts>
void refuse_foreign_leaves(const char* what, const Tensor& x, const Ts&... ts) {
  if (!x.is_cuda() || traced(x) || (traced(ts) || ...)) return;
  const c10::cuda::CUDAGuard guard(x.device());
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  refuse_foreign_leaf(what, x);
  (refuse_foreign_leaf(what, ts), ...);
}

// Whether [..., D] lies as rows at one stride; that stride.
bool row_stride_of(const Tensor& x, int64_t* stride) {
  const int64_t nd = x.dim();
  if (x.numel() == 0) { *stride = x.size(-1); return true; }
  if (x.size(-1) > 1 && x.stride(-1) != 1) return false;
  int64_t step = -1, span = 1;      // stride of the innermost row dimension, rows below
  for (int64_t d = nd - 2; d >= 0; --d) {
    if (x.size(d) == 1) continue;
    if (step < 0) step = x.stride(d);
    else if (x.stride(d) != step * span) return false;
    span *= x.size(d);
  }
  *stride = step < 0 ? x.size(-1) : step;
  return true;
}

Tensor rows_of(const Tensor& x, int64_t* stride) {
  if (row_stride_of(x, stride)) return x;
  Tensor c = x.contiguous();
  *stride = x.size(-1);
  return c;
}

// ---------------------------------------------------------------- layer norm
struct Affine { OptTensor w, b; int f32 = 0; };
struct Mod { OptTensor s, t; int f32 = 0; int64_t ss = 0, ts = 0, rows = 1, samples = 1; };

int pair_type(const Tensor& x, const OptTensor& a, const OptTensor& b, const char* names) {
  if (!has(a) && !has(b)) return 0;
  const auto t = has(a) ? a->scalar_type() : b->scalar_type();
  NEED(!has(a) || !has(b) || a->scalar_type() == b->scalar_type(), names,
       " must have one type, got ", a->scalar_type(), " and ", b->scalar_type());
  NEED(t == x.scalar_type() || t == at::kFloat, names, " must be float32 or of x's type ",
       x.scalar_type(), ", got ", t);
  return t == at::kFloat;
}

Affine affine_of(const Tensor& x, const OptTensor& w, const OptTensor& b) {
  Affine a{c10::nullopt, c10::nullopt, pair_type(x, w, b, "weight and bias")};
  const int64_t d = x.size(-1);
  const auto one = [&](const OptTensor& t, const char* name) -> OptTensor {
    if (!has(t)) return c10::nullopt;
    need_on(*t, name, x);
    NEED(t->dim() == 1 && t->size(0) == d, name, " must be [", d, "], got ", t->sizes());
    return t->contiguous();
  };
  a.w = one(w, "weight");
  a.b = one(b, "bias");
  return a;
}

// [D], [B, D] or [B, 1, ..., 1, D] with B = 1 or x's first size -> [B, D] and its sample stride
Mod mod_of(const Tensor& x, const OptTensor& s, const OptTensor& t) {
  Mod m;
  m.f32 = pair_type(x, s, t, "scale and shift");
  const int64_t d = x.size(-1), rows = d ? x.numel() / d : 0;
  m.rows = rows;
  if (!has(s) && !has(t)) return m;
  int64_t samples = -1;
  const auto one = [&](const OptTensor& p, const char* name, int64_t* stride) -> OptTensor {
    if (!has(p)) return c10::nullopt;
    need_on(*p, name, x);
    NEED(p->dim() >= 1 && p->size(-1) == d, name, " must be [", d, "] or [B, ", d, "], got ",
         p->sizes());
    const int64_t b = p->dim() == 1 ? 1 : p->size(0);
    for (int64_t i = 1; i < p->dim() - 1; ++i)
      NEED(p->size(i) == 1, name, " must be [", d, "] or [B, ", d, "], got ", p->sizes());
    NEED(b == 1 || (x.dim() >= 2 && b == x.size(0)), name, " has ", b,
         " samples, x has shape ", x.sizes());
    NEED(samples < 0 || samples == b, "scale and shift must have the same number of samples");
    samples = b;
    Tensor v = (d > 1 && p->stride(-1) != 1) ? p->contiguous() : *p;
    *stride = b == 1 ? 0 : v.stride(0);
    return v;
  };
  m.s = one(s, "scale", &m.ss);
  m.t = one(t, "shift", &m.ts);
  m.samples = samples;
  m.rows = samples ? rows / samples : 0;
  return m;
}

void check_norm_input(const Tensor& x) {
  NEED(x.is_cuda(), "x must be a CUDA tensor (no CPU path), got ", x.device());
  NEED(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., D] with D >= 1, got ", x.sizes());
  dtype_code(x, "x");
}

std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x, const OptTensor& weight,
                                                const OptTensor& bias, const OptTensor& scale,
                                                const OptTensor& shift, double eps, bool stats) {
  check_norm_input(x);
  NEED(eps >= 0, "eps must not be negative, got ", eps);
  const c10::cuda::CUDAGuard guard(x.device());
  const Affine a = affine_of(x, weight, bias);
  const Mod m = mod_of(x, scale, shift);
  int64_t xs = 0;
  const Tensor xr = rows_of(x, &xs);
  const int64_t d = x.size(-1), rows = x.numel() / d;
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor mean = stats ? at::empty({rows}, f32) : Tensor();
  Tensor rstd = stats ? at::empty({rows}, f32) : Tensor();
  if (rows)
    check_status(gwb_layer_norm(xr.const_data_ptr(), xs, ptr(a.w), ptr(a.b), a.f32, ptr(m.s), m.ss,
                                ptr(m.t), m.ts, m.f32, rows, d, m.rows, (float)eps,
                                dtype_code(x, "x"), y.data_ptr(),
                                stats ? mean.data_ptr<float>() : nullptr,
                                stats ? rstd.data_ptr<float>() : nullptr, stream_of(x)),
                 "layer_norm");
  return {y, mean, rstd};
}

Tensor layer_norm_cuda(const Tensor& x, const OptTensor& w, const OptTensor& b,
                       const OptTensor& scale, const OptTensor& shift, double eps) {
  return std::get<0>(norm_forward(x, w, b, scale, shift, eps, false));
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_stats_cuda(const Tensor& x, const OptTensor& w,
                                                         const OptTensor& b,
                                                         const OptTensor& scale,
                                                         const OptTensor& shift, double eps) {
  return norm_forward(x, w, b, scale, shift, eps, true);
}

// -> (dx, dweight, dbias, dscale, dshift); one not asked for is empty [0]
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> layer_norm_backward_cuda(
    const Tensor& dy, const Tensor& x, const Tensor& mean, const Tensor& rstd,
    const OptTensor& weight, const OptTensor& bias, const OptTensor& scale,
    const OptTensor& shift, std::array<bool, 5> mask) {
  check_norm_input(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const Affine a = affine_of(x, weight, bias);
  const Mod m = mod_of(x, scale, shift);
  const int64_t d = x.size(-1), rows = x.numel() / d;
  need_on(dy, "dy", x);
  NEED(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(),
       "dy must match x: shape ", x.sizes(), ", type ", x.scalar_type());
  for (const Tensor* t : {&mean, &rstd}) {
    need_on(*t, "mean and rstd", x);
    NEED(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == rows &&
             t->is_contiguous(),
         "mean and rstd must be contiguous float32 [", rows, "]");
  }
  NEED((!mask[1] || has(a.w)) && (!mask[2] || has(a.b)) && (!mask[3] || has(m.s)) &&
           (!mask[4] || has(m.t)),
       "a gradient was asked for of a parameter that is not given");
  int64_t xs = 0, ys = 0;
  const Tensor xr = rows_of(x, &xs), dyr = rows_of(dy, &ys);
  const auto like = [&](bool on, const OptTensor& t, at::IntArrayRef shape) {
    return on ? at::empty(shape, t->options().memory_format(at::MemoryFormat::Contiguous))
              : at::empty({0}, x.options());
  };
  Tensor dx = mask[0] ? at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous))
                      : at::empty({0}, x.options());
  Tensor dw = like(mask[1], a.w, {d}), db = like(mask[2], a.b, {d});
  Tensor ds = like(mask[3], m.s, has(m.s) ? m.s->sizes() : at::IntArrayRef{});
  Tensor dt = like(mask[4], m.t, has(m.t) ? m.t->sizes() : at::IntArrayRef{});
  Tensor work;
  if (mask[1] || mask[2] || mask[3] || mask[4])
    work = at::empty({gwb_layer_norm_backward_work(rows, d, m.rows)},
                     x.options().dtype(at::kFloat));
  if (rows == 0) {
    ds.zero_();
    dt.zero_();
  }
  const auto out = [](bool on, Tensor& t) { return on ? t.data_ptr() : nullptr; };
  check_status(gwb_layer_norm_backward(
                   dyr.const_data_ptr(), ys, xr.const_data_ptr(), xs, mean.const_data_ptr<float>(),
                   rstd.const_data_ptr<float>(), ptr(a.w), ptr(a.b), a.f32, ptr(m.s), m.ss, m.f32,
                   rows, d, m.rows, dtype_code(x, "x"), out(mask[0], dx), out(mask[1], dw),
                   out(mask[2], db), out(mask[3], ds), out(mask[4], dt),
                   work.defined() ? work.data_ptr<float>() : nullptr, stream_of(x)),
               "layer_norm_backward");
  return {dx, dw, db, ds, dt};
}

template <typename Sig>
auto op_of(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w,
                        const OptTensor& b, const OptTensor& scale, const OptTensor& shift,
                        double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = op_of<decltype(layer_norm_stats_cuda)>("gwb200::layer_norm_stats");
    auto [y, mean, rstd] = op.call(x, w, b, scale, shift, eps);
    const auto keep = [](const OptTensor& t) { return has(t) ? *t : Tensor(); };
    ctx->save_for_backward({x, mean, rstd, keep(w), keep(b), keep(scale), keep(shift)});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    refuse_second_order("layer_norm_backward", grads[0], v[0], v[3], v[4], v[5], v[6]);
    if (!grads[0].defined()) return variable_list(6);
    // needs_input_grad counts the tensors that were given, absent ones left out
    std::array<bool, 5> mask{ctx->needs_input_grad(0)};
    for (int i = 1, given = 1; i < 5; ++i)
      if (v[2 + i].defined()) mask[i] = ctx->needs_input_grad(given++);
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = op_of<decltype(layer_norm_backward_cuda)>("gwb200::layer_norm_backward");
    auto [dx, dw, db, ds, dt] = op.call(grads[0], v[0], v[1], v[2], opt(v[3]), opt(v[4]),
                                        opt(v[5]), opt(v[6]), mask);
    const auto give = [&](int i, Tensor& t) { return mask[i] ? t : Tensor(); };
    return {give(0, dx), give(1, dw), give(2, db), give(3, ds), give(4, dt), Tensor()};
  }
};

Tensor layer_norm_autograd(const Tensor& x, const OptTensor& w, const OptTensor& b,
                           const OptTensor& scale, const OptTensor& shift, double eps) {
  refuse_tangents("layer_norm", x, w, b, scale, shift);
  if (at::GradMode::is_enabled() &&
      (wants(x) || wants(w) || wants(b) || wants(scale) || wants(shift))) {
    refuse_foreign_leaves("layer_norm", x, w, b, scale, shift);
    return LayerNormFn::apply(x, w, b, scale, shift, eps);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = op_of<decltype(layer_norm_cuda)>("gwb200::layer_norm");
  return op.call(x, w, b, scale, shift, eps);
}

// ---------------------------------------------------------------- rotary
struct RotaryShape { int64_t B, S, n, dh; int64_t pos[3]; int kind; int64_t axes; };

std::array<int64_t, 3> strides_of(const Tensor& t) {
  return t.dim() == 4 ? std::array<int64_t, 3>{t.stride(0), t.stride(1), t.stride(2)}
                      : std::array<int64_t, 3>{0, t.stride(0), t.stride(1)};
}

RotaryShape rotary_shape(const Tensor& q, const OptTensor& k, const Tensor& positions,
                         const Tensor& inv_freq, const OptTensor& axis) {
  NEED(q.is_cuda(), "q must be a CUDA tensor (no CPU path), got ", q.device());
  NEED(q.dim() == 4 || q.dim() == 3, "q must be [B, S, H, D] or [S, H, D], got ", q.sizes());
  dtype_code(q, "q");
  RotaryShape r;
  const int64_t nd = q.dim();
  r.B = nd == 4 ? q.size(0) : 1;
  r.S = q.size(nd - 3);
  r.dh = q.size(nd - 1);
  if (has(k)) {
    need_on(*k, "k", q);
    NEED(k->scalar_type() == q.scalar_type() && k->dim() == nd && k->size(nd - 1) == r.dh &&
             k->size(nd - 3) == r.S && (nd == 3 || k->size(0) == r.B),
         "k must match q in type, batch, tokens and head size: q ", q.sizes(), ", k ", k->sizes());
  }
  need_on(inv_freq, "inv_freq", q);
  NEED(inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1 && inv_freq.is_contiguous(),
       "inv_freq must be contiguous float64 [rotary_dim / 2]");
  r.n = inv_freq.size(0);
  NEED(r.n >= 1 && 2 * r.n <= r.dh && r.dh <= 4096, "inv_freq has ", r.n,
       " entries; heads of ", r.dh, " features take 1 to ", r.dh / 2, " (at most 4096 features)");
  need_on(positions, "positions", q);
  switch (positions.scalar_type()) {
    case at::kLong: r.kind = 0; break;
    case at::kInt: r.kind = 1; break;
    case at::kFloat: r.kind = 2; break;
    default: NEED(false, "positions must be int64, int32 or float32, got ",
                  positions.scalar_type());
  }
  int64_t pd = positions.dim();
  r.axes = 1;
  r.pos[2] = 0;
  if (has(axis)) {
    need_on(*axis, "axis", q);
    NEED(axis->scalar_type() == at::kInt && axis->dim() == 1 && axis->size(0) == r.n &&
             axis->is_contiguous(),
         "axis must be contiguous int32 [", r.n, "]");
    NEED(pd >= 2, "positions must be [S, A] or [B, S, A] when axis is given, got ",
         positions.sizes());
    r.axes = positions.size(pd - 1);
    NEED(r.axes >= 1 && r.axes <= 64, "positions have ", r.axes, " axes (1 to 64)");
    r.pos[2] = positions.stride(pd - 1);
    --pd;
  }
  NEED(pd == 1 || pd == 2, "positions must be [S] or [B, S]",
       has(axis) ? " with a last dimension of axes" : "", ", got ", positions.sizes());
  NEED(positions.size(pd - 1) == r.S, "positions cover ", positions.size(pd - 1),
       " tokens, q has ", r.S);
  r.pos[1] = positions.stride(pd - 1);
  r.pos[0] = 0;
  if (pd == 2) {
    NEED(positions.size(0) == r.B || positions.size(0) == 1, "positions cover ",
         positions.size(0), " sequences, q has ", r.B);
    r.pos[0] = positions.size(0) == 1 ? 0 : positions.stride(0);
  }
  return r;
}

void rotary_call(const RotaryShape& r, const Tensor& q, Tensor& qo, const OptTensor& k, Tensor* ko,
                 const Tensor& positions, const Tensor& inv_freq, const OptTensor& axis,
                 bool interleaved, double scale, bool inverse) {
  if (r.B == 0 || r.S == 0) return;
  const auto qs = strides_of(q), qos = strides_of(qo);
  std::array<int64_t, 3> ks{}, kos{};
  if (has(k)) { ks = strides_of(*k); kos = strides_of(*ko); }
  check_status(gwb_rotary(q.const_data_ptr(), qs.data(), qo.data_ptr(), qos.data(),
                          q.size(q.dim() - 2), ptr(k), ks.data(),
                          has(k) ? ko->data_ptr() : nullptr, kos.data(),
                          has(k) ? k->size(k->dim() - 2) : 0, positions.const_data_ptr(), r.kind,
                          r.pos, inv_freq.const_data_ptr<double>(),
                          static_cast<const int32_t*>(ptr(axis)), r.axes, r.B, r.S, r.n, r.dh,
                          (float)scale, interleaved, inverse, dtype_code(q, "q"), stream_of(q)),
               "rotary");
}

Tensor dense_last(const Tensor& t) {
  return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t;
}

std::tuple<Tensor, Tensor> rotary_cuda(const Tensor& q, const OptTensor& k,
                                       const Tensor& positions, const Tensor& inv_freq,
                                       const OptTensor& axis, bool interleaved, double scale,
                                       bool inverse) {
  const RotaryShape r = rotary_shape(q, k, positions, inv_freq, axis);
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor qd = dense_last(q);
  const OptTensor kd = has(k) ? OptTensor(dense_last(*k)) : c10::nullopt;
  Tensor qo = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor ko = has(k) ? at::empty(k->sizes(),
                                 k->options().memory_format(at::MemoryFormat::Contiguous))
                     : at::empty({0}, q.options());
  rotary_call(r, qd, qo, kd, &ko, positions, inv_freq, axis, interleaved, scale, inverse);
  return {qo, ko};
}

// Whether `gap` is the sum of one multiple of each term's stride within that
// term's range. Terms come in order of falling stride, and what the later ones
// can reach leaves few multiples of a term to try; a search that would try many
// all the same (odd strides that mesh) says yes.
struct Term { int64_t stride, low, high; };
bool reaches(const Term* t, size_t n, int64_t gap, int* tries) {
  if (n == 0) return gap == 0;
  int64_t low = 0, high = 0;
  for (size_t i = 1; i < n; ++i) {
    low += t[i].low * t[i].stride;
    high += t[i].high * t[i].stride;
  }
  const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  const int64_t first = std::max(t->low, -floor_div(high - gap, t->stride));
  const int64_t last = std::min(t->high, floor_div(gap - low, t->stride));
  for (int64_t m = first; m <= last; ++m)
    if (--*tries < 0 || reaches(t + 1, n - 1, gap - m * t->stride, tries)) return true;
  return false;
}

// Whether two tensors of one storage have an element in common: an index of
// each whose offsets differ by their distance. A dimension of one stride in
// both is one term, the difference of its two indices.
bool share_elements(const Tensor& q, const Tensor& k) {
  if (!q.is_alias_of(k) || q.numel() == 0 || k.numel() == 0) return false;
  std::vector<Term> terms;
  const auto add = [&](int64_t stride, int64_t low, int64_t high) {
    if (stride > 0 && low < high) terms.push_back({stride, low, high});
  };
  for (int64_t d = 0; d < q.dim(); ++d) {
    const int64_t up = q.size(d) - 1, down = 1 - k.size(d);
    if (q.stride(d) == k.stride(d)) {
      add(q.stride(d), down, up);
    } else {
      add(q.stride(d), 0, up);
      add(k.stride(d), down, 0);
    }
  }
  std::sort(terms.begin(), terms.end(),
            [](const Term& a, const Term& b) { return a.stride > b.stride; });
  int tries = 10000;
  return reaches(terms.data(), terms.size(), k.storage_offset() - q.storage_offset(), &tries);
}

// Whether two indices of one tensor name the same element: an expanded
// dimension, or two indices whose first difference some later ones undo.
bool overlaps_itself(const Tensor& t) {
  if (t.numel() < 2 || t.is_non_overlapping_and_dense()) return false;
  std::vector<Term> terms;
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) < 2) continue;
    if (t.stride(d) == 0) return true;
    terms.push_back({t.stride(d), 1 - t.size(d), t.size(d) - 1});
  }
  std::sort(terms.begin(), terms.end(),
            [](const Term& a, const Term& b) { return a.stride > b.stride; });
  int tries = 10000;
  for (size_t i = 0; i < terms.size(); ++i) {
    Term& first = terms[i];
    first.low = 1;
    if (reaches(&first, terms.size() - i, 0, &tries)) return true;
  }
  return false;
}

void rotary_inplace_cuda(Tensor q, const OptTensor& k, const Tensor& positions,
                         const Tensor& inv_freq, const OptTensor& axis, bool interleaved,
                         double scale, bool inverse) {
  const RotaryShape r = rotary_shape(q, k, positions, inv_freq, axis);
  const c10::cuda::CUDAGuard guard(q.device());
  const auto writable = [](const Tensor& t, const char* name) {
    NEED(t.size(-1) <= 1 || t.stride(-1) == 1, name,
         " must be dense in its last dimension to be rotated in place");
    NEED(!overlaps_itself(t), name,
         " overlaps itself and cannot be rotated in place");
  };
  writable(q, "q");
  Tensor kt;
  if (has(k)) {
    writable(*k, "k");
    NEED(!share_elements(q, *k), "q and k share memory and cannot both be rotated in place");
    kt = *k;
  }
  rotary_call(r, q, q, k, &kt, positions, inv_freq, axis, interleaved, scale, inverse);
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k,
                               const Tensor& positions, const Tensor& inv_freq,
                               const OptTensor& axis, bool interleaved, double scale,
                               bool inverse) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = op_of<decltype(rotary_cuda)>("gwb200::rotary");
    auto [qo, ko] = op.call(q, k, positions, inv_freq, axis, interleaved, scale, inverse);
    ctx->save_for_backward({positions, inv_freq, has(axis) ? *axis : Tensor()});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["k"] = has(k);
    if (!has(k)) ctx->mark_non_differentiable({ko});
    return {qo, ko};
  }
  // The map is linear in q and k, so its gradient is the op itself by the
  // negative angle, through autograd again.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const bool with_k = ctx->saved_data["k"].toBool();
    const bool need_q = grads[0].defined() && ctx->needs_input_grad(0);
    const bool need_k = with_k && grads[1].defined() && ctx->needs_input_grad(1);
    variable_list out(8);
    if (!need_q && !need_k) return out;
    static auto op = op_of<decltype(rotary_cuda)>("gwb200::rotary");
    const Tensor& first = need_q ? grads[0] : grads[1];
    auto [a, b] = op.call(first, need_q && need_k ? OptTensor(grads[1]) : c10::nullopt, v[0], v[1],
                          opt(v[2]), ctx->saved_data["interleaved"].toBool(),
                          ctx->saved_data["scale"].toDouble(),
                          !ctx->saved_data["inverse"].toBool());
    if (need_q) out[0] = a;
    if (need_k) out[1] = need_q ? b : a;
    return out;
  }
};

void refuse_learned_angles(const Tensor& positions, const Tensor& inv_freq) {
  NEED(!(at::GradMode::is_enabled() && (wants(positions) || wants(inv_freq))),
       "positions and inv_freq get no gradient: pass them detached");
}

std::tuple<Tensor, Tensor> rotary_autograd(const Tensor& q, const OptTensor& k,
                                           const Tensor& positions, const Tensor& inv_freq,
                                           const OptTensor& axis, bool interleaved, double scale,
                                           bool inverse) {
  refuse_tangents("rotary", q, k, positions, inv_freq);
  refuse_learned_angles(positions, inv_freq);
  if (at::GradMode::is_enabled() && (wants(q) || wants(k))) {
    refuse_foreign_leaves("rotary", q, k);
    auto r = RotaryFn::apply(q, k, positions, inv_freq, axis, interleaved, scale, inverse);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = op_of<decltype(rotary_cuda)>("gwb200::rotary");
  return op.call(q, k, positions, inv_freq, axis, interleaved, scale, inverse);
}

void rotary_inplace_autograd(Tensor q, const OptTensor& k, const Tensor& positions,
                             const Tensor& inv_freq, const OptTensor& axis, bool interleaved,
                             double scale, bool inverse) {
  refuse_tangents("rotary_", q, k, positions, inv_freq);
  refuse_learned_angles(positions, inv_freq);
  NEED(!(at::GradMode::is_enabled() && (wants(q) || wants(k))),
       "rotary_ writes in place and keeps no gradient: use rotary");
  at::AutoDispatchBelowAutograd below;
  static auto op = op_of<decltype(rotary_inplace_cuda)>("gwb200::rotary_");
  op.call(q, k, positions, inv_freq, axis, interleaved, scale, inverse);
}

// Counts the change where autograd looks for it. A key of its own: inference
// mode passes the Autograd key by, but not this one, for tensors made outside it.
void rotary_inplace_counted(Tensor q, const OptTensor& k, const Tensor& positions,
                            const Tensor& inv_freq, const OptTensor& axis, bool interleaved,
                            double scale, bool inverse) {
  {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = op_of<decltype(rotary_inplace_cuda)>("gwb200::rotary_");
    op.call(q, k, positions, inv_freq, axis, interleaved, scale, inverse);
  }
  torch::autograd::increment_version(q);
  if (has(k)) torch::autograd::increment_version(*k);
}

// ---------------------------------------------------------------- gated projections
bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }

// Rows at one stride that TMA can read (16-byte steps), else a copy.
Tensor tma_rows_of(const Tensor& x, int64_t* stride) {
  const int64_t d = x.size(-1);
  if (row_stride_of(x, stride) && *stride >= d && *stride % 8 == 0 && aligned16(x)) return x;
  *stride = d;
  if (x.is_contiguous() && aligned16(x)) return x;
  // contiguous() of a dense but misaligned view would return the view itself
  return at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)).copy_(x);
}

struct GatedShape { int64_t rows, d, f; int dtype; };

GatedShape gated_shape(const Tensor& x, const Tensor& wg, const Tensor& wu, const OptTensor& bg,
                       const OptTensor& bu, int64_t act) {
  NEED(x.is_cuda(), "x must be a CUDA tensor (no CPU path), got ", x.device());
  NEED(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
       "x must be bfloat16 or float16, got ", x.scalar_type());
  NEED(x.dim() >= 1, "x must be [..., D]");
  GatedShape g{0, x.size(-1), wg.dim() == 2 ? wg.size(0) : 0, dtype_code(x, "x")};
  NEED(g.d >= 8 && g.d % 8 == 0, "x has ", g.d, " features; a positive multiple of 8 is needed");
  g.rows = x.numel() / g.d;
  const auto weight = [&](const Tensor& w, const char* name) {
    need_on(w, name, x);
    NEED(w.scalar_type() == x.scalar_type(), name, " must be ", x.scalar_type(), ", got ",
         w.scalar_type());
    NEED(w.dim() == 2 && w.size(0) == g.f && w.size(1) == g.d, name, " must be [", g.f, ", ", g.d,
         "], got ", w.sizes());
    NEED(w.is_contiguous() && aligned16(w), name, " must be contiguous and 16-byte aligned");
  };
  weight(wg, "w_gate");
  weight(wu, "w_up");
  NEED(g.f >= 8 && g.f % 8 == 0, "w_gate has ", g.f, " rows; a positive multiple of 8 is needed");
  const auto bias = [&](const OptTensor& b, const char* name) {
    if (!has(b)) return;
    need_on(*b, name, x);
    NEED(b->scalar_type() == x.scalar_type() && b->dim() == 1 && b->size(0) == g.f, name,
         " must be ", x.scalar_type(), " [", g.f, "], got ", b->scalar_type(), " ", b->sizes());
    NEED(b->is_contiguous() && aligned16(*b), name, " must be contiguous and 16-byte aligned");
  };
  bias(bg, "b_gate");
  bias(bu, "b_up");
  NEED(act >= GWB_ACT_SILU && act <= GWB_ACT_GELU_TANH, "unknown activation code ", act);
  return g;
}

Tensor gated_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const OptTensor& bg,
                     const OptTensor& bu, int64_t act, Tensor* kept) {
  const GatedShape g = gated_shape(x, wg, wu, bg, bu, act);
  const c10::cuda::CUDAGuard guard(x.device());
  int64_t xs = 0;
  const Tensor xr = tma_rows_of(x, &xs);
  auto shape = x.sizes().vec();
  shape.back() = g.f;
  Tensor h = at::empty(shape, x.options().memory_format(at::MemoryFormat::Contiguous));
  if (!kept) {
    check_status(gwb_gated_linear(xr.const_data_ptr(), xs, wg.const_data_ptr(),
                                  wu.const_data_ptr(), ptr(bg), ptr(bu), g.rows, g.d, g.f,
                                  (int)act, g.dtype, h.data_ptr(), stream_of(x)),
                 "gated_linear");
    return h;
  }
  *kept = at::empty({gwb_gated_linear_kept(g.rows, g.f, g.dtype)}, x.options().dtype(at::kByte));
  check_status(gwb_gated_linear_keep(xr.const_data_ptr(), xs, wg.const_data_ptr(),
                                     wu.const_data_ptr(), ptr(bg), ptr(bu), g.rows, g.d, g.f,
                                     (int)act, g.dtype, h.data_ptr(), kept->data_ptr(),
                                     stream_of(x)),
               "gated_linear_keep");
  return h;
}

Tensor gated_linear_cuda(const Tensor& x, const Tensor& wg, const Tensor& wu, const OptTensor& bg,
                         const OptTensor& bu, int64_t act, bool recompute) {
  return gated_forward(x, wg, wu, bg, bu, act, nullptr);
}

std::tuple<Tensor, Tensor> gated_linear_keep_cuda(const Tensor& x, const Tensor& wg,
                                                  const Tensor& wu, const OptTensor& bg,
                                                  const OptTensor& bu, int64_t act) {
  Tensor kept;
  Tensor h = gated_forward(x, wg, wu, bg, bu, act, &kept);
  return {h, kept};
}

// -> (dx, dw_gate, dw_up, db_gate, db_up); one not asked for is empty [0]
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> gated_linear_backward_cuda(
    const Tensor& dh, const Tensor& x, const Tensor& wg, const Tensor& wu, const OptTensor& bg,
    const OptTensor& bu, const OptTensor& kept, int64_t act, std::array<bool, 5> mask) {
  const GatedShape g = gated_shape(x, wg, wu, bg, bu, act);
  const c10::cuda::CUDAGuard guard(x.device());
  need_on(dh, "dh", x);
  NEED(dh.scalar_type() == x.scalar_type() && dh.dim() == x.dim() && dh.size(-1) == g.f &&
           dh.sizes().slice(0, dh.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
       "dh must be ", x.scalar_type(), " of x's shape with ", g.f, " features, got ", dh.sizes());
  NEED((!mask[3] || has(bg)) && (!mask[4] || has(bu)),
       "a gradient was asked for of a bias that is not given");
  if (has(kept)) {
    need_on(*kept, "kept", x);
    NEED(kept->scalar_type() == at::kByte && kept->dim() == 1 && kept->is_contiguous() &&
             aligned16(*kept) && kept->size(0) == gwb_gated_linear_kept(g.rows, g.f, g.dtype),
         "kept must be what gated_linear_keep gave for x and the weights");
  }
  int64_t xs = 0, ds = 0;
  const Tensor xr = tma_rows_of(x, &xs), dr = tma_rows_of(dh, &ds);
  const auto out = [&](bool on, at::IntArrayRef shape) {
    return at::empty(on ? shape : at::IntArrayRef{0},
                     x.options().memory_format(at::MemoryFormat::Contiguous));
  };
  Tensor dx = out(mask[0], x.sizes()), dwg = out(mask[1], wg.sizes()), dwu = out(mask[2], wu.sizes());
  Tensor dbg = out(mask[3], {g.f}), dbu = out(mask[4], {g.f});
  Tensor work = at::empty({gwb_gated_linear_backward_work(g.rows, g.d, g.f)},
                          x.options().dtype(at::kByte));
  const auto at_ = [](bool on, Tensor& t) { return on ? t.data_ptr() : nullptr; };
  check_status(gwb_gated_linear_backward(
                   dr.const_data_ptr(), ds, xr.const_data_ptr(), xs, wg.const_data_ptr(),
                   wu.const_data_ptr(), ptr(bg), ptr(bu), has(kept) ? kept->data_ptr() : nullptr, g.rows,
                   g.d, g.f, (int)act, g.dtype, at_(mask[0], dx), at_(mask[1], dwg), at_(mask[2], dwu), at_(mask[3], dbg),
                   at_(mask[4], dbu), work.data_ptr(), stream_of(x)),
               "gated_linear_backward");
  return {dx, dwg, dwu, dbg, dbu};
}

struct GatedLinearFn : torch::autograd::Function<GatedLinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        const OptTensor& bg, const OptTensor& bu, int64_t act, bool recompute) {
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor h, kept;
    if (recompute) {
      static auto op = op_of<decltype(gated_linear_cuda)>("gwb200::gated_linear");
      h = op.call(x, wg, wu, bg, bu, act, true);
    } else {
      static auto op = op_of<decltype(gated_linear_keep_cuda)>("gwb200::gated_linear_keep");
      std::tie(h, kept) = op.call(x, wg, wu, bg, bu, act);
    }
    ctx->save_for_backward(
        {x, wg, wu, has(bg) ? *bg : Tensor(), has(bu) ? *bu : Tensor(), kept});
    ctx->saved_data["act"] = act;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    refuse_second_order("gated_linear_backward", grads[0], v[0], v[1], v[2], v[3], v[4]);
    if (!grads[0].defined()) return variable_list(7);
    std::array<bool, 5> mask{};
    for (int i = 0, given = 0; i < 5; ++i)
      if (v[i].defined()) mask[i] = ctx->needs_input_grad(given++);
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = op_of<decltype(gated_linear_backward_cuda)>("gwb200::gated_linear_backward");
    auto [dx, dwg, dwu, dbg, dbu] =
        op.call(grads[0], v[0], v[1], v[2], opt(v[3]), opt(v[4]), opt(v[5]),
                ctx->saved_data["act"].toInt(), mask);
    const auto give = [&](int i, Tensor& t) { return mask[i] ? t : Tensor(); };
    return {give(0, dx), give(1, dwg), give(2, dwu), give(3, dbg), give(4, dbu), Tensor(), Tensor()};
  }
};

Tensor gated_linear_autograd(const Tensor& x, const Tensor& wg, const Tensor& wu,
                             const OptTensor& bg, const OptTensor& bu, int64_t act,
                             bool recompute) {
  refuse_tangents("gated_linear", x, wg, wu, bg, bu);
  if (at::GradMode::is_enabled() &&
      (wants(x) || wants(wg) || wants(wu) || wants(bg) || wants(bu))) {
    refuse_foreign_leaves("gated_linear", x, wg, wu, bg, bu);
    return GatedLinearFn::apply(x, wg, wu, bg, bu, act, recompute);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = op_of<decltype(gated_linear_cuda)>("gwb200::gated_linear");
  return op.call(x, wg, wu, bg, bu, act, recompute);
}

}  // namespace gwb200_block

TORCH_LIBRARY_FRAGMENT(gwb200, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? shift, "
        "float eps) -> Tensor");
  m.def("layer_norm_stats(Tensor x, Tensor? weight, Tensor? bias, Tensor? scale, Tensor? shift, "
        "float eps) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor dy, Tensor x, Tensor mean, Tensor rstd, Tensor? weight, "
        "Tensor? bias, Tensor? scale, Tensor? shift, bool[5] mask) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("rotary(Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, Tensor? axis, "
        "bool interleaved, float scale, bool inverse) -> (Tensor, Tensor)");
  m.def("rotary_(Tensor(a!) q, Tensor(b!)? k, Tensor positions, Tensor inv_freq, Tensor? axis, "
        "bool interleaved, float scale, bool inverse) -> ()");
  m.def("gated_linear(Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, Tensor? b_up, "
        "int activation, bool recompute) -> Tensor");
  m.def("gated_linear_keep(Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, Tensor? b_up, "
        "int activation) -> (Tensor, Tensor)");
  m.def("gated_linear_backward(Tensor dh, Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, "
        "Tensor? b_up, Tensor? kept, int activation, bool[5] mask) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(gwb200, CUDA, m) {
  m.impl("layer_norm", &gwb200_block::layer_norm_cuda);
  m.impl("layer_norm_stats", &gwb200_block::layer_norm_stats_cuda);
  m.impl("layer_norm_backward", &gwb200_block::layer_norm_backward_cuda);
  m.impl("rotary", &gwb200_block::rotary_cuda);
  m.impl("rotary_", &gwb200_block::rotary_inplace_cuda);
  m.impl("gated_linear", &gwb200_block::gated_linear_cuda);
  m.impl("gated_linear_keep", &gwb200_block::gated_linear_keep_cuda);
  m.impl("gated_linear_backward", &gwb200_block::gated_linear_backward_cuda);
}

TORCH_LIBRARY_IMPL(gwb200, ADInplaceOrView, m) {
  m.impl("rotary_", &gwb200_block::rotary_inplace_counted);
}

TORCH_LIBRARY_IMPL(gwb200, Autograd, m) {
  m.impl("layer_norm", &gwb200_block::layer_norm_autograd);
  m.impl("rotary", &gwb200_block::rotary_autograd);
  m.impl("rotary_", &gwb200_block::rotary_inplace_autograd);
  m.impl("gated_linear", &gwb200_block::gated_linear_autograd);
}
