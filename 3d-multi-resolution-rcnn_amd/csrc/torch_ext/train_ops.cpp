// `_train_ops`: layer norm, linear cross entropy and orthogonalised updates as PyTorch operators over the C ABI (include/mr3d.h).
// The autograd nodes are C++: at the sizes of a bbox head (512 x 1024) the kernels of a forward and a backward pass take 15 us, a Python
// autograd function and the engine's way back into the interpreter take 130.
#include "common.h"

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <vector>

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_code(const at::Tensor &t) { return t.scalar_type() == at::kFloat ? MR3D_DTYPE_F32 : MR3D_DTYPE_BF16; }
bool stored(const at::Tensor &t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
void *addr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
at::Tensor or_none(const std::optional<at::Tensor> &t) { return t.has_value() ? *t : at::Tensor(); }
bool wants(const at::Tensor &t) { return t.defined() && t.requires_grad(); }

at::Tensor workspace(size_t bytes, const at::Tensor &like, size_t align, void **p) {
  at::Tensor ws = at::empty({(int64_t)(bytes + align)}, like.options().dtype(at::kByte));
  const uintptr_t a = (uintptr_t)ws.data_ptr();
  *p = (void *)((a + align - 1) / align * align);
  return ws;
}

// The operators read memory, and autograd's reverse mode is all that they take part in: a forward-mode tangent would be lost, a trace would record the
// empty result and not the kernel, function transforms hand in wrappers, and a negated view keeps its sign outside of its memory
void check_plain(const char *what, const std::vector<at::Tensor> &tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), what, " cannot be traced (torch.jit.trace)");
  static const c10::DispatchKeySet wrappers({c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                             c10::DispatchKey::Python});
  for (const at::Tensor &t : tensors) {
    if (!t.defined()) continue;
    TORCH_CHECK_NOT_IMPLEMENTED(!t.key_set().has_any(wrappers), what, " has no function transforms (torch.func, vmap, fake tensors)");
    TORCH_CHECK_NOT_IMPLEMENTED(t.layout() == at::kStrided, what, " takes dense tensors, got ", t.layout());
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what, " has no forward-mode derivative");
    TORCH_CHECK_NOT_IMPLEMENTED(!t.is_neg(), what, " does not read a negated view: resolve_neg() first");
  }
}

// The nodes below give first derivatives.  A graph through their gradients (create_graph) gets a node that says so when it is used
variable_list first_derivatives_only(variable_list grads, const char *what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (auto &g : grads) in.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivatives", (int)in.size());
  return (*node)(std::move(in));
}

// ------------------------------------------------------------------------------------------------ layer norm
constexpr int64_t kLayerNormMaxCols = 16384;

// [rows, cols] with a contiguous last axis: a view where the strides allow it, else a copy.  (A one-column view may carry any last stride.)
at::Tensor rows_view(const at::Tensor &t, int64_t cols) {
  at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, cols});
  return (r.stride(1) == 1 || (cols == 1 && r.stride(0) == 1)) && r.stride(0) >= 0 ? r : r.contiguous();
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static at::Tensor compute(const at::Tensor &x, const at::Tensor &w, const at::Tensor &b, double eps, at::Tensor *stats) {
    const int64_t cols = x.size(-1);
    const at::Tensor xr = rows_view(x, cols);
    const int64_t rows = xr.size(0);
    at::Tensor y = at::empty({rows, cols}, x.options());
    if (stats) *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    if (rows) {
      Mr3dDeviceGuard guard(x.device());
      const at::Tensor wc = w.defined() ? w.contiguous() : w, bc = b.defined() ? b.contiguous() : b;
      float *m = stats ? stats->data_ptr<float>() : nullptr;
      mr3d_check_status(mr3d_layer_norm_forward(xr.data_ptr(), xr.stride(0), addr(wc), addr(bc), y.data_ptr(), m, m ? m + rows : nullptr, rows,
                                                (int)cols, (float)eps, dtype_code(x), dtype_code(w.defined() ? w : b.defined() ? b : x),
                                                mr3d_current_stream(x)),
                        "mr3d_layer_norm_forward");
    }
    return x.dim() == 2 ? y : y.view(x.sizes());
  }

  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const std::optional<at::Tensor> &w, const std::optional<at::Tensor> &b, double eps) {
    at::Tensor stats;
    const at::Tensor wt = or_none(w), bt = or_none(b);
    at::Tensor y = compute(x, wt, bt, eps, &stats);
    ctx->save_for_backward({x, wt, stats});
    ctx->saved_data["want"] = (int64_t)(wants(x) | wants(wt) << 1 | wants(bt) << 2);
    ctx->saved_data["param"] = (int64_t)(wt.defined() ? wt : bt.defined() ? bt : x).scalar_type();
    return y;
  }

  static variable_list backward(AutogradContext *ctx, variable_list g) {
    check_plain("layer_norm's backward", g);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const int64_t want = ctx->saved_data["want"].toInt(), cols = x.size(-1);
    const auto ptype = (at::ScalarType)ctx->saved_data["param"].toInt();
    at::Tensor dx, dw, db;
    {
      at::AutoGradMode off(false);
      Mr3dDeviceGuard guard(x.device());
      const at::Tensor xr = rows_view(x, cols), dy = rows_view(g[0], cols);
      const int64_t rows = xr.size(0);
      const auto popt = x.options().dtype(ptype);
      if (want & 1) dx = at::empty({rows, cols}, x.options());
      if (want & 2) dw = rows ? at::empty({cols}, popt) : at::zeros({cols}, popt);
      if (want & 4) db = rows ? at::empty({cols}, popt) : at::zeros({cols}, popt);
      if (rows) {
        const at::Tensor wc = w.defined() ? w.contiguous() : w;
        const int dt = dtype_code(x);
        const size_t need = want & 6 ? mr3d_layer_norm_workspace_bytes(rows, (int)cols, dt) : 0;
        void *p = nullptr;
        const at::Tensor ws = need ? workspace(need, x, 16, &p) : at::Tensor();
        const float *m = stats.data_ptr<float>();
        mr3d_check_status(mr3d_layer_norm_backward(xr.data_ptr(), xr.stride(0), dy.data_ptr(), dy.stride(0), addr(wc), m, m + rows, addr(dx), addr(dw),
                                                   addr(db), rows, (int)cols, dt, ptype == at::kFloat ? MR3D_DTYPE_F32 : MR3D_DTYPE_BF16, p, need,
                                                   mr3d_current_stream(x)),
                          "mr3d_layer_norm_backward");
      }
      if (dx.defined() && x.dim() != 2) dx = dx.view(x.sizes());
    }
    return first_derivatives_only({dx, dw, db, at::Tensor()}, "layer_norm");
  }
};

at::Tensor layer_norm(const at::Tensor &x, const std::optional<at::Tensor> &weight, const std::optional<at::Tensor> &bias, double eps) {
  check_plain("layer_norm", {x, or_none(weight), or_none(bias)});
  TORCH_CHECK_VALUE(x.dim() >= 1, "layer_norm: x is a tensor [..., C]");
  TORCH_CHECK_TYPE(stored(x), "layer_norm: x is float32 or bfloat16, got ", x.scalar_type());
  const int64_t cols = x.size(-1);
  TORCH_CHECK_NOT_IMPLEMENTED(cols >= 1 && cols <= kLayerNormMaxCols, "layer_norm: 1 to ", kLayerNormMaxCols, " columns, got ", cols);
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps is at least 0, got ", eps);
  for (const auto *p : {&weight, &bias}) {
    if (!p->has_value()) continue;
    const at::Tensor &t = **p;
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == cols && t.device() == x.device(), "layer_norm: weight and bias are [", cols, "] on ", x.device(), ", got ",
                      t.sizes(), " on ", t.device());
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == x.scalar_type(), "layer_norm: weight and bias are float32 or ", x.scalar_type(),
                     ", got ", t.scalar_type());
  }
  TORCH_CHECK_TYPE(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "layer_norm: weight and bias have one type");
  TORCH_CHECK_NOT_IMPLEMENTED(x.is_cuda(), "layer_norm has no CPU fallback");
  if (at::GradMode::is_enabled() && (wants(x) || wants(or_none(weight)) || wants(or_none(bias)))) return LayerNorm::apply(x, weight, bias, eps);
  return LayerNorm::compute(x, or_none(weight), or_none(bias), eps, nullptr);
}

// ------------------------------------------------------------------------------------------------ linear cross entropy
// [rows, cols] as the kernels read it.  Strides of axes of one element say nothing (contiguous() lets them be): they are set to the packed ones
at::Tensor packed_rows(const at::Tensor &t) {
  const int64_t rows = t.size(0), cols = t.size(1);
  const int64_t r = rows > 1 ? t.stride(0) : cols, c = cols > 1 ? t.stride(1) : 1;
  if (c != 1 || r < cols) return t.contiguous();
  return r == t.stride(0) && c == t.stride(1) ? t : t.as_strided({rows, cols}, {r, c});
}

struct CeArgs {
  at::Tensor label, row_weight, avg, valid;
  double avg_factor;
  int64_t ignore_index;
};

bool capturing(const at::Tensor &t) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  TORCH_CHECK(hipStreamIsCapturing((hipStream_t)mr3d_current_stream(t), &st) == hipSuccess, "hipStreamIsCapturing failed");
  return st != hipStreamCaptureStatusNone;
}

// The forward call leaves the gradients too; backward multiplies them by the incoming one, in place and once: a graph that holds only one of the two
// would multiply again at every replay, or hand out memory that the next replay overwrites, so they are captured together or not at all
struct LinearCe : torch::autograd::Function<LinearCe> {
  static at::Tensor compute(const at::Tensor &x, const at::Tensor &w, const at::Tensor &bias, const CeArgs &c, int want, at::Tensor (&grads)[3]) {
    const int64_t k = w.size(1), classes = w.size(0);
    Mr3dDeviceGuard guard(x.device());
    const auto fopt = x.options().dtype(at::kFloat);
    const at::Tensor xr = packed_rows(x.reshape({-1, k})), wr = packed_rows(w);
    const int64_t rows = xr.size(0);
    if (want & 1) grads[0] = at::empty({rows, k}, x.options());
    if (want & 2) grads[1] = rows ? at::empty({classes, k}, w.options()) : at::zeros({classes, k}, w.options());
    if (want & 4) grads[2] = rows ? at::empty({classes}, bias.options()) : at::zeros({classes}, bias.options());
    if (!rows) return at::zeros({1}, fopt);
    at::Tensor loss = at::empty({1}, fopt);
    const at::Tensor b = bias.defined() ? bias.contiguous() : bias;
    mr3d_linear_ce a{};
    a.x = xr.data_ptr(); a.weight = wr.data_ptr(); a.bias = addr(b);
    a.labels = (const long long *)c.label.data_ptr<int64_t>();
    a.row_weight = (const float *)addr(c.row_weight);
    a.avg_factor_dev = (const float *)addr(c.avg);
    a.valid_rows_dev = (const int *)addr(c.valid);
    a.loss = loss.data_ptr<float>();
    a.dx = addr(grads[0]); a.dweight = addr(grads[1]); a.dbias = addr(grads[2]);
    a.x_stride = xr.stride(0); a.weight_stride = wr.stride(0); a.ignore_index = c.ignore_index;
    a.avg_factor = (float)c.avg_factor;
    a.rows = (int)rows; a.hidden = (int)k; a.classes = (int)classes;
    a.dtype = dtype_code(x); a.param_dtype = dtype_code(b.defined() ? b : x);
    a.want_dx = want & 1; a.want_dweight = want >> 1 & 1; a.want_dbias = want >> 2 & 1;
    const size_t need = mr3d_linear_cross_entropy_workspace_bytes(&a);
    void *p;
    const at::Tensor ws = workspace(need, x, 1024, &p);
    mr3d_check_status(mr3d_linear_cross_entropy(&a, p, need, mr3d_current_stream(x)), "mr3d_linear_cross_entropy");
    return loss;
  }

  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &w, const std::optional<at::Tensor> &bias, const CeArgs &c) {
    const at::Tensor b = or_none(bias);
    at::Tensor grads[3];
    ctx->saved_data["captured"] = capturing(x);
    at::Tensor loss = compute(x, w, b, c, wants(x) | wants(w) << 1 | wants(b) << 2, grads);
    for (int i = 0; i < 3; ++i)
      if (grads[i].defined()) ctx->saved_data["g" + std::to_string(i)] = i == 0 && x.dim() != 2 ? grads[i].view(x.sizes()) : grads[i];
    return loss;
  }

  static variable_list backward(AutogradContext *ctx, variable_list g) {
    check_plain("linear_cross_entropy's backward", g);
    TORCH_CHECK(!ctx->saved_data.count("used"), "linear_cross_entropy: a second backward through the same loss (its gradients were handed over by the "
                                                "first); call linear_cross_entropy again");
    TORCH_CHECK(ctx->saved_data["captured"].toBool() == capturing(g[0]),
                "linear_cross_entropy: the call and its backward are captured into graphs together or not at all");
    ctx->saved_data["used"] = true;
    variable_list out(4);
    {
      at::AutoGradMode off(false);
      const at::Tensor f = g[0].to(at::kFloat).contiguous();
      mr3d_span spans[3];
      int n = 0;
      for (int i = 0; i < 3; ++i) {
        const std::string key = "g" + std::to_string(i);
        if (!ctx->saved_data.count(key)) continue;
        out[i] = ctx->saved_data[key].toTensor();
        ctx->saved_data.erase(key);
        if (out[i].numel()) spans[n++] = {out[i].data_ptr(), (long long)out[i].numel(), dtype_code(out[i]), 0};
      }
      if (n) {
        Mr3dDeviceGuard guard(f.device());
        mr3d_check_status(mr3d_scale_by(spans, n, f.data_ptr<float>(), mr3d_current_stream(f)), "mr3d_scale_by");
      }
    }
    return first_derivatives_only(std::move(out), "linear_cross_entropy");
  }
};

at::Tensor linear_cross_entropy(const at::Tensor &x, const at::Tensor &weight, const at::Tensor &label, const std::optional<at::Tensor> &row_weight,
                                const std::optional<at::Tensor> &bias, const std::optional<at::Tensor> &avg_dev, std::optional<double> avg_host,
                                const std::optional<at::Tensor> &valid_rows, int64_t ignore_index) {
  check_plain("linear_cross_entropy", {x, weight, label, or_none(row_weight), or_none(bias), or_none(avg_dev), or_none(valid_rows)});
#define CE "linear_cross_entropy: "
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1), CE "x is [..., K] and weight [C, K], got ", x.sizes(), " and ", weight.sizes());
  TORCH_CHECK_TYPE(stored(x) && weight.scalar_type() == x.scalar_type(), CE "x and weight are both float32 or both bfloat16, got ", x.scalar_type(), " and ",
                   weight.scalar_type());
  const int64_t classes = weight.size(0), k = weight.size(1);
  TORCH_CHECK_NOT_IMPLEMENTED(classes >= 1 && classes <= 1 << 20 && k >= 1 && k <= 1 << 16 && x.numel() / k <= 1 << 22,
                              CE "1 to 2^20 classes, 1 to 2^16 features, up to 2^22 rows");
  TORCH_CHECK_VALUE(!bias || (bias->dim() == 1 && bias->size(0) == classes && (bias->scalar_type() == at::kFloat || bias->scalar_type() == x.scalar_type())),
                    CE "bias is [", classes, "], float32 or ", x.scalar_type());
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  TORCH_CHECK_VALUE(label.sizes() == lead && label.scalar_type() == at::kLong, CE "label is ", lead, ", int64");
  CeArgs c;
  if (row_weight) {
    TORCH_CHECK_VALUE(row_weight->sizes() == lead, CE "row_weight is ", lead);
    TORCH_CHECK_NOT_IMPLEMENTED(!row_weight->requires_grad(), "linear_cross_entropy is not differentiable in row_weight");
  }
  TORCH_CHECK_VALUE(!avg_dev || (avg_dev->numel() == 1 && avg_dev->device() == x.device()), CE "avg_factor is a number or one value on the device of x");
  TORCH_CHECK_NOT_IMPLEMENTED(!avg_dev || !avg_dev->requires_grad(), "linear_cross_entropy is not differentiable in avg_factor");
  TORCH_CHECK_VALUE(!avg_host || (float)*avg_host > 0, CE "avg_factor is positive in float32");
  TORCH_CHECK_VALUE(!valid_rows || (valid_rows->numel() == 1 && valid_rows->scalar_type() == at::kInt), CE "valid_rows is one int32 value on the device");
  for (const at::Tensor &t : {weight, or_none(bias), label, or_none(row_weight), or_none(valid_rows)})
    TORCH_CHECK_VALUE(!t.defined() || t.device() == x.device(), CE "all tensors are on one device");
#undef CE
  TORCH_CHECK_NOT_IMPLEMENTED(x.is_cuda(), "linear_cross_entropy has no CPU fallback");
  c.label = label.contiguous();
  if (row_weight) c.row_weight = row_weight->to(at::kFloat).contiguous();
  if (avg_dev) c.avg = avg_dev->detach().to(at::kFloat).contiguous();
  if (valid_rows) c.valid = valid_rows->contiguous();
  c.avg_factor = avg_host ? *avg_host : 0.;
  c.ignore_index = ignore_index;
  const at::Tensor b = or_none(bias);
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(b))) return LinearCe::apply(x, weight, bias, c);
  at::Tensor none[3];
  return LinearCe::compute(x, weight, b, c, 0, none);
}

// ------------------------------------------------------------------------------------------------ orthogonalised updates
std::vector<at::Tensor> orthogonalize(const std::vector<at::Tensor> &mats, int64_t steps, double a, double b, double c, double eps,
                                      const std::optional<std::vector<at::Tensor>> &out) {
  check_plain("orthogonalize", mats);
  if (out) check_plain("orthogonalize", *out);
  at::AutoGradMode off(false);
  std::vector<at::Tensor> flat, outs;
  for (const at::Tensor &t : mats) {
    TORCH_CHECK_TYPE(t.dim() >= 2, "orthogonalize: a matrix is a tensor of two or more axes, got ", t.sizes());
    TORCH_CHECK_TYPE(stored(t), "orthogonalize: a matrix is float32 or bfloat16, got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.device() == mats[0].device(), "orthogonalize: the matrices of a list are on one device");
    flat.push_back(t.dim() == 2 ? t : t.reshape({t.size(0), t.size(0) ? t.numel() / t.size(0) : 0}));
    TORCH_CHECK_NOT_IMPLEMENTED(flat.back().size(0) <= 1 << 20 && flat.back().size(1) <= 1 << 20, "orthogonalize: up to 2^20 rows and columns");
  }
  auto small = [](double v) { return v >= -16 && v <= 16; };
  TORCH_CHECK_VALUE(steps >= 1 && steps <= 100 && eps >= 0 && small(a) && small(b) && small(c),
                    "orthogonalize: 1 to 100 steps, eps at least 0, coefficients within 16");
  if (mats.empty()) return outs;
  TORCH_CHECK_NOT_IMPLEMENTED(mats[0].is_cuda(), "orthogonalize has no CPU fallback");
  if (out) {
    TORCH_CHECK_VALUE(out->size() == mats.size(), "orthogonalize: one out per matrix");
    outs = *out;
    for (size_t i = 0; i < mats.size(); ++i)
      TORCH_CHECK_VALUE(outs[i].sizes() == mats[i].sizes() && outs[i].scalar_type() == mats[i].scalar_type() && outs[i].device() == mats[i].device() &&
                            outs[i].is_contiguous(),
                        "orthogonalize: an out is contiguous and has its matrix's shape, type and device");
    // No out may lie on another matrix or out: some are written while others are still read.  A matrix that is its own out counts once.
    struct Span {
      const char *from, *to;
      bool written;
    };
    std::vector<Span> spans;
    for (size_t i = 0; i < mats.size(); ++i) {
      const at::Tensor &m = flat[i];
      if (!m.numel()) continue;
      const char *o = (const char *)outs[i].data_ptr(), *in = (const char *)m.data_ptr();
      spans.push_back({o, o + outs[i].nbytes(), true});
      if (in == o && m.is_contiguous()) continue;
      spans.push_back({in, in + ((m.size(0) - 1) * m.stride(0) + (m.size(1) - 1) * m.stride(1) + 1) * m.element_size(), false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span &p, const Span &q) { return p.from < q.from; });
    const char *read = nullptr, *written = nullptr;
    for (const Span &s : spans) {
      TORCH_CHECK_VALUE(s.from >= written && (!s.written || s.from >= read),
                        "orthogonalize: an out overlaps another out or a matrix that is not its own, contiguous one");
      const char *&end = s.written ? written : read;
      end = std::max(end, s.to);
    }
  } else {
    // one buffer per type; every result starts on its own 256 bytes
    outs.resize(mats.size());
    for (const auto type : {at::kFloat, at::kBFloat16}) {
      int64_t total = 0;
      const int64_t unit = type == at::kFloat ? 64 : 128;
      for (const at::Tensor &t : mats)
        if (t.scalar_type() == type) total += (t.numel() + unit - 1) / unit * unit;
      if (!total) {
        for (size_t i = 0; i < mats.size(); ++i)
          if (mats[i].scalar_type() == type) outs[i] = at::empty(mats[i].sizes(), mats[i].options());
        continue;
      }
      const at::Tensor buf = at::empty({total}, mats[0].options().dtype(type));
      int64_t at = 0;
      for (size_t i = 0; i < mats.size(); ++i) {
        const at::Tensor &t = mats[i];
        if (t.scalar_type() != type) continue;
        outs[i] = buf.narrow(0, at, t.numel()).view(t.sizes());
        at += (t.numel() + unit - 1) / unit * unit;
      }
    }
  }
  std::vector<mr3d_matrix> table;
  for (size_t i = 0; i < mats.size(); ++i) {
    const at::Tensor &t = flat[i];
    if (t.numel()) table.push_back({t.data_ptr(), outs[i].data_ptr(), t.size(0), t.size(1), t.stride(0), t.stride(1), dtype_code(t), 0});
  }
  if (table.empty()) return outs;
  Mr3dDeviceGuard guard(mats[0].device());
  const size_t need = mr3d_orthogonalize_workspace_bytes(table.data(), (int)table.size());
  TORCH_CHECK(need, "orthogonalize: the list is refused");
  void *p;
  const at::Tensor ws = workspace(need, mats[0], 256, &p);
  mr3d_check_status(mr3d_orthogonalize(table.data(), (int)table.size(), (int)steps, (float)a, (float)b, (float)c, (float)eps, p, need,
                                       mr3d_current_stream(mats[0])),
                    "mr3d_orthogonalize");
  if (out)
    for (const at::Tensor &t : outs)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // a graph that saved it says so
  return outs;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
  m.def("linear_cross_entropy", &linear_cross_entropy, py::call_guard<py::gil_scoped_release>());
  m.def("orthogonalize", &orthogonalize, py::call_guard<py::gil_scoped_release>());
}
