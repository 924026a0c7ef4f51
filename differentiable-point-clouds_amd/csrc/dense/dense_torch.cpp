// dense_torch.cpp -- compiled PyTorch binding of the dense-layer operators: what dense.py does through ctypes (checks, allocations, the
// current stream, autograd bookkeeping), in C++, because a training step's calls are launch-bound at the sizes of the networks
// (80 x 4096 -> 1024 with gradients: 55 us of device work, 140 us of host work from Python, 70 from here).  No arithmetic happens here: every
// number comes out of the library, reached through dlopen on the path that Python hands over.
//
// Built by __graft_entry__.build() with torch.utils.cpp_extension (host compiler only) into csrc/dense/build_torch/.
#include <torch/extension.h>

#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <string>
#include <vector>

#include "dpc_dense.h"

namespace {
using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  std::string path;
  bool host_memory = false;
  decltype(&dpc_dense_linear_sizes) sizes = nullptr;
  decltype(&dpc_dense_linear_forward) forward = nullptr;
  decltype(&dpc_dense_linear_backward) backward = nullptr;
  decltype(&dpc_dense_linear_serve_workspace) serve_workspace = nullptr;
  decltype(&dpc_dense_linear_serve) serve = nullptr;
  decltype(&dpc_dense_orthogonal_workspace) orthogonal_workspace = nullptr;
  decltype(&dpc_dense_orthogonal) orthogonal = nullptr;
};
std::mutex g_mu;
std::vector<Api*> g_apis;      // never freed: libraries stay open

template <class F>
void sym(void* h, const char* name, F& f, const std::string& path) {
  f = reinterpret_cast<F>(dlsym(h, name));
  TORCH_CHECK(f != nullptr, path, ": symbol ", name, " not found");
}

// -> id of the library; the same path opened twice gives the same id
int64_t open_library(const std::string& path, bool host_memory) {
  std::lock_guard<std::mutex> lk(g_mu);
  for (size_t i = 0; i < g_apis.size(); ++i)
    if (g_apis[i]->path == path) return (int64_t)i;
  void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(h != nullptr, "dlopen(", path, "): ", dlerror());
  Api* a = new Api;
  a->path = path;
  a->host_memory = host_memory;
  sym(h, "dpc_dense_linear_sizes", a->sizes, path);
  sym(h, "dpc_dense_linear_forward", a->forward, path);
  sym(h, "dpc_dense_linear_backward", a->backward, path);
  sym(h, "dpc_dense_linear_serve_workspace", a->serve_workspace, path);
  sym(h, "dpc_dense_linear_serve", a->serve, path);
  sym(h, "dpc_dense_orthogonal_workspace", a->orthogonal_workspace, path);
  sym(h, "dpc_dense_orthogonal", a->orthogonal, path);
  decltype(&dpc_dense_abi_struct_bytes) bytes = nullptr;
  sym(h, "dpc_dense_abi_struct_bytes", bytes, path);
  TORCH_CHECK(bytes(0) == sizeof(DpcDenseMatrix) && bytes(1) == sizeof(DpcDenseSteps), path,
              ": the structs are laid out differently in the library and in this binding (rebuild both)");
  g_apis.push_back(a);
  return (int64_t)g_apis.size() - 1;
}
const Api& api_of(int64_t lib) {
  std::lock_guard<std::mutex> lk(g_mu);
  TORCH_CHECK(lib >= 0 && (size_t)lib < g_apis.size(), "unknown library id ", lib);
  return *g_apis[(size_t)lib];
}

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == 0, "DPC_RC:", rc, ":", what); }   // Python turns it into its own error

int code_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return DPC_DENSE_F32;
    case at::kBFloat16: return DPC_DENSE_BF16;
    case at::kHalf: return DPC_DENSE_F16;
    default: TORCH_CHECK_TYPE(false, what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
  return -1;
}

// where a tensor lies: where the library computes, and with the others
void check_place(const Api& api, const Tensor& t, const Tensor& first) {
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, "expected a dense tensor, got layout ", t.layout());
  TORCH_CHECK_VALUE(!api.host_memory || t.is_cpu(), "emulation library needs host tensors");
  TORCH_CHECK_VALUE(api.host_memory || t.is_cuda(), "the dense operators need tensors on a ROCm device (no CPU fallback)");
  TORCH_CHECK_VALUE(t.device() == first.device(), "tensors on different devices: ", first.device(), " and ", t.device());
}

// forward-mode derivatives are not computed here, and not dropped either
void check_no_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "the dense operators carry no forward-mode derivatives: pass the primal, or detach");
}

dpc_dense_stream_t stream_of(const Api& api, const Tensor& ref) {
  if (api.host_memory) return nullptr;
  return (dpc_dense_stream_t)c10::hip::getCurrentHIPStream(ref.device().index()).stream();
}

Tensor buffer(at::IntArrayRef shape, const Tensor& like, at::ScalarType type, bool poison) {
  Tensor t = at::empty(shape, like.options().dtype(type).requires_grad(false));
  if (poison) t.view(at::kByte).fill_(255);
  return t;
}
// bytes, 256-byte aligned
struct Bytes {
  Tensor hold;
  void* at = nullptr;
  size_t n = 0;
};
void* aligned(const Tensor& t) { return reinterpret_cast<void*>(((uintptr_t)t.data_ptr() + 255) & ~(uintptr_t)255); }
Bytes bytes(size_t n, const Tensor& like, bool poison) {
  Bytes b;
  b.n = n;
  if (n == 0) return b;
  b.hold = at::empty({(int64_t)n + 256}, like.options().dtype(at::kByte).requires_grad(false));
  if (poison) b.hold.fill_(255);
  b.at = aligned(b.hold);
  return b;
}

// [rows, cols] with neighbouring columns and rows that do not overlap, the values as they lie in memory
Tensor rows_of(const Tensor& t_) {
  const Tensor t = t_.resolve_neg();
  if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) return t.contiguous();
  return t;
}
size_t ld_of(const Tensor& t) { return (size_t)(t.size(0) > 1 ? t.stride(0) : t.size(1)); }
int dim_of(int64_t n) {
  TORCH_CHECK_VALUE(n <= 0x7fffffff, "an axis of ", n, " is too long");
  return (int)n;
}
// While a stream records a graph: a leaf whose earlier, eager autograd graph still lives would make the recorded backward pass wait for that
// graph's stream, which ends the process.  Refused here, where it can still be said.
void check_recording(const Api& api, const Tensor& t) {
  if (api.host_memory || !t.requires_grad() || t.grad_fn()) return;
  c10::OptionalDeviceGuard guard(t.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto leaf = torch::autograd::impl::try_get_grad_accumulator(t);
  TORCH_CHECK(!leaf || !leaf->stream().has_value() || leaf->stream()->id() == c10::hip::getCurrentHIPStream(t.device().index()).id(),
              "linear_fp8 is being recorded into a graph while the autograd graph of an earlier eager call of the same leaf lives: drop what keeps "
              "it (an output, a loss) before the recording");
}
const void* ptr(const optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// ---- the product ------------------------------------------------------------------------------------------------------------------
struct LinearFp8 : public torch::autograd::Function<LinearFp8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const optional<Tensor>& bias, int64_t lib, int64_t needs,
                        bool poison) {
    const Api& api = api_of(lib);
    const Tensor x = rows_of(x_), w = rows_of(w_);
    const int m = dim_of(x.size(0)), k = dim_of(x.size(1)), n = dim_of(w.size(0));
    const int xt = code_of(x, "x"), wt = code_of(w, "weight"), bt = bias.has_value() ? code_of(*bias, "bias") : 0;
    c10::OptionalDeviceGuard guard(x.device());
    size_t sizes[3];
    check_rc(api.sizes(m, k, n, xt, wt, (int)needs, sizes), "dpc_dense_linear_sizes");
    Tensor out = buffer({m, n}, x, x.scalar_type(), poison);
    const Bytes saved = bytes(sizes[0], x, poison), ws = bytes(sizes[1], x, poison);
    check_rc(api.forward(stream_of(api, x), m, k, n, x.data_ptr(), ld_of(x), xt, w.data_ptr(), ld_of(w), wt, ptr(bias), bt, out.data_ptr(),
                         (int)needs, saved.at, saved.n, ws.at, ws.n),
             "dpc_dense_linear_forward");
    if (needs != 0) {
      Tensor keep = saved.hold;
      if (!keep.defined()) keep = at::empty({0}, x.options().dtype(at::kByte).requires_grad(false));
      ctx->save_for_backward({keep});
      ctx->saved_data["sizes"] = std::vector<int64_t>{lib, m, k, n, (int64_t)x.scalar_type(), (int64_t)w.scalar_type(),
                                                      bias.has_value() ? (int64_t)bias->scalar_type() : -1, needs, poison ? 1 : 0,
                                                      (int64_t)sizes[0], (int64_t)sizes[2],
                                                      (int64_t)((uintptr_t)saved.at - (saved.n > 0 ? (uintptr_t)saved.hold.data_ptr() : 0))};
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const std::vector<int64_t> s = ctx->saved_data["sizes"].toIntVector();
    const Api& api = api_of(s[0]);
    const int m = (int)s[1], k = (int)s[2], n = (int)s[3], needs = (int)s[7];
    const auto xt = (at::ScalarType)s[4], wt = (at::ScalarType)s[5];
    const bool poison = s[8] != 0;
    Tensor saved = ctx->get_saved_variables()[0];
    variable_list out(6);
    const bool again = at::GradMode::is_enabled() && grads[0].requires_grad();
    {
      at::AutoGradMode off(false);
      const Tensor dy = rows_of(grads[0]);
      c10::OptionalDeviceGuard guard(dy.device());
      if (needs & 1) out[0] = buffer({m, k}, dy, xt, poison);
      if (needs & 2) out[1] = buffer({n, k}, dy, wt, poison);
      if (needs & 4) out[2] = buffer({n}, dy, (at::ScalarType)s[6], poison);
      const Bytes ws = bytes((size_t)s[10], dy, poison);
      const auto p = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
      const void* kept = nullptr;
      if (s[9] > 0) {            // (hooks on saved tensors may have brought it back at another address)
        kept = static_cast<const char*>(saved.data_ptr()) + s[11];
        if ((uintptr_t)kept % 256 != 0) {
          const Bytes again_at = bytes((size_t)s[9], dy, false);
          at::from_blob(again_at.at, {s[9]}, again_at.hold.options()).copy_(saved.narrow(0, s[11], s[9]));
          saved = again_at.hold, kept = again_at.at;
        }
      }
      check_rc(api.backward(stream_of(api, dy), m, k, n, dy.data_ptr(), ld_of(dy), code_of(dy, "dy"), wt == at::kFloat ? DPC_DENSE_F32 : wt == at::kHalf ? DPC_DENSE_F16 : DPC_DENSE_BF16,
                            out[2].defined() ? code_of(out[2], "bias") : 0, kept, (size_t)s[9], p(out[0]), p(out[1]), p(out[2]), ws.at, ws.n),
               "dpc_dense_linear_backward");
    }
    if (again) {                 // differentiable once: a second differentiation says so
      auto error = std::make_shared<torch::autograd::DelayedError>("linear_fp8 is differentiable once only", 3);
      variable_list first(out.begin(), out.begin() + 3);
      for (auto& t : first)
        if (t.defined()) t.requires_grad_(true);
      first = (*error)(std::move(first));
      std::copy(first.begin(), first.end(), out.begin());
    }
    return out;
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const optional<Tensor>& bias_, int64_t lib, bool poison) {
  const Api& api = api_of(lib);
  check_place(api, x, x);
  check_place(api, w, x);
  code_of(x, "x");
  code_of(w, "weight");
  TORCH_CHECK_VALUE(w.dim() == 2, "weight must be [out_features, in_features], got ", w.sizes());
  const int64_t n = w.size(0), k = w.size(1);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "x must be [..., ", k, "], got ", x.sizes());
  optional<Tensor> bias = bias_;
  if (bias.has_value()) {
    check_place(api, *bias, x);
    code_of(*bias, "bias");
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == n, "bias must be [", n, "], got ", bias->sizes());
    bias = bias->resolve_neg().contiguous();
  }
  const bool grad = at::GradMode::is_enabled();
  if (grad) {
    check_recording(api, x);
    check_recording(api, w);
    if (bias_.has_value()) check_recording(api, *bias_);      // (as given: a copy of a strided leaf is none)
  }
  const int64_t needs = grad ? (x.requires_grad() ? 1 : 0) | (w.requires_grad() ? 2 : 0) | (bias.has_value() && bias->requires_grad() ? 4 : 0) : 0;
  if (x.dim() == 2) return LinearFp8::apply(x, w, bias, lib, needs, poison);
  int64_t rows = 1;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
  shape.back() = n;
  return LinearFp8::apply(x.reshape({rows, k}), w, bias, lib, needs, poison).reshape(shape);
}

Tensor serve(const Tensor& x, const Tensor& values, const Tensor& scales, int64_t k, const optional<Tensor>& bias_, int64_t lib, bool poison) {
  const Api& api = api_of(lib);
  for (const Tensor& t : {x, values, scales}) check_place(api, t, x);
  const int xt = code_of(x, "x");
  const int64_t blocks = k >= 0 ? (k + 127) / 128 : -1;
  TORCH_CHECK_VALUE(k >= 0 && values.dim() == 2 && values.scalar_type() == at::kFloat8_e4m3fn && values.size(1) == blocks * 128,
                    "values must be float8_e4m3fn [out_features, ", blocks * 128, "], got ", values.scalar_type(), " ", values.sizes());
  const int64_t n = values.size(0);
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kByte && scales.dim() == 2 && scales.size(0) == blocks && scales.size(1) == n,
                    "scales must be uint8 [", blocks, ", ", n, "], got ", scales.scalar_type(), " ", scales.sizes());
  TORCH_CHECK_VALUE(values.is_contiguous() && scales.is_contiguous() && (uintptr_t)values.data_ptr() % 16 == 0 && !values.is_neg() && !scales.is_neg(),
                    "values and scales must be contiguous, values 16-byte aligned and no negative views");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "x must be [..., ", k, "], got ", x.sizes());
  optional<Tensor> bias = bias_;
  int bt = 0;
  if (bias.has_value()) {
    check_place(api, *bias, x);
    bt = code_of(*bias, "bias");
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == n, "bias must be [", n, "], got ", bias->sizes());
  }
  TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && (x.requires_grad() || (bias.has_value() && bias->requires_grad()))),
                    "a packed weight serves only: call under torch.no_grad(), or pass the weight itself");
  check_no_tangent(x);
  if (bias.has_value()) check_no_tangent(*bias);
  at::AutoGradMode off(false);
  if (bias.has_value()) bias = bias->resolve_neg().contiguous();
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  int64_t rows = 1;
  for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
  shape.back() = n;
  const Tensor x2 = rows_of(x.dim() == 2 ? x : x.reshape({rows, k}));
  c10::OptionalDeviceGuard guard(x.device());
  Tensor out = buffer(shape, x, x.scalar_type(), poison);
  const int m = dim_of(rows), ki = dim_of(k), ni = dim_of(n);
  const Bytes ws = bytes(api.serve_workspace(m, ki, ni, xt), x, poison);
  check_rc(api.serve(stream_of(api, x), m, ki, ni, x2.data_ptr(), ld_of(x2), xt, values.data_ptr(), static_cast<const uint8_t*>(scales.data_ptr()),
                     ptr(bias), bt, out.data_ptr(), ws.at, ws.n),
           "dpc_dense_linear_serve");
  return out;
}

// ---- orthogonalisation and the update ------------------------------------------------------------------------------------------------
DpcDenseSteps steps_of(int64_t steps, const std::vector<double>& coefficients, double eps) {
  DpcDenseSteps s{};
  s.steps = (int32_t)steps;
  s.eps = eps;
  for (int64_t i = 0; i < 3 * steps; ++i) s.coefficients[i / 3][i % 3] = (float)coefficients[(size_t)i];
  return s;
}

struct Entry {
  Tensor grad, momentum, out;
  int64_t rows, cols;
  double scale;
  size_t offset;              // of the matrix in grad and out, in elements
};

// the library's calls for a list of matrices; everything that can be refused is refused when they are planned, before the first of them runs
struct Call {
  std::vector<DpcDenseMatrix> matrices;
  int code;
};
struct Calls {
  std::vector<Call> list;
  size_t workspace = 0;       // one for all of them: they follow each other on the stream
};

Calls plan_orthogonal(const Api& api, const std::vector<Entry>& all, const DpcDenseSteps& s) {
  check_rc(api.orthogonal(nullptr, 0, nullptr, 0, &s, nullptr, 0), "dpc_dense_orthogonal");      // (coefficients)
  Calls calls;
  for (at::ScalarType type : {at::kFloat, at::kBFloat16, at::kHalf}) {
    const size_t width = type == at::kFloat ? 4 : 2;
    bool open = false;
    for (const Entry& e : all) {
      if (e.out.scalar_type() != type) continue;
      if (!open || calls.list.back().matrices.size() == DPC_DENSE_MAX_MATRICES) calls.list.push_back(Call{{}, code_of(e.out, "a matrix")});
      open = true;
      calls.list.back().matrices.push_back(DpcDenseMatrix{static_cast<const char*>(e.grad.data_ptr()) + e.offset * width,
                                                          e.momentum.defined() ? static_cast<float*>(e.momentum.data_ptr()) : nullptr,
                                                          static_cast<char*>(e.out.data_ptr()) + e.offset * width, dim_of(e.rows), dim_of(e.cols),
                                                          (float)e.scale, 0});
    }
  }
  for (const Call& c : calls.list) {
    const size_t need = api.orthogonal_workspace((int)c.matrices.size(), c.matrices.data(), c.code);
    check_rc(need > 0 ? DPC_DENSE_OK : DPC_DENSE_E_SHAPE, "dpc_dense_orthogonal");
    calls.workspace = std::max(calls.workspace, need);
  }
  return calls;
}

void run_orthogonal(const Api& api, const Calls& calls, const Tensor& first, const DpcDenseSteps& s, bool poison) {
  c10::OptionalDeviceGuard guard(first.device());
  const Bytes ws = bytes(calls.workspace, first, poison);
  for (const Call& c : calls.list)
    check_rc(api.orthogonal(stream_of(api, first), (int)c.matrices.size(), c.matrices.data(), c.code, &s, ws.at, ws.n), "dpc_dense_orthogonal");
}

std::vector<Tensor> newton_schulz(const std::vector<Tensor>& mats, int64_t steps, const std::vector<double>& coefficients, double eps, bool batched,
                                  int64_t lib, bool poison) {
  const Api& api = api_of(lib);
  at::AutoGradMode off(false);
  std::vector<Tensor> outs;
  std::vector<Entry> all;
  for (const Tensor& g : mats) {
    check_place(api, g, mats[0]);
    check_no_tangent(g);
    code_of(g, "a matrix");
    TORCH_CHECK_VALUE(!batched || g.dim() >= 2, "expected [..., rows, cols], got ", g.sizes());
    TORCH_CHECK_VALUE(batched || g.dim() == 2, "expected matrices, got ", g.sizes());
  }
  for (const Tensor& g_ : mats) {
    const Tensor g = g_.detach().resolve_neg().contiguous();
    outs.push_back(buffer(g.sizes(), g, g.scalar_type(), poison));
    if (g.numel() == 0) continue;
    const int64_t r = g.size(-2), c = g.size(-1);
    for (int64_t i = 0; i < g.numel() / (r * c); ++i) all.push_back(Entry{g, Tensor(), outs.back(), r, c, 1.0, (size_t)(i * r * c)});
  }
  const DpcDenseSteps s = steps_of(steps, coefficients, eps);
  const Calls calls = plan_orthogonal(api, all, s);
  if (!all.empty()) run_orthogonal(api, calls, all[0].out, s, poison);
  return outs;
}

// contiguous, or channels_last: then a weight's storage is a matrix [size(0), the rest]
optional<at::MemoryFormat> format_of(const Tensor& t) {
  if (t.is_contiguous()) return at::MemoryFormat::Contiguous;
  if (t.dim() == 4 && t.is_contiguous(at::MemoryFormat::ChannelsLast)) return at::MemoryFormat::ChannelsLast;
  return std::nullopt;
}

void muon_update(const std::vector<Tensor>& weights, const std::vector<Tensor>& grads, const std::vector<Tensor>& momenta, double lr,
                 const optional<Tensor>& lr_tensor, double momentum, bool nesterov, double weight_decay, int64_t steps,
                 const std::vector<double>& coefficients, double eps, int64_t adjust, int64_t lib, bool poison) {
  const Api& api = api_of(lib);
  at::AutoGradMode off(false);
  DpcDenseSteps s = steps_of(steps, coefficients, eps);
  s.nesterov = nesterov, s.momentum = momentum, s.weight_decay = weight_decay, s.lr = lr;
  const Tensor* first = weights.empty() ? nullptr : &weights[0];
  if (lr_tensor.has_value()) {
    check_place(api, *lr_tensor, first ? *first : *lr_tensor);
    check_no_tangent(*lr_tensor);
    s.lr_device = static_cast<const float*>(lr_tensor->data_ptr());
  }
  std::vector<Entry> all;
  struct Span {
    uintptr_t lo, hi;
    bool written;
  };
  std::vector<Span> spans;
  const auto span = [&](const Tensor& t, bool written) {
    if (t.numel() > 0) spans.push_back({(uintptr_t)t.data_ptr(), (uintptr_t)t.data_ptr() + t.nbytes(), written});
  };
  for (size_t i = 0; i < weights.size(); ++i) {
    const Tensor &w = weights[i], &m = momenta[i];
    Tensor g = grads[i];
    for (const Tensor* t : {&w, &m, static_cast<const Tensor*>(&g)}) check_place(api, *t, *first), check_no_tangent(*t);
    code_of(w, "a weight");
    TORCH_CHECK_VALUE(w.dim() >= 2, "weight ", i, " has shape ", w.sizes(), ": only matrices can be orthogonalised");
    TORCH_CHECK_VALUE(g.scalar_type() == w.scalar_type() && g.sizes() == w.sizes(), "gradient ", i, " is ", g.scalar_type(), " ", g.sizes(),
                      ", its weight ", w.scalar_type(), " ", w.sizes());
    TORCH_CHECK_VALUE(m.scalar_type() == at::kFloat && m.sizes() == w.sizes(), "momentum ", i, " must be float32 ", w.sizes(), ", got ",
                      m.scalar_type(), " ", m.sizes());
    const auto form = format_of(w);
    TORCH_CHECK_VALUE(form.has_value() && m.is_contiguous(*form), "weight ", i, " and its momentum must be contiguous, or both channels_last");
    TORCH_CHECK_VALUE(!w.is_neg() && !m.is_neg(), "weight ", i, " or its momentum is a negative view: nothing can be written through it");
    if (w.numel() == 0) continue;
    g = g.detach().resolve_neg();
    if (!g.is_contiguous(*form)) g = g.contiguous(*form);
    const int64_t r = w.size(0), c = w.numel() / r;
    const double scale = adjust == 0 ? 0.2 * std::sqrt((double)std::max(r, c)) : adjust == 1 ? std::sqrt(std::max(1.0, (double)r / c)) : 1.0;
    span(w, true);
    span(m, true);
    span(g, false);
    all.push_back(Entry{g, m, w, r, c, scale, 0});
  }
  if (lr_tensor.has_value() && !all.empty()) span(*lr_tensor, false);
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  uintptr_t end = 0, end_written = 0;
  for (const Span& p : spans) {
    TORCH_CHECK_VALUE(p.lo >= (p.written ? end : end_written), "weights and momenta must not share memory with each other or with the gradients");
    end = std::max(end, p.hi);
    if (p.written) end_written = std::max(end_written, p.hi);
  }
  const Calls calls = plan_orthogonal(api, all, s);
  if (all.empty()) return;
  for (const Entry& e : all) {   // autograd graphs that hold the old weights are told
    e.out.unsafeGetTensorImpl()->bump_version();
    e.momentum.unsafeGetTensorImpl()->bump_version();
  }
  run_orthogonal(api, calls, all[0].out, s, poison);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "compiled binding of the dense-layer operators (include/dpc_dense.h)";
  m.def("open_library", &open_library, "dlopen a build of the library; returns its id");
  m.def("linear", &linear, "dense.linear_fp8 with a weight tensor");
  m.def("serve", &serve, "dense.linear_fp8 with a packed weight");
  m.def("newton_schulz", &newton_schulz, "dense.newton_schulz over a list");
  m.def("muon_update", &muon_update, "dense.muon_update");
}
