// torch binding of the operators that a training step calls often: the gated linear
// recurrence, norm + gate + residual, and AdamW over a list of tensors, over the C ABI
// in include/mambaqc_b200.h.
//
// The other operators are bound with ctypes and torch.autograd.Function. A Python
// autograd function costs 100 us and more of host time for a forward and a backward
// with eight inputs and nothing inside, which is above what the kernels take at most
// sizes. Small tensors, forward and backward in a loop: the recurrence (four inputs with
// a gradient) 79 us, the norm (eight) 115, a built-in layer norm (two) 73, a product of
// two tensors 60. It holds no kernels and no state: arguments are
// checked in Python (kernels/*.py) before they come here, memory is torch's, and
// failures of the C ABI become RuntimeErrors with its message.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cstdlib>
#include <cstring>

#include "mambaqc_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------------ the library

struct Api {
  decltype(&mqc_last_error) last_error;
  decltype(&mqc_status_string) status_string;
  decltype(&mqc_gated_scan_fwd) gated_scan_fwd;
  decltype(&mqc_gated_scan_bwd_workspace_size) gated_scan_bwd_workspace_size;
  decltype(&mqc_gated_scan_bwd) gated_scan_bwd;
  decltype(&mqc_gated_scan_step) gated_scan_step;
  decltype(&mqc_norm_gate_fwd) norm_gate_fwd;
  decltype(&mqc_norm_gate_bwd_workspace_size) norm_gate_bwd_workspace_size;
  decltype(&mqc_norm_gate_bwd) norm_gate_bwd;
  decltype(&mqc_adamw_step) adamw_step;
  decltype(&mqc_adamw_moments) adamw_moments;
  decltype(&mqc_grad_norm_workspace_size) grad_norm_workspace_size;
  decltype(&mqc_grad_norm) grad_norm;
};
Api api = {};

template <typename F>
void resolve(void* lib, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(lib, name));
  TORCH_CHECK(f != nullptr, "mambaqc_b200: the library has no ", name);
}

// Binds the functions of the library at `path` (the one that ctypes loads).
void init(const std::string& path) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib != nullptr, "mambaqc_b200: ", dlerror());
  resolve(lib, "mqc_last_error", api.last_error);
  resolve(lib, "mqc_status_string", api.status_string);
  resolve(lib, "mqc_gated_scan_fwd", api.gated_scan_fwd);
  resolve(lib, "mqc_gated_scan_bwd_workspace_size", api.gated_scan_bwd_workspace_size);
  resolve(lib, "mqc_gated_scan_bwd", api.gated_scan_bwd);
  resolve(lib, "mqc_gated_scan_step", api.gated_scan_step);
  resolve(lib, "mqc_norm_gate_fwd", api.norm_gate_fwd);
  resolve(lib, "mqc_norm_gate_bwd_workspace_size", api.norm_gate_bwd_workspace_size);
  resolve(lib, "mqc_norm_gate_bwd", api.norm_gate_bwd);
  resolve(lib, "mqc_adamw_step", api.adamw_step);
  resolve(lib, "mqc_adamw_moments", api.adamw_moments);
  resolve(lib, "mqc_grad_norm_workspace_size", api.grad_norm_workspace_size);
  resolve(lib, "mqc_grad_norm", api.grad_norm);
}

void check(int rc, const char* what) {
  if (rc == MQC_OK) return;
  throw std::runtime_error(std::string(what) + " failed: " + api.status_string(rc) + " (" +
                           std::to_string(rc) + "): " + api.last_error());
}

// --------------------------------------------------------------------- tensors

int dtype_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? MQC_DTYPE_F32 : MQC_DTYPE_BF16;
}
template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor defined(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Counts a write in place by a kernel, so that autograd refuses a graph that saved what
// was there before. (Tensors of inference mode have no count.)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The operators have no forward-mode derivative: an input that carries a tangent is
// refused, where reading its value alone would make the derivative vanish.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what,
                ": forward-mode derivatives are not supported");
}

// Contiguous fp32 (the tensor itself where it is that already).
Tensor as_f32(const Tensor& t) {
  if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
  return t.to(at::kFloat).contiguous();
}
Tensor as_type(const Tensor& t, at::ScalarType type) {
  return !t.defined() || t.scalar_type() == type ? t : t.to(type);
}
Tensor like(const Tensor& t, at::ScalarType type) {
  return at::empty(t.sizes(), t.options().dtype(type).requires_grad(false));
}
Tensor like(const Tensor& t) { return like(t, t.scalar_type()); }
Tensor f32(const Tensor& on, at::IntArrayRef sizes) {
  return at::empty(sizes, on.options().dtype(at::kFloat).requires_grad(false));
}

// A tensor whose rows (of `width` contiguous elements, evenly spaced over all leading
// dimensions) the kernels can read in place, copied if they cannot; *row: their stride.
Tensor rows_of(const Tensor& t, int64_t width, int64_t* row) {
  *row = width;
  if (t.is_contiguous()) return t;
  const int64_t dims = t.dim();
  bool ok = t.stride(-1) == 1 && dims >= 2 && t.stride(-2) >= width;
  int64_t expect = ok ? t.stride(-2) : 0;
  *row = expect;
  for (int64_t d = dims - 2; ok && d >= 0; --d) {
    if (t.size(d) > 1 && t.stride(d) != expect) ok = false;
    expect *= t.size(d);
  }
  if (ok) return t;
  *row = width;
  return t.contiguous();
}

// Where each call is asked to check itself (MAMBAQC_B200_SYNC_CHECK=1): an error if a
// kernel has reported a wait that it gave up to the status word of the tensor's device.
void check_status(int64_t status, const Tensor& on) {
  const char* wanted = std::getenv("MAMBAQC_B200_SYNC_CHECK");
  if (wanted == nullptr || std::strcmp(wanted, "1") != 0) return;
  at::NoGradGuard no_grad;
  Tensor word = at::from_blob(reinterpret_cast<void*>(status), {1},
                              on.options().dtype(at::kInt).requires_grad(false));
  const int value = word.item<int>();
  if (value == 0) return;
  word.zero_();
  if (value & MQC_DEVICE_STATUS_TIMEOUT)
    throw std::runtime_error(
        "mambaqc_b200: a bounded device-side wait timed out; results of that launch are invalid");
}

cudaStream_t stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// What autograd's backward returned becomes an error when it is itself differentiated
// (as torch.autograd.function.once_differentiable does).
variable_list once(variable_list grads, const variable_list& given) {
  bool needed = false;
  for (const Tensor& g : given) needed = needed || wants_grad(g);
  if (!at::GradMode::is_enabled() || !needed) return grads;
  variable_list fake;
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    g = g.detach();
    g.set_requires_grad(true);
    fake.push_back(g);
  }
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "mambaqc_b200: trying to differentiate twice a function that is differentiable once",
      int64_t(fake.size()));
  variable_list marked = (*node)(std::move(fake));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[k++];
  return grads;
}

// ------------------------------------------------------------- gated recurrence

struct ScanInputs {
  Tensor x, r, i, lambda, reset;
  int64_t x_row, r_row, i_row;
};

mqc_gated_scan_args scan_args(const ScanInputs& in, double sharpness, int64_t status,
                              bool give_up) {
  mqc_gated_scan_args a = {};
  a.batch = in.x.size(0);
  a.seq_len = in.x.size(1);
  a.channels = in.x.size(2);
  a.dtype = dtype_of(in.x);
  a.sharpness = float(sharpness);
  a.x = ptr(in.x);
  a.r = ptr(in.r);
  a.i = ptr(in.i);
  a.x_row = in.x_row;
  a.r_row = in.r_row;
  a.i_row = in.i_row;
  a.lambda_ = ptr(in.lambda);
  a.reset = ptr(in.reset);
  a.status = reinterpret_cast<void*>(status);
  a.give_up = give_up;
  return a;
}

// (y, hT, ckpt); hT and ckpt are undefined where they are not wanted.
std::tuple<Tensor, Tensor, Tensor> scan_forward(const ScanInputs& in, const Tensor& h0,
                                                double sharpness, bool want_state, bool keep,
                                                int64_t status, bool give_up) {
  c10::cuda::CUDAGuard guard(in.x.device());
  const int64_t b = in.x.size(0), t = in.x.size(1), d = in.x.size(2);
  Tensor y = like(in.x), hT, ckpt;
  if (want_state) hT = f32(in.x, {b, d});
  if (keep) ckpt = f32(in.x, {b, (t + MQC_GATED_SCAN_TILE - 1) / MQC_GATED_SCAN_TILE, d});
  mqc_gated_scan_args a = scan_args(in, sharpness, status, give_up);
  a.h0 = ptr(h0);
  a.y = ptr(y);
  a.hT = ptr(hT);
  a.ckpt = ptr(ckpt);
  check(api.gated_scan_fwd(&a, stream_of(in.x)), "mqc_gated_scan_fwd");
  check_status(status, in.x);
  return {y, hT, ckpt};
}

ScanInputs scan_inputs(const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& lambda,
                       const Tensor& reset) {
  ScanInputs in;
  const int64_t d = x.size(2);
  in.x = rows_of(x, d, &in.x_row);
  in.r = rows_of(r, d, &in.r_row);
  in.i = rows_of(i, d, &in.i_row);
  in.lambda = as_f32(lambda);
  in.reset = reset.defined() ? reset.contiguous() : reset;
  return in;
}

struct GatedScan : public torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& r,
                               const Tensor& i, const Tensor& lambda, const OptTensor& h0_,
                               const OptTensor& reset, double sharpness, bool want_state,
                               int64_t status, bool give_up) {
    const Tensor h0 = defined(h0_);
    const ScanInputs in = scan_inputs(x, r, i, lambda, defined(reset));
    auto [y, hT, ckpt] = scan_forward(in, as_f32(h0), sharpness, want_state, true, status, give_up);
    ctx->save_for_backward({in.x, in.r, in.i, in.lambda, in.reset, ckpt});
    ctx->saved_data["sharpness"] = sharpness;
    ctx->saved_data["status"] = status;
    if (give_up) ctx->saved_data["give_up"] = true;
    ctx->saved_data["lambda"] = int64_t(lambda.scalar_type());
    ctx->saved_data["h0"] = h0.defined() ? int64_t(h0.scalar_type()) : int64_t(-1);
    ctx->set_materialize_grads(false);
    return want_state ? variable_list{y, hT} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const ScanInputs in = scan_inputs(saved[0], saved[1], saved[2], saved[3], saved[4]);
    c10::cuda::CUDAGuard guard(in.x.device());
    const int64_t b = in.x.size(0), t = in.x.size(1), d = in.x.size(2);
    const int64_t h0_type = ctx->saved_data["h0"].toInt();
    const int64_t status = ctx->saved_data["status"].toInt();
    mqc_gated_scan_args a = scan_args(in, ctx->saved_data["sharpness"].toDouble(), status,
                                      ctx->saved_data.count("give_up") != 0);
    a.ckpt = ptr(saved[5]);
    a.dy_row = d;
    Tensor dy;
    if (grads[0].defined()) dy = rows_of(as_type(grads[0], in.x.scalar_type()), d, &a.dy_row);
    const Tensor dhT = as_f32(grads.size() > 1 ? grads[1] : Tensor());
    Tensor dx = like(in.x), dr = like(in.x), di = like(in.x), dlambda = like(in.lambda), dh0;
    // the inputs that exist are counted: x, r, i, lambda, h0
    if (h0_type >= 0 && ctx->needs_input_grad(4)) dh0 = f32(in.x, {b, d});
    const size_t bytes = api.gated_scan_bwd_workspace_size(b, t, d);
    const Tensor ws = f32(in.x, {int64_t(bytes / 4) + 1});
    a.dy = ptr(dy);
    a.dhT = ptr(dhT);
    a.dx = ptr(dx);
    a.dr = ptr(dr);
    a.di = ptr(di);
    a.dlambda = ptr(dlambda);
    a.dh0 = ptr(dh0);
    check(api.gated_scan_bwd(&a, ptr(ws), bytes, stream_of(in.x)), "mqc_gated_scan_bwd");
    check_status(status, in.x);
    dlambda = as_type(dlambda, at::ScalarType(ctx->saved_data["lambda"].toInt()));
    if (dh0.defined()) dh0 = as_type(dh0, at::ScalarType(h0_type));
    return once({dx, dr, di, dlambda, dh0, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, grads);
  }
};

std::tuple<Tensor, OptTensor> gated_scan(const Tensor& x, const Tensor& r, const Tensor& i,
                                         const Tensor& lambda, const OptTensor& h0,
                                         const OptTensor& reset, double sharpness, bool want_state,
                                         int64_t status, bool give_up) {
  const Tensor h = defined(h0), rst = defined(reset);
  refuse_tangents("gated_linear_scan", {&x, &r, &i, &lambda, &h});
  if (at::GradMode::is_enabled() && (x.requires_grad() || r.requires_grad() || i.requires_grad() ||
                                     lambda.requires_grad() || wants_grad(h))) {
    variable_list out =
        GatedScan::apply(x, r, i, lambda, h0, reset, sharpness, want_state, status, give_up);
    return {out[0], want_state ? OptTensor(out[1]) : OptTensor()};
  }
  at::NoGradGuard no_grad;
  auto [y, hT, ckpt] = scan_forward(scan_inputs(x, r, i, lambda, rst), as_f32(h), sharpness,
                                    want_state, false, status, give_up);
  return {y, want_state ? OptTensor(hT) : OptTensor()};
}

Tensor gated_step(const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& lambda,
                  const Tensor& h, double sharpness, const OptTensor& out) {
  refuse_tangents("gated_linear_step", {&x, &r, &i, &lambda, &h});
  at::NoGradGuard no_grad;
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t d = x.size(1);
  int64_t x_row, r_row, i_row;
  const Tensor xs = rows_of(x, d, &x_row), rs = rows_of(r, d, &r_row), is = rows_of(i, d, &i_row);
  const Tensor lam = as_f32(lambda);
  Tensor y = out.has_value() ? *out : like(x);
  check(api.gated_scan_step(ptr(xs), x_row, ptr(rs), r_row, ptr(is), i_row, ptr(lam), ptr(h), ptr(y),
                            x.size(0), d, float(sharpness), dtype_of(x), stream_of(x)),
        "mqc_gated_scan_step");
  written(h);
  if (out.has_value()) written(y);
  return y;
}

// ------------------------------------------------------ norm + gate + residual

struct NormInputs {
  Tensor x, y, z, weight, bias, scale, next_weight, next_bias;
  int64_t z_row = 0;
  int kind = 0;
  double eps = 0;
  at::ScalarType branch = at::kFloat;  // of y, z, n
};

int64_t width_of(const Tensor& x) { return x.size(-1); }
int64_t row_count(const Tensor& x) { return width_of(x) ? x.numel() / width_of(x) : 0; }

mqc_norm_gate_args norm_args(const NormInputs& in) {
  mqc_norm_gate_args a = {};
  a.rows = row_count(in.x);
  a.width = width_of(in.x);
  a.z_row = in.z_row;
  a.x_dtype = dtype_of(in.x);
  a.y_dtype = in.branch == at::kFloat ? MQC_DTYPE_F32 : MQC_DTYPE_BF16;
  a.norm = in.kind;
  a.eps = float(in.eps);
  a.x = ptr(in.x);
  a.y = ptr(in.y);
  a.z = ptr(in.z);
  a.weight = ptr<float>(in.weight);
  a.bias = ptr<float>(in.bias);
  a.scale = ptr<float>(in.scale);
  a.next_weight = ptr<float>(in.next_weight);
  a.next_bias = ptr<float>(in.next_bias);
  return a;
}

NormInputs norm_inputs(const Tensor& x, const Tensor& y, const Tensor& z, const Tensor& weight,
                       const Tensor& bias, const Tensor& scale, const Tensor& next_weight,
                       const Tensor& next_bias, int64_t kind, double eps, at::ScalarType branch) {
  NormInputs in;
  in.x = x.contiguous();
  in.z_row = width_of(x);
  if (y.defined()) {
    in.y = y.contiguous();
    in.z = rows_of(z, width_of(x), &in.z_row);
  }
  in.weight = as_f32(weight);
  in.bias = as_f32(bias);
  in.scale = as_f32(scale);
  in.next_weight = as_f32(next_weight);
  in.next_bias = as_f32(next_bias);
  in.kind = int(kind);
  in.eps = eps;
  in.branch = branch;
  return in;
}

// (out, n, stats); out is undefined without y, n without a next weight.
std::tuple<Tensor, Tensor, Tensor> norm_forward(const NormInputs& in, bool keep) {
  c10::cuda::CUDAGuard guard(in.x.device());
  Tensor out, n, stats;
  if (in.y.defined()) out = like(in.x);
  if (in.next_weight.defined()) n = like(in.x, in.branch);
  if (keep) stats = f32(in.x, {row_count(in.x), 4});
  mqc_norm_gate_args a = norm_args(in);
  a.out = ptr(out);
  a.n = ptr(n);
  a.stats = ptr(stats);
  check(api.norm_gate_fwd(&a, stream_of(in.x)), "mqc_norm_gate_fwd");
  return {out, n, stats};
}

struct NormGate : public torch::autograd::Function<NormGate> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& y_,
                               const OptTensor& z_, const OptTensor& weight_,
                               const OptTensor& bias_, const OptTensor& scale_,
                               const OptTensor& next_weight_, const OptTensor& next_bias_,
                               int64_t kind, double eps, int64_t branch) {
    const Tensor y = defined(y_), z = defined(z_), weight = defined(weight_), bias = defined(bias_);
    const Tensor scale = defined(scale_), next_weight = defined(next_weight_);
    const Tensor next_bias = defined(next_bias_);
    const NormInputs in = norm_inputs(x, y, z, weight, bias, scale, next_weight, next_bias, kind,
                                      eps, at::ScalarType(branch));
    auto [out, n, stats] = norm_forward(in, true);
    ctx->save_for_backward(
        {in.x, in.y, in.z, in.weight, in.bias, in.scale, in.next_weight, in.next_bias, stats});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["branch"] = branch;
    std::vector<int64_t> types;
    for (const Tensor& t : {weight, bias, scale, next_weight, next_bias})
      types.push_back(t.defined() ? int64_t(t.scalar_type()) : -1);
    ctx->saved_data["types"] = types;
    ctx->set_materialize_grads(false);
    variable_list result;
    if (out.defined()) result.push_back(out);
    if (n.defined()) result.push_back(n);
    return result;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const NormInputs in = norm_inputs(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7],
                                      ctx->saved_data["kind"].toInt(),
                                      ctx->saved_data["eps"].toDouble(),
                                      at::ScalarType(ctx->saved_data["branch"].toInt()));
    const std::vector<int64_t> types = ctx->saved_data["types"].toIntVector();
    c10::cuda::CUDAGuard guard(in.x.device());
    const bool post = in.y.defined(), next = in.next_weight.defined();
    Tensor dout, dn;
    if (post && grads[0].defined()) dout = as_type(grads[0], in.x.scalar_type()).contiguous();
    if (next && grads[post ? 1 : 0].defined())
      dn = as_type(grads[post ? 1 : 0], in.branch).contiguous();
    Tensor dx = like(in.x), dy, dz;
    if (post) {
      dy = like(in.x, in.branch);
      dz = like(in.x, in.branch);
    }
    const Tensor params[5] = {in.weight, in.bias, in.scale, in.next_weight, in.next_bias};
    Tensor sums[5];
    size_t input = post ? 3 : 1;  // the inputs that exist are counted: x, y, z, then these
    for (int k = 0; k < 5; ++k)
      if (params[k].defined() && ctx->needs_input_grad(input++)) sums[k] = like(params[k]);
    mqc_norm_gate_args a = norm_args(in);
    const size_t bytes = api.norm_gate_bwd_workspace_size(a.rows, a.width);
    const Tensor ws = f32(in.x, {int64_t(bytes / 4) + 1});
    a.stats = ptr(s[8]);
    a.dout = ptr(dout);
    a.dn = ptr(dn);
    a.dx = ptr(dx);
    a.dy = ptr(dy);
    a.dz = ptr(dz);
    a.dweight = ptr<float>(sums[0]);
    a.dbias = ptr<float>(sums[1]);
    a.dscale = ptr<float>(sums[2]);
    a.dnext_weight = ptr<float>(sums[3]);
    a.dnext_bias = ptr<float>(sums[4]);
    check(api.norm_gate_bwd(&a, ptr(ws), bytes, stream_of(in.x)), "mqc_norm_gate_bwd");
    for (int k = 0; k < 5; ++k)
      if (sums[k].defined()) sums[k] = as_type(sums[k], at::ScalarType(types[k]));
    return once({dx, dy, dz, sums[0], sums[1], sums[2], sums[3], sums[4], Tensor(), Tensor(),
                 Tensor()},
                grads);
  }
};

// (out, n), each None where it does not exist.
std::tuple<OptTensor, OptTensor> norm_gate(const Tensor& x, const OptTensor& y, const OptTensor& z,
                                           const OptTensor& weight, const OptTensor& bias,
                                           const OptTensor& scale, const OptTensor& next_weight,
                                           const OptTensor& next_bias, int64_t kind, double eps,
                                           bool branch_f32) {
  const at::ScalarType branch = branch_f32 ? at::kFloat : at::kBFloat16;
  const Tensor t[7] = {defined(y),     defined(z),           defined(weight),   defined(bias),
                       defined(scale), defined(next_weight), defined(next_bias)};
  refuse_tangents(t[0].defined() ? "norm_gate_residual" : "residual_norm",
                  {&x, &t[0], &t[1], &t[2], &t[3], &t[4], &t[5], &t[6]});
  bool grad = x.requires_grad();
  for (const Tensor& v : t) grad = grad || wants_grad(v);
  if (at::GradMode::is_enabled() && grad) {
    const variable_list got = NormGate::apply(x, y, z, weight, bias, scale, next_weight, next_bias,
                                              kind, eps, int64_t(branch));
    if (!t[0].defined()) return {OptTensor(), got[0]};
    return {got[0], got.size() > 1 ? OptTensor(got[1]) : OptTensor()};
  }
  at::NoGradGuard no_grad;
  auto [out, n, stats] = norm_forward(
      norm_inputs(x, t[0], t[1], t[2], t[3], t[4], t[5], t[6], kind, eps, branch), false);
  return {out.defined() ? OptTensor(out) : OptTensor(), n.defined() ? OptTensor(n) : OptTensor()};
}

// ------------------------------------------------------------------------ AdamW

using List = std::vector<Tensor>;

template <typename P = void*>
std::vector<P> pointers(const List& list) {
  std::vector<P> p;
  p.reserve(list.size());
  for (const Tensor& t : list) p.push_back(t.data_ptr());
  return p;
}
std::vector<int64_t> sizes_of(const List& list) {
  std::vector<int64_t> n;
  n.reserve(list.size());
  for (const Tensor& t : list) n.push_back(t.numel());
  return n;
}

// The index of the first tensor of `list` that is not contiguous, of `count` elements
// each (or as many as `like` has), on `device` and of one of the two types; -1 if none.
int64_t misfit(const List& list, const std::vector<int64_t>& count, int64_t device,
               at::ScalarType a, at::ScalarType b) {
  for (size_t k = 0; k < list.size(); ++k) {
    const Tensor& t = list[k];
    if (!(t.is_cuda() && t.get_device() == device && t.is_contiguous() && t.numel() == count[k] &&
          (t.scalar_type() == a || t.scalar_type() == b)))
      return int64_t(k);
  }
  return -1;
}

// Whether the lists of an AdamW step fit together (else Python says what does not).
bool lists_fit(const List& params, const List& grads, const List& m, const List& v,
               const List& em, const List& ev, bool bits8) {
  const size_t n = params.size();
  if (n == 0 || !params[0].is_cuda() || grads.size() != n || m.size() != n || v.size() != n ||
      (bits8 && (em.size() != n || ev.size() != n)))
    return false;
  const std::vector<int64_t> count = sizes_of(params);
  const int64_t dev = params[0].get_device();
  const at::ScalarType state = bits8 ? at::kByte : at::kFloat;
  if (misfit(m, count, dev, state, state) >= 0 || misfit(v, count, dev, state, state) >= 0)
    return false;
  // the values of 8-bit moments alone: their codes stand in for parameters and gradients
  if (!(params[0].is_same(m[0]) && grads[0].is_same(m[0])) &&
      (misfit(params, count, dev, at::kFloat, at::kBFloat16) >= 0 ||
       misfit(grads, count, dev, at::kFloat, at::kBFloat16) >= 0))
    return false;
  if (!bits8) return true;
  std::vector<int64_t> blocks(n);
  for (size_t k = 0; k < n; ++k) blocks[k] = (count[k] + MQC_ADAMW_BLOCK - 1) / MQC_ADAMW_BLOCK;
  return misfit(em, blocks, dev, at::kByte, at::kByte) < 0 &&
         misfit(ev, blocks, dev, at::kByte, at::kByte) < 0;
}

// [norm, factor]; max_norm < 0: no clipping.
Tensor grad_norm(const List& grads, double max_norm) {
  c10::cuda::CUDAGuard guard(grads[0].device());
  const size_t bytes = api.grad_norm_workspace_size(int64_t(grads.size()));
  // the partial sums (8-byte aligned), then the two results
  const Tensor all = f32(grads[0], {int64_t(bytes / 4) + 2});
  const std::vector<int64_t> count = sizes_of(grads);
  const auto p = pointers<const void*>(grads);
  std::vector<int32_t> types;
  types.reserve(grads.size());
  for (const Tensor& g : grads) types.push_back(dtype_of(g));
  float* out = ptr<float>(all) + bytes / 4;
  check(api.grad_norm(int64_t(grads.size()), count.data(), p.data(), types.data(), max_norm,
                      out, ptr(all), bytes, stream_of(all)),
        "mqc_grad_norm");
  return all.narrow(0, int64_t(bytes / 4), 2);
}

void adamw_step(const List& params, const List& grads, const List& m, const List& v, const List& em,
                const List& ev, const std::vector<int64_t>& ordinals, const OptTensor& clip,
                int64_t step, double lr, double beta1, double beta2, double eps,
                double weight_decay, bool bits8, bool carry, int64_t seed) {
  c10::cuda::CUDAGuard guard(params[0].device());
  // one call for each pair of parameter and gradient types
  for (int kind = 0; kind < 4; ++kind) {
    std::vector<int64_t> numel, ordinal;
    std::vector<void*> p, pm, pv, pem, pev;
    std::vector<const void*> g;
    for (size_t k = 0; k < params.size(); ++k) {
      if (dtype_of(params[k]) * 2 + dtype_of(grads[k]) != kind) continue;
      numel.push_back(params[k].numel());
      ordinal.push_back(ordinals[k]);
      p.push_back(params[k].data_ptr());
      g.push_back(grads[k].data_ptr());
      pm.push_back(m[k].data_ptr());
      pv.push_back(v[k].data_ptr());
      if (bits8) {
        pem.push_back(em[k].data_ptr());
        pev.push_back(ev[k].data_ptr());
      }
    }
    if (p.empty()) continue;
    mqc_adamw_args a = {};
    a.count = int64_t(p.size());
    a.numel = numel.data();
    a.ordinal = ordinal.data();
    a.param = p.data();
    a.grad = g.data();
    a.exp_avg = pm.data();
    a.exp_avg_sq = pv.data();
    a.exp_avg_exponent = bits8 ? pem.data() : nullptr;
    a.exp_avg_sq_exponent = bits8 ? pev.data() : nullptr;
    a.clip = clip.has_value() ? static_cast<const float*>(clip->data_ptr()) : nullptr;
    a.lr = lr;
    a.beta1 = beta1;
    a.beta2 = beta2;
    a.eps = eps;
    a.weight_decay = weight_decay;
    a.step = step;
    a.param_dtype = kind / 2;
    a.grad_dtype = kind % 2;
    a.state_bits = bits8 ? 8 : 32;
    a.flags = carry ? MQC_ADAMW_CARRY : 0;
    a.seed = uint32_t(seed);
    check(api.adamw_step(&a, stream_of(params[0])), "mqc_adamw_step");
  }
  for (const List* list : {&params, &m, &v, &em, &ev})
    for (const Tensor& t : *list) written(t);
}

std::tuple<List, List> adamw_moments(const List& m, const List& v, const List& em, const List& ev) {
  c10::cuda::CUDAGuard guard(m[0].device());
  List out_m, out_r;
  for (const Tensor& t : m) {
    out_m.push_back(like(t, at::kBFloat16));
    out_r.push_back(like(t, at::kBFloat16));
  }
  const std::vector<int64_t> count = sizes_of(m);
  const auto pm = pointers<const void*>(m), pv = pointers<const void*>(v);
  const auto pem = pointers<const void*>(em), pev = pointers<const void*>(ev);
  const auto om = pointers(out_m), orr = pointers(out_r);
  check(api.adamw_moments(int64_t(m.size()), count.data(), pm.data(), pv.data(), pem.data(),
                          pev.data(), om.data(), orr.data(), stream_of(m[0])),
        "mqc_adamw_moments");
  return {out_m, out_r};
}

}  // namespace

PYBIND11_MODULE(_torch_ops, mod) {
  mod.attr("built_for") = MQC_BUILT_FOR;  // what csrc/build.py looks for in this file
  mod.def("init", &init);
  mod.def("gated_scan", &gated_scan);
  mod.def("gated_step", &gated_step);
  mod.def("norm_gate", &norm_gate);
  mod.def("lists_fit", &lists_fit);
  mod.def("grad_norm", &grad_norm);
  mod.def("adamw_step", &adamw_step);
  mod.def("adamw_moments", &adamw_moments);
}
