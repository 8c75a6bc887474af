// Host side of the package in native code: operators on torch tensors and the autograd Functions of the training
// path, each a few allocations and calls into libmega_b200.so on the current stream.
//
// At the small shapes of the path the host is what a call costs: an operator through Python (checks, allocations,
// thirty converted arguments) takes 20 - 40 us, a Python autograd Function as much again each way, against 3 - 10 us
// of device time per launch.  Here an operator takes 3 - 5 us and the backward of a training pass runs in the
// autograd engine without the interpreter.
//
// fairseq/modules/norm_layer/{timestep_norm,sequence_norm}.py, fairseq/modules/fused_ops/*.py and
// fairseq/modules/moving_average_gated_attention.py:317-414 of the reference are what the Functions stand in for.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <tuple>
#include <unordered_map>
#include <vector>

#include "mega_b200.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

namespace {

PyObject* g_error = nullptr;   // the package's MegaError

void check(int status, const char* what) {
  if (status == MEGA_OK) return;
  std::string msg = std::string(what) + ": " + mega_status_string(status);
  if (status == MEGA_ERR_CUDA) msg += std::string(" (") + mega_last_cuda_error() + ")";
  if (g_error && PyGILState_Check()) {
    PyErr_SetString(g_error, msg.c_str());
    throw py::error_already_set();
  }
  throw std::runtime_error(msg);   // (a backward in the autograd engine's threads)
}

void on_cuda(const Tensor& t) {
  if (t.defined() && !t.is_cuda())
    throw std::runtime_error("mega_b200 ops run on CUDA tensors only (there is no CPU fallback)");
}
template <typename... Ts>
void on_cuda(const Tensor& t, const Ts&... rest) {
  on_cuda(t);
  on_cuda(rest...);
}

// The library takes pointers: what it reads behind one has to be there.
void expect(bool ok, const char* what) {
  if (!ok) throw py::value_error(what);
}
void expect_numel(const Tensor& t, int64_t n, const char* what) {
  if (t.defined() && t.numel() != n)
    throw py::value_error(std::string(what) + " has " + std::to_string(t.numel()) + " values, not " + std::to_string(n));
}

// device of the call and its current stream
struct Where {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Where(const Tensor& t) : guard(t.device()), stream(at::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MEGA_F32;
    case at::kBFloat16: return MEGA_BF16;
    case at::kHalf: return MEGA_F16;
    default: throw py::type_error("mega_b200 supports float32, bfloat16 and float16 activations");
  }
}

Tensor none() { return Tensor(); }
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
float* fptr(const Tensor& t) { return ptr<float>(t); }

// fp32, contiguous (parameters, statistics, states are small)
Tensor f32c(const Tensor& t) {
  if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
  return t.detach().to(at::kFloat).contiguous();
}
// Parameters in fp32, contiguous, side by side: one launch for all that are not so already
std::vector<Tensor> f32_all(const std::vector<Tensor>& ts, void* stream) {
  std::vector<Tensor> out(ts.size());
  const void* src[8];
  float* dst[8];
  int64_t n[8], total = 0;
  int count = 0;
  auto half = [](const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; };
  for (const auto& t : ts) total += half(t) ? (t.numel() + 3) / 4 * 4 : 0;
  Tensor all;
  if (total) all = at::empty({total}, at::TensorOptions().dtype(at::kFloat).device(ts[0].device()));
  int64_t from = 0;
  int dt = -1;
  for (size_t i = 0; i < ts.size(); ++i) {
    const Tensor& t = ts[i];
    if (!half(t) || !t.is_contiguous() || (dt >= 0 && dtype_of(t) != dt) || count == 8) {
      out[i] = f32c(t);
      continue;
    }
    dt = dtype_of(t);
    out[i] = all.narrow(0, from, t.numel()).view(t.sizes());
    src[count] = t.data_ptr();
    dst[count] = fptr(all) + from;
    n[count++] = t.numel();
    from += (t.numel() + 3) / 4 * 4;
  }
  if (count) check(mega_to_float(src, dst, n, count, dt, stream), "to_float");
  return out;
}
// complex64 of `dims` dimensions as its interleaved floats; a real tensor has no imaginary part, unless it is (..., 2) fp32
// and so interleaved already
Tensor c64(const Tensor& t, int64_t dims) {
  if (!t.defined()) return t;
  Tensor d = t.detach();
  if (d.scalar_type() == at::kFloat && d.dim() > dims && d.size(-1) == 2) return d.contiguous();
  if (d.scalar_type() != at::kComplexFloat) d = d.to(at::kComplexFloat);
  return at::view_as_real(d.contiguous());
}

Tensor mask_u8(const Tensor& mask, int64_t bsz, int64_t length) {
  if (!mask.defined()) return mask;
  if (mask.dim() != 2 || mask.size(0) != bsz || mask.size(1) != length)
    throw py::value_error("padding_mask must be (batch, length) = (" + std::to_string(bsz) + ", " + std::to_string(length) + ")");
  return mask.scalar_type() == at::kBool ? mask.contiguous() : mask.ne(0).contiguous();
}

// uninitialised, strided like t (contiguous when t's strides leave gaps)
Tensor like(const Tensor& t) {
  if (t.is_contiguous()) return at::empty(t.sizes(), t.options().requires_grad(false));
  if (t.is_non_overlapping_and_dense()) return at::empty_strided(t.sizes(), t.strides(), t.options().requires_grad(false));
  return at::empty(t.sizes(), t.options().requires_grad(false));
}
Tensor floats(at::IntArrayRef size, const Tensor& t) {
  return at::empty(size, at::TensorOptions().dtype(at::kFloat).device(t.device()));
}
Tensor counts(int64_t n, const Tensor& t) { return at::empty({n}, at::TensorOptions().dtype(at::kLong).device(t.device())); }

#define STRIDES3(t) (t).stride(0), (t).stride(1), (t).stride(2)

// ------------------------------------------------------------------------------------------------ EMA
struct Coeffs {
  Tensor p, q, g;
};

void check_rows(int64_t rows, int64_t dim, bool bidir) {
  if (rows != (bidir ? 2 * dim : dim))
    throw py::value_error("coefficient rows " + std::to_string(rows) + " do not match embed_dim " + std::to_string(dim));
}
// p (K, N); q, gamma (K, N), complex ones interleaved; omega (D); a state (B, D, N)
void check_coeffs(const Tensor& p, const Tensor& q, const Tensor& g, const Tensor& omega, const Tensor& h, bool cplx, int64_t bsz,
                  int64_t dim, bool bidir) {
  expect(p.dim() >= 2, "coefficients must be (rows, ndim)");
  check_rows(p.size(0), dim, bidir);
  const int64_t m = cplx ? 2 : 1, n = p.size(1);
  expect_numel(p, p.size(0) * n, "p");
  expect_numel(q, p.numel() * m, "q");
  expect_numel(g, p.numel() * m, "gamma");
  expect_numel(omega, dim, "omega");
  expect_numel(h, bsz * dim * n * m, "the state");
}

Coeffs coeffs(const Tensor& alpha, const Tensor& delta, const Tensor& third, const Tensor& gamma, bool cplx, const Where& w) {
  const int64_t k = alpha.size(0), n = alpha.size(1);
  expect_numel(alpha, k * n, "alpha");
  expect_numel(delta, k * n, "delta");
  expect_numel(third, cplx ? k : k * n, cplx ? "theta" : "beta");
  expect_numel(gamma, cplx ? 2 * k * n : k * n, "gamma");
  const auto st = alpha.scalar_type();
  auto prep = [&](const Tensor& t) { return (t.scalar_type() == st ? t.detach() : t.detach().to(st)).contiguous(); };
  const Tensor a = prep(alpha), d = prep(delta), t = prep(third), g = prep(gamma);
  Tensor f = floats({(cplx ? 5 : 3) * k * n}, alpha);
  Coeffs c;
  c.p = f.narrow(0, 0, k * n).view({k, n});
  if (cplx) {
    c.q = f.narrow(0, k * n, 2 * k * n).view({k, n, 2});
    c.g = f.narrow(0, 3 * k * n, 2 * k * n).view({k, n, 2});
    check(mega_cema_coeffs(a.data_ptr(), d.data_ptr(), t.data_ptr(), g.data_ptr(), dtype_of(a), (int)k, (int)n, fptr(c.p),
                           fptr(c.q), fptr(c.g), w.stream), "cema_coeffs");
  } else {
    c.q = f.narrow(0, k * n, k * n).view({k, n});
    c.g = f.narrow(0, 2 * k * n, k * n).view({k, n});
    check(mega_ema_coeffs(a.data_ptr(), d.data_ptr(), t.data_ptr(), g.data_ptr(), dtype_of(a), (int)k, (int)n, fptr(c.p),
                          fptr(c.q), fptr(c.g), w.stream), "ema_coeffs");
  }
  return c;
}

// x (B, D, L); p (K, N), q / g (K, N) or interleaved (K, N, 2); states likewise
void run_ema(const Tensor& x, const Tensor& y, const Tensor& p, const Tensor& q, const Tensor& g, const Tensor& omega,
             const Tensor& mask, const Tensor& h_in, const Tensor& h_out, unsigned flags, int trunc, bool cplx, const Where& w) {
  const int B = (int)x.size(0), D = (int)x.size(1), L = (int)x.size(2), N = (int)p.size(1);
  auto fn = cplx ? mega_cema_fwd : mega_ema_fwd;
  check(fn(x.data_ptr(), y.data_ptr(), dtype_of(x), B, D, L, STRIDES3(x), STRIDES3(y), fptr(p), fptr(q), fptr(g), fptr(omega),
           N, ptr<uint8_t>(mask), fptr(h_in), fptr(h_out), flags, trunc, w.stream), cplx ? "cema_fwd" : "ema_fwd");
}

std::tuple<Tensor, OptTensor> ema_forward(const Tensor& x, const Tensor& p_, const Tensor& q_, const Tensor& g_,
                                          const Tensor& omega_, const OptTensor& mask_, const OptTensor& h_in_, bool want_state,
                                          int64_t flags, int64_t trunc, bool cplx, const OptTensor& out_) {
  on_cuda(x, p_, q_, g_, omega_, given(mask_), given(h_in_));
  const Where w(x);
  const int64_t bsz = x.size(0), dim = x.size(1);
  const Tensor p = f32c(p_), q = cplx ? c64(q_, 2) : f32c(q_), g = cplx ? c64(g_, 2) : f32c(g_), omega = f32c(omega_);
  const int64_t n = p.size(1);
  const Tensor mask = mask_u8(given(mask_), bsz, x.size(2));
  const Tensor h_in = cplx ? c64(given(h_in_), 3) : f32c(given(h_in_));
  check_coeffs(p, q, g, omega, h_in, cplx, bsz, dim, flags & MEGA_EMA_BIDIRECTIONAL);
  const Tensor y = out_.has_value() ? *out_ : like(x);
  expect(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type(), "out must be like x");
  Tensor h_out = want_state ? (cplx ? floats({bsz, dim, n, 2}, x) : floats({bsz, dim, n}, x)) : Tensor();
  run_ema(x, y, p, q, g, omega, mask, h_in, h_out, (unsigned)flags, (int)trunc, cplx, w);
  if (!want_state) return {y, std::nullopt};
  return {y, cplx ? at::view_as_complex(h_out) : h_out};
}

// y = silu(a) / its gradient over a dense tensor's memory
bool rows_of(const Tensor& t, int64_t cols, int64_t& rows) {
  const int64_t vec = 16 / t.element_size();
  if (!t.is_non_overlapping_and_dense() || t.numel() % cols != 0 || cols % vec != 0) return false;
  rows = t.numel() / cols;
  return true;
}

class EmaFn : public torch::autograd::Function<EmaFn> {
 public:
  // chan: x and y are (B, L, D) instead of (B, D, L)
  static Tensor forward(AutogradContext* ctx, Tensor x_, Tensor alpha, Tensor delta, Tensor third, Tensor gamma, Tensor omega,
                        OptTensor mask_, int64_t flags, int64_t trunc, bool cplx, bool silu, bool chan) {
    const Tensor x = chan ? x_.transpose(1, 2) : x_;
    on_cuda(x, alpha, delta, third, gamma, omega, given(mask_));
    expect(x.dim() == 3 && alpha.dim() >= 2, "x must have three dimensions, alpha (rows, ndim, 1)");
    check_rows(alpha.size(0), x.size(1), flags & MEGA_EMA_BIDIRECTIONAL);
    expect_numel(omega, x.size(1), "omega");
    const Where w(x);
    const Tensor mask = mask_u8(given(mask_), x.size(0), x.size(2));
    const Coeffs c = coeffs(alpha, delta, third, gamma, cplx, w);
    // (the result is a tensor of its own, not a view of one: a view made in here could not be changed in place)
    Tensor y_ = like(x_), y = chan ? y_.transpose(1, 2) : y_, out = y_;
    const auto f = f32_all({omega, alpha, delta, third}, w.stream);
    run_ema(x, y, c.p, c.q, c.g, f[0], mask, none(), none(), (unsigned)flags, (int)trunc, cplx, w);
    if (silu) {
      int64_t rows;
      if (rows_of(y_, x.size(1), rows)) {
        out = like(y_);
        check(mega_gate_silu(y_.data_ptr(), x.size(1), nullptr, 0, out.data_ptr(), x.size(1), dtype_of(y), rows, (int)x.size(1),
                             w.stream), "gate_silu");
      } else {
        out = at::silu(y_);
      }
    }
    ctx->save_for_backward({x_, f[1], f[2], f[3], f[0], mask, c.p, c.q, c.g, silu ? y : Tensor()});
    ctx->saved_data["flags"] = flags;
    ctx->saved_data["trunc"] = trunc;
    ctx->saved_data["cplx"] = cplx;
    ctx->saved_data["chan"] = chan;
    ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)alpha.scalar_type(), (int64_t)delta.scalar_type(),
                                                    (int64_t)third.scalar_type(), (int64_t)gamma.scalar_type(),
                                                    (int64_t)omega.scalar_type()};
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const bool chan = ctx->saved_data["chan"].toBool();
    const Tensor x = chan ? s[0].transpose(1, 2) : s[0];
    const Tensor &alpha = s[1], &delta = s[2], &third = s[3], &omega = s[4], &mask = s[5], &p = s[6], &q = s[7], &g = s[8], &y = s[9];
    const unsigned flags = (unsigned)ctx->saved_data["flags"].toInt();
    const int trunc = (int)ctx->saved_data["trunc"].toInt();
    const bool cplx = ctx->saved_data["cplx"].toBool();
    const auto types = ctx->saved_data["types"].toIntVector();
    const Where w(x);
    Tensor dy = chan ? grads[0].transpose(1, 2) : grads[0];
    if (dy.scalar_type() != x.scalar_type()) dy = dy.to(x.scalar_type());
    if (y.defined()) {   // through the SiLU, in y's memory order
      if (dy.strides() != y.strides()) {
        Tensor t = like(y);
        t.copy_(dy);
        dy = t;
      }
      int64_t rows;
      if (rows_of(y, x.size(1), rows)) {
        Tensor d = like(y);
        const int64_t c = x.size(1);
        check(mega_gate_silu_bwd(dy.data_ptr(), c, y.data_ptr(), c, d.data_ptr(), c, nullptr, dtype_of(y), rows, (int)c, w.stream),
              "gate_silu_bwd");
        dy = d;
      } else {
        dy = at::silu_backward(dy, y);
      }
    }
    const int B = (int)x.size(0), D = (int)x.size(1), L = (int)x.size(2);
    const int64_t k = p.size(0), n = p.size(1), kn = k * n, m = cplx ? 2 : 1;
    Tensor dx = like(x);
    // dp, dq, dgamma_hat and domega in one piece (the library zeroes them together), the raw parameters' behind them
    const int64_t sums = kn * (1 + 2 * m), raw = cplx ? 4 * kn + k : 4 * kn;
    Tensor f = floats({sums + D + raw}, x);
    float* at_ = f.data_ptr<float>();
    float *dp = at_, *dq = at_ + kn, *dg = at_ + kn * (1 + m), *dom = at_ + sums, *da = dom + D, *dd = da + kn;
    if (cplx) {
      float *dgm = dd + kn, *dt = dgm + 2 * kn;
      check(mega_cema_bwd(dy.data_ptr(), x.data_ptr(), dx.data_ptr(), dtype_of(x), B, D, L, STRIDES3(dy), STRIDES3(x), STRIDES3(dx),
                          fptr(p), fptr(q), fptr(g), fptr(omega), (int)n, ptr<uint8_t>(mask), flags, trunc, dp, dq, dg, dom, w.stream),
            "cema_bwd");
      check(mega_cema_coeffs_bwd(fptr(alpha), fptr(delta), fptr(third), fptr(q), dp, dq, dg, (int)k, (int)n, da, dd, dt, dgm, w.stream),
            "cema_coeffs_bwd");
    } else {
      float *db = dd + kn, *dgm = db + kn;
      check(mega_ema_bwd(dy.data_ptr(), x.data_ptr(), dx.data_ptr(), dtype_of(x), B, D, L, STRIDES3(dy), STRIDES3(x), STRIDES3(dx),
                         fptr(p), fptr(q), fptr(g), fptr(omega), (int)n, ptr<uint8_t>(mask), nullptr, nullptr, flags, trunc, dp, dq, dg,
                         dom, nullptr, w.stream), "ema_bwd");
      check(mega_ema_coeffs_bwd(fptr(alpha), fptr(delta), fptr(third), dp, dq, dg, (int)k, (int)n, da, dd, db, dgm, w.stream), "ema_coeffs_bwd");
    }
    // (one conversion where the parameters share a type; none passes through another's)
    Tensor out = f.narrow(0, sums, D + raw);
    if (std::all_of(types.begin(), types.end(), [&](int64_t t) { return t == types[0]; })) out = out.to((at::ScalarType)types[0]);
    const int64_t base = out.storage_offset();
    auto part = [&](int64_t from, at::IntArrayRef size, at::IntArrayRef stride, int64_t type) {
      Tensor v = out.as_strided(size, stride, base + from);
      return v.scalar_type() == (at::ScalarType)type ? v : v.to((at::ScalarType)type);
    };
    auto like_param = [&](int64_t from, const Tensor& t, int64_t type) { return part(from, t.sizes(), t.strides(), type); };
    const Tensor g_om = like_param(0, omega, types[4]), g_a = like_param(D, alpha, types[0]), g_d = like_param(D + kn, delta, types[1]);
    const Tensor g_3 = like_param(D + (cplx ? 4 : 2) * kn, third, types[2]);
    const Tensor g_g = cplx ? part(D + 2 * kn, {k, n, 2}, {2 * n, 2, 1}, types[3]) : part(D + 3 * kn, {k, n}, {n, 1}, types[3]);
    return {chan ? dx.transpose(1, 2) : dx, g_a, g_d, g_3, g_g, g_om, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor ema_train(const Tensor& x, const Tensor& alpha, const Tensor& delta, const Tensor& third, const Tensor& gamma,
                 const Tensor& omega, const OptTensor& mask, int64_t flags, int64_t trunc, bool cplx, bool silu,
                 bool chan) {
  return EmaFn::apply(x, alpha, delta, third, gamma, omega, mask, flags, trunc, cplx, silu, chan);
}

// ------------------------------------------------------------------------------------------------ norms
struct NormParams {
  Tensor gamma, beta, count, mean, var;
};

// The type that parameters share when the library reads it, else fp32: none of them passes through a narrower one.
at::ScalarType common_type(std::initializer_list<Tensor> ts) {
  at::ScalarType type = at::kFloat;
  bool first = true;
  for (const auto& t : ts) {
    if (!t.defined()) continue;
    const auto own = t.scalar_type();
    if ((own != at::kFloat && own != at::kBFloat16 && own != at::kHalf) || (!first && own != type)) return at::kFloat;
    type = own;
    first = false;
  }
  return type;
}
Tensor as_type(const Tensor& t, at::ScalarType type) {
  if (!t.defined()) return t;
  return (t.scalar_type() == type ? t.detach() : t.detach().to(type)).contiguous();
}

NormParams prepare(const Tensor& weight, const Tensor& bias, const Tensor& pc, const Tensor& pm, const Tensor& pl, int64_t bsz,
                   const Where& w) {
  const int64_t d = weight.size(0), g = pm.defined() ? pm.size(0) : 0;
  expect_numel(weight, d, "weight");
  expect_numel(bias, d, "bias");
  expect_numel(pm, g, "prior_mean");
  if (pm.defined()) expect_numel(pl, g, "prior_logv");
  expect(g <= d, "more prior means than features");
  const auto type = common_type({weight, bias, pm, pl});
  const Tensor wt = as_type(weight, type), b = as_type(bias, type), m = as_type(pm, type), l = as_type(pl, type);
  const Tensor c = pc.defined() ? pc.detach().to(at::kLong).contiguous() : pc;
  Tensor f = floats({2 * d + 2 * bsz * g}, weight);
  NormParams r;
  r.gamma = f.narrow(0, 0, d);
  r.beta = f.narrow(0, d, d);
  if (g) {
    r.mean = f.narrow(0, 2 * d, bsz * g).view({bsz, g});
    r.var = f.narrow(0, 2 * d + bsz * g, bsz * g).view({bsz, g});
    r.count = counts(bsz, weight);
  }
  check(mega_norm_prepare(ptr<int64_t>(c), ptr(m), ptr(l), wt.data_ptr(), b.data_ptr(), dtype_of(wt),
                          (int)(g ? bsz : 0), (int)g, (int)d, ptr<int64_t>(r.count), fptr(r.mean), fptr(r.var), fptr(r.gamma),
                          fptr(r.beta), w.stream), "norm_prepare");
  return r;
}

py::tuple norm_prepare(const Tensor& weight, const Tensor& bias, const OptTensor& pc, const OptTensor& pm, const OptTensor& pl,
                       int64_t bsz) {
  on_cuda(weight, bias, given(pc), given(pm), given(pl));
  const Where w(weight);
  const NormParams r = prepare(weight, bias, given(pc), given(pm), given(pl), bsz, w);
  if (!pm.has_value()) return py::make_tuple(r.gamma, r.beta);
  return py::make_tuple(r.gamma, r.beta, r.count, r.mean, r.var);
}

// (dweight, dbias, dprior_mean, dprior_logv), each in its parameter's type
std::vector<Tensor> finish(const Tensor& weight, const Tensor& bias, const Tensor& pm, const Tensor& logv, const float* dgamma,
                           const float* dbeta, const float* dpm, const float* dpv, int64_t bsz, int64_t g, const Where& w) {
  const int64_t d = weight.size(0);
  const auto type = common_type({weight, bias, pm, logv});
  Tensor out = at::empty({2 * d + 2 * g}, weight.options().requires_grad(false).dtype(type));
  const Tensor l = as_type(logv, type);
  char* at_ = static_cast<char*>(out.data_ptr());
  const int64_t es = out.element_size();
  check(mega_norm_finish(dpm, dpv, ptr(l), dgamma, dbeta, dtype_of(out), (int)(g ? bsz : 0), (int)g, (int)d,
                         g ? at_ + 2 * d * es : nullptr, g ? at_ + (2 * d + g) * es : nullptr, at_, at_ + d * es, w.stream),
        "norm_finish");
  auto own = [&](int64_t from, const Tensor& p) { return out.narrow(0, from, p.numel()).view(p.sizes()).to(p.scalar_type()); };
  std::vector<Tensor> r = {own(0, weight), own(d, bias)};
  if (g) {
    r.push_back(own(2 * d, pm));
    r.push_back(own(2 * d + g, logv));
  }
  return r;
}

constexpr int64_t kGridSequences = 65535;   // sequences that the kernels over time take in a launch

bool whole_rows(const Tensor& x) {   // contiguous channels in whole 16-byte pieces
  const int64_t es = x.element_size();
  return x.stride(2) == 1 && x.size(2) * es % 16 == 0 && x.stride(0) * es % 16 == 0 && x.stride(1) * es % 16 == 0 &&
         reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> timestep_norm_fwd(const Tensor& x, const Tensor& pc_, const Tensor& pm_, const Tensor& pv_,
                                                             const Tensor& gamma_, const Tensor& beta_, const OptTensor& mask_,
                                                             double eps, int64_t groups, const OptTensor& out_) {
  on_cuda(x, pc_, pm_, pv_, gamma_, beta_, given(mask_));
  const Where w(x);
  const int64_t bsz = x.size(0), length = x.size(1), dim = x.size(2), g = groups > 0 ? groups : dim;
  const Tensor pc = pc_.to(at::kLong).contiguous(), pm = f32c(pm_), pv = f32c(pv_), gamma = f32c(gamma_), beta = f32c(beta_);
  if (pm.dim() != 2 || pm.size(0) != bsz || pm.size(1) != g || pv.sizes() != pm.sizes())
    throw py::value_error("prev_mean/prev_var must be (batch, groups) = (" + std::to_string(bsz) + ", " + std::to_string(g) + ")");
  const Tensor mask = mask_u8(given(mask_), bsz, length);
  expect_numel(pc, bsz, "prev_count");
  expect_numel(gamma, dim, "gamma");
  expect_numel(beta, dim, "beta");
  const Tensor y = out_.has_value() ? *out_ : like(x);
  expect(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type(), "out must be like x");
  Tensor count = counts(bsz, x), st = floats({2, bsz, g}, x);
  Tensor mean = st.select(0, 0), var = st.select(0, 1);
  check(mega_timestep_norm_fwd(x.data_ptr(), y.data_ptr(), dtype_of(x), (int)bsz, (int)length, (int)dim, STRIDES3(x), STRIDES3(y),
                               ptr<int64_t>(pc), fptr(pm), fptr(pv), fptr(gamma), fptr(beta), ptr<uint8_t>(mask), (int)g, eps,
                               ptr<int64_t>(count), fptr(mean), fptr(var), w.stream), "timestep_norm_fwd");
  return {y, count, mean, var};
}

class TsnFn : public torch::autograd::Function<TsnFn> {
 public:
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor pcount, Tensor pmean, Tensor plogv, Tensor weight, Tensor bias,
                        OptTensor mask_, int64_t groups, double eps) {
    on_cuda(x, pcount, pmean, plogv, weight, bias, given(mask_));
    const Where w(x);
    const int64_t bsz = x.size(0), length = x.size(1), dim = x.size(2), g = groups > 0 ? groups : dim;
    expect_numel(weight, dim, "weight");
    expect_numel(pmean, g, "prior_mean");
    const NormParams r = prepare(weight, bias, pcount, pmean, plogv, bsz, w);
    const Tensor mask = mask_u8(given(mask_), bsz, length);
    const bool again = groups <= 0 && whole_rows(x) && bsz <= kGridSequences;
    Tensor y = like(x), count = counts(bsz, x);
    if (again) {   // the backward takes the statistics again: nothing is kept but the arguments
      Tensor st = floats({2, bsz, g}, x);
      check(mega_timestep_norm_fwd(x.data_ptr(), y.data_ptr(), dtype_of(x), (int)bsz, (int)length, (int)dim, STRIDES3(x), STRIDES3(y),
                                   ptr<int64_t>(r.count), fptr(r.mean), fptr(r.var), fptr(r.gamma), fptr(r.beta),
                                   ptr<uint8_t>(mask), (int)g, eps, ptr<int64_t>(count), fptr(st), fptr(st) + bsz * g, w.stream),
            "timestep_norm_fwd");
      ctx->save_for_backward({x, weight, plogv, r.gamma, mask, r.count, r.mean, r.var, bias, pmean});
    } else {
      Tensor st = floats({2, bsz, g}, x), cm = floats({bsz, length, g}, x), cr = floats({bsz, length, g}, x);
      Tensor gm = g != dim ? floats({bsz, length, g}, x) : Tensor();
      check(mega_timestep_norm_fwd_train(x.data_ptr(), y.data_ptr(), dtype_of(x), (int)bsz, (int)length, (int)dim, STRIDES3(x),
                                         STRIDES3(y), ptr<int64_t>(r.count), fptr(r.mean), fptr(r.var), fptr(r.gamma),
                                         fptr(r.beta), ptr<uint8_t>(mask), (int)g, eps, ptr<int64_t>(count), fptr(st),
                                         fptr(st) + bsz * g, fptr(cm), fptr(cr), fptr(gm), w.stream), "timestep_norm_fwd_train");
      ctx->save_for_backward({x, weight, plogv, r.gamma, mask, count, r.mean, Tensor(), bias, pmean, cm, cr, gm});
    }
    ctx->saved_data["again"] = again;
    ctx->saved_data["g"] = g;
    ctx->saved_data["eps"] = eps;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &weight = s[1], &plogv = s[2], &gamma = s[3], &mask = s[4];
    const int64_t g = ctx->saved_data["g"].toInt();
    const Where w(x);
    const int64_t bsz = x.size(0), dim = x.size(2);
    Tensor dy = grads[0];
    if (dy.scalar_type() != x.scalar_type()) dy = dy.to(x.scalar_type());
    const bool again = ctx->saved_data["again"].toBool();
    if (again && !whole_rows(dy)) dy = dy.contiguous();
    Tensor dx = like(x);
    Tensor f = floats({2 * dim + 2 * bsz * g}, x);
    float *dgamma = fptr(f), *dbeta = dgamma + dim, *dpm = dbeta + dim, *dpv = dpm + bsz * g;
    bool done = false;
    if (again) {
      const int rc = mega_timestep_norm_bwd_stats(dy.data_ptr(), x.data_ptr(), dx.data_ptr(), dtype_of(x), (int)bsz, (int)x.size(1), (int)dim,
                                                  STRIDES3(dy), STRIDES3(x), STRIDES3(dx), nullptr, nullptr, ptr<int64_t>(s[5]),
                                                  fptr(s[6]), fptr(s[7]), fptr(gamma), ptr<uint8_t>(mask),
                                                  ctx->saved_data["eps"].toDouble(), dpm, dpv, dgamma, dbeta, w.stream);
      done = rc != MEGA_ERR_UNSUPPORTED;   // (the device had no scratch memory for it: with saves, as the other forms do)
      if (done) check(rc, "timestep_norm_bwd_stats");
    }
    if (!done) {
      Tensor count = s[5], cm, cr, gm;
      if (again) {
        const int64_t length = x.size(1);
        Tensor y = like(x), st = floats({2, bsz, g}, x);
        count = counts(bsz, x);
        cm = floats({bsz, length, g}, x);
        cr = floats({bsz, length, g}, x);
        check(mega_timestep_norm_fwd_train(x.data_ptr(), y.data_ptr(), dtype_of(x), (int)bsz, (int)length, (int)dim, STRIDES3(x),
                                           STRIDES3(y), ptr<int64_t>(s[5]), fptr(s[6]), fptr(s[7]), fptr(gamma), fptr(gamma),
                                           ptr<uint8_t>(mask), (int)g, ctx->saved_data["eps"].toDouble(), ptr<int64_t>(count),
                                           fptr(st), fptr(st) + bsz * g, fptr(cm), fptr(cr), nullptr, w.stream),
              "timestep_norm_fwd_train");
      } else {
        cm = s[10];
        cr = s[11];
        gm = s[12];
      }
      check(mega_timestep_norm_bwd(dy.data_ptr(), x.data_ptr(), dx.data_ptr(), dtype_of(x), (int)bsz, (int)x.size(1), (int)dim,
                                   STRIDES3(dy), STRIDES3(x), STRIDES3(dx), nullptr, nullptr, fptr(s[6]), ptr<int64_t>(count),
                                   fptr(cm), fptr(cr), fptr(gm), fptr(gamma), ptr<uint8_t>(mask), (int)g, dpm, dpv, dgamma, dbeta,
                                   w.stream), "timestep_norm_bwd");
    }
    auto r = finish(weight, s[8], s[9], plogv, dgamma, dbeta, dpm, dpv, bsz, g, w);
    return {dx, Tensor(), r[2], r[3], r[0], r[1], Tensor(), Tensor(), Tensor()};
  }
};

Tensor timestep_norm_train(const Tensor& x, const Tensor& pc, const Tensor& pm, const Tensor& pl, const Tensor& weight,
                           const Tensor& bias, const OptTensor& mask, int64_t groups, double eps) {
  return TsnFn::apply(x, pc, pm, pl, weight, bias, mask, groups, eps);
}

// x (B, D, L), or (B, L, D) with length_last = false
struct Sqn {
  int64_t bsz, dim, length, sb, sd, sl;
};
Sqn sqn_view(const Tensor& x, bool length_last) {
  if (length_last) return {x.size(0), x.size(1), x.size(2), x.stride(0), x.stride(1), x.stride(2)};
  return {x.size(0), x.size(2), x.size(1), x.stride(0), x.stride(2), x.stride(1)};
}

void run_sqn(const Tensor& x, const Tensor& y, const Tensor& gamma, const Tensor& beta, const Tensor& mask, double eps,
             bool length_last, int64_t g, const Tensor& count, const Tensor& mean, const Tensor& rstd, const Where& w) {
  const Sqn a = sqn_view(x, length_last), o = sqn_view(y, length_last);
  check(mega_sequence_norm_fwd(x.data_ptr(), y.data_ptr(), dtype_of(x), (int)a.bsz, (int)a.dim, (int)a.length, a.sb, a.sd, a.sl, o.sb,
                               o.sd, o.sl, fptr(gamma), fptr(beta), ptr<uint8_t>(mask), (int)g, eps, ptr<int64_t>(count),
                               fptr(mean), fptr(rstd), w.stream), "sequence_norm_fwd");
}

std::tuple<Tensor, Tensor, Tensor, Tensor> sequence_norm_fwd(const Tensor& x, const Tensor& gamma_, const Tensor& beta_,
                                                             const OptTensor& mask_, double eps, bool length_last, int64_t groups,
                                                             const OptTensor& out_) {
  on_cuda(x, gamma_, beta_, given(mask_));
  const Where w(x);
  const Sqn a = sqn_view(x, length_last);
  const int64_t g = groups > 0 ? groups : a.dim;
  const Tensor mask = mask_u8(given(mask_), a.bsz, a.length);
  expect_numel(gamma_, a.dim, "gamma");
  expect_numel(beta_, a.dim, "beta");
  const Tensor y = out_.has_value() ? *out_ : like(x);
  expect(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type(), "out must be like x");
  Tensor count = counts(a.bsz, x), st = floats({2, a.bsz, g}, x);
  Tensor mean = st.select(0, 0), rstd = st.select(0, 1);
  run_sqn(x, y, f32c(gamma_), f32c(beta_), mask, eps, length_last, g, count, mean, rstd, w);
  return {y, count, mean, rstd};
}

class SqnFn : public torch::autograd::Function<SqnFn> {
 public:
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor weight, Tensor bias, OptTensor mask_, double eps, bool length_last,
                        int64_t groups) {
    on_cuda(x, weight, bias, given(mask_));
    const Where w(x);
    const Sqn a = sqn_view(x, length_last);
    const int64_t g = groups > 0 ? groups : a.dim;
    expect_numel(weight, a.dim, "weight");
    const NormParams r = prepare(weight, bias, none(), none(), none(), 0, w);
    const Tensor mask = mask_u8(given(mask_), a.bsz, a.length);
    Tensor y = like(x), count = counts(a.bsz, x), st = floats({2, a.bsz, g}, x);
    Tensor mean = st.select(0, 0), rstd = st.select(0, 1);
    run_sqn(x, y, r.gamma, r.beta, mask, eps, length_last, g, count, mean, rstd, w);
    ctx->save_for_backward({x, weight, r.gamma, mask, count, mean, rstd, bias});
    ctx->saved_data["ll"] = length_last;
    ctx->saved_data["g"] = g;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &weight = s[1];
    const bool ll = ctx->saved_data["ll"].toBool();
    const Where w(x);
    Tensor dy = grads[0];
    if (dy.scalar_type() != x.scalar_type()) dy = dy.to(x.scalar_type());
    Tensor dx = like(x);
    const Sqn a = sqn_view(x, ll), q = sqn_view(dy, ll), o = sqn_view(dx, ll);
    Tensor f = floats({2 * a.dim}, x);
    check(mega_sequence_norm_bwd(dy.data_ptr(), x.data_ptr(), dx.data_ptr(), dtype_of(x), (int)a.bsz, (int)a.dim, (int)a.length, q.sb,
                                 q.sd, q.sl, a.sb, a.sd, a.sl, o.sb, o.sd, o.sl, ptr<int64_t>(s[4]), fptr(s[5]), fptr(s[6]),
                                 fptr(s[2]), ptr<uint8_t>(s[3]), (int)ctx->saved_data["g"].toInt(), fptr(f), fptr(f) + a.dim,
                                 w.stream), "sequence_norm_bwd");
    auto r = finish(weight, s[7], none(), none(), fptr(f), fptr(f) + a.dim, nullptr, nullptr, 0, 0, w);
    return {dx, r[0], r[1], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor sequence_norm_train(const Tensor& x, const Tensor& weight, const Tensor& bias, const OptTensor& mask, double eps,
                           bool length_last, int64_t groups) {
  return SqnFn::apply(x, weight, bias, mask, eps, length_last, groups);
}

// ---------------------------------------------------------------------------------------- fused norm -> EMA
// (y, count, mean, var, h or None, xn or None)
py::tuple tsn_ema_forward(const Tensor& x, const Tensor& pc_, const Tensor& pm_, const Tensor& pv_, const Tensor& gamma_,
                          const Tensor& beta_, double eps, const Tensor& p_, const Tensor& q_, const Tensor& g_,
                          const Tensor& omega_, const OptTensor& mask_, const OptTensor& h_in_, bool want_state, bool silu,
                          bool want_normed, bool cplx) {
  on_cuda(x, pc_, pm_, pv_, gamma_, beta_, p_, q_, g_, omega_, given(mask_), given(h_in_));
  const Where w(x);
  const int64_t bsz = x.size(0), length = x.size(1), dim = x.size(2);
  const Tensor pc = pc_.to(at::kLong).contiguous(), pm = f32c(pm_), pv = f32c(pv_), gamma = f32c(gamma_), beta = f32c(beta_);
  const Tensor p = f32c(p_), q = cplx ? c64(q_, 2) : f32c(q_), g = cplx ? c64(g_, 2) : f32c(g_), omega = f32c(omega_);
  const Tensor h_in = cplx ? c64(given(h_in_), 3) : f32c(given(h_in_));
  const int64_t n = p.size(1);
  check_coeffs(p, q, g, omega, h_in, cplx, bsz, dim, false);
  expect_numel(pc, bsz, "prev_count");
  expect_numel(pm, bsz * dim, "prev_mean");
  expect_numel(pv, bsz * dim, "prev_var");
  expect_numel(gamma, dim, "gamma");
  expect_numel(beta, dim, "beta");
  const Tensor mask = mask_u8(given(mask_), bsz, length);
  Tensor y = like(x), xn = want_normed ? like(y) : Tensor();
  Tensor count = counts(bsz, x), st = floats({2, bsz, dim}, x);
  Tensor mean = st.select(0, 0), var = st.select(0, 1);
  Tensor h_out = want_state ? (cplx ? floats({bsz, dim, n, 2}, x) : floats({bsz, dim, n}, x)) : Tensor();
  auto fn = cplx ? mega_tsn_cema_fwd : mega_tsn_ema_fwd;
  check(fn(x.data_ptr(), y.data_ptr(), ptr(xn), dtype_of(x), (int)bsz, (int)length, (int)dim, STRIDES3(x), STRIDES3(y),
           ptr<int64_t>(pc), fptr(pm), fptr(pv), fptr(gamma), fptr(beta), eps, ptr<int64_t>(count), fptr(mean), fptr(var), fptr(p),
           fptr(q), fptr(g), fptr(omega), (int)n, ptr<uint8_t>(mask), fptr(h_in), fptr(h_out), silu ? MEGA_EMA_SILU : 0u,
           w.stream), cplx ? "tsn_cema_fwd" : "tsn_ema_fwd");
  py::object h = py::none(), nx = py::none();
  if (want_state) h = py::cast(cplx ? at::view_as_complex(h_out) : h_out);
  if (want_normed) nx = py::cast(xn);
  return py::make_tuple(y, count, mean, var, h, nx);
}

// y, or None outside the fused kernel's envelope
OptTensor sqn_ema_forward(const Tensor& x, const Tensor& gamma, const Tensor& beta, double eps, const Tensor& p_, const Tensor& q_,
                          const Tensor& g_, const Tensor& omega_, const OptTensor& mask_, int64_t flags) {
  on_cuda(x, gamma, beta, p_, q_, g_, omega_, given(mask_));
  if (x.stride(2) != 1) return std::nullopt;
  const Where w(x);
  const Tensor p = f32c(p_), q = f32c(q_), g = f32c(g_), omega = f32c(omega_), ga = f32c(gamma), be = f32c(beta);
  check_coeffs(p, q, g, omega, none(), false, x.size(0), x.size(1), flags & MEGA_EMA_BIDIRECTIONAL);
  expect_numel(ga, x.size(1), "gamma");
  expect_numel(be, x.size(1), "beta");
  const Tensor mask = mask_u8(given(mask_), x.size(0), x.size(2));
  Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
  const int rc = mega_sqn_ema_fwd(x.data_ptr(), y.data_ptr(), dtype_of(x), (int)x.size(0), (int)x.size(1), (int)x.size(2), STRIDES3(x),
                                  STRIDES3(y), fptr(ga), fptr(be), eps, nullptr, nullptr, nullptr, fptr(p), fptr(q), fptr(g),
                                  fptr(omega), (int)p.size(1), ptr<uint8_t>(mask), (unsigned)flags, w.stream);
  if (rc == MEGA_ERR_UNSUPPORTED) return std::nullopt;
  check(rc, "sqn_ema_fwd");
  return y;
}

// ------------------------------------------------------------------------------------------------ the block
// Row-major matrix view of a tensor's last dimension with one row pitch; copied when it is none.
struct Rows {
  Tensor t;
  int64_t rows, cols, ld;
};
Rows rows_view(const Tensor& t) {
  const int64_t cols = t.size(-1);
  bool ok = t.dim() >= 2 && (t.stride(-1) == 1 || cols == 1);
  int64_t ld = cols;
  if (ok) {
    ld = t.size(-2) > 1 ? t.stride(-2) : std::max(cols, t.stride(-2));
    int64_t exp = ld;
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
      if (t.size(i) != 1 && t.stride(i) != exp) ok = false;
      exp *= t.size(i);
    }
  }
  if (!ok || ld < cols) return {t.contiguous(), t.numel() / cols, cols, cols};
  return {t, t.numel() / cols, cols, ld};
}
Tensor fresh(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }

Tensor gate_silu(const Tensor& a, const OptTensor& b) {
  on_cuda(a, given(b));
  const Where w(a);
  const Rows ra = rows_view(a);
  Tensor y = fresh(a);
  Rows rb{Tensor(), 0, 0, 0};
  if (b.has_value()) rb = rows_view(*b);
  check(mega_gate_silu(ra.t.data_ptr(), ra.ld, ptr(rb.t), rb.ld, y.data_ptr(), ra.cols, dtype_of(a), ra.rows, (int)ra.cols, w.stream),
        "gate_silu");
  return y;
}

Tensor gate_mul_silu(const Tensor& a, const Tensor& r) {
  on_cuda(a, r);
  const Where w(a);
  const Rows ra = rows_view(a), rr = rows_view(r);
  Tensor y = fresh(a);
  check(mega_gate_mul_silu(ra.t.data_ptr(), ra.ld, rr.t.data_ptr(), rr.ld, y.data_ptr(), ra.cols, dtype_of(a), ra.rows, (int)ra.cols,
                           w.stream), "gate_mul_silu");
  return y;
}

Tensor gate_output(const Tensor& residual, const Tensor& u, const Tensor& hx, const Tensor& h_lin) {
  on_cuda(residual, u, hx, h_lin);
  const Where w(residual);
  const Rows r = rows_view(residual), ru = rows_view(u), rx = rows_view(hx), rh = rows_view(h_lin);
  Tensor y = fresh(residual);
  check(mega_gate_output(r.t.data_ptr(), r.ld, ru.t.data_ptr(), ru.ld, rx.t.data_ptr(), rx.ld, rh.t.data_ptr(), rh.ld, y.data_ptr(),
                         r.cols, dtype_of(residual), r.rows, (int)r.cols, w.stream), "gate_output");
  return y;
}

// rot: fp32 (positions, S / 2, 2), or None
std::tuple<Tensor, Tensor> gate_qk(const Tensor& z, const Tensor& gamma, const Tensor& beta, const OptTensor& rot, int64_t period,
                                   int64_t q_offset, double eps) {
  on_cuda(z, gamma, beta, given(rot));
  const Where w(z);
  const Rows r = rows_view(z);
  const Tensor g = f32c(gamma), b = f32c(beta);
  if (g.dim() != 2 || g.size(0) != 2 || g.size(1) != r.cols || b.sizes() != g.sizes())
    throw py::value_error("gate_qk: gamma and beta must be (2, " + std::to_string(r.cols) + ")");
  Tensor q = fresh(z), k = fresh(z);
  if (!rot.has_value()) {
    check(mega_gate_qk(r.t.data_ptr(), r.ld, fptr(g), fptr(b), q.data_ptr(), r.cols, k.data_ptr(), r.cols, dtype_of(z), r.rows,
                       (int)r.cols, eps, w.stream), "gate_qk");
    return {q, k};
  }
  Tensor t = rot->is_complex() ? at::view_as_real(*rot) : *rot;
  t = f32c(t);
  if (t.dim() != 3 || t.size(1) * 2 != r.cols || t.size(2) != 2)
    throw py::value_error("gate_qk_rotary: rot must be (positions, S / 2) complex or (positions, S / 2, 2) float");
  check(mega_gate_qk_rotary(r.t.data_ptr(), r.ld, fptr(g), fptr(b), fptr(t), (int)t.size(0), (int)period, (int)q_offset, q.data_ptr(),
                            r.cols, k.data_ptr(), r.cols, dtype_of(z), r.rows, (int)r.cols, eps, w.stream), "gate_qk_rotary");
  return {q, k};
}

// ------------------------------------------------------------------------------- gated linear recurrence
// (the package's other operators take what a caller hands them; these check it all, as their operands come from several places)
void same_kind(const Tensor& t, const Tensor& x, const char* what) {
  if (!t.defined()) return;
  if (t.scalar_type() != x.scalar_type()) throw py::type_error(std::string(what) + " must have x's type");
  if (t.device() != x.device()) throw py::value_error(std::string(what) + " must be on x's device");
  if (t.sizes() != x.sizes()) throw py::value_error(std::string(what) + " must have x's shape");
}
Tensor mask_on(const Tensor& mask, const Tensor& x, const char* what) {
  if (!mask.defined()) return mask;
  if (mask.device() != x.device()) throw py::value_error(std::string(what) + " must be on x's device");
  if (mask.dim() != 2 || mask.size(0) != x.size(0) || mask.size(1) != x.size(1))
    throw py::value_error(std::string(what) + " must be (batch, length) = (" + std::to_string(x.size(0)) + ", " + std::to_string(x.size(1)) + ")");
  return mask.scalar_type() == at::kBool ? mask.contiguous() : mask.ne(0).contiguous();
}
void check_state(const Tensor& h, const Tensor& x, int64_t dim, const char* what) {
  if (!h.defined()) return;
  if (h.device() != x.device()) throw py::value_error(std::string(what) + " must be on x's device");
  if (!at::isFloatingType(h.scalar_type())) throw py::type_error(std::string(what) + " must be a floating-point tensor");
  if (h.dim() != 2 || h.size(0) != x.size(0) || h.size(1) != dim)
    throw py::value_error(std::string(what) + " must be (batch, channels) = (" + std::to_string(x.size(0)) + ", " + std::to_string(dim) + ")");
}
int extent(int64_t n) {
  expect(n <= INT_MAX, "an extent does not fit 32 bits");
  return (int)n;
}
// contiguous channels; the strides of the axes before them are free
Tensor channels(const Tensor& t) { return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

struct Rec {
  Tensor x, f, i, pad, reset, h_in;
  int B, L, D;
  unsigned flags;
};
Rec rec_args(const Tensor& x, const Tensor& f, const Tensor& i, const Tensor& pad, const Tensor& reset, const Tensor& h_in, bool reverse) {
  on_cuda(x, f, i, pad, reset, h_in);
  expect(x.dim() == 3, "x must be (batch, length, channels)");
  dtype_of(x);
  same_kind(f, x, "the forget gate");
  same_kind(i, x, "the input gate");
  check_state(h_in, x, x.size(2), "h_in");
  Rec r = {channels(x.detach()), channels(f.detach()), i.defined() ? channels(i.detach()) : i};
  r.pad = mask_on(pad, x, "padding_mask");
  r.reset = mask_on(reset, x, "reset_mask");
  r.h_in = f32c(h_in);
  r.B = extent(x.size(0)), r.L = extent(x.size(1)), r.D = extent(x.size(2));
  r.flags = reverse ? MEGA_REC_REVERSE : 0u;
  return r;
}
#define STRIDES2(t) ((t).defined() ? (t).stride(0) : 0), ((t).defined() ? (t).stride(1) : 0)

void run_rec(const Rec& r, const Tensor& y, const Tensor& h_out, const Tensor& starts, const Where& w) {
  check(mega_gated_recurrence_fwd(r.x.data_ptr(), r.f.data_ptr(), ptr(r.i), y.data_ptr(), dtype_of(r.x), r.B, r.L, r.D, STRIDES2(r.x),
                                  STRIDES2(r.f), STRIDES2(r.i), STRIDES2(y), ptr<uint8_t>(r.pad), ptr<uint8_t>(r.reset), fptr(r.h_in),
                                  fptr(h_out), fptr(starts), r.flags, w.stream), "gated_recurrence_fwd");
}
// the output of (B, L, D) operands: time-major ones give a time-major result
Tensor rec_like(const Tensor& x) {
  return x.size(-1) == 1 || x.stride(-1) == 1 ? like(x) : at::empty(x.sizes(), x.options().requires_grad(false));
}

// (y, state behind the last step or None)
std::tuple<Tensor, OptTensor> gated_recurrence(const Tensor& x, const Tensor& f, const OptTensor& i, const OptTensor& pad,
                                               const OptTensor& reset, const OptTensor& h_in, bool want_state, bool reverse) {
  const Rec r = rec_args(x, f, given(i), given(pad), given(reset), given(h_in), reverse);
  const Where w(x);
  const Tensor y = rec_like(x);
  Tensor h = want_state ? floats({r.B, r.D}, x) : Tensor();
  if (x.numel() == 0) {   // (no step: the state stays)
    if (h.defined()) r.h_in.defined() ? h.copy_(r.h_in) : h.zero_();
  } else {
    run_rec(r, y, h, none(), w);
  }
  if (!want_state) return {y, std::nullopt};
  return {y, h};
}

// Whether a call that reads each value of t (B, D) where it writes that of `out` may do so: t is `out`, value for value, or elsewhere.
bool in_place_or_apart(const Tensor& out, const Tensor& t) {
  if (!t.defined() || t.numel() == 0) return true;
  const char *to = static_cast<const char*>(out.data_ptr()), *from = static_cast<const char*>(t.data_ptr());
  const int64_t span = ((t.size(0) - 1) * t.stride(0) + (t.size(1) - 1) * t.stride(1) + 1) * t.element_size();
  if (to + out.nbytes() <= from || from + span <= to) return true;
  return to == from && t.scalar_type() == out.scalar_type() && t.is_contiguous();
}

// one step: x, f, i (B, D) -> (y, h'); h' is `h_out` where given, which may be h
std::tuple<Tensor, Tensor> gated_recurrence_step(const Tensor& x_, const Tensor& f_, const OptTensor& i_, const OptTensor& h_,
                                                 const OptTensor& h_out_) {
  on_cuda(x_, f_, given(i_), given(h_), given(h_out_));
  expect(x_.dim() == 2, "x must be (batch, channels)");
  const int dt = dtype_of(x_);
  same_kind(f_, x_, "the forget gate");
  same_kind(given(i_), x_, "the input gate");
  check_state(given(h_), x_, x_.size(1), "h");
  const Where w(x_);
  const Tensor x = channels(x_), f = channels(f_), i = channels(given(i_)), h = f32c(given(h_));
  const int B = extent(x.size(0)), D = extent(x.size(1));
  Tensor y = at::empty(x.sizes(), x.options().requires_grad(false)), out = given(h_out_);
  if (out.defined()) {
    check_state(out, x_, D, "h_out");
    expect(out.scalar_type() == at::kFloat && out.is_contiguous(), "h_out must be contiguous float32");
    expect(in_place_or_apart(out, h), "h_out overlaps h and is not h");
    for (const Tensor& t : {x, f, i}) expect(in_place_or_apart(out, t), "h_out overlaps x or a gate and is not it");
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();   // (a graph that has saved it must not use the new values)
  } else {
    out = floats({B, D}, x);
  }
  if (x.numel())
    check(mega_gated_recurrence_step(x.data_ptr(), f.data_ptr(), ptr(i), y.data_ptr(), dt, B, D, x.stride(0), f.stride(0),
                                     i.defined() ? i.stride(0) : 0, D, fptr(h), fptr(out), w.stream), "gated_recurrence_step");
  return {y, out};
}

void first_order() {
  if (at::GradMode::is_enabled()) throw std::runtime_error("mega_b200: second derivatives of this operator are not available");
}
// a gradient of (B, L, D) values in x's type with contiguous channels
Tensor rec_grad(const Tensor& g, const Tensor& x) {
  return channels(g.scalar_type() == x.scalar_type() ? g : g.to(x.scalar_type()));
}

// Separate operands, or one tensor z (B, L, 2 D or 3 D) that holds x, f (and i) side by side, whose gradient then comes as
// one tensor too (the gradients of three slices would be three tensors of z's size, added up).
class RecFn : public torch::autograd::Function<RecFn> {
 public:
  static variable_list forward(AutogradContext* ctx, Tensor x, OptTensor f, OptTensor i, OptTensor pad, OptTensor reset, OptTensor h_in,
                               bool want_state, bool reverse, int64_t packed) {
    const int64_t d = packed ? x.size(2) / packed : 0;   // (x is not checked yet where it is an operand by itself)
    auto part = [&](int64_t k) { return x.detach().narrow(2, k * d, d); };
    const Rec r = packed ? rec_args(part(0), part(1), packed == 3 ? part(2) : Tensor(), given(pad), given(reset), given(h_in), reverse)
                         : rec_args(x, given(f), given(i), given(pad), given(reset), given(h_in), reverse);
    const Where w(x);
    const int64_t seg = mega_gated_recurrence_segment(dtype_of(r.x), r.i.defined());
    Tensor y = rec_like(r.x), h = want_state ? floats({r.B, r.D}, x) : Tensor(), starts = floats({r.B, (r.L + seg - 1) / seg, r.D}, x);
    run_rec(r, y, h, starts, w);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, given(f), given(i), r.pad, r.reset, starts});
    // (of the state that came in its type alone is needed: the caller may go on to write over it)
    ctx->saved_data["state"] = r.h_in.defined() ? (int64_t)h_in->scalar_type() : (int64_t)-1;
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["packed"] = packed;
    if (!want_state) return {y};
    return {y, h};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    const auto s = ctx->get_saved_variables();
    const int64_t packed = ctx->saved_data["packed"].toInt();
    const Tensor &z = s[0], &starts = s[5];
    const int64_t state = ctx->saved_data["state"].toInt();
    const Where w(z);
    const int64_t d = packed ? z.size(2) / packed : z.size(2);
    auto part = [&](const Tensor& t, int64_t k) { return t.narrow(2, k * d, d); };
    const Tensor x = channels(packed ? part(z, 0) : z), f = channels(packed ? part(z, 1) : s[1]);
    const Tensor i = channels(packed == 3 ? part(z, 2) : s[2]);
    const bool dh = grads.size() > 1 && grads[1].defined();
    const Tensor dy = grads[0].defined() ? rec_grad(grads[0], x) : at::zeros(x.sizes(), x.options());
    const Tensor dh_out = dh ? f32c(grads[1]) : Tensor();
    Tensor dz = packed ? at::empty(z.sizes(), z.options().requires_grad(false)) : Tensor();
    Tensor dx = packed ? part(dz, 0) : rec_like(x), df = packed ? part(dz, 1) : rec_like(f), di;
    if (i.defined()) di = packed ? part(dz, 2) : rec_like(i);
    Tensor dh_in = state >= 0 ? floats({x.size(0), d}, x) : Tensor();
    check(mega_gated_recurrence_bwd(dy.data_ptr(), x.data_ptr(), f.data_ptr(), ptr(i), dx.data_ptr(), df.data_ptr(), ptr(di),
                                    dtype_of(x), (int)x.size(0), (int)x.size(1), (int)d, STRIDES2(dy), STRIDES2(x), STRIDES2(f),
                                    STRIDES2(i), STRIDES2(dx), STRIDES2(df), STRIDES2(di), ptr<uint8_t>(s[3]), ptr<uint8_t>(s[4]),
                                    fptr(starts), fptr(dh_out), fptr(dh_in), ctx->saved_data["reverse"].toBool() ? MEGA_REC_REVERSE : 0u,
                                    w.stream), "gated_recurrence_bwd");
    if (dh_in.defined()) dh_in = dh_in.to((at::ScalarType)state);
    return {packed ? dz : dx, packed ? Tensor() : df, packed ? Tensor() : di, Tensor(), Tensor(), dh_in, Tensor(), Tensor(), Tensor()};
  }
};

// (y, h) or (y,); differentiable
variable_list gated_recurrence_train(const Tensor& x, const Tensor& f, const OptTensor& i, const OptTensor& pad, const OptTensor& reset,
                                     const OptTensor& h_in, bool want_state, bool reverse) {
  if (x.numel() == 0) {   // (else RecFn checks them, and converts what it has to once)
    rec_args(x, f, given(i), given(pad), given(reset), given(h_in), reverse);
    variable_list r = {i.has_value() ? x + f + *i : x + f};   // (no values, but gradients of that shape)
    if (want_state) r.push_back(h_in.has_value() ? h_in->to(at::kFloat, false, true) : at::zeros({x.size(0), x.size(2)}, x.options().dtype(at::kFloat)));
    return r;
  }
  return RecFn::apply(x, OptTensor(f), i, pad, reset, h_in, want_state, reverse, (int64_t)0);
}
variable_list gated_recurrence_packed(const Tensor& z, bool gated, const OptTensor& pad, const OptTensor& reset, const OptTensor& h_in,
                                      bool want_state, bool reverse) {
  const int64_t k = gated ? 3 : 2;
  on_cuda(z);
  expect(z.dim() == 3 && z.size(2) % k == 0, "the packed operand must be (batch, length, 2 or 3 times the channels)");
  const int64_t d = z.size(2) / k;
  if (z.numel() == 0)
    return gated_recurrence_train(z.narrow(2, 0, d), z.narrow(2, d, d), gated ? OptTensor(z.narrow(2, 2 * d, d)) : std::nullopt, pad, reset,
                                  h_in, want_state, reverse);
  return RecFn::apply(z, OptTensor(), OptTensor(), pad, reset, h_in, want_state, reverse, k);
}

// ----------------------------------------------------------------------- group norm with an activation
// x (B, ..., D) as (B, L, D) with contiguous channels
Tensor gn_rows(const Tensor& x) {
  expect(x.dim() >= 2, "x must be (batch, ..., channels)");
  if (x.dim() == 3) return channels(x);
  return channels(x.dim() == 2 ? x.unsqueeze(1) : x.reshape({x.size(0), -1, x.size(-1)}));
}
struct Gn {
  Tensor x, gamma, beta, mask;
  int B, L, D, G;
  unsigned flags;
};
Tensor gn_param(const Tensor& p) {
  return p.scalar_type() == at::kFloat && p.is_contiguous() ? p : f32c(p);
}
Gn gn_args(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups, const Tensor& mask, bool silu, bool offset) {
  on_cuda(x, weight, bias, mask);
  dtype_of(x);
  expect(x.dim() >= 2, "x must be (batch, ..., channels)");
  const int64_t d = x.size(-1);
  expect(groups >= 1 && d % groups == 0, "num_groups must divide the channels");
  expect_numel(weight, d, "weight");
  expect_numel(bias, d, "bias");
  if (weight.device() != x.device() || bias.device() != x.device()) throw py::value_error("weight and bias must be on x's device");
  Gn r;
  r.flags = (silu ? MEGA_GN_SILU : 0u) | (offset ? MEGA_GN_OFFSET : 0u);
  if (x.numel() == 0) return r;
  r.x = gn_rows(x);
  Tensor m = mask;
  if (m.defined() && m.dim() != 2 && m.dim() == x.dim() - 1) {
    expect(m.sizes() == x.sizes().slice(0, x.dim() - 1), "padding_mask must have x's shape without its channels");
    m = x.dim() == 2 ? m.unsqueeze(1) : m.reshape({m.size(0), -1});
  }
  r.mask = mask_on(m, r.x, "padding_mask");
  r.gamma = gn_param(weight), r.beta = gn_param(bias);
  r.B = extent(r.x.size(0)), r.L = extent(r.x.size(1)), r.D = extent(d), r.G = (int)groups;
  return r;
}
// A result of x's shape for rows r, and its own rows (a tensor of its own: a view could not be changed in place)
std::pair<Tensor, Tensor> gn_like(const Tensor& x, const Tensor& rows) {
  if (x.dim() == 3) {
    Tensor y = rec_like(rows);
    return {y, y};
  }
  Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
  return {y, y.view(rows.sizes())};
}
// (count (B) int64, mean, rstd (B, G) fp32) in one piece, which is one allocation to a call
struct Stats {
  int64_t* count;
  float *mean, *rstd;
  char* end;
  Stats(const Tensor& t, int64_t b, int64_t g)
      : count(static_cast<int64_t*>(t.data_ptr())), mean(reinterpret_cast<float*>(count + b)), rstd(mean + b * g),
        end(static_cast<char*>(t.data_ptr()) + bytes(b, g)) {}
  static int64_t bytes(int64_t b, int64_t g) { return (8 * b * (1 + g) + 15) / 16 * 16; }
};
Tensor bytes_of(int64_t n, const Tensor& like) { return at::empty({n}, at::TensorOptions().dtype(at::kByte).device(like.device())); }
// y like x; its statistics, with the call's workspace behind them
std::pair<Tensor, Tensor> run_gn(const Tensor& x, const Gn& r, double eps, const Where& w) {
  const int dt = dtype_of(r.x);
  auto [out, y] = gn_like(x, r.x);
  const Tensor stats = bytes_of(Stats::bytes(r.B, r.G) + mega_group_norm_work(dt, r.B, r.L, r.D, r.G, 0), r.x);
  const Stats st(stats, r.B, r.G);
  check(mega_group_norm_fwd(r.x.data_ptr(), y.data_ptr(), dt, r.B, r.L, r.D, STRIDES2(r.x), STRIDES2(y), fptr(r.gamma), fptr(r.beta),
                            ptr<uint8_t>(r.mask), r.G, eps, r.flags, st.count, st.mean, st.rstd, st.end, w.stream), "group_norm_fwd");
  return {out, stats};
}

Tensor group_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups, const OptTensor& mask, double eps, bool silu) {
  const Gn r = gn_args(x, weight, bias, groups, given(mask), silu, true);
  if (x.numel() == 0) return fresh(x);
  const Where w(x);
  return run_gn(x, r, eps, w).first;
}

// (y, count, mean, rstd)
std::tuple<Tensor, Tensor, Tensor, Tensor> group_norm_fwd(const Tensor& x, const Tensor& gamma, const Tensor& beta, int64_t groups,
                                                          const OptTensor& mask, double eps, bool silu, bool offset) {
  const Gn r = gn_args(x, gamma, beta, groups, given(mask), silu, offset);
  const Where w(x);
  const int64_t b = x.size(0);
  if (x.numel() == 0) {
    Tensor rstd = floats({b, groups}, x);
    rstd.fill_(1.0 / std::sqrt(eps));
    return {fresh(x), counts(b, x).zero_(), floats({b, groups}, x).zero_(), rstd};
  }
  auto [y, stats] = run_gn(x, r, eps, w);
  const Tensor f = stats.narrow(0, 8 * b, 8 * b * groups).view(at::kFloat).view({2, b, groups});
  return {y, stats.narrow(0, 0, 8 * b).view(at::kLong), f.select(0, 0), f.select(0, 1)};
}

class GnFn : public torch::autograd::Function<GnFn> {
 public:
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor weight, Tensor bias, int64_t groups, OptTensor mask, double eps, bool silu) {
    const Gn r = gn_args(x, weight, bias, groups, given(mask), silu, true);
    const Where w(x);
    auto [y, stats] = run_gn(x, r, eps, w);
    ctx->save_for_backward({x, weight, bias, r.mask, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["silu"] = silu;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &weight = s[1], &bias = s[2];
    const Gn r = gn_args(x, weight, bias, ctx->saved_data["groups"].toInt(), Tensor(), ctx->saved_data["silu"].toBool(), true);
    const Where w(x);
    const int dt = dtype_of(x);
    Tensor dy = grads[0];
    dy = gn_rows(dy.scalar_type() == x.scalar_type() ? dy : dy.to(x.scalar_type()));
    auto [out, dx] = gn_like(x, r.x);
    Tensor dw = floats({r.D}, x), db = floats({r.D}, x);
    const Tensor work = bytes_of(mega_group_norm_work(dt, r.B, r.L, r.D, r.G, 1), x);
    const Stats st(s[4], r.B, r.G);
    check(mega_group_norm_bwd(dy.data_ptr(), r.x.data_ptr(), dx.data_ptr(), dt, r.B, r.L, r.D, STRIDES2(dy), STRIDES2(r.x), STRIDES2(dx),
                              fptr(r.gamma), fptr(r.beta), ptr<uint8_t>(s[3]), r.G, r.flags, st.count, st.mean, st.rstd, fptr(dw), fptr(db),
                              work.data_ptr(), w.stream), "group_norm_bwd");
    auto own = [&](const Tensor& g, const Tensor& p) {
      const Tensor v = p.dim() == 1 ? g : g.view(p.sizes());
      return p.scalar_type() == at::kFloat ? v : v.to(p.scalar_type());
    };
    return {out, own(dw, weight), own(db, bias), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor group_norm_train(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups, const OptTensor& mask, double eps,
                        bool silu) {
  if (x.numel() == 0) {   // (no values, but gradients of that shape)
    on_cuda(x, weight, bias);
    return (x * (weight + bias)).to(x.scalar_type());
  }
  return GnFn::apply(x, weight, bias, groups, mask, eps, silu);
}

// ------------------------------------------------------------- linear attention with a decay for each head
struct Att {
  Tensor q, k, v, f, pad, reset, h_in;
  mega_decayed_attention_args a;
};
void put(int64_t* to, const Tensor& t, int64_t first) {   // strides of the axes in front of the last one
  for (int64_t i = 0; i < 3; ++i) to[i] = t.stride(first + i);
}
// q, k (..., H, K), v (..., H, V), f (..., H) of one type and device (the gates' type may be float32); `lead`: axes in front of the heads
void check_att(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& f, int64_t lead) {
  on_cuda(q, k, v, f);
  dtype_of(q);
  expect(q.dim() == lead + 2 && v.dim() == lead + 2,
         lead == 2 ? "q, k and v must be (batch, length, heads, width)" : "q, k and v must be (batch, heads, width)");
  if (k.scalar_type() != q.scalar_type()) throw py::type_error("k must have q's type");
  expect(k.device() == q.device(), "k must be on q's device");
  expect(k.sizes() == q.sizes(), "k must have q's shape");
  if (v.scalar_type() != q.scalar_type()) throw py::type_error("v must have q's type");
  if (f.scalar_type() != q.scalar_type() && f.scalar_type() != at::kFloat) throw py::type_error("the gates must have q's type or be float32");
  if (v.device() != q.device() || f.device() != q.device()) throw py::value_error("v and the gates must be on q's device");
  expect(v.sizes().slice(0, lead + 1) == q.sizes().slice(0, lead + 1), "v must have q's batch, length and heads");
  expect(f.sizes() == q.sizes().slice(0, lead + 1), "the gates must have q's shape without its width");
  expect(q.size(-1) >= 1 && v.size(-1) >= 1 && q.size(-1) <= MEGA_ATT_MOST && v.size(-1) <= MEGA_ATT_MOST,
         "heads have 1 to 256 keys and values");
}
void check_att_state(const Tensor& h, const Tensor& q, const Tensor& v, const char* what) {
  if (!h.defined()) return;
  if (h.device() != q.device()) throw py::value_error(std::string(what) + " must be on q's device");
  if (!at::isFloatingType(h.scalar_type())) throw py::type_error(std::string(what) + " must be a floating-point tensor");
  expect(h.dim() == 4 && h.size(0) == q.size(0) && h.size(1) == q.size(-2) && h.size(2) == q.size(-1) && h.size(3) == v.size(-1),
         "a state must be (batch, heads, keys, values)");
}
// gates of (heads), the same at every step, as (batch, length, heads)
Tensor gates_of(const Tensor& f, const Tensor& q) { return f.dim() == 1 && q.dim() >= 3 ? f.expand(q.sizes().slice(0, q.dim() - 1)) : f; }
Att att_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& f, const Tensor& pad, const Tensor& reset, const Tensor& h_in,
             double scale, bool reverse) {
  check_att(q, k, v, f, 2);
  on_cuda(pad, reset, h_in);
  check_att_state(h_in, q, v, "h_in");
  Att r = {channels(q.detach()), channels(k.detach()), channels(v.detach()), f.detach(), mask_on(pad, q, "padding_mask"),
           mask_on(reset, q, "reset_mask"), f32c(h_in), {}};
  mega_decayed_attention_args& a = r.a;
  a.dtype = dtype_of(q), a.gate_dtype = dtype_of(f);
  a.B = extent(q.size(0)), a.L = extent(q.size(1)), a.H = extent(q.size(2)), a.K = (int)q.size(3), a.V = (int)v.size(3);
  a.flags = reverse ? MEGA_ATT_REVERSE : 0u;
  a.scale = scale;
  a.q = r.q.data_ptr(), a.k = r.k.data_ptr(), a.v = r.v.data_ptr(), a.f = r.f.data_ptr();
  put(a.qs, r.q, 0), put(a.ks, r.k, 0), put(a.vs, r.v, 0), put(a.fs, r.f, 0);
  a.pad_mask = ptr<uint8_t>(r.pad), a.reset_mask = ptr<uint8_t>(r.reset);
  a.h_in = fptr(r.h_in);
  return r;
}
Tensor att_work(const mega_decayed_attention_args& a, int backward, const Tensor& like) {
  const int64_t n = mega_decayed_attention_work(&a, backward);
  return n ? at::empty({n}, at::TensorOptions().dtype(at::kByte).device(like.device())) : Tensor();
}
void run_att(Att& r, const Tensor& y, const Tensor& h_out, const Where& w) {
  r.a.y = y.data_ptr();
  put(r.a.ys, y, 0);
  r.a.h_out = fptr(h_out);
  const Tensor work = att_work(r.a, 0, y);
  r.a.work = ptr(work);
  check(mega_decayed_attention_fwd(&r.a, w.stream), "decayed_attention_fwd");
}
Tensor att_state(const Tensor& q, const Tensor& v) { return floats({q.size(0), q.size(-2), q.size(-1), v.size(-1)}, q); }

// (y, state behind the last step or None)
std::tuple<Tensor, OptTensor> decayed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& f, const OptTensor& pad,
                                                const OptTensor& reset, const OptTensor& h_in, double scale, bool want_state, bool reverse) {
  Att r = att_args(q, k, v, gates_of(f, q), given(pad), given(reset), given(h_in), scale, reverse);
  const Where w(q);
  const Tensor y = rec_like(v);
  Tensor h = want_state ? att_state(q, v) : Tensor();
  if (v.numel() == 0) {   // (no step: the state stays)
    if (h.defined()) r.h_in.defined() ? h.copy_(r.h_in) : h.zero_();
  } else {
    run_att(r, y, h, w);
  }
  if (!want_state) return {y, std::nullopt};
  return {y, h};
}

// whether t lies apart from `out` (contiguous): no place from its first value to its last is one of `out`'s
bool apart(const Tensor& out, const Tensor& t) {
  if (!t.defined() || t.numel() == 0 || out.numel() == 0) return true;
  const char *to = static_cast<const char*>(out.data_ptr()), *from = static_cast<const char*>(t.data_ptr());
  int64_t low = 0, high = 0;
  for (int64_t i = 0; i < t.dim(); ++i) (t.stride(i) < 0 ? low : high) += (t.size(i) - 1) * t.stride(i);
  return to + out.nbytes() <= from + low * t.element_size() || from + (high + 1) * t.element_size() <= to;
}

// one step: q, k (B, H, K), v (B, H, V), f (B, H) -> (y, h'); h' is `h_out` where given, which may be h
std::tuple<Tensor, Tensor> decayed_attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& f_, const OptTensor& h_,
                                                  double scale, const OptTensor& h_out_) {
  const Tensor f = gates_of(f_, q_);
  check_att(q_, k_, v_, f, 1);
  on_cuda(given(h_), given(h_out_));
  check_att_state(given(h_), q_, v_, "h");
  const Where w(q_);
  const Tensor q = channels(q_), k = channels(k_), v = channels(v_), h = f32c(given(h_));
  Tensor y = at::empty(v.sizes(), v.options().requires_grad(false)), out = given(h_out_);
  if (out.defined()) {
    check_att_state(out, q_, v_, "h_out");
    expect(out.scalar_type() == at::kFloat && out.is_contiguous(), "h_out must be contiguous float32");
    expect(!h.defined() || out.data_ptr() == h.data_ptr() || apart(out, h), "h_out overlaps h and is not h");
    for (const Tensor& t : {q, k, v, f}) expect(apart(out, t), "h_out overlaps q, k, v or the gates");
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();   // (a graph that has saved it must not use the new values)
  } else {
    out = att_state(q, v);
  }
  if (v.numel()) {
    mega_decayed_attention_args a = {};
    a.dtype = dtype_of(q), a.gate_dtype = dtype_of(f);
    a.B = extent(q.size(0)), a.L = 1, a.H = extent(q.size(1)), a.K = (int)q.size(2), a.V = (int)v.size(2);
    a.scale = scale;
    a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr(), a.f = f.data_ptr();
    auto strides = [](int64_t* to, const Tensor& t) { to[0] = t.stride(0), to[1] = 0, to[2] = t.stride(1); };
    strides(a.qs, q), strides(a.ks, k), strides(a.vs, v), strides(a.fs, f), strides(a.ys, y);
    a.y = y.data_ptr(), a.h_in = fptr(h), a.h_out = fptr(out);
    check(mega_decayed_attention_step(&a, w.stream), "decayed_attention_step");
  }
  return {y, out};
}

// Separate operands, or one tensor z (B, L, H (2 K + V + 1)) that holds q, k, v and the gates side by side, whose gradient then comes
// as one tensor too.
struct AttParts {
  Tensor q, k, v, f;
  AttParts(const Tensor& z, int64_t heads, int64_t keys) {
    const int64_t kd = heads * keys, vd = z.size(2) - 2 * kd - heads;
    q = part(z, 0, kd, heads), k = part(z, kd, kd, heads), v = part(z, 2 * kd, vd, heads), f = z.narrow(2, 2 * kd + vd, heads);
  }
  static Tensor part(const Tensor& z, int64_t from, int64_t n, int64_t heads) {
    return z.narrow(2, from, n).unflatten(2, {heads, n / heads});
  }
};
class AttFn : public torch::autograd::Function<AttFn> {
 public:
  static variable_list forward(AutogradContext* ctx, Tensor q, OptTensor k, OptTensor v, OptTensor f, OptTensor pad, OptTensor reset,
                               OptTensor h_in, double scale, bool want_state, bool reverse, int64_t heads, int64_t keys) {
    Att r;
    if (heads) {
      const AttParts p(q.detach(), heads, keys);
      r = att_args(p.q, p.k, p.v, p.f, given(pad), given(reset), given(h_in), scale, reverse);
    } else {
      r = att_args(q, *k, *v, *f, given(pad), given(reset), given(h_in), scale, reverse);
    }
    const Where w(q);
    Tensor y = rec_like(r.v), h = want_state ? att_state(r.q, r.v) : Tensor();
    run_att(r, y, h, w);
    ctx->set_materialize_grads(false);
    const Tensor state = given(h_in);
    const bool same = state.defined() && r.h_in.data_ptr() == state.data_ptr();
    ctx->save_for_backward({q, given(k), given(v), given(f), r.pad, r.reset, same ? state : r.h_in});
    ctx->saved_data["state"] = state.defined() ? (int64_t)state.scalar_type() : (int64_t)-1;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["keys"] = keys;
    if (!want_state) return {y};
    return {y, h};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    const auto s = ctx->get_saved_variables();
    const int64_t heads = ctx->saved_data["heads"].toInt(), keys = ctx->saved_data["keys"].toInt();
    const int64_t state = ctx->saved_data["state"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const bool reverse = ctx->saved_data["reverse"].toBool();
    const Where w(s[0]);
    Att r;
    Tensor dz, dq, dk, dv, df;
    if (heads) {
      const AttParts p(s[0].detach(), heads, keys);
      r = att_args(p.q, p.k, p.v, p.f, s[4], s[5], s[6], scale, reverse);
      dz = at::empty(s[0].sizes(), s[0].options().requires_grad(false));
      const AttParts d(dz, heads, keys);
      dq = d.q, dk = d.k, dv = d.v, df = d.f;
    } else {
      r = att_args(s[0], s[1], s[2], s[3], s[4], s[5], s[6], scale, reverse);
      dq = rec_like(r.q), dk = rec_like(r.k), dv = rec_like(r.v), df = at::empty(r.f.sizes(), r.f.options().requires_grad(false));
    }
    const Tensor dy = grads[0].defined() ? rec_grad(grads[0], r.v) : at::zeros(r.v.sizes(), r.v.options());
    const Tensor dh_out = grads.size() > 1 && grads[1].defined() ? f32c(grads[1]) : Tensor();
    Tensor dh_in = state >= 0 ? att_state(r.q, r.v) : Tensor();
    mega_decayed_attention_args& a = r.a;
    a.dy = dy.data_ptr(), a.dq = dq.data_ptr(), a.dk = dk.data_ptr(), a.dv = dv.data_ptr(), a.df = df.data_ptr();
    put(a.gs, dy, 0), put(a.dqs, dq, 0), put(a.dks, dk, 0), put(a.dvs, dv, 0), put(a.dfs, df, 0);
    a.dh_out = fptr(dh_out), a.dh_in = fptr(dh_in);
    const Tensor work = att_work(a, 1, dy);
    a.work = ptr(work);
    check(mega_decayed_attention_bwd(&a, w.stream), "decayed_attention_bwd");
    if (dh_in.defined()) dh_in = dh_in.to((at::ScalarType)state);
    const Tensor no;
    if (heads) return {dz, no, no, no, no, no, dh_in, no, no, no, no, no};
    return {dq, dk, dv, df, no, no, dh_in, no, no, no, no, no};
  }
};
// (y, h) or (y,); differentiable
variable_list decayed_attention_train(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& f_, const OptTensor& pad,
                                      const OptTensor& reset, const OptTensor& h_in, double scale, bool want_state, bool reverse) {
  on_cuda(q, k, v, f_);
  const Tensor f = gates_of(f_, q);
  if (q.numel() == 0 || v.numel() == 0) {   // (else AttFn checks them, and converts what it has to once)
    att_args(q, k, v, f, given(pad), given(reset), given(h_in), scale, reverse);
    variable_list r = {v * ((q * k).sum(-1, true) * f.unsqueeze(-1)).to(v.scalar_type())};   // (no values, but gradients of that shape)
    if (want_state) r.push_back(h_in.has_value() ? h_in->to(at::kFloat, false, true) : att_state(q, v).zero_());
    return r;
  }
  return AttFn::apply(q, OptTensor(k), OptTensor(v), OptTensor(f), pad, reset, h_in, scale, want_state, reverse, (int64_t)0, (int64_t)0);
}
variable_list decayed_attention_packed(const Tensor& z, int64_t heads, int64_t keys, const OptTensor& pad, const OptTensor& reset,
                                       const OptTensor& h_in, double scale, bool want_state, bool reverse) {
  on_cuda(z);
  expect(z.dim() == 3 && heads >= 1 && keys >= 1 && (z.size(2) - heads * (2 * keys + 1)) > 0 && (z.size(2) - heads * (2 * keys + 1)) % heads == 0,
         "the packed operand must be (batch, length, heads (2 keys + values + 1))");
  if (z.numel() == 0) {
    const AttParts p(z, heads, keys);
    return decayed_attention_train(p.q, p.k, p.v, p.f, pad, reset, h_in, scale, want_state, reverse);
  }
  return AttFn::apply(z, OptTensor(), OptTensor(), OptTensor(), pad, reset, h_in, scale, want_state, reverse, heads, keys);
}

// -------------------------------------------------------------------- root-mean-square norm with a residual
struct Rms {
  Tensor x, res, w;
  int B, L, D, G;
};
Rms rms_args(const Tensor& x, const Tensor& weight, const Tensor& res, int64_t groups) {
  on_cuda(x, weight, res);
  dtype_of(x);
  expect(x.dim() >= 2, "x must be (batch, ..., channels)");
  same_kind(res, x, "the residual");
  const int64_t d = x.size(-1);
  expect(groups >= 1 && d % groups == 0, "num_groups must divide the channels");
  expect_numel(weight, d, "weight");
  if (!at::isFloatingType(weight.scalar_type())) throw py::type_error("weight must be a floating-point tensor");
  if (weight.device() != x.device()) throw py::value_error("weight must be on x's device");
  Rms r;
  if (x.numel() == 0) return r;
  r.x = gn_rows(x.detach());
  if (res.defined()) r.res = gn_rows(res.detach());
  r.w = gn_param(weight.detach());
  r.B = extent(r.x.size(0)), r.L = extent(r.x.size(1)), r.D = extent(d), r.G = extent(groups);
  return r;
}
// y, and r with a residual
std::pair<Tensor, Tensor> run_rms(const Tensor& x, const Rms& r, double eps, const Where& w) {
  auto [out, y] = gn_like(x, r.x);
  Tensor total, sum;
  if (r.res.defined()) std::tie(total, sum) = gn_like(x, r.x);
  check(mega_rms_norm_fwd(r.x.data_ptr(), ptr(r.res), y.data_ptr(), ptr(sum), dtype_of(r.x), r.B, r.L, r.D, STRIDES2(r.x), STRIDES2(r.res),
                          STRIDES2(y), STRIDES2(sum), fptr(r.w), r.G, eps, w.stream), "rms_norm_fwd");
  return {out, total};
}
std::tuple<Tensor, OptTensor> rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& res, int64_t groups, double eps) {
  const Rms r = rms_args(x, weight, given(res), groups);
  const bool two = res.has_value();
  if (x.numel() == 0) return {fresh(x), two ? OptTensor(fresh(x)) : std::nullopt};
  const Where w(x);
  auto [y, sum] = run_rms(x, r, eps, w);
  return {y, two ? OptTensor(sum) : std::nullopt};
}
class RmsFn : public torch::autograd::Function<RmsFn> {
 public:
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, OptTensor res, int64_t groups, double eps) {
    const Rms r = rms_args(x, weight, given(res), groups);
    const Where w(x);
    auto [y, sum] = run_rms(x, r, eps, w);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({sum.defined() ? sum : x, weight});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["residual"] = sum.defined();
    if (!sum.defined()) return {y};
    return {y, sum};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    const auto s = ctx->get_saved_variables();
    const Rms r = rms_args(s[0], s[1], Tensor(), ctx->saved_data["groups"].toInt());
    const Where w(s[0]);
    const int dt = dtype_of(r.x);
    auto rows = [&](const Tensor& g) { return g.defined() ? gn_rows(g.scalar_type() == r.x.scalar_type() ? g : g.to(r.x.scalar_type())) : Tensor(); };
    Tensor dy = rows(grads[0]);
    const Tensor dr = grads.size() > 1 ? rows(grads[1]) : Tensor();
    if (!dy.defined()) dy = at::zeros(r.x.sizes(), r.x.options());
    auto [out, dx] = gn_like(s[0], r.x);
    Tensor dw = floats({r.D}, r.x);
    const Tensor work = bytes_of(mega_rms_norm_work(dt, r.B, r.L, r.D, r.G), r.x);
    check(mega_rms_norm_bwd(dy.data_ptr(), ptr(dr), r.x.data_ptr(), dx.data_ptr(), dt, r.B, r.L, r.D, STRIDES2(dy), STRIDES2(dr), STRIDES2(r.x),
                            STRIDES2(dx), fptr(r.w), r.G, ctx->saved_data["eps"].toDouble(), fptr(dw), work.data_ptr(), w.stream), "rms_norm_bwd");
    const Tensor& weight = s[1];
    Tensor g = weight.dim() == 1 ? dw : dw.view(weight.sizes());
    if (weight.scalar_type() != at::kFloat) g = g.to(weight.scalar_type());
    return {out, g, ctx->saved_data["residual"].toBool() ? out : Tensor(), Tensor(), Tensor()};
  }
};
variable_list rms_norm_train(const Tensor& x, const Tensor& weight, const OptTensor& res, int64_t groups, double eps) {
  if (x.numel() == 0) {   // (no values, but gradients of that shape)
    rms_args(x, weight, given(res), groups);
    const Tensor total = res.has_value() ? x + *res : x;
    const Tensor y = (total * weight.view({-1})).to(x.scalar_type());
    return res.has_value() ? variable_list{y, total} : variable_list{y};
  }
  return RmsFn::apply(x, weight, res, groups, eps);
}

Tensor softmax_fwd(const Tensor& x, bool causal) {
  on_cuda(x);
  const Where w(x);
  const Tensor xc = x.contiguous();
  const int64_t outer = xc.size(-2), inner = xc.size(-1);
  Tensor y = fresh(xc);
  check(mega_attention_softmax_fwd(xc.data_ptr(), y.data_ptr(), dtype_of(xc), xc.numel() / (outer * inner), outer, (int)inner, causal,
                                   w.stream), "attention_softmax_fwd");
  return y;
}

// the shapes that pointers into the projections' outputs rely on
void check_block(const Tensor& x, const Tensor& wv, const Tensor& wm, const Tensor& wh, const Tensor& gamma, const Tensor& beta,
                 const Tensor& bias, const Tensor& rot, int64_t period) {
  const int64_t d = x.size(2), s = gamma.size(1), e = wv.size(0);
  expect(wv.dim() == 2 && wv.size(1) == d && wm.dim() == 2 && wm.size(0) == 2 * d + s + e && wm.size(1) == d && wh.dim() == 2 &&
             wh.size(0) == d && wh.size(1) == e, "projections do not fit the block");
  expect(gamma.numel() == 2 * s && beta.numel() == 2 * s, "gamma and beta must be (2, zdim)");
  expect(period > 0 && x.size(0) * x.size(1) % period == 0, "chunks do not divide the sequence");
  expect(!bias.defined() || bias.numel() >= 2 * period - 1, "relative bias too short");
  expect(!rot.defined() || rot.numel() >= period * s, "rotary table too short");
}

// Training pass from the moving average to the output.  bias: learned relative bias (2 P - 1), or rot: rotary table
// (positions, S / 2, 2) with the causal mask; rows (b, t) sit at position t % period of their chunk.
class BlockFn : public torch::autograd::Function<BlockFn> {
 public:
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor xn, Tensor mx, Tensor wv, Tensor bv, Tensor wm, Tensor bm, Tensor wh,
                        Tensor gamma, Tensor beta, OptTensor bias_, OptTensor rot_, OptTensor mask_, int64_t period) {
    on_cuda(x, xn, mx, wv, bv, wm, bm, wh, gamma, beta, given(bias_), given(rot_), given(mask_));
    const Where w(x);
    const int64_t bsz = x.size(0), seq = x.size(1), d = x.size(2), rows = bsz * seq, s = gamma.size(1), e = wv.size(0);
    const int64_t f = 2 * d + s + e, nb = rows / period;
    check_block(x, wv, wm, wh, gamma, beta, given(bias_), given(rot_), period);
    const int dt = dtype_of(x);
    const int64_t es = x.element_size();
    const Tensor bias = given(bias_), rot = given(rot_);
    const Tensor x_ = x, xn_ = xn, mx_ = mx;
    x = x.contiguous();
    xn = xn.contiguous().view({rows, d});
    mx = mx.contiguous().view({rows, d});
    Tensor v_lin = at::addmm(bv, xn, wv.t());
    Tensor base = at::addmm(bm, mx, wm.t());
    char* bp = static_cast<char*>(base.data_ptr());
    char *u = bp, *z = bp + d * es, *r = z + s * es, *hx = r + e * es;
    Tensor v = fresh(v_lin);
    check(mega_gate_silu(v_lin.data_ptr(), e, nullptr, 0, v.data_ptr(), e, dt, rows, (int)e, w.stream), "gate_silu");
    const auto affine = f32_all({gamma, beta}, w.stream);
    const Tensor &ga = affine[0], &be = affine[1];
    Tensor q = at::empty({nb, period, s}, x.options().requires_grad(false)), k = fresh(q);
    if (rot.defined())
      check(mega_gate_qk_rotary(z, f, fptr(ga), fptr(be), fptr(rot), (int)rot.size(0), (int)period, 0, q.data_ptr(), s, k.data_ptr(), s,
                                dt, rows, (int)s, 1e-5, w.stream), "gate_qk_rotary");
    else
      check(mega_gate_qk(z, f, fptr(ga), fptr(be), q.data_ptr(), s, k.data_ptr(), s, dt, rows, (int)s, 1e-5, w.stream), "gate_qk");
    Tensor v3 = v.view({nb, period, e});
    Tensor wgt;
    {
      Tensor scores = at::bmm(q, k.transpose(1, 2));
      wgt = fresh(scores);
      if (rot.defined()) {
        check(mega_attention_softmax_fwd(scores.data_ptr(), wgt.data_ptr(), dt, nb, period, (int)period, 1, w.stream),
              "attention_softmax_fwd");
      } else {
        const Tensor mask = mask_u8(given(mask_), bsz, seq);
        const Tensor b = bias.scalar_type() == x.scalar_type() ? bias.detach().contiguous() : bias.detach().to(x.scalar_type()).contiguous();
        check(mega_attention_bias_softmax_fwd(scores.data_ptr(), wgt.data_ptr(), b.data_ptr(), (int)((b.size(0) + 1) / 2),
                                              ptr<uint8_t>(mask), dt, nb, (int)period, (int)period, w.stream),
              "attention_bias_softmax_fwd");
      }
    }
    Tensor attn = at::bmm(wgt, v3).view({rows, e});
    Tensor gated = fresh(attn);
    check(mega_gate_mul_silu(attn.data_ptr(), e, r, f, gated.data_ptr(), e, dt, rows, (int)e, w.stream), "gate_mul_silu");
    Tensor h_lin = at::mm(gated, wh.t());
    Tensor out = at::empty({bsz, seq, d}, x.options().requires_grad(false));
    check(mega_gate_output(x.data_ptr(), d, u, f, hx, f, h_lin.data_ptr(), d, out.data_ptr(), d, dt, rows, (int)d, w.stream), "gate_output");
    ctx->save_for_backward({x_, xn_, mx_, wv, wm, wh, ga, bias, rot, v_lin, base, q, k, v3, wgt, attn, gated, h_lin, bv, bm, gamma, beta,
                            rot.defined() ? Tensor() : mask_u8(given(mask_), bsz, seq)});
    ctx->saved_data["period"] = period;
    ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)bv.scalar_type(), (int64_t)bm.scalar_type(), (int64_t)gamma.scalar_type(),
                                                    (int64_t)beta.scalar_type()};
    return out;
  }

  // The pass in torch operations, for a gradient that is to be differentiated again: the gradients of the inputs as
  // functions of the inputs.  (Through aliases of them: an input that another one was computed from gets its own share.)
  static variable_list differentiable(AutogradContext* ctx, const variable_list& sv, Tensor dout) {
    const int64_t period = ctx->saved_data["period"].toInt();
    std::vector<Tensor> in = {sv[0], sv[1], sv[2], sv[3], sv[18], sv[4], sv[19], sv[5], sv[20], sv[21], sv[7]};
    for (auto& t : in)
      if (t.defined()) t = t.view_as(t);
    const Tensor &x = in[0], &xn = in[1], &mx = in[2], &wv = in[3], &bv = in[4], &wm = in[5], &bm = in[6], &wh = in[7], &gamma = in[8],
                 &beta = in[9], &bias = in[10], &rot = sv[8], &mask = sv[22];
    const int64_t bsz = x.size(0), seq = x.size(1), d = x.size(2), s = gamma.size(1), e = wv.size(0), nb = bsz * seq / period;
    const auto type = x.scalar_type();
    const Tensor v = at::silu(at::linear(xn, wv, bv)).reshape({nb, period, e}), base = at::linear(mx, wm, bm);
    const Tensor u = base.narrow(2, 0, d), z = base.narrow(2, d, s), r = base.narrow(2, d + s, e), hx = base.narrow(2, d + s + e, d);
    const Tensor zn = z / z.norm(2, {-1}, true).clamp_min(1e-5);
    auto part = [&](int64_t i) {
      Tensor t = (zn * (gamma[i] + 1.0) + beta[i]).reshape({nb, period, s});
      if (!rot.defined()) return t.to(type);
      const Tensor w = rot.narrow(0, 0, period), f = t.to(at::kFloat).reshape({nb, period, s / 2, 2});
      const Tensor a = f.select(3, 0), b = f.select(3, 1), c = w.select(2, 0), i_ = w.select(2, 1);
      return at::stack({a * c - b * i_, a * i_ + b * c}, -1).flatten(2).to(type);
    };
    Tensor scores = at::bmm(part(0), part(1).transpose(1, 2));
    const auto where = scores.options().requires_grad(false);
    if (rot.defined()) {
      scores = scores.masked_fill(at::ones({period, period}, where.dtype(at::kBool)).triu(1), -INFINITY);
    } else {
      const Tensor at_ = at::arange(period, where.dtype(at::kLong));
      scores = scores + bias.index({at_.unsqueeze(0) - at_.unsqueeze(1) + (bias.size(0) + 1) / 2 - 1});
      if (mask.defined()) {
        const Tensor m = mask.reshape({nb, period}).to(at::kBool);
        scores = scores.masked_fill(m.logical_and(m.all(1, true).logical_not()).unsqueeze(1), -INFINITY);
      }
    }
    const Tensor attn = at::bmm(scores.to(at::kFloat).softmax(-1).to(type), v).reshape({bsz, seq, e});
    const Tensor h = at::silu(hx + at::linear(attn * at::silu(r), wh));
    const Tensor out = at::addcmul(x, u.sigmoid(), h - x);
    variable_list wanted, result(14);
    std::vector<size_t> place;
    for (size_t i = 0; i < in.size(); ++i)
      if (in[i].defined() && in[i].requires_grad()) {
        wanted.push_back(in[i]);
        place.push_back(i);
      }
    const auto g = torch::autograd::grad({out}, wanted, {dout}, true, true, true);
    for (size_t i = 0; i < place.size(); ++i) result[place[i]] = g[i];
    return result;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto sv = ctx->get_saved_variables();
    if (at::GradMode::is_enabled()) return differentiable(ctx, sv, grads[0].to(sv[0].scalar_type()));
    const Tensor x = sv[0].contiguous(), xn = sv[1].contiguous().flatten(0, 1), mx = sv[2].contiguous().flatten(0, 1);
    const Tensor &wv = sv[3], &wm = sv[4], &wh = sv[5], &ga = sv[6], &bias = sv[7], &rot = sv[8],
                 &v_lin = sv[9], &base = sv[10], &q = sv[11], &k = sv[12], &v3 = sv[13], &wgt = sv[14], &attn = sv[15], &gated = sv[16],
                 &h_lin = sv[17];
    const Where w(x);
    const int64_t period = ctx->saved_data["period"].toInt();
    const auto types = ctx->saved_data["types"].toIntVector();
    const int64_t bsz = x.size(0), seq = x.size(1), d = x.size(2), rows = bsz * seq, s = ga.size(1), e = wv.size(0), nb = rows / period;
    const int64_t f = base.size(1), nbias = bias.defined() ? bias.size(0) : 0;
    const int dt = dtype_of(x);
    const int64_t es = x.element_size();
    Tensor dout = grads[0];
    if (dout.scalar_type() != x.scalar_type()) dout = dout.to(x.scalar_type());
    dout = dout.contiguous();
    // every sum in one zeroed piece: bias gradients of v_proj and mx_proj, the (2, s) affine, the relative bias
    Tensor sums = at::zeros({e + f + 4 * s + nbias}, at::TensorOptions().dtype(at::kFloat).device(x.device()));
    float *sbv = fptr(sums), *sbm = sbv + e, *sg = sbm + f, *sb = sg + 2 * s, *srel = sb + 2 * s;
    Tensor dbase = fresh(base), dx = fresh(x);
    auto cut = [&](const Tensor& t, char*& u, char*& z, char*& r, char*& hx) {
      u = static_cast<char*>(t.data_ptr());
      z = u + d * es;
      r = z + s * es;
      hx = r + e * es;
    };
    char *u, *z, *r, *hx, *du, *dz, *dr, *dhx;
    cut(base, u, z, r, hx);
    cut(dbase, du, dz, dr, dhx);
    check(mega_gate_output_bwd(dout.data_ptr(), d, x.data_ptr(), d, u, f, hx, f, h_lin.data_ptr(), d, dx.data_ptr(), d, du, f, dhx, f, sbm,
                               sbm + d + s + e, dt, rows, (int)d, w.stream), "gate_output_bwd");
    const Tensor dh = dbase.narrow(1, d + s + e, d);
    Tensor dgated = at::mm(dh, wh);
    const bool need_xn = ctx->needs_input_grad(1), need_mx = ctx->needs_input_grad(2), need_wv = ctx->needs_input_grad(3),
               need_wm = ctx->needs_input_grad(5), need_wh = ctx->needs_input_grad(7);
    Tensor dwh = need_wh ? at::mm(dh.t(), gated) : Tensor();
    check(mega_gate_mul_silu_bwd(dgated.data_ptr(), e, attn.data_ptr(), e, r, f, dgated.data_ptr(), e, dr, f, sbm + d + s, dt, rows, (int)e,
                                 w.stream), "gate_mul_silu_bwd");
    const Tensor dattn = dgated.view({nb, period, e});
    Tensor dv = at::bmm(wgt.transpose(1, 2), dattn).view({rows, e});
    Tensor ds;
    {
      Tensor dw = at::bmm(dattn, v3.transpose(1, 2));
      ds = fresh(dw);
      check(mega_attention_softmax_bwd(dw.data_ptr(), wgt.data_ptr(), ds.data_ptr(), dt, nb, period, (int)period, rot.defined() ? 1 : 0,
                                       w.stream), "attention_softmax_bwd");
    }
    if (nbias)
      check(mega_attention_bias_grad(ds.data_ptr(), srel, (int)((nbias + 1) / 2), dt, nb, (int)period, (int)period, w.stream),
            "attention_bias_grad");
    Tensor dq = at::bmm(ds, k), dk = at::bmm(ds.transpose(1, 2), q);
    check(mega_gate_qk_bwd(z, f, fptr(ga), fptr(rot), rot.defined() ? (int)rot.size(0) : 0, (int)period, 0, dq.data_ptr(), s, dk.data_ptr(),
                           s, dz, f, sg, sb, sbm + d, dt, rows, (int)s, 1e-5, w.stream), "gate_qk_bwd");
    check(mega_gate_silu_bwd(dv.data_ptr(), e, v_lin.data_ptr(), e, dv.data_ptr(), e, sbv, dt, rows, (int)e, w.stream), "gate_silu_bwd");
    Tensor dxn = need_xn ? at::mm(dv, wv).view({bsz, seq, d}) : Tensor();
    Tensor dwv = need_wv ? at::mm(dv.t(), xn) : Tensor();
    Tensor dmx = need_mx ? at::mm(dbase, wm).view({bsz, seq, d}) : Tensor();
    Tensor dwm = need_wm ? at::mm(dbase.t(), mx) : Tensor();
    const auto own = wv.scalar_type();   // (one conversion where all share it; none passes through another's type)
    const bool same = std::all_of(types.begin(), types.end(), [&](int64_t t) { return t == (int64_t)own; }) &&
                      (!nbias || bias.scalar_type() == own);
    Tensor flat = same ? sums.to(own) : sums;
    auto part = [&](int64_t from, int64_t count, int64_t type) {
      Tensor t = flat.narrow(0, from, count);
      return t.scalar_type() == (at::ScalarType)type ? t : t.to((at::ScalarType)type);
    };
    return {dx, dxn, dmx, dwv, part(0, e, types[0]), dwm, part(e, f, types[1]), dwh, part(e + f, 2 * s, types[2]).view({2, s}),
            part(e + f + 2 * s, 2 * s, types[3]).view({2, s}),
            nbias ? part(e + f + 4 * s, nbias, (int64_t)bias.scalar_type()) : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// Inference from the moving average to the output, chunked causal attention with rotary positions.  cache: the keys
// (before their rotation) and values come back too, as a decoding state keeps them.
std::tuple<Tensor, Tensor, Tensor> block_infer(Tensor x, Tensor xn, Tensor mx, const Tensor& wv, const Tensor& bv, const Tensor& wm,
                                               const Tensor& bm, const Tensor& wh, const Tensor& gamma, const Tensor& beta,
                                               const Tensor& rot, int64_t period, bool cache) {
  on_cuda(x, xn, mx, wv, bv, wm, bm, wh, gamma, beta, rot);
  check_block(x, wv, wm, wh, gamma, beta, none(), rot, period);
  const Where w(x);
  const int64_t bsz = x.size(0), seq = x.size(1), d = x.size(2), rows = bsz * seq, s = gamma.size(1), e = wv.size(0);
  const int64_t f = 2 * d + s + e, nb = rows / period;
  const int dt = dtype_of(x);
  const int64_t es = x.element_size();
  x = x.contiguous();
  const Tensor xn2 = xn.contiguous().view({rows, d}), mx2 = mx.contiguous().view({rows, d});
  // (score rows and reduction indices in whole 16-byte pieces: the library's products are several times faster on them;
  // the positions in between are of no row's causal range, and their values zero.  It takes a launch for each chunk, so at 32
  // chunks the two are level: 32 of 500 take 615 us with the pitch, 33 of 500 take 605 without)
  const int64_t pitch = period % 8 && nb <= 32 ? (period + 7) / 8 * 8 : period;
  Tensor v_lin = at::addmm(bv, xn2, wv.t()), v3 = v_lin.view({nb, period, e}), vp = v3;
  if (pitch != period) {
    vp = at::empty({nb, pitch, e}, x.options());
    vp.narrow(1, period, pitch - period).zero_();
    v3 = vp.narrow(1, 0, period);
    for (int64_t i = 0; i < nb; ++i)
      check(mega_gate_silu(static_cast<char*>(v_lin.data_ptr()) + i * period * e * es, e, nullptr, 0,
                           static_cast<char*>(vp.data_ptr()) + i * pitch * e * es, e, dt, period, (int)e, w.stream), "gate_silu");
  } else {
    check(mega_gate_silu(v_lin.data_ptr(), e, nullptr, 0, v_lin.data_ptr(), e, dt, rows, (int)e, w.stream), "gate_silu");
  }
  const Tensor base = at::addmm(bm, mx2, wm.t());
  char* bp = static_cast<char*>(base.data_ptr());
  char *u = bp, *z = bp + d * es, *r = z + s * es, *hx = r + e * es;
  const auto affine = f32_all({gamma, beta}, w.stream);
  const Tensor &ga = affine[0], &be = affine[1];
  Tensor q = at::empty({nb, pitch, s}, x.options()), k = fresh(q), raw;
  if (cache) raw = at::empty({bsz, seq, s}, x.options());
  check(mega_gate_qk_rotary_cache(z, f, fptr(ga), fptr(be), fptr(rot), (int)rot.size(0), (int)period, 0, (int)pitch, q.data_ptr(), s,
                                  k.data_ptr(), s, ptr(raw), dt, rows, (int)s, 1e-5, w.stream), "gate_qk_rotary");
  const Tensor scores = at::bmm(q, k.transpose(1, 2));
  Tensor wgt = fresh(scores);
  check(mega_attention_softmax_fwd(scores.data_ptr(), wgt.data_ptr(), dt, nb, pitch, (int)pitch, 1, w.stream), "attention_softmax_fwd");
  Tensor attn = at::bmm(wgt.narrow(1, 0, period), vp).view({rows, e});
  check(mega_gate_mul_silu(attn.data_ptr(), e, r, f, attn.data_ptr(), e, dt, rows, (int)e, w.stream), "gate_mul_silu");
  Tensor out = at::mm(attn, wh.t()).view({bsz, seq, d});
  check(mega_gate_output(x.data_ptr(), d, u, f, hx, f, out.data_ptr(), d, out.data_ptr(), d, dt, rows, (int)d, w.stream), "gate_output");
  return {out, raw, cache ? v3.reshape({bsz, seq, e}) : Tensor()};
}

Tensor block_train(const Tensor& x, const Tensor& xn, const Tensor& mx, const Tensor& wv, const Tensor& bv, const Tensor& wm,
                   const Tensor& bm, const Tensor& wh, const Tensor& gamma, const Tensor& beta, const OptTensor& bias,
                   const OptTensor& rot, const OptTensor& mask, int64_t period) {
  return BlockFn::apply(x, xn, mx, wv, bv, wm, bm, wh, gamma, beta, bias, rot, mask, period);
}

// ------------------------------------------------------------------------------------ single-token step
// TimestepNorm -> EMA on one token is one launch of 3 us, so the call is as fast as its host path: the same checks
// and the same library call took 6.6 us through the interpreter and ctypes, 2 us here.
//
// A plan is everything a step passes to the library, and what it was built from: it holds as long as the parameters
// (identity, version counters and storage: p.data = t, which is also how a module is moved, leaves the first two alone), the
// state tensors, the batch, the dtype and the options stay what they were.  The state tensors are updated in place, except
// the counts: one array is read, another written, and they alternate.
struct Names {
  PyObject *params, *modules, *groups, *bidirectional, *plan, *block_plan, *count, *mean, *var, *h, *key, *value, *key_mask,
      *forward, *hooks, *pre_hooks;
  Names() {
    auto s = [](const char* t) { return PyUnicode_InternFromString(t); };
    params = s("_parameters"); groups = s("num_groups"); bidirectional = s("bidirectional"); plan = s("_step_plan");
    modules = s("_modules"); block_plan = s("_block_plan"); key = s("prev_key"); value = s("prev_value");
    key_mask = s("prev_key_padding_mask"); forward = s("forward"); hooks = s("_forward_hooks"); pre_hooks = s("_forward_pre_hooks");
    count = s("prev_count"); mean = s("prev_mean"); var = s("prev_var"); h = s("prev_state");
  }
};
const Names& names() {
  static const Names* n = new Names;
  return *n;
}

int64_t version_of(const Tensor& t) { return (int64_t)t.unsafeGetTensorImpl()->version_counter().current_version(); }

// A parameter as it was when a plan was built; its storage stays as long as the plan, which may hold its address.
struct Mark {
  int64_t version;
  const void* at;
  c10::Storage storage;
  explicit Mark(const Tensor& t) : version(version_of(t)), at(t.data_ptr()), storage(t.storage()) {}
  bool holds(const Tensor& t) const { return version_of(t) == version && t.data_ptr() == at; }
};

struct StepPlan {
  std::vector<py::object> names, params;   // two of the norm, five of the layer
  std::vector<Mark> marks;
  py::object nkey, ekey, groups, activation;
  py::object count, count_next, mean, var, h;
  std::vector<Tensor> operands;            // gamma, beta, p, q, g, omega (fp32)
  bool kept = false;                       // (below)
  Tensor count_t, next_t, mean_t, var_t, h_t;
  int dtype, device, ndim, cplx, normed;
  int64_t batch, dim;
  double eps;
};

std::unique_ptr<StepPlan> step_plan(std::vector<py::object> names, std::vector<py::object> params, py::object nkey, py::object ekey,
                                    py::object groups, py::object activation, std::vector<py::object> state,
                                    std::vector<Tensor> operands, const Tensor& x, bool cplx, bool normed, double eps) {
  auto p = std::make_unique<StepPlan>();
  p->names = std::move(names);
  p->params = std::move(params);
  for (auto& t : p->params) p->marks.emplace_back(THPVariable_Unpack(t.ptr()));
  p->nkey = std::move(nkey); p->ekey = std::move(ekey); p->groups = std::move(groups); p->activation = std::move(activation);
  p->count = state[0]; p->count_next = state[1]; p->mean = state[2]; p->var = state[3]; p->h = state[4];
  p->count_t = THPVariable_Unpack(p->count.ptr()); p->next_t = THPVariable_Unpack(p->count_next.ptr());
  p->mean_t = THPVariable_Unpack(p->mean.ptr()); p->var_t = THPVariable_Unpack(p->var.ptr());
  p->h_t = THPVariable_Unpack(p->h.ptr());
  p->operands = std::move(operands);
  p->dtype = dtype_of(x); p->device = (int)x.get_device(); p->ndim = (int)p->operands[2].size(1);
  p->cplx = cplx; p->normed = normed; p->batch = x.size(0); p->dim = x.size(2); p->eps = eps;
  return p;
}

bool params_match(const StepPlan& p, PyObject* dict, size_t from, size_t to) {
  for (size_t i = from; i < to; ++i) {
    PyObject* t = PyDict_GetItemWithError(dict, p.names[i].ptr());
    if (t != p.params[i].ptr() || !p.marks[i].holds(THPVariable_Unpack(t))) return false;
  }
  return true;
}

// norm_ema_step(norm, move, x, incremental_state, activation, return_normed): the outputs, or None when the layer has
// no plan for this call
// A graph that holds a step works on the state's tensors, which whoever replays it has to keep, and on the plan's, which go
// with the plan: with the next generation, or a change of mode.  Those stay as long as the pole states then.
void keep_with_state(StepPlan& p) {
  using Kept = std::unordered_map<PyObject*, std::pair<py::object, std::vector<Tensor>>>;
  static Kept* const all = new Kept;
  PyObject* const h = p.h.ptr();
  auto& kept = (*all)[h];
  if (!kept.first) kept.first = py::weakref(h, py::cpp_function([h](py::handle) { all->erase(h); }));
  kept.second.insert(kept.second.end(), p.operands.begin(), p.operands.end());
  kept.second.push_back(p.count_t);
  kept.second.push_back(p.next_t);
  p.kept = true;
}

PyObject* norm_ema_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 6) throw py::type_error("norm_ema_step takes 6 arguments");
    if (!THPVariable_Check(a[2]) || !PyDict_Check(a[3]) || at::GradMode::is_enabled()) Py_RETURN_NONE;
    const Names& k = names();
    const auto norm = py::reinterpret_steal<py::object>(PyObject_GenericGetDict(a[0], nullptr));
    const auto move = py::reinterpret_steal<py::object>(PyObject_GenericGetDict(a[1], nullptr));
    PyObject* held = move ? PyDict_GetItemWithError(move.ptr(), k.plan) : nullptr;
    if (!held || held == Py_None || !norm) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    StepPlan& p = *py::cast<StepPlan*>(py::handle(held));
    const Tensor& x = THPVariable_Unpack(a[2]);
    PyObject* ns = PyDict_GetItemWithError(a[3], p.nkey.ptr());
    PyObject* es = PyDict_GetItemWithError(a[3], p.ekey.ptr());
    PyObject* np = PyDict_GetItemWithError(norm.ptr(), k.params);
    PyObject* mp = PyDict_GetItemWithError(move.ptr(), k.params);
    const bool same = ns && es && np && mp && PyDict_Check(ns) && PyDict_Check(es) &&
                      PyDict_GetItemWithError(ns, k.mean) == p.mean.ptr() && PyDict_GetItemWithError(ns, k.var) == p.var.ptr() &&
                      PyDict_GetItemWithError(ns, k.count) == p.count.ptr() && PyDict_GetItemWithError(es, k.h) == p.h.ptr() &&
                      PyDict_GetItemWithError(norm.ptr(), k.groups) == p.groups.ptr() &&
                      PyDict_GetItemWithError(move.ptr(), k.bidirectional) == Py_False &&
                      PyObject_RichCompareBool(a[4], p.activation.ptr(), Py_EQ) == 1 && PyObject_IsTrue(a[5]) == p.normed &&
                      x.is_cuda() && x.get_device() == p.device && x.dim() == 3 && x.size(1) == 1 && x.size(0) == p.batch &&
                      x.size(2) == p.dim && x.is_contiguous() && x.scalar_type() != at::kDouble && x.is_floating_point() &&
                      dtype_of(x) == p.dtype && params_match(p, np, 0, 2) && params_match(p, mp, 2, p.params.size());
    if (!same) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.device);
    void* stream = at::cuda::getCurrentCUDAStream((c10::DeviceIndex)p.device).stream();
    // (the default stream cannot be captured; asking takes 0.4 us, a twentieth of a step)
    if (stream && !p.kept && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) keep_with_state(p);
    auto like = [&] { return Tensor(at::detail::empty_cuda(x.sizes(), x.scalar_type(), x.device(), std::nullopt)); };
    Tensor y = like(), xn = p.normed ? like() : Tensor();
    const auto& o = p.operands;
    const unsigned flags = p.activation.is_none() ? 0u : MEGA_EMA_SILU;
    const auto step = p.cplx ? mega_tsn_cema_step : mega_tsn_ema_step;
    check(step(x.data_ptr(), y.data_ptr(), ptr(xn), p.dtype, (int)p.batch, (int)p.dim, ptr<int64_t>(p.count_t), ptr<int64_t>(p.next_t),
               fptr(p.mean_t), fptr(p.var_t), fptr(o[0]), fptr(o[1]), p.eps, fptr(o[2]), fptr(o[3]), fptr(o[4]), fptr(o[5]), p.ndim,
               (float*)p.h_t.data_ptr(), flags, stream), "tsn_ema_step");
    std::swap(p.count, p.count_next);
    std::swap(p.count_t, p.next_t);
    if (PyDict_SetItem(ns, k.count, p.count.ptr()) != 0) return nullptr;
    PyObject* out = THPVariable_Wrap(std::move(y));
    if (!p.normed) return out;
    PyObject* second = THPVariable_Wrap(std::move(xn));
    PyObject* both = PyTuple_Pack(2, out, second);
    Py_XDECREF(out);
    Py_XDECREF(second);
    return both;
  } catch (py::error_already_set& e) {
    e.restore();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// ------------------------------------------------------------------------------------ single-token step of a block
// Five launches of 3 - 6 us each: through the interpreter and ctypes a step took 31 us of host, more than the device.
//
// A plan belongs to a generation: to its running mean, a tensor that the steps update in place and that the state keeps
// from the first to the last of them.  The block's plans are found by it, so generations that are answered in turn keep
// theirs, and a plan goes, with the buffers of keys and values it holds, when the tensor does.
constexpr int kOwners = 7;
struct BlockPlan {
  mega_block_step_args args;
  PyObject* block;                         // (not owned: the plans live in the block's dictionary)
  py::object owners[kOwners];              // norm, move, then those a step stands for: v_proj, mx_proj, h_proj, attention, positions
  std::vector<std::pair<int, py::object>> names;   // of a parameter: owner (0: the block, 1 ...: the above), key
  std::vector<py::object> params;
  std::vector<Mark> marks;
  py::object submodules[kOwners];          // the owners' keys
  py::object nkey, ekey, akey;
  PyObject* mean;                          // (not owned: the plan goes with it)
  py::object count, count_next, var, h, last_key, last_value;
  Tensor keys, values;
  std::vector<py::object> keep;
  int64_t pos, chunk, batch, dim;
  int device;
  uintptr_t stream;
  at::ScalarType type;
};

std::shared_ptr<BlockPlan> block_plan(py::bytes args, std::vector<py::object> owners, std::vector<std::string> submodules,
                                      std::vector<std::pair<int, std::string>> names, std::vector<py::object> params,
                                      std::vector<py::object> state_keys, std::vector<py::object> state, const Tensor& keys,
                                      const Tensor& values, std::vector<py::object> keep, int64_t chunk, const Tensor& x,
                                      uintptr_t stream) {
  auto p = std::make_shared<BlockPlan>();
  const std::string raw = args;
  if (raw.size() != sizeof p->args || owners.size() != kOwners + 1 || submodules.size() != kOwners) throw py::value_error("block_plan");
  memcpy(&p->args, raw.data(), raw.size());
  auto word = [](const std::string& t) { return py::reinterpret_steal<py::object>(PyUnicode_InternFromString(t.c_str())); };
  p->block = owners[0].ptr();
  for (int i = 0; i < kOwners; ++i) p->owners[i] = owners[i + 1];
  for (int i = 0; i < kOwners; ++i) p->submodules[i] = word(submodules[i]);
  for (auto& n : names) p->names.emplace_back(n.first, word(n.second));
  p->params = std::move(params);
  for (auto& t : p->params) p->marks.emplace_back(THPVariable_Unpack(t.ptr()));
  p->nkey = state_keys[0]; p->ekey = state_keys[1]; p->akey = state_keys[2];
  p->count = state[0]; p->count_next = state[1]; p->mean = state[2].ptr(); p->var = state[3]; p->h = state[4];
  p->last_key = state[5]; p->last_value = state[6];
  p->keys = keys; p->values = values;
  p->keep = std::move(keep);
  p->pos = p->args.pos; p->chunk = chunk;
  p->batch = x.size(0); p->dim = x.size(2); p->device = (int)x.get_device(); p->stream = stream; p->type = x.scalar_type();
  return p;
}

// A block's plans.
struct BlockPlans {
  struct Entry {
    std::shared_ptr<BlockPlan> plan;
    py::object watch;   // weak reference to the mean
  };
  using Map = std::unordered_map<PyObject*, Entry>;
  std::shared_ptr<Map> plans = std::make_shared<Map>();
  py::object nkey;      // the norm's key in a state

  void add(std::shared_ptr<BlockPlan> p) {
    PyObject* const mean = p->mean;
    nkey = p->nkey;
    std::weak_ptr<Map> all = plans;
    py::object watch = py::weakref(mean, py::cpp_function([all, mean](py::handle) {
      if (auto m = all.lock()) m->erase(mean);
    }));
    (*plans)[mean] = Entry{std::move(p), std::move(watch)};
  }
};

py::object dict_of(PyObject* o) { return py::reinterpret_steal<py::object>(PyObject_GenericGetDict(o, nullptr)); }

// (an absent entry and None are the same)
bool holds(PyObject* dict, PyObject* key, PyObject* want) {
  PyObject* v = dict ? PyDict_GetItemWithError(dict, key) : nullptr;
  return (v ? v : Py_None) == want;
}

// whether a dictionary in a module's dictionary is empty
bool empty(PyObject* dict, PyObject* key) {
  PyObject* v = PyDict_GetItemWithError(dict, key);
  return v && PyDict_Check(v) && PyDict_Size(v) == 0;
}

// Whether the plan is one for this block, these inputs and this state.
bool block_matches(const BlockPlan& p, PyObject* blk, PyObject* block_dict, const Tensor& x, PyObject* inc) {
  const Names& k = names();
  if (blk != p.block || p.pos >= p.args.cap) return false;
  PyObject* ns = PyDict_GetItemWithError(inc, p.nkey.ptr());
  PyObject* es = PyDict_GetItemWithError(inc, p.ekey.ptr());
  PyObject* as = PyDict_GetItemWithError(inc, p.akey.ptr());
  if (as == Py_None) as = nullptr;
  if (!ns || !es || !PyDict_Check(ns) || !PyDict_Check(es) || (as && !PyDict_Check(as))) return false;
  if (!holds(ns, k.mean, p.mean) || !holds(ns, k.var, p.var.ptr()) || !holds(ns, k.count, p.count.ptr()) ||
      !holds(es, k.h, p.h.ptr()) || !holds(as, k.key, p.last_key.ptr()) || !holds(as, k.value, p.last_value.ptr()) ||
      !holds(as, k.key_mask, Py_None))
    return false;
  if (!x.is_cuda() || x.get_device() != p.device || x.dim() != 3 || x.size(1) != 1 || x.size(0) != p.batch || x.size(2) != p.dim ||
      x.scalar_type() != p.type || !x.is_contiguous())
    return false;
  PyObject* subs = PyDict_GetItemWithError(block_dict, k.modules);
  if (!subs) return false;
  py::object dicts[kOwners + 1];   // the owners' parameters
  for (int i = 0; i <= kOwners; ++i) {
    if (i && PyDict_GetItemWithError(subs, p.submodules[i - 1].ptr()) != p.owners[i - 1].ptr()) return false;
    const py::object d = i ? dict_of(p.owners[i - 1].ptr()) : py::reinterpret_borrow<py::object>(block_dict);
    dicts[i] = py::reinterpret_borrow<py::object>(d ? PyDict_GetItemWithError(d.ptr(), k.params) : nullptr);
    if (!dicts[i]) return false;
    if (i > 2 && (PyDict_Contains(d.ptr(), k.forward) != 0 || !empty(d.ptr(), k.hooks) || !empty(d.ptr(), k.pre_hooks))) return false;
  }
  for (size_t i = 0; i < p.params.size(); ++i) {
    PyObject* t = PyDict_GetItemWithError(dicts[p.names[i].first].ptr(), p.names[i].second.ptr());
    if (t != p.params[i].ptr() || !p.marks[i].holds(THPVariable_Unpack(t))) return false;
  }
  return true;
}

// block_step(block, x, incremental_state): the output, or None when the block has no plan for this call
PyObject* block_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    if (n != 3) throw py::type_error("block_step takes 3 arguments");
    if (!THPVariable_Check(a[1]) || !PyDict_Check(a[2]) || at::GradMode::is_enabled()) Py_RETURN_NONE;
    const Names& k = names();
    const py::object dict = dict_of(a[0]);
    PyObject* held = dict ? PyDict_GetItemWithError(dict.ptr(), k.block_plan) : nullptr;
    if (!held || held == Py_None) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const auto plans = py::cast<BlockPlans*>(py::handle(held))->plans;
    PyObject* ns = PyDict_GetItemWithError(a[2], py::cast<BlockPlans*>(py::handle(held))->nkey.ptr());
    PyObject* mean = ns && PyDict_Check(ns) ? PyDict_GetItemWithError(ns, k.mean) : nullptr;
    const auto found = plans->find(mean);
    if (found == plans->end()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const std::shared_ptr<BlockPlan> keep_plan = found->second.plan;
    BlockPlan& p = *keep_plan;
    const Tensor& x = THPVariable_Unpack(a[1]);
    if (!block_matches(p, a[0], dict.ptr(), x, a[2])) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.device);
    void* stream = at::cuda::getCurrentCUDAStream((c10::DeviceIndex)p.device).stream();
    if ((uintptr_t)stream != p.stream) Py_RETURN_NONE;
    Tensor out(at::detail::empty_cuda(x.sizes(), x.scalar_type(), x.device(), std::nullopt));
    auto at = [](PyObject* t) { return THPVariable_Unpack(t).data_ptr(); };
    p.args.count = (int64_t*)at(p.count.ptr());
    p.args.count_next = (int64_t*)at(p.count_next.ptr());
    p.args.mean = (float*)at(p.mean);
    p.args.var = (float*)at(p.var.ptr());
    p.args.h = (float*)at(p.h.ptr());
    p.args.x = x.data_ptr();
    p.args.out = out.data_ptr();
    p.args.pos = p.pos;
    check(mega_block_step(&p.args, stream), "block_step");
    std::swap(p.count, p.count_next);   // the counts alternate between two arrays, the step wrote the second one
    if (PyDict_SetItem(PyDict_GetItemWithError(a[2], p.nkey.ptr()), k.count, p.count.ptr()) != 0) return nullptr;
    PyObject* as = PyDict_GetItemWithError(a[2], p.akey.ptr());
    if (!as || as == Py_None) {
      const auto fresh = py::dict();
      if (PyDict_SetItem(a[2], p.akey.ptr(), fresh.ptr()) != 0) return nullptr;
      as = PyDict_GetItemWithError(a[2], p.akey.ptr());
    }
    const int64_t pos = ++p.pos;
    if (p.chunk < 0 || pos % p.chunk != 0) {
      p.last_key = py::reinterpret_steal<py::object>(THPVariable_Wrap(p.keys.narrow(1, 0, pos)));
      p.last_value = py::reinterpret_steal<py::object>(THPVariable_Wrap(p.values.narrow(1, 0, pos)));
      if (PyDict_SetItem(as, k.key, p.last_key.ptr()) != 0 || PyDict_SetItem(as, k.value, p.last_value.ptr()) != 0 ||
          PyDict_SetItem(as, k.key_mask, Py_None) != 0)
        return nullptr;
    } else {   // the chunk is complete: the next token starts another one, in other buffers
      for (PyObject* key : {k.key, k.value, k.key_mask})
        if (PyDict_GetItemWithError(as, key) && PyDict_DelItem(as, key) != 0) return nullptr;
      plans->erase(p.mean);
    }
    return THPVariable_Wrap(std::move(out));
  } catch (py::error_already_set& e) {
    e.restore();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyMethodDef g_raw[] = {{"norm_ema_step", (PyCFunction)(void (*)())norm_ema_step, METH_FASTCALL, nullptr},
                       {"block_step", (PyCFunction)(void (*)())block_step, METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(_mega_host, m) {
  py::class_<StepPlan>(m, "StepPlan")
      .def(py::init(&step_plan))
      .def("__deepcopy__", [](StepPlan&, py::object) { return py::none(); })   // (a copied or pickled layer builds its own)
      .def("__reduce__", [](StepPlan&) {
        return py::make_tuple(py::reinterpret_borrow<py::object>((PyObject*)Py_TYPE(Py_None)), py::tuple());
      });
  py::class_<BlockPlan, std::shared_ptr<BlockPlan>>(m, "BlockPlan").def(py::init(&block_plan));
  py::class_<BlockPlans>(m, "BlockPlans")
      .def(py::init<>())
      .def("add", &BlockPlans::add)
      .def("__len__", [](BlockPlans& b) { return b.plans->size(); })
      .def("__deepcopy__", [](BlockPlans&, py::object) { return py::none(); })
      .def("__reduce__", [](BlockPlans&) {
        return py::make_tuple(py::reinterpret_borrow<py::object>((PyObject*)Py_TYPE(Py_None)), py::tuple());
      });
  PyModule_AddFunctions(m.ptr(), g_raw);
  m.def("set_error", [](py::object e) { g_error = e.release().ptr(); });
  m.def("ema_forward", &ema_forward);
  m.def("ema_train", &ema_train);
  m.def("norm_prepare", &norm_prepare);
  m.def("timestep_norm_fwd", &timestep_norm_fwd);
  m.def("timestep_norm_train", &timestep_norm_train);
  m.def("sequence_norm_fwd", &sequence_norm_fwd);
  m.def("sequence_norm_train", &sequence_norm_train);
  m.def("tsn_ema_forward", &tsn_ema_forward);
  m.def("sqn_ema_forward", &sqn_ema_forward);
  m.def("gate_silu", &gate_silu);
  m.def("gate_mul_silu", &gate_mul_silu);
  m.def("gate_output", &gate_output);
  m.def("gate_qk", &gate_qk);
  m.def("attention_softmax_fwd", &softmax_fwd);
  m.def("gated_recurrence", &gated_recurrence);
  m.def("gated_recurrence_step", &gated_recurrence_step);
  m.def("gated_recurrence_train", &gated_recurrence_train);
  m.def("gated_recurrence_packed", &gated_recurrence_packed);
  m.def("decayed_attention", &decayed_attention);
  m.def("decayed_attention_step", &decayed_attention_step);
  m.def("decayed_attention_train", &decayed_attention_train);
  m.def("decayed_attention_packed", &decayed_attention_packed);
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_train", &rms_norm_train);
  m.def("group_norm", &group_norm);
  m.def("group_norm_fwd", &group_norm_fwd);
  m.def("group_norm_train", &group_norm_train);
  m.def("block_train", &block_train);
  m.def("block_infer", &block_infer);
}
