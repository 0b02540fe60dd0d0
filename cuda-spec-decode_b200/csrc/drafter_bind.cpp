// torch binding of the drafter's long-context operators: checks of arguments,
// outputs, streams and autograd around the C ABI (include/specdec.h).
//
// The other entry points are called from Python through ctypes. These are the
// layer's innermost calls, a few microseconds of GPU work each at the drafter's
// sizes, and there the host decides: with the same steps in Python a forward
// and backward of the norm with rotation on a [32, 528, 4 + 4, 64] batch took
// the host 146 us (GPU 51 us), of which torch's own engine needs 48. Here the
// backward also runs without the interpreter.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <array>
#include <cstdint>
#include <limits>
#include <map>
#include <mutex>
#include <optional>
#include <string>

#include "specdec.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// The reference's exception types, as specdec._lib.check raises them: contract
// violations AssertionError, values out of domain ValueError.
[[noreturn]] void raise(PyObject* type, const std::string& msg) {
  py::gil_scoped_acquire gil;
  PyErr_SetString(type, msg.c_str());
  throw py::error_already_set();
}
void require(bool ok, const char* msg) {
  if (!ok) raise(PyExc_AssertionError, msg);
}
void check(int code, const char* what) {
  if (code == SPECDEC_OK) return;
  std::string msg = specdec_last_error();
  if (msg.empty()) msg = specdec_status_string(code);
  if (code == SPECDEC_ERR_ARGUMENT) raise(PyExc_AssertionError, msg);
  if (code == SPECDEC_ERR_VALUE || code == SPECDEC_ERR_TARGET_RANGE) raise(PyExc_ValueError, msg);
  raise(PyExc_RuntimeError, std::string(what) + ": " + msg);
}

// A size as the C ABI takes it.
int32_t i32(int64_t n) {
  require(n >= std::numeric_limits<int32_t>::min() && n <= std::numeric_limits<int32_t>::max(), "sizes must fit in int32");
  return (int32_t)n;
}

// Everything below runs with the tensors' device current, on its current stream.
struct On {
  c10::cuda::CUDAGuard guard;
  cudaStream_t stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// The stream's sticky drafter status word (specdec._lib.status_words): Python
// makes it once per device and stream and keeps it for the life of the process.
int32_t* status_word(const Tensor& t, cudaStream_t stream) {
  static std::mutex mu;
  static std::map<std::pair<int, cudaStream_t>, int32_t*> words;
  const std::pair<int, cudaStream_t> key(t.device().index(), stream);
  {
    std::lock_guard<std::mutex> lock(mu);
    const auto it = words.find(key);
    if (it != words.end()) return it->second;
  }
  int32_t* p;
  {
    py::gil_scoped_acquire gil;
    p = reinterpret_cast<int32_t*>(py::module_::import("specdec.drafter").attr("_status")(t.device()).cast<uintptr_t>());
  }
  std::lock_guard<std::mutex> lock(mu);
  words[key] = p;
  return p;
}

int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? SPECDEC_DTYPE_BF16 : SPECDEC_DTYPE_F32; }

// The C ABI's three element strides; null for a contiguous tensor.
struct Strides {
  std::array<int64_t, 3> s;
  const int64_t* p = nullptr;
  explicit Strides(const Tensor& t) {
    if (t.is_contiguous()) return;
    s = {t.stride(0), t.stride(1), t.stride(2)};
    p = s.data();
  }
};

Tensor heads_contiguous(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

// t itself if every row of a head starts on a 16-byte boundary, else a copy.
Tensor rows16(const Tensor& t) {
  bool ok = reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 && t.stride(3) == 1;
  for (int d = 0; d < 3; ++d) ok = ok && (t.stride(d) % 8 == 0 || t.size(d) <= 1);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)); }
Tensor bytes(size_t n, const Tensor& on) {
  return n ? at::empty({(int64_t)n}, on.options().dtype(at::kByte)) : Tensor();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// A backward's results when a graph of the backward is being built: there is no
// second derivative, and asking for one raises.
variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice a function that has no second derivative: ") + name,
      static_cast<int>(grads.size()));
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  return (*error)(std::move(grads));
}

// Forward mode: the kernels compute no tangents. A dual tensor does not require
// a gradient, so without this check its tangent would be lost without a word.
// Raises as torch.autograd.Function (the other operators) does.
template <class... T>
void refuse_tangents(const char* name, const T&... inputs) {
  if ((... || inputs._fw_grad(0).defined()))
    raise(PyExc_NotImplementedError, std::string(name) + " has no forward-mode derivative");
}

// ---- rotary positions, norms of queries and keys ------------------------------

struct Turn {  // how to turn: positions, frequencies, layout, factor
  Tensor positions, inv_freq;
  bool interleaved;
  double scale;
  int64_t pos_stride() const { return positions.dim() == 2 ? positions.stride(0) : 0; }
  int32_t dim() const { return (int32_t)(2 * inv_freq.numel()); }
};

void check_heads(const char* name, const Tensor& x, const Tensor* q) {
  const auto t = x.scalar_type();
  if (!(x.is_cuda() && x.dim() == 4 && (t == at::kFloat || t == at::kBFloat16)))
    raise(PyExc_AssertionError, std::string(name) + " must be cuda float32 or bfloat16 [B, T, heads, D]");
  if (q && !(x.device() == q->device() && t == q->scalar_type() && x.size(0) == q->size(0) && x.size(1) == q->size(1) &&
             x.size(3) == q->size(3)))
    raise(PyExc_AssertionError, std::string(name) + " must match q's device, dtype, batch, length and head size");
}

Turn check_turn(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, bool interleaved, double scale) {
  const auto t = positions.scalar_type();
  const bool each = positions.dim() == 2 && positions.size(0) == x.size(0) && positions.size(1) == x.size(1);
  const bool shared = positions.dim() == 1 && positions.size(0) == x.size(1);
  require(positions.device() == x.device() && (t == at::kLong || t == at::kInt) && (each || shared),
          "positions must be int64 (or int32) [T] or [B, T] on the heads' device");
  require(inv_freq.device() == x.device() && inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1,
          "inv_freq must be float64 [rotary_dim / 2] on the heads' device");
  require(inv_freq.numel() > 0 && 2 * inv_freq.numel() <= x.size(3),
          "inv_freq must turn at least one pair and at most the head");
  Tensor p = t == at::kLong ? positions : positions.to(at::kLong);
  if (p.size(-1) > 1 && p.stride(-1) != 1) p = p.contiguous();
  return {p, inv_freq.contiguous(), interleaved, scale};
}

Tensor rotary_run(const Tensor& given, const Turn& how, bool inverse) {
  const Tensor x = heads_contiguous(given);
  const On on(x);
  Tensor y = like(x);
  const Strides xs(x);
  check(specdec_rotary(x.const_data_ptr(), xs.p, y.data_ptr(), how.positions.const_data_ptr<int64_t>(), how.pos_stride(),
                       how.inv_freq.const_data_ptr<double>(), i32(x.size(0)), i32(x.size(1)), i32(x.size(2)), i32(x.size(3)),
                       how.dim(), how.interleaved, (float)how.scale, inverse, dtype_of(x), on.stream),
        "specdec_rotary");
  return y;
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const Tensor& inv_freq,
                        bool interleaved, double scale) {
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["scale"] = scale;
    return rotary_run(x, {positions, inv_freq, interleaved, scale}, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    Tensor dx;
    if (g[0].defined()) {
      refuse_tangents("the gradient of rotary", g[0]);
      dx = rotary_run(g[0], {saved[0], saved[1], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["scale"].toDouble()},
                      true);
    }
    return once({dx, Tensor(), Tensor(), Tensor(), Tensor()}, "rotary");
  }
};

Tensor rotary(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, bool interleaved, double scale) {
  check_heads("x", x, nullptr);
  refuse_tangents("rotary", x, inv_freq);
  const Turn how = check_turn(x, positions, inv_freq, interleaved, scale);
  if (at::GradMode::is_enabled() && x.requires_grad())
    return RotaryFn::apply(x, how.positions, how.inv_freq, interleaved, scale);
  return rotary_run(x, how, false);
}

Tensor fp32_weight(const Tensor& w) { return w.to(at::kFloat).contiguous(); }

std::array<Tensor, 2> norm_run(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Turn& how,
                               double eps) {
  const On on(q);
  Tensor yq = like(q), yk = like(k);
  const Strides qs(q), ks(k);
  check(specdec_qk_norm_rotary_forward(q.const_data_ptr(), qs.p, k.const_data_ptr(), ks.p, wq.const_data_ptr<float>(),
                                       wk.const_data_ptr<float>(), yq.data_ptr(), yk.data_ptr(),
                                       how.positions.const_data_ptr<int64_t>(), how.pos_stride(),
                                       how.inv_freq.const_data_ptr<double>(), i32(q.size(0)), i32(q.size(1)),
                                       i32(q.size(2)), i32(k.size(2)), i32(q.size(3)), how.dim(), how.interleaved, (float)how.scale, (float)eps, dtype_of(q),
                                       on.stream),
        "specdec_qk_norm_rotary_forward");
  return {yq, yk};
}

struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& q_weight,
                               const Tensor& k_weight, const Tensor& positions, const Tensor& inv_freq, double eps,
                               bool interleaved, double scale) {
    const Tensor q = heads_contiguous(q_in), k = heads_contiguous(k_in);
    const Tensor wq = fp32_weight(q_weight), wk = fp32_weight(k_weight);
    ctx->save_for_backward({q, k, wq, wk, positions, inv_freq});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["tq"] = (int64_t)q_weight.scalar_type();
    ctx->saved_data["tk"] = (int64_t)k_weight.scalar_type();
    const auto y = norm_run(q, k, wq, wk, {positions, inv_freq, interleaved, scale}, eps);
    return {y[0], y[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &wq = saved[2], &wk = saved[3];
    const Turn how{saved[4], saved[5], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["scale"].toDouble()};
    const On on(q);
    for (const Tensor& t : g)
      if (t.defined()) refuse_tangents("the gradient of qk_norm_rotary", t);
    // an output that nothing depends on brings no gradient: zeros
    const Tensor dyq = g[0].defined() ? heads_contiguous(g[0]) : at::zeros_like(q);
    const Tensor dyk = g[1].defined() ? heads_contiguous(g[1]) : at::zeros_like(k);
    Tensor dq = like(q), dk = like(k), dwq = like(wq), dwk = like(wk);
    const size_t n = specdec_qk_norm_rotary_workspace_bytes(q.size(0), q.size(1), q.size(3), q.device().index());
    const Tensor ws = bytes(n, q);
    const Strides qs(q), ks(k), dqs(dyq), dks(dyk);
    check(specdec_qk_norm_rotary_backward(
              q.const_data_ptr(), qs.p, k.const_data_ptr(), ks.p, wq.const_data_ptr<float>(), wk.const_data_ptr<float>(),
              dyq.const_data_ptr(), dqs.p, dyk.const_data_ptr(), dks.p, dq.data_ptr(), dk.data_ptr(), dwq.data_ptr<float>(),
              dwk.data_ptr<float>(), how.positions.const_data_ptr<int64_t>(), how.pos_stride(),
              how.inv_freq.const_data_ptr<double>(), q.size(0), q.size(1), q.size(2), k.size(2), q.size(3), how.dim(),
              how.interleaved, (float)how.scale, (float)ctx->saved_data["eps"].toDouble(), dtype_of(q), ptr(ws), n, on.stream),
          "specdec_qk_norm_rotary_backward");
    return once({dq, dk, dwq.to((at::ScalarType)ctx->saved_data["tq"].toInt()),
                 dwk.to((at::ScalarType)ctx->saved_data["tk"].toInt()), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()},
                "qk_norm_rotary");
  }
};

std::tuple<Tensor, Tensor> qk_norm_rotary(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                          const Tensor& positions, const Tensor& inv_freq, std::optional<double> eps,
                                          bool interleaved, double scale) {
  check_heads("q", q, nullptr);
  check_heads("k", k, &q);
  const int64_t D = q.size(3);
  require(q_weight.dim() == 1 && q_weight.size(0) == D && k_weight.dim() == 1 && k_weight.size(0) == D &&
              q_weight.device() == q.device() && k_weight.device() == q.device(),
          "weights must be [D] on q's device");
  refuse_tangents("qk_norm_rotary", q, k, q_weight, k_weight, inv_freq);
  const Turn how = check_turn(q, positions, inv_freq, interleaved, scale);
  // as torch's rms_norm, which takes fp32's for bf16 inputs too
  const double e = eps ? *eps : (double)std::numeric_limits<float>::epsilon();
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || q_weight.requires_grad() || k_weight.requires_grad())) {
    const auto y = NormFn::apply(q, k, q_weight, k_weight, how.positions, how.inv_freq, e, interleaved, scale);
    return {y[0], y[1]};
  }
  const auto y = norm_run(heads_contiguous(q), heads_contiguous(k), fp32_weight(q_weight), fp32_weight(k_weight), how, e);
  return {y[0], y[1]};
}

// ---- sliding-window attention ---------------------------------------------------

constexpr int64_t kNoWindow = std::numeric_limits<int32_t>::max();

struct Window {
  int64_t window, sinks;
  double scale;
};

Window check_window(const Tensor& q, const Tensor& k, const Tensor& v, std::optional<int64_t> window, int64_t sinks,
                    std::optional<double> scale) {
  require(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 4, "q must be cuda bfloat16 [B, T, heads, D]");
  require(q.size(3) == 64 || q.size(3) == 128, "heads must have 64 or 128 elements");
  require(k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3),
          "k and v must be [B, T, k_heads, D] with q's batch and head size");
  require(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.device() == q.device() &&
              v.device() == q.device(),
          "k and v must have q's dtype and device");
  require(k.size(2) > 0 && q.size(2) > 0 && q.size(2) % k.size(2) == 0, "query heads must be a multiple of key heads");
  require(!window || *window >= 1, "window must be >= 1 or None");
  require(sinks >= 0, "sinks must be >= 0");
  return {window ? std::min(*window, kNoWindow) : kNoWindow, std::min(sinks, kNoWindow),
          scale ? *scale : 1.0 / std::sqrt((double)q.size(3))};
}

Tensor check_lens(const Tensor& lens, const Tensor& q) {
  require(lens.dim() == 1 && lens.size(0) == q.size(0) && (lens.scalar_type() == at::kInt || lens.scalar_type() == at::kLong) &&
              lens.device() == q.device(),
          "ctx_lens must be int32 (or int64) [B] on q's device");
  return (lens.scalar_type() == at::kInt ? lens : lens.clamp(0, kNoWindow).to(at::kInt)).contiguous();
}

const int32_t* lens_ptr(const Tensor& lens) { return lens.defined() ? lens.const_data_ptr<int32_t>() : nullptr; }
const uint16_t* bits(const Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
uint16_t* out_bits(const Tensor& t) { return static_cast<uint16_t*>(ptr(t)); }

// o; with `train` also the residual of its rounding and the log-sum-exp.
std::array<Tensor, 3> window_run(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lens, int64_t n_ctx,
                                 const Window& w, bool train) {
  const On on(q);
  Tensor o = like(q), res, lse;
  if (train) {
    res = like(q);
    lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  }
  const Strides qs(q), ks(k), vs(v);
  check(specdec_window_attention_forward(bits(q), qs.p, bits(k), ks.p, bits(v), vs.p, out_bits(o), out_bits(res),
                                         static_cast<float*>(ptr(lse)), lens_ptr(lens), i32(q.size(0)), i32(q.size(1)),
                                         i32(q.size(2)), i32(k.size(2)), i32(q.size(3)), n_ctx, w.window, w.sinks, (float)w.scale,
                                         status_word(q, on.stream), on.stream),
        "specdec_window_attention_forward");
  return {o, res, lse};
}

struct WindowFn : torch::autograd::Function<WindowFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                        const std::optional<Tensor>& ctx_lens, int64_t n_ctx, int64_t window, int64_t sinks,
                        double scale) {
    const Tensor q = rows16(q_in), k = rows16(k_in), v = rows16(v_in), lens = ctx_lens ? *ctx_lens : Tensor();
    const auto r = window_run(q, k, v, lens, n_ctx, {window, sinks, scale}, true);
    ctx->save_for_backward({q, k, v, r[0], r[1], r[2], lens});
    ctx->saved_data["n_ctx"] = n_ctx;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &lens = saved[6];
    Tensor dq, dk, dv;
    if (g[0].defined()) {
      refuse_tangents("the gradient of window_attention", g[0]);
      const On on(q);
      Tensor dout = g[0].contiguous();
      if (reinterpret_cast<uintptr_t>(dout.const_data_ptr()) % 16) dout = dout.clone();
      dq = like(q), dk = like(k), dv = like(v);
      const int64_t n_ctx = ctx->saved_data["n_ctx"].toInt(), window = ctx->saved_data["window"].toInt(),
                    sinks = ctx->saved_data["sinks"].toInt();
      const size_t n = specdec_window_attention_workspace_bytes(q.size(0), q.size(1), q.size(2), k.size(2), q.size(3), n_ctx,
                                                                window, sinks, q.device().index());
      const Tensor ws = bytes(n, q);
      const Strides qs(q), ks(k), vs(v);
      check(specdec_window_attention_backward(
                bits(q), qs.p, bits(k), ks.p, bits(v), vs.p, bits(saved[3]), bits(saved[4]), saved[5].const_data_ptr<float>(),
                bits(dout), out_bits(dq), out_bits(dk), out_bits(dv), lens_ptr(lens), q.size(0), q.size(1), q.size(2),
                k.size(2), q.size(3), n_ctx, window, sinks, (float)ctx->saved_data["scale"].toDouble(),
                status_word(q, on.stream), ptr(ws), n, on.stream),
            "specdec_window_attention_backward");
    }
    return once({dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, "window_attention");
  }
};

Tensor window_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t n_ctx, std::optional<int64_t> window,
                        int64_t sinks, std::optional<double> scale, const std::optional<Tensor>& ctx_lens) {
  const Window w = check_window(q, k, v, window, sinks, scale);
  require(k.size(1) == q.size(1), "k and v must have q's length");
  require(n_ctx >= 0 && n_ctx <= q.size(1), "n_ctx must be in [0, T]");
  refuse_tangents("window_attention", q, k, v);
  std::optional<Tensor> lens;
  if (ctx_lens) lens = check_lens(*ctx_lens, q);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return WindowFn::apply(q, k, v, lens, n_ctx, w.window, w.sinks, w.scale);
  return window_run(rows16(q), rows16(k), rows16(v), lens ? *lens : Tensor(), n_ctx, w, false)[0];
}

Tensor window_attention_cached(const Tensor& q_in, const Tensor& k_cache, const Tensor& v_cache, const Tensor& ctx_lens,
                               int64_t n_block, std::optional<int64_t> window, int64_t sinks, std::optional<double> scale) {
  const Window w = check_window(q_in, k_cache, v_cache, window, sinks, scale);
  require(!(at::GradMode::is_enabled() && (q_in.requires_grad() || k_cache.requires_grad() || v_cache.requires_grad())),
          "window_attention_cached has no backward: call it under torch.no_grad()");
  refuse_tangents("window_attention_cached", q_in, k_cache, v_cache);
  const Tensor lens = check_lens(ctx_lens, q_in);
  require(k_cache.stride(3) == 1 && v_cache.stride(3) == 1, "the cache's heads must be contiguous");
  const int32_t B = i32(q_in.size(0)), Tq = i32(q_in.size(1)), Hq = i32(q_in.size(2)), D = i32(q_in.size(3)),
                size = i32(k_cache.size(1)), Hk = i32(k_cache.size(2));
  require(n_block >= 0 && n_block <= size, "n_block must be in [0, size of the cache]");
  const Tensor q = rows16(q_in);
  const On on(q);
  Tensor o = like(q);
  const size_t n = specdec_window_attention_cached_workspace_bytes(B, Tq, size, Hq, Hk, D, n_block, w.window, w.sinks,
                                                                   q.device().index());
  const Tensor ws = bytes(n, q);
  const Strides qs(q), ks(k_cache), vs(v_cache);
  check(specdec_window_attention_cached(bits(q), qs.p, bits(k_cache), ks.p, bits(v_cache), vs.p, out_bits(o),
                                        lens_ptr(lens), B, Tq, size, Hq, Hk, D, n_block, w.window, w.sinks, (float)w.scale,
                                        status_word(q, on.stream), ptr(ws), n, on.stream),
        "specdec_window_attention_cached");
  return o;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("rotary", &rotary);
  m.def("qk_norm_rotary", &qk_norm_rotary);
  m.def("window_attention", &window_attention);
  m.def("window_attention_cached", &window_attention_cached);
}
