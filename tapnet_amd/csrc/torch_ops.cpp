// tapnet_amd.attention's operators on torch tensors: argument checks, memory from torch's allocator, autograd nodes, and the calls
// into libtapir_hip's C ABI (include/tapir_hip.h).  Host code only.  It is C++ because the operators' small calls are bound by the
// host: a layer norm of one frame's tokens with its gradients took 152 us a call through Python's autograd functions and ctypes,
// of which the kernels need a fifth.
#include <ATen/DeviceGuard.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cmath>
#include <mutex>
#include <optional>
#include <string>
#include <vector>

#include "../../include/tapir_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------------------------------------------------------ contexts
// One context per device and element type: it holds no weights and no workspaces, only the last error's text.  Contexts are not
// thread-safe: calls take turns (they only enqueue).  They live as long as the process.
constexpr int kMaxDevices = 64;
std::mutex g_lock;
tapir_ctx* g_ctx[kMaxDevices][2];

hipStream_t current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

tapir_ctx* context(const Tensor& like, hipStream_t stream) {   // (under g_lock)
  const int dev = like.device().index(), dtype = like.scalar_type() == at::kBFloat16 ? TAPIR_BF16 : TAPIR_F32;
  TORCH_CHECK(dev >= 0 && dev < kMaxDevices, "device index ", dev);
  tapir_ctx*& c = g_ctx[dev][dtype == TAPIR_BF16];
  if (c == nullptr) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    TORCH_CHECK(hipStreamIsCapturing(stream, &status) == hipSuccess && status == hipStreamCaptureStatusNone,
                "call the operator once before capturing it into a graph (the first call prepares the library)");
    tapir_cfg cfg{};
    cfg.pyramid_level = 1;
    cfg.num_pips_iter = 4;
    cfg.num_mixer_blocks = 12;
    cfg.softmax_temperature = 20.f;
    cfg.initial_h = cfg.initial_w = 256;
    cfg.dtype = dtype;
    const int rc = tapir_create(&c, &cfg, dev);
    if (rc != TAPIR_OK) c = nullptr;
    TORCH_CHECK(rc == TAPIR_OK, "tapir_create failed (", rc, ")");
  }
  return c;
}

// fn(context, stream) on the current stream of `like`'s device; a refusal becomes a ValueError, anything else a RuntimeError
template <class Fn> void call(const Tensor& like, const char* name, Fn&& fn) {
  const hipStream_t stream = current_stream(like);
  std::lock_guard<std::mutex> guard(g_lock);
  tapir_ctx* c = context(like, stream);
  const int rc = fn(c, stream);
  if (rc == TAPIR_OK) return;
  const std::string text = std::string(name) + " failed (" + std::to_string(rc) + "): " + tapir_last_error(c);
  TORCH_CHECK_VALUE(rc != TAPIR_ERR_INVALID && rc != TAPIR_ERR_UNSUPPORTED, text);
  TORCH_CHECK(false, text);
}

// ---------------------------------------------------------------------------------------------------------- arguments
void check_input(const char* name, const Tensor& t) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name, " has to be float32 or bfloat16, not ",
                    t.scalar_type());
  TORCH_CHECK_VALUE(t.device().is_cuda(), name, " has to be on the GPU: tapnet_amd has no CPU fallback");
  TORCH_CHECK_VALUE(t.layout() == at::kStrided, name, " has to be a dense tensor");
}

void check_beside(const char* name, const Tensor& t, const Tensor& like, at::ScalarType type) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", the input on ", like.device());
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, " has to be ", type, ", not ", t.scalar_type());
  TORCH_CHECK_VALUE(t.layout() == at::kStrided, name, " has to be a dense tensor");
}

void check_axes(const char* name, const Tensor& t, int64_t n) {
  TORCH_CHECK_VALUE(t.dim() == n, name, " has to have ", n, " axes, not ", t.dim());
}

// (ZeroTensors and lazily negated or conjugated views hold no such values in memory)
Tensor plain(const Tensor& t) { return t._is_zerotensor() ? t.clone() : t.is_neg() ? t.resolve_neg() : t; }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor option(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }   // (autograd takes no undefined tensor)
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

Tensor workspace(uint64_t bytes, const Tensor& like) {
  return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

// Gradients are not differentiable again: asked for a second derivative, the node behind them says so.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g.set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "the operators of tapnet_amd.attention have no second derivative", static_cast<int64_t>(grads.size()));
  return (*node)(std::move(grads));
}

// ---------------------------------------------------------------------------------------------------------- layer norm
struct Rows {   // a tensor as [rows, channels] with dense channels and one row stride; t keeps the memory alive
  Tensor t;
  int64_t rows, stride;
};

Rows as_rows(const Tensor& in) {
  Tensor t = plain(in);
  const int64_t channels = t.size(-1);
  const int64_t rows = t.numel() / channels;
  if (t.is_contiguous()) return {t, rows, channels};
  if (channels == 1 || t.stride(-1) == 1) {
    int64_t stride = channels, span = 0;   // span: what the next axis outwards has to step by
    bool one = true;
    for (int64_t d = t.dim() - 2; d >= 0 && one; --d) {
      if (t.size(d) == 1) continue;
      if (span == 0) stride = t.stride(d);
      else one = t.stride(d) == span;
      span = t.stride(d) * t.size(d);
      if (t.stride(d) == 0) span = -1;     // (a broadcast axis: nothing outwards of it joins in)
    }
    if (one) return {t, rows, stride};
  }
  return {t.contiguous(), rows, channels};
}

struct Normed { Tensor y, stats; };   // stats [2, rows]: mean, 1 / deviation

Normed norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, bool train) {
  const at::DeviceGuard guard(x.device());
  const Rows r = as_rows(x);
  Normed out{at::empty(x.sizes(), x.options()), train ? at::empty({2, r.rows}, x.options().dtype(at::kFloat)) : Tensor()};
  float* const mean = fptr(out.stats);
  call(x, "layer_norm", [&](tapir_ctx* c, hipStream_t s) {
    return tapir_layer_norm(c, ptr(r.t), r.stride, fptr(weight), fptr(bias), ptr(out.y), mean, mean ? mean + r.rows : nullptr, r.rows,
                            static_cast<int>(x.size(-1)), static_cast<float>(eps), s);
  });
  return out;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    Normed out = norm_forward(x, value(weight), value(bias), eps, true);
    ctx->save_for_backward({x, value(weight), out.stats});
    ctx->saved_data["bias"] = bias.has_value();
    return out.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
    const Tensor& dy = grads[0];
    variable_list out(4);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const at::DeviceGuard guard(x.device());
      const Rows r = as_rows(x), g = as_rows(dy);
      const int channels = static_cast<int>(x.size(-1));
      const auto f32 = x.options().dtype(at::kFloat);
      // (the node's edges are those of the tensors that were given)
      const bool has_weight = weight.defined(), has_bias = ctx->saved_data["bias"].toBool();
      if (ctx->needs_input_grad(0)) out[0] = at::empty(x.sizes(), x.options());
      if (has_weight && ctx->needs_input_grad(1)) out[1] = at::empty({channels}, f32);
      if (has_bias && ctx->needs_input_grad(1 + has_weight)) out[2] = at::empty({channels}, f32);
      uint64_t bytes = 0;
      if (out[1].defined() || out[2].defined())
        call(x, "layer_norm", [&](tapir_ctx* c, hipStream_t) { return tapir_layer_norm_workspace(c, r.rows, channels, &bytes); });
      const Tensor work = workspace(bytes, x);
      const float* mean = fptr(stats);
      call(x, "layer_norm", [&](tapir_ctx* c, hipStream_t s) {
        return tapir_layer_norm_backward(c, ptr(r.t), r.stride, ptr(g.t), g.stride, fptr(weight), mean, mean + r.rows, ptr(out[0]),
                                         fptr(out[1]), fptr(out[2]), r.rows, channels, ptr(work), bytes, s);
      });
    }
    return once(std::move(out));
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight_, const OptTensor& bias_, double eps) {
  Tensor weight = value(weight_), bias = value(bias_);
  check_input("x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x has to have a last axis of at least one channel");
  TORCH_CHECK_VALUE(x.size(-1) < (int64_t{1} << 31), "x has too many channels");
  for (auto& [name, p] : {std::pair<const char*, Tensor&>("weight", weight), std::pair<const char*, Tensor&>("bias", bias)}) {
    if (!p.defined()) continue;
    check_beside(name, p, x, at::kFloat);
    TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == x.size(-1), name, " has to be float32 [", x.size(-1), "], not ", p.sizes());
    p = plain(p).contiguous();
  }
  TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "eps has to be finite and not negative, not ", eps);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return LayerNorm::apply(x, option(weight), option(bias), eps);
  return norm_forward(x, weight, bias, eps, false).y;
}

// ---------------------------------------------------------------------------------------------------- rotary positions
struct Turn {
  std::vector<int64_t> sections;
  std::vector<double> bases;
  bool interleaved;
};

Tensor turn(const Tensor& in, const Tensor& positions, const Turn& how, bool inverse) {
  const at::DeviceGuard guard(in.device());
  Tensor x = plain(in);
  if (x.size(3) > 1 && x.stride(3) != 1) x = x.contiguous();
  Tensor y = at::empty(x.sizes(), x.options());
  const int axes = static_cast<int>(how.sections.size());
  tapir_rotary_args a{};
  a.batch = x.size(0);
  a.tokens = x.size(1);
  a.heads = static_cast<int>(x.size(2));
  a.dim = static_cast<int>(x.size(3));
  a.axes = axes;
  a.interleaved = how.interleaved;
  a.inverse = inverse;
  for (int i = 0; i < axes; ++i) {
    a.section[i] = static_cast<int>(how.sections[i]);
    a.base[i] = how.bases[i];
  }
  a.x = ptr(x);
  for (int i = 0; i < 3; ++i) a.x_stride[i] = x.stride(i);
  a.positions = fptr(positions);
  a.positions_stride = positions.dim() == 3 && positions.size(0) > 1 ? a.tokens * axes : 0;
  a.y = ptr(y);
  if (x.numel() == 0) return y;
  call(x, "rotary_positions", [&](tapir_ctx* c, hipStream_t s) { return tapir_rotary_positions(c, &a, s); });
  return y;
}

struct Rotary : torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const std::vector<int64_t>& sections,
                        const std::vector<double>& bases, bool interleaved) {
    ctx->save_for_backward({positions});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["bases"] = bases;
    ctx->saved_data["interleaved"] = interleaved;
    return turn(x, positions, {sections, bases, interleaved}, false);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      out[0] = turn(grads[0], ctx->get_saved_variables()[0],
                    {ctx->saved_data["sections"].toIntVector(), ctx->saved_data["bases"].toDoubleVector(),
                     ctx->saved_data["interleaved"].toBool()}, true);
    }
    return once(std::move(out));
  }
};

Tensor rotary_positions(const Tensor& x, const Tensor& positions_, const std::optional<std::vector<int64_t>>& sections_,
                        std::vector<double> bases, bool interleaved) {
  check_input("x", x);
  check_axes("x", x, 4);
  check_beside("positions", positions_, x, at::kFloat);
  const int64_t batch = x.size(0), tokens = x.size(1), dim = x.size(3);
  const Tensor& p = positions_;
  TORCH_CHECK_VALUE((p.dim() == 2 || p.dim() == 3) && p.size(-2) == tokens && (p.dim() == 2 || p.size(0) == 1 || p.size(0) == batch),
                    "positions have to be [", batch, ", ", tokens, ", axes] or [", tokens, ", axes], not ", p.sizes());
  TORCH_CHECK_VALUE(!p.requires_grad(), "positions have no gradient: detach them");
  const int64_t axes = p.size(-1);
  TORCH_CHECK_VALUE(axes >= 1 && axes <= 4, "1 to 4 axes of positions, not ", axes);
  TORCH_CHECK_VALUE(dim >= 1 && dim <= 256 && x.size(2) >= 1 && x.size(2) < (int64_t{1} << 31),
                    "x has to have heads of 1 to 256 channels, not ", x.sizes());
  std::vector<int64_t> sections;
  if (sections_.has_value()) {
    sections = *sections_;
  } else {
    const int64_t pairs = dim / 2;
    for (int64_t a = 0; a < axes; ++a) sections.push_back(2 * (pairs / axes + (a < pairs % axes)));
  }
  int64_t sum = 0;
  bool good = static_cast<int64_t>(sections.size()) == axes;
  for (int64_t s : sections) {
    good = good && s >= 0 && s % 2 == 0 && s <= dim;
    sum += good ? s : 0;
  }
  TORCH_CHECK_VALUE(good && sum <= dim, "sections ", sections, ": ", axes, " even channel counts are wanted, at most ", dim, " together");
  if (bases.size() == 1) bases.resize(axes, bases[0]);
  good = static_cast<int64_t>(bases.size()) == axes;
  for (double b : bases) good = good && b > 0 && std::isfinite(b);
  TORCH_CHECK_VALUE(good, "base ", bases, ": one positive number, or one per axis");
  const Tensor positions = plain(p).contiguous();
  if (at::GradMode::is_enabled() && x.requires_grad()) return Rotary::apply(x, positions, sections, bases, interleaved);
  return turn(x, positions, {sections, bases, interleaved}, false);
}

// ----------------------------------------------------------------------------------------------------- cross attention
// `t` itself where its rows (last axis) are dense, start at multiples of 16 bytes and are less than 2^22 elements apart, else a
// dense copy.  An axis of one element has no stride (torch calls such a tensor contiguous whatever number stands there).
Tensor aligned(const Tensor& in) {
  Tensor t = plain(in);
  const int64_t epc = 16 / static_cast<int64_t>(t.element_size());
  bool good = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) good = good && (t.size(d) <= 1 || t.stride(d) % epc == 0);
  good = good && (t.size(1) <= 1 || t.stride(1) < (int64_t{1} << 22));
  if (good) return t;
  t = t.contiguous();
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

tapir_attn_args attn_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Tensor& mask, double scale) {
  tapir_attn_args a{};
  a.batch = q.size(0);
  a.queries = q.size(1);
  a.keys = k.size(1);
  a.heads = static_cast<int>(q.size(2));
  a.kv_heads = static_cast<int>(k.size(2));
  a.dim = static_cast<int>(q.size(3));
  a.scale = static_cast<float>(scale);
  a.q = ptr(q);
  a.k = ptr(k);
  a.v = ptr(v);
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = q.stride(i);
    a.k_stride[i] = k.stride(i);
    a.v_stride[i] = v.stride(i);
  }
  a.key_lengths = static_cast<const int32_t*>(ptr(lengths));
  a.key_mask = static_cast<const uint8_t*>(ptr(mask));
  return a;
}

Tensor attn_workspace(const Tensor& like, tapir_attn_args& a, bool backward) {
  uint64_t bytes = 0;
  call(like, "cross_attention", [&](tapir_ctx* c, hipStream_t) { return tapir_cross_attention_workspace(c, &a, backward, &bytes); });
  Tensor work = workspace(bytes, like);
  a.workspace = ptr(work);
  a.workspace_bytes = bytes;
  return work;
}

struct Attended { Tensor q, k, v, out, out32, stats; };

Attended attn_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Tensor& mask, double scale,
                      bool train) {
  const at::DeviceGuard guard(q.device());
  Attended r{aligned(q), aligned(k), aligned(v), at::empty(q.sizes(), q.options()), Tensor(), Tensor()};
  tapir_attn_args a = attn_args(r.q, r.k, r.v, lengths, mask, scale);
  a.out = ptr(r.out);
  if (train) {
    const auto f32 = q.options().dtype(at::kFloat);
    r.out32 = q.scalar_type() == at::kFloat ? r.out : at::empty(q.sizes(), f32);
    r.stats = at::empty({q.size(0), q.size(1) * q.size(2), 2}, f32);
    a.out_f32 = fptr(r.out32);
    a.stats = fptr(r.stats);
  }
  const Tensor work = attn_workspace(q, a, false);
  call(q, "cross_attention", [&](tapir_ctx* c, hipStream_t s) { return tapir_cross_attention(c, &a, s); });
  return r;
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths_,
                        const OptTensor& mask_, double scale) {
    const Tensor lengths = value(lengths_), mask = value(mask_);
    const Attended r = attn_forward(q, k, v, lengths, mask, scale, true);
    // (f32: the result is its own unrounded form and is saved as an output)
    ctx->save_for_backward({r.q, r.k, r.v, lengths, mask, r.out32, r.stats});
    ctx->saved_data["scale"] = scale;
    return r.out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2];
    variable_list out(6);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const at::DeviceGuard guard(q.device());
      const Tensor dout = aligned(grads[0]);
      tapir_attn_args a = attn_args(q, k, v, saved[3], saved[4], ctx->saved_data["scale"].toDouble());
      a.out_f32 = fptr(saved[5]);
      a.stats = fptr(saved[6]);
      a.dout = ptr(dout);
      for (int i = 0; i < 3; ++i) a.dout_stride[i] = dout.stride(i);
      if (ctx->needs_input_grad(0)) out[0] = at::empty(q.sizes(), q.options());
      if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2))
        for (int i = 1; i < 3; ++i) out[i] = at::empty(k.sizes(), k.options());
      a.dq = ptr(out[0]);
      a.dk = ptr(out[1]);
      a.dv = ptr(out[2]);
      const Tensor work = attn_workspace(q, a, true);
      call(q, "cross_attention", [&](tapir_ctx* c, hipStream_t s) { return tapir_cross_attention_backward(c, &a, s); });
    }
    return once(std::move(out));
  }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths_, const OptTensor& mask_,
                       const std::optional<double>& scale_) {
  check_input("q", q);
  check_axes("q", q, 4);
  const int64_t batch = q.size(0), heads = q.size(2), dim = q.size(3);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>("k", k), std::pair<const char*, const Tensor&>("v", v)}) {
    check_beside(name, t, q, q.scalar_type());
    check_axes(name, t, 4);
  }
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(0) == batch && k.size(3) == dim, "k ", k.sizes(), " and v ", v.sizes(),
                    " have to be [", batch, ", keys, kv_heads, ", dim, "] both");
  const int64_t keys = k.size(1), kv_heads = k.size(2);
  TORCH_CHECK_VALUE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads < (int64_t{1} << 31), heads,
                    " query heads are not a multiple of ", kv_heads, " key heads");
  TORCH_CHECK_VALUE(dim >= 8 && dim <= 128 && dim % 8 == 0, "the head dimension has to be a multiple of 8 up to 128, not ", dim);
  Tensor lengths = value(lengths_), mask = value(mask_);
  if (lengths.defined()) {
    check_beside("key_lengths", lengths, q, at::kInt);
    TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == batch, "key_lengths have to be int32 [", batch, "], not ", lengths.sizes());
    lengths = plain(lengths).contiguous();
  }
  if (mask.defined()) {
    check_beside("key_mask", mask, q, at::kBool);
    TORCH_CHECK_VALUE(mask.dim() == 2 && mask.size(0) == batch && mask.size(1) == keys, "key_mask has to be bool [", batch, ", ", keys,
                      "], not ", mask.sizes());
    mask = mask.contiguous();
  }
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt(static_cast<double>(dim));
  TORCH_CHECK_VALUE(scale > 0 && std::isfinite(static_cast<float>(scale)) && static_cast<float>(scale) > 0,
                    "scale has to be positive and finite, not ", scale);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return CrossAttention::apply(q, k, v, option(lengths), option(mask), scale);
  return attn_forward(q, k, v, lengths, mask, scale, false).out;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  namespace py = pybind11;
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
  m.def("rotary_positions", &rotary_positions, py::arg("x"), py::arg("positions"), py::arg("sections"), py::arg("bases"),
        py::arg("interleaved"));
  m.def("cross_attention", &cross_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("key_lengths"), py::arg("key_mask"),
        py::arg("scale"));
}
