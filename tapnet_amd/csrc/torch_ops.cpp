// tapnet_amd.attention's operators on torch tensors: argument checks, memory from torch's allocator, autograd nodes, and the calls
// into libtapir_hip's C ABI (include/tapir_hip.h).  Host code only.  It is C++ because the operators' small calls are bound by the
// host: a layer norm of one frame's tokens with its gradients took 152 us a call through Python's autograd functions and ctypes,
// of which the kernels need a fifth.
//
// The operators are registered with torch's dispatcher (library `tapnet_amd`): what a caller gets (layer_norm, rotary_positions,
// cross_attention) and, below autograd, what launches kernels (..._forward, ..._backward; a Meta form says the results' shapes).  A
// recording of a program -- torch.jit.trace, make_fx -- then holds the operators themselves.  Memory that a function filled
// behind the dispatcher would be recorded as an uninitialised allocation and nothing else.
#include <ATen/DeviceGuard.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>
#include <torch/library.h>

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
  TORCH_CHECK_VALUE(t.device().is_cuda() || t.is_meta(), name, " has to be on the GPU: tapnet_amd has no CPU fallback");
  TORCH_CHECK_VALUE(t.layout() == at::kStrided, name, " has to be a dense tensor");
}

// No forward-mode derivatives: a tangent would be dropped without a word.
void check_no_tangent(const char* name, const Tensor& t) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "tapnet_amd.attention has no forward-mode derivatives, but ", name, " has a tangent");
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

// The registered operator `name`, as a C++ function.
template <class Fn> c10::TypedOperatorHandle<Fn> registered(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();
}

// A leaf's accumulation node belongs to the stream on which it was made.  Where a backward pass is captured while an eager graph of the
// same leaf is alive, torch's engine would make that stream, which is not part of the capture, wait for the captured gradient; the error
// comes up on the engine's own thread and ends the process.  Said here, before the gradient is handed on, it is an error of the call.
void check_capture(const Tensor& like) {
  if (!like.is_cuda() || c10::hip::device_count() == 0) return;      // (a recorded program's tensors)
  const hipStream_t stream = current_stream(like);
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream, &status) != hipSuccess || status != hipStreamCaptureStatusActive) return;
  const auto node = torch::autograd::get_current_node();
  if (node == nullptr) return;
  for (const auto& edge : node->next_edges()) {
    if (edge.function == nullptr || edge.function->name() != "torch::autograd::AccumulateGrad") continue;
    const auto of_leaf = edge.function->stream();
    if (!of_leaf.has_value()) continue;
    const hipStream_t other = c10::hip::HIPStreamMasqueradingAsCUDA(*of_leaf).stream();
    if (other == stream) continue;
    const hipError_t rc = hipStreamIsCapturing(other, &status);
    if (rc != hipSuccess) (void)hipGetLastError();
    TORCH_CHECK(rc == hipSuccess && status == hipStreamCaptureStatusActive,
                "a backward pass is captured while an eager autograd graph of the same leaf is alive: delete its results first");
  }
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

void check_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias) {
  check_input("x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x has to have a last axis of at least one channel");
  TORCH_CHECK_VALUE(x.size(-1) <= (int64_t{1} << 30), "x has more than 2^30 channels");
  for (const auto& [name, p] : {std::pair<const char*, const OptTensor&>("weight", weight), std::pair<const char*, const OptTensor&>("bias", bias)}) {
    if (!p.has_value()) continue;
    check_beside(name, *p, x, at::kFloat);
    TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == x.size(-1), name, " has to be float32 [", x.size(-1), "], not ", p->sizes());
  }
}

Tensor dense(const OptTensor& p) { return p.has_value() ? plain(*p).contiguous() : Tensor(); }

// -> y, and for a backward pass stats [2, rows]: mean, 1 / deviation
std::vector<Tensor> norm_shapes(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, bool train) {
  check_norm(x, weight, bias);
  TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "eps has to be finite and not negative, not ", eps);
  std::vector<Tensor> out{at::empty(x.sizes(), x.options())};
  if (train) out.push_back(at::empty({2, x.numel() / x.size(-1)}, x.options().dtype(at::kFloat)));
  return out;
}

std::vector<Tensor> norm_forward(const Tensor& x, const OptTensor& weight_, const OptTensor& bias_, double eps, bool train) {
  const at::DeviceGuard guard(x.device());
  std::vector<Tensor> out = norm_shapes(x, weight_, bias_, eps, train);
  const Tensor weight = dense(weight_), bias = dense(bias_);
  const Rows r = as_rows(x);
  float* const mean = train ? fptr(out[1]) : nullptr;
  call(x, "layer_norm", [&](tapir_ctx* c, hipStream_t s) {
    return tapir_layer_norm(c, ptr(r.t), r.stride, fptr(weight), fptr(bias), ptr(out[0]), mean, mean ? mean + r.rows : nullptr, r.rows,
                            static_cast<int>(x.size(-1)), static_cast<float>(eps), s);
  });
  return out;
}

// -> those of dx, dweight, dbias that are wanted
std::vector<Tensor> norm_gradients(const Tensor& x, const OptTensor& weight, const Tensor& stats, const Tensor& dy, bool want_x,
                                   bool want_weight, bool want_bias) {
  check_norm(x, weight, std::nullopt);
  check_beside("the gradient", dy, x, x.scalar_type());
  check_beside("stats", stats, x, at::kFloat);
  TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "the gradient has to be ", x.sizes(), ", not ", dy.sizes());
  TORCH_CHECK_VALUE(stats.dim() == 2 && stats.size(0) == 2 && stats.size(1) == x.numel() / x.size(-1) && stats.is_contiguous(),
                    "stats have to be those of the forward pass");
  std::vector<Tensor> out;
  if (want_x) out.push_back(at::empty(x.sizes(), x.options()));
  for (int i = 0; i < want_weight + want_bias; ++i) out.push_back(at::empty({x.size(-1)}, x.options().dtype(at::kFloat)));
  return out;
}

std::vector<Tensor> norm_backward(const Tensor& x, const OptTensor& weight_, const Tensor& stats, const Tensor& dy, bool want_x,
                                  bool want_weight, bool want_bias) {
  const at::DeviceGuard guard(x.device());
  const std::vector<Tensor> out = norm_gradients(x, weight_, stats, dy, want_x, want_weight, want_bias);
  const Tensor weight = dense(weight_);
  const Rows r = as_rows(x), g = as_rows(dy);
  const int channels = static_cast<int>(x.size(-1));
  uint64_t bytes = 0;
  if (want_weight || want_bias)
    call(x, "layer_norm", [&](tapir_ctx* c, hipStream_t) { return tapir_layer_norm_workspace(c, r.rows, channels, &bytes); });
  const Tensor work = workspace(bytes, x);
  const float* mean = fptr(stats);
  call(x, "layer_norm", [&](tapir_ctx* c, hipStream_t s) {
    return tapir_layer_norm_backward(c, ptr(r.t), r.stride, ptr(g.t), g.stride, fptr(weight), mean, mean + r.rows,
                                     want_x ? ptr(out[0]) : nullptr, want_weight ? fptr(out[want_x]) : nullptr,
                                     want_bias ? fptr(out[want_x + want_weight]) : nullptr, r.rows, channels, ptr(work), bytes, s);
  });
  return out;
}

std::vector<Tensor> norm_call(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, bool train) {
  static const auto op = registered<decltype(norm_forward)>("tapnet_amd::layer_norm_forward");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, weight, bias, eps, train);
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    const std::vector<Tensor> out = norm_call(x, weight, bias, eps, true);
    ctx->save_for_backward({x, value(weight), out[1]});
    ctx->saved_data["bias"] = bias.has_value();
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = registered<decltype(norm_backward)>("tapnet_amd::layer_norm_backward");
    check_capture(grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    // (the node's edges are those of the tensors that were given)
    const bool has_weight = saved[1].defined(), has_bias = ctx->saved_data["bias"].toBool();
    const bool want[3] = {ctx->needs_input_grad(0), has_weight && ctx->needs_input_grad(1), has_bias && ctx->needs_input_grad(1 + has_weight)};
    variable_list out(4);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const std::vector<Tensor> got = op.call(saved[0], option(saved[1]), saved[2], grads[0], want[0], want[1], want[2]);
      for (int i = 0, n = 0; i < 3; ++i)
        if (want[i]) out[i] = got[n++];
    }
    return once(std::move(out));
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  check_input("x", x);
  check_no_tangent("x", x);
  check_no_tangent("weight", value(weight));
  check_no_tangent("bias", value(bias));
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(value(weight)) || wants_grad(value(bias))))
    return LayerNorm::apply(x, weight, bias, eps);
  return norm_call(x, weight, bias, eps, false)[0];
}

// ---------------------------------------------------------------------------------------------------- rotary positions
Tensor turn_shape(const Tensor& x, const Tensor& p, at::IntArrayRef sections, c10::ArrayRef<double> bases, bool, bool) {
  check_input("x", x);
  check_axes("x", x, 4);
  check_beside("positions", p, x, at::kFloat);
  const int64_t batch = x.size(0), tokens = x.size(1), dim = x.size(3);
  TORCH_CHECK_VALUE((p.dim() == 2 || p.dim() == 3) && p.size(-2) == tokens && (p.dim() == 2 || p.size(0) == 1 || p.size(0) == batch),
                    "positions have to be [", batch, ", ", tokens, ", axes] or [", tokens, ", axes], not ", p.sizes());
  const int64_t axes = p.size(-1);
  TORCH_CHECK_VALUE(axes >= 1 && axes <= 4, "1 to 4 axes of positions, not ", axes);
  TORCH_CHECK_VALUE(dim >= 1 && dim <= 256 && x.size(2) >= 1 && x.size(2) < (int64_t{1} << 31),
                    "x has to have heads of 1 to 256 channels, not ", x.sizes());
  int64_t sum = 0;
  bool good = static_cast<int64_t>(sections.size()) == axes;
  for (int64_t s : sections) {
    good = good && s >= 0 && s % 2 == 0 && s <= dim;
    sum += good ? s : 0;
  }
  TORCH_CHECK_VALUE(good && sum <= dim, "sections ", sections, ": ", axes, " even channel counts are wanted, at most ", dim, " together");
  good = bases.size() == 1 || static_cast<int64_t>(bases.size()) == axes;
  for (double b : bases) good = good && b > 0 && std::isfinite(b);
  TORCH_CHECK_VALUE(good, "base ", bases, ": one positive number, or one per axis");
  return at::empty(x.sizes(), x.options());
}

Tensor turn(const Tensor& in, const Tensor& positions_, at::IntArrayRef sections, c10::ArrayRef<double> bases, bool interleaved, bool inverse) {
  const at::DeviceGuard guard(in.device());
  Tensor y = turn_shape(in, positions_, sections, bases, interleaved, inverse);
  Tensor x = plain(in);
  if (x.size(3) > 1 && x.stride(3) != 1) x = x.contiguous();
  const Tensor positions = plain(positions_).contiguous();
  const int axes = static_cast<int>(sections.size());
  tapir_rotary_args a{};
  a.batch = x.size(0);
  a.tokens = x.size(1);
  a.heads = static_cast<int>(x.size(2));
  a.dim = static_cast<int>(x.size(3));
  a.axes = axes;
  a.interleaved = interleaved;
  a.inverse = inverse;
  for (int i = 0; i < axes; ++i) {
    a.section[i] = static_cast<int>(sections[i]);
    a.base[i] = bases[bases.size() == 1 ? 0 : i];
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

Tensor turn_call(const Tensor& x, const Tensor& positions, at::IntArrayRef sections, c10::ArrayRef<double> bases, bool interleaved,
                 bool inverse) {
  static const auto op = registered<decltype(turn)>("tapnet_amd::rotary_positions_turn");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, positions, sections, bases, interleaved, inverse);
}

struct Rotary : torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const std::vector<int64_t>& sections,
                        const std::vector<double>& bases, bool interleaved) {
    ctx->save_for_backward({positions});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["bases"] = bases;
    ctx->saved_data["interleaved"] = interleaved;
    return turn_call(x, positions, sections, bases, interleaved, false);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture(grads[0]);
    variable_list out(5);
    out[0] = turn_call(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["sections"].toIntVector(),
                       ctx->saved_data["bases"].toDoubleVector(), ctx->saved_data["interleaved"].toBool(), true);
    return once(std::move(out));
  }
};

Tensor rotary_positions(const Tensor& x, const Tensor& positions, at::OptionalIntArrayRef sections_, c10::ArrayRef<double> bases,
                        bool interleaved) {
  check_input("x", x);
  check_axes("x", x, 4);
  check_no_tangent("x", x);
  check_no_tangent("positions", positions);
  TORCH_CHECK_VALUE(!positions.requires_grad(), "positions have no gradient: detach them");
  std::vector<int64_t> sections;
  if (sections_.has_value()) {
    sections.assign(sections_->begin(), sections_->end());
  } else if (positions.dim() >= 1) {
    const int64_t pairs = x.size(3) / 2, axes = positions.size(-1);
    for (int64_t a = 0; a < axes && a < 5; ++a) sections.push_back(2 * (pairs / axes + (a < pairs % axes)));
  }
  if (at::GradMode::is_enabled() && x.requires_grad())
    return Rotary::apply(x, positions, sections, std::vector<double>(bases.begin(), bases.end()), interleaved);
  return turn_call(x, positions, sections, bases, interleaved, false);
}

// ----------------------------------------------------------------------------------------------------- cross attention
// `t` itself where its rows (last axis) are dense, start at multiples of 16 bytes and are less than 2^22 elements apart, else a
// dense copy.  An axis of one element has no stride (torch calls such a tensor contiguous whatever number stands there).
// spaced() goes by the strides and the offset alone: a recorded program's tensors have no memory.
Tensor spaced(const Tensor& in) {
  const Tensor t = plain(in);
  const int64_t epc = 16 / static_cast<int64_t>(t.element_size());
  bool good = t.stride(3) == 1 && t.storage_offset() % epc == 0;
  for (int d = 0; d < 3; ++d) good = good && (t.size(d) <= 1 || t.stride(d) % epc == 0);
  good = good && (t.size(1) <= 1 || t.stride(1) < (int64_t{1} << 22));
  return good ? t : t.clone(at::MemoryFormat::Contiguous);
}
Tensor aligned(const Tensor& in) {
  const Tensor t = spaced(in);
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

void check_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths, const OptTensor& mask, double scale) {
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
  if (lengths.has_value()) {
    check_beside("key_lengths", *lengths, q, at::kInt);
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == batch, "key_lengths have to be int32 [", batch, "], not ", lengths->sizes());
  }
  if (mask.has_value()) {
    check_beside("key_mask", *mask, q, at::kBool);
    TORCH_CHECK_VALUE(mask->dim() == 2 && mask->size(0) == batch && mask->size(1) == keys, "key_mask has to be bool [", batch, ", ", keys,
                      "], not ", mask->sizes());
  }
  TORCH_CHECK_VALUE(scale >= 0x1p-60 && scale <= 0x1p60, "scale has to be within 2^-60 .. 2^60, not ", scale);
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

// -> the result, and for a backward pass (in bf16) the same unrounded and the rows' statistics.  f32: the result is its own
// unrounded form.
std::vector<Tensor> attn_shapes(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths, const OptTensor& mask, double scale,
                                bool train) {
  check_attention(q, k, v, lengths, mask, scale);
  std::vector<Tensor> out{at::empty(q.sizes(), q.options())};
  const auto f32 = q.options().dtype(at::kFloat);
  if (train && q.scalar_type() != at::kFloat) out.push_back(at::empty(q.sizes(), f32));
  if (train) out.push_back(at::empty({q.size(0), q.size(1) * q.size(2), 2}, f32));
  return out;
}

std::vector<Tensor> attn_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& lengths_, const OptTensor& mask_,
                                 double scale, bool train) {
  const at::DeviceGuard guard(q_.device());
  const std::vector<Tensor> out = attn_shapes(q_, k_, v_, lengths_, mask_, scale, train);
  const Tensor q = aligned(q_), k = aligned(k_), v = aligned(v_), lengths = dense(lengths_), mask = dense(mask_);
  tapir_attn_args a = attn_args(q, k, v, lengths, mask, scale);
  a.out = ptr(out[0]);
  if (train) {
    a.out_f32 = fptr(out[out.size() - 2]);
    a.stats = fptr(out.back());
  }
  const Tensor work = attn_workspace(q, a, false);
  call(q, "cross_attention", [&](tapir_ctx* c, hipStream_t s) { return tapir_cross_attention(c, &a, s); });
  return out;
}

// -> those of dq and (dk, dv) that are wanted
std::vector<Tensor> attn_gradients(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths, const OptTensor& mask, double scale,
                                   const Tensor& out_f32, const Tensor& stats, const Tensor& dout, bool want_q, bool want_kv) {
  check_attention(q, k, v, lengths, mask, scale);
  check_beside("the gradient", dout, q, q.scalar_type());
  check_beside("out_f32", out_f32, q, at::kFloat);
  check_beside("stats", stats, q, at::kFloat);
  TORCH_CHECK_VALUE(dout.sizes() == q.sizes(), "the gradient has to be ", q.sizes(), ", not ", dout.sizes());
  TORCH_CHECK_VALUE(out_f32.sizes() == q.sizes() && out_f32.is_contiguous() && stats.numel() == q.size(0) * q.size(1) * q.size(2) * 2 &&
                        stats.is_contiguous(), "out_f32 and stats have to be those of the forward pass");
  std::vector<Tensor> out;
  if (want_q) out.push_back(at::empty(q.sizes(), q.options()));
  for (int i = 0; i < 2 * want_kv; ++i) out.push_back(at::empty(k.sizes(), k.options()));
  return out;
}

std::vector<Tensor> attn_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& lengths_, const OptTensor& mask_,
                                  double scale, const Tensor& out_f32, const Tensor& stats, const Tensor& dout_, bool want_q, bool want_kv) {
  const at::DeviceGuard guard(q_.device());
  const std::vector<Tensor> out = attn_gradients(q_, k_, v_, lengths_, mask_, scale, out_f32, stats, dout_, want_q, want_kv);
  const Tensor q = aligned(q_), k = aligned(k_), v = aligned(v_), lengths = dense(lengths_), mask = dense(mask_), dout = aligned(dout_);
  tapir_attn_args a = attn_args(q, k, v, lengths, mask, scale);
  a.out_f32 = fptr(out_f32);
  a.stats = fptr(stats);
  a.dout = ptr(dout);
  for (int i = 0; i < 3; ++i) a.dout_stride[i] = dout.stride(i);
  if (want_q) a.dq = ptr(out[0]);
  if (want_kv) {
    a.dk = ptr(out[want_q]);
    a.dv = ptr(out[want_q + 1]);
  }
  const Tensor work = attn_workspace(q, a, true);
  call(q, "cross_attention", [&](tapir_ctx* c, hipStream_t s) { return tapir_cross_attention_backward(c, &a, s); });
  return out;
}

std::vector<Tensor> attn_call(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths, const OptTensor& mask, double scale,
                              bool train) {
  static const auto op = registered<decltype(attn_forward)>("tapnet_amd::cross_attention_forward");
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, lengths, mask, scale, train);
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& lengths,
                        const OptTensor& mask, double scale) {
    check_attention(q_, k_, v_, lengths, mask, scale);
    const Tensor q = spaced(q_), k = spaced(k_), v = spaced(v_);      // (copied once for both passes)
    const std::vector<Tensor> out = attn_call(q, k, v, lengths, mask, scale, true);
    // (f32: the result is saved as an output)
    ctx->save_for_backward({q, k, v, value(lengths), value(mask), out[out.size() - 2], out.back()});
    ctx->saved_data["scale"] = scale;
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = registered<decltype(attn_backward)>("tapnet_amd::cross_attention_backward");
    check_capture(grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    const bool want_q = ctx->needs_input_grad(0), want_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    variable_list out(6);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const std::vector<Tensor> got = op.call(saved[0], saved[1], saved[2], option(saved[3]), option(saved[4]), ctx->saved_data["scale"].toDouble(),
                                              saved[5], saved[6], grads[0], want_q, want_kv);
      if (want_q) out[0] = got[0];
      for (int i = 0; i < 2 * want_kv; ++i) out[1 + i] = got[want_q + i];
    }
    return once(std::move(out));
  }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths, const OptTensor& mask,
                       std::optional<double> scale_) {
  check_input("q", q);
  check_axes("q", q, 4);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>("q", q), std::pair<const char*, const Tensor&>("k", k),
                                std::pair<const char*, const Tensor&>("v", v)})
    check_no_tangent(name, t);
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(1, q.size(3))));
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return CrossAttention::apply(q, k, v, lengths, mask, scale);
  return attn_call(q, k, v, lengths, mask, scale, false)[0];
}

// what Python calls: the registered operators, so that a recording holds them
Tensor py_layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  static const auto op = registered<decltype(layer_norm)>("tapnet_amd::layer_norm");
  return op.call(x, weight, bias, eps);
}
Tensor py_rotary_positions(const Tensor& x, const Tensor& positions, const std::optional<std::vector<int64_t>>& sections,
                           const std::vector<double>& bases, bool interleaved) {
  static const auto op = registered<decltype(rotary_positions)>("tapnet_amd::rotary_positions");
  return op.call(x, positions, sections.has_value() ? at::OptionalIntArrayRef(*sections) : at::OptionalIntArrayRef(), bases, interleaved);
}
Tensor py_cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lengths, const OptTensor& mask,
                          const std::optional<double>& scale) {
  static const auto op = registered<decltype(cross_attention)>("tapnet_amd::cross_attention");
  return op.call(q, k, v, lengths, mask, scale);
}

}  // namespace

TORCH_LIBRARY(tapnet_amd, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", &layer_norm);
  m.def("layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps, bool train) -> Tensor[]");
  m.def("layer_norm_backward(Tensor x, Tensor? weight, Tensor stats, Tensor dy, bool want_x, bool want_weight, bool want_bias) -> Tensor[]");
  m.def("rotary_positions(Tensor x, Tensor positions, int[]? sections, float[] bases, bool interleaved) -> Tensor", &rotary_positions);
  m.def("rotary_positions_turn(Tensor x, Tensor positions, int[] sections, float[] bases, bool interleaved, bool inverse) -> Tensor");
  m.def("cross_attention(Tensor q, Tensor k, Tensor v, Tensor? key_lengths, Tensor? key_mask, float? scale) -> Tensor", &cross_attention);
  m.def("cross_attention_forward(Tensor q, Tensor k, Tensor v, Tensor? key_lengths, Tensor? key_mask, float scale, bool train) -> Tensor[]");
  m.def("cross_attention_backward(Tensor q, Tensor k, Tensor v, Tensor? key_lengths, Tensor? key_mask, float scale, Tensor out_f32, "
        "Tensor stats, Tensor dout, bool want_q, bool want_kv) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(tapnet_amd, CUDA, m) {
  m.impl("layer_norm_forward", &norm_forward);
  m.impl("layer_norm_backward", &norm_backward);
  m.impl("rotary_positions_turn", &turn);
  m.impl("cross_attention_forward", &attn_forward);
  m.impl("cross_attention_backward", &attn_backward);
}

TORCH_LIBRARY_IMPL(tapnet_amd, Meta, m) {
  m.impl("layer_norm_forward", &norm_shapes);
  m.impl("layer_norm_backward", &norm_gradients);
  m.impl("rotary_positions_turn", &turn_shape);
  m.impl("cross_attention_forward", &attn_shapes);
  m.impl("cross_attention_backward", &attn_gradients);
}

PYBIND11_MODULE(_torch_ops, m) {
  namespace py = pybind11;
  m.def("layer_norm", &py_layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
  m.def("rotary_positions", &py_rotary_positions, py::arg("x"), py::arg("positions"), py::arg("sections"), py::arg("bases"),
        py::arg("interleaved"));
  m.def("cross_attention", &py_cross_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("key_lengths"), py::arg("key_mask"),
        py::arg("scale"));
}
