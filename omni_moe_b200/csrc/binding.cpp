// Python binding of the operators whose calls are short: the argument checks, allocations and autograd nodes of the few-token
// layer, the RMS norm, the MX conversions and the MLP with 8-bit checkpoints, over the C ABI of libomni_moe_b200.so.
// For these the host side of a call costs more than its kernels at small sizes (a norm with its gradient: 122 us through
// Python autograd nodes), and a backward in C++ needs no interpreter lock in the autograd engine's thread.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <map>
#include <mutex>

#include "../../include/omni_moe_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kBlock = 32;          // values that share a scale
constexpr int64_t kMaxHidden = 16384;   // of the norm

// ValueError / TypeError of the wrong argument
#define OMNI_VALUE(cond, ...) \
  if (!(cond)) throw py::value_error(c10::str(__VA_ARGS__))
#define OMNI_TYPE(cond, ...) \
  if (!(cond)) throw py::type_error(c10::str(__VA_ARGS__))

void check(int rc) { TORCH_CHECK(rc == 0, "libomni_moe_b200 rejected the call (code ", rc, "): ", omni_last_error()); }

void require_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "omni_moe_b200 runs on CUDA tensors only (sm_100a); got a tensor on ", t.device().str());
}
void require_device(const Tensor& t, const Tensor& x) {
  if (t.device() == x.device()) return;
  require_cuda(t);
  TORCH_CHECK(false, "all tensors must be on ", x.device().str(), ", got one on ", t.device().str());
}
int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return OMNI_F32;
    case at::kBFloat16: return OMNI_BF16;
    case at::kHalf: return OMNI_F16;
    default: throw py::type_error(c10::str("unsupported dtype ", c10::toString(t)));
  }
}
void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int32_t* status_ptr(int64_t p) { return reinterpret_cast<int32_t*>(p); }
int64_t blocks_of(int64_t cols) { return (cols + kBlock - 1) / kBlock; }

// A matrix whose rows are contiguous and do not overlap (a view wherever the strides allow).
Tensor rows_of(const Tensor& t) {
  if (t.dim() == 2 && t.is_contiguous()) return t;
  Tensor m = t.reshape({-1, t.size(-1)});
  const bool whole = (m.size(1) == 1 || m.stride(1) == 1) && (m.size(0) <= 1 || m.stride(0) >= m.size(1));
  return whole ? m : m.contiguous();
}
// Contiguous bf16 on a 16-byte boundary, as the GEMMs' operands have to be.
Tensor as_bf16(const Tensor& t) {
  Tensor b = t.to(at::kBFloat16).contiguous();
  return reinterpret_cast<uintptr_t>(b.data_ptr()) % 16 ? b.clone() : b;
}
// Backward passes here are not differentiable again: better an error than a second derivative of zero.
void once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no second derivative: run its backward without create_graph");
}

std::pair<Tensor, Tensor> empty_mx(int64_t rows, int64_t cols, const Tensor& like) {
  return {at::empty({rows, cols}, like.options().dtype(at::kFloat8_e4m3fn)),
          at::empty({rows, blocks_of(cols)}, like.options().dtype(at::kFloat8_e8m0fnu))};
}
void check_mx(const Tensor& codes, const Tensor& scales) {
  require_cuda(codes);
  require_device(scales, codes);
  OMNI_VALUE(codes.dim() == 2 && codes.scalar_type() == at::kFloat8_e4m3fn && scales.scalar_type() == at::kFloat8_e8m0fnu,
                    "MX blocks are a matrix of float8_e4m3fn codes and one of float8_e8m0fnu scales");
  OMNI_VALUE(scales.dim() == 2 && scales.size(0) == codes.size(0) && scales.size(1) == blocks_of(codes.size(1)), "codes of shape ",
                    codes.sizes(), " need scales of shape [", codes.size(0), ", ", blocks_of(codes.size(1)), "], got ", scales.sizes());
}

// ---- MX blocks ----------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> mx_quantize(const Tensor& input) {
  require_cuda(input);
  OMNI_VALUE(input.dim() == 2, "mx_quantize takes a matrix, got a tensor of shape ", input.sizes());
  const int code = dtype_code(input.scalar_type());
  const at::cuda::OptionalCUDAGuard guard(input.device());
  const Tensor x = rows_of(input.detach());
  auto [codes, scales] = empty_mx(x.size(0), x.size(1), x);
  if (x.numel()) check(omni_mx_quantize(x.data_ptr(), x.stride(0), code, x.size(0), x.size(1), codes.data_ptr(), scales.data_ptr(), stream_of(x)));
  return {codes, scales};
}

Tensor mx_dequantize(const Tensor& codes_in, const Tensor& scales_in, at::ScalarType dtype) {
  check_mx(codes_in, scales_in);
  const int code = dtype_code(dtype);
  const at::cuda::OptionalCUDAGuard guard(codes_in.device());
  const Tensor codes = codes_in.contiguous(), scales = scales_in.contiguous();
  Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype));
  if (out.numel())
    check(omni_mx_dequantize(codes.data_ptr(), scales.data_ptr(), codes.size(0), codes.size(1), code, out.data_ptr(), stream_of(codes)));
  return out;
}

// ---- RMS norm -----------------------------------------------------------------------------------
struct NormOut {
  Tensor y, h, codes, scales, rstd;
};

NormOut norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps, bool quantize, bool keep) {
  const int64_t t = x.size(0), n = x.size(1);
  const at::cuda::OptionalCUDAGuard guard(x.device());
  NormOut o;
  o.y = at::empty({t, n}, x.options());
  if (residual.defined()) o.h = at::empty({t, n}, x.options());
  if (keep) o.rstd = at::empty({t}, x.options().dtype(at::kFloat));
  if (quantize) std::tie(o.codes, o.scales) = empty_mx(t, n, x);
  if (t)
    check(omni_rms_norm(x.data_ptr(), x.stride(0), ptr(residual), residual.defined() ? residual.stride(0) : 0, weight.data_ptr(),
                        dtype_code(weight.scalar_type()), dtype_code(x.scalar_type()), t, static_cast<int>(n), static_cast<float>(eps),
                        o.y.data_ptr(), ptr(o.h), static_cast<float*>(ptr(o.rstd)), ptr(o.codes), ptr(o.scales), stream_of(x)));
  return o;
}

std::pair<Tensor, Tensor> norm_backward(const Tensor& dy, const Tensor& dh, const Tensor& h, const Tensor& weight, const Tensor& rstd,
                                        bool need_weight, int64_t status) {
  const int64_t t = h.size(0), n = h.size(1);
  const at::cuda::OptionalCUDAGuard guard(h.device());
  Tensor dx = at::empty({t, n}, h.options()), dw;
  if (t == 0) return {dx, need_weight ? at::zeros_like(weight) : dw};
  Tensor scratch;
  if (need_weight) {
    dw = at::empty_like(weight);
    scratch = at::empty({static_cast<int64_t>(omni_rms_norm_bwd_scratch_bytes(t, static_cast<int>(n)))}, h.options().dtype(at::kByte));
  }
  check(omni_rms_norm_bwd(dy.data_ptr(), dy.stride(0), ptr(dh), dh.defined() ? dh.stride(0) : 0, h.data_ptr(), h.stride(0), weight.data_ptr(),
                          dtype_code(weight.scalar_type()), dtype_code(h.scalar_type()), rstd.data_ptr<float>(), t, static_cast<int>(n),
                          dx.data_ptr(), ptr(dw), ptr(scratch), need_weight ? scratch.numel() : 0, status_ptr(status), stream_of(h)));
  return {dx, dw};
}

// outputs: y, h (only with a residual), codes and scales (only if asked for; they carry no gradient)
struct RmsNormNode : torch::autograd::Function<RmsNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps, bool quantize,
                               int64_t status) {
    NormOut o = norm_forward(x, residual ? *residual : Tensor(), weight, eps, quantize, true);
    ctx->save_for_backward({o.h.defined() ? o.h : x, weight, o.rstd});
    ctx->saved_data["status"] = status;
    ctx->set_materialize_grads(false);
    variable_list out{o.y};
    if (o.h.defined()) out.push_back(o.h);
    if (quantize) {
      out.push_back(o.codes), out.push_back(o.scales);
      ctx->mark_non_differentiable({o.codes, o.scales});
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("omni_rms_norm_func");
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &weight = saved[1], &rstd = saved[2];
    // (the indices of needs_input_grad count the tensors that were given)
    const bool has_residual = grads.size() == 2 || grads.size() == 4;
    const bool need_x = ctx->needs_input_grad(0), need_r = has_residual && ctx->needs_input_grad(1), need_w = ctx->needs_input_grad(has_residual ? 2 : 1);
    const Tensor &dy = grads[0], dh = has_residual ? grads[1] : Tensor();
    Tensor dx, dw;
    if (dy.defined()) {
      std::tie(dx, dw) = norm_backward(rows_of(dy), dh.defined() ? rows_of(dh) : Tensor(), h, weight, rstd, need_w,
                                       ctx->saved_data["status"].toInt());
    } else {  // only the sum was used
      dx = dh;
      if (need_w) dw = at::zeros_like(weight);
    }
    return {need_x ? dx : Tensor(), need_r ? dx : Tensor(), dw, Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, OptTensor, OptTensor> rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps,
                                                          bool quantize, int64_t status) {
  require_cuda(x);
  require_device(weight, x);
  if (residual) require_device(*residual, x);
  dtype_code(x.scalar_type());
  const int64_t n = x.dim() ? x.size(-1) : 0;
  OMNI_VALUE(n >= 1 && n <= kMaxHidden, "the last dimension must be in [1, ", kMaxHidden, "], got shape ", x.sizes());
  OMNI_VALUE(weight.dim() == 1 && weight.size(0) == n, "weight must be [", n, "], got ", weight.sizes());
  OMNI_TYPE(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, "weight must be ",
                   c10::toString(x.scalar_type()), " or float32, got ", c10::toString(weight.scalar_type()));
  OMNI_VALUE(!residual || (residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type()),
                    "the residual must have the shape and type of x");
  OMNI_VALUE(eps >= 0.0, "eps must be >= 0, got ", eps);  // also refuses NaN
  const Tensor xr = rows_of(x), w = weight.contiguous();
  OptTensor rr;
  if (residual) rr = rows_of(*residual);
  Tensor y, h, codes, scales;
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (residual && residual->requires_grad()))) {
    const variable_list o = RmsNormNode::apply(xr, rr, w, eps, quantize, status);
    size_t i = 0;
    y = o[i++];
    if (residual) h = o[i++];
    if (quantize) codes = o[i], scales = o[i + 1];
  } else {
    NormOut o = norm_forward(xr, rr ? *rr : Tensor(), w, eps, quantize, false);
    y = o.y, h = o.h, codes = o.codes, scales = o.scales;
  }
  if (x.dim() != 2) {
    y = y.view(x.sizes());
    if (h.defined()) h = h.view(x.sizes());
  }
  return {y, h.defined() ? h : x, codes.defined() ? OptTensor(codes) : OptTensor(), scales.defined() ? OptTensor(scales) : OptTensor()};
}

// ---- MLP with 8-bit checkpoints -------------------------------------------------------------------
Tensor gemm(const Tensor& a, bool a_t, const Tensor& b, bool b_t, int64_t status) {
  const int64_t m = a_t ? a.size(1) : a.size(0), k = a_t ? a.size(0) : a.size(1), n = b_t ? b.size(1) : b.size(0);
  Tensor out = at::empty({m, n}, a.options());
  check(omni_gemm_bf16(a.data_ptr(), a_t, a.stride(0), b.data_ptr(), b_t, b.stride(0), m, n, k, out.data_ptr(), n, status_ptr(status), stream_of(a)));
  return out;
}

// (dx, d_gate, d_up, d_down), undefined where not needed.  x: as the weight gradients are to see it (for need_gate_up).
variable_list mlp_ckpt_backward(const Tensor& dy, const OptTensor& x, const Tensor& codes, const Tensor& scales, const Tensor& wg, const Tensor& wu,
                                const Tensor& wd, double limit, bool need_x, bool need_gate_up, bool need_down, int64_t status) {
  const int64_t t = codes.size(0), i = wg.size(0), h = wg.size(1);
  const at::cuda::OptionalCUDAGuard guard(dy.device());
  const auto bf = dy.options().dtype(at::kBFloat16);
  variable_list g(4);
  if (t == 0) {
    if (need_x) g[0] = at::zeros({0, h}, bf);
    if (need_gate_up) g[1] = at::zeros({i, h}, bf), g[2] = at::zeros({i, h}, bf);
    if (need_down) g[3] = at::zeros({h, i}, bf);
    return g;
  }
  const Tensor dgu = at::empty({t, 2 * i}, bf);
  Tensor act;
  if (need_down) act = at::empty({t, i}, bf);
  check(omni_mlp_dact_swiglu_mx(dy.data_ptr(), wd.data_ptr(), t, static_cast<int>(h), static_cast<int>(i), codes.data_ptr(), scales.data_ptr(),
                                static_cast<float>(limit), dgu.data_ptr(), ptr(act), status_ptr(status), stream_of(dy)));
  // order: the product that reads act right after the kernel that wrote it, the two that read (dgate | dup) back to back
  if (need_down) g[3] = gemm(dy, true, act, true, status);  // dy^T [H,T] @ act [T,I]
  if (need_x) {
    if (i % 64 == 0) {  // dgate @ Wg + dup @ Wu: the two weight matrices as one B operand stacked along K
      g[0] = at::empty({t, h}, bf);
      check(omni_gemm_bf16_stacked_b(dgu.data_ptr(), 0, 2 * i, wg.data_ptr(), wu.data_ptr(), i, h, t, h, 2 * i, g[0].data_ptr(), h,
                                     status_ptr(status), stream_of(dy)));
    } else {
      g[0] = gemm(dgu, false, at::cat({wg, wu}, 0), true, status);
    }
  }
  if (need_gate_up) {
    const Tensor d = gemm(dgu, true, *x, true, status);  // (dgate | dup)^T [2I,T] @ x [T,H]
    g[1] = d.narrow(0, 0, i), g[2] = d.narrow(0, i, i);
  }
  return g;
}

struct MlpCkptNode : torch::autograd::Function<MlpCkptNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, double limit,
                        const OptTensor& x_codes, const OptTensor& x_scales, bool keep_x, int64_t status) {
    const Tensor xb = as_bf16(x), wg = as_bf16(gate), wu = as_bf16(up), wd = as_bf16(down);
    const int64_t t = xb.size(0), h = xb.size(1), i = wg.size(0);
    const at::cuda::OptionalCUDAGuard guard(x.device());
    const Tensor codes = at::empty({t, 2 * i}, xb.options().dtype(at::kFloat8_e4m3fn));
    const Tensor scales = at::empty({t, 2 * blocks_of(i)}, xb.options().dtype(at::kFloat8_e8m0fnu));
    Tensor y = at::empty({t, h}, xb.options());
    if (t) {
      const Tensor act = at::empty({t, i}, xb.options());
      check(omni_mlp_gate_up_save_mx(xb.data_ptr(), wg.data_ptr(), wu.data_ptr(), t, static_cast<int>(h), static_cast<int>(i),
                                     static_cast<float>(limit), act.data_ptr(), codes.data_ptr(), scales.data_ptr(), status_ptr(status), stream_of(xb)));
      check(omni_mlp_down(act.data_ptr(), wd.data_ptr(), t, static_cast<int>(h), static_cast<int>(i), nullptr, y.data_ptr(), status_ptr(status),
                          stream_of(xb)));
    }
    variable_list saved{wg, wu, wd, codes, scales};
    const bool for_weights = gate.requires_grad() || up.requires_grad();
    if (for_weights && keep_x) {
      saved.push_back(xb);
    } else if (for_weights) {
      if (x_codes) {
        saved.push_back(*x_codes), saved.push_back(*x_scales);
      } else {
        const auto [c, s] = mx_quantize(xb);
        saved.push_back(c), saved.push_back(s);
      }
    }
    ctx->save_for_backward(saved);
    ctx->saved_data["limit"] = limit, ctx->saved_data["status"] = status;
    ctx->saved_data["types"] = std::vector<int64_t>{static_cast<int64_t>(x.scalar_type()), static_cast<int64_t>(gate.scalar_type()),
                                                    static_cast<int64_t>(up.scalar_type()), static_cast<int64_t>(down.scalar_type())};
    return x.scalar_type() == at::kBFloat16 ? y : y.to(x.scalar_type());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("omni_mlp_ckpt_func");
    const auto s = ctx->get_saved_variables();
    OptTensor x;
    if (s.size() == 6) x = s[5];
    if (s.size() == 7) x = mx_dequantize(s[5], s[6], at::kBFloat16);
    const bool need[4] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)};
    variable_list g = mlp_ckpt_backward(as_bf16(grads[0]), x, s[3], s[4], s[0], s[1], s[2], ctx->saved_data["limit"].toDouble(), need[0],
                                        need[1] || need[2], need[3], ctx->saved_data["status"].toInt());
    const auto types = ctx->saved_data["types"].toIntVector();
    for (int j = 0; j < 4; ++j) {
      const auto type = static_cast<at::ScalarType>(types[j]);
      if (!need[j]) g[j] = Tensor();
      else if (type != at::kBFloat16) g[j] = g[j].to(type);
    }
    for (int j = 0; j < 5; ++j) g.emplace_back();
    return g;
  }
};

Tensor mlp_ckpt(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, double limit, const OptTensor& x_codes,
                const OptTensor& x_scales, bool keep_x, int64_t status) {
  return MlpCkptNode::apply(x, gate, up, down, limit, x_codes, x_scales, keep_x, status);
}

// ---- the layer for a few tokens -------------------------------------------------------------------
// Scratch of a call on the current stream; its head holds counters that every launch finds and leaves at zero.  One
// buffer for each (device, stream): launches on one stream follow one another, launches on different streams may overlap
// and must not share.  While a graph is captured the buffer belongs to the graph (its head zeroed in every replay), so graphs that
// replay beside each other or beside eager calls share nothing.
Tensor decode_workspace(int64_t bytes, const Tensor& like, void* stream) {
  const auto fresh = [&] {
    Tensor ws = at::empty({bytes}, like.options().dtype(at::kByte));
    ws.narrow(0, 0, static_cast<int64_t>(omni_decode_counter_bytes())).zero_();
    return ws;
  };
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return fresh();
  static std::mutex mutex;
  static auto* buffers = new std::map<std::pair<int, void*>, Tensor>();  // never destroyed: CUDA may be gone by then
  const std::lock_guard<std::mutex> lock(mutex);
  const std::pair<int, void*> key(like.get_device(), stream);
  const auto it = buffers->find(key);
  if (it != buffers->end() && it->second.numel() >= bytes) return it->second;
  // a buffer that is dropped goes back to its own stream's pool: launches in flight keep it
  if (it != buffers->end()) buffers->erase(it);
  while (buffers->size() >= 16) buffers->erase(buffers->begin());
  return buffers->emplace(key, fresh()).first->second;
}

// Nothing where something has to be converted, copied or padded first.
OptTensor decode(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, const Tensor& router_x, const Tensor& router_y,
                 const Tensor& up_embed, const Tensor& down_embed, int64_t k, const OptTensor& bn_scale, const OptTensor& bn_shift,
                 int64_t status) {
  const Tensor* all[] = {&x, &gate, &up, &down, &router_x, &router_y, &up_embed, &down_embed};
  require_cuda(x);
  for (const Tensor* t : all) {
    require_device(*t, x);
    OMNI_VALUE(t->dim() == 2, "omni_decode_func takes a matrix of tokens and matrices of weights, got a tensor of shape ", t->sizes());
  }
  const int64_t t = x.size(0), h = x.size(1), i = gate.size(0), n = router_x.size(0), experts = up_embed.size(0);
  const auto is = [](const Tensor& m, int64_t r, int64_t c) { return m.size(0) == r && m.size(1) == c; };
  OMNI_VALUE(t <= omni_decode_max_tokens(), "omni_decode_func takes at most ", omni_decode_max_tokens(), " tokens, got ", t, ": use OmniMoE.forward");
  OMNI_VALUE(is(gate, i, h) && is(up, i, h) && is(down, h, i),
                    "gate_weight and up_weight must be (intermediate, hidden), down_weight (hidden, intermediate)");
  OMNI_VALUE(is(router_x, n, h) && is(router_y, n, h), "router_x and router_y must both be (sqrt_n, hidden)");
  OMNI_VALUE(is(up_embed, experts, h) && is(down_embed, experts, h) && experts >= n * n,
                    "up_embed and down_embed must both be (num_experts, hidden) with at least sqrt_n ** 2 rows");
  OMNI_VALUE(h >= 1 && i >= 1 && n >= 1 && k >= 1 && k <= std::min<int64_t>(128, n * n), "num_experts_per_token must be in [1, ",
                    std::min<int64_t>(128, n * n), "], got ", k);
  OMNI_VALUE(bn_scale.has_value() == bn_shift.has_value(), "bn_scale and bn_shift must be given together");
  Tensor scale, shift;
  if (bn_scale) {
    for (const Tensor* v : {&*bn_scale, &*bn_shift})
      OMNI_VALUE(v->dim() == 1 && v->size(0) == 2 * n && v->scalar_type() == at::kFloat && v->device() == x.device(),
                        "bn_scale and bn_shift must be float32 vectors of 2 * sqrt_n values on the device of x");
    scale = bn_scale->contiguous(), shift = bn_shift->contiguous();
  }
  if (at::GradMode::is_enabled()) {
    bool leaf = (bn_scale && bn_scale->requires_grad()) || (bn_shift && bn_shift->requires_grad());
    for (const Tensor* m : all) leaf = leaf || m->requires_grad();
    TORCH_CHECK(!leaf, "omni_decode_func has no backward: call it under torch.no_grad(), or OmniMoE.forward to train");
  }
  if (h % 8 || i % 8) return std::nullopt;
  for (const Tensor* m : all)
    if (m->scalar_type() != at::kBFloat16 || !m->is_contiguous() || reinterpret_cast<uintptr_t>(m->data_ptr()) % 16) return std::nullopt;
  const at::cuda::OptionalCUDAGuard guard(x.device());
  Tensor y = at::empty({t, h}, x.options());
  if (t == 0) return y;
  void* stream = stream_of(x);
  const int ti = static_cast<int>(t), hi = static_cast<int>(h), ii = static_cast<int>(i), ni = static_cast<int>(n), ki = static_cast<int>(k);
  const Tensor ws = decode_workspace(static_cast<int64_t>(omni_decode_workspace_bytes(ti, hi, ii, ni, ki)), x, stream);
  check(omni_decode(x.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr(), router_x.data_ptr(), router_y.data_ptr(), up_embed.data_ptr(),
                    down_embed.data_ptr(), static_cast<float*>(ptr(scale)), static_cast<float*>(ptr(shift)), ti, hi, ii, ni, ki, experts,
                    y.data_ptr(), ws.data_ptr(), ws.numel(), status_ptr(status), stream));
  return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("mx_quantize", &mx_quantize);
  m.def("mx_dequantize", [](const Tensor& c, const Tensor& s, py::object dtype) {
    return mx_dequantize(c, s, torch::python::detail::py_object_to_dtype(dtype));
  });
  m.def("rms_norm", &rms_norm);
  m.def("mlp_ckpt", &mlp_ckpt);
  m.def("mlp_ckpt_backward", &mlp_ckpt_backward);
  m.def("decode", &decode);
}
