// Windowed attention on the host: operands, tensor maps, launches and the autograd
// nodes (the kernels: attn_window_fwd.cu, attn_window_dkdv.cu, attn_window_dq.cu).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <string>

#include "attn_window.cuh"
#include "common.h"

namespace dst {
namespace attn_window {

// Operands the tensor maps and 16-byte vectors can address: [B, T, heads, D] with
// unit inner stride, the other strides and the start multiples of 16 bytes.
bool addressable(const at::Tensor& x) {
  if (x.stride(3) != 1 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (x.size(i) != 1 && (x.stride(i) <= 0 || x.stride(i) % 8 != 0)) return false;
  return true;
}

at::Tensor as_addressable(const at::Tensor& x) {
  return addressable(x) ? x : x.clone(at::MemoryFormat::Contiguous);
}

Operand operand(const at::Tensor& x) {
  return {static_cast<__nv_bfloat16*>(x.data_ptr()), {x.stride(1), x.stride(2), x.stride(0)}};
}

// q, k or v of a buffer [B, T, heads, 3, D].
Operand part_of(const at::Tensor& qkv, int which, int64_t D) {
  return {static_cast<__nv_bfloat16*>(qkv.data_ptr()) + which * D, {qkv.stride(1), 3 * D, qkv.stride(0)}};
}

CUtensorMap map_of(const Operand& x, int64_t B, int64_t T, int64_t heads, int64_t D, int rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(T), static_cast<uint64_t>(heads),
                            static_cast<uint64_t>(B)};
  const int64_t st[3] = {x.s.t, x.s.h, x.s.b};
  uint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] == 1 ? 16 : static_cast<uint64_t>(st[i]) * 2;
  const uint32_t box[4] = {64, static_cast<uint32_t>(rows), 1, 1};
  return make_tmap_bf16_4d(x.p, dims, strides, box);
}

void check_bf16(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16, "window attention: ", name, " must be a CUDA bf16 tensor");
}

Shape shape_of(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t window, int64_t sinks) {
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "window attention: head_dim must be a multiple of 8 up to 128, got ",
              std::to_string(D));
  TORCH_CHECK(T >= 1 && T < (int64_t(1) << 30) && B >= 1, "window attention: T and B must be positive");
  TORCH_CHECK(H <= 65535 && B <= 65535, "window attention: more than 65535 heads or sequences");
  TORCH_CHECK(Hk >= 1 && H >= 1 && H % Hk == 0,
              "window attention: the number of query heads must be a multiple of the number of key heads");
  TORCH_CHECK(window >= 1 && sinks >= 0, "window attention: window >= 1 and sinks >= 0 required");
  Shape s;
  s.T = static_cast<int>(T);
  s.Tp = static_cast<int>((T + 127) / 128 * 128);
  s.H = static_cast<int>(H);
  s.G = static_cast<int>(H / Hk);
  s.D = static_cast<int>(D);
  s.W = static_cast<int>(std::min(window, T));
  s.S = static_cast<int>(std::min(sinks, T));
  const double sc = 1.0 / std::sqrt(static_cast<double>(D));
  s.scale = static_cast<float>(sc);
  s.scale_log2 = static_cast<float>(sc * 1.4426950408889634);
  s.status = status_ptr();
  return s;
}

template <int DP>
void run_fwd(const Operand& q, const Operand& k, const Operand& v, const Operand& out, float* lse, int64_t B,
             const Shape& s) {
  const int Hk = s.H / s.G;
  launch_fwd<DP>(map_of(q, B, s.T, s.H, s.D, 128), map_of(k, B, s.T, Hk, s.D, 64), map_of(v, B, s.T, Hk, s.D, 64),
                 map_of(out, B, s.T, s.H, s.D, 128), lse, B, s, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// Chunks of about a key block's own window, at least 8 blocks of queries, and no
// more of them than keep the sums within T rows.
SinkChunks plan_sinks(const Shape& s) {
  SinkChunks c = {0, 0, 0, 0, nullptr};
  const int last_block = (s.T - 1) >> 6;
  for (int k0 = 0; k0 < s.S && (last_window_query(s, k0) >> 6) < last_block; k0 += 128) ++c.blocks;
  if (c.blocks == 0) return c;
  c.rows = std::min(s.S, c.blocks * 128);
  const int far = last_block - (last_window_query(s, 0) >> 6), most = std::max(1, s.T / c.rows - 1);
  c.steps = std::max({8, (127 + s.W) / 64 + 1, (far + most - 1) / most});
  c.chunks = (far + c.steps - 1) / c.steps;
  return c;
}

template <int DP>
void run_bwd(__nv_bfloat16* dout, const Operand& q, const Operand& k, const Operand& v, __nv_bfloat16* out,
             const float* lse, float* di, const Operand& dq, const Operand& dk, const Operand& dv, int64_t B,
             const Shape& s, const at::TensorOptions& f32) {
  auto st = at::cuda::getCurrentCUDAStream();
  const int Hk = s.H / s.G;
  TORCH_CHECK(B * s.H * s.Tp * (DP / 8) / 256 < (int64_t(1) << 31) - 1, "window attention: too many rows");
  const Operand go = {dout, {static_cast<int64_t>(s.H) * s.D, s.D, static_cast<int64_t>(s.T) * s.H * s.D}};
  launch_rowdot<DP>(dout, out, di, B, s, st);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  SinkChunks sinks = plan_sinks(s);
  at::Tensor partial;
  if (sinks.blocks) {
    partial = at::empty({B * Hk * sinks.rows * (1 + sinks.chunks) * 2 * DP}, f32);
    sinks.partial = partial.data_ptr<float>();
  }
  const CUtensorMap k64 = map_of(k, B, s.T, Hk, s.D, 64), v64 = map_of(v, B, s.T, Hk, s.D, 64);
  launch_dkdv<DP>(map_of(q, B, s.T, s.H, s.D, 64), map_of(go, B, s.T, s.H, s.D, 64), map_of(k, B, s.T, Hk, s.D, 128),
                  map_of(v, B, s.T, Hk, s.D, 128), lse, di, map_of(dk, B, s.T, Hk, s.D, 128),
                  map_of(dv, B, s.T, Hk, s.D, 128), B, sinks, s, st);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  launch_dq<DP>(map_of(q, B, s.T, s.H, s.D, 128), map_of(go, B, s.T, s.H, s.D, 128), k64, v64, lse, di,
                map_of(dq, B, s.T, s.H, s.D, 128), dk, dv, B, sinks, s, st);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// out [B, T, H, D] and the base-2 log-sum-exp [B, H, T rounded up to 128].
std::pair<at::Tensor, at::Tensor> forward(const Operand& q, const Operand& k, const Operand& v, int64_t B,
                                          const Shape& s, const at::TensorOptions& options) {
  at::Tensor out = at::empty({B, s.T, s.H, s.D}, options);
  at::Tensor lse = at::empty({B, s.H, s.Tp}, options.dtype(at::kFloat));
  const Operand o = operand(out);
  if (s.D <= 64)
    run_fwd<64>(q, k, v, o, lse.data_ptr<float>(), B, s);
  else
    run_fwd<128>(q, k, v, o, lse.data_ptr<float>(), B, s);
  return {out, lse};
}

void backward(const at::Tensor& dout, const Operand& q, const Operand& k, const Operand& v, const at::Tensor& out,
              const at::Tensor& lse, const Operand& dq, const Operand& dk, const Operand& dv, int64_t B, const Shape& s) {
  at::Tensor go = dout.contiguous();
  if (reinterpret_cast<uintptr_t>(go.data_ptr()) % 16) go = go.clone();
  at::Tensor di = at::empty_like(lse);
  auto *g = static_cast<__nv_bfloat16*>(go.data_ptr()), *o = static_cast<__nv_bfloat16*>(out.data_ptr());
  if (s.D <= 64)
    run_bwd<64>(g, q, k, v, o, lse.data_ptr<float>(), di.data_ptr<float>(), dq, dk, dv, B, s, lse.options());
  else
    run_bwd<128>(g, q, k, v, o, lse.data_ptr<float>(), di.data_ptr<float>(), dq, dk, dv, B, s, lse.options());
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The gradients under create_graph: as they are, with a node that refuses to be
// differentiated. Without one they would count as constants, silently.
struct FirstOnly : public torch::autograd::Function<FirstOnly> {
  static variable_list forward(AutogradContext*, at::TensorList gradients, at::TensorList /*of what*/) {
    return gradients.vec();
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "window attention: no second derivative on CUDA bf16 tensors");
    return {};
  }
};

// Separate q, k, v. The autograd nodes are C++: a Python node costs more host
// time per call than a short sequence takes on the GPU.
struct SeparateFn : public torch::autograd::Function<SeparateFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                            int64_t window, int64_t sinks) {
    c10::cuda::CUDAGuard guard(q_.device());
    const int64_t B = q_.size(0), T = q_.size(1), D = q_.size(3);
    const Shape s = shape_of(B, T, q_.size(2), k_.size(2), D, window, sinks);
    const at::Tensor q = as_addressable(q_), k = as_addressable(k_), v = as_addressable(v_);
    auto [out, lse] = attn_window::forward(operand(q), operand(k), operand(v), B, s, q.options());
    ctx->save_for_backward({q, k, v, out, lse});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4];
    c10::cuda::CUDAGuard guard(q.device());
    const Shape s = shape_of(q.size(0), q.size(1), q.size(2), k.size(2), q.size(3), ctx->saved_data["window"].toInt(),
                             ctx->saved_data["sinks"].toInt());
    at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
               dv = at::empty(v.sizes(), v.options());
    attn_window::backward(grads[0], operand(q), operand(k), operand(v), out, lse, operand(dq), operand(dk), operand(dv),
                          q.size(0), s);
    debug_check("window_attention backward");
    variable_list g = {dq, dk, dv};
    if (at::GradMode::is_enabled()) {
      const variable_list of = {grads[0], q, k, v};
      g = FirstOnly::apply(at::TensorList(g), at::TensorList(of));
    }
    return {g[0], g[1], g[2], at::Tensor(), at::Tensor()};
  }
};

// q, k, v interleaved head by head in one buffer, and their gradients likewise.
struct FusedFn : public torch::autograd::Function<FusedFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& qkv_, int64_t n_head, int64_t head_dim,
                            int64_t window, int64_t sinks) {
    c10::cuda::CUDAGuard guard(qkv_.device());
    const int64_t B = qkv_.size(0), T = qkv_.size(1);
    const Shape s = shape_of(B, T, n_head, n_head, head_dim, window, sinks);
    at::Tensor qkv = qkv_.contiguous();
    if (reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16) qkv = qkv.clone();
    auto [out, lse] = attn_window::forward(part_of(qkv, 0, head_dim), part_of(qkv, 1, head_dim),
                                           part_of(qkv, 2, head_dim), B, s, qkv.options());
    ctx->save_for_backward({qkv, out, lse});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    return out.view({B, T, n_head * head_dim});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &qkv = saved[0], &out = saved[1], &lse = saved[2];
    c10::cuda::CUDAGuard guard(qkv.device());
    const int64_t B = out.size(0), D = out.size(3);
    const Shape s = shape_of(B, out.size(1), out.size(2), out.size(2), D, ctx->saved_data["window"].toInt(),
                             ctx->saved_data["sinks"].toInt());
    at::Tensor dqkv = at::empty(qkv.sizes(), qkv.options());
    attn_window::backward(grads[0], part_of(qkv, 0, D), part_of(qkv, 1, D), part_of(qkv, 2, D), out, lse,
                          part_of(dqkv, 0, D), part_of(dqkv, 1, D), part_of(dqkv, 2, D), B, s);
    debug_check("window_attention backward");
    if (at::GradMode::is_enabled()) {
      const variable_list of = {grads[0], qkv};
      dqkv = FirstOnly::apply(at::TensorList(dqkv), at::TensorList(of))[0];
    }
    return {dqkv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace attn_window
}  // namespace dst

using namespace dst;

// q [B, T, H, D], k and v [B, T, Hk, D], any strides -> [B, T, H, D], differentiable.
at::Tensor window_attention_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window,
                                int64_t sinks) {
  attn_window::check_bf16(q, "q");
  attn_window::check_bf16(k, "k");
  attn_window::check_bf16(v, "v");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == q.size(0) &&
                  k.size(1) == q.size(1) && k.size(3) == q.size(3),
              "window attention: q [B, T, H, D] and k, v [B, T, Hk, D] must agree");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(), "window attention: q, k, v on one device");
  return attn_window::SeparateFn::apply(q, k, v, window, sinks);
}

// qkv [B, T, n_head * 3 * head_dim] -> [B, T, n_head * head_dim], differentiable.
at::Tensor window_attention(const at::Tensor& qkv, int64_t n_head, int64_t head_dim, int64_t window, int64_t sinks) {
  attn_window::check_bf16(qkv, "qkv");
  TORCH_CHECK(qkv.dim() == 3 && n_head >= 1 && head_dim >= 1 && qkv.size(2) == 3 * n_head * head_dim,
              "window attention: qkv must be [B, T, n_head * 3 * head_dim]");
  return attn_window::FusedFn::apply(qkv, n_head, head_dim, window, sinks);
}

void register_attn_window(pybind11::module& m) {
  m.def("window_attention_qkv", &window_attention_qkv, "sliding-window attention with sinks", pybind11::arg("q"),
        pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("window"), pybind11::arg("sinks"));
  m.def("window_attention", &window_attention, "sliding-window attention with sinks over a fused qkv buffer",
        pybind11::arg("qkv"), pybind11::arg("n_head"), pybind11::arg("head_dim"), pybind11::arg("window"),
        pybind11::arg("sinks"));
}
