// Layers and loss over core::Functional (reference: source/layers/*.cpp, source/loss/MSE.cpp).
#include <cmath>
#include <stdexcept>
#include <tuple>

#include "core/Functional.h"
#include "device_util.h"
#include "layers/LayerNorm.h"
#include "layers/LinearAttention.h"
#include "layers/Linear.h"
#include "layers/MHA.h"
#include "layers/ReLU.h"
#include "loss/MSE.h"

namespace layers {

namespace {
cudaStream_t stream() { return CudaContext::getStream(); }
std::shared_ptr<core::Tensor> param(std::vector<uint32_t> shape) {
  return std::make_shared<core::Tensor>(shape, true);
}
}  // namespace

// He-normal weights (std = sqrt(2 / fan_in)) and zero bias, as Linear.cpp:8-22.
Linear::Linear(uint32_t in_channels, uint32_t out_channels, bool relu_)
    : weight(param({in_channels, out_channels})), bias(param({1, out_channels})), relu(relu_) {
  core::pop_data_normal(weight, std::sqrt(2.0f / static_cast<float>(in_channels)), stream());
  core::pop_data_zeros(bias, stream());
}

// X W + bias in one fused projection (matmul and bias add of Linear.cpp:24-35).
std::shared_ptr<core::Tensor> Linear::forward(const std::shared_ptr<core::Tensor>& input) {
  std::vector<std::shared_ptr<core::Tensor>> out;
  core::linear(input, weight, bias, 1, out, stream(), relu);
  return out[0];
}

std::vector<std::shared_ptr<core::Tensor>> Linear::parameters() { return {weight, bias}; }

std::shared_ptr<core::Tensor> ReLU::forward(const std::shared_ptr<core::Tensor>& In) {
  return core::relu(In, stream());
}

LayerNorm::LayerNorm(uint32_t n, float eps)
    : gamma(param({1, n})), beta(param({1, n})), normalized_shape(n), epsilon(eps) {
  core::check_status(pa_fill(gamma->get_data_ptr(), n, 1.0f, core::ps(stream())), "LayerNorm init");
  core::pop_data_zeros(beta, stream());
}

std::shared_ptr<core::Tensor> LayerNorm::forward(const std::shared_ptr<core::Tensor>& input) {
  return core::layer_norm(input, gamma, beta, epsilon, stream());
}

std::pair<std::shared_ptr<core::Tensor>, std::shared_ptr<core::Tensor>> LayerNorm::forward_add(
    const std::shared_ptr<core::Tensor>& x, const std::shared_ptr<core::Tensor>& r) {
  return core::add_layer_norm(x, r, gamma, beta, epsilon, stream());
}

std::vector<std::shared_ptr<core::Tensor>> LayerNorm::parameters() { return {gamma, beta}; }

// Same parameter shapes and He-normal init as MHA.cpp:10-28.
MultiheadAttention::MultiheadAttention(uint32_t e, uint32_t h)
    : in_proj_weight(param({e, 3 * e})),
      in_proj_bias(param({1, 3 * e})),
      out_proj_weight(param({e, e})),
      out_proj_bias(param({1, e})),
      embed_dim(e),
      num_heads(h) {
  const float std_dev = std::sqrt(2.0f / static_cast<float>(e));
  core::pop_data_normal(in_proj_weight, std_dev, stream());
  core::pop_data_zeros(in_proj_bias, stream());
  core::pop_data_normal(out_proj_weight, std_dev, stream());
  core::pop_data_zeros(out_proj_bias, stream());
}

// Self-attention: the in-projection writes Q, K, V directly (bias added in the
// GEMM epilogue) and the out-projection adds its bias the same way - the
// reference's matmul / bias add / split passes (MHA.cpp:50-77) fused.
std::shared_ptr<core::Tensor> MultiheadAttention::forward(const std::shared_ptr<core::Tensor>& x) {
  std::vector<std::shared_ptr<core::Tensor>> qkv, out;
  std::shared_ptr<core::Tensor> attn;
  core::linear(x, in_proj_weight, in_proj_bias, 3, qkv, stream());
  core::flash_attention(qkv[0], qkv[1], qkv[2], attn, static_cast<int>(num_heads), stream());
  core::linear(attn, out_proj_weight, out_proj_bias, 1, out, stream());
  return out[0];
}

std::shared_ptr<core::Tensor> MultiheadAttention::forward(const std::shared_ptr<core::Tensor>& q,
                                                          const std::shared_ptr<core::Tensor>& k,
                                                          const std::shared_ptr<core::Tensor>& v) {
  // forward(x, x, x) (how the reference's denoise layer calls it) is self-attention
  if (q == k && k == v) return forward(q);
  std::vector<std::shared_ptr<core::Tensor>> w, b;
  core::split(in_proj_weight, 3, 1, w, stream());
  core::split(in_proj_bias, 3, 1, b, stream());
  std::shared_ptr<core::Tensor> t[3], p[3], attn, o1, out;
  const std::shared_ptr<core::Tensor>* in[3] = {&q, &k, &v};
  for (int i = 0; i < 3; ++i) {
    core::matmul(*in[i], w[i], t[i], stream());
    core::matadd(t[i], b[i], p[i], stream());
  }
  core::flash_attention(p[0], p[1], p[2], attn, static_cast<int>(num_heads), stream());
  core::matmul(attn, out_proj_weight, o1, stream());
  core::matadd(o1, out_proj_bias, out, stream());
  return out;
}

std::vector<std::shared_ptr<core::Tensor>> MultiheadAttention::parameters() {
  return {in_proj_weight, in_proj_bias, out_proj_weight, out_proj_bias};
}

namespace {
uint32_t dividing(uint32_t e, uint32_t h) {
  if (h == 0 || e == 0 || e % h)
    throw std::runtime_error("LinearAttention: embedding dim not divisible by num_heads");
  return e;
}
}  // namespace

LinearAttention::LinearAttention(uint32_t e, uint32_t h, const std::vector<float>& decay,
                                 const core::RopeSpec& rope)
    : in_proj_weight(param({dividing(e, h), 3 * e})),
      in_proj_bias(param({1, 3 * e})),
      out_proj_weight(param({e, e})),
      out_proj_bias(param({1, e})),
      log_decay(std::make_shared<core::Tensor>(std::vector<uint32_t>{h}, false)),
      embed_dim(e),
      num_heads(h),
      rope_spec(rope) {
  if (!decay.empty() && decay.size() != h)
    throw std::runtime_error("LinearAttention: one log decay per head");
  std::vector<float> l(decay);
  if (l.empty())
    for (uint32_t i = 0; i < h; ++i)
      l.push_back(-std::exp2(-8.0f * static_cast<float>(i + 1) / static_cast<float>(h)));
  log_decay->to_device(l);
  const float std_dev = std::sqrt(2.0f / static_cast<float>(e));
  core::pop_data_normal(in_proj_weight, std_dev, stream());
  core::pop_data_zeros(in_proj_bias, stream());
  core::pop_data_normal(out_proj_weight, std_dev, stream());
  core::pop_data_zeros(out_proj_bias, stream());
}

std::pair<std::shared_ptr<core::Tensor>, std::shared_ptr<core::Tensor>> LinearAttention::run(
    const std::shared_ptr<core::Tensor>& x, const std::shared_ptr<core::IntTensor>& positions,
    const std::shared_ptr<core::IntTensor>& lengths, const std::shared_ptr<core::Tensor>& state,
    bool want_state) {
  if (rope_spec.sections.empty() != (positions == nullptr))
    throw std::runtime_error("LinearAttention: positions go with rotary sections");
  std::vector<std::shared_ptr<core::Tensor>> qkv, out;
  core::linear(x, in_proj_weight, in_proj_bias, 3, qkv, stream());
  if (positions)
    std::tie(qkv[0], qkv[1]) = core::rope(qkv[0], qkv[1], static_cast<int>(embed_dim / num_heads),
                                          rope_spec, positions, stream());
  auto [o, after] = core::linear_attention(qkv[0], qkv[1], qkv[2], static_cast<int>(num_heads),
                                           log_decay, lengths, state, want_state, stream());
  core::linear(o, out_proj_weight, out_proj_bias, 1, out, stream());
  return {out[0], after};
}

std::shared_ptr<core::Tensor> LinearAttention::forward(const std::shared_ptr<core::Tensor>& x) {
  return run(x, nullptr, nullptr, nullptr, false).first;
}

std::shared_ptr<core::Tensor> LinearAttention::forward(
    const std::shared_ptr<core::Tensor>& x, const std::shared_ptr<core::IntTensor>& positions,
    const std::shared_ptr<core::IntTensor>& lengths) {
  return run(x, positions, lengths, nullptr, false).first;
}

std::pair<std::shared_ptr<core::Tensor>, std::shared_ptr<core::Tensor>>
LinearAttention::forward_state(const std::shared_ptr<core::Tensor>& x,
                               const std::shared_ptr<core::IntTensor>& positions,
                               const std::shared_ptr<core::IntTensor>& lengths,
                               const std::shared_ptr<core::Tensor>& state) {
  return run(x, positions, lengths, state, true);
}

std::vector<std::shared_ptr<core::Tensor>> LinearAttention::parameters() {
  return {in_proj_weight, in_proj_bias, out_proj_weight, out_proj_bias};
}

}  // namespace layers

namespace loss {
std::shared_ptr<core::Tensor> MSE::forward(const std::shared_ptr<core::Tensor>& predictions,
                                           const std::shared_ptr<core::Tensor>& targets) {
  return core::mse_loss(predictions, targets, CudaContext::getStream());
}
}  // namespace loss
