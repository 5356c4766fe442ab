// Operators over the positions of a sequence: rotary positions and linear
// attention with a decay per head (pa_rope_*, pa_linear_attn_*), with their
// graph nodes. Neither is in the reference, whose attention knows no positions
// and no order; they take the same [N, L, E] tensors as core::flash_attention.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include <memory>
#include <utility>
#include <vector>
#include "core/Autograd.h"
#include "core/Tensor.h"

namespace core {

// A device array of 32-bit whole numbers (positions, lengths), filled once.
class IntTensor {
 public:
  IntTensor(const std::vector<uint32_t>& shape, const std::vector<int32_t>& values);
  ~IntTensor();
  IntTensor(const IntTensor&) = delete;
  IntTensor& operator=(const IntTensor&) = delete;
  std::vector<uint32_t> get_shape() const { return shape; }
  const int32_t* get_data_ptr() const { return data_ptr; }

 private:
  std::vector<uint32_t> shape;
  int32_t* data_ptr = nullptr;
};

// How heads turn: pairs of each position axis, and the forms of pa_rope_desc.
struct RopeSpec {
  std::vector<int32_t> sections;
  double base = 10000.0;
  int layout = 0;  // pa_rope_layout
  int freqs = 0;   // pa_rope_freqs
};

// (turn(Q), turn(K)) of Q [N, L, H head_dim] and K [N, L, Hk head_dim] by
// positions [axes, N, L], in one launch.
std::pair<std::shared_ptr<Tensor>, std::shared_ptr<Tensor>> rope(
    const std::shared_ptr<Tensor>& Q, const std::shared_ptr<Tensor>& K, int head_dim,
    const RopeSpec& spec, const std::shared_ptr<IntTensor>& positions, const cudaStream_t& stream);

// Causal linear attention of Q, K, V [N, L, E] with decay exp(log_decay[h]) (a constant [H]; no
// gradient), over the first lengths[n] tokens of each sequence (null: all), from
// state [N, H, D, D] (null: zero). Returns {O, the state after the last token};
// the second is null unless want_state. One new token without gradients (set_grad_enabled)
// takes the single-token kernel.
std::pair<std::shared_ptr<Tensor>, std::shared_ptr<Tensor>> linear_attention(
    const std::shared_ptr<Tensor>& Q, const std::shared_ptr<Tensor>& K,
    const std::shared_ptr<Tensor>& V, int num_heads, const std::shared_ptr<Tensor>& log_decay,
    const std::shared_ptr<IntTensor>& lengths, const std::shared_ptr<Tensor>& state,
    bool want_state, const cudaStream_t& stream);

// dQ += turn^-1(dQ'), dK += turn^-1(dK') (written outright where nothing has
// written them yet); an output that no gradient reached adds nothing.
struct RopeFunction : public Function {
  std::shared_ptr<Tensor> Q_input, K_input;
  std::weak_ptr<Tensor> Q_output, K_output;
  int head_dim;
  RopeSpec spec;
  std::shared_ptr<IntTensor> positions;
  RopeFunction(std::shared_ptr<Tensor> q, std::shared_ptr<Tensor> k, const std::shared_ptr<Tensor>& qo,
               const std::shared_ptr<Tensor>& ko, int head_dim_, RopeSpec spec_,
               std::shared_ptr<IntTensor> pos);
  void apply_backward() override;
  std::vector<std::shared_ptr<Tensor>> inputs() const override { return {Q_input, K_input}; }
};

struct LinearAttentionFunction : public Function {
  std::shared_ptr<Tensor> Q_input, K_input, V_input, state_input;  // state_input may be null
  std::weak_ptr<Tensor> O_output, state_output;
  std::shared_ptr<Tensor> log_decay;
  std::shared_ptr<IntTensor> lengths;
  int num_heads;
  int math_mode;  // the forward's f32 math mode, which the backward uses too
  void apply_backward() override;
  std::vector<std::shared_ptr<Tensor>> inputs() const override {
    if (state_input) return {Q_input, K_input, V_input, state_input};
    return {Q_input, K_input, V_input};
  }
};

}  // namespace core
