// layers::LinearAttention: MultiheadAttention's projections (in_proj_weight
// [E, 3E], in_proj_bias [1, 3E], out_proj_weight [E, E], out_proj_bias [1, E])
// around causal linear attention with a decay per head, optionally with rotary
// positions on q and k. Not in the reference.
#pragma once
#include "core/Sequence.h"
#include "layers/Module.h"

namespace layers {
class LinearAttention : public Module {
 public:
  // log_decay: one value a head (empty: -2^(-8 (h + 1) / H), from heads that forget within a
  // few tokens to heads that keep hundreds). rope.sections empty: no rotary positions.
  LinearAttention(uint32_t embed_dim, uint32_t num_heads, const std::vector<float>& log_decay,
                  const core::RopeSpec& rope);
  // without rotary positions
  std::shared_ptr<core::Tensor> forward(const std::shared_ptr<core::Tensor>& input) override;
  // positions [axes, N, L]; lengths [N] valid tokens (null: all)
  std::shared_ptr<core::Tensor> forward(const std::shared_ptr<core::Tensor>& input,
                                        const std::shared_ptr<core::IntTensor>& positions,
                                        const std::shared_ptr<core::IntTensor>& lengths);
  // A piece of a longer sequence (a prompt, a single new token): from state [N, H, D, D]
  // (null: the start) to {output, state after it}. Generation turns set_grad_enabled off: with it
  // on, the state keeps the graph of every piece before it, to be trained through.
  std::pair<std::shared_ptr<core::Tensor>, std::shared_ptr<core::Tensor>> forward_state(
      const std::shared_ptr<core::Tensor>& input, const std::shared_ptr<core::IntTensor>& positions,
      const std::shared_ptr<core::IntTensor>& lengths, const std::shared_ptr<core::Tensor>& state);
  std::vector<std::shared_ptr<core::Tensor>> parameters() override;

 private:
  std::pair<std::shared_ptr<core::Tensor>, std::shared_ptr<core::Tensor>> run(
      const std::shared_ptr<core::Tensor>& input, const std::shared_ptr<core::IntTensor>& positions,
      const std::shared_ptr<core::IntTensor>& lengths, const std::shared_ptr<core::Tensor>& state,
      bool want_state);
  std::shared_ptr<core::Tensor> in_proj_weight, in_proj_bias, out_proj_weight, out_proj_bias, log_decay;
  const uint32_t embed_dim;
  const uint32_t num_heads;
  const core::RopeSpec rope_spec;
};
}  // namespace layers
