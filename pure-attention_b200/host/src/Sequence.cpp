#include "core/Sequence.h"

#include <stdexcept>
#include <string>

#include "device_util.h"

namespace core {

namespace {
cudaStream_t stream() { return CudaContext::getStream(); }

pa_attn_desc attn_desc(const Tensor& q, int num_heads) {
  const auto sh = q.get_shape();
  return pa_attn_desc{static_cast<int32_t>(sh[0]), static_cast<int32_t>(sh[1]), num_heads,
                      static_cast<int32_t>(sh[2]) / num_heads, PA_F32, 0.f};
}

pa_rope_desc rope_desc(const std::vector<uint32_t>& shape, int heads, int kv_heads, int head_dim,
                       const RopeSpec& spec) {
  pa_rope_desc d{};
  d.batch = static_cast<int32_t>(shape[0]);
  d.seq_len = static_cast<int32_t>(shape[1]);
  d.num_heads = heads;
  d.num_kv_heads = kv_heads;
  d.head_dim = head_dim;
  d.dtype = PA_F32;
  d.layout = spec.layout;
  d.freqs = spec.freqs;
  d.axes = static_cast<int32_t>(spec.sections.size());
  for (size_t a = 0; a < spec.sections.size(); ++a) d.sections[a] = spec.sections[a];
  d.base = spec.base;
  return d;
}
}  // namespace

IntTensor::IntTensor(const std::vector<uint32_t>& shape_, const std::vector<int32_t>& values)
    : shape(shape_) {
  size_t n = 1;
  for (uint32_t s : shape) n *= s;
  if (n != values.size() || n == 0) throw std::runtime_error("IntTensor: values must fill the shape");
  void* p = nullptr;
  retain_pool_memory();
  if (cudaMallocAsync(&p, n * sizeof(int32_t), stream()) != cudaSuccess)
    throw std::runtime_error("IntTensor: cannot allocate device memory");
  data_ptr = static_cast<int32_t*>(p);
  if (cudaMemcpyAsync(data_ptr, values.data(), n * sizeof(int32_t), cudaMemcpyHostToDevice, stream()) !=
          cudaSuccess ||
      cudaStreamSynchronize(stream()) != cudaSuccess) {
    cudaFreeAsync(data_ptr, stream());
    throw std::runtime_error("IntTensor: copy to the device failed");
  }
}

IntTensor::~IntTensor() { cudaFreeAsync(data_ptr, CudaContext::getStream()); }

std::pair<std::shared_ptr<Tensor>, std::shared_ptr<Tensor>> rope(
    const std::shared_ptr<Tensor>& Q, const std::shared_ptr<Tensor>& K, int head_dim,
    const RopeSpec& spec, const std::shared_ptr<IntTensor>& positions, const cudaStream_t& s) {
  const auto q = Q->get_shape(), k = K->get_shape();
  if (q.size() != 3 || k.size() != 3 || q[0] != k[0] || q[1] != k[1])
    throw std::runtime_error("Rope: Q, K must be [N, L, E] of the same N and L");
  if (head_dim <= 0 || q[2] % head_dim || k[2] % head_dim || q[2] == 0 || k[2] == 0)
    throw std::runtime_error("Rope: embedding dim not divisible by the head dim");
  if (spec.sections.empty() || spec.sections.size() > PA_ROPE_MAX_AXES)
    throw std::runtime_error("Rope: 1 to 4 position axes");
  if (!positions || positions->get_shape() !=
                        std::vector<uint32_t>{static_cast<uint32_t>(spec.sections.size()), q[0], q[1]})
    throw std::runtime_error("Rope: positions must be [axes, N, L]");
  const bool g = grad_enabled() && (Q->requires_grad() || K->requires_grad());
  auto Qo = std::make_shared<Tensor>(q, g, false);
  auto Ko = std::make_shared<Tensor>(k, g, false);
  const pa_rope_desc d = rope_desc(q, static_cast<int>(q[2]) / head_dim,
                                   static_cast<int>(k[2]) / head_dim, head_dim, spec);
  check_status(pa_rope_fwd(&d, Q->get_data_ptr(), K->get_data_ptr(), positions->get_data_ptr(),
                           Qo->get_data_ptr(), Ko->get_data_ptr(), ps(s)),
               "Rope");
  if (g) {
    auto node = std::make_shared<RopeFunction>(Q, K, Qo, Ko, head_dim, spec, positions);
    Qo->set_grad_fn(node);
    Ko->set_grad_fn(node);
  }
  return {Qo, Ko};
}

RopeFunction::RopeFunction(std::shared_ptr<Tensor> q, std::shared_ptr<Tensor> k,
                           const std::shared_ptr<Tensor>& qo, const std::shared_ptr<Tensor>& ko,
                           int head_dim_, RopeSpec spec_, std::shared_ptr<IntTensor> pos)
    : Q_input(std::move(q)), K_input(std::move(k)), Q_output(qo), K_output(ko), head_dim(head_dim_),
      spec(std::move(spec_)), positions(std::move(pos)) {}

void RopeFunction::apply_backward() {
  auto Qo = Q_output.lock(), Ko = K_output.lock();
  const float* dq = Q_input->requires_grad() ? grad_in(Qo) : nullptr;
  const float* dk = K_input->requires_grad() ? grad_in(Ko) : nullptr;
  const auto q = Q_input->get_shape(), k = K_input->get_shape();
  const int hq = static_cast<int>(q[2]) / head_dim, hk = static_cast<int>(k[2]) / head_dim;
  const int32_t* pos = positions->get_data_ptr();
  // one launch where both are written the same way into different tensors
  if (dq && dk && Q_input != K_input &&
      Q_input->gradient_unwritten() == K_input->gradient_unwritten()) {
    bool fresh = false;
    float* gq = Q_input->gradient_for_write(&fresh);
    float* gk = K_input->gradient_for_write(&fresh);
    const pa_rope_desc d = rope_desc(q, hq, hk, head_dim, spec);
    check_status(pa_rope_bwd(&d, dq, dk, pos, gq, gk, fresh ? 0 : 1, ps(stream())), "Rope backward");
    return;
  }
  auto one = [&](const Tensor& in, const float* dy, int heads) {
    if (!dy) return;
    bool fresh = false;
    float* g = in.gradient_for_write(&fresh);
    const pa_rope_desc d = rope_desc(q, heads, 0, head_dim, spec);
    check_status(pa_rope_bwd(&d, dy, nullptr, pos, g, nullptr, fresh ? 0 : 1, ps(stream())),
                 "Rope backward");
  };
  one(*Q_input, dq, hq);
  one(*K_input, dk, hk);
}

std::pair<std::shared_ptr<Tensor>, std::shared_ptr<Tensor>> linear_attention(
    const std::shared_ptr<Tensor>& Q, const std::shared_ptr<Tensor>& K,
    const std::shared_ptr<Tensor>& V, int num_heads, const std::shared_ptr<Tensor>& log_decay,
    const std::shared_ptr<IntTensor>& lengths, const std::shared_ptr<Tensor>& state,
    bool want_state, const cudaStream_t& s) {
  const auto sh = Q->get_shape();
  if (sh.size() != 3 || K->get_shape() != sh || V->get_shape() != sh)
    throw std::runtime_error("LinearAttention: Q, K, V must share a [N, L, E] shape");
  if (num_heads <= 0 || sh[2] % num_heads)
    throw std::runtime_error("LinearAttention: embedding dim not divisible by num_heads");
  if (log_decay->numel() != static_cast<size_t>(num_heads))
    throw std::runtime_error("LinearAttention: one log decay per head");
  if (log_decay->requires_grad())
    throw std::runtime_error("LinearAttention: the decay is a constant (no gradient)");
  if (lengths && lengths->get_shape() != std::vector<uint32_t>{sh[0]})
    throw std::runtime_error("LinearAttention: lengths must be [N]");
  const uint32_t H = static_cast<uint32_t>(num_heads), D = sh[2] / H;
  const std::vector<uint32_t> state_shape{sh[0], H, D, D};
  if (state && state->get_shape() != state_shape)
    throw std::runtime_error("LinearAttention: the state must be [N, H, D, D]");
  const bool g = grad_enabled() && (Q->requires_grad() || K->requires_grad() || V->requires_grad() ||
                                    (state && state->requires_grad()));
  auto O = std::make_shared<Tensor>(sh, g, false);
  std::shared_ptr<Tensor> out;
  if (want_state) out = std::make_shared<Tensor>(state_shape, g, false);
  const pa_attn_desc d = attn_desc(*Q, num_heads);
  int st;
  if (sh[1] == 1 && !g && state && out && !lengths) {
    // one new token (2.3 us; as a chunk of one token 9 us; 8 heads of 64 in fp32)
    st = pa_linear_attn_step(&d, Q->get_data_ptr(), K->get_data_ptr(), V->get_data_ptr(),
                             log_decay->get_data_ptr(), state->get_data_ptr(), O->get_data_ptr(),
                             out->get_data_ptr(), ps(s));
  } else {
    Scratch ws(pa_linear_attn_fwd_workspace_size(&d), s);
    st = pa_linear_attn_fwd(&d, Q->get_data_ptr(), K->get_data_ptr(), V->get_data_ptr(),
                            log_decay->get_data_ptr(), lengths ? lengths->get_data_ptr() : nullptr,
                            state ? state->get_data_ptr() : nullptr, O->get_data_ptr(),
                            out ? out->get_data_ptr() : nullptr, ws.get(), ws.size(), ps(s));
  }
  if (st == PA_ERR_UNSUPPORTED)
    throw std::runtime_error("LinearAttention: Unsupported Head Dimension");
  check_status(st, "LinearAttention");
  if (g) {
    auto node = std::make_shared<LinearAttentionFunction>();
    node->Q_input = Q;
    node->K_input = K;
    node->V_input = V;
    node->state_input = state;
    node->O_output = O;
    if (out) node->state_output = out;
    node->log_decay = log_decay;
    node->lengths = lengths;
    node->num_heads = num_heads;
    node->math_mode = pa_get_f32_math();
    O->set_grad_fn(node);
    if (out) out->set_grad_fn(node);
  }
  return {O, out};
}

// Gradients go straight into Q/K/V's grads, as in FlashAttentionFunction.
void LinearAttentionFunction::apply_backward() {
  const float* dO = grad_in(O_output.lock());
  const float* dS = grad_in(state_output.lock());
  if (!dO && !dS) return;
  const size_t n = Q_input->numel(), bytes = n * sizeof(float);
  Scratch zeros(dO ? 0 : bytes, stream());  // only the state has a gradient
  if (!dO) {
    cudaMemsetAsync(zeros.get(), 0, bytes, stream());
    dO = static_cast<const float*>(zeros.get());
  }
  const pa_attn_desc d = attn_desc(*Q_input, num_heads);
  Scratch ws(pa_linear_attn_bwd_workspace_size(&d), stream());
  const bool state_grad = state_input && state_input->requires_grad();
  const size_t sn = state_grad ? state_input->numel() : 0;
  Scratch ds(sn * sizeof(float), stream());
  auto run = [&](void* dq, void* dk, void* dv, int accumulate) {
    const int mode = pa_get_f32_math();
    pa_set_f32_math(math_mode);
    const int st = pa_linear_attn_bwd(
        &d, Q_input->get_data_ptr(), K_input->get_data_ptr(), V_input->get_data_ptr(), dO,
        log_decay->get_data_ptr(), lengths ? lengths->get_data_ptr() : nullptr,
        state_input ? state_input->get_data_ptr() : nullptr, dS, dq, dk, dv,
        static_cast<float*>(ds.get()), accumulate, ws.get(), ws.size(), ps(stream()));
    pa_set_f32_math(mode);
    check_status(st, "LinearAttention Backward");
  };
  const std::shared_ptr<Tensor>* qkv[3] = {&Q_input, &K_input, &V_input};
  const bool shared = Q_input == K_input || K_input == V_input || Q_input == V_input;
  bool all = true;
  for (auto* t : qkv) all = all && (*t)->requires_grad();
  // one tensor in several roles, or one without a gradient: separate buffers first
  Scratch g3(shared || !all ? 3 * bytes : 0, stream());
  if (shared || !all) {
    float* gp = static_cast<float*>(g3.get());
    run(gp, gp + n, gp + 2 * n, 0);
    for (int i = 0; i < 3; ++i)
      if ((*qkv[i])->requires_grad()) add_into(**qkv[i], gp + i * n, n, "LinearAttention Backward");
  } else {
    float* dst[3];
    bool unwritten[3], fresh = true;
    for (int i = 0; i < 3; ++i) {
      dst[i] = (*qkv[i])->gradient_for_write(&unwritten[i]);
      fresh = fresh && unwritten[i];
    }
    if (!fresh)
      for (int i = 0; i < 3; ++i)
        if (unwritten[i]) cudaMemsetAsync(dst[i], 0, bytes, stream());
    run(dst[0], dst[1], dst[2], fresh ? 0 : 1);
  }
  if (state_grad)
    add_into(*state_input, static_cast<const float*>(ds.get()), sn, "LinearAttention Backward");
}

}  // namespace core
