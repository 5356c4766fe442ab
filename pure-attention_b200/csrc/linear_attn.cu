// Causal linear attention with a decay per head: forward, backward and the
// single-token step.
//
//   S_t = l S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t        (l = exp(log_decay[h]))
//
// over the valid tokens of each sequence, from a carried state S_0 (or zero) to
// the state after the last token. With U_t = l U_{t+1} + scale q_t dO_t^T the
// gradients are dq_t = scale S_t dO_t, dk_t = U_t v_t, dv_t = U_t^T k_t: each is
// the same recurrence on other tensors, dq forward in time on (dO, v, k), dv on
// (k, q, dO) and dk on (v, dO, q) backward in time. One kernel therefore serves
// all four, with the order of the tokens and the form of the carried state as
// arguments (MixDir).
#include <cuda_bf16.h>
#include "host_launchers.h"

namespace pa {
namespace {

__device__ __forceinline__ float ld_f(const float* p) { return *p; }
__device__ __forceinline__ float ld_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void st_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// log2 of the decay. A decay of zero (log -inf) is held as 2^-10000, so that
// its power 0 is 1 and every other power is 0.
__device__ __forceinline__ float log2_decay(const float* log_decay, int h) {
  const float l = log_decay[h] * kLog2e;
  return l < -10000.f ? -10000.f : l;
}

__device__ __forceinline__ int valid_tokens(const int32_t* lens, int b, int L) {
  if (!lens) return L;
  const int n = lens[b];
  return n < 0 ? 0 : (n > L ? L : n);
}

// Thread e holds column e of the state (D values) and walks the tokens.
template <typename T, int D>
__global__ void __launch_bounds__(D)
    mix_scan_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* o,
                    const float* __restrict__ log_decay, const int32_t* __restrict__ lens,
                    const float* s_in, float* s_out, int L, int H, float scale, MixDir dir) {
  __shared__ float sq[D], sk[D];
  const int h = blockIdx.x % H, b = blockIdx.x / H, e = threadIdx.x;
  const int n = valid_tokens(lens, b, L);
  const float lam = exp2f(log2_decay(log_decay, h));
  const size_t st0 = static_cast<size_t>(blockIdx.x) * D * D;
  float S[D];
#pragma unroll
  for (int d = 0; d < D; ++d)
    S[d] = s_in ? dir.in_mult * s_in[st0 + (dir.transposed ? e * D + d : d * D + e)] : 0.f;
  for (int p = 0; p < n; ++p) {
    const int t = dir.reverse ? n - 1 - p : p;
    const size_t at = ((static_cast<size_t>(b) * L + t) * H + h) * D + e;
    __syncthreads();
    sq[e] = ld_f(q + at);
    sk[e] = ld_f(k + at);
    const float ve = ld_f(v + at);
    __syncthreads();
    const float w = p == 0 && dir.lead ? 1.f : lam;
    float acc = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) {
      S[d] = fmaf(w, S[d], sk[d] * ve);
      acc = fmaf(sq[d], S[d], acc);
    }
    st_f(o + at, (dir.accumulate ? ld_f(o + at) : 0.f) + scale * acc);
  }
  if (!dir.accumulate)
    for (int t = n; t < L; ++t) st_f(o + ((static_cast<size_t>(b) * L + t) * H + h) * D + e, 0.f);
  if (s_out) {
    const float w = dir.out_mult * (dir.lead && n > 0 ? lam : 1.f);
#pragma unroll
    for (int d = 0; d < D; ++d)
      s_out[st0 + (dir.transposed ? e * D + d : d * D + e)] = w * S[d];
  }
}

// One new token: a block per (sequence, head); each warp takes rows of the
// state, lanes take 16 bytes of columns.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    mix_step_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                    const float* __restrict__ log_decay, const float* s_in, T* __restrict__ o, float* s_out,
                    int H, float scale) {
  constexpr int CV = D / 4, RPI = 256 / CV, ROWS = D / RPI;  // vectors a row, rows a pass, passes
  __shared__ float4 part[256];
  const int bh = blockIdx.x, h = bh % H;
  const int c = threadIdx.x % CV, r0 = threadIdx.x / CV;
  const size_t st0 = static_cast<size_t>(bh) * D * D, at = static_cast<size_t>(bh) * D;
  float4 s[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
    s[i] = reinterpret_cast<const float4*>(s_in + st0)[(r0 + i * RPI) * CV + c];
  const float lam = exp2f(log2_decay(log_decay, h));
  float ve[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) ve[j] = ld_f(v + at + 4 * c + j);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int d = r0 + i * RPI;
    const float kd = ld_f(k + at + d), qd = ld_f(q + at + d);
    s[i].x = fmaf(lam, s[i].x, kd * ve[0]);
    s[i].y = fmaf(lam, s[i].y, kd * ve[1]);
    s[i].z = fmaf(lam, s[i].z, kd * ve[2]);
    s[i].w = fmaf(lam, s[i].w, kd * ve[3]);
    reinterpret_cast<float4*>(s_out + st0)[d * CV + c] = s[i];
    acc.x = fmaf(qd, s[i].x, acc.x);
    acc.y = fmaf(qd, s[i].y, acc.y);
    acc.z = fmaf(qd, s[i].z, acc.z);
    acc.w = fmaf(qd, s[i].w, acc.w);
  }
  part[threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.x < D) {  // fixed order: the same bits every time
    const float* p = reinterpret_cast<const float*>(part);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < RPI; ++i) sum += p[i * D + threadIdx.x];
    st_f(o + at + threadIdx.x, scale * sum);
  }
}

template <typename T, int D>
int mix(const AttnShape& sh, const void* q, const void* k, const void* v, void* o, const float* log_decay,
        const int32_t* lens, const float* s_in, float* s_out, const MixDir& dir, cudaStream_t s) {
  mix_scan_kernel<T, D><<<sh.B * sh.H, D, 0, s>>>(
      static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), static_cast<T*>(o),
      log_decay, lens, s_in, s_out, sh.L, sh.H, sh.scale, dir);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

int mix_any(const AttnShape& sh, bool f32, const void* q, const void* k, const void* v, void* o,
            const float* log_decay, const int32_t* lens, const float* s_in, float* s_out,
            const MixDir& dir, cudaStream_t s) {
  if (f32)
    return sh.D == 32 ? mix<float, 32>(sh, q, k, v, o, log_decay, lens, s_in, s_out, dir, s)
                      : mix<float, 64>(sh, q, k, v, o, log_decay, lens, s_in, s_out, dir, s);
  return sh.D == 64 ? mix<__nv_bfloat16, 64>(sh, q, k, v, o, log_decay, lens, s_in, s_out, dir, s)
                    : mix<__nv_bfloat16, 128>(sh, q, k, v, o, log_decay, lens, s_in, s_out, dir, s);
}

template <typename T, int D>
int step(const AttnShape& sh, const void* q, const void* k, const void* v, const float* log_decay,
         const float* s_in, void* o, float* s_out, cudaStream_t s) {
  mix_step_kernel<T, D><<<sh.B * sh.H, 256, 0, s>>>(static_cast<const T*>(q), static_cast<const T*>(k),
                                                    static_cast<const T*>(v), log_decay, s_in,
                                                    static_cast<T*>(o), s_out, sh.H, sh.scale);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // namespace

size_t linear_attn_workspace_bytes(const AttnShape&, bool, bool) { return 0; }

int launch_linear_attn_fwd(const AttnShape& sh, bool f32, const void* q, const void* k, const void* v,
                           const float* log_decay, const int32_t* lens, const float* s_in, void* o,
                           float* s_out, void*, uint32_t*, cudaStream_t s) {
  return mix_any(sh, f32, q, k, v, o, log_decay, lens, s_in, s_out, MixDir{}, s);
}

int launch_linear_attn_bwd(const AttnShape& sh, bool f32, const void* q, const void* k, const void* v,
                           const void* dO, const float* log_decay, const int32_t* lens,
                           const float* s_in, const float* ds_out, void* dq, void* dk, void* dv,
                           float* ds_in, bool accumulate, void*, uint32_t*, cudaStream_t s) {
  MixDir d;
  d.accumulate = accumulate;
  d.transposed = true;
  int st = mix_any(sh, f32, dO, v, k, dq, log_decay, lens, s_in, nullptr, d, s);
  if (st != PA_OK) return st;
  d.reverse = true;
  d.lead = 1;
  d.in_mult = 1.f / sh.scale;
  d.out_mult = sh.scale;
  st = mix_any(sh, f32, v, dO, q, dk, log_decay, lens, ds_out, nullptr, d, s);
  if (st != PA_OK) return st;
  d.transposed = false;
  return mix_any(sh, f32, k, q, dO, dv, log_decay, lens, ds_out, ds_in, d, s);
}

int launch_linear_attn_step(const AttnShape& sh, bool f32, const void* q, const void* k, const void* v,
                            const float* log_decay, const float* s_in, void* o, float* s_out,
                            cudaStream_t s) {
  if (f32)
    return sh.D == 32 ? step<float, 32>(sh, q, k, v, log_decay, s_in, o, s_out, s)
                      : step<float, 64>(sh, q, k, v, log_decay, s_in, o, s_out, s);
  return sh.D == 64 ? step<__nv_bfloat16, 64>(sh, q, k, v, log_decay, s_in, o, s_out, s)
                    : step<__nv_bfloat16, 128>(sh, q, k, v, log_decay, s_in, o, s_out, s);
}

}  // namespace pa
