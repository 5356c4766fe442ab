// Gradients of causal attention over packed sequences with shared key-value heads.
#include <cuda_bf16.h>
#include "host_launchers.h"

namespace pa {
namespace {

using bf16 = __nv_bfloat16;

// First and one past the last token of the sequence that holds token t (first = last: none).
__device__ __forceinline__ int2 sequence_of(const int32_t* cu, int n, int T, int t) {
  int before = min(max(cu[0], 0), T);
  for (int i = 0; i < n; ++i) {
    const int end = min(max(cu[i + 1], before), T);
    if (t >= before && t < end) return make_int2(before, end);
    before = end;
  }
  return make_int2(0, 0);
}

template <int N>
__device__ __forceinline__ void row(const bf16* p, float (&x)[N]) {
  for (int i = 0; i < N; ++i) x[i] = __bfloat162float(p[(threadIdx.x & 31) + 32 * i]);
}
template <int N>
__device__ __forceinline__ float dot(const float (&x)[N], const float (&y)[N]) {
  float s = 0.f;
  for (int i = 0; i < N; ++i) s += x[i] * y[i];
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  return s;
}
template <int N>
__device__ __forceinline__ void put(bf16* p, const float (&x)[N], bool add) {
  for (int i = 0; i < N; ++i) {
    bf16* at = p + (threadIdx.x & 31) + 32 * i;
    *at = __float2bfloat16_rn(x[i] + (add ? __bfloat162float(*at) : 0.f));
  }
}

template <int D>
__global__ void packed_dq_kernel(const PackedShape sh, const bf16* q, const bf16* k, const bf16* v, const bf16* o,
                                 const bf16* dO, const float* lse, const int32_t* cu, bf16* dq, float* delta, bool add) {
  const int t = blockIdx.x * 4 + threadIdx.x / 32, h = blockIdx.y, kh = h / (sh.H / sh.Hk);
  if (t >= sh.T) return;
  const int2 seq = sequence_of(cu, sh.n, sh.T, t);
  if (seq.x == seq.y) return;
  constexpr int N = D / 32;
  float x[N], y[N], g[N], acc[N] = {};
  const size_t at = (static_cast<size_t>(t) * sh.H + h) * D;
  row(o + at, y);
  row(dO + at, g);
  const float dl = dot(g, y), z = lse[static_cast<size_t>(h) * sh.T + t];
  row(q + t * sh.q_stride + h * D, x);
  for (int j = seq.x; j <= t; ++j) {
    row(k + j * sh.k_stride + kh * D, y);
    const float p = __expf(sh.scale * dot(x, y) - z);
    float w[N];
    row(v + j * sh.v_stride + kh * D, w);
    const float ds = sh.scale * p * (dot(g, w) - dl);
    for (int i = 0; i < N; ++i) acc[i] += ds * y[i];
  }
  put(dq + t * sh.dq_stride + h * D, acc, add);
  if ((threadIdx.x & 31) == 0) delta[static_cast<size_t>(h) * sh.T + t] = dl;
}

template <int D>
__global__ void packed_dkv_kernel(const PackedShape sh, const bf16* q, const bf16* k, const bf16* v, const bf16* dO,
                                  const float* lse, const float* delta, const int32_t* cu, bf16* dk, bf16* dv, bool add) {
  const int t = blockIdx.x * 4 + threadIdx.x / 32, kh = blockIdx.y, G = sh.H / sh.Hk;
  if (t >= sh.T) return;
  const int2 seq = sequence_of(cu, sh.n, sh.T, t);
  if (seq.x == seq.y) return;
  constexpr int N = D / 32;
  float x[N], y[N], w[N], g[N], ak[N] = {}, av[N] = {};
  row(k + t * sh.k_stride + kh * D, y);
  row(v + t * sh.v_stride + kh * D, w);
  for (int h = kh * G; h < kh * G + G; ++h)
    for (int i = t; i < seq.y; ++i) {
      row(q + i * sh.q_stride + h * D, x);
      row(dO + (static_cast<size_t>(i) * sh.H + h) * D, g);
      const size_t r = static_cast<size_t>(h) * sh.T + i;
      const float p = __expf(sh.scale * dot(x, y) - lse[r]), ds = sh.scale * p * (dot(g, w) - delta[r]);
      for (int e = 0; e < N; ++e) {
        av[e] += p * g[e];
        ak[e] += ds * x[e];
      }
    }
  put(dk + t * sh.dk_stride + kh * D, ak, add);
  put(dv + t * sh.dv_stride + kh * D, av, add);
}

}  // namespace

size_t packed_attn_bwd_workspace_bytes(const PackedShape& sh) { return 4 * static_cast<size_t>(sh.T) * sh.H; }

template <int D>
static void packed_bwd(const PackedShape& sh, const bf16* q, const bf16* k, const bf16* v, const bf16* o,
                       const bf16* dO, const float* lse, const int32_t* cu, bf16* dq, bf16* dk, bf16* dv, bool add,
                       float* delta, cudaStream_t s) {
  packed_dq_kernel<D><<<dim3((sh.T + 3) / 4, sh.H), 128, 0, s>>>(sh, q, k, v, o, dO, lse, cu, dq, delta, add);
  packed_dkv_kernel<D><<<dim3((sh.T + 3) / 4, sh.Hk), 128, 0, s>>>(sh, q, k, v, dO, lse, delta, cu, dk, dv, add);
}

int launch_packed_attn_bwd(const PackedShape& sh, const void* q, const void* k, const void* v,
                           const void* o, const void* dO, const float* lse, const int32_t* cu,
                           void* dq, void* dk, void* dv, bool accumulate, void* ws,
                           uint32_t*, cudaStream_t s) {
  auto go = [&](auto bwd) {
    bwd(sh, static_cast<const bf16*>(q), static_cast<const bf16*>(k), static_cast<const bf16*>(v),
        static_cast<const bf16*>(o), static_cast<const bf16*>(dO), lse, cu, static_cast<bf16*>(dq),
        static_cast<bf16*>(dk), static_cast<bf16*>(dv), accumulate, static_cast<float*>(ws), s);
  };
  if (sh.D == 64) go(packed_bwd<64>);
  else go(packed_bwd<128>);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // namespace pa
