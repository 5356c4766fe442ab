// Attention of one new token of each sequence over its paged cache.
#include <cuda_bf16.h>
#include "host_launchers.h"

namespace pa {
namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// A warp takes a (sequence, head of q); its lanes share the head's values.
template <typename T, int D>
__global__ void paged_step_kernel(const PagedShape sh, const T* __restrict__ q, const T* __restrict__ kc,
                                  const T* __restrict__ vc, const int32_t* __restrict__ table,
                                  const int32_t* __restrict__ lens, T* __restrict__ o, float* __restrict__ lse) {
  const int w = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
  if (w >= sh.B * sh.H) return;
  const int b = w / sh.H, h = w % sh.H, kh = h / (sh.H / sh.Hk);
  constexpr int N = D / 32;
  float x[N], acc[N] = {}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < N; ++i) x[i] = to_f(q[b * sh.q_stride + static_cast<size_t>(h) * D + lane + 32 * i]) * sh.scale;
  const int most = sh.max_pages * sh.page_size, n = max(0, min(lens[b], most));
  for (int t = 0; t < n; ++t) {
    const int page = table[static_cast<size_t>(b) * sh.max_pages + t / sh.page_size];
    if (page < 0 || page >= sh.num_pages) continue;
    const size_t row = ((static_cast<size_t>(page) * sh.page_size + t % sh.page_size) * sh.Hk + kh) * D + lane;
    float s = 0.f;
    for (int i = 0; i < N; ++i) s += x[i] * to_f(kc[row + 32 * i]);
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float top = fmaxf(m, s), old = m == -INFINITY ? 0.f : __expf(m - top), p = s == -INFINITY ? 0.f : __expf(s - top);
    l = l * old + p;
    for (int i = 0; i < N; ++i) acc[i] = acc[i] * old + p * to_f(vc[row + 32 * i]);
    m = top;
  }
  for (int i = 0; i < N; ++i) put(o + static_cast<size_t>(w) * D + lane + 32 * i, l == 0.f ? 0.f : acc[i] / l);
  if (lse && lane == 0) lse[w] = l == 0.f ? -INFINITY : m + __logf(l);
}

template <typename T, int D>
int paged_launch(const PagedShape& sh, const void* q, const void* kc, const void* vc, const int32_t* table,
                 const int32_t* lens, void* o, float* lse, cudaStream_t s) {
  paged_step_kernel<T, D><<<(sh.B * sh.H + 3) / 4, 128, 0, s>>>(sh, static_cast<const T*>(q), static_cast<const T*>(kc),
                                                              static_cast<const T*>(vc), table, lens,
                                                              static_cast<T*>(o), lse);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // namespace

size_t paged_attn_workspace_bytes(const PagedShape&) { return 256; }

int launch_paged_attn(const PagedShape& sh, const void* q, const void* kc, const void* vc, const int32_t* table,
                      const int32_t* lens, void* o, float* lse, void*, cudaStream_t s) {
  if (sh.f32)
    return sh.D == 32 ? paged_launch<float, 32>(sh, q, kc, vc, table, lens, o, lse, s)
                      : paged_launch<float, 64>(sh, q, kc, vc, table, lens, o, lse, s);
  return sh.D == 64 ? paged_launch<__nv_bfloat16, 64>(sh, q, kc, vc, table, lens, o, lse, s)
                    : paged_launch<__nv_bfloat16, 128>(sh, q, kc, vc, table, lens, o, lse, s);
}

}  // namespace pa
