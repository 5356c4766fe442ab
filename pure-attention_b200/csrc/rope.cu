// Rotary positions with one to four position axes, applied to q and k in one
// launch, and the adjoint for the gradients.
//
// Pair i of a head (i < P, 2P <= head_dim) belongs to one position axis and
// turns by the angle a = position[axis(i)] * w_i, w_i = base^-f_i:
//   y_a = x_a cos a - x_b sin a,   y_b = x_b cos a + x_a sin a,
// where (a, b) = (i, P + i) (halves) or (2i, 2i + 1) (pairs); values from 2P on
// pass through. The turn is orthogonal, so the backward turns by -a.
//
// The angles are the only part that fp32 cannot hold: at position 200000 an
// fp32 product is off by 2^-24 * 2e5 = 0.012 rad. The host passes w_i / 2 pi in
// 64 bits; the kernel takes the fraction of position * w_i / 2 pi in 64 bits
// (one multiply, one rounding to the nearest whole turn) and only then fp32
// sine and cosine, exact to about 3e-7 for every 32-bit position.
//
// Bound by HBM: q and k are read once and written once. A block computes the
// cosines and sines of its tokens once into shared memory, and all heads of q
// and k of those tokens read them there.
#include <cmath>
#include <cuda_bf16.h>
#include "host_launchers.h"

namespace pa {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 128;  // head_dim <= 256

struct RopeTable {
  double turns[kRopeMaxPairs];  // w_i / 2 pi
  uint8_t axis[kRopeMaxPairs];
};

// V values as V * sizeof(T) bytes (16 for the vector paths).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One tile of `tokens` tokens per block. V: values per load; the scalar form
// (V = 1) takes head sizes and sections whose runs are not whole 16-byte
// vectors. ACC: y += turn(x) (gradients added to what y holds).
template <typename T, int V, bool HALVES, bool ACC>
__global__ void __launch_bounds__(kRopeThreads)
    rope_kernel(const T* __restrict__ q, const T* __restrict__ k, T* qo, T* ko,
                const int32_t* __restrict__ pos, const __grid_constant__ RopeTable tab, int P, int D,
                int Hq, int Hk, long long n_tok, int tokens, float sign) {
  extern __shared__ float2 cs[];  // [tokens][P] (cos, sin)
  const long long t0 = static_cast<long long>(blockIdx.x) * tokens;
  const int nt = static_cast<int>(n_tok - t0 < tokens ? n_tok - t0 : tokens);
  for (int i = threadIdx.x; i < nt * P; i += kRopeThreads) {
    const int t = i / P, p = i - t * P;
    const double u = static_cast<double>(pos[tab.axis[p] * n_tok + t0 + t]) * tab.turns[p];
    float s, c;
    sincospif(2.f * static_cast<float>(u - rint(u)), &s, &c);
    cs[i] = make_float2(c, sign * s);
  }
  __syncthreads();
  // Work items of one head: `run` pairs of vectors (halves) or vectors (pairs)
  // to turn, then `tail` vectors to pass through.
  constexpr int W = HALVES ? V : (V == 1 ? 2 : V);  // values a pairs-layout item covers
  const int turn = HALVES ? P / V : 2 * P / W;
  const int tail = (D - 2 * P) / V;
  const int per_head = turn + tail, per_tok = (Hq + Hk) * per_head;
  for (int it = threadIdx.x; it < nt * per_tok; it += kRopeThreads) {
    const int t = it / per_tok, r = it - t * per_tok;
    const int h = r / per_head, c = r - h * per_head;
    const bool is_k = h >= Hq;
    const size_t at = (is_k ? (static_cast<size_t>(t0 + t) * Hk + (h - Hq))
                            : (static_cast<size_t>(t0 + t) * Hq + h)) * D;
    const T* src = (is_k ? k : q) + at;
    T* dst = (is_k ? ko : qo) + at;
    const float2* w = cs + t * P;
    if (c >= turn) {  // pass through
      using PV = Pack<T, V>;
      const int e = 2 * P + (c - turn) * V;
      PV x = *reinterpret_cast<const PV*>(src + e);
      if (ACC) {
        const PV o = *reinterpret_cast<const PV*>(dst + e);
#pragma unroll
        for (int i = 0; i < V; ++i) x.v[i] = from_f<T>(to_f(o.v[i]) + to_f(x.v[i]));
      }
      *reinterpret_cast<PV*>(dst + e) = x;
    } else if (HALVES) {
      using PV = Pack<T, V>;
      const int e = c * V;
      PV a = *reinterpret_cast<const PV*>(src + e), b = *reinterpret_cast<const PV*>(src + P + e);
      PV oa, ob;
      if (ACC) {
        oa = *reinterpret_cast<const PV*>(dst + e);
        ob = *reinterpret_cast<const PV*>(dst + P + e);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 m = w[e + i];
        const float fa = to_f(a.v[i]), fb = to_f(b.v[i]);
        float ya = fa * m.x - fb * m.y, yb = fb * m.x + fa * m.y;
        if (ACC) {
          ya += to_f(oa.v[i]);
          yb += to_f(ob.v[i]);
        }
        a.v[i] = from_f<T>(ya);
        b.v[i] = from_f<T>(yb);
      }
      *reinterpret_cast<PV*>(dst + e) = a;
      *reinterpret_cast<PV*>(dst + P + e) = b;
    } else {
      using PW = Pack<T, W>;
      const int e = c * W;
      PW x;
      PW o;
      if constexpr (V == 1) {  // a pair need not be aligned to its size
        x.v[0] = src[e];
        x.v[1] = src[e + 1];
        if (ACC) {
          o.v[0] = dst[e];
          o.v[1] = dst[e + 1];
        }
      } else {
        x = *reinterpret_cast<const PW*>(src + e);
        if (ACC) o = *reinterpret_cast<const PW*>(dst + e);
      }
#pragma unroll
      for (int i = 0; i < W / 2; ++i) {
        const float2 m = w[e / 2 + i];
        const float fa = to_f(x.v[2 * i]), fb = to_f(x.v[2 * i + 1]);
        float ya = fa * m.x - fb * m.y, yb = fb * m.x + fa * m.y;
        if (ACC) {
          ya += to_f(o.v[2 * i]);
          yb += to_f(o.v[2 * i + 1]);
        }
        x.v[2 * i] = from_f<T>(ya);
        x.v[2 * i + 1] = from_f<T>(yb);
      }
      if constexpr (V == 1) {
        dst[e] = x.v[0];
        dst[e + 1] = x.v[1];
      } else {
        *reinterpret_cast<PW*>(dst + e) = x;
      }
    }
  }
}

template <typename T, int V>
void rope_launch(const RopeShape& sh, const void* q, const void* k, void* qo, void* ko,
                 const int32_t* pos, const RopeTable& tab, long long n_tok, int tokens, bool inverse,
                 bool accumulate, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>((n_tok + tokens - 1) / tokens);
  const size_t smem = static_cast<size_t>(tokens) * sh.pairs * sizeof(float2);
  const float sign = inverse ? -1.f : 1.f;
  auto go = [&](auto kernel) {
    kernel<<<grid, kRopeThreads, smem, s>>>(static_cast<const T*>(q), static_cast<const T*>(k),
                                            static_cast<T*>(qo), static_cast<T*>(ko), pos, tab,
                                            sh.pairs, sh.D, sh.Hq, sh.Hk, n_tok, tokens, sign);
  };
  if (sh.halves) {
    if (accumulate) go(rope_kernel<T, V, true, true>);
    else go(rope_kernel<T, V, true, false>);
  } else {
    if (accumulate) go(rope_kernel<T, V, false, true>);
    else go(rope_kernel<T, V, false, false>);
  }
}

}  // namespace

int launch_rope(const RopeShape& sh, const void* q, const void* k, void* qo, void* ko,
                const int32_t* positions, bool inverse, bool accumulate, cudaStream_t s) {
  RopeTable tab;
  const double turn = 1.0 / 6.283185307179586476925286766559, log2_base = std::log2(sh.base);
  int i = 0;
  for (int a = 0; a < sh.axes; ++a)
    for (int j = 0; j < sh.sections[a]; ++j, ++i) {
      const double f = sh.per_axis ? static_cast<double>(j) / sh.sections[a]
                                   : static_cast<double>(i) / sh.pairs;
      tab.turns[i] = turn * std::exp2(-f * log2_base);
      tab.axis[i] = static_cast<uint8_t>(a);
    }
  const long long n_tok = static_cast<long long>(sh.B) * sh.L;
  // Tokens per block: one while that leaves blocks for the whole GPU, up to 8
  // (the table of 8 tokens x 128 pairs is 8 KB).
  const long long want = n_tok / (8ll * device_sm_count());
  const int tokens = want < 1 ? 1 : (want > 8 ? 8 : static_cast<int>(want));
  const int V = sh.f32 ? 4 : 8;
  // whole 16-byte vectors in every run that is turned or passed through
  const bool vec = sh.D % V == 0 && (sh.halves ? sh.pairs : 2 * sh.pairs) % V == 0;
  if (sh.f32) {
    if (vec) rope_launch<float, 4>(sh, q, k, qo, ko, positions, tab, n_tok, tokens, inverse, accumulate, s);
    else rope_launch<float, 1>(sh, q, k, qo, ko, positions, tab, n_tok, tokens, inverse, accumulate, s);
  } else {
    if (vec) rope_launch<__nv_bfloat16, 8>(sh, q, k, qo, ko, positions, tab, n_tok, tokens, inverse, accumulate, s);
    else rope_launch<__nv_bfloat16, 1>(sh, q, k, qo, ko, positions, tab, n_tok, tokens, inverse, accumulate, s);
  }
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // namespace pa
