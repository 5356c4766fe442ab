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
// sine and cosine: the angle is off by 1e-7 rad up to position 2^24 (the fp32
// fraction) and by 4e-7 at 2^31 (the 64-bit product).
//
// Bound by HBM: q and k are read once and written once. A block computes the
// cosines and sines of its tokens once into shared memory, and all heads of q
// and k of those tokens read them there. 8 x 4096 tokens of 16 + 16 heads of 64
// in bf16 (268 MB) take 51.7 us back to back: 5.2 TB/s, 79% of a plain copy. A
// call of a few tokens takes 3 us of the GPU, less than its launch on the host.
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
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T v[V];
};

// Values 2 j and 2 j + 1 of a vector (bf16 as one 32-bit word: unpacked and packed two at a time).
template <int V>
__device__ __forceinline__ float2 two_of(const Pack<float, V>& x, int j) {
  return make_float2(x.v[2 * j], x.v[2 * j + 1]);
}
template <int V>
__device__ __forceinline__ float2 two_of(const Pack<__nv_bfloat16, V>& x, int j) {
  const uint32_t w = reinterpret_cast<const uint32_t*>(&x)[j];
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <int V>
__device__ __forceinline__ void set_two(Pack<float, V>& x, int j, float2 y) {
  x.v[2 * j] = y.x;
  x.v[2 * j + 1] = y.y;
}
template <int V>
__device__ __forceinline__ void set_two(Pack<__nv_bfloat16, V>& x, int j, float2 y) {
  reinterpret_cast<uint32_t*>(&x)[j] = pack_bf16x2(y.x, y.y);
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// How a block's threads share its tokens: thread = (token t of T, head slot of G, vector c
// of a head). A head slot takes heads slot, slot + G, ... of q and then k, so a thread's
// vector and cosines stay the same from head to head.
struct RopeSplit {
  int T, G;
};

// V: values per load; the scalar form (V = 1) takes head sizes and sections whose runs are
// not whole 16-byte vectors. ACC: y += turn(x) (gradients added to what y holds).
//
// A vector is two runs of V values that turn together (halves: values i and P + i on),
// or W values of pairs side by side, or V values that pass through. Each thread loads
// the vectors of kRopeUnroll heads before it works on the first. With 1, 2, 4 and 8 heads
// and cold caches: 8 x 4096 tokens of 16 + 16 heads of 64 in bf16 70, 70, 58 and 73 us, of 16 + 4
// heads in fp32 85, 63, 66 and 63 us, 2 x 1177 tokens of 32 + 8 heads in bf16 17, 15, 14 and 14 us.
constexpr int kRopeUnroll = 4;
template <typename T, int V, bool HALVES, bool ACC>
__device__ __forceinline__ void rope_tokens(const T* q, const T* k, T* qo, T* ko, const int32_t* __restrict__ pos,
                                            const RopeTable& tab, int P, int D, int Hq, int Hk, long long n_tok,
                                            const RopeSplit split, float sign) {
  // 2 x (cos [T][P], sin [T][P]): one sync a tile; apart, so that the lanes of a head read
  // whole 16-byte vectors from different banks
  extern __shared__ __align__(16) float tables[];
  constexpr int W = V == 1 ? 2 : V;       // values of a pairs vector
  constexpr bool TWO = HALVES || V == 1;  // a turning vector has a second run
  constexpr int N = TWO ? V : V / 2;      // angles of a vector
  using PV = Pack<T, V>;
  using PN = Pack<float, N>;
  const int n_turn = HALVES ? P / V : 2 * P / W, per_head = n_turn + (D - 2 * P) / V;
  const int c = threadIdx.x % per_head, slot = threadIdx.x / per_head % split.G;
  const int t = threadIdx.x / (per_head * split.G);
  const bool works = t < split.T, turns = c < n_turn;
  const int e = turns ? c * (HALVES ? V : W) : 2 * P + (c - n_turn) * V, second = HALVES ? P : 1;
  const int angle = t * P + (HALVES ? e : e / 2);
  // A thread's first entry of the table has the same pair in every tile: lanes that index the
  // parameter differently are served one by one, so it is read once.
  const int my_t = threadIdx.x / P, my_p = threadIdx.x - my_t * P;
  const double my_turns = tab.turns[my_p];
  const int32_t* my_pos = pos + tab.axis[my_p] * n_tok;
  const long long n_tiles = (n_tok + split.T - 1) / split.T;
#pragma unroll 1
  for (long long tile = blockIdx.x; tile < n_tiles; tile += gridDim.x) {
    float *cosines = tables + ((tile / gridDim.x) & 1) * 2 * split.T * P, *sines = cosines + split.T * P;
    const long long t0 = tile * split.T, tok = t0 + t;
    const bool live = works && tok < n_tok;
    PN cv, sv;
#pragma unroll 1
    for (int h0 = slot; h0 - slot < Hq + Hk; h0 += kRopeUnroll * split.G) {
      PV a[kRopeUnroll], b[kRopeUnroll], oa[kRopeUnroll], ob[kRopeUnroll];
      T* dst[kRopeUnroll];
#pragma unroll
      for (int n = 0; n < kRopeUnroll; ++n) {
        const int h = h0 + n * split.G;
        const bool is_k = h >= Hq;
        const size_t at = (is_k ? static_cast<size_t>(tok) * Hk + (h - Hq) : static_cast<size_t>(tok) * Hq + h) * D + e;
        dst[n] = live && h < Hq + Hk ? (is_k ? ko : qo) + at : nullptr;
        if (dst[n]) {
          const T* src = (is_k ? k : q) + at;
          a[n] = *reinterpret_cast<const PV*>(src);
          if (TWO && turns) b[n] = *reinterpret_cast<const PV*>(src + second);
          if (ACC) {
            oa[n] = *reinterpret_cast<const PV*>(dst[n]);
            if (TWO && turns) ob[n] = *reinterpret_cast<const PV*>(dst[n] + second);
          }
        }
      }
      if (h0 == slot) {  // the table, while the first loads are on their way
        const int nt = static_cast<int>(n_tok - t0 < split.T ? n_tok - t0 : split.T);
        auto entry = [&](int i, double u) {
          float s, co;
          sincospif(2.f * static_cast<float>(u - rint(u)), &s, &co);
          cosines[i] = co;
          sines[i] = sign * s;
        };
        if (my_t < nt) entry(threadIdx.x, static_cast<double>(my_pos[t0 + my_t]) * my_turns);
        for (int i = threadIdx.x + kRopeThreads; i < nt * P; i += kRopeThreads) {
          const int ti = i / P, p = i - ti * P;
          if (p == my_p) entry(i, static_cast<double>(my_pos[t0 + ti]) * my_turns);
          else entry(i, static_cast<double>(pos[tab.axis[p] * n_tok + t0 + ti]) * tab.turns[p]);
        }
        __syncthreads();
        if (live && turns) {
          cv = *reinterpret_cast<const PN*>(cosines + angle);
          sv = *reinterpret_cast<const PN*>(sines + angle);
        }
      }
#pragma unroll
      for (int n = 0; n < kRopeUnroll; ++n) {
        if (!dst[n]) continue;
        if (turns) {
          if constexpr (V == 1) {
            const float fa = to_f(a[n].v[0]), fb = to_f(b[n].v[0]);
            a[n].v[0] = from_f<T>(fa * cv.v[0] - fb * sv.v[0] + (ACC ? to_f(oa[n].v[0]) : 0.f));
            b[n].v[0] = from_f<T>(fb * cv.v[0] + fa * sv.v[0] + (ACC ? to_f(ob[n].v[0]) : 0.f));
          } else if constexpr (HALVES) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
              const float2 fa = two_of(a[n], j), fb = two_of(b[n], j);
              const float2 co = two_of(cv, j), si = two_of(sv, j);
              float2 ya = __ffma2_rn(fb, make_float2(-si.x, -si.y), __fmul2_rn(fa, co));
              float2 yb = __ffma2_rn(fa, si, __fmul2_rn(fb, co));
              if (ACC) {
                ya = __fadd2_rn(ya, two_of(oa[n], j));
                yb = __fadd2_rn(yb, two_of(ob[n], j));
              }
              set_two(a[n], j, ya);
              set_two(b[n], j, yb);
            }
          } else {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
              const float2 f = two_of(a[n], j);
              float2 y = __ffma2_rn(make_float2(f.y, f.x), make_float2(-sv.v[j], sv.v[j]),
                                    __fmul2_rn(f, make_float2(cv.v[j], cv.v[j])));
              if (ACC) y = __fadd2_rn(y, two_of(oa[n], j));
              set_two(a[n], j, y);
            }
          }
          if (TWO) *reinterpret_cast<PV*>(dst[n] + second) = b[n];
        } else if (ACC) {
          if constexpr (V == 1) {
            a[n].v[0] = from_f<T>(to_f(oa[n].v[0]) + to_f(a[n].v[0]));
          } else {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) set_two(a[n], j, __fadd2_rn(two_of(oa[n], j), two_of(a[n], j)));
          }
        }
        *reinterpret_cast<PV*>(dst[n]) = a[n];
      }
    }
  }
}

// Outputs apart from the inputs: loads and stores may pass one another (8 x 4096 tokens of 16 + 16
// heads of 64 in bf16, pairs side by side: 45 us, 51 without __restrict__).
template <typename T, int V, bool HALVES, bool ACC>
__global__ void __launch_bounds__(kRopeThreads)
    rope_kernel(const T* __restrict__ q, const T* __restrict__ k, T* __restrict__ qo, T* __restrict__ ko,
                const int32_t* __restrict__ pos, const __grid_constant__ RopeTable tab, int P, int D,
                int Hq, int Hk, long long n_tok, const RopeSplit split, float sign) {
  rope_tokens<T, V, HALVES, ACC>(q, k, qo, ko, pos, tab, P, D, Hq, Hk, n_tok, split, sign);
}

// qo is q, or ko is k: a thread has loaded each value before it stores its turn.
template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(kRopeThreads)
    rope_in_place_kernel(const T* q, const T* k, T* qo, T* ko, const int32_t* __restrict__ pos,
                         const __grid_constant__ RopeTable tab, int P, int D, int Hq, int Hk, long long n_tok,
                         const RopeSplit split, float sign) {
  rope_tokens<T, V, HALVES, false>(q, k, qo, ko, pos, tab, P, D, Hq, Hk, n_tok, split, sign);
}

template <typename T, int V>
void rope_launch(const RopeShape& sh, const void* q, const void* k, void* qo, void* ko,
                 const int32_t* pos, const RopeTable& tab, bool inverse, bool accumulate, cudaStream_t s) {
  const int run = sh.halves ? V : (V == 1 ? 2 : V), heads = sh.Hq + sh.Hk;
  const int per_head = (sh.halves ? sh.pairs : 2 * sh.pairs) / run + (sh.D - 2 * sh.pairs) / V;  // <= 256
  const long long n_tok = static_cast<long long>(sh.B) * sh.L;
  // Head slots so that a thread has kRopeUnroll heads (all its loads in flight at once), the rest of
  // the block for tokens; with few tokens one token a block, so that more blocks share them.
  RopeSplit split;
  const int fit = kRopeThreads / per_head;
  split.G = (heads + kRopeUnroll - 1) / kRopeUnroll;
  if (split.G > fit) split.G = fit;
  split.T = fit / split.G;
  const long long spread = n_tok / device_sm_count();
  if (split.T > spread) split.T = spread < 1 ? 1 : static_cast<int>(spread);
  const long long tiles = (n_tok + split.T - 1) / split.T, blocks = 8ll * device_sm_count();
  const unsigned grid = static_cast<unsigned>(tiles < blocks ? tiles : blocks);
  const size_t smem = 4 * static_cast<size_t>(split.T) * sh.pairs * sizeof(float);
  const float sign = inverse ? -1.f : 1.f;
  const bool in_place = qo == q || (sh.Hk > 0 && ko == k);  // (never with accumulate)
  auto go = [&](auto kernel) {
    kernel<<<grid, kRopeThreads, smem, s>>>(static_cast<const T*>(q), static_cast<const T*>(k),
                                            static_cast<T*>(qo), static_cast<T*>(ko), pos, tab,
                                            sh.pairs, sh.D, sh.Hq, sh.Hk, n_tok, split, sign);
  };
  if (sh.halves) {
    if (accumulate) go(rope_kernel<T, V, true, true>);
    else if (in_place) go(rope_in_place_kernel<T, V, true>);
    else go(rope_kernel<T, V, true, false>);
  } else {
    if (accumulate) go(rope_kernel<T, V, false, true>);
    else if (in_place) go(rope_in_place_kernel<T, V, false>);
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
  const int V = sh.f32 ? 4 : 8;
  // whole 16-byte vectors in every run that is turned or passed through
  const bool vec = sh.D % V == 0 && (sh.halves ? sh.pairs : 2 * sh.pairs) % V == 0;
  if (sh.f32) {
    if (vec) rope_launch<float, 4>(sh, q, k, qo, ko, positions, tab, inverse, accumulate, s);
    else rope_launch<float, 1>(sh, q, k, qo, ko, positions, tab, inverse, accumulate, s);
  } else {
    if (vec) rope_launch<__nv_bfloat16, 8>(sh, q, k, qo, ko, positions, tab, inverse, accumulate, s);
    else rope_launch<__nv_bfloat16, 1>(sh, q, k, qo, ko, positions, tab, inverse, accumulate, s);
  }
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // namespace pa
