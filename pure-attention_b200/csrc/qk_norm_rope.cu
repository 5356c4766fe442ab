// Root-mean-square norm of each head of q and k, then their rotary positions,
// in one pass, optionally with k and v written into a paged cache; and the
// gradients of both.
//
// With x a head of D values, r = (mean(x^2) + eps)^-1/2 and R the rotation by
// the token's positions (rope.cu):
//   y = R (x r gamma)
//   dn = R^T dy,  u = dn gamma,  dgamma = sum dn x r,
//   dx = r (u - x r^2 mean(u x)).
// The statistics are sums in fp32 over the lanes that share a head; r is computed
// again in the backward, which reads x anyway, rather than stored.
//
// Bound by HBM in bytes (x once, y once; the backward x, dy and dx), and next to that by instructions: some 300 for
// 16 bytes of a head a lane (conversions, squares, shuffles, two products a value), 53% of the issue slots. 8 x
// 4096 tokens of 16 + 2 heads of 128 in bf16: 76 us (4.0 TB/s of 6.55 a plain copy; the rotation alone 66), the
// gradient 148 us (3.1 TB/s), in fp32 168 us (5.4). Slower, 89 to 122 us: inputs through a ring of bulk copies or of
// cp.async, packed pairs of fp32, vectors of 8 bytes, fewer heads in flight with more blocks. Where the turned pairs are
// no whole vectors of 16 bytes (halves: a number of pairs that 8, in fp32 4, does not divide) values move one by one: the
// same batch with heads of 80, 24 pairs turned 71 us and the gradient 136, 20 pairs 836 and 966.
#include <cmath>
#include <cstring>
#include <type_traits>
#include <cuda_bf16.h>
#include "host_launchers.h"

namespace pa {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormMaxPairs = 128;  // head_dim <= 256
// Heads that a thread loads before it works on the first.
__host__ __device__ constexpr int norm_at_once(int U, bool bwd) { return U > 1 ? 1 : bwd ? 2 : 4; }

// w_i / 2 pi as a fraction of 2^64: position * turns modulo 2^64 is the fraction of a turn, exact but for the
// table's own rounding (2^-33 of a turn at position 2^31), in integers.
struct NormTable {
  uint64_t turns[kNormMaxPairs];
  uint8_t axis[kNormMaxPairs];
};
constexpr int kNormAngles = 4;  // of a tile that a thread computes, at most

// One tensor of the call: heads of D values, tokens `stride` values apart.
template <typename T>
struct NormSide {
  const T* x;          // input; NULL: no such tensor
  T* y;                // output (forward) or dx (backward)
  const T* dy;         // backward
  const float* gamma;  // NULL: no norm
  int heads;
  long long x_stride, y_stride;
};

template <typename T>
struct NormArgs {
  NormSide<T> side[2];  // q, k
  // cache (forward)
  const T* v;
  long long v_stride, num_slots;
  const int32_t* slots;
  T *k_cache, *v_cache;
  const int32_t* pos;
  float* partial;  // backward: [block][2][D] sums of dgamma
  long long n_tok;
  int P, D, lanes, tile, G;  // lanes that share a head (a power of two); tokens of a tile, head slots of a token
  float eps;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

template <int N>
__device__ __forceinline__ void load_f32(const float* p, float (&f)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + j);
      f[j] = x.x, f[j + 1] = x.y, f[j + 2] = x.z, f[j + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = p[j];
  }
}

// A lane's unit c of a head: two runs of V values that turn together (halves: e and P + e
// on; scalar pairs: 2 c and 2 c + 1), one run of V / 2 pairs, or one run that passes through.
template <int V, bool HALVES>
struct UnitAt {
  static constexpr bool TWO = HALVES || V == 1;
  int e, second, angle;
  bool on, turns;
  __device__ UnitAt(int c, int P, int D) {
    constexpr int W = V == 1 ? 2 : V;
    const int n_turn = HALVES ? P / V : 2 * P / W;
    turns = c < n_turn;
    on = c < n_turn + (D - 2 * P) / V;
    e = turns ? c * (HALVES ? V : W) : 2 * P + (c - n_turn) * V;
    second = HALVES ? P : 1;
    angle = HALVES ? e : e / 2;
  }
};

// The unit's values in memory, as they are, and as floats: two runs of V.
template <typename T, int V>
struct Raw {
  using R = std::conditional_t<V == 1, T, uint4>;
  R r[2];
};
template <typename T, int V>
__device__ __forceinline__ void read_raw(Raw<T, V>& x, const T* p, int second, bool two) {
  using R = typename Raw<T, V>::R;
  x.r[0] = *reinterpret_cast<const R*>(p);
  if (two) x.r[1] = *reinterpret_cast<const R*>(p + second);
  else memset(&x.r[1], 0, sizeof(R));
}
template <int V>
struct Unit {
  float v[2][V];
};
template <typename T, int V>
__device__ __forceinline__ Unit<V> floats_of(const Raw<T, V>& x) {
  Unit<V> f;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    if constexpr (V == 1) {
      f.v[z][0] = to_f(x.r[z]);
    } else {
      const uint32_t w[4] = {x.r[z].x, x.r[z].y, x.r[z].z, x.r[z].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2) {
          f.v[z][2 * j] = __uint_as_float(w[j] << 16);
          f.v[z][2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
          f.v[z][j] = __uint_as_float(w[j]);
        }
      }
    }
  }
  return f;
}
template <typename T, int V>
__device__ __forceinline__ void write_run(T* p, const float (&f)[V]) {
  if constexpr (V == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  else if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  else if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(f[0]);
  else *p = f[0];
}

// What a unit's turn multiplies by, N of each: with (a, b) a pair, a' = a ca - b sb, b' = b cb + a sa, where ca
// and sa are the cosine and the sine times gamma of a, cb and sb times gamma of b. A unit that passes
// through has ca = gamma alone. Kept from head to head of a token (of the backward: without gamma).
template <int V, bool HALVES>
struct Turn {
  static constexpr int N = UnitAt<V, HALVES>::TWO ? V : V / 2;
  float ca[N], cb[N], sa[N], sb[N];
  __device__ __forceinline__ void set(const float* co, const float* si, const Unit<V>& gm, bool turns) {
    float c[N], s[N];
    if (turns) {
      load_f32<N>(co, c);
      load_f32<N>(si, s);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (!turns) c[j] = 1.f, s[j] = 0.f;
      const float ga = UnitAt<V, HALVES>::TWO ? gm.v[0][j] : gm.v[0][(2 * j) % V],
                  gb = UnitAt<V, HALVES>::TWO ? gm.v[1][j] : gm.v[0][(2 * j + 1) % V];
      ca[j] = c[j] * ga;
      sa[j] = s[j] * ga;
      cb[j] = c[j] * gb;
      sb[j] = s[j] * gb;
    }
  }
  // f (times r) turned; BACK: by the negative angles
  template <bool BACK>
  __device__ __forceinline__ void apply(Unit<V>& f, float r) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float& a = UnitAt<V, HALVES>::TWO ? f.v[0][j] : f.v[0][(2 * j) % V];
      float& b = UnitAt<V, HALVES>::TWO ? f.v[1][j] : f.v[0][(2 * j + 1) % V];
      const float x = a, y = b;
      if (BACK) {
        a = fmaf(x, ca[j], y * sa[j]);
        b = fmaf(y, cb[j], -(x * sb[j]));
      } else {
        a = r * fmaf(x, ca[j], -(y * sb[j]));
        b = r * fmaf(y, cb[j], x * sa[j]);
      }
    }
  }
};

// T: value type; V: values of a run (16 bytes of them; 1 where the runs are no whole vectors); U: units of a
// lane; BWD: gradients; ACC: added to what dx holds. Thread = (token of a tile, head slot of G, lane of a
// head): a slot takes heads slot, slot + G, ... of q and then of k, so a thread keeps its token's angles and
// its part of gamma from head to head. The loads of AT_ONCE heads are in flight.
template <typename T, int V, int U, bool HALVES, bool BWD, bool ACC>
__global__ void __launch_bounds__(kNormThreads, U > 1 ? 1 : 2)
    qk_norm_rope_kernel(const __grid_constant__ NormArgs<T> g, const __grid_constant__ NormTable tab) {
  using At = UnitAt<V, HALVES>;
  constexpr int AT_ONCE = norm_at_once(U, BWD), RUNS = At::TWO ? 2 : 1;
  extern __shared__ __align__(16) float tables[];  // 2 x (cos [tile][P], sin [tile][P])
  // the parameter's table: lanes that index it differently there would be served one by one
  __shared__ uint64_t s_turns[kNormMaxPairs];
  __shared__ int s_axis[kNormMaxPairs];
  const int P = g.P, D = g.D;
  for (int i = threadIdx.x; i < P; i += kNormThreads) {
    s_turns[i] = tab.turns[i];
    s_axis[i] = tab.axis[i];
  }
  __syncthreads();
  const int lane = threadIdx.x & (g.lanes - 1), slot = threadIdx.x / g.lanes % g.G, t = threadIdx.x / (g.lanes * g.G);
  const float inv_d = 1.f / D;
  const int first_ta = threadIdx.x / P, first_p = threadIdx.x - first_ta * P;
  const int step_ta = kNormThreads / P, step_p = kNormThreads - step_ta * P;
  const long long n_tiles = (g.n_tok + g.tile - 1) / g.tile;
  auto tokens_of = [&](long long tile) {
    const long long left = g.n_tok - tile * g.tile;
    return static_cast<int>(left < g.tile ? left : g.tile);
  };
  // The angles of a tile in two parts: the positions of a thread's are loaded before the tile before it is
  // worked on, their cosines and sines computed after it.
  int pos[kNormAngles];
  auto positions = [&](long long tile) {
    const int nt = tokens_of(tile);
    int ta = first_ta, p = first_p;
#pragma unroll
    for (int k = 0; k < kNormAngles; ++k) {
      if (ta < nt) pos[k] = g.pos[s_axis[p] * g.n_tok + tile * g.tile + ta];
      ta += step_ta;
      p += step_p;
      if (p >= P) p -= P, ++ta;
    }
  };
  auto angles = [&](long long tile, int half) {
    const int nt = tokens_of(tile);
    float* to = tables + half * 2 * g.tile * P + threadIdx.x;
    int ta = first_ta, p = first_p;
#pragma unroll
    for (int k = 0; k < kNormAngles; ++k) {
      if (ta < nt) {
        const uint64_t turn = static_cast<uint64_t>(static_cast<int64_t>(pos[k])) * s_turns[p];
        float sn, cs;
        sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * 0x1p-31f, &sn, &cs);
        to[k * kNormThreads] = cs;
        to[k * kNormThreads + g.tile * P] = sn;
      }
      ta += step_ta;
      p += step_p;
      if (p >= P) p -= P, ++ta;
    }
  };

  Unit<V> dg[2][U];
  if (BWD) memset(dg, 0, sizeof(dg));
  positions(blockIdx.x);
  angles(blockIdx.x, 0);
  int parity = 0;
#pragma unroll 1
  for (long long tile = blockIdx.x; tile < n_tiles; tile += gridDim.x, parity ^= 1) {
    const float *cosines = tables + parity * 2 * g.tile * P, *sines = cosines + g.tile * P;
    const long long tok = tile * g.tile + t;
    const bool live = t < tokens_of(tile), more = tile + gridDim.x < n_tiles;
    if (more) positions(tile + gridDim.x);
    bool first = true;  // the tile's angles have not been waited for
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const NormSide<T>& sd = g.side[w];
      if (!sd.x) continue;
      const bool normed = sd.gamma != nullptr;
      const T* src = sd.x + tok * sd.x_stride + static_cast<long long>(slot) * D;
      const T* src_dy = BWD ? sd.dy + (tok * sd.heads + slot) * D : nullptr;
      T* dst = sd.y ? sd.y + tok * sd.y_stride + static_cast<long long>(slot) * D : nullptr;
      T* row = nullptr;
      if (!BWD && w == 1 && g.slots && live) {
        const long long s = g.slots[tok];
        if (s >= 0 && s < g.num_slots) row = g.k_cache + (s * sd.heads + slot) * D;
      }
      Turn<V, HALVES> turn[U];
      Unit<V> gm[U];
      // (all lanes of a warp take the same number of turns: the sums are over whole warps)
#pragma unroll 1
      for (int h0 = 0; h0 < sd.heads; h0 += AT_ONCE * g.G) {
        Raw<T, V> rx[AT_ONCE][U], ry[AT_ONCE][U];
        auto any = [&](int n) { return n == 0 || h0 + n * g.G < sd.heads; };  // in the whole block
        auto has = [&](int n) { return live && slot + h0 + n * g.G < sd.heads; };
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
          if (!any(n)) continue;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const At at(lane + u * g.lanes, P, D);
            if (has(n) && at.on) {
              const int off = (h0 + n * g.G) * D + at.e;
              read_raw<T, V>(rx[n][u], src + off, at.second, At::TWO && at.turns);
              if (BWD) read_raw<T, V>(ry[n][u], src_dy + off, at.second, At::TWO && at.turns);
            } else {
              memset(&rx[n][u], 0, sizeof(rx[n][u]));
              if (BWD) memset(&ry[n][u], 0, sizeof(ry[n][u]));
            }
          }
        }
        if (h0 == 0) {
          if (first) __syncthreads();  // the angles are there
          first = false;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const At at(lane + u * g.lanes, P, D);
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
              for (int j = 0; j < V; ++j) gm[u].v[z][j] = z == 0 || (At::TWO && at.turns) ? 1.f : 0.f;
            if (normed && at.on) {
              load_f32<V>(sd.gamma + at.e, gm[u].v[0]);
              if (At::TWO && at.turns) load_f32<V>(sd.gamma + at.e + at.second, gm[u].v[1]);
            }
            Unit<V> one;
#pragma unroll
            for (int j = 0; j < V; ++j) one.v[0][j] = one.v[1][j] = 1.f;
            const int angle = live && at.on && at.turns ? t * P + at.angle : 0;
            turn[u].set(cosines + angle, sines + angle, BWD ? one : gm[u], at.on && at.turns);
          }
        }
        // A unit's values are unpacked for the sums, and again for the results: packed they take half the
        // registers, and twice the heads are in flight.
        float s1[AT_ONCE], s2[AT_ONCE];
        if (normed) {
#pragma unroll
          for (int n = 0; n < AT_ONCE; ++n) {
            if (!any(n)) continue;
            s1[n] = s2[n] = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const Unit<V> x = floats_of<T, V>(rx[n][u]);
              Unit<V> y;
              if (BWD) {
                y = floats_of<T, V>(ry[n][u]);
                turn[u].template apply<true>(y, 1.f);
              }
#pragma unroll
              for (int z = 0; z < RUNS; ++z)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                  s1[n] = fmaf(x.v[z][j], x.v[z][j], s1[n]);
                  if (BWD) s2[n] = fmaf(y.v[z][j] * gm[u].v[z][j], x.v[z][j], s2[n]);
                }
            }
          }
          for (int m = g.lanes / 2; m > 0; m >>= 1)
#pragma unroll
            for (int n = 0; n < AT_ONCE; ++n) {
              if (!any(n)) continue;
              s1[n] += __shfl_xor_sync(0xffffffffu, s1[n], m);
              if (BWD) s2[n] += __shfl_xor_sync(0xffffffffu, s2[n], m);
            }
        }
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
          if (!any(n) || !has(n)) continue;
          const float r = normed ? rsqrtf(s1[n] * inv_d + g.eps) : 1.f, back = BWD && normed ? r * r * s2[n] * inv_d : 0.f;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const At at(lane + u * g.lanes, P, D);
            if (!at.on) continue;
            const int off = (h0 + n * g.G) * D + at.e;
            Unit<V> x;
            if (!BWD || normed) x = floats_of<T, V>(rx[n][u]);
            if (BWD) {
              Unit<V> y = floats_of<T, V>(ry[n][u]);
              turn[u].template apply<true>(y, 1.f);
              if (normed) {
#pragma unroll
                for (int z = 0; z < RUNS; ++z)
#pragma unroll
                  for (int j = 0; j < V; ++j) {
                    const float f = x.v[z][j];
                    dg[w][u].v[z][j] = fmaf(y.v[z][j] * f, r, dg[w][u].v[z][j]);
                    x.v[z][j] = r * fmaf(f, -back, y.v[z][j] * gm[u].v[z][j]);
                  }
              } else {
                x = y;
              }
            } else {
              turn[u].template apply<false>(x, r);
            }
            if (ACC) {
              Raw<T, V> old;
              read_raw<T, V>(old, dst + off, at.second, At::TWO && at.turns);
              const Unit<V> f = floats_of<T, V>(old);
#pragma unroll
              for (int z = 0; z < RUNS; ++z)
#pragma unroll
                for (int j = 0; j < V; ++j) x.v[z][j] += f.v[z][j];
            }
#pragma unroll
            for (int z = 0; z < RUNS; ++z) {
              if (z == 1 && !at.turns) continue;
              if (dst) write_run<T, V>(dst + off + z * at.second, x.v[z]);
              if (row) write_run<T, V>(row + off + z * at.second, x.v[z]);
            }
          }
        }
      }
    }
    if (!BWD && g.slots) {  // v as it is, 16 bytes at a time
      constexpr int W = 16 / sizeof(T);
      const int per = g.side[1].heads * D / W, nt = tokens_of(tile);
      for (int i = threadIdx.x; i < nt * per; i += kNormThreads) {
        const int tv = i / per, e = (i - tv * per) * W;
        const long long s = g.slots[tile * g.tile + tv];
        if (s >= 0 && s < g.num_slots)
          *reinterpret_cast<uint4*>(g.v_cache + s * g.side[1].heads * D + e) =
              *reinterpret_cast<const uint4*>(g.v + (tile * g.tile + tv) * g.v_stride + e);
      }
    }
    if (more) angles(tile + gridDim.x, parity ^ 1);
  }
  if (BWD) {
    // this block's sums of dgamma: the threads' that share a lane, one after the other
    const int groups = kNormThreads / g.lanes, group = threadIdx.x / g.lanes;
    __syncthreads();
    float* sums = tables;  // [groups][D]
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const At at(lane + u * g.lanes, P, D);
        if (!at.on) continue;
#pragma unroll
        for (int z = 0; z < RUNS; ++z) {
          if (z == 1 && !at.turns) continue;
#pragma unroll
          for (int j = 0; j < V; ++j) sums[group * D + at.e + z * at.second + j] = dg[w][u].v[z][j];
        }
      }
      __syncthreads();
      for (int d = threadIdx.x; d < D; d += kNormThreads) {
        float s = 0.f;
        for (int i = 0; i < groups; ++i) s += sums[i * D + d];
        g.partial[(static_cast<size_t>(blockIdx.x) * 2 + w) * D + d] = s;
      }
      __syncthreads();
    }
  }
}

// dgamma (=|+=) the blocks' sums, in one order: 32 values a block, 32 lanes of blocks each.
__global__ void __launch_bounds__(1024)
    dgamma_sum_kernel(const float* __restrict__ partial, int blocks, int D, float* dgq, float* dgk, int accumulate) {
  __shared__ float sums[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  float s = 0.f;
  if (col < 2 * D)
    for (int b = part; b < blocks; b += 32) s += partial[static_cast<size_t>(b) * 2 * D + col];
  sums[part][threadIdx.x & 31] = s;
  __syncthreads();
  if (part == 0 && col < 2 * D) {
    float t = 0.f;
    for (int i = 0; i < 32; ++i) t += sums[i][threadIdx.x];
    float* out = col < D ? dgq : dgk;
    if (out) {
      out += col < D ? col : col - D;
      *out = accumulate ? *out + t : t;
    }
  }
}

// Blocks of a call at most: of the backward as many as there are sums of dgamma.
int norm_blocks(bool bwd) { return (bwd ? 2 : 16) * device_sm_count(); }

struct NormPlan {
  int V, U, lanes, tile, G;
  unsigned grid;
  int smem;
};

NormPlan norm_plan(const RopeShape& r, bool bwd) {
  NormPlan p;
  const int vec = r.f32 ? 4 : 8;
  p.V = (r.halves ? r.pairs : 2 * r.pairs) % vec == 0 ? vec : 1;
  const int run = r.halves ? p.V : (p.V == 1 ? 2 : p.V);
  const int units = (r.halves ? r.pairs : 2 * r.pairs) / run + (r.D - 2 * r.pairs) / p.V;
  p.lanes = 1;
  while (p.lanes < units && p.lanes < 32) p.lanes *= 2;
  p.U = p.V == 1 ? 8 : (units + p.lanes - 1) / p.lanes;  // V == 1: at most 255 units of 32 lanes
  // Head slots so that a thread has two turns of q's heads, and no more than there are heads of k; the rest of
  // the block for tokens; with few tokens one token a block, so that more blocks share them. 8 x 4096 tokens of
  // 16 + 2 heads of 128 in bf16: one turn 90 us, two 78; 16 + 16 heads 117 and 111, of 64 64 and 62.
  const int fit = kNormThreads / p.lanes, at_once = norm_at_once(p.U, bwd);
  p.G = (r.Hq + 2 * at_once - 1) / (2 * at_once);
  if (r.Hk > 0 && p.G > r.Hk) p.G = r.Hk;
  if (p.G > fit) p.G = fit;
  p.tile = fit / p.G;
  const long long n_tok = static_cast<long long>(r.B) * r.L, spread = n_tok / device_sm_count();
  if (p.tile > spread) p.tile = spread < 1 ? 1 : static_cast<int>(spread);
  if (p.tile > kNormAngles * kNormThreads / r.pairs) p.tile = kNormAngles * kNormThreads / r.pairs;
  if (p.tile == 1) {  // the block is one token's
    p.G = r.Hq > r.Hk ? r.Hq : r.Hk;
    if (p.G > fit) p.G = fit;
  }
  const long long tiles = (n_tok + p.tile - 1) / p.tile, blocks = norm_blocks(bwd);
  p.grid = static_cast<unsigned>(tiles < blocks ? tiles : blocks);
  p.smem = 4 * p.tile * r.pairs * 4;
  const int sums = fit * r.D * 4;  // <= 32 KB: a lane has 8 U values of a head at most
  if (bwd && sums > p.smem) p.smem = sums;
  return p;
}

// The table of a call's rotation, kept per thread for the calls that follow with the same one: 64 powers
// in long double are 8 us of host time, more than a launch.
const NormTable& norm_table(const RopeShape& r) {
  struct Kept {
    RopeShape of;
    bool valid = false;
    NormTable tab;
  };
  static thread_local Kept kept;
  const auto same = [&r](const RopeShape& o) {
    if (o.axes != r.axes || o.pairs != r.pairs || o.per_axis != r.per_axis || o.base != r.base) return false;
    for (int a = 0; a < r.axes; ++a)
      if (o.sections[a] != r.sections[a]) return false;
    return true;
  };
  if (kept.valid && same(kept.of)) return kept.tab;
  const long double turn = 1.0L / 6.28318530717958647692528676655900577L;
  int i = 0;
  for (int a = 0; a < r.axes; ++a)
    for (int j = 0; j < r.sections[a]; ++j, ++i) {
      const long double f = r.per_axis ? static_cast<long double>(j) / r.sections[a] : static_cast<long double>(i) / r.pairs;
      kept.tab.turns[i] = static_cast<uint64_t>(turn * std::pow(static_cast<long double>(r.base), -f) * 0x1p64L + 0.5L);
      kept.tab.axis[i] = static_cast<uint8_t>(a);
    }
  kept.of = r;
  kept.valid = true;
  return kept.tab;
}

template <typename T, int V, int U, bool HALVES, bool BWD, bool ACC>
int norm_go(const NormPlan& p, const NormArgs<T>& g, const NormTable& tab, cudaStream_t s) {
  qk_norm_rope_kernel<T, V, U, HALVES, BWD, ACC><<<p.grid, kNormThreads, p.smem, s>>>(g, tab);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

template <typename T, int V, int U, bool HALVES>
int norm_go(const NormPlan& p, const NormArgs<T>& g, const NormTable& tab, bool bwd, bool acc, cudaStream_t s) {
  if (!bwd) return norm_go<T, V, U, HALVES, false, false>(p, g, tab, s);
  return acc ? norm_go<T, V, U, HALVES, true, true>(p, g, tab, s) : norm_go<T, V, U, HALVES, true, false>(p, g, tab, s);
}

template <typename T, int V, int U>
int norm_go(const NormPlan& p, const NormArgs<T>& g, const NormTable& tab, bool halves, bool bwd, bool acc,
            cudaStream_t s) {
  return halves ? norm_go<T, V, U, true>(p, g, tab, bwd, acc, s) : norm_go<T, V, U, false>(p, g, tab, bwd, acc, s);
}

template <typename T>
int norm_launch(const NormRope& sh, const NormPlan& p, NormArgs<T>& g, bool bwd, bool acc, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const RopeShape& r = sh.rope;
  g.n_tok = static_cast<long long>(r.B) * r.L;
  g.P = r.pairs;
  g.D = r.D;
  g.lanes = p.lanes;
  g.tile = p.tile;
  g.G = p.G;
  g.eps = sh.eps;
  const NormTable& tab = norm_table(r);
  if (p.V == 1) return norm_go<T, 1, 8>(p, g, tab, r.halves, bwd, acc, s);
  if (p.U == 1) return norm_go<T, V, 1>(p, g, tab, r.halves, bwd, acc, s);
  return norm_go<T, V, 2>(p, g, tab, r.halves, bwd, acc, s);
}

template <typename T>
int norm_fwd(const NormRope& sh, const void* q, const void* k, const float* gq, const float* gk,
             const int32_t* positions, void* qo, void* ko, const NormRopeCache& c, cudaStream_t s) {
  const RopeShape& r = sh.rope;
  NormArgs<T> g = {};
  g.side[0] = {static_cast<const T*>(q), static_cast<T*>(qo), nullptr, gq, r.Hq, sh.q_stride,
               static_cast<long long>(r.Hq) * r.D};
  g.side[1] = {static_cast<const T*>(k), static_cast<T*>(ko), nullptr, gk, r.Hk, sh.k_stride,
               static_cast<long long>(r.Hk) * r.D};
  g.v = static_cast<const T*>(c.v);
  g.v_stride = sh.v_stride;
  g.num_slots = c.num_slots;
  g.slots = c.slots;
  g.k_cache = static_cast<T*>(c.k_cache);
  g.v_cache = static_cast<T*>(c.v_cache);
  g.pos = positions;
  return norm_launch<T>(sh, norm_plan(r, false), g, false, false, s);
}

template <typename T>
int norm_bwd(const NormRope& sh, const void* dqo, const void* dko, const void* q, const void* k, const float* gq,
             const float* gk, const int32_t* positions, void* dq, void* dk, float* dgq, float* dgk, bool acc,
             void* ws, cudaStream_t s) {
  const RopeShape& r = sh.rope;
  NormArgs<T> g = {};
  g.side[0] = {static_cast<const T*>(q), static_cast<T*>(dq), static_cast<const T*>(dqo), gq, r.Hq, sh.q_stride,
               sh.dq_stride};
  g.side[1] = {static_cast<const T*>(k), static_cast<T*>(dk), static_cast<const T*>(dko), gk, r.Hk, sh.k_stride,
               sh.dk_stride};
  g.pos = positions;
  g.partial = static_cast<float*>(ws);
  const NormPlan p = norm_plan(r, true);
  const int st = norm_launch<T>(sh, p, g, true, acc, s);
  if (st != PA_OK || (!dgq && !dgk)) return st;
  dgamma_sum_kernel<<<(2 * r.D + 31) / 32, 1024, 0, s>>>(g.partial, static_cast<int>(p.grid), r.D, dgq, dgk, acc);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // namespace

int launch_qk_norm_rope_fwd(const NormRope& sh, const void* q, const void* k, const float* gq,
                            const float* gk, const int32_t* positions, void* qo, void* ko,
                            const NormRopeCache& cache, cudaStream_t s) {
  return sh.rope.f32 ? norm_fwd<float>(sh, q, k, gq, gk, positions, qo, ko, cache, s)
                     : norm_fwd<__nv_bfloat16>(sh, q, k, gq, gk, positions, qo, ko, cache, s);
}

size_t qk_norm_rope_bwd_workspace_bytes(const NormRope& sh) {
  return static_cast<size_t>(norm_blocks(true)) * 2 * sh.rope.D * sizeof(float);
}

int launch_qk_norm_rope_bwd(const NormRope& sh, const void* dqo, const void* dko, const void* q,
                            const void* k, const float* gq, const float* gk, const int32_t* positions,
                            void* dq, void* dk, float* dgq, float* dgk, bool accumulate, void* ws,
                            cudaStream_t s) {
  return sh.rope.f32
             ? norm_bwd<float>(sh, dqo, dko, q, k, gq, gk, positions, dq, dk, dgq, dgk, accumulate, ws, s)
             : norm_bwd<__nv_bfloat16>(sh, dqo, dko, q, k, gq, gk, positions, dq, dk, dgq, dgk, accumulate, ws, s);
}

}  // namespace pa
