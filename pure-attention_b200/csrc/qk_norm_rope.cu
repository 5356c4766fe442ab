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
#include <cmath>
#include <cuda_bf16.h>
#include "host_launchers.h"

namespace pa {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormMaxPairs = 128;  // head_dim <= 256

struct NormTable {
  double turns[kNormMaxPairs];  // w_i / 2 pi
  uint8_t axis[kNormMaxPairs];
};

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
  int P, D, lanes, tile;  // lanes that share a head (a power of two); tokens of a tile
  float eps;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

// V values at p (16 bytes of them, or one) as floats, and back.
template <int V>
__device__ __forceinline__ void load_run(const float* p, float (&f)[V]) {
  if constexpr (V == 4) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
  } else {
    f[0] = *p;
  }
}
template <int V>
__device__ __forceinline__ void load_run(const __nv_bfloat16* p, float (&f)[V]) {
  if constexpr (V == 8) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  } else {
    f[0] = __bfloat162float(*p);
  }
}
template <int V>
__device__ __forceinline__ void store_run(float* p, const float (&f)[V]) {
  if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  else *p = f[0];
}
template <int V>
__device__ __forceinline__ void store_run(__nv_bfloat16* p, const float (&f)[V]) {
  if constexpr (V == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  else *p = __float2bfloat16_rn(f[0]);
}
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
  static constexpr int N = TWO ? V : V / 2;  // angles of a unit
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

template <int V, bool HALVES>
__device__ __forceinline__ void turn_unit(float (&a)[V], float (&b)[V], const float* co, const float* si, float sign) {
  constexpr int N = UnitAt<V, HALVES>::N;
  float c[N], s[N];
  load_f32<N>(co, c);
  load_f32<N>(si, s);
  if constexpr (UnitAt<V, HALVES>::TWO) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float x = a[j], y = b[j], t = sign * s[j];
      a[j] = x * c[j] - y * t;
      b[j] = y * c[j] + x * t;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = a[2 * j], y = a[2 * j + 1], t = sign * s[j];
      a[2 * j] = x * c[j] - y * t;
      a[2 * j + 1] = y * c[j] + x * t;
    }
  }
}

// T: value type; V: values of a run (16 bytes of them; 1 where the runs are no whole
// vectors); U: units of a lane; BWD: gradients; ACC: added to what dx holds.
// A tile is `tile` tokens; `lanes` lanes share a head, and the block's groups of lanes
// take the tile's heads one after the other.
template <typename T, int V, int U, bool HALVES, bool BWD, bool ACC>
__global__ void __launch_bounds__(kNormThreads)
    qk_norm_rope_kernel(const __grid_constant__ NormArgs<T> g, const __grid_constant__ NormTable tab) {
  using At = UnitAt<V, HALVES>;
  extern __shared__ __align__(16) float tables[];  // 2 x (cos [tile][P], sin [tile][P])
  const int lane = threadIdx.x & (g.lanes - 1), group = threadIdx.x / g.lanes, groups = kNormThreads / g.lanes;
  const int P = g.P, D = g.D;
  const float inv_d = 1.f / D;
  float dg[2][U][2][V];
  if (BWD) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) dg[i][u][0][j] = dg[i][u][1][j] = 0.f;
  }
  const long long n_tiles = (g.n_tok + g.tile - 1) / g.tile;
  int parity = 0;
#pragma unroll 1
  for (long long tile = blockIdx.x; tile < n_tiles; tile += gridDim.x, parity ^= 1) {
    float *cosines = tables + parity * 2 * g.tile * P, *sines = cosines + g.tile * P;
    const long long t0 = tile * g.tile;
    const int nt = static_cast<int>(g.n_tok - t0 < g.tile ? g.n_tok - t0 : g.tile);
    for (int i = threadIdx.x; i < nt * P; i += kNormThreads) {
      const int ti = i / P, p = i - ti * P;
      const double u = static_cast<double>(g.pos[tab.axis[p] * g.n_tok + t0 + ti]) * tab.turns[p];
      float s, c;
      sincospif(2.f * static_cast<float>(u - rint(u)), &s, &c);
      cosines[i] = c;
      sines[i] = s;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const NormSide<T>& sd = g.side[w];
      if (!sd.x) continue;
      // all lanes of a warp take the same number of turns: the sums are over whole warps
      const int items = nt * sd.heads, turns = (items + groups - 1) / groups;
#pragma unroll 1
      for (int k = 0; k < turns; ++k) {
        const int i = group + k * groups;
        const bool live = i < items;
        const int t = live ? i / sd.heads : 0, h = live ? i - t * sd.heads : 0;
        const long long tok = t0 + t;
        const T* src = sd.x + tok * sd.x_stride + static_cast<long long>(h) * D;
        float a[U][2][V], y[U][2][V];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const At at(lane + u * g.lanes, P, D);
#pragma unroll
          for (int j = 0; j < V; ++j) a[u][0][j] = a[u][1][j] = y[u][0][j] = y[u][1][j] = 0.f;
          if (!live || !at.on) continue;
          load_run<V>(src + at.e, a[u][0]);
          if (At::TWO && at.turns) load_run<V>(src + at.e + at.second, a[u][1]);
          if (BWD) {
            const T* dy = sd.dy + (tok * sd.heads + h) * D;
            load_run<V>(dy + at.e, y[u][0]);
            if (At::TWO && at.turns) load_run<V>(dy + at.e + at.second, y[u][1]);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const At at(lane + u * g.lanes, P, D);
          if (BWD && live && at.on && at.turns)
            turn_unit<V, HALVES>(y[u][0], y[u][1], cosines + t * P + at.angle, sines + t * P + at.angle, -1.f);
#pragma unroll
          for (int j = 0; j < V; ++j) s1 += a[u][0][j] * a[u][0][j] + a[u][1][j] * a[u][1][j];
        }
        float r = 1.f;
        if (sd.gamma) {
          float gm[U][2][V];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const At at(lane + u * g.lanes, P, D);
#pragma unroll
            for (int j = 0; j < V; ++j) gm[u][0][j] = gm[u][1][j] = 0.f;
            if (!at.on) continue;
            load_f32<V>(sd.gamma + at.e, gm[u][0]);
            if (At::TWO && at.turns) load_f32<V>(sd.gamma + at.e + at.second, gm[u][1]);
            if (BWD) {
#pragma unroll
              for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int j = 0; j < V; ++j) s2 += y[u][z][j] * gm[u][z][j] * a[u][z][j];
            }
          }
          for (int m = g.lanes / 2; m > 0; m >>= 1) {
            s1 += __shfl_xor_sync(0xffffffffu, s1, m);
            if (BWD) s2 += __shfl_xor_sync(0xffffffffu, s2, m);
          }
          r = rsqrtf(s1 * inv_d + g.eps);
          const float back = r * r * s2 * inv_d;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
              for (int j = 0; j < V; ++j) {
                if (BWD) {
                  if (live) dg[w][u][z][j] += y[u][z][j] * (a[u][z][j] * r);
                  a[u][z][j] = r * (y[u][z][j] * gm[u][z][j] - a[u][z][j] * back);
                } else {
                  a[u][z][j] = a[u][z][j] * r * gm[u][z][j];
                }
              }
        } else if (BWD) {
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) a[u][0][j] = y[u][0][j], a[u][1][j] = y[u][1][j];
        }
        if (!live) continue;
        T* dst = sd.y ? sd.y + tok * sd.y_stride + static_cast<long long>(h) * D : nullptr;
        T* row = nullptr;
        if (!BWD && w == 1 && g.slots) {
          const long long slot = g.slots[tok];
          if (slot >= 0 && slot < g.num_slots) row = g.k_cache + (slot * sd.heads + h) * D;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const At at(lane + u * g.lanes, P, D);
          if (!at.on) continue;
          if (!BWD && at.turns)
            turn_unit<V, HALVES>(a[u][0], a[u][1], cosines + t * P + at.angle, sines + t * P + at.angle, 1.f);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            if (z == 1 && !(At::TWO && at.turns)) continue;
            const int e = at.e + z * at.second;
            if (ACC) {
              float old[V];
              load_run<V>(dst + e, old);
#pragma unroll
              for (int j = 0; j < V; ++j) a[u][z][j] += old[j];
            }
            if (dst) store_run<V>(dst + e, a[u][z]);
            if (row) store_run<V>(row + e, a[u][z]);
          }
        }
      }
    }
    if (!BWD && g.slots) {  // v as it is, 16 bytes at a time
      constexpr int W = 16 / sizeof(T);
      const int per = g.side[1].heads * D / W;
      for (int i = threadIdx.x; i < nt * per; i += kNormThreads) {
        const int t = i / per, e = (i - t * per) * W;
        const long long slot = g.slots[t0 + t];
        if (slot >= 0 && slot < g.num_slots)
          *reinterpret_cast<uint4*>(g.v_cache + slot * g.side[1].heads * D + e) =
              *reinterpret_cast<const uint4*>(g.v + (t0 + t) * g.v_stride + e);
      }
    }
  }
  if (BWD) {
    // this block's sums of dgamma: the groups' one after the other
    __syncthreads();
    float* sums = tables;  // [groups][D]
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const At at(lane + u * g.lanes, P, D);
        if (!at.on) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sums[group * D + at.e + j] = dg[w][u][0][j];
          if (At::TWO && at.turns) sums[group * D + at.e + at.second + j] = dg[w][u][1][j];
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

int norm_blocks() { return 4 * device_sm_count(); }

struct NormPlan {
  int V, U, lanes, tile;
  unsigned grid;
  size_t smem;
};

NormPlan norm_plan(const RopeShape& r, bool bwd) {
  NormPlan p;
  const int vec = r.f32 ? 4 : 8;
  p.V = (r.halves ? r.pairs : 2 * r.pairs) % vec == 0 ? vec : 1;
  const int run = r.halves ? p.V : (p.V == 1 ? 2 : p.V);
  const int units = (r.halves ? r.pairs : 2 * r.pairs) / run + (r.D - 2 * r.pairs) / p.V;
  p.lanes = 1;
  while (p.lanes < units && p.lanes < 32) p.lanes *= 2;
  p.U = (units + p.lanes - 1) / p.lanes;
  const int groups = kNormThreads / p.lanes, heads = r.Hq + r.Hk;
  const long long n_tok = static_cast<long long>(r.B) * r.L;
  // a few heads a group and tile; with few tokens one token a block, so that more blocks share them
  p.tile = (4 * groups + heads - 1) / heads;
  const long long spread = n_tok / device_sm_count();
  if (p.tile > spread) p.tile = spread < 1 ? 1 : static_cast<int>(spread);
  if (p.tile > 16) p.tile = 16;  // 2 x 2 x 16 x 128 fp32 of angles at most: 32 KB
  const long long tiles = (n_tok + p.tile - 1) / p.tile;
  p.grid = static_cast<unsigned>(tiles < norm_blocks() ? tiles : norm_blocks());
  p.smem = 4 * static_cast<size_t>(p.tile) * r.pairs * sizeof(float);
  const size_t sums = static_cast<size_t>(groups) * r.D * sizeof(float);  // <= 32 KB (groups * D <= 8192)
  if (bwd && sums > p.smem) p.smem = sums;
  return p;
}

NormTable norm_table(const RopeShape& r) {
  NormTable tab;
  const double turn = 1.0 / 6.283185307179586476925286766559, log2_base = std::log2(r.base);
  int i = 0;
  for (int a = 0; a < r.axes; ++a)
    for (int j = 0; j < r.sections[a]; ++j, ++i) {
      const double f = r.per_axis ? static_cast<double>(j) / r.sections[a] : static_cast<double>(i) / r.pairs;
      tab.turns[i] = turn * std::exp2(-f * log2_base);
      tab.axis[i] = static_cast<uint8_t>(a);
    }
  return tab;
}

template <typename T, int V, int U, bool HALVES>
void norm_go(const NormPlan& p, const NormArgs<T>& g, const NormTable& tab, bool bwd, bool acc, cudaStream_t s) {
  if (!bwd) qk_norm_rope_kernel<T, V, U, HALVES, false, false><<<p.grid, kNormThreads, p.smem, s>>>(g, tab);
  else if (!acc) qk_norm_rope_kernel<T, V, U, HALVES, true, false><<<p.grid, kNormThreads, p.smem, s>>>(g, tab);
  else qk_norm_rope_kernel<T, V, U, HALVES, true, true><<<p.grid, kNormThreads, p.smem, s>>>(g, tab);
}

template <typename T, int V, int U>
void norm_go(const NormPlan& p, const NormArgs<T>& g, const NormTable& tab, bool halves, bool bwd, bool acc,
             cudaStream_t s) {
  if (halves) norm_go<T, V, U, true>(p, g, tab, bwd, acc, s);
  else norm_go<T, V, U, false>(p, g, tab, bwd, acc, s);
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
  g.eps = sh.eps;
  const NormTable tab = norm_table(r);
  if (p.V == 1) norm_go<T, 1, 8>(p, g, tab, r.halves, bwd, acc, s);  // at most 255 units of 32 lanes
  else if (p.U == 1) norm_go<T, V, 1>(p, g, tab, r.halves, bwd, acc, s);
  else norm_go<T, V, 2>(p, g, tab, r.halves, bwd, acc, s);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
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
  return static_cast<size_t>(norm_blocks()) * 2 * sh.rope.D * sizeof(float);
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
