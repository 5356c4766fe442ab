// Attention of one new token of each sequence over its paged cache.
//
//   o = sum_t exp(q.k_t scale - lse) v_t over the cached tokens t of the sequence
//
// Bound by HBM: every cached key and value is read once and used by the heads of one group.
// A unit is (sequence, kv head, up to 16 heads of its group); all units' keys
// are laid end to end in tiles of 64 and dealt out to the CTAs in equal runs, whatever the lengths
// of the sequences: a CTA may hold several units, or a piece of a long one. A unit that lies in one
// CTA is finished there; the pieces of the others (running maximum, sum, unnormalised o) go to
// the workspace and a second kernel joins them in order. Nothing is counted in
// memory, so a workspace may hold anything before the call and results do not depend on the run.
//
// Within a CTA a warp takes 16 keys of each tile through a ring of its own in shared memory
// (cp.async, no barrier between warps) and keeps its own softmax statistics; the warps are merged
// when the unit ends. bf16: the heads are the 16 rows of mma.m16n8k16 (the 5th-generation
// tensor core wants 64 rows at least, and its rate is not needed: 32 products for
// 16 keys of 128 values take a third of the time that HBM needs for them). fp32: plain FMA, exact
// to fp32 rounding.
#include <cuda_bf16.h>
#include "packed_common.cuh"

namespace pa {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kWarps = 4, kKeys = 16;         // keys of a warp and tile
constexpr int kTileKeys = kWarps * kKeys;

// n / d for 0 <= n < 2^31 as a multiplication: m = floor(2^(31 + s) / d) + 1 with 2^s >= d.
struct Divisor {
  uint32_t m, shift;
  explicit Divisor(int d = 1) {
    uint32_t s = 0;
    while ((1ll << s) < d) ++s;
    shift = 31 + s;
    m = static_cast<uint32_t>((1ull << shift) / d + 1);
  }
  __device__ int of(int n) const { return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * m >> shift); }
};

// A call's sizes, and the places of its units' pieces.
struct PagedArgs {
  PagedShape sh;
  Divisor page;
  int end_tiles;            // 1, or 0 where a unit has one tile at most
  float scale_log2;
  int chunks, chunk_heads;  // chunks of a group, heads of each
  float* pieces;            // [2 * CTAs][piece_floats]
  int2* spans;              // [units]: first and last CTA of each
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16-byte piece c of row r of a warp's K or V block (rows of ROW bytes): swizzled, so that eight rows'
// same piece lies in eight different groups of banks.
template <int ROW>
__device__ __forceinline__ uint32_t piece_at(int r, int c) {
  return static_cast<uint32_t>(r * ROW + ((c ^ (r & 7)) << 4));
}

// ---------------------------------------------------------------- bf16: one warp's softmax over its keys
// Both products are taken transposed, S^T = K Q^T and o^T = V^T P^T: keys, then values, are the 16 rows
// of mma.m16n8k16 and up to 8 heads (NB times 8) its columns, so that few heads waste little of it. Thread
// (g = lane / 4, c = lane % 4) holds heads 2 c and 2 c + 1 of each 8 in both results.
template <int D, int NB>
struct Bf16Core {
  using T = bf16;
  static constexpr int ROWS = 8 * NB, ROW = D * 2;
  static constexpr int STATE = NB * (8 * D + 16);  // floats of a warp's state: o, then each head's m and sum
  uint32_t q[NB][D / 16][2];
  float m[NB][2], l[NB][2], o[NB][D / 16][4];

  __device__ void start(const bf16* x, int heads) {  // x: the chunk's first head
    const int g = lane_id() / 4, c = lane_id() % 4;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          q[n][k][i] = 8 * n + g < heads
                           ? *reinterpret_cast<const uint32_t*>(x + (8 * n + g) * D + k * 16 + 2 * c + 8 * i)
                           : 0u;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.f;
    }
  }

  // keys: bit t = key t of the block counts
  __device__ void block(uint32_t sK, uint32_t sV, uint32_t keys, float scale_log2) {
    const int lane = lane_id(), g = lane / 4;
    // ldmatrix rows: lane's row of the 8x8 matrix lane / 8
    const int r8 = lane & 7, mat = lane >> 3;
    uint32_t kb[D / 16][4], vb[D / 16][4];
#pragma unroll
    for (int k = 0; k < D / 16; ++k)  // keys 0-7, 8-15 of values 0-7, then of values 8-15
      ldmatrix4(sK + piece_at<ROW>(r8 + 8 * (mat & 1), 2 * k + (mat >> 1)), kb[k]);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)  // values 0-7, 8-15 of keys 0-7, then of keys 8-15
      ldmatrix4_trans(sV + piece_at<ROW>(r8 + 8 * (mat >> 1), 2 * k + (mat & 1)), vb[k]);
    uint32_t p[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float s[4] = {}, s2[4] = {};  // even and odd steps: two chains of products
#pragma unroll
      for (int k = 0; k < D / 16; ++k) mma_16816(k & 1 ? s2 : s, kb[k], q[n][k][0], q[n][k][1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = (s[i] + s2[i]) * scale_log2;
      if (keys != 0xffffu) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!((keys >> (g + 8 * (i >> 1))) & 1)) s[i] = -INFINITY;
      }
      float top[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
#pragma unroll
      for (int d = 4; d < 32; d <<= 1)
#pragma unroll
        for (int h = 0; h < 2; ++h) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
      // m rises only by more than 8 (p <= 2^8 is exact in fp32 and bf16): o is seldom rescaled
      if (__any_sync(0xffffffffu, top[0] > m[n][0] + 8.f || top[1] > m[n][1] + 8.f)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float to = fmaxf(m[n][h], top[h]), a = to == -INFINITY ? 1.f : ex2(m[n][h] - to);
          m[n][h] = to;
          l[n][h] *= a;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            o[n][k][h] *= a;
            o[n][k][2 + h] *= a;
          }
        }
      }
      const float base[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = ex2(s[2 * i] - base[0]), y = ex2(s[2 * i + 1] - base[1]);
        l[n][0] += x;
        l[n][1] += y;
        // rounded once, for the product with v; key rows become head rows
        asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p[n][i]) : "r"(pack_bf16x2(x, y)));
      }
    }
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int n = 0; n < NB; ++n) mma_16816(o[n][k], vb[k], p[n][0], p[n][1]);
  }

  // A head's sum over the eight threads that hold its keys.
  __device__ float row_sum(int n, int h) const {
    float sum = l[n][h];
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
  }
  __device__ void dump(float* to) const {
    const int lane = lane_id();
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float sum = row_sum(n, h);
        if (lane < 4) *reinterpret_cast<float2*>(to + NB * 8 * D + 2 * (8 * n + 2 * lane + h)) = make_float2(m[n][h], sum);
      }
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[((n * (D / 16) + k) * 4 + i) * 32 + lane] = o[n][k][i];
    }
  }
  __device__ void merge(const float* from) {
    const int lane = lane_id();
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 other = *reinterpret_cast<const float2*>(from + NB * 8 * D + 2 * (8 * n + 2 * (lane % 4) + h));
        const float to = fmaxf(m[n][h], other.x);
        const float a = to == -INFINITY ? 1.f : ex2(m[n][h] - to), b = to == -INFINITY ? 0.f : ex2(other.x - to);
        m[n][h] = to;
        l[n][h] = l[n][h] * a + (lane < 4 ? other.y * b : 0.f);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int i = h; i < 4; i += 2)
            o[n][k][i] = o[n][k][i] * a + from[((n * (D / 16) + k) * 4 + i) * 32 + lane] * b;
      }
  }
  // f(row, m, l) once a head and f(row, column, value, l) for the warp's state
  template <typename F, typename G>
  __device__ void each(int heads, F row_of, G value_of) {
    const int g = lane_id() / 4, c = lane_id() % 4;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float sum = row_sum(n, h);
        const int row = 8 * n + 2 * c + h;
        if (row >= heads) continue;
        if (g == 0) row_of(row, m[n][h], sum);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          value_of(row, k * 16 + g, o[n][k][h], sum);
          value_of(row, k * 16 + g + 8, o[n][k][2 + h], sum);
        }
      }
  }
};

// ---------------------------------------------------------------- fp32
// HC heads. Scores: lane = (key, half of its values); products with v: lane = D / 32 values.
template <int D, int HC>
struct F32Core {
  using T = float;
  static constexpr int ROWS = HC, ROW = D * 4;
  static constexpr int N = D / 32, STATE = 32 * HC * (2 + N);
  float m[HC], l[HC], o[HC][N];
  float *q, *p;  // shared, of this warp: [HC][D] and [HC][16]

  __device__ void start(const float* x, int heads) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        o[h][i] = 0.f;
        q[h * D + i * 32 + lane_id()] = h < heads ? x[h * D + i * 32 + lane_id()] : 0.f;
      }
    }
    __syncwarp();
  }

  __device__ void block(const uint8_t* sK, const uint8_t* sV, uint32_t keys, float scale_log2) {
    const int lane = lane_id(), key = lane & 15, half = lane >> 4;
    float k[D / 2];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
      *reinterpret_cast<float4*>(&k[4 * i]) =
          *reinterpret_cast<const float4*>(sK + piece_at<ROW>(key, half * (D / 8) + i));
    const bool on = (keys >> key) & 1;
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      float2 s2 = make_float2(0.f, 0.f), t2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(q + h * D + half * (D / 2) + 4 * i);
        s2 = __ffma2_rn(make_float2(k[4 * i], k[4 * i + 1]), make_float2(x.x, x.y), s2);
        t2 = __ffma2_rn(make_float2(k[4 * i + 2], k[4 * i + 3]), make_float2(x.z, x.w), t2);
      }
      float s = (s2.x + s2.y) + (t2.x + t2.y);
      s += __shfl_xor_sync(0xffffffffu, s, 16);
      s = on ? s * scale_log2 : -INFINITY;
      float top = s;
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      if (top > m[h]) {  // the same in all lanes
        const float a = ex2(m[h] - top);
        m[h] = top;
        l[h] *= a;
#pragma unroll
        for (int i = 0; i < N; ++i) o[h][i] *= a;
      }
      const float w = ex2(s - (m[h] == -INFINITY ? 0.f : m[h]));
      if (half == 0) {
        l[h] += w;  // this key's; summed over the lanes at the end
        p[h * 16 + key] = w;
      }
    }
    __syncwarp();
#pragma unroll
    for (int t = 0; t < 16; t += 4) {
      float v[4][N];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* row = sV + piece_at<ROW>(t + j, lane * N / 4) + (lane * N % 4) * 4;
        if constexpr (N == 2) {
          const float2 x = *reinterpret_cast<const float2*>(row);
          v[j][0] = x.x;
          v[j][N - 1] = x.y;
        } else {
          v[j][0] = *reinterpret_cast<const float*>(row);
        }
      }
#pragma unroll
      for (int h = 0; h < HC; ++h) {
        const float4 w = *reinterpret_cast<const float4*>(p + h * 16 + t);
        const float ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < N; ++i) o[h][i] = fmaf(ws[j], v[j][i], o[h][i]);
      }
    }
    __syncwarp();
  }

  __device__ void dump(float* to) const {
    const int lane = lane_id();
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      to[h * 32 + lane] = m[h];
      to[(HC + h) * 32 + lane] = l[h];
#pragma unroll
      for (int i = 0; i < N; ++i) to[(2 * HC + h * N + i) * 32 + lane] = o[h][i];
    }
  }
  __device__ void merge(const float* from) {
    const int lane = lane_id();
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      const float om = from[h * 32 + lane], to = fmaxf(m[h], om);
      const float a = to == -INFINITY ? 1.f : ex2(m[h] - to), b = to == -INFINITY ? 0.f : ex2(om - to);
      m[h] = to;
      l[h] = l[h] * a + from[(HC + h) * 32 + lane] * b;
#pragma unroll
      for (int i = 0; i < N; ++i) o[h][i] = o[h][i] * a + from[(2 * HC + h * N + i) * 32 + lane] * b;
    }
  }
  template <typename F, typename G>
  __device__ void each(int heads, F row_of, G value_of) {
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      float sum = l[h];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (h >= heads) continue;
      if (lane_id() == 0) row_of(h, m[h], sum);
#pragma unroll
      for (int i = 0; i < N; ++i) value_of(h, N * static_cast<int>(lane_id()) + i, o[h][i], sum);
    }
  }
};

template <typename Core>
struct PagedSmem;
template <int D, int NB>
struct PagedSmem<Bf16Core<D, NB>> {
  static constexpr int CTAS = NB == 1 ? 3 : 2;  // that share an SM
  static constexpr int STAGES = (NB == 1 ? 2 : 3) * (128 / D), EXTRA = 0;
};
template <int D, int HC>
struct PagedSmem<F32Core<D, HC>> {
  static constexpr int CTAS = 2;
  static constexpr int STAGES = D == 64 ? 3 : 5, EXTRA = HC * (D + 16) * 4;  // q and p of a warp
};
template <typename Core>
constexpr int paged_smem() {
  return kWarps * (PagedSmem<Core>::STAGES * 2 * kKeys * Core::ROW + PagedSmem<Core>::EXTRA) +
         2 * Core::STATE * 4;
}
// Floats of a unit's piece: o, then each row's m and sum; whole 16 bytes.
template <int ROWS, int D>
__host__ __device__ constexpr int piece_floats() {
  return (ROWS * (D + 2) + 3) / 4 * 4;
}

__device__ __forceinline__ int keys_of(const PagedArgs& a, const int32_t* lens, int b) {
  return min(max(__ldg(lens + b), 0), a.sh.max_pages * a.sh.page_size);
}
// Tiles of a sequence, and one without keys: the end of a unit takes about as long as a tile, so that
// many short sequences make no CTA late. Without it (a cache of one tile) no unit is cut.
__device__ __forceinline__ int tiles_of(const PagedArgs& a, int keys) {
  return max(1 - a.end_tiles, (keys + kTileKeys - 1) / kTileKeys) + a.end_tiles;
}

// Where a tile of the whole run of tiles lies.
struct TileAt {
  int b, kh, chunk, tile, n_tiles, len;  // sequence, kv head, chunk; tile of the unit, its tiles, its keys
  long long left;                        // tiles of the CTA's run still to come, this one too
};

template <typename Core, int D>
__global__ void __launch_bounds__(kWarps * 32, PagedSmem<Core>::CTAS)
    paged_step_kernel(const __grid_constant__ PagedArgs a, const typename Core::T* __restrict__ q,
                      const typename Core::T* __restrict__ kc, const typename Core::T* __restrict__ vc,
                      const int32_t* __restrict__ table, const int32_t* __restrict__ lens,
                      typename Core::T* __restrict__ o, float* __restrict__ lse) {
  using T = typename Core::T;
  constexpr int STAGES = PagedSmem<Core>::STAGES, ROW = Core::ROW, BLOCK = kKeys * ROW;
  constexpr int PIECES = ROW / 16, ROWS_A_GO = 32 / PIECES;  // 16-byte pieces of a row, rows a warp copies at once
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ long long s_scan[kWarps], s_total;
  __shared__ TileAt s_first;
  const int warp = warp_id(), lane = lane_id();
  const int parts = a.sh.Hk * a.chunks, group = a.sh.H / a.sh.Hk;
  launch_dependents();

  // This CTA's run of tiles: every thread a run of sequences, their tiles' prefix sum, and the
  // thread that holds the first tile finds its place.
  const int per = (a.sh.B + kWarps * 32 - 1) / (kWarps * 32);
  const int lo = min(a.sh.B, static_cast<int>(threadIdx.x) * per), hi = min(a.sh.B, lo + per);
  long long mine = 0;
  for (int b = lo; b < hi; ++b) mine += tiles_of(a, keys_of(a, lens, b));
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += x;
  }
  if (lane == 31) s_scan[warp] = upto;
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += s_scan[w];
  if (threadIdx.x == kWarps * 32 - 1) s_total = upto;
  __syncthreads();
  const long long total = s_total * parts, run = (total + gridDim.x - 1) / gridDim.x;
  const long long begin = blockIdx.x * run;
  if (begin >= total) return;
  if ((upto - mine) * parts <= begin && begin < upto * parts) {
    long long at = (upto - mine) * parts;
    int b = lo, len = keys_of(a, lens, b);
    while (at + static_cast<long long>(tiles_of(a, len)) * parts <= begin) {
      at += static_cast<long long>(tiles_of(a, len)) * parts;
      len = keys_of(a, lens, ++b);
    }
    const int n = tiles_of(a, len), part = static_cast<int>((begin - at) / n);
    s_first = {b, part / a.chunks, part % a.chunks, static_cast<int>((begin - at) % n), n, len,
               min(run, total - begin)};
  }
  __syncthreads();
  TileAt use = s_first;
  auto advance = [&](TileAt& t) {
    --t.left;
    if (++t.tile < t.n_tiles || t.left <= 0) return;
    t.tile = 0;
    if (++t.chunk < a.chunks) return;
    t.chunk = 0;
    if (++t.kh < a.sh.Hk) return;
    t.kh = 0;
    t.len = keys_of(a, lens, ++t.b);
    t.n_tiles = tiles_of(a, t.len);
  };

  uint8_t* ring = smem + warp * STAGES * 2 * BLOCK;
  float* scratch = reinterpret_cast<float*>(smem + kWarps * STAGES * 2 * BLOCK);
  Core core;
  if constexpr (sizeof(T) == 4) {
    core.q = scratch + 2 * Core::STATE + warp * (Core::ROWS * (D + 16));
    core.p = core.q + Core::ROWS * D;
  }

  // The place in the pools of lane's key of a tile (lanes 0-15), or -1; loaded a tile ahead.
  auto slot_of = [&](const TileAt& t) {
    const int key = t.tile * kTileKeys + warp * kKeys + (lane & 15);
    if (t.left <= 0 || key >= t.len) return -1;
    const int i = a.page.of(key), page = __ldg(table + static_cast<size_t>(t.b) * a.sh.max_pages + i);
    return page < 0 || page >= a.sh.num_pages ? -1 : (page - i) * a.sh.page_size + key;
  };
  TileAt ahead = use;
  int slot = slot_of(ahead);
  uint32_t keys_in[STAGES];
  // Copies the tile at `ahead` into stage `st`; rows that are no keys become zeros, so that what lies
  // there cannot meet a weight of zero as NaN.
  const int my_row = lane / PIECES, my_col = lane % PIECES;
  const size_t pitch = static_cast<size_t>(a.sh.Hk) * D;
  auto fetch = [&](int st, uint32_t& keys) {
    keys = __ballot_sync(0xffffffffu, slot >= 0) & 0xffffu;
    if (keys) {
      const uint32_t dst = smem_u32(ring + st * 2 * BLOCK);
      const int head = ahead.kh * D + my_col * (16 / static_cast<int>(sizeof(T)));
      const T *k0 = kc + head, *v0 = vc + head;
#pragma unroll
      for (int i = 0; i < kKeys / ROWS_A_GO; ++i) {
        const int r = i * ROWS_A_GO + my_row;
        const int s = __shfl_sync(0xffffffffu, slot, r);
        const size_t at = static_cast<uint32_t>(max(s, 0)) * pitch;
        cp_async16(dst + piece_at<ROW>(r, my_col), k0 + at, s >= 0);
        cp_async16(dst + BLOCK + piece_at<ROW>(r, my_col), v0 + at, s >= 0);
      }
    }
    cp_async_commit();
    advance(ahead);
    slot = slot_of(ahead);
  };
#pragma unroll
  for (int st = 0; st < STAGES - 1; ++st) fetch(st, keys_in[st]);

  auto q_of = [&](const TileAt& t, int* heads, int* first) {
    *heads = min(a.chunk_heads, group - t.chunk * a.chunk_heads);
    *first = t.kh * group + t.chunk * a.chunk_heads;
    return q + t.b * a.sh.q_stride + static_cast<size_t>(*first) * D;
  };
  int heads, first;
  {
    const T* x = q_of(use, &heads, &first);
    core.start(x, heads);
  }
  bool from_before = use.tile > 0;  // the unit began in an earlier CTA
  while (use.left > 0) {
#pragma unroll
    for (int st = 0; st < STAGES; ++st) {  // unrolled: the stage is a constant
      if (use.left <= 0) break;
      cp_async_wait<STAGES - 2>();
      __syncwarp();
      {
        const int to = (st + STAGES - 1) % STAGES;
        fetch(to, keys_in[to]);
      }
      const uint32_t keys = keys_in[st];
      if (keys) {
        if constexpr (sizeof(T) == 2)
          core.block(smem_u32(ring + st * 2 * BLOCK), smem_u32(ring + st * 2 * BLOCK + BLOCK), keys, a.scale_log2);
        else
          core.block(ring + st * 2 * BLOCK, ring + st * 2 * BLOCK + BLOCK, keys, a.scale_log2);
      }
      __syncwarp();
      const TileAt was = use;
      advance(use);
      const bool ends = was.tile + 1 == was.n_tiles;
      if (!ends && use.left > 0) continue;
      // The unit, or this CTA's run, ends: merge the warps, 2 and 3 into 0 and 1, then 1 into 0.
      if (warp >= 2) core.dump(scratch + (warp - 2) * Core::STATE);
      __syncthreads();
      if (warp < 2) core.merge(scratch + warp * Core::STATE);
      __syncthreads();
      if (warp == 1) core.dump(scratch);
      __syncthreads();
      if (warp == 0) {
        core.merge(scratch);
        if (ends && !from_before) {
          const size_t out = static_cast<size_t>(was.b) * a.sh.H + first;
          core.each(
              heads,
              [&](int row, float m, float l) {
                if (lse) lse[out + row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
              },
              [&](int row, int col, float x, float l) {
                const float y = l == 0.f ? 0.f : x / l;
                if constexpr (sizeof(T) == 2) o[(out + row) * D + col] = __float2bfloat16_rn(y);
                else o[(out + row) * D + col] = y;
              });
        } else {
          // slot 0 of a CTA: a unit from before; slot 1: one that goes on in the next
          float* to = a.pieces + (2 * static_cast<size_t>(blockIdx.x) + (from_before ? 0 : 1)) * piece_floats<Core::ROWS, D>();
          core.each(
              heads,
              [&](int row, float m, float l) {
                *reinterpret_cast<float2*>(to + Core::ROWS * D + 2 * row) = make_float2(m, l);
              },
              [&](int row, int col, float x, float) { to[row * D + col] = x; });
        }
        if (!from_before && lane == 0) {  // the CTAs of a unit, told by the first
          const int later = static_cast<int>((was.n_tiles - 1 - was.tile + run - 1) / run);
          a.spans[static_cast<size_t>(was.b) * parts + was.kh * a.chunks + was.chunk] = make_int2(blockIdx.x, blockIdx.x + (ends ? 0 : later));
        }
      }
      __syncthreads();
      if (use.left > 0) {
        from_before = false;
        const T* x = q_of(use, &heads, &first);
        core.start(x, heads);
      }
    }
  }
  cp_async_wait<0>();
}

// Joins the pieces of the units that several CTAs hold: a block takes (sequence, head).
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(128)
    paged_join_kernel(const __grid_constant__ PagedArgs a, T* __restrict__ o, float* __restrict__ lse) {
  constexpr int LANES = D / 4, PARTS = 128 / LANES;  // threads that share a row, pieces at a time
  __shared__ float s_m[128], s_l[PARTS], s_o[PARTS][D];
  const int group = a.sh.H / a.sh.Hk, b = blockIdx.x / a.sh.H, h = blockIdx.x % a.sh.H, gh = h % group;
  const int part = h / group * a.chunks + gh / a.chunk_heads, row = gh % a.chunk_heads;
  wait_prerequisites();
  const int2 span = a.spans[static_cast<size_t>(b) * a.sh.Hk * a.chunks + part];
  if (span.x == span.y) return;
  const int n = span.y - span.x + 1;
  auto piece = [&](int i) {  // the first CTA's last unit, the others' first
    return a.pieces + (2 * static_cast<size_t>(span.x + i) + (i == 0 ? 1 : 0)) * piece_floats<ROWS, D>();
  };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < n; i += 128) m = fmaxf(m, piece(i)[ROWS * D + 2 * row]);
  s_m[threadIdx.x] = m;
  __syncthreads();
  for (int d = 64; d > 0; d >>= 1) {
    if (threadIdx.x < d) s_m[threadIdx.x] = fmaxf(s_m[threadIdx.x], s_m[threadIdx.x + d]);
    __syncthreads();
  }
  m = s_m[0];
  const int lane = threadIdx.x % LANES, p = threadIdx.x / LANES;
  float l = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = p; i < n; i += PARTS) {
    const float* from = piece(i);
    const float2 ml = *reinterpret_cast<const float2*>(from + ROWS * D + 2 * row);
    const float4 y = *reinterpret_cast<const float4*>(from + row * D + 4 * lane);
    const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
    l = fmaf(ml.y, w, l);
    x.x = fmaf(y.x, w, x.x), x.y = fmaf(y.y, w, x.y), x.z = fmaf(y.z, w, x.z), x.w = fmaf(y.w, w, x.w);
  }
  *reinterpret_cast<float4*>(&s_o[p][4 * lane]) = x;
  if (lane == 0) s_l[p] = l;
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) sum += s_l[i];
  for (int d = threadIdx.x; d < D; d += 128) {
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) y += s_o[i][d];
    y = sum == 0.f ? 0.f : y / sum;
    T* to = o + static_cast<size_t>(blockIdx.x) * D + d;
    if constexpr (sizeof(T) == 2) *to = __float2bfloat16_rn(y);
    else *to = y;
  }
  if (lse && threadIdx.x == 0) lse[blockIdx.x] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * kLn2;
}

// Heads of a chunk of a group, and the chunks: as even as they go.
struct PagedPlan {
  int chunks, chunk_heads, ctas;
};
PagedPlan paged_plan(const PagedShape& sh) {
  const int group = sh.H / sh.Hk, most = sh.f32 ? 8 : 16;
  PagedPlan p;
  p.chunks = (group + most - 1) / most;
  p.chunk_heads = (group + p.chunks - 1) / p.chunks;
  p.ctas = (!sh.f32 && p.chunk_heads <= 8 ? 3 : 2) * device_sm_count();
  return p;
}

template <typename Core, int D>
int paged_launch(const PagedShape& sh, const PagedPlan& p, const void* q, const void* kc, const void* vc,
                 const int32_t* table, const int32_t* lens, void* o, float* lse, void* ws, cudaStream_t s) {
  using T = typename Core::T;
  static std::atomic<uint64_t> attr{0};
  if (!ensure_smem_attr(paged_step_kernel<Core, D>, paged_smem<Core>(), attr)) return PA_ERR_LAUNCH;
  PagedArgs a;
  a.sh = sh;
  a.page = Divisor(sh.page_size);
  a.scale_log2 = sh.scale * kLog2e;
  a.chunks = p.chunks;
  a.chunk_heads = p.chunk_heads;
  a.pieces = static_cast<float*>(ws);
  a.spans = reinterpret_cast<int2*>(a.pieces + 2 * static_cast<size_t>(p.ctas) * 16 * (D + 2));
  // as many CTAs as there can be tiles of keys
  const long long unit_tiles = (static_cast<long long>(sh.max_pages) * sh.page_size + kTileKeys - 1) / kTileKeys;
  a.end_tiles = unit_tiles > 1;
  const long long tiles = static_cast<long long>(sh.B) * sh.Hk * p.chunks * (unit_tiles + a.end_tiles);
  const int grid = static_cast<int>(tiles < p.ctas ? tiles : p.ctas);
  paged_step_kernel<Core, D><<<grid, kWarps * 32, paged_smem<Core>(), s>>>(
      a, static_cast<const T*>(q), static_cast<const T*>(kc), static_cast<const T*>(vc), table, lens,
      static_cast<T*>(o), lse);
  if (cudaGetLastError() != cudaSuccess) return PA_ERR_LAUNCH;
  if (unit_tiles == 1) return PA_OK;  // no unit is cut
  return launch_beside(paged_join_kernel<T, D, Core::ROWS>, dim3(sh.B * sh.H), 128, 0, s, a, static_cast<T*>(o), lse);
}

template <int D>
int paged_bf16(const PagedShape& sh, const PagedPlan& p, const void* q, const void* kc, const void* vc,
               const int32_t* table, const int32_t* lens, void* o, float* lse, void* ws, cudaStream_t s) {
  if (p.chunk_heads <= 8) return paged_launch<Bf16Core<D, 1>, D>(sh, p, q, kc, vc, table, lens, o, lse, ws, s);
  return paged_launch<Bf16Core<D, 2>, D>(sh, p, q, kc, vc, table, lens, o, lse, ws, s);
}

template <int D>
int paged_f32(const PagedShape& sh, const PagedPlan& p, const void* q, const void* kc, const void* vc,
              const int32_t* table, const int32_t* lens, void* o, float* lse, void* ws, cudaStream_t s) {
  if (p.chunk_heads <= 1) return paged_launch<F32Core<D, 1>, D>(sh, p, q, kc, vc, table, lens, o, lse, ws, s);
  if (p.chunk_heads <= 2) return paged_launch<F32Core<D, 2>, D>(sh, p, q, kc, vc, table, lens, o, lse, ws, s);
  if (p.chunk_heads <= 4) return paged_launch<F32Core<D, 4>, D>(sh, p, q, kc, vc, table, lens, o, lse, ws, s);
  return paged_launch<F32Core<D, 8>, D>(sh, p, q, kc, vc, table, lens, o, lse, ws, s);
}

}  // namespace

size_t paged_attn_workspace_bytes(const PagedShape& sh) {
  const PagedPlan p = paged_plan(sh);
  return 2 * static_cast<size_t>(p.ctas) * 16 * (sh.D + 2) * sizeof(float) +
         (static_cast<size_t>(sh.B) * sh.Hk * p.chunks * sizeof(int2) + 255) / 256 * 256;
}

int launch_paged_attn(const PagedShape& sh, const void* q, const void* kc, const void* vc, const int32_t* table,
                      const int32_t* lens, void* o, float* lse, void* ws, cudaStream_t s) {
  const PagedPlan p = paged_plan(sh);
  if (sh.f32)
    return sh.D == 32 ? paged_f32<32>(sh, p, q, kc, vc, table, lens, o, lse, ws, s)
                      : paged_f32<64>(sh, p, q, kc, vc, table, lens, o, lse, ws, s);
  return sh.D == 64 ? paged_bf16<64>(sh, p, q, kc, vc, table, lens, o, lse, ws, s)
                    : paged_bf16<128>(sh, p, q, kc, vc, table, lens, o, lse, ws, s);
}

}  // namespace pa
