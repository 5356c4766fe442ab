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
// when the unit ends. bf16: mma.m16n8k16 with keys, and then values, as the 16 rows and up to 8 heads as
// the columns (16 heads: two), since a group of few heads fills 8 columns sooner than 16 rows; the 5th-generation
// tensor core wants 64 rows at least, and its rate is not needed (the pipe is 9% busy). fp32: plain FMA,
// exact to fp32 rounding.
//
// Measured, against 6550 GB/s of a plain copy: 64 sequences of up to 8192 tokens, 16 + 4 heads of 128 in bf16, 72 us
// (5.1 TB/s), 444 sequences of 1024 154 us (6.1 TB/s), two contexts of 131072 with 16 + 2 heads 56 us (4.8 TB/s: 50
// the step, 6 the join). What is left is the start of a CTA (lengths, their prefix sum, the first pages) and the
// join. The base of shared memory lies on a line: cp.async takes a line of memory in one request only
// where it lands in one line there, and a base 16 bytes off made four of each.
#include <cuda_bf16.h>
#include <type_traits>
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
  // Unit, first and last CTA of what the join takes: of each unit, or (cuts_by_cta) of the unit that begins
  // in a CTA and goes on in the next, of which a CTA has one at most, whichever is fewer.
  int4* cuts;
  int cuts_by_cta;
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
  static constexpr int TURN = NB == 1 ? 64 : 32;  // values of a head that are merged at a time
  uint32_t q[NB][D / 16][2];
  float m[NB][2], l[NB][2], o[NB][D / 16][4];

  __device__ void load_q(const bf16* x, int heads) {  // x: the chunk's first head
    const int g = lane_id() / 4, c = lane_id() % 4;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          q[n][k][i] = 8 * n + g < heads
                           ? *reinterpret_cast<const uint32_t*>(x + (8 * n + g) * D + k * 16 + 2 * c + 8 * i)
                           : 0u;
  }
  __device__ void start() {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.f;
    }
  }

  // A block's K and V into registers, so that the ring can be filled again at once.
  uint32_t kb[D / 16][4], vb[D / 16][4];
  __device__ void load(const uint8_t* k_block, const uint8_t* v_block) {
    // ldmatrix rows: lane's row of the 8x8 matrix lane / 8
    const int r8 = lane_id() & 7, mat = lane_id() >> 3;
    const uint32_t sK = smem_u32(k_block), sV = smem_u32(v_block);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)  // keys 0-7, 8-15 of values 0-7, then of values 8-15
      ldmatrix4(sK + piece_at<ROW>(r8 + 8 * (mat & 1), 2 * k + (mat >> 1)), kb[k]);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)  // values 0-7, 8-15 of keys 0-7, then of keys 8-15
      ldmatrix4_trans(sV + piece_at<ROW>(r8 + 8 * (mat >> 1), 2 * k + (mat & 1)), vb[k]);
  }

  // keys: bit t = key t of the block counts
  __device__ void block(uint32_t keys, float scale_log2) {
    const int g = lane_id() / 4;
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

  // A head's maximum and sum, and TURN of its values from TURN * turn on, into the warp's part of the
  // scratch memory (rows of TURN + 4 floats: no two lanes meet in a bank).
  __device__ void dump_ml(float2* to) const {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[n][h];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane_id() < 4) to[8 * n + 2 * lane_id() + h] = make_float2(m[n][h], sum);
      }
  }
  template <int TURN_NO>
  __device__ void dump(float* to) const {
    const int g = lane_id() / 4, c = lane_id() % 4;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int k = 0; k < TURN / 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          to[(8 * n + 2 * c + (i & 1)) * (TURN + 4) + k * 16 + g + 8 * (i >> 1)] = o[n][TURN_NO * (TURN / 16) + k][i];
  }
};

// ---------------------------------------------------------------- fp32
// HC heads. Scores: lane = (key, half of its values); products with v: lane = D / 32 values.
template <int D, int HC>
struct F32Core {
  using T = float;
  static constexpr int ROWS = HC, ROW = D * 4;
  static constexpr int N = D / 32, TURN = D;
  float m[HC], l[HC], o[HC][N];
  float *q, *p;  // shared, of this warp: [HC][D] and [HC][16]

  __device__ void load_q(const float* x, int heads) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < HC; ++h)
#pragma unroll
      for (int i = 0; i < N; ++i)
        q[h * D + i * 32 + lane_id()] = h < heads ? x[h * D + i * 32 + lane_id()] : 0.f;
    __syncwarp();
  }
  __device__ void start() {
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) o[h][i] = 0.f;
    }
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

  __device__ void dump_ml(float2* to) const {
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      float sum = l[h];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane_id() == 0) to[h] = make_float2(m[h], sum);
    }
  }
  template <int>
  __device__ void dump(float* to) const {
#pragma unroll
    for (int h = 0; h < HC; ++h)
#pragma unroll
      for (int i = 0; i < N; ++i) to[h * (D + 4) + N * lane_id() + i] = o[h][i];
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
         kWarps * Core::ROWS * (Core::TURN + 4) * 4;
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
  // whole lines: cp.async takes a line of memory in one request only where it lands in one line here
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_scan[kWarps], s_total;
  __shared__ TileAt s_first;
  __shared__ float2 s_ml[kWarps][Core::ROWS];
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
  if (begin >= total) {
    if (a.cuts_by_cta && threadIdx.x == 0) a.cuts[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
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
    core.q = scratch + kWarps * Core::ROWS * (Core::TURN + 4) + warp * (Core::ROWS * (D + 16));
    core.p = core.q + Core::ROWS * D;
  }

  // The page of lane's key of a tile (lanes 0-15) is loaded a tile ahead, and looked at only when that
  // tile is copied: an instruction that uses it any sooner would stop the warp until it is there.
  auto key_of = [&](const TileAt& t) {
    const int key = t.tile * kTileKeys + warp * kKeys + (lane & 15);
    return t.left > 0 && key < t.len ? key : -1;
  };
  auto page_of = [&](const TileAt& t) {
    const int key = key_of(t);
    return key < 0 ? -1 : __ldg(table + static_cast<size_t>(t.b) * a.sh.max_pages + a.page.of(key));
  };
  TileAt ahead = use;
  int page = page_of(ahead);
  uint32_t keys_in[STAGES];
  // Copies the tile at `ahead` into stage `st`; rows that are no keys become zeros, so that what lies
  // there cannot meet a weight of zero as NaN.
  const int my_row = lane / PIECES, my_col = lane % PIECES;
  const size_t pitch = static_cast<size_t>(a.sh.Hk) * D;
  auto fetch = [&](int st, uint32_t& keys) {
    const int key = key_of(ahead);  // -1 with page -1
    const int slot = page < 0 || page >= a.sh.num_pages ? -1 : (page - a.page.of(key)) * a.sh.page_size + key;
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
    page = page_of(ahead);
  };
#pragma unroll
  for (int st = 0; st < STAGES; ++st) fetch(st, keys_in[st]);

  auto q_of = [&](const TileAt& t, int* heads, int* first) {
    *heads = min(a.chunk_heads, group - t.chunk * a.chunk_heads);
    *first = t.kh * group + t.chunk * a.chunk_heads;
    return q + t.b * a.sh.q_stride + static_cast<size_t>(*first) * D;
  };
  int heads, first;
  {
    const T* x = q_of(use, &heads, &first);
    core.load_q(x, heads);
    core.start();
  }
  bool from_before = use.tile > 0;  // the unit began in an earlier CTA
  while (use.left > 0) {
#pragma unroll
    for (int st = 0; st < STAGES; ++st) {  // unrolled: the stage is a constant
      if (use.left <= 0) break;
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t keys = keys_in[st];
      const uint8_t *k_block = ring + st * 2 * BLOCK, *v_block = k_block + BLOCK;
      if constexpr (sizeof(T) == 2) {
        if (keys) core.load(k_block, v_block);
        __syncwarp();
        fetch(st, keys_in[st]);
        if (keys) core.block(keys, a.scale_log2);
      } else {
        if (keys) core.block(k_block, v_block, keys, a.scale_log2);
        __syncwarp();
        fetch(st, keys_in[st]);
      }
      const TileAt was = use;
      advance(use);
      const bool ends = was.tile + 1 == was.n_tiles;
      if (!ends && use.left > 0) continue;
      // The unit, or this CTA's run, ends. The next unit's q is loaded while the warps' states are merged
      // through the scratch memory, TURN values of each head at a time, by all threads.
      const int was_heads = heads, was_first = first;
      if (use.left > 0) {
        const T* x = q_of(use, &heads, &first);
        core.load_q(x, heads);
      }
      const bool whole = ends && !from_before;
      // slot 0 of a CTA: a unit from before; slot 1: one that goes on in the next
      float* piece = a.pieces + (2 * static_cast<size_t>(blockIdx.x) + (from_before ? 0 : 1)) * piece_floats<Core::ROWS, D>();
      const size_t out = static_cast<size_t>(was.b) * a.sh.H + was_first;
      constexpr int TURN = Core::TURN, FOURS = TURN / 4;
      auto merge = [&](auto turn) {
        constexpr int AT = decltype(turn)::value * TURN;
        __syncthreads();  // the scratch memory is free
        if (AT == 0) core.dump_ml(s_ml[warp]);
        core.template dump<decltype(turn)::value>(scratch + warp * Core::ROWS * (TURN + 4));
        __syncthreads();
        for (int i = threadIdx.x; i < was_heads * FOURS; i += kWarps * 32) {
          const int row = i / FOURS, col = i % FOURS * 4;
          float m = -INFINITY, l = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ml[w][row].x);
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float2 ml = s_ml[w][row];
            const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
            const float4 y = *reinterpret_cast<const float4*>(scratch + (w * Core::ROWS + row) * (TURN + 4) + col);
            l = fmaf(ml.y, f, l);
            x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
          }
          if (!whole) {
            *reinterpret_cast<float4*>(piece + row * D + AT + col) = x;
            if (AT == 0 && col == 0) *reinterpret_cast<float2*>(piece + Core::ROWS * D + 2 * row) = make_float2(m, l);
            continue;
          }
          const float inv = l == 0.f ? 0.f : 1.f / l;
          T* to = o + (out + row) * D + AT + col;
          if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
          else
            *reinterpret_cast<float4*>(to) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
          if (lse && AT == 0 && col == 0) lse[out + row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
        }
      };
      merge(std::integral_constant<int, 0>());
      if constexpr (D / TURN > 1) merge(std::integral_constant<int, 1>());
      if constexpr (D / TURN > 2) {
        merge(std::integral_constant<int, 2>());
        merge(std::integral_constant<int, 3>());
      }
      if (warp == 0) {
        if (!from_before && lane == 0 && (!a.cuts_by_cta || !ends)) {  // told by the first of a unit's CTAs
          const int unit = (was.b * a.sh.Hk + was.kh) * a.chunks + was.chunk;
          const int later = ends ? 0 : static_cast<int>((was.n_tiles - 1 - was.tile + run - 1) / run);
          a.cuts[a.cuts_by_cta ? blockIdx.x : unit] = make_int4(unit, blockIdx.x, blockIdx.x + later, 0);
        }
        if (a.cuts_by_cta && lane == 0 && use.left <= 0 && (from_before || ends))
          a.cuts[blockIdx.x] = make_int4(0, 0, 0, 0);  // nothing that begins here goes on
      }
      from_before = false;
      core.start();
    }
  }
  cp_async_wait<0>();
}

// Joins the pieces of the units that several CTAs hold: a block takes (cut unit, head). Its threads share
// the pieces out, each with a running maximum, so that the loads of all pieces are on their way at once.
constexpr int kJoinThreads = 256;
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads)
    paged_join_kernel(const __grid_constant__ PagedArgs a, T* __restrict__ o, float* __restrict__ lse) {
  constexpr int LANES = D / 4, PARTS = kJoinThreads / LANES;  // threads that share a row, pieces at a time
  __shared__ float2 s_ml[PARTS];
  __shared__ __align__(16) float s_o[PARTS][D];
  const int row = blockIdx.x % a.chunk_heads;
  wait_prerequisites();
  const int4 cut = a.cuts[blockIdx.x / a.chunk_heads];  // unit, first and last CTA
  const int group = a.sh.H / a.sh.Hk, chunk = cut.x % a.chunks, n = cut.z - cut.y + 1;
  if (n <= 1 || chunk * a.chunk_heads + row >= group) return;
  auto piece = [&](int i) {  // the first CTA's last unit, the others' first
    return a.pieces + (2 * static_cast<size_t>(cut.y + i) + (i == 0 ? 1 : 0)) * piece_floats<ROWS, D>();
  };
  const int lane = threadIdx.x % LANES, p = threadIdx.x / LANES;
  float m = -INFINITY, l = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 ml, float4 y) {
    const float to = fmaxf(m, ml.x);
    const float u = to == -INFINITY ? 1.f : ex2(m - to), w = ml.x == -INFINITY ? 0.f : ex2(ml.x - to);
    m = to;
    l = l * u + ml.y * w;
    x.x = x.x * u + y.x * w, x.y = x.y * u + y.y * w, x.z = x.z * u + y.z * w, x.w = x.w * u + y.w * w;
  };
  constexpr int GO = 8;
#pragma unroll 1
  for (int i0 = p; i0 < n; i0 += GO * PARTS) {
    float2 ml[GO];
    float4 y[GO];
#pragma unroll
    for (int k = 0; k < GO; ++k) {
      const int i = i0 + k * PARTS;
      if (i < n) {
        const float* from = piece(i);
        ml[k] = *reinterpret_cast<const float2*>(from + ROWS * D + 2 * row);
        y[k] = *reinterpret_cast<const float4*>(from + row * D + 4 * lane);
      }
    }
#pragma unroll
    for (int k = 0; k < GO; ++k)
      if (i0 + k * PARTS < n) add(ml[k], y[k]);
  }
  *reinterpret_cast<float4*>(&s_o[p][4 * lane]) = x;
  if (lane == 0) s_ml[p] = make_float2(m, l);
  __syncthreads();
  if (p > 0) return;
#pragma unroll
  for (int i = 1; i < PARTS; ++i) add(s_ml[i], *reinterpret_cast<const float4*>(&s_o[i][4 * lane]));
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int unit = cut.x / a.chunks;  // (sequence, kv head)
  const size_t out = static_cast<size_t>(unit / a.sh.Hk) * a.sh.H + (unit % a.sh.Hk) * group + chunk * a.chunk_heads + row;
  T* to = o + out * D + 4 * lane;
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
  else
    *reinterpret_cast<float4*>(to) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  if (lse && lane == 0) lse[out] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
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
  a.cuts = reinterpret_cast<int4*>(a.pieces + 2 * static_cast<size_t>(p.ctas) * 16 * (D + 2));
  // as many CTAs as there can be tiles of keys
  const long long unit_tiles = (static_cast<long long>(sh.max_pages) * sh.page_size + kTileKeys - 1) / kTileKeys;
  a.end_tiles = unit_tiles > 1;
  const long long tiles = static_cast<long long>(sh.B) * sh.Hk * p.chunks * (unit_tiles + a.end_tiles);
  const int grid = static_cast<int>(tiles < p.ctas ? tiles : p.ctas);
  a.cuts_by_cta = static_cast<long long>(sh.B) * sh.Hk * p.chunks > grid;
  paged_step_kernel<Core, D><<<grid, kWarps * 32, paged_smem<Core>(), s>>>(
      a, static_cast<const T*>(q), static_cast<const T*>(kc), static_cast<const T*>(vc), table, lens,
      static_cast<T*>(o), lse);
  if (cudaGetLastError() != cudaSuccess) return PA_ERR_LAUNCH;
  if (unit_tiles == 1) return PA_OK;  // no unit is cut
  const int cuts = a.cuts_by_cta ? grid : sh.B * sh.Hk * p.chunks;
  return launch_beside(true, paged_join_kernel<T, D, Core::ROWS>, dim3(cuts * p.chunk_heads), kJoinThreads, 0, s, a,
                       static_cast<T*>(o), lse);
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
         p.ctas * sizeof(int4);
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
