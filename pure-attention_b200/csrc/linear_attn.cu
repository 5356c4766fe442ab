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

// ---------------------------------------------------------------- chunked kernel
// A sequence in chunks of C = 128 tokens. With S the state entering a chunk of n
// valid tokens (rows i, j of the chunk; l the decay):
//   O   = scale (P V + diag(l^(i+1)) Q S),   P = (Q K^T) o l^(i-j) for j <= i, else 0
//   S' = l^n S + K^T V',                      V' = diag(l^(n-1-j)) V
// All four products run on the tensor cores; every power of l has a whole,
// non-negative exponent, so nothing overflows where l is small.
//
// One CTA per SM walks units (sequence, head, 64 columns of V, segment of the
// sequence); a unit's chunks follow one another through the state, and the
// rings below run on across units.
//   warps 0-3   P: load Q K^T from TMEM, times l^(i-j), bf16 back to TMEM; then the
//               previous chunk's O out
//   warps 4-7   the state in fp32 registers (thread = row of the state), its bf16
//               parts to shared memory for Q S
//   warp 8      tcgen05.mma issue
//   warps 9-12  k and q into 128-byte swizzled tiles: bf16 by cp.async, fp32 through
//               registers, split on the way
//   warps 13-16 v through registers into V and V'
//               (Rows past the sequence are zeros, rows may run backwards in
//               time, and fp32 is split: none of these fits a plain TMA box.)
// Q and K feed two products each as they lie: K as the K-major B of Q K^T and as the
// MN-major A of K^T V'.
//
// Roundings: fp32 sums and state throughout. V' and the state are two bf16
// parts (off by 2^-16), so states keep fp32-like accuracy; P is one bf16 (2^-8),
// as in the softmax kernels. NT = 3 (fp32 operands): every operand is a
// hi/lo pair and every product hi*hi + hi*lo + lo*hi.
//
// TMEM columns: Q K^T and P 2 x 128 (P of 32 tokens over their 32 scores: hi in the
// first 16 columns, lo in the others), Q S 64, P V 64, K^T V' 2 x 64.
//
// The loops below stay rolled where they can: six roles that each run a long
// straight line once per chunk miss the instruction cache (measured: 38% of the
// stall cycles, 5500 against XXXX clocks a chunk).
constexpr int kMixThreads = 17 * 32;
constexpr int kTile = 128 * 128;  // bytes of 128 rows x 64 bf16

template <int DK, int NT>
struct MixCfg {
  static constexpr int NP = NT == 3 ? 2 : 1;       // planes (hi, lo) of q, k, v
  static constexpr int KT = DK / 64;               // 64-column tiles of q and k
  static constexpr int OPER = NP * KT * kTile;     // bytes of q (or k) of a stage
  static constexpr int V_STAGE = (NP + 2) * kTile; // v, and V' hi and lo
  static constexpr int ST_PLANE = DK * 128;        // [DK, 64] bf16
  static constexpr bool SMALL = NP == 1 && DK == 64;
  static constexpr int QKS = SMALL ? 3 : 2, VS = SMALL ? 2 : 1, STB = DK == 64 ? 2 : 1;
  static constexpr int SMEM = QKS * 2 * OPER + VS * V_STAGE + STB * 2 * ST_PLANE + 1024;
  static constexpr int NC = DK == 64 ? 32 : 64;    // state columns of a thread
};
static_assert(MixCfg<64, 1>::SMEM <= 226 * 1024 && MixCfg<64, 3>::SMEM <= 226 * 1024 &&
              MixCfg<128, 1>::SMEM <= 226 * 1024, "shared memory of one CTA");

struct MixOne {  // one direction of the recurrence
  const void *q, *k, *v;
  void* o;
  const float* s_in;
  float* s_out;
  MixDir dir;
};
struct MixArgs {
  MixOne one[3];
  int n_dir;
  const float* log_decay;
  const int32_t* lens;
  float* ws;  // segment states, see seg_slot
  int B, L, H, D;
  int n_seg, seg_tokens, n_units;
  float scale;
};

struct MixUnit {
  int dir, b, h, half, seg;
  int n;          // valid tokens of the sequence
  int p0, count;  // first position and tokens of this segment
  int chunks;
};

// unit -> (segment, sequence, head, direction, column half), halves and
// directions of one head next to one another: they read the same rows, from L2
template <int DK>
__device__ __forceinline__ MixUnit mix_unit(const MixArgs& a, int u) {
  MixUnit x;
  constexpr int halves = DK / 64;
  x.half = u % halves;
  u /= halves;
  x.dir = u % a.n_dir;
  u /= a.n_dir;
  x.h = u % a.H;
  u /= a.H;
  x.b = u % a.B;
  x.seg = u / a.B;
  x.n = valid_tokens(a.lens, x.b, a.L);
  x.p0 = x.seg * a.seg_tokens;
  const int left = x.n - x.p0;
  x.count = left < 0 ? 0 : (left < a.seg_tokens ? left : a.seg_tokens);
  x.chunks = (x.count + 127) >> 7;
  return x;
}

// Workspace of a sequence cut in segments: per (sequence, head, direction, half)
// n_seg slots of [DK, 64] fp32. Slot s < n_seg - 1 holds the state of segment s
// alone (from zero), slot n_seg - 1 a copy of the carried state (state_out may
// overwrite state_in while other segments still need it).
template <int DK>
__device__ __forceinline__ float* seg_slot(const MixArgs& a, const MixUnit& x, int slot) {
  const size_t w = ((static_cast<size_t>(x.b) * a.H + x.h) * a.n_dir + x.dir) * (DK / 64) + x.half;
  return a.ws + (w * a.n_seg + slot) * (DK * 64);
}

__device__ __forceinline__ uint32_t lo_pair(float a, float b, uint32_t hi) {
  return pack_bf16x2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}

// The chunks of this CTA in order, for the loading warps.
template <int DK>
struct ChunkIter {
  MixUnit x;
  int u, chunk, g;  // g: chunks of this CTA so far
  __device__ __forceinline__ bool first(const MixArgs& a) {
    u = blockIdx.x;
    chunk = g = 0;
    return settle(a);
  }
  __device__ __forceinline__ bool settle(const MixArgs& a) {  // to a unit that has chunks
    for (; u < a.n_units; u += gridDim.x) {
      x = mix_unit<DK>(a, u);
      if (x.chunks > 0) return true;
    }
    return false;
  }
  __device__ __forceinline__ bool next(const MixArgs& a) {
    ++g;
    if (++chunk < x.chunks) return true;
    chunk = 0;
    u += gridDim.x;
    return settle(a);
  }
  __device__ __forceinline__ int valid() const {  // valid rows of the chunk
    const int left = x.count - chunk * 128;
    return left < 128 ? left : 128;
  }
};

// Rows of 64 values (one column tile) of a chunk, dealt to the 128 threads of a
// loading group in 16-byte vectors: thread t has column vector t % PER_ROW of rows
// t / PER_ROW + i * ROWS.
template <typename T>
struct Rows {
  static constexpr int PER_ROW = 64 * static_cast<int>(sizeof(T)) / 16;  // 8 or 16
  static constexpr int ROWS = 128 / PER_ROW;                             // rows a pass: 16 or 8
  const T* src;
  long long step;
  int row0, valid;  // valid = 0 past the head's columns
  template <int DK>
  __device__ __forceinline__ Rows(const MixArgs& a, const ChunkIter<DK>& it, const void* base, int tile, int t) {
    const bool rev = a.one[it.x.dir].dir.reverse;
    const int col = (t % PER_ROW) * (16 / static_cast<int>(sizeof(T)));
    row0 = t / PER_ROW;
    valid = tile * 64 + col < a.D ? it.valid() : 0;  // head dim 32 fills half a tile
    const int pos = it.x.p0 + it.chunk * 128 + row0;
    const long long tok = static_cast<long long>(it.x.b) * a.L + (rev ? it.x.n - 1 - pos : pos);
    step = static_cast<long long>(a.H) * a.D * ROWS * (rev ? -1 : 1);
    src = static_cast<const T*>(base) + (tok * a.H + it.x.h) * a.D + tile * 64 + col;
  }
  __device__ __forceinline__ int row(int i) const { return row0 + i * ROWS; }
  __device__ __forceinline__ uint4 load(int i) const {
    return row(i) < valid ? __ldg(reinterpret_cast<const uint4*>(src + i * step)) : make_uint4(0, 0, 0, 0);
  }
};

// 16 bytes global -> shared, zeros where !ok (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
// One arrival on `bar` once this thread's cp.asyncs so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Four (fp32) or eight (bf16) values of row `row` from byte column `cb` on, as
// bf16 hi and, where `lo` is not 0, lo.
__device__ __forceinline__ void put4(uint32_t hi, uint32_t lo, uint32_t off, float a, float b, float c, float d) {
  const uint32_t h0 = pack_bf16x2(a, b), h1 = pack_bf16x2(c, d);
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(hi + off), "r"(h0), "r"(h1) : "memory");
  if (lo)
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(lo + off), "r"(lo_pair(a, b, h0)),
                 "r"(lo_pair(c, d, h1)) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// V (hi, and lo where NP = 2; not for segment states) and V' = diag(l^(valid - 1 - row)) V
// in two parts, from one vector of V.
template <typename T, int NP, bool STATES>
__device__ __forceinline__ void store_v(uint4 r, int row, int t, uint32_t at, float w) {
  const uint32_t x[4] = {r.x, r.y, r.z, r.w};
  if constexpr (sizeof(T) == 2) {
    const uint32_t off = sw128_offset(row, (t % 8) * 16);
    if (!STATES) st_shared_v4(at + off, x[0], x[1], x[2], x[3]);
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = w * __uint_as_float(x[j] << 16), b = w * __uint_as_float(x[j] & 0xffff0000u);
      h[j] = pack_bf16x2(a, b);
      l[j] = lo_pair(a, b, h[j]);
    }
    st_shared_v4(at + kTile + off, h[0], h[1], h[2], h[3]);
    st_shared_v4(at + 2 * kTile + off, l[0], l[1], l[2], l[3]);
  } else {
    const uint32_t off = sw128_offset(row, (t % 16) * 8);
    const float f[4] = {__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3])};
    if (!STATES) put4(at, NP == 2 ? at + kTile : 0, off, f[0], f[1], f[2], f[3]);
    put4(at + NP * kTile, at + (NP + 1) * kTile, off, w * f[0], w * f[1], w * f[2], w * f[3]);
  }
}

// Lane l of each group of 4 holds 4 16-byte vectors of row l; afterwards lane a holds
// vector a of rows 0 .. 3, so that 4 lanes store 64 contiguous bytes (one row per
// lane would spread every store over 32 rows).
__device__ __forceinline__ void transpose4(uint4 (&v)[4]) {
#pragma unroll
  for (int s = 1; s < 4; s *= 2) {
    const bool up = (lane_id() & s) != 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & s) continue;
      const uint4 give = up ? v[i] : v[i + s];
      uint4 got;
      got.x = __shfl_xor_sync(0xffffffffu, give.x, s);
      got.y = __shfl_xor_sync(0xffffffffu, give.y, s);
      got.z = __shfl_xor_sync(0xffffffffu, give.z, s);
      got.w = __shfl_xor_sync(0xffffffffu, give.w, s);
      if (up) v[i] = got;
      else v[i + s] = got;
    }
  }
}

// f[0..15] += 16 values of an output row.
__device__ __forceinline__ void add16(const float* src, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 o = reinterpret_cast<const float4*>(src)[i];
    f[4 * i] += o.x;
    f[4 * i + 1] += o.y;
    f[4 * i + 2] += o.z;
    f[4 * i + 3] += o.w;
  }
}
__device__ __forceinline__ void add16(const __nv_bfloat16* src, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 o = reinterpret_cast<const uint4*>(src)[i];
    const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[8 * i + 2 * j] += __uint_as_float(w[j] << 16);
      f[8 * i + 2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(bar);
}

// STATES: only the segments' own states, into the workspace.
template <typename T, int DK, int NT, bool STATES>
__global__ void __launch_bounds__(kMixThreads, 1) mix_kernel(const __grid_constant__ MixArgs a, uint32_t* status) {
  using C = MixCfg<DK, NT>;
  constexpr int NP = C::NP, KT = C::KT;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[26];
  __shared__ __align__(16) float wtab[256];  // powers of the decay, a table for each P warp
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  if (cta_aborted(status, &abort_flag)) return;
  const uint32_t sm0 = smem_u32(align1024(smem_raw));
  const uint32_t sv0 = sm0 + C::QKS * 2 * C::OPER, ss0 = sv0 + C::VS * C::V_STAGE;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  // ring slot s: K planes, then Q planes; V, V' hi, V' lo; state hi, lo
  auto sK = [&](int s) { return sm0 + s * 2 * C::OPER; };
  auto sQ = [&](int s) { return sm0 + s * 2 * C::OPER + C::OPER; };
  auto sV = [&](int s) { return sv0 + s * C::V_STAGE; };
  auto sS = [&](int s) { return ss0 + s * 2 * C::ST_PLANE; };
  enum { QK_FULL = 0, QK_EMPTY = 3, V_FULL = 6, V_EMPTY = 8, S_FULL = 10, P_FULL = 12, KV_FULL = 14,
         KV_FREE = 16, ST_FULL = 18, ST_EMPTY = 20, O_FULL = 22, O_FREE = 23 };
  constexpr uint32_t T_S = 0, T_QS = 256, T_PV = 320, T_KV = 384;

  const int warp = warp_id();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) {
      mbar_init(bar(QK_FULL + i), 128);
      mbar_init(bar(QK_EMPTY + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(V_FULL + i), 4);
      mbar_init(bar(V_EMPTY + i), 1);
      mbar_init(bar(S_FULL + i), 1);
      mbar_init(bar(P_FULL + i), 4);
      mbar_init(bar(KV_FULL + i), 1);
      mbar_init(bar(KV_FREE + i), 4);
      mbar_init(bar(ST_FULL + i), 4);
      mbar_init(bar(ST_EMPTY + i), 1);
    }
    mbar_init(bar(O_FULL), 1);
    mbar_init(bar(O_FREE), 4);
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;

  if (warp >= 13) {
    // ------------------------------------------------------------ v: one chunk ahead in registers
    const int t = threadIdx.x - 13 * 32;
    constexpr int VECS = 128 / Rows<T>::ROWS;
    uint4 r[VECS];
    ChunkIter<DK> it;
    bool more = it.first(a);
    if (more) {
      const Rows<T> rows(a, it, a.one[it.x.dir].v, it.x.half, t);
#pragma unroll
      for (int i = 0; i < VECS; ++i) r[i] = rows.load(i);
    }
    float w[VECS];  // the rows' powers of the decay, kept while they stay the same
    int w_unit = -1, w_valid = 0;
    while (more) {
      const int g = it.g, vs = g % C::VS, valid = it.valid();
      if (it.u != w_unit || valid != w_valid) {
        const float l2 = log2_decay(a.log_decay, it.x.h);
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
          const int row = t / Rows<T>::PER_ROW + i * Rows<T>::ROWS;
          w[i] = row < valid ? exp2f(l2 * static_cast<float>(valid - 1 - row)) : 0.f;
        }
        w_unit = it.u;
        w_valid = valid;
      }
      if (g >= C::VS && !mbar_wait_warp(bar(V_EMPTY + vs), (g / C::VS - 1) & 1, status)) break;
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        const int row = t / Rows<T>::PER_ROW + i * Rows<T>::ROWS;
        store_v<T, NP, STATES>(r[i], row, t, sV(vs), w[i]);
      }
      fence_proxy_async_smem();
      warp_arrive(bar(V_FULL + vs));
      more = it.next(a);
      if (more) {
        const Rows<T> rows(a, it, a.one[it.x.dir].v, it.x.half, t);
#pragma unroll
        for (int i = 0; i < VECS; ++i) r[i] = rows.load(i);
      }
    }
  } else if (warp >= 9) {
    // ------------------------------------------------------------ k and q
    const int t = threadIdx.x - 9 * 32;
    constexpr int TILES = STATES ? KT : 2 * KT;  // k tiles, then q tiles
    ChunkIter<DK> it;
    bool more = it.first(a);
    auto rows_of = [&](int tile) {
      const MixOne& one = a.one[it.x.dir];
      return Rows<T>(a, it, tile < KT ? one.k : one.q, tile % KT, t);
    };
    auto tile_at = [&](int s, int tile) { return (tile < KT ? sK(s) : sQ(s)) + (tile % KT) * kTile; };
    if constexpr (sizeof(T) == 2) {
      // straight into the ring; the barrier completes as the copies land
      for (; more; more = it.next(a)) {
        const int g = it.g, s = g % C::QKS;
        if (g >= C::QKS && !mbar_wait_warp(bar(QK_EMPTY + s), (g / C::QKS - 1) & 1, status)) break;
#pragma unroll 1
        for (int tile = 0; tile < TILES; ++tile) {
          const Rows<T> rows = rows_of(tile);
          const uint32_t at = tile_at(s, tile);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool ok = rows.row(i) < rows.valid;
            cp_async16(at + sw128_offset(rows.row(i), (t % 8) * 16), ok ? rows.src + i * rows.step : rows.src, ok);
          }
        }
        cp_async_arrive(bar(QK_FULL + s));
      }
    } else {
      // through registers, half a tile at a time, the next half always in flight
      uint4 r0[8], r1[8];
      auto load_half = [&](uint4 (&r)[8], int tile, int half) {
        const Rows<T> rows = rows_of(tile);
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = rows.load(half * 8 + j);
      };
      auto put_half = [&](const uint4 (&r)[8], uint32_t at, int half) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          put4(at, NP == 2 ? at + KT * kTile : 0, sw128_offset(t / 16 + (half * 8 + j) * 8, (t % 16) * 8),
               __uint_as_float(r[j].x), __uint_as_float(r[j].y), __uint_as_float(r[j].z), __uint_as_float(r[j].w));
      };
      if (more) load_half(r0, 0, 0);
      while (more) {
        const int g = it.g, s = g % C::QKS;
        if (g >= C::QKS && !mbar_wait_warp(bar(QK_EMPTY + s), (g / C::QKS - 1) & 1, status)) break;
#pragma unroll 1
        for (int tile = 0; tile < TILES; ++tile) {
          const uint32_t at = tile_at(s, tile);
          load_half(r1, tile, 1);
          put_half(r0, at, 0);
          if (tile + 1 == TILES) more = it.next(a);
          if (more) load_half(r0, tile + 1 == TILES ? 0 : tile + 1, 0);
          put_half(r1, at, 1);
        }
        fence_proxy_async_smem();
        mbar_arrive(bar(QK_FULL + s));
      }
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------ MMA issue
    if (elect_one()) {
      int total = 0;
      for (int u = blockIdx.x; u < a.n_units; u += gridDim.x) total += mix_unit<DK>(a, u).chunks;
      constexpr uint32_t idS = make_idesc(128, 128, 1, false, false), idV = make_idesc(128, 64, 1, false, true),
                         idKV = make_idesc(128, 64, 1, true, true);
      auto wait = [&](int i, int phase) { return mbar_wait(bar(i), phase & 1, status); };
      auto issue_S = [&](int g) {
        const int s = g % C::QKS;
        if (!wait(QK_FULL + s, g / C::QKS)) return false;
        fence_proxy_async_smem();  // bf16: the copies' writes, before the tensor core reads them
        tc_fence_after();
#pragma unroll 1
        for (int term = 0; term < NT; ++term) {
          const uint64_t qd = make_sdesc(sQ(s) + (term == 2 ? KT * kTile : 0), 16, 1024);
          const uint64_t kd = make_sdesc(sK(s) + (term == 1 ? KT * kTile : 0), 16, 1024);
#pragma unroll
          for (int k = 0; k < DK / 16; ++k) {
            const uint32_t off = ((k / 4) * kTile + (k % 4) * 32) >> 4;
            umma_f16_ss(tmem + T_S + (g & 1) * 128, qd + off, kd + off, idS, (term > 0 || k > 0) ? 1u : 0u);
          }
        }
        umma_commit(bar(S_FULL + (g & 1)));
        return true;
      };
      bool ok = true;
      for (int g = 0; ok && g < total; ++g) {
        const int s = g % C::QKS, vs = g % C::VS, b = g & 1;
        if (STATES) ok = wait(QK_FULL + s, g / C::QKS);
        else if (g == 0) ok = issue_S(0);
        // K^T V' (DK = 64: both halves of the 128 rows are the same 64 rows of the
        // state, so every warp of the state finds its columns in its own lanes)
        ok = ok && wait(V_FULL + vs, g / C::VS) && (g < 2 || wait(KV_FREE + b, (g >> 1) - 1));
        if (!ok) break;
        if (STATES) fence_proxy_async_smem();
        tc_fence_after();
        constexpr int KV_TERMS = NT == 3 ? 3 : 2;
#pragma unroll 1
        for (int term = 0; term < KV_TERMS; ++term) {
          const uint64_t kd = make_sdesc(sK(s) + (term == 2 ? KT * kTile : 0), DK == 64 ? 0 : kTile, 1024);
          const uint64_t vd = make_sdesc(sV(vs) + (NP + (term == 1 ? 1 : 0)) * kTile, kTile, 1024);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ss(tmem + T_KV + b * 64, kd + (k * 2048 >> 4), vd + (k * 2048 >> 4), idKV,
                        (term > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(bar(KV_FULL + b));
        if (STATES) {
          umma_commit(bar(QK_EMPTY + s));
          umma_commit(bar(V_EMPTY + vs));
          continue;
        }
        if (g + 1 < total && !(ok = issue_S(g + 1))) break;
        // Q S from the state entering this chunk
        const int sb = g % C::STB;
        ok = wait(ST_FULL + sb, g / C::STB) && (g < 1 || wait(O_FREE, g - 1));
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int term = 0; term < KV_TERMS; ++term) {
          const uint64_t qd = make_sdesc(sQ(s) + (term == 2 ? KT * kTile : 0), 16, 1024);
          const uint64_t sd = make_sdesc(sS(sb) + (term == 1 ? C::ST_PLANE : 0), kTile, 1024);
#pragma unroll
          for (int k = 0; k < DK / 16; ++k)
            umma_f16_ss(tmem + T_QS, qd + (((k / 4) * kTile + (k % 4) * 32) >> 4), sd + (k * 2048 >> 4), idV,
                        (term > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(bar(ST_EMPTY + sb));
        umma_commit(bar(QK_EMPTY + s));
        // P V
        if (!(ok = wait(P_FULL + b, g >> 1))) break;
        tc_fence_after();
#pragma unroll 1
        for (int term = 0; term < NT; ++term) {
          const uint64_t vd = make_sdesc(sV(vs) + (term == 1 ? kTile : 0), kTile, 1024);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ts(tmem + T_PV, tmem + T_S + b * 128 + (k / 2) * 32 + (term == 2 ? 16 : 0) + (k % 2) * 8,
                        vd + (k * 2048 >> 4), idV,
                        (term > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(bar(V_EMPTY + vs));
        umma_commit(bar(O_FULL));
      }
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------ P, then the previous chunk's O
    if (!STATES) {
      const int i = threadIdx.x, lane = lane_id();
      float* tab = wtab + 64 * warp;  // tab[j] = l^(31 - j), this warp's own; past 31 not used
      int g = 0;
      bool ok = true;
      // the chunk whose output is due
      T* o_base = nullptr;     // its first row, this head and column half
      long long o_step = 0;    // values from one row to the next
      int o_valid = 0;
      float o_scale = 0.f;     // of Q S
      bool o_add = false;
      auto write_out = [&]() {
        if (!mbar_wait_warp(bar(O_FULL), (g - 1) & 1, status)) return false;
        tc_fence_after();
        constexpr int COLS = 64 / static_cast<int>(sizeof(T));  // columns of 64 bytes
        const int cols = a.D < 64 ? a.D : 64;
#pragma unroll 1
        for (int c0 = 0; c0 < cols; c0 += COLS) {
          uint4 v[4];
#pragma unroll
          for (int c = 0; c < COLS; c += 16) {
            uint32_t o1[16], o2[16];
            tmem_ld16x2_sync(tmem + T_QS + c0 + c + lane_base, tmem + T_PV + c0 + c + lane_base, o1, o2);
            float f[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              f[e] = fmaf(o_scale, __uint_as_float(o1[e]), a.scale * __uint_as_float(o2[e]));
            if (o_add && i < o_valid) add16(o_base + i * o_step + c0 + c, f);
            if constexpr (sizeof(T) == 2) {
              v[c / 8] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                                    pack_bf16x2(f[6], f[7]));
              v[c / 8 + 1] = make_uint4(pack_bf16x2(f[8], f[9]), pack_bf16x2(f[10], f[11]),
                                        pack_bf16x2(f[12], f[13]), pack_bf16x2(f[14], f[15]));
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                v[e] = make_uint4(__float_as_uint(f[4 * e]), __float_as_uint(f[4 * e + 1]),
                                  __float_as_uint(f[4 * e + 2]), __float_as_uint(f[4 * e + 3]));
            }
          }
          if (c0 + COLS >= cols) {
            tc_fence_before();
            warp_arrive(bar(O_FREE));
          }
          transpose4(v);
          const int r0 = 32 * warp + (lane & ~3);
          T* dst = o_base + r0 * o_step + c0 + (lane & 3) * (16 / static_cast<int>(sizeof(T)));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (r0 + k < o_valid) *reinterpret_cast<uint4*>(dst + k * o_step) = v[k];
        }
        return true;
      };
      for (int u = blockIdx.x; ok && u < a.n_units; u += gridDim.x) {
        const MixUnit x = mix_unit<DK>(a, u);
        if (x.chunks == 0) continue;
        const MixOne& one = a.one[x.dir];
        const float l2 = log2_decay(a.log_decay, x.h);
        __syncwarp();
        tab[lane] = exp2f(l2 * static_cast<float>(31 - lane));
        tab[32 + lane] = 0.f;
        __syncwarp();
        const float l32 = exp2f(l2 * 32.f), l_first = exp2f(l2 * static_cast<float>(lane + 1));
        for (int c = 0; c < x.chunks; ++c) {
          if (!(ok = mbar_wait_warp(bar(S_FULL + (g & 1)), (g >> 1) & 1, status))) break;
          tc_fence_after();
          const uint32_t ts = tmem + T_S + (g & 1) * 128 + lane_base;
          // P of 32 columns goes over their scores: hi in the first 16 columns, lo (NT = 3)
          // in the next
          auto put = [&](int cb, const float (&p)[32]) {
            uint32_t h[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) h[j] = pack_bf16x2(p[2 * j], p[2 * j + 1]);
            tmem_st16(ts + cb * 32, h);
            if (NT == 3) {
              uint32_t l[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) l[j] = lo_pair(p[2 * j], p[2 * j + 1], h[j]);
              tmem_st16(ts + cb * 32 + 16, l);
            }
          };
          uint32_t r[32];
          float p[32];
          // on the diagonal: column j of row `lane` has l^(lane - j) = tab[31 - lane + j]
          tmem_ld32_sync(ts + warp * 32, r);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float w = tab[31 - lane + j];
            p[j] = j <= lane ? __uint_as_float(r[j]) * w : 0.f;
          }
          put(warp, p);
          // left of it, nearest first: l^(i - j) = l^(i - 32 cb - 31) l^(31 - j), no negative exponent
          float rf = l_first;
#pragma unroll 1
          for (int cb = warp - 1; cb >= 0; --cb) {
            tmem_ld32_sync(ts + cb * 32, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 f = reinterpret_cast<const float4*>(tab)[j];
              p[4 * j] = __uint_as_float(r[4 * j]) * (rf * f.x);
              p[4 * j + 1] = __uint_as_float(r[4 * j + 1]) * (rf * f.y);
              p[4 * j + 2] = __uint_as_float(r[4 * j + 2]) * (rf * f.z);
              p[4 * j + 3] = __uint_as_float(r[4 * j + 3]) * (rf * f.w);
            }
            put(cb, p);
            rf *= l32;
          }
          // right of it: zero
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = 0;
#pragma unroll 1
          for (int cb = warp + 1; cb < 4; ++cb) {
            tmem_st16(ts + cb * 32, r);
            if (NT == 3) tmem_st16(ts + cb * 32 + 16, r);
          }
          tmem_st_wait();
          tc_fence_before();
          warp_arrive(bar(P_FULL + (g & 1)));
          if (g > 0 && !(ok = write_out())) break;
          const int pos = x.p0 + c * 128, left = x.count - c * 128;
          const long long tok = static_cast<long long>(x.b) * a.L + (one.dir.reverse ? x.n - 1 - pos : pos);
          o_step = static_cast<long long>(a.H) * a.D * (one.dir.reverse ? -1 : 1);
          o_base = static_cast<T*>(one.o) + (tok * a.H + x.h) * a.D + x.half * 64;
          o_valid = left < 128 ? left : 128;
          o_add = one.dir.accumulate;
          o_scale = a.scale * exp2f(l2 * static_cast<float>(i + 1 - (pos == 0 ? one.dir.lead : 0)));
          ++g;
        }
      }
      if (ok && g > 0) write_out();
    }
  } else {
    // ------------------------------------------------------------ state
    const int r = threadIdx.x - 128;
    constexpr int NC = C::NC;
    const int row = DK == 64 ? (r & 63) : r, col0 = DK == 64 ? (r >> 6) * 32 : 0;
    int g = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < a.n_units; u += gridDim.x) {
      const MixUnit x = mix_unit<DK>(a, u);
      const MixOne& one = a.one[x.dir];
      const float l2 = log2_decay(a.log_decay, x.h);
      const bool in_state = row < a.D && x.half * 64 + col0 < a.D;  // head dim 32: a quarter of the tile
      const size_t st0 = (static_cast<size_t>(x.b) * a.H + x.h) * a.D * a.D;
      // element (row, col) of the caller's state
      auto state_at = [&](int c) {
        const int e = x.half * 64 + col0 + c;
        return st0 + (one.dir.transposed ? static_cast<size_t>(e) * a.D + row : static_cast<size_t>(row) * a.D + e);
      };
      float S[NC];
      if (a.n_seg == 1 || (STATES && x.seg == 0)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) S[c] = one.s_in && in_state ? one.dir.in_mult * one.s_in[state_at(c)] : 0.f;
      }
      if (STATES) {
        if (x.seg == 0) {
          float4* dst = reinterpret_cast<float4*>(seg_slot<DK>(a, x, a.n_seg - 1));
#pragma unroll
          for (int c = 0; c < NC / 4; ++c) dst[c * 128 + r] = make_float4(S[4 * c], S[4 * c + 1], S[4 * c + 2], S[4 * c + 3]);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) S[c] = 0.f;
      } else if (a.n_seg > 1) {
        // the state entering this segment from the segments before it
        auto add = [&](int slot, float w, bool first) {
          const float4* src = reinterpret_cast<const float4*>(seg_slot<DK>(a, x, slot));
#pragma unroll
          for (int c = 0; c < NC / 4; ++c) {
            const float4 f = src[c * 128 + r];
            S[4 * c] = fmaf(w, f.x, first ? 0.f : S[4 * c]);
            S[4 * c + 1] = fmaf(w, f.y, first ? 0.f : S[4 * c + 1]);
            S[4 * c + 2] = fmaf(w, f.z, first ? 0.f : S[4 * c + 2]);
            S[4 * c + 3] = fmaf(w, f.w, first ? 0.f : S[4 * c + 3]);
          }
        };
        add(a.n_seg - 1, x.seg == 0 ? 1.f : exp2f(l2 * static_cast<float>(x.p0 - one.dir.lead)), true);
        for (int f = 0; f < x.seg && x.count > 0; ++f)
          add(f, exp2f(l2 * static_cast<float>(x.p0 - (f + 1) * a.seg_tokens)), false);
      }
      // the state's bf16 parts for chunk gg's Q S
      auto put_state = [&](int gg) {
        const int sb = gg % C::STB;
        if (gg >= C::STB && !mbar_wait_warp(bar(ST_EMPTY + sb), (gg / C::STB - 1) & 1, status)) return false;
#pragma unroll
        for (int c = 0; c < NC / 8; ++c) {
          uint32_t h[4], l[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            h[j] = pack_bf16x2(S[8 * c + 2 * j], S[8 * c + 2 * j + 1]);
            l[j] = lo_pair(S[8 * c + 2 * j], S[8 * c + 2 * j + 1], h[j]);
          }
          const uint32_t at = sS(sb) + sw128_offset(row, col0 * 2 + c * 16);
          st_shared_v4(at, h[0], h[1], h[2], h[3]);
          st_shared_v4(at + C::ST_PLANE, l[0], l[1], l[2], l[3]);
        }
        fence_proxy_async_smem();
        warp_arrive(bar(ST_FULL + sb));
        return true;
      };
      if (!STATES && x.chunks > 0 && !(ok = put_state(g))) break;
      for (int c = 0; c < x.chunks; ++c, ++g) {
        const int left = x.count - c * 128, valid = left < 128 ? left : 128;
        // the carried state enters the very first token without a decay (lead)
        const int lead = c == 0 && x.seg == 0 && !STATES ? one.dir.lead : 0;
        if (!(ok = mbar_wait_warp(bar(KV_FULL + (g & 1)), (g >> 1) & 1, status))) break;
        tc_fence_after();
        const float dec = exp2f(l2 * static_cast<float>(valid - lead));
#pragma unroll
        for (int j = 0; j < NC / 16; ++j) {
          uint32_t v[16];
          tmem_ld16(tmem + T_KV + (g & 1) * 64 + col0 + j * 16 + lane_base, v);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) S[16 * j + e] = fmaf(dec, S[16 * j + e], __uint_as_float(v[e]));
        }
        tc_fence_before();
        warp_arrive(bar(KV_FREE + (g & 1)));
        if (STATES) continue;
        if (c + 1 < x.chunks && !(ok = put_state(g + 1))) break;
      }
      if (!ok) break;
      if (STATES) {
        if (x.seg < a.n_seg - 1) {
          float4* dst = reinterpret_cast<float4*>(seg_slot<DK>(a, x, x.seg));
#pragma unroll
          for (int c = 0; c < NC / 4; ++c) dst[c * 128 + r] = make_float4(S[4 * c], S[4 * c + 1], S[4 * c + 2], S[4 * c + 3]);
        }
        continue;
      }
      // after the last token's segment (the first one of an empty sequence)
      if (one.s_out && in_state && x.seg == (x.n > 0 ? (x.n - 1) / a.seg_tokens : 0)) {
        const float w = one.dir.out_mult * (one.dir.lead && x.n > 0 ? exp2f(l2) : 1.f);
#pragma unroll
        for (int c = 0; c < NC; ++c) one.s_out[state_at(c)] = w * S[c];
      }
      if (!one.dir.accumulate) {  // zeros past the sequence
        const int p1 = a.L - x.p0 < a.seg_tokens ? a.L : x.p0 + a.seg_tokens;
        const int pz = x.n > x.p0 ? x.n : x.p0;
        const int vecs = (a.D < 64 ? a.D : 64) * static_cast<int>(sizeof(T)) / 16;
        const long long zeros = static_cast<long long>(p1 - pz) * vecs;
        for (long long i = r; i < zeros; i += 128) {
          const size_t tok = static_cast<size_t>(x.b) * a.L + pz + i / vecs;
          reinterpret_cast<uint4*>(static_cast<T*>(one.o) + (tok * a.H + x.h) * a.D + x.half * 64)[i % vecs] =
              make_uint4(0, 0, 0, 0);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
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

// Segments of one sequence. A sequence's chunks follow one another, so with few
// (sequence, head) pairs most of the GPU would idle: the sequence is cut, the
// segments' own states are computed first (k and v are read a second time) and
// each segment starts from their sum.
struct MixPlan {
  int n_seg, seg_tokens, units;
};
MixPlan mix_plan(const AttnShape& sh, int n_dir) {
  MixPlan p;
  const int chunks = (sh.L + 127) / 128;
  const long long pairs = static_cast<long long>(sh.B) * sh.H * n_dir * (sh.D == 128 ? 2 : 1);
  long long seg = device_sm_count() / pairs;
  if (seg > chunks / 4) seg = chunks / 4;
  if (seg < 1) seg = 1;
  const int seg_chunks = static_cast<int>((chunks + seg - 1) / seg);
  p.n_seg = (chunks + seg_chunks - 1) / seg_chunks;
  p.seg_tokens = seg_chunks * 128;
  p.units = static_cast<int>(pairs) * p.n_seg;
  return p;
}

template <typename T, int DK, int NT>
int mix_launch(MixArgs a, uint32_t* status, cudaStream_t s) {
  using C = MixCfg<DK, NT>;
  static std::atomic<uint64_t> attr_s{0}, attr{0};
  const int sms = device_sm_count();
  if (a.n_seg > 1) {
    if (!ensure_smem_attr(mix_kernel<T, DK, NT, true>, C::SMEM, attr_s)) return PA_ERR_LAUNCH;
    MixArgs f = a;
    f.n_units = a.n_units / a.n_seg * (a.n_seg - 1);
    mix_kernel<T, DK, NT, true><<<f.n_units < sms ? f.n_units : sms, kMixThreads, C::SMEM, s>>>(f, status);
    if (cudaGetLastError() != cudaSuccess) return PA_ERR_LAUNCH;
  }
  if (!ensure_smem_attr(mix_kernel<T, DK, NT, false>, C::SMEM, attr)) return PA_ERR_LAUNCH;
  mix_kernel<T, DK, NT, false><<<a.n_units < sms ? a.n_units : sms, kMixThreads, C::SMEM, s>>>(a, status);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

int mix(const AttnShape& sh, bool f32, MixArgs a, const float* log_decay, const int32_t* lens, void* ws,
        uint32_t* status, cudaStream_t s) {
  const MixPlan p = mix_plan(sh, a.n_dir);
  a.log_decay = log_decay;
  a.lens = lens;
  a.ws = static_cast<float*>(ws);
  a.B = sh.B;
  a.L = sh.L;
  a.H = sh.H;
  a.D = sh.D;
  a.n_seg = p.n_seg;
  a.seg_tokens = p.seg_tokens;
  a.n_units = p.units;
  a.scale = sh.scale;
  if (!f32)
    return sh.D == 64 ? mix_launch<__nv_bfloat16, 64, 1>(a, status, s)
                      : mix_launch<__nv_bfloat16, 128, 1>(a, status, s);
  return f32_math() == PA_F32_MATH_BF16 ? mix_launch<float, 64, 1>(a, status, s)
                                        : mix_launch<float, 64, 3>(a, status, s);
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

size_t linear_attn_workspace_bytes(const AttnShape& sh, bool, bool backward) {
  const MixPlan p = mix_plan(sh, backward ? 3 : 1);
  return p.n_seg == 1 ? 0 : static_cast<size_t>(p.units) * (sh.D == 128 ? 128 : 64) * 64 * sizeof(float);
}

int launch_linear_attn_fwd(const AttnShape& sh, bool f32, const void* q, const void* k, const void* v,
                           const float* log_decay, const int32_t* lens, const float* s_in, void* o,
                           float* s_out, void* ws, uint32_t* status, cudaStream_t s) {
  MixArgs a{};
  a.n_dir = 1;
  a.one[0] = MixOne{q, k, v, o, s_in, s_out, MixDir{}};
  return mix(sh, f32, a, log_decay, lens, ws, status, s);
}

int launch_linear_attn_bwd(const AttnShape& sh, bool f32, const void* q, const void* k, const void* v,
                           const void* dO, const float* log_decay, const int32_t* lens,
                           const float* s_in, const float* ds_out, void* dq, void* dk, void* dv,
                           float* ds_in, bool accumulate, void* ws, uint32_t* status, cudaStream_t s) {
  // The backward recurrence keeps U / scale, so one product with scale gives
  // dk and dv: the gradient of the state enters divided by it and leaves
  // multiplied.
  MixDir d;
  d.accumulate = accumulate;
  d.transposed = true;
  MixDir dk_dir = d;
  dk_dir.reverse = true;
  dk_dir.lead = 1;
  dk_dir.in_mult = 1.f / sh.scale;
  dk_dir.out_mult = sh.scale;
  MixDir dv_dir = dk_dir;
  dv_dir.transposed = false;
  MixArgs a{};
  a.n_dir = 3;
  a.one[0] = MixOne{k, q, dO, dv, ds_out, ds_in, dv_dir};
  a.one[1] = MixOne{v, dO, q, dk, ds_out, nullptr, dk_dir};
  a.one[2] = MixOne{dO, v, k, dq, s_in, nullptr, d};
  return mix(sh, f32, a, log_decay, lens, ws, status, s);
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
