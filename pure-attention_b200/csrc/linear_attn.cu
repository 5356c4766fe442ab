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
// A sequence in chunks of 128 tokens. With S the state entering a chunk of n
// valid tokens (rows i, j of the chunk; l the decay), forward in time:
//   O   = scale (P V + diag(l^(i+1)) Q S),   P = (Q K^T) o l^(i-j) for j <= i, else 0
//   S'  = l^n S + K^T V',                     V' = diag(l^(n-1-j)) V
// and backward in time, the chunks from the last on: P with l^(j-i) for j >= i,
// diag(l^(n-i)), V' = diag(l^j) V. All four products run on the tensor cores;
// every power of l has a whole, non-negative exponent, so nothing overflows where
// l is small.
//
// One CTA per SM walks units (sequence, head, 64 columns of V, segment of the
// sequence); a unit's chunks follow one another through the state, and the
// rings below run on across units.
//   warps 0-7   P: load Q K^T from TMEM, times l^|i-j|, bf16 back to TMEM; then the
//               previous chunk's O out (two warps share 32 rows: some blocks of P
//               and 32 columns of O each)
//   warps 8-11  the state in fp32 registers (thread = row of the state), its bf16
//               parts to shared memory for Q S
//               (fp32: and the splitting of k)
//   warps 12-15 V' from V (fp32: and the splitting of v)
//   warps 16-19 tcgen05.mma issue (one thread), TMA loads (one thread), the splitting of
//               fp32 q (two warps)
// Q and K feed two products each as they lie: K as the K-major B of Q K^T and as the
// MN-major A of K^T V'.
//
// Roundings: fp32 sums and state throughout. V' is two bf16 parts (off by 2^-17), so a carried
// state gains an error of 2^-17 of each token's part, not 2^-9 (one part would save a quarter of
// the products, but a state is read by every later token). As operands of the output's two products,
// P and the state entering the chunk are one bf16 each (2^-9), as P is in the softmax kernels: the
// output is rounded to bf16 itself. NT = 3 (fp32 operands): every operand is a hi/lo pair and every
// product hi*hi + hi*lo + lo*hi (2^-16 in all).
//
// What bounds it. 8 x 4096 tokens of 16 heads of 64 in bf16 (268 MB: 41 us at the copy rate) take 58
// us alone, 4.6 TB/s, 64-65 us back to back under the power limit. A chunk takes 2900 clocks, and by
// count 270 KB of it pass the 128 bytes a clock of the SM's shared memory, 2200 clocks: tiles of
// q, k and v land there, V' is made there in two parts, and the four products read their operands
// there (but P, from TMEM); 128 of 148 SMs are busy. At head dim 128 a unit is half of V's columns,
// and each half forms P anew: a state of 128 x 128 would need 128 registers of each of 128 threads.
// Chunks of fp32 move 700 KB (three products, and tiles split into parts in place), 5400 of 6000
// clocks, 3.7 us: 8 x 1024 tokens of 8 heads of 64 in one launch are 8 chunks a block and 5.5 us to
// start, 35 us, and cut in two 34. Heads of 32 in fp32 take the instance of 64 columns, half of each
// tile zeros: 33 us where heads of 64 take 34. Short calls wait for their own code: the first chunk of
// a cold launch takes 5 us.
//
// TMEM columns: Q K^T and P 2 x 128 (P of 32 tokens over their 32 scores: hi in the
// first 16 columns, lo in the others), Q S 64, P V 64, K^T [V' hi, V' lo] 128.
constexpr int kMixThreads = 20 * 32;
constexpr int kTile = 128 * 128;  // bytes of 128 rows x 64 bf16

template <typename T, int DK, int NT>
struct MixCfg {
  static constexpr int NP = NT == 3 ? 2 : 1;       // planes (hi, lo) of q, k, v
  static constexpr int KT = DK / 64;               // 64-column tiles of q and k
  // bytes of q (or k) of a stage; fp32 tiles land there whole before they are split
  static constexpr int OPER = (sizeof(T) == 4 ? 2 : 1) * KT * kTile;
  static constexpr int V_STAGE = NP * kTile;       // v
  static constexpr int VP_BYTES = 2 * kTile;       // V' hi and lo
  static constexpr int ST_PLANE = DK * 128;        // [DK, 64] bf16
  static constexpr bool SMALL = sizeof(T) == 2 && DK == 64;
  static constexpr int QKS = SMALL ? 3 : 2, VS = SMALL ? 4 : (sizeof(T) == 2 ? 2 : 1);
  // V', state planes, and 2 KB a warp through which the output goes out
  static constexpr int SMEM = QKS * 2 * OPER + VS * V_STAGE + VP_BYTES + NP * ST_PLANE + kTile + 1024;
  static constexpr int NC = DK == 64 ? 32 : 64;    // state columns of a thread
};
static_assert(MixCfg<__nv_bfloat16, 64, 1>::SMEM <= 225 * 1024 && MixCfg<__nv_bfloat16, 128, 1>::SMEM <= 225 * 1024 &&
              MixCfg<float, 64, 3>::SMEM <= 225 * 1024, "shared memory of one CTA");

struct MixOne {  // one direction of the recurrence
  const void *q, *k, *v;
  void* o;
  const float* s_in;
  float* s_out;
  MixDir dir;
  int mq, mk, mv;  // bf16: the tensor maps of q, k, v
  int mo;          // and of o
};
// Division by a number that the host knows: n / d = (high word of n mul + n) >> shift for
// n < 2^31, with shift = ceil(log2 d) and mul = floor(2^32 (2^shift - d) / d) + 1.
struct Divisor {
  uint32_t d, mul, shift;
  static Divisor of(int d) {
    Divisor x{static_cast<uint32_t>(d), 0, 0};
    while ((1ull << x.shift) < x.d) ++x.shift;
    x.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << x.shift) - x.d)) / x.d + 1);
    return x;
  }
  // n / d, and n becomes the remainder
  __device__ __forceinline__ int split(int& n) const {
    const uint32_t u = static_cast<uint32_t>(n), q = (__umulhi(u, mul) + u) >> shift;
    n = static_cast<int>(u - q * d);
    return static_cast<int>(q);
  }
};

struct MixArgs {
  MixOne one[3];
  int n_dir;
  Divisor by_dir, by_H, by_B;
  const float* log_decay;
  const int32_t* lens;
  float* ws;  // segment states, see seg_slot
  int B, L, H, D;
  int n_seg, seg_tokens, n_units;
  int fine, state_tokens, n_slots;  // segment states: `fine` pieces a segment, their tokens; see seg_slot
  float scale;
};
struct MixMaps {
  CUtensorMap m[4];  // inputs: 64 columns x 128 tokens
  CUtensorMap o[3];  // outputs: 64 bytes of columns x 32 tokens
};

struct MixUnit {
  int dir, b, h, half, seg;
  int n;          // valid tokens of the sequence
  int p0, count;  // first token and tokens of this segment
  int chunks;
  bool rev;
  // Chunk c in the order of the recurrence: its first token, its valid tokens.
  __device__ __forceinline__ int index(int c) const { return rev ? chunks - 1 - c : c; }
  __device__ __forceinline__ int token(int c) const { return p0 + index(c) * 128; }
  __device__ __forceinline__ int valid(int c) const {
    const int left = count - index(c) * 128;
    return left < 128 ? left : 128;
  }
  // the chunk that the carried state of the sequence enters
  __device__ __forceinline__ bool starts(int c) const {
    return rev ? token(c) + 128 >= n : token(c) == 0;
  }
};

// unit -> (segment, sequence, head, direction, column half), halves and
// directions of one head next to one another: they read the same rows, from L2.
// Segment states are wanted of all but the segment that comes last in time order; there
// x.seg counts pieces.
template <int DK, bool STATES>
__device__ __forceinline__ MixUnit mix_unit(const MixArgs& a, int u) {
  MixUnit x;
  constexpr int halves = DK / 64;
  x.half = u % halves;
  u /= halves;
  x.dir = u;
  x.h = a.by_dir.split(x.dir);
  x.b = a.by_H.split(x.h);
  x.seg = a.by_B.split(x.b);
  x.rev = a.one[x.dir].dir.reverse;
  if (STATES && x.rev) x.seg += a.fine;
  x.n = valid_tokens(a.lens, x.b, a.L);
  const int tokens = STATES ? a.state_tokens : a.seg_tokens;
  x.p0 = x.seg * tokens;
  const int left = x.n - x.p0;
  x.count = left < 0 ? 0 : (left < tokens ? left : tokens);
  x.chunks = (x.count + 127) >> 7;
  return x;
}

// Workspace of a sequence cut in segments: per (sequence, head, direction, half)
// n_slots = (n_seg - 1) * fine + 1 slots of [DK, 64] fp32. The last holds a copy of the
// carried state (state_out may overwrite state_in while other segments still need
// it), the others the states of single pieces of segments (from zero).
template <int DK>
__device__ __forceinline__ float* seg_slot(const MixArgs& a, const MixUnit& x, int slot) {
  const size_t w = ((static_cast<size_t>(x.b) * a.H + x.h) * a.n_dir + x.dir) * (DK / 64) + x.half;
  return a.ws + (w * a.n_slots + slot) * (DK * 64);
}

// The chunks of this CTA in order.
template <int DK, bool STATES>
struct ChunkIter {
  MixUnit x;
  int u, chunk, g;  // g: chunks of this CTA so far
  int n_units;
  __device__ __forceinline__ bool first(const MixArgs& a, int units) {
    n_units = units;
    u = blockIdx.x;
    chunk = g = 0;
    return settle(a);
  }
  __device__ __forceinline__ bool settle(const MixArgs& a) {  // to a unit that has chunks
    for (; u < n_units; u += gridDim.x) {
      x = mix_unit<DK, STATES>(a, u);
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
  __device__ __forceinline__ int valid() const { return x.valid(chunk); }
};

// Pairs of fp32 values.
__device__ __forceinline__ float2 pair_of(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ uint32_t hi_pair(float2 v) { return pack_bf16x2(v.x, v.y); }
__device__ __forceinline__ uint32_t lo_pair(float2 v, uint32_t hi) {
  const float2 d = __fadd2_rn(v, make_float2(-__uint_as_float(hi << 16), -__uint_as_float(hi & 0xffff0000u)));
  return pack_bf16x2(d.x, d.y);
}
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
// Four fp32 values as bf16 hi and, where `lo` is not 0, lo.
__device__ __forceinline__ void put4(uint32_t hi, uint32_t lo, uint32_t off, float2 a, float2 b) {
  const uint32_t h0 = hi_pair(a), h1 = hi_pair(b);
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(hi + off), "r"(h0), "r"(h1) : "memory");
  if (lo)
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(lo + off), "r"(lo_pair(a, h0)), "r"(lo_pair(b, h1))
                 : "memory");
}

// An fp32 tile (128 rows x 64 values) as TMA leaves it: columns 0-31 as rows of 128 bytes
// where the hi plane will be, 32-63 where the lo plane will be. Split in place it stays
// within its rows: 16 lanes hold a row between reading and writing it. Thread t of N
// has the 16-byte vectors t % 16 of rows t / 16 + i * N / 16.
template <int N>
struct Split {
  static constexpr int ROWS = N / 16, VECS = 128 / ROWS;
  uint32_t at;  // of the tile
  int row0, c;
  __device__ __forceinline__ Split(uint32_t tile, int t) : at(tile), row0(t / 16), c(t % 16) {}
  __device__ __forceinline__ int row(int i) const { return row0 + i * ROWS; }
  // zero past the sequence, whatever is there
  __device__ __forceinline__ float4 load(int i, int valid) const {
    const uint4 v = ld_shared_v4(at + (c >> 3) * kTile + row(i) * 128 + (c & 7) * 16);
    return row(i) < valid ? make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z),
                                        __uint_as_float(v.w))
                          : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  template <int NP>
  __device__ __forceinline__ void store(uint32_t to, int i, float4 v) const {
    put4(to, NP == 2 ? to + kTile : 0, sw128_offset(row(i), c * 8), make_float2(v.x, v.y), make_float2(v.z, v.w));
  }
  // vectors i0 .. i0 + 7 in place
  template <int NP>
  __device__ __forceinline__ void eight(int i0, int valid) const {
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load(i0 + i, valid);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) store<NP>(at, i0 + i, v[i]);
  }
};

// 32 values of an output row += f.
__device__ __forceinline__ void add_row(float* dst, const float2 (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float4 o = reinterpret_cast<const float4*>(dst)[i];
    o.x += f[2 * i].x;
    o.y += f[2 * i].y;
    o.z += f[2 * i + 1].x;
    o.w += f[2 * i + 1].y;
    reinterpret_cast<float4*>(dst)[i] = o;
  }
}
__device__ __forceinline__ void add_row(__nv_bfloat16* dst, const float2 (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 o = reinterpret_cast<const uint4*>(dst)[i];
    const uint32_t w[4] = {o.x, o.y, o.z, o.w};
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = hi_pair(__fadd2_rn(f[4 * i + j], pair_of(w[j] << 16, w[j] & 0xffff0000u)));
    reinterpret_cast<uint4*>(dst)[i] = make_uint4(y[0], y[1], y[2], y[3]);
  }
}

__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(bar);
}

// A shared-memory descriptor and the one `bytes` further on (16-byte units in the low word).
struct Desc {
  uint64_t d;
  __device__ __forceinline__ Desc at(uint32_t bytes) const {
    return Desc{(d & 0xffffffff00000000ull) | (static_cast<uint32_t>(d) + (bytes >> 4))};
  }
};

// STATES: only the segments' own states, into the workspace.
template <typename T, int DK, int NT, bool STATES>
__global__ void __launch_bounds__(kMixThreads, 1)
    mix_kernel(const __grid_constant__ MixArgs a, const __grid_constant__ MixMaps maps, uint32_t* status) {
  using C = MixCfg<T, DK, NT>;
  constexpr int NP = C::NP, KT = C::KT;
  constexpr bool BF16 = sizeof(T) == 2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[35];  // N_BARS
  __shared__ __align__(16) float wtab[4 * 64 + 4 * 32];  // powers of the decay, a table for each P warp
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const uint32_t sm0 = smem_u32(align1024(smem_raw));
  const uint32_t sv0 = sm0 + C::QKS * 2 * C::OPER, sVp = sv0 + C::VS * C::V_STAGE, ss0 = sVp + C::VP_BYTES;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  // ring slot s: K planes, then Q planes; V planes. V' hi, lo; the state's hi, lo (ss0); the stage
  auto sK = [&](int s) { return sm0 + s * 2 * C::OPER; };
  auto sQ = [&](int s) { return sm0 + s * 2 * C::OPER + C::OPER; };
  auto sV = [&](int s) { return sv0 + s * C::V_STAGE; };
  enum { QK_FULL = 0, QK_EMPTY = 3, V_FULL = 6, V_EMPTY = 10, S_FULL = 14, P_FULL = 16, VP_FULL = 18, VP_EMPTY = 20,
         KV_FULL = 22, KV_FREE = 24, ST_FULL = 26, ST_EMPTY, O_FULL, O_FREE, QK_RAW = 30, V_RAW = 32, MMA_DONE = 34, N_BARS };
  // Segment states: V' and K^T V' twice, in what Q and its scores do not use there.
  constexpr int VB = STATES ? 2 : 1;
  constexpr uint32_t VP_LO2 = C::OPER >= 2 * kTile ? kTile : 2 * C::OPER;  // hi to lo in the second V'
  auto vp_at = [&](int g) { return VB == 2 && (g & 1) ? sm0 + C::OPER : sVp; };
  auto vp_lo = [&](int g) { return VB == 2 && (g & 1) ? VP_LO2 : static_cast<uint32_t>(kTile); };
  auto kv_at = [&](int g) { return VB == 2 && (g & 1) ? 0u : 384u; };
  constexpr uint32_t T_S = 0, T_QS = 256, T_PV = 320;  // and kv_at

  // The launch that needs these states may set itself up on SMs that are free.
  if (STATES && threadIdx.x == 0) launch_dependents();
  const int warp = warp_id();
  // Role of a warp of the last warpgroup: 0 MMA issue, 1 loads, 2 and 3 splitting. The issuing warp slows the
  // other warps of its sub-partition (an MMA that waits for the queue holds up their TMEM
  // loads), so it sits with the 32 rows that have the fewest scores: the first forward in time,
  // the last backward.
  const int role = warp < 16 ? -1 : (warp - 16 + (a.n_dir == 1 ? 0 : 1)) & 3;
  // One thread loads, all tiles by TMA.
  const bool loads = role == 1 && lane_id() == 0;
  int n_qk = 0, n_v = 0;  // chunks whose tiles it has sent for
  auto load = [&](const ChunkIter<DK, STATES>& it) {
    const int g = it.g, s = g % C::QKS, vs = g % C::VS;
    const MixOne& one = a.one[it.x.dir];
    const int tok = it.x.token(it.chunk), h = it.x.h, b = it.x.b;
    const uint32_t qk = bar((BF16 ? QK_FULL : QK_RAW) + s);
    constexpr int COLS = 128 / static_cast<int>(sizeof(T));  // 128 bytes a row
    if (g >= C::QKS && !mbar_wait(bar(QK_EMPTY + s), (g / C::QKS - 1) & 1, status)) return false;
    mbar_arrive_expect_tx(qk, (STATES ? 1 : 2) * C::OPER);
#pragma unroll
    for (int tile = 0; tile < C::OPER / kTile; ++tile) {
      tma_load_4d(sK(s) + tile * kTile, &maps.m[one.mk], qk, tile * COLS, h, tok, b);
      if (!STATES) tma_load_4d(sQ(s) + tile * kTile, &maps.m[one.mq], qk, tile * COLS, h, tok, b);
    }
    ++n_qk;
    if (BF16) {
      if (g >= C::VS && !mbar_wait(bar(V_EMPTY + vs), (g / C::VS - 1) & 1, status)) return false;
      mbar_arrive_expect_tx(bar(V_FULL + vs), kTile);
      tma_load_4d(sV(vs), &maps.m[one.mv], bar(V_FULL + vs), it.x.half * 64, h, tok, b);
    } else {
      if (g >= VB && !mbar_wait(bar(VP_EMPTY + g % VB), (g / VB - 1) & 1, status)) return false;
      const uint32_t raw = bar(V_RAW + g % VB);
      mbar_arrive_expect_tx(raw, 2 * kTile);
      tma_load_4d(vp_at(g), &maps.m[one.mv], raw, 0, h, tok, b);
      tma_load_4d(vp_at(g) + vp_lo(g), &maps.m[one.mv], raw, COLS, h, tok, b);
    }
    ++n_v;
    return true;
  };
  ChunkIter<DK, STATES> load_it;
  bool load_more = false;
  if (loads) {  // the first chunk is on its way before the block has set itself up
    for (int i = 0; i < 3; ++i) {
      mbar_init(bar(QK_FULL + i), BF16 ? 1 : (STATES ? 2 : 6));  // fp32: the splitting warps
      mbar_init(bar(QK_EMPTY + i), 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(V_FULL + i), BF16 ? 1 : 4);
      mbar_init(bar(V_EMPTY + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(S_FULL + i), 1);
      mbar_init(bar(P_FULL + i), 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(QK_RAW + i), 1);
      mbar_init(bar(V_RAW + i), 1);
      mbar_init(bar(VP_FULL + i), 4);
      mbar_init(bar(VP_EMPTY + i), 1);
      mbar_init(bar(KV_FULL + i), 1);
      mbar_init(bar(KV_FREE + i), 4);
    }
    mbar_init(bar(ST_FULL), 4);
    mbar_init(bar(ST_EMPTY), 1);
    mbar_init(bar(O_FULL), 1);
    mbar_init(bar(O_FREE), 8);
    mbar_init(bar(MMA_DONE), 1);
    fence_mbar_init();
    load_more = load_it.first(a, a.n_units);
    if (load_more) {
      load(load_it);
      load_more = load_it.next(a);
    }
  } else if (role == 0) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  } else if (role == 3) {
    if (lane_id() == 0) abort_flag = aborted(status);
    if (lane_id() < 4) {
      const MixOne& one = a.one[mix_unit<DK, STATES>(a, blockIdx.x).dir];
      tma_prefetch_desc(lane_id() == 3 ? &maps.o[one.mo]
                                       : &maps.m[lane_id() == 0 ? one.mk : (lane_id() == 1 ? one.mq : one.mv)]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // an earlier kernel's failure: no work
  const int n_units = abort_flag ? 0 : a.n_units;
  const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;

  // Head dim 128: a state thread holds 64 values. 2 x 96 + 152 + 88 + 48 = 5 x 96 registers.
  constexpr bool MOVE_REGS = DK == 128 && !STATES;
  if (MOVE_REGS) {
    if (warp >= 16) regs_dec<48>();
    else if (warp >= 12) regs_dec<88>();
    else if (warp >= 8) regs_inc<152>();
  }

  if (warp < 8) {
    // ------------------------------------------------------------ P, then the previous chunk's O
    if (!STATES) {
      const int w4 = warp & 3, part = warp >> 2;  // 32 rows, and which of their two warps
      const int lane = lane_id(), i = 32 * w4 + lane;
      float* tab = wtab + (part == 0 ? 64 * w4 : 256 + 32 * w4);  // this warp's own
      int g = 0;
      bool ok = true;
      // the chunk whose output is due
      int o_dir = 0, o_col = 0, o_h = 0, o_tok = 0, o_b = 0, o_valid = 0;
      float o_scale = 0.f;   // of Q S
      auto write_out = [&]() {
        if (!mbar_wait_warp(bar(O_FULL), (g - 1) & 1, status)) return false;
        tc_fence_after();
        const float2 w2 = make_float2(o_scale, o_scale);
        uint32_t o1[32], o2[32];
        const uint32_t at = tmem + lane_base + 32 * part;
        tmem_ld32(at + T_QS, o1);
        tmem_ld32_sync(at + T_PV, o2);
        tc_fence_before();
        warp_arrive(bar(O_FREE));
        if (32 * part >= a.D) return true;  // head dim 32: no columns for part 1
        float2 f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e)
          f[e] = __ffma2_rn(w2, pair_of(o1[2 * e], o1[2 * e + 1]), pair_of(o2[2 * e], o2[2 * e + 1]));
        const bool add = a.one[o_dir].dir.accumulate;
        if (add && (sizeof(T) == 2 || o_valid < 128)) {
          // added in fp32 and rounded once, and rows past the end left alone: each lane its row
          if (i < o_valid)
            add_row(static_cast<T*>(a.one[o_dir].o) +
                        ((static_cast<size_t>(o_b) * a.L + o_tok + i) * a.H + o_h) * a.D + o_col,
                    f);
          return true;
        }
        if (i >= o_valid) {
#pragma unroll
          for (int e = 0; e < 16; ++e) f[e] = make_float2(0.f, 0.f);
        }
        // 32 rows of 64 bytes a store, 64-byte swizzled: a bf16 row's 32 columns, 16 of fp32
        const uint32_t stage = ss0 + NP * C::ST_PLANE + warp * 2048;
        constexpr int STORES = static_cast<int>(sizeof(T)) / 2;
#pragma unroll
        for (int half = 0; half < STORES; ++half) {
          if (lane == 0) bulk_wait_read<0>();  // this warp's store before
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t to = stage + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4);
            if constexpr (sizeof(T) == 2)
              st_shared_v4(to, hi_pair(f[4 * c]), hi_pair(f[4 * c + 1]), hi_pair(f[4 * c + 2]), hi_pair(f[4 * c + 3]));
            else
              st_shared_v4(to, __float_as_uint(f[8 * half + 2 * c].x), __float_as_uint(f[8 * half + 2 * c].y),
                           __float_as_uint(f[8 * half + 2 * c + 1].x), __float_as_uint(f[8 * half + 2 * c + 1].y));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && o_tok + 32 * w4 < a.L) {
            const CUtensorMap* map = &maps.o[a.one[o_dir].mo];
            if (add) tma_reduce_add_4d(map, stage, o_col + 16 * half, o_h, o_tok + 32 * w4, o_b);
            else tma_store_4d(map, stage, o_col + 16 * half, o_h, o_tok + 32 * w4, o_b);
            tma_store_commit();
          }
        }
        return true;
      };
      for (int u = blockIdx.x; ok && u < n_units; u += gridDim.x) {
        const MixUnit x = mix_unit<DK, STATES>(a, u);
        if (x.chunks == 0) continue;
        const MixOne& one = a.one[x.dir];
        const float l2 = log2_decay(a.log_decay, x.h);
        // Part 0: tab[e] with e = 31 - lane + j, forward l^(31-e) for e <= 31, backward l^(e-31) for
        // e >= 31. Part 1: l^(31-j), backward l^(j+1). All times scale.
        __syncwarp();
        const float near = a.scale * exp2f(l2 * static_cast<float>(x.rev ? lane + 1 : 31 - lane));
        if (part == 0) {
          tab[lane] = x.rev ? (lane == 31 ? a.scale : 0.f) : near;
          tab[32 + lane] = x.rev ? near : 0.f;
        } else {
          tab[lane] = near;
        }
        __syncwarp();
        const float* diag = tab + 31 - lane;
        // Part 0 takes the block on the diagonal (as dear as two others), part 1 those beside it, at
        // distance d = 1 .. nb: l^|i-j| = l^(32 (d - 1)) l_first tab, no negative exponent.
        const int nb = x.rev ? 3 - w4 : w4, dir = x.rev ? 1 : -1;
        const float l32 = exp2f(l2 * 32.f);
        const float l_first = exp2f(l2 * static_cast<float>(x.rev ? 31 - lane : lane + 1));
        for (int c = 0; c < x.chunks; ++c) {
          const int valid = x.valid(c);
          if (!(ok = mbar_wait_warp(bar(S_FULL + (g & 1)), (g >> 1) & 1, status))) break;
          tc_fence_after();
          const uint32_t ts = tmem + T_S + (g & 1) * 128 + lane_base;
          uint32_t r[32];
          float2 p[16];
          // P of 32 columns goes over their scores: hi in the first 16 columns, lo (NT = 3) in the next
          auto put = [&](int cb) {
            uint32_t h[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) h[j] = hi_pair(p[j]);
            tmem_st16(ts + cb * 32, h);
            if (NT == 3) {
              uint32_t l[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) l[j] = lo_pair(p[j], h[j]);
              tmem_st16(ts + cb * 32 + 16, l);
            }
          };
          // columns of block cb to keep: tokens up to the end of the sequence
          auto tokens = [&](int cb) {
            const int left = valid - 32 * cb;
            return left >= 32 ? 0xffffffffu : (left <= 0 ? 0u : (1u << left) - 1u);
          };
          // zeros where the mask has none (not by zero weights: a score there may be infinite)
          auto keep = [&](uint32_t mask) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              p[j].x = (mask >> (2 * j)) & 1u ? p[j].x : 0.f;
              p[j].y = (mask >> (2 * j + 1)) & 1u ? p[j].y : 0.f;
            }
          };
          if (part == 0) {
            tmem_ld32_sync(ts + w4 * 32, r);
#pragma unroll
            for (int j = 0; j < 16; ++j)
              p[j] = __fmul2_rn(pair_of(r[2 * j], r[2 * j + 1]), make_float2(diag[2 * j], diag[2 * j + 1]));
            keep(x.rev ? tokens(w4) & (0xffffffffu << lane) : 0xffffffffu >> (31 - lane));
            put(w4);
          }
          if (part == 1) {
            float rf = l_first;
#pragma unroll 1
            for (int d = 1; d <= nb; ++d) {
              const int cb = w4 + dir * d;
              tmem_ld32_sync(ts + cb * 32, r);
              const float2 rf2 = make_float2(rf, rf);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 f = reinterpret_cast<const float4*>(tab)[j];
                p[2 * j] = __fmul2_rn(pair_of(r[4 * j], r[4 * j + 1]), __fmul2_rn(rf2, make_float2(f.x, f.y)));
                p[2 * j + 1] = __fmul2_rn(pair_of(r[4 * j + 2], r[4 * j + 3]), __fmul2_rn(rf2, make_float2(f.z, f.w)));
              }
              if (x.rev && valid < 128) keep(tokens(cb));
              put(cb);
              rf *= l32;
            }
            uint32_t z[16];  // the other side of the diagonal is zero
#pragma unroll
            for (int j = 0; j < 16; ++j) z[j] = 0;
#pragma unroll 1
            for (int d = 1; d <= 3 - nb; ++d) {
              tmem_st16(ts + (w4 - dir * d) * 32, z);
              if (NT == 3) tmem_st16(ts + (w4 - dir * d) * 32 + 16, z);
            }
          }
          tmem_st_wait();
          tc_fence_before();
          warp_arrive(bar(P_FULL + (g & 1)));
          if (g > 0 && !(ok = write_out())) break;
          o_dir = x.dir;
          o_col = x.half * 64 + 32 * part;
          o_h = x.h;
          o_tok = x.token(c);
          o_b = x.b;
          o_valid = valid;
          const int lead = x.starts(c) ? one.dir.lead : 0;
          o_scale = a.scale * exp2f(l2 * static_cast<float>((x.rev ? valid - i : i + 1) - lead));
          ++g;
        }
      }
      if (ok && g > 0) write_out();
      if (lane == 0) bulk_wait_all();
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------ state
    const int r = threadIdx.x - 8 * 32;
    constexpr int NC = C::NC;
    const int row = DK == 64 ? (r & 63) : r, col0 = DK == 64 ? (r >> 6) * 32 : 0;
    int g = 0;
    bool ok = true;
    // fp32: these warps have the time to split k, a chunk ahead of the state
    ChunkIter<DK, STATES> k_it;
    bool k_more = !BF16 && !STATES && k_it.first(a, n_units);
    auto split_k = [&]() {
      if constexpr (!BF16 && !STATES) {
        if (!k_more) return true;
        const int s = k_it.g % C::QKS;
        if (!mbar_wait_warp(bar(QK_RAW + s), (k_it.g / C::QKS) & 1, status)) return false;
        const Split<128> k(sK(s), r);
#pragma unroll 1
        for (int i = 0; i < Split<128>::VECS; i += 8) k.template eight<NP>(i, k_it.valid());
        fence_proxy_async_smem();
        warp_arrive(bar(QK_FULL + s));
        k_more = k_it.next(a);
      }
      return true;
    };
    ok = split_k();
    // the segments' states: also where there is nothing to do, so that this launch ends after theirs
    if (!STATES && a.n_seg > 1) wait_prerequisites();
    for (int u = blockIdx.x; ok && u < n_units; u += gridDim.x) {
      const MixUnit x = mix_unit<DK, STATES>(a, u);
      const MixOne& one = a.one[x.dir];
      const float l2 = log2_decay(a.log_decay, x.h);
      const bool in_state = row < a.D && x.half * 64 + col0 < a.D;  // head dim 32: a quarter of the tile
      // element (row, column 0) of the caller's state
      const long long e0 = x.half * 64 + col0;
      const size_t st0 = (static_cast<size_t>(x.b) * a.H + x.h) * a.D * a.D +
                         (one.dir.transposed ? e0 * a.D + row : static_cast<long long>(row) * a.D + e0);
      float2 S[NC / 2];
      auto save = [&](int slot) {
        float4* dst = reinterpret_cast<float4*>(seg_slot<DK>(a, x, slot));
#pragma unroll
        for (int c = 0; c < NC / 4; ++c)
          dst[c * 128 + r] = make_float4(S[2 * c].x, S[2 * c].y, S[2 * c + 1].x, S[2 * c + 1].y);
      };
      const bool carried = a.n_seg == 1 || (STATES && x.seg == (x.rev ? a.fine : 0));
#pragma unroll
      for (int c = 0; c < NC / 2; ++c) S[c] = make_float2(0.f, 0.f);
      if (carried && one.s_in && in_state) {
        const float* src = one.s_in + st0;
        const float w = one.dir.in_mult;
#pragma unroll
        for (int c = 0; c < NC / 4; ++c) {
          float4 f;
          if (one.dir.transposed)  // the lanes' values lie side by side
            f = make_float4(src[4 * c * a.D], src[(4 * c + 1) * a.D], src[(4 * c + 2) * a.D], src[(4 * c + 3) * a.D]);
          else
            f = reinterpret_cast<const float4*>(src)[c];
          S[2 * c] = make_float2(w * f.x, w * f.y);
          S[2 * c + 1] = make_float2(w * f.z, w * f.w);
        }
      }
      const int last = x.n > 0 ? (x.n - 1) / a.seg_tokens : 0;  // the segment of the last token
      if (STATES) {
        if (carried) save(a.n_slots - 1);
#pragma unroll
        for (int c = 0; c < NC / 2; ++c) S[c] = make_float2(0.f, 0.f);
      } else if (a.n_seg > 1) {
        // the state entering this segment, from the carried one and the segments in between
        auto add = [&](int slot, int tokens) {
          const float w = exp2f(l2 * static_cast<float>(tokens));
          const float4* src = reinterpret_cast<const float4*>(seg_slot<DK>(a, x, slot));
#pragma unroll
          for (int c = 0; c < NC / 4; ++c) {
            const float4 f = src[c * 128 + r];
            S[2 * c] = __ffma2_rn(make_float2(w, w), make_float2(f.x, f.y), S[2 * c]);
            S[2 * c + 1] = __ffma2_rn(make_float2(w, w), make_float2(f.z, f.w), S[2 * c + 1]);
          }
        };
        const int end = x.p0 + a.seg_tokens;
        const int before = x.rev ? (x.n > end ? x.n - end : 0) : x.p0;  // tokens before this segment
        add(a.n_slots - 1, before > 0 ? before - one.dir.lead : 0);
        if (x.count > 0) {
          if (x.rev)
            for (int f = (x.seg + 1) * a.fine; f * a.state_tokens < x.n; ++f) add(f - a.fine, f * a.state_tokens - end);
          else
            for (int f = 0; f < x.seg * a.fine; ++f) add(f, x.p0 - (f + 1) * a.state_tokens);
        }
      }
      // the state's bf16 parts for chunk gg's Q S
      auto put_state = [&](int gg) {
        if (gg > 0 && !mbar_wait_warp(bar(ST_EMPTY), (gg - 1) & 1, status)) return false;
#pragma unroll
        for (int c = 0; c < NC / 8; ++c) {
          uint32_t h[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) h[j] = hi_pair(S[4 * c + j]);
          const uint32_t at = ss0 + sw128_offset(row, col0 * 2 + c * 16);
          st_shared_v4(at, h[0], h[1], h[2], h[3]);
          if (NT == 3)
            st_shared_v4(at + C::ST_PLANE, lo_pair(S[4 * c], h[0]), lo_pair(S[4 * c + 1], h[1]),
                         lo_pair(S[4 * c + 2], h[2]), lo_pair(S[4 * c + 3], h[3]));
        }
        fence_proxy_async_smem();
        warp_arrive(bar(ST_FULL));
        return true;
      };
      if (!STATES && x.chunks > 0 && !(ok = put_state(g))) break;
      for (int c = 0; c < x.chunks; ++c, ++g) {
        // the carried state enters the very first token without a decay (lead)
        const int lead = !STATES && x.starts(c) ? one.dir.lead : 0;
        const float dec = exp2f(l2 * static_cast<float>(x.valid(c) - lead));
        const float2 dec2 = make_float2(dec, dec);
        if (!(ok = split_k())) break;
        if (!(ok = mbar_wait_warp(bar(KV_FULL + g % VB), (g / VB) & 1, status))) break;
        tc_fence_after();
#pragma unroll
        for (int j = 0; j < NC / 16; ++j) {
          uint32_t vh[16], vl[16];  // K^T V' hi and K^T V' lo
          const uint32_t at = tmem + kv_at(g) + col0 + j * 16 + lane_base;
          tmem_ld16x2_sync(at, at + 64, vh, vl);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            S[8 * j + e] = __ffma2_rn(dec2, S[8 * j + e], __fadd2_rn(pair_of(vh[2 * e], vh[2 * e + 1]),
                                                                   pair_of(vl[2 * e], vl[2 * e + 1])));
        }
        tc_fence_before();
        warp_arrive(bar(KV_FREE + g % VB));
        if (!STATES && c + 1 < x.chunks && !(ok = put_state(g + 1))) break;
      }
      if (!ok) break;
      if (STATES) {
        save(x.rev ? x.seg - a.fine : x.seg);
        continue;
      }
      // the state after the last token in time order
      if (one.s_out && in_state && x.seg == (x.rev ? 0 : last)) {
        const float w = one.dir.out_mult * (one.dir.lead && x.n > 0 ? exp2f(l2) : 1.f);
        float4* dst = reinterpret_cast<float4*>(one.s_out + st0);  // (a transposed state has no output)
#pragma unroll
        for (int c = 0; c < NC / 4; ++c)
          dst[c] = make_float4(w * S[2 * c].x, w * S[2 * c].y, w * S[2 * c + 1].x, w * S[2 * c + 1].y);
      }
      if (!one.dir.accumulate) {  // zeros past the sequence
        const int p1 = a.L - x.p0 < a.seg_tokens ? a.L : x.p0 + a.seg_tokens;
        const int pz = x.n > x.p0 ? x.n : x.p0;
        const int vecs = (a.D < 64 ? a.D : 64) * static_cast<int>(sizeof(T)) / 16;
        const long long zeros = static_cast<long long>(p1 - pz) * vecs;
        for (long long z = r; z < zeros; z += 128) {
          const size_t tok = static_cast<size_t>(x.b) * a.L + pz + z / vecs;
          reinterpret_cast<uint4*>(static_cast<T*>(one.o) + (tok * a.H + x.h) * a.D + x.half * 64)[z % vecs] =
              make_uint4(0, 0, 0, 0);
        }
      }
    }
  } else if (warp < 16) {
    // ------------------------------------------------------------ V'
    const int t = threadIdx.x - 12 * 32;
    ChunkIter<DK, STATES> it;
    bool more = it.first(a, n_units);
    int w_unit = -1, w_valid = 0;
    // l^(valid - 1 - row), backward l^row; zero past the end
    auto weight = [&](float l2, int row, int valid) {
      return row < valid ? exp2f(l2 * static_cast<float>(it.x.rev ? row : valid - 1 - row)) : 0.f;
    };
    if constexpr (BF16) {
      // Each thread has 16-byte column t % 8 of rows t / 8 + 16 i. A weight w is two bf16 parts;
      // hi = bf16(v w_hi), and since v w_hi has 16 bits, v w_hi - hi is a bf16 too:
      // lo = bf16(v w_lo + (v w_hi - hi)), off by 2^-17 of v w, in three packed instructions.
      __nv_bfloat162 wh[8], wl[8];
      for (; more; more = it.next(a)) {
        const int g = it.g, vs = g % C::VS, valid = it.valid();
        if (it.u != w_unit || valid != w_valid) {
          const float l2 = log2_decay(a.log_decay, it.x.h);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float w = weight(l2, t / 8 + 16 * i, valid);
            wh[i] = __float2bfloat162_rn(w);
            wl[i] = __float2bfloat162_rn(w - __low2float(wh[i]));
          }
          w_unit = it.u;
          w_valid = valid;
        }
        if (!mbar_wait_warp(bar(V_FULL + vs), (g / C::VS) & 1, status)) break;
        uint4 v[8];  // all loads before the first store: they may not pass it
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = ld_shared_v4(sV(vs) + sw128_offset(t / 8 + 16 * i, (t % 8) * 16));
        if (valid < 128) {
          // Tokens past this sequence lie in the tiles, and may hold anything: their rows of V meet
          // zeros of P, and their rows of K zeros of V', which NaN or infinity would survive.
          const int s = g % C::QKS;
          if (!mbar_wait_warp(bar(QK_FULL + s), (g / C::QKS) & 1, status)) break;
          for (int z = t + valid * 8; z < 128 * 8; z += 128) {
            st_shared_v4(sV(vs) + z * 16, 0, 0, 0, 0);
            for (int tile = 0; tile < KT; ++tile) st_shared_v4(sK(s) + tile * kTile + z * 16, 0, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (t / 8 + 16 * i >= valid) v[i] = make_uint4(0, 0, 0, 0);
        }
        if (g >= VB && !mbar_wait_warp(bar(VP_EMPTY + g % VB), (g / VB - 1) & 1, status)) break;
        const uint32_t to = vp_at(g), to_lo = to + vp_lo(g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t off = sw128_offset(t / 8 + 16 * i, (t % 8) * 16);
          const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
          uint32_t h[4], l[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 vv = *reinterpret_cast<const __nv_bfloat162*>(&x[j]);
            const __nv_bfloat162 hh = __hmul2_rn(vv, wh[i]);
            const __nv_bfloat162 ll = __hfma2(vv, wl[i], __hfma2(vv, wh[i], __hneg2(hh)));
            h[j] = *reinterpret_cast<const uint32_t*>(&hh);
            l[j] = *reinterpret_cast<const uint32_t*>(&ll);
          }
          st_shared_v4(to + off, h[0], h[1], h[2], h[3]);
          st_shared_v4(to_lo + off, l[0], l[1], l[2], l[3]);
        }
        fence_proxy_async_smem();
        warp_arrive(bar(VP_FULL + g % VB));
      }
    } else {
      // fp32: v lands where its V' goes
      using X = Split<128>;
      float w[X::VECS];
      for (; more; more = it.next(a)) {
        const int g = it.g, valid = it.valid();
        if (it.u != w_unit || valid != w_valid) {
          const float l2 = log2_decay(a.log_decay, it.x.h);
#pragma unroll
          for (int i = 0; i < X::VECS; ++i) w[i] = weight(l2, t / 16 + i * X::ROWS, valid);
          w_unit = it.u;
          w_valid = valid;
        }
        if (!mbar_wait_warp(bar(V_RAW + g % VB), (g / VB) & 1, status)) break;
        const X v(vp_at(g), t);  // (its planes are a tile apart there in either place)
        float4 r[X::VECS];
#pragma unroll
        for (int i = 0; i < X::VECS; ++i) r[i] = v.load(i, valid);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < X::VECS; ++i)
          v.template store<2>(vp_at(g), i, make_float4(r[i].x * w[i], r[i].y * w[i], r[i].z * w[i], r[i].w * w[i]));
        fence_proxy_async_smem();
        warp_arrive(bar(VP_FULL + g % VB));
        if (!STATES) {
          if (g > 0 && !mbar_wait_warp(bar(V_EMPTY), (g - 1) & 1, status)) break;
#pragma unroll
          for (int i = 0; i < X::VECS; ++i) v.template store<NP>(sV(0), i, r[i]);
          fence_proxy_async_smem();
          warp_arrive(bar(V_FULL));
        }
      }
    }
  } else if (role == 1) {
    // ------------------------------------------------------------ TMA loads
    if (loads) {
      if (abort_flag) load_more = false;
      while (load_more && load(load_it)) load_more = load_it.next(a);
      // What is still on its way must land before the block ends, also where a failure, here or in another
      // block and at any moment, lets the other roles leave without waiting for it.
      auto landed = [&](int first, int ring, int n) {
        for (int g = n < ring ? 0 : n - ring; g < n; ++g) mbar_drain(bar(first + g % ring), (g / ring) & 1);
      };
      landed(BF16 ? QK_FULL : QK_RAW, C::QKS, n_qk);
      landed(BF16 ? V_FULL : V_RAW, BF16 ? C::VS : VB, n_v);
    }
  } else if (role >= 2) {
    // ------------------------------------------------------------ fp32: split q in place (segment states: k)
    if constexpr (!BF16) {
      const int t = (role - 2) * 32 + lane_id();
      ChunkIter<DK, STATES> it;
      for (bool more = it.first(a, n_units); more; more = it.next(a)) {
        const int g = it.g, s = g % C::QKS;
        if (!mbar_wait_warp(bar(QK_RAW + s), (g / C::QKS) & 1, status)) break;
        const Split<64> x(STATES ? sK(s) : sQ(s), t);
#pragma unroll 1
        for (int i = 0; i < Split<64>::VECS; i += 8) x.template eight<NP>(i, it.valid());
        fence_proxy_async_smem();
        warp_arrive(bar(QK_FULL + s));
      }
    }
  } else if (role == 0) {
    // ------------------------------------------------------------ MMA issue
    if (elect_one()) {
      int total = 0;
      for (int u = blockIdx.x; u < n_units; u += gridDim.x) total += mix_unit<DK, STATES>(a, u).chunks;
      constexpr uint32_t idS = make_idesc(128, 128, 1, false, false), idV = make_idesc(128, 64, 1, false, true),
                         idKV = make_idesc(128, 128, 1, true, true), idKV1 = make_idesc(128, 64, 1, true, true);
      constexpr int LO = KT * kTile;  // from a hi plane of q or k to its lo plane
      // K-step `k` of a K-major tile, of an MN-major one
      auto kmaj = [](int k) { return static_cast<uint32_t>((k / 4) * kTile + (k % 4) * 32); };
      auto mn = [](int k) { return static_cast<uint32_t>(k * 2048); };
      const Desc dQ{make_sdesc(sQ(0), 16, 1024)}, dK{make_sdesc(sK(0), 16, 1024)},
          dKt{make_sdesc(sK(0), DK == 64 ? 0 : kTile, 1024)}, dV{make_sdesc(sV(0), kTile, 1024)},
          dS{make_sdesc(ss0, kTile, 1024)};
      auto wait = [&](int i, int phase) { return mbar_wait(bar(i), phase & 1, status); };
      // Three products each make the unrolled code long, and its first pass waits for it to arrive:
      // fp32 8 x 1024 x 8 x 64 takes 45.1 us rolled, 46.5 unrolled, bf16 8 x 4096 x 16 x 64 66 and 62.
      constexpr int UNROLL_MMA = BF16 ? 8 : 1;
      auto issue_S = [&](int g) {
        const int s = g % C::QKS;
        if (!wait(QK_FULL + s, g / C::QKS)) return false;
        tc_fence_after();
        const Desc q = dQ.at(s * 2 * C::OPER), kk = dK.at(s * 2 * C::OPER);
#pragma unroll
        for (int term = 0; term < NT; ++term)
#pragma unroll UNROLL_MMA
          for (int k = 0; k < DK / 16; ++k)
            umma_f16_ss(tmem + T_S + (g & 1) * 128, q.at((term == 2 ? LO : 0) + kmaj(k)).d,
                        kk.at((term == 1 ? LO : 0) + kmaj(k)).d, idS, (term > 0 || k > 0) ? 1u : 0u);
        umma_commit(bar(S_FULL + (g & 1)));
        return true;
      };
      bool ok = true;
      for (int g = 0; ok && g < total; ++g) {
        const int s = g % C::QKS, vs = g % C::VS, b = g & 1;
        ok = wait(QK_FULL + s, g / C::QKS);
        if (!STATES && g == 0) ok = ok && issue_S(0);
        // K^T [V' hi, V' lo] (DK = 64: both halves of the 128 rows are the same 64 rows of the
        // state, so every warp of the state finds its columns in its own lanes)
        ok = ok && wait(VP_FULL + g % VB, g / VB) && (g < VB || wait(KV_FREE + g % VB, g / VB - 1));
        if (!ok) break;
        tc_fence_after();
        const Desc kt = dKt.at(s * 2 * C::OPER), vp{make_sdesc(vp_at(g), vp_lo(g), 1024)};
        const uint32_t kv = tmem + kv_at(g);
#pragma unroll UNROLL_MMA
        for (int k = 0; k < 8; ++k) umma_f16_ss(kv, kt.at(mn(k)).d, vp.at(mn(k)).d, idKV, k > 0 ? 1u : 0u);
        if (NT == 3) {
#pragma unroll UNROLL_MMA
          for (int k = 0; k < 8; ++k) umma_f16_ss(kv, kt.at(LO + mn(k)).d, vp.at(mn(k)).d, idKV1, 1u);
        }
        umma_commit(bar(KV_FULL + g % VB));
        umma_commit(bar(VP_EMPTY + g % VB));
        if (STATES) {
          umma_commit(bar(QK_EMPTY + s));
          umma_commit(bar(V_EMPTY + vs));
          continue;
        }
        // The next chunk's scores before this one's Q S, so that its P is ready in time; fp32 tiles, of
        // which there are two, the other way round: Q S frees the tiles of the chunk after next.
        if (BF16 && g + 1 < total && !(ok = issue_S(g + 1))) break;
        // Q S from the state entering this chunk
        ok = wait(ST_FULL, g) && (g < 1 || wait(O_FREE, g - 1));
        if (!ok) break;
        tc_fence_after();
        const Desc q = dQ.at(s * 2 * C::OPER);
#pragma unroll
        for (int term = 0; term < NT; ++term)
#pragma unroll UNROLL_MMA
          for (int k = 0; k < DK / 16; ++k)
            umma_f16_ss(tmem + T_QS, q.at((term == 2 ? LO : 0) + kmaj(k)).d,
                        dS.at((term == 1 ? C::ST_PLANE : 0) + mn(k)).d, idV, (term > 0 || k > 0) ? 1u : 0u);
        umma_commit(bar(ST_EMPTY));
        umma_commit(bar(QK_EMPTY + s));
        if (!BF16 && g + 1 < total && !(ok = issue_S(g + 1))) break;
        // P V
        ok = wait(V_FULL + vs, g / C::VS) && wait(P_FULL + b, g >> 1);
        if (!ok) break;
        tc_fence_after();
        const Desc v = dV.at(vs * C::V_STAGE);
#pragma unroll
        for (int term = 0; term < NT; ++term)
#pragma unroll UNROLL_MMA
          for (int k = 0; k < 8; ++k)
            umma_f16_ts(tmem + T_PV, tmem + T_S + b * 128 + (term == 2 ? 16 : 0) + (k / 2) * 32 + (k % 2) * 8,
                        v.at((term == 1 ? kTile : 0) + mn(k)).d, idV, (term > 0 || k > 0) ? 1u : 0u);
        umma_commit(bar(V_EMPTY + vs));
        umma_commit(bar(O_FULL));
      }
      if (total > 0) {  // as with the copies: no product reads tiles or writes TMEM that the block gives up
        umma_commit(bar(MMA_DONE));
        mbar_drain(bar(MMA_DONE), 0);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (role == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One new token. A block takes 32 columns of a state (sequence, head): 8 lanes a row of
// 128 bytes, 16 rows a pass, all passes' loads in flight at once. Bound by HBM: the
// state is read once and written once. 64 sequences of 16 heads of 128 (134 MB) take 24.6 us, 5.5
// TB/s, of 32 heads 39.4 us, 6.8 TB/s; one sequence of 8 heads of 64 2.3 us, less than its
// launch on the host. Whole states a block (fewer, larger) left SMs idle where users are few.
constexpr int kStepThreads = 128, kStepCols = 32;
template <typename T, int D>
__global__ void __launch_bounds__(kStepThreads)
    mix_step_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                    const float* __restrict__ log_decay, const float* s_in, T* __restrict__ o, float* s_out,
                    int H, float scale) {
  constexpr int BLOCKS = D / kStepCols, ROWS = kStepThreads / 8, PASSES = D / ROWS;
  __shared__ float part[ROWS][kStepCols];
  const int bh = blockIdx.x / BLOCKS, col = (blockIdx.x % BLOCKS) * kStepCols + (threadIdx.x % 8) * 4;
  const int r0 = threadIdx.x / 8;
  const size_t st0 = static_cast<size_t>(bh) * D * D + col, at = static_cast<size_t>(bh) * D;
  float4 s[PASSES];
  float kd[PASSES], qd[PASSES], ve[4];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) s[i] = *reinterpret_cast<const float4*>(s_in + st0 + (r0 + i * ROWS) * D);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    kd[i] = ld_f(k + at + r0 + i * ROWS);
    qd[i] = ld_f(q + at + r0 + i * ROWS);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) ve[j] = ld_f(v + at + col + j);
  const float lam = exp2f(log2_decay(log_decay, bh % H));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    s[i].x = fmaf(lam, s[i].x, kd[i] * ve[0]);
    s[i].y = fmaf(lam, s[i].y, kd[i] * ve[1]);
    s[i].z = fmaf(lam, s[i].z, kd[i] * ve[2]);
    s[i].w = fmaf(lam, s[i].w, kd[i] * ve[3]);
    *reinterpret_cast<float4*>(s_out + st0 + (r0 + i * ROWS) * D) = s[i];
    acc.x = fmaf(qd[i], s[i].x, acc.x);
    acc.y = fmaf(qd[i], s[i].y, acc.y);
    acc.z = fmaf(qd[i], s[i].z, acc.z);
    acc.w = fmaf(qd[i], s[i].w, acc.w);
  }
  *reinterpret_cast<float4*>(&part[r0][(threadIdx.x % 8) * 4]) = acc;
  __syncthreads();
  if (threadIdx.x < kStepCols) {  // fixed order: the same bits every time
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) sum += part[i][threadIdx.x];
    st_f(o + at + (blockIdx.x % BLOCKS) * kStepCols + threadIdx.x, scale * sum);
  }
}

// Segments of one sequence. A sequence's chunks follow one another, so with few
// (sequence, head) pairs most of the GPU would idle: the sequence is cut, the
// segments' own states are computed first (k and v are read a second time) and
// each segment starts from their sum.
struct MixPlan {
  int pairs;             // units of a segment: (sequence, head, direction, column half)
  int n_seg, seg_tokens;
  int fine;              // pieces of a segment whose states are computed on their own
  int n_slots;
};
MixPlan mix_plan(const AttnShape& sh, bool f32, int n_dir) {
  MixPlan p;
  const int chunks = (sh.L + 127) / 128, sms = device_sm_count();
  p.pairs = sh.B * sh.H * n_dir * (sh.D == 128 ? 2 : 1);
  // Segments for the SMs there are, of 2 chunks at least (2 heads, 64 chunks: fp32 33 us with 32
  // segments, 40 with 64; bf16 25 and 34), and so few that adding up their states stays cheap (2 heads,
  // bf16: 64 chunks 23 us with 22 segments, 25 with 32; 1024 chunks 72 with 64, 74 with 74).
  int seg = sms / p.pairs;
  if (seg > chunks / 2) seg = chunks / 2;
  while (seg > 1 && seg * seg > 8 * chunks) --seg;
  // None where the second launch and the second reading of k and v cost more than the chunks that a
  // sequence no longer waits for. bf16: 8 heads in 2 segments 8 chunks 18.6 us whole and 19.3 cut, 12
  // chunks 24.5 and 23.6; 32 heads in 4, 6 chunks 16.5 and 17.2, 8 chunks 18.5 and 17.4. A chunk of
  // fp32 takes twice as long: 32 heads in 2 segments 6 chunks 30 and 29, 8 chunks 37 and 34. With 64 heads
  // in 2 segments a cut gains less (warm, back to back): fp32 6 chunks 27.6 whole and 27.5 cut, 8 chunks
  // 35.1 and 34.0, 12 chunks 49.9 and 47.4; bf16 12 chunks 20.9 and 21.5, 16 chunks 26.1 and 24.7. From half
  // as many units as SMs on nothing is cut, and some SMs idle.
  if (seg > 1 && chunks - (chunks + seg - 1) / seg < (f32 ? 3 : 6)) seg = 1;
  if (seg < 1) seg = 1;
  int seg_chunks = (chunks + seg - 1) / seg;
  // The states' launch has one segment less: cut finer it still fills the GPU (2 x 16384 tokens of 16
  // heads of 128: 191 us, 220 without).
  p.fine = seg > 1 ? sms / (p.pairs * (seg - 1)) : 1;
  if (p.fine > seg_chunks / 4) p.fine = seg_chunks / 4;
  if (p.fine < 1) p.fine = 1;
  seg_chunks = (seg_chunks + p.fine - 1) / p.fine * p.fine;
  p.n_seg = (chunks + seg_chunks - 1) / seg_chunks;
  p.seg_tokens = seg_chunks * 128;
  p.n_slots = (p.n_seg - 1) * p.fine + 1;
  return p;
}

template <typename T, int DK, int NT>
int mix_launch(MixArgs a, const MixMaps& maps, uint32_t* status, cudaStream_t s) {
  using C = MixCfg<T, DK, NT>;
  static std::atomic<uint64_t> attr_s{0}, attr{0};
  const int sms = device_sm_count();
  if (a.n_seg > 1) {
    if (!ensure_smem_attr(mix_kernel<T, DK, NT, true>, C::SMEM, attr_s)) return PA_ERR_LAUNCH;
    MixArgs f = a;
    f.n_units = a.n_units / a.n_seg * (a.n_slots - 1);
    mix_kernel<T, DK, NT, true><<<f.n_units < sms ? f.n_units : sms, kMixThreads, C::SMEM, s>>>(f, maps, status);
    if (cudaGetLastError() != cudaSuccess) return PA_ERR_LAUNCH;
  }
  if (!ensure_smem_attr(mix_kernel<T, DK, NT, false>, C::SMEM, attr)) return PA_ERR_LAUNCH;
  // After the states' launch this one starts while that one runs (all its blocks are on SMs by then,
  // so these take none from them) and waits for it where a state is added up.
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.n_units < sms ? a.n_units : sms);
  cfg.blockDim = dim3(kMixThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = a.n_seg > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, mix_kernel<T, DK, NT, false>, a, maps, status) == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

// An input [B, L, H, D] as boxes of 128 bytes of columns x 1 head x 128 tokens, bf16 in
// the MMA operands' swizzle.
bool make_in_map(CUtensorMap* m, const void* base, const AttnShape& sh, bool f32) {
  if (!f32) return make_qkv_map(m, base, sh, 128);
  const uint64_t D = sh.D, H = sh.H, L = sh.L;
  const uint64_t dims[4] = {D, H, L, static_cast<uint64_t>(sh.B)};
  const uint64_t strides[3] = {D * 4, H * D * 4, L * H * D * 4};
  const uint32_t box[4] = {32, 1, 128, 1};
  return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// An output [B, L, H, D] as boxes of 64 bytes of columns x 1 head x 32 tokens.
bool make_out_map(CUtensorMap* m, const void* base, const AttnShape& sh, bool f32) {
  const uint64_t e = f32 ? 4 : 2, D = sh.D, H = sh.H, L = sh.L;
  const uint64_t dims[4] = {D, H, L, static_cast<uint64_t>(sh.B)};
  const uint64_t strides[3] = {D * e, H * D * e, L * H * D * e};
  const uint32_t box[4] = {static_cast<uint32_t>(64 / e), 1, 32, 1};
  return make_tmap(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides,
                   box, CU_TENSOR_MAP_SWIZZLE_64B);
}

int mix(const AttnShape& sh, bool f32, MixArgs a, const float* log_decay, const int32_t* lens, void* ws,
        uint32_t* status, cudaStream_t s) {
  const MixPlan p = mix_plan(sh, f32, a.n_dir);
  a.log_decay = log_decay;
  a.lens = lens;
  a.ws = static_cast<float*>(ws);
  a.B = sh.B;
  a.L = sh.L;
  a.H = sh.H;
  a.D = sh.D;
  a.by_dir = Divisor::of(a.n_dir);
  a.by_H = Divisor::of(sh.H);
  a.by_B = Divisor::of(sh.B);
  a.n_seg = p.n_seg;
  a.seg_tokens = p.seg_tokens;
  a.n_units = p.pairs * p.n_seg;
  a.fine = p.fine;
  a.state_tokens = p.seg_tokens / p.fine;
  a.n_slots = p.n_slots;
  a.scale = sh.scale;
  MixMaps maps{};
  for (int d = 0; d < a.n_dir; ++d) {
    if (!make_out_map(&maps.o[d], a.one[d].o, sh, f32)) return PA_ERR_ALIGN;
    a.one[d].mo = d;
  }
  // tensor maps of the distinct inputs (at most q, k, v and dO)
  const void* seen[4];
  int n = 0;
  for (int d = 0; d < a.n_dir; ++d) {
    const void* in[3] = {a.one[d].q, a.one[d].k, a.one[d].v};
    int* index[3] = {&a.one[d].mq, &a.one[d].mk, &a.one[d].mv};
    for (int j = 0; j < 3; ++j) {
      int m = 0;
      while (m < n && seen[m] != in[j]) ++m;
      if (m == n) {
        if (!make_in_map(&maps.m[n], in[j], sh, f32)) return PA_ERR_ALIGN;
        seen[n++] = in[j];
      }
      *index[j] = m;
    }
  }
  if (f32)
    return f32_math() == PA_F32_MATH_BF16 ? mix_launch<float, 64, 1>(a, maps, status, s)
                                          : mix_launch<float, 64, 3>(a, maps, status, s);
  return sh.D == 64 ? mix_launch<__nv_bfloat16, 64, 1>(a, maps, status, s)
                    : mix_launch<__nv_bfloat16, 128, 1>(a, maps, status, s);
}

template <typename T, int D>
int step(const AttnShape& sh, const void* q, const void* k, const void* v, const float* log_decay,
         const float* s_in, void* o, float* s_out, cudaStream_t s) {
  mix_step_kernel<T, D><<<sh.B * sh.H * (D / kStepCols), kStepThreads, 0, s>>>(
      static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), log_decay, s_in,
      static_cast<T*>(o), s_out, sh.H, sh.scale);
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // namespace

size_t linear_attn_workspace_bytes(const AttnShape& sh, bool f32, bool backward) {
  const MixPlan p = mix_plan(sh, f32, backward ? 3 : 1);
  return p.n_seg == 1 ? 0 : static_cast<size_t>(p.pairs) * p.n_slots * (sh.D == 128 ? 128 : 64) * 64 * sizeof(float);
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
