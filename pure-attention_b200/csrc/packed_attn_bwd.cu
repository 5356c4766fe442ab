// Gradients of causal attention over packed sequences with shared key-value
// heads, for sm_100a: bf16 in, fp32 accumulation in TMEM.
//
//   P = exp(S scale - lse),  dP = dO V^T,  Delta = rowsum(dO o),  dS = P (dP - Delta)
//   dq = scale dS K,   dk = scale sum_heads dS^T Q,   dv = sum_heads P^T dO
//
// S and dP are computed twice (seven products where five would do), for dq and for dk and dv, so
// that each output is one accumulator in TMEM with one order of its sum: no fp32 dq
// is added up in memory, results do not depend on the run, and neither
// chain of products waits for the other's.
//   packed_stats_kernel  Delta and lse log2(e) per (head, query row), laid out in
//                        blocks of 128 rows of a sequence (rows behind its end: lse =
//                        +inf, so that their P is 0)
//   packed_bwd_kernel    its first blocks packed_dq: an item is (query tile, head), walking the key tiles up to
//                        the diagonal; rows of the products are queries
//                        the others packed_dkv: an item is (key tile, kv head), walking the query tiles from
//                        the diagonal on for each head of the group; rows are keys
// Both keep P and dS in TMEM as the A operand of the products that use them.
//
// Measured, lists and statistics included: 12800 tokens in 8 sequences of up to 4096, 16 heads of 64, 332 us (553
// TFLOP/s of the five products under the mask); 8192 tokens, 16 + 4 heads of 128, 739 us (930). At 128 the tensor
// pipe is 70% busy. At 64 it is 37% (dq) and 45% (dk, dv), the exponential unit 50%: a tile's products are
// short (one of 128 x 128 x 64 takes 362 clocks in a row of them, 768 with its barrier waited for), and each waits 450
// clocks from issue to barrier, which tiles in turn hide in part. dP in two buffers, dS in columns of its own and a
// second issuing warp, which take those waits out of the chain one by one, were not faster (dq 153 to 155 us; dk
// and dv with P^T in shared memory for the room 178 to 236 us; dq and dk / dv measured as launches of their own). One pass
// over the keys with five products, as attn_bwd.cu has for lengths that are all alike (905 TFLOP/s without a mask), was
// not tried: it adds dq up in memory, in an order that would have to be fixed for results that do not depend on the run.
#include <cuda_bf16.h>
#include <type_traits>
#include "packed_common.cuh"

namespace pa {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kChunk = 128 * 128;  // bytes of one 128-row x 128-byte box

// Rows of the statistics of one head: blocks of 128 rows, each sequence from a block of its own.
// Sequence i starts at block start_i / 128 + i: every sequence before it has less than one block
// that is not full.
__host__ __device__ inline long long stat_blocks(int T, int n) { return static_cast<long long>(T) / 128 + n; }
__device__ __forceinline__ size_t stat_row(const PackedUnit& u, int tile) {
  return (static_cast<size_t>(u.start / 128) + u.seq + tile) * 128;
}

// TMEM column of the k-th 16-column K-step of packed P / dS: each warpgroup packs its 64
// columns (32 of bf16 pairs) at the start of the 64 fp32 columns that it read.
__device__ __forceinline__ uint32_t step_col(int k) { return k < 4 ? k * 8 : 64 + (k - 4) * 8; }

// ---------------------------------------------------------------- statistics
constexpr int kStatBlocks = 3;  // per SM; a thread has its piece of 4 or 8 rows of o and dO in flight
template <int D>
__global__ void __launch_bounds__(256, kStatBlocks)
    packed_stats_kernel(const bf16* __restrict__ dO, const bf16* __restrict__ O, const float* __restrict__ lse,
                        const __grid_constant__ PackedWork work, int T, int H, long long rows, float* __restrict__ lse2,
                        float* __restrict__ delta) {
  constexpr int LANES = D / 8, STEP = 256 / LANES;  // lanes that share a row; rows of a pass
  launch_dependents();
  wait_prerequisites();
  // item = (unit, head), stepped through without divisions
  const int count = work.list ? load_written(&work.list->count) : static_cast<int>(gridDim.x) / H;
  const int lane = threadIdx.x % LANES, r0 = threadIdx.x / LANES;
  const int du = static_cast<int>(gridDim.x) / H, dh = static_cast<int>(gridDim.x) % H;
  int at_unit = static_cast<int>(blockIdx.x) / H, h = static_cast<int>(blockIdx.x) % H;
  auto unit_of = [&](int i) { return i >= count ? PackedUnit{0, 0, 0, 0} : work.list ? work.listed(i) : work.direct(i); };
  PackedUnit next = unit_of(at_unit);
  while (next.work) {
    const PackedUnit u = next;
    const int tile = u.work - 1, head = h;
    at_unit += du;
    h += dh;
    if (h >= H) {
      h -= H;
      ++at_unit;
    }
    next = unit_of(at_unit);
    const size_t out = head * static_cast<size_t>(rows) + stat_row(u, tile);
    uint4 a[128 / STEP], b[128 / STEP];
    float l[128 / STEP];
#pragma unroll
    for (int k = 0; k < 128 / STEP; ++k) {
      const int row = tile * 128 + r0 + k * STEP;
      if (row < u.len) {
        const size_t at = ((static_cast<size_t>(u.start) + row) * H + head) * D + lane * 8;
        a[k] = *reinterpret_cast<const uint4*>(dO + at);
        b[k] = *reinterpret_cast<const uint4*>(O + at);
      }
      l[k] = row < u.len ? lse[static_cast<size_t>(head) * T + u.start + row] * kLog2e : INFINITY;
    }
#pragma unroll
    for (int k = 0; k < 128 / STEP; ++k) {
      const int row = tile * 128 + r0 + k * STEP;
      float s = 0.f;
      if (row < u.len) {
        const __nv_bfloat162 *x = reinterpret_cast<const __nv_bfloat162*>(&a[k]),
                             *y = reinterpret_cast<const __nv_bfloat162*>(&b[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 p = __bfloat1622float2(x[e]), q = __bfloat1622float2(y[e]);
          s = fmaf(p.x, q.x, fmaf(p.y, q.y, s));
        }
      }
#pragma unroll
      for (int m = LANES / 2; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
      if (lane == 0) {
        const int at = r0 + k * STEP;
        delta[out + at] = s;
        lse2[out + at] = l[k];
      }
    }
  }
}

// 32 values of a lane's row `row`, scaled: to[i] (=|+=) o[i] * mul. to: the columns in row 0 of the sequence. All lanes of
// the warp take part.
__device__ __forceinline__ void write_row(bf16* to, long long stride, int row, int len, const uint32_t (&o)[32],
                                          float mul, int accumulate) {
  uint4 u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[8 * i + e]) * mul;
    if (accumulate && row < len) {
      const uint4 old = reinterpret_cast<const uint4*>(to + row * stride)[i];
      const __nv_bfloat162* p2 = reinterpret_cast<const __nv_bfloat162*>(&old);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 pf = __bfloat1622float2(p2[e]);
        f[2 * e] += pf.x;
        f[2 * e + 1] += pf.y;
      }
    }
    u[i] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
  const int quad = row & ~3;
  store_rows(to + quad * stride, stride, len - quad, u);
}

// Who computes P and dS: warps 0 to 2 load, issue and clear ragged rows; from warp 4 on, pairs of
// warpgroups compute, a thread half a row of a tile. At 64 head dimensions the products of a tile are short, and
// two pairs take the tiles in turn, so that one's exponentials run beside the other's dS (sequences of up to 4096
// tokens, 12800 in all, 16 heads: dq 169 to 153 us, dk and dv 235 to 178 us). They need more than the
// 96 registers that 640 threads leave each, and the first four warps give theirs. At 128 the products take longer
// than the exponentials and TMEM has no room for another tile in flight: there one pair with 168
// registers a thread is faster (8192 tokens, 16 + 4 heads: dq 299 us, two pairs 330; dk and dv 463 us, 479).
template <int D>
struct BwdWarps {
  static constexpr int PAIRS = D == 64 ? 2 : 1;
  static constexpr int ROLES = 4, PAIR = 256, THREADS = ROLES * 32 + PAIRS * PAIR;
  static constexpr int CHUNK = PAIRS == 2 ? 16 : 32;  // columns of dP that a thread holds at a time
  static constexpr int FEW = 64, MANY = 104;
  static_assert(FEW * 128 + MANY * 512 <= 640 * 96, "an increase would wait forever");
  static __device__ __forceinline__ void roles_regs() {
    if constexpr (PAIRS == 2) regs_dec<FEW>();
  }
  static __device__ __forceinline__ void pairs_regs() {
    if constexpr (PAIRS == 2) regs_inc<MANY>();
  }
  static __device__ __forceinline__ int pair_of(int g) { return PAIRS == 2 ? g & 1 : 0; }
  // The first tile of `pair` from tile g on.
  static __device__ __forceinline__ int first(int g, int pair) { return PAIRS == 2 ? g + ((g ^ pair) & 1) : g; }
};

template <int N>
__device__ __forceinline__ void load_columns(uint32_t at, uint32_t (&v)[N]) {
  if constexpr (N == 32) tmem_ld32_sync(at, v);
  else tmem_ld16_sync(at, v);
}
template <int N>
__device__ __forceinline__ void store_columns(uint32_t at, const uint32_t (&v)[N]) {
  if constexpr (N == 16) tmem_st16(at, v);
  else PA_TMEM_ST_X8(at, v);
}

// Maps of a call's tensors.
struct BwdMaps {
  CUtensorMap q, k, v, dO;
};

// What the issuer knows of a tile of the stream it works through.
struct StreamTile {
  int it;  // item
  bool valid, first, last, ragged;
};

// ---------------------------------------------------------------- dq
// TMEM: S0 [0,128) S1 [128,256) dP [256,384) dq [384, 384 + D); dS over its S. Per tile g the
// issuer runs dP(g+1) as soon as dP(g) is read, then dq(g), then S(g+2) over dS(g): the
// exponentials of a tile never wait for its scores.
template <int D>
struct PackedDq {
  static constexpr int KCH = D / 64;
  static constexpr int TILE = 128 * D * 2;
  static constexpr int QBUF = D == 64 ? 2 : 1;  // Q and dO of an item
  static constexpr int KST = D == 64 ? 4 : 3, VST = D == 64 ? 4 : 2;
  static constexpr int SMEM = (QBUF * 2 + KST + VST) * TILE + 1024;
  static constexpr uint32_t T_S = 0, T_DP = 256, T_DQ = 384;
};

template <int D>
__device__ __forceinline__ void packed_dq(const BwdMaps& maps, bf16* __restrict__ dq, long long dq_stride,
                                          const float* lse2, const float* delta, const PackedWork& work, int H, int group,
                                          long long rows, float scale, float scale_log2, int accumulate,
                                          uint32_t* status, int block, int blocks) {
  using C = PackedDq<D>;
  using W = BwdWarps<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[36];
  __shared__ PackedUnit own;  // without a list: the CTA's only unit
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  if (cta_aborted(status, &abort_flag)) {
    wait_prerequisites();
    return;
  }
  uint8_t* smem = align1024(smem_raw);
  uint8_t* sQ = smem;  // buffer u: Q, then dO
  uint8_t* sK = sQ + C::QBUF * 2 * C::TILE;
  uint8_t* sV = sK + C::KST * C::TILE;
  auto q_full = [&](int u) { return smem_u32(&bars[0 + u]); };
  auto q_empty = [&](int u) { return smem_u32(&bars[2 + u]); };
  auto k_full = [&](int s) { return smem_u32(&bars[4 + s]); };
  auto k_empty = [&](int s) { return smem_u32(&bars[8 + s]); };
  auto v_full = [&](int s) { return smem_u32(&bars[12 + s]); };
  auto v_empty = [&](int s) { return smem_u32(&bars[16 + s]); };
  // By tile parity: each pair waits for its own tiles only, and an arriving side can be a tile ahead.
  auto s_full = [&](int g) { return smem_u32(&bars[20 + (g & 1)]); };
  auto ds_full = [&](int g) { return smem_u32(&bars[22 + (g & 1)]); };
  auto dp_full = [&](int g) { return smem_u32(&bars[24 + (g & 1)]); };
  auto dp_free = [&](int g) { return smem_u32(&bars[26 + (g & 1)]); };
  // An item's dq is there, for the pair of its last tile (which may wait for it before the item before is
  // done, so each pair has a barrier of its own); it has been read.
  auto acc_done = [&](int pair) { return smem_u32(&bars[28 + pair]); };
  const uint32_t acc_free = smem_u32(&bars[34]);
  const uint32_t mma_done = smem_u32(&bars[35]);  // all products have ended
  // the f-th ragged K tile has landed, and its rows behind the end are zero; two are on the way at most
  auto k_ragged = [&](int f) { return smem_u32(&bars[30 + (f & 1)]); };
  auto k_zeroed = [&](int f) { return smem_u32(&bars[32 + (f & 1)]); };

  const int warp = warp_id();
  if (threadIdx.x == 0) {
    for (int u = 0; u < 2; ++u) {
      mbar_init(q_full(u), 1);
      mbar_init(q_empty(u), 1);
      mbar_init(s_full(u), 1);
      mbar_init(ds_full(u), W::PAIR);
      mbar_init(dp_full(u), 1);
      mbar_init(dp_free(u), W::PAIR);
      mbar_init(k_ragged(u), 1);
      mbar_init(k_zeroed(u), 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    for (int u = 0; u < 2; ++u) mbar_init(acc_done(u), 1);
    mbar_init(acc_free, W::PAIR);
    mbar_init(mma_done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  wait_prerequisites();
  if (threadIdx.x == 64 && !work.list) own = work.direct(block / H);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const long long n_items = work.items(H);
  auto unit_of = [&](int turn) {
    const long long i = packed_turn(turn, block, blocks);
    if (!work.list) return turn == 0 ? own : PackedUnit{0, 0, 0, 0};
    return i < n_items ? work.listed(static_cast<int>(i / H)) : PackedUnit{0, 0, 0, 0};
  };
  auto head_of = [&](int turn) { return static_cast<int>(packed_turn(turn, block, blocks) % H); };
  if (warp < W::ROLES) W::roles_regs();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      tma_prefetch_desc(&maps.q);
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
      tma_prefetch_desc(&maps.dO);
      bool ok = true;
      PackedUnit next = unit_of(0);
      int it = 0, g = 0, nv = 0;  // items, tiles of K and of V sent for
      while (ok && next.work) {
        const PackedUnit u = next;
        const int h = head_of(it), kh = h / group, row = u.start + (u.work - 1) * 128;
        next = unit_of(it + 1);
        const int b = it % C::QBUF, k = it / C::QBUF;
        if (k > 0 && !(ok = mbar_wait(q_empty(b), (k - 1) & 1, status))) break;
        mbar_arrive_expect_tx(q_full(b), 2 * C::TILE);
        for (int c = 0; c < C::KCH; ++c) {
          tma_load_3d(smem_u32(sQ + b * 2 * C::TILE + c * kChunk), &maps.q, q_full(b), c * 64, h, row);
          tma_load_3d(smem_u32(sQ + (b * 2 + 1) * C::TILE + c * kChunk), &maps.dO, q_full(b), c * 64, h, row);
        }
        ++it;
        for (int j = 0; j < u.work; ++j) {
          int s = g % C::KST;
          if (g >= C::KST && !(ok = mbar_wait(k_empty(s), ((g / C::KST) - 1) & 1, status))) break;
          mbar_arrive_expect_tx(k_full(s), C::TILE);
          for (int c = 0; c < C::KCH; ++c)
            tma_load_3d(smem_u32(sK + s * C::TILE + c * kChunk), &maps.k, k_full(s), c * 64, kh, u.start + j * 128);
          ++g;
          s = nv % C::VST;
          if (nv >= C::VST && !(ok = mbar_wait(v_empty(s), ((nv / C::VST) - 1) & 1, status))) break;
          mbar_arrive_expect_tx(v_full(s), C::TILE);
          for (int c = 0; c < C::KCH; ++c)
            tma_load_3d(smem_u32(sV + s * C::TILE + c * kChunk), &maps.v, v_full(s), c * 64, kh, u.start + j * 128);
          ++nv;
        }
      }
      drain_ring<C::QBUF>(it, q_full);
      drain_ring<C::KST>(g, k_full);
      drain_ring<C::VST>(nv, v_full);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t idS = make_idesc(128, 128, 1, false, false);
      constexpr uint32_t idQ = make_idesc(128, D, 1, false, true);
      const uint64_t dQ0 = make_sdesc(smem_u32(sQ), 16, 1024);
      const uint64_t dK0 = make_sdesc(smem_u32(sK), 16, 1024);
      const uint64_t dV0 = make_sdesc(smem_u32(sV), 16, 1024);
      const uint64_t dK_MN = make_sdesc(smem_u32(sK), kChunk, 1024);
      auto product = [&](uint32_t to, uint64_t a, uint64_t b) {  // K-major x K-major over D
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k / 4) * kChunk + (k % 4) * 32) >> 4;
          umma_f16_ss(to, a + off, b + off, idS, k > 0 ? 1u : 0u);
        }
      };
      bool ok = true;
      PackedUnit unit = unit_of(0);
      int turn = 0, left = unit.work;  // tiles of the item still to come
      auto next_tile = [&] {
        StreamTile t = {turn, unit.work > 0, left == unit.work, left == 1,
                        left == 1 && unit.work * 128 > unit.len};
        if (t.valid && --left == 0) {
          unit = unit_of(++turn);
          left = unit.work;
        }
        return t;
      };
      int rg = 0, rz = 0;  // ragged tiles announced, waited for
      auto issue_S = [&](const StreamTile& t, int g) {
        if (t.first && !mbar_wait(q_full(t.it % C::QBUF), (t.it / C::QBUF) & 1, status)) return false;
        if (!mbar_wait(k_full(g % C::KST), (g / C::KST) & 1, status)) return false;
        if (t.ragged) mbar_arrive(k_ragged(rg++));
        tc_fence_after();
        product(tmem + C::T_S + (g & 1) * 128, dQ0 + (((t.it % C::QBUF) * 2 * C::TILE) >> 4),
                dK0 + (((g % C::KST) * C::TILE) >> 4));
        umma_commit(s_full(g));
        return true;
      };
      auto issue_dP = [&](const StreamTile& t, int g) {
        if (!mbar_wait(v_full(g % C::VST), (g / C::VST) & 1, status)) return false;
        tc_fence_after();
        product(tmem + C::T_DP, dQ0 + ((((t.it % C::QBUF) * 2 + 1) * C::TILE) >> 4),
                dV0 + (((g % C::VST) * C::TILE) >> 4));
        umma_commit(dp_full(g));
        umma_commit(v_empty(g % C::VST));
        if (t.last) umma_commit(q_empty(t.it % C::QBUF));  // (its last S was issued before)
        return true;
      };
      StreamTile a = next_tile(), b = next_tile();
      if (a.valid) ok = issue_S(a, 0) && issue_dP(a, 0) && (!b.valid || issue_S(b, 1));
      for (int g = 0; ok && a.valid; ++g) {
        if (b.valid && !(ok = mbar_wait(dp_free(g), (g >> 1) & 1, status) && issue_dP(b, g + 1))) break;
        if (!(ok = mbar_wait(ds_full(g), (g >> 1) & 1, status))) break;
        if (a.ragged) {
          if (!(ok = mbar_wait(k_zeroed(rz), (rz >> 1) & 1, status))) break;
          ++rz;
        }
        // dq restarts from zero: the item before has been read
        if (a.first && a.it > 0 && !(ok = mbar_wait(acc_free, (a.it - 1) & 1, status))) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_f16_ts(tmem + C::T_DQ, tmem + C::T_S + (g & 1) * 128 + step_col(k),
                      dK_MN + (((g % C::KST) * C::TILE + k * 2048) >> 4), idQ, (!a.first || k > 0) ? 1u : 0u);
        umma_commit(k_empty(g % C::KST));
        if (a.last) umma_commit(acc_done(W::pair_of(g)));
        const StreamTile c = next_tile();
        if (c.valid && !(ok = issue_S(c, g + 2))) break;
        a = b;
        b = c;
      }
      drain_products(mma_done);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ rows behind a sequence's end
    PackedUnit next = unit_of(0);
    int g = 0, f = 0;
    for (int it = 0; next.work; ++it) {
      const PackedUnit u = next;
      next = unit_of(it + 1);
      g += u.work;
      if (u.work * 128 <= u.len) continue;
      if (!mbar_wait_warp(k_ragged(f), (f >> 1) & 1, status)) break;
      zero_rows(sK + ((g - 1) % C::KST) * C::TILE, C::KCH, u.len - (u.work - 1) * 128);
      if (lane_id() == 0) mbar_arrive(k_zeroed(f));
      ++f;
    }
  } else if (warp >= W::ROLES) {
    // ------------------------------------------------------------ P and dS
    // A pair takes every other tile, its warpgroup `half` the keys [64 half, 64 half + 64); thread = query row.
    W::pairs_regs();
    const int pair = (warp - W::ROLES) >> 3, half = ((warp - W::ROLES) >> 2) & 1;
    const int r = ((warp & 3) << 5) + static_cast<int>(lane_id());
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tdP = tmem + C::T_DP + lane_base + half * 64;
    bool ok = true;
    PackedUnit next = unit_of(0);
    auto stats = [&](const PackedUnit& u, int turn) {
      if (!u.work) return make_float2(0.f, 0.f);
      const size_t at = head_of(turn) * static_cast<size_t>(rows) + stat_row(u, u.work - 1) + r;
      return make_float2(lse2[at], delta[at]);
    };
    float2 st_next = stats(next, 0);
    int g0 = 0, done = 0;  // the item's first tile; items that this pair wrote
    for (int it = 0; ok && next.work; ++it) {
      const PackedUnit u = next;
      const float neg_lse = -st_next.x, del = st_next.y;
      next = unit_of(it + 1);
      st_next = stats(next, it + 1);
      const int last = g0 + u.work - 1;
      for (int g = W::first(g0, pair); g <= last; g += W::PAIRS) {
        const uint32_t tS = tmem + C::T_S + (g & 1) * 128 + lane_base + half * 64;
        if (!(ok = mbar_wait_warp(s_full(g), (g >> 1) & 1, status))) break;
        tc_fence_after();
        float p[64];
        tmem_ld32_sync(tS, *reinterpret_cast<uint32_t(*)[32]>(&p[0]));
        tmem_ld32_sync(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&p[32]));
#pragma unroll
        for (int i = 0; i < 64; ++i) p[i] = ex2(fmaf(p[i], scale_log2, neg_lse));
        if (!(ok = mbar_wait_warp(dp_full(g), (g >> 1) & 1, status))) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 64 / W::CHUNK; ++c) {
          constexpr int N = W::CHUNK;
          uint32_t v[N], ds[N / 2];
          load_columns(tdP + c * N, v);
          if (c == 64 / N - 1) {
            tc_fence_before();
            mbar_arrive(dp_free(g));  // the next dP may overwrite it
          }
          if (g == last) {  // the block on the diagonal
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float x = p[c * N + i] * (__uint_as_float(v[i]) - del);
              v[i] = __float_as_uint(half * 64 + c * N + i > r ? 0.f : x);
            }
          } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
              v[i] = __float_as_uint(p[c * N + i] * (__uint_as_float(v[i]) - del));
          }
#pragma unroll
          for (int i = 0; i < N / 2; ++i)
            ds[i] = pack_bf16x2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
          store_columns(tS + c * (N / 2), ds);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(ds_full(g));
      }
      if (!ok) break;
      g0 = last + 1;
      if (W::pair_of(last) != pair) continue;
      // dq write-back by the pair of the last tile, each warpgroup half of the columns, while
      // the other pair begins the next item
      if (!(ok = mbar_wait_warp(acc_done(pair), done & 1, status))) break;
      ++done;
      tc_fence_after();
      const int row = (u.work - 1) * 128 + r;
      bf16* dst = dq + static_cast<size_t>(u.start) * dq_stride + static_cast<size_t>(head_of(it)) * D;
#pragma unroll 1
      for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
        uint32_t o[32];
        tmem_ld32_sync(tmem + C::T_DQ + lane_base + c * 32, o);
        write_row(dst + c * 32, dq_stride, row, u.len, o, scale, accumulate);
      }
      tc_fence_before();
      mbar_arrive(acc_free);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- dk, dv
// TMEM, d = 64: S0 [0,128) S1 [128,256) dP [256,384) dv [384,448) dk [448,512); d = 128: S [0,128)
// dP [128,256) dv [256,384) dk [384,512). P^T over its S, dS^T over dP. Per tile g: dv(g) and the
// next S into the same columns once P^T(g) is there, dk(g) and dP(g+1) once dS^T(g) is.
template <int D>
struct PackedDkv {
  static constexpr int KCH = D / 64;
  static constexpr int TILE = 128 * D * 2;
  static constexpr int SBUF = D == 64 ? 2 : 1;
  static constexpr int KVBUF = D == 64 ? 2 : 1;  // K and V of an item
  static constexpr int QST = D == 64 ? 4 : 2, OST = D == 64 ? 3 : 2;
  static constexpr int SMEM = (KVBUF * 2 + QST + OST) * TILE + QST * 1024 + 1024;
  static constexpr uint32_t T_S = 0, T_DP = 128 * SBUF, T_DV = T_DP + 128, T_DK = T_DV + D;
};

template <int D>
__device__ __forceinline__ void packed_dkv(const BwdMaps& maps, bf16* __restrict__ dk, bf16* __restrict__ dv,
                                           long long dk_stride, long long dv_stride, const float* lse2,
                                           const float* delta, const PackedWork& work, int Hk, int group, long long rows,
                                           float scale, float scale_log2, int accumulate, uint32_t* status, int block,
                                           int blocks) {
  using C = PackedDkv<D>;
  using W = BwdWarps<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[34];
  __shared__ PackedUnit own;  // without a list: the CTA's only unit
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  if (cta_aborted(status, &abort_flag)) {
    wait_prerequisites();
    return;
  }
  uint8_t* smem = align1024(smem_raw);
  uint8_t* sKV = smem;  // buffer b: K, then V
  uint8_t* sQ = sKV + C::KVBUF * 2 * C::TILE;
  uint8_t* sO = sQ + C::QST * C::TILE;
  uint8_t* sStat = sO + C::OST * C::TILE;  // stage s: lse2 and Delta of 128 queries
  auto kv_full = [&](int b) { return smem_u32(&bars[0 + b]); };
  auto kv_empty = [&](int b) { return smem_u32(&bars[2 + b]); };
  auto q_full = [&](int s) { return smem_u32(&bars[4 + s]); };
  auto q_empty = [&](int s) { return smem_u32(&bars[8 + s]); };
  auto o_full = [&](int s) { return smem_u32(&bars[12 + s]); };
  auto o_empty = [&](int s) { return smem_u32(&bars[15 + s]); };
  auto ready = [&](int s) { return smem_u32(&bars[18 + s]); };  // Q and dO of a tile, rows behind the end zero
  // By tile parity: each pair waits for its own tiles only, and an arriving side can be a tile ahead.
  auto s_full = [&](int g) { return smem_u32(&bars[22 + (g & 1)]); };
  auto p_full = [&](int g) { return smem_u32(&bars[24 + (g & 1)]); };
  auto dp_full = [&](int g) { return smem_u32(&bars[26 + (g & 1)]); };
  auto ds_full = [&](int g) { return smem_u32(&bars[28 + (g & 1)]); };
  auto acc_done = [&](int pair) { return smem_u32(&bars[30 + pair]); };  // dv and dk are there, as for dq; were read
  const uint32_t acc_free = smem_u32(&bars[32]);
  const uint32_t mma_done = smem_u32(&bars[33]);  // all products have ended

  const int warp = warp_id();
  if (threadIdx.x == 0) {
    for (int u = 0; u < 2; ++u) {
      mbar_init(kv_full(u), 1);
      mbar_init(kv_empty(u), 1);
      mbar_init(s_full(u), 1);
      mbar_init(p_full(u), W::PAIR);
      mbar_init(dp_full(u), 1);
      mbar_init(ds_full(u), W::PAIR);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(q_full(s), 1);
      mbar_init(q_empty(s), 1);
      mbar_init(ready(s), 1);
    }
    for (int s = 0; s < 3; ++s) {
      mbar_init(o_full(s), 1);
      mbar_init(o_empty(s), 1);
    }
    for (int u = 0; u < 2; ++u) mbar_init(acc_done(u), 1);
    mbar_init(acc_free, W::PAIR);
    mbar_init(mma_done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  wait_prerequisites();
  if (threadIdx.x == 64 && !work.list) own = work.direct(block / Hk);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const long long n_items = work.items(Hk);
  auto unit_of = [&](int turn) {
    const long long i = packed_turn(turn, block, blocks);
    if (!work.list) return turn == 0 ? own : PackedUnit{0, 0, 0, 0};
    return i < n_items ? work.listed(static_cast<int>(i / Hk)) : PackedUnit{0, 0, 0, 0};
  };
  auto head_of = [&](int turn) { return static_cast<int>(packed_turn(turn, block, blocks) % Hk); };
  // Unit of work w: key tile (tiles of the sequence) - w, seen by the w query tiles from its own on.
  auto tiles_of = [](const PackedUnit& u) { return (u.len + 127) / 128; };
  if (warp < W::ROLES) W::roles_regs();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      tma_prefetch_desc(&maps.q);
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
      tma_prefetch_desc(&maps.dO);
      bool ok = true;
      PackedUnit next = unit_of(0);
      int it = 0, g = 0, go = 0;  // items, tiles of Q (with their statistics) and of dO sent for
      while (ok && next.work) {
        const PackedUnit u = next;
        const int kh = head_of(it), first = tiles_of(u) - u.work;
        next = unit_of(it + 1);
        const int b = it % C::KVBUF, k = it / C::KVBUF;
        if (k > 0 && !(ok = mbar_wait(kv_empty(b), (k - 1) & 1, status))) break;
        mbar_arrive_expect_tx(kv_full(b), 2 * C::TILE);
        for (int c = 0; c < C::KCH; ++c) {
          tma_load_3d(smem_u32(sKV + b * 2 * C::TILE + c * kChunk), &maps.k, kv_full(b), c * 64, kh,
                      u.start + first * 128);
          tma_load_3d(smem_u32(sKV + (b * 2 + 1) * C::TILE + c * kChunk), &maps.v, kv_full(b), c * 64, kh,
                      u.start + first * 128);
        }
        ++it;
        for (int h = kh * group; ok && h < (kh + 1) * group; ++h)
          for (int j = first; j < first + u.work; ++j) {
            int s = g % C::QST;
            if (g >= C::QST && !(ok = mbar_wait(q_empty(s), ((g / C::QST) - 1) & 1, status))) break;
            mbar_arrive_expect_tx(q_full(s), C::TILE + 1024);
            for (int c = 0; c < C::KCH; ++c)
              tma_load_3d(smem_u32(sQ + s * C::TILE + c * kChunk), &maps.q, q_full(s), c * 64, h, u.start + j * 128);
            const size_t at = h * static_cast<size_t>(rows) + stat_row(u, j);
            bulk_load(smem_u32(sStat + s * 1024), lse2 + at, 512, q_full(s));
            bulk_load(smem_u32(sStat + s * 1024 + 512), delta + at, 512, q_full(s));
            ++g;
            s = go % C::OST;
            if (go >= C::OST && !(ok = mbar_wait(o_empty(s), ((go / C::OST) - 1) & 1, status))) break;
            mbar_arrive_expect_tx(o_full(s), C::TILE);
            for (int c = 0; c < C::KCH; ++c)
              tma_load_3d(smem_u32(sO + s * C::TILE + c * kChunk), &maps.dO, o_full(s), c * 64, h, u.start + j * 128);
            ++go;
          }
      }
      drain_ring<C::KVBUF>(it, kv_full);
      drain_ring<C::QST>(g, q_full);
      drain_ring<C::OST>(go, o_full);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t idS = make_idesc(128, 128, 1, false, false);
      constexpr uint32_t idG = make_idesc(128, D, 1, false, true);
      const uint64_t dKV0 = make_sdesc(smem_u32(sKV), 16, 1024);
      const uint64_t dQ0 = make_sdesc(smem_u32(sQ), 16, 1024);
      const uint64_t dO0 = make_sdesc(smem_u32(sO), 16, 1024);
      const uint64_t dQ_MN = make_sdesc(smem_u32(sQ), kChunk, 1024);
      const uint64_t dO_MN = make_sdesc(smem_u32(sO), kChunk, 1024);
      auto product = [&](uint32_t to, uint64_t a, uint64_t b) {  // K-major x K-major over D
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k / 4) * kChunk + (k % 4) * 32) >> 4;
          umma_f16_ss(to, a + off, b + off, idS, k > 0 ? 1u : 0u);
        }
      };
      auto add_to = [&](uint32_t to, uint32_t a, uint64_t b, bool fresh) {  // A from TMEM, over 128 queries
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_f16_ts(to, a + step_col(k), b + ((k * 2048) >> 4), idG, (!fresh || k > 0) ? 1u : 0u);
      };
      bool ok = true;
      PackedUnit unit = unit_of(0);
      int turn = 0, left = unit.work * group;
      auto next_tile = [&] {
        StreamTile t = {turn, unit.work > 0, left == unit.work * group, left == 1, false};
        if (t.valid && --left == 0) {
          unit = unit_of(++turn);
          left = unit.work * group;
        }
        return t;
      };
      auto issue_S = [&](const StreamTile& t, int g) {
        const int b = t.it % C::KVBUF;
        if (t.first && !mbar_wait(kv_full(b), (t.it / C::KVBUF) & 1, status)) return false;
        if (!mbar_wait(ready(g % C::QST), (g / C::QST) & 1, status)) return false;
        tc_fence_after();
        product(tmem + C::T_S + (g % C::SBUF) * 128, dKV0 + ((b * 2 * C::TILE) >> 4),
                dQ0 + (((g % C::QST) * C::TILE) >> 4));
        umma_commit(s_full(g));
        return true;
      };
      auto issue_dP = [&](const StreamTile& t, int g) {
        const int b = t.it % C::KVBUF;
        product(tmem + C::T_DP, dKV0 + (((b * 2 + 1) * C::TILE) >> 4), dO0 + (((g % C::OST) * C::TILE) >> 4));
        umma_commit(dp_full(g));
        if (t.last) umma_commit(kv_empty(b));  // (its last S was issued before)
      };
      StreamTile a = next_tile(), b = next_tile();
      if (a.valid && (ok = issue_S(a, 0))) {
        issue_dP(a, 0);
        if (C::SBUF == 2 && b.valid) ok = issue_S(b, 1);
      }
      for (int g = 0; ok && a.valid; ++g) {
        if (!(ok = mbar_wait(p_full(g), (g >> 1) & 1, status))) break;
        // dv and dk restart from zero: the item before has been read
        if (a.first && a.it > 0 && !(ok = mbar_wait(acc_free, (a.it - 1) & 1, status))) break;
        tc_fence_after();
        add_to(tmem + C::T_DV, tmem + C::T_S + (g % C::SBUF) * 128, dO_MN + (((g % C::OST) * C::TILE) >> 4), a.first);
        umma_commit(o_empty(g % C::OST));
        // the next S over P^T(g), in order behind dv(g); with one K / V buffer the first S of an
        // item waits for its keys behind dk(g)
        const StreamTile c = C::SBUF == 2 ? next_tile() : b;
        const bool late = C::KVBUF == 1 && c.first;
        if (c.valid && !late && !(ok = issue_S(c, g + C::SBUF))) break;
        if (!(ok = mbar_wait(ds_full(g), (g >> 1) & 1, status))) break;
        tc_fence_after();
        add_to(tmem + C::T_DK, tmem + C::T_DP, dQ_MN + (((g % C::QST) * C::TILE) >> 4), a.first);
        umma_commit(q_empty(g % C::QST));
        if (a.last) umma_commit(acc_done(W::pair_of(g)));
        if (c.valid && late && !(ok = issue_S(c, g + C::SBUF))) break;
        if (b.valid) issue_dP(b, g + 1);  // (waited for with its S)
        a = b;
        b = C::SBUF == 2 ? c : next_tile();
      }
      drain_products(mma_done);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ rows behind a sequence's end
    // Queries there are zero, with lse = +inf: their P and dS are 0 whatever lies behind the sequence.
    bool ok = true;
    PackedUnit next = unit_of(0);
    int g = 0;
    for (int it = 0; ok && next.work; ++it) {
      const PackedUnit u = next;
      const int n = tiles_of(u), first = n - u.work;
      next = unit_of(it + 1);
      for (int h = 0; ok && h < group; ++h)
        for (int j = first; j < n; ++j, ++g) {
          if (!(ok = mbar_wait_warp(q_full(g % C::QST), (g / C::QST) & 1, status) &&
                     mbar_wait_warp(o_full(g % C::OST), (g / C::OST) & 1, status)))
            break;
          if ((j + 1) * 128 > u.len) {
            zero_rows(sQ + (g % C::QST) * C::TILE, C::KCH, u.len - j * 128);
            zero_rows(sO + (g % C::OST) * C::TILE, C::KCH, u.len - j * 128);
          }
          if (lane_id() == 0) mbar_arrive(ready(g % C::QST));
        }
    }
  } else if (warp >= W::ROLES) {
    // ------------------------------------------------------------ P^T and dS^T
    // A pair takes every other tile, its warpgroup `half` the queries [64 half, 64 half + 64); thread = key row.
    W::pairs_regs();
    const int pair = (warp - W::ROLES) >> 3, half = ((warp - W::ROLES) >> 2) & 1;
    const int r = ((warp & 3) << 5) + static_cast<int>(lane_id());
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tdP = tmem + C::T_DP + lane_base + half * 64;
    bool ok = true;
    PackedUnit next = unit_of(0);
    int g0 = 0, done = 0;  // the item's first tile; items that this pair wrote
    for (int it = 0; ok && next.work; ++it) {
      const PackedUnit u = next;
      next = unit_of(it + 1);
      const int last = g0 + u.work * group - 1;
      int j = (W::first(g0, pair) - g0) % u.work;  // query tile of the head, from the diagonal on
      for (int g = W::first(g0, pair); g <= last; g += W::PAIRS) {
        const uint32_t tS = tmem + C::T_S + (g % C::SBUF) * 128 + lane_base + half * 64;
        const float* lse2s = reinterpret_cast<const float*>(sStat + (g % C::QST) * 1024) + half * 64;
        const float* dels = lse2s + 128;
        if (!(ok = mbar_wait_warp(q_full(g % C::QST), (g / C::QST) & 1, status) &&
                   mbar_wait_warp(s_full(g), (g >> 1) & 1, status)))
          break;
        tc_fence_after();
        float p[64];
        tmem_ld32_sync(tS, *reinterpret_cast<uint32_t(*)[32]>(&p[0]));
        tmem_ld32_sync(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&p[32]));
        const bool diagonal = j == 0;
        j += W::PAIRS;
        if (j >= u.work) j -= u.work;
        if (j >= u.work) j -= u.work;  // (two tiles on in a head of one)
        // Queries before the key. (dS needs no mask of its own: there P is 0 and dP - Delta finite.)
        auto exponentials = [&](auto masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 z = *reinterpret_cast<const float4*>(lse2s + 16 * c + 4 * e);
              float* x = &p[16 * c + 4 * e];
              x[0] = ex2(fmaf(x[0], scale_log2, -z.x));
              x[1] = ex2(fmaf(x[1], scale_log2, -z.y));
              x[2] = ex2(fmaf(x[2], scale_log2, -z.z));
              x[3] = ex2(fmaf(x[3], scale_log2, -z.w));
            }
            if constexpr (decltype(masked)::value) {
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (half * 64 + 16 * c + e < r) p[16 * c + e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) pk[e] = pack_bf16x2(p[16 * c + 2 * e], p[16 * c + 2 * e + 1]);
            PA_TMEM_ST_X8(tS + c * 8, pk);
          }
        };
        if (diagonal) exponentials(std::true_type{});
        else exponentials(std::false_type{});
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full(g));
        if (!(ok = mbar_wait_warp(dp_full(g), (g >> 1) & 1, status))) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 64 / W::CHUNK; ++c) {
          constexpr int N = W::CHUNK;
          uint32_t v[N], pk[N / 2];
          load_columns(tdP + c * N, v);
#pragma unroll
          for (int e = 0; e < N / 4; ++e) {
            const float4 z = *reinterpret_cast<const float4*>(dels + c * N + 4 * e);
            const float x[4] = {__uint_as_float(v[4 * e]) - z.x, __uint_as_float(v[4 * e + 1]) - z.y,
                                __uint_as_float(v[4 * e + 2]) - z.z, __uint_as_float(v[4 * e + 3]) - z.w};
            pk[2 * e] = pack_bf16x2(p[c * N + 4 * e] * x[0], p[c * N + 4 * e + 1] * x[1]);
            pk[2 * e + 1] = pack_bf16x2(p[c * N + 4 * e + 2] * x[2], p[c * N + 4 * e + 3] * x[3]);
          }
          store_columns(tdP + c * (N / 2), pk);  // over columns that have been read
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(ds_full(g));
      }
      if (!ok) break;
      g0 = last + 1;
      if (W::pair_of(last) != pair) continue;
      // Write-back by the pair of the last tile, half 0 dv and half 1 dk, while the other pair begins
      // the next item.
      if (!(ok = mbar_wait_warp(acc_done(pair), done & 1, status))) break;
      ++done;
      tc_fence_after();
      const int row = (tiles_of(u) - u.work) * 128 + r;
      const size_t start = static_cast<size_t>(u.start), col = static_cast<size_t>(head_of(it)) * D;
      const long long stride = half == 0 ? dv_stride : dk_stride;
      bf16* dst = (half == 0 ? dv : dk) + start * stride + col;
      const uint32_t src = tmem + (half == 0 ? C::T_DV : C::T_DK) + lane_base;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32_sync(src + c * 32, o);
        write_row(dst + c * 32, stride, row, u.len, o, half == 0 ? 1.f : scale, accumulate);
      }
      tc_fence_before();
      mbar_arrive(acc_free);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One launch for both: an SM takes a block of dk and dv as soon as its block of dq ends, and each waits for the
// statistics by itself. As two launches, the second waiting for all of the first: 100 tokens of 8 + 2 heads of 64 19.3 us
// on the GPU instead of 13.4; as called 8192 tokens of 16 + 4 heads of 128 878 instead of 842, 12800 tokens of 16
// heads of 64 355 instead of 350.
template <int D>
__global__ void __launch_bounds__(BwdWarps<D>::THREADS, 1)
    packed_bwd_kernel(const __grid_constant__ BwdMaps maps, bf16* __restrict__ dq, bf16* __restrict__ dk,
                      bf16* __restrict__ dv, long long dq_stride, long long dk_stride, long long dv_stride,
                      const float* lse2, const float* delta, const __grid_constant__ PackedWork work, int H, int Hk,
                      long long rows, float scale, float scale_log2, int accumulate, int dq_blocks, uint32_t* status) {
  const int block = static_cast<int>(blockIdx.x);
  if (block < dq_blocks)
    packed_dq<D>(maps, dq, dq_stride, lse2, delta, work, H, H / Hk, rows, scale, scale_log2, accumulate, status, block,
                 dq_blocks);
  else
    packed_dkv<D>(maps, dk, dv, dk_stride, dv_stride, lse2, delta, work, Hk, H / Hk, rows, scale, scale_log2, accumulate,
                  status, block - dq_blocks, static_cast<int>(gridDim.x) - dq_blocks);
}

size_t stat_bytes(const PackedShape& sh) {
  return (static_cast<size_t>(stat_blocks(sh.T, sh.n)) * 128 * sh.H * sizeof(float) + 255) / 256 * 256;
}

template <int D>
int packed_bwd(const PackedShape& sh, const void* q, const void* k, const void* v, const void* o, const void* dO,
               const float* lse, const int32_t* cu, void* dq, void* dk, void* dv, bool accumulate, void* ws,
               uint32_t* status, cudaStream_t s) {
  BwdMaps maps;
  if (!make_packed_map(&maps.q, q, sh.T, sh.H, D, sh.q_stride) ||
      !make_packed_map(&maps.k, k, sh.T, sh.Hk, D, sh.k_stride) ||
      !make_packed_map(&maps.v, v, sh.T, sh.Hk, D, sh.v_stride) ||
      !make_packed_map(&maps.dO, dO, sh.T, sh.H, D, static_cast<long long>(sh.H) * D))
    return PA_ERR_ALIGN;
  constexpr int SMEM = PackedDq<D>::SMEM > PackedDkv<D>::SMEM ? PackedDq<D>::SMEM : PackedDkv<D>::SMEM;
  static std::atomic<uint64_t> attr{0};
  if (!ensure_smem_attr(packed_bwd_kernel<D>, SMEM, attr)) return PA_ERR_LAUNCH;
  uint8_t* w = static_cast<uint8_t*>(ws);
  float* lse2 = reinterpret_cast<float*>(w + packed_list_bytes(sh, 128));
  float* delta = reinterpret_cast<float*>(w + packed_list_bytes(sh, 128) + stat_bytes(sh));
  const long long rows = stat_blocks(sh.T, sh.n) * 128;
  auto grid = [&](long long heads, long long most) {
    const long long items = static_cast<long long>(packed_units(sh, 128)) * heads;
    return static_cast<int>(items < most ? items : most);
  };
  const int sms = device_sm_count();
  PackedWork work;
  int st = packed_work(&work, sh, cu, 128, sh.H, sms, ws, s);
  if (st != PA_OK) return st;
  st = launch_beside(work.list != nullptr, packed_stats_kernel<D>, dim3(grid(sh.H, kStatBlocks * sms)), 256, 0, s,
                     static_cast<const bf16*>(dO), static_cast<const bf16*>(o), lse, work, sh.T, sh.H, rows, lse2, delta);
  if (st != PA_OK) return st;
  const int dq_blocks = grid(sh.H, sms);
  return launch_beside(true, packed_bwd_kernel<D>, dim3(dq_blocks + grid(sh.Hk, sms)), BwdWarps<D>::THREADS, SMEM, s, maps,
                       static_cast<bf16*>(dq), static_cast<bf16*>(dk), static_cast<bf16*>(dv), sh.dq_stride,
                       sh.dk_stride, sh.dv_stride, static_cast<const float*>(lse2), static_cast<const float*>(delta),
                       work, sh.H, sh.Hk, rows, sh.scale, sh.scale * kLog2e, static_cast<int>(accumulate), dq_blocks,
                       status);
}

}  // namespace

size_t packed_attn_bwd_workspace_bytes(const PackedShape& sh) {
  return packed_list_bytes(sh, 128) + 2 * stat_bytes(sh);
}

int launch_packed_attn_bwd(const PackedShape& sh, const void* q, const void* k, const void* v,
                           const void* o, const void* dO, const float* lse, const int32_t* cu,
                           void* dq, void* dk, void* dv, bool accumulate, void* ws,
                           uint32_t* status, cudaStream_t s) {
  return sh.D == 64 ? packed_bwd<64>(sh, q, k, v, o, dO, lse, cu, dq, dk, dv, accumulate, ws, status, s)
                    : packed_bwd<128>(sh, q, k, v, o, dO, lse, cu, dq, dk, dv, accumulate, ws, status, s);
}

}  // namespace pa
