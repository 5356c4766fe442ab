// Causal attention over packed sequences with shared key-value heads, forward,
// for sm_100a: bf16 in, fp32 accumulation in TMEM.
//
//   S = Q K^T scale,  o_i = sum_{j <= i} exp(S_ij - lse_i) v_j
// with one pass over the keys: a row keeps its running maximum m and sum l, and
// O is rescaled where m rises (in the log2 domain, and only by more than 8, as
// fp32 and bf16 hold 2^8 exactly). Only the block on the diagonal is masked; blocks
// behind it are not touched.
//
// Persistent, one CTA per SM: an item is two 128-query tiles that walk the same
// key tiles, either one tile of two heads of a group (an even group: the tiles
// have the same keys and the same length, so nothing is wasted) or two
// neighbouring tiles of one head. Roles:
//   warp 0      TMA producer (Q per item, K/V ring)
//   warp 1      TMEM allocator + tcgen05.mma issuer
//   warp 2      zeroes the rows of V behind a sequence's end: they belong to
//               another sequence or to none, and 0 x NaN would reach O
//   warps 4-7   softmax of tile 0 (thread = one query row), warps 8-11 of tile 1
// The two softmax warpgroups ping-pong so that the tensor core computes one
// tile's S or P V while the other tile's softmax runs. TMEM, d = 64: S0 [0,128)
// S1 [128,256) O0, O1 [256,384) P0, P1 [384,512); d = 128: O takes 128 columns
// each and P is written over its own S.
//
// Measured, against 1618 TFLOP/s of a large matrix product (1344 under the power cap): 16384 tokens, 16 + 4 heads of
// 128, 925 us (1188 TFLOP/s of the pairs under the mask); 22764 tokens in 16 sequences of all lengths, 16 + 2 heads
// of 128, 251 us (925). Bound by a tile's chain: softmax 1850 clocks, then P V and the next S 1140 and some 450
// from a product's issue to its barrier, with two tiles in turn and no TMEM for a third; the exponentials and
// the tensor core are each busy for half of it. Handing P over in two to four parts, so that P V starts under the
// exponentials, was not faster (both sides 251, and 925 to 928). Ragged sequences add the masked halves of the
// diagonal tiles (7%) and the ends of some 10 items a CTA. Heads of 64: 12800 tokens in 8 sequences, 16 heads, 128 us (574
// TFLOP/s), 16384 tokens of 16 + 4 heads 716 us (768): the exponentials are the same for half of the products.
#include <type_traits>
#include "packed_common.cuh"

namespace pa {
namespace {

using bf16 = __nv_bfloat16;

// ---------------------------------------------------------------- the list of work
constexpr int kListThreads = 1024, kListBins = 2048;

__device__ __forceinline__ int units_of(int len, int unit) { return (len + unit - 1) / unit; }

// Inclusive prefix maximum (or sum) over the block's threads.
template <bool MAX>
__device__ int block_scan(int v, int* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v = MAX ? max(v, o) : v + o;
  }
  if (lane == 31) warps[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = warps[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w = MAX ? max(w, o) : w + o;
    }
    warps[lane] = w;
  }
  __syncthreads();
  if (warp > 0) v = MAX ? max(v, warps[warp - 1]) : v + warps[warp - 1];
  __syncthreads();
  return v;
}

// One block: sequences from cu (their starts a running maximum, clamped to the
// tokens), a histogram of the units' work, and the units in descending order.
__global__ void __launch_bounds__(kListThreads)
    packed_list_kernel(const int32_t* __restrict__ cu, int n, int T, int unit, int most, PackedList* list) {
  __shared__ int bins[kListBins], warps[32], longest;
  launch_dependents();
  int4* out = reinterpret_cast<int4*>(list + 1);
  int2* seqs = reinterpret_cast<int2*>(out + most);  // start, length
  const int tid = threadIdx.x;
  if (tid == 0) longest = 0;
  for (int b = tid; b < kListBins; b += kListThreads) bins[b] = 0;
  __syncthreads();
  // a thread takes a run of sequences; starts before its run are the maximum of the runs before
  const int per = (n + kListThreads - 1) / kListThreads, lo = min(n, tid * per), hi = min(n, lo + per);
  int m = 0;
  for (int i = lo; i < hi; ++i) m = max(m, min(max(cu[i], 0), T));
  int before = block_scan<true>(m, warps);
  before = __shfl_up_sync(0xffffffffu, before, 1);
  if ((tid & 31) == 0) before = tid ? warps[(tid >> 5) - 1] : 0;
  int top = 0;
  for (int i = lo; i < hi; ++i) {
    const int len = packed_seq(cu, i, T, before);
    seqs[i] = make_int2(before, len);
    top = max(top, units_of(len, unit));
  }
  atomicMax(&longest, top);
  __syncthreads();
  int shift = 0;
  while ((longest >> shift) >= kListBins) ++shift;
  const int lane = tid & 31;
  for (int i = tid >> 5; i < n; i += kListThreads / 32)
    for (int w = 1 + lane; w <= units_of(seqs[i].y, unit); w += 32) atomicAdd(&bins[w >> shift], 1);
  __syncthreads();
  // entries before those of bin b: all of larger work
  int mine[kListBins / kListThreads], sum = 0;
#pragma unroll
  for (int k = 0; k < kListBins / kListThreads; ++k) {
    mine[k] = sum;
    sum += bins[kListBins - 1 - (tid * (kListBins / kListThreads) + k)];
  }
  const int upto = block_scan<false>(sum, warps);
#pragma unroll
  for (int k = 0; k < kListBins / kListThreads; ++k)
    bins[kListBins - 1 - (tid * (kListBins / kListThreads) + k)] = upto - sum + mine[k];
  if (tid == kListThreads - 1) list->count = min(upto, most);
  __syncthreads();
  for (int i = tid >> 5; i < n; i += kListThreads / 32) {
    const int2 s = seqs[i];
    for (int w = 1 + lane; w <= units_of(s.y, unit); w += 32) {
      const int at = atomicAdd(&bins[w >> shift], 1);
      if (at < most) out[at] = make_int4(s.x, s.y, w, i);
    }
  }
}

// ---------------------------------------------------------------- forward
template <int D>
struct PackedFwd {
  static constexpr int KCH = D / 64;  // 128-byte column chunks of a row
  static constexpr int STAGES = D == 64 ? 3 : 2;
  static constexpr int CHUNK = 128 * 128;  // bytes of one 128-row x 128-byte box
  static constexpr int TILE = 128 * D * 2;
  static constexpr int Q_ITEM = 2 * TILE;
  static constexpr int KV_RING = STAGES * 2 * TILE;
  static constexpr int QBUF = 2 * Q_ITEM + KV_RING + 1024 <= 227 * 1024 ? 2 : 1;
  static constexpr int SMEM = QBUF * Q_ITEM + KV_RING + 1024;
  static constexpr int THREADS = 384;
  // Registers of a thread: a softmax thread holds a row of S (128 values), and the first four warps give
  // theirs; the shares add up to the 384 x 168 of the launch.
  static constexpr int FEW = 88, MANY = 208;
  static_assert((FEW + 2 * MANY) * 128 <= THREADS * 168, "an increase would wait forever");
  static constexpr bool SEP_P = D == 64;  // P in its own TMEM columns
  static constexpr uint32_t T_S = 0, T_O = 256;
  static constexpr uint32_t T_P = SEP_P ? 384 : 0;
};

// What an item's two tiles are.
struct PackedItem {
  int start, len;
  int head[2], row[2];  // head of q; first query row within the sequence
  int n[2], n_kv;       // key tiles of each (0: no such tile), of both
  int kv_head;
  bool ragged;          // the last key tile passes the sequence's end
};
__device__ __forceinline__ PackedItem packed_item(const PackedUnit& u, int hh, bool pair_heads, int group) {
  PackedItem it;
  it.start = u.start;
  it.len = u.len;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    it.head[t] = pair_heads ? 2 * hh + t : hh;
    const int tile = pair_heads ? u.work - 1 : 2 * (u.work - 1) + t;
    it.row[t] = tile * 128;
    it.n[t] = it.row[t] < u.len ? tile + 1 : 0;
  }
  it.n_kv = max(it.n[0], it.n[1]);
  it.kv_head = it.head[0] / group;
  it.ragged = it.n_kv * 128 > u.len;
  return it;
}

template <int D>
__global__ void __launch_bounds__(384, 1)
    packed_fwd_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK,
                      const __grid_constant__ CUtensorMap mapV, bf16* __restrict__ O, float* __restrict__ lse,
                      const __grid_constant__ PackedWork work, int T, int H, int group, int pair_heads,
                      float scale_log2, uint32_t* status) {
  using C = PackedFwd<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[23];
  __shared__ PackedUnit own;  // without a list: the CTA's only unit
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  if (cta_aborted(status, &abort_flag)) {
    wait_prerequisites();
    return;
  }

  uint8_t* smem = align1024(smem_raw);
  uint8_t* sQ = smem;  // tile t of Q buffer u at sQ + u * Q_ITEM + t * TILE
  uint8_t* sK = smem + C::QBUF * C::Q_ITEM;
  uint8_t* sV = sK + C::STAGES * C::TILE;

  auto q_full = [&](int u) { return smem_u32(&bars[0 + u]); };
  auto q_empty = [&](int u) { return smem_u32(&bars[2 + u]); };
  auto kv_full = [&](int s) { return smem_u32(&bars[4 + s]); };
  auto kv_empty = [&](int s) { return smem_u32(&bars[7 + s]); };
  auto s_full = [&](int t) { return smem_u32(&bars[10 + t]); };
  auto p_full = [&](int t) { return smem_u32(&bars[12 + t]); };
  auto o_done = [&](int t) { return smem_u32(&bars[14 + t]); };
  auto s_free = [&](int t) { return smem_u32(&bars[16 + t]); };
  auto pv_done = [&](int t) { return smem_u32(&bars[18 + t]); };
  const uint32_t v_ragged = smem_u32(&bars[20]);  // a ragged V tile has landed
  const uint32_t v_zeroed = smem_u32(&bars[21]);  // and its rows behind the end are zero
  const uint32_t mma_done = smem_u32(&bars[22]);  // all products have ended

  const int warp = warp_id();
  if (threadIdx.x == 0) {
    for (int u = 0; u < C::QBUF; ++u) {
      mbar_init(q_full(u), 1);
      mbar_init(q_empty(u), 1);
    }
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t), 128);
      mbar_init(o_done(t), 1);
      mbar_init(s_free(t), 128);
      mbar_init(pv_done(t), 1);
    }
    mbar_init(v_ragged, 1);
    mbar_init(v_zeroed, 1);
    mbar_init(mma_done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  const int n_hh = pair_heads ? H / 2 : H;
  wait_prerequisites();  // the list
  if (threadIdx.x == 64 && !work.list) own = work.direct(static_cast<int>(blockIdx.x) / n_hh);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const long long n_items = work.items(n_hh);
  const int block = static_cast<int>(blockIdx.x), blocks = static_cast<int>(gridDim.x);
  // Items in turn; the next one's unit is fetched while the current one runs.
  auto unit_of = [&](int turn) {
    const long long i = packed_turn(turn, block, blocks);
    if (!work.list) return turn == 0 ? own : PackedUnit{0, 0, 0, 0};
    return i < n_items ? work.listed(static_cast<int>(i / n_hh)) : PackedUnit{0, 0, 0, 0};
  };
  auto item_of = [&](int turn, const PackedUnit& u) {
    return packed_item(u, static_cast<int>(packed_turn(turn, block, blocks) % n_hh), pair_heads, group);
  };

  // Counters that run over all items: it, items; g, key tiles (ring slot and its
  // phase); gt, key tiles of query tile t; f, ragged tiles.
  if (warp < 4) regs_dec<C::FEW>();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      tma_prefetch_desc(&mapQ);
      tma_prefetch_desc(&mapK);
      tma_prefetch_desc(&mapV);
      bool ok = true;
      PackedUnit unit = unit_of(0);
      int it = 0, g = 0;  // items, key tiles sent for
      while (ok && unit.work) {
        const PackedItem w = item_of(it, unit);
        unit = unit_of(it + 1);
        const int u = it % C::QBUF, k = it / C::QBUF;
        if (k > 0 && !(ok = mbar_wait(q_empty(u), (k - 1) & 1, status))) break;
        mbar_arrive_expect_tx(q_full(u), (w.n[1] ? 2 : 1) * C::TILE);
        for (int t = 0; t < 2; ++t)
          if (w.n[t])
            for (int c = 0; c < C::KCH; ++c)
              tma_load_3d(smem_u32(sQ + u * C::Q_ITEM + t * C::TILE + c * C::CHUNK), &mapQ, q_full(u), c * 64,
                          w.head[t], w.start + w.row[t]);
        ++it;
        for (int j = 0; j < w.n_kv; ++j, ++g) {
          const int s = g % C::STAGES;
          if (g >= C::STAGES && !(ok = mbar_wait(kv_empty(s), ((g / C::STAGES) - 1) & 1, status))) break;
          mbar_arrive_expect_tx(kv_full(s), 2 * C::TILE);
          for (int c = 0; c < C::KCH; ++c) {
            tma_load_3d(smem_u32(sK + s * C::TILE + c * C::CHUNK), &mapK, kv_full(s), c * 64, w.kv_head,
                        w.start + j * 128);
            tma_load_3d(smem_u32(sV + s * C::TILE + c * C::CHUNK), &mapV, kv_full(s), c * 64, w.kv_head,
                        w.start + j * 128);
          }
        }
      }
      drain_ring<C::QBUF>(it, q_full);
      drain_ring<C::STAGES>(g, kv_full);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t idS = make_idesc(128, 128, 1, false, false);
      constexpr uint32_t idO = make_idesc(128, D, 1, false, true);
      const uint64_t dQ0 = make_sdesc(smem_u32(sQ), 16, 1024);
      const uint64_t dK0 = make_sdesc(smem_u32(sK), 16, 1024);
      const uint64_t dV0 = make_sdesc(smem_u32(sV), C::CHUNK, 1024);
      auto issue_S = [&](int t, int u, int g) {
        const uint64_t qd = dQ0 + ((u * C::Q_ITEM + t * C::TILE) >> 4);
        const uint64_t kd = dK0 + (((g % C::STAGES) * C::TILE) >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k / 4) * C::CHUNK + (k % 4) * 32) >> 4;
          umma_f16_ss(tmem + C::T_S + t * 128, qd + off, kd + off, idS, k > 0 ? 1u : 0u);
        }
      };
      auto issue_PV = [&](int t, int g, int j) {  // j == 0 starts O from zero
        const uint32_t tp = C::SEP_P ? (tmem + C::T_P + t * 64) : (tmem + C::T_S + t * 128);
        const uint64_t vd = dV0 + (((g % C::STAGES) * C::TILE) >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_f16_ts(tmem + C::T_O + t * D, tp + k * 8, vd + ((k * 2048) >> 4), idO, (j > 0 || k > 0) ? 1u : 0u);
      };
      bool ok = true;
      PackedUnit unit = unit_of(0);
      int g = 0, gt[2] = {0, 0}, f = 0;
      for (int it = 0; ok && unit.work; ++it) {
        const PackedItem w = item_of(it, unit);
        unit = unit_of(it + 1);
        const int u = it % C::QBUF;
        ok = mbar_wait(q_full(u), (it / C::QBUF) & 1, status) &&
             mbar_wait(kv_full(g % C::STAGES), (g / C::STAGES) & 1, status);
        if (!ok) break;
        if (w.ragged && w.n_kv == 1) mbar_arrive(v_ragged);
        // S of the first key tile. Separate P: S's columns are free once the softmax has
        // loaded the previous S. P over S: the P V that reads them was issued before (in order).
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!w.n[t]) continue;
          if (C::SEP_P && gt[t] > 0 && !(ok = mbar_wait(s_free(t), (gt[t] - 1) & 1, status))) break;
          tc_fence_after();
          issue_S(t, u, g);
          umma_commit(s_full(t));
        }
        if (!ok) break;
        if (w.n_kv == 1) umma_commit(q_empty(u));
        for (int j = 0; ok && j < w.n_kv; ++j, ++g) {
          const bool any_more = j + 1 < w.n_kv;
          if (any_more && !(ok = mbar_wait(kv_full((g + 1) % C::STAGES), ((g + 1) / C::STAGES) & 1, status))) break;
          if (w.ragged && j + 2 == w.n_kv) mbar_arrive(v_ragged);
          if (w.ragged && !any_more && !(ok = mbar_wait(v_zeroed, f++ & 1, status))) break;
          // P V of the first tile starts O from zero: its p_full is arrived only after the softmax
          // has read the previous item's O, so O is free then.
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >= w.n[t]) continue;
            const bool more = j + 1 < w.n[t];
            if (C::SEP_P) {
              if (more) {  // next S first (its columns were released by s_free), then P V
                if (!(ok = mbar_wait(s_free(t), gt[t] & 1, status))) break;
                tc_fence_after();
                issue_S(t, u, g + 1);
                umma_commit(s_full(t));
              }
              if (!(ok = mbar_wait(p_full(t), gt[t] & 1, status))) break;
              tc_fence_after();
              issue_PV(t, g, j);
              umma_commit(pv_done(t));
            } else {  // P lives in S's columns: P V first, then the next S overwrites them
              if (!(ok = mbar_wait(p_full(t), gt[t] & 1, status))) break;
              tc_fence_after();
              issue_PV(t, g, j);
              umma_commit(pv_done(t));
              if (more) {
                issue_S(t, u, g + 1);
                umma_commit(s_full(t));
              }
            }
            if (!more) umma_commit(o_done(t));
            ++gt[t];
          }
          if (!ok) break;
          umma_commit(kv_empty(g % C::STAGES));
          if (j + 2 == w.n_kv) umma_commit(q_empty(u));  // the item's last S products are issued
        }
      }
      drain_products(mma_done);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ rows behind a sequence's end
    PackedUnit unit = unit_of(0);
    int g = 0, f = 0;
    for (int it = 0; unit.work; ++it) {
      const PackedItem w = item_of(it, unit);
      unit = unit_of(it + 1);
      g += w.n_kv;
      if (!w.ragged) continue;
      if (!mbar_wait_warp(v_ragged, f++ & 1, status)) break;
      zero_rows(sV + ((g - 1) % C::STAGES) * C::TILE, C::KCH, w.len - (w.n_kv - 1) * 128);
      if (lane_id() == 0) mbar_arrive(v_zeroed);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax
    regs_inc<C::MANY>();
    const int t = (warp - 4) / 4;               // query tile of this warpgroup
    const int r = threadIdx.x - 128 * (t + 1);  // row within the tile == TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + C::T_S + t * 128 + lane_base;
    const uint32_t tO = tmem + C::T_O + t * D + lane_base;
    const uint32_t tP = C::SEP_P ? (tmem + C::T_P + t * 64 + lane_base) : tS;
    bool ok = true;
    PackedUnit unit = unit_of(0);
    int gt = 0, done = 0;
    for (int it = 0; ok && unit.work; ++it) {
      const PackedItem w = item_of(it, unit);
      unit = unit_of(it + 1);
      const int n = t ? w.n[1] : w.n[0];
      if (!n) continue;
      float m = -INFINITY;  // running max of S * scale * log2(e)
      float l = 0.f;        // running row sum (relative to m)
      for (int j = 0; j < n; ++j, ++gt) {
        if (!(ok = mbar_wait_warp(s_full(t), gt & 1, status))) break;
        tc_fence_after();
        float s[128];
        tmem_ld128_sync(tS, reinterpret_cast<uint32_t(&)[128]>(s));
        if (C::SEP_P) {
          tc_fence_before();
          mbar_arrive(s_free(t));  // S may now be overwritten by the next tile's product
        }
        if (j == n - 1) {  // the block on the diagonal
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i > r) s[i] = -INFINITY;
        }
        // row max over eight independent chains of three-input max
        float mk[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mk[k] = fmaxf(s[k], s[8 + k]);
#pragma unroll
        for (int i = 16; i < 128; i += 16)
#pragma unroll
          for (int k = 0; k < 8; ++k) mk[k] = max3f(mk[k], s[i + k], s[i + 8 + k]);
        const float mx = max3f(max3f(mk[0], mk[1], mk[2]), max3f(mk[3], mk[4], mk[5]), fmaxf(mk[6], mk[7]));
        const float m_new = fmaxf(m, mx * scale_log2);
        const bool need = m_new > m + 8.f;
        const bool warp_need = __any_sync(0xffffffffu, need);
        const float alpha = need ? ex2(m - m_new) : 1.f;
        if (need) {
          l *= alpha;
          m = m_new;
        }
        // P of the previous tile and O are read / accumulated by its P V product
        if (C::SEP_P && gt > 0) {
          if (!(ok = mbar_wait_warp(pv_done(t), (gt - 1) & 1, status))) break;
          tc_fence_after();
        }
        const float neg_m = m == -INFINITY ? 0.f : -m;  // no key so far: P is 0, not exp(-inf + inf)
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p0 = ex2(fmaf(s[c * 16 + 2 * i], scale_log2, neg_m));
            const float p1 = ex2(fmaf(s[c * 16 + 2 * i + 1], scale_log2, neg_m));
            sum += p0 + p1;
            pk[i] = pack_bf16x2(p0, p1);
          }
          PA_TMEM_ST_X8(tP + c * 8, pk);
        }
        l += sum;
        if (warp_need && j > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32_sync(tO + c * 32, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + c * 32, o);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full(t));
      }
      // O write-back. The TMEM loads complete before this warpgroup's next p_full
      // arrive, which the next item's first P V waits for.
      if (!ok || !(ok = mbar_wait_warp(o_done(t), done & 1, status))) break;
      ++done;
      tc_fence_after();
      const int row = (t ? w.row[1] : w.row[0]) + r, head = t ? w.head[1] : w.head[0];
      const bool live = row < w.len;
      const float inv_l = l == 0.f ? 0.f : 1.f / l;  // (0: all its scores are -infinity)
      const size_t token = static_cast<size_t>(w.start) + row;
      bf16* oquad = O + ((token - (r & 3)) * H + head) * D;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        uint4 u[4];
        tmem_ld32_sync(tO + c * 32, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w4[e] = pack_bf16x2(__uint_as_float(o[8 * i + 2 * e]) * inv_l, __uint_as_float(o[8 * i + 2 * e + 1]) * inv_l);
          u[i] = make_uint4(w4[0], w4[1], w4[2], w4[3]);
        }
        store_rows(oquad + c * 32, static_cast<long long>(H) * D, w.len - (row & ~3), u);
      }
      if (live) lse[static_cast<size_t>(head) * T + token] = (m + __log2f(l)) * kLn2;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
int packed_fwd(const PackedShape& sh, const void* q, const void* k, const void* v, const int32_t* cu, void* o,
               float* lse, void* ws, uint32_t* status, cudaStream_t s) {
  using C = PackedFwd<D>;
  CUtensorMap mq, mk, mv;
  if (!make_packed_map(&mq, q, sh.T, sh.H, D, sh.q_stride) || !make_packed_map(&mk, k, sh.T, sh.Hk, D, sh.k_stride) ||
      !make_packed_map(&mv, v, sh.T, sh.Hk, D, sh.v_stride))
    return PA_ERR_ALIGN;
  static std::atomic<uint64_t> attr{0};
  if (!ensure_smem_attr(packed_fwd_kernel<D>, C::SMEM, attr)) return PA_ERR_LAUNCH;
  const int group = sh.H / sh.Hk;
  const bool pair_heads = group % 2 == 0;
  const int unit = pair_heads ? 128 : 256, heads = pair_heads ? sh.H / 2 : sh.H;
  const size_t items = packed_units(sh, unit) * heads, sms = device_sm_count();
  PackedWork work;
  const int st = packed_work(&work, sh, cu, unit, heads, static_cast<int>(sms), ws, s);
  if (st != PA_OK) return st;
  const dim3 grid(static_cast<unsigned>(items < sms ? items : sms));
  return launch_beside(work.list != nullptr, packed_fwd_kernel<D>, grid, C::THREADS, C::SMEM, s, mq, mk, mv,
                       static_cast<bf16*>(o), lse, work, sh.T, sh.H, group, static_cast<int>(pair_heads),
                       sh.scale * kLog2e, status);
}

}  // namespace

int launch_packed_list(const PackedShape& sh, const int32_t* cu, int unit, void* list, cudaStream_t s) {
  packed_list_kernel<<<1, kListThreads, 0, s>>>(cu, sh.n, sh.T, unit, static_cast<int>(packed_units(sh, unit)),
                                                static_cast<PackedList*>(list));
  return cudaGetLastError() == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

size_t packed_attn_fwd_workspace_bytes(const PackedShape& sh) { return packed_list_bytes(sh, 128); }

int launch_packed_attn_fwd(const PackedShape& sh, const void* q, const void* k, const void* v,
                           const int32_t* cu, void* o, float* lse, void* ws, uint32_t* status,
                           cudaStream_t s) {
  return sh.D == 64 ? packed_fwd<64>(sh, q, k, v, cu, o, lse, ws, status, s)
                    : packed_fwd<128>(sh, q, k, v, cu, o, lse, ws, status, s);
}

}  // namespace pa
