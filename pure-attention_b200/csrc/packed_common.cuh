// What the kernels of packed causal attention share: the list of their work and
// the maps of their tensors.
//
// A sequence of n tokens has ceil(n / unit) units of `unit` tokens (128 or 256,
// counted from its own start). A causal unit's work grows with its place: unit i
// of queries sees keys up to its own end, unit i of keys is seen by queries from
// its own start. The list holds each sequence's units as (sequence, work), work =
// 1 .. units, most work first, and a persistent kernel deals it out in turns
// (snake): every CTA then ends within one unit's work of the others, with no
// counter shared between CTAs. (Units of equal work may change places from run to run; no result depends on it.)
// Where the units cannot be more than the SMs, a CTA takes one at most and finds it from the lengths by itself:
// a launch less (a prompt of 100 tokens: 10.7 to 7.0 us on the GPU, 6.5 to 3.8 of host time).
#pragma once
#include "host_launchers.h"

namespace pa {

// An entry: first token, length of the sequence, work (1 .. units of the sequence), sequence.
struct PackedUnit {
  int start, len, work, seq;
};
struct PackedList {
  int count;  // entries
  int pad[63];
  // PackedUnit units[packed_units(...)], then scratch
};
// Most units that sequences of T tokens can have: each has less than one that is not full.
inline size_t packed_units(const PackedShape& sh, int unit) { return static_cast<size_t>(sh.T) / unit + sh.n; }
inline size_t packed_list_bytes(const PackedShape& sh, int unit) {
  return (sizeof(PackedList) + 16 * packed_units(sh, unit) + 8 * static_cast<size_t>(sh.n) + 255) / 256 * 256;
}
// packed_attn.cu: writes the list into `list` (packed_list_bytes); the kernel after it may start beside it.
int launch_packed_list(const PackedShape& sh, const int32_t* cu, int unit, void* list, cudaStream_t s);

// Sequence i of the tokens: starts are a running maximum, clamped to the tokens. `before` is the start of the
// sequence before it (0 at first), and its own afterwards.
__device__ __forceinline__ int packed_seq(const int32_t* cu, int i, int T, int& before) {
  before = max(before, min(max(__ldcg(cu + i), 0), T));
  return max(before, min(__ldcg(cu + i + 1), T)) - before;
}

// Where a kernel has its units from: the list, or (NULL) the lengths, which every kernel then walks by itself. Sequences of
// 10 tokens, 2 + 1 heads of 64, us on the GPU without and with the list: 4 of them 7.7 and 9.6 forward, 11.4 and 14.6
// gradients; 8 8.4 and 9.8, 13.1 and 14.7; 16 10.0 and 9.9, 16.5 and 14.6; 32 13.5 and 10.2, 23.1 and 15.4. So the list
// pays from 16 on forward, and for gradients a few sequences sooner.
constexpr int kDirectSeqs = 16;
struct PackedWork {
  const PackedList* list;
  const int32_t* cu;
  int n, T, unit;

  // Items of `heads` heads a unit in the list.
  __device__ __forceinline__ long long items(int heads) const {
    return list ? static_cast<long long>(load_written(&list->count)) * heads : 0;
  }
  __device__ __forceinline__ PackedUnit listed(int i) const {
    const int4 u = load_written(reinterpret_cast<const int4*>(list + 1) + i);
    return {u.x, u.y, u.z, u.w};
  }
  __device__ __forceinline__ PackedUnit direct(int i) const {
    int start = 0;
    for (int s = 0; s < n; ++s) {
      const int len = packed_seq(cu, s, T, start), units = (len + unit - 1) / unit;
      if (i < units) return {start, len, i + 1, s};
      i -= units;
    }
    return {0, 0, 0, 0};
  }
};
// The work of a call whose kernels have at most `heads` items a unit; launches the list where there is one.
inline int packed_work(PackedWork* w, const PackedShape& sh, const int32_t* cu, int unit, int heads, int sms, void* ws,
                       cudaStream_t s) {
  const bool direct = sh.n <= kDirectSeqs && packed_units(sh, unit) * heads <= static_cast<size_t>(sms);
  *w = {direct ? nullptr : static_cast<const PackedList*>(ws), cu, sh.n, sh.T, unit};
  return direct ? PA_OK : launch_packed_list(sh, cu, unit, ws, s);
}
// Item of a CTA's turn, CTA `block` of the `blocks` that share the work out.
__device__ __forceinline__ long long packed_turn(int turn, int block, int blocks) {
  return static_cast<long long>(turn) * blocks + ((turn & 1) ? blocks - 1 - block : block);
}

// 3-D TMA map over [T, H, D] bf16 with `stride` values from token to token: box of 64 columns x 1
// head x 128 tokens, 128-byte swizzle. Tokens past T read as zero.
inline bool make_packed_map(CUtensorMap* m, const void* base, int T, int H, int D, long long stride) {
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(H), static_cast<uint64_t>(T)};
  const uint64_t strides[2] = {static_cast<uint64_t>(D) * 2, static_cast<uint64_t>(stride) * 2};
  const uint32_t box[3] = {64, 1, 128};
  return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Launches `kernel`; beside: so that it may start beside the kernel before it in the stream
// (it waits for that one's results where it needs them).
template <typename K, typename... A>
int launch_beside(bool beside, K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = beside ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

// Waits for the copies of a ring of SLOTS buffers that may still be on their way when `sent` fills were sent
// for: the last SLOTS of them, and none that was not. full(slot) is the barrier of a slot. A block does so whatever
// was recorded: a failure, in it or in another block and at any moment, lets the roles that would have waited leave.
template <int SLOTS, typename F>
__device__ __forceinline__ void drain_ring(int sent, F full) {
  for (int i = max(0, sent - SLOTS); i < sent; ++i) mbar_drain(full(i % SLOTS), (i / SLOTS) & 1);
}

// The same for the tensor products of the issuing thread, which read shared memory and write TMEM that the block
// gives up at its end: `done` is a barrier for this alone.
__device__ __forceinline__ void drain_products(uint32_t done) {
  umma_commit(done);
  mbar_drain(done, 0);
}

// Stores 32 columns of bf16 of a warp's 32 consecutive rows, a lane's row as four 16-byte pieces in u.
// The lanes of a quad exchange pieces first, so that a store covers 64 bytes of 8 rows and not 16
// of 32: the write-back of an item is bound by the lines that its stores touch. to: the columns in the
// quad's first row; rows: rows that exist from there on. All lanes of the warp take part.
__device__ __forceinline__ void store_rows(__nv_bfloat16* to, long long stride, int rows, uint4 (&u)[4]) {
  const int q = static_cast<int>(lane_id() & 3);
#pragma unroll
  for (int b = 1; b < 4; b <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j & b) continue;
      const bool up = q & b;
      uint4 v = up ? u[j] : u[j | b];
      v.x = __shfl_xor_sync(0xffffffffu, v.x, b);
      v.y = __shfl_xor_sync(0xffffffffu, v.y, b);
      v.z = __shfl_xor_sync(0xffffffffu, v.z, b);
      v.w = __shfl_xor_sync(0xffffffffu, v.w, b);
      if (up) u[j] = v;
      else u[j | b] = v;
    }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < rows) *reinterpret_cast<uint4*>(to + j * stride + q * 8) = u[j];
}

// Zeroes rows [from, 128) of a swizzled tile of `chunks` 128-row x 128-byte boxes (one warp), and
// orders the zeros before the tensor core's reads.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int chunks, int from) {
  for (int c = 0; c < chunks; ++c)
    for (int i = from * 8 + static_cast<int>(lane_id()); i < 128 * 8; i += 32)
      *reinterpret_cast<uint4*>(tile + c * 16384 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace pa
