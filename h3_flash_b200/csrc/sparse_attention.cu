// Block-sparse attention for B200 (sm_100a): every block of query rows attends to its own
// list of key blocks. tcgen05 MMA with TMEM accumulators, TMA-fed operands, fp32 online
// softmax.
//
//   out[r] = sum_{j in list} sum_{c in block j} p_rc v_c / sum p_rc,
//   p_rc = 2^(scale log2(e) q_r . k_c - m_r),   lse[r] = ln(2) (m_r + log2(sum p_rc))
//
// The unit of work along a list is 64 keys: a listed block of 64, or half of one of 128. A
// work item is a pair of neighbouring 128-row query tiles of one (batch, head), or a range
// of units of such a pair; where the queries are one tile (a few rows against a long list)
// the two tiles of an item are that tile with two ranges of its list. The grid has a CTA per
// item, but a CTA that nears its item's end takes over the next one that has not started
// (cluster launch control), and its loads start while the one before ends: lists and padded
// batches are uneven, and items that are dealt out beforehand leave SMs idle (a batch of 4097,
// 0, 3700 and 2900 rows with lists of 0 to 12 blocks: 33 us dealt out, 26.5 us taken over).
//
//   warp 8      loads: what an item is, read from global memory and handed to the other warps
//               through shared memory; its Q tiles; then a ring of slots. Slot u of a tile holds
//               V of unit u and K of unit u + 2, which the tile's MMA warp reads one after
//               the other (a first slot holds K of units 0 and 1). Where the tiles of a pair
//               have one list (block_q = 256) one slot serves both; with lists of their own
//               slots of tile 0 and tile 1 alternate.
//   warps 9, 10 MMA issuers of tile 0 and 1, one elected lane each: O_t += P_t(u) V(u), then
//               S_t(u + 2) = Q_t K(u + 2)^T into the TMEM columns P_t(u) came from. The
//               tensor core takes only an MMA or two ahead, so issuing a unit lasts as long
//               as its MMAs (about 690 clocks) and the waits before it (about 420) would
//               leave it idle: with a warp per tile the other's MMAs fill them.
//   warps 0-3   softmax of tile 0, warps 4-7 of tile 1, a thread per row: scores from TMEM,
//               row max, p, row sum; P goes back over the S columns; O is rescaled in TMEM
//               only when the running max grew by more than 2^8. P is rounded to the type
//               of V (the MMA's operand type); sums, max and O stay fp32.
//
// Why 64 keys: scores of a tile are double-buffered, two units of 64 fp32 columns beside
// O, so the softmax of unit u + 1 has its scores while P V of unit u and the scores of u + 2
// are computed; with units of 128 keys TMEM holds one buffer, and each tile's softmax and
// MMAs wait for one another. The price is that an N = 64 score MMA reads its Q operand from
// shared memory for half as many columns. Measured on 592 pairs of tiles, 64 blocks a list,
// under the power cap: 590 us with one list per pair and 640 us with a list per tile, against
// 678 and 694 us with units of 128 keys (before the steps noted below, now 538 and 581 us).
//
// TMEM (512 columns): S of tile t, buffer b at 128 t + 64 b; O of tile t at 256 + 128 t.
//
// What does not exist is never read into a result: list entries outside the sequence load
// zeros (a TMA box behind the end of the tensor), and their scores are replaced by -inf.
// Keys behind k_lens inside a block may hold NaN: their scores are replaced, and their V rows
// are overwritten with zeros in shared memory before the tensor core sees them (0 * NaN is
// NaN).
//
// Every mbarrier wait is bounded; on expiry the status word gets kStatusAttentionTimeout,
// the CTA's abort flag is raised and all roles unwind, free TMEM and return.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>

#include "attention_ptx.cuh"
#include "common.cuh"

namespace h3b {
namespace attn {
namespace sparse {

constexpr int kTile = 128;  // query rows per tile
constexpr int kUnit = 64;   // keys per unit
constexpr int kTiles = 2;
constexpr int kSoftmaxWarps = 4 * kTiles;
constexpr int kThreads = (kSoftmaxWarps + 1 + kTiles) * 32;
constexpr int kLoadWarp = kSoftmaxWarps;
constexpr int kMmaWarp = kSoftmaxWarps + 1;  // + tile
constexpr uint32_t kQHalf = kTile * 128;   // 128 rows x 64 columns, 128-byte swizzle
constexpr uint32_t kKvHalf = kUnit * 128;  // 64 rows x 64 columns
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemS = 0;    // + t*128 + buffer*64
constexpr uint32_t kTmemO = 256;  // + t*128
// Rescale O only when the running row max (log2 units) grew by more than this; P then
// stays within 2^8, exact in the fp32 accumulator and inside fp16's range.
constexpr float kRescaleThreshold = 8.0f;

// What the MMA and softmax warps know of an item.
struct Info {
  int batch, head, row0[kTiles];  // first query row of the tiles; batch < 0: no more items
  int q_rows;                     // rows of the batch entry that exist
  int units[kTiles];
  int part;  // workspace part of tile 0 (tile 1: the next), or -1: rows are final
};
// Keys of the units ahead, per tile: more than the slots of the ring and the scores in TMEM
// can be ahead of the softmax (10 + 2 units).
constexpr int kKeyRing = 16;

template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kQBytes = kHalves * kQHalf;
  static constexpr uint32_t kPartBytes = kHalves * kKvHalf;  // K or V rows of a unit
  static constexpr uint32_t kSlotBytes = 2 * kPartBytes;
  // Slots: what fits beside the two Q tiles (five of 32 KB at D = 128).
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr uint32_t kSmemQ = 0;
  static constexpr uint32_t kSmemRing = kTiles * kQBytes;
  static constexpr uint32_t kSmemBar = kSmemRing + kSlots * kSlotBytes;
  // qfull[2] qempty[2] s[2][2] p[2][2] pv[2][2] fix ifull[2] iempty[2] next full[slots] empty[slots]
  static constexpr int kNumBars = 22 + 2 * kSlots;
  static constexpr uint32_t kSmemNext = (kSmemBar + kNumBars * 8 + 15) / 16 * 16;  // 16 bytes
  static constexpr uint32_t kSmemInfo = kSmemNext + 16;                    // Info[2]
  static constexpr uint32_t kSmemKeys = kSmemInfo + 2 * sizeof(Info);      // u8 [2][kKeyRing]
  static constexpr uint32_t kSmemTag = kSmemKeys + kTiles * kKeyRing;      // u32 [slots]
  static constexpr uint32_t kSmemTail = kSmemTag + 4 * kSlots;             // tmem slot, abort flag
  static constexpr uint32_t kSmemBytes = (kSmemTail + 16 + 127) / 128 * 128;
  static constexpr uint32_t kSmemAlloc = kSmemBytes + 1024;
  static_assert(kSmemAlloc <= 232448, "shared memory per CTA");
};

// Instruction descriptor, kind::f16, f32 accumulator, M = 128; A and B of one type.
__host__ __device__ constexpr uint32_t instr_desc(bool fp16, int n, bool b_mn_major) {
  return (1u << 4) | ((fp16 ? 0u : 1u) << 7) | ((fp16 ? 0u : 1u) << 10) |
         ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTile >> 4) << 24);
}

struct Params {
  void* out;
  float* lse;
  const int32_t* indices;
  const int32_t* counts;
  const int32_t* q_lens;
  const int32_t* k_lens;
  int64_t o_batch_stride, o_row_stride, o_head_stride;
  int list_len, nq, tiles_per_list;  // query tiles (1 or 2) that share a list
  int heads, group;                  // query heads, query heads per key head
  int seq_q, seq_k, nk;
  float scale_log2;
  unsigned int* status;
  // Items [0, n_full) are whole pairs of tiles; pair n_full + i is split into `splits` items
  // of entries_per_split list entries. With `duo` (one query tile) both tiles of an item are
  // that tile, with entries_per_split entries each. Split items write unnormalised fp32 O
  // and (max, sum) of `ws_rows` rows per tile to ws: ws_rows * D, then ws_rows * 4 floats of
  // which two are used (a part starts on 16 bytes).
  int pairs, n_items, n_full, splits, entries_per_split, duo, ws_rows, wide_out;
  float* ws;
};

__device__ __forceinline__ int rows_of(const int32_t* lens, int b, int seq) {
  if (lens == nullptr) return seq;
  const int n = lens[b];
  return n < 0 ? 0 : (n > seq ? seq : n);
}

// One item as the load warp reads it: everything that comes from global memory is asked for
// at once, list entries a lane each (entries lane and 32 + lane of both lists).
struct Item {
  int batch, head, row0[kTiles], q_len, k_len, part;
  int count[kTiles];            // as it stands in memory
  int first[kTiles], most[kTiles];  // the item's first entry, and how many it may use
  const int32_t* list[kTiles];  // from the first entry on
  int chunk[kTiles], ahead[kTiles];

  __device__ __forceinline__ void load(const Params& p, int item, int lane) {
    int whole = item, rank = 0;
    const bool split = item >= p.n_full;
    part = -1;
    if (split) {
      const int i = item - p.n_full;
      whole = p.n_full + i / p.splits;
      rank = i % p.splits;
      part = i * kTiles;
    }
    const int pair = whole % p.pairs;
    const int bh = whole / p.pairs;
    head = bh % p.heads;
    batch = bh / p.heads;
    q_len = p.q_lens != nullptr ? p.q_lens[batch] : p.seq_q;
    k_len = p.k_lens != nullptr ? p.k_lens[batch] : p.seq_k;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int tile = p.duo ? 0 : kTiles * pair + t;
      row0[t] = tile * kTile;
      first[t] = split ? (p.duo ? kTiles * rank + t : rank) * p.entries_per_split : 0;
      // A tile behind the last row has no list of its own; it gets no entries either.
      const int64_t at = (int64_t)bh * p.nq + min(tile / p.tiles_per_list, p.nq - 1);
      count[t] = p.counts != nullptr ? p.counts[at] : p.list_len;
      most[t] = split ? min(p.entries_per_split, p.list_len - first[t]) : p.list_len;
      list[t] = p.indices + at * p.list_len + first[t];
      chunk[t] = lane < most[t] ? list[t][lane] : -1;
      ahead[t] = 32 + lane < most[t] ? list[t][32 + lane] : -1;
    }
  }
  __device__ __forceinline__ int q_rows(const Params& p) const { return min(max(q_len, 0), p.seq_q); }
  __device__ __forceinline__ int k_rows(const Params& p) const { return min(max(k_len, 0), p.seq_k); }
  __device__ __forceinline__ int entries(const Params& p, int t) const {
    return row0[t] < q_rows(p)
               ? max(0, min(min(max(count[t], 0), p.list_len) - first[t], most[t]))
               : 0;
  }
};

// The 64 keys of a unit: first row, and how many rows exist (0 for an entry that names no block).
template <int BK>
__device__ __forceinline__ int unit_keys(int entry, int unit, int nk, int k_rows, int& row) {
  row = (unsigned)entry < (unsigned)nk ? entry * BK + (unit & (BK / kUnit - 1)) * kUnit : k_rows;
  return max(0, min(kUnit, k_rows - row));
}

// Two fp32 values as a pair of the operand type.
template <bool FP16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if (FP16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_bf16(lo, hi);
}

// SHARED: the tiles of a pair have one list (block_q = 256), and one slot serves both.
template <bool FP16, int D, int BK, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1)
    sparse_fwd(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map, const Params prm) {
  using L = Layout<D>;
  constexpr int kPer = BK / kUnit;  // units per list entry
  constexpr int kSlots = L::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bars = sbase + L::kSmemBar;
  auto bar_qfull = [&](int t) { return bars + 8u * t; };
  auto bar_qempty = [&](int t) { return bars + 8u * (2 + t); };
  auto bar_s = [&](int t, uint32_t buf) { return bars + 8u * (4 + 2 * t + buf); };
  auto bar_p = [&](int t, uint32_t buf) { return bars + 8u * (8 + 2 * t + buf); };
  auto bar_pv = [&](int t, uint32_t buf) { return bars + 8u * (12 + 2 * t + buf); };
  const uint32_t bar_fix = bars + 8u * 16;
  auto bar_ifull = [&](uint32_t i) { return bars + 8u * (17 + (i & 1)); };
  auto bar_iempty = [&](uint32_t i) { return bars + 8u * (19 + (i & 1)); };
  const uint32_t bar_next = bars + 8u * 21;
  auto bar_full = [&](int s) { return bars + 8u * (22 + s); };
  auto bar_empty = [&](int s) { return bars + 8u * (22 + kSlots + s); };
  volatile Info* info = reinterpret_cast<volatile Info*>(smem + L::kSmemInfo);
  volatile uint8_t* key_ring = smem + L::kSmemKeys;  // [tile][unit % kKeyRing]
  volatile uint32_t* slot_tag = reinterpret_cast<uint32_t*>(smem + L::kSmemTag);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSmemTail);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(bar_qfull(t), 1);
      mbar_init(bar_qempty(t), 1);
      for (int buf = 0; buf < 2; ++buf) {
        mbar_init(bar_s(t, buf), 1);
        mbar_init(bar_p(t, buf), 4);
        mbar_init(bar_pv(t, buf), 1);
      }
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(bar_full(s), 1);
      slot_tag[s] = 0xffffffffu;
      mbar_init(bar_empty(s), SHARED ? 2 : 1);  // the tiles that wait for a slot
    }
    mbar_init(bar_fix, 1);
    mbar_init(bar_next, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_ifull(i), 1);
      mbar_init(bar_iempty(i), kSoftmaxWarps + kTiles);
    }
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kLoadWarp && lane == 0) {
    prefetch_map(&q_map);
    prefetch_map(&k_map);
    prefetch_map(&v_map);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_wait();  // everything above touched nothing but this CTA's own memory

  auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, prm.status));
  };
  // Slots are filled and read in one order; `pos` counts them since the start.
  auto slot_of = [](uint32_t pos) { return (int)(pos % kSlots); };
  auto phase_of = [](uint32_t pos) { return (pos / kSlots) & 1u; };
  // The next item of this warp, `i` counting them: read from shared memory, then released.
  // False at the end.
  auto take_info = [&](uint32_t i, Info& it) -> bool {
    if (!wait_all(bar_ifull(i), (i >> 1) & 1)) return false;
    const volatile Info& src = info[i & 1];
    it.batch = src.batch;
    it.head = src.head;
    it.row0[0] = src.row0[0];
    it.row0[1] = src.row0[1];
    it.q_rows = src.q_rows;
    it.units[0] = src.units[0];
    it.units[1] = src.units[1];
    it.part = src.part;
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_iempty(i));
    return it.batch >= 0;
  };

  if (warp == kLoadWarp) {
    // ---------------- loads: the whole warp walks, one lane issues ----------------
    uint32_t pos = 0;
    uint32_t q_phase[kTiles] = {0, 0};
    uint32_t fix_phase = 0;
    bool ok = true;
    // A tile's walk along its list: entries of units u, u + 1, u + 2 (-1 behind the end), and
    // two chunks of 32 entries, a lane each, the second on its way while the first is used.
    struct Walk {
      const int32_t* list;
      int entries, units, e[3], chunk, ahead, base;
      uint32_t keys_at;  // units handed to the softmax so far
    };
    Walk walk[kTiles];
    walk[0].keys_at = walk[1].keys_at = 0;
    uint32_t n_items = 0;
    uint32_t next_phase = 0;
    for (int item = blockIdx.x; item >= 0 && ok; ++n_items) {
      Item it;
      it.load(prm, item, lane);
      const int kv_head = it.head / prm.group;
      const int k_rows = it.k_rows(prm);
      auto entry = [&](Walk& w, int unit) -> int {  // called with ascending units
        const int i = unit / kPer;
        if (i >= w.entries) return -1;
        if (i >= w.base + 32) {
          w.base += 32;
          w.chunk = w.ahead;
          w.ahead = w.base + 32 + lane < w.entries ? w.list[w.base + 32 + lane] : -1;
        }
        return __shfl_sync(0xffffffffu, w.chunk, i & 31);
      };
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        Walk& w = walk[t];
        w.list = it.list[t];
        w.entries = it.entries(prm, t);
        w.units = w.entries * kPer;
        w.base = 0;
        w.chunk = it.chunk[t];
        w.ahead = it.ahead[t];
        w.e[0] = entry(w, 0);
        w.e[1] = entry(w, 1);
        w.e[2] = entry(w, 2);
      }
      ok = wait_all(bar_iempty(n_items), ((n_items >> 1) & 1) ^ 1);
      if (!ok) break;
      if (lane == 0) {
        volatile Info& dst = info[n_items & 1];
        dst.batch = it.batch;
        dst.head = it.head;
        dst.row0[0] = it.row0[0];
        dst.row0[1] = it.row0[1];
        dst.q_rows = it.q_rows(prm);
        dst.units[0] = walk[0].units;
        dst.units[1] = walk[1].units;
        dst.part = it.part;
        mbar_arrive(bar_ifull(n_items));
      }
      __syncwarp();
      // The next slot: V of `unit` and K of unit + 2 (none from the end on), or, with unit -1,
      // K of units 0 and 1. The keys of the K units go to the softmax of the tiles that read it.
      auto push = [&](int t, int unit) -> bool {
        Walk& w = walk[t];
        const bool first = unit < 0;
        const bool two = first ? w.units > 1 : unit + 2 < w.units;  // both parts are there
        int row0, row1;
        const int keys0 = unit_keys<BK>(w.e[0], first ? 0 : unit, prm.nk, k_rows, row0);
        const int keys1 = first ? unit_keys<BK>(w.e[1], 1, prm.nk, k_rows, row1)
                                : unit_keys<BK>(w.e[2], unit + 2, prm.nk, k_rows, row1);
        if (keys0 == 0) row0 = prm.seq_k;  // behind the end: zeros
        if (keys1 == 0) row1 = prm.seq_k;
        const bool cut = !first && keys0 > 0 && keys0 < kUnit && k_rows < prm.seq_k;
        const int slot = slot_of(pos);
        if (!wait_all(bar_empty(slot), phase_of(pos) ^ 1)) return false;
        const uint32_t dst = sbase + L::kSmemRing + slot * L::kSlotBytes;
        const uint32_t full = bar_full(slot);
        // Visible to the softmax through this slot's barrier, the MMA warp and its commit: written by the
        // lane that arms the barrier.
        auto hand_keys = [&](const Walk& reader, int tile) {
          if (first) key_ring[tile * kKeyRing + reader.keys_at % kKeyRing] = (uint8_t)keys0;
          if (two) key_ring[tile * kKeyRing + (reader.keys_at + (first ? 1 : 0)) % kKeyRing] = (uint8_t)keys1;
        };
        const bool both = SHARED && walk[1].units > 0;
        if (elect_one()) {
          hand_keys(w, t);
          if (both) hand_keys(walk[1], 1);
          slot_tag[slot] = pos;
          const uint32_t bar = cut ? bar_fix : full;
          mbar_expect_tx(bar, two ? L::kSlotBytes : L::kPartBytes);
          const CUtensorMap* map0 = first ? &k_map : &v_map;
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h)
            tma_load_4d(dst + h * kKvHalf, map0, bar, 64 * h, kv_head, row0, it.batch);
          if (two) {
#pragma unroll
            for (int h = 0; h < L::kHalves; ++h)
              tma_load_4d(dst + L::kPartBytes + h * kKvHalf, &k_map, bar, 64 * h, kv_head, row1,
                          it.batch);
          }
        }
        __syncwarp();
        const uint32_t handed = (first ? 1u : 0u) + (two ? 1u : 0u);
        w.keys_at += handed;
        if (both) walk[1].keys_at += handed;
        if (cut) {
          // V rows behind the last key: zeros, then hand the slot over.
          if (!wait_all(bar_fix, fix_phase)) return false;
          fix_phase ^= 1;
          for (int i = lane; i < (kUnit - keys0) * 8 * L::kHalves; i += 32) {
            const int r = keys0 + i / (8 * L::kHalves), c = i % (8 * L::kHalves);
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(
                             dst + (c >> 3) * kKvHalf + r * 128 + (c & 7) * 16),
                         "r"(0)
                         : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (elect_one()) mbar_arrive(full);
          __syncwarp();
        }
        ++pos;
        return true;
      };
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        if (walk[t].units == 0 || !ok) continue;
        ok = wait_all(bar_qempty(t), q_phase[t] ^ 1);
        if (!ok) break;
        q_phase[t] ^= 1;
        if (elect_one()) {
          const uint32_t dst = sbase + L::kSmemQ + t * L::kQBytes;
          mbar_expect_tx(bar_qfull(t), L::kQBytes);
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h)
            tma_load_4d(dst + h * kQHalf, &q_map, bar_qfull(t), 64 * h, it.head,
                        it.row0[t], it.batch);
        }
        __syncwarp();
        if (t == 0 || !SHARED) ok = push(t, -1);
      }
      const int units = max(walk[0].units, walk[1].units);
      // Asks for the next item two units before the last: late enough to leave it to a CTA
      // that is free sooner, early enough to have the answer when this item's loads are out.
      const int ask = max(units - 2, 0);
      auto request = [&]() {
        if (elect_one()) {
          mbar_expect_tx(bar_next, 16);
          asm volatile(
              "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 "
              "[%0], [%1];" ::"r"(sbase + L::kSmemNext),
              "r"(bar_next)
              : "memory");
        }
        __syncwarp();
      };
      if (units == 0) request();
      for (int u = 0; u < units && ok; ++u) {
        if (u == ask) request();
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          Walk& w = walk[t];
          if (u < w.units && ok && (t == 0 || !SHARED)) ok = push(t, u);
          w.e[0] = w.e[1];
          w.e[1] = w.e[2];
          w.e[2] = entry(w, u + 3);
        }
      }
      ok = ok && wait_all(bar_next, next_phase);
      if (!ok) break;
      next_phase ^= 1;
      uint32_t taken, cta;
      asm volatile(
          "{\n\t.reg .b128 answer;\n\t.reg .pred p;\n\t"
          "ld.shared.b128 answer, [%2];\n\t"
          "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, answer;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t"
          "mov.u32 %1, 0;\n\t"
          "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, answer;\n\t}"
          : "=r"(taken), "=r"(cta)
          : "r"(sbase + L::kSmemNext)
          : "memory");
      // The answer has been read before the next one may be written.
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      item = taken ? (int)cta : -1;
    }
    if (ok && wait_all(bar_iempty(n_items), ((n_items >> 1) & 1) ^ 1)) {
      if (lane == 0) {
        info[n_items & 1].batch = -1;
        mbar_arrive(bar_ifull(n_items));
      }
      __syncwarp();
    }
  } else if (warp >= kMmaWarp) {
    // ---------------- MMA issuer of tile t ----------------
    const int t = warp - kMmaWarp;
    constexpr uint32_t idesc_qk = instr_desc(FP16, kUnit, false);
    constexpr uint32_t idesc_pv = instr_desc(FP16, D, true);
    const uint64_t q_desc = smem_desc(sbase + L::kSmemQ + t * L::kQBytes, 16, 1024);
    const uint64_t k_desc0 = smem_desc(sbase + L::kSmemRing, 16, 1024);
    const uint64_t v_desc0 = smem_desc(sbase + L::kSmemRing, kKvHalf, 1024);
    const uint32_t t_s = tmem + kTmemS + t * 128;
    const uint32_t t_o = tmem + kTmemO + t * 128;
    uint32_t base = 0;           // slots of the items before
    uint32_t n_s = 0, n_pv = 0;  // units issued so far
    uint32_t q_phase = 0;
    bool ok = true;
    // Waits for the slot at `at`. With slots of its own a tile never looks at the other's, so
    // it can be here before the slot's use before this one (the other's) has landed, and the
    // parity of that phase is the one it would take for its own: the tag comes first.
    auto wait_slot = [&](uint32_t at) -> bool {
      const int slot = slot_of(at);
      if (!SHARED && __any_sync(0xffffffffu, slot_tag[slot] != at)) {
        const unsigned long long t0 = globaltimer();
        while (__any_sync(0xffffffffu, slot_tag[slot] != at)) {
          const bool late = globaltimer() - t0 > kWaitLimitNs;
          if (late && lane == 0) {
            *abort_flag = 1u;
            if (prm.status) atomicOr(prm.status, kStatusAttentionTimeout);
          }
          if (__any_sync(0xffffffffu, late || *abort_flag != 0u)) return false;
        }
      }
      return wait_all(bar_full(slot), phase_of(at));
    };
    // One lane: S = Q K^T, K being part `part` of the slot.
    auto issue_s = [&](int slot, int part) {
      const uint64_t kd =
          k_desc0 + (uint64_t)((slot * L::kSlotBytes + part * L::kPartBytes) >> 4);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t in = (kk & 3) * 32;
        mma_ss(t_s + (n_s & 1) * 64, q_desc + (uint64_t)(((kk >> 2) * kQHalf + in) >> 4),
               kd + (uint64_t)(((kk >> 2) * kKvHalf + in) >> 4), idesc_qk, kk > 0 ? 1u : 0u);
      }
      mma_commit(bar_s(t, n_s & 1));
    };
    for (uint32_t n_items = 0; ok; ++n_items) {
      Info it;
      if (!take_info(n_items, it)) break;
      const int units0 = it.units[0], units1 = it.units[1];
      const int units = t == 0 ? units0 : units1;
      // Where this tile's slots are: its first at base + lead, slot u at `next`, which steps
      // over the other tile's while that has units left.
      const int other = t == 0 ? units1 : units0;
      const uint32_t lead = t == 1 && !SHARED && units0 > 0 ? 1u : 0u;
      const uint32_t firsts = SHARED ? 1u : (units0 > 0) + (units1 > 0);
      uint32_t next = base + firsts + (t == 1 && !SHARED && units0 > 0 ? 1u : 0u);
      const uint32_t slots = units0 == 0 && units1 == 0 ? 0u
                             : firsts + (SHARED ? max(units0, units1) : units0 + units1);
      auto release = [&](int slot) { mma_commit(bar_empty(slot)); };  // one lane
      // A tile without rows passes its item's shared slots one by one. It must not step over them:
      // a parity names a phase only to a warp that has seen the phase before, and in a later
      // item it could take a slot whose use in this one has not landed for its own. (592
      // pairs of tiles with lists of 64 blocks of 128 keys: 458 us, stepping over 473 us. Testing
      // the tag of shared slots instead: 506 us where stepping over took 482 us.)
      for (uint32_t i = 0; SHARED && units == 0 && i < slots; ++i) {
        const int slot = slot_of(base + i);
        ok = wait_slot(base + i);
        if (!ok) break;
        if (lane == 0) mbar_arrive(bar_empty(slot));
        __syncwarp();
      }
      if (!ok) break;
      if (units > 0) {
        const uint32_t first = base + lead;
        const int slot = slot_of(first);
        ok = wait_all(bar_qfull(t), q_phase) && wait_slot(first);
        if (!ok) break;
        q_phase ^= 1;
        tc_fence_after();
        if (elect_one()) issue_s(slot, 0);
        __syncwarp();
        ++n_s;
        if (units > 1) {
          if (elect_one()) issue_s(slot, 1);
          __syncwarp();
          ++n_s;
        }
        if (elect_one()) {
          release(slot);
          if (units <= 2) mma_commit(bar_qempty(t));
        }
        __syncwarp();
      }
      for (int u = 0; u < units; ++u) {
        const int slot = slot_of(next);
        ok = wait_all(bar_p(t, n_pv & 1), (n_pv >> 1) & 1) && wait_slot(next);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = v_desc0 + (uint64_t)((slot * L::kSlotBytes) >> 4);
#pragma unroll
          for (int kk = 0; kk < kUnit / 16; ++kk)
            mma_ts(t_o, t_s + (n_pv & 1) * 64 + kk * 8, vd + (uint64_t)((kk * 2048) >> 4),
                   idesc_pv, (u > 0 || kk > 0) ? 1u : 0u);
          mma_commit(bar_pv(t, n_pv & 1));
          if (u + 2 < units) issue_s(slot, 1);
          release(slot);
          if (u + 3 == units) mma_commit(bar_qempty(t));
        }
        __syncwarp();
        ++n_pv;
        if (u + 2 < units) ++n_s;
        // Slots in order: unit u of tile 0, of tile 1, unit u + 1 of tile 0, ...
        if (SHARED) {
          next += 1;
        } else {
          next += 1u + (t == 0 ? u < other : u + 1 < other);
        }
      }
      base += slots;
    }
  } else {
    // ---------------- softmax: warp -> (tile, lane quadrant), thread -> query row ----------------
    const int t = warp >> 2;
    const int quad = warp & 3;
    const int row_in_tile = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t t_o = tmem + lanes + kTmemO + t * 128;
    const float c = prm.scale_log2;
    const float2 c2 = make_float2(c, c);
    uint32_t n = 0;  // units so far: buffer n & 1, phase n >> 1
    bool ok = true;
    for (uint32_t n_items = 0; ok; ++n_items) {
      Info it;
      if (!take_info(n_items, it)) break;
      const int units = t == 0 ? it.units[0] : it.units[1];
      const int row = (t == 0 ? it.row0[0] : it.row0[1]) + row_in_tile;
      const bool live = row < it.q_rows;
      const bool idle = !__any_sync(0xffffffffu, live);  // no row of this warp exists
      float m_use = -INFINITY;  // running row max, log2 units, that P is taken against
      float l_sum = 0.f;
      // Nobody reads the rows of a warp without rows: whatever stands in TMEM will do for P.
      for (int u = 0; idle && u < units; ++u, ++n) {
        ok = wait_all(bar_s(t, n & 1), (n >> 1) & 1);
        if (!ok) break;
        if (lane == 0) mbar_arrive(bar_p(t, n & 1));
      }
      // Whether this unit's scores were seen complete during the last one's
      // exponentials: a wait costs 90 to 180 clocks even where nothing is left to wait for
      // (561 against 580 us with one list per pair, 593 against 597 us with a list per tile).
      bool ready = false;
      for (int u = 0; !idle && u < units; ++u, ++n) {
        const uint32_t t_s = tmem + lanes + kTmemS + t * 128 + (n & 1) * 64;
        // tcgen05.ld/st below are warp-collective.
        if (!__all_sync(0xffffffffu, ready)) {
          ok = wait_all(bar_s(t, n & 1), (n >> 1) & 1);
          if (!ok) break;
        }
        tc_fence_after();
        const int keys = key_ring[t * kKeyRing + n % kKeyRing];
        uint32_t sv[2][32];
        tmem_ld32(t_s, sv[0]);
        tmem_ld32(t_s + 32, sv[1]);
        tmem_ld_wait(sv[0]);
        tmem_pin(sv[1]);
        if (keys < kUnit) {  // columns from `keys` on do not exist
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= keys) sv[i >> 5][i & 31] = __float_as_uint(-INFINITY);
        }
        float mx[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const uint32_t* r = sv[a >> 1] + (a & 1) * 16;
          float m = max3(__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[2]));
#pragma unroll
          for (int k = 3; k < 15; k += 2)
            m = max3(m, __uint_as_float(r[k]), __uint_as_float(r[k + 1]));
          mx[a] = fmaxf(m, __uint_as_float(r[15]));
        }
        const float m_new = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * c;
        const bool need = m_new > m_use + kRescaleThreshold;
        if (__any_sync(0xffffffffu, need)) {
          const float m_next = need ? m_new : m_use;
          if (u > 0) {
            // O is at rest once P V of the unit before is complete. That one's buffer was last
            // used two units before it, which these scores certify: the parity names the phase.
            ok = wait_all(bar_pv(t, (n - 1) & 1), ((n - 1) >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            const float alpha = need ? ex2(m_use - m_next) : 1.f;
#pragma unroll 1
            for (int q8 = 0; q8 < D / 16; ++q8) {
              uint32_t o[16];
              tmem_ld16(t_o + 16 * q8, o);
              tmem_ld_wait16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(t_o + 16 * q8, o);
            }
            l_sum *= alpha;
          }
          m_use = m_next;
        }
        const float base = m_use == -INFINITY ? 0.f : m_use;  // no key yet: all p are 0
        const float2 nm2 = make_float2(-base, -base);
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (i == 8) {
            ready = u + 1 < units && mbar_try(bar_s(t, (n + 1) & 1), ((n + 1) >> 1) & 1);
          }
          const uint32_t* src = sv[i >> 4] + 2 * (i & 15);
          const float2 x = __ffma2_rn(
              make_float2(__uint_as_float(src[0]), __uint_as_float(src[1])), c2, nm2);
          float2 p;
          p.x = ex2(x.x);
          p.y = ex2(x.y);
          acc[i & 1] = __fadd2_rn(acc[i & 1], p);
          pk[i] = pack_pair<FP16>(p.x, p.y);
        }
        // P over the first 32 of the unit's S columns, all of them read. One arrival per warp:
        // with one per thread, and the MMA warps waiting for the slot before P, 560 and 601 us
        // against 556 and 580.
        tmem_st32(t_s, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p(t, n & 1));
        l_sum += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
      }
      // ---------------- epilogue ----------------
      if (ok && units > 0) ok = wait_all(bar_pv(t, (n - 1) & 1), ((n - 1) >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (it.part >= 0) {
        float* ws = prm.ws + (int64_t)(it.part + t) * prm.ws_rows * (D + 4);
        if (units > 0 && !idle) {
#pragma unroll 1
          for (int q4 = 0; q4 < D / 32; ++q4) {
            uint32_t o[32];
            tmem_ld32(t_o + 32 * q4, o);
            tmem_ld_wait(o);
            float* dst = ws + row_in_tile * D + 32 * q4;
            if (live) {
#pragma unroll
              for (int v4 = 0; v4 < 8; ++v4)
                *reinterpret_cast<float4*>(dst + v4 * 4) =
                    make_float4(__uint_as_float(o[v4 * 4 + 0]), __uint_as_float(o[v4 * 4 + 1]),
                                __uint_as_float(o[v4 * 4 + 2]), __uint_as_float(o[v4 * 4 + 3]));
            }
          }
        }
        if (live)
          *reinterpret_cast<float2*>(ws + prm.ws_rows * D + 2 * row_in_tile) =
              make_float2(m_use, l_sum);
        continue;
      }
      const bool some = live && l_sum != 0.f;  // the row has a key
      const float inv_l = some ? 1.f / l_sum : 0.f;
      uint16_t* dst = row < prm.seq_q
                          ? reinterpret_cast<uint16_t*>(prm.out) +
                                (int64_t)it.batch * prm.o_batch_stride +
                                (int64_t)row * prm.o_row_stride +
                                (int64_t)it.head * prm.o_head_stride
                          : nullptr;
#pragma unroll 1
      for (int q4 = 0; q4 < D / 32; ++q4) {
        uint32_t o[32];
        if (units > 0) {
          tmem_ld32(t_o + 32 * q4, o);
          tmem_ld_wait(o);
        }
        if (units == 0 || !some) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (dst != nullptr) {
          Chunk32 w[2];
          uint32_t* words = reinterpret_cast<uint32_t*>(w);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            words[i] = pack_pair<FP16>(__uint_as_float(o[2 * i]) * inv_l,
                                       __uint_as_float(o[2 * i + 1]) * inv_l);
          // A thread per row: 32-byte stores are whole sectors, half as many as 16-byte ones.
          if (prm.wide_out) {
            st32(dst + 32 * q4, w[0]);
            st32(dst + 32 * q4 + 16, w[1]);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              *reinterpret_cast<uint4*>(dst + 32 * q4 + 16 * i) = w[i].lo;
              *reinterpret_cast<uint4*>(dst + 32 * q4 + 16 * i + 8) = w[i].hi;
            }
          }
        }
      }
      if (dst != nullptr && prm.lse != nullptr)
        prm.lse[((int64_t)it.batch * prm.heads + it.head) * prm.seq_q + row] =
            some ? (m_use + log2f(l_sum)) * 0.6931471805599453f : -INFINITY;
    }
  }

  grid_done();
  if (*abort_flag != 0u) {
    // Unwinding: let copies in flight land before shared memory is given up.
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  }
}

// Joins the parts of the split pairs: one warp per query row, D/32 columns per lane.
// O = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s. Up to kMaxParts parts: lane s holds the
// max and sum of part s, and the O of four parts is on its way at a time.
constexpr int kMaxParts = 32;
template <bool FP16, int D>
__global__ void __launch_bounds__(256) sparse_combine(const Params prm, int split_pairs) {
  grid_wait();
  const int gw = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int pair_rows = min(prm.duo ? kTile : kTiles * kTile, prm.seq_q);
  if (gw >= split_pairs * pair_rows) return;
  const int ui = gw / pair_rows;
  const int rr = gw - ui * pair_rows;
  const int t = rr / kTile;
  const int r_in_tile = rr - t * kTile;
  const int whole = prm.n_full + ui;
  const int bh = whole / prm.pairs;
  const int head = bh % prm.heads;
  const int batch = bh / prm.heads;
  const int row = whole % prm.pairs * (kTiles * kTile) + rr;
  if (row >= prm.seq_q) return;
  const bool live = row < rows_of(prm.q_lens, batch, prm.seq_q);
  const int parts = prm.duo ? prm.splits * kTiles : prm.splits;
  const int64_t part_floats = (int64_t)prm.ws_rows * (D + 4);
  const int64_t step = prm.duo ? part_floats : part_floats * kTiles;
  const float* first = prm.ws + (int64_t)ui * prm.splits * kTiles * part_floats + t * part_floats;
  constexpr int kCols = D / 32;
  float acc[kCols] = {};
  float m = -INFINITY, l = 0.f;
  if (live && lane < parts) {
    const float2 ml =
        *reinterpret_cast<const float2*>(first + lane * step + prm.ws_rows * D + 2 * r_in_tile);
    m = ml.x;
    l = ml.y;
  }
  float m_max = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m_max = fmaxf(m_max, __shfl_xor_sync(0xffffffffu, m_max, o));
  // A part without keys wrote no O and has no weight.
  const float weight = l == 0.f ? 0.f : ex2(m - m_max);
  const float l_tot = warp_sum(l == 0.f ? 0.f : weight * l);
  const unsigned with_keys = __ballot_sync(0xffffffffu, l != 0.f);
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float w = __shfl_sync(0xffffffffu, weight, s);
    if ((with_keys >> s & 1u) == 0u) continue;
    const float* o = first + s * step + r_in_tile * D + lane * kCols;
#pragma unroll
    for (int i = 0; i < kCols; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(o + i);
      acc[i] += w * v.x;
      acc[i + 1] += w * v.y;
    }
  }
  const float inv = l_tot == 0.f ? 0.f : 1.f / l_tot;
  uint16_t* dst = reinterpret_cast<uint16_t*>(prm.out) + (int64_t)batch * prm.o_batch_stride +
                  (int64_t)row * prm.o_row_stride + (int64_t)head * prm.o_head_stride +
                  lane * kCols;
#pragma unroll
  for (int i = 0; i < kCols; i += 2)
    *reinterpret_cast<uint32_t*>(dst + i) = pack_pair<FP16>(acc[i] * inv, acc[i + 1] * inv);
  if (prm.lse != nullptr && lane == 0)
    prm.lse[(int64_t)bh * prm.seq_q + row] =
        l_tot != 0.f ? (m_max + log2f(l_tot)) * 0.6931471805599453f : -INFINITY;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

struct Plan {
  int pairs, total, n_full, splits, entries_per_split, items, split_pairs, duo, ws_rows;
  int64_t ws_bytes;
};

// Whole pairs of tiles fill waves of SMs; when the last wave would leave at least half of
// them idle, its pairs may be split along their lists, down to 128 keys per part, and joined.
// Queries of one tile are split in two even where SMs are short, half a list for each of the
// two tiles of an item. Both only as far as an estimate says that it saves more than the join
// costs: a step is one unit of 64 keys of both tiles (or of a lone one), the join another launch
// and the parts written and read. (Whole lists of 16 and 128 units on 2048 rows, 6 heads, at full
// clock: 0.74 us a step with D = 64, 0.76 to 0.80 with D = 128; long calls that draw the power cap take
// more, but they fill the SMs without a split.) Measured split into as many parts as fit, and whole (us):
// 2048 rows, 6 heads, D = 64, lists of 256 keys 14.9 and 8.2, of 1536 keys 21.5 and 23.1, of
// 8192 keys 50 and 100; one row, 6 heads, 256 keys 8.7 and 6.7, 768 keys 9.2 and 11.3.
Plan make_plan(int64_t batch, int64_t seq_q, int64_t heads, int64_t head_dim, int64_t block_k,
               int64_t list_len, bool can_split) {
  Plan pl{};
  pl.pairs = (int)((seq_q + kTiles * kTile - 1) / (kTiles * kTile));
  pl.total = (int)(pl.pairs * heads * batch);
  const int least = (int)(2 * kUnit / block_k);  // entries of 128 keys
  const int parts = (int)((list_len + least - 1) / least);
  const int sms = num_sms();
  pl.ws_rows = (int)std::min<int64_t>(kTile, seq_q);
  pl.splits = 1;
  pl.entries_per_split = (int)list_len;
  pl.n_full = pl.items = pl.total;
  const int64_t units = list_len * block_k / kUnit;
  constexpr int64_t kPairStepNs = 740, kTileStepNs = 580, kJoinNs = 4000, kJoinNsPerMb = 600;
  const bool one_tile = seq_q <= kTile;
  const int each = one_tile ? kTiles : 1;  // ranges per item
  const int rem = one_tile ? pl.total : pl.total % sms;
  auto waves = [&](int64_t items) { return (items + sms - 1) / sms; };
  const int64_t part_bytes = (int64_t)pl.ws_rows * (head_dim + 4) * 4;
  int64_t best = waves(rem) * units * (one_tile ? kTileStepNs : kPairStepNs);
  const int most = rem == 0 || !can_split
                       ? 0
                       : std::min(std::min(std::max(sms / rem, 1) * each, kMaxParts), parts);
  for (int want = 2; want <= most; ++want) {
    const int entries = (parts + want - 1) / want * least;
    const int ranges = (int)((list_len + entries - 1) / entries);
    const int splits = (ranges + each - 1) / each;
    const int64_t bytes = (int64_t)rem * splits * kTiles * part_bytes;
    if (bytes > (256ll << 20)) break;
    const int64_t ns = waves((int64_t)rem * splits) * (entries * block_k / kUnit) * kPairStepNs +
                       kJoinNs + bytes * kJoinNsPerMb / 1000000;
    if (ns < best) {
      best = ns;
      pl.duo = one_tile;
      pl.splits = splits;
      pl.entries_per_split = entries;
    }
  }
  if (pl.duo || pl.splits >= 2) {
    pl.split_pairs = rem;
    pl.n_full = pl.total - rem;
    pl.items = pl.n_full + rem * pl.splits;
    pl.ws_bytes = (int64_t)rem * pl.splits * kTiles * part_bytes;
  }
  return pl;
}

// 4-D map over (head_dim, heads, rows, batch) with a (64, 1, box_rows, 1) box.
int make_map(CUtensorMap* map, const void* base, int64_t batch, int64_t seq, int64_t heads,
             int64_t head_dim, int64_t bs, int64_t rs, int64_t hs, int box_rows, bool fp16,
             const char* name) {
  auto fn = encode_fn();
  if (fn == nullptr) {
    set_error("h3b_block_sparse_attention: cuTensorMapEncodeTiled is unavailable");
    return H3B_ERR_CUDA;
  }
  // Size-1 dimensions never step their stride; give them a valid one.
  if (heads == 1) hs = head_dim;
  if (seq == 1) rs = heads * hs;
  if (batch == 1) bs = rs * seq;
  cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)seq,
                        (cuuint64_t)batch};
  cuuint64_t strides[3] = {(cuuint64_t)hs * 2, (cuuint64_t)rs * 2, (cuuint64_t)bs * 2};
  cuuint32_t box[4] = {64, 1, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                  4, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    char buf[256];
    snprintf(buf, sizeof(buf),
             "h3b_block_sparse_attention: tensor map for %s rejected (CUresult %d)", name, (int)r);
    set_error(buf);
    return H3B_ERR_CUDA;
  }
  return H3B_OK;
}

template <bool FP16, int D, int BK, bool SHARED>
int launch(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const Params& p,
           int split_pairs, cudaStream_t stream) {
  static ContextSlot slots[kMaxDevices];
  cudaError_t e = cudaErrorInvalidDevice;
  if (context_cached(slots, [&]() -> void* {
        e = cudaFuncSetAttribute(sparse_fwd<FP16, D, BK, SHARED>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)Layout<D>::kSmemAlloc);
        return e == cudaSuccess ? reinterpret_cast<void*>(1) : nullptr;
      }) == nullptr) {
    set_error(std::string("h3b_block_sparse_attention: cannot reserve shared memory: ") +
              cudaGetErrorString(e));
    return H3B_ERR_CUDA;
  }
  launch_after(sparse_fwd<FP16, D, BK, SHARED>, dim3((unsigned)p.n_items), kThreads, Layout<D>::kSmemAlloc, stream, qm, km,
               vm, p);
  int rc = check_launch("h3b_block_sparse_attention");
  if (rc != H3B_OK || split_pairs == 0) return rc;
  const int rows = split_pairs * std::min(p.duo ? kTile : kTiles * kTile, p.seq_q);
  launch_after(sparse_combine<FP16, D>, dim3((unsigned)((rows + 7) / 8)), 256, 0, stream, p,
               split_pairs);
  return check_launch("h3b_block_sparse_attention");
}

template <bool FP16, int D, int BK>
int launch_lists(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm,
                 const Params& p, int split_pairs, cudaStream_t s) {
  return p.tiles_per_list == kTiles && !p.duo
             ? launch<FP16, D, BK, true>(qm, km, vm, p, split_pairs, s)
             : launch<FP16, D, BK, false>(qm, km, vm, p, split_pairs, s);
}

template <bool FP16>
int launch_dims(int64_t head_dim, int64_t block_k, const CUtensorMap& qm, const CUtensorMap& km,
                const CUtensorMap& vm, const Params& p, int split_pairs, cudaStream_t s) {
  if (head_dim == 128)
    return block_k == 128 ? launch_lists<FP16, 128, 128>(qm, km, vm, p, split_pairs, s)
                          : launch_lists<FP16, 128, 64>(qm, km, vm, p, split_pairs, s);
  return block_k == 128 ? launch_lists<FP16, 64, 128>(qm, km, vm, p, split_pairs, s)
                        : launch_lists<FP16, 64, 64>(qm, km, vm, p, split_pairs, s);
}

}  // namespace sparse
}  // namespace attn
}  // namespace h3b

extern "C" int h3b_block_sparse_attention_workspace_size(int64_t batch, int64_t seq_q,
                                                         int64_t heads, int64_t head_dim,
                                                         int64_t block_k, int64_t list_len,
                                                         int64_t* bytes_out) {
  H3B_REQUIRE(bytes_out != nullptr,
              "block_sparse_attention_workspace_size: null output pointer");
  H3B_REQUIRE(batch >= 0 && seq_q >= 0 && heads >= 0 && list_len >= 0,
              "block_sparse_attention: negative shape");
  *bytes_out = 0;
  if (batch == 0 || seq_q == 0 || heads == 0 || list_len == 0 ||
      !(head_dim == 64 || head_dim == 128) || !(block_k == 64 || block_k == 128))
    return H3B_OK;
  *bytes_out = h3b::attn::sparse::make_plan(batch, seq_q, heads, head_dim, block_k, list_len, true).ws_bytes;
  return H3B_OK;
}

extern "C" int h3b_block_sparse_attention(
    void* out, float* lse, const void* q, const void* k, const void* v, const int32_t* indices,
    const int32_t* counts, int64_t list_len, int64_t batch, int64_t seq_q, int64_t seq_k,
    int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t block_q, int64_t block_k,
    int64_t q_batch_stride, int64_t q_row_stride, int64_t q_head_stride, int64_t k_batch_stride,
    int64_t k_row_stride, int64_t k_head_stride, int64_t v_batch_stride, int64_t v_row_stride,
    int64_t v_head_stride, int64_t o_batch_stride, int64_t o_row_stride, int64_t o_head_stride,
    const int32_t* q_lens, const int32_t* k_lens, float softmax_scale, int64_t dtype,
    void* workspace, int64_t workspace_bytes, h3b_stream_t stream) {
  using namespace h3b::attn::sparse;
  H3B_REQUIRE(batch >= 0 && seq_q >= 0 && seq_k >= 0 && heads >= 0 && kv_heads >= 0 && list_len >= 0,
              "block_sparse_attention: negative shape");
  if (!(head_dim == 64 || head_dim == 128) || !(block_q == 128 || block_q == 256) ||
      !(block_k == 64 || block_k == 128) ||
      !(dtype == H3B_DTYPE_BF16 || dtype == H3B_DTYPE_FP16)) {
    h3b::set_error("h3b_block_sparse_attention: needs bf16 or fp16, head_dim 64 or 128, block_q "
                   "128 or 256, block_k 64 or 128");
    return H3B_ERR_UNSUPPORTED;
  }
  if (batch == 0 || seq_q == 0 || heads == 0) return H3B_OK;
  H3B_REQUIRE(seq_k > 0, "block_sparse_attention: empty key sequence");
  H3B_REQUIRE(list_len > 0, "block_sparse_attention: empty lists");
  H3B_REQUIRE(kv_heads > 0 && heads % kv_heads == 0,
              "block_sparse_attention: heads (%lld) must be a multiple of kv_heads (%lld)",
              (long long)heads, (long long)kv_heads);
  H3B_REQUIRE(softmax_scale > 0.f && std::isfinite(softmax_scale),
              "block_sparse_attention: softmax_scale must be positive and finite");
  H3B_REQUIRE(seq_q < (1LL << 31) - 256 && seq_k < (1LL << 31) - 256 && list_len <= (1LL << 20) &&
                  batch <= (1LL << 24) / heads &&
                  ((seq_q + 255) / 256) * heads * batch < (1LL << 30),
              "block_sparse_attention: shape exceeds launch limits");
  H3B_REQUIRE(out != nullptr && q != nullptr && k != nullptr && v != nullptr && indices != nullptr,
              "block_sparse_attention: null argument");
  H3B_REQUIRE(h3b::aligned16(q) && h3b::aligned16(k) && h3b::aligned16(v) && h3b::aligned16(out),
              "block_sparse_attention: q, k, v, out must be 16-byte aligned");
  const int64_t strides[12] = {q_batch_stride, q_row_stride, q_head_stride, k_batch_stride,
                               k_row_stride,   k_head_stride, v_batch_stride, v_row_stride,
                               v_head_stride,  o_batch_stride, o_row_stride, o_head_stride};
  for (int i = 0; i < 12; ++i) {
    const int64_t seq = i / 3 == 0 || i / 3 == 3 ? seq_q : seq_k;
    const int64_t size = i % 3 == 0 ? batch
                         : i % 3 == 1 ? seq : (i / 3 == 0 || i / 3 == 3 ? heads : kv_heads);
    H3B_REQUIRE(size == 1 || (strides[i] % 8 == 0 && strides[i] > 0),
                "block_sparse_attention: strides must be positive multiples of 8 elements");
  }
  const bool fp16 = dtype == H3B_DTYPE_FP16;
  CUtensorMap qm, km, vm;
  int rc;
  if ((rc = make_map(&qm, q, batch, seq_q, heads, head_dim, q_batch_stride, q_row_stride,
                     q_head_stride, kTile, fp16, "q")) != H3B_OK)
    return rc;
  if ((rc = make_map(&km, k, batch, seq_k, kv_heads, head_dim, k_batch_stride, k_row_stride,
                     k_head_stride, kUnit, fp16, "k")) != H3B_OK)
    return rc;
  if ((rc = make_map(&vm, v, batch, seq_k, kv_heads, head_dim, v_batch_stride, v_row_stride,
                     v_head_stride, kUnit, fp16, "v")) != H3B_OK)
    return rc;
  Plan pl = make_plan(batch, seq_q, heads, head_dim, block_k, list_len, true);
  if (pl.ws_bytes > 0 && (workspace == nullptr || workspace_bytes < pl.ws_bytes ||
                          !h3b::aligned16(workspace)))
    // No (or too small a) workspace: run every pair whole.
    pl = make_plan(batch, seq_q, heads, head_dim, block_k, list_len, false);
  Params p{};
  p.out = out;
  p.lse = lse;
  p.indices = indices;
  p.counts = counts;
  p.q_lens = q_lens;
  p.k_lens = k_lens;
  p.o_batch_stride = o_batch_stride;
  p.o_row_stride = o_row_stride;
  p.o_head_stride = o_head_stride;
  p.list_len = (int)list_len;
  p.nq = (int)((seq_q + block_q - 1) / block_q);
  p.tiles_per_list = (int)(block_q / kTile);
  p.heads = (int)heads;
  p.group = (int)(heads / kv_heads);
  p.seq_q = (int)seq_q;
  p.seq_k = (int)seq_k;
  p.nk = (int)((seq_k + block_k - 1) / block_k);
  p.scale_log2 = (float)((double)softmax_scale * 1.4426950408889634);
  p.status = h3b::status_ptr();
  p.pairs = pl.pairs;
  p.n_items = pl.items;
  p.n_full = pl.n_full;
  p.splits = pl.splits;
  p.entries_per_split = pl.entries_per_split;
  p.duo = pl.duo;
  p.ws_rows = pl.ws_rows;
  p.wide_out = h3b::aligned32(out) && (batch == 1 || o_batch_stride % 16 == 0) &&
               (seq_q == 1 || o_row_stride % 16 == 0) && (heads == 1 || o_head_stride % 16 == 0);
  p.ws = reinterpret_cast<float*>(workspace);
  return fp16 ? launch_dims<true>(head_dim, block_k, qm, km, vm, p, pl.split_pairs, stream)
              : launch_dims<false>(head_dim, block_k, qm, km, vm, p, pl.split_pairs, stream);
}
