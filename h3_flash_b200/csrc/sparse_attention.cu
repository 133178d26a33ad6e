// Block-sparse attention for B200 (sm_100a): every block of query rows attends to its own
// list of key blocks. tcgen05 MMA with TMEM accumulators, TMA-fed operands, fp32 online
// softmax.
//
//   out[r] = sum_{j in list} sum_{c in block j} p_rc v_c / sum p_rc,
//   p_rc = 2^(scale log2(e) q_r . k_c - m_r),   lse[r] = ln(2) (m_r + log2(sum p_rc))
//
// A step is 128 keys: one listed block of 128, or two of 64, each fetched by its own TMA
// load from wherever its list entry points. A work item is a pair of neighbouring 128-row
// query tiles of one (batch, head), or a range of steps of such a pair. CTAs are
// persistent: item i runs on CTA i mod gridDim, and the loads of an item start while the
// one before it ends.
//
//   warp 8      loads: the Q tiles of the item, then K and V tiles in the order the MMAs
//               read them, into a ring of slots that hold one K or one V tile each. Where
//               both tiles of the pair are at the same list entry the slot is filled once
//               and read by both ("shared"); the list decides, so no entry needs sorting.
//   warp 9      MMA issuer, one elected lane: S_t = Q_t K^T, O_t += P_t V, tiles t = 0, 1
//               in turn, so that the tensor core works on one while the other's softmax runs.
//   warps 0-3   softmax of tile 0, warps 4-7 of tile 1, a thread per row: scores from TMEM,
//               row max, p, row sum; P goes back over the S columns; O is rescaled in TMEM
//               only when the running max grew by more than 2^8. P is rounded to the type
//               of V (the MMA's operand type); sums, max and O stay fp32.
//
// TMEM (512 columns): S0 [0,128) S1 [128,256) O0 [256,384) O1 [384,512).
//
// What does not exist is never read into a result: list entries outside the sequence and
// the upper half of an odd last step load zeros (a TMA box behind the end of the tensor),
// and their scores are replaced by -inf. Keys behind k_lens inside a block may hold NaN:
// their scores are replaced, and their V rows are overwritten with zeros in shared memory
// before the tensor core sees them (0 * NaN is NaN).
//
// Every mbarrier wait is bounded; on expiry the status word gets kStatusAttentionTimeout,
// the CTA's abort flag is raised and all roles unwind, free TMEM and return.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <cmath>
#include <cstdio>
#include <cstring>

#include "attention_ptx.cuh"
#include "common.cuh"

namespace h3b {
namespace attn {
namespace sparse {

constexpr int kTile = 128;  // query rows per tile and keys per step
constexpr int kTiles = 2;
constexpr int kSoftmaxWarps = 4 * kTiles;
constexpr int kThreads = (kSoftmaxWarps + 2) * 32;
constexpr int kLoadWarp = kSoftmaxWarps;
constexpr int kMmaWarp = kSoftmaxWarps + 1;
constexpr uint32_t kHalfBytes = kTile * 128;  // 128 rows x 64 columns, 128-byte swizzle
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemS = 0;    // + t*128
constexpr uint32_t kTmemO = 256;  // + t*128
// Rescale O only when the running row max (log2 units) grew by more than this; P then
// stays within 2^8, exact in the fp32 accumulator and inside fp16's range.
constexpr float kRescaleThreshold = 8.0f;

template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;
  static constexpr uint32_t kTileBytes = kHalves * kHalfBytes;
  // Slots: what fits beside the two Q tiles (five of 32 KB at D = 128).
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr uint32_t kSmemQ = 0;
  static constexpr uint32_t kSmemRing = kTiles * kTileBytes;
  static constexpr uint32_t kSmemBar = kSmemRing + kSlots * kTileBytes;
  // qfull[2] qempty[2] full[slots] empty[slots] s[2] p[2][2] o[2] fix
  static constexpr int kNumBars = 2 * kTiles + 2 * kSlots + 4 * kTiles + 1;
  static constexpr uint32_t kSmemShared = kSmemBar + kNumBars * 8;  // u32 per slot
  static constexpr uint32_t kSmemTail = kSmemShared + kSlots * 4;   // tmem slot, abort flag
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
  // Items [0, n_full) are whole units; unit n_full + u is split into `splits` items of
  // steps_per_split steps, which write unnormalised fp32 O and (max, sum) to ws.
  int pairs, n_items, n_full, splits, steps_per_split;
  float* ws;
};

template <int D>
constexpr int kWsTileFloats = kTile * D + 2 * kTile;

__device__ __forceinline__ int rows_of(const int32_t* lens, int b, int seq) {
  if (lens == nullptr) return seq;
  const int n = lens[b];
  return n < 0 ? 0 : (n > seq ? seq : n);
}

// One item: which (batch, head, pair), which lists and which steps of them.
template <int SUB>
struct Item {
  int batch, head, pair, split;  // split < 0: a whole unit
  int q_rows, k_rows;            // rows that exist
  int step0;
  int entries[kTiles];           // list entries of tile t from step0 on
  int steps[kTiles];
  const int32_t* list[kTiles];   // from step0 on

  __device__ __forceinline__ void load(const Params& p, int item) {
    int unit = item, rank = 0;
    split = -1;
    if (item >= p.n_full) {
      const int r = item - p.n_full;
      unit = p.n_full + r / p.splits;
      rank = r % p.splits;
      split = r;
    }
    pair = unit % p.pairs;
    const int bh = unit / p.pairs;
    head = bh % p.heads;
    batch = bh / p.heads;
    q_rows = rows_of(p.q_lens, batch, p.seq_q);
    k_rows = rows_of(p.k_lens, batch, p.seq_k);
    step0 = split < 0 ? 0 : rank * p.steps_per_split;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int tile = kTiles * pair + t;
      entries[t] = 0;
      list[t] = p.indices;
      if (tile * kTile < q_rows) {
        const int64_t at = (int64_t)bh * p.nq + tile / p.tiles_per_list;
        int n = p.counts != nullptr ? p.counts[at] : p.list_len;
        n = min(max(n, 0), p.list_len) - step0 * SUB;
        if (split >= 0) n = min(n, p.steps_per_split * SUB);
        entries[t] = max(n, 0);
        list[t] = p.indices + at * p.list_len + step0 * SUB;
      }
      steps[t] = (entries[t] + SUB - 1) / SUB;
    }
  }
};

// Keys of a listed block that exist: 0 for an entry that names no block.
__device__ __forceinline__ int block_keys(int entry, int block_k, int nk, int k_rows) {
  return (unsigned)entry < (unsigned)nk ? max(0, min(block_k, k_rows - entry * block_k)) : 0;
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

template <bool FP16, int D, int BK>
__global__ void __launch_bounds__(kThreads, 1)
    sparse_fwd(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map, const Params prm) {
  using L = Layout<D>;
  constexpr int kSub = kTile / BK;  // list entries per step
  constexpr int kSlots = L::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bars = sbase + L::kSmemBar;
  auto bar_qfull = [&](int t) { return bars + 8u * t; };
  auto bar_qempty = [&](int t) { return bars + 8u * (kTiles + t); };
  auto bar_full = [&](int s) { return bars + 8u * (2 * kTiles + s); };
  auto bar_empty = [&](int s) { return bars + 8u * (2 * kTiles + kSlots + s); };
  auto bar_s = [&](int t) { return bars + 8u * (2 * kTiles + 2 * kSlots + t); };
  auto bar_p = [&](int t, int h) {
    return bars + 8u * (2 * kTiles + 2 * kSlots + kTiles + 2 * t + h);
  };
  auto bar_o = [&](int t) { return bars + 8u * (2 * kTiles + 2 * kSlots + 3 * kTiles + t); };
  const uint32_t bar_fix = bars + 8u * (2 * kTiles + 2 * kSlots + 4 * kTiles);
  volatile uint32_t* shared_flag = reinterpret_cast<uint32_t*>(smem + L::kSmemShared);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSmemTail);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(bar_qfull(t), 1);
      mbar_init(bar_qempty(t), 1);
      mbar_init(bar_s(t), 1);
      mbar_init(bar_p(t, 0), 4 * 32);
      mbar_init(bar_p(t, 1), 4 * 32);
      mbar_init(bar_o(t), 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    mbar_init(bar_fix, 1);
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

  // Both sides of the ring walk it in the same order; a slot index and its phase parity.
  struct Ring {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
    }
  };

  if (warp == kLoadWarp) {
    // ---------------- loads: the whole warp walks, one lane issues ----------------
    Ring ring;
    uint32_t q_phase[kTiles] = {0, 0};  // parity of the next qempty wait, minus one use
    uint32_t fix_phase = 0;
    bool ok = true;
    auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, prm.status));
    };
    for (int item = blockIdx.x; item < prm.n_items && ok; item += gridDim.x) {
      Item<kSub> it;
      it.load(prm, item);
      const int kv_head = it.head / prm.group;
      // List entries ahead: lane l holds entry base + l of tile t's list.
      int chunk[kTiles], chunk_base[kTiles];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        chunk_base[t] = 0;
        chunk[t] = lane < it.entries[t] ? it.list[t][lane] : -1;
      }
      auto entry = [&](int t, int e) -> int {  // e never decreases by more than a chunk
        if (e >= it.entries[t]) return -1;
        if (e < chunk_base[t] || e >= chunk_base[t] + 32) {
          chunk_base[t] = e & ~31;
          chunk[t] = chunk_base[t] + lane < it.entries[t] ? it.list[t][chunk_base[t] + lane] : -1;
        }
        return __shfl_sync(0xffffffffu, chunk[t], e & 31);
      };
      // K or V rows of step `step` of tile t into the next slot.
      auto push = [&](const CUtensorMap* map, int t, int step, bool is_v, bool shared) -> bool {
        if (!wait_all(bar_empty(ring.slot), ring.phase ^ 1)) return false;
        const uint32_t dst = sbase + L::kSmemRing + ring.slot * L::kTileBytes;
        const uint32_t full = bar_full(ring.slot);
        int row[kSub], keys[kSub];
        bool cut = false;
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const int e = entry(t, step * kSub + s);
          keys[s] = block_keys(e, BK, prm.nk, it.k_rows);
          row[s] = keys[s] > 0 ? e * BK : prm.seq_k;  // behind the end: zeros
          cut = cut || (is_v && keys[s] > 0 && keys[s] < BK && it.k_rows < prm.seq_k);
        }
        if (elect_one()) {
          shared_flag[ring.slot] = shared ? 1u : 0u;
          const uint32_t bar = cut ? bar_fix : full;
          mbar_expect_tx(bar, L::kTileBytes);
#pragma unroll
          for (int s = 0; s < kSub; ++s)
#pragma unroll
            for (int h = 0; h < L::kHalves; ++h)
              tma_load_4d(dst + h * kHalfBytes + s * BK * 128, map, bar, 64 * h, kv_head, row[s],
                          it.batch);
        }
        __syncwarp();
        if (cut) {
          // V rows behind the last key: zeros, then hand the slot over.
          if (!wait_all(bar_fix, fix_phase)) return false;
          fix_phase ^= 1;
#pragma unroll
          for (int s = 0; s < kSub; ++s)
            for (int i = lane; i < (BK - keys[s]) * 8 * L::kHalves; i += 32) {
              const int r = keys[s] + i / (8 * L::kHalves), c = i % (8 * L::kHalves);
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(
                               dst + (c >> 3) * kHalfBytes + (s * BK + r) * 128 + (c & 7) * 16),
                           "r"(0)
                           : "memory");
            }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (elect_one()) mbar_arrive(full);
          __syncwarp();
        }
        ring.next();
        return true;
      };
      auto same = [&](int step) -> bool {  // both tiles at the same entries
        if (step >= it.steps[0] || step >= it.steps[1]) return false;
        bool eq = true;
#pragma unroll
        for (int s = 0; s < kSub; ++s)
          eq = (entry(0, step * kSub + s) == entry(1, step * kSub + s)) && eq;
        return eq;
      };
      bool share = same(0);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        if (it.steps[t] == 0 || !ok) continue;
        ok = wait_all(bar_qempty(t), q_phase[t] ^ 1);
        if (!ok) break;
        q_phase[t] ^= 1;
        if (elect_one()) {
          const uint32_t dst = sbase + L::kSmemQ + t * L::kTileBytes;
          mbar_expect_tx(bar_qfull(t), L::kTileBytes);
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h)
            tma_load_4d(dst + h * kHalfBytes, &q_map, bar_qfull(t), 64 * h, it.head,
                        (kTiles * it.pair + t) * kTile, it.batch);
        }
        __syncwarp();
        if (t == 0 || !share) ok = push(&k_map, t, 0, false, share);
      }
      const int steps = max(it.steps[0], it.steps[1]);
      for (int j = 0; j < steps && ok; ++j) {
        const bool share_next = same(j + 1);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          if (j >= it.steps[t] || !ok) continue;
          if (t == 0 || !share) ok = push(&v_map, t, j, true, share);
          if (ok && j + 1 < it.steps[t] && (t == 0 || !share_next))
            ok = push(&k_map, t, j + 1, false, share_next);
        }
        share = share_next;
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------- MMA issuer ----------------
    constexpr uint32_t idesc_qk = instr_desc(FP16, kTile, false);
    constexpr uint32_t idesc_pv = instr_desc(FP16, D, true);
    auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag, prm.status));
    };
    const uint64_t q_desc0 = smem_desc(sbase + L::kSmemQ, 16, 1024);
    const uint64_t k_desc0 = smem_desc(sbase + L::kSmemRing, 16, 1024);
    const uint64_t v_desc0 = smem_desc(sbase + L::kSmemRing, kHalfBytes, 1024);
    Ring ring;
    uint32_t q_phase[kTiles] = {0, 0}, p_phase[kTiles] = {0, 0};
    int k_held = 0;  // K slot tile 0 left for tile 1
    bool ok = true;
    // Takes the next slot of the ring and says whether both tiles read it.
    auto take = [&](bool& shared) -> int {
      if (!wait_all(bar_full(ring.slot), ring.phase)) {
        ok = false;
        return 0;
      }
      tc_fence_after();
      const int slot = ring.slot;
      shared = shared_flag[slot] != 0;
      ring.next();
      return slot;
    };
    auto commit = [&](uint32_t bar) {
      if (elect_one()) mma_commit(bar);
      __syncwarp();
    };
    for (int item = blockIdx.x; item < prm.n_items && ok; item += gridDim.x) {
      Item<kSub> it;
      it.load(prm, item);
      bool share = false, share_next = false;
      auto issue_s = [&](int t, int step, bool& shared) {
        const int slot = t == 1 && shared ? k_held : take(shared);
        if (!ok) return;
        if (t == 0) k_held = slot;
        const uint64_t qd = q_desc0 + (uint64_t)((t * L::kTileBytes) >> 4);
        const uint64_t kd = k_desc0 + (uint64_t)((slot * L::kTileBytes) >> 4);
        const uint32_t d = tmem + kTmemS + t * 128;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = (uint64_t)(((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4);
            mma_ss(d, qd + off, kd + off, idesc_qk, kk > 0 ? 1u : 0u);
          }
          mma_commit(bar_s(t));
          if (t == 1 || !shared) mma_commit(bar_empty(slot));
          if (step + 1 == it.steps[t]) mma_commit(bar_qempty(t));
        }
        __syncwarp();
      };
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        if (it.steps[t] == 0 || !ok) continue;
        ok = wait_all(bar_qfull(t), q_phase[t]);
        if (!ok) break;
        q_phase[t] ^= 1;
        tc_fence_after();
        issue_s(t, 0, share);
      }
      const int steps = max(it.steps[0], it.steps[1]);
      int v_slot = 0;
      for (int j = 0; j < steps && ok; ++j) {
        share_next = false;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          if (j >= it.steps[t] || !ok) continue;
          // O_t += P_t V in two 64-key halves as the softmax hands them over.
          if (t == 0 || !share) {
            bool v_shared = false;
            v_slot = take(v_shared);
            if (!ok) break;
          }
          const uint64_t vd = v_desc0 + (uint64_t)((v_slot * L::kTileBytes) >> 4);
          const uint32_t d = tmem + kTmemO + t * 128;
#pragma unroll
          for (int h = 0; h < 2 && ok; ++h) {
            ok = wait_all(bar_p(t, h), p_phase[t]);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k4 = 0; k4 < 4; ++k4) {
                const int kk = h * 4 + k4;
                mma_ts(d, tmem + kTmemS + t * 128 + kk * 8, vd + (uint64_t)((kk * 2048) >> 4),
                       idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
          p_phase[t] ^= 1;
          if (t == 1 || !share) commit(bar_empty(v_slot));
          if (j + 1 < it.steps[t]) {
            issue_s(t, j + 1, share_next);
          } else {
            commit(bar_o(t));
          }
        }
        share = share_next;
      }
    }
  } else {
    // ---------------- softmax: warp -> (tile, lane quadrant), thread -> query row ----------------
    const int t = warp >> 2;
    const int quad = warp & 3;
    const int row_in_tile = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t t_s = tmem + lanes + kTmemS + t * 128;
    const uint32_t t_o = tmem + lanes + kTmemO + t * 128;
    const float c = prm.scale_log2;
    const float2 c2 = make_float2(c, c);
    uint32_t s_phase = 0, o_phase = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < prm.n_items && ok; item += gridDim.x) {
      Item<kSub> it;
      it.load(prm, item);
      const int n_steps = it.steps[t];
      const int32_t* list = it.list[t];
      float m_use = -INFINITY;  // running row max, log2 units, that P is taken against
      float l_sum = 0.f;
      int e_next[kSub];
      auto fetch = [&](int step) {
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const int e = step * kSub + s;
          e_next[s] = e < it.entries[t] ? __ldg(list + e) : -1;
        }
      };
      fetch(0);
      for (int j = 0; j < n_steps && ok; ++j) {
        int keys[kSub];
        bool whole = true;
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          keys[s] = block_keys(e_next[s], BK, prm.nk, it.k_rows);
          whole = whole && keys[s] == BK;
        }
        fetch(j + 1);
        ok = wait_bar(bar_s(t), s_phase, abort_flag, prm.status);
        // tcgen05.ld/st below are warp-collective.
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        s_phase ^= 1;
        tc_fence_after();
        uint32_t sv[4][32];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) tmem_ld32(t_s + 32 * q4, sv[q4]);
        tmem_ld_wait(sv[0]);
        tmem_pin(sv[1]);
        tmem_pin(sv[2]);
        tmem_pin(sv[3]);
        // Column 32*q4 + i exists if it is below the keys of its block.
        auto mask = [&](int q4) {
          const int limit = (kSub == 1 || q4 < 2) ? keys[0] : BK + keys[kSub - 1];
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (32 * q4 + i >= limit) sv[q4][i] = __float_as_uint(-INFINITY);
        };
        if (!whole) {
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) mask(q4);
        }
        float2 acc[2];
        uint32_t pk[32];
        auto exponentiate = [&](int h, float m) {
          const float base = m == -INFINITY ? 0.f : m;  // nothing seen yet: all p are 0
          const float2 nm2 = make_float2(-base, -base);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int key = 64 * h + 2 * i;
            const uint32_t* src = sv[key >> 5] + (key & 31);
            const float2 x = __ffma2_rn(
                make_float2(__uint_as_float(src[0]), __uint_as_float(src[1])), c2, nm2);
            float2 p;
            p.x = ex2(x.x);
            p.y = ex2(x.y);
            acc[i & 1] = __fadd2_rn(acc[i & 1], p);
            pk[i] = pack_pair<FP16>(p.x, p.y);
          }
        };
        // The row max and, independent of it, the first half of P against the running
        // max; that half is redone when the max moved by more than the threshold.
        float mx[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          const uint32_t* r = sv[a >> 1] + (a & 1) * 16;
          float m = max3(__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[2]));
#pragma unroll
          for (int k = 3; k < 15; k += 2)
            m = max3(m, __uint_as_float(r[k]), __uint_as_float(r[k + 1]));
          mx[a] = fmaxf(m, __uint_as_float(r[15]));
        }
        acc[0] = acc[1] = make_float2(0.f, 0.f);
        exponentiate(0, m_use);
        const float row_max =
            fmaxf(max3(mx[0], mx[1], mx[2]), max3(mx[3], max3(mx[4], mx[5], mx[6]), mx[7]));
        const float m_new = row_max * c;
        const bool need = m_new > m_use + kRescaleThreshold;
        if (__any_sync(0xffffffffu, need)) {
          const float m_next = need ? m_new : m_use;
          if (j > 0) {
            // The PV of the step before is complete: the commit of this S covers it.
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
          // S columns [0, 64) are still intact.
          tmem_ld32(t_s, sv[0]);
          tmem_ld32(t_s + 32, sv[1]);
          tmem_ld_wait(sv[0]);
          tmem_pin(sv[1]);
          if (!whole) {
            mask(0);
            mask(1);
          }
          acc[0] = acc[1] = make_float2(0.f, 0.f);
          exponentiate(0, m_use);
        }
        // P of keys [64h, 64h+64) -> S columns [32h, 32h+32), already read.
        tmem_st32(t_s, pk);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar_p(t, 0));
        exponentiate(1, m_use);
        tmem_st32(t_s + 32, pk);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar_p(t, 1));
        l_sum += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
      }
      // ---------------- epilogue ----------------
      if (ok && n_steps > 0) {
        ok = wait_bar(bar_o(t), o_phase, abort_flag, prm.status);
        ok = __all_sync(0xffffffffu, ok);
        o_phase ^= 1;
      }
      if (!ok) break;
      tc_fence_after();
      const int row = (kTiles * it.pair + t) * kTile + row_in_tile;
      const bool live = row < it.q_rows;
      if (it.split >= 0) {
        float* ws = prm.ws + ((int64_t)it.split * kTiles + t) * kWsTileFloats<D>;
        if (n_steps > 0) {
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
          *reinterpret_cast<float2*>(ws + kTile * D + 2 * row_in_tile) = make_float2(m_use, l_sum);
        continue;
      }
      const float inv_l = live && l_sum != 0.f ? 1.f / l_sum : 0.f;
      uint16_t* dst = row < prm.seq_q
                          ? reinterpret_cast<uint16_t*>(prm.out) +
                                (int64_t)it.batch * prm.o_batch_stride +
                                (int64_t)row * prm.o_row_stride +
                                (int64_t)it.head * prm.o_head_stride
                          : nullptr;
#pragma unroll 1
      for (int q4 = 0; q4 < D / 32; ++q4) {
        uint32_t o[32];
        if (n_steps > 0) {
          tmem_ld32(t_o + 32 * q4, o);
          tmem_ld_wait(o);
        }
        if (n_steps == 0 || !live || l_sum == 0.f) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (dst != nullptr) {
#pragma unroll
          for (int v8 = 0; v8 < 4; ++v8) {
            uint4 u;
            u.x = pack_pair<FP16>(__uint_as_float(o[v8 * 8 + 0]) * inv_l,
                                  __uint_as_float(o[v8 * 8 + 1]) * inv_l);
            u.y = pack_pair<FP16>(__uint_as_float(o[v8 * 8 + 2]) * inv_l,
                                  __uint_as_float(o[v8 * 8 + 3]) * inv_l);
            u.z = pack_pair<FP16>(__uint_as_float(o[v8 * 8 + 4]) * inv_l,
                                  __uint_as_float(o[v8 * 8 + 5]) * inv_l);
            u.w = pack_pair<FP16>(__uint_as_float(o[v8 * 8 + 6]) * inv_l,
                                  __uint_as_float(o[v8 * 8 + 7]) * inv_l);
            *reinterpret_cast<uint4*>(dst + 32 * q4 + v8 * 8) = u;
          }
        }
      }
      if (dst != nullptr && prm.lse != nullptr)
        prm.lse[((int64_t)it.batch * prm.heads + it.head) * prm.seq_q + row] =
            live && l_sum != 0.f ? (m_use + log2f(l_sum)) * 0.6931471805599453f : -INFINITY;
    }
  }

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

// Joins the parts of the split units: one warp per query row, D/32 columns per lane.
// O = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.
template <bool FP16, int D>
__global__ void __launch_bounds__(256) sparse_combine(const Params prm, int split_units) {
  const int gw = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  constexpr int kUnitRows = kTiles * kTile;
  const int unit_rows = min(kUnitRows, prm.seq_q);
  if (gw >= split_units * unit_rows) return;
  const int ui = gw / unit_rows;
  const int rr = gw - ui * unit_rows;
  const int t = rr / kTile;
  const int r_in_tile = rr - t * kTile;
  const int unit = prm.n_full + ui;
  const int bh = unit / prm.pairs;
  const int head = bh % prm.heads;
  const int batch = bh / prm.heads;
  const int row = unit % prm.pairs * kUnitRows + rr;
  if (row >= prm.seq_q) return;
  const bool live = row < rows_of(prm.q_lens, batch, prm.seq_q);
  auto part = [&](int s) {
    return prm.ws + ((int64_t)(ui * prm.splits + s) * kTiles + t) * kWsTileFloats<D>;
  };
  constexpr int kCols = D / 32;
  float m_max = -INFINITY, l_tot = 0.f, acc[kCols] = {};
  if (live) {
    for (int s = 0; s < prm.splits; ++s) {
      const float2 ml = *reinterpret_cast<const float2*>(part(s) + kTile * D + 2 * r_in_tile);
      m_max = fmaxf(m_max, ml.x);
    }
    for (int s = 0; s < prm.splits; ++s) {
      const float2 ml = *reinterpret_cast<const float2*>(part(s) + kTile * D + 2 * r_in_tile);
      if (ml.y == 0.f) continue;  // a part without keys wrote no O
      const float w = ex2(ml.x - m_max);
      l_tot += w * ml.y;
      const float* o = part(s) + r_in_tile * D + lane * kCols;
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] += w * o[i];
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
  int pairs, units, n_full, splits, steps_per_split, items, split_units;
  int64_t ws_bytes;
};

// Whole units fill waves of SMs; when the last wave would leave at least half of them
// idle, its units are split along their lists.
Plan make_plan(int64_t batch, int64_t seq_q, int64_t heads, int64_t head_dim, int64_t block_k,
               int64_t list_len) {
  Plan pl{};
  pl.pairs = (int)((seq_q + kTiles * kTile - 1) / (kTiles * kTile));
  pl.units = (int)(pl.pairs * heads * batch);
  const int sub = (int)(kTile / block_k);
  const int steps = (int)((list_len + sub - 1) / sub);
  const int sms = num_sms();
  const int rem = pl.units % sms;
  pl.splits = 1;
  pl.steps_per_split = steps;
  pl.n_full = pl.items = pl.units;
  if (rem > 0 && 2 * rem <= sms && steps >= 2) {
    const int want = std::min(std::min(sms / rem, 32), steps);
    pl.steps_per_split = (steps + want - 1) / want;
    pl.splits = (steps + pl.steps_per_split - 1) / pl.steps_per_split;
  }
  if (pl.splits >= 2) {
    pl.split_units = rem;
    pl.n_full = pl.units - rem;
    pl.items = pl.n_full + rem * pl.splits;
    pl.ws_bytes = (int64_t)rem * pl.splits * kTiles * (kTile * head_dim + 2 * kTile) * 4;
  } else {
    pl.splits = 1;
    pl.steps_per_split = steps;
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

template <bool FP16, int D, int BK>
int launch(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const Params& p,
           int split_units, cudaStream_t stream) {
  static ContextSlot slots[kMaxDevices];
  cudaError_t e = cudaErrorInvalidDevice;
  if (context_cached(slots, [&]() -> void* {
        e = cudaFuncSetAttribute(sparse_fwd<FP16, D, BK>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)Layout<D>::kSmemAlloc);
        return e == cudaSuccess ? reinterpret_cast<void*>(1) : nullptr;
      }) == nullptr) {
    set_error(std::string("h3b_block_sparse_attention: cannot reserve shared memory: ") +
              cudaGetErrorString(e));
    return H3B_ERR_CUDA;
  }
  const unsigned grid = (unsigned)std::min(p.n_items, num_sms());
  sparse_fwd<FP16, D, BK><<<grid, kThreads, Layout<D>::kSmemAlloc, stream>>>(qm, km, vm, p);
  int rc = check_launch("h3b_block_sparse_attention");
  if (rc != H3B_OK || split_units == 0) return rc;
  const int rows = split_units * std::min(kTiles * kTile, p.seq_q);
  sparse_combine<FP16, D><<<(unsigned)((rows + 7) / 8), 256, 0, stream>>>(p, split_units);
  return check_launch("h3b_block_sparse_attention");
}

template <bool FP16>
int launch_dims(int64_t head_dim, int64_t block_k, const CUtensorMap& qm, const CUtensorMap& km,
                const CUtensorMap& vm, const Params& p, int split_units, cudaStream_t s) {
  if (head_dim == 128)
    return block_k == 128 ? launch<FP16, 128, 128>(qm, km, vm, p, split_units, s)
                          : launch<FP16, 128, 64>(qm, km, vm, p, split_units, s);
  return block_k == 128 ? launch<FP16, 64, 128>(qm, km, vm, p, split_units, s)
                        : launch<FP16, 64, 64>(qm, km, vm, p, split_units, s);
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
  *bytes_out = h3b::attn::sparse::make_plan(batch, seq_q, heads, head_dim, block_k, list_len).ws_bytes;
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
  H3B_REQUIRE(seq_q < (1LL << 31) - 256 && seq_k < (1LL << 31) - 256 && list_len < (1LL << 30) &&
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
                     k_head_stride, (int)block_k, fp16, "k")) != H3B_OK)
    return rc;
  if ((rc = make_map(&vm, v, batch, seq_k, kv_heads, head_dim, v_batch_stride, v_row_stride,
                     v_head_stride, (int)block_k, fp16, "v")) != H3B_OK)
    return rc;
  Plan pl = make_plan(batch, seq_q, heads, head_dim, block_k, list_len);
  if (pl.ws_bytes > 0 && (workspace == nullptr || workspace_bytes < pl.ws_bytes ||
                          !h3b::aligned16(workspace))) {
    // No (or too small a) workspace: run every unit whole.
    pl.splits = 1;
    pl.split_units = 0;
    pl.n_full = pl.items = pl.units;
  }
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
  p.steps_per_split = pl.steps_per_split;
  p.ws = reinterpret_cast<float*>(workspace);
  return fp16 ? launch_dims<true>(head_dim, block_k, qm, km, vm, p, pl.split_units, stream)
              : launch_dims<false>(head_dim, block_k, qm, km, vm, p, pl.split_units, stream);
}
