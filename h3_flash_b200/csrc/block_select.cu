// Which key blocks each block of queries attends to: mean query and mean key of every
// block, their products, the top_k best per query block.
//
//   Qm[i] = mean of the rows of query block i that exist     (fp64 sum, held in fp32)
//   Km[j] = mean of the rows of key block j that exist       (the same)
//   s[i, j] = Qm[i] . Km[j]                                  (fp64)
//   list[i] = the top_k blocks by (kept, s, lowest index), written in ascending order
//
// The choice is discrete, so scores are compared where rounding cannot move them: a mean
// of at most 256 16-bit values is summed in fp64 and the products of two fp32 means are
// exact in fp64, which leaves 2^-52 relative in a score. Two devices, two batch layouts
// or another summation order then choose alike. Most of it is done in fp32 all the same:
// only scores too close to the border for fp32 to tell are taken in fp64 (score_select).
//
// Two kernels. block_means reads q and k once (bound by HBM: everything else is small);
// one warp per (block, head), heads of one block in neighbouring warps so that whole rows
// are read together. score_select holds the scores of up to 16 query blocks in shared
// memory as order-preserving keys and selects with one warp per row.
#include <cuda_fp16.h>

#include <cstdio>

#include "common.cuh"

namespace h3b {
namespace select {

constexpr int kMeanWarps = 4;

struct MeanSide {
  const void* x;
  float* mean;  // q: [batch, heads, blocks, D]; k: [batch, heads, D, pitch]
  int64_t batch_stride, row_stride, head_stride;
  const int32_t* lens;
  int seq, heads, block, blocks, pitch;
  bool transposed;
  int64_t warps;  // batch * blocks * heads
};

struct MeanArgs {
  MeanSide side[2];
  int64_t total;
};

__device__ __forceinline__ int rows_of(const int32_t* lens, int b, int seq) {
  if (lens == nullptr) return seq;
  const int n = lens[b];
  return n < 0 ? 0 : (n > seq ? seq : n);
}

template <bool FP16>
__device__ __forceinline__ void add8(double (&acc)[8], uint4 u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float2 f;
    if (FP16) {
      f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
    } else {
      f = make_float2(bf16lo(w[j]), bf16hi(w[j]));
    }
    acc[2 * j] += (double)f.x;
    acc[2 * j + 1] += (double)f.y;
  }
}

// One warp per (batch, block, head): D/8 lanes hold the columns of a row, the others further rows.
template <bool FP16, int D>
__global__ void __launch_bounds__(kMeanWarps * 32) block_means(MeanArgs a) {
  int64_t w = (int64_t)blockIdx.x * kMeanWarps + (threadIdx.x >> 5);
  if (w >= a.total) return;
  const int lane = threadIdx.x & 31;
  const bool is_k = w >= a.side[0].warps;
  const MeanSide& s = a.side[is_k ? 1 : 0];
  if (is_k) w -= a.side[0].warps;
  const int head = (int)(w % s.heads);
  const int block = (int)(w / s.heads % s.blocks);
  const int b = (int)(w / s.heads / s.blocks);
  constexpr int kLanes = D / 8;          // lanes per row
  constexpr int kRows = 32 / kLanes;     // rows per load
  constexpr int kUnroll = 8;
  const int col = (lane % kLanes) * 8;
  const int row0 = block * s.block;
  const int count = min(s.block, rows_of(s.lens, b, s.seq) - row0);
  double acc[8] = {};
  const char* base = (const char*)s.x + 2 * ((int64_t)b * s.batch_stride +
                                             (int64_t)row0 * s.row_stride +
                                             (int64_t)head * s.head_stride + col);
  for (int r0 = lane / kLanes; r0 < count; r0 += kRows * kUnroll) {
    uint4 u[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int r = r0 + i * kRows;
      u[i] = r < count ? ld_cached(base + 2 * (int64_t)r * s.row_stride) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) add8<FP16>(acc, u[i]);
  }
#pragma unroll
  for (int o = 16; o >= kLanes; o >>= 1)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
  if (lane >= kLanes) return;
  const double n = count > 0 ? (double)count : 1.0;
  if (s.transposed) {
    float* out = s.mean + (((int64_t)b * s.heads + head) * D + col) * s.pitch + block;
#pragma unroll
    for (int j = 0; j < 8; ++j) out[(int64_t)j * s.pitch] = (float)(acc[j] / n);
  } else {
    float* out = s.mean + (((int64_t)b * s.heads + head) * s.blocks + block) * D + col;
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = (float)(acc[j] / n);
  }
}

struct SelectArgs {
  int32_t* indices;
  int32_t* counts;
  const float* q_mean;
  const float* k_mean;
  const int32_t* q_lens;
  const int32_t* k_lens;
  const uint8_t* keep;
  int heads, kv_heads, seq_q, seq_k, block_q, block_k, nq, nk, pitch, top_k;
  int row_groups;  // CTAs per (batch, head)
};

// Order-preserving keys of a score. -0 and +0 are the same score, NaN ranks as -inf.
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) s = -INFINITY;
  s += 0.0;
  const long long bits = __double_as_longlong(s);
  return bits < 0 ? ~(unsigned long long)bits : (unsigned long long)bits | (1ull << 63);
}
__device__ __forceinline__ uint32_t score_key(float s) {
  if (s != s) s = -INFINITY;
  s += 0.f;
  const int bits = __float_as_int(s);
  return bits < 0 ? ~(uint32_t)bits : (uint32_t)bits | (1u << 31);
}
__device__ __forceinline__ float key_score(uint32_t key) {
  return __int_as_float((key >> 31) ? (int)(key & 0x7fffffffu) : (int)~key);
}
// Besides scores: 0 for blocks that are out, kInKey for blocks that are in.
constexpr uint32_t kInKey = 0xffffffffu;

// Highest fp64 key t such that at least `want` of n_keys keys are >= t, and how many exceed
// it: bit by bit from the first bit in which keys differ. count(key, mask) gives the number
// of keys that equal `key` in the bits of `mask`.
template <class Count>
__device__ __forceinline__ unsigned long long kth_key(unsigned long long common, int bit,
                                                      int n_keys, int want, int& above,
                                                      unsigned long long& decided, Count count) {
  unsigned long long prefix = common;
  int equal = n_keys;
  above = 0;
  for (; bit >= 0 && above + equal > want; --bit) {
    const unsigned long long probe = prefix | (1ull << bit);
    const int n = count(probe, ~((1ull << bit) - 1ull));
    if (above + n >= want) {
      prefix = probe;
      equal = n;
    } else {
      above += n;
      equal -= n;
    }
  }
  decided = bit < 0 ? ~0ull : ~(((1ull << bit) << 1) - 1ull);  // bits of prefix above `bit`
  return prefix;
}

template <int D, int ROWS>
struct SelectShape {
  static constexpr int kThreads = ROWS == 1 ? 512 : 256;
  static constexpr int kCols = ROWS == 1 ? 1 : 2;  // columns per thread
  static constexpr int kWarps = kThreads / 32;
  // CTAs per SM that registers should allow: three of 16 rows fit in shared memory at 800 columns.
  static constexpr int kCtas = ROWS == 1 ? 2 : 3;
};
constexpr int kBins = 256;

// ROWS query blocks of one (batch, head) per CTA. Scores are first taken in fp32, whose
// rounding leaves at most E = D 2^-24 |q| max|k| (Cauchy-Schwarz). An order statistic moves
// by no more than the values do, so with T the k-th largest fp32 score, blocks above T + 2E
// are in and blocks below T - 2E are out whatever the rounding did; the few between are
// scored again in fp64 and ranked. A bound that is not finite makes every block one of those.
template <int D, int ROWS>
__global__ void __launch_bounds__(SelectShape<D, ROWS>::kThreads, SelectShape<D, ROWS>::kCtas)
    score_select(SelectArgs a) {
  using S = SelectShape<D, ROWS>;
  extern __shared__ __align__(16) unsigned char smem[];
  float* q_tile = reinterpret_cast<float*>(smem);                 // [D][ROWS]
  uint32_t* keys = reinterpret_cast<uint32_t*>(q_tile + D * ROWS);  // [ROWS][pitch]
  __shared__ unsigned int k_square;                               // bits of max |k|^2
  __shared__ int close[S::kWarps][32];                            // columns to score again
  __shared__ uint32_t bins[S::kWarps][kBins];
  const int group = blockIdx.x % a.row_groups;
  const int64_t bh = blockIdx.x / a.row_groups;
  const int head = (int)(bh % a.heads);
  const int b = (int)(bh / a.heads);
  const int row0 = group * ROWS;
  const int q_rows = rows_of(a.q_lens, b, a.seq_q);
  const int k_rows = rows_of(a.k_lens, b, a.seq_k);
  const int k_blocks = (k_rows + a.block_k - 1) / a.block_k;  // blocks that exist

  if (threadIdx.x == 0) k_square = 0u;
  for (int i = threadIdx.x; i < D * ROWS; i += S::kThreads) {
    const int r = i / D, d = i % D;
    q_tile[d * ROWS + r] = row0 + r < a.nq ? a.q_mean[(bh * a.nq + row0 + r) * D + d] : 0.f;
  }
  // More kept blocks than a list holds: only they compete, by score.
  int kept_count = 0;
  if (a.keep != nullptr)
    for (int c = threadIdx.x; c < (k_blocks + S::kThreads - 1) / S::kThreads * S::kThreads;
         c += S::kThreads)
      kept_count += __syncthreads_count(c < k_blocks && a.keep[c] != 0);
  const bool only_kept = kept_count > a.top_k;
  if (only_kept) kept_count = 0;
  __syncthreads();
  const float* km = a.k_mean +
                    ((int64_t)b * a.kv_heads + head / (a.heads / a.kv_heads)) * D * a.pitch;
  for (int col = threadIdx.x * S::kCols; col < k_blocks; col += S::kThreads * S::kCols) {
    if constexpr (S::kCols == 2) {
      // Columns col, col + 1 (the pitch is even; a column behind the last is scored and
      // ignored), rows in pairs: a pair of q comes as it lies in shared memory.
      float2 acc[ROWS / 2][2] = {}, square = make_float2(0.f, 0.f);
#pragma unroll 8
      for (int d = 0; d < D; ++d) {
        const float2 k2 = __ldg(reinterpret_cast<const float2*>(km + (int64_t)d * a.pitch + col));
        square = __ffma2_rn(k2, k2, square);
        const float2 first = make_float2(k2.x, k2.x), second = make_float2(k2.y, k2.y);
#pragma unroll
        for (int r = 0; r < ROWS / 2; r += 2) {
          const float4 q = *reinterpret_cast<const float4*>(q_tile + d * ROWS + 2 * r);
          acc[r][0] = __ffma2_rn(make_float2(q.x, q.y), first, acc[r][0]);
          acc[r][1] = __ffma2_rn(make_float2(q.x, q.y), second, acc[r][1]);
          acc[r + 1][0] = __ffma2_rn(make_float2(q.z, q.w), first, acc[r + 1][0]);
          acc[r + 1][1] = __ffma2_rn(make_float2(q.z, q.w), second, acc[r + 1][1]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = col + i;
        if (c >= k_blocks) continue;
        const bool kept = a.keep != nullptr && a.keep[c] != 0;
        if (kept || !only_kept) atomicMax(&k_square, __float_as_uint(i == 0 ? square.x : square.y));
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          keys[r * a.pitch + c] =
              only_kept && !kept ? 0u
              : kept && !only_kept ? kInKey
                                   : score_key(r % 2 == 0 ? acc[r / 2][i].x : acc[r / 2][i].y);
      }
    } else {
      float acc[ROWS] = {}, square = 0.f;
#pragma unroll 32
      for (int d = 0; d < D; ++d) {
        const float k1 = __ldg(km + (int64_t)d * a.pitch + col);
        square = fmaf(k1, k1, square);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) acc[r] = fmaf(q_tile[d * ROWS + r], k1, acc[r]);
      }
      const bool kept = a.keep != nullptr && a.keep[col] != 0;
      if (kept || !only_kept) atomicMax(&k_square, __float_as_uint(square));
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        keys[r * a.pitch + col] = only_kept && !kept ? 0u
                                  : kept && !only_kept ? kInKey : score_key(acc[r]);
    }
  }
  __syncthreads();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned below = (1u << lane) - 1u;
  for (int r = warp; r < ROWS; r += S::kWarps) {
    if (row0 + r >= a.nq) break;
    uint32_t* row = keys + r * a.pitch;
    const int64_t list = bh * a.nq + row0 + r;
    int32_t* out = a.indices + list * a.top_k;
    const bool exists = (row0 + r) * a.block_q < q_rows;
    const int want = exists ? min(a.top_k, k_blocks) : 0;
    // Calls f(column) for every lane's columns, warp-uniformly: a column >= k_blocks has no key.
    auto each = [&](auto f) {
      for (int c = lane; c < k_blocks; c += 32) f(c);
    };
    uint32_t least_in = kInKey;  // keys from here on are in
    if (want > kept_count) {
      // T, the k-th largest score: count the scores in equal bins of their range, go on
      // inside the bin that holds the k-th, rank what is left when a warp holds it. The bin
      // of a score never decreases with it, whatever the rounding.
      float low = -INFINITY, high = INFINITY;
      int left = want - kept_count;  // the rank of T among the scores in [low, high]
      uint32_t kth;
      for (;;) {
        uint32_t least = kInKey, most = 0u;
        int n = 0;
        const uint32_t low_key = score_key(low), high_key = score_key(high);
        each([&](int c) {
          const uint32_t k = row[c];
          if (k >= low_key && k <= high_key) {
            least = min(least, k);
            most = max(most, k);
            ++n;
          }
        });
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        n = __reduce_add_sync(0xffffffffu, n);
        if (least == most || left == n) {
          kth = least;
          break;
        }
        if (left == 1) {
          kth = most;
          break;
        }
        if (n <= 32) {
          int at = 0;
          for (int c0 = 0; c0 < k_blocks; c0 += 32) {
            const uint32_t k = c0 + lane < k_blocks ? row[c0 + lane] : 0u;
            const bool mine = k >= least && k <= most;
            const unsigned mask = __ballot_sync(0xffffffffu, mine);
            if (mine) bins[warp][at + __popc(mask & below)] = k;
            at += __popc(mask);
          }
          __syncwarp();
          const uint32_t mine = lane < n ? bins[warp][lane] : 0u;
          int rank = 0;
          for (int i = 0; i < n; ++i) {
            const uint32_t k = __shfl_sync(0xffffffffu, mine, i);
            rank += k > mine || (k == mine && i < lane);
          }
          const unsigned found = __ballot_sync(0xffffffffu, lane < n && rank == left - 1);
          kth = __shfl_sync(0xffffffffu, mine, __ffs((int)found) - 1);
          __syncwarp();
          break;
        }
        low = key_score(least);
        high = key_score(most);
        const float span = high - low;
        const float scale = (float)kBins / span;
        // A range too wide or too narrow for fp32: every block is scored again in fp64.
        if (!(span < INFINITY) || !(scale < INFINITY)) {
          kth = 0u;
          break;
        }
        auto bin_of = [&](uint32_t k) { return min((int)((key_score(k) - low) * scale), kBins - 1); };
        for (int i = lane; i < kBins; i += 32) bins[warp][i] = 0u;
        __syncwarp();
        each([&](int c) {
          const uint32_t k = row[c];
          if (k >= least && k <= most) atomicAdd(&bins[warp][bin_of(k)], 1u);
        });
        __syncwarp();
        // Lane l sums bins [8l, 8l + 8); from the top, the lane and then the bin that reach `left`.
        uint32_t mine[kBins / 32];
        int sum = 0;
#pragma unroll
        for (int i = 0; i < kBins / 32; ++i) {
          mine[i] = bins[warp][lane * (kBins / 32) + i];
          sum += (int)mine[i];
        }
        int up = sum;  // scores in this lane's bins and above
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int other = __shfl_down_sync(0xffffffffu, up, o);
          if (lane + o < 32) up += other;
        }
        const unsigned reach = __ballot_sync(0xffffffffu, up >= left);
        const int owner = 31 - __clz((int)reach);
        int bin = 0, over = up - sum;
        if (lane == owner) {
          bool done = false;
#pragma unroll
          for (int i = kBins / 32 - 1; i >= 0; --i) {
            if (!done && over + (int)mine[i] >= left) {
              bin = lane * (kBins / 32) + i;
              done = true;
            }
            if (!done) over += (int)mine[i];
          }
        }
        bin = __shfl_sync(0xffffffffu, bin, owner);
        left -= __shfl_sync(0xffffffffu, over, owner);
        // The bin's own range.
        uint32_t bin_least = kInKey, bin_most = 0u;
        each([&](int c) {
          const uint32_t k = row[c];
          if (k >= least && k <= most && bin_of(k) == bin) {
            bin_least = min(bin_least, k);
            bin_most = max(bin_most, k);
          }
        });
        low = key_score(__reduce_min_sync(0xffffffffu, bin_least));
        high = key_score(__reduce_max_sync(0xffffffffu, bin_most));
        __syncwarp();
      }
      float q_square = 0.f;
      for (int d = lane; d < D; d += 32) q_square += q_tile[d * ROWS + r] * q_tile[d * ROWS + r];
      q_square = warp_sum(q_square);
      // 2E, rounded up: D 2^-23 sqrt(|q|^2 |k|^2), 1% for the rounding of the norms, and the
      // underflow of D products.
      const float twice = 1.01f * D * 1.1920929e-7f * sqrtf(q_square) *
                              sqrtf(__uint_as_float(k_square)) + 1.2e-38f;
      const float t = key_score(kth);
      const bool bounded = kth != 0u && twice < INFINITY && fabsf(t) < INFINITY;
      const uint32_t hi = bounded ? score_key(__fadd_ru(t, twice)) : kInKey - 1u;
      const uint32_t lo = bounded ? score_key(__fadd_rd(t, -twice)) : 1u;
      int n_in = 0, n_close = 0;
      for (int c0 = 0; c0 < k_blocks; c0 += 32) {
        const int c = c0 + lane;
        const uint32_t k = c < k_blocks ? row[c] : 0u;
        const bool is_close = k >= lo && k <= hi;
        const unsigned mask = __ballot_sync(0xffffffffu, is_close);
        if (is_close) {
          const int at = n_close + __popc(mask & below);
          if (at < 32) close[warp][at] = c;
        }
        n_close += __popc(mask);
        n_in += __popc(__ballot_sync(0xffffffffu, k > hi));
      }
      __syncwarp();
      const int open = want - n_in;  // places left for the close ones
      least_in = hi == kInKey ? kInKey : hi + 1u;
      if (n_close == open) {
        least_in = lo;
      } else {
        // fp64 score of a column, the same sum in every lane.
        auto score = [&](int c) -> unsigned long long {
          double s = 0.0;
          for (int d = lane; d < D; d += 32)
            s = fma((double)q_tile[d * ROWS + r], (double)km[(int64_t)d * a.pitch + c], s);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          return score_key(s);
        };
        if (n_close <= 32) {
          unsigned long long mine = 0ull;
          for (int i = 0; i < n_close; ++i) {
            const unsigned long long s = score(close[warp][i]);
            if (i == lane) mine = s;
          }
          int rank = 0;  // close[] ascends: of equal scores the lower lane goes first
          for (int i = 0; i < n_close; ++i) {
            const unsigned long long s = __shfl_sync(0xffffffffu, mine, i);
            rank += s > mine || (s == mine && i < lane);
          }
          if (lane < n_close) row[close[warp][lane]] = rank < open ? kInKey : 0u;
        } else {
          // Many scores within the bound (equal blocks, say): the same search on fp64 keys,
          // which are computed again in every pass.
          auto each_close = [&](auto f) {
            for (int c0 = 0; c0 < k_blocks; c0 += 32) {
              const uint32_t k = c0 + lane < k_blocks ? row[c0 + lane] : 0u;
              unsigned mask = __ballot_sync(0xffffffffu, k >= lo && k <= hi);
              for (; mask != 0u; mask &= mask - 1u) {
                const int c = c0 + __ffs((int)mask) - 1;
                f(c, score(c));
              }
            }
          };
          unsigned long long one = 0ull, zero = 0ull;
          each_close([&](int, unsigned long long s) {
            one |= s;
            zero |= ~s;
          });
          const int top = 63 - __clzll((long long)(one & zero));  // -1: all equal
          const unsigned long long same64 = top >= 63 ? 0ull : ~((2ull << top) - 1ull);
          int above64;
          unsigned long long decided64;
          const unsigned long long prefix64 = kth_key(
              one & (top < 0 ? ~0ull : same64), top, n_close, open, above64, decided64,
              [&](unsigned long long key, unsigned long long mask) {
                int n = 0;
                each_close([&](int, unsigned long long s) { n += (s & mask) == key; });
                return n;
              });
          int ties = open - above64;
          each_close([&](int c, unsigned long long s) {
            const unsigned long long high = s & decided64;
            const bool in = high > prefix64 || (high == prefix64 && ties-- > 0);
            if (lane == (c & 31)) row[c] = in ? kInKey : 0u;
          });
        }
        __syncwarp();
      }
    }
    int done = 0;
    for (int c0 = 0; c0 < k_blocks && done < want; c0 += 32) {
      const int c = c0 + lane;
      const bool take = c < k_blocks && row[c] >= least_in;
      const unsigned mask = __ballot_sync(0xffffffffu, take);
      if (take) out[done + __popc(mask & below)] = c;
      done += __popc(mask);
    }
    for (int c = done + lane; c < a.top_k; c += 32) out[c] = -1;
    if (lane == 0) a.counts[list] = done;
  }
}

constexpr int kMaxKeyBlocks = 24576;  // scores of one query block fit in shared memory

size_t select_smem(int head_dim, int rows, int64_t pitch) {
  return 4 * (size_t)rows * (head_dim + pitch);
}

template <int D, int ROWS>
int launch_select(const SelectArgs& a, int64_t batch, size_t smem, cudaStream_t s) {
  static ContextSlot slots[kMaxDevices];
  cudaError_t e = cudaErrorInvalidDevice;
  if (context_cached(slots, [&]() -> void* {
        e = cudaFuncSetAttribute(score_select<D, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 200 * 1024);
        return e == cudaSuccess ? reinterpret_cast<void*>(1) : nullptr;
      }) == nullptr) {
    set_error(std::string("h3b_select_key_blocks: cannot reserve shared memory: ") +
              cudaGetErrorString(e));
    return H3B_ERR_CUDA;
  }
  const int64_t grid = batch * a.heads * a.row_groups;
  H3B_REQUIRE(grid <= 0x7fffffffLL, "select_key_blocks: shape exceeds launch limits");
  score_select<D, ROWS><<<(unsigned)grid, SelectShape<D, ROWS>::kThreads, smem, s>>>(a);
  return check_launch("h3b_select_key_blocks");
}

template <bool FP16, int D>
int launch_all(const MeanArgs& m, SelectArgs a, int64_t batch, cudaStream_t s) {
  const int64_t grid = (m.total + kMeanWarps - 1) / kMeanWarps;
  H3B_REQUIRE(grid <= 0x7fffffffLL, "select_key_blocks: shape exceeds launch limits");
  block_means<FP16, D><<<(unsigned)grid, kMeanWarps * 32, 0, s>>>(m);
  int rc = check_launch("h3b_select_key_blocks");
  if (rc != H3B_OK) return rc;
  // Query blocks per CTA: as many as there are and as shared memory holds; each reads the
  // key means once.
  int rows = 16;
  while (rows > 1 && (rows / 2 >= a.nq || select_smem(D, rows, a.pitch) > 200 * 1024)) rows /= 4;
  a.row_groups = (a.nq + rows - 1) / rows;
  const size_t smem = select_smem(D, rows, a.pitch);
  if (rows == 16) return launch_select<D, 16>(a, batch, smem, s);
  if (rows == 4) return launch_select<D, 4>(a, batch, smem, s);
  return launch_select<D, 1>(a, batch, smem, s);
}

}  // namespace select
}  // namespace h3b

extern "C" int h3b_select_key_blocks_workspace_size(int64_t batch, int64_t seq_q, int64_t seq_k,
                                                    int64_t heads, int64_t kv_heads,
                                                    int64_t head_dim, int64_t block_q,
                                                    int64_t block_k, int64_t* bytes_out) {
  H3B_REQUIRE(bytes_out != nullptr, "select_key_blocks_workspace_size: null output pointer");
  H3B_REQUIRE(batch >= 0 && seq_q >= 0 && seq_k >= 0 && heads >= 0 && kv_heads >= 0 &&
                  head_dim >= 0 && block_q > 0 && block_k > 0,
              "select_key_blocks: negative shape");
  const int64_t nq = (seq_q + block_q - 1) / block_q, nk = (seq_k + block_k - 1) / block_k;
  const int64_t pitch = (nk + 31) / 32 * 32;
  *bytes_out = 4 * batch * head_dim * (heads * nq + kv_heads * pitch);
  return H3B_OK;
}

extern "C" int h3b_select_key_blocks(
    int32_t* indices, int32_t* counts, const void* q, const void* k, int64_t batch, int64_t seq_q,
    int64_t seq_k, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t block_q,
    int64_t block_k, int64_t top_k, int64_t q_batch_stride, int64_t q_row_stride,
    int64_t q_head_stride, int64_t k_batch_stride, int64_t k_row_stride, int64_t k_head_stride,
    const int32_t* q_lens, const int32_t* k_lens, const uint8_t* keep, int64_t dtype,
    void* workspace, int64_t workspace_bytes, h3b_stream_t stream) {
  using namespace h3b::select;
  int64_t need = 0;
  H3B_REQUIRE(batch >= 0 && seq_q >= 0 && seq_k >= 0 && heads >= 0 && kv_heads >= 0,
              "select_key_blocks: negative shape");
  if (!(head_dim == 64 || head_dim == 128) || !(block_q == 128 || block_q == 256) ||
      !(block_k == 64 || block_k == 128) ||
      !(dtype == H3B_DTYPE_BF16 || dtype == H3B_DTYPE_FP16)) {
    h3b::set_error("h3b_select_key_blocks: needs bf16 or fp16, head_dim 64 or 128, block_q 128 or "
                   "256, block_k 64 or 128");
    return H3B_ERR_UNSUPPORTED;
  }
  if (batch == 0 || seq_q == 0 || heads == 0) return H3B_OK;
  H3B_REQUIRE(seq_k > 0, "select_key_blocks: empty key sequence");
  H3B_REQUIRE(kv_heads > 0 && heads % kv_heads == 0,
              "select_key_blocks: heads (%lld) must be a multiple of kv_heads (%lld)",
              (long long)heads, (long long)kv_heads);
  H3B_REQUIRE(seq_q < (1LL << 31) - 256 && seq_k < (1LL << 31) - 256,
              "select_key_blocks: shape exceeds launch limits");
  const int64_t nq = (seq_q + block_q - 1) / block_q, nk = (seq_k + block_k - 1) / block_k;
  H3B_REQUIRE(top_k >= 1 && top_k <= nk, "select_key_blocks: top_k (%lld) must be 1..%lld",
              (long long)top_k, (long long)nk);
  if (nk > kMaxKeyBlocks) {
    h3b::set_error("h3b_select_key_blocks: more than 24576 key blocks");
    return H3B_ERR_UNSUPPORTED;
  }
  H3B_REQUIRE(batch <= (1LL << 31) / heads && batch * heads <= (1LL << 31) / nq,
              "select_key_blocks: shape exceeds launch limits");
  H3B_REQUIRE(indices != nullptr && counts != nullptr && q != nullptr && k != nullptr,
              "select_key_blocks: null argument");
  H3B_REQUIRE(h3b::aligned16(q) && h3b::aligned16(k), "select_key_blocks: q and k must be 16-byte aligned");
  const int64_t strides[6] = {q_batch_stride, q_row_stride, q_head_stride,
                              k_batch_stride, k_row_stride, k_head_stride};
  for (int i = 0; i < 6; ++i)
    H3B_REQUIRE(strides[i] % 8 == 0 && strides[i] >= 0,
                "select_key_blocks: strides must be multiples of 8 elements");
  int rc = h3b_select_key_blocks_workspace_size(batch, seq_q, seq_k, heads, kv_heads, head_dim,
                                                block_q, block_k, &need);
  if (rc != H3B_OK) return rc;
  H3B_REQUIRE(workspace != nullptr && workspace_bytes >= need && h3b::aligned16(workspace),
              "select_key_blocks: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  const int pitch = (int)((nk + 31) / 32 * 32);
  float* q_mean = static_cast<float*>(workspace);
  float* k_mean = q_mean + batch * heads * nq * head_dim;
  MeanArgs m{};
  m.side[0] = MeanSide{q, q_mean, q_batch_stride, q_row_stride, q_head_stride, q_lens,
                       (int)seq_q, (int)heads, (int)block_q, (int)nq, 0, false, batch * nq * heads};
  m.side[1] = MeanSide{k, k_mean, k_batch_stride, k_row_stride, k_head_stride, k_lens,
                       (int)seq_k, (int)kv_heads, (int)block_k, (int)nk, pitch, true,
                       batch * nk * kv_heads};
  m.total = m.side[0].warps + m.side[1].warps;
  SelectArgs a{};
  a.indices = indices;
  a.counts = counts;
  a.q_mean = q_mean;
  a.k_mean = k_mean;
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.keep = keep;
  a.heads = (int)heads;
  a.kv_heads = (int)kv_heads;
  a.seq_q = (int)seq_q;
  a.seq_k = (int)seq_k;
  a.block_q = (int)block_q;
  a.block_k = (int)block_k;
  a.nq = (int)nq;
  a.nk = (int)nk;
  a.pitch = pitch;
  a.top_k = (int)top_k;
  if (dtype == H3B_DTYPE_FP16)
    return head_dim == 128 ? launch_all<true, 128>(m, a, batch, stream)
                           : launch_all<true, 64>(m, a, batch, stream);
  return head_dim == 128 ? launch_all<false, 128>(m, a, batch, stream)
                         : launch_all<false, 64>(m, a, batch, stream);
}
