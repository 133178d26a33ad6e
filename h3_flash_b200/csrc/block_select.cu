// Which key blocks each block of queries attends to: mean query and mean key of every
// block, their products, the top_k best per query block.
//
//   Qm[i] = mean of the rows of query block i that exist     (fp64 sum, held in fp32)
//   Km[j] = mean of the rows of key block j that exist       (the same)
//   s[i, j] = Qm[i] . Km[j]                                  (fp64)
//   list[i] = the top_k blocks by (kept, s, lowest index), written in ascending order
//
// The choice is discrete, so scores are compared where rounding hardly moves them. The fp64 sum
// of at most 256 values is exact for fp16 (multiples of 2^-24 below 2^16: 48 bits), and for bf16
// where the nonzero values of a column of a block lie within a factor of 2^37 (8 bits a value and 8
// more for the sum beside these 37). The means then do not depend on the order of summation,
// which differs between short and long sequences (block_means). (One order for both: 24 heads of
// 51,200 rows 168 us in place of 165, with D = 64 119 in place of 115.) The products of two fp32
// means are exact in fp64; their sum, always taken in one order, is off by at most
// D 2^-53 sum |Qm_i Km_j|. Blocks whose scores lie closer than that may rank either way, but the
// same way in any batch. Most of it is done in fp32 all the same: only scores too close to the
// border for fp32 to tell are taken in fp64 (block_choose).
//
// Three kernels:
//   block_means   reads q and k once; bound by HBM, and two thirds of the time at long
//                 sequences. Heads of one block lie next to each other in the grid, so that
//                 whole rows are read together. Leaves each mean in fp32, its norm, and the
//                 mean as a sum of two bf16.
//   block_scores  s in fp32 from the bf16 parts, hi hi + hi mid + mid hi, on the tensor cores
//                 (tcgen05, a tile per CTA). The query heads that share a key head are rows
//                 of one product.
//   block_choose  a warp per query block, its scores in registers: counts them in bins, ranks
//                 those next to the border. Rows that this does not settle, or of more than
//                 4096 key blocks, go through the workspace (choose_any).
// 24 heads of 51,200 rows, 80 of 800 blocks: 117, 24 and 31 us, 165 together, each kernel starting
// while the one before drains. The steps of different groups of heads in one launch, to overlap
// HBM and latencies, took 186 us with three groups and 192 us with four (173 us apart then): a
// launch costs some 12 us however little it does.
#include <cuda_fp16.h>

#include <cstdio>

#include "attention_ptx.cuh"
#include "common.cuh"

namespace h3b {
namespace select {

constexpr int kMeanWarps = 4;

// Where the means of one side (queries or keys) go: per row, D values each.
struct Means {
  float* mean;
  __nv_bfloat16* hi;
  __nv_bfloat16* mid;
  float* norm;
};

struct MeanSide {
  const void* x;
  Means out;
  int64_t batch_stride, row_stride, head_stride;
  const int32_t* lens;
  int seq, heads, block, blocks;
  int64_t blocks_total;  // batch * blocks * heads
};

struct MeanArgs {
  MeanSide side[2];
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

// WARPS warps per (batch, block, head) take turns at its rows: D/8 lanes hold the columns of a
// row, the others further rows. One warp where there are blocks enough to fill the GPU (24
// heads of 51,200 rows, 64-key blocks: 105 us, with four 155 us), four for short sequences
// (4352 rows, three heads: 4.6 us, with one 9.3 us). Eight loads of 16 bytes a lane and seven
// CTAs per SM keep HBM busy; four loads with eight CTAs (119 us), sixteen with five (122 us)
// are slower than 116 us, and so are fewer conversions to fp64, whose unit is busy 71% of the
// time: with some done on the bits by integer instructions 125 us and more.
template <bool FP16, int D, int WARPS>
__global__ void __launch_bounds__(kMeanWarps * 32, 7) block_means(const MeanArgs a) {
  __shared__ double part[WARPS > 1 ? WARPS : 1][WARPS > 1 ? D : 1];
  const int warp = threadIdx.x >> 5 & (WARPS - 1), lane = threadIdx.x & 31;
  grid_wait();
  int64_t w = (int64_t)blockIdx.x * (kMeanWarps / WARPS) + (threadIdx.x >> 5) / WARPS;
  if (w >= a.side[0].blocks_total + a.side[1].blocks_total) return;
  const bool is_k = w >= a.side[0].blocks_total;
  const MeanSide& s = a.side[is_k ? 1 : 0];
  if (is_k) w -= a.side[0].blocks_total;
  const int head = (int)(w % s.heads);
  const int block = (int)(w / s.heads % s.blocks);
  const int b = (int)(w / s.heads / s.blocks);
  constexpr int kLanes = D / 8;                     // lanes per row
  constexpr int kRows = 32 / kLanes * WARPS;       // rows per load of these warps
  constexpr int kUnroll = 8;
  const int col = (lane % kLanes) * 8;
  const int row0 = block * s.block;
  const int count = min(s.block, rows_of(s.lens, b, s.seq) - row0);
  double acc[8] = {};
  const char* base = (const char*)s.x + 2 * ((int64_t)b * s.batch_stride +
                                             (int64_t)row0 * s.row_stride +
                                             (int64_t)head * s.head_stride + col);
  for (int r0 = warp * (32 / kLanes) + lane / kLanes; r0 < count; r0 += kRows * kUnroll) {
    uint4 u[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int r = r0 + i * kRows;
      // (Not through the read-only path: a kernel before this one in the stream may have written
      // these rows while this grid had already started.)
      u[i] = r < count ? *reinterpret_cast<const uint4*>(base + 2 * (int64_t)r * s.row_stride)
                       : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) add8<FP16>(acc, u[i]);
  }
#pragma unroll
  for (int o = 16; o >= kLanes; o >>= 1)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
  if (WARPS > 1) {
    if (lane < kLanes) {
#pragma unroll
      for (int j = 0; j < 8; ++j) part[warp][col + j] = acc[j];
    }
    __syncthreads();
    if (warp != 0) return;
    if (lane < kLanes) {
#pragma unroll
      for (int i = 1; i < WARPS; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += part[i][col + j];
    }
  }
  grid_done();
  const int64_t out = ((int64_t)b * s.heads + head) * s.blocks + block;
  double square = 0.0;
  if (lane < kLanes) {
    // (A power of two divides exactly as its reciprocal multiplies.)
    const bool exact = (count & (count - 1)) == 0;
    const double n = count > 0 ? (double)count : 1.0;
    const double inv = 1.0 / (double)(count > 0 ? count : 1);
    float m[8], hi[8], mid[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = (float)(exact ? acc[j] * inv : acc[j] / n);
      hi[j] = __bfloat162float(__float2bfloat16_rn(m[j]));
      mid[j] = m[j] - hi[j];
      square += (double)m[j] * (double)m[j];
    }
    float4* mean = reinterpret_cast<float4*>(s.out.mean + out * D + col);
    mean[0] = make_float4(m[0], m[1], m[2], m[3]);
    mean[1] = make_float4(m[4], m[5], m[6], m[7]);
    *reinterpret_cast<uint4*>(s.out.hi + out * D + col) = pack8(hi);
    *reinterpret_cast<uint4*>(s.out.mid + out * D + col) = pack8(mid);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) square += __shfl_xor_sync(0xffffffffu, square, o);
  // (Squares of tiny or huge means leave fp32.)
  if (lane == 0)
    s.out.norm[out] = square > 1e-30 && square < 1e30 ? sqrtf((float)square) : (float)sqrt(square);
}

// ---- scores ---------------------------------------------------------------

constexpr int kScoreM = 128, kScoreN = 128, kScoreThreads = 256;
constexpr int kScoreDepth = 64;  // columns of the means in shared memory at a time
constexpr uint32_t kScoreRow = 2 * kScoreDepth;  // bytes
static_assert(kScoreM == 128 && kScoreDepth == 64, "the layout below");
constexpr uint32_t kScoreBuffer = 2 * (kScoreM + kScoreN) * kScoreRow;

struct ScoreArgs {
  Means q, k;
  float* scores;    // [products][m][pitch]
  uint32_t* norms;  // [products][pitch / kScoreN]: bits of the largest |k| of a tile's columns
  unsigned int* status;
  int m, nk, pitch;
};

// 16 bytes into shared memory, or zeros where the row does not exist.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}

// A 128 x 128 tile of scores per CTA: tcgen05 products of 64 columns at a time, hi hi, hi mid
// and mid hi into one accumulator of 128 TMEM columns. The parts lie in shared memory as the
// tensor core reads them, rows of 128 bytes with 16-byte chunks xor-swizzled by row. With one
// buffer of 64 columns (64 KB) three CTAs fit an SM and overlap their loads, products and
// stores; where there is no more than a CTA per SM, a buffer for all columns lets all loads
// start at once. Measured, one buffer against two at D = 128: 672 tiles 24 and 28 us, 32 tiles
// 7.9 and 7.3 us (mma.sync on tiles of 64 x 128: 30 and 6.9 us).
template <int D, int BUFFERS>
__global__ void __launch_bounds__(kScoreThreads, BUFFERS == 1 ? 3 : 1)
    block_scores(const __grid_constant__ ScoreArgs a) {
  constexpr int kSteps = D / kScoreDepth;
  static_assert(BUFFERS == 1 || BUFFERS == kSteps, "");
  constexpr int N = kScoreN;
  constexpr uint32_t kQPart = kScoreM * kScoreRow, kKPart = N * kScoreRow;
  extern __shared__ uint8_t tiles[];
  __shared__ __align__(8) uint64_t done_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_flag;
  const uint32_t base = (attn::smem_u32(tiles) + 1023u) / 1024u * 1024u;
  const uint32_t bar = attn::smem_u32(&done_bar);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    attn::mbar_init(bar, 1);
    abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     attn::smem_u32(&tmem_slot)),
                 "r"(N)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int m0 = blockIdx.y * kScoreM, n0 = blockIdx.x * N;
  const int64_t product = blockIdx.z;
  attn::tc_fence_before();
  __syncthreads();
  attn::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  grid_wait();
  // Parts of a buffer: q hi, q mid, k hi, k mid. Eight threads a row.
  auto load = [&](int step) {
    const uint32_t buffer = base + (BUFFERS > 1 ? step : 0) * kScoreBuffer;
    const int chunk = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < (kScoreM + N) * 8 / kScoreThreads; ++i) {
      constexpr int kRows = kScoreThreads / 8;
      const bool is_q = i < kScoreM / kRows;
      const int row = (threadIdx.x >> 3) + (is_q ? i : i - kScoreM / kRows) * kRows;
      const int r = (is_q ? m0 : n0) + row;
      const bool there = r < (is_q ? a.m : a.nk);
      const Means& side = is_q ? a.q : a.k;
      const int64_t off =
          there ? (product * (is_q ? a.m : a.nk) + r) * D + step * kScoreDepth + chunk * 8 : 0;
      const uint32_t dst =
          buffer + (is_q ? 0u : 2 * kQPart) + row * kScoreRow + (uint32_t)((chunk ^ (row & 7)) << 4);
      copy16(dst, side.hi + off, there);
      copy16(dst + (is_q ? kQPart : kKPart), side.mid + off, there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  load(0);
  if (BUFFERS > 1) load(1);
  if (blockIdx.y == 0 && warp == 0) {
    uint32_t norm = 0u;  // the bits order like the values, NaN above all
#pragma unroll
    for (int i = 0; i < N / 32; ++i) {
      const int c = n0 + 32 * i + lane;
      if (c < a.nk) norm = max(norm, __float_as_uint(a.k.norm[product * a.nk + c]));
    }
    norm = __reduce_max_sync(0xffffffffu, norm);
    if (lane == 0) a.norms[product * gridDim.x + blockIdx.x] = norm;
  }
  bool ok = true;
#pragma unroll
  for (int step = 0; step < kSteps; ++step) {
    if (BUFFERS == 1 && step > 0) {
      // The products before have read their columns.
      ok = __syncthreads_and(attn::wait_bar(bar, (step - 1) & 1, &abort_flag, a.status));
      if (!ok) break;
      load(step);
    }
    if (BUFFERS > 1 && step == 0)
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
      if (attn::elect_one()) {
        // kind::f16, bf16 operands, both with their columns innermost, f32 accumulator.
        constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) |
                                    ((uint32_t)(kScoreM >> 4) << 24);
        const uint32_t buffer = base + (BUFFERS > 1 ? step : 0) * kScoreBuffer;
        const uint64_t qd = attn::smem_desc(buffer, 16, 1024);
        const uint64_t kd = attn::smem_desc(buffer + 2 * kQPart, 16, 1024);
        auto q = [&](int n, int kk) { return qd + (uint64_t)((n * kQPart + kk * 32) >> 4); };
        auto k = [&](int n, int kk) { return kd + (uint64_t)((n * kKPart + kk * 32) >> 4); };
#pragma unroll
        for (int kk = 0; kk < kScoreDepth / 16; ++kk) {
          attn::mma_ss(tmem, q(1, kk), k(0, kk), kIdesc, step > 0 || kk > 0 ? 1u : 0u);
          attn::mma_ss(tmem, q(0, kk), k(1, kk), kIdesc, 1u);
          attn::mma_ss(tmem, q(0, kk), k(0, kk), kIdesc, 1u);
        }
        if (BUFFERS == 1 || step + 1 == kSteps) attn::mma_commit(bar);
      }
      __syncwarp();
    }
  }
  if (ok)
    ok = __syncthreads_and(
        attn::wait_bar(bar, BUFFERS == 1 ? (kSteps - 1) & 1 : 0, &abort_flag, a.status));
  grid_done();
  if (ok) {
    attn::tc_fence_after();
    // Warp w: rows 32 (w & 3), half w >> 2 of the columns; a row a thread, 32-byte stores.
    const int row = m0 + 32 * (warp & 3) + lane, column = N / 2 * (warp >> 2);
    float* dst = a.scores + (product * a.m + row) * a.pitch + n0 + column;
#pragma unroll
    for (int c = 0; c < N / 2; c += 32) {
      uint32_t s[32];
      attn::tmem_ld32(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + column + c, s);
      attn::tmem_ld_wait(s);
      if (row < a.m) {
#pragma unroll
        for (int i = 0; i < 32; i += 8)
          st32(dst + c + i, Chunk32{make_uint4(s[i], s[i + 1], s[i + 2], s[i + 3]),
                                    make_uint4(s[i + 4], s[i + 5], s[i + 6], s[i + 7])});
      }
    }
  }
  if (!ok) {  // unwinding: let products in flight end before their memory is given up
    const unsigned long long t0 = attn::globaltimer();
    while (attn::globaltimer() - t0 < 200000ull) __nanosleep(1000);
  }
  attn::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    attn::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(N)
                 : "memory");
  }
}

// ---- choice ---------------------------------------------------------------

struct ChooseArgs {
  int32_t* indices;
  int32_t* counts;
  Means q, k;
  uint32_t* scores;  // [rows][pitch]: fp32 scores, overwritten with keys by choose_any
  const uint32_t* norms;  // [batch * kv_heads][norm_tiles]
  int norm_tiles;
  const int32_t* q_lens;
  const int32_t* k_lens;
  const uint8_t* keep;
  int heads, kv_heads, seq_q, seq_k, head_dim, block_q, block_k, nq, nk, pitch, top_k;
  uint32_t rows;  // batch * heads * nq
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

constexpr int kBins = 256;
// Bins for a row of 32 KEYS columns: three of them should rarely hold more than a warp ranks
// (2036 columns, 6108 rows: 27 on average around the best tenth with 256 bins; 288 us with
// these, 73 us with twice as many).
template <int KEYS>
constexpr int kBinsOf = KEYS <= 32 ? kBins : kBins * KEYS / 32;
constexpr int kChooseWarps = 4;

// What a warp's row of scores is about.
struct Row {
  int64_t list, k_row0;  // which query block, and the first key block of its key head
  int k_blocks, want, kept;  // blocks that exist, places in the list, kept blocks
  float q_norm, k_norm;      // k_norm: the largest of the blocks that exist
};

// fp64 scores of four columns (c of lane 8g for group g of eight lanes) as order-preserving
// keys, in all lanes of a group. Every column is summed in the same order.
__device__ __forceinline__ unsigned long long exact_keys(const ChooseArgs& a, const Row& r, int c,
                                                         int lane) {
  const float* q = a.q.mean + r.list * a.head_dim;
  const float* k = a.k.mean + (r.k_row0 + c) * a.head_dim;
  float4 x[4], y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = 4 * (lane & 7) + 32 * i;
    const bool there = d < a.head_dim;
    x[i] = there ? *reinterpret_cast<const float4*>(q + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    y[i] = there ? *reinterpret_cast<const float4*>(k + d) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fma((double)x[i].x, (double)y[i].x, s);
    s = fma((double)x[i].y, (double)y[i].y, s);
    s = fma((double)x[i].z, (double)y[i].z, s);
    s = fma((double)x[i].w, (double)y[i].w, s);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return score_key(s);
}

// Of n columns (n <= 32, ascending or not), which are the `open` best by fp64 score, ties to
// the lower column: a mask by position.
__device__ __forceinline__ unsigned best_of(const ChooseArgs& a, const Row& r, const int* columns,
                                            int n, int open, int lane) {
  unsigned long long mine = 0ull;
  for (int i = 0; i < n; i += 4) {
    const unsigned long long s = exact_keys(a, r, columns[min(i + (lane >> 3), n - 1)], lane);
    const unsigned long long at = __shfl_sync(0xffffffffu, s, (lane & 3) * 8);
    if (lane >= i && lane < i + 4) mine = at;
  }
  const int column = columns[min(lane, n - 1)];
  int rank = 0;
  for (int i = 0; i < n; ++i) {
    const unsigned long long s = __shfl_sync(0xffffffffu, mine, i);
    const int c = __shfl_sync(0xffffffffu, column, i);
    rank += s > mine || (s == mine && c < column);
  }
  return __ballot_sync(0xffffffffu, lane < n && rank < open);
}

// The bound on the difference of two scores from their fp32 values, 2E with
//   E = 6e-5 |q| max|k| + 1e-35:
// dropping mid mid and what two bf16 leave of a mean, 3 2^-18 of |q| |k| (Cauchy-Schwarz);
// 384 products summed in fp32, 2^-23 each if every addition truncates (1.14e-5 + 4.58e-5);
// products below fp32's range. Infinite where it does not hold: means too small for two bf16 to
// hold their digits, and norms whose product is near or beyond fp32's range. (Below 1e38 no
// partial sum leaves the range: by Cauchy-Schwarz they stay under 1.02 |q| |k|.)
__device__ __forceinline__ float twice_error(const Row& r) {
  const bool sound = (r.q_norm >= 1e-30f || r.q_norm == 0.f) && (r.k_norm >= 1e-30f || r.k_norm == 0.f) &&
                     r.q_norm * r.k_norm < 1e38f;
  return sound ? 1.21e-4f * r.q_norm * r.k_norm + 2e-35f : INFINITY;
}

// Any row: keys of the scores in the workspace, where each lane reads and writes columns
// lane, lane + 32, ... only. Returns how many blocks it listed.
__device__ __noinline__ int choose_any(const ChooseArgs& a, const Row& r, uint32_t* bins,
                                       int* close, int lane) {
  const unsigned below = (1u << lane) - 1u;
  const int k_blocks = r.k_blocks, want = r.want;
  int32_t* out = a.indices + r.list * a.top_k;
  uint32_t* row = a.scores + r.list * a.pitch;
  // More kept blocks than a list holds: only they compete, by score.
  const bool only_kept = r.kept > a.top_k;
  const int kept = only_kept ? 0 : r.kept;
  for (int c = lane; c < k_blocks; c += 32) {
    const bool keep = a.keep != nullptr && a.keep[c] != 0;
    row[c] = only_kept && !keep ? 0u
             : keep && !only_kept ? kInKey : score_key(__uint_as_float(row[c]));
  }
  // f(column, key) for all columns; a column behind the last block has key 0.
  auto each_column = [&](auto f) {
#pragma unroll 4
    for (int c0 = 0; c0 < k_blocks; c0 += 32) f(c0 + lane, c0 + lane < k_blocks ? row[c0 + lane] : 0u);
  };
  auto each = [&](auto f) { each_column([&](int, uint32_t k) { f(k); }); };
  uint32_t least_in = kInKey;  // keys from here on are in
  int done = 0;
  if (want > kept) {
    // T, the k-th largest score: count the scores in equal bins of their range, go on
    // inside the bin that holds the k-th, rank what is left when a warp holds it. The bin
    // of a score never decreases with it, whatever the rounding.
    float low = -INFINITY, high = INFINITY;
    int left = want - kept;  // the rank of T among the scores in [low, high]
    uint32_t kth;
    for (;;) {
      uint32_t least = kInKey, most = 0u;
      int n = 0;
      const uint32_t low_key = score_key(low), high_key = score_key(high);
      each([&](uint32_t k) {
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
        each([&](uint32_t k) {
          const bool mine = k >= least && k <= most;
          const unsigned mask = __ballot_sync(0xffffffffu, mine);
          if (mine) bins[at + __popc(mask & below)] = k;
          at += __popc(mask);
        });
        __syncwarp();
        const uint32_t mine = lane < n ? bins[lane] : 0u;
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
      for (int i = lane; i < kBins; i += 32) bins[i] = 0u;
      __syncwarp();
      each([&](uint32_t k) {
        if (k >= least && k <= most) atomicAdd(&bins[bin_of(k)], 1u);
      });
      __syncwarp();
      // Lane l sums bins [8l, 8l + 8); from the top, the lane and then the bin that reach `left`.
      uint32_t mine[kBins / 32];
      int sum = 0;
#pragma unroll
      for (int i = 0; i < kBins / 32; ++i) {
        mine[i] = bins[lane * (kBins / 32) + i];
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
      each([&](uint32_t k) {
        if (k >= least && k <= most && bin_of(k) == bin) {
          bin_least = min(bin_least, k);
          bin_most = max(bin_most, k);
        }
      });
      low = key_score(__reduce_min_sync(0xffffffffu, bin_least));
      high = key_score(__reduce_max_sync(0xffffffffu, bin_most));
      __syncwarp();
    }
    const float twice = twice_error(r);
    const float t = key_score(kth);
    const bool bounded = kth != 0u && twice < INFINITY && fabsf(t) < INFINITY;
    const uint32_t hi = bounded ? score_key(__fadd_ru(t, twice)) : kInKey - 1u;
    const uint32_t lo = bounded ? score_key(__fadd_rd(t, -twice)) : 1u;
    int n_in = 0, n_close = 0;
    each_column([&](int c, uint32_t k) {
      const bool is_close = k >= lo && k <= hi;
      const unsigned mask = __ballot_sync(0xffffffffu, is_close);
      if (is_close) {
        const int at = n_close + __popc(mask & below);
        if (at < 32) close[at] = c;
      }
      n_close += __popc(mask);
      n_in += __popc(__ballot_sync(0xffffffffu, k > hi));
    });
    __syncwarp();
    const int open = want - n_in;  // places left for the close ones
    least_in = hi + 1u;
    if (n_close == open) {
      least_in = lo;
    } else {
      if (n_close <= 32) {
        const unsigned in = best_of(a, r, close, n_close, open, lane);
        for (int i = 0; i < n_close; ++i) {
          const int c = close[i];
          if (lane == (c & 31)) row[c] = (in >> i & 1u) ? kInKey : 0u;
        }
      } else {
        // Many scores within the bound (equal blocks, say): a search on fp64 keys, which are
        // computed again in every pass.
        auto each_close = [&](auto f) {
          each_column([&](int c0, uint32_t k) {
            unsigned mask = __ballot_sync(0xffffffffu, k >= lo && k <= hi);
            for (; mask != 0u; mask &= mask - 1u) {
              const int c = c0 - lane + __ffs((int)mask) - 1;
              f(c, exact_keys(a, r, c, lane));
            }
          });
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
    }
  }
  each_column([&](int c, uint32_t k) {
    const bool take = k >= least_in;
    const unsigned mask = __ballot_sync(0xffffffffu, take);
    if (take) out[done + __popc(mask & below)] = c;
    done += __popc(mask);
  });
  return done;
}

// Eight floats, 32-byte aligned.
__device__ __forceinline__ void ld_floats8(const float* p, float* v) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]),
                 "=f"(v[6]), "=f"(v[7])
               : "l"(p)
               : "memory");
}
// The smallest of three, NaN passed over (and max3, the largest).
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A row of at most 32 KEYS finite scores, KEYS neighbouring columns in the registers of each
// lane: counts them in bins of their range, gathers the bin that holds the k-th and its
// neighbours, and ranks these, one a lane. Sets of columns are bit masks, a word for 32 columns
// of a lane. Returns -1 where that does not settle it (scores bunched in a bin, all alike, a
// border wider than a bin): choose_any does. (Bound by the latency of its steps.
// 9600 rows of 800 columns: 30 us, with marked floats in place of masks and 16-byte loads 51 us.)
template <int KEYS>
__device__ __forceinline__ int choose_fast(const ChooseArgs& a, const Row& r, uint32_t* bins,
                                           int* columns, int* gathered, int lane) {
  constexpr int kWords = (KEYS + 31) / 32;
  constexpr int kBins = kBinsOf<KEYS>, kHeld = kBins / 32;
  const float* row = reinterpret_cast<const float*>(a.scores) + r.list * a.pitch;
  const int c0 = lane * KEYS;
  const int mine = min(max(r.k_blocks - c0, 0), KEYS);  // columns of this lane that exist
  const int left = r.want - r.kept;
  uint32_t in[kWords];  // columns of this lane that are in
#pragma unroll
  for (int w = 0; w < kWords; ++w) in[w] = 0u;
  if (r.kept > 0) {
#pragma unroll 8
    for (int i = 0; i < mine; ++i) {
      const uint32_t bit = (a.keep[c0 + i] != 0 ? 1u : 0u) << (i & 31);
#pragma unroll
      for (int w = 0; w < kWords; ++w) in[w] |= i >> 5 == w ? bit : 0u;
    }
  }
  if (r.want == r.k_blocks) {
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      in[w] = mine >= 32 * w + 32 ? ~0u : mine <= 32 * w ? 0u : (1u << (mine - 32 * w)) - 1u;
  } else if (left > 0) {
    const float twice = twice_error(r);
    const float nan = __int_as_float(0x7fffffff);
    float v[KEYS];  // NaN where a column does not compete: it is in no range and in no bin
#pragma unroll
    for (int i = 0; i < KEYS; i += 8) {
      if (mine > 0 && c0 + i < a.pitch) {
        ld_floats8(row + c0 + i, v + i);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i + j] = nan;
      }
    }
    if (r.k_blocks % KEYS != 0) {
#pragma unroll
      for (int i = 0; i < KEYS; ++i) v[i] = i < mine ? v[i] : nan;
    }
    if (r.kept > 0) {
#pragma unroll
      for (int i = 0; i < KEYS; ++i) v[i] = in[i >> 5] >> (i & 31) & 1u ? nan : v[i];
    }
    float low = nan, high = nan;
#pragma unroll
    for (int i = 0; i < KEYS; i += 2) {
      low = min3(low, v[i], v[i + 1]);
      high = attn::max3(high, v[i], v[i + 1]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    const float scale = (float)(kBins - 3) / (high - low);
    // The bin is what s scale + shift rounds to, 0 to kBins - 1: read from the low bits of a float in
    // [2^23, 2^24), where the rounding is to integers, that of `shift` too. It never decreases
    // with the score. (A range that small beside the scores is within their error.)
    if (!(twice < INFINITY) || !(scale < 1e30f) || !(scale > 1e-30f) || !(fabsf(low) * scale < 1e6f))
      return -1;
    constexpr float kOne = 12582912.f;  // 1.5 2^23
    const float shift = kOne + (1.f - low * scale);
    auto place = [&](float s) { return fmaf(s, scale, shift); };  // kOne + bin
    auto bin_of = [&](float s) {  // (of a score of the row, or NaN)
      return __float_as_int(place(s)) - __float_as_int(kOne);
    };
#pragma unroll
    for (int i = 0; i < kBins / 128; ++i)
      *reinterpret_cast<uint4*>(bins + 128 * i + 4 * lane) = make_uint4(0u, 0u, 0u, 0u);
    if (lane == 0) *gathered = 0;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int bin = bin_of(v[i]);
      if ((unsigned)bin < (unsigned)kBins) atomicAdd(&bins[bin], 1u);
    }
    __syncwarp();
    // From the top, the bin that reaches the k-th: lane l looks at kHeld neighbouring bins.
    int held[kHeld], sum = 0;
#pragma unroll
    for (int i = 0; i < kHeld; i += 4) {
      const int4 four = *reinterpret_cast<const int4*>(bins + kHeld * lane + i);
      held[i] = four.x;
      held[i + 1] = four.y;
      held[i + 2] = four.z;
      held[i + 3] = four.w;
      sum += (four.x + four.y) + (four.z + four.w);
    }
    int up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_down_sync(0xffffffffu, up, o);
      if (lane + o < 32) up += other;
    }
    const int total = __shfl_sync(0xffffffffu, up, 0);
    if (total != r.k_blocks - r.kept) return -1;  // (NaN)
    const unsigned reach = __ballot_sync(0xffffffffu, up >= left);
    const int owner = 31 - __clz((int)reach);
    int bin = 0, over = up - sum;
    bool found = false;
#pragma unroll
    for (int i = kHeld - 1; i >= 0; --i) {
      if (!found && over + held[i] >= left) {
        bin = kHeld * lane + i;
        found = true;
      }
      if (!found) over += held[i];
    }
    bin = __shfl_sync(0xffffffffu, bin, owner);
    over = __shfl_sync(0xffffffffu, over, owner);  // scores in the bins above
    const int next = bin + 1 < kBins ? (int)bins[bin + 1] : 0;
    const int n = next + (int)bins[bin] + (bin > 0 ? (int)bins[bin - 1] : 0);
    if (n > 32) return -1;
    uint32_t near[kWords];
#pragma unroll
    for (int w = 0; w < kWords; ++w) near[w] = 0u;
    const int below = bin - 1;
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
      if ((unsigned)(bin_of(v[i]) - below) < 3u) near[i >> 5] |= 1u << (i & 31);
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      if (near[w] == 0u) continue;
      int at = atomicAdd(gathered, __popc(near[w]));
      for (uint32_t m = near[w]; m != 0u; m &= m - 1u) columns[at++] = c0 + 32 * w + __ffs((int)m) - 1;
    }
    __syncwarp();
    const int my_column = lane < n ? columns[lane] : 0x7fffffff;
    const float my_value = lane < n ? row[my_column] : -INFINITY;
    int rank = 0;
    for (int i = 0; i < n; ++i) {
      const float s = __shfl_sync(0xffffffffu, my_value, i);
      rank += s > my_value || (s == my_value && columns[i] < my_column);
    }
    const int first = over - next;  // scores above all that were gathered
    const unsigned kth = __ballot_sync(0xffffffffu, lane < n && rank == left - first - 1);
    const float t = __shfl_sync(0xffffffffu, my_value, __ffs((int)kth) - 1);
    const float hi = __fadd_ru(t, twice), lo = __fadd_rd(t, -twice);
    // All that is close has to be among the gathered.
    if ((bin > 0 && place(lo) < kOne + (float)(bin - 1)) ||
        (bin + 1 < kBins && place(hi) > kOne + (float)(bin + 1)))
      return -1;
    const unsigned close = __ballot_sync(0xffffffffu, lane < n && my_value >= lo && my_value <= hi);
    const int open = left - first - __popc(__ballot_sync(0xffffffffu, lane < n && my_value > hi));
    const int n_close = __popc(close);
    // In: what lies above hi, and where all the close ones fit, what reaches lo.
    const bool all_close = n_close == open;
    float least = lo;
    if (!all_close)  // the next float above hi
      least = hi == 0.f ? 1e-45f : __int_as_float(__float_as_int(hi) + (hi > 0.f ? 1 : -1));
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
      if (v[i] >= least) in[i >> 5] |= 1u << (i & 31);
    if (!all_close) {
      // The close columns move to the front of `columns`.
      __syncwarp();
      if (close >> lane & 1u) columns[__popc(close & ((1u << lane) - 1u))] = my_column;
      __syncwarp();
      const unsigned best = best_of(a, r, columns, n_close, open, lane);
      for (unsigned m = best; m != 0u; m &= m - 1u) {
        const unsigned at = (unsigned)(columns[__ffs((int)m) - 1] - c0);
#pragma unroll
        for (int w = 0; w < kWords; ++w)
          if (at >> 5 == (unsigned)w && at < (unsigned)KEYS) in[w] |= 1u << (at & 31);
      }
    }
  }
  int count = 0;
#pragma unroll
  for (int w = 0; w < kWords; ++w) count += __popc(in[w]);
  int before = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += other;
  }
  const int done = __shfl_sync(0xffffffffu, before, 31);
  int32_t* out = a.indices + r.list * a.top_k + (before - count);
#pragma unroll
  for (int w = 0; w < kWords; ++w)
    for (uint32_t m = in[w]; m != 0u; m &= m - 1u) *out++ = c0 + 32 * w + __ffs((int)m) - 1;
  return done;
}

// A warp per query block. An order statistic moves by no more than the values do: with T the
// k-th largest fp32 score and E its error (twice_error), blocks above T + 2E are in and blocks
// below T - 2E are out whatever the rounding did; the few between are scored again in fp64 and
// ranked.
// CTAs per SM that the registers should allow: a row is a chain of short steps, and many rows at
// once hide it (6108 rows of 2036 columns: two CTAs 63 us, three 48 us, four 43 us, five 43 us).
// Eight warps a CTA are slower, 33 against 30 us for 9600 rows of 800: a CTA lasts as long as its
// slowest row.
// Rows of 32, 64 and 128 columns a lane spill 60, 84 and 124 bytes a thread under these bounds. Rows of
// more than 4096 columns (KEYS = 0) are slow: every pass of choose_any reads them from global
// memory. 24 heads of 354,206 rows: 0.90 ms for lists of 138 of 2768 blocks (128 columns a lane), 5.0
// ms for 276 of 5535 blocks (choose_any), beside an HBM pass of 0.7 ms.
template <int KEYS>
__global__ void __launch_bounds__(kChooseWarps * 32, KEYS <= 16 ? 8 : KEYS <= 32 ? 6 : KEYS <= 64 ? 4 : 3)
    block_choose(const __grid_constant__ ChooseArgs a) {
  __shared__ __align__(16) uint32_t bins[kChooseWarps][kBinsOf<KEYS>];
  __shared__ int columns[kChooseWarps][32];
  __shared__ int gathered[kChooseWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t list = blockIdx.x * kChooseWarps + warp;
  if (list >= a.rows) return;
  const uint32_t bh = list / (uint32_t)a.nq, block = list % (uint32_t)a.nq;
  const int head = (int)(bh % (uint32_t)a.heads), b = (int)(bh / (uint32_t)a.heads);
  const int64_t kv = (int64_t)b * a.kv_heads + head / (a.heads / a.kv_heads);
  grid_wait();
  uint32_t norm = 0u;
  for (int i = lane; i < a.norm_tiles; i += 32) norm = max(norm, a.norms[kv * a.norm_tiles + i]);
  Row r;
  r.list = list;
  r.q_norm = a.q.norm[list];
  r.k_row0 = kv * a.nk;
  r.k_blocks = (rows_of(a.k_lens, b, a.seq_k) + a.block_k - 1) / a.block_k;
  r.want = (int)block * a.block_q < rows_of(a.q_lens, b, a.seq_q) ? min(a.top_k, r.k_blocks) : 0;
  r.kept = 0;
  r.k_norm = __uint_as_float(__reduce_max_sync(0xffffffffu, norm));
  int done = 0;
  if (r.want > 0) {
    if (a.keep != nullptr) {
#pragma unroll 8
      for (int c = lane; c < r.k_blocks; c += 32) r.kept += a.keep[c] != 0;
      r.kept = __reduce_add_sync(0xffffffffu, r.kept);
    }
    done = -1;
    if constexpr (KEYS > 0) {
      if (r.kept <= r.want)
        done = choose_fast<KEYS>(a, r, bins[warp], columns[warp], &gathered[warp], lane);
    }
    if (done < 0) {
      __syncwarp();
      done = choose_any(a, r, bins[warp], columns[warp], lane);
    }
  }
  grid_done();
  int32_t* out = a.indices + r.list * a.top_k;
  for (int c = done + lane; c < a.top_k; c += 32) out[c] = -1;
  if (lane == 0) a.counts[r.list] = done;
}

// ---- host side --------------------------------------------------------------

struct Sizes {
  int64_t q_rows, k_rows, pitch, norms_at, scores_at, bytes;
};
Sizes sizes_of(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t nq,
               int64_t nk) {
  Sizes s;
  s.q_rows = batch * heads * nq;
  s.k_rows = batch * kv_heads * nk;
  s.pitch = (nk + kScoreN - 1) / kScoreN * kScoreN;
  // Per row: D fp32, D + D bf16, a norm (rounded up so that every part starts on 16 bytes).
  s.norms_at = (s.q_rows + s.k_rows) * head_dim * 8 + ((s.q_rows + s.k_rows) * 4 + 31) / 16 * 16;
  s.scores_at = s.norms_at + (batch * kv_heads * (s.pitch / kScoreN) * 4 + 15) / 16 * 16;
  // Scores start at the next 32 bytes, wherever the workspace starts.
  s.bytes = s.scores_at + 16 + s.q_rows * s.pitch * 4;
  return s;
}

template <int KEYS>
int launch_choose(const ChooseArgs& a, cudaStream_t s) {
  launch_after(block_choose<KEYS>, dim3((a.rows + kChooseWarps - 1) / kChooseWarps),
               kChooseWarps * 32, 0, s, a);
  return check_launch("h3b_select_key_blocks");
}

template <int D, int BUFFERS>
int launch_scores(const ScoreArgs& sc, int64_t m_tiles, int64_t products, cudaStream_t s) {
  constexpr int kSmem = (int)(BUFFERS * kScoreBuffer + 1024);
  static ContextSlot slots[kMaxDevices];
  cudaError_t e = cudaErrorInvalidDevice;
  if (context_cached(slots, [&]() -> void* {
        e = cudaFuncSetAttribute(block_scores<D, BUFFERS>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        return e == cudaSuccess ? reinterpret_cast<void*>(1) : nullptr;
      }) == nullptr) {
    set_error(std::string("h3b_select_key_blocks: cannot reserve shared memory: ") +
              cudaGetErrorString(e));
    return H3B_ERR_CUDA;
  }
  launch_after(block_scores<D, BUFFERS>,
               dim3((unsigned)(sc.pitch / kScoreN), (unsigned)m_tiles, (unsigned)products), kScoreThreads,
               kSmem, s, sc);
  return check_launch("h3b_select_key_blocks");
}

template <bool FP16, int D>
int launch_all(const MeanArgs& m, const ScoreArgs& sc, const ChooseArgs& a, int64_t products,
               cudaStream_t s) {
  const int64_t blocks = m.side[0].blocks_total + m.side[1].blocks_total;
  const int warps = blocks >= (int64_t)num_sms() * 16 ? 1 : kMeanWarps;  // per block
  const int64_t grid = (blocks * warps + kMeanWarps - 1) / kMeanWarps;
  const int64_t m_tiles = (sc.m + kScoreM - 1) / kScoreM;
  H3B_REQUIRE(grid <= 0x7fffffffLL && products <= 65535 && m_tiles <= 65535,
              "select_key_blocks: shape exceeds launch limits");
  if (warps == 1)
    launch_after(block_means<FP16, D, 1>, dim3((unsigned)grid), kMeanWarps * 32, 0, s, m);
  else
    launch_after(block_means<FP16, D, kMeanWarps>, dim3((unsigned)grid), kMeanWarps * 32, 0, s, m);
  int rc = check_launch("h3b_select_key_blocks");
  if (rc != H3B_OK) return rc;
  if (sc.pitch / kScoreN * m_tiles * products <= num_sms())
    rc = launch_scores<D, D / kScoreDepth>(sc, m_tiles, products, s);
  else
    rc = launch_scores<D, 1>(sc, m_tiles, products, s);
  if (rc != H3B_OK) return rc;
  // Registers for a row's scores: as few as hold it, up to 128 a lane.
  if (a.nk <= 8 * 32) return launch_choose<8>(a, s);
  if (a.nk <= 16 * 32) return launch_choose<16>(a, s);
  if (a.nk <= 32 * 32) return launch_choose<32>(a, s);
  if (a.nk <= 64 * 32) return launch_choose<64>(a, s);
  if (a.nk <= 128 * 32) return launch_choose<128>(a, s);
  return launch_choose<0>(a, s);
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
  *bytes_out = h3b::select::sizes_of(batch, heads, kv_heads, head_dim, nq, nk).bytes;
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
  H3B_REQUIRE(batch <= (1LL << 31) / heads && batch * heads <= ((1LL << 31) - 64) / nq,
              "select_key_blocks: shape exceeds launch limits");
  H3B_REQUIRE(indices != nullptr && counts != nullptr && q != nullptr && k != nullptr,
              "select_key_blocks: null argument");
  H3B_REQUIRE(h3b::aligned16(q) && h3b::aligned16(k), "select_key_blocks: q and k must be 16-byte aligned");
  const int64_t strides[6] = {q_batch_stride, q_row_stride, q_head_stride,
                              k_batch_stride, k_row_stride, k_head_stride};
  const int64_t sizes[6] = {batch, seq_q, heads, batch, seq_k, kv_heads};
  for (int i = 0; i < 6; ++i)
    H3B_REQUIRE(sizes[i] == 1 || (strides[i] % 8 == 0 && strides[i] >= 0),
                "select_key_blocks: strides must be multiples of 8 elements");
  int rc = h3b_select_key_blocks_workspace_size(batch, seq_q, seq_k, heads, kv_heads, head_dim,
                                                block_q, block_k, &need);
  if (rc != H3B_OK) return rc;
  H3B_REQUIRE(workspace != nullptr && workspace_bytes >= need && h3b::aligned16(workspace),
              "select_key_blocks: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  const Sizes sz = sizes_of(batch, heads, kv_heads, head_dim, nq, nk);
  char* at = static_cast<char*>(workspace);
  auto take = [&](int64_t bytes) {
    char* p = at;
    at += bytes;
    return p;
  };
  Means qm, km;
  qm.mean = reinterpret_cast<float*>(take(sz.q_rows * head_dim * 4));
  km.mean = reinterpret_cast<float*>(take(sz.k_rows * head_dim * 4));
  qm.hi = reinterpret_cast<__nv_bfloat16*>(take(sz.q_rows * head_dim * 2));
  qm.mid = reinterpret_cast<__nv_bfloat16*>(take(sz.q_rows * head_dim * 2));
  km.hi = reinterpret_cast<__nv_bfloat16*>(take(sz.k_rows * head_dim * 2));
  km.mid = reinterpret_cast<__nv_bfloat16*>(take(sz.k_rows * head_dim * 2));
  qm.norm = reinterpret_cast<float*>(take(sz.q_rows * 4));
  km.norm = reinterpret_cast<float*>(take(sz.k_rows * 4));
  auto* norms = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + sz.norms_at);
  auto* scores = reinterpret_cast<uint32_t*>(
      (reinterpret_cast<uintptr_t>(workspace) + (uintptr_t)sz.scores_at + 31) / 32 * 32);
  MeanArgs m{};
  m.side[0] = MeanSide{q, qm, q_batch_stride, q_row_stride, q_head_stride, q_lens, (int)seq_q,
                       (int)heads, (int)block_q, (int)nq, batch * nq * heads};
  m.side[1] = MeanSide{k, km, k_batch_stride, k_row_stride, k_head_stride, k_lens, (int)seq_k,
                       (int)kv_heads, (int)block_k, (int)nk, batch * nk * kv_heads};
  // The heads of a group lie behind one another: one product per (batch, key head).
  ScoreArgs sc{qm, km, reinterpret_cast<float*>(scores), norms, h3b::status_ptr(), (int)(heads / kv_heads * nq), (int)nk,
               (int)sz.pitch};
  ChooseArgs a{};
  a.indices = indices;
  a.counts = counts;
  a.q = qm;
  a.k = km;
  a.scores = scores;
  a.norms = norms;
  a.norm_tiles = (int)(sz.pitch / kScoreN);
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.keep = keep;
  a.heads = (int)heads;
  a.kv_heads = (int)kv_heads;
  a.seq_q = (int)seq_q;
  a.seq_k = (int)seq_k;
  a.head_dim = (int)head_dim;
  a.block_q = (int)block_q;
  a.block_k = (int)block_k;
  a.nq = (int)nq;
  a.nk = (int)nk;
  a.pitch = (int)sz.pitch;
  a.top_k = (int)top_k;
  a.rows = (uint32_t)sz.q_rows;
  if (dtype == H3B_DTYPE_FP16)
    return head_dim == 128 ? launch_all<true, 128>(m, sc, a, batch * kv_heads, stream)
                           : launch_all<true, 64>(m, sc, a, batch * kv_heads, stream);
  return head_dim == 128 ? launch_all<false, 128>(m, sc, a, batch * kv_heads, stream)
                         : launch_all<false, 64>(m, sc, a, batch * kv_heads, stream);
}
