// Norms after and before a branch fused with its gate and the scaled residual.
//
//   b      = RMSNorm(branch) * post_weight
//   hidden = residual_scale * residual + gate[idx] * b                        (out0)
//   normed = RMSNorm(hidden) * weight * (1 + scale[idx]) + shift[idx]         (out1, optional)
//
// Bound by HBM: a row of branch and of residual is read once, hidden and normed are
// written once; the two reductions and everything between them stay in registers. Sums of
// squares and all products are fp32, each output is rounded once to its own type, and
// normed is taken from the unrounded hidden.
#include <cuda_fp16.h>

#include <cstdio>

#include "common.cuh"

namespace h3b {
namespace {

struct SandwichArgs {
  void* hidden;
  void* normed;  // null: no second norm
  const void* residual;
  const void* branch;
  const void* post_weight;
  const void* gate;
  const void* weight;
  const void* scale;
  const void* shift;
  const int64_t* index;
  int64_t rows, cols, n_index, n_table;
  int64_t residual_stride, branch_stride, hidden_stride, normed_stride;
  int64_t gate_stride, scale_stride, shift_stride;
  float residual_scale, post_eps, eps;
};

// 16 bytes of T as pairs of floats and back: pairs, since Blackwell's packed fp32 instructions
// halve the arithmetic, which at the clock of a busy GPU is not far below what HBM takes.
template <class T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void unpack(uint4 u, float2 (&v)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = make_float2(bf16lo(w[j]), bf16hi(w[j]));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[4]) {
    return make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[1].x, v[1].y),
                      pack_bf16(v[2].x, v[2].y), pack_bf16(v[3].x, v[3].y));
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void unpack(uint4 u, float2 (&v)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(v[j].x, v[j].y);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void unpack(uint4 u, float2 (&v)[2]) {
    v[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    v[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[2]) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x),
                      __float_as_uint(v[1].y));
  }
};
__device__ __forceinline__ float2 pair(float x) { return make_float2(x, x); }

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_float(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ float from_float(float x) {
  return x;
}

// Table row of activation row `row`. An entry outside the table reads the nearest row
// instead of memory past it.
__device__ __forceinline__ int64_t table_row(const SandwichArgs& a, int64_t row) {
  // (row < 2^31; a remainder costs some 30 instructions a thread, in 64 bits three times that.)
  const int64_t at = row < a.n_index ? row : (uint32_t)row % (uint32_t)a.n_index;
  const int64_t t = a.index[at];
  return t < 0 ? 0 : (t >= a.n_table ? a.n_table - 1 : t);
}

// Sum over the whole CTA (`warps` warps); red holds one float per warp.
template <int WARPS>
__device__ __forceinline__ float cta_sum(float v, float* red) {
  v = warp_sum(v);
  if (WARPS == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) s += red[w];
  return s;
}

// Any width and alignment: one CTA per row, scalar accesses, hidden recomputed from L1/L2. Bound by
// its 2- and 4-byte accesses: 51,200 rows of 3071 take 757 us in bf16 and 767 us in fp32 (455 and 500 us
// without the second norm), where their bytes take 192 and 384 us.
constexpr int kScalarWarps = 8;
template <class T>
__global__ void __launch_bounds__(kScalarWarps * 32) sandwich_scalar(SandwichArgs a) {
  __shared__ float red[2][kScalarWarps];
  const int64_t row = blockIdx.x;
  const int64_t t = table_row(a, row);
  const T* residual = (const T*)a.residual + row * a.residual_stride;
  const T* branch = (const T*)a.branch + row * a.branch_stride;
  const T* gate = (const T*)a.gate + t * a.gate_stride;
  const T* post_weight = (const T*)a.post_weight;
  float ss = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
    const float x = to_float(branch[c]);
    ss += x * x;
  }
  ss = cta_sum<kScalarWarps>(ss, red[0]);
  const float post_rstd = rsqrtf(ss / (float)a.cols + a.post_eps);
  auto hidden_at = [&](int64_t c) {
    return a.residual_scale * to_float(residual[c]) +
           to_float(gate[c]) * (to_float(branch[c]) * post_rstd * to_float(post_weight[c]));
  };
  T* hidden = (T*)a.hidden + row * a.hidden_stride;
  float hh = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
    const float h = hidden_at(c);
    hidden[c] = from_float<T>(h);
    hh += h * h;
  }
  if (a.normed == nullptr) return;
  hh = cta_sum<kScalarWarps>(hh, red[1]);
  const float rstd = rsqrtf(hh / (float)a.cols + a.eps);
  const T* weight = (const T*)a.weight;
  const T* scale = (const T*)a.scale + t * a.scale_stride;
  const T* shift = (const T*)a.shift + t * a.shift_stride;
  T* normed = (T*)a.normed + row * a.normed_stride;
  for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x)
    normed[c] = from_float<T>(hidden_at(c) * rstd * to_float(weight[c]) *
                                  (1.f + to_float(scale[c])) + to_float(shift[c]));
}

// The row in registers: WARPS warps per row, NCH 16-byte chunks per thread; after the first
// reduction the 8 registers that held a chunk of branch and residual hold hidden in fp32.
// 51,200 rows of 3072 bf16: 209-213 us (1259 MB, 6.0 TB/s), with single fp32 instructions 216;
// with eight CTAs an SM instead of seven 216, with the second tables loaded before the second
// sum 230 (more registers, fewer rows at once).
template <class T, int WARPS, int NCH, bool NORMED>
__global__ void __launch_bounds__(WARPS * 32) sandwich_vec(SandwichArgs a) {
  constexpr int kN = Vec<T>::kN;
  constexpr int kThreads = WARPS * 32;
  __shared__ float red[2][WARPS];
  const int64_t row = blockIdx.x;
  const int cols = (int)a.cols;
  const T* residual = (const T*)a.residual + row * a.residual_stride;
  const T* branch = (const T*)a.branch + row * a.branch_stride;
  uint4 raw_b[NCH], raw_r[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * kThreads + threadIdx.x) * kN;
    if (col < cols) {
      raw_b[c] = ld_stream(branch + col);
      raw_r[c] = ld_stream(residual + col);
    } else {
      raw_b[c] = raw_r[c] = make_uint4(0, 0, 0, 0);
    }
  }
  const int64_t t = table_row(a, row);
  const T* gate = (const T*)a.gate + t * a.gate_stride;
  const T* post_weight = (const T*)a.post_weight;
  constexpr int kPairs = kN / 2;
  float2 ss2 = pair(0.f);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    float2 x[kPairs];
    Vec<T>::unpack(raw_b[c], x);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) ss2 = __ffma2_rn(x[j], x[j], ss2);
  }
  const float ss = cta_sum<WARPS>(ss2.x + ss2.y, red[0]);
  const float2 post_rstd = pair(rsqrtf(ss / (float)cols + a.post_eps));
  const float2 residual_scale = pair(a.residual_scale);
  T* hidden = (T*)a.hidden + row * a.hidden_stride;
  float2 h[NCH][kPairs];
  float2 hh2 = pair(0.f);
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * kThreads + threadIdx.x) * kN;
    if (col < cols) {
      float2 x[kPairs], r[kPairs], g[kPairs], w[kPairs];
      Vec<T>::unpack(raw_b[c], x);
      Vec<T>::unpack(raw_r[c], r);
      Vec<T>::unpack(ld_cached(gate + col), g);
      Vec<T>::unpack(ld_cached(post_weight + col), w);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float2 b = __fmul2_rn(__fmul2_rn(x[j], post_rstd), w[j]);
        h[c][j] = __ffma2_rn(g[j], b, __fmul2_rn(residual_scale, r[j]));
        hh2 = __ffma2_rn(h[c][j], h[c][j], hh2);
      }
      st_stream(hidden + col, Vec<T>::pack(h[c]));
    }
  }
  if (!NORMED) return;
  const float hh = cta_sum<WARPS>(hh2.x + hh2.y, red[1]);
  const float2 rstd = pair(rsqrtf(hh / (float)cols + a.eps));
  const T* weight = (const T*)a.weight;
  const T* scale = (const T*)a.scale + t * a.scale_stride;
  const T* shift = (const T*)a.shift + t * a.shift_stride;
  T* normed = (T*)a.normed + row * a.normed_stride;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * kThreads + threadIdx.x) * kN;
    if (col < cols) {
      float2 w[kPairs], sc[kPairs], sh[kPairs], o[kPairs];
      Vec<T>::unpack(ld_cached(weight + col), w);
      Vec<T>::unpack(ld_cached(scale + col), sc);
      Vec<T>::unpack(ld_cached(shift + col), sh);
#pragma unroll
      for (int j = 0; j < kPairs; ++j)
        o[j] = __ffma2_rn(__fmul2_rn(__fmul2_rn(h[c][j], rstd), w[j]), __fadd2_rn(pair(1.f), sc[j]),
                          sh[j]);
      st_stream(normed + col, Vec<T>::pack(o));
    }
  }
}

template <class T, int WARPS, int NCH>
void launch_vec(const SandwichArgs& a, cudaStream_t s) {
  if (a.normed != nullptr)
    sandwich_vec<T, WARPS, NCH, true><<<(unsigned)a.rows, WARPS * 32, 0, s>>>(a);
  else
    sandwich_vec<T, WARPS, NCH, false><<<(unsigned)a.rows, WARPS * 32, 0, s>>>(a);
}

// Fewest chunks per thread that up to four keep the row in registers: threads first.
template <class T, int WARPS>
void launch_chunks(const SandwichArgs& a, int chunks, cudaStream_t s) {
  const int nch = (chunks + WARPS * 32 - 1) / (WARPS * 32);
  if (nch == 1) launch_vec<T, WARPS, 1>(a, s);
  else if (nch == 2) launch_vec<T, WARPS, 2>(a, s);
  else if (nch == 3) launch_vec<T, WARPS, 3>(a, s);
  else launch_vec<T, WARPS, 4>(a, s);
}

template <class T>
bool vector_rows(const SandwichArgs& a) {
  constexpr int kN = Vec<T>::kN;
  const bool second = a.normed != nullptr;
  const void* bases[] = {a.hidden, a.residual, a.branch, a.post_weight, a.gate,
                         second ? a.normed : a.hidden, second ? a.weight : a.gate,
                         second ? a.scale : a.gate, second ? a.shift : a.gate};
  for (const void* p : bases)
    if (!aligned16(p)) return false;
  const int64_t strides[] = {a.hidden_stride, a.residual_stride, a.branch_stride, a.gate_stride,
                             second ? a.scale_stride : 0, second ? a.shift_stride : 0};
  for (int64_t v : strides)
    if (v % kN != 0) return false;
  return a.cols % kN == 0 && a.cols / kN <= 4 * 512;
}

template <class T>
int launch_sandwich(const SandwichArgs& a, cudaStream_t s, const char* name) {
  H3B_REQUIRE(a.rows <= 0x7fffffffLL, "%s: too many rows (%lld)", name, (long long)a.rows);
  if (!vector_rows<T>(a)) {
    sandwich_scalar<T><<<(unsigned)a.rows, kScalarWarps * 32, 0, s>>>(a);
    return check_launch(name);
  }
  const int chunks = (int)(a.cols / Vec<T>::kN);
  if (chunks <= 4 * 32) launch_chunks<T, 1>(a, chunks, s);
  else if (chunks <= 4 * 128) launch_chunks<T, 4>(a, chunks, s);
  else if (chunks <= 4 * 256) launch_chunks<T, 8>(a, chunks, s);
  else launch_chunks<T, 16>(a, chunks, s);
  return check_launch(name);
}

}  // namespace
}  // namespace h3b

extern "C" int h3b_sandwich_residual_rmsnorm_modulate(
    void* hidden_out, void* normed_out, const void* residual, const void* branch,
    const void* post_weight, const void* gate, const void* weight, const void* scale,
    const void* shift, const int64_t* index, int64_t rows, int64_t cols, int64_t n_index,
    int64_t n_table, int64_t residual_row_stride, int64_t branch_row_stride,
    int64_t out_row_stride, int64_t gate_row_stride, int64_t scale_row_stride,
    int64_t shift_row_stride, float residual_scale, float post_eps, float eps, int64_t dtype,
    h3b_stream_t stream) {
  const char* name = "h3b_sandwich_residual_rmsnorm_modulate";
  H3B_REQUIRE(rows >= 0 && cols >= 0, "sandwich_residual_rmsnorm_modulate: negative shape");
  H3B_REQUIRE(dtype >= 0 && dtype <= 2, "sandwich_residual_rmsnorm_modulate: unknown dtype %lld",
              (long long)dtype);
  if (rows == 0 || cols == 0) return H3B_OK;
  H3B_REQUIRE(n_index > 0 && n_table > 0,
              "sandwich_residual_rmsnorm_modulate: empty index or table");
  H3B_REQUIRE(hidden_out != nullptr && residual != nullptr && branch != nullptr &&
                  post_weight != nullptr && gate != nullptr && index != nullptr,
              "sandwich_residual_rmsnorm_modulate: null argument");
  H3B_REQUIRE(normed_out == nullptr ||
                  (weight != nullptr && scale != nullptr && shift != nullptr),
              "sandwich_residual_rmsnorm_modulate: normed needs weight, scale and shift");
  h3b::SandwichArgs a{};
  a.hidden = hidden_out;
  a.normed = normed_out;
  a.residual = residual;
  a.branch = branch;
  a.post_weight = post_weight;
  a.gate = gate;
  a.weight = weight;
  a.scale = scale;
  a.shift = shift;
  a.index = index;
  a.rows = rows;
  a.cols = cols;
  a.n_index = n_index;
  a.n_table = n_table;
  a.residual_stride = residual_row_stride;
  a.branch_stride = branch_row_stride;
  a.hidden_stride = a.normed_stride = out_row_stride;
  a.gate_stride = gate_row_stride;
  a.scale_stride = scale_row_stride;
  a.shift_stride = shift_row_stride;
  a.residual_scale = residual_scale;
  a.post_eps = post_eps;
  a.eps = eps;
  if (dtype == H3B_DTYPE_BF16) return h3b::launch_sandwich<__nv_bfloat16>(a, stream, name);
  if (dtype == H3B_DTYPE_FP16) return h3b::launch_sandwich<__half>(a, stream, name);
  return h3b::launch_sandwich<float>(a, stream, name);
}
