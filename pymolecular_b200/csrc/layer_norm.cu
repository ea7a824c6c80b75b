// Layer normalisation of node features, forward and backward.
//
//   mu = mean_j x_j,  s = 1 / sqrt(mean_j (x_j - mu)^2 + eps),  u_j = (x_j - mu) s
//   y_j  = u_j w_j + b_j
//   dx_j = s (g_j - mean g - u_j mean(g u)),  g_j = dy_j w_j
//   dw_j = sum_rows dy_j u_j,  db_j = sum_rows dy_j
//
// One pass over the data in each direction: a row lives in the registers of
// the threads that share it, the variance is taken from the centred values
// (two reductions, no cancellation at large means), all sums in fp32.
// The forward keeps (mu, s) per row for the backward.  Both directions are
// bound by HBM (8 or 20 flops per element): 2^20 x 128 float32 takes 169 us
// forward and 263 us backward, 97 % and 94 % of the measured copy rate; small
// calls by latency (1850 x 64 forward: 2.3 us).
//
// Rows are shared by TPR threads: 8, 16 or 32 lanes of a warp with NV
// vectors each, or a whole block for wide rows.  The weight's gradient is
// kept by each thread for its own columns over all rows the block visits, summed
// over the block's row groups in order, written as one partial per block, and
// the partials are summed in block order by a second kernel: no atomics,
// bit-identical reruns.
#include <algorithm>
#include <type_traits>

#include <cuda_fp16.h>

#include "common.cuh"

namespace egnn {
namespace {

constexpr int kMaxCols = 8192;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
  else return __float2half_rn(v);
}

// VEC consecutive elements: one 16-byte access (VEC > 1) or one scalar.
template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void widen(const Vec<T, VEC>& r, float* out) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) out[k] = to_f(r.v[k]);
}
// The vectors of R rows (base, base + step, ...) that belong to thread l of a
// row; zeros past the row's end and past the last row.
template <typename T, int VEC, int NV, int TPR, int R>
__device__ __forceinline__ void load_rows(const T* __restrict__ p, int64_t ld, int64_t base, int step, int64_t rows,
                                          int cols, int l, Vec<T, VEC> (&to)[R][NV]) {
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int64_t r = base + k * step;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + l) * VEC;
      if (r < rows && c < cols) {
        to[k][v] = *reinterpret_cast<const Vec<T, VEC>*>(p + r * ld + c);
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) to[k][v].v[q] = from_f<T>(0.f);
      }
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* in) {
  Vec<T, VEC> r;
#pragma unroll
  for (int k = 0; k < VEC; ++k) r.v[k] = from_f<T>(in[k]);
  *reinterpret_cast<Vec<T, VEC>*>(p) = r;
}

// Element i of a parameter vector of type float (same = 0) or T (same = 1);
// `none` where there is no such vector.
template <typename T>
__device__ __forceinline__ float param(const void* p, int same, int i, float none) {
  if (!p) return none;
  return same ? to_f(static_cast<const T*>(p)[i]) : static_cast<const float*>(p)[i];
}

// Sums over the TPR threads of a row, for R rows at once; every thread gets
// them.  Fixed order.
template <int TPR, int R>
__device__ __forceinline__ void row_sum(float (&a)[R], float* red) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int d = W / 2; d > 0; d >>= 1)
#pragma unroll
    for (int k = 0; k < R; ++k) a[k] += __shfl_xor_sync(0xffffffffu, a[k], d);
  if constexpr (TPR > 32) {
    __syncthreads();   // the previous sums have been read
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < R; ++k) red[(threadIdx.x >> 5) * R + k] = a[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 32; ++w) s += red[w * R + k];
      a[k] = s;
    }
  }
}

template <int TPR>
constexpr int block_threads() { return TPR > 32 ? TPR : 256; }

template <typename T, int VEC, int NV, int TPR, int R>
__global__ void __launch_bounds__(block_threads<TPR>())
    layer_norm_fwd_kernel(int64_t rows, int cols, const T* __restrict__ x, int64_t ldx, const void* __restrict__ w,
                          const void* __restrict__ b, int same, float eps, T* __restrict__ y,
                          float2* __restrict__ stats) {
  constexpr int GROUPS = block_threads<TPR>() / TPR;
  __shared__ float red[TPR > 32 ? TPR / 32 * R : 1];
  const int g = threadIdx.x / TPR, l = threadIdx.x % TPR;
  const float inv = 1.f / (float)cols;
  pdl_enter();
  float wv[NV * VEC], bv[NV * VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = (v * TPR + l) * VEC + k;
      wv[v * VEC + k] = c < cols ? param<T>(w, same, c, 1.f) : 0.f;
      bv[v * VEC + k] = c < cols ? param<T>(b, same, c, 0.f) : 0.f;
    }
  const int64_t stride = (int64_t)gridDim.x * GROUPS * R;
  int64_t base = (int64_t)blockIdx.x * GROUPS * R;
  Vec<T, VEC> next[R][NV];   // the next rows are on their way while these are summed
  load_rows<T, VEC, NV, TPR, R>(x, ldx, base + g, GROUPS, rows, cols, l, next);
#pragma unroll 1
  for (; base < rows; base += stride) {
    float xv[R][NV * VEC];
    float sum[R], sq[R];
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int v = 0; v < NV; ++v) widen(next[k][v], &xv[k][v * VEC]);
    load_rows<T, VEC, NV, TPR, R>(x, ldx, base + stride + g, GROUPS, rows, cols, l, next);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      sum[k] = 0.f;
#pragma unroll
      for (int q = 0; q < NV * VEC; ++q) sum[k] += xv[k][q];
    }
    row_sum<TPR, R>(sum, red);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const float mu = sum[k] * inv;
      sum[k] = mu;
      sq[k] = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if ((v * TPR + l) * VEC < cols)
#pragma unroll
          for (int q = 0; q < VEC; ++q) {
            xv[k][v * VEC + q] -= mu;
            sq[k] = fmaf(xv[k][v * VEC + q], xv[k][v * VEC + q], sq[k]);
          }
    }
    row_sum<TPR, R>(sq, red);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t r = base + k * GROUPS + g;
      const float s = rsqrtf(fmaf(sq[k], inv, eps));
      if (r >= rows) continue;
      if (stats && l == 0) stats[r] = make_float2(sum[k], s);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * TPR + l) * VEC;
        if (c >= cols) continue;
        float o[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) o[q] = fmaf(xv[k][v * VEC + q] * s, wv[v * VEC + q], bv[v * VEC + q]);
        store_vec<T, VEC>(y + r * cols + c, o);
      }
    }
  }
}

template <typename T, int VEC, int NV, int TPR, int R>
__global__ void __launch_bounds__(block_threads<TPR>())
    layer_norm_bwd_kernel(int64_t rows, int cols, const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                          int64_t lddy, const void* __restrict__ w, int same, const float2* __restrict__ stats,
                          T* __restrict__ dx, float* __restrict__ part) {
  constexpr int GROUPS = block_threads<TPR>() / TPR;
  constexpr int E = NV * VEC;
  __shared__ float red[TPR > 32 ? TPR / 32 * 2 * R : 1];
  __shared__ float fold[GROUPS > 1 ? block_threads<TPR>() * E : 1];
  const int g = threadIdx.x / TPR, l = threadIdx.x % TPR;
  const float inv = 1.f / (float)cols;
  pdl_enter();
  float wv[E], dw[E], db[E];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = (v * TPR + l) * VEC + k;
      wv[v * VEC + k] = c < cols ? param<T>(w, same, c, 1.f) : 0.f;
      dw[v * VEC + k] = db[v * VEC + k] = 0.f;
    }
  const int64_t stride = (int64_t)gridDim.x * GROUPS * R;
  int64_t base = (int64_t)blockIdx.x * GROUPS * R;
  // A block's row keeps the next one on its way (60000 x 1000: 114 us against
  // 153); lanes of a warp, many rows to an SM, do better without (2^20 x 128: 263 us
  // against 279).
  constexpr bool AHEAD = TPR > 32;
  Vec<T, VEC> nx[R][NV], nd[R][NV];
  if (AHEAD) {
    load_rows<T, VEC, NV, TPR, R>(x, ldx, base + g, GROUPS, rows, cols, l, nx);
    load_rows<T, VEC, NV, TPR, R>(dy, lddy, base + g, GROUPS, rows, cols, l, nd);
  }
#pragma unroll 1
  for (; base < rows; base += stride) {
    float u[R][E], d[R][E], sums[2 * R];
    float2 st[R];
    if (!AHEAD) {
      load_rows<T, VEC, NV, TPR, R>(x, ldx, base + g, GROUPS, rows, cols, l, nx);
      load_rows<T, VEC, NV, TPR, R>(dy, lddy, base + g, GROUPS, rows, cols, l, nd);
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t r = base + k * GROUPS + g;
      st[k] = r < rows ? stats[r] : make_float2(0.f, 0.f);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        widen(nx[k][v], &u[k][v * VEC]);
        widen(nd[k][v], &d[k][v * VEC]);
      }
    }
    if (AHEAD) {
      load_rows<T, VEC, NV, TPR, R>(x, ldx, base + stride + g, GROUPS, rows, cols, l, nx);
      load_rows<T, VEC, NV, TPR, R>(dy, lddy, base + stride + g, GROUPS, rows, cols, l, nd);
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      sums[2 * k] = sums[2 * k + 1] = 0.f;
      const bool row = base + k * GROUPS + g < rows;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (row && (v * TPR + l) * VEC < cols)
#pragma unroll
          for (int q = 0; q < VEC; ++q) {
            const int e = v * VEC + q;
            u[k][e] = (u[k][e] - st[k].x) * st[k].y;
            dw[e] = fmaf(d[k][e], u[k][e], dw[e]);
            db[e] += d[k][e];
            d[k][e] *= wv[e];
            sums[2 * k] += d[k][e];
            sums[2 * k + 1] = fmaf(d[k][e], u[k][e], sums[2 * k + 1]);
          }
    }
    if (!dx) continue;
    row_sum<TPR, 2 * R>(sums, red);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t r = base + k * GROUPS + g;
      if (r >= rows) continue;
      const float m0 = sums[2 * k] * inv, m1 = sums[2 * k + 1] * inv;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * TPR + l) * VEC;
        if (c >= cols) continue;
        float o[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) o[q] = st[k].y * (d[k][v * VEC + q] - m0 - u[k][v * VEC + q] * m1);
        store_vec<T, VEC>(dx + r * cols + c, o);
      }
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = ((e / VEC) * TPR + l) * VEC + e % VEC;
      if (c < cols) {
        out[c] = dw[e];
        out[cols + c] = db[e];
      }
    }
  } else {
    // fold[e][thread]: the block's row groups are added in order
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) fold[e * block_threads<TPR>() + threadIdx.x] = half ? db[e] : dw[e];
      __syncthreads();
      for (int i = threadIdx.x; i < E * TPR; i += block_threads<TPR>()) {
        const int e = i / TPR, lane = i % TPR;
        const int c = ((e / VEC) * TPR + lane) * VEC + e % VEC;
        if (c >= cols) continue;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) s += fold[e * block_threads<TPR>() + q * TPR + lane];
        out[half * cols + c] = s;
      }
    }
  }
}

// dw, db = the blocks' partials added in block order: warp k of a block takes
// the k-th 32nd of them for 32 columns, the pieces are added in order.
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_fold_kernel(int n, int cols, const float* __restrict__ part,
                                                               void* __restrict__ dw, void* __restrict__ db, int same) {
  pdl_enter();
  __shared__ float red[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;   // 0 .. 2 cols - 1: dw then db
  const int per = (n + 31) / 32, lo = warp * per, hi = min(n, lo + per);
  float s = 0.f;
  if (c < 2 * cols) {
#pragma unroll 8
    for (int i = lo; i < hi; ++i) s += part[(int64_t)i * 2 * cols + c];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp || c >= 2 * cols) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) s += red[k][lane];
  void* to = c < cols ? dw : db;
  const int i = c < cols ? c : c - cols;
  if (!to) return;
  if (same) static_cast<T*>(to)[i] = from_f<T>(s);
  else static_cast<float*>(to)[i] = s;
}

// Most blocks of a backward, which is also the number of partials.
constexpr int kMaxPartials = 8;   // to an SM
int bwd_max_blocks(int num_sms) { return num_sms * kMaxPartials; }

struct FwdArgs {
  int64_t rows;
  int cols;
  const void* x;
  int64_t ldx;
  const void *w, *b;
  int same;
  float eps;
  void* y;
  float2* stats;
};
struct BwdArgs {
  int64_t rows;
  int cols;
  const void* x;
  int64_t ldx;
  const void* dy;
  int64_t lddy;
  const void* w;
  int same;
  const float2* stats;
  void* dx;
  float* part;
  int* n_part;
};

// Blocks of a kernel that an SM holds: a grid of that many keeps
// every block at work to the end (60000 x 1000 backward: 114 us; one that is
// not a multiple, 135).
template <class K>
int blocks_per_sm(K kernel, int threads) {
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess) n = 2;
  return std::max(1, n);
}

template <typename T, int VEC, int NV, int TPR, int R>
int launch_fwd(const FwdArgs& a, cudaStream_t s) {
  constexpr int GROUPS = block_threads<TPR>() / TPR;
  const int64_t need = (a.rows + GROUPS * R - 1) / (GROUPS * R);
  static const int fit = blocks_per_sm(layer_norm_fwd_kernel<T, VEC, NV, TPR, R>, block_threads<TPR>());
  const int blocks = (int)std::min<int64_t>(need, (int64_t)num_sms_current() * fit);
  EGNN_CHECK_CUDA(launch_pdl(layer_norm_fwd_kernel<T, VEC, NV, TPR, R>, dim3(blocks), dim3(block_threads<TPR>()), 0, s,
                             a.rows, a.cols, static_cast<const T*>(a.x), a.ldx, a.w, a.b, a.same, a.eps,
                             static_cast<T*>(a.y), a.stats));
  EGNN_CHECK_LAUNCH();
  return EGNN_OK;
}

template <typename T, int VEC, int NV, int TPR, int R>
int launch_bwd(const BwdArgs& a, cudaStream_t s) {
  constexpr int GROUPS = block_threads<TPR>() / TPR;
  const int64_t need = (a.rows + GROUPS * R - 1) / (GROUPS * R);
  // as many blocks as are resident, but 16 rounds of rows to each, so that the
  // partials stay few, as far as two blocks to an SM allow it
  static const int fit = std::min(kMaxPartials, blocks_per_sm(layer_norm_bwd_kernel<T, VEC, NV, TPR, R>, block_threads<TPR>()));
  const int64_t sms = num_sms_current();
  const int blocks =
      (int)std::min<int64_t>(need, std::max<int64_t>(std::min(fit, 2) * sms, std::min<int64_t>(need / 16, fit * sms)));
  *a.n_part = blocks;
  EGNN_CHECK_CUDA(launch_pdl(layer_norm_bwd_kernel<T, VEC, NV, TPR, R>, dim3(blocks), dim3(block_threads<TPR>()), 0, s,
                             a.rows, a.cols, static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.dy), a.lddy,
                             a.w, a.same, a.stats, static_cast<T*>(a.dx), a.part));
  EGNN_CHECK_LAUNCH();
  return EGNN_OK;
}

// Rows that a group of threads takes at once: 32 bytes to a thread in the
// forward (2^20 x 128 float32: 169 us; 64 bytes 178, 16 bytes 187), 8 elements
// in the backward (263 us; 16 elements 277, 4 elements 288), or twice that where
// it keeps two rows together (32117 x 256: 19.4 us against 21.1).
constexpr int rows_at_once(int size, int tpr, int most) { return tpr > 32 || size >= most ? 1 : most / size; }

struct Fwd {
  const FwdArgs& a;
  cudaStream_t s;
  template <typename T>
  static constexpr bool twelve() { return true; }
  template <typename T, int VEC, int NV, int TPR>
  int run() const { return launch_fwd<T, VEC, NV, TPR, rows_at_once(VEC * NV * (int)sizeof(T), TPR, 32)>(a, s); }
};
struct Bwd {
  const BwdArgs& a;
  cudaStream_t s;
  template <typename T>
  static constexpr bool twelve() { return sizeof(T) == 2; }
  template <typename T, int VEC, int NV, int TPR>
  int run() const { return launch_bwd<T, VEC, NV, TPR, rows_at_once(VEC * NV, TPR, sizeof(T) == 2 || VEC * NV == 8 ? 16 : 8)>(a, s); }
};

// The sharing of a row: lanes of a warp while they hold at most 16 elements
// each, else a block with 8 to a thread.  Narrow rows are taken several at a
// time so that each thread keeps enough loads in flight.  257 to 384 scalars are
// 12 to a lane and not 16 (30011 x 321 bf16: forward 11.3 us against 15.2, backward
// 20.8 against 21.9), but in a float32 backward (47.0 against 35.2).
template <typename T, int VEC, class F>
int dispatch_cols(int cols, const F& f) {
  const int v = (cols + VEC - 1) / VEC;   // vectors in a row
  if (v <= 8) return f.template run<T, VEC, 1, 8>();
  if (v <= 16) return f.template run<T, VEC, 1, 16>();
  if (v <= 32) return f.template run<T, VEC, 1, 32>();
  if (v <= 64) return f.template run<T, VEC, 2, 32>();
  if constexpr (VEC < 8) {
    if (v <= 128) return f.template run<T, VEC, 4, 32>();
  }
  if constexpr (VEC == 1) {
    if (v <= 256) return f.template run<T, VEC, 8, 32>();
    if constexpr (F::template twelve<T>())
      if (v <= 384) return f.template run<T, VEC, 12, 32>();
    if (v <= 512) return f.template run<T, VEC, 16, 32>();
  }
  if (cols <= 1024) return f.template run<T, VEC, 8 / VEC, 128>();
  if (cols <= 2048) return f.template run<T, VEC, 8 / VEC, 256>();
  if (cols <= 4096) return f.template run<T, VEC, 8 / VEC, 512>();
  return f.template run<T, VEC, 8 / VEC, 1024>();
}

// 16-byte accesses where every row of every operand starts on a 16-byte
// boundary, scalars elsewhere.
template <typename T, class F>
int dispatch_vec(int cols, bool aligned, const F& f) {
  if (aligned) return dispatch_cols<T, 16 / sizeof(T)>(cols, f);
  return dispatch_cols<T, 1>(cols, f);
}

template <class F>
int dispatch(int dtype, int cols, bool aligned, const F& f) {
  if (dtype == EGNN_DTYPE_F32) return dispatch_vec<float>(cols, aligned, f);
  if (dtype == EGNN_DTYPE_BF16) return dispatch_vec<__nv_bfloat16>(cols, aligned, f);
  return dispatch_vec<__half>(cols, aligned, f);
}

size_t dtype_size(int dtype) { return dtype == EGNN_DTYPE_F32 ? 4 : 2; }

bool rows_aligned(const void* p, int64_t ld, int cols, size_t size) {
  return !(reinterpret_cast<uintptr_t>(p) & 15u) && (size_t)cols * size % 16 == 0 && (size_t)ld * size % 16 == 0;
}

int check_shape(const char* what, int64_t rows, int32_t cols, int64_t ld, int32_t dtype, int32_t param_dtype) {
  if (rows < 0 || cols < 1) return fail(EGNN_ERR_INVALID_ARG, "%s: bad shape", what);
  if (cols > kMaxCols) return fail(EGNN_ERR_UNSUPPORTED, "%s: %d columns (at most %d)", what, cols, kMaxCols);
  if (ld < cols && rows > 1) return fail(EGNN_ERR_INVALID_ARG, "%s: row stride below the row's length", what);
  if (dtype < EGNN_DTYPE_F32 || dtype > EGNN_DTYPE_F16) return fail(EGNN_ERR_INVALID_ARG, "%s: unknown dtype", what);
  if (param_dtype != EGNN_DTYPE_F32 && param_dtype != dtype)
    return fail(EGNN_ERR_INVALID_ARG, "%s: parameters are float32 or of the rows' type", what);
  return EGNN_OK;
}

}  // namespace
}  // namespace egnn

using namespace egnn;

extern "C" int egnn_layer_norm_fwd(int64_t rows, int32_t cols, const void* x, int64_t ldx, int32_t dtype,
                                   const void* weight, const void* bias, int32_t param_dtype, float eps, void* y,
                                   float* stats, void* stream) {
  EGNN_TRY(check_shape("egnn_layer_norm_fwd", rows, cols, ldx, dtype, param_dtype));
  if (!(eps >= 0.f)) return fail(EGNN_ERR_INVALID_ARG, "egnn_layer_norm_fwd: eps must not be negative");
  if (rows == 0) return EGNN_OK;
  if (!x || !y) return fail(EGNN_ERR_INVALID_ARG, "egnn_layer_norm_fwd: null pointer");
  cudaStream_t s = (cudaStream_t)stream;
  const size_t size = dtype_size(dtype);
  const FwdArgs a{rows, cols, x, ldx, weight, bias, param_dtype == dtype && dtype != EGNN_DTYPE_F32, eps, y,
                  reinterpret_cast<float2*>(stats)};
  const bool aligned = rows_aligned(x, rows > 1 ? ldx : cols, cols, size) && rows_aligned(y, cols, cols, size);
  TimerScope ts("layer_norm", s);
  return dispatch(dtype, cols, aligned, Fwd{a, s});
}

extern "C" size_t egnn_layer_norm_workspace_size(int64_t rows, int32_t cols) {
  if (rows < 0 || cols < 1 || cols > kMaxCols) return 0;
  Carver c(nullptr);
  c.take<float>((size_t)std::min<int64_t>(std::max<int64_t>(rows, 1), bwd_max_blocks(num_sms_current())) * 2 * cols);
  return c.size();
}

extern "C" int egnn_layer_norm_bwd(int64_t rows, int32_t cols, const void* x, int64_t ldx, const void* dy,
                                   int64_t lddy, int32_t dtype, const void* weight, int32_t param_dtype,
                                   const float* stats, void* dx, void* dw, void* db, void* ws, size_t ws_bytes,
                                   void* stream) {
  EGNN_TRY(check_shape("egnn_layer_norm_bwd", rows, cols, std::min(ldx, lddy), dtype, param_dtype));
  cudaStream_t s = (cudaStream_t)stream;
  const size_t size = dtype_size(dtype);
  const int same = param_dtype == dtype && dtype != EGNN_DTYPE_F32;
  if (rows == 0) {
    const size_t bytes = (size_t)cols * dtype_size(param_dtype);
    if (dw) EGNN_CHECK_CUDA(cudaMemsetAsync(dw, 0, bytes, s));
    if (db) EGNN_CHECK_CUDA(cudaMemsetAsync(db, 0, bytes, s));
    return EGNN_OK;
  }
  if (!x || !dy || !stats) return fail(EGNN_ERR_INVALID_ARG, "egnn_layer_norm_bwd: null pointer");
  if (!dx && !dw && !db) return EGNN_OK;
  Carver c(ws);
  float* part = nullptr;
  if (dw || db) {
    if (!ws || ws_bytes < egnn_layer_norm_workspace_size(rows, cols))
      return fail(EGNN_ERR_WORKSPACE, "egnn_layer_norm_bwd: workspace too small");
    part = c.take<float>(0);
  }
  int n = 0;
  const BwdArgs a{rows, cols, x, ldx, dy, lddy, weight, same, reinterpret_cast<const float2*>(stats), dx, part, &n};
  const bool aligned = rows_aligned(x, rows > 1 ? ldx : cols, cols, size) &&
                       rows_aligned(dy, rows > 1 ? lddy : cols, cols, size) &&
                       (!dx || rows_aligned(dx, cols, cols, size));
  TimerScope ts("layer_norm", s);
  EGNN_TRY(dispatch(dtype, cols, aligned, Bwd{a, s}));
  if (!part) return EGNN_OK;
  const dim3 grid((2 * cols + 31) / 32);
  if (dtype == EGNN_DTYPE_BF16)
    EGNN_CHECK_CUDA(launch_pdl(layer_norm_fold_kernel<__nv_bfloat16>, grid, dim3(1024), 0, s, n, cols, (const float*)part,
                               dw, db, same));
  else
    EGNN_CHECK_CUDA(launch_pdl(layer_norm_fold_kernel<__half>, grid, dim3(1024), 0, s, n, cols, (const float*)part, dw,
                               db, same));
  EGNN_CHECK_LAUNCH();
  return EGNN_OK;
}
