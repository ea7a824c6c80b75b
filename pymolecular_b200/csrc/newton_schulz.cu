// Orthogonalised updates: Newton-Schulz products on batches of weight
// matrices, alone or inside the momentum step that uses them.
//
//   X0 = U / (|U|_F + eps)  (m x n with m <= n: transposed where rows > cols)
//   A = X X^T,  X <- a X + (b A + c A A) X      `steps` times
//
// Simple form: the matrices in float32 in the workspace, one launch over all
// matrices' tiles for each product.
#include <algorithm>
#include <cmath>

#include <cuda_fp16.h>

#include "common.cuh"

namespace egnn {
namespace {

constexpr int kItems = 48;      // matrices of one launch (kernel parameters)
constexpr int kMaxSide = 16384;
constexpr int kMaxSmall = 1024;
constexpr int kMaxSteps = 64;

struct NsItem {
  const void* in;        // the matrix, or the gradient (float32) of a step
  void* out;             // its orthogonalised form; NULL in a step
  float* weight;
  float* mom;
  int64_t ld_in, ld_out, ld_mom;   // ld_out: of `out` or `weight`
  int rows, cols, dtype;
  float gain;
  float *x[2], *a, *b;   // workspace: X twice, A, b A + c A A
};

struct NsBatch {
  NsItem it[kItems];
  int tile0[kItems + 1];   // first block of each matrix
  int count;
};

struct NsScalars {
  float a, b, c;
  double eps;
  float mu, nu;             // nu = 1 - mu
  double decay, lr;
  const float* lr_device;
  int nesterov;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == EGNN_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == EGNN_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == EGNN_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == EGNN_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Element (r, c) of U from the gradient and the momentum already updated.
__device__ __forceinline__ float update_value(const NsItem& it, const NsScalars& q, int r, int c) {
  const float g = load_any(it.in, it.dtype, r * it.ld_in + c);
  if (!it.mom) return g;
  const float m = it.mom[r * it.ld_mom + c];
  return q.nesterov ? fmaf(q.mu, m, q.nu * g) : m;
}

__device__ __forceinline__ int item_of(const NsBatch& b, int block) {
  int k = 0;
  while (k + 1 < b.count && b.tile0[k + 1] <= block) ++k;
  return k;
}

// One block per matrix: momentum, |U|_F (squares added in float64: no
// overflow or underflow at any scale of the gradient), X0.
__global__ void __launch_bounds__(512) ns_start_kernel(const __grid_constant__ NsBatch batch, NsScalars q) {
  pdl_enter();
  __shared__ double red[512];
  const NsItem& it = batch.it[blockIdx.x];
  const int n = it.rows * it.cols;
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 512) {
    const int r = i / it.cols, c = i % it.cols;
    if (it.mom) {
      float* m = it.mom + r * it.ld_mom + c;
      *m = fmaf(q.mu, *m, q.nu * load_any(it.in, it.dtype, r * it.ld_in + c));
    }
    const double u = update_value(it, q, r, c);
    s += u * u;
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 256; w > 0; w >>= 1) {
    if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  const double inv = 1.0 / (sqrt(red[0]) + q.eps);
  const bool turn = it.rows > it.cols;
  for (int i = threadIdx.x; i < n; i += 512) {
    const int r = i / it.cols, c = i % it.cols;
    it.x[0][turn ? c * it.rows + r : i] = (float)(update_value(it, q, r, c) * inv);
  }
}

// MODE 0: A = X X^T;  1: B = b A + c A A;  2: X' = a X + B X.
template <int MODE>
__global__ void __launch_bounds__(256) ns_product_kernel(const __grid_constant__ NsBatch batch, NsScalars q, int cur) {
  pdl_enter();
  __shared__ float sa[32][33], sb[32][33];
  const int k = item_of(batch, blockIdx.x);
  const NsItem& it = batch.it[k];
  const int m = min(it.rows, it.cols), n = max(it.rows, it.cols);
  const int N = MODE == 2 ? n : m, K = MODE == 0 ? n : m;
  const int tn = (N + 31) / 32, t = blockIdx.x - batch.tile0[k];
  const int r0 = t / tn * 32, c0 = t % tn * 32;
  const float* L = MODE == 0 ? it.x[cur] : MODE == 1 ? it.a : it.b;   // m x K
  const float* R = MODE == 1 ? it.a : it.x[cur];                     // K x N, or N x K (MODE 0)
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < K; k0 += 32) {
    for (int p = ty; p < 32; p += 8) {
      sa[p][tx] = r0 + p < m && k0 + tx < K ? L[(int64_t)(r0 + p) * K + k0 + tx] : 0.f;
      if (MODE == 0) sb[tx][p] = c0 + p < N && k0 + tx < K ? R[(int64_t)(c0 + p) * K + k0 + tx] : 0.f;
      else sb[p][tx] = k0 + p < K && c0 + tx < N ? R[(int64_t)(k0 + p) * N + c0 + tx] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 32; ++kk)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = fmaf(sa[ty + 8 * j][kk], sb[kk][tx], acc[j]);
    __syncthreads();
    if ((k0 & 480) == 480 || k0 + 32 >= K)   // pieces of 512 terms, so that long sums keep float32's exactness
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[j] += acc[j];
        acc[j] = 0.f;
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    acc[j] = sum[j];
    const int r = r0 + ty + 8 * j, c = c0 + tx;
    if (r >= m || c >= N) continue;
    const int64_t i = (int64_t)r * N + c;
    if (MODE == 0) it.a[i] = acc[j];
    else if (MODE == 1) it.b[i] = fmaf(q.b, it.a[i], q.c * acc[j]);
    else it.x[cur ^ 1][i] = fmaf(q.a, it.x[cur][i], acc[j]);
  }
}

// The result written out, or the weight moved by it.
__global__ void __launch_bounds__(512) ns_finish_kernel(const __grid_constant__ NsBatch batch, NsScalars q, int cur) {
  pdl_enter();
  const NsItem& it = batch.it[blockIdx.x];
  const int n = it.rows * it.cols;
  const bool turn = it.rows > it.cols;
  const double lr = q.lr_device ? (double)*q.lr_device : q.lr;
  const float keep = (float)(1.0 - lr * q.decay), move = (float)(-lr * it.gain);
  for (int i = threadIdx.x; i < n; i += 512) {
    const int r = i / it.cols, c = i % it.cols;
    const float o = it.x[cur][turn ? c * it.rows + r : i];
    if (it.weight) {
      float* w = it.weight + r * it.ld_out + c;
      *w = fmaf(move, o, keep * *w);
    } else {
      store_any(it.out, it.dtype, r * it.ld_out + c, o);
    }
  }
}

// Largest |p| of the odd polynomial on [0, r]: at r or at a root of its
// derivative a + 3 b s^2 + 5 c s^4.
double odd_poly_max(const egnn_ns_options& o, double r) {
  auto p = [&](double s) { return std::fabs(s * (o.a + s * s * (o.b + s * s * o.c))); };
  double most = p(r);
  double roots[2] = {-1.0, -1.0};
  if (o.c != 0.0) {
    const double d = 9.0 * o.b * o.b - 20.0 * o.a * o.c;
    if (d >= 0.0) {
      roots[0] = (-3.0 * o.b + std::sqrt(d)) / (10.0 * o.c);
      roots[1] = (-3.0 * o.b - std::sqrt(d)) / (10.0 * o.c);
    }
  } else if (o.b != 0.0) {
    roots[0] = -o.a / (3.0 * o.b);
  }
  for (double t : roots)
    if (t > 0.0 && t < r * r) most = std::max(most, p(std::sqrt(t)));
  return most;
}

int check_options(const char* what, const egnn_ns_options& o) {
  if (o.steps < 0 || o.steps > kMaxSteps) return fail(EGNN_ERR_INVALID_ARG, "%s: steps must be 0 .. %d", what, kMaxSteps);
  if (!(o.eps >= 0.0) || !std::isfinite(o.eps)) return fail(EGNN_ERR_INVALID_ARG, "%s: eps must not be negative", what);
  if (!std::isfinite(o.a) || !std::isfinite(o.b) || !std::isfinite(o.c))
    return fail(EGNN_ERR_INVALID_ARG, "%s: coefficients must be finite", what);
  double r = 1.0;
  for (int k = 0; k < o.steps; ++k) {
    r = odd_poly_max(o, r);
    if (!(r < 1024.0))
      return fail(EGNN_ERR_INVALID_ARG, "%s: these coefficients let the singular values grow past 1024", what);
  }
  return EGNN_OK;
}

bool size_built(int rows, int cols) {
  return rows >= 0 && cols >= 0 && rows <= kMaxSide && cols <= kMaxSide && std::min(rows, cols) <= kMaxSmall;
}

void carve(Carver& c, int rows, int cols, NsItem* it) {
  const size_t m = std::min(rows, cols), n = std::max(rows, cols);
  float* p[4] = {c.take<float>(m * n), c.take<float>(m * n), c.take<float>(m * m), c.take<float>(m * m)};
  if (it) {
    it->x[0] = p[0];
    it->x[1] = p[1];
    it->a = p[2];
    it->b = p[3];
  }
}

int tiles(int r, int c) { return (r + 31) / 32 * ((c + 31) / 32); }

int run_batch(NsBatch& b, const NsScalars& q, int steps, cudaStream_t s) {
  TimerScope ts("newton_schulz", s);
  EGNN_CHECK_CUDA(launch_pdl(ns_start_kernel, dim3(b.count), dim3(512), 0, s, b, q));
  EGNN_CHECK_LAUNCH();
  int cur = 0;
  for (int k = 0; k < steps; ++k) {
    for (int mode = 0; mode < 3; ++mode) {
      int t = 0;
      for (int i = 0; i < b.count; ++i) {
        const int m = std::min(b.it[i].rows, b.it[i].cols), n = std::max(b.it[i].rows, b.it[i].cols);
        b.tile0[i] = t;
        t += tiles(m, mode == 2 ? n : m);
      }
      b.tile0[b.count] = t;
      auto kernel = mode == 0 ? ns_product_kernel<0> : mode == 1 ? ns_product_kernel<1> : ns_product_kernel<2>;
      EGNN_CHECK_CUDA(launch_pdl(kernel, dim3(t), dim3(256), 0, s, b, q, cur));
      EGNN_CHECK_LAUNCH();
    }
    cur ^= 1;
  }
  EGNN_CHECK_CUDA(launch_pdl(ns_finish_kernel, dim3(b.count), dim3(512), 0, s, b, q, cur));
  EGNN_CHECK_LAUNCH();
  return EGNN_OK;
}

// The matrices in batches of kItems, each with its own part of the workspace.
template <class Fill>
int run_all(const char* what, int64_t count, const Fill& fill, const NsScalars& q, int steps, void* ws,
            size_t ws_bytes, cudaStream_t s) {
  Carver need(nullptr);
  NsItem it;
  for (int64_t i = 0; i < count; ++i) {
    EGNN_TRY(fill(i, it));
    carve(need, it.rows, it.cols, nullptr);
  }
  if (need.size() > 0 && (!ws || ws_bytes < need.size())) return fail(EGNN_ERR_WORKSPACE, "%s: workspace too small", what);
  Carver c(ws);
  NsBatch b;
  b.count = 0;
  for (int64_t i = 0; i < count; ++i) {
    EGNN_TRY(fill(i, b.it[b.count]));
    if (b.it[b.count].rows == 0 || b.it[b.count].cols == 0) continue;
    carve(c, b.it[b.count].rows, b.it[b.count].cols, &b.it[b.count]);
    if (++b.count == kItems) {
      EGNN_TRY(run_batch(b, q, steps, s));
      b.count = 0;
    }
  }
  return b.count ? run_batch(b, q, steps, s) : EGNN_OK;
}

}  // namespace
}  // namespace egnn

using namespace egnn;

extern "C" size_t egnn_orthogonalize_workspace_size(int64_t count, const int32_t* sizes) {
  if (count < 0 || (count > 0 && !sizes)) return 0;
  Carver c(nullptr);
  c.take<float>(1);
  for (int64_t i = 0; i < count; ++i) {
    if (!size_built(sizes[2 * i], sizes[2 * i + 1])) return 0;
    carve(c, sizes[2 * i], sizes[2 * i + 1], nullptr);
  }
  return c.size();
}

extern "C" int egnn_orthogonalize(int64_t count, const egnn_matrix* m, const egnn_ns_options* o, void* ws,
                                  size_t ws_bytes, void* stream) {
  const char* what = "egnn_orthogonalize";
  if (count < 0 || !o || (count > 0 && !m)) return fail(EGNN_ERR_INVALID_ARG, "%s: null pointer or negative count", what);
  EGNN_TRY(check_options(what, *o));
  const NsScalars q{(float)o->a, (float)o->b, (float)o->c, o->eps, 0.f, 0.f, 0.0, 0.0, nullptr, 0};
  auto fill = [&](int64_t i, NsItem& it) -> int {
    const egnn_matrix& x = m[i];
    if (x.dtype < EGNN_DTYPE_F32 || x.dtype > EGNN_DTYPE_F16) return fail(EGNN_ERR_INVALID_ARG, "%s: unknown dtype", what);
    if (x.rows < 0 || x.cols < 0) return fail(EGNN_ERR_INVALID_ARG, "%s: bad shape", what);
    if (!size_built(x.rows, x.cols)) return fail(EGNN_ERR_UNSUPPORTED, "%s: %d x %d is not built", what, x.rows, x.cols);
    if (x.rows > 0 && x.cols > 0) {
      if (!x.in || !x.out) return fail(EGNN_ERR_INVALID_ARG, "%s: null pointer", what);
      if (x.rows > 1 && (x.ld_in < x.cols || x.ld_out < x.cols))
        return fail(EGNN_ERR_INVALID_ARG, "%s: row stride below the row's length", what);
    }
    it = NsItem{};
    it.in = x.in;
    it.out = x.out;
    it.ld_in = x.ld_in;
    it.ld_out = x.ld_out;
    it.rows = x.rows;
    it.cols = x.cols;
    it.dtype = x.dtype;
    return EGNN_OK;
  };
  return run_all(what, count, fill, q, o->steps, ws, ws_bytes, (cudaStream_t)stream);
}

extern "C" int egnn_muon_step(int64_t count, const egnn_muon_matrix* m, const egnn_muon_options* o, void* ws,
                              size_t ws_bytes, void* stream) {
  const char* what = "egnn_muon_step";
  if (count < 0 || !o || (count > 0 && !m)) return fail(EGNN_ERR_INVALID_ARG, "%s: null pointer or negative count", what);
  EGNN_TRY(check_options(what, o->ns));
  if (!(o->momentum >= 0.0 && o->momentum < 1.0)) return fail(EGNN_ERR_INVALID_ARG, "%s: momentum must be in [0, 1)", what);
  const NsScalars q{(float)o->ns.a, (float)o->ns.b, (float)o->ns.c, o->ns.eps, (float)o->momentum,
                    (float)(1.0 - o->momentum), o->weight_decay, o->lr, o->lr_device, o->nesterov != 0};
  auto fill = [&](int64_t i, NsItem& it) -> int {
    const egnn_muon_matrix& x = m[i];
    if (x.rows < 0 || x.cols < 0) return fail(EGNN_ERR_INVALID_ARG, "%s: bad shape", what);
    if (!size_built(x.rows, x.cols)) return fail(EGNN_ERR_UNSUPPORTED, "%s: %d x %d is not built", what, x.rows, x.cols);
    if (x.rows > 0 && x.cols > 0) {
      if (!x.weight || !x.grad || !x.momentum) return fail(EGNN_ERR_INVALID_ARG, "%s: null pointer", what);
      if (x.rows > 1 && (x.ld_weight < x.cols || x.ld_grad < x.cols || x.ld_momentum < x.cols))
        return fail(EGNN_ERR_INVALID_ARG, "%s: row stride below the row's length", what);
    }
    it = NsItem{};
    it.in = x.grad;
    it.weight = x.weight;
    it.mom = x.momentum;
    it.ld_in = x.ld_grad;
    it.ld_out = x.ld_weight;
    it.ld_mom = x.ld_momentum;
    it.rows = x.rows;
    it.cols = x.cols;
    it.dtype = EGNN_DTYPE_F32;
    it.gain = x.gain;
    return EGNN_OK;
  };
  return run_all(what, count, fill, q, o->ns.steps, ws, ws_bytes, (cudaStream_t)stream);
}
