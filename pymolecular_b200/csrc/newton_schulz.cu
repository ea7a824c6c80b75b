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

#include "newton_schulz.cuh"

namespace egnn {
namespace {

constexpr int kMaxSide = 16384;
constexpr int kMaxSmall = 1024;
constexpr int kMaxSteps = 64;

struct NsWork {
  float *x[2], *a, *b;   // X twice, A, b A + c A A
};
struct NsLarge {
  NsBatch n;
  NsWork w[kNsItems];
  int tile0[kNsItems + 1];   // first block of each matrix
};

__device__ __forceinline__ float update_value(const NsItem& it, const NsScalars& q, int r, int c) {
  const float g = ns_load(it.in, it.dtype, r * it.ld_in + c);
  return it.mom ? ns_update(q, g, it.mom[r * it.ld_mom + c]) : g;
}

__device__ __forceinline__ int item_of(const NsLarge& b, int block) {
  int k = 0;
  while (k + 1 < b.n.count && b.tile0[k + 1] <= block) ++k;
  return k;
}

// One block per matrix: momentum, |U|_F (squares added in float64: no
// overflow or underflow at any scale of the gradient), X0.
__global__ void __launch_bounds__(512) ns_start_kernel(const __grid_constant__ NsLarge batch, NsScalars q) {
  pdl_enter();
  __shared__ double red[512];
  const NsItem& it = batch.n.it[blockIdx.x];
  const NsWork& wk = batch.w[blockIdx.x];
  const int n = it.rows * it.cols;
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 512) {
    const int r = i / it.cols, c = i % it.cols;
    if (it.mom) {
      float* m = it.mom + r * it.ld_mom + c;
      *m = ns_momentum(q, ns_load(it.in, it.dtype, r * it.ld_in + c), *m);
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
    wk.x[0][turn ? c * it.rows + r : i] = (float)(update_value(it, q, r, c) * inv);
  }
}

// MODE 0: A = X X^T;  1: B = b A + c A A;  2: X' = a X + B X.
template <int MODE>
__global__ void __launch_bounds__(256) ns_product_kernel(const __grid_constant__ NsLarge batch, NsScalars q, int cur) {
  pdl_enter();
  __shared__ float sa[32][33], sb[32][33];
  const int k = item_of(batch, blockIdx.x);
  const NsItem& it = batch.n.it[k];
  const NsWork& wk = batch.w[k];
  const int m = min(it.rows, it.cols), n = max(it.rows, it.cols);
  const int N = MODE == 2 ? n : m, K = MODE == 0 ? n : m;
  const int tn = (N + 31) / 32, t = blockIdx.x - batch.tile0[k];
  const int r0 = t / tn * 32, c0 = t % tn * 32;
  const float* L = MODE == 0 ? wk.x[cur] : MODE == 1 ? wk.a : wk.b;   // m x K
  const float* R = MODE == 1 ? wk.a : wk.x[cur];                     // K x N, or N x K (MODE 0)
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
    if (MODE == 0) wk.a[i] = acc[j];
    else if (MODE == 1) wk.b[i] = fmaf(q.b, wk.a[i], q.c * acc[j]);
    else wk.x[cur ^ 1][i] = fmaf(q.a, wk.x[cur][i], acc[j]);
  }
}

// The result written out, or the weight moved by it.
__global__ void __launch_bounds__(512) ns_finish_kernel(const __grid_constant__ NsLarge batch, NsScalars q, int cur) {
  pdl_enter();
  const NsItem& it = batch.n.it[blockIdx.x];
  const NsWork& wk = batch.w[blockIdx.x];
  const int n = it.rows * it.cols;
  const bool turn = it.rows > it.cols;
  float keep = 0.f, move = 0.f;
  if (it.mom) ns_rates(it, q, keep, move);
  for (int i = threadIdx.x; i < n; i += 512) {
    const int r = i / it.cols, c = i % it.cols;
    const float o = wk.x[cur][turn ? c * it.rows + r : i];
    if (it.mom) {
      float* w = static_cast<float*>(it.out) + r * it.ld_out + c;
      *w = fmaf(move, o, keep * *w);
    } else {
      ns_store(it.out, it.dtype, r * it.ld_out + c, o);
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

// 2^e with size 2^e near 2^14: a factor 4 below fp16's largest value.
float scale_for(double size) {
  if (!(size > 0.0)) return 1.f;
  const int e = 14 - (int)std::ceil(std::log2(size));
  return (float)std::ldexp(1.0, std::max(-60, std::min(60, e)));
}

// Checks the options and derives the scales from how far the singular values can grow.
int scalars(const char* what, const egnn_ns_options& o, NsScalars& q) {
  if (o.steps < 0 || o.steps > kMaxSteps) return fail(EGNN_ERR_INVALID_ARG, "%s: steps must be 0 .. %d", what, kMaxSteps);
  if (!(o.eps >= 0.0) || !std::isfinite(o.eps)) return fail(EGNN_ERR_INVALID_ARG, "%s: eps must not be negative", what);
  if (!std::isfinite(o.a) || !std::isfinite(o.b) || !std::isfinite(o.c))
    return fail(EGNN_ERR_INVALID_ARG, "%s: coefficients must be finite", what);
  double r = 1.0, most = 1.0;
  for (int k = 0; k < o.steps; ++k) {
    r = odd_poly_max(o, r);
    if (!(r < 1024.0))
      return fail(EGNN_ERR_INVALID_ARG, "%s: these coefficients let the singular values grow past 1024", what);
    most = std::max(most, r);
  }
  q = NsScalars{};
  q.a = (float)o.a;
  q.b = (float)o.b;
  q.c = (float)o.c;
  q.eps = o.eps;
  q.steps = o.steps;
  q.sx = scale_for(most);
  q.sa = scale_for(most * most);
  q.sb = scale_for(std::fabs(o.b) * most * most + std::fabs(o.c) * most * most * most * most);
  return EGNN_OK;
}

bool size_built(int rows, int cols) {
  return rows >= 0 && cols >= 0 && rows <= kMaxSide && cols <= kMaxSide && std::min(rows, cols) <= kMaxSmall;
}

bool is_large(int rows, int cols) { return !ns_fused_fits(std::min(rows, cols), std::max(rows, cols)); }

// Workspace of a matrix that a block's shared memory does not hold.
void carve(Carver& c, int rows, int cols, NsWork* w) {
  const size_t m = std::min(rows, cols), n = std::max(rows, cols);
  if (m == 0 || !is_large(rows, cols)) return;
  float* p[4] = {c.take<float>(m * n), c.take<float>(m * n), c.take<float>(m * m), c.take<float>(m * m)};
  if (w) *w = NsWork{{p[0], p[1]}, p[2], p[3]};
}

int tiles(int r, int c) { return (r + 31) / 32 * ((c + 31) / 32); }

int run_large(NsLarge& b, const NsScalars& q, cudaStream_t s) {
  TimerScope ts("newton_schulz", s);
  EGNN_CHECK_CUDA(launch_pdl(ns_start_kernel, dim3(b.n.count), dim3(512), 0, s, b, q));
  EGNN_CHECK_LAUNCH();
  int cur = 0;
  for (int k = 0; k < q.steps; ++k) {
    for (int mode = 0; mode < 3; ++mode) {
      int t = 0;
      for (int i = 0; i < b.n.count; ++i) {
        const int m = std::min(b.n.it[i].rows, b.n.it[i].cols), n = std::max(b.n.it[i].rows, b.n.it[i].cols);
        b.tile0[i] = t;
        t += tiles(m, mode == 2 ? n : m);
      }
      b.tile0[b.n.count] = t;
      auto kernel = mode == 0 ? ns_product_kernel<0> : mode == 1 ? ns_product_kernel<1> : ns_product_kernel<2>;
      EGNN_CHECK_CUDA(launch_pdl(kernel, dim3(t), dim3(256), 0, s, b, q, cur));
      EGNN_CHECK_LAUNCH();
    }
    cur ^= 1;
  }
  EGNN_CHECK_CUDA(launch_pdl(ns_finish_kernel, dim3(b.n.count), dim3(512), 0, s, b, q, cur));
  EGNN_CHECK_LAUNCH();
  return EGNN_OK;
}

// The matrices that fit a block's shared memory in batches of one launch, the
// large ones in batches of their own.  Everything is checked before the first
// launch.
template <class Fill>
int run_all(const char* what, int64_t count, const Fill& fill, const NsScalars& q, void* ws, size_t ws_bytes,
            cudaStream_t s) {
  if (count == 0) return EGNN_OK;
  Carver need(nullptr);
  need.take<float>(1);
  NsItem it;
  for (int64_t i = 0; i < count; ++i) {
    EGNN_TRY(fill(i, it));
    carve(need, it.rows, it.cols, nullptr);
  }
  if (!ws || ws_bytes < need.size()) return fail(EGNN_ERR_WORKSPACE, "%s: workspace too small", what);
  Carver c(ws);
  c.take<float>(1);
  NsBatch small;
  NsLarge large;
  small.count = large.n.count = 0;
  for (int64_t i = 0; i < count; ++i) {
    EGNN_TRY(fill(i, it));
    if (it.rows == 0 || it.cols == 0) continue;
    if (is_large(it.rows, it.cols)) {
      carve(c, it.rows, it.cols, &large.w[large.n.count]);
      large.n.it[large.n.count] = it;
      if (++large.n.count == kNsItems) {
        EGNN_TRY(run_large(large, q, s));
        large.n.count = 0;
      }
    } else {
      small.it[small.count] = it;
      if (++small.count == kNsItems) {
        EGNN_TRY(ns_fused(small, q, s));
        small.count = 0;
      }
    }
  }
  if (small.count) EGNN_TRY(ns_fused(small, q, s));
  return large.n.count ? run_large(large, q, s) : EGNN_OK;
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
  NsScalars q;
  EGNN_TRY(scalars(what, *o, q));
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
  return run_all(what, count, fill, q, ws, ws_bytes, (cudaStream_t)stream);
}

extern "C" int egnn_muon_step(int64_t count, const egnn_muon_matrix* m, const egnn_muon_options* o, void* ws,
                              size_t ws_bytes, void* stream) {
  const char* what = "egnn_muon_step";
  if (count < 0 || !o || (count > 0 && !m)) return fail(EGNN_ERR_INVALID_ARG, "%s: null pointer or negative count", what);
  NsScalars q;
  EGNN_TRY(scalars(what, o->ns, q));
  if (!(o->momentum >= 0.0 && o->momentum < 1.0)) return fail(EGNN_ERR_INVALID_ARG, "%s: momentum must be in [0, 1)", what);
  q.mu = (float)o->momentum;
  q.nu = (float)(1.0 - o->momentum);
  q.decay = o->weight_decay;
  q.lr = o->lr;
  q.lr_device = o->lr_device;
  q.nesterov = o->nesterov != 0;
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
    it.out = x.weight;
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
  return run_all(what, count, fill, q, ws, ws_bytes, (cudaStream_t)stream);
}
