// Orthogonalised updates: Newton-Schulz products on batches of weight
// matrices, alone or inside the momentum step that uses them.  The entry
// points: checks, scales, and the choice between the two kernels.
//
//   X0 = U / (|U|_F + eps)  (m x n with m <= n: transposed where rows > cols)
//   A = X X^T,  X <- a X + (b A + c A A) X      `steps` times
//
// A matrix whose X and A fit a block's shared memory (m <= 128 and n a few
// hundred: every weight of a model with H <= 128) is iterated there by one
// block; a larger one by a group of blocks, through L2.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "newton_schulz.cuh"

namespace egnn {
namespace {

constexpr int kMaxSide = 16384;
constexpr int kMaxSmall = 1024;

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

// Largest |p(s) / s| of it on [0, r]: at the ends or where its derivative in s^2 is zero.
double even_poly_max(const egnn_ns_options& o, double r) {
  auto p = [&](double t) { return std::fabs(o.a + t * (o.b + t * o.c)); };
  double most = std::max(p(0.0), p(r * r));
  const double t = o.c != 0.0 ? -o.b / (2.0 * o.c) : -1.0;
  if (t > 0.0 && t < r * r) most = std::max(most, p(t));
  return most;
}

// The least e with x <= 2^e, within what the kernels work with.
int exponent_above(double x) {
  if (!(x > 0.0)) return -kNsMostExp;
  return (int)std::max<double>(-kNsMostExp, std::min<double>(kNsMostExp, std::ceil(std::log2(x))));
}

// Checks the options and derives the bounds of the scales from how far the singular values can grow.
int scalars(const char* what, const egnn_ns_options& o, NsScalars& q) {
  if (o.steps < 0 || o.steps > kNsMaxSteps) return fail(EGNN_ERR_INVALID_ARG, "%s: steps must be 0 .. %d", what, kNsMaxSteps);
  if (!(o.eps >= 0.0) || !std::isfinite(o.eps)) return fail(EGNN_ERR_INVALID_ARG, "%s: eps must not be negative", what);
  if (!std::isfinite(o.a) || !std::isfinite(o.b) || !std::isfinite(o.c))
    return fail(EGNN_ERR_INVALID_ARG, "%s: coefficients must be finite", what);
  q = NsScalars{};
  // A scale follows the largest value that the bound allows, while small ones go with |a| in a
  // step.  Entries near 2^-12 of the bound (1 / sqrt(m n) at the largest sides) keep their 22 bits
  // down to another 2^-4; behind that the error grows past float32's
  // (14 times at 2^-5: 1024 x 4096, coefficients 0.141, -4.726, 0.285).
  double r = 1.0, small = 1.0;
  for (int k = 0; k < o.steps; ++k) {
    q.growth[k] = (int8_t)exponent_above(even_poly_max(o, r));
    r = odd_poly_max(o, r);
    if (!(r < 1024.0))
      return fail(EGNN_ERR_INVALID_ARG, "%s: these coefficients let the singular values grow past 1024", what);
    q.bound[k + 1] = (int8_t)exponent_above(r);
    small *= std::fabs(o.a);
    if (k + 1 < o.steps && r > 16.0 * small)
      return fail(EGNN_ERR_INVALID_ARG, "%s: these coefficients let small singular values fall too far behind the largest", what);
  }
  q.a_exp = exponent_above(std::fabs(o.a));
  q.b_exp = exponent_above(std::fabs(o.b));
  q.c_exp = exponent_above(std::fabs(o.c));
  q.a = (float)o.a;
  q.b = (float)o.b;
  q.c = (float)o.c;
  q.eps = o.eps;
  q.steps = o.steps;
  // the debugging aid of the edge kernels' waits (read at every call): 0 makes the readers give up at once
  const char* polls = std::getenv("EGNN_DEBUG_WAIT_POLLS");
  const long limit = polls && *polls ? std::strtol(polls, nullptr, 10) : -1;
  q.wait_polls = limit < 0 ? 1 << 22 : (int)std::min<long>(limit, 1L << 22);
  return EGNN_OK;
}

bool size_built(int rows, int cols) {
  return rows >= 0 && cols >= 0 && rows <= kMaxSide && cols <= kMaxSide && std::min(rows, cols) <= kMaxSmall;
}

bool is_large(int rows, int cols) { return !ns_fused_fits(std::min(rows, cols), std::max(rows, cols)); }

// Workspace of the matrices that a block's shared memory does not hold: that of the
// batch of them which needs most, since batches run one after another.
struct Need {
  Carver c{nullptr};
  size_t most;
  int64_t large = 0;
  Need() {
    c.take<float>(1);
    most = c.size();
  }
  void add(int rows, int cols) {
    if (!rows || !cols || !is_large(rows, cols)) return;
    if (large++ % kNsLarge == 0) c.off = 0;
    ns_grid_carve(c, rows, cols);
    most = std::max(most, c.size());
  }
};

// The matrices that fit a block's shared memory in batches of one launch, the
// large ones in batches of their own.  Everything is checked before the first
// launch.
template <class Fill>
int run_all(const char* what, int64_t count, const Fill& fill, const NsScalars& q, void* ws, size_t ws_bytes,
            cudaStream_t s) {
  if (count == 0) return EGNN_OK;
  Need need;
  NsItem it;
  int64_t small_count = 0;
  for (int64_t i = 0; i < count; ++i) {
    EGNN_TRY(fill(i, it));
    need.add(it.rows, it.cols);
    small_count += it.rows && it.cols && !is_large(it.rows, it.cols);
  }
  if (!ws || ws_bytes < need.most) return fail(EGNN_ERR_WORKSPACE, "%s: workspace too small", what);
  if (reinterpret_cast<uintptr_t>(ws) & 255u)
    return fail(EGNN_ERR_INVALID_ARG, "%s: the workspace must start on a 256-byte boundary", what);
  const Carver c(ws);
  // A few small matrices among large ones (embeddings among wide layers) run beside
  // them, on SMs that the large ones leave: five of up to 128 x 31 with 200 x 333,
  // 64 x 1100 and 513 x 97 take 120 us, one kernel after the other 139; 18 of 128 x 257
  // with six H = 256 layers 190 and 241.
  struct Side {
    cudaStream_t main_s, stream;
    int status = EGNN_OK;
    bool on;
    Side(cudaStream_t s, bool want) : main_s(s), stream(s), on(want) {
      if (on) status = fork_side(main_s, &stream);
    }
    int join() {
      const bool was = on;
      on = false;
      return was ? join_side(main_s) : EGNN_OK;
    }
    ~Side() { join(); }   // also on an early return, so that no capture is left forked
  } side(s, need.large > 0 && small_count > 0 && small_count <= num_sms_current() / 8);
  EGNN_TRY(side.status);
  const int spare = side.on ? (int)small_count : 0;
  NsBatch small, large;
  small.count = large.count = 0;
  for (int64_t i = 0; i < count; ++i) {
    EGNN_TRY(fill(i, it));
    if (it.rows == 0 || it.cols == 0) continue;
    NsBatch& b = is_large(it.rows, it.cols) ? large : small;
    b.it[b.count] = it;
    if (++b.count == (&b == &large ? kNsLarge : kNsItems)) {
      EGNN_TRY(&b == &large ? ns_grid(b, c, q, spare, s) : ns_fused(b, q, side.stream));
      b.count = 0;
    }
  }
  if (small.count) EGNN_TRY(ns_fused(small, q, side.stream));
  if (large.count) EGNN_TRY(ns_grid(large, c, q, spare, s));
  return side.join();
}

}  // namespace
}  // namespace egnn

using namespace egnn;

extern "C" size_t egnn_orthogonalize_workspace_size(int64_t count, const int32_t* sizes) {
  if (count < 0 || (count > 0 && !sizes)) return 0;
  Need need;
  for (int64_t i = 0; i < count; ++i) {
    if (!size_built(sizes[2 * i], sizes[2 * i + 1])) return 0;
    need.add(sizes[2 * i], sizes[2 * i + 1]);
  }
  return need.most;
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
