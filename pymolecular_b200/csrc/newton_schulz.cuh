// Shared between the Newton-Schulz kernels: descriptors of the matrices of a
// launch, the scalars of a call, element access.
#pragma once

#include <algorithm>
#include <type_traits>

#include <cuda_fp16.h>

#include "common.cuh"

namespace egnn {

// Matrices of one batch: as many as fill the device with one block each (10 KB of kernel
// parameters; 140 of 128 x 257 take 60 us, in batches of 64 166 us).
constexpr int kNsItems = 160;
constexpr int kNsLarge = 64;   // matrices of a batch that go through the workspace, which batches share
constexpr int kNsMaxSteps = 64;

struct NsItem {
  const void* in;        // the matrix, or the gradient (float32) of a step
  void* out;             // its orthogonalised form, or the weight of a step
  float* mom;            // momentum of a step; NULL: no step
  int64_t ld_in, ld_out, ld_mom;
  int rows, cols, dtype;
  float gain;
};

struct NsBatch {
  NsItem it[kNsItems];
  int count;
};

// X, A and B = b A + c A A are kept as fp16 pairs hi + lo (22 bits) scaled by
// powers of two, chosen so that their largest entries stay near 2^14: the
// iteration bounds the singular values, hence every entry, beforehand.
struct NsScalars {
  float a, b, c;
  double eps;
  float sx, sa, sb;         // scales of X, A and b A + c A A
  float mu, nu;             // nu = 1 - mu
  double decay, lr;
  const float* lr_device;
  int nesterov;
  int steps;
  int wait_polls;           // limit of the accumulator readers' waits
};

__device__ __forceinline__ float ns_float(float v) { return v; }
__device__ __forceinline__ float ns_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float ns_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T ns_from(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// M <- mu M + nu G, and U = mu M + nu G (Nesterov) or M from the moved M.
__device__ __forceinline__ float ns_momentum(const NsScalars& q, float g, float m) { return fmaf(q.mu, m, q.nu * g); }
__device__ __forceinline__ float ns_update(const NsScalars& q, float g, float m) {
  return q.nesterov ? fmaf(q.mu, m, q.nu * g) : m;
}

// Factors of W <- keep W + move O.
__device__ __forceinline__ void ns_rates(const NsItem& it, const NsScalars& q, float& keep, float& move) {
  const double lr = q.lr_device ? (double)*q.lr_device : q.lr;
  keep = (float)(1.0 - lr * q.decay);
  move = (float)(-lr * it.gain);
}

// A sum in tensor memory is rounded towards zero at each of its L instructions.
// On average one loses half a unit in the last place of the sum so far, which
// is 2^-23 / (4 ln 2) of it, and sums so far average (L + 1) / 2L of the whole:
// the mean loss, relative to the sum, that the readers add back.  What is left
// is its scatter.
__host__ __device__ inline float ns_mean_loss(int instructions) {
  return 0x1p-23f * 0.3607f * 0.5f * (float)(instructions + 1);
}

// Whether one block's shared memory holds the whole iteration of an m x n
// matrix (m <= n).
bool ns_fused_fits(int m, int n);
// The matrices of the batch, one block each.
int ns_fused(const NsBatch& b, const NsScalars& q, cudaStream_t s);
// The matrices of the batch on the whole device but `spare` SMs, with workspace
// from `c`; ns_grid_carve takes what one matrix needs.
int ns_grid(const NsBatch& b, Carver c, const NsScalars& q, int spare, cudaStream_t s);
void ns_grid_carve(Carver& c, int rows, int cols);
// Waits that ran out since the last call.
int ns_fused_take_timeouts();
int ns_grid_take_timeouts();

}  // namespace egnn
