// Shared between the Newton-Schulz kernels: descriptors of the matrices of a
// launch, the scalars of a call, element access.
#pragma once

#include <algorithm>
#include <type_traits>

#include <cuda_fp16.h>

#include "common.cuh"

namespace egnn {

// Matrices of one batch: as many as fill the device with one block each (10 KB of kernel
// parameters; 140 of 128 x 257 take 54 us, in batches of 64 158 us).
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

// X, A and B = b A + c A A are kept as fp16 pairs hi + lo (22 bits), scaled by
// powers of two of their own in every step, a factor 4 below fp16's largest value.
// With the singular values, hence the entries, of X up to 2^e: X by 2^(14 - e),
// A by 2^(14 - 2e), B by 2^(14 - eb) with 2^eb above |b| 2^2e + |c| 2^4e.  e starts
// from |G| / (|G| + eps) and goes by the polynomial's bounds; one bound of all
// steps would leave the early ones, or a gradient below eps, to fp16's smallest numbers
// (coefficients 6, -3, 0.3 in two steps of 1024 x 4096: error 8.4e-6, so 1.4e-7;
// |G| = 1e-14, eps = 1e-7: 2e-3, so 1.3e-7).
struct NsScalars {
  float a, b, c;
  double eps;
  int8_t bound[kNsMaxSteps + 1];   // before step k the singular values are below 2^bound[k]
  int8_t growth[kNsMaxSteps];      // and grow by at most 2^growth[k] in it
  int a_exp, b_exp, c_exp;         // |a| <= 2^a_exp, ...
  float mu, nu;                    // nu = 1 - mu
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

// Smaller singular values than 2^kNsLeast are held with fewer bits: 2^(14 - kNsLeast) is a
// float32, and |G| / (|G| + 1e-7) is above it for any float32 |G| above the smallest normal one.
constexpr int kNsLeast = -112, kNsMostExp = 64;
// 2^e; 0 below float32's range.
__device__ __forceinline__ float ns_pow2(int e) {
  return e < -149 ? 0.f : __int_as_float(e < -126 ? 1 << (e + 149) : (min(e, 127) + 127) << 23);
}
// The weights of a step whose X is below 2^e, of the scaled terms, and e for the next step.
struct NsStep {
  float b, cc;     // B = b A + cc (A A)
  float x, bx;     // X' = x X + bx (B X), scaled for the next step, or X' itself after the last
  __device__ NsStep() {}
  __device__ __forceinline__ NsStep(const NsScalars& q, int step, int& e) {
    const int eb = max(q.b_exp + 2 * e, q.c_exp + 4 * e) + 1;
    // the polynomial's factor of s: its most over the step's whole range, or at 2^e and below
    const int grown = e + min((int)q.growth[step], max(q.a_exp, eb - 1) + 2);
    // 2^14: X' itself, not scaled
    const int next = step + 1 < q.steps ? max(kNsLeast, min((int)q.bound[step + 1], grown)) : 14;
    b = q.b * ns_pow2(2 * e - eb);
    cc = q.c * ns_pow2(4 * e - eb - 14);
    x = q.a * ns_pow2(e - next);
    bx = ns_pow2(eb + e - next - 14);
    e = next;
  }
};
constexpr float kNsGram = 0x1p-14f;   // X X^T of scaled X -> scaled A, in every step

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
