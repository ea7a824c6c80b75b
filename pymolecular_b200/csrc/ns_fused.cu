// Newton-Schulz iteration of one matrix in one block, on the tensor cores.
//
//   A = X X^T,  B = b A + c A A,  X <- a X + B X      (X m x n, m <= n)
//
// Every product takes float32-like operands as pairs of fp16 tiles, v = hi + lo
// with hi = fp16(v), lo = fp16(v - hi): 22 bits, against float32's 24.  The
// three products lo hi, hi lo, hi hi accumulate in that order into one float32
// accumulator in tensor memory, so that the small terms go in while the sum is
// small; lo lo (2^-22 of the result) is left out.  Measured error against
// float64 at 128 x 257: see the table of the design notes; float32 products
// give the same.
//
// X (hi, lo) and A, then B, (hi, lo) stay in shared memory through all steps:
// global memory sees the matrix once on the way in and once on the way out.
// The same X tile is the K-major operand of X X^T and the MN-major operand of
// B X.  A block's shared memory bounds n: 7 column blocks of 64 for m > 64, 13
// for m > 32, 27 below.
#include <atomic>

#include "newton_schulz.cuh"
#include "tc.cuh"

namespace egnn {

__device__ int g_ns_fused_timeouts = 0;

namespace {

using namespace tc;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kSlots = 4, kSlotCols = 128;   // X' accumulators in tensor memory
constexpr int kSmemMax = 232448 - 1024;      // a block's shared memory less the static part

// Rows of a tile: all column blocks are `rows` x 128 bytes.
__host__ __device__ inline int tile_rows(int m) { return m <= 32 ? 32 : m <= 64 ? 64 : 128; }

// X hi + lo, A hi + lo, what a 128-row operand read runs past the last block,
// and the alignment of the first tile.
__host__ __device__ inline size_t smem_bytes(int m, int n) {
  const int R = tile_rows(m);
  return (size_t)((n + 63) / 64 + (m + 63) / 64) * R * 256 + (128 - R) * 128 + 1024;
}

// hi and lo tiles at (row, c0 .. c0 + 31) <- v.
__device__ __forceinline__ void store_pairs32(char* hi, char* lo, int R, int row, int c0, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = v[8 * j + 2 * k], y = v[8 * j + 2 * k + 1];
      const __half2 p = __floats2half2_rn(x, y);
      const float2 f = __half22float2(p);
      const __half2 r = __floats2half2_rn(x - f.x, y - f.y);
      h[k] = *reinterpret_cast<const uint32_t*>(&p);
      l[k] = *reinterpret_cast<const uint32_t*>(&r);
    }
    const uint32_t at = sw128_offset(row, c0 + 8 * j, R);
    *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

__device__ __forceinline__ void load_pairs32(const char* hi, const char* lo, int R, int row, int c0, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t at = sw128_offset(row, c0 + 8 * j, R);
    const uint4 h = *reinterpret_cast<const uint4*>(hi + at), l = *reinterpret_cast<const uint4*>(lo + at);
    const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&hh[k]));
      const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&ll[k]));
      v[8 * j + 2 * k] = p.x + r.x;
      v[8 * j + 2 * k + 1] = p.y + r.y;
    }
  }
}

__device__ __forceinline__ uint64_t desc_k(const char* tile, int R, int kk) {
  return make_desc(smem_u32(tile) + (kk >> 2) * R * 128 + (kk & 3) * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t desc_mn(const char* tile, int R, int c0, int kk) {
  return make_desc(smem_u32(tile) + (c0 >> 6) * R * 128 + kk * 2048, R * 128, 1024);
}

constexpr int kBatch = 8;

// The elements tid, tid + kThreads, ... of a matrix, kBatch at a time.
struct Walk {
  int r[kBatch];
  int c[kBatch];
  int rows, cols, dr, dc;
  __device__ __forceinline__ Walk(const NsItem& it, int tid)
      : rows(it.rows), cols(it.cols), dr(kThreads / it.cols), dc(kThreads % it.cols) {
    r[0] = tid / it.cols;
    c[0] = tid % it.cols;
    spread();
  }
  __device__ __forceinline__ void step(int to, int from) {
    r[to] = r[from] + dr;
    c[to] = c[from] + dc;
    if (c[to] >= cols) {
      c[to] -= cols;
      ++r[to];
    }
  }
  __device__ __forceinline__ void spread() {
#pragma unroll
    for (int k = 1; k < kBatch; ++k) step(k, k - 1);
  }
  __device__ __forceinline__ bool any() const { return r[0] < rows; }
  __device__ __forceinline__ bool has(int k) const { return r[k] < rows; }
  __device__ __forceinline__ void next() {
    step(0, kBatch - 1);
    spread();
  }
};

// Thread-uniform wait for the commit on `bar`; false when it ran out.
__device__ __forceinline__ bool wait_commit(uint64_t* bar, uint32_t parity) {
  const bool ok = mbar_wait(bar, parity);
  const bool bad = __syncthreads_or(!ok);
  fence_after_sync();
  return !bad;
}
// Tile writes and accumulator reads done by every thread -> the next products may go.
__device__ __forceinline__ void hand_over() {
  fence_proxy_async();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
}

__global__ void __launch_bounds__(kThreads, 1) ns_fused_kernel(const __grid_constant__ NsBatch batch,
                                                               const __grid_constant__ NsScalars q) {
  extern __shared__ char raw[];
  __shared__ uint64_t bar[kSlots];
  __shared__ uint32_t tmem_s;
  __shared__ double red[kWarps];
  const NsItem& it = batch.it[blockIdx.x];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool turn = it.rows > it.cols;
  const int m = turn ? it.cols : it.rows, n = turn ? it.rows : it.cols;
  const int R = tile_rows(m);
  const int m16 = (m + 15) & ~15, n16 = (n + 15) & ~15;
  const int xt = (n + 63) / 64 * R * 128, at = (m + 63) / 64 * R * 128;
  char* const Xh = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  char* const Xl = Xh + xt;
  char* const Ah = Xl + xt;
  char* const Al = Ah + at;

  // padding rows and columns of X are zeros, and every product keeps them so
  for (int i = tid; i < 2 * xt / 16; i += kThreads) reinterpret_cast<uint4*>(Xh)[i] = make_uint4(0, 0, 0, 0);
  if (warp == 0) tmem_alloc(&tmem_s, 512);
  if (tid == 0) {
    for (int k = 0; k < kSlots; ++k) mbar_init(&bar[k], 1);
    fence_mbar_init();
  }
  pdl_enter();

  // ---- U, its norm (squares added in float64: no overflow or underflow at any
  // scale of the gradient), X0.  Element i is thread i % kThreads's in both
  // passes; kBatch elements are loaded before any of them is used.
  Walk walk(it, tid);
  double ss = 0.0;
  for (; walk.any(); walk.next()) {
    float g[kBatch], mo[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      g[k] = walk.has(k) ? ns_load(it.in, it.dtype, walk.r[k] * it.ld_in + walk.c[k]) : 0.f;
      mo[k] = it.mom && walk.has(k) ? it.mom[walk.r[k] * it.ld_mom + walk.c[k]] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      float u = g[k];
      if (it.mom && walk.has(k)) {
        const float mv = ns_momentum(q, g[k], mo[k]);
        it.mom[walk.r[k] * it.ld_mom + walk.c[k]] = mv;
        u = ns_update(q, g[k], mv);
      }
      ss += (double)u * u;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
  if (lane == 0) red[warp] = ss;
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_s;
  ss = 0.0;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) ss += red[k];
  const double inv = 1.0 / (sqrt(ss) + q.eps);
  for (walk = Walk(it, tid); walk.any(); walk.next()) {
    float u[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      u[k] = walk.has(k) ? ns_load(it.in, it.dtype, walk.r[k] * it.ld_in + walk.c[k]) : 0.f;
      if (it.mom && walk.has(k)) u[k] = ns_update(q, u[k], it.mom[walk.r[k] * it.ld_mom + walk.c[k]]);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (!walk.has(k)) continue;
      const float v = (float)(u[k] * inv) * q.sx;
      const uint32_t o = turn ? sw128_offset(walk.c[k], walk.r[k], R) : sw128_offset(walk.r[k], walk.c[k], R);
      const __half h = __float2half_rn(v);
      *reinterpret_cast<__half*>(Xh + o) = h;
      *reinterpret_cast<__half*>(Xl + o) = __float2half_rn(v - __half2float(h));
    }
  }
  hand_over();

  // warp w reads accumulator lanes 32 (w % 4) .. + 31 = tile rows, and of each
  // group of four 32-column pieces the (w / 4)-th
  const int row = (warp & 3) * 32 + lane, piece = warp >> 2;
  const bool rows_here = (warp & 3) * 32 < R;
  const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  const uint32_t tA = 0, tAA = 128;
  const uint32_t idesc_m = make_idesc_f16(128, m16, 0, 0);
  const float fA = q.sa / (q.sx * q.sx);                    // accumulator -> A scaled
  const float fbA = q.b * q.sb / (q.sx * q.sx), fcAA = q.c * q.sb / (q.sa * q.sa);
  const float fX = 1.f / q.sb;
  const int n_slots = (n16 + kSlotCols - 1) / kSlotCols;
  uint32_t phase = 0, pending = 0;   // bit k: parity of bar[k]; a commit on it not yet waited for
  bool ok = true;

  // X' columns [128 k, 128 k + 128) into slot k % kSlots
  auto issue_update = [&](int k) {
    pending |= 1u << (k % kSlots);
    if (tid != 0) return;
    const int c0 = k * kSlotCols, N = min(kSlotCols, n16 - c0);
    const uint32_t d = tmem + (k % kSlots) * kSlotCols;
    const uint32_t idesc = make_idesc_f16(128, N, 0, 1);
    for (int p = 0; p < 3; ++p) {
      const char* L = p == 0 ? Al : Ah;
      const char* X = p == 1 ? Xl : Xh;
      for (int kk = 0; kk < m16 / 16; ++kk)
        mma_f16(d, desc_k(L, R, kk), desc_mn(X, R, c0, kk), idesc, (p | kk) ? 1u : 0u);
    }
    mma_commit(&bar[k % kSlots]);
  };
  auto wait_slot = [&](int k) {
    const bool good = wait_commit(&bar[k], (phase >> k) & 1u);
    if (good) {
      phase ^= 1u << k;
      pending &= ~(1u << k);
    }
    return good;
  };

#pragma unroll 1
  for (int step = 0; step < q.steps && ok; ++step) {
    if (tid == 0) {
      for (int p = 0; p < 3; ++p) {
        const char* L = p == 0 ? Xl : Xh;
        const char* Rr = p == 1 ? Xl : Xh;
        for (int kk = 0; kk < n16 / 16; ++kk)
          mma_f16(tmem + tA, desc_k(L, R, kk), desc_k(Rr, R, kk), idesc_m, (p | kk) ? 1u : 0u);
      }
      mma_commit(&bar[0]);
    }
    pending |= 1u;
    if (!(ok = wait_slot(0))) break;
    if (rows_here && piece * 32 < m16) {
      float v[32];
      tmem_ld32(tl + tA + piece * 32, v);
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] *= fA;
      store_pairs32(Ah, Al, R, row, piece * 32, v);
    }
    hand_over();
    if (tid == 0) {
      for (int p = 0; p < 3; ++p) {
        const char* L = p == 0 ? Al : Ah;
        const char* Rr = p == 1 ? Al : Ah;
        for (int kk = 0; kk < m16 / 16; ++kk)
          mma_f16(tmem + tAA, desc_k(L, R, kk), desc_k(Rr, R, kk), idesc_m, (p | kk) ? 1u : 0u);
      }
      mma_commit(&bar[0]);
    }
    pending |= 1u;
    if (!(ok = wait_slot(0))) break;
    if (rows_here && piece * 32 < m16) {
      float v[32], w[32];
      tmem_ld32(tl + tA + piece * 32, v);
      tmem_ld32(tl + tAA + piece * 32, w);
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = fmaf(fbA, v[k], fcAA * w[k]);
      store_pairs32(Ah, Al, R, row, piece * 32, v);
    }
    hand_over();
    for (int k = 0; k < min(n_slots, kSlots); ++k) issue_update(k);
    for (int k = 0; k < n_slots; ++k) {
      if (!(ok = wait_slot(k % kSlots))) break;
      const int c0 = k * kSlotCols + piece * 32;
      if (rows_here && c0 < n16) {
        float v[32], x[32];
        tmem_ld32(tl + (k % kSlots) * kSlotCols + piece * 32, v);
        load_pairs32(Xh, Xl, R, row, c0, x);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = fmaf(q.a, x[j], fX * v[j]);
        store_pairs32(Xh, Xl, R, row, c0, v);
      }
      if (k + kSlots < n_slots) {   // the slot is free once every thread has read it
        fence_before_sync();
        __syncthreads();
        fence_after_sync();
        issue_update(k + kSlots);
      }
    }
    hand_over();
  }

  if (!ok) {
    if (tid == 0) {   // what is still in flight ends before the tensor memory goes
      atomicAdd(&g_ns_fused_timeouts, 1);
      for (int k = 0; k < kSlots; ++k)
        if (pending >> k & 1u) mbar_wait(&bar[k], (phase >> k) & 1u);
    }
  } else {
    const float back = 1.f / q.sx;
    float keep = 0.f, move = 0.f;
    if (it.mom) ns_rates(it, q, keep, move);
    for (walk = Walk(it, tid); walk.any(); walk.next()) {
      float w[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        w[k] = it.mom && walk.has(k) ? static_cast<const float*>(it.out)[walk.r[k] * it.ld_out + walk.c[k]] : 0.f;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (!walk.has(k)) continue;
        const uint32_t o = turn ? sw128_offset(walk.c[k], walk.r[k], R) : sw128_offset(walk.r[k], walk.c[k], R);
        const float v = (__half2float(*reinterpret_cast<const __half*>(Xh + o)) +
                         __half2float(*reinterpret_cast<const __half*>(Xl + o))) * back;
        const int64_t io = walk.r[k] * it.ld_out + walk.c[k];
        if (it.mom) static_cast<float*>(it.out)[io] = fmaf(move, v, keep * w[k]);
        else ns_store(it.out, it.dtype, io, v);
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

}  // namespace

bool ns_fused_fits(int m, int n) { return m <= 128 && smem_bytes(m, n) <= (size_t)kSmemMax; }

int ns_fused(const NsBatch& b, const NsScalars& q, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  const uint64_t bit = device_bit();
  if (!(ready.load() & bit)) {
    EGNN_CHECK_CUDA(cudaFuncSetAttribute(ns_fused_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax));
    ready.fetch_or(bit);
  }
  size_t smem = 0;
  for (int i = 0; i < b.count; ++i)
    smem = std::max(smem, smem_bytes(std::min(b.it[i].rows, b.it[i].cols), std::max(b.it[i].rows, b.it[i].cols)));
  TimerScope ts("newton_schulz", s);
  EGNN_CHECK_CUDA(launch_pdl(ns_fused_kernel, dim3(b.count), dim3(kThreads), smem, s, b, q));
  EGNN_CHECK_LAUNCH();
  return EGNN_OK;
}

int ns_fused_take_timeouts() {
  int n = 0;
  if (cudaMemcpyFromSymbol(&n, g_ns_fused_timeouts, sizeof(int)) != cudaSuccess) return 0;
  if (n) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_ns_fused_timeouts, &zero, sizeof(int));
  }
  return n;
}

}  // namespace egnn
