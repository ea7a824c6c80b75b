// Newton-Schulz iteration of one matrix in one block, on the tensor cores.
//
//   A = X X^T,  B = b A + c A A,  X <- a X + B X      (X m x n, m <= n)
//
// Every product takes float32-like operands as pairs of fp16 tiles, v = hi + lo
// with hi = fp16(v), lo = fp16(v - hi): 22 bits, against float32's 24.  lo lo
// (2^-22 of the result) is left out.  Sums in tensor memory are rounded towards
// zero at every instruction, by the size of the sum so far: lo hi + hi lo goes
// into an accumulator of its own, or in before hi hi, so that only one
// instruction per 16 terms costs a rounding of the full sum.  The hi hi terms of
// X X^T are one sum up to n = 384 and three beyond, those of the other products one.
//
// X (hi, lo) and A, then B, (hi, lo) stay in shared memory through all steps:
// global memory sees the matrix once on the way in and once on the way out.
// The same X tile is the K-major operand of X X^T and the MN-major operand of
// B X.  Shared memory bounds the blocks of 64 columns of X and A to 7 for m > 64
// and 13 for m > 32, tensor memory n to 1024.
//
// What bounds it: a chain of three dependent products a step, on one SM.  A step of
// 128 x 257 takes 14,000 cycles, its products alone 8,300 (three half-precision
// products each), the rest are accumulators on their way through the registers.
// 5 steps of one 64 x 129 take 30 us, of one 128 x 257 and of 35 of them 53 us, against
// 77, 99 and 134 us in the kernel for large matrices, which takes 102 us for 128 x 321.  A matrix on a cluster of two blocks was slower (65 us for the 35, then 55 without): 64 KB
// through distributed shared memory cost 9,000 cycles a step.
#include <atomic>

#include "ns_tiles.cuh"

namespace egnn {

__device__ int g_ns_fused_timeouts = 0;

namespace {

using namespace tc;
using namespace ns;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kSlots = 3, kSlotCols = 128;   // X' accumulators in tensor memory; B comes after them
constexpr int kMaxChunks = 8;                // of 128 columns of X
constexpr int kSmemMax = 232448 - 1024;      // a block's shared memory less the static part

// Rows of a tile: all column blocks are `rows` x 128 bytes.
__host__ __device__ inline int tile_rows(int m) { return m <= 32 ? 32 : m <= 64 ? 64 : 128; }

// X hi + lo, A hi + lo, what a 128-row operand read runs past the last block,
// and the alignment of the first tile.
__host__ __device__ inline size_t smem_bytes(int m, int n) {
  const int R = tile_rows(m);
  return (size_t)((n + 63) / 64 + (m + 63) / 64) * R * 256 + (128 - R) * 128 + 1024;
}

// Issues D (+)= L R over the K-steps h, h + 2, h + 4, h + 6 (those below nk) of
// 128 columns of L, both K-major from their descriptors; blk16 is a column
// block in descriptor units.
__device__ __forceinline__ void issue(uint32_t one, uint32_t d, uint64_t l, uint64_t r, uint32_t blk16, int h, int nk,
                                      uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int p = 0; p < 4; ++p)
    if (2 * p + h < nk) {
      const uint32_t o = (p >> 1) * blk16 + (p & 1) * 4 + h * 2;
      mma_f16_elected(one, d, l + o, r + o, idesc, accumulate);
      accumulate = 1;
    }
}
// The same with L in tensor memory and R MN-major.
__device__ __forceinline__ void issue_mn(uint32_t one, uint32_t d, uint32_t l, uint64_t r, int h, int nk, uint32_t idesc,
                                         uint32_t accumulate) {
#pragma unroll
  for (int p = 0; p < 4; ++p)
    if (2 * p + h < nk) {
      mma_f16_ts_elected(one, d, l + (2 * p + h) * 8, r + (2 * p + h) * 128, idesc, accumulate);
      accumulate = 1;
    }
}

// The units of a matrix two at a time, the next two's loads in flight while
// two are worked on: load(unit, slot) and work(unit, slot).
template <class Load, class Work>
__device__ __forceinline__ void units(int rows, int cols, const Load& load, const Work& work) {
  Unit u[2] = {Unit(cols, threadIdx.x >> 5, kWarps), Unit(cols, (threadIdx.x >> 5) + kWarps, kWarps)};
  if (u[0].r0 < rows) load(u[0], 0);
  if (u[1].r0 < rows) load(u[1], 1);
#pragma unroll 1
  while (u[0].r0 < rows) {
    Unit t[2] = {u[0], u[1]};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      t[i].id += kWarps;
      t[i].next();
      if (t[i].r0 < rows) load(t[i], 2 + i);
    }
    work(u[0], 0);
    if (u[1].r0 < rows) work(u[1], 1);
    u[0] = t[0];
    u[1] = t[1];
  }
}

// U into the tiles (raw); returns this thread's sum of squares, added in
// float64: no overflow or underflow at any scale of the gradient.
template <typename T, bool MOM>
__device__ __forceinline__ double take_in(const NsItem& it, const NsScalars& q, char* Xh, char* Xl, uint32_t blk,
                                          bool turn) {
  const int rows = it.rows, cols = it.cols;
  const T* const in = static_cast<const T*>(it.in);
  float* const mom = it.mom;
  const int64_t ld_in = it.ld_in, ld_mom = it.ld_mom;
  const float mu = q.mu, nu = q.nu;
  const bool nesterov = q.nesterov;
  double ss = 0.0;
  float g[4][8], m[4][8];
  units(
      rows, cols,
      [&](const Unit& u, int i) {
        unit_load(in, ld_in, u, rows, cols, g[i]);
        if (MOM) unit_load(mom, ld_mom, u, rows, cols, m[i]);
      },
      [&](const Unit& u, int i) {
        if (MOM) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            m[i][k] = fmaf(mu, m[i][k], nu * g[i][k]);
            g[i][k] = nesterov ? fmaf(mu, m[i][k], nu * g[i][k]) : m[i][k];
          }
          unit_store(mom, ld_mom, u, rows, cols, m[i]);
        }
        ss += squares(g[i]);
        // rows past the matrix get the zeros that are there already
        if (u.c < cols) unit_to_raw(Xh, Xl, blk, turn, u, g[i]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          g[i][k] = g[2 + i][k];
          if (MOM) m[i][k] = m[2 + i][k];
        }
      });
  return ss;
}

// The tiles (raw) to the result, or the weight moved by them.
template <typename T, bool MOM>
__device__ __forceinline__ void give_out(const NsItem& it, const NsScalars& q, const char* Xh, const char* Xl,
                                         uint32_t blk, bool turn) {
  const int rows = it.rows, cols = it.cols;
  T* const out = static_cast<T*>(it.out);
  const int64_t ld = it.ld_out;
  float keep = 0.f, move = 0.f;
  if (MOM) ns_rates(it, q, keep, move);
  float w[4][8];
  units(
      rows, cols,
      [&](const Unit& u, int i) {
        if (MOM) unit_load(out, ld, u, rows, cols, w[i]);
      },
      [&](const Unit& u, int i) {
        if (u.c < cols) {
          float v[8];
          unit_from_raw(Xh, Xl, blk, turn, u, v);
          if (MOM)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = fmaf(move, v[k], keep * w[i][k]);
          unit_store(out, ld, u, rows, cols, v);
        }
        if (MOM)
#pragma unroll
          for (int k = 0; k < 8; ++k) w[i][k] = w[2 + i][k];
      });
}

struct Barriers {
  uint64_t a_done, aa_done;              // commits of X X^T and A A
  uint64_t slot_done[kSlots];            // commits of X' columns
  uint64_t a_ready[2], b_ready[2];       // halves of the A and B tiles are written
  uint64_t x_ready[kMaxChunks][2];       // halves of each 128 columns of X
  uint64_t drained;
};

// This warp's tile writes and accumulator reads are done.
__device__ __forceinline__ void arrive(uint64_t* bar) {
  fence_proxy_async();
  fence_before_sync();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Warps 0 .. 15 take the matrix in, turn accumulators into operand tiles and
// give the result out; warp 16 issues the products.  Operands are handed over
// in halves (even and odd K-steps), so that products run while the second
// half is still being written, and X X^T of the next step runs while the last
// columns of X' are.
__global__ void __launch_bounds__(kThreads + 32, 1) ns_fused_kernel(const __grid_constant__ NsBatch batch,
                                                                    const __grid_constant__ NsScalars q) {
  extern __shared__ char raw[];
  __shared__ Barriers bar;
  __shared__ uint32_t tmem_s;
  __shared__ int gave_up_s;
  __shared__ double red[kWarps];
  const NsItem& it = batch.it[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // known to be uniform
  const bool turn = it.rows > it.cols;
  const int m = turn ? it.cols : it.rows, n = turn ? it.rows : it.cols;
  const int R = tile_rows(m);
  const int m16 = (m + 15) & ~15, n16 = (n + 15) & ~15;
  const int xt = (n + 63) / 64 * R * 128, at = (m + 63) / 64 * R * 128;
  char* const Xh = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  char* const Xl = Xh + xt;
  char* const Ah = Xl + xt;
  char* const Al = Ah + at;
  volatile int* const gave_up = &gave_up_s;
  const int chunks = (n16 + kSlotCols - 1) / kSlotCols;

  // padding rows and columns of X are zeros, and every product keeps them so
  for (int i = tid; i < 2 * xt / 16; i += kThreads + 32) reinterpret_cast<uint4*>(Xh)[i] = make_uint4(0, 0, 0, 0);
  if (warp == kWarps) {
    tmem_alloc(&tmem_s, 512);
    if (lane == 0) {
      gave_up_s = 0;
      mbar_init(&bar.a_done, 1);
      mbar_init(&bar.aa_done, 1);
      mbar_init(&bar.drained, 1);
      for (int k = 0; k < kSlots; ++k) mbar_init(&bar.slot_done[k], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bar.a_ready[h], kWarps);
        mbar_init(&bar.b_ready[h], kWarps);
        for (int k = 0; k < chunks; ++k) mbar_init(&bar.x_ready[k][h], kWarps);
      }
      fence_mbar_init();
    }
  }
  pdl_enter();
  __syncthreads();
  if (warp < kWarps) {
    double ss = it.mom                            ? take_in<float, true>(it, q, Xh, Xl, R * 128, turn)
                : it.dtype == EGNN_DTYPE_F32  ? take_in<float, false>(it, q, Xh, Xl, R * 128, turn)
                : it.dtype == EGNN_DTYPE_BF16 ? take_in<__nv_bfloat16, false>(it, q, Xh, Xl, R * 128, turn)
                                              : take_in<__half, false>(it, q, Xh, Xl, R * 128, turn);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    if (lane == 0) red[warp] = ss;
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_s;
  // The slots hold X' only after B is made, so A and A A, their small terms apart, go there.  Long sums
  // are spread over three accumulators.
  const int sums = chunks > kSlots ? kSlots : 1;
  const uint32_t tA = tmem, tAA = tmem + kSlotCols, tAAx = tmem + 2 * kSlotCols, tAx = tmem + 3 * kSlotCols;
  const uint32_t tB = tAx, tBl = tB + 64;   // hi and lo of B
  // which use of its slot X' columns k are in a step
  auto slot_use = [&](int step, int k) {
    const int slot = k % kSlots;
    return step * ((chunks - slot + kSlots - 1) / kSlots) + k / kSlots;
  };

  if (warp == kWarps) {
    const uint32_t one = elect_one();
    const uint32_t blk16 = R * 8;
    const uint32_t idesc_m = make_idesc_f16(128, m16, 0, 0);
    const int nk = n16 >> 4, mk = m16 >> 4;
    const uint64_t xh = make_desc(smem_u32(Xh), 16, 1024), xl = make_desc(smem_u32(Xl), 16, 1024);
    const uint64_t ah = make_desc(smem_u32(Ah), 16, 1024), al = make_desc(smem_u32(Al), 16, 1024);
    const uint64_t xh_mn = make_desc(smem_u32(Xh), R * 128, 1024), xl_mn = make_desc(smem_u32(Xl), R * 128, 1024);
    bool ok = true;
#pragma unroll 1
    for (int step = 0; step < q.steps && ok; ++step) {
      // slots used more than once: their last X' columns have to be read before A goes there
      for (int k = kSlots; k < chunks && ok; ++k)
        ok = wait_bar(&bar.x_ready[k][0], step, gave_up) && wait_bar(&bar.x_ready[k][1], step, gave_up);
      // B has been read by the last of the products
      if (step > 0 && ok) ok = wait_bar(&bar.slot_done[(chunks - 1) % kSlots], slot_use(step - 1, chunks - 1), gave_up);
#pragma unroll 1
      for (int k = 0; k < chunks && ok; ++k)
#pragma unroll 1
        for (int h = 0; h < 2 && ok; ++h) {
          if (!(ok = wait_bar(&bar.x_ready[k][h], step, gave_up))) break;
          const uint32_t o = 2 * k * blk16, d = tmem + (k % sums) * kSlotCols;
          issue(one, tAx, xl + o, xh + o, blk16, h, nk - 8 * k, idesc_m, k | h);
          issue(one, tAx, xh + o, xl + o, blk16, h, nk - 8 * k, idesc_m, 1);
          issue(one, d, xh + o, xh + o, blk16, h, nk - 8 * k, idesc_m, k >= sums || h);
        }
      if (!ok) break;
      if (one) mma_commit(&bar.a_done);
#pragma unroll 1
      for (int h = 0; h < 2 && ok; ++h) {
        if (!(ok = wait_bar(&bar.a_ready[h], step, gave_up))) break;
        issue(one, tAAx, al, ah, blk16, h, mk, idesc_m, h);
        issue(one, tAAx, ah, al, blk16, h, mk, idesc_m, 1);
        issue(one, tAA, ah, ah, blk16, h, mk, idesc_m, h);
      }
      if (!ok) break;
      if (one) mma_commit(&bar.aa_done);
      // X' columns [128 k, 128 k + 128) into slot k % kSlots
      if (!(ok = wait_bar(&bar.b_ready[0], step, gave_up))) break;
#pragma unroll 1
      for (int k0 = 0; k0 < chunks && ok; k0 += kSlots) {
        const int k1 = min(chunks, k0 + kSlots);
#pragma unroll 1
        for (int h = 0; h < 2 && ok; ++h) {
          if (h == 1 && k0 == 0 && !(ok = wait_bar(&bar.b_ready[1], step, gave_up))) break;
#pragma unroll 1
          for (int k = k0; k < k1 && ok; ++k) {
            // a slot that was used in this step is free once X' has been read out of it
            if (h == 0 && k >= kSlots &&
                !(ok = wait_bar(&bar.x_ready[k - kSlots][0], step + 1, gave_up) &&
                       wait_bar(&bar.x_ready[k - kSlots][1], step + 1, gave_up)))
              break;
            const uint32_t o = 2 * k * blk16, d = tmem + (k - k0) * kSlotCols;
            const uint32_t idesc = make_idesc_f16(128, min(kSlotCols, n16 - k * kSlotCols), 0, 1);
            issue_mn(one, d, tBl, xh_mn + o, h, mk, idesc, h);
            issue_mn(one, d, tB, xl_mn + o, h, mk, idesc, 1);
            if (h == 1) {
              issue_mn(one, d, tB, xh_mn + o, 0, mk, idesc, 1);
              issue_mn(one, d, tB, xh_mn + o, 1, mk, idesc, 1);
              if (one) mma_commit(&bar.slot_done[k - k0]);
            }
          }
        }
      }
    }
    // nothing may be in flight when the tensor memory goes
    if (one) mma_commit(&bar.drained);
    wait_bar(&bar.drained, 0, gave_up);
  } else {
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) ss += red[k];
    float pre, f;
    int e;   // X is below 2^e
    norm_scale(ss, q.eps, pre, f, e);
    const float sx = ns_pow2(14 - e);
    // warp w owns tile rows 32 (w % 4) .. + 31, which are its accumulator lanes,
    // and of each group of four 32-column pieces the (w / 4)-th
    const int row = (warp & 3) * 32 + lane, piece = warp >> 2;
    const bool rows_here = (warp & 3) * 32 < R;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    // this thread's pieces of X (128 columns apart) and of A
    const uint32_t xh = row_at(smem_u32(Xh), R, row, piece * 32), ah = row_at(smem_u32(Ah), R, row, piece * 32);
    for (int k = 0; k < chunks; ++k) {
      const int c0 = k * kSlotCols + piece * 32;
      const uint32_t hi = xh + k * (2 * R * 128), lo = hi + xt;
      float v[32];
      if (rows_here && c0 < n16) {
        load_raw32(hi, lo, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = v[j] * pre * f;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (rows_here && c0 < n16) {
          if (q.steps == 0) {
            store_raw16(hi, lo, h, v + 16 * h);
          } else {
#pragma unroll
            for (int j = 16 * h; j < 16 * h + 16; ++j) v[j] *= sx;
            store_pairs16(hi, lo, h, v + 16 * h);
          }
        }
        arrive(&bar.x_ready[k][h]);
      }
    }

    const float loss_n = ns_mean_loss((n16 >> 4) / sums), loss_m = ns_mean_loss(m16 >> 4);
    const bool a_here = rows_here && piece * 32 < m16;
    bool ok = true;
#pragma unroll 1
    for (int step = 0; step < q.steps && ok; ++step) {
      const NsStep w(q, step, e);
      // What does not wait for a product is fetched before the wait.  An accumulator is read
      // to its end before the first half is handed over, where the products of that half
      // write to its place.
      float v[32];   // A, then B, then X
      auto read_a = [&](int h) {
        float t[16], x[16];
        const uint32_t c = lanes + piece * 32 + 16 * h;
        tmem_ld16x2(tA + c, tAx + c, t, x);
        for (int j = 1; j < sums; ++j) {
          float u[16];
          tmem_ld16(tmem + j * kSlotCols + c, u);
#pragma unroll
          for (int k = 0; k < 16; ++k) t[k] += u[k];
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) v[16 * h + k] = (fmaf(t[k], loss_n, t[k]) + x[k]) * kNsGram;
      };
      if (!(ok = wait_bar(&bar.a_done, step, gave_up, q.wait_polls))) break;
      if (a_here) {
        read_a(0);
        if (sums > 1) read_a(1);   // A A goes where the sums are
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (a_here) {
          if (h == 1 && sums == 1) read_a(1);
          store_pairs16(ah, ah + at, h, v + 16 * h);
        }
        arrive(&bar.a_ready[h]);
      }
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] *= w.b;
      if (!(ok = wait_bar(&bar.aa_done, step, gave_up))) break;
      if (a_here) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float t[16], x[16];
          const uint32_t c = lanes + piece * 32 + 16 * h;
          tmem_ld16x2(tAA + c, tAAx + c, t, x);
#pragma unroll
          for (int k = 0; k < 16; ++k)
            v[16 * h + k] = fmaf(w.cc, x[k], fmaf(w.cc, fmaf(t[k], loss_m, t[k]), v[16 * h + k]));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (a_here) {
          uint32_t hw[8], lw[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) split2(v[16 * h + 2 * k], v[16 * h + 2 * k + 1], hw[k], lw[k]);
          tmem_st8u(tB + lanes + piece * 16 + 8 * h, hw);
          tmem_st8u(tBl + lanes + piece * 16 + 8 * h, lw);
        }
        arrive(&bar.b_ready[h]);
      }
#pragma unroll 1
      for (int k = 0; k < chunks; ++k) {
        const int slot = k % kSlots;
        const int c0 = k * kSlotCols + piece * 32;
        const bool here = rows_here && c0 < n16;
        const uint32_t hi = xh + k * (2 * R * 128), lo = hi + xt;
        if (here) {   // this thread's own
          load_pairs32(hi, lo, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= w.x;
        }
        if (!(ok = wait_bar(&bar.slot_done[slot], slot_use(step, k), gave_up))) break;
        if (here) {
          float t[16], u[16];
          const uint32_t c = tmem + lanes + slot * kSlotCols + piece * 32;
          tmem_ld16x2(c, c + 16, t, u);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            v[j] = fmaf(w.bx, fmaf(t[j], loss_m, t[j]), v[j]);
            v[16 + j] = fmaf(w.bx, fmaf(u[j], loss_m, u[j]), v[16 + j]);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (here) {
            if (step + 1 < q.steps) store_pairs16(hi, lo, h, v + 16 * h);
            else store_raw16(hi, lo, h, v + 16 * h);
          }
          arrive(&bar.x_ready[k][h]);
        }
      }
    }
  }

  fence_before_sync();
  __syncthreads();
  if (warp == kWarps) {
    if (lane == 0 && *gave_up) atomicAdd(&g_ns_fused_timeouts, 1);
    tmem_dealloc(tmem, 512);
  } else if (!*gave_up) {
    if (it.mom) give_out<float, true>(it, q, Xh, Xl, R * 128, turn);
    else if (it.dtype == EGNN_DTYPE_F32) give_out<float, false>(it, q, Xh, Xl, R * 128, turn);
    else if (it.dtype == EGNN_DTYPE_BF16) give_out<__nv_bfloat16, false>(it, q, Xh, Xl, R * 128, turn);
    else give_out<__half, false>(it, q, Xh, Xl, R * 128, turn);
  }
}

}  // namespace

bool ns_fused_fits(int m, int n) { return m <= 128 && n <= kMaxChunks * kSlotCols && smem_bytes(m, n) <= (size_t)kSmemMax; }

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
  EGNN_CHECK_CUDA(launch_pdl(ns_fused_kernel, dim3(b.count), dim3(kThreads + 32), smem, s, b, q));
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
