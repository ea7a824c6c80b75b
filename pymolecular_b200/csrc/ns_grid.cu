// Newton-Schulz iteration of matrices that a block's shared memory does not
// hold: one cooperative launch whose blocks share out the matrices, each group
// of blocks running all steps of its matrix on the tensor cores.
//
//   A = X X^T,  B = b A + c A A,  X <- a X + B X      (X m x n, m <= n)
//
// X (two buffers), A and B lie in the workspace as images: 128-row bands of
// 64-column blocks, each block the 16 KB shared-memory form of an fp16 operand
// (hi, and lo after all hi blocks), so that a bulk copy moves a block and the
// same block serves as K-major and as MN-major operand.  Products are lo hi +
// hi lo + hi hi as in the one-block kernel.  At these sizes images stay in L2.
//
// A block computes 128 x 128 tiles of its group's products: one warp streams
// operands through a ring of 64-column stages, one issues the products, sixteen
// turn accumulators (two, used in turn) into blocks of an image, which leave
// through shared memory as bulk copies (16-byte stores from the accumulators'
// rows and the fence behind them took 8,300 cycles a tile, these 6,300).  Blocks
// of a group meet after each product at a counter in global memory; only the copies
// of the next product wait for it.  The wait is bounded, and the launch is
// cooperative, so all blocks are resident.
//
// What bounds it: at one to three tiles a product the chain of copy latency,
// products, accumulator reads and the meeting, not the tensor cores.
//
// Sums in tensor memory are rounded towards zero at every instruction, by the
// size of the sum so far.  So lo hi + hi lo has an accumulator of its own, and
// an accumulator takes at most 128 terms, in 8 instructions; the pieces are
// added in float32 registers, and what truncation loses on average is added back.
#include <atomic>

#include "ns_tiles.cuh"

namespace egnn {

__device__ int g_ns_grid_timeouts = 0;

namespace {

using namespace tc;
using namespace ns;

constexpr int kReaders = 16;           // warps that read accumulators
constexpr int kThreads = 64 + 32 * kReaders;   // and one of copies, one of products
constexpr int kMaxStages = 8;
constexpr int kBlk = 16384;            // bytes of a 128 x 64 block
constexpr int kRing = 12 * kBlk;
constexpr size_t kSmem = kRing + 2 * kBlk + 1024;   // the ring, the blocks on their way out, alignment

__host__ __device__ inline int up(int a, int b) { return (a + b - 1) / b; }

struct Work {
  char* x[2];            // images: hi blocks, then lo blocks
  char *a, *b;
  unsigned* counter;     // arrivals of the group's blocks, for each product
  double* partial;       // sums of squares of the parts of U
};
struct Grid {
  NsItem it[kNsItems];
  Work w[kNsItems];
  int first[kNsItems + 1];   // first block of each matrix's group
  int count;
};
constexpr int kParts = 32;   // blocks of a matrix in the norm

struct Shape {
  int m, n, m16, n16, bands, xc, ac;   // 128-row bands, 64-column blocks of X and of A
  bool turn;
  __host__ __device__ explicit Shape(const NsItem& it) {
    turn = it.rows > it.cols;
    m = turn ? it.cols : it.rows;
    n = turn ? it.rows : it.cols;
    m16 = (m + 15) & ~15;
    n16 = (n + 15) & ~15;
    bands = up(m, 128);
    xc = up(n, 64);
    ac = up(m, 64);
  }
  __host__ __device__ size_t x_bytes() const { return (size_t)bands * xc * kBlk; }   // of hi alone
  __host__ __device__ size_t a_bytes() const { return (size_t)bands * ac * kBlk; }
  // tiles of a product (0: A, 1: B, 2: X') and its 64-column chunks of K
  __host__ __device__ int tile_cols(int mode) const { return mode == 2 ? up(n16, 128) : bands; }
  __host__ __device__ int tiles(int mode) const { return bands * tile_cols(mode); }
  // rows of a band that hold anything (those a copy moves), and the ring's stages
  __host__ __device__ int band_rows(int band) const { return m16 - 128 * band < 128 ? m16 - 128 * band : 128; }
  __host__ __device__ int stage_bytes(int mode) const {
    const int rows = band_rows(0) * 128;   // a block of the highest band
    return 2 * rows + (mode == 2 ? 2 * kBlk : bands > 1 ? 2 * rows : 0);
  }
  __host__ __device__ int stages(int mode) const {
    const int s = kRing / stage_bytes(mode);
    return s < kMaxStages ? s : kMaxStages;
  }
  // 64-column chunks of one accumulator.  One band has few accumulators to add up,
  // and shorter ones (128 x 2000: error 2.6e-6 with two chunks, 1.8e-6 with one) cost it little.
  __host__ __device__ int segment() const { return bands > 1 ? 2 : 1; }
  __host__ __device__ int k16(int mode) const { return (mode == 0 ? n16 : m16) >> 4; }
};

// The band of an image that a unit lies in; its row there becomes a tile row.
__device__ __forceinline__ size_t to_band(Unit& u, int blocks, bool turn) {
  int& r = turn ? u.c : u.r0;
  const size_t band = (size_t)(r >> 7) * blocks * kBlk;
  r &= 127;
  return band;
}

// ---- U: momentum, and the sums of squares of kParts parts of each matrix ------
__global__ void __launch_bounds__(256) ns_norm_kernel(const __grid_constant__ Grid g, const __grid_constant__ NsScalars q) {
  pdl_enter();
  __shared__ double red[8];
  const NsItem& it = g.it[blockIdx.y];
  const Work& w = g.w[blockIdx.y];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x == 0)
    for (int k = threadIdx.x; k < 3 * q.steps; k += 256) w.counter[k] = 0;
  double ss = 0.0;
  for (Unit u(it.cols, blockIdx.x * 8 + warp, kParts * 8); u.r0 < it.rows; u.next()) {
    float v[8];
    if (it.dtype == EGNN_DTYPE_F32) unit_load(static_cast<const float*>(it.in), it.ld_in, u, it.rows, it.cols, v);
    else if (it.dtype == EGNN_DTYPE_BF16) unit_load(static_cast<const __nv_bfloat16*>(it.in), it.ld_in, u, it.rows, it.cols, v);
    else unit_load(static_cast<const __half*>(it.in), it.ld_in, u, it.rows, it.cols, v);
    if (it.mom) {
      float mo[8];
      unit_load(it.mom, it.ld_mom, u, it.rows, it.cols, mo);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        mo[k] = ns_momentum(q, v[k], mo[k]);
        v[k] = ns_update(q, v[k], mo[k]);
      }
      unit_store(it.mom, it.ld_mom, u, it.rows, it.cols, mo);
    }
    ss += squares(v);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  if (threadIdx.x) return;
  for (int k = 1; k < 8; ++k) ss += red[k];
  w.partial[blockIdx.x] = ss;
}

// ---- X0 as an image, zeros around the matrix ----------------------------------
__global__ void __launch_bounds__(256) ns_image_kernel(const __grid_constant__ Grid g, const __grid_constant__ NsScalars q) {
  pdl_enter();
  const NsItem& it = g.it[blockIdx.y];
  const Shape sh(it);
  double ss = 0.0;
  for (int k = 0; k < kParts; ++k) ss += g.w[blockIdx.y].partial[k];
  float pre, f;
  norm_scale(ss, q.eps, pre, f);
  char* const hi = g.w[blockIdx.y].x[0];
  char* const lo = hi + sh.x_bytes();
  const int rows = sh.turn ? sh.xc * 64 : sh.bands * 128, cols = sh.turn ? sh.bands * 128 : sh.xc * 64;
  for (Unit u(cols, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8); u.r0 < rows; u.next()) {
    float v[8];
    if (it.dtype == EGNN_DTYPE_F32) unit_load(static_cast<const float*>(it.in), it.ld_in, u, it.rows, it.cols, v);
    else if (it.dtype == EGNN_DTYPE_BF16) unit_load(static_cast<const __nv_bfloat16*>(it.in), it.ld_in, u, it.rows, it.cols, v);
    else unit_load(static_cast<const __half*>(it.in), it.ld_in, u, it.rows, it.cols, v);
    if (it.mom) {
      float mo[8];
      unit_load(it.mom, it.ld_mom, u, it.rows, it.cols, mo);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = ns_update(q, v[k], mo[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] * pre * f;
    Unit t = u;
    const size_t band = to_band(t, sh.xc, sh.turn);
    if (q.steps) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= q.sx;
      unit_to_pairs(hi + band, lo + band, 128, sh.turn, t, v);
    } else {
      unit_to_raw(hi + band, lo + band, kBlk, sh.turn, t, v);
    }
  }
}

// ---- the result out of the image, or the weight moved by it --------------------
template <typename T>
__device__ __forceinline__ void give(const NsItem& it, const NsScalars& q, const Shape& sh, const char* hi, const char* lo) {
  T* const out = static_cast<T*>(it.out);
  float keep = 0.f, move = 0.f;
  if (it.mom) ns_rates(it, q, keep, move);
  for (Unit u(it.cols, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8); u.r0 < it.rows; u.next()) {
    float v[8], w[8];
    if (u.c >= it.cols) continue;
    if (it.mom) unit_load(out, it.ld_out, u, it.rows, it.cols, w);
    Unit t = u;
    const size_t band = to_band(t, sh.xc, sh.turn);
    unit_from_raw(hi + band, lo + band, kBlk, sh.turn, t, v);
    if (it.mom)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = fmaf(move, v[k], keep * w[k]);
    unit_store(out, it.ld_out, u, it.rows, it.cols, v);
  }
}
__global__ void __launch_bounds__(256) ns_give_kernel(const __grid_constant__ Grid g, const __grid_constant__ NsScalars q) {
  pdl_enter();
  const NsItem& it = g.it[blockIdx.y];
  const Shape sh(it);
  const char* hi = g.w[blockIdx.y].x[q.steps & 1];
  const char* lo = hi + sh.x_bytes();
  if (it.dtype == EGNN_DTYPE_F32) give<float>(it, q, sh, hi, lo);
  else if (it.dtype == EGNN_DTYPE_BF16) give<__nv_bfloat16>(it, q, sh, hi, lo);
  else give<__half>(it, q, sh, hi, lo);
}

// ---- the steps ------------------------------------------------------------------
struct Barriers {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t old_read[kMaxStages];         // the readers have taken A or X out of the stage
  uint64_t acc_full[2], acc_empty[2];
  uint64_t written, out_free;            // the blocks on their way out
  uint64_t drained;
};

// Generic accesses of global memory <-> bulk copies.
__device__ __forceinline__ void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void bulk_copy_s2g(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

// B and X' add a multiple of the same tile of A or X to their product.  That
// tile comes through the ring anyhow: as two chunks of L (A: columns 2 tj, 2 tj + 1)
// or of R (X: rows of the band ti), from where the readers take it.
__device__ __forceinline__ bool old_chunk(int mode, int ti, int tj, int kc) {
  return mode != 0 && (kc >> 1) == (mode == 1 ? tj : ti);
}

__global__ void __launch_bounds__(kThreads, 1) ns_grid_kernel(const __grid_constant__ Grid g,
                                                              const __grid_constant__ NsScalars q) {
  extern __shared__ char raw[];
  __shared__ Barriers bar;
  __shared__ uint32_t tmem_s;
  __shared__ int gave_up_s;
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  int item = 0;
  while (item + 1 < g.count && g.first[item + 1] <= (int)blockIdx.x) ++item;
  const Shape sh(g.it[item]);
  const Work& w = g.w[item];
  const int group = g.first[item + 1] - g.first[item], rank = blockIdx.x - g.first[item];
  char* const ring = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  char* const out = ring + kRing;
  volatile int* const gave_up = &gave_up_s;

  if (warp == 1) {
    tmem_alloc(&tmem_s, 512);
    if (lane == 0) {
      gave_up_s = 0;
      for (int k = 0; k < kMaxStages; ++k) {
        mbar_init(&bar.full[k], 1);
        mbar_init(&bar.empty[k], 1);
        mbar_init(&bar.old_read[k], kReaders);
      }
      for (int k = 0; k < 2; ++k) {
        mbar_init(&bar.acc_full[k], 1);
        mbar_init(&bar.acc_empty[k], kReaders);
      }
      mbar_init(&bar.written, kReaders);
      mbar_init(&bar.out_free, 1);
      mbar_init(&bar.drained, 1);
      fence_mbar_init();
    }
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_s;
  const int phases = 3 * q.steps, segment = sh.segment();
  bool ok = true;

  if (warp == 0) {
    // ---- copies.  Before a product's first copy all of the last one's are read
    // (this block's own arrival says so), so the ring is cut anew for each.
    uint32_t used = 0, parity = 0;   // bit k: stage k has been filled; the parity of its last filling
    uint32_t old = 0, old_parity = 0;   // the same of its fillings with a chunk that the readers take from
#pragma unroll 1
    for (int p = 0; p < phases && ok; ++p) {
      const int mode = p % 3, cur = (p / 3) & 1;
      if (p > 0) {   // every block of the group has written its tiles of the last product
        bool here = false;
        for (uint32_t i = 0; i < (1u << 23) && !here; ++i) {
          here = load_acquire(w.counter + p - 1) == (unsigned)group;
          if (!here && (i & 255u) == 255u && *gave_up) break;
        }
        here = __all_sync(0xffffffffu, here);
        if (!here) {
          *gave_up = 1;
          ok = false;
          break;
        }
        fence_proxy_async_all();
      }
      const char* Lh = mode == 0 ? w.x[cur] : mode == 1 ? w.a : w.b;
      const char* Rh = mode == 1 ? w.a : w.x[cur];
      const size_t lsize = mode == 0 ? sh.x_bytes() : sh.a_bytes(), rsize = mode == 1 ? sh.a_bytes() : sh.x_bytes();
      const int lc = mode == 0 ? sh.xc : sh.ac;   // column blocks of L (and of a K-major R)
      const int chunks = up(sh.k16(mode), 4), tn = sh.tile_cols(mode);
      const int stages = sh.stages(mode), stage_bytes = sh.stage_bytes(mode), full_rows = sh.band_rows(0) * 128;
      int st = 0;
#pragma unroll 1
      for (int t = rank; t < sh.tiles(mode) && ok; t += group) {
        const int ti = t / tn, tj = t % tn;
        const int rcols = mode == 2 ? min(2, sh.xc - 2 * tj) : 0;   // 64-column blocks of an MN-major R
        const bool shared = mode != 2 && ti == tj;
        const uint32_t lbytes = sh.band_rows(ti) * 128, rbytes = mode == 2 || shared ? 0 : sh.band_rows(tj) * 128;
        const uint32_t bytes = 2 * lbytes + 2 * rbytes + rcols * kBlk;
#pragma unroll 1
        for (int kc = 0; kc < chunks && ok; ++kc) {
          if ((used >> st & 1u) && !(ok = wait_bar(&bar.empty[st], parity >> st & 1u, gave_up))) break;
          if (old >> st & 1u) {
            if (!(ok = wait_bar(&bar.old_read[st], old_parity >> st & 1u, gave_up))) break;
            old &= ~(1u << st);
            old_parity ^= 1u << st;
          }
          if (old_chunk(mode, ti, tj, kc)) old |= 1u << st;
          if (used >> st & 1u) parity ^= 1u << st;
          used |= 1u << st;
          if (lane == 0) {
            char* const to = ring + st * stage_bytes;
            const size_t l = (size_t)(ti * lc + kc) * kBlk;
            mbar_expect_tx_bytes(&bar.full[st], bytes);
            bulk_copy_g2s(to, Lh + l, lbytes, &bar.full[st]);
            bulk_copy_g2s(to + full_rows, Lh + lsize + l, lbytes, &bar.full[st]);
            char* const rt = to + 2 * full_rows;
            if (mode == 2) {   // 64 rows of X: half of a block for each column block
              for (int c = 0; c < rcols; ++c) {
                const size_t r = (size_t)((kc >> 1) * sh.xc + 2 * tj + c) * kBlk + (kc & 1) * (kBlk / 2);
                bulk_copy_g2s(rt + c * (kBlk / 2), Rh + r, kBlk / 2, &bar.full[st]);
                bulk_copy_g2s(rt + kBlk + c * (kBlk / 2), Rh + rsize + r, kBlk / 2, &bar.full[st]);
              }
            } else if (!shared) {
              const size_t r = (size_t)(tj * lc + kc) * kBlk;
              bulk_copy_g2s(rt, Rh + r, rbytes, &bar.full[st]);
              bulk_copy_g2s(rt + full_rows, Rh + rsize + r, rbytes, &bar.full[st]);
            }
          }
          if (++st == stages) st = 0;
        }
      }
    }
    if (*gave_up)   // no copy may still be landing when the block ends
      for (int k = 0; k < kMaxStages; ++k) {
        bool in = !(used >> k & 1u);
        for (uint32_t i = 0; i < (1u << 16) && !in; ++i) in = mbar_try_wait(&bar.full[k], parity >> k & 1u);
      }
  } else if (warp == 1) {
    // ---- products
    const uint32_t one = elect_one();
    int seg = 0;
    uint32_t parity = 0;   // of each stage's next filling
#pragma unroll 1
    for (int p = 0; p < phases && ok; ++p) {
      const int mode = p % 3, tn = sh.tile_cols(mode), k16 = sh.k16(mode), chunks = up(k16, 4);
      const int stages = sh.stages(mode), stage_bytes = sh.stage_bytes(mode), full_rows = sh.band_rows(0) * 128;
      int st = 0;
#pragma unroll 1
      for (int t = rank; t < sh.tiles(mode) && ok; t += group) {
        const int ti = t / tn, tj = t % tn;
        const bool shared = mode != 2 && ti == tj;
        const uint32_t idesc = make_idesc_f16(128, min(128, (mode == 2 ? sh.n16 : sh.m16) - 128 * tj), 0, mode == 2);
#pragma unroll 1
        for (int kc = 0; kc < chunks && ok; ++kc) {
          const bool start = kc % segment == 0;
          // the accumulator's last user has been read
          if (start && !(ok = wait_bar(&bar.acc_empty[seg & 1], ((seg >> 1) & 1) ^ 1, gave_up))) break;
          if (!(ok = wait_bar(&bar.full[st], parity >> st & 1u, gave_up))) break;
          parity ^= 1u << st;
          const uint32_t d = tmem + (seg & 1) * 256;   // hi hi, and the small terms 128 columns further
          const uint32_t at = smem_u32(ring + st * stage_bytes), rt = shared ? at : at + 2 * full_rows;
          const uint64_t lh = make_desc(at, 16, 1024), ll = make_desc(at + full_rows, 16, 1024);
          const uint64_t rh = mode == 2 ? make_desc(rt, kBlk / 2, 1024) : make_desc(rt, 16, 1024);
          const uint64_t rl = mode == 2 ? make_desc(rt + kBlk, kBlk / 2, 1024) : make_desc(rt + full_rows, 16, 1024);
          const int nk = k16 - 4 * kc;
          const uint32_t rstep = mode == 2 ? 128 : 2;
#pragma unroll
          for (int pr = 0; pr < 3; ++pr)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < nk)
                mma_f16_elected(one, pr == 2 ? d : d + 128, (pr == 0 ? ll : lh) + 2 * j, (pr == 1 ? rl : rh) + rstep * j,
                                idesc, !(start && pr != 1 && j == 0));
          if (one) mma_commit(&bar.empty[st]);
          if (++st == stages) st = 0;
          if ((kc + 1) % segment == 0 || kc + 1 == chunks) {
            if (one) mma_commit(&bar.acc_full[seg & 1]);
            ++seg;
          }
        }
      }
    }
    // nothing may be in flight when the tensor memory goes
    if (one) mma_commit(&bar.drained);
    wait_bar(&bar.drained, 0, gave_up);
  } else {
    // ---- accumulators into images: warp w reads the rows 32 (w % 4) .. + 31 of
    // one 32-column piece
    const int row = (warp & 3) * 32 + lane, c = ((warp - 2) >> 2) * 32;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const float loss = ns_mean_loss(4 * segment);
    int seg = 0, outs = 0, frees = 0;
    uint32_t parity = 0;   // of each stage's next filling
#pragma unroll 1
    for (int p = 0; p < phases && ok; ++p) {
      const int mode = p % 3, cur = (p / 3) & 1, tn = sh.tile_cols(mode), chunks = up(sh.k16(mode), 4);
      const int blocks = mode == 2 ? sh.xc : sh.ac;
      const size_t size = mode == 2 ? sh.x_bytes() : sh.a_bytes();
      const int stages = sh.stages(mode), stage_bytes = sh.stage_bytes(mode), full_rows = sh.band_rows(0) * 128;
      int st = 0;
      char* const dst = mode == 0 ? w.a : mode == 1 ? w.b : w.x[cur ^ 1];
      const bool last = p + 1 == phases;   // X' itself, not scaled
      // weights of the product and of the old tile
      const float end = last ? 1.f / q.sx : 1.f;
      const float wp = mode == 0 ? q.sa / (q.sx * q.sx) : mode == 1 ? q.c * q.sb / (q.sa * q.sa) : end / q.sb;
      const float wo = mode == 1 ? q.b * q.sb / q.sa : q.a * end;
#pragma unroll 1
      for (int t = rank; t < sh.tiles(mode) && ok; t += group) {
        const int ti = t / tn, tj = t % tn;
        const int N = min(128, (mode == 2 ? sh.n16 : sh.m16) - 128 * tj);
        const bool here = c < N;
        const size_t band = (size_t)ti * blocks * kBlk;
        float acc[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) acc[k] = 0.f;
        const int mine = mode == 1 ? 2 * tj + (c >> 6) : 2 * ti + (row >> 6);   // the chunk with this warp's part
#pragma unroll 1
        for (int kc = 0; kc < chunks; ++kc) {
          if (old_chunk(mode, ti, tj, kc)) {
            if (here && kc == mine) {
              if (!(ok = wait_bar(&bar.full[st], parity >> st & 1u, gave_up))) break;
              const uint32_t stage = smem_u32(ring) + st * stage_bytes;
              const uint32_t from = mode == 1 ? row_at(stage, 128, row, c & 63)
                                              : row_at(stage + 2 * full_rows + (c >> 6) * (kBlk / 2), 128, row & 63, c & 63);
              float x[32];
              load_pairs32(from, from + (mode == 1 ? full_rows : kBlk), x);
#pragma unroll
              for (int k = 0; k < 32; ++k) acc[k] = fmaf(wo, x[k], acc[k]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.old_read[st]);
          }
          parity ^= 1u << st;
          if (++st == stages) st = 0;
          if ((kc + 1) % segment && kc + 1 < chunks) continue;
          if (!(ok = wait_bar(&bar.acc_full[seg & 1], (seg >> 1) & 1, gave_up, q.wait_polls))) break;
          if (here) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {   // small terms and hi hi, 16 columns each
              float v[16];
              tmem_ld16(tmem + (seg & 1) * 256 + (h & 1 ? 0 : 128) + lanes + c + (h >> 1) * 16, v);
              const float l = h & 1 ? loss : 0.f;
#pragma unroll
              for (int k = 0; k < 16; ++k) acc[(h >> 1) * 16 + k] = fmaf(wp, fmaf(v[k], l, v[k]), acc[(h >> 1) * 16 + k]);
            }
          }
          fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.acc_empty[seg & 1]);
          ++seg;
        }
        if (!ok) break;
        // The block's last tile of the product leaves through the ring, which is
        // idle until the group has met, hi and lo at once; others, while the ring
        // serves the next tile, through the two blocks behind it, one after the other.
        const uint32_t bytes = sh.band_rows(ti) * 128;
        const bool ring_free = t + group >= sh.tiles(mode);
        uint32_t words[2][16];   // hi and lo of 32 columns; at the end float32 columns 0 .. 15 and 16 .. 31
        auto write = [&](char* at, int part) {
          if (!here) return;
          const uint32_t to = row_at(smem_u32(at), 128, row, c);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sts16(to ^ (j << 4), words[part][4 * j], words[part][4 * j + 1], words[part][4 * j + 2], words[part][4 * j + 3]);
        };
        auto meet = [&]() {   // of the readers
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.written);
          return wait_bar(&bar.written, outs++, gave_up);
        };
        auto hand_on = [&]() {   // true in warp 2 when all have written
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.written);
          if (warp == 2) ok = wait_bar(&bar.written, outs, gave_up);
          ++outs;
          return warp == 2 && ok;
        };
        auto send = [&](char* from, int part) {
          char* const to = dst + part * size + band + (size_t)2 * tj * kBlk;
          bulk_copy_s2g(to, from, bytes);
          if (N > 64) bulk_copy_s2g(to + kBlk, from + kBlk, bytes);
        };
        auto emit = [&]() {
          if (last) {
#pragma unroll
            for (int k = 0; k < 32; ++k) words[k >> 4][k & 15] = __float_as_uint(acc[k]);
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) split2(acc[2 * k], acc[2 * k + 1], words[0][k], words[1][k]);
          }
          if (ring_free) {
            // every reader has taken its part of the old tile out of the ring
            if (mode != 0 && !(ok = meet())) return;
            write(ring, 0);
            write(ring + 2 * kBlk, 1);
            if (hand_on() && lane == 0) {
              send(ring, 0);
              send(ring + 2 * kBlk, 1);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
            __syncwarp();
            return;
          }
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            if (frees && !(ok = wait_bar(&bar.out_free, frees - 1, gave_up))) return;
            ++frees;
            write(out, part);
            if (hand_on() && lane == 0) {
              send(out, part);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
              asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
              mbar_arrive(&bar.out_free);
            }
            __syncwarp();
          }
        };
        emit();
        if (!ok) break;
      }
      if (!ok) break;
      if (warp == 2 && lane == 0) {
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        fence_proxy_async_all();
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(w.counter + p) : "memory");
      }
      __syncwarp();
    }
    if (!ok && warp == 2 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    if (lane == 0 && *gave_up) atomicAdd(&g_ns_grid_timeouts, 1);
    tmem_dealloc(tmem, 512);
  }
}

// The time of a matrix's step with a group of g blocks, in chunks of K.
int step_time(const Shape& s, int g) {
  int t = 0;
  for (int mode = 0; mode < 3; ++mode) t += up(s.tiles(mode), g) * up(s.k16(mode), 4);
  return t;
}

// Shares `blocks` out: again and again to the matrix that takes longest, as
// many more as shorten its step.
void share_out(Grid& g, int blocks) {
  int size[kNsItems], time[kNsItems], left = blocks - g.count;
  for (int i = 0; i < g.count; ++i) {
    size[i] = 1;
    time[i] = step_time(Shape(g.it[i]), 1);
  }
  while (left > 0) {
    int worst = 0;
    for (int i = 1; i < g.count; ++i)
      if (time[i] > time[worst]) worst = i;
    const Shape s(g.it[worst]);
    const int most = std::min(size[worst] + left, std::max(s.tiles(0), s.tiles(2)));
    int next = size[worst] + 1;
    while (next <= most && step_time(s, next) >= time[worst]) ++next;
    if (next > most) break;
    left -= next - size[worst];
    size[worst] = next;
    time[worst] = step_time(s, next);
  }
  g.first[0] = 0;
  for (int i = 0; i < g.count; ++i) g.first[i + 1] = g.first[i] + size[i];
}

Work carve_work(Carver& c, const Shape& s) {
  Work w;
  w.x[0] = c.take<char>(2 * s.x_bytes());
  w.x[1] = c.take<char>(2 * s.x_bytes());
  w.a = c.take<char>(2 * s.a_bytes());
  w.b = c.take<char>(2 * s.a_bytes());
  w.partial = c.take<double>(kParts);
  w.counter = c.take<unsigned>(3 * kNsMaxSteps);
  return w;
}

int run(Grid& g, const NsScalars& q, int blocks, cudaStream_t s) {
  share_out(g, blocks);
  int units = 1;
  for (int i = 0; i < g.count; ++i) units = std::max(units, up(g.it[i].rows, 8) * up(g.it[i].cols, 32));
  const dim3 grid(std::min(128, up(units, 16)), g.count);
  TimerScope ts("newton_schulz", s);
  EGNN_CHECK_CUDA(launch_pdl(ns_norm_kernel, dim3(kParts, g.count), dim3(256), 0, s, g, q));
  EGNN_CHECK_LAUNCH();
  EGNN_CHECK_CUDA(launch_pdl(ns_image_kernel, grid, dim3(256), 0, s, g, q));
  EGNN_CHECK_LAUNCH();
  if (q.steps) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(g.first[g.count]);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    EGNN_CHECK_CUDA(cudaLaunchKernelEx(&cfg, ns_grid_kernel, (const Grid&)g, q));
    EGNN_CHECK_LAUNCH();
  }
  EGNN_CHECK_CUDA(launch_pdl(ns_give_kernel, grid, dim3(256), 0, s, g, q));
  EGNN_CHECK_LAUNCH();
  return EGNN_OK;
}

}  // namespace

void ns_grid_carve(Carver& c, int rows, int cols) {
  NsItem it = {};
  it.rows = rows;
  it.cols = cols;
  carve_work(c, Shape(it));
}

int ns_grid(const NsBatch& b, Carver& c, const NsScalars& q, int spare, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  const uint64_t bit = device_bit();
  if (!(ready.load() & bit)) {
    EGNN_CHECK_CUDA(cudaFuncSetAttribute(ns_grid_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    ready.fetch_or(bit);
  }
  const int blocks = std::max(1, num_sms_current() - spare);
  Grid g;
  g.count = 0;
  for (int i = 0; i < b.count; ++i) {
    g.it[g.count] = b.it[i];
    g.w[g.count] = carve_work(c, Shape(b.it[i]));
    if (++g.count == std::min(kNsItems, blocks) || i + 1 == b.count) {
      EGNN_TRY(run(g, q, blocks, s));
      g.count = 0;
    }
  }
  return EGNN_OK;
}

int ns_grid_take_timeouts() {
  int n = 0;
  if (cudaMemcpyFromSymbol(&n, g_ns_grid_timeouts, sizeof(int)) != cudaSuccess) return 0;
  if (n) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_ns_grid_timeouts, &zero, sizeof(int));
  }
  return n;
}

}  // namespace egnn
