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
// A block computes tiles of 128 rows and 64 or 128 columns of its group's products:
// one warp streams operands through a ring of 64-column stages, one issues the
// products, sixteen turn accumulators (two, used in turn) into blocks of an image,
// which leave through shared memory as bulk copies (16-byte stores from the
// accumulators' rows and the fence behind them took 8,300 cycles a tile, these 6,300).
// Blocks of a group meet after each product at a counter in global memory; only the
// copies of the next product wait for it.  The wait is bounded, and the launch is
// cooperative, so all blocks are resident.
//
// What bounds it: the chain of a product, some 13,000 cycles of which the tensor cores
// work 2,000 to 7,000: meeting and first copies 3,400, the last accumulator's way into
// shared memory 2,800, from there into L2 3,500.  One 200 x 333 takes 114 us for 5 steps,
// the 30 matrices of six H = 256 layers 187 us, 30 of 256 x 513 201 to 212 us: the six layers' 13 GF,
// three times in half precision, are 24 us of the measured matrix rate.
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
  unsigned* counter;     // arrivals of the group's blocks, for each phase
  int* start;            // X0 is below 2^start; kGaveUp: a wait ran out, the image is not complete
  float* part;           // pieces of A
  double* partial;       // sums of squares of the parts of U
};
constexpr int kGaveUp = 1 << 20;
constexpr int kItems = kNsLarge;   // matrices of one launch
struct Grid {
  NsItem it[kItems];
  Work w[kItems];
  int first[kItems + 1];   // first block of each matrix's group
  int count, tile;           // tile: columns of a product that a block computes at once
};
constexpr int kParts = 32;   // blocks of a matrix in the norm

// A's sum runs over the long side.  It is split into pieces of at least kSplit chunks
// of 64 columns, which a group's blocks compute side by side, as float32, and add up,
// in order, in a phase of its own.  The pieces' number follows from the matrix alone,
// and with it the result.  In pieces and whole: 64 x 1100 107 and 135 us, 128 x 900 130
// and 141, 1 x 16384 164 and 861.  It is no gain where bands fill the device: 1024 x 1024
// 280 and 238; pieces of 4 make 30 matrices of 256 x 513 slower (238 and 201), of 9 leave
// 64 x 1100 at 119.
constexpr int kSplit = 6, kMostPieces = 64;   // of them all tiles

struct Shape {
  int m, n, m16, n16, bands, xc, ac;   // 128-row bands, 64-column blocks of X and of A
  int tile;                            // 64 or 128
  int pieces, piece;                   // of A, and the chunks of each
  bool turn;
  __host__ __device__ explicit Shape(const NsItem& it, int tile_ = 128) : tile(tile_) {
    turn = it.rows > it.cols;
    m = turn ? it.cols : it.rows;
    n = turn ? it.rows : it.cols;
    m16 = (m + 15) & ~15;
    n16 = (n + 15) & ~15;
    bands = up(m, 128);
    xc = up(n, 64);
    ac = up(m, 64);
    pieces = xc / kSplit < kMostPieces / (bands * bands) ? xc / kSplit : kMostPieces / (bands * bands);
    piece = pieces > 1 ? up(xc, pieces) : xc;
    pieces = up(xc, piece);
  }
  __host__ __device__ size_t x_bytes() const { return (size_t)bands * xc * kBlk; }   // of hi alone
  __host__ __device__ size_t a_bytes() const { return (size_t)bands * ac * kBlk; }
  __host__ __device__ size_t part_bytes() const { return pieces > 1 ? (size_t)pieces * bands * bands * 65536 : 0; }
  // Phases of a step: the products 0: A, 1: B, 2: X', and 3: the pieces of A added up.
  __host__ __device__ int per_step() const { return pieces > 1 ? 4 : 3; }
  __host__ __device__ int mode(int p) const {
    const int k = p % per_step();
    return pieces > 1 && k ? k == 1 ? 3 : k - 1 : k;
  }
  // tiles of a product
  __host__ __device__ int tile_cols(int mode) const { return up(mode == 2 ? n16 : m16, tile); }
  __host__ __device__ int tiles(int mode) const { return bands * tile_cols(mode) * (mode == 0 ? pieces : 1); }
  // rows of a band that hold anything (those a copy moves), and the ring's stages:
  // hi and lo of a band of L, then of R
  __host__ __device__ int band_rows(int band) const { return m16 - 128 * band < 128 ? m16 - 128 * band : 128; }
  __host__ __device__ int l_bytes() const { return band_rows(0) * 128; }
  __host__ __device__ int r_bytes(int mode) const { return mode != 2 && bands == 1 ? 0 : tile * 128; }
  __host__ __device__ int stage_bytes(int mode) const { return 2 * (l_bytes() + r_bytes(mode)); }
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
    for (int k = threadIdx.x; k < 4 * q.steps; k += 256) w.counter[k] = 0;
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
  int e;
  norm_scale(ss, q.eps, pre, f, e);
  if (blockIdx.x == 0 && threadIdx.x == 0) *g.w[blockIdx.y].start = e;
  const float sx = ns_pow2(14 - e);
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
      for (int k = 0; k < 8; ++k) v[k] *= sx;
      unit_to_pairs(hi + band, lo + band, 128, sh.turn, t, v);
    } else {
      unit_to_raw(hi + band, lo + band, kBlk, sh.turn, t, v);
    }
  }
}

// ---- the result out of the image, or the weight moved by it --------------------
// A matrix whose iteration gave up is left alone: there are no numbers in its image.
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
  if (*g.w[blockIdx.y].start == kGaveUp) return;
  const Shape sh(it);
  const char* hi = g.w[blockIdx.y].x[q.steps & 1];
  const char* lo = hi + sh.x_bytes();
  if (it.dtype == EGNN_DTYPE_F32) give<float>(it, q, sh, hi, lo);
  else if (it.dtype == EGNN_DTYPE_BF16) give<__nv_bfloat16>(it, q, sh, hi, lo);
  else give<__half>(it, q, sh, hi, lo);
}

// What the warps of a block need to know of each phase of a step, in shared memory.
struct Phase {
  int mode, tn, round, tiles;       // tile columns, tiles of a piece, of all pieces
  int k16, piece, chunks;           // K in steps of 16; chunks of a piece, and in all
  int stages, stage_bytes, r_bytes; // the ring
  __device__ void set(const Shape& sh, int k) {
    mode = sh.mode(k);
    tn = sh.tile_cols(mode);
    round = sh.bands * tn;
    tiles = sh.tiles(mode);
    k16 = sh.k16(mode);
    chunks = up(k16, 4);
    piece = mode == 0 ? sh.piece : chunks;
    stages = sh.stages(mode);
    stage_bytes = sh.stage_bytes(mode);
    r_bytes = sh.r_bytes(mode);
  }
};
// The t-th tile of a product: its place, and its chunks of K.
struct Tile {
  int ti, tj, k0, k1;
  __device__ __forceinline__ Tile(const Phase& f, int t) {
    k0 = 0;
    for (; t >= f.round; t -= f.round) k0 += f.piece;
    k1 = min(k0 + f.piece, f.chunks);
    ti = t / f.tn;
    tj = t - ti * f.tn;
  }
};

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

// Whether every block of the group has arrived at `counter`; the wait is bounded.
__device__ __forceinline__ bool wait_group(const unsigned* counter, int group, volatile int* gave_up) {
  bool here = false;
  for (uint32_t i = 0; i < (1u << 23) && !here; ++i) {
    here = load_acquire(counter) == (unsigned)group;
    if (!here && (i & 255u) == 255u && *gave_up) break;
  }
  here = __all_sync(0xffffffffu, here);
  if (!here) *gave_up = 1;
  return here;
}

// B and X' add a multiple of the same tile of A or X to their product.  That
// tile comes through the ring anyhow: as chunks of L (A: the tile's columns)
// or of R (X: rows of the band ti), from where the readers take it.
__device__ __forceinline__ bool old_chunk(int mode, int ti, int tj, int kc, int tile) {
  return mode == 1 ? kc / (tile >> 6) == tj : mode == 2 && (kc >> 1) == ti;
}

// Pieces of A: 16 readers' elements of each tile, four columns of a reader's 32 rows after one another.
__device__ __forceinline__ float4* piece_at(float* part, int tile, int t, int reader) {
  return reinterpret_cast<float4*>(part) + ((size_t)t * kReaders + reader) * (2 * tile) + (threadIdx.x & 31);
}
// A (hi; lo `size` bytes further) from its pieces, eight columns of a reader's rows at a time.
template <int tile>
__device__ __noinline__ void add_pieces(float* part, char* a, size_t size, int tn, int tiles, int pieces, int m16, int blocks,
                                        int first, int stride) {
  constexpr int W = tile / 4, units = W / 8;   // of a reader
#pragma unroll 1
  for (int u = first; u < tiles * kReaders * units; u += stride) {
    const int at = u / units, t = at / kReaders, reader = at % kReaders;
    // a reader is a warp, of which the first two do not read: its rows follow from the warp
    const int row = (reader + 2 & 3) * 32 + (threadIdx.x & 31);
    const int c = tile * (t % tn) + (reader >> 2) * W + u % units * 8;
    if (c >= m16) continue;
    const float4* from = piece_at(part, tile, t, reader) + u % units * 64;
    float v[8] = {};
#pragma unroll 4
    for (int k = 0; k < pieces; ++k, from += tiles * kReaders * 2 * tile) {
      const float4 x = __ldcg(from), y = __ldcg(from + 32);
      v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
      v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) split2(v[2 * k], v[2 * k + 1], h[k], l[k]);
    char* const to = a + (size_t)(t / tn) * blocks * kBlk + sw128_offset(row, c, 128);
    *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(to + size) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

template <int tile>   // columns of a product that a block computes at once: 64 or 128
__global__ void __launch_bounds__(kThreads, 1) ns_grid_kernel(const __grid_constant__ Grid g,
                                                              const __grid_constant__ NsScalars q) {
  extern __shared__ char raw[];
  __shared__ Barriers bar;
  __shared__ uint32_t tmem_s;
  __shared__ Phase phase[4];
  __shared__ NsStep weights[kNsMaxSteps];
  __shared__ int gave_up_s;
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  int item = 0;
  while (item + 1 < g.count && g.first[item + 1] <= (int)blockIdx.x) ++item;
  const Shape sh(g.it[item], tile);
  const Work& w = g.w[item];
  const int group = g.first[item + 1] - g.first[item], rank = blockIdx.x - g.first[item];
  char* const ring = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  char* const out = ring + kRing;
  volatile int* const gave_up = &gave_up_s;

  if (warp == 0 && lane < sh.per_step()) phase[lane].set(sh, lane);
  if (warp == 2) {
    int e = *w.start;
    for (int k = 0; k < q.steps; ++k) {
      const NsStep s(q, k, e);
      if (lane == 0) weights[k] = s;
    }
  }
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
  const int per_step = sh.per_step(), phases = per_step * q.steps, segment = sh.segment(), l_all = sh.l_bytes();
  bool ok = true;

  if (warp == 0) {
    // ---- copies.  Before a product's first copy all of the last one's are read
    // (this block's own arrival says so), so the ring is cut anew for each.
    uint32_t used = 0, parity = 0;   // bit k: stage k has been filled; the parity of its last filling
    uint32_t old = 0, old_parity = 0;   // the same of its fillings with a chunk that the readers take from
#pragma unroll 1
    for (int p = 0, k = 0, cur = 0; p < phases && ok; ++p, ++k) {
      if (k == per_step) k = 0, cur ^= 1;
      const Phase& f = phase[k];
      const int mode = f.mode;
      if (mode == 3) continue;
      if (p > 0) {   // every block of the group has written its tiles of the last phase
        if (!(ok = wait_group(w.counter + p - 1, group, gave_up))) break;
        fence_proxy_async_all();
      }
      const char* Lh = mode == 0 ? w.x[cur] : mode == 1 ? w.a : w.b;
      const char* Rh = mode == 1 ? w.a : w.x[cur];
      const size_t lsize = mode == 0 ? sh.x_bytes() : sh.a_bytes(), rsize = mode == 1 ? sh.a_bytes() : sh.x_bytes();
      const int lc = mode == 0 ? sh.xc : sh.ac;   // column blocks of L (and of a K-major R)
      const int stages = f.stages, stage_bytes = f.stage_bytes, r_all = f.r_bytes;
      int st = 0;
#pragma unroll 1
      for (int t = rank; t < f.tiles && ok; t += group) {
        const Tile at(f, t);
        const int ti = at.ti, tj = at.tj;
        const int rcols = mode == 2 ? min(tile >> 6, sh.xc - (tile >> 6) * tj) : 0;   // 64-column blocks of an MN-major R
        const int rrow = tile * tj & 127;                                             // first row in its band of a K-major R
        const bool shared = mode != 2 && ti == tile * tj >> 7;
        const uint32_t lbytes = sh.band_rows(ti) * 128, rbytes = mode == 2 || shared ? 0 : min(tile, sh.m16 - tile * tj) * 128;
        const uint32_t bytes = 2 * lbytes + 2 * rbytes + rcols * kBlk;
#pragma unroll 1
        for (int kc = at.k0; kc < at.k1 && ok; ++kc) {
          if ((used >> st & 1u) && !(ok = wait_bar(&bar.empty[st], parity >> st & 1u, gave_up))) break;
          if (old >> st & 1u) {
            if (!(ok = wait_bar(&bar.old_read[st], old_parity >> st & 1u, gave_up))) break;
            old &= ~(1u << st);
            old_parity ^= 1u << st;
          }
          if (old_chunk(mode, ti, tj, kc, tile)) old |= 1u << st;
          if (used >> st & 1u) parity ^= 1u << st;
          used |= 1u << st;
          if (lane == 0) {
            char* const to = ring + st * stage_bytes;
            const size_t l = (size_t)(ti * lc + kc) * kBlk;
            mbar_expect_tx_bytes(&bar.full[st], bytes);
            bulk_copy_g2s(to, Lh + l, lbytes, &bar.full[st]);
            bulk_copy_g2s(to + l_all, Lh + lsize + l, lbytes, &bar.full[st]);
            char* const rt = to + 2 * l_all;
            if (mode == 2) {   // 64 rows of X: half of a block for each column block
              for (int c = 0; c < rcols; ++c) {
                const size_t r = (size_t)((kc >> 1) * sh.xc + (tile >> 6) * tj + c) * kBlk + (kc & 1) * (kBlk / 2);
                bulk_copy_g2s(rt + c * (kBlk / 2), Rh + r, kBlk / 2, &bar.full[st]);
                bulk_copy_g2s(rt + r_all + c * (kBlk / 2), Rh + rsize + r, kBlk / 2, &bar.full[st]);
              }
            } else if (!shared) {
              const size_t r = (size_t)((tile * tj >> 7) * lc + kc) * kBlk + rrow * 128;
              bulk_copy_g2s(rt, Rh + r, rbytes, &bar.full[st]);
              bulk_copy_g2s(rt + r_all, Rh + rsize + r, rbytes, &bar.full[st]);
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
    for (int p = 0, k = 0; p < phases && ok; ++p, ++k) {
      if (k == per_step) k = 0;
      const Phase& f = phase[k];
      const int mode = f.mode, k16 = f.k16;
      if (mode == 3) continue;
      const int stages = f.stages, stage_bytes = f.stage_bytes, r_all = f.r_bytes;
      int st = 0;
#pragma unroll 1
      for (int t = rank; t < f.tiles && ok; t += group) {
        const Tile x(f, t);
        const int ti = x.ti, tj = x.tj;
        const bool shared = mode != 2 && ti == tile * tj >> 7;
        const uint32_t idesc = make_idesc_f16(128, min(tile, (mode == 2 ? sh.n16 : sh.m16) - tile * tj), 0, mode == 2);
#pragma unroll 1
        for (int kc = x.k0; kc < x.k1 && ok; ++kc) {
          const bool start = (kc - x.k0) % segment == 0;
          // the accumulator's last user has been read
          if (start && !(ok = wait_bar(&bar.acc_empty[seg & 1], ((seg >> 1) & 1) ^ 1, gave_up))) break;
          if (!(ok = wait_bar(&bar.full[st], parity >> st & 1u, gave_up))) break;
          parity ^= 1u << st;
          const uint32_t d = tmem + (seg & 1) * 256;   // hi hi, and the small terms 128 columns further
          // a K-major R of the band ti is part of L
          const uint32_t at = smem_u32(ring + st * stage_bytes), rt = shared ? at + (tile * tj & 127) * 128 : at + 2 * l_all;
          const uint32_t rlo = rt + (shared ? l_all : r_all), lbo = mode == 2 ? kBlk / 2 : 16;
          const uint64_t lh = make_desc(at, 16, 1024), ll = make_desc(at + l_all, 16, 1024);
          const uint64_t rh = make_desc(rt, lbo, 1024), rl = make_desc(rlo, lbo, 1024);
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
          if ((kc + 1 - x.k0) % segment == 0 || kc + 1 == x.k1) {
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
    // a quarter of the tile's columns
    constexpr int W = tile / 4;
    const int row = (warp & 3) * 32 + lane, c = ((warp - 2) >> 2) * W, c16 = c >> 4 & 1;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const float loss = ns_mean_loss(4 * segment);
    int seg = 0, outs = 0, sent = 0;
    const NsStep* step = weights;
    // The readers' arrival at `written`.  A warp arrives again only when the last round is
    // complete: arrivals are counted, not the warps, and a fast one's second would stand for a slow
    // one's first.
    auto arrive_written = [&]() {
      __syncwarp();
      if (outs && !(ok = wait_bar(&bar.written, outs - 1, gave_up))) return false;
      if (lane == 0) mbar_arrive(&bar.written);
      ++outs;
      return true;
    };
    uint32_t parity = 0;   // of each stage's next filling
#pragma unroll 1
    for (int p = 0, phase_of_step = 0, cur = 0; p < phases && ok; ++p, ++phase_of_step) {
      if (phase_of_step == per_step) {
        phase_of_step = 0;
        cur ^= 1;
        ++step;
      }
      const Phase& f = phase[phase_of_step];
      const int mode = f.mode;
      if (mode == 3) {
        if (!(ok = wait_group(w.counter + p - 1, group, gave_up))) break;
        add_pieces<tile>(w.part, w.a, sh.a_bytes(), phase[0].tn, phase[0].round, sh.pieces, sh.m16, sh.ac,
                         rank + group * (warp - 2), group * kReaders);
        fence_proxy_async_all();
      }
      const bool apart = mode == 0 && sh.pieces > 1;
      const int blocks = mode == 2 ? sh.xc : sh.ac;
      const size_t size = mode == 2 ? sh.x_bytes() : sh.a_bytes();
      const int stages = f.stages, stage_bytes = f.stage_bytes, r_all = f.r_bytes;
      int st = 0;
      char* const dst = mode == 0 ? w.a : mode == 1 ? w.b : w.x[cur ^ 1];
      const bool last = p + 1 == phases;   // X' itself, not scaled
      // weights of the product and of the old tile
      const float wp = mode == 0 ? kNsGram : mode == 1 ? step->cc : step->bx;
      const float wo = mode == 1 ? step->b : step->x;
#pragma unroll 1
      for (int t = rank; mode != 3 && t < f.tiles && ok; t += group) {
        const Tile at(f, t);
        const int ti = at.ti, tj = at.tj;
        const int N = min(tile, (mode == 2 ? sh.n16 : sh.m16) - tile * tj);
        const bool here = c < N;
        const size_t band = (size_t)ti * blocks * kBlk;
        float acc[W];
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k] = 0.f;
        const int mine = mode == 1 ? (tile * tj + c) >> 6 : 2 * ti + (row >> 6);   // the chunk with this warp's part
#pragma unroll 1
        for (int kc = at.k0; kc < at.k1; ++kc) {
          if (old_chunk(mode, ti, tj, kc, tile)) {
            if (here && kc == mine) {
              if (!(ok = wait_bar(&bar.full[st], parity >> st & 1u, gave_up))) break;
              const uint32_t stage = smem_u32(ring) + st * stage_bytes;
              const uint32_t from = mode == 1 ? row_at(stage, 128, row, c & 63)
                                              : row_at(stage + 2 * l_all + (c >> 6) * (kBlk / 2), 128, row & 63, c & 63);
#pragma unroll
              for (int h = 0; h < W; h += 16) {
                float x[16];
                load_pairs16(from, from + (mode == 1 ? l_all : r_all), c16 + (h >> 4), x);
#pragma unroll
                for (int k = 0; k < 16; ++k) acc[h + k] = fmaf(wo, x[k], acc[h + k]);
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.old_read[st]);
          }
          parity ^= 1u << st;
          if (++st == stages) st = 0;
          if ((kc + 1 - at.k0) % segment && kc + 1 < at.k1) continue;
          if (!(ok = wait_bar(&bar.acc_full[seg & 1], (seg >> 1) & 1, gave_up, q.wait_polls))) break;
          if (here) {
#pragma unroll
            for (int h = 0; h < W; h += 16) {
              float small[16], v[16];
              const uint32_t at16 = tmem + (seg & 1) * 256 + lanes + c + h;
              tmem_ld16x2(at16 + 128, at16, small, v);
#pragma unroll
              for (int k = 0; k < 16; ++k)
                acc[h + k] = fmaf(wp, fmaf(v[k], loss, v[k]), fmaf(wp, small[k], acc[h + k]));
            }
          }
          fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.acc_empty[seg & 1]);
          ++seg;
        }
        if (!ok) break;
        if (apart) {
          if (here) {
            float4* const to = piece_at(w.part, tile, t, warp - 2);
#pragma unroll
            for (int k = 0; k < W / 4; ++k) to[32 * k] = make_float4(acc[4 * k], acc[4 * k + 1], acc[4 * k + 2], acc[4 * k + 3]);
          }
          continue;
        }
        // A tile leaves as hi and lo through the blocks behind the ring.  They hold one of
        // two 128 columns wide: those go one after the other, but for the block's last
        // tile of the product, which takes the ring, idle until the group has met.
        const uint32_t bytes = sh.band_rows(ti) * 128;
        const bool ring_free = t + group >= f.tiles;
        auto hand_on = [&]() {   // true in warp 2 when all have written
          fence_proxy_async();
          if (!arrive_written()) return false;
          if (warp == 2) ok = wait_bar(&bar.written, outs - 1, gave_up);
          return warp == 2 && ok;
        };
        auto out_free = [&]() {   // the copies out of the blocks behind the ring have read them
          if (sent) {
            if (warp == 2 && lane == 0) {
              asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
              mbar_arrive(&bar.out_free);
            }
            __syncwarp();
            ok = wait_bar(&bar.out_free, sent - 1, gave_up);
          }
          ++sent;
          return ok;
        };
        auto send = [&](char* from, int part) {
          char* const to = dst + part * size + band + (size_t)(tile * tj >> 6) * kBlk;
          bulk_copy_s2g(to, from, bytes);
          if (N > 64) bulk_copy_s2g(to + kBlk, from + kBlk, bytes);
        };
        auto commit = []() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); };
        auto emit = [&]() {
          if (tile == 64 || ring_free) {
            if (tile == 64) {
              if (!out_free()) return;
            } else if (mode != 0) {   // every reader has taken its part of the old tile out of the ring
              if (!arrive_written() || !(ok = wait_bar(&bar.written, outs - 1, gave_up))) return;
            }
            char* const from = tile == 64 ? out : ring;
            if (here) {
              const uint32_t hi = row_at(smem_u32(from), 128, row, c), lo = hi + tile * 256;
#pragma unroll
              for (int h = 0; h < W; h += 16)
                if (last) store_raw16(hi, lo, c16 + (h >> 4), acc + h);
                else store_pairs16(hi, lo, c16 + (h >> 4), acc + h);
            }
            if (hand_on() && lane == 0) {
              send(from, 0);
              send(from + tile * 256, 1);
              commit();
            }
            __syncwarp();
            return;
          }
          uint32_t words[2][W / 2];   // hi and lo; at the end float32 columns 0 .. 15 and 16 .. 31
          if (last) {
#pragma unroll
            for (int k = 0; k < W; ++k) words[2 * k / W][k % (W / 2)] = __float_as_uint(acc[k]);
          } else {
#pragma unroll
            for (int k = 0; k < W / 2; ++k) split2(acc[2 * k], acc[2 * k + 1], words[0][k], words[1][k]);
          }
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            if (!out_free()) return;
            if (here) {
              const uint32_t to = row_at(smem_u32(out), 128, row, c);
#pragma unroll
              for (int j = 0; j < W / 8; ++j)
                sts16(to ^ (j << 4), words[part][4 * j], words[part][4 * j + 1], words[part][4 * j + 2], words[part][4 * j + 3]);
            }
            if (hand_on() && lane == 0) {
              send(out, part);
              commit();
            }
            __syncwarp();
          }
        };
        emit();
        if (!ok) break;
      }
      if (!ok) break;
      if (apart || mode == 3) {   // what all readers have stored
        if (!arrive_written()) break;
        if (warp == 2 && !(ok = wait_bar(&bar.written, outs - 1, gave_up))) break;
      }
      if (warp == 2 && lane == 0) {
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        fence_proxy_async_all();
        if (!last) asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(w.counter + p) : "memory");
      }
      __syncwarp();
    }
    if (!ok && warp == 2 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    if (lane == 0 && *gave_up) {
      *w.start = kGaveUp;
      atomicAdd(&g_ns_grid_timeouts, 1);
    }
    tmem_dealloc(tmem, 512);
  }
}

// The time of a matrix's step with a group of g blocks, in cycles, fitted to lists of
// 200 x 333 and 256 x 513: a phase's meeting and first copies, and for each tile of a
// block its chunks of K and its way out.
int step_time(const Shape& s, int g) {
  const int tile = s.tile == 64 ? 5000 : 5500, chunk = s.tile == 64 ? 550 : 1000;
  int t = 0;
  for (int mode = 0; mode < 3; ++mode)
    t += 8000 + 30 * g + up(s.tiles(mode), g) * (tile + chunk * (mode == 0 ? s.piece : up(s.k16(mode), 4)));
  return t;
}

// Shares `blocks` out, size[i] to matrix i: again and again to the matrix that takes
// longest, as many more as shorten its step.  Returns the longest step's time.
int allot(const Grid& g, int blocks, int tile, int* size) {
  int time[kItems], left = blocks - g.count, most = 0;
  bool done[kItems] = {};
  for (int i = 0; i < g.count; ++i) {
    size[i] = 1;
    time[i] = step_time(Shape(g.it[i], tile), 1);
  }
  while (left > 0) {
    int worst = -1;
    for (int i = 0; i < g.count; ++i)
      if (!done[i] && (worst < 0 || time[i] > time[worst])) worst = i;
    if (worst < 0) break;
    const Shape s(g.it[worst], tile);
    const int end = std::min(size[worst] + left, std::max(s.tiles(0), s.tiles(2)));
    int next = size[worst] + 1, t = 0;
    while (next <= end && (t = step_time(s, next)) >= time[worst]) ++next;
    if (next > end) {
      done[worst] = true;
      continue;
    }
    left -= next - size[worst];
    size[worst] = next;
    time[worst] = t;
  }
  for (int i = 0; i < g.count; ++i) most = std::max(most, time[i]);
  return most;
}

// Tiles 64 or 128 columns wide, whichever let the longest step end first: 64 make more
// of them, each sooner done.  64 and 128: 200 x 333 114 and 134 us, 16 matrices of 256 x 513
// 151 and 182, 30 of them 239 and 201, six H = 256 layers 213 and 187.
void share_out(Grid& g, int blocks) {
  int size64[kItems], size128[kItems];
  g.tile = allot(g, blocks, 64, size64) < allot(g, blocks, 128, size128) ? 64 : 128;
  const int* const size = g.tile == 64 ? size64 : size128;
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
  w.counter = c.take<unsigned>(4 * kNsMaxSteps);   // the last of 4 kNsMaxSteps phases has none
  w.start = reinterpret_cast<int*>(w.counter + 4 * kNsMaxSteps - 1);
  w.part = c.take<float>(s.part_bytes() / 4);
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
    EGNN_CHECK_CUDA(cudaLaunchKernelEx(&cfg, g.tile == 64 ? ns_grid_kernel<64> : ns_grid_kernel<128>, (const Grid&)g, q));
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

int ns_grid(const NsBatch& b, Carver c, const NsScalars& q, int spare, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  const uint64_t bit = device_bit();
  if (!(ready.load() & bit)) {
    EGNN_CHECK_CUDA(cudaFuncSetAttribute(ns_grid_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    EGNN_CHECK_CUDA(cudaFuncSetAttribute(ns_grid_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    ready.fetch_or(bit);
  }
  const int blocks = std::max(1, num_sms_current() - spare);
  Grid g;
  g.count = 0;
  for (int i = 0; i < b.count; ++i) {
    g.it[g.count] = b.it[i];
    g.w[g.count] = carve_work(c, Shape(b.it[i]));
    if (++g.count == std::min(kItems, blocks) || i + 1 == b.count) {
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
