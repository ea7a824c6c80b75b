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

// The same places hold a float32's upper and lower 16 bits before the first
// product and after the last.
__device__ __forceinline__ void store_raw32(char* hi, char* lo, int R, int row, int c0, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t x = __float_as_uint(v[8 * j + 2 * k]), y = __float_as_uint(v[8 * j + 2 * k + 1]);
      h[k] = __byte_perm(x, y, 0x7632);
      l[k] = __byte_perm(x, y, 0x5410);
    }
    const uint32_t at = sw128_offset(row, c0 + 8 * j, R);
    *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}
__device__ __forceinline__ void load_raw32(const char* hi, const char* lo, int R, int row, int c0, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t at = sw128_offset(row, c0 + 8 * j, R);
    const uint4 h = *reinterpret_cast<const uint4*>(hi + at), l = *reinterpret_cast<const uint4*>(lo + at);
    const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[8 * j + 2 * k] = __uint_as_float(__byte_perm(ll[k], hh[k], 0x5410));
      v[8 * j + 2 * k + 1] = __uint_as_float(__byte_perm(ll[k], hh[k], 0x7632));
    }
  }
}

// Issues D (+)= L R over nk K-steps of 16.  L is K-major; R is K-major, or
// MN-major from column c0 on.  Tiles of `rows` rows; only the address field of
// the descriptors moves.
template <bool MN>
__device__ __forceinline__ void issue(uint32_t one, uint32_t d, const char* L, const char* Rt, int rows, int c0, int nk, uint32_t idesc,
                                      bool accumulate) {
  const uint32_t blk = rows * 128;
  uint64_t l = make_desc(smem_u32(L), 16, 1024);
  uint64_t r = MN ? make_desc(smem_u32(Rt) + (c0 >> 6) * blk, blk, 1024) : make_desc(smem_u32(Rt), 16, 1024);
  uint32_t acc = accumulate;
#pragma unroll 1
  for (int k0 = 0; k0 < nk; k0 += 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k0 + j < nk) {
        mma_f16_elected(one, d, l + 2 * j, r + (MN ? 128 : 2) * j, idesc, acc);
        acc = 1;
      }
    l += blk >> 4;
    r += MN ? 512 : blk >> 4;
  }
}
// lo hi + hi lo + hi hi, in this order.
template <bool MN>
__device__ __forceinline__ void issue3(uint32_t one, uint32_t d, const char* Lh, const char* Ll, const char* Rh, const char* Rl, int rows,
                                       int c0, int nk, uint32_t idesc) {
  issue<MN>(one, d, Ll, Rh, rows, c0, nk, idesc, false);
  issue<MN>(one, d, Lh, Rl, rows, c0, nk, idesc, true);
  issue<MN>(one, d, Lh, Rh, rows, c0, nk, idesc, true);
}

// A warp's share of a matrix in global memory: units of 8 rows x 32 columns,
// a column to a lane, so that an element costs few instructions besides its
// access: the swizzle of row k of a unit is a constant of k.  In a turned
// matrix the 8 rows are one 16-byte chunk of a tile row.
struct Unit {
  int id, per_row, r0, c;
  __device__ __forceinline__ Unit(int cols) : id(threadIdx.x >> 5), per_row((cols + 31) >> 5) { place(); }
  __device__ __forceinline__ void place() {
    r0 = id / per_row * 8;
    c = id % per_row * 32 + (threadIdx.x & 31);
  }
  __device__ __forceinline__ void next() {
    id += kWarps;
    place();
  }
};
// Tile offset of element (r0 + k, c): chunk (k, in the low bits) of a tile whose column blocks are blk bytes.
__device__ __forceinline__ uint32_t unit_row(const Unit& u, uint32_t blk, int k) {
  return (u.c >> 6) * blk + ((u.r0 + k) << 7) + ((((u.c >> 3) & 7) ^ k) << 4) + ((u.c & 7) << 1);
}
__device__ __forceinline__ uint32_t unit_chunk(const Unit& u, uint32_t blk) {
  return (u.r0 >> 6) * blk + (u.c << 7) + ((((u.r0 >> 3) & 7) ^ (u.c & 7)) << 4);
}

// The unit's 8 elements of this lane; zeros outside the matrix.
template <typename T>
__device__ __forceinline__ void unit_load(const T* p, int64_t ld, const Unit& u, int rows, int cols, float (&v)[8]) {
  const int n = u.c < cols ? rows - u.r0 : 0;
  p += u.r0 * ld + u.c;
#pragma unroll
  for (int k = 0; k < 8; ++k, p += ld) v[k] = k < n ? ns_float(*p) : 0.f;
}
template <typename T>
__device__ __forceinline__ void unit_store(T* p, int64_t ld, const Unit& u, int rows, int cols, const float (&v)[8]) {
  const int n = u.c < cols ? rows - u.r0 : 0;
  p += u.r0 * ld + u.c;
#pragma unroll
  for (int k = 0; k < 8; ++k, p += ld)
    if (k < n) *p = ns_from<T>(v[k]);
}

// U into the tiles (raw); returns this thread's sum of squares, added in
// float64: no overflow or underflow at any scale of the gradient.  The next
// unit's loads are in flight while a unit is worked on.
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
  float g[8], m[8];
  Unit u(cols);
  if (u.r0 < rows) {
    unit_load(in, ld_in, u, rows, cols, g);
    if (MOM) unit_load(mom, ld_mom, u, rows, cols, m);
  }
#pragma unroll 1
  while (u.r0 < rows) {
    float g2[8], m2[8];
    Unit t = u;
    t.next();
    if (t.r0 < rows) {
      unit_load(in, ld_in, t, rows, cols, g2);
      if (MOM) unit_load(mom, ld_mom, t, rows, cols, m2);
    }
    if (MOM) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = fmaf(mu, m[k], nu * g[k]);
        g[k] = nesterov ? fmaf(mu, m[k], nu * g[k]) : m[k];
      }
      unit_store(mom, ld_mom, u, rows, cols, m);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fma((double)g[k], (double)g[k], ss);
    if (u.c < cols) {   // rows past the matrix get the zeros that are there already
      if (turn) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t x = __float_as_uint(g[2 * k]), y = __float_as_uint(g[2 * k + 1]);
          h[k] = __byte_perm(x, y, 0x7632);
          l[k] = __byte_perm(x, y, 0x5410);
        }
        const uint32_t o = unit_chunk(u, blk);
        *reinterpret_cast<uint4*>(Xh + o) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(Xl + o) = make_uint4(l[0], l[1], l[2], l[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t o = unit_row(u, blk, k), x = __float_as_uint(g[k]);
          *reinterpret_cast<uint16_t*>(Xh + o) = (uint16_t)(x >> 16);
          *reinterpret_cast<uint16_t*>(Xl + o) = (uint16_t)x;
        }
      }
    }
    u = t;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      g[k] = g2[k];
      if (MOM) m[k] = m2[k];
    }
  }
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
  float w[8];
  Unit u(cols);
  if (MOM && u.r0 < rows) unit_load(out, ld, u, rows, cols, w);
#pragma unroll 1
  while (u.r0 < rows) {
    float w2[8], v[8];
    Unit t = u;
    t.next();
    if (MOM && t.r0 < rows) unit_load(out, ld, t, rows, cols, w2);
    if (u.c < cols) {
      if (turn) {
        const uint32_t o = unit_chunk(u, blk);
        const uint4 h = *reinterpret_cast<const uint4*>(Xh + o), l = *reinterpret_cast<const uint4*>(Xl + o);
        const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[2 * k] = __uint_as_float(__byte_perm(ll[k], hh[k], 0x5410));
          v[2 * k + 1] = __uint_as_float(__byte_perm(ll[k], hh[k], 0x7632));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t o = unit_row(u, blk, k);
          v[k] = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(Xh + o) << 16 |
                                 *reinterpret_cast<const uint16_t*>(Xl + o));
        }
      }
      if (MOM)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fmaf(move, v[k], keep * w[k]);
      unit_store(out, ld, u, rows, cols, v);
    }
    u = t;
    if (MOM)
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = w2[k];
  }
}

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

  __syncthreads();
  double ss = it.mom                            ? take_in<float, true>(it, q, Xh, Xl, R * 128, turn)
              : it.dtype == EGNN_DTYPE_F32  ? take_in<float, false>(it, q, Xh, Xl, R * 128, turn)
              : it.dtype == EGNN_DTYPE_BF16 ? take_in<__nv_bfloat16, false>(it, q, Xh, Xl, R * 128, turn)
                                            : take_in<__half, false>(it, q, Xh, Xl, R * 128, turn);
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
  // a power of two first, so that the rest of the scale is a float32 at any norm
  const float pre = inv > 1.0 ? 0x1p64f : inv < 0x1p-64 ? 0x1p-64f : 1.f, f = (float)(inv / (double)pre);
  // warp w owns tile rows 32 (w % 4) .. + 31, which are its accumulator lanes,
  // and of each group of four 32-column pieces the (w / 4)-th
  const int row = (warp & 3) * 32 + lane, piece = warp >> 2;
  const bool rows_here = (warp & 3) * 32 < R;
  const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  if (rows_here)
    for (int c0 = piece * 32; c0 < n16; c0 += 128) {
      float v[32];
      load_raw32(Xh, Xl, R, row, c0, v);
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = v[k] * pre * f;
      if (q.steps == 0) {
        store_raw32(Xh, Xl, R, row, c0, v);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] *= q.sx;
        store_pairs32(Xh, Xl, R, row, c0, v);
      }
    }
  hand_over();

  const uint32_t tA = 0, tAA = 128;
  const uint32_t idesc_m = make_idesc_f16(128, m16, 0, 0);
  const float fA = q.sa / (q.sx * q.sx);                    // accumulator -> A scaled
  const float fbA = q.b * q.sb / (q.sx * q.sx), fcAA = q.c * q.sb / (q.sa * q.sa);
  const float fX = 1.f / q.sb, back = 1.f / q.sx;
  const int n_slots = (n16 + kSlotCols - 1) / kSlotCols;
  const int uwarp = __shfl_sync(0xffffffffu, warp, 0);   // the same, known to be uniform
  uint32_t phase = 0, pending = 0;   // bit k: parity of bar[k]; a commit on it not yet waited for
  bool ok = true;

  // X' columns [128 k, 128 k + 128) into slot k % kSlots
  auto issue_update = [&](int k) {
    pending |= 1u << (k % kSlots);
    if (uwarp != 0) return;
    const int c0 = k * kSlotCols, N = min(kSlotCols, n16 - c0);
    const uint32_t one = elect_one();
    issue3<true>(one, tmem + (k % kSlots) * kSlotCols, Ah, Al, Xh, Xl, R, c0, m16 / 16, make_idesc_f16(128, N, 0, 1));
    if (one) mma_commit(&bar[k % kSlots]);
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
    if (uwarp == 0) {
      const uint32_t one = elect_one();
      issue3<false>(one, tmem + tA, Xh, Xl, Xh, Xl, R, 0, n16 / 16, idesc_m);
      if (one) mma_commit(&bar[0]);
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
    if (uwarp == 0) {
      const uint32_t one = elect_one();
      issue3<false>(one, tmem + tAA, Ah, Al, Ah, Al, R, 0, m16 / 16, idesc_m);
      if (one) mma_commit(&bar[0]);
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
        if (step + 1 < q.steps) {
          store_pairs32(Xh, Xl, R, row, c0, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= back;
          store_raw32(Xh, Xl, R, row, c0, v);
        }
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
    if (it.mom) give_out<float, true>(it, q, Xh, Xl, R * 128, turn);
    else if (it.dtype == EGNN_DTYPE_F32) give_out<float, false>(it, q, Xh, Xl, R * 128, turn);
    else if (it.dtype == EGNN_DTYPE_BF16) give_out<__nv_bfloat16, false>(it, q, Xh, Xl, R * 128, turn);
    else give_out<__half, false>(it, q, Xh, Xl, R * 128, turn);
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
