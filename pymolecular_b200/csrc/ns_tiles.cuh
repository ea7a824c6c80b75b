// Element access of the Newton-Schulz kernels: fp16 hi / lo pairs in swizzled
// tiles, and the way of a matrix between its own layout and those tiles.
#pragma once

#include "newton_schulz.cuh"
#include "tc.cuh"

namespace egnn {
namespace ns {

using tc::sw128_offset;

// hi and lo tiles at (row, c0 .. c0 + 15) <- v[at .. at + 15].
__device__ __forceinline__ void store_pairs16(char* hi, char* lo, int R, int row, int c0, const float* v) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
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
__device__ __forceinline__ void store_raw16(char* hi, char* lo, int R, int row, int c0, const float* v) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
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

// A warp's share of a matrix in global memory: units of 8 rows x 32 columns,
// a column to a lane, so that an element costs few instructions besides its
// access: the swizzle of row k of a unit is a constant of k.  In a turned
// matrix the 8 rows are one 16-byte chunk of a tile row.
struct Unit {
  int id, per_row, stride, r0, c;
  __device__ __forceinline__ Unit(int cols, int first, int stride_)
      : id(first), per_row((cols + 31) >> 5), stride(stride_) {
    place();
  }
  __device__ __forceinline__ void place() {
    r0 = id / per_row * 8;
    c = id % per_row * 32 + (threadIdx.x & 31);
  }
  __device__ __forceinline__ void next() {
    id += stride;
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

// 8 float32 <-> one chunk of a tile row (raw halves).
__device__ __forceinline__ void store_chunk_raw(char* hi, char* lo, const float (&v)[8]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t x = __float_as_uint(v[2 * k]), y = __float_as_uint(v[2 * k + 1]);
    h[k] = __byte_perm(x, y, 0x7632);
    l[k] = __byte_perm(x, y, 0x5410);
  }
  *reinterpret_cast<uint4*>(hi) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4*>(lo) = make_uint4(l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ void load_chunk_raw(const char* hi, const char* lo, float (&v)[8]) {
  const uint4 h = *reinterpret_cast<const uint4*>(hi), l = *reinterpret_cast<const uint4*>(lo);
  const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = __uint_as_float(__byte_perm(ll[k], hh[k], 0x5410));
    v[2 * k + 1] = __uint_as_float(__byte_perm(ll[k], hh[k], 0x7632));
  }
}
__device__ __forceinline__ void store_raw(char* hi, char* lo, float v) {
  const uint32_t x = __float_as_uint(v);
  *reinterpret_cast<uint16_t*>(hi) = (uint16_t)(x >> 16);
  *reinterpret_cast<uint16_t*>(lo) = (uint16_t)x;
}
__device__ __forceinline__ float load_raw(const char* hi, const char* lo) {
  return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(hi) << 16 |
                         *reinterpret_cast<const uint16_t*>(lo));
}

// The scale 1 / (norm + eps) as pre * f: a power of two first, so that f is a
// float32 at any norm.
__device__ __forceinline__ void norm_scale(double ss, double eps, float& pre, float& f) {
  const double inv = 1.0 / (sqrt(ss) + eps);
  pre = inv > 1.0 ? 0x1p64f : inv < 0x1p-64 ? 0x1p-64f : 1.f;
  f = (float)(inv / (double)pre);
}

// ---- waits -------------------------------------------------------------------
// Bounded wait, the same answer in the whole warp; false when it or another
// warp's wait ran out.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  bool ok = false;
  for (uint32_t i = 0; i < (1u << 22) && !ok; ++i) {
    ok = tc::mbar_try_wait(bar, parity & 1u);
    if (!ok && (i & 255u) == 255u && *gave_up) break;
  }
  ok = __all_sync(0xffffffffu, ok);
  if (!ok) *gave_up = 1;
  tc::fence_after_sync();
  return ok;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}

}  // namespace ns
}  // namespace egnn
