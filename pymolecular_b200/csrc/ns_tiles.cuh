// Element access of the Newton-Schulz kernels: fp16 hi / lo pairs in swizzled
// tiles, and the way of a matrix between its own layout and those tiles.
#pragma once

#include "newton_schulz.cuh"
#include "tc.cuh"

namespace egnn {
namespace ns {

using tc::sw128_offset;

// hi + c and hi - c with hi one half of a word of two fp16, in float32.
__device__ __forceinline__ float add_low(uint32_t w, float c) {
  float d;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tadd.f32.f16 %0, a, %2;\n\t}" : "=f"(d) : "r"(w), "f"(c));
  return d;
}
__device__ __forceinline__ float add_high(uint32_t w, float c) {
  float d;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tadd.f32.f16 %0, b, %2;\n\t}" : "=f"(d) : "r"(w), "f"(c));
  return d;
}
// x, y as fp16 pairs hi + lo, x in the lower half of the words.
__device__ __forceinline__ void split2(float x, float y, uint32_t& h, uint32_t& l) {
  const __half2 p = __floats2half2_rn(x, y);
  h = *reinterpret_cast<const uint32_t*>(&p);
  const __half2 r = __floats2half2_rn(-add_low(h, -x), -add_high(h, -y));
  l = *reinterpret_cast<const uint32_t*>(&r);
}

// ---- 32 columns of a tile row in shared memory -----------------------------------
// They are 4 chunks of 16 bytes in the hi tile and 4 in the lo tile, chunk j at the
// row's address ^ (j << 4).  As float32 (before the first product and after the
// last) the same bytes hold columns 0 .. 15 in hi and 16 .. 31 in lo.
__device__ __forceinline__ uint32_t row_at(uint32_t tile, int R, int row, int c0) {
  return tile + (c0 >> 6) * (R * 128) + (row << 7) + (((c0 >> 3 & 4) ^ (row & 7)) << 4);
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Columns 16 half .. + 15 as pairs.
__device__ __forceinline__ void store_pairs16(uint32_t hi, uint32_t lo, int half, const float* v) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) split2(v[8 * j + 2 * k], v[8 * j + 2 * k + 1], h[k], l[k]);
    const uint32_t chunk = (2 * half + j) << 4;
    sts16(hi ^ chunk, h[0], h[1], h[2], h[3]);
    sts16(lo ^ chunk, l[0], l[1], l[2], l[3]);
  }
}
__device__ __forceinline__ void load_pairs16(uint32_t hi, uint32_t lo, int half, float* v) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t chunk = (2 * half + j) << 4;
    const uint4 h = lds16(hi ^ chunk), l = lds16(lo ^ chunk);
    const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[8 * j + 2 * k] = add_low(hh[k], add_low(ll[k], 0.f));
      v[8 * j + 2 * k + 1] = add_high(hh[k], add_high(ll[k], 0.f));
    }
  }
}
__device__ __forceinline__ void load_pairs32(uint32_t hi, uint32_t lo, float (&v)[32]) {
  load_pairs16(hi, lo, 0, v);
  load_pairs16(hi, lo, 1, v + 16);
}
// Columns 16 half .. + 15 as float32.
__device__ __forceinline__ void store_raw16(uint32_t hi, uint32_t lo, int half, const float* v) {
  const uint32_t t = half ? lo : hi;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    sts16(t ^ (j << 4), __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
          __float_as_uint(v[4 * j + 3]));
}
__device__ __forceinline__ void load_raw32(uint32_t hi, uint32_t lo, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint4 x = lds16((j & 4 ? lo : hi) ^ ((j & 3) << 4));
    v[4 * j] = __uint_as_float(x.x);
    v[4 * j + 1] = __uint_as_float(x.y);
    v[4 * j + 2] = __uint_as_float(x.z);
    v[4 * j + 3] = __uint_as_float(x.w);
  }
}
// Offset of float32 column c in its tile.
__device__ __forceinline__ uint32_t raw_offset(int row, int c, uint32_t blk) {
  return (c >> 6) * blk + (row << 7) + ((((c >> 3 & 4) | (c >> 2 & 3)) ^ (row & 7)) << 4) + ((c & 3) << 2);
}

// A warp's share of a matrix in global memory: units of 8 rows x 32 columns,
// a column to a lane, so that an element costs few instructions besides its
// access: the swizzle of row k of a unit is a constant of k.  Two units share
// 64 columns, 16 of each 32 to a unit: those lie in one tile and in all its
// banks.  In a turned matrix the 8 rows are two chunks of a tile row.
struct Unit {
  int id, per_row, stride, r0, c;
  __device__ __forceinline__ Unit(int cols, int first, int stride_)
      : id(first), per_row((cols + 63) / 64 * 2), stride(stride_) {
    place();
  }
  __device__ __forceinline__ void place() {
    const int lane = threadIdx.x & 31, j = id % per_row;
    r0 = id / per_row * 8;
    c = (j >> 1) * 64 + (lane & 16) * 2 + (j & 1) * 16 + (lane & 15);
  }
  __device__ __forceinline__ void next() {
    id += stride;
    place();
  }
};
// The raw elements (r0 .. r0 + 7, c) of a tile, or (c, r0 .. r0 + 7) of a turned one.
__device__ __forceinline__ void unit_to_raw(char* hi, char* lo, uint32_t blk, bool turn, const Unit& u, const float (&v)[8]) {
  if (turn) {
    char* const t = u.r0 & 16 ? lo : hi;
    *reinterpret_cast<float4*>(t + raw_offset(u.c, u.r0, blk)) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(t + raw_offset(u.c, u.r0 + 4, blk)) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    char* const t = u.c & 16 ? lo : hi;
#pragma unroll
    for (int k = 0; k < 8; ++k) *reinterpret_cast<float*>(t + raw_offset(u.r0 + k, u.c, blk)) = v[k];
  }
}
__device__ __forceinline__ void unit_from_raw(const char* hi, const char* lo, uint32_t blk, bool turn, const Unit& u,
                                              float (&v)[8]) {
  if (turn) {
    const char* const t = u.r0 & 16 ? lo : hi;
    const float4 x = *reinterpret_cast<const float4*>(t + raw_offset(u.c, u.r0, blk));
    const float4 y = *reinterpret_cast<const float4*>(t + raw_offset(u.c, u.r0 + 4, blk));
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  } else {
    const char* const t = u.c & 16 ? lo : hi;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const float*>(t + raw_offset(u.r0 + k, u.c, blk));
  }
}
// The same of pairs.
__device__ __forceinline__ void unit_to_pairs(char* hi, char* lo, int R, bool turn, const Unit& u, const float (&v)[8]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) split2(v[2 * k], v[2 * k + 1], h[k], l[k]);
  if (turn) {
    const uint32_t at = sw128_offset(u.c, u.r0, R);
    *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t at = sw128_offset(u.r0 + k, u.c, R);
      *reinterpret_cast<uint16_t*>(hi + at) = (uint16_t)(h[k >> 1] >> (k & 1) * 16);
      *reinterpret_cast<uint16_t*>(lo + at) = (uint16_t)(l[k >> 1] >> (k & 1) * 16);
    }
  }
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

// The sum of 8 squares, for a sum in float64: in float32 where that neither
// overflows nor loses small ones (conversions and float64 products would cost
// more than the rest of an element).
__device__ __forceinline__ double squares(const float (&v)[8]) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s = fmaf(v[k], v[k], s);
  if (s > 0x1p-80f && s < 0x1p100f) return (double)s;
  uint32_t any = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) any |= __float_as_uint(v[k]) << 1;
  if (!any) return 0.0;
  double d = 0.0;
#pragma unroll 1
  for (int k = 0; k < 8; ++k) {
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) x = j == k ? v[j] : x;
    d = fma((double)x, (double)x, d);
  }
  return d;
}

// x 2^-e for |e| < 1000.
__device__ __forceinline__ float scaled_down(double x, int e) {
  return (float)(x * __hiloint2double((1023 - e) << 20, 0));
}
// 1 / (sqrt(ss) + eps) as pre * f, so that both are float32 at any norm: norm and
// eps are brought near 1 by the power of two h of the larger, and half of it goes
// to each factor.  Float32 arithmetic: a float64 square root and division took
// 3,000 cycles of a block's time.  bound: the norm after it is at most 2^bound.
__device__ __forceinline__ void norm_scale(double ss, double eps, float& pre, float& f, int& bound) {
  bound = 0;
  const int e = ((__double2hiint(ss) >> 20) & 0x7ff) - 1023;   // -1023: zero; 1024: infinity or NaN
  if (e == 1024) {
    pre = 1.f;
    f = (float)(1.0 / ss);
    return;
  }
  const int eh = ((__double2hiint(eps) >> 20) & 0x7ff) - 1023;
  int h = max(e >> 1, eh);
  h = min(max(h, -200), 200);
  const float norm = e == -1023 ? 0.f : ldexpf(sqrtf(scaled_down(ss, e & ~1)), max((e >> 1) - h, -200));
  const float t = 1.f / (norm + scaled_down(eps, h));
  const int h1 = h / 2;
  pre = ldexpf(1.f, -h1);
  f = ldexpf(t, h1 - h);
  bound = max(kNsLeast, min(0, (__float_as_int(norm * t) >> 23 & 255) - 126));
}

// ---- waits -------------------------------------------------------------------
constexpr int kWaitPolls = 1 << 22;
// Bounded wait, the same answer in the whole warp; false when it or another
// warp's wait ran out.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* gave_up, int polls = kWaitPolls) {
  bool ok = false;
  for (int i = 0; i < polls && !ok; ++i) {
    ok = tc::mbar_try_wait(bar, parity & 1u);
    if (!ok && (i & 255) == 255 && *gave_up) break;
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
