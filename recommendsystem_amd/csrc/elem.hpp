// Element types of the sequence kernels (layernorm.hip, recurrence.hip, pack8.hip): fp32, bf16 and
// fp16 rows, computed in fp32 and rounded to nearest even once, on the store.
#pragma once
#include "common.hpp"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

enum { RS_F32 = 0, RS_BF16 = 1, RS_F16 = 2 };

typedef uint32_t rs_u32x4 __attribute__((ext_vector_type(4)));

// A 16-byte vector of V elements.  Rows may start at any element (an odd width, a column slice):
// gfx950 reads and writes global vectors at any alignment, so the access only promises the
// element's own.
template <int BYTES, int ALIGN>
struct __attribute__((packed, aligned(ALIGN))) RsVec {
  uint32_t w[BYTES / 4];
};

struct ElemF32 {
  typedef float T;
  static constexpr int V = 4;  // elements of 16 bytes
  static __device__ __forceinline__ float load(T x) { return x; }
  static __device__ __forceinline__ T store(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ void pack(const float* x, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
  }
};

struct ElemBF16 {
  typedef __bf16 T;
  static constexpr int V = 8;
  static __device__ __forceinline__ float load(T x) { return (float)x; }
  static __device__ __forceinline__ T store(float x) { return (__bf16)x; }
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ void pack(const float* x, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(pack_bf16(x[2 * i], x[2 * i + 1]));
  }
};

struct ElemF16 {
  typedef _Float16 T;
  static constexpr int V = 8;
  static __device__ __forceinline__ float load(T x) { return (float)x; }
  static __device__ __forceinline__ T store(float x) { return (_Float16)x; }
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
      x[2 * i] = (float)h[0];
      x[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ void pack(const float* x, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 h = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
      w[i] = __builtin_bit_cast(uint32_t, h);
    }
  }
};

// FN<Elem>(...) for the run-time type code; an unknown code is a bad argument
#define RS_DISPATCH_ELEM(dtype, FN, ...)                     \
  ((dtype) == RS_F32    ? FN<ElemF32>(__VA_ARGS__)           \
   : (dtype) == RS_BF16 ? FN<ElemBF16>(__VA_ARGS__)          \
   : (dtype) == RS_F16  ? FN<ElemF16>(__VA_ARGS__)           \
                        : (int)RS_ERR_ARG)

// ---------------------------------------------------------------------------------------------
// The 8-bit form of a row: blocks of 128 columns (the last one short), each with one fp32 scale
//   s = max|x| / 127,   code = x / s to the nearest whole number, ties to even,   x ~ code * s.
// The codes are exactly those of the definition, not of a rounded quotient: the first guess
// rint(x * (1/s)) is off by one at most, and the remainder x - code * s, which one fma gives
// without error there, says which way.  A block whose largest magnitude is below 2^-100 is kept
// as zeros; one with an infinity or NaN gets that as its scale, so all of it reads back as NaN.
// ---------------------------------------------------------------------------------------------
#define RS_PACK_BLOCK 128
#define RS_PACK_TINY 7.888609052210118e-31f  // 2^-100

static __device__ __forceinline__ float pack8_scale(uint32_t top_bits) {
  const float top = __uint_as_float(top_bits);
  return top < RS_PACK_TINY ? 0.f : top / 127.0f;
}
static __device__ __forceinline__ float pack8_inverse(float s) {
  return s == 0.f ? 0.f : __builtin_amdgcn_rcpf(s);
}
static __device__ __forceinline__ int pack8_code(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, s, x), half = 0.5f * s;
  if (fabsf(r) >= half) {  // one step further, or a tie: only then is q looked at
    const bool odd = ((int)q) & 1;
    if (r > half || (r == half && odd)) q += 1.f;
    else if (r < -half || (r == -half && odd)) q -= 1.f;
  }
  // 0 for a block kept as zeros (s = 0) and for the NaN of one that is not finite
  return s > 0.f && fabsf(q) <= 127.f ? (int)q : 0;
}
