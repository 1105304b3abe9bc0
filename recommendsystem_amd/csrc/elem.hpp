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
  template <int W = 4>
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* x) {
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = __uint_as_float(w[i]);
  }
  template <int W = 4>
  static __device__ __forceinline__ void pack(const float* x, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = __float_as_uint(x[i]);
  }
};

struct ElemBF16 {
  typedef __bf16 T;
  static constexpr int V = 8;
  static __device__ __forceinline__ float load(T x) { return (float)x; }
  static __device__ __forceinline__ T store(float x) { return (__bf16)x; }
  template <int W = 4>
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* x) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  template <int W = 4>
  static __device__ __forceinline__ void pack(const float* x, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = __float_as_uint(pack_bf16(x[2 * i], x[2 * i + 1]));
  }
};

struct ElemF16 {
  typedef _Float16 T;
  static constexpr int V = 8;
  static __device__ __forceinline__ float load(T x) { return (float)x; }
  static __device__ __forceinline__ T store(float x) { return (_Float16)x; }
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  template <int W = 4>
  static __device__ __forceinline__ void unpack(const uint32_t* w, float* x) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const f16x2 h = __builtin_bit_cast(f16x2, w[i]);
      x[2 * i] = (float)h[0];
      x[2 * i + 1] = (float)h[1];
    }
  }
  template <int W = 4>
  static __device__ __forceinline__ void pack(const float* x, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
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

typedef RsVec<16, 1> Raw;  // 16 bytes of a row as loaded

// 16 bytes of a row at p, or `fill` where they are not wanted (in = false; p then points at some 16
// bytes that may be read).  PART (D is no multiple of V): a lane with fewer than V elements left
// picks its nv elements one by one (none for nv <= 0); without it every lane reads 16 bytes.
template <class E, bool PART>
__device__ __forceinline__ void load16(Raw& r, const typename E::T* p, int nv, bool in,
                                       uint32_t fill) {
  constexpr int V = E::V, S = 16 / V;
  if (!PART || nv >= V) {
    const RsVec<16, S> x = *reinterpret_cast<const RsVec<16, S>*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = in ? x.w[i] : fill;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = fill;
    if (in) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < nv) {
          if (S == 4) r.w[j] = reinterpret_cast<const uint32_t*>(p)[j];
          else {
            const uint32_t h = reinterpret_cast<const uint16_t*>(p)[j];
            const uint32_t old = r.w[j * S / 4];
            r.w[j * S / 4] = (j & 1) ? (old & 0xFFFFu) | (h << 16) : (old & 0xFFFF0000u) | h;
          }
        }
    }
  }
}

template <class E>
__device__ __forceinline__ void store16(typename E::T* p, const float* x, int nv) {
  constexpr int V = E::V, S = 16 / V;
  RsVec<16, S> y;
  E::pack(x, y.w);
  if (nv >= V) *reinterpret_cast<RsVec<16, S>*>(p) = y;
  else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < nv) p[j] = E::store(x[j]);
  }
}

// V floats (a state, a gradient of one) at p
template <int V>
__device__ __forceinline__ void load_f(float* x, const float* p, int nv) {
  if (nv >= V) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const RsVec<16, 4> r = reinterpret_cast<const RsVec<16, 4>*>(p)[q];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * q + i] = __uint_as_float(r.w[i]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = j < nv ? p[j] : 0.f;
  }
}
template <int V>
__device__ __forceinline__ void store_f(float* p, const float* x, int nv) {
  if (nv >= V) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      RsVec<16, 4> r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = __float_as_uint(x[4 * q + i]);
      reinterpret_cast<RsVec<16, 4>*>(p)[q] = r;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < nv) p[j] = x[j];
  }
}

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
// The codes of V elements of one block, as bytes.  Adding 1.5 * 2^23 leaves the whole number in the
// sum's low bits.
template <int V>
__device__ __forceinline__ void pack8_codes(const float* x, float s, float inv, uint32_t* out) {
  const float magic = 12582912.0f, half = s > 0.f ? 0.5f * s : __builtin_inff();
  uint32_t t[V];
  float far = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float m = fmaf(x[j], inv, magic);
    t[j] = __float_as_uint(m);
    far = fmaxf(far, fabsf(fmaf(magic - m, s, x[j])));
  }
  if (far >= half) {  // an element is one step further, or a tie
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float r = fmaf(magic - __uint_as_float(t[j]), s, x[j]);
      const bool odd = t[j] & 1;
      if (r > half || (r == half && odd)) t[j] += 1;
      else if (r < -half || (r == -half && odd)) t[j] -= 1;
    }
  }
#pragma unroll
  for (int j = 0; j < V; j += 4)  // the low bytes of four words
    out[j / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[j + 3], t[j + 2], 0x0C0C0400u),
                                       __builtin_amdgcn_perm(t[j + 1], t[j], 0x0C0C0400u),
                                       0x05040100u);
}

// V codes to / from memory, nv of them in range
template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, const uint32_t* w, int nv) {
  if (nv >= V) {
    RsVec<V, 1> r;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) r.w[i] = w[i];
    *reinterpret_cast<RsVec<V, 1>*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < nv) p[j] = (int8_t)(w[j / 4] >> (8 * (j % 4)));
  }
}
template <int V>
__device__ __forceinline__ void load_codes(uint32_t* w, const int8_t* p, int nv) {
  if (nv >= V) {
    const RsVec<V, 1> r = *reinterpret_cast<const RsVec<V, 1>*>(p);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) w[i] = r.w[i];
  } else {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) w[i] = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < nv) w[j / 4] |= (uint32_t)(uint8_t)p[j] << (8 * (j % 4));
  }
}
// (rounded, as rs_unpack8 gives them: not as part of an fma with what is done to them next)
template <int V>
__device__ __forceinline__ void unpack_codes(const uint32_t* w, float s, float* x) {
#pragma clang fp contract(off)
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = (float)(int8_t)(w[j / 4] >> (8 * (j % 4))) * s;
}

// The largest of W aligned lanes' words (W a power of two, at most 64), in every lane
template <int W>
__device__ __forceinline__ uint32_t group_umax(uint32_t v) {
#define RS_UMAX_DPP(CTRL) \
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false))
  if (W >= 2) RS_UMAX_DPP(0xB1);    // as in group_sum
  if (W >= 4) RS_UMAX_DPP(0x4E);
  if (W >= 8) RS_UMAX_DPP(0x141);
  if (W >= 16) RS_UMAX_DPP(0x140);
#undef RS_UMAX_DPP
#pragma unroll
  for (int o = 16; o < W; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}

// The largest magnitude of V elements (NaN if one is NaN) as a bit pattern: the order of the patterns
// is that of the numbers, with NaN above infinity
template <int V>
__device__ __forceinline__ uint32_t top_bits(const float* x) {
  float t = fabsf(x[0]);
#pragma unroll
  for (int j = 1; j < V; ++j) t = __builtin_elementwise_maximum(t, fabsf(x[j]));
  return __float_as_uint(t) & 0x7FFFFFFFu;
}
