// 8-bit activation checkpoints: rs_pack8 keeps [rows, D] as one byte an element and one fp32 scale
// a block of 128 columns (the form and its rounding: elem.hpp), rs_unpack8 gives it back.
#include "elem.hpp"

template <class E>
__global__ void __launch_bounds__(64) pack8_kernel(const typename E::T* __restrict__ x, int64_t ld,
                                                   int64_t nblocks, int nb, int D,
                                                   int8_t* __restrict__ codes,
                                                   float* __restrict__ scales) {
  for (int64_t id = blockIdx.x; id < nblocks; id += gridDim.x) {
    const int64_t row = id / nb;
    const int c = (int)(id % nb) * RS_PACK_BLOCK + (int)threadIdx.x;
    const float a = c < D ? E::load(x[row * ld + c]) : 0.f;
    const float b = c + 64 < D ? E::load(x[row * ld + c + 64]) : 0.f;
    // magnitudes as bit patterns: their order is that of the numbers, with NaN above infinity
    uint32_t top = max(__float_as_uint(a) & 0x7FFFFFFFu, __float_as_uint(b) & 0x7FFFFFFFu);
    for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    const float s = pack8_scale(top), inv = pack8_inverse(s);
    if (threadIdx.x == 0) scales[id] = s;
    if (c < D) codes[row * D + c] = (int8_t)pack8_code(a, s, inv);
    if (c + 64 < D) codes[row * D + c + 64] = (int8_t)pack8_code(b, s, inv);
  }
}

template <class E>
__global__ void __launch_bounds__(256) unpack8_kernel(const int8_t* __restrict__ codes,
                                                      const float* __restrict__ scales, int64_t n,
                                                      int nb, int D, typename E::T* __restrict__ y,
                                                      int64_t ld) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / D;
    const int c = (int)(i % D);
    y[row * ld + c] = E::store((float)codes[i] * scales[row * nb + c / RS_PACK_BLOCK]);
  }
}

template <class E>
static int pack8(hipStream_t s, const void* x, int64_t ld, int64_t rows, int D, int8_t* codes,
                 float* scales) {
  const int nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  const int64_t n = rows * nb;
  pack8_kernel<E><<<(unsigned)(n < 65536 ? n : 65536), 64, 0, s>>>((const typename E::T*)x, ld, n,
                                                                   nb, D, codes, scales);
  return rs_status_after_launch();
}

template <class E>
static int unpack8(hipStream_t s, const int8_t* codes, const float* scales, int64_t rows, int D,
                   void* y, int64_t ld) {
  const int nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  const int64_t n = rows * D, g = (n + 255) / 256;
  unpack8_kernel<E><<<(unsigned)(g < 65536 ? g : 65536), 256, 0, s>>>(
      codes, scales, n, nb, D, (typename E::T*)y, ld);
  return rs_status_after_launch();
}

RS_API int rs_pack8(void* stream, int dtype, const void* x, int64_t ld_x, int64_t rows, int D,
                    int8_t* codes, float* scales) {
  if (rows < 0 || D <= 0 || dtype < RS_F32 || dtype > RS_F16) return RS_ERR_ARG;
  if (rows == 0) return RS_OK;
  if (!x || !codes || !scales || ld_x < 0) return RS_ERR_ARG;
  return RS_DISPATCH_ELEM(dtype, pack8, rs_stream(stream), x, ld_x, rows, D, codes, scales);
}

RS_API int rs_unpack8(void* stream, int dtype, const int8_t* codes, const float* scales,
                      int64_t rows, int D, void* y, int64_t ld_y) {
  if (rows < 0 || D <= 0 || dtype < RS_F32 || dtype > RS_F16) return RS_ERR_ARG;
  if (rows == 0) return RS_OK;
  if (!codes || !scales || !y || ld_y < D) return RS_ERR_ARG;
  return RS_DISPATCH_ELEM(dtype, unpack8, rs_stream(stream), codes, scales, rows, D, y, ld_y);
}
