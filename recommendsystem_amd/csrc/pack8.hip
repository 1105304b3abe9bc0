// 8-bit activation checkpoints: rs_pack8 keeps [rows, D] as one byte an element and one fp32 scale
// a block of 128 columns (the form and its rounding: elem.hpp), rs_unpack8 gives it back.
// Bound by memory.  A block's 128 columns are 16 bytes each of 128 / V lanes of a wave (fewer for
// narrow rows), whose largest magnitude is found by lane exchanges alone; a thread has several
// blocks' loads in flight.  131072 x 1024 bf16: pack 77 us at best and 90 in the
// median (5.3 and 4.5 TB/s), unpack 63 us (6.4 TB/s).
#include "elem.hpp"

namespace {
constexpr int PACK_MANY = 4;  // blocks a lane group takes at a time

// LB lanes a block.  Blocks are numbered row by row.
template <class E, int LB>
__global__ void __launch_bounds__(256) pack8_kernel(const typename E::T* __restrict__ x, int64_t ld,
                                                    int64_t nblocks, int nb, int D,
                                                    int8_t* __restrict__ codes,
                                                    float* __restrict__ scales) {
  constexpr int V = E::V, GROUPS = 256 / LB;
  const int lane = (int)threadIdx.x % LB, grp = (int)threadIdx.x / LB;
  for (int64_t base = (int64_t)blockIdx.x * GROUPS * PACK_MANY; base < nblocks;
       base += (int64_t)gridDim.x * GROUPS * PACK_MANY) {
    Raw r[PACK_MANY];
    int64_t id[PACK_MANY], row[PACK_MANY];
    int col[PACK_MANY];
#pragma unroll
    for (int k = 0; k < PACK_MANY; ++k) {
      id[k] = base + k * GROUPS + grp;
      const int64_t i = id[k] < nblocks ? id[k] : nblocks - 1;
      // (a 64-bit division is long on the GPU; most shapes do without)
      row[k] = (nblocks >> 31) == 0 ? (int64_t)((uint32_t)i / (uint32_t)nb) : i / nb;
      col[k] = (int)(i - row[k] * nb) * RS_PACK_BLOCK + lane * V;
      load16<E, true>(r[k], x + row[k] * ld + col[k], D - col[k], true, 0u);
    }
#pragma unroll
    for (int k = 0; k < PACK_MANY; ++k) {
      float v[V];
      uint32_t w[V / 4];
      E::unpack(r[k].w, v);
      const float s = pack8_scale(group_umax<LB>(top_bits<V>(v)));
      pack8_codes<V>(v, s, pack8_inverse(s), w);
      if (id[k] < nblocks) {
        store_codes<V>(codes + row[k] * D + col[k], w, D - col[k]);
        if (lane == 0) scales[id[k]] = s;
      }
    }
  }
}

// A thread takes V elements of a row at a time; pieces are numbered row by row.
template <class E>
__global__ void __launch_bounds__(256) unpack8_kernel(const int8_t* __restrict__ codes,
                                                      const float* __restrict__ scales, int64_t n,
                                                      int nch, int nb, int D,
                                                      typename E::T* __restrict__ y, int64_t ld) {
  constexpr int V = E::V;
  for (int64_t base = (int64_t)blockIdx.x * 256 * PACK_MANY; base < n;
       base += (int64_t)gridDim.x * 256 * PACK_MANY) {
    uint32_t w[PACK_MANY][V / 4];
    float s[PACK_MANY];
    int64_t id[PACK_MANY], row[PACK_MANY];
    int col[PACK_MANY];
#pragma unroll
    for (int k = 0; k < PACK_MANY; ++k) {
      id[k] = base + k * 256 + threadIdx.x;
      const int64_t i = id[k] < n ? id[k] : n - 1;
      row[k] = (n >> 31) == 0 ? (int64_t)((uint32_t)i / (uint32_t)nch) : i / nch;
      col[k] = (int)(i - row[k] * nch) * V;
      load_codes<V>(w[k], codes + row[k] * D + col[k], D - col[k]);
      s[k] = scales[row[k] * nb + col[k] / RS_PACK_BLOCK];
    }
#pragma unroll
    for (int k = 0; k < PACK_MANY; ++k) {
      float v[V];
      unpack_codes<V>(w[k], s[k], v);
      if (id[k] < n) store16<E>(y + row[k] * ld + col[k], v, D - col[k]);
    }
  }
}

template <class E, int LB>
void pack8_launch(hipStream_t s, const void* x, int64_t ld, int64_t nblocks, int nb, int D,
                  int8_t* codes, float* scales) {
  const int64_t per = 256 / LB * PACK_MANY, n = (nblocks + per - 1) / per;
  pack8_kernel<E, LB><<<(unsigned)(n < 8192 ? n : 8192), 256, 0, s>>>((const typename E::T*)x, ld,
                                                                      nblocks, nb, D, codes, scales);
}

template <class E>
int pack8(hipStream_t s, const void* x, int64_t ld, int64_t rows, int D, int8_t* codes,
          float* scales) {
  constexpr int FULL = RS_PACK_BLOCK / E::V;
  const int nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK, ch = (D + E::V - 1) / E::V;
  const int64_t n = rows * nb;
  if (ch <= 1) pack8_launch<E, 1>(s, x, ld, n, nb, D, codes, scales);
  else if (ch <= 2) pack8_launch<E, 2>(s, x, ld, n, nb, D, codes, scales);
  else if (ch <= 4) pack8_launch<E, 4>(s, x, ld, n, nb, D, codes, scales);
  else if (ch <= 8) pack8_launch<E, 8>(s, x, ld, n, nb, D, codes, scales);
  else pack8_launch<E, FULL>(s, x, ld, n, nb, D, codes, scales);
  return rs_status_after_launch();
}

template <class E>
int unpack8(hipStream_t s, const int8_t* codes, const float* scales, int64_t rows, int D, void* y,
            int64_t ld) {
  const int nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK, nch = (D + E::V - 1) / E::V;
  const int64_t n = rows * nch, g = (n + 256 * PACK_MANY - 1) / (256 * PACK_MANY);
  unpack8_kernel<E><<<(unsigned)(g < 8192 ? g : 8192), 256, 0, s>>>(codes, scales, n, nch, nb, D,
                                                                    (typename E::T*)y, ld);
  return rs_status_after_launch();
}
}  // namespace

RS_API int rs_pack8(void* stream, int dtype, const void* x, int64_t ld_x, int64_t rows, int D,
                    int8_t* codes, float* scales) {
  if (rows < 0 || D <= 0 || D > 1 << 30 || dtype < RS_F32 || dtype > RS_F16) return RS_ERR_ARG;
  if (rows == 0) return RS_OK;
  if (!x || !codes || !scales || ld_x < 0) return RS_ERR_ARG;
  return RS_DISPATCH_ELEM(dtype, pack8, rs_stream(stream), x, ld_x, rows, D, codes, scales);
}

RS_API int rs_unpack8(void* stream, int dtype, const int8_t* codes, const float* scales,
                      int64_t rows, int D, void* y, int64_t ld_y) {
  if (rows < 0 || D <= 0 || D > 1 << 30 || dtype < RS_F32 || dtype > RS_F16) return RS_ERR_ARG;
  if (rows == 0) return RS_OK;
  if (!codes || !scales || !y || ld_y < D) return RS_ERR_ARG;
  return RS_DISPATCH_ELEM(dtype, unpack8, rs_stream(stream), codes, scales, rows, D, y, ld_y);
}
