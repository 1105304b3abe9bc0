// Layer normalisation of [rows, D] and its gradients.
//   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), xh = (x - mean) rstd
//   y = xh gamma + beta
//   w = dy gamma;  dx = rstd (w - mean(w) - xh mean(w xh));  dgamma = sum_rows dy xh;  dbeta = sum_rows dy
// All sums are held in fp32.  The mean is corrected by the mean of x - mean (which subtracts
// without error when the row's spread is small against its offset), in both passes, so a row with
// a large offset loses nothing to the rounding of its own mean.
#include "elem.hpp"

#define LN_MAX_D 32768

namespace {
// the sum of v[0..N) over the block, in every thread
template <int N, int THREADS>
__device__ __forceinline__ void block_sum(float* v) {
  __shared__ float red[N][THREADS / 64];
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = group_sum<64>(v[k]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
    for (int k = 0; k < N; ++k) red[k][threadIdx.x >> 6] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = 0.f;
    for (int w = 0; w < THREADS / 64; ++w) v[k] += red[k][w];
  }
}
}  // namespace

template <class E>
__global__ void __launch_bounds__(256) ln_fwd_kernel(
    const typename E::T* __restrict__ x, int64_t ldx, int64_t rows, int D,
    const float* __restrict__ gamma, const float* __restrict__ beta, float eps,
    typename E::T* __restrict__ y, int64_t ldy, float* __restrict__ mean, float* __restrict__ rstd,
    int8_t* __restrict__ codes, float* __restrict__ scales) {
  const int nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const typename E::T* xr = x + r * ldx;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < D; c += 256) s[0] += E::load(xr[c]);
    block_sum<1, 256>(s);
    const float m0 = s[0] / (float)D;
    float q[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += 256) {
      const float d = E::load(xr[c]) - m0;
      q[0] += d;
      q[1] += d * d;
    }
    block_sum<2, 256>(q);
    const float dl = q[0] / (float)D, var = fmaxf(q[1] / (float)D - dl * dl, 0.f);
    // (fmaxf would turn a NaN row's variance into 0)
    const float rs = 1.0f / sqrtf((q[1] != q[1] ? q[1] : var) + eps);
    for (int c = threadIdx.x; c < D; c += 256)
      y[r * ldy + c] = E::store((E::load(xr[c]) - m0 - dl) * rs * gamma[c] + beta[c]);
    if (threadIdx.x == 0 && mean) {
      mean[r] = m0 + dl;
      rstd[r] = rs;
    }
    if (codes) {
      for (int b = threadIdx.x >> 6; b < nb; b += 4) {
        const int c = b * RS_PACK_BLOCK + (int)(threadIdx.x & 63);
        const float a0 = c < D ? E::load(xr[c]) : 0.f, a1 = c + 64 < D ? E::load(xr[c + 64]) : 0.f;
        uint32_t top = max(__float_as_uint(a0) & 0x7FFFFFFFu, __float_as_uint(a1) & 0x7FFFFFFFu);
        for (int o = 32; o; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        const float sc = pack8_scale(top), inv = pack8_inverse(sc);
        if ((threadIdx.x & 63) == 0) scales[r * nb + b] = sc;
        if (c < D) codes[r * D + c] = (int8_t)pack8_code(a0, sc, inv);
        if (c + 64 < D) codes[r * D + c + 64] = (int8_t)pack8_code(a1, sc, inv);
      }
    }
  }
}

// Q8: x is read from its 8-bit form; the mean is then that of the exact row and not corrected
template <class E, bool Q8>
__device__ __forceinline__ float ln_in(const typename E::T* x, int64_t ldx, const int8_t* codes,
                                       const float* scales, int nb, int64_t r, int c, int D) {
  return Q8 ? (float)codes[r * D + c] * scales[r * nb + c / RS_PACK_BLOCK] : E::load(x[r * ldx + c]);
}

template <class E, bool Q8>
__global__ void __launch_bounds__(256) ln_bwd_dx_kernel(
    const typename E::T* __restrict__ dy, int64_t lddy, const typename E::T* __restrict__ x,
    int64_t ldx, const int8_t* __restrict__ codes, const float* __restrict__ scales, int64_t rows,
    int D, const float* __restrict__ gamma, const float* __restrict__ mean,
    const float* __restrict__ rstd, typename E::T* __restrict__ dx, int64_t lddx,
    float* __restrict__ delta) {
  const int nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float m = mean[r], rs = rstd[r];
    float s[3] = {0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += 256) {
      const float w = E::load(dy[r * lddy + c]) * gamma[c];
      const float d = ln_in<E, Q8>(x, ldx, codes, scales, nb, r, c, D) - m;
      s[0] += w;
      s[1] += w * d;
      s[2] += d;
    }
    block_sum<3, 256>(s);
    const float dl = Q8 ? 0.f : s[2] / (float)D;
    const float c1 = s[0] / (float)D, c2 = (s[1] / (float)D - dl * c1) * rs * rs;
    for (int c = threadIdx.x; c < D; c += 256) {
      const float w = E::load(dy[r * lddy + c]) * gamma[c];
      const float d = ln_in<E, Q8>(x, ldx, codes, scales, nb, r, c, D) - m - dl;
      dx[r * lddx + c] = E::store(rs * (w - c1 - d * c2));
    }
    if (threadIdx.x == 0) delta[r] = m + dl;
  }
}

template <class E, bool Q8>
__global__ void __launch_bounds__(256) ln_bwd_params_kernel(
    const typename E::T* __restrict__ dy, int64_t lddy, const typename E::T* __restrict__ x,
    int64_t ldx, const int8_t* __restrict__ codes, const float* __restrict__ scales, int64_t rows,
    int D, const float* __restrict__ mean, const float* __restrict__ rstd,
    float* __restrict__ dgamma, float* __restrict__ dbeta, int accumulate) {
  const int nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  const int c = (int)blockIdx.x * 4 + (int)(threadIdx.x & 3);
  float s[2] = {0.f, 0.f};
  if (c < D)
    for (int64_t r = threadIdx.x >> 2; r < rows; r += 64) {
      const float g = E::load(dy[r * lddy + c]);
      s[0] += g * (ln_in<E, Q8>(x, ldx, codes, scales, nb, r, c, D) - mean[r]) * rstd[r];
      s[1] += g;
    }
  __shared__ float red[2][256];
  red[0][threadIdx.x] = s[0];
  red[1][threadIdx.x] = s[1];
  for (int o = 128; o >= 4; o >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < o) {
      red[0][threadIdx.x] += red[0][threadIdx.x + o];
      red[1][threadIdx.x] += red[1][threadIdx.x + o];
    }
  }
  if (threadIdx.x < 4 && c < D) {
    dgamma[c] = red[0][threadIdx.x] + (accumulate ? dgamma[c] : 0.f);
    dbeta[c] = red[1][threadIdx.x] + (accumulate ? dbeta[c] : 0.f);
  }
}

template <class E>
static int ln_fwd(hipStream_t s, const void* x, int64_t ldx, int64_t rows, int D,
                  const float* gamma, const float* beta, float eps, void* y, int64_t ldy,
                  float* mean, float* rstd, int8_t* codes, float* scales) {
  ln_fwd_kernel<E><<<(unsigned)(rows < 65536 ? rows : 65536), 256, 0, s>>>(
      (const typename E::T*)x, ldx, rows, D, gamma, beta, eps, (typename E::T*)y, ldy, mean, rstd,
      codes, scales);
  return rs_status_after_launch();
}

template <class E>
static int ln_bwd(hipStream_t s, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                  const int8_t* codes, const float* scales, int64_t rows, int D, const float* gamma,
                  const float* mean, const float* rstd, void* dx, int64_t lddx, float* dgamma,
                  float* dbeta, int accumulate, float* ws) {
  typedef typename E::T T;
  const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536), cols = (unsigned)((D + 3) / 4);
  const T *dyt = (const T*)dy, *xt = (const T*)x;
  if (codes) {
    if (rows) ln_bwd_dx_kernel<E, true><<<grid, 256, 0, s>>>(dyt, lddy, xt, ldx, codes, scales, rows, D,
                                                   gamma, mean, rstd, (T*)dx, lddx, ws);
    ln_bwd_params_kernel<E, true><<<cols, 256, 0, s>>>(dyt, lddy, xt, ldx, codes, scales, rows, D, ws,
                                                       rstd, dgamma, dbeta, accumulate);
  } else {
    if (rows) ln_bwd_dx_kernel<E, false><<<grid, 256, 0, s>>>(dyt, lddy, xt, ldx, codes, scales, rows, D,
                                                    gamma, mean, rstd, (T*)dx, lddx, ws);
    ln_bwd_params_kernel<E, false><<<cols, 256, 0, s>>>(dyt, lddy, xt, ldx, codes, scales, rows, D,
                                                        ws, rstd, dgamma, dbeta, accumulate);
  }
  return rs_status_after_launch();
}

RS_API int rs_layernorm_fwd(void* stream, int dtype, const void* x, int64_t ld_x, int64_t rows,
                            int D, const float* gamma, const float* beta, float eps, void* y,
                            int64_t ld_y, float* mean, float* rstd, int8_t* codes, float* scales) {
  if (rows < 0 || D <= 0 || dtype < RS_F32 || dtype > RS_F16 || !(eps > 0.f)) return RS_ERR_ARG;
  if (D > LN_MAX_D) return RS_ERR_UNSUPPORTED;
  if (rows == 0) return RS_OK;
  if (!x || !gamma || !beta || !y || ld_x < 0 || ld_y < D || !mean != !rstd || !codes != !scales)
    return RS_ERR_ARG;
  return RS_DISPATCH_ELEM(dtype, ln_fwd, rs_stream(stream), x, ld_x, rows, D, gamma, beta, eps, y,
                          ld_y, mean, rstd, codes, scales);
}

RS_API int64_t rs_layernorm_bwd_workspace_floats(int64_t rows, int D) {
  if (rows < 0 || D <= 0 || D > LN_MAX_D) return 0;
  return rows;
}

RS_API int rs_layernorm_bwd(void* stream, int dtype, const void* dy, int64_t ld_dy, const void* x,
                            int64_t ld_x, const int8_t* codes, const float* scales, int64_t rows,
                            int D, const float* gamma, const float* mean, const float* rstd,
                            void* dx, int64_t ld_dx, float* dgamma, float* dbeta, int accumulate,
                            float* workspace, int64_t workspace_floats) {
  if (rows < 0 || D <= 0 || dtype < RS_F32 || dtype > RS_F16) return RS_ERR_ARG;
  if (D > LN_MAX_D) return RS_ERR_UNSUPPORTED;
  if (!dgamma || !dbeta) return RS_ERR_ARG;
  if (rows > 0 && (!dy || !gamma || !mean || !rstd || !dx || ld_dy < 0 || ld_x < 0 || ld_dx < D ||
                   !x == !codes || !codes != !scales || !workspace ||
                   workspace_floats < rs_layernorm_bwd_workspace_floats(rows, D)))
    return RS_ERR_ARG;
  return RS_DISPATCH_ELEM(dtype, ln_bwd, rs_stream(stream), dy, ld_dy, x, ld_x, codes, scales, rows,
                          D, gamma, mean, rstd, dx, ld_dx, dgamma, dbeta, accumulate, workspace);
}
