// Layer normalisation of [rows, D] and its gradients.
//   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), xh = (x - mean) rstd
//   y = xh gamma + beta
//   w = dy gamma;  dx = rstd (w - mean(w) - xh mean(w xh));  dgamma = sum_rows dy xh;  dbeta = sum_rows dy
// All sums are held in fp32.  The mean is corrected by the mean of x - mean (which subtracts
// without error when the row's spread is small against its offset), in both passes, so a row with
// a large offset loses nothing to the rounding of its own mean.
//
// Bound by memory.  A row lives in the registers of TPR threads (4 .. 64 lanes of a wave, or a
// workgroup of 256 or 512), NCH x 16 bytes each, so it is read once; workgroups stay and walk the
// rows, with gamma and beta in registers and the next row's loads in flight.  In the backward every
// thread also keeps its columns' share of dgamma and dbeta in registers over all of its rows; one
// partial row a workgroup then goes to the workspace and a second launch adds them in a fixed order.
#include "elem.hpp"

#define LN_MAX_D 32768
#define LN_REG_D 16384  // rows up to here fit the registers of one workgroup

namespace {

struct LnArgs {
  const void *x, *dy;
  int64_t ldx, lddy, rows;
  int D, accumulate;
  const float *gamma, *beta;
  float eps;
  void *y, *dx;
  int64_t ldy, lddx;
  float *mean, *rstd;
  int8_t* codes;
  float* scales;
  float *dgamma, *dbeta, *ws;
};

// sums of v[0..N) over the TPR threads of a row, in each of them.  red: [2][N][waves], used in turn
// (flip), so one barrier a call is enough.
template <int N, int TPR>
__device__ __forceinline__ void row_sum(float* v, float* red, int& flip) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = group_sum<(TPR < 64 ? TPR : 64)>(v[k]);
  if (TPR > 64) {
    constexpr int W = TPR / 64;
    float* r = red + flip * N * W;
    flip ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) r[k * W + (threadIdx.x >> 6)] = v[k];
    }
    lds_barrier();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[k] += r[k * W + w];
    }
  }
}

template <int TPR>
struct LnShape {
  static constexpr int THREADS = TPR < 256 ? 256 : TPR;
  static constexpr int RPB = THREADS / TPR;  // rows a workgroup holds at a time
};

}  // namespace

template <class E, int TPR, int NCH, bool PACK>
__global__ void __launch_bounds__(LnShape<TPR>::THREADS) ln_fwd_kernel(const LnArgs a) {
  constexpr int V = E::V, RPB = LnShape<TPR>::RPB;
  constexpr int LB = RS_PACK_BLOCK / V < TPR ? RS_PACK_BLOCK / V : TPR;  // lanes of an 8-bit block
  typedef typename E::T X;
  __shared__ float red[2 * 2 * (TPR + 63) / 64];
  const int tr = (int)threadIdx.x % TPR, nb = (a.D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  const float inv = 1.0f / (float)a.D;
  int flip = 0;
  float gm[NCH][V], bt[NCH][V];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * TPR + tr) * V;
    load_f<V>(gm[c], a.gamma + col, a.D - col);
    load_f<V>(bt[c], a.beta + col, a.D - col);
  }
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + (int)threadIdx.x / TPR;
  Raw next[NCH];
  auto load = [&](int64_t r) {  // (behind the last row: the last row again, and not stored)
    const X* p = (const X*)a.x + (r < a.rows ? r : a.rows - 1) * a.ldx;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + tr) * V;
      load16<E, true>(next[c], p + col, a.D - col, true, 0u);
    }
  };
  load(row);
  // every thread of the workgroup runs the same number of rounds
  for (int64_t first = (int64_t)blockIdx.x * RPB; first < a.rows; first += step, row += step) {
    float x[NCH][V];
#pragma unroll
    for (int c = 0; c < NCH; ++c) E::unpack(next[c].w, x[c]);
    if (first + step < a.rows) load(row + step);
    float s[1] = {0.f}, q[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += x[c][j];
    row_sum<1, TPR>(s, red, flip);
    const float m0 = s[0] * inv;
    const bool live = row < a.rows;
    if (PACK) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int col = (c * TPR + tr) * V, nv = a.D - col;
        const float sc = pack8_scale(group_umax<LB>(top_bits<V>(x[c])));
        uint32_t w[V / 4];
        pack8_codes<V>(x[c], sc, pack8_inverse(sc), w);
        if (live) {
          store_codes<V>(a.codes + row * a.D + col, w, nv);
          if (tr % LB == 0 && nv > 0) a.scales[row * nb + col / RS_PACK_BLOCK] = sc;
        }
      }
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int nv = a.D - (c * TPR + tr) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[c][j] = j < nv ? x[c][j] - m0 : 0.f;
        q[0] += x[c][j];
        q[1] = fmaf(x[c][j], x[c][j], q[1]);
      }
    }
    row_sum<2, TPR>(q, red, flip);
    const float dl = q[0] * inv, var = q[1] * inv - dl * dl;
    // (not fmaxf: it would make a NaN row's variance 0)
    const float rs = 1.0f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
    if (live) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int col = (c * TPR + tr) * V;
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = fmaf((x[c][j] - dl) * rs, gm[c][j], bt[c][j]);
        if (col < a.D) store16<E>((X*)a.y + row * a.ldy + col, y, a.D - col);
      }
      if (tr == 0 && a.mean) {
        a.mean[row] = m0 + dl;
        a.rstd[row] = rs;
      }
    }
  }
}

// Q8: x is read from its 8-bit form; the mean is then that of the exact row and not corrected
template <class E, int TPR, int NCH, bool Q8>
__global__ void __launch_bounds__(LnShape<TPR>::THREADS) ln_bwd_kernel(const LnArgs a) {
  constexpr int V = E::V, RPB = LnShape<TPR>::RPB, THREADS = LnShape<TPR>::THREADS;
  typedef typename E::T X;
  __shared__ float red[2 * 3 * (TPR + 63) / 64];
  __shared__ float fold[RPB > 1 ? THREADS * V : 1];
  const int tr = (int)threadIdx.x % TPR, nb = (a.D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  const float inv = 1.0f / (float)a.D;
  int flip = 0;
  float gm[NCH][V], ag[NCH][V], ab[NCH][V];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int col = (c * TPR + tr) * V;
    load_f<V>(gm[c], a.gamma + col, a.D - col);
#pragma unroll
    for (int j = 0; j < V; ++j) ag[c][j] = ab[c][j] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + (int)threadIdx.x / TPR;
  Raw nx[Q8 ? 1 : NCH], ny[NCH];
  uint32_t nq[Q8 ? NCH : 1][V / 4];
  float nsc[Q8 ? NCH : 1], nmean, nrs;
  auto load = [&](int64_t r) {  // (behind the last row: the last row again, with dy = 0)
    const bool in = r < a.rows;
    if (!in) r = a.rows - 1;
    const X *px = (const X*)a.x + r * a.ldx, *py = (const X*)a.dy + r * a.lddy;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + tr) * V, nv = a.D - col;
      load16<E, true>(ny[c], py + col, nv, in, 0u);
      if (Q8) {
        load_codes<V>(nq[c], a.codes + r * a.D + col, nv);
        nsc[c] = nv > 0 ? a.scales[r * nb + col / RS_PACK_BLOCK] : 0.f;
      } else {
        load16<E, true>(nx[c], px + col, nv, true, 0u);
      }
    }
    nmean = a.mean[r];
    nrs = a.rstd[r];
  };
  load(row);
  for (int64_t first = (int64_t)blockIdx.x * RPB; first < a.rows; first += step, row += step) {
    float x[NCH][V], y[NCH][V], s[3] = {0.f, 0.f, 0.f};
    const float mean = nmean, rs = nrs;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (Q8) unpack_codes<V>(nq[c], nsc[c], x[c]);
      else E::unpack(nx[c].w, x[c]);
      E::unpack(ny[c].w, y[c]);
    }
    if (first + step < a.rows) load(row + step);
    const bool live = row < a.rows;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int nv = a.D - (c * TPR + tr) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float w = y[c][j] * gm[c][j];
        x[c][j] = j < nv ? x[c][j] - mean : 0.f;
        s[0] += w;
        s[1] = fmaf(w, x[c][j], s[1]);
        if (!Q8) s[2] += x[c][j];
      }
    }
    row_sum<(Q8 ? 2 : 3), TPR>(s, red, flip);
    const float dl = Q8 ? 0.f : s[2] * inv;
    const float c1 = s[0] * inv, c2 = (s[1] * inv - dl * c1) * rs * rs;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + tr) * V;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = x[c][j] - dl;
        o[j] = rs * (fmaf(y[c][j], gm[c][j], -c1) - d * c2);
        if (live) {  // (the last row again must not add its NaN to another's zeros)
          ag[c][j] = fmaf(y[c][j], d * rs, ag[c][j]);
          ab[c][j] += y[c][j];
        }
      }
      if (live && col < a.D) store16<E>((X*)a.dx + row * a.lddx + col, o, a.D - col);
    }
  }
  // this workgroup's partial row [dgamma | dbeta]
  float* part = a.ws + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + tr) * V;
      float* v = k ? ab[c] : ag[c];
      if (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) fold[j * THREADS + threadIdx.x] = v[j];
        __syncthreads();
        if ((int)threadIdx.x < TPR) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            v[j] = 0.f;
            for (int r = 0; r < RPB; ++r) v[j] += fold[j * THREADS + r * TPR + tr];
          }
        }
      }
      if ((int)threadIdx.x < TPR && col < a.D) store_f<V>(part + (k ? a.D : 0) + col, v, a.D - col);
    }
}

// Sums of the n partial rows: 32 columns x 32 groups of rows a workgroup
__global__ void __launch_bounds__(1024) ln_params_kernel(const float* __restrict__ part, int n,
                                                         int D, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta,
                                                         int accumulate) {
  __shared__ float red[32][33];
  const int lc = (int)threadIdx.x & 31, g = (int)threadIdx.x >> 5;
  const int c = (int)blockIdx.x * 32 + lc;
  float s = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int r = g; r < n; r += 32) s += part[(int64_t)r * 2 * D + c];
  }
  red[g][lc] = s;
  __syncthreads();
  if (g == 0 && c < 2 * D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][lc];
    float* d = c < D ? dgamma + c : dbeta + (c - D);
    *d = accumulate ? *d + t : t;
  }
}

// ---------------------------------------------------------------------------------------------
// Rows beyond LN_REG_D: one workgroup a row, which it reads three times (from cache after the first)
// ---------------------------------------------------------------------------------------------
template <class E>
__global__ void __launch_bounds__(256) ln_wide_fwd_kernel(const LnArgs a) {
  typedef typename E::T X;
  __shared__ float red[2 * 2 * 4];
  int flip = 0;
  const int D = a.D, nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const X* xr = (const X*)a.x + r * a.ldx;
    float s[1] = {0.f}, q[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += 256) s[0] += E::load(xr[c]);
    row_sum<1, 256>(s, red, flip);
    const float m0 = s[0] / (float)D;
    for (int c = threadIdx.x; c < D; c += 256) {
      const float d = E::load(xr[c]) - m0;
      q[0] += d;
      q[1] = fmaf(d, d, q[1]);
    }
    row_sum<2, 256>(q, red, flip);
    const float dl = q[0] / (float)D, var = q[1] / (float)D - dl * dl;
    const float rs = 1.0f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
    for (int c = threadIdx.x; c < D; c += 256)
      ((X*)a.y)[r * a.ldy + c] = E::store(fmaf((E::load(xr[c]) - m0 - dl) * rs, a.gamma[c], a.beta[c]));
    if (threadIdx.x == 0 && a.mean) {
      a.mean[r] = m0 + dl;
      a.rstd[r] = rs;
    }
    if (a.codes) {  // 32 lanes x 4 elements a block
      for (int b = (int)threadIdx.x >> 5; b < nb; b += 8) {
        const int c = b * RS_PACK_BLOCK + ((int)threadIdx.x & 31) * 4;
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = c + j < D ? E::load(xr[c + j]) : 0.f;
        const float sc = pack8_scale(group_umax<32>(top_bits<4>(x)));
        uint32_t w[1];
        pack8_codes<4>(x, sc, pack8_inverse(sc), w);
        store_codes<4>(a.codes + r * D + c, w, D - c);
        if ((threadIdx.x & 31) == 0) a.scales[r * nb + b] = sc;
      }
    }
  }
}

template <class E, bool Q8>
__device__ __forceinline__ float ln_in(const LnArgs& a, int nb, int64_t r, int c) {
  return Q8 ? (float)a.codes[r * a.D + c] * a.scales[r * nb + c / RS_PACK_BLOCK]
            : E::load(((const typename E::T*)a.x)[r * a.ldx + c]);
}

// dx of a row, and its corrected mean into ws
template <class E, bool Q8>
__global__ void __launch_bounds__(256) ln_wide_bwd_kernel(const LnArgs a) {
  typedef typename E::T X;
  __shared__ float red[2 * 3 * 4];
  int flip = 0;
  const int D = a.D, nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const X* dy = (const X*)a.dy + r * a.lddy;
    const float m = a.mean[r], rs = a.rstd[r];
    float s[3] = {0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += 256) {
      const float w = E::load(dy[c]) * a.gamma[c], d = ln_in<E, Q8>(a, nb, r, c) - m;
      s[0] += w;
      s[1] = fmaf(w, d, s[1]);
      s[2] += d;
    }
    row_sum<3, 256>(s, red, flip);
    const float dl = Q8 ? 0.f : s[2] / (float)D;
    const float c1 = s[0] / (float)D, c2 = (s[1] / (float)D - dl * c1) * rs * rs;
    for (int c = threadIdx.x; c < D; c += 256) {
      const float d = ln_in<E, Q8>(a, nb, r, c) - m - dl;
      ((X*)a.dx)[r * a.lddx + c] = E::store(rs * (fmaf(E::load(dy[c]), a.gamma[c], -c1) - d * c2));
    }
    if (threadIdx.x == 0) a.ws[r] = m + dl;
  }
}

// dgamma and dbeta of 4 columns
template <class E, bool Q8>
__global__ void __launch_bounds__(256) ln_wide_params_kernel(const LnArgs a) {
  const int nb = (a.D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  const int c = (int)blockIdx.x * 4 + (int)(threadIdx.x & 3);
  float s[2] = {0.f, 0.f};
  if (c < a.D)
    for (int64_t r = threadIdx.x >> 2; r < a.rows; r += 64) {
      const float g = E::load(((const typename E::T*)a.dy)[r * a.lddy + c]);
      s[0] = fmaf(g, (ln_in<E, Q8>(a, nb, r, c) - a.ws[r]) * a.rstd[r], s[0]);
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
  if (threadIdx.x < 4 && c < a.D) {
    a.dgamma[c] = red[0][threadIdx.x] + (a.accumulate ? a.dgamma[c] : 0.f);
    a.dbeta[c] = red[1][threadIdx.x] + (a.accumulate ? a.dbeta[c] : 0.f);
  }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
namespace {

// threads of a row
int ln_tpr(int D, int V) {
  const int ch = (D + V - 1) / V;  // 16-byte pieces; at most 4 a thread (fp32 rows over 8192: 8)
  return ch <= 4 ? 4 : ch <= 8 ? 8 : ch <= 16 ? 16 : ch <= 32 ? 32 : ch <= 256 ? 64 : ch <= 1024 ? 256 : 512;
}

int64_t ln_grid(int64_t rows, int tpr, int64_t most) {
  const int64_t rpb = tpr < 256 ? 256 / tpr : 1, n = (rows + rpb - 1) / rpb;
  return n < most ? n : most;
}

// workgroups of the backward: two a compute unit, which is what its registers allow
int64_t ln_bwd_grid(int64_t rows, int D, int V) { return ln_grid(rows, ln_tpr(D, V), 512); }

// KERNEL<E, TPR, NCH, FLAG> for the width
#define LN_LAUNCH(KERNEL, FLAG)                                                                \
  do {                                                                                         \
    const int ch = (a.D + E::V - 1) / E::V, tpr = ln_tpr(a.D, E::V);                           \
    if (tpr == 4) KERNEL<E, 4, 1, FLAG><<<grid, 256, 0, s>>>(a);                               \
    else if (tpr == 8) KERNEL<E, 8, 1, FLAG><<<grid, 256, 0, s>>>(a);                          \
    else if (tpr == 16) KERNEL<E, 16, 1, FLAG><<<grid, 256, 0, s>>>(a);                        \
    else if (tpr == 32) KERNEL<E, 32, 1, FLAG><<<grid, 256, 0, s>>>(a);                        \
    else if (tpr == 64 && ch <= 64) KERNEL<E, 64, 1, FLAG><<<grid, 256, 0, s>>>(a);            \
    else if (tpr == 64 && ch <= 128) KERNEL<E, 64, 2, FLAG><<<grid, 256, 0, s>>>(a);           \
    else if (tpr == 64) KERNEL<E, 64, 4, FLAG><<<grid, 256, 0, s>>>(a);                        \
    else if (tpr == 256 && ch <= 512) KERNEL<E, 256, 2, FLAG><<<grid, 256, 0, s>>>(a);         \
    else if (tpr == 256) KERNEL<E, 256, 4, FLAG><<<grid, 256, 0, s>>>(a);                      \
    else if (ch <= 2048) KERNEL<E, 512, 4, FLAG><<<grid, 512, 0, s>>>(a);                      \
    else KERNEL<E, 512, E::V == 4 ? 8 : 4, FLAG><<<grid, 512, 0, s>>>(a);                      \
  } while (0)

template <class E>
int ln_fwd(hipStream_t s, const LnArgs& a) {
  if (a.D > LN_REG_D) {
    ln_wide_fwd_kernel<E><<<(unsigned)(a.rows < 65536 ? a.rows : 65536), 256, 0, s>>>(a);
    return rs_status_after_launch();
  }
  const unsigned grid = (unsigned)ln_grid(a.rows, ln_tpr(a.D, E::V), 2048);
  if (a.codes) LN_LAUNCH(ln_fwd_kernel, true);
  else LN_LAUNCH(ln_fwd_kernel, false);
  return rs_status_after_launch();
}

template <class E>
int ln_bwd(hipStream_t s, const LnArgs& a) {
  if (a.D > LN_REG_D) {
    const unsigned grid = (unsigned)(a.rows < 65536 ? a.rows : 65536), cols = (unsigned)((a.D + 3) / 4);
    if (a.codes) {
      if (a.rows) ln_wide_bwd_kernel<E, true><<<grid, 256, 0, s>>>(a);
      ln_wide_params_kernel<E, true><<<cols, 256, 0, s>>>(a);
    } else {
      if (a.rows) ln_wide_bwd_kernel<E, false><<<grid, 256, 0, s>>>(a);
      ln_wide_params_kernel<E, false><<<cols, 256, 0, s>>>(a);
    }
    return rs_status_after_launch();
  }
  const unsigned grid = (unsigned)ln_bwd_grid(a.rows, a.D, E::V);
  if (grid) {
    if (a.codes) LN_LAUNCH(ln_bwd_kernel, true);
    else LN_LAUNCH(ln_bwd_kernel, false);
  }
  ln_params_kernel<<<(unsigned)((2 * a.D + 31) / 32), 1024, 0, s>>>(a.ws, (int)grid, a.D, a.dgamma,
                                                                    a.dbeta, a.accumulate);
  return rs_status_after_launch();
}

}  // namespace

RS_API int rs_layernorm_fwd(void* stream, int dtype, const void* x, int64_t ld_x, int64_t rows,
                            int D, const float* gamma, const float* beta, float eps, void* y,
                            int64_t ld_y, float* mean, float* rstd, int8_t* codes, float* scales) {
  if (rows < 0 || D <= 0 || dtype < RS_F32 || dtype > RS_F16 || !(eps > 0.f)) return RS_ERR_ARG;
  if (D > LN_MAX_D) return RS_ERR_UNSUPPORTED;
  if (rows == 0) return RS_OK;
  if (!x || !gamma || !beta || !y || ld_x < 0 || ld_y < D || !mean != !rstd || !codes != !scales)
    return RS_ERR_ARG;
  LnArgs a = {};
  a.x = x, a.ldx = ld_x, a.rows = rows, a.D = D, a.gamma = gamma, a.beta = beta, a.eps = eps;
  a.y = y, a.ldy = ld_y, a.mean = mean, a.rstd = rstd, a.codes = codes, a.scales = scales;
  return RS_DISPATCH_ELEM(dtype, ln_fwd, rs_stream(stream), a);
}

// the partial rows of whichever type needs more
RS_API int64_t rs_layernorm_bwd_workspace_floats(int64_t rows, int D) {
  if (rows < 0 || D <= 0 || D > LN_MAX_D) return 0;
  if (D > LN_REG_D) return rows;
  const int64_t g4 = ln_bwd_grid(rows, D, 4), g8 = ln_bwd_grid(rows, D, 8);
  return (g4 > g8 ? g4 : g8) * 2 * D;
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
  LnArgs a = {};
  a.dy = dy, a.lddy = ld_dy, a.x = x, a.ldx = ld_x, a.rows = rows, a.D = D, a.gamma = gamma;
  a.codes = const_cast<int8_t*>(codes), a.scales = const_cast<float*>(scales);
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  a.dx = dx, a.lddx = ld_dx, a.dgamma = dgamma, a.dbeta = dbeta, a.accumulate = accumulate;
  a.ws = workspace;
  return RS_DISPATCH_ELEM(dtype, ln_bwd, rs_stream(stream), a);
}
