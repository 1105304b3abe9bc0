// Layer normalisation of [rows, D] and its gradients.
//   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), xh = (x - mean) rstd
//   y = xh gamma + beta
//   w = dy gamma;  dx = rstd (w - mean(w) - xh mean(w xh));  dgamma = sum_rows dy xh;  dbeta = sum_rows dy
// All sums are held in fp32.  The forward takes a first mean m = x[0] + mean(x - x[0]), and both
// passes correct it by the mean of x - m (both differences have no error when the row's spread is
// small against its offset), so a row with a large offset loses nothing to the rounding of its own
// mean, and a constant row is normalised to exact zeros.  x[0] serves for m alone: the differences that
// are kept are those of x itself from m, so a first column far off the others costs them no digits.
//
// Bound by memory.  A row lives in the registers of TPR threads (1 .. 64 lanes of a wave, or 2 to 8
// waves), NCH x 16 bytes each, so it is read once; workgroups stay and walk the rows, with gamma and
// beta in registers and the next row's loads in flight.  In the backward every thread also keeps its
// columns' share of dgamma and dbeta in registers over all of its rows; one partial row a workgroup
// then goes to the workspace and a second launch adds them in a fixed order.
// 65536 x 1024 bf16: forward 46 us (5.8 TB/s), backward 80 + 4 us (5.0 TB/s); a large copy of torch's
// runs at 5.4 TB/s.  Rows that start off 16 bytes cost more, each load then touching two pieces of 64
// bytes: 40000 x 1500 bf16 forward 5.5, backward 3.5 TB/s; 4099 x 5003 fp16 3.6 and 2.9 TB/s.  Rows wider
// than any shape are read two or three times: 4096 x 12000 fp32 forward 126 us (3.1 TB/s of what a pass
// moves once), backward 220 (2.7); 4096 x 32768 bf16 210 (2.6) and 361 us (2.2).
#include "elem.hpp"

#define LN_MAX_D 32768

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

template <int TPR>
struct LnShape {
  static constexpr int THREADS = TPR < 256 ? 256 : TPR;
  static constexpr int RPB = THREADS / TPR;  // rows a workgroup holds at a time
};

// dy gamma, rounded: as part of an fma it would not cancel against the mean of the rounded ones (in a
// row of one column, whose input's gradient is zero, it has to)
__device__ __forceinline__ float ln_weighted(float y, float gm) {
#pragma clang fp contract(off)
  return y * gm;
}
// The same, computed again: kept over the row's sums the products would take as many registers as
// the row (32768 x 2048 bf16 from 8 bits: 136 us, 86 so)
__device__ __forceinline__ float ln_weighted_again(float y, float gm) {
  asm("" : "+v"(y));
  return ln_weighted(y, gm);
}

// sums of v[0..N) over the TPR threads of a row, in each of them.  red: two buffers of N floats a
// wave, used in turn (flip), so one barrier a call is enough.
template <int N, int TPR>
__device__ __forceinline__ void row_sum(float* v, float* red, int& flip) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = group_sum<(TPR < 64 ? TPR : 64)>(v[k]);
  if (TPR > 64) {
    constexpr int W = TPR / 64, ALL = LnShape<TPR>::THREADS / 64;
    float* r = red + flip * N * ALL;
    const int wave = wave_id();
    flip ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) r[k * ALL + wave] = v[k];
    }
    lds_barrier();
    r += wave / W * W;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[k] += r[k * ALL + w];
    }
  }
}

}  // namespace

template <class E, int TPR, int NCH, bool PACK>
__global__ void __launch_bounds__(LnShape<TPR>::THREADS) ln_fwd_kernel(const LnArgs a) {
  constexpr int V = E::V, RPB = LnShape<TPR>::RPB;
  // an 8-bit block is 16 bytes of LB lanes, CPB times over
  constexpr int LB = RS_PACK_BLOCK / V < TPR ? RS_PACK_BLOCK / V : TPR;
  constexpr int CPB = RS_PACK_BLOCK / V / LB;
  typedef typename E::T X;
  __shared__ float red[2 * 2 * LnShape<TPR>::THREADS / 64];
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
  float next0;
  auto load = [&](int64_t r) {  // (behind the last row: the last row again, and not stored)
    const X* p = (const X*)a.x + (r < a.rows ? r : a.rows - 1) * a.ldx;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = (c * TPR + tr) * V;
      load16<E, true>(next[c], p + col, a.D - col, true, 0u);
    }
    next0 = E::load(p[0]);
  };
  load(row);
  // every thread of the workgroup runs the same number of rounds
  for (int64_t first = (int64_t)blockIdx.x * RPB; first < a.rows; first += step, row += step) {
    float x[NCH][V];
#pragma unroll
    for (int c = 0; c < NCH; ++c) E::unpack(next[c].w, x[c]);
    const float x0 = next0;
    if (first + step < a.rows) load(row + step);
    const bool live = row < a.rows;
    if (PACK) {
#pragma unroll
      for (int c0 = 0; c0 < NCH; c0 += CPB) {
        uint32_t top = 0;
#pragma unroll
        for (int c = c0; c < c0 + CPB && c < NCH; ++c) top = max(top, top_bits<V>(x[c]));
        const float sc = pack8_scale(group_umax<LB>(top)), inv8 = pack8_inverse(sc);
#pragma unroll
        for (int c = c0; c < c0 + CPB && c < NCH; ++c) {
          const int col = (c * TPR + tr) * V, nv = a.D - col;
          uint32_t w[V / 4];
          pack8_codes<V>(x[c], sc, inv8, w);
          if (live) {
            store_codes<V>(a.codes + row * a.D + col, w, nv);
            if (c == c0 && tr % LB == 0 && nv > 0) a.scales[row * nb + col / RS_PACK_BLOCK] = sc;
          }
        }
      }
    }
    float s[1] = {0.f}, q[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int nv = a.D - (c * TPR + tr) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += j < nv ? x[c][j] - x0 : 0.f;
    }
    row_sum<1, TPR>(s, red, flip);
    const float m = fmaf(s[0], inv, x0);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int nv = a.D - (c * TPR + tr) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[c][j] = j < nv ? x[c][j] - m : 0.f;
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
        a.mean[row] = m + dl;
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
  __shared__ float red[2 * 3 * LnShape<TPR>::THREADS / 64];
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
        const float w = ln_weighted(y[c][j], gm[c][j]);
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
        o[j] = rs * fmaf(-d, c2, ln_weighted_again(y[c][j], gm[c][j]) - c1);
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
      // over the rows of a wave by exchanges, over the waves through LDS
#pragma unroll
      for (int o = TPR; o < 64; o <<= 1)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += __shfl_xor(v[j], o, 64);
      if (RPB > 1) {
        constexpr int SPAN = TPR < 64 ? 64 : TPR, N = THREADS / SPAN;  // threads between equal columns
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) fold[j * THREADS + threadIdx.x] = v[j];
        __syncthreads();
        if ((int)threadIdx.x < TPR) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            v[j] = 0.f;
#pragma unroll
            for (int r = 0; r < N; ++r) v[j] += fold[j * THREADS + r * SPAN + tr];
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
// Wider rows: one workgroup a row, which it reads two or three times (from cache after the first);
// the parameters' gradients are summed by columns in a launch of their own.
// ---------------------------------------------------------------------------------------------
namespace {
constexpr int LN_WIDE = 1024;  // threads

// f(x, col, nv) for 16 bytes after 16 bytes of a row
template <class E, class F>
__device__ __forceinline__ void for_row(const typename E::T* p, int D, F f) {
#pragma unroll 2
  for (int col = (int)threadIdx.x * E::V; col < D; col += LN_WIDE * E::V) {
    Raw r;
    float x[E::V];
    load16<E, true>(r, p + col, D - col, true, 0u);
    E::unpack(r.w, x);
    f(x, col, D - col);
  }
}
// the row's input at col: 16 bytes of x, or as many codes
template <class E, bool Q8>
__device__ __forceinline__ void ln_in(const LnArgs& a, int nb, int64_t r, int col, float* x) {
  if (Q8) {
    uint32_t w[E::V / 4];
    load_codes<E::V>(w, a.codes + r * a.D + col, a.D - col);
    unpack_codes<E::V>(w, a.scales[r * nb + col / RS_PACK_BLOCK], x);
  } else {
    Raw q;
    load16<E, true>(q, (const typename E::T*)a.x + r * a.ldx + col, a.D - col, true, 0u);
    E::unpack(q.w, x);
  }
}
}  // namespace

template <class E>
__global__ void __launch_bounds__(LN_WIDE) ln_wide_fwd_kernel(const LnArgs a) {
  typedef typename E::T X;
  constexpr int V = E::V;
  __shared__ float red[2 * 2 * LN_WIDE / 64];
  int flip = 0;
  const int D = a.D, nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const X* xr = (const X*)a.x + r * a.ldx;
    float s[1] = {0.f}, q[2] = {0.f, 0.f};
    const float x0 = E::load(xr[0]);
    for_row<E>(xr, D, [&](const float* x, int, int nv) {
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += j < nv ? x[j] - x0 : 0.f;
    });
    row_sum<1, LN_WIDE>(s, red, flip);
    const float m = x0 + s[0] / (float)D;
    for_row<E>(xr, D, [&](const float* x, int, int nv) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = j < nv ? x[j] - m : 0.f;
        q[0] += d;
        q[1] = fmaf(d, d, q[1]);
      }
    });
    row_sum<2, LN_WIDE>(q, red, flip);
    const float dl = q[0] / (float)D, var = q[1] / (float)D - dl * dl;
    const float rs = 1.0f / sqrtf((var < 0.f ? 0.f : var) + a.eps);
    for_row<E>(xr, D, [&](const float* x, int col, int nv) {
      float y[V], gm[V], bt[V];
      load_f<V>(gm, a.gamma + col, nv);
      load_f<V>(bt, a.beta + col, nv);
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = fmaf((x[j] - m - dl) * rs, gm[j], bt[j]);
      store16<E>((X*)a.y + r * a.ldy + col, y, nv);
    });
    if (threadIdx.x == 0 && a.mean) {
      a.mean[r] = m + dl;
      a.rstd[r] = rs;
    }
    if (a.codes) {  // 32 lanes x 4 elements a block
      for (int b = (int)threadIdx.x >> 5; b < nb; b += LN_WIDE / 32) {
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

// dx of a row, and its corrected mean into ws
template <class E, bool Q8>
__global__ void __launch_bounds__(LN_WIDE) ln_wide_bwd_kernel(const LnArgs a) {
  typedef typename E::T X;
  constexpr int V = E::V;
  __shared__ float red[2 * 3 * LN_WIDE / 64];
  int flip = 0;
  const int D = a.D, nb = (D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const X* dy = (const X*)a.dy + r * a.lddy;
    const float m = a.mean[r], rs = a.rstd[r];
    float s[3] = {0.f, 0.f, 0.f};
    for_row<E>(dy, D, [&](const float* y, int col, int nv) {
      float gm[V], x[V];
      load_f<V>(gm, a.gamma + col, nv);
      ln_in<E, Q8>(a, nb, r, col, x);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float w = ln_weighted(y[j], gm[j]), d = j < nv ? x[j] - m : 0.f;
        s[0] += w;
        s[1] = fmaf(w, d, s[1]);
        s[2] += d;
      }
    });
    row_sum<3, LN_WIDE>(s, red, flip);
    const float dl = Q8 ? 0.f : s[2] / (float)D;
    const float c1 = s[0] / (float)D, c2 = (s[1] / (float)D - dl * c1) * rs * rs;
    for_row<E>(dy, D, [&](const float* y, int col, int nv) {
      float gm[V], x[V], o[V];
      load_f<V>(gm, a.gamma + col, nv);
      ln_in<E, Q8>(a, nb, r, col, x);
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = rs * fmaf(-(x[j] - m - dl), c2, ln_weighted(y[j], gm[j]) - c1);
      store16<E>((X*)a.dx + r * a.lddx + col, o, nv);
    });
    if (threadIdx.x == 0) a.ws[r] = m + dl;
  }
}

// Partial rows [dgamma | dbeta] of 16 bytes of columns a thread, over every gridDim.y-th row
template <class E, bool Q8>
__global__ void __launch_bounds__(64) ln_wide_params_kernel(const LnArgs a) {
  constexpr int V = E::V;
  const int nb = (a.D + RS_PACK_BLOCK - 1) / RS_PACK_BLOCK;
  const int col = ((int)blockIdx.x * 64 + (int)threadIdx.x) * V, nv = a.D - col;
  if (nv <= 0) return;
  float ag[V], ab[V];
#pragma unroll
  for (int j = 0; j < V; ++j) ag[j] = ab[j] = 0.f;
#pragma unroll 4
  for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    Raw q;
    float y[V], x[V];
    load16<E, true>(q, (const typename E::T*)a.dy + r * a.lddy + col, nv, true, 0u);
    E::unpack(q.w, y);
    ln_in<E, Q8>(a, nb, r, col, x);
    const float m = a.ws[r], rs = a.rstd[r];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      ag[j] = fmaf(y[j], (x[j] - m) * rs, ag[j]);
      ab[j] += y[j];
    }
  }
  float* part = a.ws + a.rows + (int64_t)blockIdx.y * 2 * a.D + col;
  store_f<V>(part, ag, nv);
  store_f<V>(part + a.D, ab, nv);
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
namespace {

// X(threads of a row, 16-byte pieces a thread, pieces from, pieces to): the first that holds the row,
// with at most a third of the lanes without work.  A power of two of pieces takes a lane each up to a
// wave (131072 x 256 fp32, forward + backward: 127 us, half the lanes with two pieces 147 us), other
// widths few lanes with several (200000 x 100 bf16: 60 us, 16 lanes with one piece 76 us).
#define LN_SHAPES(X)                                                                              \
  X(1, 1, 1, 1) X(4, 1, 4, 4) X(8, 1, 8, 8) X(16, 1, 16, 16) X(32, 1, 32, 32) X(64, 1, 64, 64)    \
  X(1, 2, 1, 2) X(1, 3, 1, 3) X(2, 3, 1, 6) X(4, 2, 1, 8) X(4, 3, 1, 12) X(8, 2, 1, 16)           \
  X(8, 3, 1, 24) X(16, 2, 1, 32) X(16, 3, 1, 48) X(32, 2, 1, 64) X(32, 3, 1, 96)                  \
  X(64, 2, 1, 128) X(64, 3, 1, 192) X(64, 4, 1, 256) X(128, 3, 1, 384) X(128, 4, 1, 512)          \
  X(256, 3, 1, 768) X(256, 4, 1, 1024) X(512, 3, 1, 1536) X(512, 4, 1, 2048)

int ln_pieces(int D, int V) { return (D + V - 1) / V; }

struct LnPlan {
  int tpr, nch;  // 0: wider than any shape
};
LnPlan ln_plan(int pieces) {
#define LN_PLAN(TPR, NCH, FROM, TO) \
  if (pieces >= FROM && pieces <= TO) return {TPR, NCH};
  LN_SHAPES(LN_PLAN)
#undef LN_PLAN
  return {0, 0};
}

int64_t ln_rounds(int64_t rows, int tpr) {  // of one workgroup over all rows
  const int64_t rpb = tpr < 256 ? 256 / tpr : 1;
  return (rows + rpb - 1) / rpb;
}
int64_t ln_grid(int64_t rows, int tpr, int64_t most) {
  const int64_t n = ln_rounds(rows, tpr);
  return n < most ? n : most;
}

// Partial rows of the parameters' gradients = workgroups of the backward: two a compute unit, which
// is what its registers allow with 32 elements a thread, and more of them measured slower down to 8
// elements (65536 x 1024 bf16: 78 us, with 1024 workgroups 95; 400000 x 64 bf16: 34 us, with 2048 38).
// Narrow rows of 4 elements a thread have too few bytes in flight so (400000 x 64 fp32: 90 us, with
// 2048 63).  For rows wider than any shape, as many groups of rows as give 1024 waves or so.
int64_t ln_parts(int64_t rows, int D, int V) {
  const LnPlan p = ln_plan(ln_pieces(D, V));
  if (!p.tpr) {
    const int64_t most = 65536 / ln_pieces(D, V) + 1;
    return rows < most ? rows : most;
  }
  return ln_grid(rows, p.tpr, p.nch * V <= 4 && D <= 128 ? 2048 : 512);
}

template <class E>
int ln_fwd(hipStream_t s, const LnArgs& a) {
  const int pieces = ln_pieces(a.D, E::V), tpr = ln_plan(pieces).tpr;
  if (!tpr) {
    ln_wide_fwd_kernel<E><<<(unsigned)(a.rows < 65536 ? a.rows : 65536), LN_WIDE, 0, s>>>(a);
    return rs_status_after_launch();
  }
  const unsigned grid = (unsigned)ln_grid(a.rows, tpr, 2048);
#define LN_FWD(TPR, NCH, FROM, TO)                                                     \
  if (pieces >= FROM && pieces <= TO) {                                                \
    if (a.codes) ln_fwd_kernel<E, TPR, NCH, true><<<grid, LnShape<TPR>::THREADS, 0, s>>>(a); \
    else ln_fwd_kernel<E, TPR, NCH, false><<<grid, LnShape<TPR>::THREADS, 0, s>>>(a);  \
    return rs_status_after_launch();                                                   \
  }
  LN_SHAPES(LN_FWD)
#undef LN_FWD
  return RS_ERR_UNSUPPORTED;
}

template <class E>
void ln_bwd_rows(hipStream_t s, const LnArgs& a, unsigned grid) {
  const int pieces = ln_pieces(a.D, E::V);
#define LN_BWD(TPR, NCH, FROM, TO)                                                     \
  if (pieces >= FROM && pieces <= TO) {                                                \
    if (a.codes) ln_bwd_kernel<E, TPR, NCH, true><<<grid, LnShape<TPR>::THREADS, 0, s>>>(a); \
    else ln_bwd_kernel<E, TPR, NCH, false><<<grid, LnShape<TPR>::THREADS, 0, s>>>(a);  \
    return;                                                                            \
  }
  LN_SHAPES(LN_BWD)
#undef LN_BWD
}

template <class E>
int ln_bwd(hipStream_t s, const LnArgs& a) {
  const bool wide = !ln_plan(ln_pieces(a.D, E::V)).tpr;
  const unsigned parts = (unsigned)ln_parts(a.rows, a.D, E::V);
  if (a.rows && wide) {
    const unsigned grid = (unsigned)(a.rows < 65536 ? a.rows : 65536);
    const dim3 cols((unsigned)((ln_pieces(a.D, E::V) + 63) / 64), parts);
    if (a.codes) {
      ln_wide_bwd_kernel<E, true><<<grid, LN_WIDE, 0, s>>>(a);
      ln_wide_params_kernel<E, true><<<cols, 64, 0, s>>>(a);
    } else {
      ln_wide_bwd_kernel<E, false><<<grid, LN_WIDE, 0, s>>>(a);
      ln_wide_params_kernel<E, false><<<cols, 64, 0, s>>>(a);
    }
  } else if (a.rows) {
    ln_bwd_rows<E>(s, a, parts);
  }
  ln_params_kernel<<<(unsigned)((2 * a.D + 31) / 32), 1024, 0, s>>>(
      wide ? a.ws + a.rows : a.ws, (int)parts, a.D, a.dgamma, a.dbeta, a.accumulate);
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

// for whichever element size needs more
RS_API int64_t rs_layernorm_bwd_workspace_floats(int64_t rows, int D) {
  if (rows < 0 || D <= 0 || D > LN_MAX_D) return 0;
  int64_t most = 0;
  for (int V = 4; V <= 8; V += 4) {
    const int64_t n = ln_parts(rows, D, V) * 2 * D + (ln_plan(ln_pieces(D, V)).tpr ? 0 : rows);
    if (n > most) most = n;
  }
  return most;
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
