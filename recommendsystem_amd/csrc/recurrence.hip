// Gated linear recurrence over [B, T, D] and its gradients, all channels independent:
//   i_t = sigmoid(-g_t) = 1 - f_t        h_t = f_t h_{t-1} + (1 - f_t) v_t = h_{t-1} + i_t (v_t - h_{t-1})
//   r_t = the gradient that reaches h_t from later steps, a_t = dh_t + r_t
//   dv_t = i_t a_t     dg_t = a_t (h_{t-1} - v_t) i_t (1 - i_t)     r_{t-1} = a_t - i_t a_t
// The state and its gradient are fp32 throughout.  Written with i rather than f: a gate that is
// almost open (f rounds to 1) still moves the state by its own small i.
// Steps from lengths[b] on are not read: h, dv and dg are zero there and the state stands still.
//
// A run of steps takes the state in front of it, s, to A s + H: A = f_1 f_2 ... is what it keeps, H
// where it takes a zero state.  Two runs join to A = A1 A2, H = A2 H1 + H2; the gradient runs the
// other way through the same A.  A is held as one signed number m: as A itself up to 1/2 (m > 0), as
// -C, C = 1 - A, above (m <= 0), so that neither a long memory (A close to 1) nor a state that has
// been forgotten (A close to 0) loses digits:  A s + H = (m <= 0 ? s : 0) + m s + H.  A workgroup owns one tile of channels and
// walks the time axis in tiles of NG x K steps: a thread takes K consecutive steps of 16 bytes of
// channels into registers, reduces them to (A, H), the NG runs are joined by wave shuffles and one
// LDS exchange, and every thread then replays its own steps from the state in front of them.  So
// everything is read once and written once, whatever the length.
//
// The backward computes the states again from v and g, tile by tile, from the fp32 states that
// the forward kept in front of every tile; h itself (rounded to the rows' type) is not used.
//
// Where B and D give too few workgroups to fill the chip, the time axis is cut into segments: a
// first launch reduces every segment to its (A, H), and each workgroup of the second folds those in
// front of its own.  The input is then read twice.
#include "elem.hpp"

namespace {

struct RecArgs {
  const void *v, *g, *dh;
  int64_t v_sb, v_st, g_sb, g_st, dh_sb, dh_st;
  int64_t B, T;
  int D, nct;       // width, channel tiles
  int tiles, tps;   // time tiles, time tiles of a segment
  int segs;
  const int32_t* lengths;
  const float *h0, *dlast;  // the state before the first step; the gradient of the one after the last
  float* states;
  void *h, *dv, *dg;
  int64_t dv_sb, dv_st, dg_sb, dg_st;
  float *last, *dh0;
  float* ws;  // [segs][2][B D]: (m, H) of every segment
};

template <class E>
__device__ __forceinline__ float rec_input_gate(float g) {
  // exp = inf gives 0.  16-bit rows: the exponential's argument is rounded once, |g| half steps of fp32
  return __builtin_amdgcn_rcpf(1.0f + (E::V == 4 ? expf(g) : __expf(g)));
}

// the bits of a gate that lets nothing in (+infinity), twice for 16-bit elements
template <class E>
struct ShutGate;
template <> struct ShutGate<ElemF32> { static constexpr uint32_t W = 0x7F800000u; };
template <> struct ShutGate<ElemBF16> { static constexpr uint32_t W = 0x7F807F80u; };
template <> struct ShutGate<ElemF16> { static constexpr uint32_t W = 0x7C007C00u; };

#define REC_TINY 1e-37f  // an A that underflows stays positive: 0 would read as C = 0, "keeps all"

// A and C of a run (each exact to its own last digits) as m
__device__ __forceinline__ float keep_of(float A, float C) {
  return C < 0.5f ? -C : fmaxf(A, REC_TINY);
}
// the state behind a run
__device__ __forceinline__ float pass(float s, float m, float h) {
  return (m <= 0.f ? s : 0.f) + fmaf(m, s, h);
}
// run 1, then run 2, into run 2:  A1 A2 out of A or -C on either side
__device__ __forceinline__ void join(float m1, float h1, float& m2, float& h2) {
  h2 = pass(h1, m2, h2);
  const bool c1 = m1 <= 0.f, c2 = m2 <= 0.f;
  const float p = fmaf(m1, m2, (c2 ? m1 : 0.f) + (c1 ? m2 : 0.f));
  m2 = c1 && c2 ? (p < -0.5f ? p + 1.0f : p) : fmaxf(p, REC_TINY);
}

// Which (b, channels, segment) a thread works on.
template <class E, int LC, int NG>
struct Place {
  int64_t b;
  int c0, nv;  // first channel, channels in range (<= 0: none)
  int cl;      // the channel to load from: c0, or 0 where there is none in range
  int seg, grp;
  int64_t n;   // steps of this sequence
  __device__ __forceinline__ Place(const RecArgs& a) {
    const int tid = (int)threadIdx.x;
    if (NG == 1) {  // every thread for itself: (b, 16 bytes of channels) in one flat range
      const int nch = (a.D + E::V - 1) / E::V;
      const int64_t id = (int64_t)blockIdx.x * LC + tid;
      b = id / nch;
      c0 = (int)(id % nch) * E::V;
      nv = b < a.B ? a.D - c0 : 0;
      if (b >= a.B) b = a.B - 1;
      seg = 0;
      grp = 0;
    } else {
      int64_t id = blockIdx.x;
      const int64_t per = a.B * a.nct;
      seg = a.segs > 1 ? (int)(id / per) : 0;
      id -= seg * per;
      b = id / a.nct;
      c0 = ((int)(id % a.nct) * LC + tid % LC) * E::V;
      nv = a.D - c0;
      grp = tid / LC;
    }
    cl = nv > 0 ? c0 : 0;
    n = a.T;
    if (a.lengths) {
      n = a.lengths[b];
      n = n < 0 ? 0 : (n > a.T ? a.T : n);
    }
  }
};

// Inclusive join over the groups of a wave, in time order (UP) or against it.
template <int LC, int NG, int V, bool UP>
__device__ __forceinline__ void wave_scan(float* C, float* H) {
  constexpr int GW = NG == 1 ? 1 : 64 / LC;  // groups of a wave
  const int grp = (int)(threadIdx.x & 63) / LC;
#pragma unroll
  for (int d = 1; d < GW; d <<= 1) {
    const bool has = UP ? grp >= d : grp + d < GW;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float c1 = UP ? __shfl_up(C[j], d * LC, 64) : __shfl_down(C[j], d * LC, 64);
      const float h1 = UP ? __shfl_up(H[j], d * LC, 64) : __shfl_down(H[j], d * LC, 64);
      if (has) join(c1, h1, C[j], H[j]);
    }
  }
}

// The state in front of this thread's run (into `in`) and, into s, behind the whole tile, from s
// in front of the tile and the run's own (m, H); UP: in time order.  lds: [waves][2][LC * V].
template <int LC, int NG, int V, bool UP>
__device__ __forceinline__ void tile_scan(float* C, float* H, float* s, float* in, float* lds) {
  if (NG == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      in[j] = s[j];
      s[j] = pass(s[j], C[j], H[j]);
    }
    return;
  }
  constexpr int GW = 64 / LC, W = NG / GW;
  const int lane = (int)(threadIdx.x & 63), grp = lane / LC, wave = wave_id();
  wave_scan<LC, NG, V, UP>(C, H);
  const bool edge = UP ? grp == GW - 1 : grp == 0;  // holds the wave's total
  if (W > 1) {
    float* mine = lds + wave * 2 * LC * V + (lane % LC) * V;
    if (edge) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        mine[j] = C[j];
        mine[LC * V + j] = H[j];
      }
    }
    lds_barrier();
    float sw[V];
    // two waves' totals at a time: unrolled fully they would take 2 V registers a wave
#pragma unroll 2
    for (int k = 0; k < W; ++k) {
      const int w = UP ? k : W - 1 - k;
      const float* t = lds + w * 2 * LC * V + (lane % LC) * V;
      if (w == wave) {
#pragma unroll
        for (int j = 0; j < V; ++j) sw[j] = s[j];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = pass(s[j], t[j], t[LC * V + j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) in[j] = sw[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      in[j] = s[j];
      const int src = (UP ? 64 - LC : 0) + lane % LC;
      s[j] = pass(s[j], __shfl(C[j], src, 64), __shfl(H[j], src, 64));
    }
  }
  // what lies between the wave's edge and this thread's run
  const bool first = UP ? grp == 0 : grp == GW - 1;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float c1 = UP ? __shfl_up(C[j], LC, 64) : __shfl_down(C[j], LC, 64);
    const float h1 = UP ? __shfl_up(H[j], LC, 64) : __shfl_down(H[j], LC, 64);
    if (!first) in[j] = pass(in[j], c1, h1);
  }
}

// The (m, H) of all of the workgroup's runs in order, in every thread.  lds as in tile_scan.
template <int LC, int NG, int V, bool UP>
__device__ __forceinline__ void tile_total(float* C, float* H, float* lds) {
  constexpr int GW = 64 / LC, W = NG / GW;
  const int lane = (int)(threadIdx.x & 63), grp = lane / LC, wave = wave_id();
  wave_scan<LC, NG, V, UP>(C, H);
  float* mine = lds + wave * 2 * LC * V + (lane % LC) * V;
  if (UP ? grp == GW - 1 : grp == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      mine[j] = C[j];
      mine[LC * V + j] = H[j];
    }
  }
  lds_barrier();
#pragma unroll
  for (int j = 0; j < V; ++j) C[j] = H[j] = 0.f;
#pragma unroll 2
  for (int k = 0; k < W; ++k) {
    const float* t = lds + (UP ? k : W - 1 - k) * 2 * LC * V + (lane % LC) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float c = t[j], h = t[LC * V + j];
      join(C[j], H[j], c, h);
      C[j] = c;
      H[j] = h;
    }
  }
}

template <int LC, int NG, int V>
struct ScanLds {  // two buffers: one barrier a tile is enough
  static constexpr int W = NG == 1 ? 1 : NG / (64 / LC);
  static constexpr int FLOATS = W * 2 * LC * V;
};

}  // namespace

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------
template <class E, int LC, int NG, int K, bool PART>
__global__ void __launch_bounds__(LC * NG) rec_fwd_kernel(const RecArgs a) {
  constexpr int V = E::V, STEPS = NG * K;
  typedef typename E::T X;
  __shared__ __attribute__((aligned(16))) float lds[2][ScanLds<LC, NG, V>::FLOATS];
  const Place<E, LC, NG> p(a);
  const X* vp = (const X*)a.v + p.b * a.v_sb + p.cl;
  const X* gp = (const X*)a.g + p.b * a.g_sb + p.cl;
  X* hp = (X*)a.h + p.b * a.T * a.D + p.c0;
  const int64_t ch = p.b * a.D + p.c0;
  const int t0 = p.seg * a.tps, t1 = min(a.tiles, t0 + a.tps);

  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  if (a.h0) load_f<V>(s, a.h0 + ch, p.nv);
  for (int k = 0; k < p.seg; ++k) {
    float C[V], H[V];
    const float* w = a.ws + (int64_t)k * 2 * a.B * a.D + ch;
    load_f<V>(C, w, p.nv);
    load_f<V>(H, w + a.B * a.D, p.nv);
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = pass(s[j], C[j], H[j]);
  }

  Raw nv_[K], ng_[K];
  auto load = [&](int tile) {
    const int64_t t = (int64_t)tile * STEPS + p.grp * K;
    const X *vt = vp + t * a.v_st, *gt = gp + t * a.g_st;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool in = t + k < p.n;
      load16<E, PART>(nv_[k], in ? vt + k * a.v_st : vp, p.nv, in, 0u);
      load16<E, PART>(ng_[k], in ? gt + k * a.g_st : gp, p.nv, in, ShutGate<E>::W);
    }
  };
  if (t1 > t0) load(t0);
  for (int tile = t0; tile < t1; ++tile) {
    Raw rv[K];
    float in[K][V], A[V], C[V], H[V], st[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      A[j] = 1.f;
      C[j] = H[j] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float g[V], v[V];
      rv[k] = nv_[k];
      E::unpack(ng_[k].w, g);
      E::unpack(rv[k].w, v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float i = in[k][j] = rec_input_gate<E>(g[j]);
        H[j] = fmaf(i, v[j] - H[j], H[j]);
        A[j] = fmaf(-i, A[j], A[j]);
        C[j] = fmaf(i, 1.0f - C[j], C[j]);
      }
    }
    if (tile + 1 < t1) load(tile + 1);
    if (a.states && p.grp == 0)
      store_f<V>(a.states + (p.b * a.tiles + tile) * a.D + p.c0, s, p.nv);
#pragma unroll
    for (int j = 0; j < V; ++j) C[j] = keep_of(A[j], C[j]);
    tile_scan<LC, NG, V, true>(C, H, s, st, lds[tile & 1]);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t t = (int64_t)tile * STEPS + p.grp * K + k;
      float v[V], o[V];
      E::unpack(rv[k].w, v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        st[j] = fmaf(in[k][j], v[j] - st[j], st[j]);
        o[j] = t < p.n ? st[j] : 0.f;
      }
      if (t < a.T) store16<E>(hp + t * a.D, o, p.nv);
    }
  }
  if (p.grp == 0 && t1 == a.tiles) store_f<V>(a.last + ch, s, p.nv);
}

// (A, H) of every segment but the last (backward: of every one but the first, over dh, against
// time).  A group takes one run of consecutive steps of the segment, so the runs are joined once.
template <class E, int LC, int NG, int K, bool FWD, bool PART>
__global__ void __launch_bounds__(LC * NG) rec_sum_kernel(const RecArgs a) {
  constexpr int V = E::V, STEPS = NG * K;
  typedef typename E::T X;
  __shared__ __attribute__((aligned(16))) float lds[ScanLds<LC, NG, V>::FLOATS];
  Place<E, LC, NG> p(a);
  if (!FWD) p.seg += 1;
  // (no dh: the gates' rows are read in its place, and not used)
  const bool none = !FWD && !a.dh;
  const X* gp = (const X*)a.g + p.b * a.g_sb + p.cl;
  const X* xp = FWD ? (const X*)a.v + p.b * a.v_sb + p.cl
                    : none ? gp : (const X*)a.dh + p.b * a.dh_sb + p.cl;
  const int64_t x_st = FWD ? a.v_st : none ? a.g_st : a.dh_st;
  const int run = a.tps * K;  // steps of a group
  const int64_t first = (int64_t)p.seg * a.tps * STEPS + (int64_t)p.grp * run;
  float A[V], C[V], H[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    A[j] = 1.f;
    C[j] = H[j] = 0.f;
  }
  for (int q = 0; q < a.tps; ++q) {
    Raw rx[K], rg[K];
    const int64_t t = first + (FWD ? q * K : run - 1 - q * K);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      {
        const int64_t tk = FWD ? t + k : t - k;
        const bool in = tk < p.n;
        load16<E, PART>(rx[k], in ? xp + tk * x_st : xp, p.nv, in && !none, 0u);
        load16<E, PART>(rg[k], in ? gp + tk * a.g_st : gp, p.nv, in, ShutGate<E>::W);
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float g[V], x[V];
      E::unpack(rg[k].w, g);
      E::unpack(rx[k].w, x);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float i = rec_input_gate<E>(g[j]);
        if (FWD) H[j] = fmaf(i, x[j] - H[j], H[j]);
        else H[j] = fmaf(-i, x[j] + H[j], x[j] + H[j]);
        A[j] = fmaf(-i, A[j], A[j]);
        C[j] = fmaf(i, 1.0f - C[j], C[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) C[j] = keep_of(A[j], C[j]);
  tile_total<LC, NG, V, FWD>(C, H, lds);
  if (p.grp == 0) {
    float* w = a.ws + (int64_t)p.seg * 2 * a.B * a.D + p.b * a.D + p.c0;
    store_f<V>(w, C, p.nv);
    store_f<V>(w + a.B * a.D, H, p.nv);
  }
}

// ---------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------
template <class E, int LC, int NG, int K, bool PART>
__global__ void __launch_bounds__(LC * NG) rec_bwd_kernel(const RecArgs a) {
  constexpr int V = E::V, STEPS = NG * K;
  typedef typename E::T X;
  __shared__ __attribute__((aligned(16))) float lds[2][2][ScanLds<LC, NG, V>::FLOATS];
  const Place<E, LC, NG> p(a);
  const X* vp = (const X*)a.v + p.b * a.v_sb + p.cl;
  const X* gp = (const X*)a.g + p.b * a.g_sb + p.cl;
  // (no dh: the gates' rows are read in its place, and not used)
  const bool none = !a.dh;
  const X* dp = none ? gp : (const X*)a.dh + p.b * a.dh_sb + p.cl;
  const int64_t d_st = none ? a.g_st : a.dh_st;
  X* dvp = (X*)a.dv + p.b * a.dv_sb + p.c0;
  X* dgp = (X*)a.dg + p.b * a.dg_sb + p.c0;
  const int64_t ch = p.b * a.D + p.c0;
  const int t0 = p.seg * a.tps, t1 = min(a.tiles, t0 + a.tps);

  float r[V];  // the gradient from behind the tile
#pragma unroll
  for (int j = 0; j < V; ++j) r[j] = 0.f;
  if (a.dlast) load_f<V>(r, a.dlast + ch, p.nv);
  for (int k = a.segs - 1; k > p.seg; --k) {
    float C[V], G[V];
    const float* w = a.ws + (int64_t)k * 2 * a.B * a.D + ch;
    load_f<V>(C, w, p.nv);
    load_f<V>(G, w + a.B * a.D, p.nv);
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = pass(r[j], C[j], G[j]);
  }

  Raw nv_[K], ng_[K], nd_[K];
  float ns[V];
  auto load = [&](int tile) {
    const int64_t t = (int64_t)tile * STEPS + p.grp * K;
    const X *vt = vp + t * a.v_st, *gt = gp + t * a.g_st, *dt = dp + t * d_st;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool in = t + k < p.n;
      load16<E, PART>(ng_[k], in ? gt + k * a.g_st : gp, p.nv, in, ShutGate<E>::W);
      load16<E, PART>(nv_[k], in ? vt + k * a.v_st : vp, p.nv, in, 0u);
      load16<E, PART>(nd_[k], in ? dt + k * d_st : dp, p.nv, in && !none, 0u);
    }
    load_f<V>(ns, a.states + (p.b * a.tiles + tile) * a.D + p.c0, p.nv);
  };
  if (t1 > t0) load(t1 - 1);
  for (int tile = t1 - 1; tile >= t0; --tile) {
    Raw rd[K];
    float in[K][V], e[K][V], A[V], C[V], H[V], G[V], s[V], st[V], rt[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      A[j] = 1.f;
      C[j] = H[j] = G[j] = 0.f;
      s[j] = ns[j];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float g[V];
      rd[k] = nd_[k];
      E::unpack(ng_[k].w, g);
      E::unpack(nv_[k].w, e[k]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float i = in[k][j] = rec_input_gate<E>(g[j]);
        H[j] = fmaf(i, e[k][j] - H[j], H[j]);
        A[j] = fmaf(-i, A[j], A[j]);
        C[j] = fmaf(i, 1.0f - C[j], C[j]);
      }
    }
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
      float d[V];
      E::unpack(rd[k].w, d);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float x = d[j] + G[j];
        G[j] = fmaf(-in[k][j], x, x);
      }
    }
    if (tile > t0) load(tile - 1);
    float C2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) C2[j] = C[j] = keep_of(A[j], C[j]);
    tile_scan<LC, NG, V, true>(C, H, s, st, lds[tile & 1][0]);
    tile_scan<LC, NG, V, false>(C2, G, r, rt, lds[tile & 1][1]);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = st[j] - e[k][j];  // h_{t-1} - v_t
        e[k][j] = d;
        st[j] = fmaf(-in[k][j], d, st[j]);
      }
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
      const int64_t t = (int64_t)tile * STEPS + p.grp * K + k;
      float d[V], gv[V], gg[V];
      E::unpack(rd[k].w, d);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float i = in[k][j], x = d[j] + rt[j];
        gv[j] = i * x;
        gg[j] = gv[j] * e[k][j] * (1.0f - i);
        rt[j] = x - gv[j];
      }
      if (t < a.T) {
        store16<E>(dvp + t * a.dv_st, gv, p.nv);
        store16<E>(dgp + t * a.dg_st, gg, p.nv);
      }
    }
  }
  if (p.grp == 0 && t0 == 0 && a.dh0) store_f<V>(a.dh0 + ch, r, p.nv);
}

// ---------------------------------------------------------------------------------------------
// one step
// ---------------------------------------------------------------------------------------------
template <class E>
__global__ void __launch_bounds__(256) rec_step_kernel(const RecArgs a, float* new_state) {
  constexpr int V = E::V;
  typedef typename E::T X;
  const int nch = (a.D + V - 1) / V;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.B * nch) return;
  const int64_t b = id / nch;
  const int c0 = (int)(id % nch) * V, nv = a.D - c0;
  float s[V], v[V], g[V];
  Raw rv, rg;
  load16<E, true>(rv, (const X*)a.v + b * a.v_sb + c0, nv, true, 0u);
  load16<E, true>(rg, (const X*)a.g + b * a.g_sb + c0, nv, true, 0u);
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  if (a.h0) load_f<V>(s, a.h0 + b * a.D + c0, nv);
  E::unpack(rv.w, v);
  E::unpack(rg.w, g);
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = fmaf(rec_input_gate<E>(g[j]), v[j] - s[j], s[j]);
  store16<E>((X*)a.h + b * a.D + c0, s, nv);
  store_f<V>(new_state + b * a.D + c0, s, nv);
}

// ---------------------------------------------------------------------------------------------
// Launch plans, a function of the element size, B, T and D alone (the backward finds the states
// where the forward's plan put them).
// ---------------------------------------------------------------------------------------------
namespace {

enum { REC_FLAT, REC_WAVE, REC_BLOCK };
struct RecPlan {
  int kind, steps;  // steps: of a time tile
  int nct, segs, tps;
  int64_t tiles;
};

RecPlan rec_plan(int dtype, int64_t B, int64_t T, int D) {
  const int V = dtype == RS_F32 ? 4 : 8;
  RecPlan p;
  p.nct = (D + 8 * V - 1) / (8 * V);
  const int64_t blocks = B * p.nct;
  p.kind = T <= 8 ? REC_FLAT : T <= 64 || blocks >= 2048 ? REC_WAVE : REC_BLOCK;
  p.steps = p.kind == REC_FLAT ? 8 : p.kind == REC_WAVE ? 64 : 256;
  p.tiles = (T + p.steps - 1) / p.steps;
  p.segs = 1;
  p.tps = (int)p.tiles;
  if (p.kind == REC_BLOCK && blocks < 256 && p.tiles > 1) {
    const int64_t want = (512 + blocks - 1) / blocks;
    p.tps = (int)((p.tiles + want - 1) / want);
    p.segs = (int)((p.tiles + p.tps - 1) / p.tps);
  }
  return p;
}

void rec_fill(RecArgs& a, const RecPlan& p, int64_t B, int64_t T, int D) {
  a.B = B;
  a.T = T;
  a.D = D;
  a.nct = p.nct;
  a.tiles = (int)p.tiles;
  a.tps = p.tps;
  a.segs = p.segs;
}

template <class E, bool PART>
int rec_fwd_as(hipStream_t s, const RecPlan& p, const RecArgs& a) {
  const unsigned per = (unsigned)(a.B * a.nct);
  if (p.kind == REC_FLAT) {
    const int64_t n = a.B * ((a.D + E::V - 1) / E::V);
    rec_fwd_kernel<E, 64, 1, 8, PART><<<(unsigned)((n + 63) / 64), 64, 0, s>>>(a);
  } else if (p.kind == REC_WAVE) {
    rec_fwd_kernel<E, 8, 8, 8, PART><<<per, 64, 0, s>>>(a);
  } else {
    if (p.segs > 1) rec_sum_kernel<E, 8, 32, 8, true, PART><<<per * (p.segs - 1), 256, 0, s>>>(a);
    rec_fwd_kernel<E, 8, 32, 8, PART><<<per * p.segs, 256, 0, s>>>(a);
  }
  return rs_status_after_launch();
}

template <class E, bool PART>
int rec_bwd_as(hipStream_t s, const RecPlan& p, const RecArgs& a) {
  const unsigned per = (unsigned)(a.B * a.nct);
  if (p.kind == REC_FLAT) {
    const int64_t n = a.B * ((a.D + E::V - 1) / E::V);
    rec_bwd_kernel<E, 64, 1, 8, PART><<<(unsigned)((n + 63) / 64), 64, 0, s>>>(a);
  } else if (p.kind == REC_WAVE) {
    rec_bwd_kernel<E, 8, 16, 4, PART><<<per, 128, 0, s>>>(a);
  } else {
    if (p.segs > 1) rec_sum_kernel<E, 8, 32, 8, false, PART><<<per * (p.segs - 1), 256, 0, s>>>(a);
    rec_bwd_kernel<E, 8, 64, 4, PART><<<per * p.segs, 512, 0, s>>>(a);
  }
  return rs_status_after_launch();
}

template <class E>
int rec_fwd(hipStream_t s, const RecPlan& p, const RecArgs& a) {
  return a.D % E::V ? rec_fwd_as<E, true>(s, p, a) : rec_fwd_as<E, false>(s, p, a);
}
template <class E>
int rec_bwd(hipStream_t s, const RecPlan& p, const RecArgs& a) {
  return a.D % E::V ? rec_bwd_as<E, true>(s, p, a) : rec_bwd_as<E, false>(s, p, a);
}

template <class E>
int rec_step(hipStream_t s, const RecArgs& a, float* new_state) {
  const int64_t n = a.B * ((a.D + E::V - 1) / E::V);
  rec_step_kernel<E><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a, new_state);
  return rs_status_after_launch();
}

// what the launches index: workgroups and time tiles in 31 bits
bool rec_shape_ok(int dtype, int64_t B, int64_t T, int D) {
  return dtype >= RS_F32 && dtype <= RS_F16 && B >= 0 && T >= 0 && D > 0 && T < (1ll << 31) &&
         B < (1ll << 30) && B * ((D + 31) / 32) < (1ll << 30);
}

}  // namespace

RS_API int64_t rs_gated_rec_states_floats(int dtype, int64_t B, int64_t T, int D) {
  if (!rec_shape_ok(dtype, B, T, D)) return 0;
  return B * rec_plan(dtype, B, T, D).tiles * D;
}

RS_API int64_t rs_gated_rec_workspace_floats(int dtype, int64_t B, int64_t T, int D) {
  if (!rec_shape_ok(dtype, B, T, D)) return 0;
  const RecPlan p = rec_plan(dtype, B, T, D);
  return p.segs > 1 ? p.segs * 2 * B * D : 0;
}

RS_API int rs_gated_rec_fwd(void* stream, int dtype, const void* v, int64_t v_sb, int64_t v_st,
                            const void* g, int64_t g_sb, int64_t g_st, int64_t B, int64_t T, int D,
                            const int32_t* lengths, const float* h0, void* h, float* last,
                            float* states, float* workspace, int64_t workspace_floats) {
  if (!rec_shape_ok(dtype, B, T, D)) return RS_ERR_ARG;
  if (B == 0) return RS_OK;
  if (!last || (T > 0 && (!v || !g || !h || v_sb < 0 || v_st < 0 || g_sb < 0 || g_st < 0)))
    return RS_ERR_ARG;
  const int64_t need = rs_gated_rec_workspace_floats(dtype, B, T, D);
  if (need > 0 && (!workspace || workspace_floats < need)) return RS_ERR_ARG;
  const RecPlan p = rec_plan(dtype, B, T, D);
  RecArgs a = {};
  rec_fill(a, p, B, T, D);
  a.v = v, a.v_sb = v_sb, a.v_st = v_st;
  a.g = g, a.g_sb = g_sb, a.g_st = g_st;
  a.lengths = lengths, a.h0 = h0, a.h = h, a.last = last, a.states = states, a.ws = workspace;
  return RS_DISPATCH_ELEM(dtype, rec_fwd, rs_stream(stream), p, a);
}

RS_API int rs_gated_rec_bwd(void* stream, int dtype, const void* v, int64_t v_sb, int64_t v_st,
                            const void* g, int64_t g_sb, int64_t g_st, int64_t B, int64_t T, int D,
                            const int32_t* lengths, const float* states, const void* dh,
                            int64_t dh_sb, int64_t dh_st, const float* dlast, void* dv,
                            int64_t dv_sb, int64_t dv_st, void* dg, int64_t dg_sb, int64_t dg_st,
                            float* dh0, float* workspace, int64_t workspace_floats) {
  if (!rec_shape_ok(dtype, B, T, D)) return RS_ERR_ARG;
  if (B == 0) return RS_OK;
  if (T > 0 && (!v || !g || !states || !dv || !dg || v_sb < 0 || v_st < 0 || g_sb < 0 ||
                g_st < 0 || dh_sb < 0 || dh_st < 0 || (T > 1 && (dv_st < D || dg_st < D)) ||
                (B > 1 && (dv_sb < D || dg_sb < D))))
    return RS_ERR_ARG;
  if (T == 0 && !dh0) return RS_OK;
  const int64_t need = rs_gated_rec_workspace_floats(dtype, B, T, D);
  if (need > 0 && (!workspace || workspace_floats < need)) return RS_ERR_ARG;
  const RecPlan p = rec_plan(dtype, B, T, D);
  RecArgs a = {};
  rec_fill(a, p, B, T, D);
  a.v = v, a.v_sb = v_sb, a.v_st = v_st;
  a.g = g, a.g_sb = g_sb, a.g_st = g_st;
  a.dh = dh, a.dh_sb = dh_sb, a.dh_st = dh_st;
  a.lengths = lengths, a.states = const_cast<float*>(states), a.dlast = dlast;
  a.dv = dv, a.dv_sb = dv_sb, a.dv_st = dv_st;
  a.dg = dg, a.dg_sb = dg_sb, a.dg_st = dg_st;
  a.dh0 = dh0, a.ws = workspace;
  return RS_DISPATCH_ELEM(dtype, rec_bwd, rs_stream(stream), p, a);
}

RS_API int rs_gated_rec_step(void* stream, int dtype, const void* v, int64_t ld_v, const void* g,
                             int64_t ld_g, int64_t B, int D, const float* state, void* h,
                             float* new_state) {
  if (!rec_shape_ok(dtype, B, 1, D)) return RS_ERR_ARG;
  if (B == 0) return RS_OK;
  if (!v || !g || !h || !new_state || ld_v < 0 || ld_g < 0) return RS_ERR_ARG;
  RecArgs a = {};
  a.B = B, a.T = 1, a.D = D;
  a.v = v, a.v_sb = ld_v, a.g = g, a.g_sb = ld_g, a.h0 = state, a.h = h;
  return RS_DISPATCH_ELEM(dtype, rec_step, rs_stream(stream), a, new_state);
}
