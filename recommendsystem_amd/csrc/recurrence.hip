// Gated linear recurrence over [B, T, D] and its gradients, all channels independent:
//   i_t = sigmoid(-g_t) = 1 - f_t        h_t = f_t h_{t-1} + (1 - f_t) v_t = h_{t-1} + i_t (v_t - h_{t-1})
//   r_t = the gradient that reaches h_t from later steps, a_t = dh_t + r_t
//   dv_t = i_t a_t     dg_t = a_t (h_{t-1} - v_t) i_t f_t     r_{t-1} = f_t a_t
// The state and its gradient are fp32 throughout.  A step is kept as the smaller one of i and f, to its
// own digits, and the other one is never formed where it would round to 1: an almost open gate still
// moves the state by its small i, an almost shut one still passes its small f of the state and of the
// gradient.
// Steps from lengths[b] on are not read: h, dv and dg are zero there and the state stands still.
//
// A run of steps takes the state in front of it, s, to A s + H: A = f_1 f_2 ... is what it keeps, H
// where it takes a zero state.  Two runs join to A = A1 A2, H = A2 H1 + H2; the gradient runs the
// other way through the same A.  A workgroup owns a tile of channels and walks the time axis in
// tiles of NG x K steps: a thread takes K consecutive steps of 8 bytes of channels into registers
// and reduces them to (A, H), the NG runs are joined by wave shuffles and one LDS exchange, and every
// thread then replays its own steps from the state in front of them, while the next tile's loads are
// in flight.  So everything is read once and written once, whatever the length.
//
// The backward computes the states again from v and g, tile by tile, from the fp32 states that
// the forward kept in front of every tile (of a sequence in one tile that is h0); h itself (rounded
// to the rows' type) is not used.
//
// Where B and D give too few workgroups to fill the chip, the time axis is cut into segments: a
// first launch reduces every segment to its (A, H), and each workgroup of the second folds those in
// front of its own.  The input is then read twice.
//
// Bound by memory; 8 bytes a lane (16 lanes to a line of 128 bytes) rather than 16 because the join
// costs a fixed number of operations a channel and thread: twice the steps a thread, half the joins.
// Tiles that are wholly part of the sequence go through a loop of their own with nothing conditional
// around its loads and stores: only then does the compiler know how many are in flight, and waits for
// the next tile's loads without waiting for this tile's stores (forward and backward, bf16, 10 x 4096 x
// 2048: 123 and 215 us, 145 and 247 with every tile masked; 8 x 4096 x 2048: 93 and 155 against 98 and 161;
// 37 x 1021 x 520 fp32: the same).  Widths that are no multiple of 8 bytes still have such conditions
// everywhere (PART): 8 x 4096 x 2046 bf16 takes 169 and 354 us.
// 8 x 4096 x 2048 bf16 (256 workgroups, pieces of 128 bytes): forward 93 us (4.4 TB/s), backward 155 us
// (4.4 TB/s).  8 x 4096 x 4096 in pieces of 256 bytes: 149 us (5.4 TB/s) and 257 us (5.2 TB/s), as fast
// as a copy of that size.  Holding a step as the smaller of i and f costs 0 to 7 percent of this, at some
// shapes up to 14 (10 x 4096 x 2048 bf16 forward 112 -> 123 us, 4096 x 50 x 8 backward 11.6 -> 13.4).
#include "elem.hpp"

namespace {

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

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
  float* ws;  // [segs][2][B D]: (A, H) of every segment
};

// A step's gate as one signed number: i for an open gate (g >= 0), -f for a shut one, with -0 where f
// vanishes; at most 1/2 in magnitude, m.
template <class E>
__device__ __forceinline__ float rec_gate(float g) {
  // exp = inf gives i = 0.  16-bit rows take the hardware's exp2 of the rounded g log2(e), off by |g|
  // half steps of fp32 relative to the gate; the reciprocal is off by one step
  const float e = sizeof(typename E::T) == 4 ? expf(g) : __expf(g), i = __builtin_amdgcn_rcpf(1.0f + e);
  return g < 0.f ? -(e * i) : i;
}
__device__ __forceinline__ bool gate_shut(float w) { return __float_as_int(w) < 0; }
// The same gate of which the compiler does not know the sign: it tests it again, rather than keep a
// lane mask for every step of a tile from one pass over the steps to the next.
__device__ __forceinline__ float gate_again(float w) {
  asm("" : "+v"(w));
  return w;
}
// f s + i v, as s + i (v - s) or v + f (s - v); d = s - v
__device__ __forceinline__ float gate_step(float w, bool shut, float s, float v, float d) {
  return fmaf(-w, d, shut ? v : s);
}
// f x
__device__ __forceinline__ float gate_keep(float w, bool shut, float x) { return fmaf(-w, x, shut ? 0.f : x); }

// the bits of a gate that lets nothing in (+infinity), twice for 16-bit elements
template <class E>
struct ShutGate;
template <> struct ShutGate<ElemF32> { static constexpr uint32_t W = 0x7F800000u; };
template <> struct ShutGate<ElemBF16> { static constexpr uint32_t W = 0x7F807F80u; };
template <> struct ShutGate<ElemF16> { static constexpr uint32_t W = 0x7C007C00u; };

// 8 bytes of channels of a row: VC<E> elements
template <class E>
struct VC { static constexpr int V = 8 / (int)sizeof(typename E::T); };
struct Half { uint32_t w[2]; };

// The row's channels at p (8 bytes).  PART (D is no multiple of V): a lane with fewer than V channels
// left picks its nv elements one by one (none for nv <= 0).  Without it every lane has V channels
// (Place), and nothing is conditional: a load or store behind a branch would leave the number of
// memory operations in flight unknown, and the next tile's loads could then only be waited for
// together with all of this tile's stores.  For the same reason steps that are not part of the
// sequence are loaded from some row that is, and masked where they are used.
template <class E, bool PART>
__device__ __forceinline__ void load8(Half& r, const typename E::T* p, int nv) {
  constexpr int V = VC<E>::V, S = 8 / V;
  if (!PART || nv >= V) {
    const RsVec<8, S> x = *reinterpret_cast<const RsVec<8, S>*>(p);
    r.w[0] = x.w[0];
    r.w[1] = x.w[1];
  } else {
    r.w[0] = r.w[1] = 0;
    if (nv > 0) {
      if (S == 4) r.w[0] = reinterpret_cast<const uint32_t*>(p)[0];
      else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
        r.w[0] = h[0];
        if (nv > 1) r.w[0] |= (uint32_t)h[1] << 16;
        if (nv > 2) r.w[1] = h[2];
      }
    }
  }
}
__device__ __forceinline__ void mask8(Half& r, bool in, uint32_t fill) {
  r.w[0] = in ? r.w[0] : fill;
  r.w[1] = in ? r.w[1] : fill;
}
template <class E, bool PART>
__device__ __forceinline__ void store8(typename E::T* p, const float* x, int nv) {
  constexpr int V = VC<E>::V, S = 8 / V;
  if (!PART || nv >= V) {
    RsVec<8, S> y;
    E::template pack<2>(x, y.w);
    *reinterpret_cast<RsVec<8, S>*>(p) = y;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < nv) p[j] = E::store(x[j]);
  }
}
// V floats (states, gradients of them)
template <int V, bool PART>
__device__ __forceinline__ void load_n(float* x, const float* p, int nv) {
  if (!PART || nv >= V) {
    const RsVec<4 * V, 4> r = *reinterpret_cast<const RsVec<4 * V, 4>*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = __uint_as_float(r.w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = j < nv ? p[j] : 0.f;
  }
}
template <int V, bool PART>
__device__ __forceinline__ void store_n(float* p, const float* x, int nv) {
  if (!PART || nv >= V) {
    RsVec<4 * V, 4> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.w[j] = __float_as_uint(x[j]);
    *reinterpret_cast<RsVec<4 * V, 4>*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < nv) p[j] = x[j];
  }
}

// the state behind a run
__device__ __forceinline__ float pass(float s, float A, float h) { return fmaf(A, s, h); }
// run 1, then run 2, into run 2
__device__ __forceinline__ void join(float A1, float h1, float& A2, float& h2) {
  h2 = fmaf(A2, h1, h2);
  A2 *= A1;
}

// Workgroups are dealt out to the 8 XCDs in turn, each with an L2 of its own.  Numbering them so that
// an XCD gets a run of consecutive ones puts the channel tiles of a row side by side: where rows do
// not start on lines of 128 bytes, neighbours share a line, which two XCDs would both fetch
// (65521 x 1000 fp16: 1.8 times the bytes).
__device__ __forceinline__ unsigned xcd_run(unsigned id, unsigned n) {
  const unsigned x = id & 7u, q = n >> 3, r = n & 7u;
  return x * q + (x < r ? x : r) + (id >> 3);
}

// Which (b, channels, segment) a thread works on.
// Lanes beyond the width (PART excepted) or the batch do the last ones' work once more, and write the
// same values to the same places.
template <class E, int LC, int NG, bool PART>
struct Place {
  int64_t b;
  int c0, nv;  // first channel, channels in range (PART: down to 0 or below)
  int cl;      // the channel to load from: c0, or 0 where there is none in range
  int seg, grp;
  int64_t n;   // steps of this sequence
  __device__ __forceinline__ Place(const RecArgs& a) {
    const int tid = (int)threadIdx.x;
    if (NG == 1) {  // every thread for itself: (b, 8 bytes of channels) in one flat range
      const int nch = (a.D + VC<E>::V - 1) / VC<E>::V;
      int64_t id = (int64_t)blockIdx.x * LC + tid;
      if (id >= a.B * nch) id = a.B * nch - 1;
      b = id / nch;
      c0 = (int)(id % nch) * VC<E>::V;
      seg = 0;
      grp = 0;
    } else {
      int64_t id = xcd_run(blockIdx.x, gridDim.x);
      const int64_t per = a.B * a.nct;
      seg = a.segs > 1 ? (int)(id / per) : 0;
      id -= seg * per;
      b = id / a.nct;
      c0 = ((int)(id % a.nct) * LC + tid % LC) * VC<E>::V;
      grp = tid / LC;
    }
    if (!PART && c0 > a.D - VC<E>::V) c0 = a.D - VC<E>::V;
    nv = a.D - c0;
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
__device__ __forceinline__ void wave_scan(float* A, float* H) {
  constexpr int GW = NG == 1 ? 1 : 64 / LC;  // groups of a wave
  const int grp = (int)(threadIdx.x & 63) / LC;
#pragma unroll
  for (int d = 1; d < GW; d <<= 1) {
    const bool has = UP ? grp >= d : grp + d < GW;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float a1 = UP ? __shfl_up(A[j], d * LC, 64) : __shfl_down(A[j], d * LC, 64);
      const float h1 = UP ? __shfl_up(H[j], d * LC, 64) : __shfl_down(H[j], d * LC, 64);
      if (has) join(a1, h1, A[j], H[j]);
    }
  }
}

// What lies between the edge of the wave and this thread's run, onto the state at that edge.
template <int LC, int NG, int V, bool UP>
__device__ __forceinline__ void wave_inner(const float* A, const float* H, float* in) {
  constexpr int GW = 64 / LC;
  const int grp = (int)(threadIdx.x & 63) / LC;
  const bool first = UP ? grp == 0 : grp == GW - 1;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float a1 = UP ? __shfl_up(A[j], LC, 64) : __shfl_down(A[j], LC, 64);
    const float h1 = UP ? __shfl_up(H[j], LC, 64) : __shfl_down(H[j], LC, 64);
    if (!first) in[j] = pass(in[j], a1, h1);
  }
}

// The state at the edge of this wave's runs, into `in`, and behind the whole tile, into s, from s
// in front of the tile and the waves' totals in lds, [waves][NT][LC * V] with the A in front: H is
// the hi-th.  UP: in time order.
template <int LC, int NG, int V, bool UP, int NT>
__device__ __forceinline__ void tile_fold(const float* lds, int hi, float* s, float* in) {
  constexpr int W = NG / (64 / LC);
  const int lane = (int)(threadIdx.x & 63), wave = wave_id();
#pragma unroll
  for (int j = 0; j < V; ++j) in[j] = s[j];
  // two waves' totals at a time: unrolled fully they would take 2 V registers a wave
#pragma unroll 2
  for (int k = 0; k < W; ++k) {
    const int w = UP ? k : W - 1 - k;
    const float* t = lds + w * NT * LC * V + (lane % LC) * V;
    if (w == wave) {
#pragma unroll
      for (int j = 0; j < V; ++j) in[j] = s[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = pass(s[j], t[j], t[hi * LC * V + j]);
  }
}

template <int LC, int NG, int V, bool UP>
__device__ __forceinline__ bool wave_edge() {  // holds the wave's total after wave_scan
  const int grp = (int)(threadIdx.x & 63) / LC;
  return UP ? grp == 64 / LC - 1 : grp == 0;
}

// This wave's part of lds: the V values of a channel lane at [which][LC * V]
template <int LC, int NG, int V, int NT>
__device__ __forceinline__ float* wave_part(float* lds, int which) {
  return lds + (wave_id() * NT + which) * LC * V + (int)(threadIdx.x % LC) * V;
}

// The state in front of this thread's run (into `in`) and, into s, behind the whole tile, from s
// in front of the tile and the run's own (A, H).
template <int LC, int NG, int V>
__device__ __forceinline__ void tile_scan(float* A, float* H, float* s, float* in, float* lds) {
  if (NG == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      in[j] = s[j];
      s[j] = pass(s[j], A[j], H[j]);
    }
    return;
  }
  wave_scan<LC, NG, V, true>(A, H);
  if (wave_edge<LC, NG, V, true>()) {
    store_n<V, false>(wave_part<LC, NG, V, 2>(lds, 0), A, V);
    store_n<V, false>(wave_part<LC, NG, V, 2>(lds, 1), H, V);
  }
  lds_barrier();
  tile_fold<LC, NG, V, true, 2>(lds, 1, s, in);
  wave_inner<LC, NG, V, true>(A, H, in);
}

// Both directions at once, behind one barrier: (A, H) from s in time order and (A, G) from r
// against it.
template <int LC, int NG, int V>
__device__ __forceinline__ void tile_scan_both(float* A, float* H, float* G, float* s, float* r,
                                               float* in_s, float* in_r, float* lds) {
  if (NG == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      in_s[j] = s[j];
      in_r[j] = r[j];
      r[j] = pass(r[j], A[j], G[j]);
    }
    return;
  }
  float A2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) A2[j] = A[j];
  wave_scan<LC, NG, V, true>(A, H);
  wave_scan<LC, NG, V, false>(A2, G);
  if (wave_edge<LC, NG, V, true>()) {
    store_n<V, false>(wave_part<LC, NG, V, 3>(lds, 0), A, V);
    store_n<V, false>(wave_part<LC, NG, V, 3>(lds, 1), H, V);
  }
  if (wave_edge<LC, NG, V, false>()) store_n<V, false>(wave_part<LC, NG, V, 3>(lds, 2), G, V);
  lds_barrier();
  tile_fold<LC, NG, V, true, 3>(lds, 1, s, in_s);
  tile_fold<LC, NG, V, false, 3>(lds, 2, r, in_r);
  wave_inner<LC, NG, V, true>(A, H, in_s);
  wave_inner<LC, NG, V, false>(A2, G, in_r);
}

// The (A, H) of all of the workgroup's runs in order, in every thread.
template <int LC, int NG, int V, bool UP>
__device__ __forceinline__ void tile_total(float* A, float* H, float* lds) {
  constexpr int W = NG / (64 / LC);
  wave_scan<LC, NG, V, UP>(A, H);
  if (wave_edge<LC, NG, V, UP>()) {
    store_n<V, false>(wave_part<LC, NG, V, 2>(lds, 0), A, V);
    store_n<V, false>(wave_part<LC, NG, V, 2>(lds, 1), H, V);
  }
  lds_barrier();
#pragma unroll
  for (int j = 0; j < V; ++j) {
    A[j] = 1.f;
    H[j] = 0.f;
  }
#pragma unroll 2
  for (int k = 0; k < W; ++k) {
    const float* t = lds + (UP ? k : W - 1 - k) * 2 * LC * V + (int)(threadIdx.x % LC) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float a2 = t[j], h2 = t[LC * V + j];
      join(A[j], H[j], a2, h2);
      A[j] = a2;
      H[j] = h2;
    }
  }
}

// One [B, T, D] array as a thread reads or writes it: its K steps of every tile.  The workgroup's
// sequence and a wave's first step are the same in all lanes, so addresses are a scalar base and one
// 32-bit offset a lane (rec_strides_ok bounds the strides); only where every thread works for itself
// (NG == 1) they are 64-bit a lane.
template <class E, int LC, int NG, int K, class Ptr>
struct Rows {
  typedef typename E::T X;
  Ptr base;
  int64_t st;
  uint32_t off;  // of the lane's first step and channel
  int c, ls;     // its channel; its first step of the wave's
  __device__ __forceinline__ Rows(Ptr p, int64_t b, int64_t sb, int64_t st_, int c_) : st(st_), c(c_) {
    ls = NG == 1 ? 0 : (int)(threadIdx.x & 63) / LC * K;
    base = NG == 1 ? p + b * sb + c : p + b * sb;
    off = NG == 1 ? 0u : (uint32_t)ls * (uint32_t)st + (uint32_t)c;
  }
  // step k of the thread; t: the wave's first step (NG == 1: the thread's)
  __device__ __forceinline__ Ptr at(int64_t t, int k) const { return base + (t + k) * st + off; }
  // the same within 0 .. n - 1 (n >= 1)
  __device__ __forceinline__ Ptr in(int64_t t, int k, int64_t n) const {
    const int64_t tb = t < n - 1 ? t : n - 1;
    if (NG == 1) return base + (t + k < n ? t + k : n - 1) * st;
    const int64_t most = n - 1 - tb;
    const uint32_t d = (uint32_t)(ls + k < most ? ls + k : most);
    return base + tb * st + (d * (uint32_t)st + (uint32_t)c);
  }
};
// the first step of a wave (NG == 1: of a thread) in a tile
template <int LC, int NG, int K>
__device__ __forceinline__ int64_t wave_step(int tile) {
  return NG == 1 ? (int64_t)tile * K : (int64_t)tile * (NG * K) + wave_id() * (64 / LC) * K;
}

// floats of NT values a channel and wave; kernels that join tile after tile use two in turn, so that
// one barrier a tile is enough
template <int LC, int NG, int V, int NT>
struct ScanLds {
  static constexpr int FLOATS = NG == 1 ? 1 : NG / (64 / LC) * NT * LC * V;
};

// s behind the segments from .. to - 1 (against time for !UP), whose (A, H) are in the workspace:
// every group joins a run of them, the groups are joined as those of a tile.  lds: the buffer that
// the first tile does not use.
template <class E, int LC, int NG, bool PART, bool UP>
__device__ __forceinline__ void segment_fold(const RecArgs& a, const Place<E, LC, NG, PART>& p,
                                             int from, int to, int64_t ch, float* s, float* lds) {
  constexpr int V = VC<E>::V;
  const int per = (to - from + NG - 1) / NG;
  const int lo = min(to, from + p.grp * per), hi = min(to, lo + per);
  float A[V], H[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    A[j] = 1.f;
    H[j] = 0.f;
  }
  for (int k = 0; k < hi - lo; ++k) {
    float A2[V], H2[V];
    const float* w = a.ws + (int64_t)(UP ? lo + k : hi - 1 - k) * 2 * a.B * a.D + ch;
    load_n<V, PART>(A2, w, p.nv);
    load_n<V, PART>(H2, w + a.B * a.D, p.nv);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      join(A[j], H[j], A2[j], H2[j]);
      A[j] = A2[j];
      H[j] = H2[j];
    }
  }
  tile_total<LC, NG, V, UP>(A, H, lds);
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = pass(s[j], A[j], H[j]);
}

}  // namespace

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------
template <class E, int LC, int NG, int K, bool PART>
__global__ void __launch_bounds__(LC * NG) rec_fwd_kernel(const RecArgs a) {
  constexpr int V = VC<E>::V, STEPS = NG * K;
  typedef typename E::T X;
  __shared__ __attribute__((aligned(16))) float lds[2][ScanLds<LC, NG, V, 2>::FLOATS];
  const Place<E, LC, NG, PART> p(a);
  typedef Rows<E, LC, NG, K, const X*> In;
  const In rv_((const X*)a.v, p.b, a.v_sb, a.v_st, p.cl), rg_((const X*)a.g, p.b, a.g_sb, a.g_st, p.cl);
  const Rows<E, LC, NG, K, X*> rh_((X*)a.h, p.b, a.T * a.D, a.D, p.c0);
  const int64_t ch = p.b * a.D + p.c0;
  const int t0 = p.seg * a.tps, t1 = min(a.tiles, t0 + a.tps);

  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  if (a.h0) load_n<V, PART>(s, a.h0 + ch, p.nv);
  if (NG > 1 && p.seg > 0)
    segment_fold<E, LC, NG, PART, true>(a, p, 0, p.seg, ch, s, lds[(t0 & 1) ^ 1]);

  Half nv_[K], ng_[K];
  // (whole: every step of the tile is part of the sequence)
  auto load = [&](int tile, auto whole) __attribute__((always_inline)) {
    constexpr bool W = decltype(whole)::value;
    const int64_t t = wave_step<LC, NG, K>(tile);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      load8<E, PART>(nv_[k], W ? rv_.at(t, k) : rv_.in(t, k, p.n), p.nv);
      load8<E, PART>(ng_[k], W ? rg_.at(t, k) : rg_.in(t, k, p.n), p.nv);
    }
  };
  // one tile; next: starts the next tile's loads, in between
  auto run = [&](int tile, auto whole, auto next) __attribute__((always_inline)) {
    constexpr bool W = decltype(whole)::value;
    const int64_t t = wave_step<LC, NG, K>(tile);
    Half rv[K];
    float in[K][V], A[V], H[V], st[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      A[j] = 1.f;
      H[j] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float g[V], v[V];
      if (!W) {
        mask8(nv_[k], t + rv_.ls + k < p.n, 0u);
        mask8(ng_[k], t + rv_.ls + k < p.n, ShutGate<E>::W);
      }
      rv[k] = nv_[k];
      E::template unpack<2>(ng_[k].w, g);
      E::template unpack<2>(rv[k].w, v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float w = in[k][j] = rec_gate<E>(g[j]);
        const bool shut = g[j] < 0.f;
        H[j] = gate_step(w, shut, H[j], v[j], H[j] - v[j]);
        A[j] = gate_keep(w, shut, A[j]);
      }
    }
    if (a.states && p.grp == 0)
      store_n<V, PART>(a.states + (p.b * a.tiles + tile) * a.D + p.c0, s, p.nv);
    next();
    tile_scan<LC, NG, V>(A, H, s, st, lds[tile & 1]);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float v[V], o[V];
      E::template unpack<2>(rv[k].w, v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        st[j] = gate_step(in[k][j], gate_shut(in[k][j]), st[j], v[j], st[j] - v[j]);
        o[j] = W || t + rh_.ls + k < p.n ? st[j] : 0.f;
      }
      if (W || t + rh_.ls + k < a.T) store8<E, PART>(rh_.at(t, k), o, p.nv);
    }
  };
  // whole tiles up to tw, then those with the sequence's end inside, up to te, then nothing to read
  const int tw = NG == 1 ? t0 : max(t0, (int)min((int64_t)t1, p.n / STEPS));
  const int te = (int)min((int64_t)t1, (p.n + STEPS - 1) / STEPS);
  if (tw > t0 + 1) {
    // (the first by itself: the loop then starts with as many stores in flight as it goes on with)
    load(t0, Yes());
    run(t0, Yes(), [&]() { load(t0 + 1, Yes()); });
    for (int tile = t0 + 1; tile + 1 < tw; ++tile) run(tile, Yes(), [&]() { load(tile + 1, Yes()); });
  } else if (tw > t0) {
    load(t0, Yes());
  }
  if (tw > t0) run(tw - 1, Yes(), [&]() { if (te > tw) load(tw, No()); });
  else if (te > t0) load(t0, No());
  for (int tile = tw; tile < te; ++tile) run(tile, No(), [&]() { if (tile + 1 < te) load(tile + 1, No()); });
  for (int tile = max(te, t0); tile < t1; ++tile) {
    const int64_t t = wave_step<LC, NG, K>(tile);
    const float zero[V] = {};
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (t + rh_.ls + k < a.T) store8<E, PART>(rh_.at(t, k), zero, p.nv);
  }
  if (p.grp == 0 && t1 == a.tiles) store_n<V, PART>(a.last + ch, s, p.nv);
}

// (A, H) of every segment but the last (backward: of every one but the first, over dh, against
// time).  A group takes one run of consecutive steps of the segment, so the runs are joined once.
template <class E, int LC, int NG, int K, bool FWD, bool PART>
__global__ void __launch_bounds__(LC * NG) rec_sum_kernel(const RecArgs a) {
  constexpr int V = VC<E>::V, STEPS = NG * K;
  typedef typename E::T X;
  __shared__ __attribute__((aligned(16))) float lds[ScanLds<LC, NG, V, 2>::FLOATS];
  Place<E, LC, NG, PART> p(a);
  if (!FWD) p.seg += 1;
  // (no dh: the gates' rows are read in its place, and not used)
  const bool none = !FWD && !a.dh;
  const X* gp = (const X*)a.g + p.b * a.g_sb + p.cl;
  const X* xp = FWD ? (const X*)a.v + p.b * a.v_sb + p.cl
                    : none ? gp : (const X*)a.dh + p.b * a.dh_sb + p.cl;
  const int64_t x_st = FWD ? a.v_st : none ? a.g_st : a.dh_st;
  const int run = a.tps * K;  // steps of a group
  const bool whole = (int64_t)(p.seg + 1) * a.tps * STEPS <= p.n;
  const int64_t first = (int64_t)p.seg * a.tps * STEPS + (int64_t)p.grp * run;
  float A[V], H[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    A[j] = 1.f;
    H[j] = 0.f;
  }
  // (a segment wholly behind the end changes nothing)
  const int rounds = (int64_t)p.seg * a.tps * STEPS < p.n ? a.tps : 0;
  for (int q = 0; q < rounds; ++q) {
    Half rx[K], rg[K];
    const int64_t t = first + (FWD ? q * K : run - 1 - q * K);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t tk = FWD ? t + k : t - k;
      const bool in = whole || tk < p.n;
      load8<E, PART>(rx[k], in ? xp + tk * x_st : xp, p.nv);
      load8<E, PART>(rg[k], in ? gp + tk * a.g_st : gp, p.nv);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float g[V], x[V];
      const bool in = whole || (FWD ? t + k : t - k) < p.n;
      mask8(rx[k], in && !none, 0u);
      mask8(rg[k], in, ShutGate<E>::W);
      E::template unpack<2>(rg[k].w, g);
      E::template unpack<2>(rx[k].w, x);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float w = rec_gate<E>(g[j]);
        const bool shut = g[j] < 0.f;
        H[j] = FWD ? gate_step(w, shut, H[j], x[j], H[j] - x[j]) : gate_keep(w, shut, x[j] + H[j]);
        A[j] = gate_keep(w, shut, A[j]);
      }
    }
  }
  tile_total<LC, NG, V, FWD>(A, H, lds);
  if (p.grp == 0) {
    float* w = a.ws + (int64_t)p.seg * 2 * a.B * a.D + p.b * a.D + p.c0;
    store_n<V, PART>(w, A, p.nv);
    store_n<V, PART>(w + a.B * a.D, H, p.nv);
  }
}

// ---------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------
// (two waves a SIMD: a register more than its 256 would leave the short forms one)
template <class E, int LC, int NG, int K, bool PART>
__global__ void __launch_bounds__(LC * NG, 2) rec_bwd_kernel(const RecArgs a) {
  constexpr int V = VC<E>::V, STEPS = NG * K;
  typedef typename E::T X;
  __shared__ __attribute__((aligned(16))) float lds[2][ScanLds<LC, NG, V, 3>::FLOATS];
  const Place<E, LC, NG, PART> p(a);
  typedef Rows<E, LC, NG, K, const X*> In;
  typedef Rows<E, LC, NG, K, X*> Out;
  // (no dh: the gates' rows are read in its place, and not used)
  const bool none = !a.dh;
  const In rv_((const X*)a.v, p.b, a.v_sb, a.v_st, p.cl), rg_((const X*)a.g, p.b, a.g_sb, a.g_st, p.cl),
      rd_((const X*)(none ? a.g : a.dh), p.b, none ? a.g_sb : a.dh_sb, none ? a.g_st : a.dh_st, p.cl);
  const Out rdv_((X*)a.dv, p.b, a.dv_sb, a.dv_st, p.c0), rdg_((X*)a.dg, p.b, a.dg_sb, a.dg_st, p.c0);
  const int64_t ch = p.b * a.D + p.c0;
  const int t0 = p.seg * a.tps, t1 = min(a.tiles, t0 + a.tps);

  float r[V];  // the gradient from behind the tile
#pragma unroll
  for (int j = 0; j < V; ++j) r[j] = 0.f;
  if (a.dlast) load_n<V, PART>(r, a.dlast + ch, p.nv);
  // tiles wholly behind the sequence's end: nothing to read
  const int te = (int)min((int64_t)t1, (p.n + STEPS - 1) / STEPS);
  if (NG > 1 && p.seg + 1 < a.segs)
    segment_fold<E, LC, NG, PART, false>(a, p, p.seg + 1, a.segs, ch, r, lds[te & 1]);

  Half nv_[K], ng_[K], nd_[K];
  float ns[V];
#pragma unroll
  for (int j = 0; j < V; ++j) ns[j] = 0.f;
  auto load = [&](int tile, auto whole) __attribute__((always_inline)) {
    constexpr bool W = decltype(whole)::value;
    const int64_t t = wave_step<LC, NG, K>(tile);
    if (a.states) load_n<V, PART>(ns, a.states + (p.b * a.tiles + tile) * a.D + p.c0, p.nv);
    else if (a.h0) load_n<V, PART>(ns, a.h0 + ch, p.nv);  // one tile
#pragma unroll
    for (int k = 0; k < K; ++k) {
      load8<E, PART>(ng_[k], W ? rg_.at(t, k) : rg_.in(t, k, p.n), p.nv);
      load8<E, PART>(nv_[k], W ? rv_.at(t, k) : rv_.in(t, k, p.n), p.nv);
      load8<E, PART>(nd_[k], W ? rd_.at(t, k) : rd_.in(t, k, p.n), p.nv);
    }
  };
  // one tile; next: starts the loads of the tile in front, in between
  auto run = [&](int tile, auto whole, auto next) __attribute__((always_inline)) {
    constexpr bool W = decltype(whole)::value;
    const int64_t t = wave_step<LC, NG, K>(tile);
    Half rd[K];
    float in[K][V], e[K][V], A[V], H[V], G[V], s[V], st[V], rt[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      A[j] = 1.f;
      H[j] = G[j] = 0.f;
      s[j] = ns[j];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float g[V];
      const bool in_k = W || t + rv_.ls + k < p.n;
      if (!W) {
        mask8(ng_[k], in_k, ShutGate<E>::W);
        mask8(nv_[k], in_k, 0u);
      }
      mask8(nd_[k], in_k && !none, 0u);
      rd[k] = nd_[k];
      E::template unpack<2>(ng_[k].w, g);
      E::template unpack<2>(nv_[k].w, e[k]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float w = in[k][j] = rec_gate<E>(g[j]);
        const bool shut = g[j] < 0.f;
        H[j] = gate_step(w, shut, H[j], e[k][j], H[j] - e[k][j]);
        A[j] = gate_keep(w, shut, A[j]);
      }
    }
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
      float d[V];
      E::template unpack<2>(rd[k].w, d);
#pragma unroll
      for (int j = 0; j < V; ++j) G[j] = gate_keep(in[k][j], gate_shut(in[k][j]), d[j] + G[j]);
    }
    next();
    tile_scan_both<LC, NG, V>(A, H, G, s, r, st, rt, lds[tile & 1]);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float w = in[k][j], v = e[k][j];
        e[k][j] = st[j] - v;  // h_{t-1} - v_t
        st[j] = gate_step(w, gate_shut(w), st[j], v, e[k][j]);
      }
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
      float d[V], gv[V], gg[V];
      const bool in_k = W || t + rv_.ls + k < p.n;  // (behind the end also an infinite gradient stands still)
      E::template unpack<2>(rd[k].w, d);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // the smaller and the larger part of x, f x and i x or the other way round
        const float w = gate_again(in[k][j]), m = fabsf(w), x = d[j] + rt[j], lo = m * x, hi = fmaf(-m, x, x);
        const bool shut = gate_shut(w);
        gv[j] = !in_k ? 0.f : shut ? hi : lo;
        gg[j] = in_k ? m * hi * e[k][j] : 0.f;
        rt[j] = !in_k ? rt[j] : shut ? lo : hi;
      }
      if (W || t + rdv_.ls + k < a.T) {
        store8<E, PART>(rdv_.at(t, k), gv, p.nv);
        store8<E, PART>(rdg_.at(t, k), gg, p.nv);
      }
    }
  };
  for (int tile = max(te, t0); tile < t1; ++tile) {
    const int64_t t = wave_step<LC, NG, K>(tile);
    const float zero[V] = {};
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (t + rdv_.ls + k < a.T) {
        store8<E, PART>(rdv_.at(t, k), zero, p.nv);
        store8<E, PART>(rdg_.at(t, k), zero, p.nv);
      }
  }
  // those with the sequence's end inside, then whole ones from tw on
  const int tw = NG == 1 ? t0 : max(t0, (int)min((int64_t)t1, p.n / STEPS));
  if (te > tw) {
    load(te - 1, No());
    for (int tile = te - 1; tile > tw; --tile) run(tile, No(), [&]() { load(tile - 1, No()); });
    run(tw, No(), [&]() { if (tw > t0) load(tw - 1, Yes()); });
  } else if (tw > t0) {
    load(tw - 1, Yes());
  }
  if (tw > t0 + 1) {
    // (the first by itself: the loop then starts with as many stores in flight as it goes on with)
    run(tw - 1, Yes(), [&]() { load(tw - 2, Yes()); });
    for (int tile = tw - 2; tile > t0; --tile) run(tile, Yes(), [&]() { load(tile - 1, Yes()); });
  }
  if (tw > t0) run(t0, Yes(), [&]() {});
  if (p.grp == 0 && t0 == 0 && a.dh0) store_n<V, PART>(a.dh0 + ch, r, p.nv);
}

// ---------------------------------------------------------------------------------------------
// one step
// ---------------------------------------------------------------------------------------------
template <class E>
__global__ void __launch_bounds__(256) rec_step_kernel(const RecArgs a, float* new_state) {
  constexpr int V = VC<E>::V;
  typedef typename E::T X;
  const int nch = (a.D + V - 1) / V;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.B * nch) return;
  const int64_t b = id / nch;
  const int c0 = (int)(id % nch) * V, nv = a.D - c0;
  float s[V], v[V], g[V];
  Half rv, rg;
  load8<E, true>(rv, (const X*)a.v + b * a.v_sb + c0, nv);
  load8<E, true>(rg, (const X*)a.g + b * a.g_sb + c0, nv);
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  if (a.h0) load_n<V, true>(s, a.h0 + b * a.D + c0, nv);
  E::template unpack<2>(rv.w, v);
  E::template unpack<2>(rg.w, g);
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = gate_step(rec_gate<E>(g[j]), g[j] < 0.f, s[j], v[j], s[j] - v[j]);
  store8<E, true>((X*)a.h + b * a.D + c0, s, nv);
  store_n<V, true>(new_state + b * a.D + c0, s, nv);
}

// ---------------------------------------------------------------------------------------------
// Launch plans, a function of the element size, B, T and D alone (the backward finds the states
// where the forward's plan put them).
// ---------------------------------------------------------------------------------------------
namespace {

//   FLAT  tiles of 8 steps, a thread per 8 bytes of channels, nothing to join: T <= 8, or narrow rows
//         and threads enough to hide that each of them waits for its own loads
//   SLIM  rows of up to 64 bytes: tiles of 64 steps x 32 bytes of channels, one wave
//   SLIM_LONG  the same with 1024 steps, 512 threads, for long sequences
//   SHORT T <= 32: tiles of 32 steps x 128 bytes of channels, one wave
//   WAVE  tiles of 64 steps x 128 bytes of channels, 128 threads, several workgroups a compute unit:
//         short sequences, or middling ones of many workgroups, whose first loads then overlap
//   LONG  256 steps x 128 bytes, 512 threads, one workgroup a compute unit
//   WIDE  128 steps x 256 bytes, 512 threads: rows are read in longer pieces, which memory likes, but
//         it takes twice the channels for as many workgroups, and an odd number of 128 bytes leaves
//         half of a tile beyond the width
// Forward + backward, us, bf16 (number of 128-byte tiles), and fp32 rows of the same bytes:
//                                          WAVE   LONG   WIDE      WAVE   LONG   WIDE
//   1024 x   50 x 1024 (16384)              218    959    491       193    655    350
//    256 x  256 x 1024 (4096)               224    275    254       227    232    225
//    128 x  512 x  512 (1024)               122    143    119       118    119    108
//     64 x 1024 x 2048 (2048)               487    465    422       480    435    415
//     12 x 4096 x 2048 (384)                495    393    367       410    372    342
//     60 x 2000 x  512 (480)                262    234    205       237    222    201
//     60 x 2000 x  520 (540)                344    331    361       335    302    329
//    100 x 1000 x  264 (500)                145    131    185       120    112    154
//      8 x 4096 x 2048 (256)                340    252    294       279    246    282
//     37 x  300 x  333 (222)                 87     50     70        42     31     48
// narrow rows                     FLAT   SLIM   SLIM_LONG   the best of the others
//  12000 x    16 x  8               19     49      669        74 (SHORT)
//   5000 x    20 x 32               26     43      574        38 (SHORT)
//  20000 x    50 x  8               56     76     1137       192 (SHORT)     SLIM is taken
//   9000 x   100 x 16               90     72      537       156 (SHORT)
//  40000 x    50 x 16 fp32         241    286     3157       296 (SHORT)
//    512 x    50 x 16               43     11       33        17 (WAVE)
//     64 x   100 x 16               75     14       18        17 (LONG)
//    512 x   300 x 16              210     28       36        50 (WAVE)
//    512 x   300 x  8 fp32         152     24       28        36 (WAVE)
//     32 x   300 x 16              208     25       18        29 (LONG)
//    512 x  1000 x 16              675     67       47        97 (LONG)
//    512 x  1000 x  8 fp32         485     56       39        67 (LONG)
//    256 x  4000 x 32             2722    231      153       179 (LONG)
//     16 x  4000 x 32             2673    219       35        32 (LONG)      SLIM_LONG is taken
//     64 x 20000 x  8            13346   1057      103       299 (LONG)
//     64 x 20000 x  4 fp32        9555    835       88       230 (LONG)
// Up to 128 workgroups the time axis is cut so that there are at most 256, one round (1 x 65521 x 1000
// fp16 forward, WIDE: 139 us with 32 segments, 256 workgroups; 218 with 128 workgroups, 141 with 512 in
// two rounds); above 128 a cut would read the input twice to fill less than half of the chip more.
enum { REC_FLAT, REC_SHORT, REC_WAVE, REC_LONG, REC_WIDE, REC_SLIM, REC_SLIM_LONG };
struct RecPlan {
  int kind, steps;  // steps: of a time tile
  int nct, segs, tps;
  int64_t tiles;
};

RecPlan rec_plan(int dtype, int64_t B, int64_t T, int D) {
  const int V = dtype == RS_F32 ? 2 : 4;
  const int n4 = (D + 4 * V - 1) / (4 * V), n16 = (D + 16 * V - 1) / (16 * V), n32 = (n16 + 1) / 2;
  const int64_t b16 = B * n16, b32 = B * n32;  // channel tiles
  // (a cut sequence has workgroups enough either way)
  const bool wide = n16 % 2 == 0 && (b32 >= 160 || (b16 <= 128 && n16 >= 8));
  const int64_t threads = B * ((D + V - 1) / V);  // of FLAT
  const bool flat = n4 <= 2 && (T <= 32 ? threads >= 16384 : T <= 512 && threads >= 65536);
  const bool slim = n4 == 1 || (n4 == 2 && T > 32);
  RecPlan p;
  if (T <= 8 || flat) p.kind = REC_FLAT;
  else if (slim) p.kind = T <= 128 || (T <= 512 && B * n4 >= 256) ? REC_SLIM : REC_SLIM_LONG;
  else if (T <= 32) p.kind = REC_SHORT;
  else if (T <= 64 || (T <= 512 && b16 >= 512)) p.kind = REC_WAVE;
  else p.kind = wide ? REC_WIDE : REC_LONG;
  constexpr int STEPS[] = {8, 32, 64, 256, 128, 64, 1024};  // by kind
  p.steps = STEPS[p.kind];
  p.nct = p.kind == REC_WIDE ? n32 : p.kind >= REC_SLIM ? n4 : n16;
  p.tiles = (T + p.steps - 1) / p.steps;
  p.segs = 1;
  p.tps = (int)p.tiles;
  const int64_t blocks = B * p.nct;  // 0 for an empty batch, which has nothing to cut
  const bool cut = p.kind == REC_LONG || p.kind == REC_WIDE || p.kind == REC_SLIM_LONG;
  if (cut && blocks > 0 && blocks <= 128 && p.tiles > 1) {
    const int64_t want = 256 / blocks;
    p.tps = (int)((p.tiles + want - 1) / want);
    p.segs = (int)((p.tiles + p.tps - 1) / p.tps);
  }
  return p;
}

// Whether the backward starts a tile from a kept state rather than from h0.  SLIM_LONG keeps that of its
// only tile too (B D floats): a backward of long rows without states is refused whatever their width.
bool rec_keeps_states(const RecPlan& p) { return p.tiles > 1 || p.kind == REC_SLIM_LONG; }

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
    const int64_t n = a.B * ((a.D + VC<E>::V - 1) / VC<E>::V);
    rec_fwd_kernel<E, 64, 1, 8, PART><<<(unsigned)((n + 63) / 64), 64, 0, s>>>(a);
  } else if (p.kind == REC_SHORT) {
    rec_fwd_kernel<E, 16, 4, 8, PART><<<per, 64, 0, s>>>(a);
  } else if (p.kind == REC_WAVE) {
    rec_fwd_kernel<E, 16, 8, 8, PART><<<per, 128, 0, s>>>(a);
  } else if (p.kind == REC_LONG) {
    if (p.segs > 1) rec_sum_kernel<E, 16, 32, 8, true, PART><<<per * (p.segs - 1), 512, 0, s>>>(a);
    rec_fwd_kernel<E, 16, 32, 8, PART><<<per * p.segs, 512, 0, s>>>(a);
  } else if (p.kind == REC_SLIM) {
    rec_fwd_kernel<E, 4, 16, 4, PART><<<per, 64, 0, s>>>(a);
  } else if (p.kind == REC_SLIM_LONG) {
    if (p.segs > 1) rec_sum_kernel<E, 4, 128, 8, true, PART><<<per * (p.segs - 1), 512, 0, s>>>(a);
    rec_fwd_kernel<E, 4, 128, 8, PART><<<per * p.segs, 512, 0, s>>>(a);
  } else {
    if (p.segs > 1) rec_sum_kernel<E, 32, 16, 8, true, PART><<<per * (p.segs - 1), 512, 0, s>>>(a);
    rec_fwd_kernel<E, 32, 16, 8, PART><<<per * p.segs, 512, 0, s>>>(a);
  }
  return rs_status_after_launch();
}

template <class E, bool PART>
int rec_bwd_as(hipStream_t s, const RecPlan& p, const RecArgs& a) {
  const unsigned per = (unsigned)(a.B * a.nct);
  if (p.kind == REC_FLAT) {
    const int64_t n = a.B * ((a.D + VC<E>::V - 1) / VC<E>::V);
    rec_bwd_kernel<E, 64, 1, 8, PART><<<(unsigned)((n + 63) / 64), 64, 0, s>>>(a);
  } else if (p.kind == REC_SHORT) {
    rec_bwd_kernel<E, 16, 4, 8, PART><<<per, 64, 0, s>>>(a);
  } else if (p.kind == REC_WAVE) {
    rec_bwd_kernel<E, 16, 8, 8, PART><<<per, 128, 0, s>>>(a);
  } else if (p.kind == REC_LONG) {
    if (p.segs > 1) rec_sum_kernel<E, 16, 32, 8, false, PART><<<per * (p.segs - 1), 512, 0, s>>>(a);
    rec_bwd_kernel<E, 16, 32, 8, PART><<<per * p.segs, 512, 0, s>>>(a);
  } else if (p.kind == REC_SLIM) {
    rec_bwd_kernel<E, 4, 16, 4, PART><<<per, 64, 0, s>>>(a);
  } else if (p.kind == REC_SLIM_LONG) {
    if (p.segs > 1) rec_sum_kernel<E, 4, 128, 8, false, PART><<<per * (p.segs - 1), 512, 0, s>>>(a);
    rec_bwd_kernel<E, 4, 128, 8, PART><<<per * p.segs, 512, 0, s>>>(a);
  } else {
    if (p.segs > 1) rec_sum_kernel<E, 32, 16, 8, false, PART><<<per * (p.segs - 1), 512, 0, s>>>(a);
    rec_bwd_kernel<E, 32, 16, 8, PART><<<per * p.segs, 512, 0, s>>>(a);
  }
  return rs_status_after_launch();
}

template <class E>
int rec_fwd(hipStream_t s, const RecPlan& p, const RecArgs& a) {
  return a.D % VC<E>::V ? rec_fwd_as<E, true>(s, p, a) : rec_fwd_as<E, false>(s, p, a);
}
template <class E>
int rec_bwd(hipStream_t s, const RecPlan& p, const RecArgs& a) {
  return a.D % VC<E>::V ? rec_bwd_as<E, true>(s, p, a) : rec_bwd_as<E, false>(s, p, a);
}

template <class E>
int rec_step(hipStream_t s, const RecArgs& a, float* new_state) {
  const int64_t n = a.B * ((a.D + VC<E>::V - 1) / VC<E>::V);
  rec_step_kernel<E><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a, new_state);
  return rs_status_after_launch();
}

// a wave's 128 steps (SLIM_LONG) of 2^23 elements: 2^32 bytes of fp32, which a lane's 32-bit offset holds.
// The step stride of a single step is never used.
bool rec_strides_ok(int64_t T, int64_t a, int64_t b, int64_t c, int D) {
  return D < (1 << 23) && (T <= 1 || (a < (1 << 23) && b < (1 << 23) && c < (1 << 23)));
}

// what the launches index: workgroups and time tiles in 31 bits
bool rec_shape_ok(int dtype, int64_t B, int64_t T, int D) {
  return dtype >= RS_F32 && dtype <= RS_F16 && B >= 0 && T >= 0 && D > 0 && T < (1ll << 31) &&
         B < (1ll << 30) && B * ((D + 31) / 32) < (1ll << 30);
}

}  // namespace

RS_API int64_t rs_gated_rec_states_floats(int dtype, int64_t B, int64_t T, int D) {
  if (!rec_shape_ok(dtype, B, T, D)) return 0;
  const RecPlan p = rec_plan(dtype, B, T, D);
  return rec_keeps_states(p) ? B * p.tiles * D : 0;
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
  if (!rec_strides_ok(T, v_st, g_st, 0, D)) return RS_ERR_UNSUPPORTED;
  const int64_t need = rs_gated_rec_workspace_floats(dtype, B, T, D);
  if (need > 0 && (!workspace || workspace_floats < need)) return RS_ERR_ARG;
  const RecPlan p = rec_plan(dtype, B, T, D);
  RecArgs a = {};
  rec_fill(a, p, B, T, D);
  a.v = v, a.v_sb = v_sb, a.v_st = v_st;
  a.g = g, a.g_sb = g_sb, a.g_st = g_st;
  a.lengths = lengths, a.h0 = h0, a.h = h, a.last = last, a.ws = workspace;
  a.states = rec_keeps_states(p) ? states : nullptr;
  return RS_DISPATCH_ELEM(dtype, rec_fwd, rs_stream(stream), p, a);
}

RS_API int rs_gated_rec_bwd(void* stream, int dtype, const void* v, int64_t v_sb, int64_t v_st,
                            const void* g, int64_t g_sb, int64_t g_st, int64_t B, int64_t T, int D,
                            const int32_t* lengths, const float* h0, const float* states,
                            const void* dh, int64_t dh_sb, int64_t dh_st, const float* dlast, void* dv,
                            int64_t dv_sb, int64_t dv_st, void* dg, int64_t dg_sb, int64_t dg_st,
                            float* dh0, float* workspace, int64_t workspace_floats) {
  if (!rec_shape_ok(dtype, B, T, D)) return RS_ERR_ARG;
  if (B == 0) return RS_OK;
  if (T > 0 && (!v || !g || !dv || !dg || v_sb < 0 || v_st < 0 || g_sb < 0 ||
                g_st < 0 || dh_sb < 0 || dh_st < 0 || (T > 1 && (dv_st < D || dg_st < D)) ||
                (B > 1 && (dv_sb < D || dg_sb < D))))
    return RS_ERR_ARG;
  if (T == 0 && !dh0) return RS_OK;
  const bool kept = rs_gated_rec_states_floats(dtype, B, T, D) > 0;
  if (kept && !states) return RS_ERR_ARG;
  if (!rec_strides_ok(T, v_st, g_st, dh_st, D) || !rec_strides_ok(T, dv_st, dg_st, 0, D))
    return RS_ERR_UNSUPPORTED;
  const int64_t need = rs_gated_rec_workspace_floats(dtype, B, T, D);
  if (need > 0 && (!workspace || workspace_floats < need)) return RS_ERR_ARG;
  const RecPlan p = rec_plan(dtype, B, T, D);
  RecArgs a = {};
  rec_fill(a, p, B, T, D);
  a.v = v, a.v_sb = v_sb, a.v_st = v_st;
  a.g = g, a.g_sb = g_sb, a.g_st = g_st;
  a.dh = dh, a.dh_sb = dh_sb, a.dh_st = dh_st;
  a.lengths = lengths, a.states = kept ? const_cast<float*>(states) : nullptr, a.h0 = h0;
  a.dlast = dlast;
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
