// Gated linear recurrence over [B, T, D] and its gradients, all channels independent:
//   i_t = sigmoid(-g_t) = 1 - f_t        h_t = f_t h_{t-1} + (1 - f_t) v_t = h_{t-1} + i_t (v_t - h_{t-1})
//   r_t = the gradient that reaches h_t from later steps, a_t = dh_t + r_t
//   dv_t = i_t a_t     dg_t = a_t (h_{t-1} - v_t) i_t (1 - i_t)     r_{t-1} = a_t - i_t a_t
// The state and its gradient are fp32 throughout.  Written with i rather than f: a gate that is
// almost open (f rounds to 1) still moves the state by its own small i.
// Steps from lengths[b] on are not read: h, dv and dg are zero there and the state stands still.
// The forward keeps the fp32 state in front of every RS_REC_INTERVAL-th step, from which the
// backward computes the states again; h itself, rounded to the rows' type, is not used.
#include "elem.hpp"

#define RS_REC_INTERVAL 16

namespace {
__device__ __forceinline__ float rec_input_gate(float g) {
  return __builtin_amdgcn_rcpf(1.0f + expf(g));  // exp = inf: 0
}
__device__ __forceinline__ int64_t rec_length(const int32_t* lengths, int64_t b, int64_t T) {
  if (!lengths) return T;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > T ? T : n);
}
}  // namespace

template <class E>
__global__ void __launch_bounds__(64) rec_fwd_kernel(
    const typename E::T* __restrict__ v, int64_t v_sb, int64_t v_st,
    const typename E::T* __restrict__ g, int64_t g_sb, int64_t g_st, int64_t B, int64_t T, int D,
    const int32_t* __restrict__ lengths, const float* __restrict__ h0,
    typename E::T* __restrict__ h, float* __restrict__ last, float* __restrict__ states) {
  const int64_t id = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (id >= B * D) return;
  const int64_t b = id / D, c = id % D, n = rec_length(lengths, b, T);
  const int64_t kept = (T + RS_REC_INTERVAL - 1) / RS_REC_INTERVAL;
  float s = h0 ? h0[id] : 0.f;
  for (int64_t t = 0; t < T; ++t) {
    if (states && t % RS_REC_INTERVAL == 0) states[(b * kept + t / RS_REC_INTERVAL) * D + c] = s;
    float out = 0.f;
    if (t < n) {
      const float i = rec_input_gate(E::load(g[b * g_sb + t * g_st + c]));
      out = s = fmaf(i, E::load(v[b * v_sb + t * v_st + c]) - s, s);
    }
    h[(b * T + t) * D + c] = E::store(out);
  }
  last[id] = s;
}

template <class E>
__global__ void __launch_bounds__(64) rec_bwd_kernel(
    const typename E::T* __restrict__ v, int64_t v_sb, int64_t v_st,
    const typename E::T* __restrict__ g, int64_t g_sb, int64_t g_st, int64_t B, int64_t T, int D,
    const int32_t* __restrict__ lengths, const float* __restrict__ states,
    const typename E::T* __restrict__ dh, int64_t dh_sb, int64_t dh_st,
    const float* __restrict__ dlast, typename E::T* __restrict__ dv, int64_t dv_sb, int64_t dv_st,
    typename E::T* __restrict__ dg, int64_t dg_sb, int64_t dg_st, float* __restrict__ dh0) {
  const int64_t id = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (id >= B * D) return;
  const int64_t b = id / D, c = id % D, n = rec_length(lengths, b, T);
  const int64_t kept = (T + RS_REC_INTERVAL - 1) / RS_REC_INTERVAL;
  float r = dlast ? dlast[id] : 0.f;
  for (int64_t k = kept - 1; k >= 0; --k) {
    float e[RS_REC_INTERVAL], in[RS_REC_INTERVAL];
    float s = states[(b * kept + k) * D + c];
#pragma unroll
    for (int j = 0; j < RS_REC_INTERVAL; ++j) {
      const int64_t t = k * RS_REC_INTERVAL + j;
      in[j] = e[j] = 0.f;
      if (t < n) {
        in[j] = rec_input_gate(E::load(g[b * g_sb + t * g_st + c]));
        e[j] = s - E::load(v[b * v_sb + t * v_st + c]);
        s = fmaf(-in[j], e[j], s);
      }
    }
#pragma unroll
    for (int j = RS_REC_INTERVAL - 1; j >= 0; --j) {
      const int64_t t = k * RS_REC_INTERVAL + j;
      if (t >= T) continue;
      float gv = 0.f, gg = 0.f;
      if (t < n) {
        const float a = r + (dh ? E::load(dh[b * dh_sb + t * dh_st + c]) : 0.f);
        gv = in[j] * a;
        gg = gv * e[j] * (1.0f - in[j]);
        r = a - gv;
      }
      dv[b * dv_sb + t * dv_st + c] = E::store(gv);
      dg[b * dg_sb + t * dg_st + c] = E::store(gg);
    }
  }
  if (dh0) dh0[id] = r;
}

template <class E>
__global__ void __launch_bounds__(256) rec_step_kernel(const typename E::T* __restrict__ v,
                                                       int64_t ldv,
                                                       const typename E::T* __restrict__ g,
                                                       int64_t ldg, int64_t B, int D,
                                                       const float* state,
                                                       typename E::T* __restrict__ h,
                                                       float* new_state) {
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < B * D;
       id += (int64_t)gridDim.x * 256) {
    const int64_t b = id / D, c = id % D;
    const float i = rec_input_gate(E::load(g[b * ldg + c])), s = state ? state[id] : 0.f;
    const float o = fmaf(i, E::load(v[b * ldv + c]) - s, s);
    h[id] = E::store(o);
    new_state[id] = o;
  }
}

template <class E>
static int rec_fwd(hipStream_t s, const void* v, int64_t v_sb, int64_t v_st, const void* g,
                   int64_t g_sb, int64_t g_st, int64_t B, int64_t T, int D, const int32_t* lengths,
                   const float* h0, void* h, float* last, float* states) {
  typedef typename E::T X;
  rec_fwd_kernel<E><<<(unsigned)((B * D + 63) / 64), 64, 0, s>>>(
      (const X*)v, v_sb, v_st, (const X*)g, g_sb, g_st, B, T, D, lengths, h0, (X*)h, last, states);
  return rs_status_after_launch();
}

template <class E>
static int rec_bwd(hipStream_t s, const void* v, int64_t v_sb, int64_t v_st, const void* g,
                   int64_t g_sb, int64_t g_st, int64_t B, int64_t T, int D, const int32_t* lengths,
                   const float* states, const void* dh, int64_t dh_sb, int64_t dh_st,
                   const float* dlast, void* dv, int64_t dv_sb, int64_t dv_st, void* dg,
                   int64_t dg_sb, int64_t dg_st, float* dh0) {
  typedef typename E::T X;
  rec_bwd_kernel<E><<<(unsigned)((B * D + 63) / 64), 64, 0, s>>>(
      (const X*)v, v_sb, v_st, (const X*)g, g_sb, g_st, B, T, D, lengths, states, (const X*)dh,
      dh_sb, dh_st, dlast, (X*)dv, dv_sb, dv_st, (X*)dg, dg_sb, dg_st, dh0);
  return rs_status_after_launch();
}

template <class E>
static int rec_step(hipStream_t s, const void* v, int64_t ldv, const void* g, int64_t ldg,
                    int64_t B, int D, const float* state, void* h, float* new_state) {
  typedef typename E::T X;
  const int64_t n = (B * D + 255) / 256;
  rec_step_kernel<E><<<(unsigned)(n < 65536 ? n : 65536), 256, 0, s>>>(
      (const X*)v, ldv, (const X*)g, ldg, B, D, state, (X*)h, new_state);
  return rs_status_after_launch();
}

// B, T, D within what the launches index: B * D threads in 2^31 workgroups, T in 31 bits
static bool rec_shape_ok(int dtype, int64_t B, int64_t T, int D) {
  return dtype >= RS_F32 && dtype <= RS_F16 && B >= 0 && T >= 0 && D > 0 && T < (1ll << 31) &&
         B < (1ll << 31) && B * (int64_t)D < (1ll << 36);
}

RS_API int64_t rs_gated_rec_states_floats(int dtype, int64_t B, int64_t T, int D) {
  if (!rec_shape_ok(dtype, B, T, D)) return 0;
  return B * ((T + RS_REC_INTERVAL - 1) / RS_REC_INTERVAL) * D;
}

RS_API int64_t rs_gated_rec_workspace_floats(int dtype, int64_t B, int64_t T, int D) {
  if (!rec_shape_ok(dtype, B, T, D)) return 0;
  return 0;
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
  return RS_DISPATCH_ELEM(dtype, rec_fwd, rs_stream(stream), v, v_sb, v_st, g, g_sb, g_st, B, T, D,
                          lengths, h0, h, last, states);
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
  return RS_DISPATCH_ELEM(dtype, rec_bwd, rs_stream(stream), v, v_sb, v_st, g, g_sb, g_st, B, T, D,
                          lengths, states, dh, dh_sb, dh_st, dlast, dv, dv_sb, dv_st, dg, dg_sb, dg_st, dh0);
}

RS_API int rs_gated_rec_step(void* stream, int dtype, const void* v, int64_t ld_v, const void* g,
                             int64_t ld_g, int64_t B, int D, const float* state, void* h,
                             float* new_state) {
  if (!rec_shape_ok(dtype, B, 1, D)) return RS_ERR_ARG;
  if (B == 0) return RS_OK;
  if (!v || !g || !h || !new_state || ld_v < 0 || ld_g < 0) return RS_ERR_ARG;
  return RS_DISPATCH_ELEM(dtype, rec_step, rs_stream(stream), v, ld_v, g, ld_g, B, D, state, h,
                          new_state);
}
