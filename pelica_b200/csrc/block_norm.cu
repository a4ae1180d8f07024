// block_norm.cu - the norms before and after a block, fused with the block's gate and the scaled residual stream, and
// their gradient.
//
// Forward, a row at a time (x the stream in front of the block, f the block's output):
//   p = f / sqrt(mean f^2 + e1) * (o1 + w_post)  (or f),   r = alpha x + beta g p,   n = r / sqrt(mean r^2 + e2) * (o2 + w_pre).
// n is made from r before r is rounded to the stream's type. Backward, from r, f and the gradients dr, dn that arrive at r and n,
// with s = 1 / sqrt(mean + e), u = dn (o2 + w_pre):
//   D = dr + s2 (u - r s2^2 mean(u r)),   dx = alpha D,   q = beta g D,   dg = beta sum D p,   dw_pre = sum_t dn r s2,
//   v = q (o1 + w_post),   df = s1 (v - f s1^2 mean(v f)),   dw_post = sum_t q f s1.
// Both norms' sums are made again from r and f: the forward keeps nothing. All sums in f32.
// Bound by HBM: 4 streams forward, 6 backward, a few operations a value.
#include <cooperative_groups.h>

#include "block_norm.cuh"
#include "vec.cuh"

namespace cg = cooperative_groups;

// A thread holds 8 values of a row; a row's group has tpr threads (whole warps) in each of cl CTAs (a cluster, for rows of
// more than 8,192 values), a CTA has rpb groups, each with rows of its own.
#define NORM_VALUES 8
struct NormShape {
  int tpr, rpb, cl;
};
static NormShape norm_shape(int d) {
  NormShape s;
  const int need = (d + NORM_VALUES - 1) / NORM_VALUES;
  s.cl = 1;
  while ((need + s.cl - 1) / s.cl > 1024) s.cl *= 2;
  s.tpr = ((need + s.cl - 1) / s.cl + 31) / 32 * 32;
  s.rpb = s.cl == 1 && s.tpr < 256 ? 256 / s.tpr : 1;
  return s;
}

// the group's place in the launch
struct NormPlace {
  int lane, warp, group, tpr, cl, rank, col0;
};

// Sums of N values over a row's group, in every thread: lanes, then warps through red (two turns used alternately,
// so that one barrier a sum is enough), then the cluster's CTAs.
template <int N, bool CLUSTER>
__device__ __forceinline__ void norm_sum(float (&v)[N], const NormPlace &at, float (*red)[32][N], float (*peer)[8][N], int &turn) {
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = pm_warp_sum_16_1(v[i]);
  const int warps = at.tpr >> 5;
  if (warps == 1 && !CLUSTER) return;
  float (*mine)[N] = red[turn] + at.group * warps;
  if (at.lane == 0) {
#pragma unroll
    for (int i = 0; i < N; i++) mine[at.warp][i] = v[i];
  }
  if constexpr (CLUSTER) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(at.group + 1), "r"(at.tpr) : "memory");
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = pm_warp_sum_16_1(at.lane < warps ? mine[at.lane][i] : 0.0f);
  if constexpr (CLUSTER) {
    cg::cluster_group cluster = cg::this_cluster();
    if (at.warp == 0 && at.lane < at.cl) {
      float *to = cluster.map_shared_rank(&peer[turn][at.rank][0], at.lane);
#pragma unroll
      for (int i = 0; i < N; i++) to[i] = v[i];
    }
    cluster.sync();
#pragma unroll
    for (int i = 0; i < N; i++) {
      float s = 0.0f;
      for (int q = 0; q < at.cl; q++) s = __fadd_rn(s, peer[turn][q][i]);
      v[i] = s;
    }
  }
  turn ^= 1;
}

__device__ __forceinline__ float norm_inv(float sum, int d, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)d), eps)));
}

// the thread's 8 values of a row as vectors of V: vector j is columns col0 + j * step ...
template <typename E, int V> struct NormRow {
  static constexpr int J = NORM_VALUES / V;
  Raw<E, V> v[J];
  __device__ __forceinline__ void load(const void *base, size_t at, const NormPlace &p, int d) {
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int col = p.col0 + j * p.tpr * p.cl * V;
      if (col < d) v[j] = pm_load<E, V>((const E *)base + at + col);
      else {
        const float z[V] = {};
        v[j] = pm_narrow<E, V>(z);
      }
    }
  }
  __device__ __forceinline__ void widen(float (&f)[NORM_VALUES]) const {
#pragma unroll
    for (int j = 0; j < J; j++) {
      float g[V];
      pm_widen<E, V>(v[j], g);
#pragma unroll
      for (int i = 0; i < V; i++) f[j * V + i] = g[i];
    }
  }
  __device__ __forceinline__ static void store(void *base, size_t at, const NormPlace &p, int d, const float (&f)[NORM_VALUES]) {
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int col = p.col0 + j * p.tpr * p.cl * V;
      float g[V];
#pragma unroll
      for (int i = 0; i < V; i++) g[i] = f[j * V + i];
      if (col < d) pm_store<E, V>((E *)base + at + col, pm_narrow<E, V>(g));
    }
  }
};
// weights of the thread's columns, offset added; `one` where there are none
template <typename W, int V>
__device__ __forceinline__ void norm_weights(float (&f)[NORM_VALUES], const void *w, float offset, const NormPlace &p, int d) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < NORM_VALUES; i++) f[i] = 1.0f;
    return;
  }
  NormRow<W, V> r;
  r.load(w, 0, p, d);
  r.widen(f);
#pragma unroll
  for (int i = 0; i < NORM_VALUES; i++) f[i] = __fadd_rn(f[i], offset);
}

template <bool CLUSTER> __device__ __forceinline__ NormPlace norm_place(int tpr, int cl, int v) {
  NormPlace p;
  p.tpr = tpr;
  p.cl = CLUSTER ? cl : 1;
  p.group = threadIdx.x / tpr;
  const int in = threadIdx.x - p.group * tpr;
  p.lane = in & 31;
  p.warp = in >> 5;
  p.rank = CLUSTER ? (int)(blockIdx.x % cl) : 0;
  p.col0 = (p.rank * tpr + in) * v;
  return p;
}

template <typename W> __device__ __forceinline__ float norm_token_gate(const NormCall &c, int t) {
  return c.D.gate == PM_NORM_GATE_TOKEN ? pm_to_f32(((const W *)c.gate)[t]) : 1.0f;
}

template <typename E, typename W, int V, bool CLUSTER>
__global__ void __launch_bounds__(1024) k_block_norm(NormCall c, int tpr, int rpb, int cl) {
  pm_pdl();
  __shared__ float red[2][32][1], peer[2][8][1];
  const NormPlace at = norm_place<CLUSTER>(tpr, cl, V);
  const int d = c.D.d, groups = (int)(gridDim.x / at.cl) * rpb;
  const bool post = c.D.flags & PM_NORM_POST, pre = c.D.flags & PM_NORM_PRE;
  float wp[NORM_VALUES], wn[NORM_VALUES];  // gate and post weight; pre weight
  norm_weights<W, V>(wp, post ? c.w_post : nullptr, c.D.offset_post, at, d);
  norm_weights<W, V>(wn, pre ? c.w_pre : nullptr, c.D.offset_pre, at, d);
  if (c.D.gate == PM_NORM_GATE_CHANNEL) {
    float g[NORM_VALUES];
    norm_weights<W, V>(g, c.gate, 0.0f, at, d);
#pragma unroll
    for (int i = 0; i < NORM_VALUES; i++) wp[i] = __fmul_rn(wp[i], g[i]);
  }
  int turn = 0;
  for (int t = (int)(blockIdx.x / at.cl) * rpb + at.group; t < c.T; t += groups) {
    NormRow<E, V> xr, fr;
    float r[NORM_VALUES], p[NORM_VALUES], sum[1];
    if (c.f) fr.load(c.f, (size_t)t * c.D.f_stride, at, d);
    if (c.x) xr.load(c.x, (size_t)t * c.D.x_stride, at, d);
    if (c.x) {
      xr.widen(r);
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) r[i] = __fmul_rn(c.D.alpha, r[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) r[i] = 0.0f;
    }
    if (c.f) {
      fr.widen(p);
      float s = __fmul_rn(c.D.beta, norm_token_gate<W>(c, t));
      if (post) {
        sum[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < NORM_VALUES; i++) sum[0] = __fmaf_rn(p[i], p[i], sum[0]);
        norm_sum<1, CLUSTER>(sum, at, red, peer, turn);
        const float inv = norm_inv(sum[0], d, c.D.eps_post);
#pragma unroll
        for (int i = 0; i < NORM_VALUES; i++) p[i] = __fmul_rn(p[i], inv);
      }
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) r[i] = __fmaf_rn(__fmul_rn(p[i], wp[i]), s, r[i]);
    }
    if (c.r) NormRow<E, V>::store(c.r, (size_t)t * c.D.r_stride, at, d, r);
    if (pre) {
      sum[0] = 0.0f;
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) sum[0] = __fmaf_rn(r[i], r[i], sum[0]);
      norm_sum<1, CLUSTER>(sum, at, red, peer, turn);
      const float inv = norm_inv(sum[0], d, c.D.eps_pre);
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) p[i] = __fmul_rn(__fmul_rn(r[i], inv), wn[i]);
      NormRow<E, V>::store(c.n, (size_t)t * c.D.n_stride, at, d, p);
    }
  }
  if constexpr (CLUSTER) cg::this_cluster().sync();  // no CTA leaves while another may still write its sums here
}

// Each group adds up the weights' gradients of its rows in registers; a CTA adds its groups and leaves a row of sums in
// parts[kind][CTA][d], which k_norm_sum_parts adds up. No atomics.
template <typename E, typename W, int V, bool CLUSTER>
__global__ void __launch_bounds__(1024) k_block_norm_grad(NormCall c, int tpr, int rpb, int cl) {
  pm_pdl();
  extern __shared__ float fold[];  // [threads][8]
  __shared__ float red3[2][32][3], peer3[2][8][3], red[2][32][1], peer[2][8][1];
  const NormPlace at = norm_place<CLUSTER>(tpr, cl, V);
  const int d = c.D.d, n_parts = (int)(gridDim.x / at.cl), part = (int)(blockIdx.x / at.cl), groups = n_parts * rpb;
  const bool post = c.D.flags & PM_NORM_POST, pre = c.D.flags & PM_NORM_PRE;
  const bool channel = c.D.gate == PM_NORM_GATE_CHANNEL;
  float a_pre[NORM_VALUES] = {}, a_post[NORM_VALUES] = {}, a_gate[NORM_VALUES] = {};
  float wp[NORM_VALUES], wn[NORM_VALUES], wg[NORM_VALUES];
  norm_weights<W, V>(wp, post ? c.w_post : nullptr, c.D.offset_post, at, d);
  norm_weights<W, V>(wn, pre ? c.w_pre : nullptr, c.D.offset_pre, at, d);
  norm_weights<W, V>(wg, channel ? c.gate : nullptr, 0.0f, at, d);
  int turn3 = 0, turn = 0;
  for (int t = part * rpb + at.group; t < c.T; t += groups) {
    NormRow<E, V> rr, fr, drr, dnr;
    float r[NORM_VALUES], f[NORM_VALUES], D[NORM_VALUES], u[NORM_VALUES];
    const size_t at_r = (size_t)t * c.D.r_stride, at_f = (size_t)t * c.D.f_stride;
    if (pre) {
      rr.load(c.x, at_r, at, d);
      dnr.load(c.dn, (size_t)t * c.D.n_stride, at, d);
    }
    if (c.f) fr.load(c.f, at_f, at, d);
    if (c.dr) {
      drr.load(c.dr, at_r, at, d);
      drr.widen(D);
    } else {
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) D[i] = 0.0f;
    }
    float sum[3] = {0.0f, 0.0f, 0.0f};
    if (pre) {
      rr.widen(r);
      dnr.widen(u);
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) {
        sum[0] = __fmaf_rn(r[i], r[i], sum[0]);
        sum[1] = __fmaf_rn(__fmul_rn(u[i], wn[i]), r[i], sum[1]);
      }
    }
    if (c.f) {
      fr.widen(f);
      if (post) {
#pragma unroll
        for (int i = 0; i < NORM_VALUES; i++) sum[2] = __fmaf_rn(f[i], f[i], sum[2]);
      }
    }
    if (pre || post) norm_sum<3, CLUSTER>(sum, at, red3, peer3, turn3);
    if (pre) {
      const float s2 = norm_inv(sum[0], d, c.D.eps_pre);
      const float m = __fmul_rn(__fmul_rn(s2, s2), __fdiv_rn(sum[1], (float)d));
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) {
        a_pre[i] = __fmaf_rn(u[i], __fmul_rn(r[i], s2), a_pre[i]);
        D[i] = __fmaf_rn(s2, __fmaf_rn(-r[i], m, __fmul_rn(u[i], wn[i])), D[i]);
      }
    }
    if (c.dx) {
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) u[i] = __fmul_rn(c.D.alpha, D[i]);
      NormRow<E, V>::store(c.dx, (size_t)t * c.D.x_stride, at, d, u);
    }
    if (!c.f) continue;
    const float s1 = post ? norm_inv(sum[2], d, c.D.eps_post) : 1.0f;
    const float gt = norm_token_gate<W>(c, t);
    // u = beta D, q = beta g D (g of the channel; the token's gate is one factor of the row)
    float dot[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NORM_VALUES; i++) {
      u[i] = __fmul_rn(c.D.beta, D[i]);
      const float pw = __fmul_rn(__fmul_rn(f[i], s1), wp[i]);
      if (channel) a_gate[i] = __fmaf_rn(u[i], pw, a_gate[i]);
      u[i] = __fmul_rn(u[i], wg[i]);
      dot[0] = __fmaf_rn(u[i], pw, dot[0]);
      a_post[i] = __fmaf_rn(__fmul_rn(u[i], gt), __fmul_rn(f[i], s1), a_post[i]);
    }
    if (post || c.D.gate == PM_NORM_GATE_TOKEN) norm_sum<1, CLUSTER>(dot, at, red, peer, turn);  // sum of u (f s1 w) over the row
    if (c.D.gate == PM_NORM_GATE_TOKEN && c.dgate && at.rank == 0 && at.warp == 0 && at.lane == 0) c.dgate[t] = dot[0];
    const float m = __fdiv_rn(__fmul_rn(dot[0], gt), (float)d);  // mean(v f) s1
#pragma unroll
    for (int i = 0; i < NORM_VALUES; i++) {
      const float q = __fmul_rn(u[i], gt);
      f[i] = post ? __fmul_rn(s1, __fmaf_rn(-__fmul_rn(f[i], s1), m, __fmul_rn(q, wp[i]))) : q;
    }
    if (c.df) NormRow<E, V>::store(c.df, at_f, at, d, f);
  }
  // the CTA's groups, kind by kind, columns of a thread as it holds them
#pragma unroll
  for (int kind = 0; kind < 3; kind++) {
    const bool on = kind == 0 ? pre && c.dw_pre : kind == 1 ? post && c.dw_post && c.f : channel && c.dgate;
    if (!on) continue;
    float *a = kind == 0 ? a_pre : kind == 1 ? a_post : a_gate;
    if (rpb > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NORM_VALUES; i++) fold[i * blockDim.x + threadIdx.x] = a[i];
      __syncthreads();
      if (at.group == 0)
        for (int g = 1; g < rpb; g++)
#pragma unroll
          for (int i = 0; i < NORM_VALUES; i++) a[i] = __fadd_rn(a[i], fold[i * blockDim.x + g * tpr + threadIdx.x]);
    }
    if (at.group == 0) {
      float *to = c.parts + ((size_t)kind * n_parts + part) * d;
#pragma unroll
      for (int j = 0; j < NORM_VALUES / V; j++) {
        const int col = at.col0 + j * tpr * at.cl * V;
#pragma unroll
        for (int i = 0; i < V; i++)
          if (col + i < d) to[col + i] = a[j * V + i];
      }
    }
  }
  if constexpr (CLUSTER) cg::this_cluster().sync();
}

// out[kind][col] = sum over the parts, 8 runs of parts a CTA of 32 columns, runs added in order
__global__ void __launch_bounds__(256) k_norm_sum_parts(const float *__restrict__ parts, int n_parts, int d, float *o0, float *o1, float *o2) {
  pm_pdl();
  __shared__ float red[8][32];
  float *out = blockIdx.y == 0 ? o0 : blockIdx.y == 1 ? o1 : o2;
  if (!out) return;
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  const float *p = parts + (size_t)blockIdx.y * n_parts * d;
  float s = 0.0f;
  if (col < d) {
#pragma unroll 4
    for (int i = run; i < n_parts; i += 8) s = __fadd_rn(s, p[(size_t)i * d + col]);
  }
  red[run][lane] = s;
  __syncthreads();
  if (run == 0 && col < d) {
#pragma unroll
    for (int i = 1; i < 8; i++) s = __fadd_rn(s, red[i][lane]);
    out[col] = s;
  }
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
// CTAs (clusters) of a call: rows there are, at most what 1,024 threads an SM make resident
static int norm_parts(const NormShape &s, int T, int n_sm) {
  const int per_sm = 1024 / (s.tpr * s.rpb);
  const int most = s.cl > 1 ? n_sm / s.cl : n_sm * (per_sm > 0 ? per_sm : 1);
  const int need = (T + s.rpb - 1) / s.rpb;
  return need < most ? need : most;
}
size_t norm_parts_floats(const pm_norm_desc &D, int T, int n_sm) { return (size_t)3 * norm_parts(norm_shape(D.d), T, n_sm) * D.d; }

template <typename... P>
static cudaError_t norm_launch(const Launch &L, void (*kern)(P...), int parts, const NormShape &s, size_t smem, NormCall c) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts * s.cl);
  cfg.blockDim = dim3(s.tpr * s.rpb);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = L.stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = s.cl;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = s.cl > 1 ? 2 : 1;
  if (L.count) ++*L.count;
  return cudaLaunchKernelEx(&cfg, kern, c, s.tpr, s.rpb, s.cl);
}

template <typename E, typename W, int V> static cudaError_t norm_forward(const Launch &L, const NormCall &c) {
  const NormShape s = norm_shape(c.D.d);
  const int parts = norm_parts(s, c.T, L.n_sm);
  return s.cl > 1 ? norm_launch(L, k_block_norm<E, W, V, true>, parts, s, 0, c) : norm_launch(L, k_block_norm<E, W, V, false>, parts, s, 0, c);
}
template <typename E, typename W, int V> static cudaError_t norm_backward(const Launch &L, const NormCall &c) {
  const NormShape s = norm_shape(c.D.d);
  const int parts = norm_parts(s, c.T, L.n_sm);
  const size_t fold = s.rpb > 1 ? (size_t)s.tpr * s.rpb * NORM_VALUES * sizeof(float) : 0;  // 8 KB: rpb is 1 from 256 threads on
  cudaError_t e = cudaSuccess;  // (no rows: the sums alone, zeros)
  if (parts) e = s.cl > 1 ? norm_launch(L, k_block_norm_grad<E, W, V, true>, parts, s, fold, c)
                          : norm_launch(L, k_block_norm_grad<E, W, V, false>, parts, s, fold, c);
  if (e != cudaSuccess) return e;
  float *channel = c.D.gate == PM_NORM_GATE_CHANNEL ? c.dgate : nullptr;
  if (!c.dw_pre && !c.dw_post && !channel) return cudaSuccess;
  return pm_launch(L, k_norm_sum_parts, dim3((c.D.d + 31) / 32, 3), 256, 0, (const float *)c.parts, parts, c.D.d, c.dw_pre, c.dw_post, channel);
}

#define NORM_TYPES(F)                                                                                                      \
  do {                                                                                                                     \
    const bool wide = c.D.wtype == PM_TYPE_F32;                                                                            \
    switch (c.D.dtype) {                                                                                                   \
      case PM_TYPE_F32: return c.vec ? F<float, float, 4>(L, c) : F<float, float, 1>(L, c);                                \
      case PM_TYPE_F16:                                                                                                    \
        if (wide) return c.vec ? F<__half, float, 8>(L, c) : F<__half, float, 1>(L, c);                                    \
        return c.vec ? F<__half, __half, 8>(L, c) : F<__half, __half, 1>(L, c);                                            \
      default:                                                                                                             \
        if (wide) return c.vec ? F<__nv_bfloat16, float, 8>(L, c) : F<__nv_bfloat16, float, 1>(L, c);                      \
        return c.vec ? F<__nv_bfloat16, __nv_bfloat16, 8>(L, c) : F<__nv_bfloat16, __nv_bfloat16, 1>(L, c);                \
    }                                                                                                                      \
  } while (0)

cudaError_t launch_block_norm(const Launch &L, const NormCall &c) {
  if (c.T == 0) return cudaSuccess;
  NORM_TYPES(norm_forward);
}
cudaError_t launch_block_norm_grad(const Launch &L, const NormCall &c) {
  NORM_TYPES(norm_backward);
}
