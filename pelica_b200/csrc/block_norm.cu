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

// A thread holds N values of a row; a row's group has tpr threads (whole warps) in each of cl CTAs (a cluster, for rows that
// the registers of an SM do not hold), a CTA has rpb groups, each with rows of its own. Rows of a group follow one another; a
// thread copies its own values of the next ones into its own slots of shared memory (cp.async) while it works on one, so that
// the bytes in flight do not depend on registers and no thread waits for another's copy.
// Values of rows that an SM holds, in whole CTAs: forward 16 values a thread in 896 threads (two rows of 7,168 values: 4096 x 7168 bf16 41 us, one
// row at a time 58), in 1,024 for wider rows (4096 x 8192 51 us, with 896 62; 4096 x 7168 47), 8 values in 1,024; backward, whose column sums
// take registers, 16 values in 512, 8 in 896.
#define NORM_FWD 14336
#define NORM_FWD_WIDE 16384
#define NORM_FWD_8 8192
#define NORM_GRAD 8192
#define NORM_GRAD_8 7168
#define NORM_SMEM 233472      // bytes of shared memory of an SM, of which every CTA takes
#define NORM_SMEM_CTA 3584    // ... these for its sums and for itself
struct NormShape {
  int tpr, rpb, cl;   // threads of a row's group in a CTA, groups of a CTA, CTAs of a row
  int stages;         // rows in a group's ring, 0: none
  int slots;          // of shared memory, a thread
  int per_sm;         // CTAs resident on an SM
  int threads() const { return tpr * rpb; }
};
static NormShape norm_shape(int d, int n, int sm_values) {
  NormShape s = {};
  const int need = (d + n - 1) / n, most = sm_values / n;
  s.cl = 1;
  while ((need + s.cl - 1) / s.cl > most) s.cl *= 2;
  s.tpr = ((need + s.cl - 1) / s.cl + 31) / 32 * 32;
  s.rpb = s.cl == 1 && s.tpr < 256 ? 256 / s.tpr : 1;
  s.per_sm = most / s.threads();
  return s;
}

// the group's place in the launch
struct NormPlace {
  int lane, warp, group, tpr, cl, rank, col0;
};

// sums over a warp: of one value, in every lane; of up to eight, value q in the lanes with lane & 7 == q
template <int N> __device__ __forceinline__ float norm_warp_sums(const float (&v)[N], int lane) {
  static_assert(N <= 6, "");
  if constexpr (N == 1) return pm_warp_sum_16_1(v[0]);
  else {  // lanes of eight keep one value each: 3 + 2 + 1 + 2 exchanges for 30
    const bool b0 = lane & 1, b1 = lane & 2, b2 = lane & 4;
    float a[3], b[2];
#pragma unroll
    for (int j = 0; j < 3; j++) {
      const float e = 2 * j < N ? v[2 * j < N ? 2 * j : 0] : 0.0f, o = 2 * j + 1 < N ? v[2 * j + 1 < N ? 2 * j + 1 : 0] : 0.0f;
      a[j] = 2 * j < N ? __fadd_rn(b0 ? o : e, __shfl_xor_sync(PM_FULL, b0 ? e : o, 1)) : 0.0f;
    }
    b[0] = __fadd_rn(b1 ? a[1] : a[0], __shfl_xor_sync(PM_FULL, b1 ? a[0] : a[1], 2));
    b[1] = N > 4 ? __fadd_rn(b1 ? 0.0f : a[2], __shfl_xor_sync(PM_FULL, b1 ? a[2] : 0.0f, 2)) : 0.0f;
    float s = __fadd_rn(b2 ? b[1] : b[0], __shfl_xor_sync(PM_FULL, b2 ? b[0] : b[1], 4));
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) s = __fadd_rn(s, __shfl_xor_sync(PM_FULL, s, o));
    return s;
  }
}

// A CTA may write to another's shared memory only once all of the cluster are known to run: every thread arrives when it begins and
// waits in front of the first sums, behind the loads of the weights. (Nothing written is handed over: the arrival is relaxed.)
__device__ __forceinline__ void norm_cluster_arrive() {
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void norm_cluster_wait() {
  asm volatile("barrier.cluster.wait;" ::: "memory");
}

// Sums of N values over a row's group, in every thread: lanes, then warps through red (two turns used alternately, so that one
// barrier a sum is enough), then the cluster's CTAs.
template <int N> using NormRed = float[2][N == 1 ? 1 : 8][32];
template <int N> using NormPeer = float[2][8][N];
template <int N, bool CLUSTER>
__device__ __forceinline__ void norm_sum(float (&v)[N], const NormPlace &at, NormRed<N> &red, NormPeer<N> &peer, int &turn) {
  constexpr int Q = N == 1 ? 1 : 8;
  float s = norm_warp_sums<N>(v, at.lane);
  const int warps = at.tpr >> 5;
  if (warps > 1 || CLUSTER) {
    const int first = at.group * warps;
    if (at.lane < Q) red[turn][at.lane][first + at.warp] = s;
    if constexpr (CLUSTER) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(at.group + 1), "r"(at.tpr) : "memory");
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = at.lane < warps ? red[turn][i][first + at.lane] : 0.0f;
    s = norm_warp_sums<N>(v, at.lane);
  }
  if constexpr (CLUSTER) {
    cg::cluster_group cluster = cg::this_cluster();
    // the first warp's lanes give sum i % Q to CTA i / Q
    if (at.warp == 0 && (at.lane & (Q - 1)) < N)
      for (int i = at.lane; i < at.cl * Q; i += 32) cluster.map_shared_rank(&peer[turn][at.rank][0], i / Q)[i & (Q - 1)] = s;
    cluster.sync();
#pragma unroll
    for (int i = 0; i < N; i++) {
      float sum = 0.0f;
      for (int q = 0; q < at.cl; q++) sum = __fadd_rn(sum, peer[turn][q][i]);
      v[i] = sum;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = N == 1 ? s : __shfl_sync(PM_FULL, s, i);
  }
  turn ^= 1;
}

// 1 / sqrt(sum / d + eps): the hardware's estimate and one step of Newton's iteration (left out where it has no value: 0, infinity)
__device__ __forceinline__ float norm_inv(float sum, float inv_d, float eps) {
  const float x = __fmaf_rn(sum, inv_d, eps), y = rsqrtf(x);
  const float e = __fmaf_rn(-__fmul_rn(x, y), y, 1.0f);
  return fabsf(e) < 1.0f ? __fmaf_rn(__fmul_rn(0.5f, y), e, y) : y;
}

// the thread's N values of a row as vectors of V: vector j is columns col0 + j * step ...
template <typename E, int V, int N> struct NormRow {
  static constexpr int J = N / V;
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
  __device__ __forceinline__ VecF<N> widen() const {
    VecF<N> f;
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      if constexpr (V == 1) f.p[i] = pm_pack2(pm_to_f32(v[2 * i].v[0]), pm_to_f32(v[2 * i + 1].v[0]));
      else f.p[i] = pm_widen2(&v[2 * i / V].v[2 * i % V]);
    }
    return f;
  }
  __device__ __forceinline__ static void store(void *base, size_t at, const NormPlace &p, int d, const VecF<N> &f) {
    float g[N];
#pragma unroll
    for (int i = 0; i < N / 2; i++) pm_unpack2(f.p[i], g[2 * i], g[2 * i + 1]);
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int col = p.col0 + j * p.tpr * p.cl * V;
      float h[V];
#pragma unroll
      for (int i = 0; i < V; i++) h[i] = g[j * V + i];
      if (col < d) pm_store<E, V>((E *)base + at + col, pm_narrow<E, V>(h));
    }
  }
};
// weights of the thread's columns, offset added; ones where there are none
template <typename W, int V, int N>
__device__ __forceinline__ VecF<N> norm_weights(const void *w, float offset, const NormPlace &p, int d) {
  if (!w) return vf_all<N>(1.0f);
  NormRow<W, V, N> r;
  r.load(w, 0, p, d);
  return r.widen() + vf_all<N>(offset);
}

// The thread's slots of shared memory: 16 bytes each, `pitch` bytes (all threads' of the CTA) apart. Addresses of the shared
// window throughout; the accesses are volatile: a value that is read a second time is read, not kept in registers.
struct NormSlots {
  uint32_t mine, pitch;
  __device__ __forceinline__ uint32_t at(int i) const { return mine + i * pitch; }
  __device__ __forceinline__ static uint4 get(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
  }
  __device__ __forceinline__ static void put(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
  }
  template <int N> __device__ __forceinline__ void put_vec(int i, const VecF<N> &f) const {
#pragma unroll
    for (int j = 0; j < N / 4; j++)
      asm volatile("st.shared.v2.u64 [%0], {%1, %2};" ::"r"(at(i + j)), "l"(f.p[2 * j]), "l"(f.p[2 * j + 1]) : "memory");
  }
  template <int N> __device__ __forceinline__ VecF<N> get_vec(int i) const {
    VecF<N> f;
#pragma unroll
    for (int j = 0; j < N / 4; j++) asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(f.p[2 * j]), "=l"(f.p[2 * j + 1]) : "r"(at(i + j)));
    return f;
  }
};
__device__ __forceinline__ NormSlots norm_slots(uint4 *all) { return {(uint32_t)__cvta_generic_to_shared(all + threadIdx.x), blockDim.x * 16}; }
// The streams of a group's rows: with RING, stream k of a stage is slot k * J behind the stage's `row`; without, a load.
template <typename E, int V, int N, bool RING> struct NormRing {
  static constexpr int J = N / V;
  NormSlots slots;
  int first, streams, stages;
  // (columns behind the row are never copied: they stay zero)
  __device__ __forceinline__ void clear() const {
    if constexpr (RING)
      for (int i = 0; i < stages * streams * J; i++) NormSlots::put(slots.at(first + i), make_uint4(0, 0, 0, 0));
  }
  __device__ __forceinline__ uint32_t row(int stage) const { return slots.at(first + stage * streams * J); }
  __device__ __forceinline__ void copy(uint32_t row, int k, const void *base, size_t at, const NormPlace &p, int d) const {
    if constexpr (RING) {
#pragma unroll
      for (int j = 0; j < J; j++) {
        const int col = p.col0 + j * p.tpr * p.cl * V;
        if (col < d) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(row + (k * J + j) * slots.pitch), "l"((const E *)base + at + col) : "memory");
      }
    }
  }
  __device__ __forceinline__ static void commit() {
    if constexpr (RING) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // until the oldest of the rows in flight is here
  __device__ __forceinline__ void wait() const {
    if constexpr (RING) {
      if (stages >= 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
      else if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  }
  __device__ __forceinline__ void get(NormRow<E, V, N> &r, uint32_t row, int k, const void *base, size_t at, const NormPlace &p, int d) const {
    if constexpr (RING) {
#pragma unroll
      for (int j = 0; j < J; j++) *(uint4 *)&r.v[j] = NormSlots::get(row + (k * J + j) * slots.pitch);
    } else {
      r.load(base, at, p, d);
    }
  }
};

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

// (strides are 31 bits: one multiplication)
__device__ __forceinline__ size_t norm_row(int t, int64_t stride) { return (size_t)(uint32_t)t * (uint32_t)stride; }

template <typename W> __device__ __forceinline__ float norm_token_gate(const NormCall &c, int t) {
  return c.D.gate == PM_NORM_GATE_TOKEN ? pm_to_f32(((const W *)c.gate)[t]) : 1.0f;
}

// What a call has, known when the kernel is compiled: a row costs half the instructions where the streams need no questions.
//   NORM_ANY       whatever the call gives
//   NORM_SANDWICH  both norms and every stream
//   NORM_BEFORE    the norm before the next block only, every stream
enum NormMode { NORM_ANY, NORM_SANDWICH, NORM_BEFORE };

// SM: values of rows that an SM holds
template <typename E, typename W, int V, int N, int SM, bool CLUSTER, bool RING, NormMode MODE>
__global__ void __launch_bounds__(SM / N) k_block_norm(NormCall c, int tpr, int rpb, int cl, int stages) {
  if constexpr (CLUSTER) norm_cluster_arrive();
  pm_pdl();
  extern __shared__ uint4 slots[];
  __shared__ NormRed<1> red;
  __shared__ NormPeer<1> peer;
  const NormPlace at = norm_place<CLUSTER>(tpr, cl, V);
  const int d = c.D.d, groups = (int)(gridDim.x / at.cl) * rpb;
  constexpr bool ANY = MODE == NORM_ANY;
  const bool post = ANY ? c.D.flags & PM_NORM_POST : MODE == NORM_SANDWICH, pre = ANY ? c.D.flags & PM_NORM_PRE : true;
  const bool has_x = ANY ? c.x != nullptr : true, has_f = ANY ? c.f != nullptr : true, has_r = ANY ? c.r != nullptr : true;
  const int i_x = has_f ? 1 : 0;
  const NormRing<E, V, N, RING> ring = {norm_slots(slots), N / 2, i_x + (has_x ? 1 : 0), stages};
  const int t0 = (int)(blockIdx.x / at.cl) * rpb + at.group;
  auto copy = [&](int stage, int t) {
    if (t < c.T) {
      uint32_t row = ring.row(stage);
      if (has_f) ring.copy(row, 0, c.f, norm_row(t, c.D.f_stride), at, d);
      if (has_x) ring.copy(row, i_x, c.x, norm_row(t, c.D.x_stride), at, d);
    }
    ring.commit();
  };
  // without a ring a group of 16-byte words has one row: its loads go in front of the weights' (one token 6.2 -> 5.8 us)
  NormRow<E, V, N> xr, fr;
  auto fetch = [&](int t) {
    if (t >= c.T) return;
    if (has_f) fr.load(c.f, norm_row(t, c.D.f_stride), at, d);
    if (has_x) xr.load(c.x, norm_row(t, c.D.x_stride), at, d);
  };
  if constexpr (!RING && V > 1) fetch(t0);
  ring.clear();
  if constexpr (RING)
    for (int s = 0; s < stages; s++) copy(s, t0 + s * groups);
  VecF<N> wp = norm_weights<W, V, N>(post ? c.w_post : nullptr, c.D.offset_post, at, d);  // gate and post weight
  VecF<N> wn = norm_weights<W, V, N>(pre ? c.w_pre : nullptr, c.D.offset_pre, at, d);
  if (c.D.gate == PM_NORM_GATE_CHANNEL) wp = wp * norm_weights<W, V, N>(c.gate, 0.0f, at, d);
  if constexpr (RING) {  // (read again for each row: the registers are the rows')
    ring.slots.template put_vec<N>(0, wp);
    ring.slots.template put_vec<N>(N / 4, wn);
  }
  if constexpr (CLUSTER) norm_cluster_wait();
  int turn = 0, stage = 0;
  for (int t = t0; t < c.T; t += groups) {
    ring.wait();
    if (!RING && (V == 1 || t != t0)) fetch(t);
    if constexpr (RING) {
      const uint32_t row = ring.row(stage);
      if (has_f) ring.get(fr, row, 0, c.f, 0, at, d);
      if (has_x) ring.get(xr, row, i_x, c.x, 0, at, d);
      copy(stage, t + stages * groups);
      stage = stage + 1 == stages ? 0 : stage + 1;
      wp = ring.slots.template get_vec<N>(0);
    }
    VecF<N> r = has_x ? xr.widen() * c.D.alpha : vf_all<N>(0.0f);
    const VecF<N> f = has_f ? fr.widen() : vf_all<N>(0.0f);
    if (has_f) {
      float s = __fmul_rn(c.D.beta, norm_token_gate<W>(c, t));
      if (post) {
        float sum[1] = {vf_dot(f, f)};
        norm_sum<1, CLUSTER>(sum, at, red, peer, turn);
        s = __fmul_rn(s, norm_inv(sum[0], c.inv_d, c.D.eps_post));
      }
      r = vf_fma(f * wp, s, r);
    }
    if (has_r) NormRow<E, V, N>::store(c.r, norm_row(t, c.D.r_stride), at, d, r);
    if (pre) {
      float sum[1] = {vf_dot(r, r)};
      norm_sum<1, CLUSTER>(sum, at, red, peer, turn);
      if constexpr (RING) wn = ring.slots.template get_vec<N>(N / 4);
      NormRow<E, V, N>::store(c.n, norm_row(t, c.D.n_stride), at, d, r * wn * norm_inv(sum[0], c.inv_d, c.D.eps_pre));
    }
  }
  if constexpr (CLUSTER) cg::this_cluster().sync();  // no CTA leaves while another may still write its sums here
}

// Two sweeps over a row's values. The first makes all sums that the row needs at once: with q = g f (o1 + w_post), the sum of v f is linear
// in D, so <D, q> = <dr, q> + s2 (<u, q> - s2^2 mean(u r) <r, q>) needs no D, and one exchange between the warps does where
// two lay on the chain. The second sweep makes dx, df and the weights' gradients. The values are read from the ring each time and
// the weights lie beside it (f32, the thread's own columns): the sums of the weights' gradients fill the registers. A CTA adds up
// its groups and leaves a row of sums in parts[kind][CTA][d], which k_norm_sum_parts adds up. No atomics.
template <typename E, typename W, int V, int N, int SM, bool CLUSTER, bool RING, NormMode MODE>
__global__ void __launch_bounds__(SM / N) k_block_norm_grad(NormCall c, int tpr, int rpb, int cl, int stages) {
  if constexpr (CLUSTER) norm_cluster_arrive();
  pm_pdl();
  extern __shared__ uint4 slots[];
  constexpr int SUMS = MODE == NORM_BEFORE ? 2 : 6;  // r r, u r; f f, dr q, u q, r q
  __shared__ NormRed<SUMS> red;
  __shared__ NormPeer<SUMS> peer;
  const NormPlace at = norm_place<CLUSTER>(tpr, cl, V);
  const int d = c.D.d, n_parts = (int)(gridDim.x / at.cl), part = (int)(blockIdx.x / at.cl), groups = n_parts * rpb;
  constexpr bool ANY = MODE == NORM_ANY;
  const bool post = ANY ? c.D.flags & PM_NORM_POST : MODE == NORM_SANDWICH, pre = ANY ? c.D.flags & PM_NORM_PRE : true;
  const bool channel = c.D.gate == PM_NORM_GATE_CHANNEL, token = MODE != NORM_BEFORE && c.D.gate == PM_NORM_GATE_TOKEN;
  const bool use_f = ANY ? post || channel || token : MODE == NORM_SANDWICH;  // (plain: df = beta D)
  const bool has_dr = ANY ? c.dr != nullptr : true, has_dx = ANY ? c.dx != nullptr : true, has_df = ANY ? c.df != nullptr : true;
  const NormSlots own = norm_slots(slots);
  // slots: the pre weight, post weight times the channel's gate, the ring
  const int i_f = pre ? 2 : 0, i_dr = i_f + (use_f ? 1 : 0);
  const NormRing<E, V, N, RING> ring = {own, N / 2, i_dr + (has_dr ? 1 : 0), stages};
  const int t0 = part * rpb + at.group;
  auto copy = [&](int stage, int t) {
    if (t < c.T) {
      uint32_t row = ring.row(stage);
      if (pre) {
        ring.copy(row, 0, c.x, norm_row(t, c.D.r_stride), at, d);
        ring.copy(row, 1, c.dn, norm_row(t, c.D.n_stride), at, d);
      }
      if (use_f) ring.copy(row, i_f, c.f, norm_row(t, c.D.f_stride), at, d);
      if (has_dr) ring.copy(row, i_dr, c.dr, norm_row(t, c.D.r_stride), at, d);
    }
    ring.commit();
  };
  ring.clear();
  if constexpr (RING)
    for (int s = 0; s < stages; s++) copy(s, t0 + s * groups);
  own.template put_vec<N>(0, norm_weights<W, V, N>(pre ? c.w_pre : nullptr, c.D.offset_pre, at, d));
  own.template put_vec<N>(N / 4, norm_weights<W, V, N>(post ? c.w_post : nullptr, c.D.offset_post, at, d) * norm_weights<W, V, N>(channel ? c.gate : nullptr, 0.0f, at, d));
  VecF<N> a_pre = vf_all<N>(0.0f), a_dk = vf_all<N>(0.0f);
  if constexpr (CLUSTER) norm_cluster_wait();
  int turn = 0, stage = 0;
  for (int t = t0; t < c.T; t += groups) {
    const size_t at_r = norm_row(t, c.D.r_stride), at_f = norm_row(t, c.D.f_stride), at_n = norm_row(t, c.D.n_stride);
    const uint32_t row = ring.row(stage);
    NormRow<E, V, N> raw;
    float sum[SUMS] = {};
    ring.wait();
    {
      VecF<N> q;
      if (use_f) {
        ring.get(raw, row, i_f, c.f, at_f, at, d);
        q = raw.widen();
        if (post) sum[SUMS > 2 ? 2 : 0] = vf_dot(q, q);
        q = q * own.template get_vec<N>(N / 4);
        if (has_dr) {
          ring.get(raw, row, i_dr, c.dr, at_r, at, d);
          sum[SUMS > 2 ? 3 : 0] = vf_dot(raw.widen(), q);
        }
      }
      if (pre) {
        ring.get(raw, row, 0, c.x, at_r, at, d);
        const VecF<N> r = raw.widen();
        ring.get(raw, row, 1, c.dn, at_n, at, d);
        const VecF<N> u = raw.widen() * own.template get_vec<N>(0);
        sum[0] = vf_dot(r, r);
        sum[1] = vf_dot(u, r);
        if (use_f) {
          sum[SUMS > 2 ? 4 : 0] = vf_dot(u, q);
          sum[SUMS > 2 ? 5 : 0] = vf_dot(r, q);
        }
      }
    }
    if (pre || post || token) norm_sum<SUMS, CLUSTER>(sum, at, red, peer, turn);
    VecF<N> D = vf_all<N>(0.0f);
    if (has_dr) {
      ring.get(raw, row, i_dr, c.dr, at_r, at, d);
      D = raw.widen();
    }
    float s2 = 0.0f, m = 0.0f;
    if (pre) {
      s2 = norm_inv(sum[0], c.inv_d, c.D.eps_pre);
      m = __fmul_rn(__fmul_rn(s2, s2), __fmul_rn(sum[1], c.inv_d));
      ring.get(raw, row, 0, c.x, at_r, at, d);
      const VecF<N> r = raw.widen();
      ring.get(raw, row, 1, c.dn, at_n, at, d);
      const VecF<N> dn = raw.widen();
      a_pre = vf_fma(dn, r * s2, a_pre);
      D = vf_fma(vf_fma(r, -m, dn * own.template get_vec<N>(0)), s2, D);
    }
    if (has_dx) NormRow<E, V, N>::store(c.dx, norm_row(t, c.D.x_stride), at, d, D * c.D.alpha);
    // k = f s1; D becomes beta g D (o1 + w_post); gt: the token's gate
    const float gt = MODE == NORM_BEFORE ? 1.0f : norm_token_gate<W>(c, t);
    D = D * __fmul_rn(c.D.beta, gt);
    if constexpr (SUMS > 2) {
      if (use_f) {
        const float s1 = post ? norm_inv(sum[2], c.inv_d, c.D.eps_post) : 1.0f;
        const float dot = __fmul_rn(__fmul_rn(c.D.beta, s1), __fmaf_rn(s2, __fmaf_rn(-m, sum[5], sum[4]), sum[3]));
        if (token && c.dgate && at.rank == 0 && at.warp == 0 && at.lane == 0) c.dgate[t] = dot;
        ring.get(raw, row, i_f, c.f, at_f, at, d);
        const VecF<N> k = raw.widen() * s1;
        if (post || channel) a_dk = vf_fma(D, k, a_dk);
        D = D * own.template get_vec<N>(N / 4);
        if (post) D = vf_fma(k, -__fmul_rn(__fmul_rn(dot, gt), c.inv_d), D) * s1;
      }
    }
    if constexpr (RING) {
      copy(stage, t + stages * groups);
      stage = stage + 1 == stages ? 0 : stage + 1;
    }
    if (has_df) NormRow<E, V, N>::store(c.df, at_f, at, d, D);
  }
  // The CTA's groups, kind by kind, columns of a thread as it holds them. With K = sum over t of beta g_t D k, dw_post is K times
  // the channel's gate and the channel's dgate is K times the post weight.
  if constexpr (RING) asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
  for (int kind = 0; kind < 2; kind++) {
    const bool on = kind == 0 ? pre && c.dw_pre : (post && c.dw_post) || (channel && c.dgate);
    if (!on) continue;
    VecF<N> sums = kind == 0 ? a_pre : a_dk;
    if (rpb > 1) {
      __syncthreads();
      own.template put_vec<N>(0, sums);  // (the weights have served)
      __syncthreads();
      if (at.group == 0)
        for (int g = 1; g < rpb; g++) sums = sums + NormSlots{own.mine + g * tpr * 16, own.pitch}.template get_vec<N>(0);
    }
    auto leave = [&](int which, const VecF<N> &s) { NormRow<float, V, N>::store(c.parts, ((size_t)which * n_parts + part) * d, at, d, s); };
    if (at.group) continue;
    if (kind == 0) leave(0, sums);
    else {
      if (post && c.dw_post) leave(1, channel ? sums * norm_weights<W, V, N>(c.gate, 0.0f, at, d) : sums);
      if (channel && c.dgate) leave(2, post ? sums * norm_weights<W, V, N>(c.w_post, c.D.offset_post, at, d) : sums);
    }
  }
  if constexpr (CLUSTER) cg::this_cluster().sync();
}

// out[kind][col] = sum over the parts: a CTA has 32 columns, a warp the parts 32 apart, warps are added in order (8 warps a CTA:
// 17 us instead of 14 for the gradient of 4096 x 512)
__global__ void __launch_bounds__(1024) k_norm_sum_parts(const float *__restrict__ parts, int n_parts, int d, float *o0, float *o1, float *o2) {
  pm_pdl();
  __shared__ float red[32][32];
  float *out = blockIdx.y == 0 ? o0 : blockIdx.y == 1 ? o1 : o2;
  if (!out) return;
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  const float *p = parts + (size_t)blockIdx.y * n_parts * d;
  float s = 0.0f;
  if (col < d) {
#pragma unroll 4
    for (int i = run; i < n_parts; i += 32) s = __fadd_rn(s, p[(size_t)i * d + col]);
  }
  red[run][lane] = s;
  __syncthreads();
  if (run == 0 && col < d) {
#pragma unroll
    for (int i = 1; i < 32; i++) s = __fadd_rn(s, red[i][lane]);
    out[col] = s;
  }
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
// CTAs (clusters) of a call: rows there are, at most what is resident
static int norm_parts(const NormShape &s, int T, int n_sm) {
  const int most = s.cl > 1 ? n_sm / s.cl : n_sm * s.per_sm;
  const int need = (T + s.rpb - 1) / s.rpb;
  return need < most ? need : most;
}
size_t norm_parts_floats(const pm_norm_desc &D, int T, int n_sm) {
  size_t most = 0;  // (of both forms of a row: which one is taken goes by the buffers)
  for (int n : {8, 16}) {
    const size_t f = (size_t)3 * norm_parts(norm_shape(D.d, n, n == 16 ? NORM_GRAD : NORM_GRAD_8), T, n_sm) * D.d;
    if (f > most) most = f;
  }
  return most;
}

// the rows of `row` slots that fit into a ring beside `fixed` slots a thread, 3 at most; fewer CTAs on an SM where not one would fit
// (two CTAs with a row ahead each are better than one with three: forward 4096 x 7168 41 us, 58)
static void norm_ring(NormShape &s, int fixed, int row) {
  auto fit = [&](int per_sm) { return ((NORM_SMEM / per_sm - NORM_SMEM_CTA) / (s.threads() * 16) - fixed) / row; };
  while (s.per_sm > 1 && fit(s.per_sm) < 1) s.per_sm--;
  const int n = fit(s.per_sm);
  s.stages = n > 3 ? 3 : n < 1 ? 1 : n;
  s.slots = fixed + s.stages * row;
}

template <typename... P>
static cudaError_t norm_launch(const Launch &L, SmemOptIn &opt, void (*kern)(P...), int parts, const NormShape &s, NormCall c) {
  const size_t smem = (size_t)s.threads() * s.slots * 16;
  const cudaError_t e = smem_optin(opt, kern, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts * s.cl);
  cfg.blockDim = dim3(s.threads());
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
  return cudaLaunchKernelEx(&cfg, kern, c, s.tpr, s.rpb, s.cl, s.stages);
}
template <typename E, typename W, int V, int N, int SM, bool RING, NormMode MODE, bool GRAD>
static cudaError_t norm_go(const Launch &L, int parts, const NormShape &s, const NormCall &c) {
  static SmemOptIn one, many;
  if constexpr (GRAD)
    return s.cl > 1 ? norm_launch(L, many, k_block_norm_grad<E, W, V, N, SM, true, RING, MODE>, parts, s, c)
                    : norm_launch(L, one, k_block_norm_grad<E, W, V, N, SM, false, RING, MODE>, parts, s, c);
  else
    return s.cl > 1 ? norm_launch(L, many, k_block_norm<E, W, V, N, SM, true, RING, MODE>, parts, s, c)
                    : norm_launch(L, one, k_block_norm<E, W, V, N, SM, false, RING, MODE>, parts, s, c);
}
// the kernels of 16-byte words that go by what the call has
template <typename E, typename W, int V, int N, int SM, bool GRAD>
static cudaError_t norm_go_mode(const Launch &L, int parts, const NormShape &s, const NormCall &c) {
  const bool all = GRAD ? c.dr && c.dx && c.df : c.x && c.f && c.r;
  const bool post = c.D.flags & PM_NORM_POST, pre = c.D.flags & PM_NORM_PRE;
  if (all && pre && post) return norm_go<E, W, V, N, SM, true, NORM_SANDWICH, GRAD>(L, parts, s, c);
  if (all && pre && c.D.gate == PM_NORM_GATE_NONE) return norm_go<E, W, V, N, SM, true, NORM_BEFORE, GRAD>(L, parts, s, c);
  return norm_go<E, W, V, N, SM, true, NORM_ANY, GRAD>(L, parts, s, c);
}

// rows of 16-byte words, more of them than groups: through rings
template <typename E, typename W, int V, int N, int SM> static cudaError_t norm_forward_ring(const Launch &L, const NormCall &c) {
  NormShape s = norm_shape(c.D.d, N, SM);
  norm_ring(s, N / 2, ((c.x ? 1 : 0) + (c.f ? 1 : 0)) * N / V);
  return norm_go_mode<E, W, V, N, SM, false>(L, norm_parts(s, c.T, L.n_sm), s, c);
}
// 16 values a thread of the 16-bit types, half the threads for the same sums (gradient of 4096 x 2048 bf16 31 -> 28 us, x 4096 60 -> 56); 8 of
// f32, whose rings are twice the size (gradient of 4096 x 7168: 145 us, 159 with 16), of rows value by value, and of a row a group (no ring).
template <typename E, typename W, int V> static cudaError_t norm_forward(const Launch &L, const NormCall &c) {
  const NormShape s = norm_shape(c.D.d, 8, NORM_FWD_8);
  const int parts = norm_parts(s, c.T, L.n_sm);
  if constexpr (V > 1) {
    if (c.T > parts * s.rpb) {
      if constexpr (V == 4) return norm_forward_ring<E, W, V, 8, NORM_FWD_8>(L, c);
      else if (c.D.d > NORM_FWD / 2) return norm_forward_ring<E, W, V, 16, NORM_FWD_WIDE>(L, c);
      else return norm_forward_ring<E, W, V, 16, NORM_FWD>(L, c);
    }
  }
  return norm_go<E, W, V, 8, NORM_FWD_8, false, NORM_ANY, false>(L, parts, s, c);
}
template <typename E, typename W, int V> static cudaError_t norm_backward_rows(const Launch &L, const NormCall &c, int *parts) {
  constexpr int N = V == 8 ? 16 : 8, SM = V == 8 ? NORM_GRAD : NORM_GRAD_8;
  NormShape s = norm_shape(c.D.d, N, SM);
  const bool post = c.D.flags & PM_NORM_POST, pre = c.D.flags & PM_NORM_PRE, gate = c.D.gate != PM_NORM_GATE_NONE;
  const int row = ((pre ? 2 : 0) + (post || gate ? 1 : 0) + (c.dr ? 1 : 0)) * N / V;
  s.slots = N / 2;
  if (V > 1 && row) norm_ring(s, N / 2, row);
  *parts = norm_parts(s, c.T, L.n_sm);
  if constexpr (V > 1) return norm_go_mode<E, W, V, N, SM, true>(L, *parts, s, c);
  else return norm_go<E, W, V, N, SM, false, NORM_ANY, true>(L, *parts, s, c);
}
template <typename E, typename W, int V> static cudaError_t norm_backward(const Launch &L, const NormCall &c) {
  int parts = 0;
  float *channel = c.D.gate == PM_NORM_GATE_CHANNEL ? c.dgate : nullptr;
  if (c.T) {  // (no rows: the sums alone, zeros)
    const cudaError_t e = norm_backward_rows<E, W, V>(L, c, &parts);
    if (e != cudaSuccess) return e;
  }
  if (!c.dw_pre && !c.dw_post && !channel) return cudaSuccess;
  return pm_launch(L, k_norm_sum_parts, dim3((c.D.d + 31) / 32, 3), 1024, 0, (const float *)c.parts, parts, c.D.d, c.dw_pre, c.dw_post, channel);
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
