// rows.cu - tokens sorted by expert and back, with their gradients.
//
// Pair p = t * K + k goes to local expert e(p) = ids[p] - first; a pair of another rank's expert, or of no expert
// (PM_ROWS_NONE: the padding of a batch), has no row. With c_e the pairs of expert e and A the alignment of its group,
//   offset_e = sum over e' < e of ceil(c_e' / A) * A,   pos_p = offset_e(p) + #{q < p : e(q) = e(p)}   (a stable counting sort).
//   dispatch       rows[pos_p] = s_p x[t]                      collect       y[t]  = add[t] + sum_k w_p rows[pos_p]
//   its gradient   dx[t]  = sum_k s_p drows[pos_p]             its gradient  drows[pos_p] = w_p dy[t]
//                  dw_p   = <drows[pos_p], x[t]>                             dw_p = <rows[pos_p], dy[t]>
// A group's padding rows are zeros, so that a product over whole groups adds nothing for them. Sums are made in f32, over
// k in ascending order, without atomics: the same bits in every run. Bound by HBM: one multiply-add a value moved.
#include <cooperative_groups.h>

#include "rows.cuh"
#include "vec.cuh"

namespace cg = cooperative_groups;

#define ROWS_NO_EXPERT 0xffffu

// expert id -> local index, ROWS_NO_EXPERT for a pair without a row; an id that no expert has is reported
__device__ __forceinline__ uint32_t rows_local(const RowsCall &c, uint32_t id) {
  if (id >= (uint32_t)c.D.n_exp) {
    if (id != PM_ROWS_NONE) atomicCAS(c.err, 0, PM_DEVERR_BAD_EXPERT_ID);
    return ROWS_NO_EXPERT;
  }
  const uint32_t e = id - (uint32_t)c.D.first_expert;
  return e < (uint32_t)c.D.n_local ? e : ROWS_NO_EXPERT;
}
// a position from a plan buffer: one that the rows do not have is reported and has no row
__device__ __forceinline__ uint32_t rows_pos(const RowsCall &c, uint32_t pos) {
  if (pos == PM_ROWS_NONE || (int64_t)pos < c.pl.max_rows) return pos;
  atomicCAS(c.err, 0, PM_DEVERR_BAD_ROW);
  return PM_ROWS_NONE;
}
__device__ __forceinline__ uint32_t rows_padded(uint32_t n, uint32_t align) { return (n + align - 1) / align * align; }

// exclusive sums of the padded counts of PM_MAX_EXPERTS experts in shared memory; every thread of a CTA of >= 256 calls it.
// off: PM_MAX_EXPERTS + 1 words; part: 8 words
__device__ __forceinline__ void rows_scan(const uint32_t *cnt, uint32_t align, uint32_t *off, uint32_t *part) {
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t a = 0, b = 0, sum = 0;
  if (tid < PM_MAX_EXPERTS / 2) {
    a = rows_padded(cnt[2 * tid], align);
    b = rows_padded(cnt[2 * tid + 1], align);
    sum = a + b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(PM_FULL, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) part[tid >> 5] = sum;
  }
  __syncthreads();
  if (tid < PM_MAX_EXPERTS / 2) {
    uint32_t before = sum - a - b;
    for (int i = 0; i < (tid >> 5); i++) before += part[i];
    off[2 * tid] = before;
    off[2 * tid + 1] = before + a;
    if (tid == PM_MAX_EXPERTS / 2 - 1) off[PM_MAX_EXPERTS] = before + a + b;
  }
  __syncthreads();
}

// a pair's entries in the plan's lists
__device__ __forceinline__ void rows_write_pair(const RowsCall &c, const float *w, uint32_t p, uint32_t id, uint32_t pos) {
  c.pl.pos[p] = pos;
  if (pos == PM_ROWS_NONE) return;
  if (c.pl.row_pair) c.pl.row_pair[pos] = p;
  if (c.pl.row_expert) c.pl.row_expert[pos] = id;
  if (c.pl.row_weight) c.pl.row_weight[pos] = w ? w[p] : 1.0f;
}
// ... and those of a padding row: no pair, the group's expert, no weight
__device__ __forceinline__ void rows_write_pad(const RowsCall &c, uint32_t e, uint32_t row) {
  if (c.pl.row_pair) c.pl.row_pair[row] = PM_ROWS_NONE;
  if (c.pl.row_expert) c.pl.row_expert[row] = e + (uint32_t)c.D.first_expert;
  if (c.pl.row_weight) c.pl.row_weight[row] = 0.0f;
}

// a row of zeros, by all threads of the CTA
template <typename E, int V> __device__ __forceinline__ void rows_zero(const RowsCall &c, E *rows, uint32_t r) {
  const Raw<E, V> zero = vf_narrow<E, V>(vf_zero<V>());
  const uint32_t dv = (uint32_t)c.D.d / V;
  for (uint32_t v = threadIdx.x; v < dv; v += blockDim.x) pm_store<E, V>(rows + (size_t)r * c.D.rows_stride + (size_t)v * V, zero);
}

// ---------------------------------------------------------------------------
// plan and rows of a few pairs in one launch
// ---------------------------------------------------------------------------
// Grid (token, slab of 256 vectors), and as many CTAs without a token as spread the padding over the GPU. Every CTA sorts all pairs
// for itself - at most PM_ROWS_SMALL_PAIRS, in shared memory - and copies its piece of its token: no CTA waits for another.
#define ROWS_PAD_CTAS 256  // at least, where groups are padded
#define ROWS_PAD_LIST PM_MAX_EXPERTS  // padding rows of one CTA: no group has ROWS_PAD_CTAS of them
static_assert(ROWS_PAD_CTAS >= PM_ROWS_MAX_ALIGN, "a CTA has one padding row of a group");
template <typename E, int V>
__global__ void __launch_bounds__(256) k_rows_dispatch_small(RowsCall c, const uint32_t *__restrict__ ids, const float *__restrict__ w, bool scale,
                                                             const E *__restrict__ x, E *__restrict__ rows) {
  pm_pdl();
  __shared__ uint16_t le[PM_ROWS_SMALL_PAIRS];
  __shared__ uint32_t cnt[PM_MAX_EXPERTS], off[PM_MAX_EXPERTS + 1], part[8];
  __shared__ uint32_t at[PM_MAX_TOPK], pad[ROWS_PAD_LIST], n_pad;
  __shared__ float ws[PM_MAX_TOPK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = c.D.top_k;
  const uint32_t P = (uint32_t)c.T * K, t = blockIdx.x, p0 = t * K, dv = (uint32_t)c.D.d / V;
  const uint32_t v0 = blockIdx.y * 256 + tid;
  Raw<E, V> mine;
  const bool live = x && t < (uint32_t)c.T;
  if (live && v0 < dv) mine = pm_load<E, V>(x + (size_t)t * c.D.x_stride + (size_t)v0 * V);
  for (int e = tid; e < PM_MAX_EXPERTS; e += 256) cnt[e] = 0;
  __syncthreads();
  for (uint32_t p = tid; p < P; p += 256) {
    const uint32_t e = rows_local(c, ids[p]);
    le[p] = (uint16_t)e;
    if (e != ROWS_NO_EXPERT) atomicAdd(&cnt[e], 1u);
  }
  __syncthreads();
  rows_scan(cnt, c.D.align, off, part);
  for (int k = warp; k < K && t < (uint32_t)c.T; k += 8) {  // a warp a pair of this token: the pairs of the same expert before it
    const uint32_t e = le[p0 + k];
    uint32_t n = 0;
    for (uint32_t q = lane; q < p0 + k; q += 32) n += le[q] == e;
    n = __reduce_add_sync(PM_FULL, n);
    if (lane == 0) {
      const uint32_t pos = e == ROWS_NO_EXPERT ? PM_ROWS_NONE : off[e] + n;
      at[k] = pos;
      ws[k] = scale ? w[p0 + k] : 1.0f;
      if (blockIdx.y == 0) rows_write_pair(c, w, p0 + k, e + (uint32_t)c.D.first_expert, pos);
    }
  }
  const uint32_t cta = blockIdx.y * gridDim.x + blockIdx.x, n_cta = gridDim.x * gridDim.y;
  if (cta == 0) {
    for (int e = tid; e < c.D.n_local; e += 256) {
      c.pl.offset[e] = off[e];
      c.pl.count[e] = cnt[e];
    }
    if (tid == 0) c.pl.offset[c.D.n_local] = off[c.D.n_local];
  }
  if (c.D.align > 1) {  // padding row r is CTA r % n_cta's
    if (tid == 0) n_pad = 0;
    __syncthreads();
    for (uint32_t e = tid; e < (uint32_t)c.D.n_local; e += 256) {
      const uint32_t from = off[e] + cnt[e], to = off[e + 1];
      for (uint32_t r = from + (cta + n_cta - from % n_cta) % n_cta; r < to; r += n_cta) {
        rows_write_pad(c, e, r);
        if (x) pad[atomicAdd(&n_pad, 1u)] = r;
      }
    }
    __syncthreads();
    if (x)
      for (uint32_t i = 0; i < n_pad; i++) rows_zero<E, V>(c, rows, pad[i]);
  }
  if (!live) return;
  __syncthreads();
  for (uint32_t v = v0; v < dv; v += gridDim.y * 256) {
    if (v != v0) mine = pm_load<E, V>(x + (size_t)t * c.D.x_stride + (size_t)v * V);
    const VecF<V> f = vf_widen<E, V>(mine);
    for (int k = 0; k < K; k++)
      if (at[k] != PM_ROWS_NONE)
        pm_store<E, V>(rows + (size_t)at[k] * c.D.rows_stride + (size_t)v * V, scale ? vf_narrow<E, V>(vf_mul<V>(f, ws[k])) : mine);
  }
}

// ---------------------------------------------------------------------------
// the plan of many pairs
// ---------------------------------------------------------------------------
// Clusters of 8 (4) CTAs x 32 warps, each of which places a run of 8,192 pairs times `steps`; a warp owns 32 pairs a step. A pair's
// rank within its warp (match.any: the lanes with the same expert) comes from the warp's counts, u16 in shared memory; then
// sums over a CTA's warps and over the CTAs through distributed shared memory. A cluster counts the pairs in front of its run
// and behind it itself - no ranks, so shared-memory additions do - instead of waiting for the other clusters: nothing is
// exchanged in global memory, and a recorded graph holds no pointer of the library's. 131,072 pairs: 25 us in one
// cluster, whose 8 SMs wait for match.any (votes bit by bit: as long).
#define SORT_CTAS 8
#define SORT_WARPS 32
#define SORT_THREADS (SORT_WARPS * 32)
#define SORT_CLUSTERS 8
#define SORT_STEPS (PM_MAX_TOKENS * PM_MAX_TOPK / (SORT_CTAS * SORT_THREADS * SORT_CLUSTERS))
__global__ void __launch_bounds__(SORT_THREADS)
    k_rows_sort(RowsCall c, uint32_t steps, const uint32_t *__restrict__ ids, const float *__restrict__ w) {
  pm_pdl();
  __shared__ uint16_t hist[SORT_WARPS][PM_MAX_EXPERTS];
  __shared__ uint32_t ours[PM_MAX_EXPERTS], front[PM_MAX_EXPERTS], behind[PM_MAX_EXPERTS];
  __shared__ uint32_t cnt[PM_MAX_EXPERTS], off[PM_MAX_EXPERTS + 1], part[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks(), stride = ctas * SORT_THREADS, run = blockIdx.x / ctas;
  const uint32_t P = (uint32_t)c.T * c.D.top_k;
  const uint32_t begin = run * steps * stride, end = min(begin + steps * stride, P);
  const uint32_t first = begin + (rank * SORT_WARPS + warp) * steps * 32 + lane;
  uint32_t mine[SORT_STEPS];  // ids, then expert << 16 | rank
#pragma unroll
  for (int s = 0; s < SORT_STEPS; s++) mine[s] = s < (int)steps && first + s * 32 < P ? ids[first + s * 32] : PM_ROWS_NONE;
  for (int i = tid; i < SORT_WARPS * PM_MAX_EXPERTS / 2; i += SORT_THREADS) ((uint32_t *)hist)[i] = 0;
  if (tid < PM_MAX_EXPERTS) front[tid] = behind[tid] = 0;
  __syncthreads();
  for (uint32_t p0 = rank * SORT_THREADS + tid; p0 < P && gridDim.x > ctas; p0 += 4 * stride) {
    uint32_t id[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t p = p0 + i * stride;
      id[i] = p < P && (p < begin || p >= end) ? ids[p] : PM_ROWS_NONE;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t e = id[i] - (uint32_t)c.D.first_expert;  // (an id that no expert has is its own cluster's to report)
      if (id[i] < (uint32_t)c.D.n_exp && e < (uint32_t)c.D.n_local) atomicAdd(p0 + i * stride < begin ? &front[e] : &behind[e], 1u);
    }
  }
#pragma unroll
  for (int s = 0; s < SORT_STEPS; s++) {
    if (s >= (int)steps) break;
    const uint32_t e = rows_local(c, mine[s]), same = __match_any_sync(PM_FULL, e), before = __popc(same & ((1u << lane) - 1));
    uint32_t have = 0;
    if (e != ROWS_NO_EXPERT) have = hist[warp][e];
    __syncwarp();
    if (e != ROWS_NO_EXPERT && before == 0) hist[warp][e] = (uint16_t)(have + __popc(same));
    __syncwarp();
    mine[s] = e << 16 | (have + before);
  }
  __syncthreads();
  if (tid < PM_MAX_EXPERTS) {  // the warps' counts become what lies before each warp (a CTA has 4,096 pairs at most)
    uint32_t sum = 0;
#pragma unroll 8
    for (int i = 0; i < SORT_WARPS; i++) {
      const uint32_t n = hist[i][tid];
      hist[i][tid] = (uint16_t)sum;
      sum += n;
    }
    ours[tid] = sum;
  }
  cluster.sync();
  uint32_t ahead = 0;  // pairs of expert tid in front of this CTA's
  if (tid < PM_MAX_EXPERTS) {
    uint32_t all = 0;
#pragma unroll 8
    for (int i = 0; i < (int)ctas; i++) {
      const uint32_t n = cluster.map_shared_rank(ours, i)[tid], f = cluster.map_shared_rank(front, i)[tid];
      ahead += f + (i < (int)rank ? n : 0);
      all += f + n + cluster.map_shared_rank(behind, i)[tid];
    }
    cnt[tid] = all;
  }
  cluster.sync();  // nobody reads another CTA's counts any more
  rows_scan(cnt, c.D.align, off, part);
  if (tid < PM_MAX_EXPERTS) ours[tid] = off[tid] + ahead;
  if (blockIdx.x == 0) {
    for (int e = tid; e < c.D.n_local; e += SORT_THREADS) {
      c.pl.offset[e] = off[e];
      c.pl.count[e] = cnt[e];
    }
    if (tid == 0) c.pl.offset[c.D.n_local] = off[c.D.n_local];
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < SORT_STEPS; s++) {
    const uint32_t p = first + s * 32, e = mine[s] >> 16;
    if (s >= (int)steps || p >= P) break;
    rows_write_pair(c, w, p, e + (uint32_t)c.D.first_expert, e == ROWS_NO_EXPERT ? PM_ROWS_NONE : ours[e] + hist[warp][e] + (mine[s] & 0xffffu));
  }
  if (c.D.align > 1 && (c.pl.row_pair || c.pl.row_expert || c.pl.row_weight))
    for (uint32_t e = blockIdx.x * SORT_WARPS + warp; e < (uint32_t)c.D.n_local; e += gridDim.x * SORT_WARPS)
      for (uint32_t r = off[e] + cnt[e] + lane; r < off[e + 1]; r += 32) rows_write_pad(c, e, r);
}

// ---------------------------------------------------------------------------
// rows out and rows back: G threads a token
// ---------------------------------------------------------------------------
// A token's threads walk its row and its K rows together, vector by vector, the K accesses of a step in flight at once: the
// positions and weights are read once a token, and the K dot products stay in a thread's registers until the end.
//   SPREAD   out[pos] = w src[t]                         otherwise   out[t] = add[t] + sum_k w rows[pos]
//   DOT      dw[t][k] = <rows[pos], src[t]>
// G: a power of two, 256 at most (a CTA); grid.y cuts the rows of a few tokens without DOT further. Behind the tokens' CTAs
// (SPREAD), some for each expert's padding. KB: K rounded up to one of five (10 pairs in a kernel for 16: 147 us instead of 126
// for 8192 x 2048 bf16 with dot products). Rows that do not start on 16 bytes go value by value, two values of a row a step and 32 warps an
// SM (8000 x 1001 f16 with dot products, 5 pairs: 66 us, of 27 of bytes; four values a step and 8 warps 112).
// CTAs that an SM is to hold: registers against reads in flight. Rows read as 16-byte words: 2 (8192 x 2048 bf16 with dot products 101 us; 1:
// 130, 3: 104). Value by value: 4, of many pairs 2 (10 pairs: 4 spilled, 538 us against 363). Rows that are only written: any.
__host__ __device__ constexpr int rows_ctas(int V, int KB, bool SPREAD, bool DOT) {
  return SPREAD && !DOT ? 1 : V == 1 && KB <= 8 ? 4 : 2;
}
template <typename E, int V, int KB, bool SPREAD, bool DOT>
__global__ void __launch_bounds__(256, rows_ctas(V, KB, SPREAD, DOT))
    k_rows(RowsCall c, uint32_t token_ctas, int G, const float *__restrict__ w, const E *__restrict__ src, const E *__restrict__ rows, const E *add,
           E *out, float *__restrict__ dw) {
  pm_pdl();
  __shared__ float sums[DOT ? 8 : 1][KB];
  const int tid = threadIdx.x;
  const uint32_t dv = (uint32_t)c.D.d / V, K = c.D.top_k;
  if (SPREAD && blockIdx.x >= token_ctas) {
    if (blockIdx.y) return;
    const uint32_t e = (blockIdx.x - token_ctas) % c.D.n_local, s = (blockIdx.x - token_ctas) / c.D.n_local;
    const uint32_t to = (uint32_t)min((int64_t)c.pl.offset[e + 1], c.pl.max_rows);
    for (uint32_t r = c.pl.offset[e] + c.pl.count[e] + s; r < to; r += (gridDim.x - token_ctas) / c.D.n_local) rows_zero<E, V>(c, out, r);
    return;
  }
  const uint32_t t = blockIdx.x * (256 / G) + tid / G;
  const bool live = t < (uint32_t)c.T;
  const uint32_t first = blockIdx.y * G + tid % G, step = gridDim.y * G;
  uint32_t pos[KB];
  float wk[KB];
  DotOf<V> dot[KB];
#pragma unroll
  for (int k = 0; k < KB; k++) {
    const bool in = live && k < (int)K;
    pos[k] = in ? c.pl.pos[t * K + k] : PM_ROWS_NONE;
    wk[k] = in && w ? w[t * K + k] : 1.0f;
    dot[k] = 0;
  }
#pragma unroll
  for (int k = 0; k < KB; k++) {
    pos[k] = rows_pos(c, pos[k]);
    if (pos[k] == PM_ROWS_NONE) wk[k] = 0.0f;  // (whatever its weight is, a NaN of a padded token's routing)
  }
  // vectors of a step: single values come two at a time, so that their reads are in flight together
  constexpr int J = V > 1 ? 1 : 2;
  if (live)
    for (uint32_t v0 = first; v0 < dv; v0 += step * J) {
      const size_t row = (size_t)t * c.D.x_stride;
      Raw<E, V> s[J], r[KB][J];
#pragma unroll
      for (int j = 0; j < J; j++) {
        const uint32_t v = v0 + j * step;
        if (J > 1 && v >= dv) break;
        if (SPREAD || DOT) s[j] = pm_load<E, V>(src + row + (size_t)v * V);
        else if (add) s[j] = pm_load<E, V>(add + row + (size_t)v * V);
        if (!SPREAD || DOT) {
#pragma unroll
          for (int k = 0; k < KB; k++) {  // (a pair without a row: zeros, which add nothing)
            r[k][j] = vf_narrow<E, V>(vf_zero<V>());
            if (pos[k] != PM_ROWS_NONE) r[k][j] = pm_load<E, V>(rows + (size_t)pos[k] * c.D.rows_stride + (size_t)v * V);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < J; j++) {
        const uint32_t v = v0 + j * step;
        if (J > 1 && v >= dv) break;
        const VecF<V> f = (SPREAD || DOT || add) ? vf_widen<E, V>(s[j]) : vf_zero<V>();
        VecF<V> acc = DOT ? vf_zero<V>() : f;
#pragma unroll
        for (int k = 0; k < KB; k++) {
          if (V == 1 && k >= (int)K) break;
          if (!SPREAD || DOT) {
            const VecF<V> g = vf_widen<E, V>(r[k][j]);
            if (DOT) vf_dot_add<V>(dot[k], g, f);
            if (!SPREAD) vf_add<V>(acc, g, wk[k]);
          }
          if (SPREAD && pos[k] != PM_ROWS_NONE)
            pm_store<E, V>(out + (size_t)pos[k] * c.D.rows_stride + (size_t)v * V, w ? vf_narrow<E, V>(vf_mul<V>(f, wk[k])) : s[j]);
        }
        if (!SPREAD) pm_store<E, V>(out + row + (size_t)v * V, vf_narrow<E, V>(acc));
      }
    }
  if constexpr (DOT) {
    const int lanes = G < 32 ? G : 32;
#pragma unroll
    for (int k = 0; k < KB; k++) {
      float a = vf_sum(dot[k]);
      for (int o = lanes / 2; o >= 1; o >>= 1) a = __fadd_rn(a, __shfl_xor_sync(PM_FULL, a, o));
      if (pos[k] == PM_ROWS_NONE) a = 0.0f;  // (not 0 times an infinity of src)
      if (G <= 32) {
        if (live && tid % G == 0 && k < (int)K) dw[t * K + k] = a;
      } else if ((tid & 31) == 0) {
        sums[tid >> 5][k] = a;
      }
    }
    if (G <= 32) return;
    __syncthreads();
    const int in = tid % G;
    if (live && in < (int)K) {
      float a = 0.0f;
      for (int i = 0; i < G / 32; i++) a = __fadd_rn(a, sums[tid / G * (G / 32) + i][in]);
      dw[t * K + in] = a;
    }
  }
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
#define ROWS_TYPES(call)                                                                          \
  do {                                                                                            \
    switch (c.D.dtype) {                                                                          \
      case PM_TYPE_F32: return c.vec ? call(float, 4) : call(float, 1);                           \
      case PM_TYPE_F16: return c.vec ? call(__half, 8) : call(__half, 1);                         \
      default: return c.vec ? call(__nv_bfloat16, 8) : call(__nv_bfloat16, 1);                    \
    }                                                                                             \
  } while (0)

static uint32_t rows_vectors(const RowsCall &c) { return c.vec ? (uint32_t)c.D.d / (c.D.dtype == PM_TYPE_F32 ? 4 : 8) : (uint32_t)c.D.d; }

// The threads of a token: as many as its row has vectors, but doubled only until the launch has 32 warps for every SM (4096 x 2048 bf16
// back to their tokens: 28 us; 8 warps 31, all 30; with dot products, 8192 tokens: 101, 101, 145). Not all of them are on the
// SMs at once: the kernels of 16-byte rows with dot products hold 16 warps an SM. Rows that are only written have one read in
// flight a thread, so they take all (prompt of 4096 x 7168: 101 us, 112 with 32 warps). Where even CTAs of 256
// threads leave SMs without work, a row without dot products is cut (grid.y).
template <typename E, int V, int KB, bool SPREAD, bool DOT>
static cudaError_t rows_go(const Launch &L, const RowsCall &c, const float *w, const void *src, const void *rows, const void *add, void *out,
                           float *dw) {
  const uint32_t dv = rows_vectors(c);
  uint32_t pad = 0;  // CTAs of the padding: two an SM, a group's rows cut as often as that takes
  if (SPREAD && c.D.align > 1) {
    const uint32_t cuts = 2u * L.n_sm / c.D.n_local;
    pad = c.D.n_local * (cuts < 1 ? 1 : cuts < (uint32_t)c.D.align - 1 ? cuts : c.D.align - 1);
  }
  int G = 4;
  while (G < 256 && (uint32_t)G < dv && (G < 32 || (SPREAD && !DOT) || (int64_t)c.T * G < (int64_t)32 * 32 * L.n_sm)) G *= 2;
  const uint32_t ctas = ((uint32_t)c.T * G + 255) / 256;
  uint32_t cuts = 1;
  if (!DOT)
    while (ctas * cuts < 2u * L.n_sm && cuts * G < dv) cuts *= 2;
  if (ctas + pad == 0) return cudaSuccess;
  return pm_launch(L, k_rows<E, V, KB, SPREAD, DOT>, dim3(ctas + pad, cuts), 256, 0, c, ctas, G, w, (const E *)src, (const E *)rows, (const E *)add,
                   (E *)out, dw);
}
template <typename E, int V, bool SPREAD, bool DOT>
static cudaError_t rows_k(const Launch &L, const RowsCall &c, const float *w, const void *src, const void *rows, const void *add, void *out,
                          float *dw) {
  if (c.D.top_k <= 4) return rows_go<E, V, 4, SPREAD, DOT>(L, c, w, src, rows, add, out, dw);
  if (c.D.top_k <= 6) return rows_go<E, V, 6, SPREAD, DOT>(L, c, w, src, rows, add, out, dw);
  if (c.D.top_k <= 8) return rows_go<E, V, 8, SPREAD, DOT>(L, c, w, src, rows, add, out, dw);
  if (c.D.top_k <= 12) return rows_go<E, V, 12, SPREAD, DOT>(L, c, w, src, rows, add, out, dw);
  return rows_go<E, V, 16, SPREAD, DOT>(L, c, w, src, rows, add, out, dw);
}

template <typename E, int V>
static cudaError_t dispatch_small(const Launch &L, const RowsCall &c, const uint32_t *ids, const float *w, bool scale, const void *x, void *rows) {
  // (a call without tokens or rows still writes its offsets; slabs: what eight CTAs an SM hold, each CTA sorts)
  uint32_t ctas = c.T > 0 ? c.T : 1, slabs = x && c.T ? (rows_vectors(c) + 255) / 256 : 1;
  if (slabs > 8u * L.n_sm / ctas) slabs = 8u * L.n_sm / ctas > 1 ? 8u * L.n_sm / ctas : 1;
  if (c.D.align > 1 && c.T && ctas * slabs < ROWS_PAD_CTAS) ctas = (ROWS_PAD_CTAS + slabs - 1) / slabs;
  return pm_launch(L, k_rows_dispatch_small<E, V>, dim3(ctas, slabs), 256, 0, c, ids, w, scale, (const E *)(c.T ? x : nullptr), (E *)rows);
}

static cudaError_t rows_sort(const Launch &L, uint32_t clusters, uint32_t ctas, const RowsCall &c, uint32_t steps, const uint32_t *ids,
                             const float *w) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * ctas);
  cfg.blockDim = dim3(SORT_THREADS);
  cfg.stream = L.stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = ctas;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (L.count) ++*L.count;
  return cudaLaunchKernelEx(&cfg, k_rows_sort, c, steps, ids, w);
}

cudaError_t launch_rows_dispatch(const Launch &L, const RowsCall &c, const uint32_t *ids, const float *w, bool scale, const void *x, void *rows) {
  if ((size_t)c.T * c.D.top_k <= PM_ROWS_SMALL_PAIRS) {
#define CALL(E, V) dispatch_small<E, V>(L, c, ids, w, scale, x, rows)
    ROWS_TYPES(CALL);
#undef CALL
  }
  const uint32_t P = (uint32_t)c.T * c.D.top_k;
  // few pairs: one cluster of four CTAs, whose barriers are cheaper (2,048 pairs 6.3 us, eight CTAs 7.9, two 6.2, one 8.3; 8,192: 7.6, 8.0, 9.5)
  const uint32_t ctas = P <= 8 * SORT_THREADS ? 4 : SORT_CTAS, step = ctas * SORT_THREADS;
  const uint32_t most = ctas == 4 ? 1 : SORT_CLUSTERS, steps = (P + step * most - 1) / (step * most);
  const uint32_t clusters = (P + step * steps - 1) / (step * steps);
  const cudaError_t e = rows_sort(L, clusters, ctas, c, steps, ids, w);
  if (e != cudaSuccess || !x) return e;
  return launch_rows_spread(L, c, scale ? w : nullptr, x, nullptr, rows, nullptr);
}

cudaError_t launch_rows_gather(const Launch &L, const RowsCall &c, const float *w, const void *rows, const void *add, const void *x, void *out,
                               float *dw) {
#define CALL(E, V) (dw ? rows_k<E, V, false, true>(L, c, w, x, rows, nullptr, out, dw) : rows_k<E, V, false, false>(L, c, w, nullptr, rows, add, out, nullptr))
  ROWS_TYPES(CALL);
#undef CALL
}

cudaError_t launch_rows_spread(const Launch &L, const RowsCall &c, const float *w, const void *src, const void *rows, void *out, float *dw) {
#define CALL(E, V) (dw ? rows_k<E, V, true, true>(L, c, w, src, rows, nullptr, out, dw) : rows_k<E, V, true, false>(L, c, w, src, nullptr, nullptr, out, nullptr))
  ROWS_TYPES(CALL);
#undef CALL
}
