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

// zeros in rows [from, to), by all threads of the CTA
template <typename E, int V> __device__ __forceinline__ void rows_zero(const RowsCall &c, E *rows, uint32_t from, uint32_t to) {
  const float z[V] = {};
  const Raw<E, V> zero = pm_narrow<E, V>(z);
  const uint32_t dv = (uint32_t)c.D.d / V;
  for (uint32_t r = from; r < to; r++)
    for (uint32_t v = threadIdx.x; v < dv; v += blockDim.x) pm_store<E, V>(rows + (size_t)r * c.D.rows_stride + (size_t)v * V, zero);
}

// ---------------------------------------------------------------------------
// plan and rows of a few pairs in one launch
// ---------------------------------------------------------------------------
// Grid (token, slab of 256 vectors). Every CTA sorts all pairs for itself - at most PM_ROWS_SMALL_PAIRS, in shared memory -
// and copies its piece of its token: no CTA waits for another.
template <typename E, int V>
__global__ void __launch_bounds__(256) k_rows_dispatch_small(RowsCall c, const uint32_t *__restrict__ ids, const float *__restrict__ w, bool scale,
                                                             const E *__restrict__ x, E *__restrict__ rows) {
  pm_pdl();
  __shared__ uint16_t le[PM_ROWS_SMALL_PAIRS];
  __shared__ uint32_t cnt[PM_MAX_EXPERTS], off[PM_MAX_EXPERTS + 1], part[8];
  __shared__ uint32_t at[PM_MAX_TOPK];
  __shared__ float ws[PM_MAX_TOPK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = c.D.top_k;
  const uint32_t P = (uint32_t)c.T * K, t = blockIdx.x, p0 = t * K, dv = (uint32_t)c.D.d / V;
  const uint32_t v0 = blockIdx.y * 256 + tid;
  Raw<E, V> mine;
  if (x && v0 < dv) mine = pm_load<E, V>(x + (size_t)t * c.D.x_stride + (size_t)v0 * V);
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
  if (c.D.align > 1)
    for (uint32_t e = cta; e < (uint32_t)c.D.n_local; e += n_cta) {
      const uint32_t from = off[e] + cnt[e], to = off[e + 1];
      if (from + tid < to) rows_write_pad(c, e, from + tid);  // (less than the alignment, 256 at most)
      if (x) rows_zero<E, V>(c, rows, from, to);
    }
  if (!x) return;
  __syncthreads();
  for (uint32_t v = v0; v < dv; v += gridDim.y * 256) {
    if (v != v0) mine = pm_load<E, V>(x + (size_t)t * c.D.x_stride + (size_t)v * V);
    float f[V];
    pm_widen<E, V>(mine, f);
    for (int k = 0; k < K; k++) {
      if (at[k] == PM_ROWS_NONE) continue;
      Raw<E, V> o = mine;
      if (scale) {
        float g[V];
#pragma unroll
        for (int i = 0; i < V; i++) g[i] = __fmul_rn(f[i], ws[k]);
        o = pm_narrow<E, V>(g);
      }
      pm_store<E, V>(rows + (size_t)at[k] * c.D.rows_stride + (size_t)v * V, o);
    }
  }
}

// ---------------------------------------------------------------------------
// the plan of many pairs
// ---------------------------------------------------------------------------
// One cluster of 8 CTAs x 32 warps; a warp owns a run of pairs. First pass: a pair's rank within its warp (match.any: the
// lanes with the same expert) and the warp's counts, u16 in shared memory. Then sums over a CTA's warps, over the CTAs
// through distributed shared memory, over the experts. Second pass: positions. No scratch in global memory, so a recorded
// graph holds no pointer of the library's; a pair's rank waits for the second pass in its place of `pos`.
#define SORT_CTAS 8
#define SORT_WARPS 32
__global__ void __cluster_dims__(SORT_CTAS, 1, 1) __launch_bounds__(SORT_WARPS * 32)
    k_rows_sort(RowsCall c, const uint32_t *__restrict__ ids, const float *__restrict__ w) {
  pm_pdl();
  __shared__ uint16_t hist[SORT_WARPS][PM_MAX_EXPERTS];
  __shared__ uint32_t total[PM_MAX_EXPERTS], cnt[PM_MAX_EXPERTS], off[PM_MAX_EXPERTS + 1], part[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster.block_rank(), P = (uint32_t)c.T * c.D.top_k;
  // a run of 32 * steps pairs a warp
  const uint32_t steps = (P + SORT_CTAS * SORT_WARPS * 32 - 1) / (SORT_CTAS * SORT_WARPS * 32);
  const uint32_t first = (rank * SORT_WARPS + warp) * steps * 32 + lane;
  for (int i = tid; i < SORT_WARPS * PM_MAX_EXPERTS / 2; i += SORT_WARPS * 32) ((uint32_t *)hist)[i] = 0;
  __syncthreads();
  for (uint32_t s = 0; s < steps; s++) {
    const uint32_t p = first + s * 32, e = p < P ? rows_local(c, ids[p]) : ROWS_NO_EXPERT;
    const uint32_t same = __match_any_sync(PM_FULL, e);
    const uint32_t before = __popc(same & ((1u << lane) - 1));
    uint32_t have = 0;
    if (e != ROWS_NO_EXPERT) have = hist[warp][e];
    __syncwarp();
    if (e != ROWS_NO_EXPERT && before == 0) hist[warp][e] = (uint16_t)(have + __popc(same));
    __syncwarp();
    if (p < P) c.pl.pos[p] = e != ROWS_NO_EXPERT ? have + before : PM_ROWS_NONE;
  }
  __syncthreads();
  if (tid < PM_MAX_EXPERTS) {  // the warps' counts become what lies before each warp (a CTA has 32,768 pairs at most)
    uint32_t sum = 0;
#pragma unroll 8
    for (int i = 0; i < SORT_WARPS; i++) {
      const uint32_t n = hist[i][tid];
      hist[i][tid] = (uint16_t)sum;
      sum += n;
    }
    total[tid] = sum;
  }
  cluster.sync();
  uint32_t ahead = 0;  // pairs of expert tid in the CTAs before this one
  if (tid < PM_MAX_EXPERTS) {
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < SORT_CTAS; i++) {
      const uint32_t n = cluster.map_shared_rank(total, i)[tid];
      if (i < (int)rank) ahead += n;
      all += n;
    }
    cnt[tid] = all;
  }
  cluster.sync();  // nobody reads another CTA's counts any more
  rows_scan(cnt, c.D.align, off, part);
  if (tid < PM_MAX_EXPERTS) total[tid] = off[tid] + ahead;
  if (rank == 0) {
    for (int e = tid; e < c.D.n_local; e += SORT_WARPS * 32) {
      c.pl.offset[e] = off[e];
      c.pl.count[e] = cnt[e];
    }
    if (tid == 0) c.pl.offset[c.D.n_local] = off[c.D.n_local];
  }
  __syncthreads();
  for (uint32_t s = 0; s < steps; s++) {
    const uint32_t p = first + s * 32;
    if (p >= P) break;
    const uint32_t r = c.pl.pos[p];
    if (r == PM_ROWS_NONE) continue;
    const uint32_t e = rows_local(c, ids[p]);
    rows_write_pair(c, w, p, e + (uint32_t)c.D.first_expert, total[e] + hist[warp][e] + r);
  }
  if (c.D.align > 1 && (c.pl.row_pair || c.pl.row_expert || c.pl.row_weight))
    for (uint32_t e = rank * SORT_WARPS + warp; e < (uint32_t)c.D.n_local; e += SORT_CTAS * SORT_WARPS)
      for (uint32_t r = off[e] + cnt[e] + lane; r < off[e + 1]; r += 32) rows_write_pad(c, e, r);
}

// ---------------------------------------------------------------------------
// copies and sums without a dot product: a thread a vector of a token
// ---------------------------------------------------------------------------
// Grid: CTAs of 256 vectors, behind them (SPREAD) one CTA an expert for the padding of its group.
template <typename E, int V>
__global__ void __launch_bounds__(256) k_rows_spread(RowsCall c, uint32_t copy_ctas, const float *__restrict__ w, const E *__restrict__ src,
                                                     E *__restrict__ out) {
  pm_pdl();
  const uint32_t dv = (uint32_t)c.D.d / V, K = c.D.top_k;
  if (blockIdx.x >= copy_ctas) {
    const uint32_t e = blockIdx.x - copy_ctas;
    const uint32_t from = c.pl.offset[e] + c.pl.count[e], to = c.pl.offset[e + 1];
    rows_zero<E, V>(c, out, from, (uint32_t)min((int64_t)to, c.pl.max_rows));
    return;
  }
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, t = i / dv, v = i - t * dv;
  if (t >= (uint32_t)c.T) return;
  const Raw<E, V> mine = pm_load<E, V>(src + (size_t)t * c.D.x_stride + (size_t)v * V);
  float f[V];
  pm_widen<E, V>(mine, f);
  for (uint32_t k = 0; k < K; k++) {
    const uint32_t pos = rows_pos(c, c.pl.pos[t * K + k]);
    if (pos == PM_ROWS_NONE) continue;
    Raw<E, V> o = mine;
    if (w) {
      const float wk = w[t * K + k];
      float g[V];
#pragma unroll
      for (int j = 0; j < V; j++) g[j] = __fmul_rn(f[j], wk);
      o = pm_narrow<E, V>(g);
    }
    pm_store<E, V>(out + (size_t)pos * c.D.rows_stride + (size_t)v * V, o);
  }
}

// KB: pairs whose reads are in flight together
template <typename E, int V, int KB>
__global__ void __launch_bounds__(256) k_rows_gather(RowsCall c, const float *__restrict__ w, const E *__restrict__ rows, const E *add, E *out) {
  pm_pdl();
  const uint32_t dv = (uint32_t)c.D.d / V, K = c.D.top_k;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, t = i / dv, v = i - t * dv;
  if (t >= (uint32_t)c.T) return;
  float acc[V] = {};
  if (add) pm_widen<E, V>(pm_load<E, V>(add + (size_t)t * c.D.x_stride + (size_t)v * V), acc);
  for (uint32_t k0 = 0; k0 < K; k0 += KB) {
    Raw<E, V> r[KB];
    float wk[KB];
    bool has[KB];
#pragma unroll
    for (int k = 0; k < KB; k++) {
      const uint32_t pos = k0 + k < K ? rows_pos(c, c.pl.pos[t * K + k0 + k]) : PM_ROWS_NONE;
      has[k] = pos != PM_ROWS_NONE;
      if (has[k]) {
        r[k] = pm_load<E, V>(rows + (size_t)pos * c.D.rows_stride + (size_t)v * V);
        wk[k] = w ? w[t * K + k0 + k] : 1.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < KB; k++)
      if (has[k]) {
        float f[V];
        pm_widen<E, V>(r[k], f);
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] = __fmaf_rn(wk[k], f[j], acc[j]);
      }
  }
  pm_store<E, V>(out + (size_t)t * c.D.x_stride + (size_t)v * V, pm_narrow<E, V>(acc));
}

// ---------------------------------------------------------------------------
// gradients with the weights' dot products: W warps a token
// ---------------------------------------------------------------------------
// A lane walks its vectors of the token's row and of its K rows, so the K dot products stay in its registers; lanes are
// summed once a token. SPREAD: rows read, out[pos] = w src[t] written (the gradient of collect). Otherwise out[t] = sum of
// w rows[pos] (the gradient of dispatch). Behind the tokens' CTAs (SPREAD), one an expert for the padding.
template <typename E, int V, int KB, bool SPREAD>
__global__ void __launch_bounds__(256) k_rows_dot(RowsCall c, uint32_t token_ctas, int W, const float *__restrict__ w, const E *__restrict__ src,
                                                  const E *__restrict__ rows, E *__restrict__ out, float *__restrict__ dw) {
  pm_pdl();
  __shared__ float sums[8][KB];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t dv = (uint32_t)c.D.d / V, K = c.D.top_k;
  if (SPREAD && blockIdx.x >= token_ctas) {
    const uint32_t e = blockIdx.x - token_ctas;
    const uint32_t from = c.pl.offset[e] + c.pl.count[e], to = c.pl.offset[e + 1];
    rows_zero<E, V>(c, out, from, (uint32_t)min((int64_t)to, c.pl.max_rows));
    return;
  }
  const uint32_t t = blockIdx.x * (8 / W) + warp / W;
  const int part = warp % W;
  uint32_t pos[KB];
  float wk[KB], dot[KB];
#pragma unroll
  for (int k = 0; k < KB; k++) {
    const bool in = t < (uint32_t)c.T && k < (int)K;
    pos[k] = in ? rows_pos(c, c.pl.pos[t * K + k]) : PM_ROWS_NONE;
    wk[k] = in && w ? w[t * K + k] : 1.0f;
    dot[k] = 0.0f;
  }
  if (t < (uint32_t)c.T)
    for (uint32_t v = part * 32 + lane; v < dv; v += 32 * W) {
      const Raw<E, V> s = pm_load<E, V>(src + (size_t)t * c.D.x_stride + (size_t)v * V);
      Raw<E, V> r[KB];
#pragma unroll
      for (int k = 0; k < KB; k++)
        if (pos[k] != PM_ROWS_NONE) r[k] = pm_load<E, V>(rows + (size_t)pos[k] * c.D.rows_stride + (size_t)v * V);
      float f[V], acc[V] = {};
      pm_widen<E, V>(s, f);
#pragma unroll
      for (int k = 0; k < KB; k++)
        if (pos[k] != PM_ROWS_NONE) {
          float g[V], o[V];
          pm_widen<E, V>(r[k], g);
#pragma unroll
          for (int j = 0; j < V; j++) {
            dot[k] = __fmaf_rn(f[j], g[j], dot[k]);
            if (SPREAD) o[j] = __fmul_rn(wk[k], f[j]);
            else acc[j] = __fmaf_rn(wk[k], g[j], acc[j]);
          }
          if (SPREAD) pm_store<E, V>(out + (size_t)pos[k] * c.D.rows_stride + (size_t)v * V, pm_narrow<E, V>(o));
        }
      if (!SPREAD) pm_store<E, V>(out + (size_t)t * c.D.x_stride + (size_t)v * V, pm_narrow<E, V>(acc));
    }
#pragma unroll
  for (int k = 0; k < KB; k++) dot[k] = pm_warp_sum_16_1(dot[k]);
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < KB; k++) sums[warp][k] = dot[k];
  }
  __syncthreads();
  if (part == 0 && lane < (int)K && t < (uint32_t)c.T) {
    float s = 0.0f;
    for (int i = 0; i < W; i++) s = __fadd_rn(s, sums[warp + i][lane]);
    dw[t * K + lane] = s;
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
static uint32_t rows_pad_ctas(const RowsCall &c) { return c.D.align > 1 ? (uint32_t)c.D.n_local : 0; }

template <typename E, int V>
static cudaError_t spread(const Launch &L, const RowsCall &c, const float *w, const void *src, void *out) {
  const uint32_t ctas = (uint32_t)(((size_t)c.T * rows_vectors(c) + 255) / 256);
  if (ctas + rows_pad_ctas(c) == 0) return cudaSuccess;
  return pm_launch(L, k_rows_spread<E, V>, ctas + rows_pad_ctas(c), 256, 0, c, ctas, w, (const E *)src, (E *)out);
}

template <typename E, int V>
static cudaError_t dispatch_small(const Launch &L, const RowsCall &c, const uint32_t *ids, const float *w, bool scale, const void *x, void *rows) {
  // (a call without tokens or rows still writes its offsets)
  const uint32_t slabs = x && c.T ? (rows_vectors(c) + 255) / 256 : 1;
  return pm_launch(L, k_rows_dispatch_small<E, V>, dim3(c.T > 0 ? c.T : 1, slabs), 256, 0, c, ids, w, scale, (const E *)(c.T ? x : nullptr), (E *)rows);
}

cudaError_t launch_rows_dispatch(const Launch &L, const RowsCall &c, const uint32_t *ids, const float *w, bool scale, const void *x, void *rows) {
  if ((size_t)c.T * c.D.top_k <= PM_ROWS_SMALL_PAIRS) {
#define CALL(E, V) dispatch_small<E, V>(L, c, ids, w, scale, x, rows)
    ROWS_TYPES(CALL);
#undef CALL
  }
  const cudaError_t e = pm_launch(L, k_rows_sort, SORT_CTAS, SORT_WARPS * 32, 0, c, ids, w);
  if (e != cudaSuccess || !x) return e;
#define CALL(E, V) spread<E, V>(L, c, scale ? w : nullptr, x, rows)
  ROWS_TYPES(CALL);
#undef CALL
}

template <typename E, int V, int KB, bool SPREAD>
static cudaError_t dot(const Launch &L, const RowsCall &c, const float *w, const void *src, const void *rows, void *out, float *dw) {
  // warps a token: as many as give every SM 16 warps, while each has a vector a lane
  int W = 1;
  while (W < 8 && (int64_t)c.T * W < 16 * L.n_sm && rows_vectors(c) > (uint32_t)(32 * W)) W *= 2;
  const uint32_t ctas = ((uint32_t)c.T * W + 7) / 8, pad = SPREAD ? rows_pad_ctas(c) : 0;
  if (ctas + pad == 0) return cudaSuccess;
  return pm_launch(L, k_rows_dot<E, V, KB, SPREAD>, ctas + pad, 256, 0, c, ctas, W, w, (const E *)src, (const E *)rows, (E *)out, dw);
}
template <typename E, int V, bool SPREAD>
static cudaError_t dot_k(const Launch &L, const RowsCall &c, const float *w, const void *src, const void *rows, void *out, float *dw) {
  if (c.D.top_k <= 4) return dot<E, V, 4, SPREAD>(L, c, w, src, rows, out, dw);
  if (c.D.top_k <= 8) return dot<E, V, 8, SPREAD>(L, c, w, src, rows, out, dw);
  return dot<E, V, 16, SPREAD>(L, c, w, src, rows, out, dw);
}

template <typename E, int V>
static cudaError_t gather(const Launch &L, const RowsCall &c, const float *w, const void *rows, const void *add, void *out) {
  const uint32_t ctas = (uint32_t)(((size_t)c.T * rows_vectors(c) + 255) / 256);
  if (ctas == 0) return cudaSuccess;
  if (c.D.top_k <= 4) return pm_launch(L, k_rows_gather<E, V, 4>, ctas, 256, 0, c, w, (const E *)rows, (const E *)add, (E *)out);
  return pm_launch(L, k_rows_gather<E, V, 8>, ctas, 256, 0, c, w, (const E *)rows, (const E *)add, (E *)out);
}

cudaError_t launch_rows_gather(const Launch &L, const RowsCall &c, const float *w, const void *rows, const void *add, const void *x, void *out,
                               float *dw) {
  if (dw) {
#define CALL(E, V) dot_k<E, V, false>(L, c, w, x, rows, out, dw)
    ROWS_TYPES(CALL);
#undef CALL
  }
#define CALL(E, V) gather<E, V>(L, c, w, rows, add, out)
  ROWS_TYPES(CALL);
#undef CALL
}

cudaError_t launch_rows_spread(const Launch &L, const RowsCall &c, const float *w, const void *src, const void *rows, void *out, float *dw) {
  if (dw) {
#define CALL(E, V) dot_k<E, V, true>(L, c, w, src, rows, out, dw)
    ROWS_TYPES(CALL);
#undef CALL
  }
#define CALL(E, V) spread<E, V>(L, c, w, src, out)
  ROWS_TYPES(CALL);
#undef CALL
}
