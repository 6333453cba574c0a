// Softmax of attention scores with a learned bias per bucket of relative positions, and its backward pass.
//
//   a[i, j] = softmax_j(scale s[i, j] + table[bucket(j - i - q_offset), head] + mask[i, j]);   causal: j <= i + q_offset only
//   backward, g = the gradient of a:  ds = a (g - sum_j a g),   scores get scale ds,   table[k, head] the sum of ds over the
//   batch, the rows and the columns whose distance falls into bucket k
// bucket(d) is the number of a side's lower edges at or below |d|, less one; edges: see hyc.h.
//
// Bound by memory: one pass over the map (two of them in backward), a row in registers between its reduction and its store,
// fp32 between the loads and the one rounding.  A warp covers SPAN = 32 V NV columns: V adjacent elements per lane and access (8
// where rows are a multiple of 8 long; 2 and 1 where they are not, so that accesses stay aligned), NV accesses.  Rows up to SPAN
// belong to one warp; longer ones (WIDE) to the warps of a block, or of a cluster of blocks, which exchange one pair (largest
// element, sum) per warp and row.
//
// Forward: the bias depends on j - i alone and is constant beyond the last edge, so that a table of 2 L + 1 values in shared
// memory (L = the last edge) serves every row of a head; pieces of a row that lie beyond take the constant.
//
// Backward: the table's gradient needs the sums of ds along diagonals.  A warp takes consecutive rows, and from row to row the
// running sum of each diagonal moves one column to the right: within a lane's V columns that is an operand of the addition, between
// lanes one shuffle per V elements, and what leaves the warp's last column is put aside in shared memory.  After the last row the
// sums of SPAN + R - 1 diagonals are there, and each bucket's are added up: no atomics, the same bits on every run.  A small
// second launch adds the warps' sums per head (in 64 bits: whole maps that nearly cancel).
#include "elem.cuh"
#include <type_traits>

namespace hyc {

constexpr int kRbMaxSide = 128;          // buckets of one side
constexpr int kRbNarrowWarps = 8;        // warps of a block whose warps have rows of their own
constexpr int kRbMaxWarps = 16;          // warps of a block that share a row
constexpr int kRbMaxCluster = 8;

struct RbParams {
  const void *x, *grad, *table, *mask;
  void* out;
  float* part;                           // backward: [unit][buckets]
  int64_t mask_b, mask_h, mask_row;
  int64_t units;                         // backward: warps (narrow), blocks or clusters (wide) with rows
  int heads, n, cols, q_offset;
  int rows_per, chunks;                  // rows of a warp (narrow: of a warp; wide: of a block or cluster), chunks of a head's rows
  int cluster;                           // blocks that share a row
  int table_type, mask_type, mask_vec;
  int side, both, causal, buckets;
  float scale;
  int edges[kRbMaxSide];
};

template <typename T, int V> struct Piece;
template <typename T> struct Piece<T, 8> { Octet<T> raw; };
template <> struct Piece<float, 2> { float2 raw; };
template <> struct Piece<__half, 2> { uint32_t raw; };
template <> struct Piece<__nv_bfloat16, 2> { uint32_t raw; };
template <typename T> struct Piece<T, 1> { T raw; };

template <typename T> __device__ __forceinline__ void ld_piece(const T* p, Piece<T, 8>& o) { o.raw = ld_octet(p); }
template <typename T> __device__ __forceinline__ void ld_piece(const T* p, Piece<T, 2>& o) { o.raw = *reinterpret_cast<const decltype(o.raw)*>(p); }
template <typename T> __device__ __forceinline__ void ld_piece(const T* p, Piece<T, 1>& o) { o.raw = *p; }
template <typename T> __device__ __forceinline__ void piece_f32(const Piece<T, 8>& o, float (&f)[8]) { octet_to_f32(o.raw, f); }
__device__ __forceinline__ void piece_f32(const Piece<float, 2>& o, float (&f)[2]) { f[0] = o.raw.x; f[1] = o.raw.y; }
__device__ __forceinline__ void piece_f32(const Piece<__half, 2>& o, float (&f)[2]) { const float2 t = half2_bits_to_f32(o.raw); f[0] = t.x; f[1] = t.y; }
__device__ __forceinline__ void piece_f32(const Piece<__nv_bfloat16, 2>& o, float (&f)[2]) { f[0] = bf16lo_to_f32(o.raw); f[1] = bf16hi_to_f32(o.raw); }
template <typename T> __device__ __forceinline__ void piece_f32(const Piece<T, 1>& o, float (&f)[1]) { f[0] = to_f32(o.raw); }
template <typename T> __device__ __forceinline__ void st_piece(T* p, const float (&f)[8]) { st_octet(p, f); }
__device__ __forceinline__ void st_piece(float* p, const float (&f)[2]) { *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]); }
__device__ __forceinline__ void st_piece(__half* p, const float (&f)[2]) { *reinterpret_cast<uint32_t*>(p) = f32_to_half2_bits(f[0], f[1]); }
__device__ __forceinline__ void st_piece(__nv_bfloat16* p, const float (&f)[2]) { *reinterpret_cast<uint32_t*>(p) = pack_bf16x2_rn(f[0], f[1]); }
template <typename T> __device__ __forceinline__ void st_piece(T* p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// e^v for v <= 0 (or NaN): two roundings and the two units in the last place of the instruction; below 2^-126 it is 0
__device__ __forceinline__ float exp_neg(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
  return r;
}

// ---- exchange between the warps that share a row: every warp gives a pair and receives all of them combined.  `turn` alternates,
// so that the next row's values cannot meet this one's readers.
struct RbExchange {
  float2 warp[2][kRbMaxWarps];
  float2 block[2][kRbMaxCluster];
};
__device__ __forceinline__ void rb_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void rb_put(float2* slot, int rank, float2 v) {      // into block `rank` of the cluster
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(slot)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(v.x), "f"(v.y) : "memory");
}
template <typename F>
__device__ __forceinline__ float2 rb_exchange(RbExchange& ex, int turn, int warps, int cluster, int rank, float2 mine, F&& join) {
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) ex.warp[turn][warp] = mine;
  __syncthreads();
  float2 all = ex.warp[turn][0];
  for (int w = 1; w < warps; ++w) all = join(all, ex.warp[turn][w]);
  if (cluster == 1) return all;
  if ((int)threadIdx.x < cluster) rb_put(&ex.block[turn][rank], (int)threadIdx.x, all);
  rb_cluster_sync();
  all = ex.block[turn][0];
  for (int c = 1; c < cluster; ++c) all = join(all, ex.block[turn][c]);
  return all;
}
// (largest element, sum of exponentials relative to it)
__device__ __forceinline__ float2 join_softmax(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(m, a.y + b.y);
  return make_float2(m, a.y * exp_neg(a.x - m) + b.y * exp_neg(b.x - m));
}

// the bias table, spread so that lanes eight columns apart meet in no bank
__device__ __forceinline__ int lut_at(int x) { return x + (x >> 3); }

__device__ __forceinline__ int rb_bucket(const int* edges, int side, int distance) {      // number of edges <= distance, less one
  int lo = 0, hi = side;                                                                // edges[lo] <= distance < edges[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (edges[mid] <= distance) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T, int V, int NV, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 32 * kRbMaxWarps : 32 * kRbNarrowWarps)
relbias_fwd_kernel(const __grid_constant__ RbParams p) {
  extern __shared__ float s_lut[];
  __shared__ int s_edges[kRbMaxSide];
  __shared__ RbExchange s_ex;
  constexpr int SPAN = 32 * V * NV;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rank = WIDE ? (int)(blockIdx.x % (unsigned)p.cluster) : 0;
  const uint32_t unit = blockIdx.x / (unsigned)p.cluster;
  const int bh = (int)(unit / (uint32_t)p.chunks), chunk = (int)(unit - (uint32_t)bh * (uint32_t)p.chunks);
  const int b = bh / p.heads, h = bh - b * p.heads;
  const int step = WIDE ? 1 : kRbNarrowWarps;
  const int first = chunk * p.rows_per * step + (WIDE ? 0 : warp);
  const int last = min((chunk + 1) * p.rows_per * step, p.n);
  const int far = p.edges[p.side - 1], ahead = p.both ? far : 0;      // distances are told apart from -far to ahead
  for (int i = threadIdx.x; i < p.side; i += blockDim.x) s_edges[i] = p.edges[i];
  pdl_wait();
  __syncthreads();
  for (int i = threadIdx.x; i <= far + ahead; i += blockDim.x) {
    const int d = i - far;
    const int k = rb_bucket(s_edges, p.side, d < 0 ? -d : (p.both ? d : 0)) + (p.both && d > 0 ? p.side : 0);
    s_lut[lut_at(i)] = ld_any(p.table, (int64_t)k * p.heads + h, p.table_type);
  }
  __syncthreads();
  if (WIDE && p.cluster > 1) rb_cluster_sync();      // the other blocks have started: their shared memory may be written
  const float bias_behind = s_lut[0], bias_ahead = s_lut[lut_at(far + ahead)];
  const int c0 = WIDE ? (rank * warps + warp) * SPAN : 0;
  const int64_t map = (int64_t)bh * p.n;
  const T* x = reinterpret_cast<const T*>(p.x) + map * p.cols;
  T* out = reinterpret_cast<T*>(p.out) + map * p.cols;
  int turn = 0;
  for (int i = first; i < last; i += step, turn ^= 1) {
    const int q = i + p.q_offset;
    const int end = p.causal ? (q < -1 ? 0 : (q + 1 < p.cols ? q + 1 : p.cols)) : p.cols;      // columns that count
    const T* row = x + (int64_t)i * p.cols;
    Piece<T, V> raw[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * 32 * V + lane * V;
      if (c < end) ld_piece(row + c, raw[k]);
    }
    float f[NV][V], m = -INFINITY;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int cb = c0 + k * 32 * V, c = cb + lane * V;
      if (cb >= end) {                   // (the whole warp)
#pragma unroll
        for (int e = 0; e < V; ++e) f[k][e] = -INFINITY;
        continue;
      }
      float bias[V];
      const int dmin = cb - q, dmax = cb + 32 * V - 1 - q;
      if (dmax <= -far || dmin >= ahead) {
        const float v = dmax <= -far ? bias_behind : bias_ahead;
#pragma unroll
        for (int e = 0; e < V; ++e) bias[e] = v;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) bias[e] = s_lut[lut_at(min(max(c + e - q, -far), ahead) + far)];
      }
      if (p.mask != nullptr && c < end) {
        const int64_t at = b * p.mask_b + h * p.mask_h + (int64_t)i * p.mask_row + c;
        if (V == 8 && p.mask_vec) {
          float mk[8];
          ld_any8(p.mask, at, p.mask_type, mk);
#pragma unroll
          for (int e = 0; e < V; ++e) bias[e] += mk[e & 7];
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) bias[e] += ld_any(p.mask, at + e, p.mask_type);
        }
      }
      if (c < end) piece_f32(raw[k], f[k]);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[k][e] = c + e < end ? fmaf(f[k][e], p.scale, bias[e]) : -INFINITY;
        m = fmaxf(m, f[k][e]);
      }
    }
    m = warp_max(m);
    const float mm = m == -INFINITY ? 0.f : m;      // nothing counts: e^-inf = 0 everywhere
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) { f[k][e] = exp_neg(f[k][e] - mm); sum += f[k][e]; }
    sum = warp_sum(sum);
    float factor;
    if (WIDE) {
      const float2 all = rb_exchange(s_ex, turn, warps, p.cluster, rank, make_float2(m, sum), join_softmax);
      factor = (m == -INFINITY ? 1.f : exp_neg(m - all.x)) / all.y;
      if (all.y == 0.f) factor = 0.f;
    } else {
      factor = sum == 0.f ? 0.f : 1.f / sum;        // a row that nothing is visible to: zeros
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * 32 * V + lane * V;
      if (c >= p.cols) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) f[k][e] = c + e < end ? f[k][e] * factor : 0.f;      // (zero in a row that became NaN, too)
      st_piece(out + (int64_t)i * p.cols + c, f[k]);
    }
  }
}

// the distances of bucket k: from .. to
__device__ __forceinline__ void rb_range(const RbParams& p, const int* edges, int k, int& from, int& to) {
  if (p.both && k >= p.side) {
    k -= p.side;
    from = max(1, edges[k]);
    to = k + 1 < p.side ? edges[k + 1] - 1 : 0x3fffffff;
  } else {
    to = k == 0 && !p.both ? 0x3fffffff : -edges[k];
    from = k + 1 < p.side ? 1 - edges[k + 1] : -0x3fffffff;
  }
}

template <typename T, int V, int NV, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 32 * kRbMaxWarps : 32 * kRbNarrowWarps)
relbias_bwd_kernel(const __grid_constant__ RbParams p) {
  extern __shared__ float s_diag_all[];
  __shared__ int s_edges[kRbMaxSide];
  __shared__ RbExchange s_ex;
  constexpr int SPAN = 32 * V * NV;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rank = WIDE ? (int)(blockIdx.x % (unsigned)p.cluster) : 0;
  for (int i = threadIdx.x; i < p.side; i += blockDim.x) s_edges[i] = p.edges[i];
  __syncthreads();
  pdl_wait();
  if (WIDE && p.cluster > 1) rb_cluster_sync();      // the other blocks have started: their shared memory may be written
  // a unit: `rows_per` consecutive rows of one map, for a warp or for the warps that share a row
  const int64_t unit = WIDE ? blockIdx.x / (unsigned)p.cluster : (int64_t)blockIdx.x * kRbNarrowWarps + warp;
  const int bh = (int)(unit / p.chunks), chunk = (int)(unit - (int64_t)bh * p.chunks);
  const int first = chunk * p.rows_per, last = min(first + p.rows_per, p.n) - 1;
  if (!WIDE && unit >= p.units) return;
  float* s_diag = s_diag_all + warp * (SPAN + p.rows_per);
  const int c0 = WIDE ? (rank * warps + warp) * SPAN : 0;
  const int64_t map = (int64_t)bh * p.n;
  const T *a = reinterpret_cast<const T*>(p.x) + map * p.cols, *g = reinterpret_cast<const T*>(p.grad) + map * p.cols;
  T* out = reinterpret_cast<T*>(p.out) + map * p.cols;
  float acc[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[k][e] = 0.f;
  int turn = 0;
  for (int i = first; i <= last; ++i, turn ^= 1) {
    const int q = i + p.q_offset;
    const int end = p.causal ? (q < -1 ? 0 : (q + 1 < p.cols ? q + 1 : p.cols)) : p.cols;
    float ds[NV][V], dot = 0.f;
    Piece<T, V> ra[NV], rg[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * 32 * V + lane * V;
      if (c < end) {
        ld_piece(a + (int64_t)i * p.cols + c, ra[k]);
        ld_piece(g + (int64_t)i * p.cols + c, rg[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * 32 * V + lane * V;
      if (c >= end) continue;
      float fa[V], fg[V];
      piece_f32(ra[k], fa);
      piece_f32(rg[k], fg);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e < end) dot = fmaf(fa[e], fg[e], dot);
    }
    dot = warp_sum(dot);
    if (WIDE) dot = rb_exchange(s_ex, turn, warps, p.cluster, rank, make_float2(dot, 0.f), [](float2 u, float2 v) { return make_float2(u.x + v.x, 0.f); }).x;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * 32 * V + lane * V;
      float fa[V], fg[V];
      if (c < end) { piece_f32(ra[k], fa); piece_f32(rg[k], fg); }
#pragma unroll
      for (int e = 0; e < V; ++e) ds[k][e] = c + e < end ? fa[e] * (fg[e] - dot) : 0.f;
      if (c < p.cols) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = ds[k][e] * p.scale;
        st_piece(out + (int64_t)i * p.cols + c, o);
      }
    }
    // the diagonals' running sums one column to the right, this row's share added
    float left = 0.f;                    // lane 0: what leaves the piece of columns before
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const float moved = __shfl_sync(0xffffffffu, acc[k][V - 1], (lane + 31) & 31);
      const float carry = lane == 0 ? left : moved;
      left = moved;
#pragma unroll
      for (int e = V - 1; e > 0; --e) acc[k][e] = acc[k][e - 1] + ds[k][e];
      acc[k][0] = carry + ds[k][0];
    }
    if (lane == 0 && i > first) s_diag[SPAN + last - i] = left;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) s_diag[k * 32 * V + lane * V + e] = acc[k][e];
  __syncwarp();
  // s_diag[x] is the sum of the diagonal at distance x + dmin
  const int dmin = c0 - last - p.q_offset, dmax = dmin + SPAN - 1 + (last - first);
  float* part = p.part + ((WIDE ? unit * p.cluster * warps + rank * warps + warp : unit)) * p.buckets;
  float mine = 0.f;
  for (int k = 0; k < p.buckets; ++k) {
    int from, to;
    rb_range(p, s_edges, k, from, to);
    from = max(from, dmin); to = min(to, dmax);
    float sum = 0.f;
    if (from <= to) {
      for (int d = from + lane; d <= to; d += 32) sum += s_diag[d - dmin];
      sum = warp_sum(sum);
    }
    if ((k & 31) == lane) mine = sum;
    if ((k & 31) == 31 || k == p.buckets - 1) {
      if ((k & ~31) + lane < p.buckets) part[(k & ~31) + lane] = mine;
    }
  }
}

// table[k, head]: the units' sums of a head, 32 buckets per block
__global__ void __launch_bounds__(1024)
relbias_table_kernel(const float* __restrict__ part, int batch, int heads, int per_map, int buckets, float* __restrict__ table) {
  __shared__ double s_sum[32][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = (int)blockIdx.x, k = (int)blockIdx.y * 32 + lane;
  double sum = 0.0;
  if (k < buckets)
    for (int b = 0; b < batch; ++b) {
      const float* src = part + ((int64_t)(b * heads + h) * per_map) * buckets + k;
      for (int u = warp; u < per_map; u += 32) sum += (double)src[(int64_t)u * buckets];
    }
  s_sum[warp][lane] = sum;
  __syncthreads();
  sum = s_sum[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int at = (int)blockIdx.y * 32 + warp;
  if (lane == 0 && at < buckets) table[(int64_t)at * heads + h] = (float)sum;
}

// ---- host side
static int rb_check(const hyc_relative_bias* a, bool backward) {
  if (a == nullptr || a->host_edges == nullptr) return HYC_ERR_NULL;
  if (!elem_type_ok(a->type)) return HYC_ERR_UNSUPPORTED;
  if (!backward && (!elem_type_ok(a->table_type) || (a->mask != nullptr && !elem_type_ok(a->mask_type)))) return HYC_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->heads < 1 || a->n < 0 || a->cols < 1 || a->batch > 0x7fffffffll || a->n > 0x3fffffffll || a->cols > HYC_RELATIVE_BIAS_MAX_COLS ||
      (a->batch * a->n != 0 && a->batch * a->n > 0x7fffffffll / a->heads) || a->q_offset < -0x1fffffffll || a->q_offset > 0x1fffffffll)
    return HYC_ERR_SHAPE;
  if (a->side < 1 || a->side > kRbMaxSide || a->host_edges[0] != 0 || a->host_edges[a->side - 1] > HYC_RELATIVE_BIAS_MAX_DISTANCE) return HYC_ERR_SHAPE;
  for (int i = 1; i < a->side; ++i)
    if (a->host_edges[i] < a->host_edges[i - 1]) return HYC_ERR_SHAPE;
  if (a->batch * a->n == 0) return HYC_OK;
  if (a->x == nullptr || a->out == nullptr || (backward ? a->grad == nullptr : a->table == nullptr)) return HYC_ERR_NULL;
  const size_t e = (size_t)elem_bytes(a->type);
  if (!aligned(a->x, e) || !aligned(a->out, e) || (backward && !aligned(a->grad, e))) return HYC_ERR_ALIGN;
  if (!backward && (!aligned(a->table, (size_t)elem_bytes(a->table_type)) || (a->mask != nullptr && !aligned(a->mask, (size_t)elem_bytes(a->mask_type)))))
    return HYC_ERR_ALIGN;
  return HYC_OK;
}

// How a map is cut: V adjacent elements per access, accesses per lane, warps (and blocks of a cluster) of a row
struct RbPlan { int v, nv, warps, cluster; bool wide; };
static RbPlan rb_plan(const hyc_relative_bias* a, bool backward) {
  RbPlan r;
  const size_t e = (size_t)elem_bytes(a->type);
  auto fits = [&](int v) {
    const size_t bytes = v == 8 ? 16 : v * e;      // (a piece of 8 fp32 values is two accesses)
    return a->cols % v == 0 && aligned(a->x, bytes) && aligned(a->out, bytes) && (!backward || aligned(a->grad, bytes));
  };
  r.v = fits(8) ? 8 : fits(2) ? 2 : 1;
  const int64_t rows = a->batch * a->heads * a->n, cols = a->cols;
  r.cluster = 1;
  if (cols <= 1024) {
    r.wide = false;
    r.warps = kRbNarrowWarps;
    r.nv = (cols <= 256 ? 256 : cols <= 512 && r.v == 8 ? 512 : 1024) / (32 * r.v);
    return r;
  }
  // few rows: as many warps as a block may have; many: as few as can hold a row, for fewer exchanges
  r.wide = true;
  int span = 1024;
  if (cols <= 256 * kRbMaxWarps && rows * ((cols + 1023) / 1024) < (int64_t)num_sms() * 16) span = 256;
  while (cols > (int64_t)r.cluster * kRbMaxWarps * span) r.cluster *= 2;
  r.warps = (int)((cols + (int64_t)r.cluster * span - 1) / ((int64_t)r.cluster * span));
  r.nv = span / (32 * r.v);
  return r;
}
// rows of a unit, so that there are a few times as many units as can be resident
static int rb_rows_per(const RbPlan& r, int64_t rows, int n, int most) {
  const int64_t resident = (int64_t)num_sms() * 32 / (r.wide ? r.warps * r.cluster : 1);
  int64_t per = rows / (resident < 1 ? 1 : 2 * resident);
  per = per < 1 ? 1 : per > most ? most : per;
  return (int)(per > n ? n : per);
}
constexpr int kRbRowsFwd = 16, kRbRowsBwd = 32;

static void rb_fill(RbParams& p, const hyc_relative_bias* a, const RbPlan& r) {
  p.x = a->x; p.grad = a->grad; p.table = a->table; p.mask = a->mask; p.out = a->out; p.part = nullptr;
  p.mask_b = a->mask_b; p.mask_h = a->mask_h; p.mask_row = a->mask_row;
  p.heads = a->heads; p.n = (int)a->n; p.cols = (int)a->cols; p.q_offset = (int)a->q_offset;
  p.cluster = r.cluster;
  p.table_type = a->table_type; p.mask_type = a->mask_type;
  p.mask_vec = a->mask != nullptr && aligned(a->mask, 16) && ((a->mask_b | a->mask_h | a->mask_row) & 7) == 0;
  p.side = a->side; p.both = a->both != 0; p.causal = a->causal != 0; p.buckets = a->both ? 2 * a->side : a->side;
  p.scale = a->scale;
  for (int i = 0; i < a->side; ++i) p.edges[i] = a->host_edges[i];
}

template <typename K>
static int rb_launch(K kern, const RbPlan& r, int64_t blocks, size_t smem, const RbParams& p, cudaStream_t st) {
  if (blocks > 0x7fffffffll) return HYC_ERR_SHAPE;
  if (smem > 32768 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    hyc_set_last_cuda_error((int)cudaGetLastError());
    return HYC_ERR_LAUNCH;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)(32 * r.warps));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)r.cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = r.cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) {
    hyc_set_last_cuda_error((int)cudaGetLastError());
    return HYC_ERR_LAUNCH;
  }
  return HYC_OK;
}

// f(element, V, NV, WIDE) for the plan's kernel
template <typename F>
static int rb_by_plan(int type, const RbPlan& r, F&& f) {
  auto by_shape = [&](auto elem) -> int {
    auto wide = [&](auto v, auto nv) -> int {
      if (r.wide) return f(elem, v, nv, std::true_type());
      return f(elem, v, nv, std::false_type());
    };
    using std::integral_constant;
    if (r.v == 8) {
      if (r.nv == 1) return wide(integral_constant<int, 8>(), integral_constant<int, 1>());
      if (r.nv == 2) return f(elem, integral_constant<int, 8>(), integral_constant<int, 2>(), std::false_type());
      return wide(integral_constant<int, 8>(), integral_constant<int, 4>());
    }
    if (r.v == 2) {
      if (r.nv == 4) return wide(integral_constant<int, 2>(), integral_constant<int, 4>());
      return wide(integral_constant<int, 2>(), integral_constant<int, 16>());
    }
    if (r.nv == 8) return wide(integral_constant<int, 1>(), integral_constant<int, 8>());
    return wide(integral_constant<int, 1>(), integral_constant<int, 32>());
  };
  if (type == HYC_F32) return by_shape(float());
  if (type == HYC_F16) return by_shape(__half());
  return by_shape(__nv_bfloat16());
}

// backward: rows of a unit and the warps' sums that the workspace holds
struct RbUnits { int rows_per, chunks; int64_t units, sums; };
static RbUnits rb_units(const hyc_relative_bias* a, const RbPlan& r) {
  RbUnits u;
  u.rows_per = rb_rows_per(r, a->batch * a->heads * a->n, (int)a->n, kRbRowsBwd);
  u.chunks = (int)((a->n + u.rows_per - 1) / u.rows_per);
  u.units = a->batch * a->heads * u.chunks;
  u.sums = u.units * (r.wide ? r.warps * r.cluster : 1);
  return u;
}

}  // namespace hyc

using namespace hyc;

extern "C" HYC_API int hyc_softmax_relative_bias_fwd(const hyc_relative_bias* a, void* stream) {
  const int rc = rb_check(a, false);
  if (rc != HYC_OK || a->batch * a->n == 0) return rc;
  const RbPlan r = rb_plan(a, false);
  RbParams p;
  rb_fill(p, a, r);
  p.rows_per = rb_rows_per(r, a->batch * a->heads * a->n, (int)a->n, kRbRowsFwd);
  const int step = p.rows_per * (r.wide ? 1 : kRbNarrowWarps);
  p.chunks = (int)((a->n + step - 1) / step);
  const int far = p.edges[p.side - 1], values = far + (p.both ? far : 0) + 1;
  const size_t smem = (size_t)(values + values / 8 + 1) * sizeof(float);
  return rb_by_plan(a->type, r, [&](auto elem, auto v, auto nv, auto wide) -> int {
    return rb_launch(relbias_fwd_kernel<decltype(elem), decltype(v)::value, decltype(nv)::value, decltype(wide)::value>, r,
                     a->batch * a->heads * p.chunks * r.cluster, smem, p, (cudaStream_t)stream);
  });
}

extern "C" HYC_API size_t hyc_softmax_relative_bias_workspace_bytes(const hyc_relative_bias* a) {
  if (rb_check(a, true) != HYC_OK || a->batch * a->n == 0) return 0;
  return (size_t)rb_units(a, rb_plan(a, true)).sums * (size_t)(a->both ? 2 * a->side : a->side) * sizeof(float);
}

extern "C" HYC_API int hyc_softmax_relative_bias_bwd(const hyc_relative_bias* a, float* dtable, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = rb_check(a, true);
  if (rc != HYC_OK) return rc;
  if (dtable == nullptr) return HYC_ERR_NULL;
  if (!aligned(dtable, 4)) return HYC_ERR_ALIGN;
  const int buckets = a->both ? 2 * a->side : a->side;
  RbUnits u = {0, 0, 0, 0};
  RbPlan r = {8, 1, 1, 1, false};
  if (a->batch * a->n != 0) {
    r = rb_plan(a, true);
    u = rb_units(a, r);
    if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < (size_t)u.sums * (size_t)buckets * sizeof(float)) return HYC_ERR_WORKSPACE;
    RbParams p;
    rb_fill(p, a, r);
    p.part = (float*)workspace;
    p.rows_per = u.rows_per; p.chunks = u.chunks; p.units = u.units;
    const int64_t blocks = r.wide ? u.units * r.cluster : (u.units + kRbNarrowWarps - 1) / kRbNarrowWarps;
    const size_t smem = (size_t)r.warps * (size_t)(32 * r.v * r.nv + u.rows_per) * sizeof(float);
    const int rl = rb_by_plan(a->type, r, [&](auto elem, auto v, auto nv, auto wide) -> int {
      return rb_launch(relbias_bwd_kernel<decltype(elem), decltype(v)::value, decltype(nv)::value, decltype(wide)::value>, r, blocks, smem, p,
                       (cudaStream_t)stream);
    });
    if (rl != HYC_OK) return rl;
  }
  const int per_map = u.chunks * (r.wide ? r.warps * r.cluster : 1);
  launch_pdl(relbias_table_kernel, dim3((unsigned)a->heads, (unsigned)((buckets + 31) / 32)), dim3(1024), 0, (cudaStream_t)stream, (const float*)workspace,
             u.units > 0 ? (int)a->batch : 0, a->heads, per_map, buckets, dtable);
  HYC_CHECK_LAUNCH();
  return HYC_OK;
}
