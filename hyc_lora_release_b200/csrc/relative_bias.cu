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
// Forward: the bias depends on j - i alone, so that one vector of (columns + rows) values in shared memory serves all rows of a block;
// an element's bias is one load from it, eight columns apart from lane to lane and spread over the banks.  A block of fewer than four rows
// (single tokens) keeps the bias by distance instead, which is constant beyond the last edge ([4,32,1,32768] 20 -> 14 us).
//
// Backward: the table's gradient needs the sums of ds along diagonals.  A warp takes consecutive rows, and from row to row the
// running sum of each diagonal moves one column to the right: within a lane's V columns that is an operand of the addition, between
// lanes one shuffle per V elements, and what leaves the warp's last column is put aside in shared memory.  After the last row the
// sums of SPAN + R - 1 diagonals are there, and each bucket's are added up: no atomics, the same bits on every run.  A small
// second launch adds the warps' sums per head, in 64 bits.  Buckets hold long ranges whose sums nearly cancel: where warps share a row (WIDE: rows
// beyond a warp's span, and rows of more than 512 columns of which there are fewer than eight per SM) the row's product sum and the
// buckets' are in 64 bits too (in 32 the table's gradient of single tokens over 1277 columns and more was up to 15 times as far off as the formula's
// in 32 bits with sums in 64; everywhere it would cost 2 to 7 %).  Of many rows the sums average out; rows of up to 512 columns keep 32
// bits even if there is one of them: over 25 inputs each of 37 to 512 columns the gradient is 0.6 to 1.4 times as far off as that formula's (median).
//
// B200, us in a row of passes, share of the copy peak, forward / backward (with the second launch, 5 us): bf16 [4,32,512,512] 27 (padding, 0.77) / 47
// (0.66); [1,32,2048,2048] 103 (0.80) / 146 (0.84), causal 85 (0.72) / 112 (0.73); [2,32,696,696] causal 32 (0.45) / 37 (0.51); fp32 [4,16,1000,1000] 90
// (0.87) / 126 (0.93); fp16 [2,32,1002,1002] 50 (0.78) / 73 (0.80), [2,32,1001,1001] causal 62 (0.48) / 87 (0.45): single elements per access cost
// instructions.  Forward is bound by instruction issue (15 per element, exponentials a third of their unit), backward by the latency of its rows.
// (Figures of single choices, at the places, are launches alone.)
#include "elem.cuh"
#include <type_traits>

namespace hyc {

constexpr int kRbMaxSide = 128;          // buckets of one side
constexpr int kRbNarrowWarps = 8;        // forward: warps of a block whose warps have rows of their own
constexpr int kRbBwdWarps = 4;           // backward: the same
constexpr int kRbMaxWarps = 16;          // warps of a block that share a row
constexpr int kRbMaxCluster = 8;

struct RbParams {
  const void *x, *grad, *table, *mask;
  void* out;
  double* part;                          // backward: [unit][buckets]
  int64_t mask_b, mask_h, mask_row;
  int64_t units;                         // backward: warps (narrow), blocks or clusters (wide) with rows
  int heads, n, cols, q_offset;
  int rows_per, chunks;                  // rows of a warp (narrow: of a warp; wide: of a block or cluster), chunks of a head's rows
  int cluster;                           // blocks that share a row
  int table_type, mask_type, mask_vec;
  int mask_staged;                       // values of the mask that a block keeps in shared memory, or 0
  int compact;                           // the bias in shared memory is by distance up to the last edge, not by column
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

__device__ __forceinline__ float warp_max(float v) {      // (a NaN among the values is passed over)
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Exponents are kept times log2(e) / 256, so that an exponential is one fused multiply-add and one instruction (two units in the last place;
// below 2^-126 it is 0), and scores, biases and masks up to the ends of fp32's range stay finite and keep their order: only what is -infinity
// counts as nothing.
constexpr float kSteps = 256.f, kUnit = 1.4426950408889634f / kSteps;
__device__ __forceinline__ float exp2_neg(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 2^(kSteps (x - top)) is exp2_neg(x s + b): the product is exact, so that the largest element gives 1.  Where kSteps top is beyond fp32,
// two exponents are equal or so far apart that a quarter of the difference gives 0 as well.
struct Exponents { float s, b; };
__device__ __forceinline__ Exponents exponents(float top) {
  const float s = fabsf(top) > 1e36f ? 0.25f : kSteps;
  return {s, -top * s};
}

// ---- two fp32 operations per instruction, over the V values of a piece
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void halves(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
template <int V>
__device__ __forceinline__ void fma_all(float (&x)[V], float s, const float (&b)[V]) {      // x = x s + b
  if constexpr (V == 1) { x[0] = fmaf(x[0], s, b[0]); }
  else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      uint64_t r;
      asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(two(x[e], x[e + 1])), "l"(two(s, s)), "l"(two(b[e], b[e + 1])));
      halves(r, x[e], x[e + 1]);
    }
  }
}
template <int V>
__device__ __forceinline__ void add_all(float (&x)[V], const float (&b)[V]) {
  if constexpr (V == 1) { x[0] += b[0]; }
  else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      uint64_t r;
      asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(x[e], x[e + 1])), "l"(two(b[e], b[e + 1])));
      halves(r, x[e], x[e + 1]);
    }
  }
}
template <int V>
__device__ __forceinline__ void fma_one(float (&x)[V], float s, float b) {
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = b;
  fma_all(x, s, v);
}
template <int V>
__device__ __forceinline__ void add_one(float (&x)[V], float b) {
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = b;
  add_all(x, v);
}
template <int V>
__device__ __forceinline__ void mul_one(float (&x)[V], float b) {
  if constexpr (V == 1) { x[0] *= b; }
  else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      uint64_t r;
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(x[e], x[e + 1])), "l"(two(b, b)));
      halves(r, x[e], x[e + 1]);
    }
  }
}
template <int V>
__device__ __forceinline__ void mul_all(float (&x)[V], const float (&b)[V]) {
  if constexpr (V == 1) { x[0] *= b[0]; }
  else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      uint64_t r;
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(x[e], x[e + 1])), "l"(two(b[e], b[e + 1])));
      halves(r, x[e], x[e + 1]);
    }
  }
}

// ---- exchange between the warps that share a row: every warp gives a value of 8 bytes and receives all of them combined.  `turn` alternates,
// so that the next row's values cannot meet this one's readers.
template <typename E>
struct RbExchange {
  E warp[2][kRbMaxWarps];
  E block[2][kRbMaxCluster];
};
__device__ __forceinline__ void rb_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void rb_put(void* slot, int rank, float2 v) {      // into block `rank` of the cluster
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(slot)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ void rb_put(void* slot, int rank, double v) {
  const long long bits = __double_as_longlong(v);
  rb_put(slot, rank, make_float2(__int_as_float((int)bits), __int_as_float((int)(bits >> 32))));
}
template <typename E, typename F>
__device__ __forceinline__ E rb_exchange(RbExchange<E>& ex, int turn, int warps, int cluster, int rank, E mine, F&& join) {
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) ex.warp[turn][warp] = mine;
  __syncthreads();
  E all = ex.warp[turn][0];
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
  return make_float2(m, a.y * exp2_neg((a.x - m) * kSteps) + b.y * exp2_neg((b.x - m) * kSteps));
}

// the bias table, spread for lanes eight columns apart so that they meet in no bank
template <int V> __device__ __forceinline__ int lut_at(int x) { return V == 8 ? x + (x >> 3) : x; }

__device__ __forceinline__ int rb_bucket(const int* edges, int side, int distance) {      // number of edges <= distance, less one
  int lo = 0, hi = side;                                                                // edges[lo] <= distance < edges[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (edges[mid] <= distance) lo = mid; else hi = mid;
  }
  return lo;
}

// columns of row i that count
__device__ __forceinline__ int rb_end(const RbParams& p, int i) {
  const int q = i + p.q_offset;
  return p.causal ? max(0, min(q + 1, p.cols)) : p.cols;
}

template <typename T, int V, int NV, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 32 * kRbMaxWarps : 32 * kRbNarrowWarps, WIDE ? 1 : V * NV <= 8 ? 5 : V * NV <= 16 ? 4 : 2)
relbias_fwd_kernel(const __grid_constant__ RbParams p) {
  extern __shared__ __align__(16) float s_mem[];
  __shared__ int s_edges[kRbMaxSide];
  __shared__ float s_table[2 * kRbMaxSide];
  __shared__ RbExchange<float2> s_ex;
  constexpr int SPAN = 32 * V * NV;
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), warps = blockDim.x >> 5;
  const int rank = WIDE ? (int)(blockIdx.x % (unsigned)p.cluster) : 0;
  float *s_mask = s_mem, *s_lut = s_mem + p.mask_staged;      // a mask that all rows share, the block's columns; the bias
  const uint32_t unit = blockIdx.x / (unsigned)p.cluster;
  const int bh = (int)(unit / (uint32_t)p.chunks), chunk = p.chunks - 1 - (int)(unit - (uint32_t)bh * (uint32_t)p.chunks);      // (causal: long rows first)
  const int b = bh / p.heads, h = bh - b * p.heads;
  const int first = (WIDE ? chunk : chunk * kRbNarrowWarps + warp) * p.rows_per, last = min(first + p.rows_per, p.n);
  const int block_rows = WIDE ? p.rows_per : kRbNarrowWarps * p.rows_per;
  const int q_last = min((chunk + 1) * block_rows, p.n) - 1 + p.q_offset;      // of the block's rows
  const int block_c0 = WIDE ? rank * warps * SPAN : 0;
  const int c0 = WIDE ? block_c0 + warp * SPAN : 0;
  const int64_t map = (int64_t)bh * p.n;
  // (at the lane's first column of the row to be read, of the row to be written)
  const int cl = c0 + lane * V;
  const T* src = reinterpret_cast<const T*>(p.x) + (map + first) * p.cols + cl;
  T* dst = reinterpret_cast<T*>(p.out) + (map + first) * p.cols + cl;
  for (int i = threadIdx.x; i < p.side; i += blockDim.x) s_edges[i] = p.edges[i];
  pdl_wait();
  Piece<T, V> raw[NV];                  // the row to come
  if (first < last) {
    const int end = rb_end(p, first);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (cl + k * 32 * V < end) ld_piece(src + k * 32 * V, raw[k]);
  }
  for (int i = threadIdx.x; i < p.buckets; i += blockDim.x) s_table[i] = ld_any(p.table, (int64_t)i * p.heads + h, p.table_type) * kUnit;
  if (p.mask_staged) {
    const int64_t at = b * p.mask_b + h * p.mask_h;
    for (int i = threadIdx.x; i < p.mask_staged && block_c0 + i < p.cols; i += blockDim.x) s_mask[i] = ld_any(p.mask, at + block_c0 + i, p.mask_type) * kUnit;
  }
  __syncthreads();
  // the bias: of every distance that the block meets, from its first column and last row on; compact: of every distance up to the last edge
  const int far = p.edges[p.side - 1], ahead = p.both ? far : 0, width = WIDE ? warps * SPAN : SPAN;
  const int from = p.compact ? -far : block_c0 - q_last, values = p.compact ? far + ahead + 1 : min(width, p.cols - block_c0) + block_rows;
  for (int i = threadIdx.x; i < values; i += blockDim.x) {
    const int d = from + i;
    const int r = d < 0 ? -d : (p.both ? d : 0);
    const int k = r >= far ? p.side - 1 : rb_bucket(s_edges, p.side, r);
    s_lut[p.compact ? i : lut_at<V>(i)] = s_table[k + (p.both && d > 0 ? p.side : 0)];
  }
  __syncthreads();
  if (WIDE && p.cluster > 1) rb_cluster_sync();      // the other blocks have started: their shared memory may be written
  const float scale = p.scale * kUnit;
  const float* my_mask = s_mask + (cl - block_c0);
  int turn = 0;
  for (int i = first; i < last; ++i, turn ^= 1, dst += p.cols) {
    const int q = i + p.q_offset, end = rb_end(p, i), end_next = i + 1 < last ? rb_end(p, i + 1) : 0;
    // the lane's columns in the bias table: eight apart, so that the shift within eight is the same for all of them
    const int shift = q_last - q, within = V == 8 ? shift & 7 : 0;
    const float* lut = V == 8 ? s_lut + 9 * ((cl - block_c0) / 8 + (shift >> 3)) : s_lut + (cl - block_c0 + shift);
    src += p.cols;
    // The first NA pieces of the row, in one straight line.  A causal row that ends in its first half leaves the other half out; a branch
    // per piece would cost more than it saves ([1,32,2048,2048] 87 -> 96 us).
    auto row = [&](auto pieces) {
      constexpr int NA = decltype(pieces)::value;
    float f[NA][V], m, tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};      // (four chains)
#pragma unroll
    for (int k = 0; k < NA; ++k) {
      piece_f32(raw[k], f[k]);
      if (cl + k * 32 * V < end_next) ld_piece(src + k * 32 * V, raw[k]);      // (its place is free: the next row's is on its way from here on)
    }
    if (p.compact) {
#pragma unroll
      for (int k = 0; k < NA; ++k) {
        float bias[V];
#pragma unroll
        for (int e = 0; e < V; ++e) bias[e] = s_lut[min(max(cl + k * 32 * V + e - q, -far), ahead) + far];
        fma_all(f[k], scale, bias);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NA; ++k) {
        float bias[V];
#pragma unroll
        for (int e = 0; e < V; ++e) bias[e] = V == 8 ? lut[k * 32 * 9 + lut_at<V>(within + e)] : lut[k * 32 * V + e];
        fma_all(f[k], scale, bias);
      }
    }
    if (p.mask_staged) {
#pragma unroll
      for (int k = 0; k < NA; ++k) {
        // (behind the row's last column: whatever lies there, the columns do not count)
        float mk[V];
        if constexpr (V == 8) {
          *reinterpret_cast<float4*>(mk) = *reinterpret_cast<const float4*>(my_mask + k * 32 * V);
          *reinterpret_cast<float4*>(mk + 4) = *reinterpret_cast<const float4*>(my_mask + k * 32 * V + 4);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) mk[e] = my_mask[k * 32 * V + e];
        }
        add_all(f[k], mk);
      }
    } else if (p.mask != nullptr) {
      const int64_t at = b * p.mask_b + h * p.mask_h + (int64_t)i * p.mask_row + cl;
#pragma unroll
      for (int k = 0; k < NA; ++k) {
        if (cl + k * 32 * V >= end) continue;
        float mk[V];
        if constexpr (V == 8) {
          if (p.mask_vec) {
            ld_any8(p.mask, at + k * 32 * V, p.mask_type, mk);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) mk[e] = ld_any(p.mask, at + k * 32 * V + e, p.mask_type);
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) mk[e] = ld_any(p.mask, at + k * 32 * V + e, p.mask_type);
        }
        mul_one(mk, kUnit);
        add_all(f[k], mk);
      }
    }
    // what lies across the row's end or behind it is decided once for 256 columns (per piece: [4,3,1470,1707] 68 us, so 53)
    constexpr int SUB = 8 / V;
#pragma unroll
    for (int o = 0; o < NA; o += SUB) {
      if (c0 + (o + SUB) * 32 * V > end) {      // (else all of the warp's columns count)
#pragma unroll
        for (int k = o; k < o + SUB; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) f[k][e] = cl + k * 32 * V + e < end ? f[k][e] : -INFINITY;
      }
#pragma unroll
      for (int k = o; k < o + SUB; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) tops[(k * V + e) & 3] = fmaxf(tops[(k * V + e) & 3], f[k][e]);
    }
    m = warp_max(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
    const Exponents ex = exponents(m == -INFINITY ? 0.f : m);      // nothing counts: 2^-inf = 0 everywhere
    float sums[V < 4 ? 4 : V], sum = 0.f;
#pragma unroll
    for (int e = 0; e < (V < 4 ? 4 : V); ++e) sums[e] = 0.f;
#pragma unroll
    for (int k = 0; k < NA; ++k) {
      fma_one(f[k], ex.s, ex.b);
#pragma unroll
      for (int e = 0; e < V; ++e) f[k][e] = exp2_neg(f[k][e]);
      if constexpr (V == 8) {
        add_all(sums, f[k]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) sums[(k * V + e) & 3] += f[k][e];
      }
    }
#pragma unroll
    for (int e = 0; e < (V < 4 ? 4 : V); ++e) sum += sums[e];
    sum = warp_sum(sum);
    float factor;
    if (WIDE) {
      const float2 all = rb_exchange(s_ex, turn, warps, p.cluster, rank, make_float2(m, sum), join_softmax);
      factor = (m == -INFINITY ? 1.f : exp2_neg((m - all.x) * kSteps)) / all.y;
      if (all.y == 0.f) factor = 0.f;
    } else {
      factor = sum == 0.f ? 0.f : __fdividef(1.f, sum);        // a row that nothing is visible to: zeros
    }
#pragma unroll
    for (int o = 0; o < NA; o += SUB) {
#pragma unroll
      for (int k = o; k < o + SUB; ++k) mul_one(f[k], factor);
      if (c0 + (o + SUB) * 32 * V > end) {
#pragma unroll
        for (int k = o; k < o + SUB; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) f[k][e] = cl + k * 32 * V + e < end ? f[k][e] : 0.f;      // (zero in a row that became NaN, too)
      }
#pragma unroll
      for (int k = o; k < o + SUB; ++k)
        if (cl + k * 32 * V < p.cols) st_piece(dst + k * 32 * V, f[k]);
    }
#pragma unroll
    for (int k = NA; k < NV; ++k) {      // columns behind the row's end
      const int c = cl + k * 32 * V;
      if (c < end_next) ld_piece(src + k * 32 * V, raw[k]);
      if (c < p.cols) {
        float zero[V];
#pragma unroll
        for (int e = 0; e < V; ++e) zero[e] = 0.f;
        st_piece(dst + k * 32 * V, zero);
      }
    }
    };
    // (not where warps meet: all of them have to be on the same line)
    if (!WIDE && SPAN >= 512 && end <= SPAN / 2) row(std::integral_constant<int, SPAN >= 512 ? NV / 2 : NV>());
    else row(std::integral_constant<int, NV>());
  }
}

// Backward's rows to come.  Short ones wait in registers; from 32 elements per lane on they would take a quarter of all registers, so they
// travel into shared memory (cp.async), where every lane reads only what it copied itself, and more warps fit on an SM ([1,32,2048,2048]
// 162 -> 135 us, causal 120 -> 103).  Not fp32, whose octets are two copies that share their sectors (1000 columns 117 -> 206 us), and not
// rows that several warps share, whose registers are few enough.
template <typename T, int V, int NV, bool WIDE>
struct RbRow {
  static constexpr bool STAGED = V == 8 && NV >= 4 && sizeof(T) == 2 && !WIDE;
  static constexpr int BYTES = STAGED ? 2 * NV * 512 : 0;               // of a warp, both operands
  Piece<T, V> reg[STAGED ? 1 : 2 * NV];
  uint32_t at;
  __device__ __forceinline__ explicit RbRow(uint32_t warp_base) : at(warp_base + (threadIdx.x & 31) * 16) {}
  // slot: 2 k for the probabilities, 2 k + 1 for their gradient, of piece k
  __device__ __forceinline__ void fetch(int slot, const T* from) {
    if constexpr (STAGED) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + (uint32_t)(slot * 512)), "l"(from) : "memory");
    } else {
      ld_piece(from, reg[slot]);
    }
  }
  __device__ __forceinline__ void wait() {
    if constexpr (STAGED) asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __device__ __forceinline__ void get(int slot, float (&f)[V]) const {
    if constexpr (STAGED) {
      Octet<T> o;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(o.v[0].x), "=r"(o.v[0].y), "=r"(o.v[0].z), "=r"(o.v[0].w) : "r"(at + (uint32_t)(slot * 512)) : "memory");
      octet_to_f32(o, f);
    } else {
      piece_f32(reg[slot], f);
    }
  }
};
// floats of shared memory per warp: the row to come, and after the last row the diagonals' sums in its place; sums that left the warp's columns
__host__ __device__ constexpr int rb_warp_floats(int span, int rows, int staged_bytes) {
  return ((staged_bytes / 4 > span ? staged_bytes / 4 : span) + rows + 3) / 4 * 4;
}

// the distances of bucket k: from .. to
__device__ __forceinline__ void rb_range(const RbParams& p, const int* edges, int k, int& from, int& to) {
  if (p.both && k >= p.side) {
    k -= p.side;
    from = max(1, edges[k]);
    to = k + 1 < p.side ? edges[k + 1] - 1 : 0x7ffffff0;
  } else {
    to = k == 0 && !p.both ? 0x7ffffff0 : -edges[k];
    from = k + 1 < p.side ? 1 - edges[k + 1] : -0x7ffffff0;
  }
}

// blocks per SM that the registers of a narrow kernel are cut for
__host__ __device__ constexpr int rb_bwd_blocks(int bytes, int v, int nv) { return v * nv < 32 ? 4 : bytes == 4 || v == 1 ? 3 : v == 8 && nv == 4 ? 5 : 4; }
template <typename T, int V, int NV, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 32 * kRbMaxWarps : 32 * kRbBwdWarps, WIDE ? 1 : rb_bwd_blocks(sizeof(T), V, NV))
relbias_bwd_kernel(const __grid_constant__ RbParams p) {
  extern __shared__ __align__(16) float s_diag_all[];
  __shared__ int s_edges[kRbMaxSide];
  __shared__ RbExchange<double> s_ex;
  constexpr int SPAN = 32 * V * NV;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rank = WIDE ? (int)(blockIdx.x % (unsigned)p.cluster) : 0;
  for (int i = threadIdx.x; i < p.side; i += blockDim.x) s_edges[i] = p.edges[i];
  __syncthreads();
  pdl_wait();
  if (WIDE && p.cluster > 1) rb_cluster_sync();      // the other blocks have started: their shared memory may be written
  // a unit: `rows_per` consecutive rows of one map, for a warp or for the warps that share a row
  const int64_t unit = WIDE ? blockIdx.x / (unsigned)p.cluster : (int64_t)blockIdx.x * kRbBwdWarps + warp;
  if (!WIDE && unit >= p.units) return;
  const int bh = (int)(unit / p.chunks), chunk = p.chunks - 1 - (int)(unit - (int64_t)bh * p.chunks);      // (causal: long rows first)
  const int first = chunk * p.rows_per, last = min(first + p.rows_per, p.n) - 1;
  typedef RbRow<T, V, NV, WIDE> Row;
  float* s_diag = s_diag_all + warp * rb_warp_floats(SPAN, p.rows_per, Row::BYTES);
  float* s_flush = s_diag + (Row::STAGED ? max(SPAN, Row::BYTES / 4) : SPAN);
  const int c0 = WIDE ? (rank * warps + warp) * SPAN : 0;
  const int64_t map = (int64_t)bh * p.n;
  const int cl = c0 + lane * V;
  const T *a = reinterpret_cast<const T*>(p.x) + (map + first) * p.cols + cl, *g = reinterpret_cast<const T*>(p.grad) + (map + first) * p.cols + cl;
  T* dst = reinterpret_cast<T*>(p.out) + (map + first) * p.cols + cl;
  Row next((uint32_t)__cvta_generic_to_shared(s_diag));
  {
    const int end = rb_end(p, first);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (cl + k * 32 * V < end) { next.fetch(2 * k, a + k * 32 * V); next.fetch(2 * k + 1, g + k * 32 * V); }
  }
  float acc[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[k][e] = 0.f;
  int turn = 0;
  for (int i = first; i <= last; ++i, turn ^= 1, dst += p.cols) {
    const int end = rb_end(p, i);
    const int end_next = i < last ? rb_end(p, i + 1) : 0;
    next.wait();
    a += p.cols;
    g += p.cols;
    // 256 columns at a time (SUB pieces, KO times): what lies before a row's end, across it or behind it is decided once for them
    constexpr int SUB = 8 / V, KO = NV / SUB;
    float dots[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) dots[e] = 0.f;
#pragma unroll
    for (int o = 0; o < KO; ++o) {
      const int cb = c0 + o * 256;
      if (cb >= end) continue;           // (the whole warp, as below)
      float fa[SUB][V], fg[SUB][V];
#pragma unroll
      for (int j = 0; j < SUB; ++j) {
        next.get(2 * (o * SUB + j), fa[j]);
        next.get(2 * (o * SUB + j) + 1, fg[j]);
        mul_all(fa[j], fg[j]);
      }
      if (cb + 256 > end) {
#pragma unroll
        for (int j = 0; j < SUB; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) fa[j][e] = cl + (o * SUB + j) * 32 * V + e < end ? fa[j][e] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < SUB; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) dots[j * V + e] += fa[j][e];
    }
#pragma unroll
    for (int o = 4; o > 1; o >>= 1)
#pragma unroll
      for (int e = 0; e < o; ++e) dots[e] += dots[e + o];
    float dot;
    if constexpr (WIDE) {                // (few rows: what a row's sum is off by averages out in no bucket)
      dot = (float)rb_exchange(s_ex, turn, warps, p.cluster, rank, warp_sum((double)dots[0] + (double)dots[1]), [](double u, double v) { return u + v; });
    } else {
      dot = warp_sum(dots[0] + dots[1]);
    }
    // the gradient, and the diagonals' running sums: one column to the right, this row's share added
    float left = 0.f;                    // lane 0: what leaves the piece of columns before
#pragma unroll
    for (int o = 0; o < KO; ++o) {
      const int cb = c0 + o * 256;
      float ds[SUB][V], fg[SUB][V];
      auto to_come = [&]() {               // (the places are free: the next row's are on their way)
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
          const int k = o * SUB + j;
          if (cl + k * 32 * V < end_next) { next.fetch(2 * k, a + k * 32 * V); next.fetch(2 * k + 1, g + k * 32 * V); }
        }
      };
      auto store = [&]() {
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
          const int k = o * SUB + j;
#pragma unroll
          for (int e = 0; e < V; ++e) fg[j][e] = ds[j][e];
          mul_one(fg[j], p.scale);
          if (cl + k * 32 * V < p.cols) st_piece(dst + k * 32 * V, fg[j]);
        }
      };
      if (cb >= end) {
#pragma unroll
        for (int j = 0; j < SUB; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) ds[j][e] = 0.f;
        to_come();
        store();
        // columns that no row so far has seen: no sums either.  (Rows that lie behind the last column all end with it: their sums move on.)
        if (p.causal && end < p.cols) { left = 0.f; continue; }
      } else {
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
          next.get(2 * (o * SUB + j), ds[j]);
          next.get(2 * (o * SUB + j) + 1, fg[j]);
        }
        to_come();
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
          if constexpr (sizeof(T) == 2) {      // a g is exact: one rounding
            mul_all(fg[j], ds[j]);
            fma_all(ds[j], -dot, fg[j]);
          } else {
            add_one(fg[j], -dot);
            mul_all(ds[j], fg[j]);
          }
        }
        if (cb + 256 > end) {
#pragma unroll
          for (int j = 0; j < SUB; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) ds[j][e] = cl + (o * SUB + j) * 32 * V + e < end ? ds[j][e] : 0.f;
        }
        store();
      }
#pragma unroll
      for (int j = 0; j < SUB; ++j) {
        const int k = o * SUB + j;
        const float moved = __shfl_sync(0xffffffffu, acc[k][V - 1], (lane + 31) & 31);
        const float carry = lane == 0 ? left : moved;
        left = moved;
#pragma unroll
        for (int e = V - 1; e > 0; --e) acc[k][e] = acc[k][e - 1] + ds[j][e];
        acc[k][0] = carry + ds[j][0];
      }
    }
    if (lane == 0 && i > first) s_flush[last - i] = left;
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) s_diag[k * 32 * V + lane * V + e] = acc[k][e];
  __syncwarp();
  // the sum of the diagonal at distance dmin + x: s_diag[x], behind the warp's columns s_flush[x - SPAN]
  auto diagonal = [&](int x) { return x < SPAN ? s_diag[x] : s_flush[x - SPAN]; };
  // .. of every step-th distance from..to: long ranges nearly cancel, in 64 bits where nothing averages out (few rows)
  typedef typename std::conditional<WIDE, double, float>::type Sum;
  auto every = [&](int from, int to, int step) {
    Sum sum = 0;
    for (int x = from; x <= to; x += 4 * step) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = x + j * step <= to ? diagonal(x + j * step) : 0.f;
      sum += ((Sum)v[0] + (Sum)v[1]) + ((Sum)v[2] + (Sum)v[3]);
    }
    return sum;
  };
  const int dmin = c0 - last - p.q_offset, dmax = dmin + SPAN - 1 + (last - first);
  double* part = p.part + ((WIDE ? unit * p.cluster * warps + rank * warps + warp : unit)) * p.buckets;
  // short ranges by a lane each, long ones by the warp
  for (int k0 = 0; k0 < p.buckets; k0 += 32) {
    const int k = k0 + lane;
    int from = 1, to = 0;
    if (k < p.buckets) rb_range(p, s_edges, k, from, to);
    from = max(from, dmin); to = min(to, dmax);
    const bool wide_range = to - from >= 48;
    Sum sum = wide_range ? (Sum)0 : every(from - dmin, to - dmin, 1);
    for (unsigned left = __ballot_sync(0xffffffffu, wide_range); left != 0u; left &= left - 1u) {
      const int l = __ffs(left) - 1, lo = __shfl_sync(0xffffffffu, from, l), hi = __shfl_sync(0xffffffffu, to, l);
      const Sum v = warp_sum(every(lo + lane - dmin, hi - dmin, 32));
      if (lane == l) sum = v;
    }
    if (k < p.buckets) part[k] = sum;
  }
}

// table[k, head]: the units' sums of a head, 32 buckets per block
__global__ void __launch_bounds__(1024)
relbias_table_kernel(const double* __restrict__ part, int batch, int heads, int per_map, int buckets, float* __restrict__ table) {
  __shared__ double s_sum[32][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = (int)blockIdx.x, k = (int)blockIdx.y * 32 + lane;
  double sum = 0.0;
  const uint32_t units = (uint32_t)batch * (uint32_t)per_map;
  if (k < buckets) {
#pragma unroll 4
    for (uint32_t u = warp; u < units; u += 32) {
      const uint32_t b = u / (uint32_t)per_map;
      sum += part[((int64_t)(b * heads + h) * per_map + (u - b * per_map)) * buckets + k];
    }
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

// How a map is cut: V adjacent elements per access, accesses per lane, warps (and blocks of a cluster) of a row.  A warp whose lanes have
// more elements spends less on what every row costs (reductions, addresses) and has fewer companions to wait for; what limits it is
// registers: 64 elements of 16-bit octets, 32 of the rest.
struct RbPlan { int v, nv, warps, cluster; bool wide; };
static RbPlan rb_plan(const hyc_relative_bias* a, bool backward) {
  RbPlan r;
  const size_t e = (size_t)elem_bytes(a->type);
  auto fits = [&](int v) {
    const size_t bytes = v == 8 ? 16 : v * e;      // (a piece of 8 fp32 values is two accesses)
    return a->cols % v == 0 && aligned(a->x, bytes) && aligned(a->out, bytes) && (!backward || aligned(a->grad, bytes));
  };
  r.v = fits(8) ? 8 : fits(2) ? 2 : 1;
  const int64_t cols = a->cols, rows = a->batch * a->heads * a->n;
  r.cluster = 1;
  r.warps = backward ? kRbBwdWarps : kRbNarrowWarps;
  // few rows: several warps each, for what a row takes
  const bool few = cols > 512 && rows < (int64_t)num_sms() * 8;
  int span = 256;
  while (span < cols && span < (e == 2 && r.v == 8 ? 2048 : 1024)) span *= 2;
  r.wide = few || cols > span;
  if (r.wide) {
    span = few && cols <= 256 * kRbMaxWarps ? 256 : 1024;
    while (cols > (int64_t)r.cluster * kRbMaxWarps * span) r.cluster *= 2;
    r.warps = (int)((cols + (int64_t)r.cluster * span - 1) / ((int64_t)r.cluster * span));
  }
  r.nv = span / (32 * r.v);
  return r;
}
// Rows of a unit (narrow: a warp, wide: the warps that share a row): what a unit takes to start and end, in rows, against units that do not
// fill the last wave.  warps: units of a block of forward; slots: blocks (backward: units) that are resident at once; causal rows are unlike,
// long ones come first, so the waves overlap.
static int rb_rows_per(int64_t maps, int n, int warps, int64_t slots, float fixed, bool causal) {
  int best = 1;
  float best_cost = 1e30f;
  for (int per = 1; per <= 32; ++per) {
    const int64_t units = maps * ((n + per * warps - 1) / (per * warps));
    const float waves = (float)units / (float)slots, whole = (float)((units + slots - 1) / slots);
    const float cost = (causal && waves > 1.f ? waves + 0.5f : whole) * ((float)per + fixed);
    if (cost < best_cost * 0.999f) { best_cost = cost; best = per; }
  }
  return best < n ? best : n;
}

static void rb_fill(RbParams& p, const hyc_relative_bias* a, const RbPlan& r) {
  p.x = a->x; p.grad = a->grad; p.table = a->table; p.mask = a->mask; p.out = a->out; p.part = nullptr;
  p.mask_b = a->mask_b; p.mask_h = a->mask_h; p.mask_row = a->mask_row;
  p.heads = a->heads; p.n = (int)a->n; p.cols = (int)a->cols; p.q_offset = (int)a->q_offset;
  p.cluster = r.cluster;
  p.table_type = a->table_type; p.mask_type = a->mask_type;
  p.mask_vec = a->mask != nullptr && aligned(a->mask, 16) && ((a->mask_b | a->mask_h | a->mask_row) & 7) == 0;
  p.side = a->side; p.both = a->both != 0; p.causal = a->causal != 0; p.buckets = a->both ? 2 * a->side : a->side;
  p.scale = a->scale;
  p.mask_staged = 0;
  p.compact = 0;
  for (int i = 0; i < a->side; ++i) p.edges[i] = a->host_edges[i];
}

// the most dynamic shared memory of any plan: forward a mask and the bias of 16384 columns, backward the diagonals of 16 warps
constexpr int kRbSmemFwd = (16384 + (16384 + 32 * kRbNarrowWarps) * 9 / 8 + 2) * 4, kRbSmemBwd = kRbMaxWarps * (1024 + 32) * 4;
template <auto KERN>
static int rb_launch(const RbPlan& r, int64_t blocks, size_t smem, const RbParams& p, cudaStream_t st) {
  if (blocks > 0x7fffffffll) return HYC_ERR_SHAPE;
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
  if (cudaLaunchKernelEx(&cfg, KERN, p) != cudaSuccess) {
    hyc_set_last_cuda_error((int)cudaGetLastError());
    return HYC_ERR_LAUNCH;
  }
  return HYC_OK;
}

// f(element, V, NV, WIDE) for the plan's kernel: narrow spans of 256 to 1024 columns, 2048 of 16-bit octets; wide ones of 256 and 1024
template <typename F>
static int rb_by_plan(int type, const RbPlan& r, F&& f) {
  auto by_shape = [&](auto elem) -> int {
    auto span = [&](auto v) -> int {
      constexpr int V = decltype(v)::value;
      auto of = [&](auto nv) -> int {
        if constexpr (decltype(nv)::value * V == 16) return f(elem, v, nv, std::false_type());
        else if constexpr (decltype(nv)::value * V == 64) return f(elem, v, nv, std::false_type());
        else return r.wide ? f(elem, v, nv, std::true_type()) : f(elem, v, nv, std::false_type());
      };
      if (r.nv == 8 / V) return of(std::integral_constant<int, 8 / V>());
      if (r.nv == 16 / V) return of(std::integral_constant<int, 16 / V>());
      if constexpr (V == 8 && sizeof(elem) == 2)
        if (r.nv == 64 / V) return of(std::integral_constant<int, 64 / V>());
      return of(std::integral_constant<int, 32 / V>());
    };
    if (r.v == 8) return span(std::integral_constant<int, 8>());
    if (r.v == 2) return span(std::integral_constant<int, 2>());
    return span(std::integral_constant<int, 1>());
  };
  if (type == HYC_F32) return by_shape(float());
  if (type == HYC_F16) return by_shape(__half());
  return by_shape(__nv_bfloat16());
}

// backward: rows of a unit and the warps' sums that the workspace holds (the same for a query and for a launch: nothing here asks the runtime)
struct RbUnits { int rows_per, chunks; int64_t units, sums; };
static RbUnits rb_units(const hyc_relative_bias* a, const RbPlan& r) {
  RbUnits u;
  const int64_t warps = r.wide ? 16 : kRbBwdWarps * rb_bwd_blocks(elem_bytes(a->type), r.v, r.nv);      // resident per SM
  const int64_t slots = (int64_t)num_sms() * warps / (r.wide ? r.warps * r.cluster : 1);
  u.rows_per = rb_rows_per(a->batch * a->heads, (int)a->n, 1, slots < 1 ? 1 : slots, 6.f, a->causal != 0);
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
  const int width = 32 * r.v * r.nv * (r.wide ? r.warps : 1);      // columns of a block
  const int far = p.edges[p.side - 1], distances = far + (p.both ? far : 0) + 1;
  const bool one_mask = a->mask != nullptr && a->mask_row == 0;
  return rb_by_plan(a->type, r, [&](auto elem, auto v, auto nv, auto wide) -> int {
    constexpr auto kern = relbias_fwd_kernel<decltype(elem), decltype(v)::value, decltype(nv)::value, decltype(wide)::value>;
    auto bytes = [&](int mask, int values) { return (size_t)(mask + values * 9 / 8 + 2) * sizeof(float); };
    const int block_warps = r.wide ? 1 : kRbNarrowWarps;      // warps with rows of their own
    const size_t most = bytes(one_mask ? width : 0, width + 32 * block_warps);
    const int rs = more_shared_memory<kern>(kRbSmemFwd);      // (before the question: the answer counts on it)
    if (rs != HYC_OK) return rs;
    const int64_t slots = (int64_t)num_sms() * resident_blocks(kern, 32 * r.warps, most, 1) / r.cluster;
    p.rows_per = rb_rows_per(a->batch * a->heads, (int)a->n, block_warps, slots < 1 ? 1 : slots, 3.f, a->causal != 0);
    const int rows = p.rows_per * block_warps;      // of a block
    p.chunks = (int)((a->n + rows - 1) / rows);
    // few rows: neither a vector of the bias per column nor a copy of the mask is read often enough to be worth making
    const bool few = rows < 4 || a->n < 4;
    p.compact = few && distances < width;
    p.mask_staged = one_mask && !few ? width : 0;
    const size_t smem = bytes(p.mask_staged, p.compact ? distances : width + rows);
    return rb_launch<kern>(r, a->batch * a->heads * p.chunks * r.cluster, smem, p, (cudaStream_t)stream);
  });
}

extern "C" HYC_API size_t hyc_softmax_relative_bias_workspace_bytes(const hyc_relative_bias* a) {
  if (rb_check(a, true) != HYC_OK || a->batch * a->n == 0) return 0;
  return (size_t)rb_units(a, rb_plan(a, true)).sums * (size_t)(a->both ? 2 * a->side : a->side) * sizeof(double);
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
    if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < (size_t)u.sums * (size_t)buckets * sizeof(double)) return HYC_ERR_WORKSPACE;
    RbParams p;
    rb_fill(p, a, r);
    p.part = (double*)workspace;
    p.rows_per = u.rows_per; p.chunks = u.chunks; p.units = u.units;
    const int64_t blocks = r.wide ? u.units * r.cluster : (u.units + kRbBwdWarps - 1) / kRbBwdWarps;
    const int rl = rb_by_plan(a->type, r, [&](auto elem, auto v, auto nv, auto wide) -> int {
      constexpr auto kern = relbias_bwd_kernel<decltype(elem), decltype(v)::value, decltype(nv)::value, decltype(wide)::value>;
      constexpr int V = decltype(v)::value, NV = decltype(nv)::value;
      const size_t smem = (size_t)r.warps * (size_t)rb_warp_floats(32 * V * NV, u.rows_per, RbRow<decltype(elem), V, NV, decltype(wide)::value>::BYTES) * sizeof(float);
      const int rs = more_shared_memory<kern>(kRbSmemBwd);
      return rs != HYC_OK ? rs : rb_launch<kern>(r, blocks, smem, p, (cudaStream_t)stream);
    });
    if (rl != HYC_OK) return rl;
  }
  const int per_map = u.chunks * (r.wide ? r.warps * r.cluster : 1);
  launch_pdl(relbias_table_kernel, dim3((unsigned)a->heads, (unsigned)((buckets + 31) / 32)), dim3(1024), 0, (cudaStream_t)stream, (const double*)workspace,
             u.units > 0 ? (int)a->batch : 0, a->heads, per_map, buckets, dtable);
  HYC_CHECK_LAUNCH();
  return HYC_OK;
}
