// RMS norms of the query and key heads with the rotary embedding in the same pass, and their backward pass.
//
//   r = 1 / sqrt(mean(x^2) + eps) over the d channels of one head,   n = x r w
//   y[j]     = n[j] c - n[j + h] s,   y[j + h] = n[j + h] c + n[j] s      j < h = rot / 2;   y[j] = n[j] from rot on
// with c, s = cos[p, j], sin[p, j] at the token's position p.  Backward, g = dy turned back by the same angle:
//   dw = sum g x r,   dx = r (g w - x r mean(g w x r))
// The row sums r needs are taken again from x, which backward reads anyway: nothing is kept between the passes but q and k.
// Everything is fp32 between the loads and the one rounding at the store.
//
// Bound by memory: x is read and y written once (backward: x, dy, dx).  A head belongs to G = 2 .. 32 adjacent lanes, each
// with the channels [4 i, 4 i + 4) and their partners h further (behind rot: 8 channels in a row), so that the pairs of the
// rotation meet in one lane and a mean is log2 G shuffles; the arithmetic is on pairs of fp32 values, two per instruction.  A warp keeps to one of the two
// tensors, so that the norm's weight, and in backward its gradient, stay in registers; the angles are loaded once per token
// and used for the heads that the warp takes of it.  Backward's gradients of the weights: per lane over all its heads, then
// per block in a fixed order, then one small launch over the blocks: the same bits on every run.
#include "elem.cuh"
#include <type_traits>

namespace hyc {

constexpr int kQkThreads = 256, kQkWarps = kQkThreads / 32;
constexpr int kQkBwdBlocks = 3;      // blocks per SM that backward's registers are cut for and its workspace counts on

// one instruction, two units in the last place (the root and the quotient, each rounded, take two dozen per head)
__device__ __forceinline__ float qk_rsqrt(float v) {
  float r;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

struct QkTensor {
  const void *x, *dy, *w;
  void* out;                       // contiguous [tokens, heads, d]
  int64_t xb, xm, xh, gb, gm, gh;  // strides of x and dy: batch, token, head
  int heads;
  int splits, per_split;           // a token's head groups as `splits` items of `per_split` groups
  int blocks;                      // blocks that work on this tensor
};
struct QkParams {
  QkTensor t[2];
  const void *cos_t, *sin_t, *pos;
  int64_t ld_cos, ld_sin, pb, pm;  // strides of the positions: batch, token
  int pos64, table_type, w_type, table_rows;
  int tokens, seq, d, half;
  float eps;
  float* part;                     // backward: [blocks][d] sums of the weights' gradients, q's blocks first; or null
};

// The lane's channels of a head: NQ pairs of quads, from o1 and from o2 on.  FULL: the head's size is a power of two and all of it is
// turned, so that every lane has channels, all of one kind, and partners at a distance known when this is compiled.
template <int NQ, int G, bool FULL> struct QkLane {
  int first[NQ], second[NQ];
  bool is_live[NQ], is_turned[NQ];
  __device__ __forceinline__ QkLane(int li, int d, int half) {
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const int at = li + j * G, i = at - half / 4;
      is_live[j] = at < d / 8;
      is_turned[j] = at < half / 4;
      first[j] = is_turned[j] ? 4 * at : 2 * half + 8 * i;
      second[j] = is_turned[j] ? 4 * at + half : 2 * half + 8 * i + 4;
      if (!is_live[j]) { first[j] = 0; second[j] = 0; }
    }
  }
  __device__ __forceinline__ bool live(int j) const { return FULL || is_live[j]; }
  __device__ __forceinline__ bool turned(int j) const { return FULL || is_turned[j]; }
  __device__ __forceinline__ int o1(int j) const { return first[j]; }
  __device__ __forceinline__ int o2(int j) const { return FULL ? first[j] + 4 * G * NQ : second[j]; }
};

// cos, sin and -sin of a token at the lane's channels; a position outside of the tables gives NaN, and reads nothing
template <int NQ> struct QkAngles { f32x2 c[NQ][2], s[NQ][2], ns[NQ][2]; };
template <int NQ, typename L>
__device__ __forceinline__ void qk_angles(const QkParams& p, int b, int m, const L& l, QkAngles<NQ>& a) {
  int64_t at = m;
  if (p.pos != nullptr) {
    const int64_t i = b * p.pb + m * p.pm;
    at = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[i] : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[i];
  }
  const bool known = at >= 0 && at < p.table_rows;
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    a.c[j][0] = a.c[j][1] = both(1.f);
    a.s[j][0] = a.s[j][1] = both(0.f);
    if (l.turned(j)) {
      if (known) {
        ld_any4(p.cos_t, at * p.ld_cos + l.o1(j), p.table_type, a.c[j]);
        ld_any4(p.sin_t, at * p.ld_sin + l.o1(j), p.table_type, a.s[j]);
      } else {
        a.c[j][0] = a.c[j][1] = a.s[j][0] = a.s[j][1] = both(__int_as_float(0x7fc00000));
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) a.ns[j][e] = a.s[j][e] ^ 0x8000000080000000ull;
  }
}

template <int G>
__device__ __forceinline__ float qk_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float qk_total(f32x2 v) {
  const float2 t = unpair(v);
  return t.x + t.y;
}
// where a warp's items lie
struct QkItem { uint32_t token; int first, b, m; };
__device__ __forceinline__ QkItem qk_item(const QkParams& p, const QkTensor& t, uint32_t item) {
  QkItem i;
  i.token = item / (uint32_t)t.splits;
  i.first = (int)(item - i.token * (uint32_t)t.splits) * t.per_split;
  i.b = (int)(i.token / (uint32_t)p.seq);
  i.m = (int)(i.token - (uint32_t)i.b * (uint32_t)p.seq);
  return i;
}

// UNROLL head groups are on their way at any time
template <typename T, int G, int NQ, bool FULL, int UNROLL>
__global__ void __launch_bounds__(kQkThreads)
qk_norm_fwd_kernel(const __grid_constant__ QkParams p) {
  pdl_wait();
  constexpr int PER = 32 / G;      // heads of a warp at a time
  const bool second = (int)blockIdx.x >= p.t[0].blocks;
  const QkTensor& t = p.t[second ? 1 : 0];
  const int block = (int)blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & 31, sub = lane / G;
  const QkLane<NQ, G, FULL> l(lane % G, p.d, p.half);
  f32x2 w1[NQ][2], w2[NQ][2];
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    ld_any4(t.w, l.o1(j), p.w_type, w1[j]);
    ld_any4(t.w, l.o2(j), p.w_type, w2[j]);
  }
  const float inv_d = 1.f / (float)p.d;
  const uint32_t items = (uint32_t)p.tokens * (uint32_t)t.splits;
  for (uint32_t item = (uint32_t)block * kQkWarps + (threadIdx.x >> 5); item < items; item += (uint32_t)t.blocks * kQkWarps) {
    const QkItem it = qk_item(p, t, item);
    const T* xt = reinterpret_cast<const T*>(t.x) + it.b * t.xb + it.m * t.xm;
    T* ot = reinterpret_cast<T*>(t.out) + (int64_t)it.token * t.heads * p.d;
    QkAngles<NQ> a;
    qk_angles<NQ>(p, it.b, it.m, l, a);
    const int head0 = it.first * PER + sub;
    int left = min((it.first + t.per_split) * PER, t.heads) - head0;      // heads of this lane's kind: left > u PER
    const T* src = xt + head0 * t.xh;
    T* dst = ot + head0 * p.d;
    const int64_t step = PER * t.xh;
    const int out_step = PER * p.d;
    Quad<T> x1[UNROLL][NQ], x2[UNROLL][NQ];
    auto fetch = [&](int u, bool there) {
#pragma unroll
      for (int j = 0; j < NQ; ++j)
        if (l.live(j) && there) {
          x1[u][j] = ld_quad(src + l.o1(j));
          x2[u][j] = ld_quad(src + l.o2(j));
        }
      src += step;
    };
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) fetch(u, left > u * PER);
    for (; left > -sub; left -= UNROLL * PER) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        f32x2 f1[NQ][2], f2[NQ][2], ss = both(0.f);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          quad_to_f32(x1[u][j], f1[j]);
          quad_to_f32(x2[u][j], f2[j]);
          f32x2 s = both(0.f);
#pragma unroll
          for (int e = 0; e < 2; ++e) s = fma2f(f1[j][e], f1[j][e], fma2f(f2[j][e], f2[j][e], s));
          if (l.live(j)) ss = add2f(ss, s);
        }
        fetch(u, left > (UNROLL + u) * PER);      // its place is free: the heads UNROLL groups on
        const float r = qk_rsqrt(fmaf(qk_sum<G>(qk_total(ss)), inv_d, p.eps));
        const f32x2 rr = both(r);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          f32x2 y1[2], y2[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const f32x2 n1 = mul2f(mul2f(f1[j][e], rr), w1[j][e]), n2 = mul2f(mul2f(f2[j][e], rr), w2[j][e]);
            y1[e] = fma2f(n2, a.ns[j][e], mul2f(n1, a.c[j][e]));
            y2[e] = fma2f(n1, a.s[j][e], mul2f(n2, a.c[j][e]));
          }
          if (l.live(j) && left > u * PER) {
            st_quad(dst + l.o1(j), y1);
            st_quad(dst + l.o2(j), y2);
          }
        }
        dst += out_step;
      }
    }
  }
}

template <typename T, int G, int NQ, bool FULL>
__global__ void __launch_bounds__(kQkThreads, NQ == 1 ? kQkBwdBlocks : 1)
qk_norm_bwd_kernel(const __grid_constant__ QkParams p) {
  __shared__ float s_part[kQkWarps][8 * G * NQ];
  pdl_wait();
  constexpr int PER = 32 / G;
  const bool second = (int)blockIdx.x >= p.t[0].blocks;
  const QkTensor& t = p.t[second ? 1 : 0];
  const int block = (int)blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / G;
  const QkLane<NQ, G, FULL> l(lane % G, p.d, p.half);
  f32x2 w1[NQ][2], w2[NQ][2], dw1[NQ][2], dw2[NQ][2];
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    ld_any4(t.w, l.o1(j), p.w_type, w1[j]);
    ld_any4(t.w, l.o2(j), p.w_type, w2[j]);
    dw1[j][0] = dw1[j][1] = dw2[j][0] = dw2[j][1] = both(0.f);
  }
  const float inv_d = 1.f / (float)p.d;
  const uint32_t items = (uint32_t)p.tokens * (uint32_t)t.splits;
  for (uint32_t item = (uint32_t)block * kQkWarps + warp; item < items; item += (uint32_t)t.blocks * kQkWarps) {
    const QkItem it = qk_item(p, t, item);
    const T *xt = reinterpret_cast<const T*>(t.x) + it.b * t.xb + it.m * t.xm, *gt = reinterpret_cast<const T*>(t.dy) + it.b * t.gb + it.m * t.gm;
    T* ot = reinterpret_cast<T*>(t.out) + (int64_t)it.token * t.heads * p.d;
    QkAngles<NQ> a;
    qk_angles<NQ>(p, it.b, it.m, l, a);
    const int head0 = it.first * PER + sub;
    int left = min((it.first + t.per_split) * PER, t.heads) - head0;
    const T *src = xt + head0 * t.xh, *grad = gt + head0 * t.gh;
    T* dst = ot + head0 * p.d;
    const int64_t step = PER * t.xh, grad_step = PER * t.gh;
    const int out_step = PER * p.d;
    Quad<T> x1[NQ], x2[NQ], d1[NQ], d2[NQ];
    auto fetch = [&](bool there) {
#pragma unroll
      for (int j = 0; j < NQ; ++j)
        if (l.live(j) && there) {
          x1[j] = ld_quad(src + l.o1(j)); x2[j] = ld_quad(src + l.o2(j));
          d1[j] = ld_quad(grad + l.o1(j)); d2[j] = ld_quad(grad + l.o2(j));
        }
      src += step;
      grad += grad_step;
    };
    fetch(left > 0);
    for (; left > -sub; left -= PER) {
      const bool ok = left > 0;
      f32x2 f1[NQ][2], f2[NQ][2], g1[NQ][2], g2[NQ][2], ss = both(0.f), sg = both(0.f);
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        quad_to_f32(x1[j], f1[j]); quad_to_f32(x2[j], f2[j]); quad_to_f32(d1[j], g1[j]); quad_to_f32(d2[j], g2[j]);
      }
      fetch(left > PER);      // the next heads while these are computed
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        f32x2 s1 = both(0.f), s2 = both(0.f);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x2 u = fma2f(g2[j][e], a.s[j][e], mul2f(g1[j][e], a.c[j][e])), v = fma2f(g1[j][e], a.ns[j][e], mul2f(g2[j][e], a.c[j][e]));
          s1 = fma2f(f1[j][e], f1[j][e], fma2f(f2[j][e], f2[j][e], s1));
          const f32x2 p1 = mul2f(u, f1[j][e]), p2 = mul2f(v, f2[j][e]);
          s2 = fma2f(p1, w1[j][e], fma2f(p2, w2[j][e], s2));
          g1[j][e] = u; g2[j][e] = v;
        }
        if (l.live(j)) { ss = add2f(ss, s1); sg = add2f(sg, s2); }
      }
      // dx = r g w - x r^2 mean(g w x r)
      const float r = qk_rsqrt(fmaf(qk_sum<G>(qk_total(ss)), inv_d, p.eps));
      const float pull = qk_sum<G>(qk_total(sg)) * (r * inv_d) * (r * -r);
      const f32x2 rr = both(r), pp = both(pull);
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        f32x2 y1[2], y2[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x2 u = mul2f(g1[j][e], rr), v = mul2f(g2[j][e], rr);
          if (ok) { dw1[j][e] = fma2f(u, f1[j][e], dw1[j][e]); dw2[j][e] = fma2f(v, f2[j][e], dw2[j][e]); }
          y1[e] = fma2f(f1[j][e], pp, mul2f(u, w1[j][e]));
          y2[e] = fma2f(f2[j][e], pp, mul2f(v, w2[j][e]));
        }
        if (ok && l.live(j)) {
          st_quad(dst + l.o1(j), y1);
          st_quad(dst + l.o2(j), y2);
        }
      }
      dst += out_step;
    }
  }
  if (p.part == nullptr) return;
#pragma unroll
  for (int j = 0; j < NQ; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int o = G; o < 32; o <<= 1) {
        dw1[j][e] = add2f(dw1[j][e], __shfl_xor_sync(0xffffffffu, (unsigned long long)dw1[j][e], o));
        dw2[j][e] = add2f(dw2[j][e], __shfl_xor_sync(0xffffffffu, (unsigned long long)dw2[j][e], o));
      }
      if (sub == 0 && l.live(j)) {
        const float2 u = unpair(dw1[j][e]), v = unpair(dw2[j][e]);
        s_part[warp][l.o1(j) + 2 * e] = u.x; s_part[warp][l.o1(j) + 2 * e + 1] = u.y;
        s_part[warp][l.o2(j) + 2 * e] = v.x; s_part[warp][l.o2(j) + 2 * e + 1] = v.y;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < p.d; i += kQkThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kQkWarps; ++w) sum += s_part[w][i];
    p.part[(int64_t)blockIdx.x * p.d + i] = sum;
  }
}

// The blocks' sums of one tensor (blockIdx.y) for 32 channels: a warp takes every 32nd block, a thread one channel
__global__ void __launch_bounds__(1024)
qk_norm_weight_kernel(const float* __restrict__ part, int blocks0, int blocks1, int d, int type, void* dw0, void* dw1) {
  __shared__ float s_sum[32][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = (int)blockIdx.x * 32 + lane;
  const int first = blockIdx.y ? blocks0 : 0, blocks = blockIdx.y ? blocks1 : blocks0;
  float sum = 0.f;
  if (i < d)
    for (int b = warp; b < blocks; b += 32) sum += part[(int64_t)(first + b) * d + i];
  s_sum[warp][lane] = sum;
  __syncthreads();
  sum = s_sum[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int at = (int)blockIdx.x * 32 + warp;
  if (lane == 0 && at < d) st_any(blockIdx.y ? dw1 : dw0, at, type, sum);
}

// ---- host side
static int qk_check(const hyc_qk_norm* a, bool backward) {
  if (a == nullptr) return HYC_ERR_NULL;
  if (!elem_type_ok(a->type) || !elem_type_ok(a->w_type) || !elem_type_ok(a->table_type)) return HYC_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->seq < 0 || a->heads[0] < 1 || a->heads[1] < 1 || a->head_dim < 16 || a->head_dim > 512 || (a->head_dim & 15) != 0 ||
      a->rotary_dim < 16 || a->rotary_dim > a->head_dim || (a->rotary_dim & 15) != 0 || a->table_rows < 0)
    return HYC_ERR_SHAPE;
  // (tokens and heads of a token are counted in 32 bits, offsets in 64)
  if (a->heads[0] > 65536 || a->heads[1] > 65536 || a->batch > 0x7fffffffll || a->seq > 0x7fffffffll || a->batch * a->seq > 0x7fffffffll)
    return HYC_ERR_SHAPE;
  if (a->batch * a->seq == 0) return HYC_OK;
  const int e = 16 / elem_bytes(a->type), et = 16 / elem_bytes(a->table_type);
  if (a->cos_t == nullptr || a->sin_t == nullptr) return HYC_ERR_NULL;
  if (a->ld_cos < a->rotary_dim / 2 || a->ld_sin < a->rotary_dim / 2) return HYC_ERR_SHAPE;
  if (a->position_ids == nullptr && a->table_rows < a->seq) return HYC_ERR_SHAPE;
  if (a->ld_cos % et != 0 || a->ld_sin % et != 0 || !aligned(a->cos_t, 16) || !aligned(a->sin_t, 16)) return HYC_ERR_ALIGN;
  for (int i = 0; i < 2; ++i) {
    if (a->x[i] == nullptr || a->weight[i] == nullptr || a->out[i] == nullptr || (backward && a->dy[i] == nullptr)) return HYC_ERR_NULL;
    if (!aligned(a->x[i], 16) || !aligned(a->weight[i], 16) || !aligned(a->out[i], 16)) return HYC_ERR_ALIGN;
    for (int j = 0; j < 3; ++j) {
      if (a->x_stride[i][j] % e != 0) return HYC_ERR_ALIGN;
      if (backward && a->dy_stride[i][j] % e != 0) return HYC_ERR_ALIGN;
    }
    if (backward && !aligned(a->dy[i], 16)) return HYC_ERR_ALIGN;
  }
  return HYC_OK;
}

// lanes of a head: one per eight channels, a power of two; 32 of them with twice as many above 256 channels
static int qk_group(int d) {
  int g = 2;
  while (g < d / 8 && g < 32) g <<= 1;
  return g;
}

// Blocks for the two tensors in proportion to their heads, at most one resident wave and no more than there is work for; a token's head
// groups are dealt to several warps where that evens out what the warps have to do.
static void qk_plan(QkParams& p, int wave) {
  const int per = 32 / qk_group(p.d), heads = p.t[0].heads + p.t[1].heads;
  for (int i = 0; i < 2; ++i) {
    QkTensor& t = p.t[i];
    const int groups = (t.heads + per - 1) / per;
    int blocks = (int)((int64_t)wave * t.heads / heads);
    if (blocks < 1) blocks = 1;
    // a warp's share is a whole number of items: small ones fill the last round, each costs about two groups more (division, angles)
    const int64_t warps = (int64_t)blocks * kQkWarps;
    int64_t best = 0;
    for (int per_split = 1; per_split <= groups; ++per_split) {
      const int splits = (groups + per_split - 1) / per_split;
      const int64_t cost = ((int64_t)p.tokens * splits + warps - 1) / warps * (per_split + 2);
      if (best == 0 || cost <= best) { best = cost; t.per_split = per_split; t.splits = splits; }
    }
    const int64_t need = ((int64_t)p.tokens * t.splits + kQkWarps - 1) / kQkWarps;
    t.blocks = (int)(need < blocks ? need : blocks);
  }
}

static void qk_fill(QkParams& p, const hyc_qk_norm* a) {
  for (int i = 0; i < 2; ++i) {
    QkTensor& t = p.t[i];
    t.x = a->x[i]; t.dy = a->dy[i]; t.w = a->weight[i]; t.out = a->out[i]; t.heads = a->heads[i];
    t.xb = a->x_stride[i][0]; t.xm = a->x_stride[i][1]; t.xh = a->x_stride[i][2];
    t.gb = a->dy_stride[i][0]; t.gm = a->dy_stride[i][1]; t.gh = a->dy_stride[i][2];
  }
  p.cos_t = a->cos_t; p.sin_t = a->sin_t; p.pos = a->position_ids;
  p.ld_cos = a->ld_cos; p.ld_sin = a->ld_sin; p.pb = a->pos_stride[0]; p.pm = a->pos_stride[1];
  p.pos64 = a->pos_is_int64; p.table_type = a->table_type; p.w_type = a->w_type;
  p.table_rows = a->table_rows > 0x7fffffffll ? 0x7fffffff : (int)a->table_rows;
  p.tokens = (int)(a->batch * a->seq); p.seq = (int)a->seq; p.d = a->head_dim; p.half = a->rotary_dim / 2;
  p.eps = a->eps;
  p.part = nullptr;
}

// f(element, lanes of a head, pairs of quads per lane, FULL)
template <typename F>
static int qk_by_type(int type, int d, int rot, F&& f) {
  auto by_group = [&](auto elem) -> int {
    using std::integral_constant;
    auto full = [&](auto group, auto quads) -> int {
      if (rot == d && d == 8 * decltype(group)::value * decltype(quads)::value) return f(elem, group, quads, std::true_type());
      return f(elem, group, quads, std::false_type());
    };
    constexpr integral_constant<int, 1> one{};
    switch (qk_group(d)) {
      case 2: return full(integral_constant<int, 2>(), one);
      case 4: return full(integral_constant<int, 4>(), one);
      case 8: return full(integral_constant<int, 8>(), one);
      case 16: return full(integral_constant<int, 16>(), one);
      default: return d <= 256 ? full(integral_constant<int, 32>(), one) : full(integral_constant<int, 32>(), integral_constant<int, 2>());
    }
  };
  if (type == HYC_F32) return by_group(float());
  if (type == HYC_F16) return by_group(__half());
  return by_group(__nv_bfloat16());
}

}  // namespace hyc

using namespace hyc;

extern "C" HYC_API int hyc_qk_norm_rope_fwd(const hyc_qk_norm* a, void* stream) {
  const int rc = qk_check(a, false);
  if (rc != HYC_OK || a->batch * a->seq == 0) return rc;
  QkParams p;
  qk_fill(p, a);
  return qk_by_type(a->type, p.d, 2 * p.half, [&](auto elem, auto group, auto quads, auto full) -> int {
    auto kern = qk_norm_fwd_kernel<decltype(elem), decltype(group)::value, decltype(quads)::value, decltype(full)::value, 2>;
    qk_plan(p, num_sms() * resident_blocks(kern, kQkThreads, 0, 2));
    launch_pdl(kern, dim3((unsigned)(p.t[0].blocks + p.t[1].blocks)), dim3(kQkThreads), 0, (cudaStream_t)stream, p);
    HYC_CHECK_LAUNCH();
    return HYC_OK;
  });
}

extern "C" HYC_API size_t hyc_qk_norm_rope_workspace_bytes(int head_dim) {
  return head_dim < 16 || head_dim > 512 ? 0 : (size_t)(num_sms() * kQkBwdBlocks + 2) * (size_t)head_dim * sizeof(float);
}

extern "C" HYC_API int hyc_qk_norm_rope_bwd(const hyc_qk_norm* a, void* dweight_q, void* dweight_k, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = qk_check(a, true);
  if (rc != HYC_OK) return rc;
  const bool weights = dweight_q != nullptr;
  if (weights != (dweight_k != nullptr)) return HYC_ERR_NULL;
  if (weights && (workspace == nullptr || workspace_bytes < hyc_qk_norm_rope_workspace_bytes(a->head_dim) || !aligned(workspace, 16)))
    return HYC_ERR_WORKSPACE;
  QkParams p;
  qk_fill(p, a);
  if (p.tokens > 0) {
    p.part = weights ? (float*)workspace : nullptr;
    const int r = qk_by_type(a->type, p.d, 2 * p.half, [&](auto elem, auto group, auto quads, auto full) -> int {
      auto kern = qk_norm_bwd_kernel<decltype(elem), decltype(group)::value, decltype(quads)::value, decltype(full)::value>;
      const int res = resident_blocks(kern, kQkThreads, 0, 1);
      qk_plan(p, num_sms() * (res < kQkBwdBlocks ? res : kQkBwdBlocks));
      launch_pdl(kern, dim3((unsigned)(p.t[0].blocks + p.t[1].blocks)), dim3(kQkThreads), 0, (cudaStream_t)stream, p);
      HYC_CHECK_LAUNCH();
      return HYC_OK;
    });
    if (r != HYC_OK) return r;
  } else {
    p.t[0].blocks = p.t[1].blocks = 0;      // no tokens: the sums are empty
  }
  if (weights) {
    launch_pdl(qk_norm_weight_kernel, dim3((unsigned)((a->head_dim + 31) / 32), 2), dim3(1024), 0, (cudaStream_t)stream, (const float*)workspace,
               p.t[0].blocks, p.t[1].blocks, a->head_dim, a->w_type, dweight_q, dweight_k);
    HYC_CHECK_LAUNCH();
  }
  return HYC_OK;
}
