// RMS norms of the query and key heads with the rotary embedding in the same pass, and their backward pass.
//
//   r = 1 / sqrt(mean(x^2) + eps) over the d channels of one head,   n = x r w
//   y[j]     = n[j] c - n[j + h] s,   y[j + h] = n[j + h] c + n[j] s      j < h = rot / 2;   y[j] = n[j] from rot on
// with c, s = cos[p, j], sin[p, j] at the token's position p.  Backward, g = dy turned back by the same angle:
//   dw = sum g x r,   dx = r (g w - x r mean(g w x r))
// The row sums r needs are taken again from x, which backward reads anyway: nothing is kept between the passes but q and k.
// Everything is fp32 between the loads and the one rounding at the store.
//
// Bound by memory: x is read and y written once (backward: x, dy, dx).  A head belongs to G = 1 .. 32 adjacent lanes, each with E channels
// from 16 bytes on (E = 8; fp32: 4) and their partners h further (behind rot: 2 E channels in a row), so that the pairs of the rotation meet in
// one lane and a mean is log2 G shuffles; the arithmetic is on pairs of fp32 values, two per instruction.  A warp keeps to one of the two
// tensors, so that the norm's weight, and in backward its gradient, stay in registers; the angles are loaded once per token and used for the
// heads that the warp takes of it; the heads to come travel into a ring in shared memory (with the next ones in registers there were too few
// warps to hide the memory: 4 x 2048 tokens of 32 + 8 heads 36 against 33 us, backward 60 against 51).  Backward's gradients of the weights: per
// lane over all its heads, then per block in a fixed order, then one small launch over the blocks: the same bits on every run.
//
// B200, us in a row of passes, share of the copy peak, forward / backward with the weights' gradients (5 of them the second launch): bf16, heads of 128,
// 4 x 2048 tokens of 32 + 8 heads 30 (0.84) / 47 (0.82), 2048 tokens of 32 + 32 heads 15 (0.70) / 22 (0.69); alone they take 26 to 32 and 20 to 21 + 5 on
// different boxes.  fp32 heads of 96, 4096 tokens of 24 + 8: 21 (0.74) / 31 (0.75).  4 x 2048 tokens of 32 + 8 heads of 80, six of them per
// warp: 24 (0.66) / 42 (0.57); four per warp, on lanes by powers of two: 31 and 43.
#include "elem.cuh"
#include <type_traits>

namespace hyc {

constexpr int kQkThreads = 256, kQkWarps = kQkThreads / 32;
constexpr int kQkBwdBlocks = 2;      // blocks per SM that backward's registers are cut for and its workspace counts on

// one instruction, two units in the last place (the root and the quotient, each rounded, take two dozen per head)
__device__ __forceinline__ float qk_rsqrt(float v) {
  float r;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// n / d for n < 2^31 and d >= 1: a multiplication by a rounded-up reciprocal of 33 bits (T. Granlund and P. Montgomery, Division by
// invariant integers using multiplication)
struct QkDivisor { uint32_t d, mul, shift; };
__device__ __forceinline__ uint32_t qk_divide(uint32_t n, const QkDivisor& v) {
  const uint32_t hi = __umulhi(n, v.mul);
  return (hi + ((n - hi) >> (v.shift > 0 ? 1 : 0))) >> (v.shift > 0 ? v.shift - 1 : 0);
}

struct QkTensor {
  const void *x, *dy, *w;
  void* out;                       // contiguous [tokens, heads, d]
  int64_t xb, xm, xh, gb, gm, gh;  // strides of x and dy: batch, token, head
  int heads;
  int groups;                      // of heads, per token
  int splits, per_split;           // a token's head groups as `splits` items of `per_split` groups
  QkDivisor by_splits;
  int blocks;                      // blocks that work on this tensor
};
struct QkParams {
  QkTensor t[2];
  const void *cos_t, *sin_t, *pos;
  int64_t ld_cos, ld_sin, pb, pm;  // strides of the positions: batch, token
  int pos64, table_type, w_type, table_rows;
  int tokens, seq, d, half;
  QkDivisor by_seq;
  float eps;
  float* part;                     // backward: [blocks][d] sums of the weights' gradients, q's blocks first; or null
};

// The lane's channels of a head: E adjacent ones from o1 and E from o2 on.  FULL: the head's size is 2 E G and all of it is turned,
// so that every lane has channels, all of one kind, and partners at a distance known when this is compiled.
template <int E, int G, bool FULL> struct QkLane {
  int first, second;
  bool is_live, is_turned;
  __device__ __forceinline__ QkLane(int li, int d, int half) {
    const int i = li - half / E;
    is_live = li < d / (2 * E);
    is_turned = li < half / E;
    first = is_turned ? E * li : 2 * half + 2 * E * i;
    second = is_turned ? E * li + half : 2 * half + 2 * E * i + E;
    if (!is_live) { first = 0; second = 0; }
  }
  __device__ __forceinline__ bool live() const { return FULL || is_live; }
  __device__ __forceinline__ bool turned() const { return FULL || is_turned; }
  __device__ __forceinline__ int o1() const { return first; }
  __device__ __forceinline__ int o2() const { return FULL ? first + E * G : second; }
};

// cos, sin and -sin of a token at the lane's channels; a position outside of the tables gives NaN, and reads nothing
template <int N> struct QkAngles { f32x2 c[N], s[N], ns[N]; };
template <int N, typename L>
__device__ __forceinline__ void qk_angles(const QkParams& p, int b, int m, const L& l, QkAngles<N>& a) {
  int64_t at = m;
  if (p.pos != nullptr) {
    const int64_t i = b * p.pb + m * p.pm;
    at = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[i] : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[i];
  }
  const bool known = at >= 0 && at < p.table_rows;
  if (l.turned() && known) {
    ld_any_pairs(p.cos_t, at * p.ld_cos + l.o1(), p.table_type, a.c);
    ld_any_pairs(p.sin_t, at * p.ld_sin + l.o1(), p.table_type, a.s);
  } else {
    const float nan = __int_as_float(0x7fc00000);
#pragma unroll
    for (int e = 0; e < N; ++e) a.c[e] = a.s[e] = both(nan);      // (channels that are not turned do not look)
  }
#pragma unroll
  for (int e = 0; e < N; ++e) a.ns[e] = a.s[e] ^ 0x8000000080000000ull;
}

// the sum over the lanes of a head; `base`: the first of them
template <int G>
__device__ __forceinline__ float qk_sum(float v, int base) {
  if constexpr ((G & (G - 1)) == 0) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  } else {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < G; ++j) sum += __shfl_sync(0xffffffffu, v, base + j);
    return sum;
  }
}
__device__ __forceinline__ float qk_total(f32x2 v) {
  const float2 t = unpair(v);
  return t.x + t.y;
}
// where a warp's items lie
struct QkItem { uint32_t token; int first, groups, b, m; };      // token, its first head group and their number; batch entry and index in it
__device__ __forceinline__ QkItem qk_item(const QkParams& p, const QkTensor& t, uint32_t item) {
  QkItem i;
  i.token = qk_divide(item, t.by_splits);
  i.first = (int)(item - i.token * (uint32_t)t.splits) * t.per_split;
  i.groups = min(t.per_split, t.groups - i.first);
  i.b = (int)qk_divide(i.token, p.by_seq);
  i.m = (int)(i.token - (uint32_t)i.b * (uint32_t)p.seq);
  return i;
}

// ---- a warp's head groups, those of all its items in a row, on their way into shared memory kQkRing at a time: every lane copies the
// pieces that it will read itself, so that nobody waits for another lane
template <typename T> constexpr int kQkRing = sizeof(T) == 4 ? 3 : 4;      // (by shared memory)
__device__ __forceinline__ void qk_copy(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// E: channels of a piece; PER: heads of a warp at a time; BWD: x and dy, else x
template <typename T, int E, int PER, bool BWD, typename L>
struct QkFeed {
  static constexpr int PIECES = BWD ? 4 : 2, PARTS = E * (int)sizeof(T) / 16, STRIDE = kQkThreads * 16;      // 16-byte parts of a piece; of the block's lanes
  static constexpr int PLACE = PIECES * PARTS * STRIDE, RING = kQkRing<T>;
  const QkParams& p;
  const QkTensor& t;
  const L& l;
  const T *src, *grad;
  int64_t step, grad_step;
  uint32_t item, items, item_step, base, put, got, top;
  int left, todo, sub;                 // heads of the item from the lane's on; groups of the item
  __device__ __forceinline__ QkFeed(const QkParams& p_, const QkTensor& t_, const L& l_, uint32_t first, uint32_t items_, uint32_t item_step_, int sub_, uint32_t smem)
      : p(p_), t(t_), l(l_), step(PER * t_.xh), grad_step(BWD ? PER * t_.gh : 0), item(first), items(items_), item_step(item_step_),
        base(smem + threadIdx.x * 16), put(base), got(base), top(base + RING * PLACE), sub(sub_) {
    open();
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) send();
  }
  __device__ __forceinline__ void open() {
    if (item >= items) return;
    const QkItem it = qk_item(p, t, item);
    const int head0 = it.first * PER + sub;
    left = sub < PER ? t.heads - head0 : 0;      // (lanes that no head belongs to: none)
    todo = it.groups;
    src = reinterpret_cast<const T*>(t.x) + it.b * t.xb + it.m * t.xm + head0 * t.xh;
    if (BWD) grad = reinterpret_cast<const T*>(t.dy) + it.b * t.gb + it.m * t.gm + head0 * t.gh;
  }
  __device__ __forceinline__ void copy(int piece, const T* from) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) qk_copy(put + (uint32_t)((piece * PARTS + i) * STRIDE), from + i * (16 / (int)sizeof(T)));
  }
  // the next group's copies, into the ring's next place (nothing once all are under way: the groups stay countable)
  __device__ __forceinline__ void send() {
    if (item < items) {
      if (l.live() && left > 0) {
        copy(0, src + l.o1());
        copy(1, src + l.o2());
        if (BWD) {
          copy(2, grad + l.o1());
          copy(3, grad + l.o2());
        }
      }
      src += step;
      if (BWD) grad += grad_step;
      left -= PER;
      if (--todo == 0) { item += item_step; open(); }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    put += PLACE;
    if (put == top) put = base;
  }
  __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory"); }
  __device__ __forceinline__ void take(int piece, f32x2 (&f)[E / 2]) const {
    uint4 o[PARTS];
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(o[i].x), "=r"(o[i].y), "=r"(o[i].z), "=r"(o[i].w) : "r"(got + (uint32_t)((piece * PARTS + i) * STRIDE)) : "memory");
    bits_to_pairs(o, f, T());
  }
  __device__ __forceinline__ void next() {
    got += PLACE;
    if (got == top) got = base;
  }
};

template <typename T, int E, int G, bool FULL>
__global__ void __launch_bounds__(kQkThreads, 3)
qk_norm_fwd_kernel(const __grid_constant__ QkParams p) {
  extern __shared__ __align__(16) uint8_t s_ring[];
  pdl_wait();
  constexpr int PER = 32 / G;      // heads of a warp at a time
  const bool second = (int)blockIdx.x >= p.t[0].blocks;
  const QkTensor& t = p.t[second ? 1 : 0];
  const int block = (int)blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & 31, sub = lane / G;
  typedef QkLane<E, G, FULL> Lane;
  constexpr int N = E / 2;
  const Lane l(lane % G, p.d, p.half);
  const uint32_t items = (uint32_t)p.tokens * (uint32_t)t.splits, item_step = (uint32_t)t.blocks * kQkWarps;
  const uint32_t first = (uint32_t)block * kQkWarps + (threadIdx.x >> 5);
  QkFeed<T, E, PER, false, Lane> feed(p, t, l, first, items, item_step, sub, (uint32_t)__cvta_generic_to_shared(s_ring));
  f32x2 w1[N], w2[N];
  ld_any_pairs(t.w, l.o1(), p.w_type, w1);
  ld_any_pairs(t.w, l.o2(), p.w_type, w2);
  const float inv_d = 1.f / (float)p.d;
  const int out_step = PER * p.d;
  for (uint32_t item = first; item < items; item += item_step) {
    const QkItem it = qk_item(p, t, item);
    QkAngles<N> a;
    qk_angles(p, it.b, it.m, l, a);
    const int head0 = it.first * PER + sub;
    int left = sub < PER ? t.heads - head0 : 0;
    T* dst = reinterpret_cast<T*>(t.out) + (int64_t)it.token * t.heads * p.d + head0 * p.d + l.o1();
    for (int group = 0; group < it.groups; ++group, left -= PER, dst += out_step) {
      f32x2 f1[N], f2[N], ss = both(0.f);
      feed.wait();
      feed.take(0, f1);
      feed.take(1, f2);
      feed.next();
      feed.send();
#pragma unroll
      for (int e = 0; e < N; ++e) ss = fma2f(f1[e], f1[e], fma2f(f2[e], f2[e], ss));
      const f32x2 rr = both(qk_rsqrt(fmaf(qk_sum<G>(l.live() ? qk_total(ss) : 0.f, lane - lane % G), inv_d, p.eps)));
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const f32x2 n1 = mul2f(mul2f(f1[e], rr), w1[e]), n2 = mul2f(mul2f(f2[e], rr), w2[e]);
        f1[e] = l.turned() ? fma2f(n2, a.ns[e], mul2f(n1, a.c[e])) : n1;      // (not by way of n2 * 0: it may be infinite)
        f2[e] = l.turned() ? fma2f(n1, a.s[e], mul2f(n2, a.c[e])) : n2;
      }
      if (l.live() && left > 0) {
        st_pairs(dst, f1);
        st_pairs(dst + (l.o2() - l.o1()), f2);
      }
    }
  }
}

template <typename T, int E, int G, bool FULL>
__global__ void __launch_bounds__(kQkThreads, kQkBwdBlocks)
qk_norm_bwd_kernel(const __grid_constant__ QkParams p) {
  extern __shared__ __align__(16) uint8_t s_ring[];
  pdl_wait();
  constexpr int PER = 32 / G;
  const bool second = (int)blockIdx.x >= p.t[0].blocks;
  const QkTensor& t = p.t[second ? 1 : 0];
  const int block = (int)blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / G;
  typedef QkLane<E, G, FULL> Lane;
  constexpr int N = E / 2;
  const Lane l(lane % G, p.d, p.half);
  const uint32_t items = (uint32_t)p.tokens * (uint32_t)t.splits, item_step = (uint32_t)t.blocks * kQkWarps;
  const uint32_t first = (uint32_t)block * kQkWarps + (uint32_t)warp;
  QkFeed<T, E, PER, true, Lane> feed(p, t, l, first, items, item_step, sub, (uint32_t)__cvta_generic_to_shared(s_ring));
  f32x2 w1[N], w2[N], dw1[N], dw2[N];
  ld_any_pairs(t.w, l.o1(), p.w_type, w1);
  ld_any_pairs(t.w, l.o2(), p.w_type, w2);
#pragma unroll
  for (int e = 0; e < N; ++e) dw1[e] = dw2[e] = both(0.f);
  const float inv_d = 1.f / (float)p.d;
  const int out_step = PER * p.d;
  for (uint32_t item = first; item < items; item += item_step) {
    const QkItem it = qk_item(p, t, item);
    QkAngles<N> a;
    qk_angles(p, it.b, it.m, l, a);
    const int head0 = it.first * PER + sub;
    int left = sub < PER ? t.heads - head0 : 0;
    T* dst = reinterpret_cast<T*>(t.out) + (int64_t)it.token * t.heads * p.d + head0 * p.d + l.o1();
    for (int group = 0; group < it.groups; ++group, left -= PER, dst += out_step) {
      const bool ok = left > 0;
      f32x2 f1[N], f2[N], g1[N], g2[N], ss = both(0.f), sg = both(0.f);
      feed.wait();
      feed.take(0, f1);
      feed.take(1, f2);
      feed.take(2, g1);
      feed.take(3, g2);
      feed.next();
      feed.send();
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const f32x2 u = l.turned() ? fma2f(g2[e], a.s[e], mul2f(g1[e], a.c[e])) : g1[e];
        const f32x2 v = l.turned() ? fma2f(g1[e], a.ns[e], mul2f(g2[e], a.c[e])) : g2[e];
        ss = fma2f(f1[e], f1[e], fma2f(f2[e], f2[e], ss));
        sg = fma2f(mul2f(u, f1[e]), w1[e], fma2f(mul2f(v, f2[e]), w2[e], sg));
        g1[e] = u; g2[e] = v;
      }
      // dx = r g w - x r^2 mean(g w x r)
      const float r = qk_rsqrt(fmaf(qk_sum<G>(l.live() ? qk_total(ss) : 0.f, lane - lane % G), inv_d, p.eps));
      const float pull = qk_sum<G>(l.live() ? qk_total(sg) : 0.f, lane - lane % G) * (r * inv_d) * (r * -r);
      const f32x2 rr = both(r), pp = both(pull);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const f32x2 u = mul2f(g1[e], rr), v = mul2f(g2[e], rr);
        if (ok) { dw1[e] = fma2f(u, f1[e], dw1[e]); dw2[e] = fma2f(v, f2[e], dw2[e]); }
        f1[e] = fma2f(f1[e], pp, mul2f(u, w1[e]));
        f2[e] = fma2f(f2[e], pp, mul2f(v, w2[e]));
      }
      if (ok && l.live()) {
        st_pairs(dst, f1);
        st_pairs(dst + (l.o2() - l.o1()), f2);
      }
    }
  }
  if (p.part == nullptr) return;
  __syncthreads();      // (the ring is empty: nothing is on its way that a warp has not waited for)
  float* s_part = reinterpret_cast<float*>(s_ring);      // [warp][channel]
#pragma unroll
  for (int e = 0; e < N; ++e) {
    // (lanes of the first head: the others' sums, the next head's first)
    const f32x2 mine1 = dw1[e], mine2 = dw2[e];
#pragma unroll
    for (int h = 1; h < PER; ++h) {
      dw1[e] = add2f(dw1[e], __shfl_sync(0xffffffffu, (unsigned long long)mine1, lane % G + h * G));
      dw2[e] = add2f(dw2[e], __shfl_sync(0xffffffffu, (unsigned long long)mine2, lane % G + h * G));
    }
    if (sub == 0 && l.live()) {
      const float2 u = unpair(dw1[e]), v = unpair(dw2[e]);
      float *at1 = s_part + warp * p.d + l.o1() + 2 * e, *at2 = s_part + warp * p.d + l.o2() + 2 * e;
      at1[0] = u.x; at1[1] = u.y;
      at2[0] = v.x; at2[1] = v.y;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.d; i += kQkThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kQkWarps; ++w) sum += s_part[w * p.d + i];
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

// Channels of a lane's piece: 16 bytes, so that the lanes of a head read whole lines; fp32 heads of more than 256 channels 32 bytes, for 32 lanes
static int qk_piece(int type, int d) { return type == HYC_F32 && d <= 256 ? 4 : 8; }
// lanes of a head: a power of two, or as many as it has pieces where more heads fit into a warp that way (five and six lanes: heads of 80 and 96
// channels, 6 and 5 of them instead of 4)
static int qk_group(int type, int d) {
  const int pieces = d / (2 * qk_piece(type, d));
  int g = 1;
  while (g < pieces) g <<= 1;
  return 32 / pieces > 32 / g ? pieces : g;
}
static QkDivisor qk_divisor(uint32_t d) {
  uint32_t shift = 0;
  while ((1ull << shift) < d) ++shift;
  return {d, (uint32_t)((((1ull << shift) - d) << 32) / d + 1), shift};
}

// How one tensor's items are cut, for `blocks` blocks: a warp's share is a whole number of items, so that small ones fill the last round, and each
// costs about two groups more (division, angles).  Returns what the busiest warp has to do, in groups.
static int64_t qk_cut(QkTensor& t, int tokens, int groups, int blocks) {
  const int64_t warps = (int64_t)blocks * kQkWarps;
  int64_t best = 0;
  for (int i = 1; i <= 9; ++i) {
    const int want = i <= 8 ? i : groups;      // items of a token
    if (want > groups) continue;
    const int per_split = (groups + want - 1) / want, splits = (groups + per_split - 1) / per_split;
    const int64_t cost = ((int64_t)tokens * splits + warps - 1) / warps * (per_split + 2);
    if (best == 0 || cost < best) { best = cost; t.per_split = per_split; t.splits = splits; }
  }
  return best;
}
// Blocks for the two tensors, at most one resident wave and no more than there is work for: in proportion to what their tokens cost, moved
// by what the whole numbers of items make of it.
static void qk_plan(QkParams& p, int group, int wave) {
  const int per = 32 / group;
  int groups[2];
  for (int i = 0; i < 2; ++i) groups[i] = (p.t[i].heads + per - 1) / per;
  // (few tokens: a warp for each group)
  const bool each = (int64_t)p.tokens * (groups[0] + groups[1]) <= (int64_t)(wave - 1) * kQkWarps;
  const int even = (int)((int64_t)wave * (groups[0] + 2) / (groups[0] + groups[1] + 4)), step = wave / 32;
  int64_t best = 0;
  int first = even;
  for (int i = -2; i <= 2 && !each; ++i) {
    int blocks = even + i * step;
    blocks = blocks < 1 ? 1 : blocks > wave - 1 ? wave - 1 : blocks;
    const int64_t q = qk_cut(p.t[0], p.tokens, groups[0], blocks), k = qk_cut(p.t[1], p.tokens, groups[1], wave - blocks), cost = q > k ? q : k;
    if (best == 0 || cost < best) { best = cost; first = blocks; }
  }
  for (int i = 0; i < 2; ++i) {
    QkTensor& t = p.t[i];
    int blocks = i == 0 ? first : wave - first;
    t.groups = groups[i];
    if (each) {
      t.per_split = 1;
      t.splits = groups[i];
      blocks = wave;
    } else {
      qk_cut(t, p.tokens, groups[i], blocks);
    }
    t.by_splits = qk_divisor((uint32_t)t.splits);
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
  p.by_seq = qk_divisor(p.seq > 0 ? (uint32_t)p.seq : 1u);
  p.part = nullptr;
}

// bytes of the ring, and of backward's sums over the warps, which take its place
template <typename T>
constexpr int qk_smem(int piece, bool backward) { return kQkRing<T> * (backward ? 4 : 2) * kQkThreads * piece * (int)sizeof(T); }
static_assert(qk_smem<__half>(8, true) >= kQkWarps * 512 * 4 && qk_smem<float>(4, true) >= kQkWarps * 256 * 4, "the sums fit in the ring");

// f(element, channels of a piece, lanes of a head, FULL)
template <typename F>
static int qk_by_type(int type, int d, int rot, F&& f) {
  using std::integral_constant;
  auto by_group = [&](auto elem, auto piece) -> int {
    auto full = [&](auto group) -> int {
      if (rot == d && d == 2 * decltype(piece)::value * decltype(group)::value) return f(elem, piece, group, std::true_type());
      return f(elem, piece, group, std::false_type());
    };
    constexpr bool wide_only = sizeof(elem) == 4 && decltype(piece)::value == 8;      // (fp32 heads of more than 256 channels)
    if constexpr (!wide_only) {
      switch (qk_group(type, d)) {
        case 1: return full(integral_constant<int, 1>());
        case 2: return full(integral_constant<int, 2>());
        case 3: return full(integral_constant<int, 3>());
        case 5: return full(integral_constant<int, 5>());
        case 6: return full(integral_constant<int, 6>());
        case 9: return full(integral_constant<int, 9>());
        case 10: return full(integral_constant<int, 10>());
        case 4: return full(integral_constant<int, 4>());
        case 8: return full(integral_constant<int, 8>());
        case 16: return full(integral_constant<int, 16>());
        default: break;
      }
    }
    return full(integral_constant<int, 32>());
  };
  if (type == HYC_F32) return qk_piece(type, d) == 4 ? by_group(float(), integral_constant<int, 4>()) : by_group(float(), integral_constant<int, 8>());
  if (type == HYC_F16) return by_group(__half(), integral_constant<int, 8>());
  return by_group(__nv_bfloat16(), integral_constant<int, 8>());
}

}  // namespace hyc

using namespace hyc;

extern "C" HYC_API int hyc_qk_norm_rope_fwd(const hyc_qk_norm* a, void* stream) {
  const int rc = qk_check(a, false);
  if (rc != HYC_OK || a->batch * a->seq == 0) return rc;
  QkParams p;
  qk_fill(p, a);
  return qk_by_type(a->type, p.d, 2 * p.half, [&](auto elem, auto piece, auto group, auto full) -> int {
    constexpr auto kern = qk_norm_fwd_kernel<decltype(elem), decltype(piece)::value, decltype(group)::value, decltype(full)::value>;
    constexpr int smem = qk_smem<decltype(elem)>(decltype(piece)::value, false);
    const int rs = more_shared_memory<kern>(smem);
    if (rs != HYC_OK) return rs;
    qk_plan(p, decltype(group)::value, num_sms() * resident_blocks(kern, kQkThreads, smem, 1));
    launch_pdl(kern, dim3((unsigned)(p.t[0].blocks + p.t[1].blocks)), dim3(kQkThreads), smem, (cudaStream_t)stream, p);
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
    const int r = qk_by_type(a->type, p.d, 2 * p.half, [&](auto elem, auto piece, auto group, auto full) -> int {
      constexpr auto kern = qk_norm_bwd_kernel<decltype(elem), decltype(piece)::value, decltype(group)::value, decltype(full)::value>;
      constexpr int smem = qk_smem<decltype(elem)>(decltype(piece)::value, true);
      const int rs = more_shared_memory<kern>(smem);
      if (rs != HYC_OK) return rs;
      const int res = resident_blocks(kern, kQkThreads, smem, 1);
      qk_plan(p, decltype(group)::value, num_sms() * (res < kQkBwdBlocks ? res : kQkBwdBlocks));
      launch_pdl(kern, dim3((unsigned)(p.t[0].blocks + p.t[1].blocks)), dim3(kQkThreads), smem, (cudaStream_t)stream, p);
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
