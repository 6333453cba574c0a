// RMS norms of the query and key heads with the rotary embedding in the same pass, and their backward pass.
//
//   r = 1 / sqrt(mean(x^2) + eps) over the d channels of one head,   n = x r w
//   y[j]     = n[j] c - n[j + h] s,   y[j + h] = n[j + h] c + n[j] s      j < h = rot / 2;   y[j] = n[j] from rot on
// with c, s = cos[p, j], sin[p, j] at the token's position p.  Backward, g = dy turned back by the same angle:
//   dw = sum g x r,   dx = r (g w - x r mean(g w x r))
// The row sums r needs are taken again from x, which backward reads anyway: nothing is kept between the passes but q and k.
// Everything is fp32 between the loads and the one rounding at the store.
//
// Bound by memory: x is read and y written once (backward: x, dy, dx).  A head belongs to G = 1 .. 32 adjacent lanes, each
// with the 16 channels [8 i, 8 i + 8) and their partners h further (behind rot: 16 channels in a row), so that the pairs of the
// rotation meet in one lane, all accesses are 128 bits wide, and a mean is log2 G shuffles.  A warp keeps to one of the two
// tensors, so that the norm's weight, and in backward its gradient, stay in registers; the angles are loaded once per token
// and used for the heads that the warp takes of it.  Backward's gradients of the weights: per lane over all its heads, then
// per block in a fixed order, then one small launch over the blocks: the same bits on every run.
#include "elem.cuh"
#include <type_traits>

namespace hyc {

constexpr int kQkThreads = 256, kQkWarps = kQkThreads / 32;

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

// The lane's two octets of a head: channels o1 .. o1 + 7 and o2 .. o2 + 7
struct QkLane { int o1, o2; bool live, turned; };
__device__ __forceinline__ QkLane qk_lane(int li, int d, int half) {
  QkLane l;
  l.live = li < d / 16;
  l.turned = li < half / 8;
  const int i = li - half / 8;
  l.o1 = l.turned ? 8 * li : 2 * half + 16 * i;
  l.o2 = l.turned ? l.o1 + half : l.o1 + 8;
  if (!l.live) { l.o1 = 0; l.o2 = 0; }
  return l;
}

// cos and sin of a token at the lane's channels; a position outside of the tables gives NaN, and reads nothing
__device__ __forceinline__ void qk_angles(const QkParams& p, int b, int m, const QkLane& l, float (&c)[8], float (&s)[8]) {
  if (!l.turned) {
#pragma unroll
    for (int e = 0; e < 8; ++e) { c[e] = 1.f; s[e] = 0.f; }
    return;
  }
  int64_t at = m;
  if (p.pos != nullptr) {
    const int64_t i = b * p.pb + m * p.pm;
    at = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[i] : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[i];
  }
  if (at < 0 || at >= p.table_rows) {
#pragma unroll
    for (int e = 0; e < 8; ++e) { c[e] = __int_as_float(0x7fc00000); s[e] = c[e]; }
    return;
  }
  ld_any8(p.cos_t, at * p.ld_cos + l.o1, p.table_type, c);
  ld_any8(p.sin_t, at * p.ld_sin + l.o1, p.table_type, s);
}

template <int G>
__device__ __forceinline__ float qk_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// UNROLL head groups are on their way at once
template <typename T, int G, int UNROLL>
__global__ void __launch_bounds__(kQkThreads)
qk_norm_fwd_kernel(const __grid_constant__ QkParams p) {
  pdl_wait();
  constexpr int PER = 32 / G;      // heads of a warp at a time
  const bool second = (int)blockIdx.x >= p.t[0].blocks;
  const QkTensor& t = p.t[second ? 1 : 0];
  const int block = (int)blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & 31, sub = lane / G;
  const QkLane l = qk_lane(lane % G, p.d, p.half);
  const T* x = reinterpret_cast<const T*>(t.x);
  T* out = reinterpret_cast<T*>(t.out);
  float w1[8], w2[8];
  ld_any8(t.w, l.o1, p.w_type, w1);
  ld_any8(t.w, l.o2, p.w_type, w2);
  const float inv_d = 1.f / (float)p.d;
  const uint32_t items = (uint32_t)p.tokens * (uint32_t)t.splits;
  for (uint32_t item = (uint32_t)block * kQkWarps + (threadIdx.x >> 5); item < items; item += (uint32_t)t.blocks * kQkWarps) {
    const uint32_t token = item / (uint32_t)t.splits;
    const int first = (int)(item - token * (uint32_t)t.splits) * t.per_split;
    const int b = (int)(token / (uint32_t)p.seq), m = (int)(token - (uint32_t)b * (uint32_t)p.seq);
    const T* xt = x + b * t.xb + m * t.xm;
    T* ot = out + (int64_t)token * t.heads * p.d;
    float c[8], s[8];
    qk_angles(p, b, m, l, c, s);
    for (int g0 = first; g0 < first + t.per_split; g0 += UNROLL) {
      Octet<T> a[UNROLL], bb[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int head = (g0 + u) * PER + sub;
        const bool ok = l.live && head < t.heads && g0 + u < first + t.per_split;
        a[u] = ok ? ld_octet(xt + head * t.xh + l.o1) : zero_octet<T>();
        bb[u] = ok ? ld_octet(xt + head * t.xh + l.o2) : zero_octet<T>();
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int head = (g0 + u) * PER + sub;
        const bool ok = l.live && head < t.heads && g0 + u < first + t.per_split;
        float f1[8], f2[8], ss = 0.f;
        octet_to_f32(a[u], f1);
        octet_to_f32(bb[u], f2);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f1[e], f1[e], fmaf(f2[e], f2[e], ss));
        const float r = 1.f / sqrtf(fmaf(qk_sum<G>(ss), inv_d, p.eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float n1 = f1[e] * r * w1[e], n2 = f2[e] * r * w2[e];
          f1[e] = n1 * c[e] - n2 * s[e];
          f2[e] = n2 * c[e] + n1 * s[e];
        }
        if (ok) {
          st_octet(ot + head * p.d + l.o1, f1);
          st_octet(ot + head * p.d + l.o2, f2);
        }
      }
    }
  }
}

template <typename T, int G>
__global__ void __launch_bounds__(kQkThreads)
qk_norm_bwd_kernel(const __grid_constant__ QkParams p) {
  __shared__ float s_part[kQkWarps][512];
  pdl_wait();
  constexpr int PER = 32 / G;
  const bool second = (int)blockIdx.x >= p.t[0].blocks;
  const QkTensor& t = p.t[second ? 1 : 0];
  const int block = (int)blockIdx.x - (second ? p.t[0].blocks : 0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / G;
  const QkLane l = qk_lane(lane % G, p.d, p.half);
  const T *x = reinterpret_cast<const T*>(t.x), *dy = reinterpret_cast<const T*>(t.dy);
  T* out = reinterpret_cast<T*>(t.out);
  float w1[8], w2[8], dw1[8], dw2[8];
  ld_any8(t.w, l.o1, p.w_type, w1);
  ld_any8(t.w, l.o2, p.w_type, w2);
#pragma unroll
  for (int e = 0; e < 8; ++e) { dw1[e] = 0.f; dw2[e] = 0.f; }
  const float inv_d = 1.f / (float)p.d;
  const uint32_t items = (uint32_t)p.tokens * (uint32_t)t.splits;
  for (uint32_t item = (uint32_t)block * kQkWarps + warp; item < items; item += (uint32_t)t.blocks * kQkWarps) {
    const uint32_t token = item / (uint32_t)t.splits;
    const int first = (int)(item - token * (uint32_t)t.splits) * t.per_split;
    const int b = (int)(token / (uint32_t)p.seq), m = (int)(token - (uint32_t)b * (uint32_t)p.seq);
    const T *xt = x + b * t.xb + m * t.xm, *gt = dy + b * t.gb + m * t.gm;
    T* ot = out + (int64_t)token * t.heads * p.d;
    float c[8], s[8];
    qk_angles(p, b, m, l, c, s);
    for (int g0 = first; g0 < first + t.per_split; ++g0) {
      const int head = g0 * PER + sub;
      const bool ok = l.live && head < t.heads;
      float f1[8], f2[8], g1[8], g2[8], ss = 0.f, sg = 0.f;
      {
        const Octet<T> xa = ok ? ld_octet(xt + head * t.xh + l.o1) : zero_octet<T>(), xb = ok ? ld_octet(xt + head * t.xh + l.o2) : zero_octet<T>();
        const Octet<T> ga = ok ? ld_octet(gt + head * t.gh + l.o1) : zero_octet<T>(), gb = ok ? ld_octet(gt + head * t.gh + l.o2) : zero_octet<T>();
        octet_to_f32(xa, f1); octet_to_f32(xb, f2); octet_to_f32(ga, g1); octet_to_f32(gb, g2);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = g1[e] * c[e] + g2[e] * s[e], d = g2[e] * c[e] - g1[e] * s[e];
        g1[e] = a; g2[e] = d;
        ss = fmaf(f1[e], f1[e], fmaf(f2[e], f2[e], ss));
        sg = fmaf(a * w1[e], f1[e], fmaf(d * w2[e], f2[e], sg));
      }
      const float r = 1.f / sqrtf(fmaf(qk_sum<G>(ss), inv_d, p.eps));
      const float mean = qk_sum<G>(sg) * r * inv_d;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n1 = f1[e] * r, n2 = f2[e] * r;
        if (ok) { dw1[e] = fmaf(g1[e], n1, dw1[e]); dw2[e] = fmaf(g2[e], n2, dw2[e]); }      // (an idle lane: its NaN angles times zero)
        f1[e] = r * (g1[e] * w1[e] - n1 * mean);
        f2[e] = r * (g2[e] * w2[e] - n2 * mean);
      }
      if (ok) {
        st_octet(ot + head * p.d + l.o1, f1);
        st_octet(ot + head * p.d + l.o2, f2);
      }
    }
  }
  if (p.part == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) {
      dw1[e] += __shfl_xor_sync(0xffffffffu, dw1[e], o);
      dw2[e] += __shfl_xor_sync(0xffffffffu, dw2[e], o);
    }
    if (sub == 0 && l.live) { s_part[warp][l.o1 + e] = dw1[e]; s_part[warp][l.o2 + e] = dw2[e]; }
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

// lanes of a head
static int qk_group(int d) {
  int g = 1;
  while (g < d / 16) g <<= 1;
  return g;
}

// Blocks for the two tensors in proportion to their heads, at most one resident wave and no more than there is work for; a token's head
// groups are dealt to several warps where there are fewer tokens than warps.
static void qk_plan(QkParams& p, int wave) {
  const int per = 32 / qk_group(p.d), heads = p.t[0].heads + p.t[1].heads;
  for (int i = 0; i < 2; ++i) {
    QkTensor& t = p.t[i];
    const int groups = (t.heads + per - 1) / per;
    int blocks = (int)((int64_t)wave * t.heads / heads);
    if (blocks < 1) blocks = 1;
    const int64_t warps = (int64_t)blocks * kQkWarps;
    int64_t splits = p.tokens >= warps ? 1 : (warps + p.tokens - 1) / p.tokens;
    if (splits > groups) splits = groups;
    t.per_split = (int)((groups + splits - 1) / splits);
    t.splits = (groups + t.per_split - 1) / t.per_split;
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

template <typename F>
static int qk_by_type(int type, int group, F&& f) {
  auto by_group = [&](auto elem) -> int {
    using T = decltype(elem);
    switch (group) {
      case 1: return f(elem, std::integral_constant<int, 1>());
      case 2: return f(elem, std::integral_constant<int, 2>());
      case 4: return f(elem, std::integral_constant<int, 4>());
      case 8: return f(elem, std::integral_constant<int, 8>());
      case 16: return f(elem, std::integral_constant<int, 16>());
      default: return f(elem, std::integral_constant<int, 32>());
    }
  };
  if (type == HYC_F32) return by_group(float());
  if (type == HYC_F16) return by_group(__half());
  return by_group(__nv_bfloat16());
}

constexpr int kQkBwdWave = 4;      // resident blocks per SM that backward counts on at most (its workspace does not ask the device)

}  // namespace hyc

using namespace hyc;

extern "C" HYC_API int hyc_qk_norm_rope_fwd(const hyc_qk_norm* a, void* stream) {
  const int rc = qk_check(a, false);
  if (rc != HYC_OK || a->batch * a->seq == 0) return rc;
  QkParams p;
  qk_fill(p, a);
  return qk_by_type(a->type, qk_group(p.d), [&](auto elem, auto group) -> int {
    auto kern = qk_norm_fwd_kernel<decltype(elem), decltype(group)::value, sizeof(elem) == 4 ? 1 : 2>;
    qk_plan(p, num_sms() * resident_blocks(kern, kQkThreads, 0, 2));
    launch_pdl(kern, dim3((unsigned)(p.t[0].blocks + p.t[1].blocks)), dim3(kQkThreads), 0, (cudaStream_t)stream, p);
    HYC_CHECK_LAUNCH();
    return HYC_OK;
  });
}

extern "C" HYC_API size_t hyc_qk_norm_rope_workspace_bytes(int head_dim) {
  return head_dim < 16 || head_dim > 512 ? 0 : (size_t)(num_sms() * kQkBwdWave + 2) * (size_t)head_dim * sizeof(float);
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
    const int r = qk_by_type(a->type, qk_group(p.d), [&](auto elem, auto group) -> int {
      auto kern = qk_norm_bwd_kernel<decltype(elem), decltype(group)::value>;
      const int res = resident_blocks(kern, kQkThreads, 0, 2);
      qk_plan(p, num_sms() * (res < kQkBwdWave ? res : kQkBwdWave));
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
