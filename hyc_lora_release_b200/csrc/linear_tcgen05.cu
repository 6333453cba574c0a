// Products with bias, activation and residual in the epilogue, and the products of their backward pass, on tcgen05.
//
//   forward   pre = x W^T + bias,  y = act(pre) + residual          backward   dpre = dy act'(pre)
//             (pre kept on demand, rounded; act takes the fp32 sum)            dx = dpre W,  dW = dpre^T x,  dbias = sum dpre
//
// All three products are C[r, c] = sum_k A[r, k] B[c, k] with operands whose contraction index is either adjacent in memory (K-major) or
// not (MN-major: W for dx, both operands for dW): no operand is copied or transposed.  bf16 or fp16 operands, fp32 accumulators in tensor
// memory, one rounding at the store.  dpre is rounded to 16 bits before its two products, as tensor-core operands are: its error, half a
// step per element, averages out in the sums, which carry about 1.4 times the error of their own rounding
// (up to 1.5 with one to four tokens); a second product with what the rounding took would double the work.
//
// Two kernels, both fed by TMA (128-byte swizzle, 64-wide k-blocks; what lies outside of an operand arrives as zero, so that any number of
// rows and any multiple of 8 columns is right), every wait bounded (hyc_linear_status; tc_settle before a CTA leaves):
//   tiles    persistent CTA pairs, 256 x 256 or 256 x 128 results per pair by tcgen05.mma.cta_group::2, two accumulators, so that the
//            epilogue of one tile overlaps the main loop of the next
//   slices   few rows or few tiles: one tile of 128 result COLUMNS x up to 256 rows per CTA (256 per CTA pair), the columns on the lanes of
//            tensor memory and the rows in its columns (a product of one row costs N = 16, not 128), K shared by the CTAs or pairs of a
//            cluster, whose partial sums meet in distributed shared memory in a fixed order
//
// B200, bf16, us of one launch alone, on different boxes (share of the measured burst rate or copy peak): tiles 2048 x 4096 -> 11008 with gelu and pre 112-127
// (0.99-0.88), its dx 111-128, dW 104-120, 8192 x 4096 -> 14336 573-609, with gelu and pre 604-640; the tensor pipe is busy 92 % of the cycles.  In a row of
// passes, under the power cap: 154, 125, 125, 719 and 744-768.  Slices, in a row of passes: 1 x 4096 -> 11008 19 (0.74 of the copy peak), 1 x 4096
// -> 4096 10, 128 x 4096 -> 4096 16, 333 x 11008 -> 4096 38 (alone 22, 13, 17, 31-35): bound by the weight's bytes and the start and end of a launch
// (about 6 us), from 200 rows on by operands from L2.  dpre of 2048 x 11008 with silu 25 alone (0.83).  Backward of 1 to 128 tokens, 4096 -> 11008: dx 20-24
// (0.67-0.58), dW 38-39 (0.36): its 90 MB of results leave through the epilogue, eight warps per SM that take 32 x 32 of them at a time.
#include "tc_common.cuh"
#include "elem.cuh"
#include <type_traits>

namespace hyc {
namespace lin {

using namespace tc;

__device__ int g_status;      // of the bounded waits of this file's kernels; 0 unless one gave up

struct Epilogue {
  const void* bias;           // [C] or null
  const void* residual;       // [R, C], or null
  void* pre;                  // [R, C], or null
  void* out;                  // [R, C]
  int64_t ld_res;             // (pre and out are contiguous)
  int act;
};
struct Shape { int R, C, K; };

// ---- activations, fp32
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
// erfc(|x| / sqrt 2) / 2 = q(t) e^(-x^2 / 2), t = 1 / (1 + 0.36 |x| / sqrt 2).  q / t is a polynomial of degree 6, fitted for the least maximum of the
// relative error over |x| < 14, weighted towards 0 (a linear program over its Chebyshev coefficients): with fp32's roundings q is off by 4.9e-6 of
// itself, the tail by 2.1e-7.  x Phi(x) = max(x, 0) - |x| erfc(..) / 2, with no cancellation on either side.
__device__ __forceinline__ float normal_tail(float x, float& density) {      // density: e^(-x^2 / 2)
  const float ax = fabsf(x);
  const float t = __fdividef(1.f, fmaf(0.36f * 0.70710678118654752f, ax, 1.f));
  float q = fmaf(t, -0.08069140564f, 0.277714377f);
  q = fmaf(t, q, -0.1709972366f);
  q = fmaf(t, q, 0.2089158673f);
  q = fmaf(t, q, 0.05609946922f);
  q = fmaf(t, q, 0.1078153617f);
  q = t * fmaf(t, q, 0.1011436123f);
  density = __expf(-0.5f * x * x);
  return q * density;
}
constexpr float kTanhA = 1.5957691216057308f, kTanhB = 0.0713548162726009f;      // 2 sqrt(2 / pi), the same times 0.044715
template <int ACT>
__device__ __forceinline__ float act_of(float x) {
  if constexpr (ACT == HYC_ACT_RELU) return x > 0.f || x != x ? x : 0.f;      // (NaN stays)
  else if constexpr (ACT == HYC_ACT_GELU) {
    float density;
    const float tail = normal_tail(x, density);
    return fmaf(-fminf(fabsf(x), 100.f), tail, fmaxf(x, 0.f));      // (far out the tail is 0; NaN is in it)
  }
  else if constexpr (ACT == HYC_ACT_GELU_TANH) return x * sigmoid(x * fmaf(kTanhB, x * x, kTanhA));      // (1 + tanh u) / 2 = sigmoid(2 u)
  else if constexpr (ACT == HYC_ACT_SILU) return x * sigmoid(x);
  else return x;
}
template <int ACT>
__device__ __forceinline__ float slope_of(float x) {
  if constexpr (ACT == HYC_ACT_RELU) return x > 0.f ? 1.f : x != x ? x : 0.f;
  else if constexpr (ACT == HYC_ACT_GELU) {
    float density;
    const float tail = normal_tail(x, density);
    return fmaf(x * 0.39894228040143268f, density, x > 0.f ? 1.f - tail : tail);
  }
  else if constexpr (ACT == HYC_ACT_GELU_TANH) {
    if (fabsf(x) > 30.f) return x > 0.f ? 1.f : 0.f;      // (x^2 may be infinite)
    const float s = sigmoid(x * fmaf(kTanhB, x * x, kTanhA));
    return s + x * s * (1.f - s) * fmaf(3.f * kTanhB, x * x, kTanhA);
  } else if constexpr (ACT == HYC_ACT_SILU) {
    const float s = sigmoid(x);
    return fmaf(x * s, 1.f - s, s);
  } else return 1.f;
}
template <typename F>
__device__ __forceinline__ void by_act(int act, F&& f) {      // (the same for a whole launch)
  switch (act) {
    case HYC_ACT_RELU: f(std::integral_constant<int, HYC_ACT_RELU>()); break;
    case HYC_ACT_GELU: f(std::integral_constant<int, HYC_ACT_GELU>()); break;
    case HYC_ACT_GELU_TANH: f(std::integral_constant<int, HYC_ACT_GELU_TANH>()); break;
    case HYC_ACT_SILU: f(std::integral_constant<int, HYC_ACT_SILU>()); break;
    default: f(std::integral_constant<int, HYC_ACT_NONE>()); break;
  }
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2_rn(a, b); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return f32_to_half2_bits(a, b); }
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) { return make_float2(bf16lo_to_f32(w), bf16hi_to_f32(w)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return half2_bits_to_f32(w); }

// instruction descriptor: fp32 accumulators, M rows, N columns, element type, which operands are MN-major
template <typename T, bool A_MN, bool B_MN>
__device__ __forceinline__ uint32_t instruction(int m, int n) {
  constexpr uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <bool MN> __device__ __forceinline__ uint64_t operand_desc(uint32_t at) { return MN ? make_desc(at, 64 * 128, 1024) : make_desc(at, 16, 1024); }
// 16 k further: 32 bytes along a swizzled row, or 16 rows of 128 bytes
template <bool MN> constexpr uint64_t kStep = MN ? 128 : 2;

// ------------------------------------------------------------------ tiles
constexpr int T_STAGE = 32768, T_STAGES = 6;                              // 128 rows of A and 128 of B per CTA and k-block
constexpr int T_EPI_BYTES = EPI_WARPS * 2048 + BN * 4;                    // a [32][32] 16-bit tile per epilogue warp; the columns' bias
constexpr int T_SMEM = 1024 + T_STAGES * T_STAGE + T_EPI_BYTES + 256;

struct TileParams {
  Shape s;
  Epilogue e;
  int tiles_m, n_wide, n_tiles, group;      // column tiles: the first n_wide are 256 wide, the others 128; row tiles of a raster group
};

// tile number -> row tile and column tile: groups of `group` row tiles, in each the row tile runs fastest (operands of neighbours stay in L2)
__device__ __forceinline__ void tile_of(const TileParams& p, int tile, int columns, int& mt, int& ct) {
  const int per = p.group * columns, g = tile / per, rest = tile - g * per;
  const int rows = min(p.group, p.tiles_m - g * p.group);
  ct = rest / rows;
  mt = g * p.group + rest - ct * rows;
}

template <typename T>
__device__ __forceinline__ void flush_tile(const uint32_t* R, T* out, int64_t row0, int R_rows, int64_t ld, int n, int C, int lane) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = 8 * k + (lane >> 2), c = lane & 3;
    const uint4 v = *reinterpret_cast<const uint4*>(R + gd_chunk(r, c));
    if (row0 + r < R_rows && n + 8 * c < C) *reinterpret_cast<uint4*>(out + (row0 + r) * ld + n + 8 * c) = v;
  }
}
template <typename T>
__device__ __forceinline__ void fetch_tile(const T* src, int64_t row0, int R_rows, int64_t ld, int n, int C, int lane, uint4 (&v)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = 8 * k + (lane >> 2), c = lane & 3;
    v[k] = make_uint4(0u, 0u, 0u, 0u);
    if (row0 + r < R_rows && n + 8 * c < C) v[k] = *reinterpret_cast<const uint4*>(src + (row0 + r) * ld + n + 8 * c);
  }
}

// One [32 rows][32 columns] block of results by a warp: the accumulators of the lane's row in, results out through the warp's tile
template <typename T>
__device__ __forceinline__ void tile_block(const TileParams& p, const uint32_t (&acc)[32], const float* bias, uint32_t* R, int64_t row0, int n, int lane,
                                           const uint4 (&res)[4]) {
  float v[32];
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float4 b = *reinterpret_cast<const float4*>(bias + c);
    v[c] = __uint_as_float(acc[c]) + b.x; v[c + 1] = __uint_as_float(acc[c + 1]) + b.y;
    v[c + 2] = __uint_as_float(acc[c + 2]) + b.z; v[c + 3] = __uint_as_float(acc[c + 3]) + b.w;
  }
  auto out = [&](void* dst) {
#pragma unroll
    for (int c8 = 0; c8 < 4; ++c8)
      *reinterpret_cast<uint4*>(R + gd_chunk(lane, c8)) = make_uint4(pack2<T>(v[8 * c8], v[8 * c8 + 1]), pack2<T>(v[8 * c8 + 2], v[8 * c8 + 3]),
                                                                     pack2<T>(v[8 * c8 + 4], v[8 * c8 + 5]), pack2<T>(v[8 * c8 + 6], v[8 * c8 + 7]));
    __syncwarp();
    flush_tile<T>(R, (T*)dst, row0, p.s.R, p.s.C, n, p.s.C, lane);
    __syncwarp();
  };
  if (p.e.pre != nullptr) out(p.e.pre);
  by_act(p.e.act, [&](auto a) {
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] = act_of<decltype(a)::value>(v[c]);
  });
  if (p.e.residual != nullptr) {
    tile_put(R, lane, res);
    __syncwarp();
#pragma unroll
    for (int c8 = 0; c8 < 4; ++c8) {
      const uint4 r = *reinterpret_cast<const uint4*>(R + gd_chunk(lane, c8));
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2<T>(w[j]);
        v[8 * c8 + 2 * j] += f.x;
        v[8 * c8 + 2 * j + 1] += f.y;
      }
    }
    __syncwarp();
  }
  out(p.e.out);
}

template <typename T, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(THREADS, 1)
linear_tiles_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_b_narrow,
                    const TileParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align_shared(smem_raw);
  uint8_t* epi = smem + T_STAGES * T_STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi + T_EPI_BYTES);
  uint64_t *full = bars, *empty = bars + T_STAGES, *acc_full = bars + 2 * T_STAGES, *acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();      // 0: leader of the pair, issues the MMAs
  const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
  const int columns = p.n_tiles, tiles = p.tiles_m * columns, kbs = (p.s.K + BK - 1) / BK;
  auto first_column = [&](int ct) { return ct < p.n_wide ? ct * BN : p.n_wide * BN + (ct - p.n_wide) * (BN / 2); };

  if (warp == 0 && elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_a)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_b)) : "memory");
  }
  if (threadIdx.x == 0) {
    // full and acc_empty are used in the leader: both CTAs' loads and epilogue warps arrive there; the leader's commits arrive in both CTAs
    for (int s = 0; s < T_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * EPI_WARPS); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();      // before tensor memory is taken: see launch_pdl
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();      // the peer's barriers exist before anything is signalled there
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto give_up = [&](int code) {
    if (lane == 0 && !*abort_flag) { *abort_flag = 1; atomicExch(&g_status, code); }
  };

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs) {
      int mt, ct;
      tile_of(p, tile, columns, mt, ct);
      const bool wide = ct < p.n_wide;
      const int m0 = mt * 2 * BM + (int)rank * BM, cols = wide ? 128 : 64, n0 = first_column(ct) + (int)rank * cols;
      for (int kb = 0; kb < kbs; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1u, abort_flag)) { give_up(ST_TIMEOUT_PRODUCER); ok = false; break; }
        const uint32_t sa = smem_u32(smem + stage * T_STAGE), sb = sa + STAGE_A_BYTES, bar = map_to_cta(&full[stage], 0);
        const int k0 = kb * BK;
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(&full[stage], (uint32_t)(2 * (STAGE_A_BYTES + cols * BK * 2)));
          if (A_MN) {
            tma_load_2d<true>(sa, &map_a, bar, m0, k0);
            tma_load_2d<true>(sa + 8192, &map_a, bar, m0 + 64, k0);
          } else {
            tma_load_2d<true>(sa, &map_a, bar, k0, m0);
          }
          if (B_MN) {
            tma_load_2d<true>(sb, &map_b, bar, n0, k0);
            if (wide) tma_load_2d<true>(sb + 8192, &map_b, bar, n0 + 64, k0);
          } else {
            tma_load_2d<true>(sb, wide ? &map_b : &map_b_narrow, bar, k0, n0);
          }
        }
        __syncwarp();
        if (++stage == T_STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc_wide = instruction<T, A_MN, B_MN>(2 * BM, BN), idesc_narrow = instruction<T, A_MN, B_MN>(2 * BM, BN / 2);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs, ++it) {
        int mt, ct;
        tile_of(p, tile, columns, mt, ct);
        const uint32_t idesc = ct < p.n_wide ? idesc_wide : idesc_narrow;
        const int buf = it & 1;
        if (!mbar_wait_warp(&acc_empty[buf], ((uint32_t)(it >> 1) & 1u) ^ 1u, abort_flag)) { give_up(ST_TIMEOUT_MMA); break; }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(buf * BN);
        for (int kb = 0; kb < kbs; ++kb) {
          if (!mbar_wait_warp(&full[stage], phase, abort_flag)) { give_up(ST_TIMEOUT_MMA); ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * T_STAGE);
          const uint64_t a = operand_desc<A_MN>(sa), b = operand_desc<B_MN>(sa + STAGE_A_BYTES);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) tc_mma<true>(d, a + kk * kStep<A_MN>, b + kk * kStep<B_MN>, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
            tc_commit<true>(&empty[stage]);
          }
          __syncwarp();
          if (++stage == T_STAGES) { stage = 0; phase ^= 1u; }
        }
        if (ok && elect_one()) tc_commit<true>(&acc_full[buf]);
        __syncwarp();
      }
    }
  } else {
    const int quad = warp & 3, chalf = (warp - 2) >> 2, et = (int)threadIdx.x - 64;
    uint32_t* R = reinterpret_cast<uint32_t*>(epi) + (warp - 2) * 512;
    float* bias = reinterpret_cast<float*>(epi + EPI_WARPS * 2048);
    const uint32_t acc_empty_leader[2] = {map_to_cta(&acc_empty[0], 0), map_to_cta(&acc_empty[1], 0)};
    bool fine = true;      // false: a wait gave up; the barriers below are still kept
    int it = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++it) {
      int mt, ct;
      tile_of(p, tile, columns, mt, ct);
      const int n0 = first_column(ct), cols = ct < p.n_wide ? BN : BN / 2, buf = it & 1;
      const int64_t row0 = (int64_t)mt * 2 * BM + (int)rank * BM + quad * 32;
      const int cb0 = cols / 2 * chalf, cb1 = cb0 + cols / 2;
      bias[et] = p.e.bias != nullptr && et < cols && n0 + et < p.s.C ? to_f32(reinterpret_cast<const T*>(p.e.bias)[n0 + et]) : 0.f;
      uint4 res[4];
      if (p.e.residual != nullptr) fetch_tile<T>((const T*)p.e.residual, row0, p.s.R, p.e.ld_res, n0 + cb0, p.s.C, lane, res);
      epi_bar_sync();
      if (fine && !mbar_wait(&acc_full[buf], (uint32_t)(it >> 1) & 1u, abort_flag)) {
        if (!*abort_flag) { *abort_flag = 1; atomicExch(&g_status, ST_TIMEOUT_EPILOGUE); }
        fine = false;
      }
      fine = __all_sync(0xffffffffu, fine);
      tc_fence_after();
      const uint32_t t_lane = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN);
      if (fine) {
#pragma unroll 1
        for (int cb = cb0; cb < cb1; cb += 32) {
          uint32_t acc[32];
          tc_ld32(t_lane + (uint32_t)cb, acc);
          const uint4 now[4] = {res[0], res[1], res[2], res[3]};
          if (p.e.residual != nullptr && cb + 32 < cb1)
            fetch_tile<T>((const T*)p.e.residual, row0, p.s.R, p.e.ld_res, n0 + cb + 32, p.s.C, lane, res);
          tile_block<T>(p, acc, bias + cb, R, row0, n0 + cb, lane, now);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty_leader[buf]);
      epi_bar_sync();      // everyone is done with the bias before the next tile's is staged
    }
  }
  // both CTAs are done with each other's barriers and tensor memory before either leaves
  tc_fence_before();
  __syncthreads();
  tc_settle(abort_flag);
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

// ------------------------------------------------------------------ slices
constexpr int S_EPI_WARPS = 8, S_THREADS = 64 + 32 * S_EPI_WARPS, S_STAGES_MAX = 12;
constexpr int S_PIPE_ONE = 196608, S_PIPE_TWO = 98304;                    // one CTA per SM, or two
constexpr int s_smem(int pipe) { return 1024 + pipe + 512; }

struct SliceParams {
  Shape s;
  Epilogue e;
  int tn, tiles_c, split;      // result rows of a tile (a multiple of 16 up to 256), column tiles, CTAs (or pairs) that share K
  int stages, stage_bytes, tmem_cols;
};

__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// the residual of 16 rows of the lane's column
template <typename T>
__device__ __forceinline__ void slice_residual(const SliceParams& p, int row0, int rows, int64_t col, T (&r)[16]) {
  const T* res = (const T*)p.e.residual;
  if (res == nullptr || col >= p.s.C) return;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < rows) r[j] = res[(int64_t)(row0 + j) * p.e.ld_res + col];
}
// 16 rows of results of the lane's column
template <typename T>
__device__ __forceinline__ void slice_block(const SliceParams& p, float (&v)[16], const T (&r)[16], float bias, int row0, int rows, int64_t col) {
  T *pre = (T*)p.e.pre, *out = (T*)p.e.out;
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] += bias;
  if (pre != nullptr) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < rows) pre[(int64_t)(row0 + j) * p.s.C + col] = from_f32<T>(v[j]);
  }
  by_act(p.e.act, [&](auto a) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = act_of<decltype(a)::value>(v[j]);
  });
  if (p.e.residual != nullptr) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] += to_f32(r[j]);
  }
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < rows) out[(int64_t)(row0 + j) * p.s.C + col] = from_f32<T>(v[j]);
}

// C_MN: the operand that gives the result's columns (B of the product) is MN-major; R_MN: the one that gives its rows (A).  PAIR: two CTAs
// share a tile of 256 columns, each loading half of the rows' operand; else a CTA has a tile of 128 columns of its own.
template <typename T, bool C_MN, bool R_MN, bool PAIR>
__global__ void __launch_bounds__(S_THREADS)
linear_slices_kernel(const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_r, const SliceParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[S_STAGES_MAX], empty[S_STAGES_MAX], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  constexpr int CTAS = PAIR ? 2 : 1;
  uint8_t* smem = align_shared(smem_raw);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const bool clustered = CTAS * p.split > 1;
  const int crank = clustered ? (int)cluster_ctarank() : 0, half = PAIR ? crank & 1 : 0, slice = PAIR ? crank >> 1 : crank;
  const uint32_t leader = (uint32_t)(PAIR ? crank & ~1 : crank);
  const int tile = (int)blockIdx.x / (CTAS * p.split), tc = tile % p.tiles_c, tr = tile / p.tiles_c;
  const int c0 = (tc * CTAS + half) * BM, r0 = tr * p.tn, rh = p.tn / CTAS;
  const int kbs = (p.s.K + BK - 1) / BK;
  const int kb_lo = (int)((int64_t)kbs * slice / p.split), kb_hi = (int)((int64_t)kbs * (slice + 1) / p.split);

  if (warp == 0 && elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_c)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_r)) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(&acc_full, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();      // before tensor memory is taken: see launch_pdl
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(p.tmem_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(p.tmem_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();      // the peer's barriers exist before anything is signalled there
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* flag = &abort_flag;
  auto give_up = [&](int code) {
    if (lane == 0 && !*flag) { *flag = 1; atomicExch(&g_status, code); }
  };
  float* part = reinterpret_cast<float*>(smem);      // [row][column] partial sums, over the drained stages
  const int quad = warp & 3, row_half = (warp - 2) >> 2;      // epilogue: 32 columns, and every other block of 16 rows
  const int64_t col = (int64_t)c0 + quad * 32 + lane;
  const uint32_t t_lane = tmem + ((uint32_t)(quad * 32) << 16);
  // the epilogue's blocks of 16 rows, dealt to the slices and their two groups of warps in turn
  const int end = min(p.s.R - r0, p.tn), first_row = 16 * (2 * slice + row_half), row_step = 32 * p.split;
  float bias = 0.f;
  T res[16];
  bool ok = true;

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb_lo; kb < kb_hi; ++kb) {
      if (!mbar_wait_warp(&empty[stage], phase ^ 1u, flag)) { give_up(ST_TIMEOUT_PRODUCER); break; }
      const uint32_t sc = smem_u32(smem + stage * p.stage_bytes), sr = sc + STAGE_A_BYTES, bar = PAIR ? map_to_cta(&full[stage], leader) : smem_u32(&full[stage]);
      const int k0 = kb * BK, rr = r0 + half * rh;
      if (elect_one()) {
        if (half == 0) mbar_expect_tx(&full[stage], (uint32_t)(CTAS * (STAGE_A_BYTES + rh * BK * 2)));
        if (C_MN) {
          tma_load_2d<PAIR>(sc, &map_c, bar, c0, k0);
          tma_load_2d<PAIR>(sc + 8192, &map_c, bar, c0 + 64, k0);
        } else {
          tma_load_2d<PAIR>(sc, &map_c, bar, k0, c0);
        }
        if (R_MN) {
          for (int j = 0; j < rh; j += 64) tma_load_2d<PAIR>(sr + (uint32_t)(j * 128), &map_r, bar, rr + j, k0);
        } else {
          tma_load_2d<PAIR>(sr, &map_r, bar, k0, rr);
        }
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    if (half == 0) {
      const uint32_t idesc = instruction<T, C_MN, R_MN>(CTAS * BM, p.tn);
      int stage = 0;
      uint32_t phase = 0;
      bool fine = true;
      for (int kb = kb_lo; kb < kb_hi; ++kb) {
        if (!mbar_wait_warp(&full[stage], phase, flag)) { give_up(ST_TIMEOUT_MMA); fine = false; break; }
        tc_fence_after();
        const uint32_t sc = smem_u32(smem + stage * p.stage_bytes);
        const uint64_t a = operand_desc<C_MN>(sc), b = operand_desc<R_MN>(sc + STAGE_A_BYTES);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) tc_mma<PAIR>(tmem, a + kk * kStep<C_MN>, b + kk * kStep<R_MN>, idesc, (kb > kb_lo || kk > 0) ? 1u : 0u);
          tc_commit<PAIR>(&empty[stage], leader);
        }
        __syncwarp();
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
      if (fine && elect_one()) tc_commit<PAIR>(&acc_full, leader);
      __syncwarp();
    }
  } else {
    if (p.e.bias != nullptr && col < p.s.C) bias = to_f32(reinterpret_cast<const T*>(p.e.bias)[col]);
    slice_residual<T>(p, r0 + first_row, end - first_row, col, res);      // (on its way during the main loop)
    ok = mbar_wait(&acc_full, 0, flag);
    if (!ok && !*flag) { *flag = 1; atomicExch(&g_status, ST_TIMEOUT_EPILOGUE); }
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    if (ok && p.split > 1) {
      // the stages are drained (the accumulators are complete): they hold the partial sums now
#pragma unroll 1
      for (int j0 = 16 * row_half; j0 < p.tn; j0 += 32) {
        uint32_t v[16];
        tc_ld16(t_lane + (uint32_t)j0, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(j0 + j) * BM + quad * 32 + lane] = __uint_as_float(v[j]);
      }
    }
  }
  // every CTA of the cluster has its partial sums in place (or has given up: the status says so)
  if (p.split > 1) cluster_sync_all();
  if (warp >= 2 && ok) {
    for (int j0 = first_row; j0 < end; j0 += row_step) {
      T now[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) now[j] = res[j];
      if (j0 + row_step < end) slice_residual<T>(p, r0 + j0 + row_step, end - j0 - row_step, col, res);
      float v[16];
      if (p.split == 1) {
        uint32_t u[16];
        tc_ld16(t_lane + (uint32_t)j0, u);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(u[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = 0.f;
        for (int s = 0; s < p.split; ++s) {      // rank 0, 1, ...: the same order on every run
          const uint32_t base = map_to_cta(part + j0 * BM + quad * 32 + lane, (uint32_t)(CTAS * s + half));
          float f[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[j]) : "r"(base + (uint32_t)(j * BM * 4)));
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] += f[j];
        }
      }
      if (col < p.s.C) slice_block<T>(p, v, now, bias, r0 + j0, end - j0, col);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_settle(flag);
  if (clustered) cluster_sync_all();      // nobody leaves while a peer may still read its partial sums or use its barriers
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
  }
}

// ------------------------------------------------------------------ dpre and the bias gradient
// dpre = dy act'(pre) and the column sums of dpre, in one pass.  A thread has eight columns (128-bit accesses) of every eighth row of the
// block's rows; sums per thread, per block in a fixed order, then over the blocks by a small launch.
constexpr int D_ROWS = 8, D_COLS = 256, D_BLOCKS = 4;      // blocks per SM
template <typename T>
__global__ void __launch_bounds__(256, D_BLOCKS)
linear_dpre_kernel(const T* __restrict__ dy, int64_t ld_dy, const T* __restrict__ pre, T* __restrict__ dpre, float* __restrict__ part, T* __restrict__ dbias,
                   int rows, int n, int per, int act) {
  __shared__ float s_sum[D_ROWS][D_COLS];
  pdl_wait();
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int c = (int)blockIdx.x * D_COLS + 8 * cl;
  const int first = (int)blockIdx.y * per, last = min(first + per, rows);
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  if (c < n) {
    by_act(act, [&](auto a) {
      constexpr int ACT = decltype(a)::value;
#pragma unroll 4
      for (int r = first + rl; r < last; r += D_ROWS) {
        float g[8], x[8];
        octet_to_f32(ld_octet(dy + r * ld_dy + c), g);
        if (ACT != HYC_ACT_NONE) {
          octet_to_f32(ld_octet(pre + (int64_t)r * n + c), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] *= slope_of<ACT>(x[e]);
          st_octet(dpre + (int64_t)r * n + c, g);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += g[e];
      }
    });
  }
  if (part == nullptr && dbias == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) s_sum[rl][8 * cl + e] = sum[e];
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int r = 0; r < D_ROWS; ++r) total += s_sum[r][threadIdx.x];
  const int at = (int)blockIdx.x * D_COLS + (int)threadIdx.x;
  if (at < n) {
    if (dbias != nullptr) dbias[at] = from_f32<T>(total);      // (all rows are this block's)
    else part[(int64_t)blockIdx.y * n + at] = total;
  }
}
template <typename T>
__global__ void __launch_bounds__(1024)
linear_dbias_kernel(const float* __restrict__ part, int parts, int n, T* __restrict__ dbias) {
  __shared__ float s_sum[32][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < n)
    for (int r = warp; r < parts; r += 32) sum += part[(int64_t)r * n + c];
  s_sum[warp][lane] = sum;
  __syncthreads();
  sum = s_sum[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int at = (int)blockIdx.x * 32 + warp;
  if (lane == 0 && at < n) dbias[at] = from_f32<T>(sum);
}

// ------------------------------------------------------------------ host side
static bool operand_map(CUtensorMap* m, const void* ptr, int type, bool mn, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)(mn ? rows : k), (cuuint64_t)(mn ? k : rows)};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64u, mn ? 64u : (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1u, 1u};
  return enc(m, type == HYC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K, typename... A>
static int launch_cluster(K kern, unsigned blocks, unsigned threads, unsigned cluster, int smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) {
    hyc_set_last_cuda_error((int)cudaGetLastError());
    return HYC_ERR_LAUNCH;
  }
  return HYC_OK;
}

// ---- which kernel, by estimated cycles.  The constants were fitted to the two kernels in all their forms at fourteen sizes (1 to 1500 rows,
// 1024 to 11008 deep and wide, cold, us):
//              tiles   slices: best            1 / 2 / 4 CTAs share K
//   1 x 4096 x 11008    33.6    20.5      21.3 / 20.9 / 26.9           256 x 4096 x 4096    20.3    16.8     33.2 / 23.8 / 34.1 (pairs)
//   8 x 11008 x 4096    41.2    21.0      34.9 / 23.3 / 21.1           333 x 11008 x 4096   42.6    30.8     47.1 / 30.8 / 60.9 (pairs)
//   64 x 4096 x 11008   27.8    22.7      23.5 / 22.7 / 30.1           512 x 4096 x 4096    21.0    22.7     34.2 / 24.9 / 49.7 (pairs)
//   128 x 4096 x 4096   20.3    14.2      22.4 / 17.0 / 16.3           1500 x 4096 x 512    19.3    16.0     33.2 / 23.3 / 19.0 (pairs)
// What the rule picks is 5 % from the best form on average.  (Clusters of 8 were never the best: only 15 of them are resident.)
struct TilePlan { int n_wide, n_tiles; float cost; };
static TilePlan plan_tiles(const Shape& s) {
  const int tiles_m = (s.R + 2 * BM - 1) / (2 * BM), halves = (s.C + BN / 2 - 1) / (BN / 2), pairs = num_sms() / 2;
  const float block = 547.f * (float)((s.K + BK - 1) / BK), half = 0.71f;
  TilePlan best = {0, halves, 1e30f};
  const int fewest = (int64_t)tiles_m * (halves / 2) > 16ll * pairs ? halves / 2 : 0;      // (of many rounds the last one does not matter)
  for (int w = halves / 2; w >= fewest; --w) {
    const int64_t wide = (int64_t)tiles_m * w, narrow = (int64_t)tiles_m * (halves - 2 * w);
    const int64_t rounds = wide / pairs, rest = wide % pairs, behind = narrow - (pairs - rest);      // wide tiles are dealt first
    float rest_cost = rounds + half * (float)((narrow + pairs - 1) / pairs);
    if (rest > 0) {
      const float c = rounds + 1 + half * (float)(behind > 0 ? (behind + pairs - 1) / pairs : 0);
      if (c > rest_cost) rest_cost = c;
    }
    const float cost = rest_cost * block + 14000.f;
    if (cost < best.cost * 0.98f) best = {w, halves - w, cost};
  }
  const float stream = 2.f * (float)s.C * (float)s.K / 1500.f;      // few tiles: the loads of their pairs alone do not fill the memory's pipe
  if (stream > best.cost) best.cost = stream;
  return best;
}
// two CTAs per SM: the partial sums, 512 bytes per row, have to fit in half of the shared memory
static bool slice_two(int tn, bool pair) { return tn <= (pair ? 128 : 64); }
// clusters of 4 CTAs do not reach every SM (33 of them are resident on a B200, one CTA per SM)
static int slice_clusters(int ctas) { return ctas <= 2 ? num_sms() / ctas : num_sms() * 33 / 148; }
struct SlicePlan { int tn, split; bool pair; float cost; };
static SlicePlan plan_slices(const Shape& s, bool r_mn) {
  const int kbs = (s.K + BK - 1) / BK, base = (s.R + 255) / 256;
  SlicePlan best = {0, 0, false, 1e30f};
  for (int form = 0; form < 4; ++form) {
    const bool pair = (form & 1) != 0;
    const int ctas = pair ? 2 : 1, tiles_c = (s.C + ctas * BM - 1) / (ctas * BM), row_tiles = base << (form >> 1);
    int tn = ((s.R + row_tiles - 1) / row_tiles + 15) / 16 * 16;
    if (r_mn) tn = tn <= 64 && !pair ? 64 : tn <= 128 ? 128 : 256;
    const int64_t tiles_r = (s.R + tn - 1) / tn, clusters = tiles_c * tiles_r;
    for (int split = 1; split * ctas <= 4; split *= 2) {
      if (split > 1 && kbs < 4 * split) break;
      const int64_t at_once = (int64_t)slice_clusters(split * ctas) * (slice_two(tn, pair) ? 2 : 1), waves = (clusters + at_once - 1) / at_once;
      const int64_t running = (clusters < at_once ? clusters : at_once) * split * ctas;
      const float per_sm = running > num_sms() ? (float)running / (float)num_sms() : 1.f;
      // a k-block: the tensor pipe, operands from L2 at 64 bytes per cycle and SM, all SMs' columns once from HBM
      const float operands = (float)(STAGE_A_BYTES + tn / ctas * BK * 2) / 64.f, hbm = (float)STAGE_A_BYTES * (float)running / 3200.f / (float)tiles_r;
      float block = (2.f * tn > operands ? 2.f * tn : operands) * per_sm;
      if (hbm > block) block = hbm;
      const float cost = 9300.f + (float)waves * ((float)((kbs + split - 1) / split) * block + 50.f * (float)tn / (float)split * per_sm + 5300.f) +
                         (split > 1 ? 3000.f + 22.f * (float)tn : 0.f);
      if (cost < best.cost) best = {tn, split, pair, cost};
    }
  }
  return best;
}

template <typename T, bool A_MN, bool B_MN, bool PAIR>
static int launch_slices(const hyc_linear* a, const Shape& s, const Epilogue& e, const SlicePlan& sp, cudaStream_t st) {
  constexpr auto kern = linear_slices_kernel<T, B_MN, A_MN, PAIR>;
  constexpr int CTAS = PAIR ? 2 : 1;
  const int rc = more_shared_memory<kern>(s_smem(S_PIPE_ONE));
  if (rc != HYC_OK) return rc;
  SliceParams p;
  p.s = s; p.e = e; p.tn = sp.tn; p.split = sp.split;
  p.tiles_c = (s.C + CTAS * BM - 1) / (CTAS * BM);
  const int64_t ctas = (int64_t)CTAS * p.split * p.tiles_c * ((s.R + p.tn - 1) / p.tn);
  if (ctas > 0x7fffffff) return HYC_ERR_SHAPE;
  const int pipe = ctas > num_sms() && slice_two(p.tn, PAIR) ? S_PIPE_TWO : S_PIPE_ONE;
  p.stage_bytes = STAGE_A_BYTES + p.tn / CTAS * BK * 2;
  p.stages = pipe / p.stage_bytes < S_STAGES_MAX ? pipe / p.stage_bytes : S_STAGES_MAX;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.tn) p.tmem_cols *= 2;
  CUtensorMap mc, mr;
  if (!operand_map(&mc, a->b, a->type, B_MN, s.C, s.K, a->ld_b, BM) || !operand_map(&mr, a->a, a->type, A_MN, s.R, s.K, a->ld_a, p.tn / CTAS))
    return HYC_ERR_UNSUPPORTED;
  return launch_cluster(kern, (unsigned)ctas, S_THREADS, (unsigned)(CTAS * p.split), s_smem(pipe), st, mc, mr, p);
}

template <typename T, bool A_MN, bool B_MN>
static int launch_product(const hyc_linear* a, cudaStream_t st) {
  const Shape s = {(int)a->rows, a->cols, a->depth};
  const Epilogue e = {a->bias, a->residual, a->pre, a->out, a->ld_res, a->act};
  const TilePlan tp = plan_tiles(s);
  const SlicePlan sp = plan_slices(s, A_MN);
  if (sp.cost < tp.cost) return sp.pair ? launch_slices<T, A_MN, B_MN, true>(a, s, e, sp, st) : launch_slices<T, A_MN, B_MN, false>(a, s, e, sp, st);
  constexpr auto kern = linear_tiles_kernel<T, A_MN, B_MN>;
  const int rc = more_shared_memory<kern>(T_SMEM);
  if (rc != HYC_OK) return rc;
  TileParams p;
  p.s = s; p.e = e;
  p.tiles_m = (s.R + 2 * BM - 1) / (2 * BM);
  p.n_wide = tp.n_wide; p.n_tiles = tp.n_tiles;
  p.group = tp.n_wide == 0 || tp.n_wide == tp.n_tiles ? 8 : p.tiles_m;      // (of mixed widths the wide ones come first)
  if (p.group > p.tiles_m) p.group = p.tiles_m;
  const int64_t tiles = (int64_t)p.tiles_m * p.n_tiles;
  if (tiles > 0x3fffffff) return HYC_ERR_SHAPE;
  CUtensorMap ma, mb, mn;
  if (!operand_map(&ma, a->a, a->type, A_MN, s.R, s.K, a->ld_a, BM) || !operand_map(&mb, a->b, a->type, B_MN, s.C, s.K, a->ld_b, 128) ||
      !operand_map(&mn, a->b, a->type, B_MN, s.C, s.K, a->ld_b, 64))
    return HYC_ERR_UNSUPPORTED;
  const int pairs = num_sms() / 2;
  return launch_cluster(kern, (unsigned)(2 * (tiles < pairs ? tiles : pairs)), THREADS, 2, T_SMEM, st, ma, mb, mn, p);
}

constexpr int kDpreParts = 64;      // most row ranges whose column sums are kept apart
static int dpre_rows(int64_t rows, int n) {
  const int64_t blocks = (n + D_COLS - 1) / D_COLS;
  int64_t parts = (int64_t)num_sms() * D_BLOCKS / blocks;      // one wave
  parts = parts > kDpreParts ? kDpreParts : parts < 1 ? 1 : parts;
  int64_t per = (rows + parts - 1) / parts;
  if (rows <= 64) per = 64;      // eight rows per thread take less than the launch that adds up blocks
  return (int)((per + D_ROWS - 1) / D_ROWS * D_ROWS);
}

template <typename T>
static int launch_dpre(const void* dy, int64_t ld_dy, const void* pre, void* dpre, void* dbias, int64_t rows, int n, int act, float* part, cudaStream_t st) {
  int parts = 0;
  if (rows > 0) {
    const int per = dpre_rows(rows, n);
    parts = (int)((rows + per - 1) / per);
    launch_pdl(linear_dpre_kernel<T>, dim3((unsigned)((n + D_COLS - 1) / D_COLS), (unsigned)parts), dim3(256), 0, st, (const T*)dy, ld_dy, (const T*)pre, (T*)dpre,
               dbias != nullptr && parts > 1 ? part : nullptr, dbias != nullptr && parts == 1 ? (T*)dbias : (T*)nullptr, (int)rows, n, per, act);
    HYC_CHECK_LAUNCH();
  }
  if (dbias != nullptr && parts != 1) {
    launch_pdl(linear_dbias_kernel<T>, dim3((unsigned)((n + 31) / 32)), dim3(1024), 0, st, (const float*)part, parts, n, (T*)dbias);
    HYC_CHECK_LAUNCH();
  }
  return HYC_OK;
}

}  // namespace lin
}  // namespace hyc

using namespace hyc;
using namespace hyc::lin;

extern "C" HYC_API int hyc_linear_act_tcgen05(const hyc_linear* a, void* stream) {
  if (a == nullptr) return HYC_ERR_NULL;
  if ((a->type != HYC_BF16 && a->type != HYC_F16) || a->act < HYC_ACT_NONE || a->act > HYC_ACT_SILU || (a->a_mn && !a->b_mn)) return HYC_ERR_UNSUPPORTED;
  const int64_t rows = a->rows;
  if (rows < 0 || rows > 0x3fffffffll || a->cols < 8 || a->cols > (1 << 24) || a->cols % 8 != 0 || a->depth < 1 || a->depth > 0x3fffffff || (!a->a_mn && a->depth % 8 != 0) ||
      (a->a_mn && rows % 8 != 0))
    return HYC_ERR_SHAPE;
  if (a->ld_a < (a->a_mn ? rows : a->depth) || a->ld_b < (a->b_mn ? a->cols : a->depth) || (a->residual != nullptr && a->ld_res < a->cols)) return HYC_ERR_SHAPE;
  if (rows == 0) return HYC_OK;
  if (a->a == nullptr || a->b == nullptr || a->out == nullptr) return HYC_ERR_NULL;
  if (a->ld_a % 8 != 0 || a->ld_b % 8 != 0 || !aligned(a->a, 16) || !aligned(a->b, 16) || !aligned(a->out, 16) || !aligned(a->pre, 16) || !aligned(a->bias, 2) ||
      !aligned(a->residual, 16) || (a->residual != nullptr && a->ld_res % 8 != 0))
    return HYC_ERR_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  auto form = [&](auto elem) -> int {
    using T = decltype(elem);
    if (a->a_mn) return launch_product<T, true, true>(a, st);
    if (a->b_mn) return launch_product<T, false, true>(a, st);
    return launch_product<T, false, false>(a, st);
  };
  return a->type == HYC_BF16 ? form(__nv_bfloat16()) : form(__half());
}

extern "C" HYC_API size_t hyc_linear_act_dpre_workspace_bytes(int cols) { return cols < 1 ? 0 : (size_t)cols * kDpreParts * sizeof(float); }

extern "C" HYC_API int hyc_linear_act_dpre(const void* dy, int64_t ld_dy, const void* pre, void* dpre, void* dbias, int64_t rows, int cols, int type, int act,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  if ((type != HYC_BF16 && type != HYC_F16) || act < HYC_ACT_NONE || act > HYC_ACT_SILU) return HYC_ERR_UNSUPPORTED;
  if (rows < 0 || rows > 0x3fffffffll || cols < 8 || cols > (1 << 24) || cols % 8 != 0 || ld_dy < 0) return HYC_ERR_SHAPE;
  if (rows > 0 && (dy == nullptr || (act != HYC_ACT_NONE && (pre == nullptr || dpre == nullptr)))) return HYC_ERR_NULL;
  if (ld_dy % 8 != 0 || !aligned(dy, 16) || !aligned(pre, 16) || !aligned(dpre, 16) || !aligned(dbias, 2)) return HYC_ERR_ALIGN;
  if (dbias != nullptr && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < hyc_linear_act_dpre_workspace_bytes(cols))) return HYC_ERR_WORKSPACE;
  if (type == HYC_BF16) return launch_dpre<__nv_bfloat16>(dy, ld_dy, pre, dpre, dbias, rows, cols, act, (float*)workspace, (cudaStream_t)stream);
  return launch_dpre<__half>(dy, ld_dy, pre, dpre, dbias, rows, cols, act, (float*)workspace, (cudaStream_t)stream);
}

extern "C" HYC_API int hyc_linear_status(int* host_status) {
  if (host_status == nullptr) return HYC_ERR_NULL;
  cudaError_t e = cudaDeviceSynchronize();      // (a copy alone would not wait for streams that do not wait for the default one)
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(host_status, g_status, sizeof(int));
  if (e != cudaSuccess) { hyc_set_last_cuda_error((int)e); cudaGetLastError(); return HYC_ERR_LAUNCH; }
  return HYC_OK;
}
