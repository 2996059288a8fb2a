// Differential attention, backward: the row statistics, the gradient of lam, and the FP32-FMA kernels that take any type, stride and
// head dim up to 128 (fp32 inputs, and 16-bit ones that the tensor-core kernels of diff_bwd_tc.cu do not take).
//
// With G = g V^T (g the gradient of out, shared by both maps) and D_m = g . (P_m V), row by row,
//     dS1 = P1 (G - D1),  dS2 = -lam P2 (G - D2)          dQ_m = scale dS_m K_m,  dK_m = scale dS_m^T Q_m
//     dV = (P1 - lam P2)^T g                              dlam = -sum of D2 over the head's rows
// P is recomputed from the scores and each row's log2 sum, P = 2^(S scale log2 e - LSE).  D2 = g . out2 with out2 = P2 V from the
// forward, and D1 = g . out + lam D2, since out = P1 V - lam P2 V.  Gradients of shared key heads are summed in the kernels that own
// them, in a fixed order: no atomics anywhere.
//
// The FMA kernels work on 32 x 32 tiles with 256 threads: a thread has one row and four columns of S1, S2 and G, then 16 columns of its
// row's gradients.  Eight threads of a warp share a row's operands and four rows share a column's (broadcasts), so a quarter of a
// load is issued for each multiply-add; they are bound by that.
#include <algorithm>

#include "diff.cuh"

namespace elsa {

namespace {

constexpr int kThreads = 256, kRows = 32, kCols = 32, kDim = 128, kPitch = kDim + 4, kTilePitch = kCols + 1;

// stats: [B * heads][-LSE1, -LSE2, -D1, -D2][n_pad]; padding rows hold -inf, -inf, 0, 0.  A warp per row.
template <typename T>
__global__ void __launch_bounds__(256)
diff_stats_kernel(const DiffParams p, float* __restrict__ stats, int n_pad) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t bh = i / n_pad;
  const int r = static_cast<int>(i - bh * n_pad);
  if (bh >= static_cast<int64_t>(p.batch) * p.heads) return;
  float* dst = stats + bh * 4 * n_pad + r;
  if (r >= p.nq) {
    if (lane == 0) { dst[0] = -CUDART_INF_F; dst[n_pad] = -CUDART_INF_F; dst[2 * n_pad] = 0.f; dst[3 * n_pad] = 0.f; }
    return;
  }
  const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh - static_cast<int64_t>(b) * p.heads);
  const T* out = static_cast<const T*>(p.out) + b * p.os.b + h * p.os.h + r * p.os.r;
  const T* g = static_cast<const T*>(p.dout) + b * p.gs.b + h * p.gs.h + r * p.gs.r;
  const T* out2 = static_cast<const T*>(p.out2) + (bh * p.nq + r) * p.v_dim;
  float d = 0.f, d2 = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int col = lane + 32 * e;
    if (col < p.v_dim) {
      const float x = to_f32<T>(g[col]);
      d = fmaf(x, to_f32<T>(out[col]), d);
      d2 = fmaf(x, to_f32<T>(out2[col]), d2);
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    d += __shfl_xor_sync(0xffffffffu, d, x);
    d2 += __shfl_xor_sync(0xffffffffu, d2, x);
  }
  if (lane == 0) {
    const int64_t ro = bh * p.nq + r, maps = static_cast<int64_t>(p.batch) * p.heads * p.nq;
    const float l1 = p.lse[ro], l2 = p.lse[maps + ro];
    dst[0] = l1 == -CUDART_INF_F ? l1 : -l1;              // (a row without keys: P = 2^-inf = 0)
    dst[n_pad] = l2 == -CUDART_INF_F ? l2 : -l2;
    dst[2 * n_pad] = -(d + diff_lam(p, h) * d2);
    dst[3 * n_pad] = -d2;
  }
}

// dlam[h] = sum of -D2 over the batch and the rows (padding is 0): a block per head, or one for all heads where lam is one value
__global__ void __launch_bounds__(512)
diff_dlam_kernel(const float* __restrict__ stats, void* dlam, int dlam_dtype, int batch, int heads, int n_pad, int all) {
  __shared__ float part[16];
  const int h0 = all ? 0 : blockIdx.x, h1 = all ? heads : h0 + 1;
  float sum = 0.f;
  for (int b = 0; b < batch; ++b)
    for (int h = h0; h < h1; ++h) {
      const float* src = stats + ((static_cast<int64_t>(b) * heads + h) * 4 + 3) * n_pad;
      for (int r = threadIdx.x; r < n_pad; r += 512) sum += src[r];
    }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.f;
    for (int w = 0; w < 16; ++w) sum += part[w];
    if (dlam_dtype == ELSA_F32) static_cast<float*>(dlam)[h0] = sum;
    else if (dlam_dtype == ELSA_F16) static_cast<__half*>(dlam)[h0] = from_f32<__half>(sum);
    else static_cast<__nv_bfloat16*>(dlam)[h0] = from_f32<__nv_bfloat16>(sum);
  }
}

// rows x0 .. x0 + 32 of a matrix into shared memory as fp32; rows from n on and columns from dim to the next multiple of 4 are zeros
template <typename T>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t stride, int x0, int n, int dim, int dim4) {
  for (int i = threadIdx.x; i < kRows * dim4; i += kThreads) {
    const int col = i % dim4, r = i / dim4;
    dst[r * kPitch + col] = x0 + r < n && col < dim ? to_f32<T>(src[(x0 + r) * stride + col]) : 0.f;
  }
}
// four dot products of one row of `a` with rows c, c + 8, c + 16, c + 24 of `b`
__device__ __forceinline__ void dots(float (&s)[4], const float* a, const float* b, int dim4) {
  for (int d = 0; d < dim4; d += 4) {
    const float4 x = *reinterpret_cast<const float4*>(a + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 y = *reinterpret_cast<const float4*>(b + 8 * e * kPitch + d);
      s[e] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[e]))));
    }
  }
}
// acc += w[0 .. 32) . tile, columns 4 c + 32 {0..3} of it (columns beyond the real ones hold what a tile before left: never stored)
__device__ __forceinline__ void accumulate(float (&acc)[16], const float* w, const float* tile, int c, int dim4) {
  for (int j = 0; j < 32; ++j) {
    const float x = w[j];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (32 * e >= dim4) continue;
      const float4 y = *reinterpret_cast<const float4*>(tile + j * kPitch + 4 * c + 32 * e);
      acc[4 * e] = fmaf(x, y.x, acc[4 * e]); acc[4 * e + 1] = fmaf(x, y.y, acc[4 * e + 1]);
      acc[4 * e + 2] = fmaf(x, y.z, acc[4 * e + 2]); acc[4 * e + 3] = fmaf(x, y.w, acc[4 * e + 3]);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store_row(T* dst, const float (&acc)[16], int c, int dim, float f) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int col = 4 * c + 32 * (e / 4) + e % 4;
    if (col < dim) dst[col] = from_f32<T>(acc[e] * f);
  }
}

// dQ1, dQ2 of 32 query rows of one head
template <typename T>
__global__ void __launch_bounds__(kThreads)
diff_dq_simt_kernel(const DiffParams p, const float* __restrict__ stats, int n_pad) {
  extern __shared__ __align__(16) float smem[];
  float* sq = smem;                                     // [map][query][dim]
  float* sg = sq + 2 * kRows * kPitch;                  // [query][value dim]
  float* sk = sg + kRows * kPitch;                      // [map][key][dim]
  float* sv = sk + 2 * kCols * kPitch;                  // [key][value dim]
  float* sd = sv + kCols * kPitch;                      // [map][query][key]
  const int h = blockIdx.y, b = blockIdx.z, g = h / (p.heads / p.kv_heads), q0 = (gridDim.x - 1 - blockIdx.x) * kRows;
  const int r = threadIdx.x / 8, c = threadIdx.x % 8, qi = q0 + r, shift = p.nk - p.nq;
  const int dim4 = (p.head_dim + 3) / 4 * 4, v4 = (p.v_dim + 3) / 4 * 4;
  for (int m = 0; m < 2; ++m)
    load_tile(sq + m * kRows * kPitch, static_cast<const T*>(p.q) + b * p.qs.b + (2 * h + m) * p.qs.h, p.qs.r, q0, p.nq, p.head_dim, dim4);
  load_tile(sg, static_cast<const T*>(p.dout) + b * p.gs.b + h * p.gs.h, p.gs.r, q0, p.nq, p.v_dim, v4);
  const float* st = stats + (static_cast<int64_t>(b) * p.heads + h) * 4 * n_pad + qi;      // (q0 + 31 < n_pad)
  const float nlse[2] = {st[0], st[n_pad]}, nd[2] = {st[2 * n_pad], st[3 * n_pad]};
  const float lam = diff_lam(p, h);
  float dq[2][16] = {};
  const int end = p.causal ? min(p.nk, min(q0 + kRows, p.nq) + shift) : p.nk;
  const int lim = p.causal ? min(p.nk - 1, qi + shift) : p.nk - 1;
  for (int k0 = 0; k0 < end; k0 += kCols) {
    __syncthreads();
    for (int m = 0; m < 2; ++m)
      load_tile(sk + m * kCols * kPitch, static_cast<const T*>(p.k) + b * p.ks.b + (2 * g + m) * p.ks.h, p.ks.r, k0, p.nk, p.head_dim, dim4);
    load_tile(sv, static_cast<const T*>(p.v) + b * p.vs.b + g * p.vs.h, p.vs.r, k0, p.nk, p.v_dim, v4);
    __syncthreads();
    float gv[4] = {};
    dots(gv, sg + r * kPitch, sv + c * kPitch, v4);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float s[4] = {};
      dots(s, sq + (m * kRows + r) * kPitch, sk + (m * kCols + c) * kPitch, dim4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = k0 + c + 8 * e <= lim ? exp2f(fmaf(s[e], p.scale_log2, nlse[m])) : 0.f;
        sd[(m * kRows + r) * kTilePitch + c + 8 * e] = x * (gv[e] + nd[m]) * (m ? -lam : 1.f);
      }
    }
    __syncwarp();                                       // (a row's weights come from eight lanes of one warp)
#pragma unroll
    for (int m = 0; m < 2; ++m) accumulate(dq[m], sd + (m * kRows + r) * kTilePitch, sk + m * kCols * kPitch, c, dim4);
  }
  if (qi < p.nq)
#pragma unroll
    for (int m = 0; m < 2; ++m)
      store_row(static_cast<T*>(p.dq) + b * p.dqs.b + (2 * h + m) * p.dqs.h + qi * p.dqs.r, dq[m], c, p.head_dim, p.scale);
}

// dK1, dK2, dV of 32 keys of one key head: over the query heads that share it, and their rows
template <typename T>
__global__ void __launch_bounds__(kThreads)
diff_dkv_simt_kernel(const DiffParams p, const float* __restrict__ stats, int n_pad) {
  extern __shared__ __align__(16) float smem[];
  float* sk = smem;                                     // [map][key][dim]
  float* sv = sk + 2 * kRows * kPitch;                  // [key][value dim]
  float* sq = sv + kRows * kPitch;                      // [map][query][dim]
  float* sg = sq + 2 * kCols * kPitch;                  // [query][value dim]
  float* sd = sg + kCols * kPitch;                      // [P1 - lam P2, dS1, dS2][key][query]
  const int g = blockIdx.y, b = blockIdx.z, group = p.heads / p.kv_heads, k0 = blockIdx.x * kRows;
  const int r = threadIdx.x / 8, c = threadIdx.x % 8, key = k0 + r, shift = p.nk - p.nq;
  const int dim4 = (p.head_dim + 3) / 4 * 4, v4 = (p.v_dim + 3) / 4 * 4;
  for (int m = 0; m < 2; ++m)
    load_tile(sk + m * kRows * kPitch, static_cast<const T*>(p.k) + b * p.ks.b + (2 * g + m) * p.ks.h, p.ks.r, k0, p.nk, p.head_dim, dim4);
  load_tile(sv, static_cast<const T*>(p.v) + b * p.vs.b + g * p.vs.h, p.vs.r, k0, p.nk, p.v_dim, v4);
  float dk[2][16] = {}, dv[16] = {};
  const int begin = p.causal ? max(0, k0 - shift) / kCols * kCols : 0;      // queries before it see none of these keys
  for (int h = g * group; h < (g + 1) * group; ++h) {
    const float lam = diff_lam(p, h);
    const float* st = stats + (static_cast<int64_t>(b) * p.heads + h) * 4 * n_pad;
    for (int q0 = begin; q0 < p.nq; q0 += kCols) {
      __syncthreads();
      for (int m = 0; m < 2; ++m)
        load_tile(sq + m * kCols * kPitch, static_cast<const T*>(p.q) + b * p.qs.b + (2 * h + m) * p.qs.h, p.qs.r, q0, p.nq, p.head_dim, dim4);
      load_tile(sg, static_cast<const T*>(p.dout) + b * p.gs.b + h * p.gs.h, p.gs.r, q0, p.nq, p.v_dim, v4);
      __syncthreads();
      float gv[4] = {}, s[2][4] = {};
      dots(gv, sv + r * kPitch, sg + c * kPitch, v4);
#pragma unroll
      for (int m = 0; m < 2; ++m) dots(s[m], sk + (m * kRows + r) * kPitch, sq + (m * kCols + c) * kPitch, dim4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int qi = q0 + c + 8 * e;                  // (below n_pad; rows from nq on have P = 0)
        const bool seen = key < p.nk && (!p.causal || key <= qi + shift);
        const float x1 = seen ? exp2f(fmaf(s[0][e], p.scale_log2, st[qi])) : 0.f;
        const float x2 = seen ? exp2f(fmaf(s[1][e], p.scale_log2, st[n_pad + qi])) : 0.f;
        float* at = sd + r * kTilePitch + c + 8 * e;
        at[0] = x1 - lam * x2;
        at[kRows * kTilePitch] = x1 * (gv[e] + st[2 * n_pad + qi]);
        at[2 * kRows * kTilePitch] = -lam * x2 * (gv[e] + st[3 * n_pad + qi]);
      }
      __syncwarp();
      accumulate(dv, sd + r * kTilePitch, sg, c, v4);
#pragma unroll
      for (int m = 0; m < 2; ++m) accumulate(dk[m], sd + ((1 + m) * kRows + r) * kTilePitch, sq + m * kCols * kPitch, c, dim4);
    }
  }
  if (key < p.nk) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
      store_row(static_cast<T*>(p.dk) + b * p.dks.b + (2 * g + m) * p.dks.h + key * p.dks.r, dk[m], c, p.head_dim, p.scale);
    store_row(static_cast<T*>(p.dv) + b * p.dvs.b + g * p.dvs.h + key * p.dvs.r, dv, c, p.v_dim, 1.f);
  }
}

template <typename T>
int simt_t(const DiffParams& p, const float* stats, cudaStream_t st) {
  const int n_pad = static_cast<int>(align_up(p.nq, 128));
  const int tiles = 6 * kRows * kPitch * 4;
  const int dq_smem = tiles + 2 * kRows * kTilePitch * 4, dkv_smem = tiles + 3 * kRows * kTilePitch * 4;
  int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&diff_dq_simt_kernel<T>), dq_smem);
  if (rc == ELSA_OK) rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&diff_dkv_simt_kernel<T>), dkv_smem);
  if (rc != ELSA_OK) return rc;
  const dim3 qgrid(static_cast<unsigned>(cdiv64(p.nq, kRows)), static_cast<unsigned>(p.heads), static_cast<unsigned>(p.batch));
  diff_dq_simt_kernel<T><<<qgrid, kThreads, dq_smem, st>>>(p, stats, n_pad);
  ELSA_LAUNCH_CHECK();
  if (p.nk > 0) {
    const dim3 kgrid(static_cast<unsigned>(cdiv64(p.nk, kRows)), static_cast<unsigned>(p.kv_heads), static_cast<unsigned>(p.batch));
    diff_dkv_simt_kernel<T><<<kgrid, kThreads, dkv_smem, st>>>(p, stats, n_pad);
    ELSA_LAUNCH_CHECK();
  }
  return ELSA_OK;
}

}  // namespace

int diff_stats(const DiffParams& p, float* stats, int dtype, cudaStream_t st) {
  const int n_pad = static_cast<int>(align_up(p.nq, 128));
  const int64_t blocks = static_cast<int64_t>(p.batch) * p.heads * n_pad / 8;
  if (blocks > 0x7fffffffll) return ELSA_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(blocks);
  if (dtype == ELSA_F32) diff_stats_kernel<float><<<grid, 256, 0, st>>>(p, stats, n_pad);
  else if (dtype == ELSA_F16) diff_stats_kernel<__half><<<grid, 256, 0, st>>>(p, stats, n_pad);
  else diff_stats_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p, stats, n_pad);
  ELSA_LAUNCH_CHECK();
  if (p.dlam) {
    diff_dlam_kernel<<<p.lam_stride == 0 ? 1 : p.heads, 512, 0, st>>>(stats, p.dlam, p.lam_dtype, p.batch, p.heads, n_pad, p.lam_stride == 0);
    ELSA_LAUNCH_CHECK();
  }
  return ELSA_OK;
}

int diff_bwd_simt(const DiffParams& p, const float* stats, int dtype, cudaStream_t st) {
  if (dtype == ELSA_F32) return simt_t<float>(p, stats, st);
  return dtype == ELSA_F16 ? simt_t<__half>(p, stats, st) : simt_t<__nv_bfloat16>(p, stats, st);
}

}  // namespace elsa
