// Differential attention, backward: the row statistics, the gradient of lam, and the kernels that take any type, stride and head dim
// up to 128 (fp32 inputs, and 16-bit ones that the kernels of diff_bwd_tc.cu do not take).
//
// With G = g V^T (g the gradient of out, shared by both maps) and D_m = g . (P_m V), row by row,
//     dS1 = P1 (G - D1),  dS2 = -lam P2 (G - D2)          dQ_m = scale dS_m K_m,  dK_m = scale dS_m^T Q_m
//     dV = (P1 - lam P2)^T g                              dlam = -sum over rows and keys of P2 G
// P is recomputed from the scores and each row's log2 sum, P = 2^(S scale log2 e - LSE).  D2 = g . out2 with out2 = P2 V from the
// forward, and D1 = g . out + lam D2, since out = P1 V - lam P2 V.  dlam is the sum of D2 too, of terms of either sign that may cancel to
// next to nothing, while the D2 of a 16-bit out2 is known to 2^-9 only: it is summed from P2 and G in fp32, as the dQ kernels have them.
// Gradients of shared key heads are summed in the kernels that own them, in a fixed order: no atomics anywhere.
//
// The kernels of any type work in fp32 on split tf32 operands (tf32.cuh): a block of eight warps owns 32 rows and streams 64 of the
// other side at a time, a warp has a 16 x 16 block of S1, S2 and G in its accumulators, turns them into dS1, dS2 (and P1 - lam P2)
// there, and uses them as they are as operands of the gradients' products; a row's four warps add up their sums at the end.
// They are bound by the latency of the splitting and of the products' chains, with 8 (dK, dV: 252 registers) or 16 (dQ) warps on an SM that
// issue in 0.27 and 0.43 of the cycles.  Where there are few tiles, up to four blocks share one, each with every team-th tile of the other
// side; their sums are added through distributed shared memory, in order.  At (1, 4 heads, 1000 tokens, 64 / 128, causal, fp32) dQ takes
// 92 us and dK, dV 143; with one block for each tile, whose longest decides, 125 and 162; eight blocks 105 and 220; FMAs on 32 x 32 tiles
// took 296 and 530 (five 16-byte shared-memory reads for 16 multiply-adds of a thread).
#include <cooperative_groups.h>

#include <algorithm>

#include "diff.cuh"
#include "tf32.cuh"

namespace elsa {

namespace {

constexpr int kThreads = 256, kOwn = kDiffAnyRows, kStream = 64, kValue = 128;   // rows a block owns, rows of a streamed tile, most value columns

// stats: [B * heads][-LSE1, -LSE2, -D1, -D2][n_pad]; padding rows hold -inf, -inf, 0, 0.  A warp takes eight consecutive rows, two at a
// time with 16 lanes each: all its loads (16 bytes, where rows allow that) are in flight at once and each statistic of the eight rows
// is one store.  131072 rows of 128 in bf16, 100 MB: 25 us; 47 with a row per warp and 8-byte loads.
template <typename T>
__global__ void __launch_bounds__(256)
diff_stats_kernel(const DiffParams p, float* __restrict__ stats, int n_pad) {
  constexpr int kRows = 8, kVec = 16 / static_cast<int>(sizeof(T)), kSteps = kValue / (16 * kVec);      // (1, or 2 in fp32)
  const int lane = threadIdx.x & 31, part = lane & 15, side = lane >> 4, per = n_pad / 64;               // blocks of 64 rows of a head
  const int64_t bh = blockIdx.x / per;
  const int r0 = (blockIdx.x - static_cast<int>(bh) * per) * 64 + (threadIdx.x >> 5) * kRows;
  const int b = static_cast<int>(bh / p.heads), h = static_cast<int>(bh - static_cast<int64_t>(b) * p.heads);
  const T* out = static_cast<const T*>(p.out) + b * p.os.b + h * p.os.h;
  const T* g = static_cast<const T*>(p.dout) + b * p.gs.b + h * p.gs.h;
  const T* out2 = static_cast<const T*>(p.out2) + bh * p.nq * p.v_dim;
  const bool vec = p.v_dim % kVec == 0 && (p.os.r | p.gs.r) % kVec == 0 &&
                   ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(out2)) & 15u) == 0;
  float d[kRows / 2], d2[kRows / 2];
  if (vec) {
    uint4 x[kRows / 2][kSteps], y[kRows / 2][kSteps], z[kRows / 2][kSteps];
#pragma unroll
    for (int i = 0; i < kRows / 2; ++i)
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        const int r = r0 + 2 * i + side, col = (part + 16 * e) * kVec;
        const bool real = r < p.nq && col < p.v_dim;
        x[i][e] = real ? *reinterpret_cast<const uint4*>(g + r * p.gs.r + col) : make_uint4(0, 0, 0, 0);
        y[i][e] = real ? *reinterpret_cast<const uint4*>(out + r * p.os.r + col) : make_uint4(0, 0, 0, 0);
        z[i][e] = real ? *reinterpret_cast<const uint4*>(out2 + static_cast<int64_t>(r) * p.v_dim + col) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
    for (int i = 0; i < kRows / 2; ++i) {
      d[i] = d2[i] = 0.f;
#pragma unroll
      for (int e = 0; e < kSteps; ++e)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float xe = to_f32<T>(reinterpret_cast<const T*>(&x[i][e])[j]);
          d[i] = fmaf(xe, to_f32<T>(reinterpret_cast<const T*>(&y[i][e])[j]), d[i]);
          d2[i] = fmaf(xe, to_f32<T>(reinterpret_cast<const T*>(&z[i][e])[j]), d2[i]);
        }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRows / 2; ++i) {
      d[i] = d2[i] = 0.f;
      const int r = r0 + 2 * i + side;
      if (r >= p.nq) continue;
      for (int col = part; col < p.v_dim; col += 16) {
        const float xe = to_f32<T>(g[r * p.gs.r + col]);
        d[i] = fmaf(xe, to_f32<T>(out[r * p.os.r + col]), d[i]);
        d2[i] = fmaf(xe, to_f32<T>(out2[static_cast<int64_t>(r) * p.v_dim + col]), d2[i]);
      }
    }
  }
  float mine = 0.f, mine2 = 0.f;                           // of row r0 + lane, in the first eight lanes
#pragma unroll
  for (int i = 0; i < kRows / 2; ++i) {
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) {
      d[i] += __shfl_xor_sync(0xffffffffu, d[i], x);
      d2[i] += __shfl_xor_sync(0xffffffffu, d2[i], x);
    }
    const float a = __shfl_sync(0xffffffffu, d[i], (lane & 1) << 4), c = __shfl_sync(0xffffffffu, d2[i], (lane & 1) << 4);
    if (lane >> 1 == i) { mine = a; mine2 = c; }
  }
  if (lane < kRows) {
    const int r = r0 + lane;
    float* dst = stats + bh * 4 * n_pad + r;
    const bool real = r < p.nq;
    const int64_t ro = bh * p.nq + r, maps = static_cast<int64_t>(p.batch) * p.heads * p.nq;
    const float l1 = real ? p.lse[ro] : -CUDART_INF_F, l2 = real ? p.lse[maps + ro] : -CUDART_INF_F;
    dst[0] = l1 == -CUDART_INF_F ? l1 : -l1;              // (a row without keys: P = 2^-inf = 0)
    dst[n_pad] = l2 == -CUDART_INF_F ? l2 : -l2;
    dst[2 * n_pad] = real ? -(mine + diff_lam(p, h) * mine2) : 0.f;
    dst[3 * n_pad] = real ? -mine2 : 0.f;
  }
}

// dlam[h] = -(sum of its parts): a block per head, or one for all heads where lam is one value.  (One walk over all parts, not one for
// each sequence and head: their loads are independent.)
__global__ void __launch_bounds__(256)
diff_dlam_kernel(const float* __restrict__ parts, void* dlam, int dlam_dtype, int batch, int heads, int tiles, int all) {
  __shared__ float part[8];
  const int h0 = all ? 0 : blockIdx.x;
  float sum = 0.f;                                       // (there are fewer than 2^30 parts)
  if (all) {
#pragma unroll 8
    for (int i = threadIdx.x; i < batch * heads * tiles; i += 256) sum += parts[i];
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < batch * tiles; i += 256) sum += parts[(i / tiles * heads + h0) * tiles + i % tiles];
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.f;
    for (int w = 0; w < 8; ++w) sum += part[w];
    if (dlam_dtype == ELSA_F32) static_cast<float*>(dlam)[h0] = -sum;
    else if (dlam_dtype == ELSA_F16) static_cast<__half*>(dlam)[h0] = from_f32<__half>(-sum);
    else static_cast<__nv_bfloat16*>(dlam)[h0] = from_f32<__nv_bfloat16>(-sum);
  }
}

// DP: head dim rounded up to 64 or 128.  Pitches are 4 mod 32 (tf32.cuh).
template <int DP> struct AnyTile {
  static constexpr int kPitch = DP + 4, kVPitch = kValue + 4;
  static constexpr int kFloats = 2 * kOwn * kPitch + kOwn * kVPitch + 2 * kStream * kPitch + kStream * kVPitch;
  static constexpr int kSmem = kFloats * 4;
};

// S1, S2 and G of a warp's 16 x 16 block: rows of (a1, a2, ag) against rows of (b1, b2, bg)
template <int DP>
__device__ __forceinline__ void scores(float (&s)[2][2][4], float (&gv)[2][4], const float* a, const float* ag, const float* b, const float* bg,
                                       int a_map, int b_map, int d8, int v8, int lane) {
  constexpr int kPitch = AnyTile<DP>::kPitch, kVPitch = AnyTile<DP>::kVPitch;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[0][n][e] = s[1][n][e] = gv[n][e] = 0.f;
#pragma unroll 2
  for (int k = 0; k < d8; k += 8) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      tf32::Split x[4], y[2];
      tf32::load_a(x, a + m * a_map + k, kPitch, lane);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        tf32::load_bt(y, b + m * b_map + 8 * n * kPitch + k, kPitch, lane);
        tf32::mma3(s[m][n], x, y);
      }
    }
  }
#pragma unroll 2
  for (int k = 0; k < v8; k += 8) {
    tf32::Split x[4], y[2];
    tf32::load_a(x, ag + k, kVPitch, lane);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      tf32::load_bt(y, bg + 8 * n * kVPitch + k, kVPitch, lane);
      tf32::mma3(gv[n], x, y);
    }
  }
}
// acc[16 x 8 N] += w[16 x 16] rows[16 x 8 N], the first n8 columns
template <int N>
__device__ __forceinline__ void accumulate(float (&acc)[N][4], const float (&w)[2][4], const float* rows, int pitch, int n8, int lane) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    tf32::Split x[4], y[2];
    tf32::acc_as_a(x, w[k]);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (8 * n >= n8) continue;
      tf32::load_b(y, rows + 8 * k * pitch + 8 * n, pitch, lane);
      tf32::mma3(acc[n], x, y);
    }
  }
}
__device__ __forceinline__ void team_sync(int team) {
  if (team > 1) cooperative_groups::this_cluster().sync();
  else __syncthreads();
}
__device__ __forceinline__ float* of_member(float* p, int team, int member) {
  return team > 1 ? cooperative_groups::this_cluster().map_shared_rank(p, member) : p;
}
// The four warps of a row half hold sums over their own columns of the tiles: added up in shared memory, in order, then over the blocks
// that share the rows (`team` of them, a cluster), in order, and stored: a block of every kThreads-th elements
template <typename T, int N>
__device__ __forceinline__ void finish(float* buffer, const float (&acc)[N][4], int half, int part, T* dst, int64_t stride, int row0, int rows, int dim,
                                       float f, int lane, int team, int member) {
  constexpr int kPitch = 8 * N + 4;
  const int r = half * 16 + (lane >> 2), c = 2 * (lane & 3);
  for (int turn = 0; turn < 4; ++turn) {
    __syncthreads();
    if (part != turn) continue;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float* at = buffer + (r + 8 * (e >> 1)) * kPitch + 8 * n + c + (e & 1);
        *at = turn == 0 ? acc[n][e] : *at + acc[n][e];
      }
  }
  team_sync(team);
  for (int i = threadIdx.x + member * kThreads; i < kOwn * 8 * N; i += kThreads * team) {
    const int row = i / (8 * N), col = i % (8 * N);
    if (row0 + row >= rows || col >= dim) continue;
    float x = 0.f;
    for (int r = 0; r < team; ++r) x += *(of_member(buffer, team, r) + row * kPitch + col);
    dst[(row0 + row) * stride + col] = from_f32<T>(x * f);
  }
  team_sync(team);                                      // (others read this block's buffer)
}

// dQ1, dQ2 of 32 query rows of one head
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, DP == 64 ? 2 : 1)
diff_dq_any_kernel(const DiffParams p, const float* __restrict__ stats, int n_pad, int team) {
  using Tile = AnyTile<DP>;
  constexpr int kPitch = Tile::kPitch, kVPitch = Tile::kVPitch;
  extern __shared__ __align__(16) float smem[];
  float* sq = smem;                                     // [map][query][dim]
  float* sg = sq + 2 * kOwn * kPitch;                   // [query][value dim]
  float* sk = sg + kOwn * kVPitch;                      // [map][key][dim]
  float* sv = sk + 2 * kStream * kPitch;                // [key][value dim]
  const int h = blockIdx.y, b = blockIdx.z, g = h / (p.heads / p.kv_heads), tiles = gridDim.x / team, member = blockIdx.x % team;
  const int q0 = (tiles - 1 - static_cast<int>(blockIdx.x) / team) * kOwn;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp & 1, part = warp >> 1, shift = p.nk - p.nq;
  const int d8 = (p.head_dim + 7) / 8 * 8, v8 = (p.v_dim + 7) / 8 * 8;
  for (int m = 0; m < 2; ++m) tf32::Rows<T, kThreads, kOwn, DP>(p.q, b * p.qs.b + (2 * h + m) * p.qs.h, p.qs.r, p.nq, p.head_dim).load(sq + m * kOwn * kPitch, kPitch, q0);
  tf32::Rows<T, kThreads, kOwn, kValue>(p.dout, b * p.gs.b + h * p.gs.h, p.gs.r, p.nq, p.v_dim).load(sg, kVPitch, q0);
  using KeyRows = tf32::Rows<T, kThreads, kStream, DP>;
  using ValueRows = tf32::Rows<T, kThreads, kStream, kValue>;
  const KeyRows k1(p.k, b * p.ks.b + 2 * g * p.ks.h, p.ks.r, p.nk, p.head_dim), k2(p.k, b * p.ks.b + (2 * g + 1) * p.ks.h, p.ks.r, p.nk, p.head_dim);
  const ValueRows vr(p.v, b * p.vs.b + g * p.vs.h, p.vs.r, p.nk, p.v_dim);
  const float lam = diff_lam(p, h);
  const int row = q0 + 16 * half + (lane >> 2);         // and row + 8   (q0 + 31 < n_pad)
  float nlse[2][2], nd[2][2];
  int lim[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float* st = stats + (static_cast<int64_t>(b) * p.heads + h) * 4 * n_pad + row + 8 * j;
    nlse[0][j] = st[0]; nlse[1][j] = st[n_pad]; nd[0][j] = st[2 * n_pad]; nd[1][j] = st[3 * n_pad];
    lim[j] = p.causal ? min(p.nk - 1, row + 8 * j + shift) : p.nk - 1;
  }
  float dq[2][DP / 8][4] = {}, dl = 0.f;
  const int end = p.causal ? min(p.nk, min(q0 + kOwn, p.nq) + shift) : p.nk;
  for (int k0 = member * kStream; k0 < end; k0 += team * kStream) {
    __syncthreads();
    k1.load(sk, kPitch, k0);
    k2.load(sk + kStream * kPitch, kPitch, k0);
    vr.load(sv, kVPitch, k0);
    __syncthreads();
    if (k0 + 16 * part >= end) continue;                // (uniform for the warp: none of its keys is seen)
    float s[2][2][4], gv[2][4];
    scores<DP>(s, gv, sq + 16 * half * kPitch, sg + 16 * half * kVPitch, sk + 16 * part * kPitch, sv + 16 * part * kVPitch, kOwn * kPitch, kStream * kPitch,
               d8, v8, lane);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = e >> 1;
        const bool seen = k0 + 16 * part + 8 * n + 2 * (lane & 3) + (e & 1) <= lim[j];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float x = seen ? exp2f(fmaf(s[m][n][e], p.scale_log2, nlse[m][j])) : 0.f;
          if (m == 1) dl = fmaf(x, gv[n][e], dl);
          s[m][n][e] = x * (gv[n][e] + nd[m][j]) * (m ? -lam : 1.f);
        }
      }
#pragma unroll
    for (int m = 0; m < 2; ++m) accumulate(dq[m], s[m], sk + m * kStream * kPitch + 16 * part * kPitch, kPitch, d8, lane);
  }
  if (p.dlam_parts) {
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) dl += __shfl_xor_sync(0xffffffffu, dl, x);
    __shared__ float part_of[kThreads / 32];
    if (lane == 0) part_of[warp] = dl;
    team_sync(team);
    if (threadIdx.x == 0 && member == 0) {
      dl = 0.f;
      for (int r = 0; r < team; ++r)
        for (int x = 0; x < kThreads / 32; ++x) dl += *(of_member(part_of, team, r) + x);
      p.dlam_parts[(static_cast<int64_t>(b) * p.heads + h) * tiles + q0 / kOwn] = dl;
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
    finish<T>(smem, dq[m], half, part, static_cast<T*>(p.dq) + b * p.dqs.b + (2 * h + m) * p.dqs.h, p.dqs.r, q0, p.nq, p.head_dim, p.scale, lane, team, member);
}

// dK1, dK2, dV of 32 keys of one key head: over the query heads that share it, and their rows
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads)
diff_dkv_any_kernel(const DiffParams p, const float* __restrict__ stats, int n_pad, int team) {
  using Tile = AnyTile<DP>;
  constexpr int kPitch = Tile::kPitch, kVPitch = Tile::kVPitch;
  extern __shared__ __align__(16) float smem[];
  float* sk = smem;                                     // [map][key][dim]
  float* sv = sk + 2 * kOwn * kPitch;                   // [key][value dim]
  float* sq = sv + kOwn * kVPitch;                      // [map][query][dim]
  float* sg = sq + 2 * kStream * kPitch;                // [query][value dim]
  const int g = blockIdx.y, b = blockIdx.z, group = p.heads / p.kv_heads, member = blockIdx.x % team, k0 = static_cast<int>(blockIdx.x) / team * kOwn;
  int turn = 0;                                         // of the members, tile by tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp & 1, part = warp >> 1, shift = p.nk - p.nq;
  const int d8 = (p.head_dim + 7) / 8 * 8, v8 = (p.v_dim + 7) / 8 * 8;
  for (int m = 0; m < 2; ++m) tf32::Rows<T, kThreads, kOwn, DP>(p.k, b * p.ks.b + (2 * g + m) * p.ks.h, p.ks.r, p.nk, p.head_dim).load(sk + m * kOwn * kPitch, kPitch, k0);
  tf32::Rows<T, kThreads, kOwn, kValue>(p.v, b * p.vs.b + g * p.vs.h, p.vs.r, p.nk, p.v_dim).load(sv, kVPitch, k0);
  const int key = k0 + 16 * half + (lane >> 2);         // and key + 8
  float dk[2][DP / 8][4] = {}, dv[kValue / 8][4] = {};
  const int begin = p.causal ? max(0, k0 - shift) / kStream * kStream : 0;      // queries before it see none of these keys
  for (int h = g * group; h < (g + 1) * group; ++h) {
    const float lam = diff_lam(p, h);
    const float* st = stats + (static_cast<int64_t>(b) * p.heads + h) * 4 * n_pad;
    const tf32::Rows<T, kThreads, kStream, DP> q1(p.q, b * p.qs.b + 2 * h * p.qs.h, p.qs.r, p.nq, p.head_dim), q2(p.q, b * p.qs.b + (2 * h + 1) * p.qs.h, p.qs.r, p.nq, p.head_dim);
    const tf32::Rows<T, kThreads, kStream, kValue> gr(p.dout, b * p.gs.b + h * p.gs.h, p.gs.r, p.nq, p.v_dim);
    for (int q0 = begin; q0 < p.nq; q0 += kStream) {
      const bool mine = turn == member;
      turn = turn + 1 == team ? 0 : turn + 1;
      if (!mine) continue;
      __syncthreads();
      q1.load(sq, kPitch, q0);
      q2.load(sq + kStream * kPitch, kPitch, q0);
      gr.load(sg, kVPitch, q0);
      __syncthreads();
      const int qc = q0 + 16 * part;                    // first query of the warp's block
      if (qc >= p.nq || (p.causal && qc + 15 + shift < k0 + 16 * half)) continue;   // (uniform for the warp: nothing seen)
      float s[2][2][4], gv[2][4];
      scores<DP>(s, gv, sk + 16 * half * kPitch, sv + 16 * half * kVPitch, sq + 16 * part * kPitch, sg + 16 * part * kVPitch, kOwn * kPitch, kStream * kPitch,
                 d8, v8, lane);
      float w[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int qi = qc + 8 * n + 2 * (lane & 3) + (e & 1), kr = key + 8 * (e >> 1);   // (qi below n_pad; rows from nq on have P = 0)
          const bool seen = kr < p.nk && (!p.causal || kr <= qi + shift);
          const float x1 = seen ? exp2f(fmaf(s[0][n][e], p.scale_log2, st[qi])) : 0.f;
          const float x2 = seen ? -lam * exp2f(fmaf(s[1][n][e], p.scale_log2, st[n_pad + qi])) : 0.f;
          w[n][e] = x1 + x2;
          s[0][n][e] = x1 * (gv[n][e] + st[2 * n_pad + qi]);
          s[1][n][e] = x2 * (gv[n][e] + st[3 * n_pad + qi]);
        }
      accumulate(dv, w, sg + 16 * part * kVPitch, kVPitch, v8, lane);
#pragma unroll
      for (int m = 0; m < 2; ++m) accumulate(dk[m], s[m], sq + m * kStream * kPitch + 16 * part * kPitch, kPitch, d8, lane);
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
    finish<T>(smem, dk[m], half, part, static_cast<T*>(p.dk) + b * p.dks.b + (2 * g + m) * p.dks.h, p.dks.r, k0, p.nk, p.head_dim, p.scale, lane, team, member);
  finish<T>(smem, dv, half, part, static_cast<T*>(p.dv) + b * p.dvs.b + g * p.dvs.h, p.dvs.r, k0, p.nk, p.v_dim, 1.f, lane, team, member);
}

// Blocks that share the rows of one tile, each with every team-th tile of the other side: as many as fill the SMs, and with a causal
// mask even out rows of many and of few tiles.
int team_of(int64_t blocks, int64_t streamed) {
  int team = 1;
  while (team < 4 && blocks * team < 4 * sm_count() && 2 * team <= cdiv64(streamed, kStream)) team *= 2;
  return team;
}

template <typename Kernel>
int launch_team(Kernel kernel, size_t smem, int team, int64_t tiles, int heads, int batch, cudaStream_t st, const DiffParams& p, const float* stats, int n_pad) {
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (rc != ELSA_OK) return rc;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(team); attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * team), static_cast<unsigned>(heads), static_cast<unsigned>(batch));
  cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cfg.attrs = &attr; cfg.numAttrs = team > 1 ? 1 : 0;
  ELSA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p, stats, n_pad, team));
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

template <typename T, int DP>
int any_t(const DiffParams& p, const float* stats, cudaStream_t st) {
  const int n_pad = static_cast<int>(align_up(p.nq, 128));
  constexpr int kSmem = AnyTile<DP>::kSmem;
  const int64_t q_tiles = cdiv64(p.nq, kOwn), k_tiles = cdiv64(p.nk, kOwn);
  const int rc = launch_team(&diff_dq_any_kernel<T, DP>, kSmem, team_of(q_tiles * p.heads * p.batch, p.nk), q_tiles, p.heads, p.batch, st, p, stats, n_pad);
  if (rc != ELSA_OK || p.nk == 0) return rc;
  return launch_team(&diff_dkv_any_kernel<T, DP>, kSmem, team_of(k_tiles * p.kv_heads * p.batch, static_cast<int64_t>(p.nq) * (p.heads / p.kv_heads)), k_tiles,
                     p.kv_heads, p.batch, st, p, stats, n_pad);
}

template <typename T>
int any_t(const DiffParams& p, const float* stats, cudaStream_t st) {
  return p.head_dim > 64 ? any_t<T, 128>(p, stats, st) : any_t<T, 64>(p, stats, st);
}

}  // namespace

int diff_stats(const DiffParams& p, float* stats, int dtype, cudaStream_t st) {
  const int n_pad = static_cast<int>(align_up(p.nq, 128));
  const int64_t blocks = static_cast<int64_t>(p.batch) * p.heads * n_pad / 64;
  if (blocks > 0x7fffffffll) return ELSA_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(blocks);
  if (dtype == ELSA_F32) diff_stats_kernel<float><<<grid, 256, 0, st>>>(p, stats, n_pad);
  else if (dtype == ELSA_F16) diff_stats_kernel<__half><<<grid, 256, 0, st>>>(p, stats, n_pad);
  else diff_stats_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p, stats, n_pad);
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

int diff_dlam(const DiffParams& p, int tiles, cudaStream_t st) {
  diff_dlam_kernel<<<p.lam_stride == 0 ? 1 : p.heads, 256, 0, st>>>(p.dlam_parts, p.dlam, p.lam_dtype, p.batch, p.heads, tiles, p.lam_stride == 0);
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

int diff_bwd_any(const DiffParams& p, const float* stats, int dtype, cudaStream_t st) {
  if (dtype == ELSA_F32) return any_t<float>(p, stats, st);
  return dtype == ELSA_F16 ? any_t<__half>(p, stats, st) : any_t<__nv_bfloat16>(p, stats, st);
}

}  // namespace elsa
