// Few query rows over long key caches: each CTA folds one range of keys of one kv head into the (m, z, s) summaries of up to
// 16 (tensor cores) or 32 (FMA) rows -- all query heads that share the kv head, and all query tokens, are rows of one tile, so
// a cache is read once -- and a second launch merges a row's summaries.
//
// Bound: the bytes of the caches; rows are few, so the products are small.
//
//   split_mma_kernel   fp16 / bf16.  Four warps, each a pipeline of its own: a warp copies 16 keys at a time (cp.async, three
//                      stages, no barrier but the warp's) and multiplies them on mma.sync m16n8k16 -- S = Q K^T, O += P V --
//                      with running max, sum and O in registers; the four are merged through shared memory at the end.  mma.sync
//                      and not tcgen05: a tile has 16 rows here and not 128, a warp's products stay in its registers, and 8
//                      bytes are loaded for every row's multiply-add that either could do.
//   split_simt_kernel  any type, any head dim up to 128, any stride: FP32 FMAs on 32 x 32 tiles.
//   merge_kernel       a warp per row.
//
// Softmax statistics, sums and O are fp32; P is rounded to the inputs' type for the second product (its error, half a step of
// that type in each weight, averages out over the keys).  The reference max of a row moves only when it is exceeded by more than
// 2^8 (P <= 256 there), which saves most of the rescaling; any reference gives the same summary.
#include <algorithm>

#include "decode.cuh"
#include "tc_common.cuh"

namespace elsa {

namespace {

constexpr int kMmaWarps = 4, kMmaThreads = 32 * kMmaWarps, kMmaRows = 16, kMmaKeys = 16, kStages = 3;
constexpr int kSimtThreads = 128, kSimtRows = 32, kSimtKeys = 32, kSimtDim = 128;
constexpr float kRescaleThreshold = 8.f;

struct Block { int seg, g, b, row0, n_rows, k0, k1, part, len; };   // rows row0 .. row0 + n_rows of kv head g, keys k0 .. k1

// what a block works on; false: nothing (a split behind the sequence's last key)
__device__ __forceinline__ bool locate(const DecodeParams& p, int tile_rows, Block& w) {
  int64_t i = blockIdx.x;
  w.seg = p.n_segs > 1 && i >= p.seg[0].blocks;
  if (w.seg) i -= p.seg[0].blocks;
  const DecodeSegment& sg = p.seg[w.seg];
  const int rows_b = p.heads / p.kv_heads * p.nq;        // rows of one sequence
  const int tile = static_cast<int>(i % sg.row_tiles); i /= sg.row_tiles;
  const int split = static_cast<int>(i % sg.n_splits); i /= sg.n_splits;
  w.g = static_cast<int>(i % p.kv_heads); i /= p.kv_heads;
  w.b = static_cast<int>(i);
  const int all = sg.shared ? rows_b * p.batch : rows_b;
  w.row0 = (sg.shared ? 0 : w.b * rows_b) + tile * tile_rows;
  w.n_rows = min(tile_rows, all - tile * tile_rows);
  w.len = sg.shared || !sg.lengths ? sg.n_keys : max(0, min(sg.n_keys, sg.lengths[w.b]));
  w.k0 = split * sg.split_width;
  w.k1 = min(w.len, w.k0 + sg.split_width);
  w.part = sg.first_part + split;
  return w.k0 < w.len;
}

// the first key that row `row` (numbered within its kv head) does not see
__device__ __forceinline__ int row_limit(const DecodeParams& p, const DecodeSegment& sg, int len, int row) {
  return sg.causal ? len - p.nq + row % p.nq + 1 : len;
}

__device__ __forceinline__ int64_t q_offset(const DecodeParams& p, int g, int row, int map) {
  const int group = p.heads / p.kv_heads, per = group * p.nq;
  const int b = row / per, r = row - b * per, gi = r / p.nq, i = r - gi * p.nq;
  return b * p.qs.b + static_cast<int64_t>(p.maps * (g * group + gi) + map) * p.qs.h + i * p.qs.r;
}

// ---- tensor cores -----------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}

// DP, VP: head dim of q and k, and of v, rounded up to 64 or 128 (the columns beyond the real ones are zeros in shared memory,
// written once).  Rows of a stage are an odd number of 16-byte pieces apart: the eight rows of an ldmatrix touch all 32 banks.
template <int MAPS, int DP, int VP> struct MmaTile {
  static constexpr int kPitchK = (DP / 8 + 1) * 16, kPitchV = (VP / 8 + 1) * 16;
  static constexpr int kStage = kMmaKeys * (MAPS * kPitchK + kPitchV);
  static constexpr int kRing = kMmaWarps * kStages * kStage;
  static constexpr int kMerge = kMmaWarps * MAPS * kMmaRows * (VP + 2) * 4;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

template <typename T, int MAPS, int DP, int VP>
__global__ void __launch_bounds__(kMmaThreads, 2)
split_mma_kernel(const DecodeParams p) {
  using Tile = MmaTile<MAPS, DP, VP>;
  extern __shared__ __align__(16) uint8_t smem[];
  Block w;
  if (!locate(p, kMmaRows, w)) return;
  const DecodeSegment& sg = p.seg[w.seg];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, qrow = lane >> 2;
  const uint32_t ring = tc::smem_u32(smem) + warp * kStages * Tile::kStage;
  const int d_pieces = p.head_dim / 8, v_pieces = p.v_dim / 8;
  const T* kp[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
    kp[m] = static_cast<const T*>(sg.k) + (sg.shared ? 0 : w.b * sg.ks.b) + static_cast<int64_t>(MAPS * w.g + m) * sg.ks.h;
  const T* vp = static_cast<const T*>(sg.v) + (sg.shared ? 0 : w.b * sg.vs.b) + static_cast<int64_t>(w.g) * sg.vs.h;

  if (p.head_dim < DP || p.v_dim < VP) {                // columns that no copy writes
    for (int i = lane; i < kStages * Tile::kStage / 16; i += 32)
      *reinterpret_cast<uint4*>(smem + warp * kStages * Tile::kStage + i * 16) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  const int n_chunks = (w.k1 - w.k0 + kMmaKeys - 1) / kMmaKeys;
  const int mine = n_chunks > warp ? (n_chunks - warp + kMmaWarps - 1) / kMmaWarps : 0;   // chunks warp, warp + 4, ...
  auto copy = [&](int it) {
    if (it < mine) {
      const uint32_t st = ring + (it % kStages) * Tile::kStage;
      const int key0 = w.k0 + (warp + it * kMmaWarps) * kMmaKeys;
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
#pragma unroll
        for (int i = 0; i < kMmaKeys * DP / 8; i += 32) {
          const int r = (i + lane) / (DP / 8), c = (i + lane) % (DP / 8), key = key0 + r;
          // (keys beyond the last one: nothing is read, zeros are written)
          if (c < d_pieces)
            cp16(st + m * kMmaKeys * Tile::kPitchK + r * Tile::kPitchK + c * 16, kp[m] + static_cast<int64_t>(min(key, w.k1 - 1)) * sg.ks.r + c * 8, key < w.k1 ? 16 : 0);
        }
      }
#pragma unroll
      for (int i = 0; i < kMmaKeys * VP / 8; i += 32) {
        const int r = (i + lane) / (VP / 8), c = (i + lane) % (VP / 8), key = key0 + r;
        if (c < v_pieces)
          cp16(st + MAPS * kMmaKeys * Tile::kPitchK + r * Tile::kPitchV + c * 16, vp + static_cast<int64_t>(min(key, w.k1 - 1)) * sg.vs.r + c * 8, key < w.k1 ? 16 : 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");   // (an empty group keeps the count)
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) copy(s);

  // Q as the A operand of every K-step; rows and columns that do not exist are zeros
  uint32_t qf[MAPS][DP / 16][4];
  int lim[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = qrow + 8 * half;
    const bool real = r < w.n_rows;
    lim[half] = real ? row_limit(p, sg, w.len, w.row0 + r) : 0;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      const T* qp = static_cast<const T*>(p.q) + (real ? q_offset(p, w.g, w.row0 + r, m) : 0);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = kk * 16 + c * 8 + quad * 2;
          qf[m][kk][half + 2 * c] = real && col < p.head_dim ? *reinterpret_cast<const uint32_t*>(qp + col) : 0u;
        }
    }
  }
  float m_ref[MAPS][2], z[MAPS][2], o[MAPS][VP / 8][4];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    m_ref[m][0] = m_ref[m][1] = -CUDART_INF_F;
    z[m][0] = z[m][1] = 0.f;
#pragma unroll
    for (int n = 0; n < VP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][n][e] = 0.f;
  }
  const uint32_t k_lane = ((lane & 7) + ((lane >> 4) << 3)) * Tile::kPitchK + ((lane >> 3) & 1) * 16;
  const uint32_t v_lane = ((lane & 7) + (((lane >> 3) & 1) << 3)) * Tile::kPitchV + (lane >> 4) * 16;
  const float c = p.scale_log2;

  for (int it = 0; it < mine; ++it) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();                                       // every lane's copies of this stage are there, and the stage before it has been read
    copy(it + kStages - 1);                             // over that one: two stages are on their way while this one is used
    const uint32_t st = ring + (it % kStages) * Tile::kStage;
    const int key0 = w.k0 + (warp + it * kMmaWarps) * kMmaKeys + quad * 2;
    uint32_t pf[MAPS][4];
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t kf[4];
        ldsm_x4(kf, st + m * kMmaKeys * Tile::kPitchK + k_lane + kk * 32);
        mma16816<T>(s[0], qf[m][kk], kf[0], kf[1]);
        mma16816<T>(s[1], qf[m][kk], kf[2], kf[3]);
      }
      float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n * 8 + (e & 1);
          s[n][e] = key < min(lim[e >> 1], w.k1) ? s[n][e] * c : -CUDART_INF_F;
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
      bool move[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        move[h] = top[h] > m_ref[m][h] + kRescaleThreshold;
      }
      if (__any_sync(0xffffffffu, move[0] || move[1])) {
        float alpha[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float m_new = move[h] ? top[h] : m_ref[m][h];   // (a row's result does not depend on the rows beside it)
          alpha[h] = move[h] ? fast_exp2(m_ref[m][h] - m_new) : 1.f;
          m_ref[m][h] = m_new;
          z[m][h] *= alpha[h];
        }
#pragma unroll
        for (int n = 0; n < VP / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[m][n][e] *= alpha[e >> 1];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float m_use = m_ref[m][h] == -CUDART_INF_F ? 0.f : m_ref[m][h];
        float e0 = fast_exp2(s[0][2 * h] - m_use), e1 = fast_exp2(s[0][2 * h + 1] - m_use);
        float e2 = fast_exp2(s[1][2 * h] - m_use), e3 = fast_exp2(s[1][2 * h + 1] - m_use);
        z[m][h] += (e0 + e1) + (e2 + e3);
        pf[m][h] = tc::pack2<T>(e0, e1);
        pf[m][2 + h] = tc::pack2<T>(e2, e3);
      }
    }
#pragma unroll
    for (int n = 0; n < VP / 16; ++n) {
      uint32_t vf[4];
      ldsm_x4_t(vf, st + MAPS * kMmaKeys * Tile::kPitchK + v_lane + n * 32);
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        mma16816<T>(o[m][2 * n], pf[m], vf[0], vf[1]);
        mma16816<T>(o[m][2 * n + 1], pf[m], vf[2], vf[3]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();                                      // the ring becomes the merge buffer

  // [warp][map][row]: VP sums, then the max and the sum of weights
  float* merge = reinterpret_cast<float*>(smem);
  auto slot = [&](int wp, int m, int r) { return merge + ((wp * MAPS + m) * kMmaRows + r) * (VP + 2); };
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      z[m][h] += __shfl_xor_sync(0xffffffffu, z[m][h], 1);
      z[m][h] += __shfl_xor_sync(0xffffffffu, z[m][h], 2);
      if (qrow + 8 * h >= w.n_rows) continue;
      float* dst = slot(warp, m, qrow + 8 * h);
#pragma unroll
      for (int n = 0; n < VP / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8 + quad * 2) = make_float2(o[m][n][2 * h], o[m][n][2 * h + 1]);
      if (quad == 0) *reinterpret_cast<float2*>(dst + VP) = make_float2(m_ref[m][h], z[m][h]);
    }
  __syncthreads();
  const int64_t base = (static_cast<int64_t>(w.part) * p.kv_heads + w.g) * decode_rows(p) + w.row0;
  for (int i = threadIdx.x; i < w.n_rows * MAPS * VP / 4; i += kMmaThreads) {
    const int col = i % (VP / 4) * 4, rm = i / (VP / 4), m = rm % MAPS, r = rm / MAPS;
    float top = -CUDART_INF_F;
#pragma unroll
    for (int wp = 0; wp < kMmaWarps; ++wp) top = fmaxf(top, slot(wp, m, r)[VP]);
    float zs = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int wp = 0; wp < kMmaWarps; ++wp) {
      const float* src = slot(wp, m, r);
      const float f = src[VP + 1] != 0.f ? fast_exp2(src[VP] - top) : 0.f;
      zs += f * src[VP + 1];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += f * src[col + e];
    }
    const int64_t at = (base + r) * MAPS + m;
    if (col < p.v_dim) *reinterpret_cast<float4*>(p.s + at * p.v_dim + col) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (col == 0) {
      p.m[at] = zs != 0.f ? top : -CUDART_INF_F;
      p.z[at] = zs;
    }
  }
}

// ---- FMA --------------------------------------------------------------------------------------------------------------
// 32 rows x 32 keys; a thread has rows (t / 8) * 2 + {0, 1} and keys t % 8 + 8 {0..3} of the scores, then the same rows and
// value columns (t % 8) * 4 + 32 {0..3} of O.  Shared rows are 4 floats longer than their columns (no bank is met twice by the
// eight threads of a row).
template <typename T, int MAPS>
__global__ void __launch_bounds__(kSimtThreads)
split_simt_kernel(const DecodeParams p) {
  extern __shared__ __align__(16) float fsmem[];
  constexpr int kPitch = kSimtDim + 4, kScorePitch = kSimtKeys + 1;
  float* sq = fsmem;                                    // [map][row][dim]
  float* sk = sq + MAPS * kSimtRows * kPitch;           // [map][key][dim]
  float* sv = sk + MAPS * kSimtKeys * kPitch;           // [key][dim]
  float* sp = sv + kSimtKeys * kPitch;                  // [map][row][key]
  Block w;
  if (!locate(p, kSimtRows, w)) return;
  const DecodeSegment& sg = p.seg[w.seg];
  const int tid = threadIdx.x, r0 = tid / 8 * 2, kc = tid % 8;
  const int dim4 = (p.head_dim + 3) / 4 * 4;
  for (int i = tid; i < MAPS * kSimtRows * dim4; i += kSimtThreads) {
    const int col = i % dim4, rm = i / dim4, r = rm % kSimtRows, m = rm / kSimtRows;
    const bool real = r < w.n_rows && col < p.head_dim;
    sq[(m * kSimtRows + r) * kPitch + col] = real ? to_f32<T>(static_cast<const T*>(p.q)[q_offset(p, w.g, w.row0 + r, m) + col]) : 0.f;
  }
  int lim[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) lim[j] = r0 + j < w.n_rows ? min(w.k1, row_limit(p, sg, w.len, w.row0 + r0 + j)) : 0;
  float m_run[MAPS][2], z[MAPS][2], o[MAPS][2][16];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      m_run[m][j] = -CUDART_INF_F; z[m][j] = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) o[m][j][e] = 0.f;
    }
  const T* vp = static_cast<const T*>(sg.v) + (sg.shared ? 0 : w.b * sg.vs.b) + static_cast<int64_t>(w.g) * sg.vs.h;
  for (int key0 = w.k0; key0 < w.k1; key0 += kSimtKeys) {
    __syncthreads();
    for (int i = tid; i < MAPS * kSimtKeys * dim4; i += kSimtThreads) {
      const int col = i % dim4, km = i / dim4, j = km % kSimtKeys, m = km / kSimtKeys;
      const T* kp = static_cast<const T*>(sg.k) + (sg.shared ? 0 : w.b * sg.ks.b) + static_cast<int64_t>(MAPS * w.g + m) * sg.ks.h;
      sk[(m * kSimtKeys + j) * kPitch + col] = key0 + j < w.k1 && col < p.head_dim ? to_f32<T>(kp[static_cast<int64_t>(key0 + j) * sg.ks.r + col]) : 0.f;
    }
    for (int i = tid; i < kSimtKeys * kSimtDim; i += kSimtThreads) {
      const int col = i % kSimtDim, j = i / kSimtDim;
      sv[j * kPitch + col] = key0 + j < w.k1 && col < p.v_dim ? to_f32<T>(vp[static_cast<int64_t>(key0 + j) * sg.vs.r + col]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      float s[2][4] = {};
      for (int d = 0; d < dim4; d += 4) {
        float4 a[2], b[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) a[j] = *reinterpret_cast<const float4*>(sq + (m * kSimtRows + r0 + j) * kPitch + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = *reinterpret_cast<const float4*>(sk + (m * kSimtKeys + kc + 8 * e) * kPitch + d);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] = fmaf(a[j].x, b[e].x, fmaf(a[j].y, b[e].y, fmaf(a[j].z, b[e].z, fmaf(a[j].w, b[e].w, s[j][e]))));
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = -CUDART_INF_F;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[j][e] = key0 + kc + 8 * e < lim[j] ? s[j][e] * p.scale_log2 : -CUDART_INF_F;
          top = fmaxf(top, s[j][e]);
        }
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float m_new = fmaxf(m_run[m][j], top), m_use = m_new == -CUDART_INF_F ? 0.f : m_new;
        const float alpha = m_new == -CUDART_INF_F ? 1.f : exp2f(m_run[m][j] - m_new);
        m_run[m][j] = m_new;
        z[m][j] *= alpha;
#pragma unroll
        for (int e = 0; e < 16; ++e) o[m][j][e] *= alpha;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = exp2f(s[j][e] - m_use);
          z[m][j] += x;
          sp[(m * kSimtRows + r0 + j) * kScorePitch + kc + 8 * e] = x;
        }
      }
    }
    __syncwarp();                                       // a row's weights come from eight lanes of one warp
    for (int j = 0; j < kSimtKeys; ++j) {
      float4 b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = *reinterpret_cast<const float4*>(sv + j * kPitch + kc * 4 + 32 * e);
#pragma unroll
      for (int m = 0; m < MAPS; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float x = sp[(m * kSimtRows + r0 + r) * kScorePitch + j];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[m][r][4 * e] = fmaf(x, b[e].x, o[m][r][4 * e]); o[m][r][4 * e + 1] = fmaf(x, b[e].y, o[m][r][4 * e + 1]);
            o[m][r][4 * e + 2] = fmaf(x, b[e].z, o[m][r][4 * e + 2]); o[m][r][4 * e + 3] = fmaf(x, b[e].w, o[m][r][4 * e + 3]);
          }
        }
    }
  }
  const int64_t base = (static_cast<int64_t>(w.part) * p.kv_heads + w.g) * decode_rows(p) + w.row0;
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) z[m][j] += __shfl_xor_sync(0xffffffffu, z[m][j], x);
      if (r0 + j >= w.n_rows) continue;
      const int64_t at = (base + r0 + j) * MAPS + m;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = kc * 4 + 32 * (e / 4) + e % 4;
        if (col < p.v_dim) p.s[at * p.v_dim + col] = o[m][j][e];
      }
      if (kc == 0) {
        p.m[at] = z[m][j] != 0.f ? m_run[m][j] : -CUDART_INF_F;
        p.z[at] = z[m][j];
      }
    }
}

// ---- merge ------------------------------------------------------------------------------------------------------------
// A warp per (kv head, row): the weights of the parts first (a lane per part, 32 parts at a time), then their sums, VEC value
// columns of each lane (VEC 4 where a row of sums is a multiple of 16 bytes), eight parts' loads in flight.  A row that sees no
// key (every z = 0) is zeros; a NaN stays one.
template <typename T, int MAPS, int VEC>
__global__ void __launch_bounds__(128)
merge_kernel(const DecodeParams p, int n_parts) {
  constexpr int kAhead = 8, kCols = 4 / VEC;            // column groups of a lane: VEC (lane + 32 e) ..., at most 128 columns
  const int64_t rows = decode_rows(p);
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= rows * p.kv_heads) return;
  const int g = i / static_cast<int>(rows), row = i - g * static_cast<int>(rows);
  const int group = p.heads / p.kv_heads, per = group * p.nq;
  const int b = row / per, r = row - b * per, gi = r / p.nq, t = r - gi * p.nq, h = g * group + gi;
  // parts [from, to) of a segment whose splits begin behind the sequence's last key were not written
  int from[2] = {0, 0}, to[2] = {0, 0};
#pragma unroll
  for (int s = 0; s < 2; ++s)
    if (s < p.n_segs) {
      const DecodeSegment& sg = p.seg[s];
      const int len = sg.shared || !sg.lengths ? sg.n_keys : max(0, min(sg.n_keys, sg.lengths[b]));
      from[s] = sg.first_part + (len + sg.split_width - 1) / sg.split_width;
      to[s] = sg.first_part + sg.n_splits;
    }
  auto written = [&](int part) { return !(part >= from[0] && part < to[0]) && !(part >= from[1] && part < to[1]); };
  const int64_t step = static_cast<int64_t>(p.kv_heads) * rows * MAPS;      // from one part to the next
  const int64_t first = (static_cast<int64_t>(g) * rows + row) * MAPS;
  float total[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    const float* pm = p.m + first + m;
    const float* pz = p.z + first + m;
    const float* ps = p.s + (first + m) * p.v_dim + lane * VEC;
    float top = -CUDART_INF_F, zs = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < n_parts; p0 += 32) {
      float m_part = -CUDART_INF_F, z_part = 0.f;
      if (p0 + lane < n_parts && written(p0 + lane)) {
        m_part = pm[(p0 + lane) * step];
        z_part = pz[(p0 + lane) * step];
      }
      float best = m_part;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, x));
      if (best > top) {                                 // (more than 32 parts: what came before is rescaled)
        const float alpha = exp2f(top - best);
        zs *= alpha;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= alpha;
        top = best;
      }
      const float f = z_part != 0.f ? exp2f(m_part - top) : 0.f;
      zs += z_part != 0.f ? f * z_part : 0.f;
      const int n = min(32, n_parts - p0);
      for (int j0 = 0; j0 < n; j0 += kAhead) {
        float x[kAhead][4];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const bool take = __shfl_sync(0xffffffffu, f, j0 + u) != 0.f;       // (lanes beyond n have f = 0)
          const float* src = ps + (p0 + j0 + u) * step * p.v_dim;
          if (VEC == 4) {
            const float4 v = take && lane * 4 < p.v_dim ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[u][0] = v.x; x[u][1] = v.y; x[u][2] = v.z; x[u][3] = v.w;
          } else {
#pragma unroll
            for (int e = 0; e < kCols; ++e) x[u][e] = take && lane + 32 * e < p.v_dim ? src[32 * e] : 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const float fj = __shfl_sync(0xffffffffu, f, j0 + u);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = fmaf(fj, x[u][e], acc[e]);
        }
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) zs += __shfl_xor_sync(0xffffffffu, zs, x);
    const float inv = 1.f / zs;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = zs != 0.f ? inv * acc[e] : 0.f;
    if (MAPS == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) total[e] = acc[e];
    } else {
      const int64_t ro = (static_cast<int64_t>(b) * p.heads + h) * p.nq + t;
      if (p.lse && lane == 0) p.lse[m * (static_cast<int64_t>(p.batch) * p.heads * p.nq) + ro] = zs != 0.f ? top + log2f(zs) : -CUDART_INF_F;
      if (m == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) total[e] = acc[e];
      } else {
        const int64_t at = static_cast<int64_t>(h) * p.lam_stride;
        const float lam = p.lam_dtype == ELSA_F32 ? static_cast<const float*>(p.lam)[at] : p.lam_dtype == ELSA_F16 ? to_f32(static_cast<const __half*>(p.lam)[at])
                                                                                                              : to_f32(static_cast<const __nv_bfloat16*>(p.lam)[at]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = VEC == 4 ? lane * 4 + e : lane + 32 * e;
          if (p.out2 && col < p.v_dim) static_cast<T*>(p.out2)[ro * p.v_dim + col] = from_f32<T>(acc[e]);
          total[e] -= lam * acc[e];
        }
      }
    }
  }
  T* dst = static_cast<T*>(p.out) + b * p.os.b + h * p.os.h + t * p.os.r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int col = VEC == 4 ? lane * 4 + e : lane + 32 * e;
    if (col < p.v_dim) dst[col] = from_f32<T>(total[e]);
  }
}

// q as [kv head][row][head_dim], E the elements of one access
template <typename E>
__global__ void __launch_bounds__(256)
pack_q_kernel(const DecodeParams p, E* packed, int row_elements) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int rows = static_cast<int>(decode_rows(p));
  if (i >= static_cast<int64_t>(rows) * p.kv_heads * row_elements) return;
  const int gr = static_cast<int>(i / row_elements), col = static_cast<int>(i - static_cast<int64_t>(gr) * row_elements);
  const int g = gr / rows, row = gr - g * rows;
  packed[i] = reinterpret_cast<const E*>(static_cast<const __half*>(p.q) + q_offset(p, g, row, 0))[col];
}

template <typename T, int MAPS, int DP, int VP>
int launch_mma(const DecodeParams& p, int64_t blocks, cudaStream_t st) {
  const auto kernel = &split_mma_kernel<T, MAPS, DP, VP>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), MmaTile<MAPS, DP, VP>::kSmem);
  if (rc != ELSA_OK) return rc;
  kernel<<<static_cast<unsigned>(blocks), kMmaThreads, MmaTile<MAPS, DP, VP>::kSmem, st>>>(p);
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

template <typename T>
int launch_mma_t(const DecodeParams& p, int64_t blocks, cudaStream_t st) {
  if (p.maps == 2) return p.v_dim > 64 ? launch_mma<T, 2, 64, 128>(p, blocks, st) : launch_mma<T, 2, 64, 64>(p, blocks, st);
  return p.head_dim > 64 || p.v_dim > 64 ? launch_mma<T, 1, 128, 128>(p, blocks, st) : launch_mma<T, 1, 64, 64>(p, blocks, st);
}

template <typename T>
int launch_simt_t(const DecodeParams& p, int64_t blocks, cudaStream_t st) {
  const auto kernel = p.maps == 2 ? &split_simt_kernel<T, 2> : &split_simt_kernel<T, 1>;
  const int smem = 4 * ((p.maps * (kSimtRows + kSimtKeys) + kSimtKeys) * (kSimtDim + 4) + p.maps * kSimtRows * (kSimtKeys + 1));
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (rc != ELSA_OK) return rc;
  kernel<<<static_cast<unsigned>(blocks), kSimtThreads, smem, st>>>(p);
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

}  // namespace

bool decode_mma_ok(const DecodeParams& p, int dtype) {
  if (dtype == ELSA_F32 || p.head_dim % 8 || p.v_dim % 8 || p.head_dim > (p.maps == 2 ? 64 : 128) || p.v_dim > 128) return false;
  // Q is read in pairs of elements, keys and values in 16-byte pieces
  if (((p.qs.b | p.qs.h | p.qs.r) & 1) || (reinterpret_cast<uintptr_t>(p.q) & 3u)) return false;
  for (int i = 0; i < p.n_segs; ++i) {
    const DecodeSegment& s = p.seg[i];
    if (s.n_keys > 0 && (((s.ks.b | s.ks.h | s.ks.r | s.vs.b | s.vs.h | s.vs.r) & 7) ||
                         ((reinterpret_cast<uintptr_t>(s.k) | reinterpret_cast<uintptr_t>(s.v)) & 15u)))
      return false;
  }
  return true;
}

int decode_split(DecodeParams& p, int dtype, cudaStream_t st) {
  if (p.head_dim > kSimtDim || p.v_dim > kSimtDim) return ELSA_ERR_UNSUPPORTED;
  const bool mma = decode_mma_ok(p, dtype);
  const int tile = mma ? kMmaRows : kSimtRows;
  const int rows_b = p.heads / p.kv_heads * p.nq;
  int64_t blocks = 0;
  for (int i = 0; i < p.n_segs; ++i) {
    DecodeSegment& s = p.seg[i];
    s.row_tiles = static_cast<int>(cdiv64(s.shared ? decode_rows(p) : rows_b, tile));
    s.blocks = static_cast<int64_t>(s.row_tiles) * s.n_splits * p.kv_heads * (s.shared ? 1 : p.batch);
    blocks += s.blocks;
  }
  if (blocks == 0) return ELSA_OK;
  if (blocks > 0x7fffffffll) return ELSA_ERR_UNSUPPORTED;
  if (mma) return dtype == ELSA_F16 ? launch_mma_t<__half>(p, blocks, st) : launch_mma_t<__nv_bfloat16>(p, blocks, st);
  if (dtype == ELSA_F32) return launch_simt_t<float>(p, blocks, st);
  return dtype == ELSA_F16 ? launch_simt_t<__half>(p, blocks, st) : launch_simt_t<__nv_bfloat16>(p, blocks, st);
}

int decode_pack_q(const DecodeParams& p, void* packed, cudaStream_t st) {
  if (p.maps != 1) return ELSA_ERR_UNSUPPORTED;
  const bool wide = p.head_dim % 8 == 0 && !((p.qs.b | p.qs.h | p.qs.r) & 7) && !(reinterpret_cast<uintptr_t>(p.q) & 15u);
  const int row_elements = wide ? p.head_dim / 8 : p.head_dim;
  const int64_t blocks = cdiv64(decode_rows(p) * p.kv_heads * row_elements, 256);
  if (blocks > 0x7fffffffll) return ELSA_ERR_UNSUPPORTED;
  // (16-bit elements are moved, not looked at)
  if (wide) pack_q_kernel<uint4><<<static_cast<unsigned>(blocks), 256, 0, st>>>(p, static_cast<uint4*>(packed), row_elements);
  else pack_q_kernel<uint16_t><<<static_cast<unsigned>(blocks), 256, 0, st>>>(p, static_cast<uint16_t*>(packed), row_elements);
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

template <typename T>
static int merge_t(const DecodeParams& p, int n_parts, unsigned grid, cudaStream_t st) {
  const bool vec = p.v_dim % 4 == 0;                    // (the sums start on a 256-byte boundary)
  const auto kernel = p.maps == 2 ? (vec ? &merge_kernel<T, 2, 4> : &merge_kernel<T, 2, 1>) : (vec ? &merge_kernel<T, 1, 4> : &merge_kernel<T, 1, 1>);
  kernel<<<grid, 128, 0, st>>>(p, n_parts);
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

int decode_merge(const DecodeParams& p, int n_parts, int dtype, cudaStream_t st) {
  if (decode_rows(p) * p.kv_heads > 0x3fffffff) return ELSA_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(cdiv64(decode_rows(p) * p.kv_heads, 4));
  if (dtype == ELSA_F32) return merge_t<float>(p, n_parts, grid, st);
  return dtype == ELSA_F16 ? merge_t<__half>(p, n_parts, grid, st) : merge_t<__nv_bfloat16>(p, n_parts, grid, st);
}

}  // namespace elsa
