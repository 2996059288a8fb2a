// Few query rows over long key caches: each CTA folds one range of keys of one kv head into the (m, z, s) summaries of up to
// 16 (16-bit types) or 32 (any type) rows -- all query heads that share the kv head, and all query tokens, are rows of one tile, so
// a cache is read once -- and a second launch merges a row's summaries.
//
// Bound: the bytes of the caches; rows are few, so the products are small.
//
//   split_mma_kernel   fp16 / bf16.  Four warps, each a pipeline of its own: a warp copies 16 keys at a time (cp.async, three
//                      stages, no barrier but the warp's) and multiplies them on mma.sync m16n8k16 -- S = Q K^T, O += P V --
//                      with running max, sum and O in registers; the four are merged through shared memory at the end.  mma.sync
//                      and not tcgen05: a tile has 16 rows here and not 128, a warp's products stay in its registers, and 8
//                      bytes are loaded for every row's multiply-add that either could do.
//                      A warp needs about 2300 cycles for 16 keys, a chain of products, shuffles and exponentials.
//   split_any_kernel   any type, any head dim up to 128, any stride, in fp32 (split tf32 operands) on 32 x 32 tiles.
//   merge_kernel       a warp per row, on the device early (it waits for the launch before it): 1 us less for a call.
//
// Measured, bf16, head dim 128: 256 x 8 caches of up to 2048 keys, 1.1 GB, 172 us = 6.3 TB/s, 0.96 of a plain copy's rate; 16 x 4
// caches of up to 8192 keys of two maps (head dim 64, values of 128), 167 MB, 41 us: about 310 blocks of 960 keys in 296 places, 1.05
// waves that take the time of two (33 to 46 us with 256 to 2048 keys a block, by chance).
//
// Softmax statistics, sums and O are fp32.  P is rounded to the inputs' type for the second product: with up to 8 rows of a tile in two
// parts, the second in the product's other rows; with more in one (its error, half a step of that type in each weight, averages out
// over the keys; a second product for the rest took 55 us where the first alone takes 45).  The reference max of a row moves only when it is exceeded by more than
// 2^8 (P <= 256 there), which saves most of the rescaling; any reference gives the same summary.
#include <algorithm>

#include "decode.cuh"
#include "tc_common.cuh"
#include "tf32.cuh"

namespace elsa {

namespace {

constexpr int kMmaWarps = 4, kMmaThreads = 32 * kMmaWarps, kMmaRows = 16, kMmaKeys = 16, kStages = 3;
constexpr int kAnyThreads = 128, kAnyRows = 32, kAnyKeys = 32, kAnyDim = 128;
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
  w.len = keys_of(sg, w.b);
  w.k0 = split * sg.split_width;
  w.k1 = min(w.len, w.k0 + sg.split_width);
  w.part = sg.first_part + split;
  if (w.k0 >= w.len) return false;
  // keys that no row of the tile sees are left out (a tile that spans a query head's end has the last token); with none left the summary says so
  const int last = (w.row0 + w.n_rows - 1) % p.nq;
  if (sg.causal && last >= w.n_rows - 1) w.k1 = min(w.k1, max(w.k0, w.len - p.nq + last + 1));
  return true;
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

// The last block ends after the launch before this one: what waits for this launch has waited for that one too.
__device__ __forceinline__ void end_behind_previous() {
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) wait_for_previous();
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
// what rounding a and b to T (`rounded`) left of them, also in T
template <typename T>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t rounded) {
  const T* e = reinterpret_cast<const T*>(&rounded);
  return tc::pack2<T>(a - to_f32<T>(e[0]), b - to_f32<T>(e[1]));
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
// PAIRED: the tile has 8 rows, each twice: row r + 8 of P is what rounding row r to T left of it, so that the product has P to twice
// the bits, at no cost, and the other 8 rows' exponentials are not there at all.
template <int MAPS, int DP, int VP, bool PAIRED> struct MmaTile {
  static constexpr int kRows = PAIRED ? kMmaRows / 2 : kMmaRows;
  static constexpr int kPitchK = (DP / 8 + 1) * 16, kPitchV = (VP / 8 + 1) * 16;
  static constexpr int kStage = kMmaKeys * (MAPS * kPitchK + kPitchV);
  static constexpr int kRing = kMmaWarps * kStages * kStage;
  static constexpr int kMerge = kMmaWarps * MAPS * kRows * (VP + 2) * 4;
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

template <typename T, int MAPS, int DP, int VP, bool PAIRED>
__global__ void __launch_bounds__(kMmaThreads, 2)
split_mma_kernel(const DecodeParams p) {
  using Tile = MmaTile<MAPS, DP, VP, PAIRED>;
  constexpr int kHalves = PAIRED ? 1 : 2;               // rows of a lane: qrow, and qrow + 8
  extern __shared__ __align__(16) uint8_t smem[];
  Block w;
  let_next_begin();
  if (!locate(p, Tile::kRows, w)) {
    end_behind_previous();
    return;
  }
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
  // A lane copies one 16-byte piece of every kPassK-th (kPassV-th) key of a chunk.  Chunks come in order: the sources move on by as much each
  // time.  Keys beyond the last one (of the last chunk): nothing is read, zeros are written.
  constexpr int kPassK = 256 / DP, kPassV = 256 / VP;    // keys of one pass of the warp
  const int k_row = lane / (DP / 8), k_col = lane % (DP / 8), v_row = lane / (VP / 8), v_col = lane % (VP / 8);
  const bool k_real = k_col < d_pieces, v_real = v_col < v_pieces;
  const int64_t k_pass = kPassK * sg.ks.r, v_pass = kPassV * sg.vs.r, k_step = kMmaWarps * kMmaKeys * sg.ks.r, v_step = kMmaWarps * kMmaKeys * sg.vs.r;
  int next = w.k0 + warp * kMmaKeys;                     // first key of the next chunk
#pragma unroll
  for (int m = 0; m < MAPS; ++m) kp[m] += (next + k_row) * sg.ks.r + k_col * 8;
  vp += (next + v_row) * sg.vs.r + v_col * 8;
  const uint32_t k_dst = k_row * Tile::kPitchK + k_col * 16, v_dst = MAPS * kMmaKeys * Tile::kPitchK + v_row * Tile::kPitchV + v_col * 16;
  auto copy = [&](int it) {
    if (it < mine) {
      const uint32_t st = ring + (it % kStages) * Tile::kStage;
      const int valid = w.k1 - next;
      if (valid >= kMmaKeys) {
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
#pragma unroll
          for (int i = 0; i < kMmaKeys / kPassK; ++i)
            if (k_real) cp16(st + k_dst + (m * kMmaKeys + i * kPassK) * Tile::kPitchK, kp[m] + i * k_pass, 16);
#pragma unroll
        for (int i = 0; i < kMmaKeys / kPassV; ++i)
          if (v_real) cp16(st + v_dst + i * kPassV * Tile::kPitchV, vp + i * v_pass, 16);
      } else {
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
#pragma unroll
          for (int i = 0; i < kMmaKeys / kPassK; ++i) {
            const bool there = i * kPassK + k_row < valid;
            if (k_real) cp16(st + k_dst + (m * kMmaKeys + i * kPassK) * Tile::kPitchK, there ? kp[m] + i * k_pass : static_cast<const T*>(sg.k), there ? 16 : 0);
          }
#pragma unroll
        for (int i = 0; i < kMmaKeys / kPassV; ++i) {
          const bool there = i * kPassV + v_row < valid;
          if (v_real) cp16(st + v_dst + i * kPassV * Tile::kPitchV, there ? vp + i * v_pass : static_cast<const T*>(sg.v), there ? 16 : 0);
        }
      }
#pragma unroll
      for (int m = 0; m < MAPS; ++m) kp[m] += k_step;
      vp += v_step;
      next += kMmaWarps * kMmaKeys;
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
    const bool real = half < kHalves && r < w.n_rows;
    lim[half] = real ? min(w.k1, row_limit(p, sg, w.len, w.row0 + r)) : w.k1;
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
  float m_ref[MAPS][kHalves], z[MAPS][kHalves], o[MAPS][VP / 8][4];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) { m_ref[m][h] = -CUDART_INF_F; z[m][h] = 0.f; }
#pragma unroll
    for (int n = 0; n < VP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][n][e] = 0.f;
  }
  const uint32_t k_lane = ((lane & 7) + ((lane >> 4) << 3)) * Tile::kPitchK + ((lane >> 3) & 1) * 16;
  const uint32_t v_lane = ((lane & 7) + (((lane >> 3) & 1) << 3)) * Tile::kPitchV + (lane >> 4) * 16;
  const float c = p.scale_log2;
  const int seen = __reduce_min_sync(0xffffffffu, min(lim[0], lim[1]));      // keys before it are seen by every row

  for (int it = 0; it < mine; ++it) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();                                       // every lane's copies of this stage are there, and the stage before it has been read
    copy(it + kStages - 1);                             // over that one: two stages are on their way while this one is used
    const uint32_t st = ring + (it % kStages) * Tile::kStage;
    const int chunk0 = w.k0 + (warp + it * kMmaWarps) * kMmaKeys;
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
      if (chunk0 + kMmaKeys > seen) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (chunk0 + quad * 2 + n * 8 + (e & 1) >= lim[e >> 1]) s[n][e] = -CUDART_INF_F;
      }
      float top[kHalves];
      bool move[kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        top[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1])) * c;
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        move[h] = top[h] > m_ref[m][h] + kRescaleThreshold;
      }
      if (__any_sync(0xffffffffu, move[0] || move[kHalves - 1])) {
        float alpha[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const float m_new = move[h] ? top[h] : m_ref[m][h];   // (a row's result does not depend on the rows beside it)
          alpha[h] = move[h] ? fast_exp2(m_ref[m][h] - m_new) : 1.f;
          m_ref[m][h] = m_new;
          z[m][h] *= alpha[h];
        }
#pragma unroll
        for (int n = 0; n < VP / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[m][n][e] *= alpha[PAIRED ? 0 : e >> 1];
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const float nm = m_ref[m][h] == -CUDART_INF_F ? 0.f : -m_ref[m][h];
        const float e0 = fast_exp2(fmaf(s[0][2 * h], c, nm)), e1 = fast_exp2(fmaf(s[0][2 * h + 1], c, nm));
        const float e2 = fast_exp2(fmaf(s[1][2 * h], c, nm)), e3 = fast_exp2(fmaf(s[1][2 * h + 1], c, nm));
        z[m][h] += (e0 + e1) + (e2 + e3);
        pf[m][h] = tc::pack2<T>(e0, e1);
        pf[m][2 + h] = tc::pack2<T>(e2, e3);
        if (PAIRED) {
          pf[m][1] = rest2<T>(e0, e1, pf[m][0]);
          pf[m][3] = rest2<T>(e2, e3, pf[m][2]);
        }
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
  auto slot = [&](int wp, int m, int r) { return merge + ((wp * MAPS + m) * Tile::kRows + r) * (VP + 2); };
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      z[m][h] += __shfl_xor_sync(0xffffffffu, z[m][h], 1);
      z[m][h] += __shfl_xor_sync(0xffffffffu, z[m][h], 2);
      if (qrow + 8 * h >= w.n_rows) continue;
      float* dst = slot(warp, m, qrow + 8 * h);
#pragma unroll
      for (int n = 0; n < VP / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8 + quad * 2) = PAIRED ? make_float2(o[m][n][0] + o[m][n][2], o[m][n][1] + o[m][n][3]) : make_float2(o[m][n][2 * h], o[m][n][2 * h + 1]);
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
  end_behind_previous();
}

// ---- any type ---------------------------------------------------------------------------------------------------------
// 32 rows x 32 keys in fp32, products on split tf32 operands (tf32.cuh).  Four warps: 16 rows each, and of two maps one, or of one
// map's keys the first or the second 16 (whose summaries are merged at the end).  A warp's weights go from its score accumulators
// straight into the second product.
// DP, VP: head dims rounded up to 64 or 128.
template <int MAPS, int DP, int VP> struct AnyShape {
  static constexpr int kPitch = DP + 4, kVPitch = VP + 4;
  static constexpr int kSmem = 4 * (MAPS * (kAnyRows + kAnyKeys) * kPitch + kAnyKeys * kVPitch);
};

template <typename T, int MAPS, int DP, int VP>
__global__ void __launch_bounds__(kAnyThreads)
split_any_kernel(const DecodeParams p) {
  extern __shared__ __align__(16) float fsmem[];
  constexpr int kPitch = AnyShape<MAPS, DP, VP>::kPitch, kVPitch = AnyShape<MAPS, DP, VP>::kVPitch;
  constexpr int kBlocks = MAPS == 2 ? 4 : 2;            // 8-key blocks of a warp's scores
  static_assert(MAPS == 2 || VP <= DP, "the merge of the two halves of the keys goes over the rows of Q");
  float* sq = fsmem;                                    // [map][row][dim]
  float* sk = sq + MAPS * kAnyRows * kPitch;            // [map][key][dim]
  float* sv = sk + MAPS * kAnyKeys * kPitch;            // [key][dim]
  Block w;
  let_next_begin();
  if (!locate(p, kAnyRows, w)) {
    end_behind_previous();
    return;
  }
  const DecodeSegment& sg = p.seg[w.seg];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp & 1, map = MAPS == 2 ? warp >> 1 : 0, part = MAPS == 2 ? 0 : warp >> 1;
  const int d8 = (p.head_dim + 7) / 8 * 8, v8 = (p.v_dim + 7) / 8 * 8;
  const int kc = threadIdx.x % 8;
  // (query rows are not evenly spaced: row by row)
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
    for (int r = threadIdx.x / 8; r < kAnyRows; r += kAnyThreads / 8) {
      const bool real = r < w.n_rows;
      const T* src = static_cast<const T*>(p.q) + (real ? q_offset(p, w.g, w.row0 + r, m) : 0);
      for (int col = kc; col < DP; col += 8) sq[(m * kAnyRows + r) * kPitch + col] = real && col < p.head_dim ? to_f32<T>(src[col]) : 0.f;
    }
  using KeyRows = tf32::Rows<T, kAnyThreads, kAnyKeys, DP>;
  using ValueRows = tf32::Rows<T, kAnyThreads, kAnyKeys, VP>;
  const int64_t k_base = (sg.shared ? 0 : w.b * sg.ks.b) + static_cast<int64_t>(MAPS * w.g) * sg.ks.h;
  const KeyRows k1(sg.k, k_base, sg.ks.r, w.k1, p.head_dim), k2(sg.k, k_base + (MAPS - 1) * sg.ks.h, sg.ks.r, w.k1, p.head_dim);
  const ValueRows vr(sg.v, (sg.shared ? 0 : w.b * sg.vs.b) + static_cast<int64_t>(w.g) * sg.vs.h, sg.vs.r, w.k1, p.v_dim);
  const int row = 16 * half + (lane >> 2);              // and row + 8
  int lim[2];
  float m_run[2] = {-CUDART_INF_F, -CUDART_INF_F}, z[2] = {0.f, 0.f}, o[VP / 8][4] = {};
#pragma unroll
  for (int j = 0; j < 2; ++j) lim[j] = row + 8 * j < w.n_rows ? min(w.k1, row_limit(p, sg, w.len, w.row0 + row + 8 * j)) : 0;
  for (int key0 = w.k0; key0 < w.k1; key0 += kAnyKeys) {
    __syncthreads();
    k1.load(sk, kPitch, key0);
    if (MAPS == 2) k2.load(sk + kAnyKeys * kPitch, kPitch, key0);
    vr.load(sv, kVPitch, key0);
    __syncthreads();
    float s[kBlocks][4] = {};
    const float* a = sq + (map * kAnyRows + 16 * half) * kPitch;
    const float* b = sk + (map * kAnyKeys + 16 * part) * kPitch;
#pragma unroll 2
    for (int k = 0; k < d8; k += 8) {
      tf32::Split x[4], y[2];
      tf32::load_a(x, a + k, kPitch, lane);
#pragma unroll
      for (int n = 0; n < kBlocks; ++n) {
        tf32::load_bt(y, b + 8 * n * kPitch + k, kPitch, lane);
        tf32::mma3(s[n], x, y);
      }
    }
    const int key = key0 + 16 * part + 2 * (lane & 3);
    float top[2] = {-CUDART_INF_F, -CUDART_INF_F}, alpha[2];
#pragma unroll
    for (int n = 0; n < kBlocks; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = key + 8 * n + (e & 1) < lim[e >> 1] ? s[n][e] * p.scale_log2 : -CUDART_INF_F;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 1));
      top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 2));
      const float m_new = fmaxf(m_run[j], top[j]);
      alpha[j] = m_new > m_run[j] ? exp2f(m_run[j] - m_new) : 1.f;
      m_run[j] = m_new;
      z[j] *= alpha[j];
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int n = 0; n < VP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= alpha[e >> 1];
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = exp2f(s[n][e] - (m_run[e >> 1] == -CUDART_INF_F ? 0.f : m_run[e >> 1]));
        z[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      tf32::Split x[4], y[2];
      tf32::acc_as_a(x, s[k]);
#pragma unroll
      for (int n = 0; n < VP / 8; ++n) {
        if (8 * n >= v8) continue;
        tf32::load_b(y, sv + (16 * part + 8 * k) * kVPitch + 8 * n, kVPitch, lane);
        tf32::mma3(o[n], x, y);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    z[j] += __shfl_xor_sync(0xffffffffu, z[j], 1);
    z[j] += __shfl_xor_sync(0xffffffffu, z[j], 2);
  }
  if (MAPS == 1) {                                      // the second 16 keys' summaries through shared memory (over the rows of Q)
    __syncthreads();
    float* buffer = fsmem;
    const int c = 2 * (lane & 3);
    if (part == 1) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* dst = buffer + (row + 8 * j) * kVPitch;
#pragma unroll
        for (int n = 0; n < VP / 8; ++n) { dst[8 * n + c] = o[n][2 * j]; dst[8 * n + c + 1] = o[n][2 * j + 1]; }
        if ((lane & 3) == 0) { dst[VP] = m_run[j]; dst[VP + 1] = z[j]; }
      }
    }
    __syncthreads();
    if (part == 1) return;                              // (no barrier follows)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float* src = buffer + (row + 8 * j) * kVPitch;
      const float m2 = src[VP], z2 = src[VP + 1], m_new = fmaxf(m_run[j], m2);
      const float f1 = z[j] != 0.f ? exp2f(m_run[j] - m_new) : 0.f, f2 = z2 != 0.f ? exp2f(m2 - m_new) : 0.f;
      z[j] = z[j] * f1 + z2 * f2;
      m_run[j] = m_new;
#pragma unroll
      for (int n = 0; n < VP / 8; ++n) {
        o[n][2 * j] = o[n][2 * j] * f1 + src[8 * n + c] * f2;
        o[n][2 * j + 1] = o[n][2 * j + 1] * f1 + src[8 * n + c + 1] * f2;
      }
    }
  }
  const int64_t base = (static_cast<int64_t>(w.part) * p.kv_heads + w.g) * decode_rows(p) + w.row0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (row + 8 * j >= w.n_rows) continue;
    const int64_t at = (base + row + 8 * j) * MAPS + map;
#pragma unroll
    for (int n = 0; n < VP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = 8 * n + 2 * (lane & 3) + e;
        if (col < p.v_dim) p.s[at * p.v_dim + col] = o[n][2 * j + e];
      }
    if ((lane & 3) == 0) {
      p.m[at] = z[j] != 0.f ? m_run[j] : -CUDART_INF_F;
      p.z[at] = z[j];
    }
  }
  end_behind_previous();
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
  wait_for_previous();
  const int g = i / static_cast<int>(rows), row = i - g * static_cast<int>(rows);
  const int group = p.heads / p.kv_heads, per = group * p.nq;
  const int b = row / per, r = row - b * per, gi = r / p.nq, t = r - gi * p.nq, h = g * group + gi;
  // parts [from, to) of a segment whose splits begin behind the sequence's last key were not written
  int from[2] = {0, 0}, to[2] = {0, 0};
#pragma unroll
  for (int s = 0; s < 2; ++s)
    if (s < p.n_segs) {
      const DecodeSegment& sg = p.seg[s];
      from[s] = sg.first_part + (keys_of(sg, b) + sg.split_width - 1) / sg.split_width;
      to[s] = sg.first_part + sg.n_splits;
    }
  auto written = [&](int part) { return !(part >= from[0] && part < to[0]) && !(part >= from[1] && part < to[1]); };
  const int64_t step = static_cast<int64_t>(p.kv_heads) * rows * MAPS;      // from one part to the next
  const int64_t first = (static_cast<int64_t>(g) * rows + row) * MAPS;
  // eight parts' sums on their way (of parts that were not written too: whatever stands there is not used)
  auto load8 = [&](float (&x)[kAhead][4], const float* ps, int p0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float* src = ps + min(p0 + u, n_parts - 1) * step * p.v_dim;
      if (VEC == 4) {
        const float4 v = lane * 4 < p.v_dim ? __ldcg(reinterpret_cast<const float4*>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[u][0] = v.x; x[u][1] = v.y; x[u][2] = v.z; x[u][3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < kCols; ++e) x[u][e] = lane + 32 * e < p.v_dim ? __ldcg(src + 32 * e) : 0.f;
      }
    }
  };
  float total[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    const float* pm = p.m + first + m;
    const float* pz = p.z + first + m;
    const float* ps = p.s + (first + m) * p.v_dim + lane * VEC;
    float top = -CUDART_INF_F, zs = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < n_parts; p0 += 32) {
      float x[kAhead][4];
      load8(x, ps, p0);                                 // (beside the weights: one latency less)
      float m_part = -CUDART_INF_F, z_part = 0.f;
      if (p0 + lane < n_parts && written(p0 + lane)) {
        m_part = __ldcg(pm + (p0 + lane) * step);
        z_part = __ldcg(pz + (p0 + lane) * step);
      }
      float best = m_part;
#pragma unroll
      for (int y = 16; y > 0; y >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, y));
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
        if (j0 > 0) load8(x, ps, p0 + j0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const float fj = __shfl_sync(0xffffffffu, f, j0 + u);               // (lanes beyond n have f = 0)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = fj != 0.f ? fmaf(fj, x[u][e], acc[e]) : acc[e];
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
      const int64_t ro = (static_cast<int64_t>(b) * p.heads + h) * p.nq_all + t;
      if (p.lse && lane == 0) p.lse[m * p.map_rows + ro] = zs != 0.f ? top + log2f(zs) : -CUDART_INF_F;
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

template <typename T, int MAPS, int DP, int VP>
int launch_mma(const DecodeParams& p, int64_t blocks, bool paired, bool behind, cudaStream_t st) {
  const auto kernel = paired ? &split_mma_kernel<T, MAPS, DP, VP, true> : &split_mma_kernel<T, MAPS, DP, VP, false>;
  const int smem = paired ? MmaTile<MAPS, DP, VP, true>::kSmem : MmaTile<MAPS, DP, VP, false>::kSmem;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (rc != ELSA_OK) return rc;
  return launch_behind(behind, kernel, static_cast<unsigned>(blocks), kMmaThreads, smem, st, p);
}

template <typename T>
int launch_mma_t(const DecodeParams& p, int64_t blocks, bool paired, bool behind, cudaStream_t st) {
  if (p.maps == 2) return p.v_dim > 64 ? launch_mma<T, 2, 64, 128>(p, blocks, paired, behind, st) : launch_mma<T, 2, 64, 64>(p, blocks, paired, behind, st);
  return p.head_dim > 64 || p.v_dim > 64 ? launch_mma<T, 1, 128, 128>(p, blocks, paired, behind, st) : launch_mma<T, 1, 64, 64>(p, blocks, paired, behind, st);
}

template <typename T, int MAPS, int DP, int VP>
int launch_any(const DecodeParams& p, int64_t blocks, bool behind, cudaStream_t st) {
  const auto kernel = &split_any_kernel<T, MAPS, DP, VP>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), AnyShape<MAPS, DP, VP>::kSmem);
  if (rc != ELSA_OK) return rc;
  return launch_behind(behind, kernel, static_cast<unsigned>(blocks), kAnyThreads, AnyShape<MAPS, DP, VP>::kSmem, st, p);
}

template <typename T>
int launch_any_t(const DecodeParams& p, int64_t blocks, bool behind, cudaStream_t st) {
  if (p.maps == 1) return p.head_dim > 64 || p.v_dim > 64 ? launch_any<T, 1, 128, 128>(p, blocks, behind, st) : launch_any<T, 1, 64, 64>(p, blocks, behind, st);
  if (p.head_dim > 64) return launch_any<T, 2, 128, 128>(p, blocks, behind, st);
  return p.v_dim > 64 ? launch_any<T, 2, 64, 128>(p, blocks, behind, st) : launch_any<T, 2, 64, 64>(p, blocks, behind, st);
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

int decode_split(DecodeParams& p, int dtype, bool behind, cudaStream_t st) {
  if (p.head_dim > kAnyDim || p.v_dim > kAnyDim) return ELSA_ERR_UNSUPPORTED;
  const bool mma = decode_mma_ok(p, dtype);
  const int rows_b = p.heads / p.kv_heads * p.nq;
  // (a shared cache is for the rows of all sequences: with more than 8 of them, tiles of 8 would read it twice as often)
  bool paired = mma && rows_b <= kMmaRows / 2;
  for (int i = 0; i < p.n_segs; ++i) paired = paired && (!p.seg[i].shared || decode_rows(p) <= kMmaRows / 2);
  const int tile = paired ? kMmaRows / 2 : mma ? kMmaRows : kAnyRows;
  int64_t blocks = 0;
  for (int i = 0; i < p.n_segs; ++i) {
    DecodeSegment& s = p.seg[i];
    s.row_tiles = static_cast<int>(cdiv64(s.shared ? decode_rows(p) : rows_b, tile));
    s.blocks = static_cast<int64_t>(s.row_tiles) * s.n_splits * p.kv_heads * (s.shared ? 1 : p.batch);
    blocks += s.blocks;
  }
  if (blocks == 0) return ELSA_OK;
  if (blocks > 0x7fffffffll) return ELSA_ERR_UNSUPPORTED;
  if (mma) return dtype == ELSA_F16 ? launch_mma_t<__half>(p, blocks, paired, behind, st) : launch_mma_t<__nv_bfloat16>(p, blocks, paired, behind, st);
  if (dtype == ELSA_F32) return launch_any_t<float>(p, blocks, behind, st);
  return dtype == ELSA_F16 ? launch_any_t<__half>(p, blocks, behind, st) : launch_any_t<__nv_bfloat16>(p, blocks, behind, st);
}

template <typename T>
static int merge_t(const DecodeParams& p, int n_parts, unsigned grid, bool behind, cudaStream_t st) {
  const bool vec = p.v_dim % 4 == 0;                    // (the sums start on a 256-byte boundary)
  const auto kernel = p.maps == 2 ? (vec ? &merge_kernel<T, 2, 4> : &merge_kernel<T, 2, 1>) : (vec ? &merge_kernel<T, 1, 4> : &merge_kernel<T, 1, 1>);
  return launch_behind(behind, kernel, grid, 128, 0, st, p, n_parts);
}

int decode_merge(const DecodeParams& p, int n_parts, int dtype, bool behind, cudaStream_t st) {
  if (decode_rows(p) * p.kv_heads > 0x3fffffff) return ELSA_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(cdiv64(decode_rows(p) * p.kv_heads, 4));
  if (dtype == ELSA_F32) return merge_t<float>(p, n_parts, grid, behind, st);
  return dtype == ELSA_F16 ? merge_t<__half>(p, n_parts, grid, behind, st) : merge_t<__nv_bfloat16>(p, n_parts, grid, behind, st);
}

}  // namespace elsa
