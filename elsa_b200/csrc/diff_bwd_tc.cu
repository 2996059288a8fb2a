// Differential attention, backward, on the 5th-generation tensor cores (fp16 / bf16, head dim <= 64, value dim <= 128, multiples of 8).
// The formulas are in diff_any.cu.  Eleven products for each pair of tiles, G = g V^T shared by the two maps, no atomics:
//
//   dq body    one CTA per 128 query rows of an output head, 64-key tiles streamed through a 4-stage ring:
//                S1 = Q1 K1^T, S2 = Q2 K2^T, G = g V^T                                (N = 64)
//                dS1, dS2 in the inputs' type, into TMEM;  dQ_m += dS_m K_m           (accumulated in TMEM)
//   dkv body   one CTA per 128 keys of a key head, over 64-query tiles of every output head that shares it:
//                S1^T = K1 Q1^T, S2^T = K2 Q2^T, G^T = V g^T                          (N = 64)
//                dV += (P1 - lam P2)^T g (N = 128), dK_m += dS_m^T Q_m                (accumulated in TMEM)
//
// One body that made all gradients would need dQ1, dQ2 of a query tile beside dV, dK1, dK2 and the three score tiles: 576 columns
// of the 512.  Two bodies recompute the exponentials (2 x 128 x 64 for each pair, 1024 cycles of the ex2 unit, twice), keep every sum
// in TMEM and in a fixed order, and a shared key head's gradients never leave their CTA.
//
// dq body, TMEM: two sets [S1 S2 G] of 3 x 64 columns, tile j in set j % 2; a thread's 16 columns of S_m give way to its 8 columns of
// packed dS_m (so K-steps are 16 columns apart and no other thread's scores are touched); dQ1 [384,448) dQ2 [448,512).  The
// scores of tile j + 1 go to the other set while tile j is worked on.
// dkv body, TMEM: S1^T S2^T G^T [0,192), (P1 - lam P2)^T [192,224), dS1^T [224,256), dV [256,384), dK1 [384,448), dK2 [448,512);
// dS2^T, for which no columns are left, goes through shared memory (128 rows of 128 bytes, swizzled as an operand).
//
// Both bodies: 16 fold warps (four threads per row, 16 columns each), a TMA producer warp, an MMA-issuing warp; all waits bounded.
// P, dS and P1 - lam P2 are rounded to the inputs' type for the second products; statistics and sums are fp32.
//
// Measured, (2, 8 heads, 8192 tokens, 64 / 128) causal bf16: 1040 to 1100 us under the power cap, 900 TFLOP/s of its eleven products; 1200 before the folds
// took pairs (fma.f32x2).  A tile takes 1670 cycles in the dq body and 2090 in the dkv body: the products that read both operands from shared
// memory, and the folds, 54 % of the ex2 unit.  A part of the exponentials on the FMA pipe (every 2nd, 4th or 8th pair): 1100 to 1180.
#include <algorithm>
#include <type_traits>

#include "diff.cuh"
#include "tc_common.cuh"

namespace elsa {

using namespace tc;

namespace {

constexpr int kSlotBytes = 64 * 64 * 2;      // one 64 x 64 16-bit tile (streamed)
constexpr int kTileBytes = 128 * 64 * 2;     // one 128 x 64 16-bit tile (resident)
constexpr int kStageBytes = 4 * kSlotBytes;  // dq: K1 K2 V V; dkv: Q1 Q2 g g
constexpr int kStages = 4;
constexpr int kVecBytes = 4 * 64 * 4;        // -LSE1 -LSE2 -D1 -D2 of 64 queries
constexpr int kFoldWarps = 16, kFoldThreads = kFoldWarps * 32, kThreads = kFoldThreads + 64;
constexpr int kProducerWarp = 16, kIssuerWarp = 17;
constexpr uint32_t kTmemCols = 512;
constexpr uint64_t kSlotStep = kSlotBytes >> 4, kStageStep = kStageBytes >> 4;    // shared-memory descriptors count 16-byte units
constexpr int kSmem = 4 * kTileBytes + kStages * (kStageBytes + kVecBytes) + kTileBytes + 1024;   // (+ dS2^T, + alignment slack)

enum BarId { BAR_STAGE = 81, BAR_FULL = 82, BAR_FREE = 83, BAR_SG = 84, BAR_SFREE = 85, BAR_DS = 86, BAR_ACC = 87 };

struct BwdParams2 {
  DiffParams d;
  const float* stats;
  int n_pad, group;
  int* status;
};

__device__ __forceinline__ void bulk_load_1d(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ float2 pair(const uint32_t (&r)[16], int i) { return make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])); }
__device__ __forceinline__ float2 exp2_pair(float2 x) { return make_float2(fast_exp2(x.x), fast_exp2(x.y)); }

// the first n (a multiple of 8, possibly <= 0) of 16 consecutive gradient values, times f
template <typename T>
__device__ __forceinline__ void store16(T* dst, const uint32_t (&r)[16], float f, int n) {
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    if (i >= n) continue;
    uint4 t;
    t.x = pack2<T>(__uint_as_float(r[i]) * f, __uint_as_float(r[i + 1]) * f);
    t.y = pack2<T>(__uint_as_float(r[i + 2]) * f, __uint_as_float(r[i + 3]) * f);
    t.z = pack2<T>(__uint_as_float(r[i + 4]) * f, __uint_as_float(r[i + 5]) * f);
    t.w = pack2<T>(__uint_as_float(r[i + 6]) * f, __uint_as_float(r[i + 7]) * f);
    *reinterpret_cast<uint4*>(dst + i) = t;
  }
}

template <typename T>
__device__ __forceinline__ void diff_dq_body(const CUtensorMap& tmap_q, const CUtensorMap& tmap_g, const CUtensorMap& tmap_k, const CUtensorMap& tmap_v,
                                             const BwdParams2& prm, int bi) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 6];
  __shared__ float dlam_part[kFoldWarps];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const DiffParams& p = prm.d;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int warp_u = __shfl_sync(0xffffffffu, warp, 0);   // (known to be warp-uniform)
  const int n_qt = (p.nq + 127) / 128;
  if (static_cast<int>(blockIdx.x) >= n_qt) return;
  const int hi = blockIdx.y, gi = hi / prm.group;
  const int q0 = (p.causal ? n_qt - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x)) * 128;   // the long tiles first
  const int shift = p.nk - p.nq;
  int ke = p.nk;
  if (p.causal) ke = min(ke, min(q0 + 128, p.nq) + shift);
  const int n_t = ke > 0 ? (ke + 63) / 64 : 0;
  const int v_tiles = p.v_dim > 64 ? 2 : 1;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  auto sQ = [&](int m) { return smem_base + m * kTileBytes; };
  auto sG = [&](int h) { return smem_base + (2 + h) * kTileBytes; };
  auto sStage = [&](int st) { return smem_base + 4 * kTileBytes + st * kStageBytes; };   // K1, K2, V (0-63), V (64-127)
  const uint32_t bar0 = smem_u32(bars);
  auto bar_full = [&](int st) { return bar0 + 8 * st; };
  auto bar_free = [&](int st) { return bar0 + 8 * (kStages + st); };
  const uint32_t barx = bar0 + 8 * 2 * kStages;
  const uint32_t bar_stage = barx, bar_dq = barx + 8;       // Q and g are in shared memory; every dQ product has retired
  // one of each for either set of score columns: the one for tile j can complete before the last thread has seen tile j - 1's
  auto bar_sg = [&](int b) { return barx + 16 + 8 * b; };   // S1, S2, G of a tile are in TMEM
  auto bar_ds = [&](int b) { return barx + 32 + 8 * b; };   // its dS1, dS2 have been delivered

  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < kStages; ++i) { mbar_init(bar_full(i), 1); mbar_init(bar_free(i), 1); }
    mbar_init(bar_stage, 1);
    mbar_init(bar_dq, 1);
    for (int b = 0; b < 2; ++b) { mbar_init(bar_sg(b), 1); mbar_init(bar_ds(b), kFoldWarps); }
    fence_mbar_init();
  }
  if (warp == kProducerWarp) {
    tmem_alloc(smem_u32(&tmem_base_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  auto tSet = [&](int b) { return tmem_base + 192 * b; };   // S1, S2 + 64, G + 128
  const uint32_t tdQ = tmem_base + 384;

  if (warp == kProducerWarp) {
    if (n_t > 0 && lane == 0) {
      prefetch_tmap(&tmap_q); prefetch_tmap(&tmap_g); prefetch_tmap(&tmap_k); prefetch_tmap(&tmap_v);
      mbar_arrive_expect_tx(bar_stage, (2 + v_tiles) * kTileBytes);
      for (int m = 0; m < 2; ++m) tma_load_4d(sQ(m), &tmap_q, bar_stage, 0, q0, 2 * hi + m, bi);
      for (int h = 0; h < v_tiles; ++h) tma_load_4d(sG(h), &tmap_g, bar_stage, 64 * h, q0, hi, bi);
      for (int j = 0; j < n_t; ++j) {
        const int st = j % kStages;
        if (j >= kStages && !mbar_wait(bar_free(st), ((j / kStages) - 1) & 1, &abort_flag, prm.status, BAR_FREE)) break;
        mbar_arrive_expect_tx(bar_full(st), (2 + v_tiles) * kSlotBytes);
        for (int m = 0; m < 2; ++m) tma_load_4d(sStage(st) + m * kSlotBytes, &tmap_k, bar_full(st), 0, j * 64, 2 * gi + m, bi);
        for (int h = 0; h < v_tiles; ++h) tma_load_4d(sStage(st) + (2 + h) * kSlotBytes, &tmap_v, bar_full(st), 64 * h, j * 64, gi, bi);
      }
    }
  } else if (warp_u == kIssuerWarp) {
    if (n_t > 0) {
      const bool leader = elect_one();
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_k = make_idesc(fmt, 0, 0, 128, 64);    // S_m, G: A, B K-major, N = 64 keys
      constexpr uint32_t idesc_mn = make_idesc(fmt, 0, 1, 128, 64);   // dQ_m: A in TMEM, B (K_m) MN-major
      const uint64_t dq[2] = {make_sdesc(sQ(0), 16, 1024), make_sdesc(sQ(1), 16, 1024)};
      const uint64_t dg[2] = {make_sdesc(sG(0), 16, 1024), make_sdesc(sG(1), 16, 1024)};
      const uint64_t dk0 = make_sdesc(sStage(0), 16, 1024), dkmn0 = make_sdesc(sStage(0), kSlotBytes, 1024);
      bool ok = mbar_wait_warp(bar_stage, 0, &abort_flag, prm.status, BAR_STAGE);
      auto issue_sg = [&](int j) {
        const int st = j % kStages;
        if (!(ok = mbar_wait_warp(bar_full(st), (j / kStages) & 1, &abort_flag, prm.status, BAR_FULL))) return;
        tc_fence_after();
        const uint32_t t = tSet(j & 1);
        const uint64_t dk = dk0 + st * kStageStep;
        for (int h = 0; h < v_tiles; ++h)
          if (leader) mma_ss_x4<2, 2>(t + 128, dg[h], dk + (2 + h) * kSlotStep, idesc_k, h == 0 ? 0u : 1u);
        for (int m = 0; m < 2; ++m)
          if (leader) mma_ss_x4<2, 2>(t + 64 * m, dq[m], dk + m * kSlotStep, idesc_k, 0u);
        if (leader) mma_commit(bar_sg(j & 1));
      };
      if (ok) {
        tc_fence_after();
        issue_sg(0);
      }
      for (int j = 0; ok && j < n_t; ++j) {
        // The other set held tile j - 1: its scores were read before its dS was delivered, and the dQ products that read that dS are
        // ahead in the tensor pipe.
        if (j + 1 < n_t) {
          issue_sg(j + 1);
          if (!ok) break;
        }
        if (!(ok = mbar_wait_warp(bar_ds(j & 1), (j >> 1) & 1, &abort_flag, prm.status, BAR_DS))) break;
        tc_fence_after();
        const int st = j % kStages;
        for (int m = 0; m < 2; ++m)
          if (leader) mma_ts_x4<16, 128>(tdQ + 64 * m, tSet(j & 1) + 64 * m, dkmn0 + st * kStageStep + m * kSlotStep, idesc_mn, j == 0 ? 0u : 1u);
        if (leader) mma_commit(bar_free(st));
      }
      if (ok && leader) mma_commit(bar_dq);
    }
  } else {
    // ---------------- fold warps: four threads per query row, 16 keys each ----------------
    const int qd = warp & 3, cq = warp >> 2;
    const int row = qd * 32 + lane;
    const int qi = q0 + row;
    const uint32_t lane_off = (static_cast<uint32_t>(qd * 32) << 16) + 16 * cq;
    const float c = p.scale_log2;
    const float* st = prm.stats + (static_cast<int64_t>(bi) * p.heads + hi) * 4 * prm.n_pad + qi;   // q0 + 127 < n_pad
    const float nlse1 = st[0], nlse2 = st[prm.n_pad], nd1 = st[2 * prm.n_pad], nd2 = st[3 * prm.n_pad];
    const float nlam = -diff_lam(p, hi);
    const float2 c2 = make_float2(c, c), nl1 = make_float2(nlse1, nlse1), nl2 = make_float2(nlse2, nlse2);
    const float2 nd1_2 = make_float2(nd1, nd1), lam2 = make_float2(nlam, nlam), lam_nd2 = make_float2(nlam * nd2, nlam * nd2);
    const int lim = p.causal ? min(p.nk - 1, qi + shift) : p.nk - 1;   // last key of this row
    float2 dl[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};     // sum of P2 G: dlam's part of these rows
    bool alive = true;
    for (int j = 0; j < n_t; ++j) {
      if (!mbar_wait_warp(bar_sg(j & 1), (j >> 1) & 1, &abort_flag, prm.status, BAR_SG)) { alive = false; break; }
      tc_fence_after();
      const uint32_t t = tSet(j & 1) + lane_off;
      uint32_t s1[16], s2[16], g[16];
      tmem_ld16(t, s1);
      tmem_ld16(t + 64, s2);
      tmem_ld16(t + 128, g);
      tmem_wait_ld();
      const int kb = j * 64 + 16 * cq;
      const bool masked = j * 64 + 64 > p.nk || (p.causal && j * 64 + 63 > q0 + shift);
      uint32_t d1[8], d2[8];
      // (pairs: fma.f32x2 and its kind; lam goes into the second map's G - D)
      auto tile = [&](auto with_mask) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 gv = pair(g, i);
          float2 x1 = exp2_pair(__ffma2_rn(pair(s1, i), c2, nl1)), x2 = exp2_pair(__ffma2_rn(pair(s2, i), c2, nl2));
          if (decltype(with_mask)::value) {
            if (kb + i > lim) x1.x = x2.x = 0.f;
            if (kb + i + 1 > lim) x1.y = x2.y = 0.f;
          }
          const float2 a = __fmul2_rn(x1, __fadd2_rn(gv, nd1_2)), b = __fmul2_rn(x2, __ffma2_rn(gv, lam2, lam_nd2));
          dl[i >> 1 & 1] = __ffma2_rn(x2, gv, dl[i >> 1 & 1]);
          d1[i >> 1] = pack2<T>(a.x, a.y);
          d2[i >> 1] = pack2<T>(b.x, b.y);
        }
      };
      if (masked) tile(std::true_type{});
      else tile(std::false_type{});
      tmem_st8(t, d1);
      tmem_st8(t + 64, d2);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive_warp(bar_ds(j & 1), lane);
    }
    if (p.dlam_parts) {
      float sum = (dl[0].x + dl[0].y) + (dl[1].x + dl[1].y);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      if (lane == 0) dlam_part[warp] = sum;
      named_barrier_sync(1, kFoldThreads);
      if (warp == 0 && lane == 0) {
        sum = 0.f;
        for (int x = 0; x < kFoldWarps; ++x) sum += dlam_part[x];
        p.dlam_parts[(static_cast<int64_t>(bi) * p.heads + hi) * n_qt + q0 / 128] = sum;
      }
    }
    uint32_t r[2][16];
#pragma unroll
    for (int i = 0; i < 16; ++i) { r[0][i] = 0u; r[1][i] = 0u; }
    if (alive && n_t > 0) {
      alive = mbar_wait_warp(bar_dq, 0, &abort_flag, prm.status, BAR_ACC);
      if (alive) {
        tc_fence_after();
        tmem_ld16(tdQ + lane_off, r[0]);
        tmem_ld16(tdQ + 64 + lane_off, r[1]);
        tmem_wait_ld();
      }
    }
    if (qi < p.nq && alive) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
        store16<T>(static_cast<T*>(p.dq) + bi * p.dqs.b + (2 * hi + m) * p.dqs.h + static_cast<int64_t>(qi) * p.dqs.r + 16 * cq, r[m], p.scale, p.head_dim - 16 * cq);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kProducerWarp) tmem_dealloc(tmem_base, kTmemCols);
}

template <typename T>
__device__ __forceinline__ void diff_dkv_body(const CUtensorMap& tmap_q, const CUtensorMap& tmap_g, const CUtensorMap& tmap_k, const CUtensorMap& tmap_v,
                                              const BwdParams2& prm, int bi) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 5];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const DiffParams& p = prm.d;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int warp_u = __shfl_sync(0xffffffffu, warp, 0);   // (known to be warp-uniform)
  const int gi = blockIdx.y, k0 = blockIdx.x * 128;
  if (k0 >= p.nk || gi >= p.kv_heads) return;
  const int shift = p.nk - p.nq;
  const int n_q64 = (p.nq + 63) / 64;
  const int q_begin = p.causal ? min(n_q64, max(0, k0 - shift) / 64) : 0;   // 64-query tiles before it see none of these keys
  const int per_head = n_q64 - q_begin, n_it = per_head * prm.group;
  const int v_tiles = p.v_dim > 64 ? 2 : 1;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  auto sK = [&](int m) { return smem_base + m * kTileBytes; };
  auto sV = [&](int h) { return smem_base + (2 + h) * kTileBytes; };
  const uint32_t sDS2 = smem_base + 4 * kTileBytes;
  auto sStage = [&](int st) { return smem_base + 5 * kTileBytes + st * kStageBytes; };   // Q1, Q2, g (0-63), g (64-127)
  const uint32_t vec_off = 5 * kTileBytes + kStages * kStageBytes;
  const uint32_t bar0 = smem_u32(bars);
  auto bar_full = [&](int st) { return bar0 + 8 * st; };
  auto bar_free = [&](int st) { return bar0 + 8 * (kStages + st); };
  const uint32_t barx = bar0 + 8 * 2 * kStages;
  const uint32_t bar_kv = barx;               // K1, K2, V are in shared memory
  const uint32_t bar_sg = barx + 8;           // S1^T, S2^T, G^T of tile i are in TMEM
  const uint32_t bar_sfree = barx + 16;       // the fold warps hold them in registers
  const uint32_t bar_ds = barx + 24;          // P1 - lam P2, dS1, dS2 of tile i have been delivered
  const uint32_t bar_acc = barx + 32;         // the dV, dK products of tile i have retired

  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < kStages; ++i) { mbar_init(bar_full(i), 1); mbar_init(bar_free(i), 1); }
    mbar_init(bar_kv, 1);
    mbar_init(bar_sg, 1); mbar_init(bar_sfree, kFoldWarps);
    mbar_init(bar_ds, kFoldWarps); mbar_init(bar_acc, 1);
    fence_mbar_init();
  }
  if (warp == kProducerWarp) {
    tmem_alloc(smem_u32(&tmem_base_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  const uint32_t tS = tmem_base, tG = tmem_base + 128, tP = tmem_base + 192, tDS1 = tmem_base + 224;
  const uint32_t tdV = tmem_base + 256, tdK = tmem_base + 384;

  if (warp == kProducerWarp) {
    if (n_it > 0 && lane == 0) {
      prefetch_tmap(&tmap_q); prefetch_tmap(&tmap_g); prefetch_tmap(&tmap_k); prefetch_tmap(&tmap_v);
      mbar_arrive_expect_tx(bar_kv, (2 + v_tiles) * kTileBytes);
      for (int m = 0; m < 2; ++m) tma_load_4d(sK(m), &tmap_k, bar_kv, 0, k0, 2 * gi + m, bi);
      for (int h = 0; h < v_tiles; ++h) tma_load_4d(sV(h), &tmap_v, bar_kv, 64 * h, k0, gi, bi);
      int hi = gi * prm.group, qt = q_begin;
      for (int it = 0; it < n_it; ++it) {
        const int st = it % kStages, qrow = qt * 64;
        if (it >= kStages && !mbar_wait(bar_free(st), ((it / kStages) - 1) & 1, &abort_flag, prm.status, BAR_FREE)) break;
        mbar_arrive_expect_tx(bar_full(st), (2 + v_tiles) * kSlotBytes + kVecBytes);
        for (int h = 0; h < v_tiles; ++h) tma_load_4d(sStage(st) + (2 + h) * kSlotBytes, &tmap_g, bar_full(st), 64 * h, qrow, hi, bi);
        for (int m = 0; m < 2; ++m) tma_load_4d(sStage(st) + m * kSlotBytes, &tmap_q, bar_full(st), 0, qrow, 2 * hi + m, bi);
        const float* src = prm.stats + (static_cast<int64_t>(bi) * p.heads + hi) * 4 * prm.n_pad + qrow;
        for (int a = 0; a < 4; ++a) bulk_load_1d(smem_base + vec_off + st * kVecBytes + 256 * a, src + a * prm.n_pad, 256, bar_full(st));
        if (++qt == n_q64) { qt = q_begin; ++hi; }
      }
    }
  } else if (warp_u == kIssuerWarp) {
    if (n_it > 0) {
      const bool leader = elect_one();
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_k = make_idesc(fmt, 0, 0, 128, 64);    // S_m^T, G^T: A, B K-major, N = 64 queries
      constexpr uint32_t idesc_mn = make_idesc(fmt, 0, 1, 128, 64);   // dK_m: B (Q_m) MN-major, N = 64
      const uint32_t idesc_v = v_tiles == 2 ? make_idesc(fmt, 0, 1, 128, 128) : idesc_mn;   // dV: B (g) MN-major
      const uint64_t dk[2] = {make_sdesc(sK(0), 16, 1024), make_sdesc(sK(1), 16, 1024)};
      const uint64_t dv[2] = {make_sdesc(sV(0), 16, 1024), make_sdesc(sV(1), 16, 1024)};
      const uint64_t dds2 = make_sdesc(sDS2, 16, 1024);
      const uint64_t ds0 = make_sdesc(sStage(0), 16, 1024);
      const uint64_t dmn0 = make_sdesc(sStage(0), kSlotBytes, 1024);  // (leading offset: from g's one 64-column half to the other)
      bool ok = mbar_wait_warp(bar_kv, 0, &abort_flag, prm.status, BAR_STAGE);
      auto issue_sg = [&](int it) {
        const int st = it % kStages;
        if (!(ok = mbar_wait_warp(bar_full(st), (it / kStages) & 1, &abort_flag, prm.status, BAR_FULL))) return;
        tc_fence_after();
        const uint64_t d = ds0 + st * kStageStep;
        for (int h = 0; h < v_tiles; ++h)
          if (leader) mma_ss_x4<2, 2>(tG, dv[h], d + (2 + h) * kSlotStep, idesc_k, h == 0 ? 0u : 1u);
        for (int m = 0; m < 2; ++m)
          if (leader) mma_ss_x4<2, 2>(tS + 64 * m, dk[m], d + m * kSlotStep, idesc_k, 0u);
        if (leader) mma_commit(bar_sg);
      };
      if (ok) {
        tc_fence_after();
        issue_sg(0);
      }
      for (int it = 0; ok && it < n_it; ++it) {
        if (it + 1 < n_it) {
          if (!(ok = mbar_wait_warp(bar_sfree, it & 1, &abort_flag, prm.status, BAR_SFREE))) break;
          tc_fence_after();
          issue_sg(it + 1);
          if (!ok) break;
        }
        if (!(ok = mbar_wait_warp(bar_ds, it & 1, &abort_flag, prm.status, BAR_DS))) break;
        tc_fence_after();
        const int st = it % kStages;
        const uint32_t acc = it == 0 ? 0u : 1u;
        const uint64_t d = dmn0 + st * kStageStep;
        if (leader) mma_ts_x4<8, 128>(tdV, tP, d + 2 * kSlotStep, idesc_v, acc);
        if (leader) mma_ts_x4<8, 128>(tdK, tDS1, d, idesc_mn, acc);
        if (leader) mma_ss_x4<2, 128>(tdK + 64, dds2, d + kSlotStep, idesc_mn, acc);
        if (leader) mma_commit(bar_free(st));
        if (leader) mma_commit(bar_acc);
      }
    }
  } else {
    // ---------------- fold warps: four threads per key row, 16 queries each ----------------
    const int qd = warp & 3, cq = warp >> 2;
    const int row = qd * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(qd * 32) << 16;
    const int key = k0 + row;
    const float c = p.scale_log2;
    // this thread's 32 bytes of row `row` of dS2^T: 16-byte pieces 2 cq and 2 cq + 1, swizzled
    const uint32_t ds2_row = sDS2 + row * 128, piece0 = ((2 * cq) ^ (row & 7)) * 16, piece1 = ((2 * cq + 1) ^ (row & 7)) * 16;
    bool alive = true;
    int hi = gi * prm.group, qt = q_begin;
    float nlam = n_it > 0 ? -diff_lam(p, hi) : 0.f;
    for (int it = 0; it < n_it; ++it) {
      const int st = it % kStages, q_tile0 = qt * 64;
      if (!mbar_wait_warp(bar_sg, it & 1, &abort_flag, prm.status, BAR_SG)) { alive = false; break; }
      // (the row statistics came by bulk copies that complete on the stage's barrier: observe it directly)
      if (!mbar_wait_warp(bar_full(st), (it / kStages) & 1, &abort_flag, prm.status, BAR_FULL)) { alive = false; break; }
      tc_fence_after();
      uint32_t pk[8], d1[8], d2[8];
      {
        uint32_t s1[16], s2[16], g[16];
        tmem_ld16(tS + lane_off + 16 * cq, s1);
        tmem_ld16(tS + 64 + lane_off + 16 * cq, s2);
        tmem_ld16(tG + lane_off + 16 * cq, g);
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive_warp(bar_sfree, lane);
        const float4* vec = reinterpret_cast<const float4*>(smem_gen + vec_off + st * kVecBytes) + 4 * cq;
        const int qc = q_tile0 + 16 * cq;
        const bool masked = p.causal && q_tile0 + shift < k0 + 127;    // some query of the tile does not see some key
        const float2 c2 = make_float2(c, c), lam2 = make_float2(nlam, nlam);
        auto tile = [&](auto with_mask) {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            const float4 l1 = vec[i4], l2 = vec[16 + i4], e1 = vec[32 + i4], e2 = vec[48 + i4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int i = 4 * i4 + 2 * h;
              const float2 nl1 = h ? make_float2(l1.z, l1.w) : make_float2(l1.x, l1.y), nl2 = h ? make_float2(l2.z, l2.w) : make_float2(l2.x, l2.y);
              const float2 nd1 = h ? make_float2(e1.z, e1.w) : make_float2(e1.x, e1.y), nd2 = h ? make_float2(e2.z, e2.w) : make_float2(e2.x, e2.y);
              const float2 gv = pair(g, i);
              float2 x1 = exp2_pair(__ffma2_rn(pair(s1, i), c2, nl1)), x2 = exp2_pair(__ffma2_rn(pair(s2, i), c2, nl2));
              if (decltype(with_mask)::value) {
                if (key > qc + i + shift) x1.x = x2.x = 0.f;
                if (key > qc + i + 1 + shift) x1.y = x2.y = 0.f;
              }
              x2 = __fmul2_rn(x2, lam2);
              const float2 pv = __fadd2_rn(x1, x2), a = __fmul2_rn(x1, __fadd2_rn(gv, nd1)), b = __fmul2_rn(x2, __fadd2_rn(gv, nd2));
              pk[i >> 1] = pack2<T>(pv.x, pv.y);
              d1[i >> 1] = pack2<T>(a.x, a.y);
              d2[i >> 1] = pack2<T>(b.x, b.y);
            }
          }
        };
        if (masked) tile(std::true_type{});
        else tile(std::false_type{});
      }
      if (it > 0) {
        // the products of the tile before have read what is overwritten now
        if (!mbar_wait_warp(bar_acc, (it - 1) & 1, &abort_flag, prm.status, BAR_ACC)) { alive = false; break; }
        tc_fence_after();
      }
      tmem_st8(tP + lane_off + 8 * cq, pk);
      tmem_st8(tDS1 + lane_off + 8 * cq, d1);
      st_shared_v4(ds2_row + piece0, d2[0], d2[1], d2[2], d2[3]);
      st_shared_v4(ds2_row + piece1, d2[4], d2[5], d2[6], d2[7]);
      tmem_wait_st();
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive_warp(bar_ds, lane);
      if (++qt == n_q64) {
        qt = q_begin;
        if (++hi < (gi + 1) * prm.group) nlam = -diff_lam(p, hi);
      }
    }
    if (alive && n_it > 0) alive = mbar_wait_warp(bar_acc, (n_it - 1) & 1, &abort_flag, prm.status, BAR_ACC);
    if (alive) {
      tc_fence_after();
#pragma unroll
      for (int x = 0; x < 4; ++x) {            // dK1, dK2, dV (0-63), dV (64-127); tcgen05.ld is warp-collective: only the stores are predicated
        uint32_t r[16];
        if (n_it > 0) {
          tmem_ld16((x < 2 ? tdK + 64 * x : tdV + 64 * (x - 2)) + lane_off + 16 * cq, r);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) r[i] = 0u;         // no query sees these keys: zero gradients
        }
        if (key < p.nk) {
          if (x < 2) store16<T>(static_cast<T*>(p.dk) + bi * p.dks.b + (2 * gi + x) * p.dks.h + static_cast<int64_t>(key) * p.dks.r + 16 * cq, r, p.scale, p.head_dim - 16 * cq);
          else store16<T>(static_cast<T*>(p.dv) + bi * p.dvs.b + gi * p.dvs.h + static_cast<int64_t>(key) * p.dvs.r + 64 * (x - 2) + 16 * cq, r, 1.f, p.v_dim - 64 * (x - 2) - 16 * cq);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kProducerWarp) tmem_dealloc(tmem_base, kTmemCols);
}

// Both bodies in one launch, the longer CTAs (dK, dV) first
template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
diff_bwd_kernel(const __grid_constant__ CUtensorMap tmap_q128, const __grid_constant__ CUtensorMap tmap_g128,
                const __grid_constant__ CUtensorMap tmap_q64, const __grid_constant__ CUtensorMap tmap_g64,
                const __grid_constant__ CUtensorMap tmap_k128, const __grid_constant__ CUtensorMap tmap_v128,
                const __grid_constant__ CUtensorMap tmap_k64, const __grid_constant__ CUtensorMap tmap_v64, const BwdParams2 prm) {
  const int z = blockIdx.z;
  if (z < prm.d.batch) diff_dkv_body<T>(tmap_q64, tmap_g64, tmap_k128, tmap_v128, prm, z);
  else diff_dq_body<T>(tmap_q128, tmap_g128, tmap_k64, tmap_v64, prm, z - prm.d.batch);
}

}  // namespace

int diff_bwd_tc(const DiffParams& p, const float* stats, int dtype, cudaStream_t st) {
  CUtensorMap mq[2], mg[2], mk[2], mv[2];                  // boxes of 128 and of 64 rows
  int rc;
  for (int i = 0; i < 2; ++i) {
    const int box = i == 0 ? 128 : 64;
    if ((rc = make_tmap_rows64(&mq[i], p.q, dtype, p.nq, 2 * p.heads, p.batch, p.qs, box, p.head_dim)) != ELSA_OK) return rc;
    if ((rc = make_tmap_rows64(&mg[i], p.dout, dtype, p.nq, p.heads, p.batch, p.gs, box, p.v_dim)) != ELSA_OK) return rc;
    if (p.nk > 0) {
      if ((rc = make_tmap_rows64(&mk[i], p.k, dtype, p.nk, 2 * p.kv_heads, p.batch, p.ks, box, p.head_dim)) != ELSA_OK) return rc;
      if ((rc = make_tmap_rows64(&mv[i], p.v, dtype, p.nk, p.kv_heads, p.batch, p.vs, box, p.v_dim)) != ELSA_OK) return rc;
    } else {
      mk[i] = mv[i] = mq[i];                               // no key tile is visited
    }
  }
  BwdParams2 prm;
  prm.d = p;
  prm.stats = stats;
  prm.n_pad = static_cast<int>(align_up(p.nq, 128));
  prm.group = p.heads / p.kv_heads;
  if ((rc = device_status_word(&prm.status, nullptr)) != ELSA_OK) return rc;
  if (2 * static_cast<int64_t>(p.batch) > 65535) return ELSA_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>((std::max(p.nq, p.nk) + 127) / 128), static_cast<unsigned>(p.heads), static_cast<unsigned>(2 * p.batch));
  auto launch = [&](auto kernel) -> int {
    const int r = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmem);
    if (r != ELSA_OK) return r;
    kernel<<<grid, kThreads, kSmem, st>>>(mq[0], mg[0], mq[1], mg[1], mk[0], mv[0], mk[1], mv[1], prm);
    return ELSA_OK;
  };
  rc = dtype == ELSA_F16 ? launch(&diff_bwd_kernel<__half>) : launch(&diff_bwd_kernel<__nv_bfloat16>);
  if (rc != ELSA_OK) return rc;
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

}  // namespace elsa
