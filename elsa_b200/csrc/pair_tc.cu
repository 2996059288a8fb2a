// Two softmax chains over one stream of keys and values, on the 5th-generation tensor cores (fp16 / bf16):
//
//   Diff        the two maps of 128 query rows of one head of the differential attention: keys of their own, the values shared
//   Rows64/128  two tiles of 128 query rows that read the same key head of a shared cache (head dim <= 64, <= 128): keys and values shared
//
// One CTA, one per SM.  64-key tiles through a ring (TMA, 128-byte swizzle):
//
//   warp 8      TMA producer
//   warp 9, 10  MMA issuers   one for each chain t:  S_t(j) = Q_t K_t^T   (tcgen05.mma 128x64x16, shared-memory operands)
//                                                    O_t   += P_t V       (tcgen05.mma 128xDx16, P from TMEM, V MN-major)
//   warps 0-3   fold of chain 0  one thread per query row: 64 scores into registers, running max, exp2, row sum, P (16-bit) into TMEM,
//   warps 4-7   fold of chain 1  rescale of O when the max moved
//
// TMEM columns: chain t has S_t at 128 t, two tiles of P_t at 128 t + 64 and + 96, and O_t at 256 + 128 t.  S_t(j + 1) is issued as soon as the
// fold holds S_t(j) in registers and runs during the exponentials of tile j; a fold warp waits for the tensor pipe only when its
// maximum moves.  Measured, (2, 8, 8192, 64 / 128) causal bf16: 128-key tiles, whose P has no columns of its own, so that scores,
// exponentials and P V of a chain follow one another, 460 us; 64-key tiles with two S_t, P over the scores it comes from, 460 (the
// scores of tile j + 1 wait for P V of tile j - 1); the latter with the next scores read ahead of the exponentials 550;
// this form 460 to 490 by the card and its clock (1.75 GHz under the power cap).  Rows128: 0.72 us a tile with few CTAs on the card, 0.9 with
// all of them, and about 10 us of a CTA besides its tiles (14 when each thread fetched its own query row and wrote its own row of sums).
//
// Bound: the ex2 unit, 2 x 128 x 64 exponentials for each tile (1024 cycles; the tensor pipe, limited by its shared-memory operands,
// needs 900 for Diff and 1280 for Rows128).
//
// The reference max of a row moves only when it is exceeded by more than 2^8; a row's result does not depend on the rows beside it.
// P is rounded to the inputs' type (its error, half a step in each weight, averages out over the keys); sums and statistics are fp32.
// Diff: each map is normalised by its own sum at the end; lam O_1 / z_1 goes through shared memory to the threads that hold the same rows
// of O_0.  Rows: a warp gathers its query rows into the swizzled operand (rows of a kv head are not evenly spaced in q) and writes its rows'
// summaries through shared memory.
#include <type_traits>

#include "pair_tc.cuh"
#include "tc_common.cuh"

namespace elsa {

using namespace tc;

namespace {

enum Mode { kDiff, kRows64, kRows128 };

constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;
constexpr int kProducerWarp = 8, kIssuerWarp = 9;
constexpr float kRescaleThreshold = 8.0f;
constexpr int kTileBytes = 128 * 64 * 2;                           // 128 query rows x 64 columns
constexpr int kSlotBytes = 64 * 64 * 2;                            // 64 keys x 64 columns

template <int MODE> struct Shape {
  static constexpr int kQHalves = MODE == kRows128 ? 2 : 1;        // 64-column halves of a query row
  static constexpr int kKSlots = MODE == kRows64 ? 1 : 2;          // K slots of a stage: of either chain (Diff), or halves
  static constexpr int kVSlots = MODE == kRows64 ? 1 : 2;          // halves of V
  static constexpr int kStageSlots = kKSlots + kVSlots;
  static constexpr int kStageBytes = kStageSlots * kSlotBytes;
  static constexpr int kStages = MODE == kRows128 ? 5 : MODE == kDiff ? 6 : 8;
  static constexpr int kSmem = 2 * kQHalves * kTileBytes + kStages * kStageBytes + 1024;   // + alignment slack
};

enum BarId { BAR_Q = 71, BAR_KV_FULL = 72, BAR_KV_FREE = 73, BAR_S = 74, BAR_P = 75, BAR_PV = 76, BAR_STAGGER = 77, BAR_O = 78, BAR_SFREE = 79 };

struct PairParams {
  DiffParams d;                  // Diff
  DecodeParams r;                // Rows
  int part_width;
  int group;
  int* status;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 32 consecutive values of a row, of which the first n (a multiple of 8, possibly <= 0) exist
template <typename T>
__device__ __forceinline__ void store32(T* dst, const float (&v)[32], int n) {
  constexpr int kStep = sizeof(T) == 4 ? 4 : 8;
#pragma unroll
  for (int i = 0; i < 32; i += kStep) {
    if (i >= n) continue;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
      uint4 t;
      t.x = pack2<T>(v[i], v[i + 1]); t.y = pack2<T>(v[i + 2], v[i + 3]);
      t.z = pack2<T>(v[i + 4], v[i + 5]); t.w = pack2<T>(v[i + 6], v[i + 7]);
      *reinterpret_cast<uint4*>(dst + i) = t;
    }
  }
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
pair_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
            const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PairParams prm) {
  using Sh = Shape<MODE>;
  constexpr int kStages = Sh::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 14];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const DiffParams& p = prm.d;
  const DecodeParams& rp = prm.r;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int warp_u = __shfl_sync(0xffffffffu, warp, 0);   // (known to be warp-uniform)
  // Diff: x = query tile, y = head, z = batch.  Rows: x = 256-row tile, y = part, z = kv head.
  int q0, k_begin = 0, k_end, bi = 0, hi = 0, gi, shift = 0;
  if constexpr (MODE == kDiff) {
    hi = blockIdx.y; bi = blockIdx.z; gi = hi / prm.group;
    // causal: the long tiles first
    q0 = (p.causal ? static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x)) * 128;
    shift = p.nk - p.nq;                                   // causal: row i sees keys up to i + shift
    k_end = p.causal ? min(p.nk, min(q0 + 128, p.nq) + shift) : p.nk;
  } else {
    gi = blockIdx.z;
    q0 = blockIdx.x * 256;
    k_begin = blockIdx.y * prm.part_width;
    k_end = min(rp.seg[0].n_keys, k_begin + prm.part_width);
  }
  const int n_t = k_end > k_begin ? (k_end - k_begin + 63) / 64 : 0;   // 64-key tiles, the same for both chains
  const int v_dim = MODE == kDiff ? p.v_dim : rp.v_dim;
  const int v_halves = Sh::kVSlots == 1 ? 1 : v_dim > 64 ? 2 : 1;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  auto q_off = [&](int t, int h) { return static_cast<uint32_t>((t * Sh::kQHalves + h) * kTileBytes); };
  const uint32_t ring = smem_base + 2 * Sh::kQHalves * kTileBytes;
  auto sK = [&](int st) { return ring + st * Sh::kStageBytes; };
  auto sV = [&](int st) { return ring + st * Sh::kStageBytes + Sh::kKSlots * kSlotBytes; };
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t bar_q = bar0, bar_stagger = bar0 + 8;
  auto bar_kv_full = [&](int st) { return bar0 + 8 * (2 + st); };
  auto bar_kv_free = [&](int st) { return bar0 + 8 * (2 + kStages + st); };
  auto bar_s = [&](int t) { return bar0 + 8 * (2 + 2 * kStages + t); };                    // S_t(j) is in TMEM
  auto bar_sfree = [&](int t) { return bar0 + 8 * (4 + 2 * kStages + t); };                // the fold warps hold it in registers
  // P_t(j) has been delivered: one for either tile, because P_t(j + 1) can be there before the issuer has looked at P_t(j)'s
  auto bar_p = [&](int t, int b) { return bar0 + 8 * (6 + 2 * kStages + 2 * t + b); };
  auto bar_pv = [&](int t) { return bar0 + 8 * (10 + 2 * kStages + t); };                  // P_t V of tile j has retired
  auto bar_o = [&](int t) { return bar0 + 8 * (12 + 2 * kStages + t); };                   // ... of the last tile

  if (MODE != kDiff) let_next_begin();                  // (the split kernel of the sequences' own keys, on the SMs that are free)
  if (tid == 0) {
    abort_flag = 0;
    mbar_init(bar_q, MODE == kDiff ? 1 : 8);
    mbar_init(bar_stagger, 1);
    for (int st = 0; st < kStages; ++st) { mbar_init(bar_kv_full(st), 1); mbar_init(bar_kv_free(st), 2); }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar_s(t), 1); mbar_init(bar_sfree(t), 4);
      for (int b = 0; b < 2; ++b) mbar_init(bar_p(t, b), 4);
      mbar_init(bar_pv(t), 1); mbar_init(bar_o(t), 1);
    }
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
  auto tS = [&](int t) { return tmem_base + 128 * t; };
  auto tP = [&](int t, int b) { return tmem_base + 128 * t + 64 + 32 * b; };
  auto tO = [&](int t) { return tmem_base + 256 + 128 * t; };

  // registers: 3 x 128 threads, 232 + 232 + 40 = 3 x 168, the launch allocation (see fold_tc.cu)
  if (warp_u >= 8) {
    reg_dec<40>();
    if (n_t > 0 && warp == kProducerWarp) {
      // ---------------- TMA producer ----------------
      if (lane == 0) {
        if constexpr (MODE == kDiff) {
          prefetch_tmap(&tmap_q);
          mbar_arrive_expect_tx(bar_q, 2 * kTileBytes);
          for (int t = 0; t < 2; ++t) tma_load_4d(smem_base + q_off(t, 0), &tmap_q, bar_q, 0, q0, 2 * hi + t, bi);
        }
        prefetch_tmap(&tmap_k); prefetch_tmap(&tmap_v);
        for (int j = 0; j < n_t; ++j) {
          const int st = j % kStages, key = k_begin + j * 64;
          if (j >= kStages && !mbar_wait(bar_kv_free(st), ((j / kStages) - 1) & 1, &abort_flag, prm.status, BAR_KV_FREE)) break;
          mbar_arrive_expect_tx(bar_kv_full(st), (Sh::kKSlots + v_halves) * kSlotBytes);
          for (int s = 0; s < Sh::kKSlots; ++s)            // Diff: the chains' keys; Rows: the key's halves
            tma_load_4d(sK(st) + s * kSlotBytes, &tmap_k, bar_kv_full(st), MODE == kDiff ? 0 : 64 * s, key, MODE == kDiff ? 2 * gi + s : gi, bi);
          for (int h = 0; h < v_halves; ++h) tma_load_4d(sV(st) + h * kSlotBytes, &tmap_v, bar_kv_full(st), 64 * h, key, gi, bi);
        }
      }
    } else if (n_t > 0 && (warp_u == kIssuerWarp || warp_u == kIssuerWarp + 1)) {
      // ---------------- MMA issuers: one for each chain ----------------
      const int t = warp_u - kIssuerWarp;
      const bool leader = elect_one();
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_s = make_idesc(fmt, 0, 0, 128, 64);                                          // S = Q K^T : A, B K-major
      const uint32_t idesc_o = v_halves == 2 ? make_idesc(fmt, 0, 1, 128, 128) : make_idesc(fmt, 0, 1, 128, 64);   // O += P V : A in TMEM, B MN-major
      const uint64_t dq = make_sdesc(smem_base + q_off(t, 0), 16, 1024);
      const uint64_t dk0 = make_sdesc(sK(0) + (MODE == kDiff ? t * kSlotBytes : 0), 16, 1024);
      const uint64_t dv0 = make_sdesc(sV(0), kSlotBytes, 1024);       // (leading offset: from one 64-column half to the other)
      constexpr uint64_t kStageStep = Sh::kStageBytes >> 4;           // descriptor address field counts 16-byte units
      bool ok = mbar_wait_warp(bar_q, 0, &abort_flag, prm.status, BAR_Q);
      auto issue_s = [&](int j) {
        const int st = j % kStages;
        if (!(ok = mbar_wait_warp(bar_kv_full(st), (j / kStages) & 1, &abort_flag, prm.status, BAR_KV_FULL))) return;
        if (j > 0 && !(ok = mbar_wait_warp(bar_sfree(t), (j - 1) & 1, &abort_flag, prm.status, BAR_SFREE))) return;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < Sh::kQHalves; ++h)
          if (leader) mma_ss_x4<2, 2>(tS(t), dq + h * (kTileBytes >> 4), dk0 + st * kStageStep + h * (kSlotBytes >> 4), idesc_s, h == 0 ? 0u : 1u);
        if (leader) mma_commit(bar_s(t));
      };
      // chain 1 starts half a period after chain 0: in step they would want the ex2 unit at the same time
      if (ok && t == 1) ok = mbar_wait_warp(bar_stagger, 0, &abort_flag, prm.status, BAR_STAGGER);
      if (ok) issue_s(0);
      for (int j = 0; ok && j < n_t; ++j) {
        const int st = j % kStages;
        if (j + 1 < n_t) {
          issue_s(j + 1);
          if (!ok) break;
        }
        if (t == 0 && j == 0 && leader) mbar_arrive(bar_stagger);
        if (!(ok = mbar_wait_warp(bar_p(t, j & 1), (j >> 1) & 1, &abort_flag, prm.status, BAR_P))) break;
        tc_fence_after();
        if (leader) mma_ts_x4<8, 128>(tO(t), tP(t, j & 1), dv0 + st * kStageStep, idesc_o, j > 0 ? 1u : 0u);
        if (leader) mma_commit(bar_pv(t));
        if (leader) mma_commit(bar_kv_free(st));  // this chain no longer reads the stage
      }
      if (ok && leader) mma_commit(bar_o(t));
    }
  } else {
    reg_inc<232>();
    // ---------------- fold warps: one thread per query row and chain ----------------
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;                 // row within the tile == TMEM lane
    const int qi = MODE == kDiff ? q0 + row : q0 + 128 * t + row;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float c = MODE == kDiff ? p.scale_log2 : rp.scale_log2;
    if constexpr (MODE != kDiff) {
      // this warp's query rows into the operand tile: 16-byte piece x of row r of a 64-column half at piece x ^ (r & 7).  A lane finds its own
      // row's place in q; then 8 or 16 lanes fetch a row together.
      const int rows = static_cast<int>(decode_rows(rp)), pieces = rp.head_dim / 8;
      unsigned long long src = 0;
      if (qi < rows) {
        const int per = prm.group * rp.nq, b = qi / per, r = qi - b * per, h = r / rp.nq, i = r - h * rp.nq;
        src = reinterpret_cast<unsigned long long>(static_cast<const T*>(rp.q) + b * rp.qs.b + static_cast<int64_t>(gi * prm.group + h) * rp.qs.h + i * rp.qs.r);
      }
      constexpr int kLanes = 8 * Sh::kQHalves, kPass = 32 / kLanes;      // lanes of a row, rows of one access
      const int piece = lane % kLanes;
      uint4 v[kLanes];
#pragma unroll
      for (int x = 0; x < kLanes; ++x) {
        const unsigned long long at = __shfl_sync(0xffffffffu, src, x * kPass + lane / kLanes);
        v[x] = at && piece < pieces ? reinterpret_cast<const uint4*>(at)[piece] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int x = 0; x < kLanes; ++x) {
        const int r = (warp & 3) * 32 + x * kPass + lane / kLanes;
        *reinterpret_cast<uint4*>(smem_gen + q_off(t, piece / 8) + r * 128 + ((piece % 8 ^ (r & 7)) << 4)) = v[x];
      }
      fence_proxy_async_smem();
      mbar_arrive_warp(bar_q, lane);
    }
    float m_ref = -CUDART_INF_F, zsum = 0.f;
    bool alive = true;
    // last key of this row
    const int lim = MODE == kDiff && p.causal ? min(p.nk - 1, qi + shift) : k_end - 1;

    for (int j = 0; j < n_t; ++j) {
      // (S(j) was issued behind P V of tile j - 2: its P may be overwritten)
      if (!mbar_wait_warp(bar_s(t), j & 1, &abort_flag, prm.status, BAR_S)) { alive = false; break; }
      tc_fence_after();
      float sv[64];
      {
        uint32_t ra[32], rb[32];
        tmem_ld32(tS(t) + lane_off, ra);
        tmem_ld32(tS(t) + lane_off + 32, rb);
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive_warp(bar_sfree(t), lane);      // S_t may be overwritten with the next tile's scores
#pragma unroll
        for (int i = 0; i < 32; ++i) { sv[i] = __uint_as_float(ra[i]); sv[32 + i] = __uint_as_float(rb[i]); }
      }
      const int k0 = k_begin + j * 64;
      if (__builtin_expect(k0 + 64 > k_end || (MODE == kDiff && p.causal && k0 + 63 > q0 + shift), 0)) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (k0 + i > lim) sv[i] = -CUDART_INF_F;
      }
      float mx[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
      for (int i = 4; i < 60; i += 8) {                      // (four independent chains of three-input maxima)
        mx[0] = max3(mx[0], sv[i], sv[i + 1]); mx[1] = max3(mx[1], sv[i + 2], sv[i + 3]);
        mx[2] = max3(mx[2], sv[i + 4], sv[i + 5]); mx[3] = max3(mx[3], sv[i + 6], sv[i + 7]);
      }
      mx[0] = max3(mx[0], sv[60], sv[61]); mx[1] = max3(mx[1], sv[62], sv[63]);
      const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
      const bool move = tmax > m_ref + kRescaleThreshold;   // also true for the first tile with a key of this row (m_ref = -inf)
      if (__builtin_expect(__any_sync(0xffffffffu, move), 0)) {
        const float m_new = move ? tmax : m_ref;             // (a row's result does not depend on the rows beside it)
        const float alpha = move ? fast_exp2(m_ref - m_new) : 1.f;
        zsum *= alpha;
        if (j > 0) {
          // O_t holds P V of the tiles before: the last of them has to have retired.  (Its phase is the
          // one that is awaited: the P V before it has retired, since S(j) was issued behind it.)
          if (!mbar_wait_warp(bar_pv(t), (j - 1) & 1, &abort_flag, prm.status, BAR_PV)) { alive = false; break; }
          tc_fence_after();
          for (int h = 0; h < 2 * v_halves; ++h) {
            uint32_t r[32];
            tmem_ld32(tO(t) + lane_off + 32 * h, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st32(tO(t) + lane_off + 32 * h, r);
          }
        }
        m_ref = m_new;
      }
      const float m_use = (m_ref == -CUDART_INF_F) ? 0.f : m_ref;
      const float2 c2 = make_float2(c, c), nm2 = make_float2(-m_use, -m_use);
      float2 ps[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t pk[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float2 x = __ffma2_rn(make_float2(sv[2 * i], sv[2 * i + 1]), c2, nm2);
        const float2 pp = make_float2(fast_exp2(x.x), fast_exp2(x.y));
        ps[i & 3] = __fadd2_rn(ps[i & 3], pp);
        pk[i] = pack2<T>(pp.x, pp.y);
      }
      tmem_st32(tP(t, j & 1) + lane_off, pk);
      tmem_wait_st();               // (also covers the O rescale stores above)
      tc_fence_before();
      mbar_arrive_warp(bar_p(t, j & 1), lane);
      const float2 s01 = __fadd2_rn(ps[0], ps[1]), s23 = __fadd2_rn(ps[2], ps[3]);
      const float2 s = __fadd2_rn(s01, s23);
      zsum += s.x + s.y;
    }
    if (alive && n_t > 0) alive = mbar_wait_warp(bar_o(t), 0, &abort_flag, prm.status, BAR_O);
    tc_fence_after();

    if constexpr (MODE == kDiff) {
      // Map 1 leaves lam O_1 / z_1 in shared memory, [column][row] (over the ring: every load has been waited for, and every MMA that read
      // it has to have retired), map 0 takes it.
      const bool row_ok = qi < p.nq;
      const int64_t ro = (static_cast<int64_t>(bi) * p.heads + hi) * p.nq + qi;
      float* exchange = reinterpret_cast<float*>(smem_gen + 2 * kTileBytes);
      const float inv = zsum != 0.f ? 1.f / zsum : 0.f;       // (NaN stays NaN)
      if (p.lse && row_ok && alive) p.lse[t * (static_cast<int64_t>(p.batch) * p.heads * p.nq) + ro] = zsum != 0.f ? m_ref + log2f(zsum) : -CUDART_INF_F;
      if (t == 1 && n_t > 0) {
        if (alive) alive = mbar_wait_warp(bar_o(0), 0, &abort_flag, prm.status, BAR_O);
        const float lam = diff_lam(p, hi);
        for (int h = 0; h < 2 * v_halves; ++h) {
          uint32_t r[32];
          tmem_ld32(tO(1) + lane_off + 32 * h, r);
          tmem_wait_ld();
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = zsum != 0.f ? __uint_as_float(r[i]) * inv : 0.f;
          if (alive) {
#pragma unroll
            for (int i = 0; i < 32; ++i) exchange[(32 * h + i) * 128 + row] = lam * o[i];
          }
          if (p.out2 && row_ok && alive) store32<T>(static_cast<T*>(p.out2) + ro * p.v_dim + 32 * h, o, p.v_dim - 32 * h);
        }
      } else if (t == 1 && p.out2 && row_ok) {
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.f;
        for (int h = 0; h < 4; ++h) store32<T>(static_cast<T*>(p.out2) + ro * p.v_dim + 32 * h, o, p.v_dim - 32 * h);
      }
      named_barrier_sync(1, 256);
      if (t == 0) {
        T* dst = static_cast<T*>(p.out) + bi * p.os.b + hi * p.os.h + static_cast<int64_t>(qi) * p.os.r;
        for (int h = 0; h < 2 * v_halves; ++h) {
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
          if (n_t > 0) {
            uint32_t r[32];
            tmem_ld32(tO(0) + lane_off + 32 * h, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = (zsum != 0.f ? __uint_as_float(r[i]) * inv : 0.f) - exchange[(32 * h + i) * 128 + row];
          }
          if (row_ok && alive) store32<T>(dst + 32 * h, o, p.v_dim - 32 * h);
        }
      }
    } else {
      const int rows = static_cast<int>(decode_rows(rp));
      const bool row_ok = qi < rows && alive;
      const int64_t ro = (static_cast<int64_t>(blockIdx.y) * rp.kv_heads + gi) * rows + qi;
      if (row_ok) {
        rp.m[ro] = zsum != 0.f ? m_ref : -CUDART_INF_F;
        rp.z[ro] = zsum;
      }
      // The warp's 32 rows of sums stand side by side in memory: through shared memory (over the ring, which neither chain reads any more),
      // so that whole lines are written.
      if (alive && n_t > 0) alive = mbar_wait_warp(bar_o(1 - t), 0, &abort_flag, prm.status, BAR_O);
      constexpr int kPitch = 64 * Sh::kVSlots + 4;         // (rows 16 bytes apart in the banks)
      float* buffer = reinterpret_cast<float*>(smem_gen + 2 * Sh::kQHalves * kTileBytes) + warp * 32 * kPitch;
      for (int h = 0; h < 2 * v_halves; ++h) {
        uint32_t r[32];
        tmem_ld32(tO(t) + lane_off + 32 * h, r);
        tmem_wait_ld();
        if (alive) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<uint4*>(buffer + lane * kPitch + 32 * h + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
      }
      __syncwarp();
      const int vecs = v_dim / 4, first = qi - lane, n_vecs = alive ? min(32, rows - first) * vecs : 0;
      float4* dst = reinterpret_cast<float4*>(rp.s + (ro - lane) * v_dim);
#pragma unroll 1
      for (int i = lane; i < n_vecs; i += 32) dst[i] = *reinterpret_cast<const float4*>(buffer + i / vecs * kPitch + i % vecs * 4);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kProducerWarp) tmem_dealloc(tmem_base, kTmemCols);
}

template <typename T, int MODE>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PairParams& prm, dim3 grid, cudaStream_t st) {
  const auto kernel = &pair_kernel<T, MODE>;
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), Shape<MODE>::kSmem);
  if (rc != ELSA_OK) return rc;
  kernel<<<grid, kThreads, Shape<MODE>::kSmem, st>>>(mq, mk, mv, prm);
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

}  // namespace

bool diff_tc_sizes(int dtype, int head_dim, int v_dim) {
  return head_dim <= 64 && v_dim <= 128 && v_dim >= 8 && v_dim % 8 == 0 && fold_tc_supported(dtype, head_dim, false);
}

// 16-byte rows for the tensor maps; an axis of one may have any stride
bool diff_rows_ok(const void* base, const Strides& s, int row, int heads, int batch) {
  return !(reinterpret_cast<uintptr_t>(base) & 15u) && s.r >= row && s.r % 8 == 0 && (heads == 1 || (s.h > 0 && s.h % 8 == 0)) &&
         (batch == 1 || (s.b > 0 && s.b % 8 == 0));
}

int diff_tc_fwd(const DiffParams& p, int dtype, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  int rc;
  if ((rc = make_tmap_rows64(&mq, p.q, dtype, p.nq, 2 * p.heads, p.batch, p.qs, 128, p.head_dim)) != ELSA_OK) return rc;
  if (p.nk > 0) {
    if ((rc = make_tmap_rows64(&mk, p.k, dtype, p.nk, 2 * p.kv_heads, p.batch, p.ks, 64, p.head_dim)) != ELSA_OK) return rc;
    if ((rc = make_tmap_rows64(&mv, p.v, dtype, p.nk, p.kv_heads, p.batch, p.vs, 64, p.v_dim)) != ELSA_OK) return rc;
  } else {
    mk = mv = mq;                                          // no key tile is visited
  }
  PairParams prm{};
  prm.d = p;
  prm.group = p.heads / p.kv_heads;
  if ((rc = device_status_word(&prm.status, nullptr)) != ELSA_OK) return rc;
  const dim3 grid(static_cast<unsigned>((p.nq + 127) / 128), static_cast<unsigned>(p.heads), static_cast<unsigned>(p.batch));
  return dtype == ELSA_F16 ? launch<__half, kDiff>(mq, mk, mv, prm, grid, st) : launch<__nv_bfloat16, kDiff>(mq, mk, mv, prm, grid, st);
}

bool rows_tc_ok(const DecodeParams& p, int dtype) {
  const DecodeSegment& s = p.seg[0];
  if (p.maps != 1 || p.v_dim != p.head_dim || !(fold_tc_supported(dtype, p.head_dim, false) || fold_tcw_supported(dtype, p.head_dim, false))) return false;
  return !((p.qs.b | p.qs.h | p.qs.r) & 7) && !(reinterpret_cast<uintptr_t>(p.q) & 15u) && diff_rows_ok(s.k, s.ks, p.head_dim, p.kv_heads, 1) &&
         diff_rows_ok(s.v, s.vs, p.v_dim, p.kv_heads, 1);
}

int rows_tc(const DecodeParams& p, int part_width, int parts, int dtype, cudaStream_t st) {
  const DecodeSegment& s = p.seg[0];
  if (part_width % 64 || parts < 1 || parts > 65535 || static_cast<int64_t>(parts) * part_width < s.n_keys) return ELSA_ERR_INVALID_ARGUMENT;
  CUtensorMap mk, mv;
  int rc;
  if ((rc = make_tmap_rows64(&mk, s.k, dtype, s.n_keys, p.kv_heads, 1, s.ks, 64, p.head_dim)) != ELSA_OK) return rc;
  if ((rc = make_tmap_rows64(&mv, s.v, dtype, s.n_keys, p.kv_heads, 1, s.vs, 64, p.v_dim)) != ELSA_OK) return rc;
  PairParams prm{};
  prm.r = p;
  prm.part_width = part_width;
  prm.group = p.heads / p.kv_heads;
  if ((rc = device_status_word(&prm.status, nullptr)) != ELSA_OK) return rc;
  const dim3 grid(static_cast<unsigned>(cdiv64(decode_rows(p), 256)), static_cast<unsigned>(parts), static_cast<unsigned>(p.kv_heads));
  if (p.head_dim <= 64) return dtype == ELSA_F16 ? launch<__half, kRows64>(mk, mk, mv, prm, grid, st) : launch<__nv_bfloat16, kRows64>(mk, mk, mv, prm, grid, st);
  return dtype == ELSA_F16 ? launch<__half, kRows128>(mk, mk, mv, prm, grid, st) : launch<__nv_bfloat16, kRows128>(mk, mk, mv, prm, grid, st);
}

}  // namespace elsa
