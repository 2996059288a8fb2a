// Differential attention, forward, on the 5th-generation tensor cores (fp16 / bf16, head dim <= 64, value dim <= 128, multiples of 8).
//
// One CTA owns the 128 query rows of one output head, both maps: what the unbiased forward (fold_tc.cu) does with two query tiles
// is done here with the two maps of one tile, which have keys of their own and share the values, read once for both:
//
//   warp 8      TMA producer   Q1, Q2 once; K1, K2 and the two 64-column halves of V into a 3-stage ring (64 KB each)
//   warp 9, 10  MMA issuers    one for each map m:  S_m = Q_m K_m^T  (4 x tcgen05.mma 128x128x16, shared-memory operands)
//                                                   O_m += P_m V     (8 x tcgen05.mma 128x128x16, P from TMEM, V MN-major)
//   warps 0-3   fold of map 1  one thread per query row: S row into registers, running max, exp2, row sum, P (16-bit) over the
//   warps 4-7   fold of map 2  columns of the S it came from, rescale of O when the max moved
//
// TMEM columns: S1 / P1 [0,128) S2 / P2 [128,256) O1 [256,384) O2 [384,512).  Two accumulators of 128 columns leave none for P, so P_m
// lies over S_m and the next scores of a map are issued behind its P V; the other map's exponentials run meanwhile, and the two
// maps start half a period apart.  Each map is normalised by its own row sum at the end: O2 / z2 goes through shared memory to the
// threads that hold the same row of O1, which write (O1 / z1) - lam (O2 / z2).
//
// Bound: the ex2 unit, 2 x 128 x 128 exponentials for each (query tile, key tile) pair (2048 cycles; the tensor pipe needs 1536).
// As in fold_tc.cu the reference max moves only when it is exceeded by more than 2^8.  P is rounded to the inputs' type, sums and
// statistics are fp32.
#include <type_traits>

#include "diff.cuh"
#include "tc_common.cuh"

namespace elsa {

using namespace tc;

namespace {

constexpr int kStages = 3;
constexpr int kTileBytes = 128 * 64 * 2;                           // one 128 x 64 16-bit tile
constexpr int kStageBytes = 4 * kTileBytes;                        // K1, K2, V (columns 0-63), V (64-127)
constexpr int kFwdSmem = 2 * kTileBytes + kStages * kStageBytes + 1024;   // + alignment slack
constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;
constexpr int kProducerWarp = 8, kIssuerWarp = 9;
constexpr float kRescaleThreshold = 8.0f;

enum BarId { BAR_Q = 71, BAR_KV_FULL = 72, BAR_KV_FREE = 73, BAR_S = 74, BAR_P = 75, BAR_O = 76, BAR_STAGGER = 77 };

struct FwdParams {
  DiffParams d;
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
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    if (i >= n) continue;
    uint4 t;
    t.x = pack2<T>(v[i], v[i + 1]); t.y = pack2<T>(v[i + 2], v[i + 3]);
    t.z = pack2<T>(v[i + 4], v[i + 5]); t.w = pack2<T>(v[i + 6], v[i + 7]);
    *reinterpret_cast<uint4*>(dst + i) = t;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
diff_fwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                const __grid_constant__ CUtensorMap tmap_v, const FwdParams prm) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 8];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const DiffParams& p = prm.d;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int warp_u = __shfl_sync(0xffffffffu, warp, 0);   // (known to be warp-uniform)
  const int hi = blockIdx.y, bi = blockIdx.z, gi = hi / prm.group;
  // causal: the long tiles first
  const int bx = p.causal ? static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x);
  const int q0 = bx * 128;
  const int shift = p.nk - p.nq;                           // causal: row i sees keys up to i + shift
  int ke = p.nk;
  if (p.causal) ke = min(ke, min(q0 + 128, p.nq) + shift);
  const int n_t = ke > 0 ? (ke + 127) / 128 : 0;           // 128-key tiles, the same for both maps
  const int v_tiles = p.v_dim > 64 ? 2 : 1;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  auto sQ = [&](int m) { return smem_base + m * kTileBytes; };
  auto sK = [&](int st, int m) { return smem_base + 2 * kTileBytes + st * kStageBytes + m * kTileBytes; };
  auto sV = [&](int st) { return smem_base + 2 * kTileBytes + st * kStageBytes + 2 * kTileBytes; };
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t bar_q = bar0, bar_stagger = bar0 + 8;
  auto bar_kv_full = [&](int st) { return bar0 + 8 * (2 + st); };
  auto bar_kv_free = [&](int st) { return bar0 + 8 * (2 + kStages + st); };
  auto bar_s = [&](int m) { return bar0 + 8 * (2 + 2 * kStages + m); };       // S_m(j) is in TMEM, and P_m V of the key tile before has retired
  auto bar_p = [&](int m) { return bar0 + 8 * (4 + 2 * kStages + m); };       // P_m(j) has been delivered
  auto bar_o = [&](int m) { return bar0 + 8 * (6 + 2 * kStages + m); };       // every MMA of the map has retired

  if (tid == 0) {
    abort_flag = 0;
    mbar_init(bar_q, 1);
    mbar_init(bar_stagger, 1);
    for (int st = 0; st < kStages; ++st) { mbar_init(bar_kv_full(st), 1); mbar_init(bar_kv_free(st), 2); }
    for (int m = 0; m < 2; ++m) { mbar_init(bar_s(m), 1); mbar_init(bar_p(m), 4); mbar_init(bar_o(m), 1); }
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
  auto tS = [&](int m) { return tmem_base + 128 * m; };
  auto tO = [&](int m) { return tmem_base + 256 + 128 * m; };

  // registers: 3 x 128 threads, 232 + 232 + 40 = 3 x 168, the launch allocation (see fold_tc.cu)
  if (warp_u >= 8) {
    reg_dec<40>();
    if (n_t > 0 && warp == kProducerWarp) {
      // ---------------- TMA producer ----------------
      if (lane == 0) {
        prefetch_tmap(&tmap_q); prefetch_tmap(&tmap_k); prefetch_tmap(&tmap_v);
        mbar_arrive_expect_tx(bar_q, 2 * kTileBytes);
        for (int m = 0; m < 2; ++m) tma_load_4d(sQ(m), &tmap_q, bar_q, 0, q0, 2 * hi + m, bi);
        for (int j = 0; j < n_t; ++j) {
          const int st = j % kStages;
          if (j >= kStages && !mbar_wait(bar_kv_free(st), ((j / kStages) - 1) & 1, &abort_flag, prm.status, BAR_KV_FREE)) break;
          mbar_arrive_expect_tx(bar_kv_full(st), (2 + v_tiles) * kTileBytes);
          for (int m = 0; m < 2; ++m) tma_load_4d(sK(st, m), &tmap_k, bar_kv_full(st), 0, j * 128, 2 * gi + m, bi);
          for (int h = 0; h < v_tiles; ++h) tma_load_4d(sV(st) + h * kTileBytes, &tmap_v, bar_kv_full(st), 64 * h, j * 128, gi, bi);
        }
      }
    } else if (n_t > 0 && (warp_u == kIssuerWarp || warp_u == kIssuerWarp + 1)) {
      // ---------------- MMA issuers: one for each map ----------------
      const int m = warp_u - kIssuerWarp;
      const bool leader = elect_one();
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_s = make_idesc(fmt, 0, 0, 128, 128);                                  // S = Q K^T : A, B K-major
      const uint32_t idesc_o = v_tiles == 2 ? make_idesc(fmt, 0, 1, 128, 128) : make_idesc(fmt, 0, 1, 128, 64);   // O += P V : A in TMEM, B MN-major
      const uint64_t dq = make_sdesc(sQ(m), 16, 1024), dk0 = make_sdesc(sK(0, m), 16, 1024);
      const uint64_t dv0 = make_sdesc(sV(0), kTileBytes, 1024);       // (leading offset: from one 64-column half to the other)
      constexpr uint64_t kStageStep = kStageBytes >> 4;               // descriptor address field counts 16-byte units
      bool ok = mbar_wait_warp(bar_q, 0, &abort_flag, prm.status, BAR_Q) && mbar_wait_warp(bar_kv_full(0), 0, &abort_flag, prm.status, BAR_KV_FULL);
      // map 2 starts half a period after map 1: in step they would want the ex2 unit at the same time
      if (ok && m == 1) ok = mbar_wait_warp(bar_stagger, 0, &abort_flag, prm.status, BAR_STAGGER);
      if (ok) {
        tc_fence_after();
        if (leader) mma_ss_x4<2, 2>(tS(m), dq, dk0, idesc_s, 0u);
        if (leader) mma_commit(bar_s(m));
      }
      for (int j = 0; ok && j < n_t; ++j) {
        const int u = j % kStages, un = (j + 1) % kStages;
        if (!(ok = mbar_wait_warp(bar_p(m), j & 1, &abort_flag, prm.status, BAR_P))) break;
        if (m == 0 && j == 0 && leader) mbar_arrive(bar_stagger);
        tc_fence_after();
        if (leader) mma_ts_x4<8, 128>(tO(m), tS(m), dv0 + u * kStageStep, idesc_o, j > 0 ? 1u : 0u);
        if (leader) mma_ts_x4<8, 128>(tO(m), tS(m) + 32, dv0 + u * kStageStep + 512, idesc_o, 1u);
        if (leader) mma_commit(bar_kv_free(u));   // this map no longer reads K_m(j), V(j)
        if (j + 1 < n_t) {
          // the next scores over P(j): the tensor pipe takes them after the P V that reads it
          if (!(ok = mbar_wait_warp(bar_kv_full(un), ((j + 1) / kStages) & 1, &abort_flag, prm.status, BAR_KV_FULL))) break;
          tc_fence_after();
          if (leader) mma_ss_x4<2, 2>(tS(m), dq, dk0 + un * kStageStep, idesc_s, 0u);
          if (leader) mma_commit(bar_s(m));
        }
      }
      if (ok && leader) mma_commit(bar_o(m));
    }
  } else {
    reg_inc<232>();
    // ---------------- fold warps: one thread per query row and map ----------------
    const int m = warp >> 2;
    const int row = (warp & 3) * 32 + lane;                 // row within the tile == TMEM lane
    const int qi = q0 + row;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float c = p.scale_log2;
    float m_ref = -CUDART_INF_F, zsum = 0.f;
    bool alive = true;

    for (int j = 0; j < n_t; ++j) {
      // (the barrier's commit covers every MMA issued before: P V of the key tile before has retired, O may be rescaled)
      if (!mbar_wait_warp(bar_s(m), j & 1, &abort_flag, prm.status, BAR_S)) { alive = false; break; }
      tc_fence_after();
      float sv[128];
      float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
      {
        uint32_t ra[32], rb[32], rc[32], rd[32];
        tmem_ld32(tS(m) + lane_off, ra);
        tmem_ld32(tS(m) + lane_off + 32, rb);
        tmem_wait_ld();
        tmem_ld32(tS(m) + lane_off + 64, rc);
        tmem_ld32(tS(m) + lane_off + 96, rd);
#pragma unroll
        for (int i = 0; i < 32; ++i) { sv[i] = __uint_as_float(ra[i]); sv[32 + i] = __uint_as_float(rb[i]); }
#pragma unroll
        for (int i = 0; i < 64; i += 8) {
          mx[0] = max3(mx[0], sv[i], sv[i + 1]); mx[1] = max3(mx[1], sv[i + 2], sv[i + 3]);
          mx[2] = max3(mx[2], sv[i + 4], sv[i + 5]); mx[3] = max3(mx[3], sv[i + 6], sv[i + 7]);
        }
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) { sv[64 + i] = __uint_as_float(rc[i]); sv[96 + i] = __uint_as_float(rd[i]); }
#pragma unroll
        for (int i = 64; i < 128; i += 8) {
          mx[0] = max3(mx[0], sv[i], sv[i + 1]); mx[1] = max3(mx[1], sv[i + 2], sv[i + 3]);
          mx[2] = max3(mx[2], sv[i + 4], sv[i + 5]); mx[3] = max3(mx[3], sv[i + 6], sv[i + 7]);
        }
      }
      const int k0 = j * 128;
      const bool tail = k0 + 128 > p.nk;
      const bool diag = p.causal && (k0 + 127 > q0 + shift);
      if (__builtin_expect(tail || diag, 0)) {
        const int lim = p.causal ? min(p.nk - 1, qi + shift) : p.nk - 1;   // last key of this row
        mx[0] = mx[1] = mx[2] = mx[3] = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < 128; ++i) {
          if (k0 + i > lim) sv[i] = -CUDART_INF_F;
          mx[i & 3] = fmaxf(mx[i & 3], sv[i]);
        }
      }
      const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
      const bool move = tmax > m_ref + kRescaleThreshold;   // also true for the first tile with a key of this row (m_ref = -inf)
      if (__builtin_expect(__any_sync(0xffffffffu, move), 0)) {
        const float m_new = move ? tmax : m_ref;             // (a row's result does not depend on the rows beside it)
        const float alpha = move ? fast_exp2(m_ref - m_new) : 1.f;
        zsum *= alpha;
        if (j > 0) {
          for (int h = 0; h < 2 * v_tiles; ++h) {
            uint32_t r[32];
            tmem_ld32(tO(m) + lane_off + 32 * h, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st32(tO(m) + lane_off + 32 * h, r);
          }
        }
        m_ref = m_new;
      }
      const float m_use = (m_ref == -CUDART_INF_F) ? 0.f : m_ref;
      const float2 c2 = make_float2(c, c), nm2 = make_float2(-m_use, -m_use);
      float2 ps[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float2 x = __ffma2_rn(make_float2(sv[64 * h + 2 * i], sv[64 * h + 2 * i + 1]), c2, nm2);
          const float2 pp = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          ps[i & 3] = __fadd2_rn(ps[i & 3], pp);
          pk[i] = pack2<T>(pp.x, pp.y);
        }
        tmem_st32(tS(m) + lane_off + 32 * h, pk);
      }
      tmem_wait_st();               // (also covers the O rescale stores above)
      tc_fence_before();
      mbar_arrive_warp(bar_p(m), lane);
      {
        const float2 s01 = __fadd2_rn(ps[0], ps[1]), s23 = __fadd2_rn(ps[2], ps[3]);
        const float2 s = __fadd2_rn(s01, s23);
        zsum += s.x + s.y;
      }
    }

    // epilogue.  Map 2 leaves lam O2 / z2 in shared memory, [column][row] (the ring is free: every MMA that read it has retired,
    // and every load has been waited for), map 1 takes it.
    const bool row_ok = qi < p.nq;
    const int64_t ro = (static_cast<int64_t>(bi) * p.heads + hi) * p.nq + qi;
    if (alive && n_t > 0) alive = mbar_wait_warp(bar_o(m), 0, &abort_flag, prm.status, BAR_O);
    float* exchange = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)) + 2 * kTileBytes);
    const float inv = zsum != 0.f ? 1.f / zsum : 0.f;       // (NaN stays NaN)
    if (p.lse && row_ok && alive) p.lse[m * (static_cast<int64_t>(p.batch) * p.heads * p.nq) + ro] = zsum != 0.f ? m_ref + log2f(zsum) : -CUDART_INF_F;
    tc_fence_after();
    if (m == 1 && n_t > 0) {
      // (map 1's last P V reads the ring's V: it has to have retired as well before the ring is written)
      if (alive) alive = mbar_wait_warp(bar_o(0), 0, &abort_flag, prm.status, BAR_O);
      const float lam = diff_lam(p, hi);
      for (int h = 0; h < 2 * v_tiles; ++h) {
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
    } else if (m == 1 && p.out2 && row_ok) {
      float o[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0.f;
      for (int h = 0; h < 4; ++h) store32<T>(static_cast<T*>(p.out2) + ro * p.v_dim + 32 * h, o, p.v_dim - 32 * h);
    }
    named_barrier_sync(1, 256);
    if (m == 0) {
      T* dst = static_cast<T*>(p.out) + bi * p.os.b + hi * p.os.h + static_cast<int64_t>(qi) * p.os.r;
      for (int h = 0; h < 2 * v_tiles; ++h) {
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
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kProducerWarp) tmem_dealloc(tmem_base, kTmemCols);
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
    if ((rc = make_tmap_rows64(&mk, p.k, dtype, p.nk, 2 * p.kv_heads, p.batch, p.ks, 128, p.head_dim)) != ELSA_OK) return rc;
    if ((rc = make_tmap_rows64(&mv, p.v, dtype, p.nk, p.kv_heads, p.batch, p.vs, 128, p.v_dim)) != ELSA_OK) return rc;
  } else {
    mk = mv = mq;                                          // no key tile is visited
  }
  FwdParams prm;
  prm.d = p;
  prm.group = p.heads / p.kv_heads;
  if ((rc = device_status_word(&prm.status, nullptr)) != ELSA_OK) return rc;
  const dim3 grid(static_cast<unsigned>((p.nq + 127) / 128), static_cast<unsigned>(p.heads), static_cast<unsigned>(p.batch));
  auto launch = [&](auto kernel) -> int {
    const int r = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kFwdSmem);
    if (r != ELSA_OK) return r;
    kernel<<<grid, kThreads, kFwdSmem, st>>>(mq, mk, mv, prm);
    return ELSA_OK;
  };
  rc = dtype == ELSA_F16 ? launch(&diff_fwd_kernel<__half>) : launch(&diff_fwd_kernel<__nv_bfloat16>);
  if (rc != ELSA_OK) return rc;
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

}  // namespace elsa
