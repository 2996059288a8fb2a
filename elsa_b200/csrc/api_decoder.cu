// C-ABI layer of the operators of decoder models (rotary positions, attention over a shared prefix, differential attention):
// argument validation and host orchestration.  Stream-ordered like api.cu; nothing allocates device memory or synchronises.
#include <algorithm>
#include <cfloat>

#include "decode.cuh"
#include "diff.cuh"
#include "kernels.cuh"
#include "pair_tc.cuh"

using namespace elsa;

namespace {

bool inputs_ok(const void* p, int heads, int n, int head_dim, int batch, int dtype) {
  return p && heads > 0 && n > 0 && batch > 0 && head_dim > 0 && dtype_ok(dtype);
}

// positive and finite in fp32, with log2 e too (a scale that is zero there would make NaN of a masked score)
bool scale_ok(double scale) { return scale >= static_cast<double>(FLT_MIN) && scale * 1.4426950408889634 <= static_cast<double>(FLT_MAX); }

// a tensor-core kernel's wait that gave up is reported by every later call that would launch one (api.cu)
int device_status_ok() {
  volatile int* host = nullptr;
  const int rc = device_status_word(nullptr, &host);
  if (rc != ELSA_OK) return rc;
  return *host != 0 ? ELSA_ERR_DEVICE_TIMEOUT : ELSA_OK;
}

// Keys of one split.  A block costs about 4 us besides its keys (launch, first loads, merge of its warps), so there are as few
// splits as give two waves of two blocks on an SM, whose second wave evens out caches of different lengths.  Measured, bf16, head
// dim 128: 256 x 8 caches of up to 2048 keys 174 us at 1024 keys a split, 238 at 256, 550 at 64; 64 x 8 of up to 1024 keys 33 us at
// 512 or 1024, 49 at 128; 24 x 3 of up to 333 keys 8.9 us at 512, 9.3 at 128, 13.3 at 64.
// fp32: a block's time is in its products, and keys that a causal mask hides are left out tile by tile: eight blocks for each SM
// ((1, 4 heads, 1000 tokens, 64 / 128, causal): 80 us at 128 keys a split, 127 at 512).
int split_width(int dtype, int64_t blocks_of_one_split, int n_keys) {
  const int64_t wanted = std::max<int64_t>(1, (dtype == ELSA_F32 ? 8ll : 4ll) * sm_count() / blocks_of_one_split);
  const int64_t width = align_up(cdiv64(n_keys, wanted), 64);
  return static_cast<int>(std::max<int64_t>(64, std::min<int64_t>(width, 1024)));
}

// Summaries grow with queries times keys: the split kernels walk a call's queries in chunks -- whole sequences, or tokens of one --
// whose summaries fit 1 GiB, as the forward of api.cu does, through the same workspace.  A row's result is the same in any chunk (but
// in one of at most 8 rows of a key head, whose weights the 16-bit split kernel holds to twice the bits).  Measured, fp32, causal,
// (1, 16 heads, 16384 tokens, 64 / 128): 41.2 ms in five chunks, 41.4 with all summaries, 4 GiB, at once.
constexpr int64_t kSummaryBytes = 1ll << 30;

struct Chunk { int seqs, tokens; };

// token_bytes: the summaries of one token, all heads and parts
Chunk chunk_of(int batch, int nq, int64_t token_bytes) {
  const int64_t tokens = std::max<int64_t>(1, kSummaryBytes / std::max<int64_t>(1, token_bytes));
  if (tokens >= nq) return {static_cast<int>(std::min<int64_t>(batch, tokens / nq)), nq};
  return {1, static_cast<int>(tokens >= 32 ? tokens / 32 * 32 : tokens)};      // (whole tiles of rows)
}
// so few parts that one token's summaries (head_bytes of a head and part) fit
int bounded_width(int width, int n_keys, int heads, int64_t head_bytes) {
  const int64_t parts = std::max<int64_t>(1, kSummaryBytes / (heads * head_bytes));
  return static_cast<int>(std::max<int64_t>(width, align_up(cdiv64(n_keys, parts), 64)));
}
template <typename F>
int for_chunks(const Chunk& c, int batch, int nq, F run) {
  for (int b = 0; b < batch; b += c.seqs)
    for (int t = 0; t < nq; t += c.tokens) {
      const int rc = run(b, std::min(c.seqs, batch - b), t, std::min(c.tokens, nq - t));
      if (rc != ELSA_OK) return rc;
    }
  return ELSA_OK;
}
const void* offset(const void* p, int64_t elements, int dtype) { return p ? static_cast<const char*>(p) + elements * dtype_size(dtype) : nullptr; }

// ---- attention over a shared prefix ------------------------------------------------------------------------------------
struct PrefixPlan {
  bool tiles;                   // the prefix on the 256-row tensor-core kernel (pair_tc.cu)
  int prefix_width, prefix_parts, own_width, own_parts;
  Chunk chunk;
  int64_t mz_bytes, s_bytes;
  int64_t bytes() const { return 2 * mz_bytes + s_bytes; }
};

// More rows for each key head than two 16-row tiles: the split kernel would read the prefix once for each tile.
constexpr int kTileRows = 32;

int plan_prefix(int dtype, int batch, int heads, int kv_heads, int nq, int head_dim, int n_prefix, int n_own, PrefixPlan* pl) {
  if (!dtype_ok(dtype) || batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || nq < 1 || head_dim < 1 || n_prefix < 0 || n_own < 0)
    return ELSA_ERR_INVALID_ARGUMENT;
  if (head_dim > 128) return ELSA_ERR_UNSUPPORTED;
  const int64_t rows = static_cast<int64_t>(batch) * (heads / kv_heads) * nq;
  if (rows * heads > 0x3fffffff || kv_heads > 65535 || n_prefix > 0x3fffffff || n_own > 0x3fffffff) return ELSA_ERR_UNSUPPORTED;
  pl->tiles = rows > kTileRows && n_prefix >= 128 && (fold_tc_supported(dtype, head_dim, false) || fold_tcw_supported(dtype, head_dim, false));
  pl->prefix_width = pl->prefix_parts = pl->own_width = pl->own_parts = 0;
  const int tile = dtype == ELSA_F32 ? 32 : 16;          // rows of a block of the split kernels
  const int64_t head_bytes = (head_dim + 2) * 4;         // a summary (the prefix and the own keys have half of a chunk's each)
  if (n_own > 0) {
    pl->own_width = bounded_width(split_width(dtype, static_cast<int64_t>(batch) * kv_heads * cdiv64(heads / kv_heads * nq, tile), n_own), n_own, heads, 2 * head_bytes);
    pl->own_parts = static_cast<int>(cdiv64(n_own, pl->own_width));
  }
  if (pl->tiles) {
    // One CTA for each 256 rows, key head and part, one CTA on an SM: waves x (64-key tiles of a part + what a CTA costs besides, about
    // 13 of them).  The split kernel of the sequences' own keys runs beside it, on the SMs that it leaves free: 0.8 of them read at full
    // speed, fewer in proportion.  So few parts may be the best, a prefix that takes long on some SMs while the caches stream through
    // the others.  Measured, us a call in a long run: 256 sequences with up to 2048 keys behind 32768 (8 heads of 128), 32 CTAs a part:
    // 288 with 2 parts, 294 with 3, 317 with 9 (two full waves, then the caches); 64 with up to 1024 behind 8192, 8 CTAs a part: 44.2 with
    // 5, 50 with 4, 46 with 7, 59 with 17; 24 with up to 333 behind 4097 (3 heads of 96, five tokens), 6 CTAs a part: 22.5 with 8 to 11,
    // 24.6 with 5, 26.7 with 17.  (With caches all but empty the first of these loses, 241 us against 198 one after the other; half full it
    // is 247 against 280, full 335 against 386.)
    const double tile_us = 0.8, bytes_us = 6.3e6;
    const double own = n_own > 0 ? (2.0 * head_dim * batch * kv_heads * n_own / bytes_us + 9.0) / tile_us : 0.0;    // in tiles too, of caches half full
    const int64_t ctas = cdiv64(rows, 256) * kv_heads, tiles = cdiv64(n_prefix, 64), sms = sm_count();
    int64_t best = 0;
    double best_cost = 0.0;
    for (int64_t parts = 1; parts <= std::min<int64_t>(tiles, 64); ++parts) {
      const int64_t per = cdiv64(tiles, parts), all = ctas * cdiv64(tiles, per);
      const double prefix = static_cast<double>(cdiv64(all, sms) * (per + 13));
      const double beside = prefix * std::min(1.0, std::max<int64_t>(0, sms - all) / (0.8 * sms));    // of the caches, meanwhile
      const double cost = prefix + std::max(0.0, own - beside);
      if (best == 0 || cost < best_cost) { best = per; best_cost = cost; }
    }
    pl->prefix_width = static_cast<int>(best * 64);
  } else if (n_prefix > 0) {
    pl->prefix_width = bounded_width(split_width(dtype, kv_heads * cdiv64(rows, tile), n_prefix), n_prefix, heads, 2 * head_bytes);
  }
  if (n_prefix > 0) pl->prefix_parts = static_cast<int>(cdiv64(n_prefix, pl->prefix_width));
  const int64_t parts = pl->prefix_parts + pl->own_parts;
  pl->chunk = chunk_of(batch, nq, parts * heads * head_bytes);
  const int64_t summaries = parts * heads * pl->chunk.seqs * pl->chunk.tokens;
  pl->mz_bytes = align_up(summaries * 4, 256);
  pl->s_bytes = align_up(summaries * head_dim * 4, 256);
  return ELSA_OK;
}

// ---- differential attention -------------------------------------------------------------------------------------------
struct DiffPlan {
  bool tensor_tiles;            // the 128-row tensor-core kernels by sizes (pair_tc.cu); else the split kernels (decode.cu)
  int split_width, parts;       // of the split kernels
  Chunk chunk;
  int64_t mz_bytes, s_bytes;
  int64_t bytes() const { return 2 * mz_bytes + s_bytes; }
};

// Up to four 16-row tiles for each key head the split kernel, which works on keys side by side, is ahead of one CTA that walks over
// them in 128-row tiles.
constexpr int kSplitRows = 64;

int plan_diff(int dtype, int batch, int heads, int kv_heads, int nq, int nk, int head_dim, int v_dim, DiffPlan* pl) {
  if (!dtype_ok(dtype) || batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || nq < 1 || nk < 0 || head_dim < 1 || v_dim < 1)
    return ELSA_ERR_INVALID_ARGUMENT;
  if (head_dim > 128 || v_dim > 128) return ELSA_ERR_UNSUPPORTED;
  const int64_t rows_b = static_cast<int64_t>(heads / kv_heads) * nq, rows = rows_b * batch;
  // (nq: the backward's four statistics of a head are indexed in 32 bits)
  if (rows * kv_heads > 0x1fffffff || heads > 65535 || batch > 65535 || nk > 0x3fffffff || nq > 0xfffffff) return ELSA_ERR_UNSUPPORTED;
  pl->tensor_tiles = rows_b > kSplitRows && diff_tc_sizes(dtype, head_dim, v_dim);
  const int64_t head_bytes = 2 * (v_dim + 2) * 4;
  pl->split_width = nk > 0 ? bounded_width(split_width(dtype, static_cast<int64_t>(batch) * kv_heads * cdiv64(rows_b, dtype == ELSA_F32 ? 32 : 16), nk), nk, heads, head_bytes) : 1;
  pl->parts = static_cast<int>(cdiv64(nk, pl->split_width));
  pl->chunk = chunk_of(batch, nq, static_cast<int64_t>(pl->parts) * heads * head_bytes);
  const int64_t summaries = 2 * static_cast<int64_t>(pl->parts) * heads * pl->chunk.seqs * pl->chunk.tokens;
  pl->mz_bytes = align_up(summaries * 4, 256);
  pl->s_bytes = align_up(summaries * v_dim * 4, 256);
  return ELSA_OK;
}

DiffParams diff_params(const void* q, const void* k, const void* v, const void* lam, int lam_dtype, int lam_stride, const int64_t* st,
                       int batch, int heads, int kv_heads, int nq, int nk, int head_dim, int v_dim, int is_causal, double scale) {
  DiffParams p{};
  p.q = q; p.k = k; p.v = v;
  p.qs = Strides{st[0], st[1], st[2]}; p.ks = Strides{st[3], st[4], st[5]}; p.vs = Strides{st[6], st[7], st[8]};
  p.lam = lam; p.lam_dtype = lam_dtype; p.lam_stride = lam_stride;
  p.batch = batch; p.heads = heads; p.kv_heads = kv_heads; p.nq = nq; p.nk = nk; p.head_dim = head_dim; p.v_dim = v_dim; p.causal = is_causal;
  p.scale = static_cast<float>(scale); p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  return p;
}

bool diff_inputs_in_tiles(const DiffParams& p) {
  return diff_rows_ok(p.q, p.qs, p.head_dim, 2 * p.heads, p.batch) &&
         (p.nk == 0 || (diff_rows_ok(p.k, p.ks, p.head_dim, 2 * p.kv_heads, p.batch) && diff_rows_ok(p.v, p.vs, p.v_dim, p.kv_heads, p.batch)));
}

// whether the forward runs on the tile kernel, which needs no workspace
// (what stands behind a sequence's last key must not be read: the tile kernel's loads are bounded by the tensors only)
bool diff_forward_in_tiles(const DiffPlan& pl, const DiffParams& p, const int* lengths) {
  return pl.tensor_tiles && !lengths && diff_inputs_in_tiles(p) && diff_rows_ok(p.out, p.os, p.v_dim, p.heads, p.batch);
}

}  // namespace

extern "C" int elsa_rotary(const void* q, void* q_out, const int64_t* q_strides, int q_heads, const void* k, void* k_out,
                           const int64_t* k_strides, int k_heads, const double* frequencies, const void* positions,
                           int position_bytes, int64_t position_stride_b, int64_t position_stride_n, double magnitude, int dtype,
                           int batch, int n, int head_dim, int rotary_dim, int interleaved, int inverse, void* stream) {
  if (!inputs_ok(q, q_heads, n, head_dim, batch, dtype) || !q_out || !q_strides || !frequencies) return ELSA_ERR_INVALID_ARGUMENT;
  if (k && (!k_out || !k_strides || k_heads <= 0)) return ELSA_ERR_INVALID_ARGUMENT;
  if (head_dim > 1024 || rotary_dim < 2 || rotary_dim > 256 || rotary_dim > head_dim || rotary_dim % 2) return ELSA_ERR_UNSUPPORTED;
  if ((position_bytes != 0 && position_bytes != 4 && position_bytes != 8) || (position_bytes != 0) != (positions != nullptr))
    return ELSA_ERR_INVALID_ARGUMENT;
  // in place means the same elements: a row written where another one is still to be read would be lost
  if (q == q_out && !std::equal(q_strides, q_strides + 3, q_strides + 3)) return ELSA_ERR_INVALID_ARGUMENT;
  if (k && k == k_out && !std::equal(k_strides, k_strides + 3, k_strides + 3)) return ELSA_ERR_INVALID_ARGUMENT;
  if (static_cast<int64_t>(q_heads) + (k ? k_heads : 0) > 2048) return ELSA_ERR_UNSUPPORTED;
  return rotary(q, q_out, q_strides, q_heads, k, k_out, k_strides, k_heads, frequencies, positions, position_bytes,
                position_stride_b, position_stride_n, magnitude, dtype, batch, n, head_dim, rotary_dim, interleaved, inverse,
                static_cast<cudaStream_t>(stream));
}

extern "C" int64_t elsa_shared_prefix_workspace_bytes(int dtype, int batch, int heads, int kv_heads, int nq, int head_dim, int n_prefix,
                                                      int n_own) {
  PrefixPlan pl;
  return plan_prefix(dtype, batch, heads, kv_heads, nq, head_dim, n_prefix, n_own, &pl) == ELSA_OK ? pl.bytes() : -1;
}

extern "C" int elsa_shared_prefix_attention(const void* q, const void* k_prefix, const void* v_prefix, const void* k, const void* v,
                                            void* out, const int64_t* strides, const int* lengths, void* workspace,
                                            int64_t workspace_bytes, int dtype, int batch, int heads, int kv_heads, int nq,
                                            int head_dim, int n_prefix, int n_own, double scale, void* stream) {
  PrefixPlan pl;
  int rc = plan_prefix(dtype, batch, heads, kv_heads, nq, head_dim, n_prefix, n_own, &pl);
  if (rc != ELSA_OK) return rc;
  if (!q || !out || !strides || (n_prefix > 0 && (!k_prefix || !v_prefix)) || (n_own > 0 && (!k || !v)) || !scale_ok(scale)) return ELSA_ERR_INVALID_ARGUMENT;
  if (pl.bytes() > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < pl.bytes())) return ELSA_ERR_WORKSPACE;
  auto st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const Strides qs{strides[0], strides[1], strides[2]}, ks{strides[7], strides[8], strides[9]}, vs{strides[10], strides[11], strides[12]};
  const Strides os{strides[13], strides[14], strides[15]};
  return for_chunks(pl.chunk, batch, nq, [&](int b0, int seqs, int t0, int tokens) -> int {
    DecodeParams p{};
    p.q = offset(q, b0 * qs.b + t0 * qs.r, dtype); p.qs = qs;
    p.batch = seqs; p.heads = heads; p.kv_heads = kv_heads; p.nq = tokens; p.head_dim = p.v_dim = head_dim; p.maps = 1;
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    p.m = reinterpret_cast<float*>(ws);
    p.z = reinterpret_cast<float*>(ws + pl.mz_bytes);
    p.s = reinterpret_cast<float*>(ws + 2 * pl.mz_bytes);
    p.out = const_cast<void*>(offset(out, b0 * os.b + t0 * os.r, dtype)); p.os = os;
    int rc;
    bool beside = false;                                // the prefix's kernel has been launched
    if (n_prefix > 0) {
      DecodeSegment& s = p.seg[0];
      s.k = k_prefix; s.v = v_prefix; s.ks = Strides{0, strides[3], strides[4]}; s.vs = Strides{0, strides[5], strides[6]}; s.n_keys = n_prefix; s.shared = 1;
      s.split_width = pl.prefix_width; s.n_splits = pl.prefix_parts; s.first_part = 0;
      // (a layout that the tensor maps do not take goes through the split kernel with the same parts)
      if (pl.tiles && rows_tc_ok(p, dtype)) {
        if ((rc = device_status_ok()) != ELSA_OK) return rc;
        if ((rc = rows_tc(p, pl.prefix_width, pl.prefix_parts, dtype, st)) != ELSA_OK) return rc;
        beside = true;
      } else {
        p.n_segs = 1;
      }
    }
    if (n_own > 0) {
      DecodeSegment& s = p.seg[p.n_segs++];
      s = DecodeSegment{};
      s.k = offset(k, b0 * ks.b, dtype); s.v = offset(v, b0 * vs.b, dtype); s.ks = ks; s.vs = vs;
      s.lengths = lengths ? lengths + b0 : nullptr; s.n_keys = n_own; s.causal = 1; s.tail = nq - t0 - tokens;
      s.split_width = pl.own_width; s.n_splits = pl.own_parts; s.first_part = pl.prefix_parts;
    }
    if ((rc = decode_split(p, dtype, beside, st)) != ELSA_OK) return rc;
    return decode_merge(p, pl.prefix_parts + pl.own_parts, dtype, n_prefix + n_own > 0, st);
  });
}

extern "C" int64_t elsa_differential_workspace_bytes(int dtype, int batch, int heads, int kv_heads, int nq, int nk, int head_dim, int v_dim) {
  DiffPlan pl;
  return plan_diff(dtype, batch, heads, kv_heads, nq, nk, head_dim, v_dim, &pl) == ELSA_OK ? pl.bytes() : -1;
}

extern "C" int64_t elsa_differential_workspace_bytes_for(const void* q, const void* k, const void* v, const int* lengths, const void* out,
                                                         const int64_t* strides, int dtype, int batch, int heads, int kv_heads, int nq, int nk,
                                                         int head_dim, int v_dim) {
  DiffPlan pl;
  if (plan_diff(dtype, batch, heads, kv_heads, nq, nk, head_dim, v_dim, &pl) != ELSA_OK || !strides) return -1;
  DiffParams d = diff_params(q, k, v, nullptr, 0, 0, strides, batch, heads, kv_heads, nq, nk, head_dim, v_dim, 0, 1.0);
  d.out = const_cast<void*>(out); d.os = Strides{strides[9], strides[10], strides[11]};
  return diff_forward_in_tiles(pl, d, lengths) ? 0 : pl.bytes();
}

extern "C" int elsa_differential_forward(const void* q, const void* k, const void* v, const void* lam, int lam_dtype, int lam_stride,
                                         const int* lengths, void* out, const int64_t* strides, void* out2, float* lse, void* workspace,
                                         int64_t workspace_bytes, int dtype, int batch, int heads, int kv_heads, int nq, int nk,
                                         int head_dim, int v_dim, int is_causal, double scale, void* stream) {
  DiffPlan pl;
  int rc = plan_diff(dtype, batch, heads, kv_heads, nq, nk, head_dim, v_dim, &pl);
  if (rc != ELSA_OK) return rc;
  if (!q || !lam || !out || !strides || (nk > 0 && (!k || !v)) || !dtype_ok(lam_dtype) || !scale_ok(scale)) return ELSA_ERR_INVALID_ARGUMENT;
  auto st = static_cast<cudaStream_t>(stream);
  DiffParams d = diff_params(q, k, v, lam, lam_dtype, lam_stride, strides, batch, heads, kv_heads, nq, nk, head_dim, v_dim, is_causal, scale);
  d.out = out; d.os = Strides{strides[9], strides[10], strides[11]};
  d.out2 = out2; d.lse = lse;
  if (diff_forward_in_tiles(pl, d, lengths)) {
    if ((rc = device_status_ok()) != ELSA_OK) return rc;
    return diff_tc_fwd(d, dtype, st);
  }
  if (pl.bytes() > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < pl.bytes())) return ELSA_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  return for_chunks(pl.chunk, batch, nq, [&](int b0, int seqs, int t0, int tokens) -> int {
    DecodeParams p{};
    p.q = offset(q, b0 * d.qs.b + t0 * d.qs.r, dtype); p.qs = d.qs;
    p.batch = seqs; p.heads = heads; p.kv_heads = kv_heads; p.nq = tokens; p.head_dim = head_dim; p.v_dim = v_dim; p.maps = 2;
    p.scale_log2 = d.scale_log2;
    p.m = reinterpret_cast<float*>(ws); p.z = reinterpret_cast<float*>(ws + pl.mz_bytes); p.s = reinterpret_cast<float*>(ws + 2 * pl.mz_bytes);
    p.lam = lam; p.lam_dtype = lam_dtype; p.lam_stride = lam_stride;
    const int64_t row0 = static_cast<int64_t>(b0) * heads * nq + t0;
    p.out = const_cast<void*>(offset(out, b0 * d.os.b + t0 * d.os.r, dtype)); p.os = d.os;
    p.out2 = const_cast<void*>(offset(out2, row0 * v_dim, dtype));
    p.lse = lse ? lse + row0 : nullptr; p.nq_all = nq; p.map_rows = static_cast<int64_t>(batch) * heads * nq;
    if (nk > 0) {
      DecodeSegment& s = p.seg[p.n_segs++];
      s.k = offset(k, b0 * d.ks.b, dtype); s.v = offset(v, b0 * d.vs.b, dtype); s.ks = d.ks; s.vs = d.vs;
      s.lengths = lengths ? lengths + b0 : nullptr; s.n_keys = nk; s.causal = is_causal; s.tail = is_causal ? nq - t0 - tokens : 0;
      s.split_width = pl.split_width; s.n_splits = pl.parts;
    }
    const int rc = decode_split(p, dtype, false, st);
    return rc != ELSA_OK ? rc : decode_merge(p, pl.parts, dtype, nk > 0, st);
  });
}

extern "C" int64_t elsa_differential_backward_workspace_bytes(int dtype, int batch, int heads, int kv_heads, int nq, int nk, int head_dim,
                                                              int v_dim) {
  DiffPlan pl;
  return plan_diff(dtype, batch, heads, kv_heads, nq, nk, head_dim, v_dim, &pl) == ELSA_OK ? diff_stats_bytes(batch, heads, nq) + diff_dlam_bytes(batch, heads, nq) : -1;
}

extern "C" int elsa_differential_backward(const void* q, const void* k, const void* v, const void* lam, int lam_dtype, int lam_stride,
                                          const void* out, const void* out2, const float* lse, const void* dout, void* dq, void* dk,
                                          void* dv, void* dlam, const int64_t* strides, void* workspace, int64_t workspace_bytes,
                                          int dtype, int batch, int heads, int kv_heads, int nq, int nk, int head_dim, int v_dim,
                                          int is_causal, double scale, void* stream) {
  DiffPlan pl;
  int rc = plan_diff(dtype, batch, heads, kv_heads, nq, nk, head_dim, v_dim, &pl);
  if (rc != ELSA_OK) return rc;
  if (!q || !lam || !out || !out2 || !lse || !dout || !dq || !strides || (nk > 0 && (!k || !v || !dk || !dv)) || !dtype_ok(lam_dtype) || !scale_ok(scale))
    return ELSA_ERR_INVALID_ARGUMENT;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) ||
      workspace_bytes < diff_stats_bytes(batch, heads, nq) + diff_dlam_bytes(batch, heads, nq))
    return ELSA_ERR_WORKSPACE;
  auto st = static_cast<cudaStream_t>(stream);
  DiffParams d = diff_params(q, k, v, lam, lam_dtype, lam_stride, strides, batch, heads, kv_heads, nq, nk, head_dim, v_dim, is_causal, scale);
  auto at = [&](int i) { return Strides{strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]}; };
  d.out = const_cast<void*>(out); d.os = at(3); d.out2 = const_cast<void*>(out2); d.lse = const_cast<float*>(lse);
  d.dout = dout; d.gs = at(4);
  d.dq = dq; d.dk = dk; d.dv = dv; d.dqs = at(5); d.dks = at(6); d.dvs = at(7);
  d.dlam = dlam;
  d.dlam_parts = dlam ? reinterpret_cast<float*>(static_cast<char*>(workspace) + diff_stats_bytes(batch, heads, nq)) : nullptr;
  float* stats = static_cast<float*>(workspace);
  // (the tile kernel has two bodies for each sequence in a grid of 65535)
  const bool tiles = batch <= 32767 && diff_tc_sizes(dtype, head_dim, v_dim) && diff_inputs_in_tiles(d) && diff_rows_ok(dout, d.gs, v_dim, heads, batch) &&
                     diff_rows_ok(dq, d.dqs, head_dim, 2 * heads, batch) &&
                     (nk == 0 || (diff_rows_ok(dk, d.dks, head_dim, 2 * kv_heads, batch) && diff_rows_ok(dv, d.dvs, v_dim, kv_heads, batch)));
  if (tiles && (rc = device_status_ok()) != ELSA_OK) return rc;
  if ((rc = diff_stats(d, stats, dtype, st)) != ELSA_OK) return rc;
  if ((rc = tiles ? diff_bwd_tc(d, stats, dtype, st) : diff_bwd_any(d, stats, dtype, st)) != ELSA_OK || !dlam) return rc;
  return diff_dlam(d, static_cast<int>(cdiv64(nq, tiles ? kDiffTcRows : kDiffAnyRows)), st);
}
