// Differential attention: out = (P1 - lam P2) V with P_m = softmax(Q_m K_m^T scale), the two maps of output head h being query heads
// 2h, 2h + 1 and key heads 2g, 2g + 1 of its key group g = h / (heads / kv_heads).
#pragma once

#include "kernels.cuh"

namespace elsa {

struct DiffParams {
  const void* q; const void* k; const void* v;   // [B, 2 heads, nq, d], [B, 2 kv_heads, nk, d], [B, kv_heads, nk, dv]
  Strides qs, ks, vs;
  const void* lam; int lam_dtype, lam_stride;    // a value for each head, or one (stride 0)
  int batch, heads, kv_heads, nq, nk, head_dim, v_dim, causal;   // causal: query i sees keys 0 .. i + nk - nq
  float scale, scale_log2;
  void* out; Strides os;                         // [B, heads, nq, dv]
  // what the backward needs (null: not wanted): P2 V, contiguous [B, heads, nq, dv] in the inputs' type, and the log2 of each row's
  // sum of 2^score, [2][B * heads * nq] (-inf: the row sees no key)
  void* out2; float* lse;
  // backward
  const void* dout; Strides gs;
  void* dq; void* dk; void* dv; Strides dqs, dks, dvs;
  void* dlam;                                    // like lam: a value for each head, or one (null: not wanted)
  float* dlam_parts;                             // [B * heads][query tiles of the backward kernel]: sums of P2 G over a tile's rows and all keys
};

// sizes that the tcgen05 kernels take (16-bit types), and the strides and addresses that their tensor maps ask for
bool diff_tc_sizes(int dtype, int head_dim, int v_dim);
bool diff_rows_ok(const void* base, const Strides& s, int row, int heads, int batch);
// row statistics of the backward, [B * heads][-LSE1, -LSE2, -D1, -D2][n_pad] with n_pad = nq rounded up to 128 (diff_any.cu)
inline int64_t diff_stats_bytes(int batch, int heads, int nq) { return align_up(static_cast<int64_t>(batch) * heads * 4 * align_up(nq, 128) * 4, 256); }
int diff_stats(const DiffParams& p, float* stats, int dtype, cudaStream_t st);
// the most parts that a backward kernel leaves, and their sum, once it has run: dlam[h] = -(sum over the batch and the tiles)
inline int64_t diff_dlam_bytes(int batch, int heads, int nq) { return align_up(static_cast<int64_t>(batch) * heads * cdiv64(nq, 32) * 4, 256); }
int diff_dlam(const DiffParams& p, int tiles, cudaStream_t st);
// dq, dk, dv from them: of any type (diff_any.cu), 16-bit in tiles (diff_bwd_tc.cu)
constexpr int kDiffAnyRows = 32, kDiffTcRows = 128;    // query rows of one of dlam's parts
int diff_bwd_any(const DiffParams& p, const float* stats, int dtype, cudaStream_t st);
int diff_bwd_tc(const DiffParams& p, const float* stats, int dtype, cudaStream_t st);

__device__ __forceinline__ float diff_lam(const DiffParams& p, int h) {
  const int64_t at = static_cast<int64_t>(h) * p.lam_stride;
  if (p.lam_dtype == ELSA_F32) return static_cast<const float*>(p.lam)[at];
  return p.lam_dtype == ELSA_F16 ? to_f32(static_cast<const __half*>(p.lam)[at]) : to_f32(static_cast<const __nv_bfloat16*>(p.lam)[at]);
}

}  // namespace elsa
