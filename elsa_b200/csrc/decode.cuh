// Attention of few query rows over long key caches, split along the keys: the per-split (m, z, s) summaries (decode.cu) and
// their merge.  Used by the shared-prefix attention (one softmax map) and by the single-token form of the differential
// attention (two maps over one value cache).
#pragma once

#include "kernels.cuh"

namespace elsa {

// One key cache.  shared: [kv heads, n_keys, .] for all sequences (batch strides unused), every query sees every key.
// Otherwise [batch, kv heads, n_keys, .]: sequence b has lengths[b] keys (null: n_keys) and, where causal, its query i of nq
// sees the first lengths[b] - tail - nq + i + 1 of them.  Keys from lengths[b] on are never read.
struct DecodeSegment {
  const void* k; const void* v;
  Strides ks, vs;                       // head axis of k: maps * kv heads, of v: kv heads
  const int* lengths;
  int n_keys, causal, shared;
  int tail;                             // causal: tokens of a sequence behind the last query of this launch (0 where it has them all)
  int split_width, n_splits, first_part;
  int row_tiles;                        // set by the launcher
  int64_t blocks;                       // set by the launcher
};

// Rows are numbered within their kv head: row = (b * group + query head within the group) * nq + i, `rows` of them.
// Summaries: m, z [part][kv head][row][map], s [part][kv head][row][map][v_dim], fp32; m in the log2 domain.
struct DecodeParams {
  const void* q; Strides qs;            // [batch, maps * heads, nq, head_dim]
  int batch, heads, kv_heads, nq, head_dim, v_dim, maps;
  float scale_log2;
  DecodeSegment seg[2]; int n_segs;
  float* m; float* z; float* s;
  // the merge
  const void* lam; int lam_dtype, lam_stride;   // maps == 2: out = s1 / z1 - lam[h] s2 / z2, a value for each head or for all (lam_stride 0)
  void* out; Strides os;                // [batch, heads, nq, v_dim]
  // maps == 2, for a backward (null: not wanted): s2 / z2 as contiguous [batch, heads, nq, v_dim], log2 of each row's sum of 2^score as
  // [map][batch * heads * nq] (-inf: no key); a launch for some of a call's rows: from its first row on, nq_all tokens of a head, map_rows
  // rows of a map
  void* out2; float* lse;
  int nq_all; int64_t map_rows;
};

__host__ __device__ inline int64_t decode_rows(const DecodeParams& p) { return static_cast<int64_t>(p.batch) * (p.heads / p.kv_heads) * p.nq; }

// the keys of sequence b that some query of the launch may see (a tail's queries see more)
__device__ __forceinline__ int keys_of(const DecodeSegment& s, int b) {
  return max(0, (s.shared || !s.lengths ? s.n_keys : min(s.n_keys, s.lengths[b])) - s.tail);
}

// A kernel that was launched by launch_behind may begin while the launch before it in the stream still runs, once all of that one's blocks
// have called let_next_begin (or ended); wait_for_previous returns when it has ended and its writes can be read.  Both do nothing in
// other launches.
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
int launch_behind(bool behind, void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st, const Args&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cfg.attrs = &attr; cfg.numAttrs = behind ? 1 : 0;
  ELSA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

// whether the tensor-core kernel takes this: 16-bit types, rows on 16-byte boundaries, head and value dims it has
bool decode_mma_ok(const DecodeParams& p, int dtype);
// summaries of all segments in one launch; parts that begin beyond a sequence's keys are not written.  behind: it may run beside the launch
// before it, one of these files' that does not write what it reads
int decode_split(DecodeParams& p, int dtype, bool behind, cudaStream_t st);
// all parts of a row merged (of a segment that is not shared: those that begin before the sequence's last key).  behind: it may come
// onto the device early; the launch before it is one of these files'
int decode_merge(const DecodeParams& p, int n_parts, int dtype, bool behind, cudaStream_t st);

}  // namespace elsa
