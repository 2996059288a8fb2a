// Two softmax chains over one stream of keys and values on the tensor cores (pair_tc.cu).
#pragma once

#include "decode.cuh"
#include "diff.cuh"

namespace elsa {

// differential attention, forward: the two maps of 128 query rows of a head (16-bit types, diff_tc_sizes)
int diff_tc_fwd(const DiffParams& p, int dtype, cudaStream_t st);

// A shared key cache for many query rows (16-bit types, head_dim <= 128 and a multiple of 8): the rows of a kv head, 256 at a time,
// against the keys of p.seg[0], which are cut into `parts` of `part_width` (a multiple of 64) keys.  Summaries [part][kv head][row], s with
// v_dim == head_dim columns, in p.m, p.z, p.s, as the split kernels write them.
bool rows_tc_ok(const DecodeParams& p, int dtype);
int rows_tc(const DecodeParams& p, int part_width, int parts, int dtype, cudaStream_t st);

}  // namespace elsa
