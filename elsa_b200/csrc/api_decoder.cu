// C-ABI layer of the operators of decoder models (rotary positions, attention over a shared prefix, differential attention):
// argument validation and host orchestration.  Stream-ordered like api.cu; nothing allocates device memory or synchronises.
#include <algorithm>

#include "kernels.cuh"

using namespace elsa;

namespace {

bool inputs_ok(const void* p, int heads, int n, int head_dim, int batch, int dtype) {
  return p && heads > 0 && n > 0 && batch > 0 && head_dim > 0 && dtype_ok(dtype);
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
