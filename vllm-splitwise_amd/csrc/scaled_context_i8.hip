#include "scaled_context.cuh"

namespace sw {
int sc_context_i8(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  return sc_context_by_size<false, 4>(a, block_size, num_seqs, stream);
}
int sc_context_i8_wide(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  return sc_context_by_size<false, 8>(a, block_size, num_seqs, stream);
}
}  // namespace sw
