#include "scaled_context.cuh"

namespace sw {
int sc_context_i8(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  return sc_context_by_size<false>(a, block_size, num_seqs, stream);
}
}  // namespace sw
