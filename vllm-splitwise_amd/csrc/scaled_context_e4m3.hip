#include "scaled_context.cuh"

namespace sw {
int sc_context_e4m3(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  return sc_context_by_size<true>(a, block_size, num_seqs, stream);
}
}  // namespace sw
