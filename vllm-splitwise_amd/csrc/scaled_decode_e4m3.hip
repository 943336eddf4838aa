#include "scaled_decode.cuh"

namespace sw {
int sc_decode_e4m3(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  return sc_decode_by_size<true, 4>(a, block_size, num_seqs, stream);
}
int sc_decode_e4m3_wide(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  return sc_decode_by_size<true, 8>(a, block_size, num_seqs, stream);
}
}  // namespace sw
