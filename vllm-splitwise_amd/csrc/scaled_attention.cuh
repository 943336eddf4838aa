// Attention over the 8-bit cache with one scale for each (block, kv head): what its two kernels share.
#pragma once

#include "scaled_cache.cuh"

namespace sw {

using sc_f32x4 = __attribute__((ext_vector_type(4))) float;
using sc_f16x8 = __attribute__((ext_vector_type(8))) _Float16;

struct ScAttention {
  void* out;                       // [rows, heads, head_size]
  const void* query;
  const uint8_t *key_cache, *value_cache;
  const float *key_scales, *value_scales, *slopes;
  const int32_t *tables, *starts, *new_lens, *lens;      // starts null: sequence i has one new token, in row i
  float* partial;                  // null or the workspace, which then takes the sums: [rows, heads, parts, head_size + 4], sums, the
                                   // scores' maximum (powers of two), the weights' sum
  int64_t q_stride, out_stride, num_rows, table_stride;
  int num_blocks, width, heads, kv_heads, group, head_size;
  int window;                      // 0: none
  int part_tokens, parts, tiles, tile_rows, most_new;
  float scale2;                    // the softmax's scale times log2(e): everything below is in powers of two
  bool bf16;
};

// A sequence as the kernels see it: its first row, new tokens and whole length, held to what the arguments can address.
// `first`: the position of its first row (below 0 if there are more new tokens than tokens; such rows see nothing).
struct ScSequence { int64_t row0; int fresh, len, first; };

template <int BS>
__device__ __forceinline__ ScSequence sc_sequence(const ScAttention& a, int seq) {
  ScSequence s;
  s.len = (int)max((int64_t)0, min((int64_t)a.lens[seq], (int64_t)a.width * BS));
  if (a.starts == nullptr) {
    s.row0 = seq, s.fresh = 1, s.first = s.len - 1;
  } else {
    s.row0 = a.starts[seq], s.fresh = max(a.new_lens[seq], 0), s.first = s.len - s.fresh;
    if (s.row0 < 0) s.row0 = 0, s.fresh = 0;
    s.fresh = (int)min((int64_t)min(s.fresh, a.most_new), a.num_rows - s.row0);
  }
  return s;
}

__device__ __forceinline__ float sc_from16(uint32_t half, bool bf16) {
  return bf16 ? bf16_bits_to_float((uint16_t)half) : f16_bits_to_float((uint16_t)half);
}
__device__ __forceinline__ uint32_t sc_pack_f16(float a, float b) {
  using f32x2 = __attribute__((ext_vector_type(2))) float;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), sc_f16x2));     // one instruction, to the nearest
}
__device__ __forceinline__ uint32_t sc_pack16(float a, float b, bool bf16) {
  using f32x2 = __attribute__((ext_vector_type(2))) float;
  using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
  return bf16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2)) : sc_pack_f16(a, b);
}

__device__ __forceinline__ sc_f32x4 sc_mfma(sc_u32x4 a, sc_u32x4 b, sc_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(sc_f16x8, a), __builtin_bit_cast(sc_f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ sc_u32x4 sc_join(sc_u32x2 a, sc_u32x2 b) { return sc_u32x4{a[0], a[1], b[0], b[1]}; }

// The first of the tokens that rows from position `pos_low` on see, down to a multiple of 64; the end of what part `part` does for rows
// up to position `pos_high` (the last part goes on to the end, whatever the parts were planned for).
__device__ __forceinline__ int sc_seen_from(const ScAttention& a, int pos_low) {
  return a.window > 0 ? max(0, pos_low - a.window + 1) & ~63 : 0;
}
__device__ __forceinline__ int sc_part_end(const ScAttention& a, const ScSequence& s, int part, int pos_high) {
  const int end = min(s.len, pos_high + 1);
  return part == a.parts - 1 ? end : min(end, (part + 1) * a.part_tokens);
}

// A value scale as a power of two.  Less than any write leaves is that of a block of zeros: further down than any sum reaches.
constexpr float kScNone = -300.f;
__device__ __forceinline__ float sc_log_scale(float s) {
  return s < kScLeast ? kScNone : __builtin_amdgcn_logf(s);  // (a NaN stays one)
}
// A value scale further below the row's reference than this counts as that far below it: its weights are 0 as halves either way, and
// their sum, brought back by the scale, is still far from the smallest number.
constexpr float kScDeep = 80.f;

// exp2 of the difference to the running maximum, which is minus infinity while nothing has been seen
__device__ __forceinline__ float sc_base(float m) { return m == -INFINITY ? 0.f : m; }

}  // namespace sw
