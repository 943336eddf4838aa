// Entry points of the attention over the 8-bit cache with one scale for each (block, kv head), the choice of its launches, and the
// kernel that joins the parts of a context.
#include "scaled_attention.cuh"

#include <algorithm>

namespace sw {

int sc_decode_i8(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream);
int sc_decode_e4m3(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream);
int sc_context_i8(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream);
int sc_context_e4m3(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream);

namespace {

// One workgroup for each (row, head): o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p over the parts that its tile had.
template <int BS>
__global__ void __launch_bounds__(256) scaled_join_kernel(const ScAttention a) {
  const int seq = blockIdx.z, tok = blockIdx.x, head = blockIdx.y, d = threadIdx.x;
  const ScSequence s = sc_sequence<BS>(a, seq);
  if (tok >= s.fresh) return;
  const int rows = s.fresh * a.group, mine = tok * a.group + head % a.group, tile = mine / a.tile_rows;
  const int pos_low = s.first + tile * a.tile_rows / a.group;
  const int pos_high = s.first + min(rows - 1, tile * a.tile_rows + a.tile_rows - 1) / a.group;
  const int from = sc_seen_from(a, pos_low);
  const int64_t row = s.row0 + tok;
  const float* parts = a.partial + (row * a.heads + head) * a.parts * (a.head_size + 4);
  const int64_t step = a.head_size + 4;
  auto there = [&](int p) { return max(p * a.part_tokens, from) < sc_part_end(a, s, p, pos_high); };
  float m = -INFINITY;
  for (int p = 0; p < a.parts; ++p)
    if (there(p)) m = fmaxf(m, parts[p * step + a.head_size]);
  const float base = sc_base(m);
  float l = 0.f, o = 0.f;
  for (int p = 0; p < a.parts; ++p) {
    if (!there(p)) continue;
    const float f = __builtin_amdgcn_exp2f(parts[p * step + a.head_size] - base);
    l += parts[p * step + a.head_size + 1] * f;
    if (d < a.head_size) o += parts[p * step + d] * f;
  }
  if (d >= a.head_size) return;
  const float res = l > 0.f ? o / l : l != l ? l : 0.f;
  reinterpret_cast<uint16_t*>(a.out)[row * a.out_stride + (int64_t)head * a.head_size + d] =
      a.bf16 ? float_to_bf16_bits(res) : float_to_f16_bits(res);
}

// Rows of a tile for `rows` rows of a (sequence, kv head): 16 of the kernel for few rows or 128 of the one for many.
int sc_tile_rows(int64_t rows) { return rows <= 16 ? 16 : 128; }

int sc_attend(const char* what, ScAttention a, int num_seqs, int64_t num_blocks, int block_size, int max_new_len, int max_context_len,
              int act, int cache, int num_parts, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  SW_CHECK_ARG(cache == SW_I8_SCALED || cache == SW_E4M3_SCALED, "%s: the cache type must be scaled int8 or e4m3", what);
  SW_CHECK_ARG(act == SW_F16 || act == SW_BF16, "%s: f16 and bf16 only", what);
  SW_CHECK_ARG(sc_head_size(a.head_size), "%s: Unsupported head size: %d", what, a.head_size);
  SW_CHECK_ARG(block_size == 8 || block_size == 16 || block_size == 32, "%s: Unsupported block size: %d", what, block_size);
  SW_CHECK_ARG(a.kv_heads > 0 && a.heads > 0 && a.heads % a.kv_heads == 0 && a.heads <= 65535,
               "%s: %d query heads on %d kv heads", what, a.heads, a.kv_heads);
  SW_CHECK_ARG(num_blocks > 0 && num_blocks <= INT32_MAX, "%s: %lld blocks", what, (long long)num_blocks);
  SW_CHECK_ARG(num_seqs >= 0 && num_seqs <= 65535, "%s: %d sequences, at most 65535 in a call", what, num_seqs);
  SW_CHECK_ARG(max_new_len >= 0 && max_context_len >= 0 && a.width >= 0 && a.num_rows >= 0, "%s: negative sizes", what);
  // positions and the tokens of whole tables are 32-bit numbers, with a group's 64 to spare
  SW_CHECK_ARG((int64_t)a.width * block_size < INT32_MAX - 4096, "%s: block tables of %d blocks are too wide", what, a.width);
  SW_CHECK_ARG((uintptr_t)a.query % 16 == 0 && a.q_stride % 8 == 0 && (uintptr_t)a.out % 16 == 0 && a.out_stride % 8 == 0 &&
                   (uintptr_t)a.key_cache % 16 == 0 && (uintptr_t)a.value_cache % 16 == 0,
               "%s: rows of query and out, and the caches, must begin on multiples of 16 bytes", what);
  SW_CHECK_ARG(num_parts >= 1 && num_parts <= 65535, "%s: %d parts", what, num_parts);
  SW_CHECK_ARG(num_parts == 1 || (workspace && (uintptr_t)workspace % 16 == 0 &&
                                  workspace_bytes >= sw_scaled_attention_workspace_bytes(num_parts, a.num_rows, a.heads, a.head_size)),
               "%s: the workspace for %d parts is missing, too small or not aligned", what, num_parts);
  a.group = a.heads / a.kv_heads;
  a.tile_rows = sc_tile_rows((int64_t)max_new_len * a.group);
  const int64_t tiles = ((int64_t)max_new_len * a.group + a.tile_rows - 1) / a.tile_rows;
  SW_CHECK_ARG((int64_t)max_new_len * a.group < INT32_MAX / 2 && tiles * a.kv_heads <= INT32_MAX, "%s: %d new tokens", what, max_new_len);
  if (num_seqs == 0 || max_new_len == 0 || a.num_rows == 0) return SW_OK;
  a.num_blocks = (int)num_blocks;
  a.tiles = (int)tiles;
  a.parts = num_parts;
  a.part_tokens = num_parts == 1 ? 0 : std::max(64, (int)((((int64_t)max_context_len + num_parts - 1) / num_parts + 63) / 64 * 64));
  a.partial = num_parts == 1 ? nullptr : (float*)workspace;
  a.bf16 = act == SW_BF16;
  const bool e4m3 = cache == SW_E4M3_SCALED;
  const int rc = a.tile_rows == 16 ? (e4m3 ? sc_decode_e4m3 : sc_decode_i8)(a, block_size, num_seqs, stream)
                                   : (e4m3 ? sc_context_e4m3 : sc_context_i8)(a, block_size, num_seqs, stream);
  if (rc != SW_OK || num_parts == 1) return rc;
  const dim3 grid(max_new_len, a.heads, num_seqs);
  const int threads = (a.head_size + 63) / 64 * 64;
  if (block_size == 8) scaled_join_kernel<8><<<grid, threads, 0, stream>>>(a);
  else if (block_size == 16) scaled_join_kernel<16><<<grid, threads, 0, stream>>>(a);
  else scaled_join_kernel<32><<<grid, threads, 0, stream>>>(a);
  SW_CHECK_LAUNCH();
  return SW_OK;
}

ScAttention sc_arguments(void* out, const void* query, const void* key_cache, const void* value_cache, const float* key_scales,
                         const float* value_scales, int num_heads, int num_kv_heads, int head_size, float scale,
                         const int32_t* block_tables, const int32_t* lens, int max_blocks_per_seq, int64_t table_stride,
                         const float* alibi_slopes, int64_t q_stride, int64_t out_stride) {
  ScAttention a = {};
  a.out = out, a.query = query;
  a.key_cache = (const uint8_t*)key_cache, a.value_cache = (const uint8_t*)value_cache;
  a.key_scales = key_scales, a.value_scales = value_scales, a.slopes = alibi_slopes;
  a.tables = block_tables, a.lens = lens;
  a.q_stride = q_stride, a.out_stride = out_stride, a.table_stride = table_stride;
  a.width = max_blocks_per_seq, a.heads = num_heads, a.kv_heads = num_kv_heads, a.head_size = head_size;
  a.scale2 = scale * 1.44269504088896340736f;
  return a;
}

}  // namespace

}  // namespace sw

extern "C" {

int sw_scaled_attention_parts(int num_seqs, int max_new_len, int num_heads, int num_kv_heads, int head_size, int max_context_len) {
  if (num_seqs <= 0 || max_new_len <= 0 || num_kv_heads <= 0 || num_heads < num_kv_heads || max_context_len <= 0) return 1;
  const int64_t rows = (int64_t)max_new_len * (num_heads / num_kv_heads), tile = sw::sc_tile_rows(rows);
  const int64_t tiles = (rows + tile - 1) / tile;
  const int64_t workgroups = (int64_t)num_seqs * num_kv_heads * tiles;
  const int64_t most = ((int64_t)max_context_len + 255) / 256;
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, 1024 / workgroups));
}

int64_t sw_scaled_attention_workspace_bytes(int num_parts, int64_t num_rows, int num_heads, int head_size) {
  return num_parts <= 1 ? 0 : (int64_t)num_parts * num_rows * num_heads * (head_size + 4) * 4;
}

int sw_paged_attention_scaled(void* out, const void* query, const void* key_cache, const void* value_cache, const float* key_scales,
                              const float* value_scales, int num_seqs, int num_heads, int num_kv_heads, int head_size, float scale,
                              const int32_t* block_tables, const int32_t* context_lens, int block_size, int64_t num_blocks,
                              int max_context_len, int max_blocks_per_seq, int64_t table_stride, const float* alibi_slopes,
                              int64_t q_stride, int64_t out_stride, int act_dtype, int cache_dtype, int num_parts, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  using namespace sw;
  ScAttention a = sc_arguments(out, query, key_cache, value_cache, key_scales, value_scales, num_heads, num_kv_heads, head_size, scale,
                               block_tables, context_lens, max_blocks_per_seq, table_stride, alibi_slopes, q_stride, out_stride);
  a.num_rows = num_seqs;
  return sc_attend("paged_attention_scaled", a, num_seqs, num_blocks, block_size, 1, max_context_len, act_dtype, cache_dtype, num_parts,
                   workspace, workspace_bytes, (hipStream_t)stream);
}

int sw_context_attention_scaled(void* out, const void* query, const void* key_cache, const void* value_cache, const float* key_scales,
                                const float* value_scales, int num_seqs, int64_t num_rows, int num_heads, int num_kv_heads,
                                int head_size, float scale, const int32_t* block_tables, const int32_t* seq_starts,
                                const int32_t* new_lens, const int32_t* seq_lens, int block_size, int64_t num_blocks, int max_new_len,
                                int max_context_len, int max_blocks_per_seq, int64_t table_stride, const float* alibi_slopes,
                                int sliding_window, int64_t q_stride, int64_t out_stride, int act_dtype, int cache_dtype, int num_parts,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace sw;
  ScAttention a = sc_arguments(out, query, key_cache, value_cache, key_scales, value_scales, num_heads, num_kv_heads, head_size, scale,
                               block_tables, seq_lens, max_blocks_per_seq, table_stride, alibi_slopes, q_stride, out_stride);
  a.starts = seq_starts, a.new_lens = new_lens, a.num_rows = num_rows, a.window = sliding_window;
  a.most_new = max_new_len;
  return sc_attend("context_attention_scaled", a, num_seqs, num_blocks, block_size, max_new_len, max_context_len, act_dtype, cache_dtype,
                   num_parts, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
