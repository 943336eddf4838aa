// Entry points of the attention over the 8-bit cache with one scale for each (block, kv head), the choice of its launches, and the
// kernel that joins the parts of a context.
#include "scaled_attention.cuh"

#include <algorithm>

namespace sw {

using ScLaunch = int(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream);
ScLaunch sc_decode_i8, sc_decode_i8_wide, sc_decode_e4m3, sc_decode_e4m3_wide, sc_context_i8, sc_context_i8_wide, sc_context_e4m3,
    sc_context_e4m3_wide;

namespace {

constexpr int kScMostParts = 1024;

// One workgroup for each (row, head): o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p over the parts that its tile had.  A wave
// finds the factors, a part a lane; then 8 groups of 32 threads take every 8th part, 4 dims a thread (twice for heads over 128), and
// are added up through LDS.
constexpr int kScJoinThreads = 256;

template <int BS>
__global__ void __launch_bounds__(kScJoinThreads) scaled_join_kernel(const ScAttention a) {
  __shared__ float factor[kScMostParts];
  __shared__ sc_f32x4 sums[kScJoinThreads];
  const int seq = blockIdx.z, tok = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  const ScSequence s = sc_sequence<BS>(a, seq);
  if (tok >= s.fresh) return;
  const int rows = s.fresh * a.group, mine = tok * a.group + head % a.group, tile = mine / a.tile_rows;
  const int pos_low = s.first + tile * a.tile_rows / a.group;
  const int pos_high = s.first + min(rows - 1, tile * a.tile_rows + a.tile_rows - 1) / a.group;
  const int from = sc_seen_from(a, pos_low);
  const int64_t row = s.row0 + tok, step = a.head_size + 4;
  const float* parts = a.partial + (row * a.heads + head) * a.parts * step;
  auto there = [&](int p) { return max(p * a.part_tokens, from) < sc_part_end(a, s, p, pos_high); };
  if (tid < 64) {
    float m = -INFINITY, l = 0.f;
    for (int p = tid; p < a.parts; p += 64)
      if (there(p)) m = fmaxf(m, parts[p * step + a.head_size]);
    const float base = sc_base(wave_max(m));
    for (int p = tid; p < a.parts; p += 64) {
      const float f = there(p) ? __builtin_amdgcn_exp2f(parts[p * step + a.head_size] - base) : 0.f;
      if (there(p)) l += parts[p * step + a.head_size + 1] * f;
      factor[p] = f;
    }
    l = wave_sum(l);
    const float inv = l > 0.f ? 1.f / l : l != l ? l : 0.f;     // a row that sees nothing gives zeros
    for (int p = tid; p < a.parts; p += 64) factor[p] *= inv;
  }
  __syncthreads();
  for (int d = 4 * (tid & 31); d < (a.head_size + 127) / 128 * 128; d += 128) {
    sc_f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (d < a.head_size) {
#pragma unroll 4
      for (int p = tid >> 5; p < a.parts; p += 8)
        if (there(p)) o += *reinterpret_cast<const sc_f32x4*>(parts + p * step + d) * factor[p];
    }
    sums[tid] = o;
    __syncthreads();
    if (tid < 32 && d < a.head_size) {
#pragma unroll
      for (int g = 1; g < kScJoinThreads / 32; ++g) o += sums[tid + 32 * g];
      *reinterpret_cast<sc_u32x2*>(reinterpret_cast<uint16_t*>(a.out) + row * a.out_stride + (int64_t)head * a.head_size + d) =
          sc_u32x2{sc_pack16(o[0], o[1], a.bf16), sc_pack16(o[2], o[3], a.bf16)};
    }
    __syncthreads();
  }
}

// The same for few parts of many rows: a wave for each (row, head), 4 dims a lane.
template <int BS>
__global__ void __launch_bounds__(256) scaled_join_few_kernel(const ScAttention a) {
  const int seq = blockIdx.z, tok = blockIdx.x, lane = threadIdx.x & 63;
  const int head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ScSequence s = sc_sequence<BS>(a, seq);
  if (tok >= s.fresh || head >= a.heads) return;
  const int rows = s.fresh * a.group, mine = tok * a.group + head % a.group, tile = mine / a.tile_rows;
  const int pos_low = s.first + tile * a.tile_rows / a.group;
  const int pos_high = s.first + min(rows - 1, tile * a.tile_rows + a.tile_rows - 1) / a.group;
  const int from = sc_seen_from(a, pos_low);
  const int64_t row = s.row0 + tok, step = a.head_size + 4;
  const float* parts = a.partial + (row * a.heads + head) * a.parts * step;
  auto there = [&](int p) { return max(p * a.part_tokens, from) < sc_part_end(a, s, p, pos_high); };
  float m = -INFINITY, l = 0.f;
  sc_f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const bool mine_d = 4 * lane < a.head_size;
  for (int p = 0; p < a.parts; ++p) {
    if (!there(p)) continue;
    const float* at = parts + p * step;
    const sc_f32x4 v = mine_d ? *reinterpret_cast<const sc_f32x4*>(at + 4 * lane) : sc_f32x4{0.f, 0.f, 0.f, 0.f};
    const float mp = at[a.head_size], lp = at[a.head_size + 1], m_new = fmaxf(m, mp), base = sc_base(m_new);
    const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(mp - base);
    m = m_new;
    l = l * f + lp * g;
    o = o * f + v * g;
  }
  const float inv = l > 0.f ? 1.f / l : l != l ? l : 0.f;     // a row that sees nothing gives zeros
  if (mine_d)
    *reinterpret_cast<sc_u32x2*>(reinterpret_cast<uint16_t*>(a.out) + row * a.out_stride + (int64_t)head * a.head_size + 4 * lane) =
        sc_u32x2{sc_pack16(o[0] * inv, o[1] * inv, a.bf16), sc_pack16(o[2] * inv, o[3] * inv, a.bf16)};
}

template <int BS>
void sc_join(const ScAttention& a, int max_new_len, int num_seqs, hipStream_t stream) {
  if (a.parts <= 8) scaled_join_few_kernel<BS><<<dim3(max_new_len, (a.heads + 3) / 4, num_seqs), 256, 0, stream>>>(a);
  else scaled_join_kernel<BS><<<dim3(max_new_len, a.heads, num_seqs), kScJoinThreads, 0, stream>>>(a);
}

// What a call of some shape launches: which kernel, on tiles of how many rows (16: the one for few rows, else the one for many), with
// how many waves a workgroup, and over how many parts of a context.
struct ScPlan { int tile_rows, waves, parts; };

ScPlan sc_plan(int num_seqs, int max_new_len, int num_heads, int num_kv_heads, int head_size, int max_context_len) {
  ScPlan p;
  const int64_t rows = (int64_t)max_new_len * (num_heads / num_kv_heads), pairs = (int64_t)num_seqs * num_kv_heads;
  auto workgroups = [&](int tile) { return std::max<int64_t>(1, pairs * ((rows + tile - 1) / tile)); };
  // Rows of 16: all tiles of a kv head read its codes again, from the L2 but for the first, and are many workgroups where the others are
  // few (us, 16 / 128 rows: 15 x 8 tokens of 8 heads behind 1803 38 / 56, 1 x 40 behind 4000 36 / 35, 16 x 21 behind 2000 54 / 77,
  // 2 x 159 of one head behind 4000 84 / 67, 8 x 214 behind 1000 83 / 65).
  if (rows <= (head_size > 128 ? 16 : 96) || (head_size <= 128 && rows <= 160 && workgroups(16) >= 1024)) {
    p.tile_rows = 16;
    // Few workgroups take 8 waves; a context is shared out until there are about 256 of them (us, 8 waves by parts: 1 x 2001 tokens of 8
    // kv heads 1 17.2, 4 12.2, 8 10.9, 32 11.9; 4 x 6001 1 60.9, 4 25.5, 8 18.1, 16 23.1; 32 heads, 1 x 501 1 8.6, 2 10.6; 4 and 8 waves:
    // 64 x 1000 of 8 heads 38.9 / 41.5, 32 x 8192 143 / 117, 128 x 4096 220 / 212).
    const int64_t w = workgroups(16);
    p.waves = head_size <= 128 && w <= (max_context_len >= 4096 && rows <= 16 ? 1024 : 256) ? 8 : 4;
    p.parts = (int)std::min<int64_t>(max_context_len < 1024 ? 1 : ((int64_t)max_context_len + 255) / 256, 256 / w);
  } else {
    // 256 rows where there are enough of them: half the widening a row (us, 128 / 256 rows: 2041 tokens of 8 heads behind 14003 1063 / 1002,
    // 8 x 1024 behind 1000 331 / 324, 6 x 301 78 / 80, 30 x 50 behind 10 33 / 37; heads of 64, 8 x 1024, 212 / 248).
    // Fewer than the 512 that run at once (256 of heads of 256): parts, for whose sums each row costs 2 x 4 bytes a dim and part; short ones up to 256 workgroups, which
    // have few rows, and long ones up to 512 (us by parts: 120 tokens of 8 heads behind 3000 1 78.5, 4 30.7, 16 25.0, 48 25.2; behind 800 1 32.6,
    // 4 21.7, 12 21.5; 2 x 42 of 8 heads of 256 on 2 behind 2007 1 139, 3 59, 10 35, 32 31; 2 x 1000 of 4 behind 1500 1 175, 3 81, 4 101; 400 of 32 on 8 behind 12000 1 282, 4 120, 6 133, 12 142;
    // 500 of 32 behind 4000 1 110, 2 76, 4 67, 8 78; 512 of 64 on 8 behind 8000 1 198, 2 180, 4 185; 800 behind 600 1 51, 2 77; 1000 of 32 heads
    // behind 100 1 39, 2 51).
    const int64_t w = workgroups(128);
    p.tile_rows = head_size >= 80 && head_size <= 128 && w >= 512 && max_context_len >= 1024 ? 256 : 128;
    p.waves = p.tile_rows / 32;
    p.parts = (int)std::max(std::min<int64_t>(max_context_len / 192, 256 / w), std::min<int64_t>(max_context_len / 768, 512 / w));
  }
  p.parts = std::max(1, std::min(p.parts, kScMostParts));
  return p;
}

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
  SW_CHECK_ARG(num_parts >= 1 && num_parts <= kScMostParts, "%s: %d parts, at most %d", what, num_parts, kScMostParts);
  SW_CHECK_ARG(num_parts == 1 || (workspace && (uintptr_t)workspace % 16 == 0 &&
                                  workspace_bytes >= sw_scaled_attention_workspace_bytes(num_parts, a.num_rows, a.heads, a.head_size)),
               "%s: the workspace for %d parts is missing, too small or not aligned", what, num_parts);
  // (a window of all that a table holds hides nothing, and positions less it stay within 32 bits)
  if (a.window >= a.width * block_size) a.window = 0;
  a.group = a.heads / a.kv_heads;
  SW_CHECK_ARG((int64_t)max_new_len * a.group < INT32_MAX / 2, "%s: %d new tokens", what, max_new_len);
  const ScPlan plan = sc_plan(num_seqs, max_new_len, a.heads, a.kv_heads, a.head_size, max_context_len);
  a.tile_rows = plan.tile_rows;
  const int64_t tiles = ((int64_t)max_new_len * a.group + a.tile_rows - 1) / a.tile_rows;
  SW_CHECK_ARG(tiles * a.kv_heads <= kScMostWorkgroups && max_new_len <= kScMostWorkgroups, "%s: %d new tokens", what, max_new_len);
  if (num_seqs == 0 || max_new_len == 0 || a.num_rows == 0) return SW_OK;
  a.num_blocks = (int)num_blocks;
  a.tiles = (int)tiles;
  a.parts = num_parts;
  a.part_tokens = num_parts == 1 ? 0 : std::max(64, (int)((((int64_t)max_context_len + num_parts - 1) / num_parts + 63) / 64 * 64));
  a.partial = num_parts == 1 ? nullptr : (float*)workspace;
  a.bf16 = act == SW_BF16;
  const bool e4m3 = cache == SW_E4M3_SCALED;
  ScLaunch* launch = plan.tile_rows > 16 ? (plan.waves == 8 ? (e4m3 ? sc_context_e4m3_wide : sc_context_i8_wide)
                                                            : (e4m3 ? sc_context_e4m3 : sc_context_i8))
                                         : (plan.waves == 8 ? (e4m3 ? sc_decode_e4m3_wide : sc_decode_i8_wide)
                                                            : (e4m3 ? sc_decode_e4m3 : sc_decode_i8));
  const int rc = launch(a, block_size, num_seqs, stream);
  if (rc != SW_OK || num_parts == 1) return rc;
  (block_size == 8 ? sc_join<8> : block_size == 16 ? sc_join<16> : sc_join<32>)(a, max_new_len, num_seqs, stream);
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
  return sw::sc_plan(num_seqs, max_new_len, num_heads, num_kv_heads, head_size, max_context_len).parts;
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
