// Attention of many rows over the 8-bit cache with one scale for each (block, kv head) (included by scaled_context_*.hip).
//
// The mathematics of scaled_decode.cuh, for prompts: rows (new tokens times the query heads of a kv head) in tiles of 128, 32 a wave,
// bound by the matrix products and the vector work beside them, 4 head_size operations a (row, token) on the one and some 8
// instructions a (row, token) / 64 on the other.  So what can be done once for the workgroup is done once:
//   * a stage of 64 tokens goes global -> registers (one stage ahead) -> halves -> LDS, where all waves read it as operands of
//     v_mfma_f32_32x32x16_f16: S^T = K . Q^T [32 tokens x 32 rows], O^T += V^T . P^T [32 dims x 32 rows].  A row is a lane's column in both;
//   * the accumulator of S^T is P^T's operand as it stands: lane half h has tokens 8 b + 4 h + j, so values are laid down with the tokens of
//     a run of 16 in the order 0-3, 8-11, 4-7, 12-15;
//   * scales come as three numbers for each 8 tokens, made by 8 threads for all: the key scale; log2 of the value scale over the reference
//     (the largest so far), which goes into the weight's exponent; and its reciprocal, which takes it out of the weights' sum again.
//     A score costs one product-and-sum, one exp2, one addition, half a maximum and half a packing;
//   * sums are rescaled only where a row's maximum has grown by more than 2^8 or the reference has.
#pragma once

#include "scaled_attention.cuh"

namespace sw {

using sc_f32x16 = __attribute__((ext_vector_type(16))) float;

constexpr int kScWaves = 4, kScRows = 32, kScTileRows = kScWaves * kScRows;
constexpr float kScLazy = 8.f;                                // powers of two by which a weight may pass 1
constexpr float kScDeep = 40.f;                               // below the reference by more a value scale counts as that much below it

__host__ __device__ constexpr int sc_stage(int head) { return head <= 128 ? 64 : 32; }
__host__ __device__ constexpr int sc_padded(int head) { return (head + 31) / 32 * 32; }
__host__ __device__ constexpr int sc_kstride(int head) { return head * 2 + 16; }            // bytes; 16 rows on 64 banks
__host__ __device__ constexpr int sc_vstride(int head) { return sc_stage(head) * 2 + 16; }
__host__ __device__ constexpr int sc_buffer(int head) {
  return sc_stage(head) * sc_kstride(head) + sc_padded(head) * sc_vstride(head) + 128;      // and the scales
}

template <bool E4M3, int HEAD, int BS>
__global__ void __launch_bounds__(kScWaves * 64, 2) scaled_context_kernel(const ScAttention a) {
  using C = ScCode<E4M3>;
  constexpr int KT = sc_stage(HEAD), NT = KT / 32, KS = HEAD / 16, DB = sc_padded(HEAD) / 32;
  constexpr int THREADS = kScWaves * 64, PIECES = KT * HEAD / 16, NP = (PIECES + THREADS - 1) / THREADS;
  constexpr int KSTRIDE = sc_kstride(HEAD), VSTRIDE = sc_vstride(HEAD), BUFFER = sc_buffer(HEAD);
  constexpr int PB = BS == 8 ? 2 : 1, SB = KT / 8;            // blocks of a run of 16 tokens; eights of a stage
  extern __shared__ __attribute__((aligned(16))) char smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int seq = blockIdx.y, part = blockIdx.z;
  // the last rows, which see most, first; a kv head's tiles on one XCD where their number is a multiple of 8
  const int tile = a.tiles - 1 - blockIdx.x / a.kv_heads, kv_head = blockIdx.x % a.kv_heads;
  const ScSequence s = sc_sequence<BS>(a, seq);
  const int rows = s.fresh * a.group;
  if (tile * kScTileRows >= rows) return;

  const int row0 = tile * kScTileRows;
  const int pos_low = s.first + row0 / a.group, pos_high = s.first + min(rows - 1, row0 + kScTileRows - 1) / a.group;
  const int begin = max(part * a.part_tokens, sc_seen_from(a, pos_low)), end = sc_part_end(a, s, part, pos_high);
  if (a.partial && begin >= end) return;                      // (the join knows)

  // this lane's row, and the wave's range of positions
  const int w0 = row0 + wave * kScRows, my = w0 + col;
  const bool active = w0 < rows, real = my < rows;
  const int row_tok = real ? my / a.group : 0, head = kv_head * a.group + (real ? my - row_tok * a.group : 0);
  const int pos = s.first + row_tok;
  const int wave_low = s.first + w0 / a.group, wave_high = s.first + min(rows - 1, w0 + kScRows - 1) / a.group;
  const int wave_from = a.window > 0 ? max(0, wave_low - a.window + 1) : 0;
  const int none_hidden = a.window > 0 ? wave_high - a.window + 1 : 0;

  sc_u32x4 qf[KS];
  float row_scale = a.scale2;
  {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.query) + (s.row0 + row_tok) * a.q_stride + (int64_t)head * HEAD + 8 * half;
    float largest = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = real ? *reinterpret_cast<const sc_u32x4*>(q + 16 * ks) : sc_u32x4{0u, 0u, 0u, 0u};
      if (a.bf16) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          largest = fmaxf(largest, fmaxf(fabsf(bf16_bits_to_float((uint16_t)(qf[ks][w] & 0xffffu))),
                                         fabsf(bf16_bits_to_float((uint16_t)(qf[ks][w] >> 16)))));
      }
    }
    float up = 1.f;
    if (a.bf16) {
      largest = fmaxf(largest, __shfl_xor(largest, 32, 64));
      if (largest > 0.f && largest < INFINITY) {
        const int e = min(15 - (int)__builtin_amdgcn_frexp_expf(largest), 126);
        up = ldexpf(1.f, e);
        row_scale = ldexpf(row_scale, -e);
      }
    }
    // (the maximum of products with a factor is that of the products only if the factor is not negative)
    const bool flip = row_scale < 0.f;
    row_scale = fabsf(row_scale);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (a.bf16)
          qf[ks][w] = sc_pack_f16(bf16_bits_to_float((uint16_t)(qf[ks][w] & 0xffffu)) * up,
                                  bf16_bits_to_float((uint16_t)(qf[ks][w] >> 16)) * up);
        if (flip) qf[ks][w] ^= 0x80008000u;
      }
  }
  const float slope = a.slopes ? a.slopes[head] * 1.44269504088896340736f : 0.f;

  // ---- staging
  const int64_t head_bytes = (int64_t)HEAD * BS, block_bytes = head_bytes * a.kv_heads;
  const uint8_t* const k_base = a.key_cache + kv_head * head_bytes;
  const uint8_t* const v_base = a.value_cache + kv_head * head_bytes;
  const int32_t* table = a.tables + (int64_t)seq * a.table_stride;
  const int last_block = (s.len - 1) / BS;
  auto entry = [&](int t) -> int { return table[min(t / BS, last_block)]; };
  auto exists = [&](int b) { return b >= 0 && b < a.num_blocks; };
  // a thread's pieces: 16 dims of token kt[i] of the stage; dim vd[i] of the tokens of run vr[i]
  int kblock[NP], vblock[NP][PB], sblock = 0;                 // their blocks, one stage further ahead than the pieces
  sc_u32x4 kraw[NP], vraw[NP];
  float kscale = 0.f, vscale = 0.f;
  bool sgood = false;
  float reference = -INFINITY;                                // of threads 0 .. SB - 1: log2 of the largest value scale so far
  auto k_token = [&](int u) { return (u / 16 / KS) * 16 + u % 16; };
  auto look = [&](int t0) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int u = i * THREADS + tid;
      if (PIECES % THREADS != 0 && u >= PIECES) continue;
      kblock[i] = entry(t0 + k_token(u));
#pragma unroll
      for (int b = 0; b < PB; ++b) vblock[i][b] = entry(t0 + (u / HEAD) * 16 + 8 * b);
    }
    if (tid < SB) sblock = entry(t0 + 8 * tid);
  };
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int u = i * THREADS + tid;
      if (PIECES % THREADS != 0 && u >= PIECES) continue;
      {
        const int off = (t0 + k_token(u)) % BS, c = u / 16 % KS;
        const int b = exists(kblock[i]) ? kblock[i] : 0;
        kraw[i] = *reinterpret_cast<const sc_u32x4*>(k_base + b * block_bytes + (c * BS + off) * 16);
      }
      const int d = u % HEAD, off = (t0 + (u / HEAD) * 16) % BS;
      if constexpr (PB == 2) {
        sc_u32x2 w[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
          w[b] = exists(vblock[i][b]) ? *reinterpret_cast<const sc_u32x2*>(v_base + vblock[i][b] * block_bytes + d * BS) : sc_u32x2{0u, 0u};
        vraw[i] = sc_join(w[0], w[1]);
      } else {
        vraw[i] = exists(vblock[i][0]) ? *reinterpret_cast<const sc_u32x4*>(v_base + vblock[i][0] * block_bytes + d * BS + off)
                                       : sc_u32x4{0u, 0u, 0u, 0u};
      }
    }
    if (tid < SB) {
      sgood = exists(sblock);
      kscale = sgood ? a.key_scales[(int64_t)sblock * a.kv_heads + kv_head] : 0.f;
      vscale = sgood ? a.value_scales[(int64_t)sblock * a.kv_heads + kv_head] : 0.f;
    }
  };
  auto commit = [&](int t0, int buf) {
    char* k_img = smem + buf * BUFFER;
    char* v_img = k_img + KT * KSTRIDE;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int u = i * THREADS + tid;
      if (PIECES % THREADS != 0 && u >= PIECES) continue;
      sc_u32x4* kp = reinterpret_cast<sc_u32x4*>(k_img + k_token(u) * KSTRIDE + (u / 16 % KS) * 32);
      kp[0] = sc_join(C::widen(kraw[i][0]), C::widen(kraw[i][1]));
      kp[1] = sc_join(C::widen(kraw[i][2]), C::widen(kraw[i][3]));
      const int run = u / HEAD;
      sc_u32x4 v = vraw[i];
      if (E4M3 && t0 + KT > s.len) {                          // slots that hold no token may hold a NaN's code
        const int left = s.len - t0 - 16 * run;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          v[w] = left >= 4 * w + 4 ? v[w] : left <= 4 * w ? 0u : v[w] & ((1u << (8 * (left - 4 * w))) - 1u);
      }
      sc_u32x4* vp = reinterpret_cast<sc_u32x4*>(v_img + (u % HEAD) * VSTRIDE + run * 32);
      vp[0] = sc_join(C::widen(v[0]), C::widen(v[2]));
      vp[1] = sc_join(C::widen(v[1]), C::widen(v[3]));
    }
    if (tid < SB) {
      float* f = reinterpret_cast<float*>(v_img + sc_padded(HEAD) * VSTRIDE);
      const float there = t0 + 8 * tid < s.len && vscale > 0.f ? __builtin_amdgcn_logf(vscale) : -INFINITY;
      float top = there;
#pragma unroll
      for (int m = 1; m < SB; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
      reference = fmaxf(reference, top);
      const float from = sc_base(reference), below = fmaxf(there - from, -kScDeep);
      f[tid] = kscale;
      f[8 + tid] = vscale != vscale ? vscale : below;         // (a NaN of a scale reaches the rows that see its block)
      f[16 + tid] = __builtin_amdgcn_exp2f(-below);
      const uint64_t missing = __ballot(!sgood);
      if (tid == 0) {
        f[24] = from;
        reinterpret_cast<uint32_t*>(f)[25] = (uint32_t)(missing & ((1u << SB) - 1u));
      }
    }
  };

  float m_run = -INFINITY, l_run = 0.f, ref_run = 0.f;
  sc_f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[b][i] = 0.f;

  const int first = begin / KT * KT;
  const int stages = end > first ? (end - first + KT - 1) / KT : 0;
  if (stages > 0) {
    look(first);
    fetch(first);
    if (stages > 1) look(first + KT);
    commit(first, 0);
    if (stages > 1) {
      fetch(first + KT);
      if (stages > 2) look(first + 2 * KT);
    }
    __syncthreads();
  }
  int buf = 0;
  for (int st = 0; st < stages; ++st, buf ^= 1) {
    const int t0 = first + st * KT;
    if (st + 1 < stages) commit(t0 + KT, buf ^ 1);
    if (st + 2 < stages) {
      fetch(t0 + 2 * KT);
      if (st + 3 < stages) look(t0 + 3 * KT);
    }
    if (active && t0 <= wave_high && t0 + KT > wave_from) {
      const char* k_img = smem + buf * BUFFER;
      const char* v_img = k_img + KT * KSTRIDE;
      const float* f = reinterpret_cast<const float*>(v_img + sc_padded(HEAD) * VSTRIDE);
      const char* kp = k_img + col * KSTRIDE + half * 16;
      sc_f32x16 x[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int u = 0; u < NT; ++u)
          x[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const sc_f16x8*>(kp + u * 32 * KSTRIDE + ks * 32),
                                                        __builtin_bit_cast(sc_f16x8, qf[ks]), x[u], 0, 0, 0);

      // scores in powers of two: x fs (+ nothing more, where no row has anything to hide or to add)
      float fs[SB];
#pragma unroll
      for (int b = 0; b < SB; ++b) fs[b] = f[b] * row_scale;
      const uint32_t missing = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t*>(f)[25]);
      const float ref = f[24];
      if (t0 + KT > wave_low + 1 || t0 < none_hidden || missing || a.slopes) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int b = u * 4 + (i >> 2), t = t0 + 8 * b + 4 * half + (i & 3);
            float v = x[u][i] * fs[b];
            if (a.slopes) v += slope * (float)(t - pos);
            const bool see = t <= pos && (a.window <= 0 || t > pos - a.window) && !(missing >> b & 1u);
            x[u][i] = see ? v : -INFINITY;
          }
#pragma unroll
        for (int b = 0; b < SB; ++b) fs[b] = 1.f;
      }
      float top = -INFINITY;
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        const int u = b >> 2, i = (b & 3) * 4;
        top = fmaxf(top, fmaxf(fmaxf(x[u][i], x[u][i + 1]), fmaxf(x[u][i + 2], x[u][i + 3])) * fs[b]);
      }
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > m_run + kScLazy) || ref != ref_run) {
        const float m_new = fmaxf(m_run, top);
        const float alpha = __builtin_amdgcn_exp2f(m_run - sc_base(m_new));
        m_run = m_new;
        l_run *= alpha;
        const float shrink = alpha > 0.f ? alpha * __builtin_amdgcn_exp2f(ref_run - ref) : 0.f;   // (the first reference may be any)
        ref_run = ref;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[b][i] *= shrink;
      }
      const float base = sc_base(m_run);
      sc_u32x4 pf[NT][2];
#pragma unroll
      for (int b = 0; b < SB; ++b) {
        const int u = b >> 2, i = (b & 3) * 4;
        const float c = f[8 + b] - base;
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(x[u][i + j], fs[b], c));
        l_run = fmaf((p[0] + p[1]) + (p[2] + p[3]), f[16 + b], l_run);
        pf[u][(b & 3) >> 1][2 * (b & 1)] = sc_pack_f16(p[0], p[1]);
        pf[u][(b & 3) >> 1][2 * (b & 1) + 1] = sc_pack_f16(p[2], p[3]);
      }
      const char* vp = v_img + col * VSTRIDE + half * 16;
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int b = 0; b < DB; ++b)
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const sc_f16x8*>(vp + b * 32 * VSTRIDE + u * 64 + h * 32),
                                                          __builtin_bit_cast(sc_f16x8, pf[u][h]), o[b], 0, 0, 0);
    }
    __syncthreads();
  }

  l_run += __shfl_xor(l_run, 32, 64);
  if (!real) return;
  const float unit = __builtin_amdgcn_exp2f(ref_run);
  const float inv = a.partial ? unit : l_run > 0.f ? unit / l_run : l_run != l_run ? l_run : 0.f;   // a row that sees nothing gives zeros
  float* to = nullptr;
  uint16_t* out = nullptr;
  if (a.partial) {
    to = a.partial + (((s.row0 + row_tok) * a.heads + head) * a.parts + part) * (HEAD + 4);
    if (half == 0) {
      to[HEAD] = m_run;
      to[HEAD + 1] = l_run;
    }
  } else {
    out = reinterpret_cast<uint16_t*>(a.out) + (s.row0 + row_tok) * a.out_stride + (int64_t)head * HEAD;
  }
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * b + 8 * q + 4 * half;
      if (HEAD % 32 != 0 && d >= HEAD) continue;
      const float v0 = o[b][4 * q] * inv, v1 = o[b][4 * q + 1] * inv, v2 = o[b][4 * q + 2] * inv, v3 = o[b][4 * q + 3] * inv;
      if (a.partial) *reinterpret_cast<sc_f32x4*>(to + d) = sc_f32x4{v0, v1, v2, v3};
      else *reinterpret_cast<sc_u32x2*>(out + d) = sc_u32x2{sc_pack16(v0, v1, a.bf16), sc_pack16(v2, v3, a.bf16)};
    }
}

template <bool E4M3, int HEAD, int BS>
int sc_launch_context(const ScAttention& a, int num_seqs, hipStream_t stream) {
  constexpr int lds = 2 * sc_buffer(HEAD);
  static_assert(lds <= 160 * 1024, "two stages must fit a compute unit's LDS");
  auto kernel = scaled_context_kernel<E4M3, HEAD, BS>;
  if (lds > 64 * 1024)
    SW_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  kernel<<<dim3(a.kv_heads * a.tiles, num_seqs, a.parts), kScWaves * 64, lds, stream>>>(a);
  SW_CHECK_LAUNCH();
  return SW_OK;
}

template <bool E4M3, int BS>
int sc_context_by_head(const ScAttention& a, int num_seqs, hipStream_t stream) {
  switch (a.head_size) {
    case 64: return sc_launch_context<E4M3, 64, BS>(a, num_seqs, stream);
    case 80: return sc_launch_context<E4M3, 80, BS>(a, num_seqs, stream);
    case 96: return sc_launch_context<E4M3, 96, BS>(a, num_seqs, stream);
    case 112: return sc_launch_context<E4M3, 112, BS>(a, num_seqs, stream);
    case 128: return sc_launch_context<E4M3, 128, BS>(a, num_seqs, stream);
    default: return sc_launch_context<E4M3, 256, BS>(a, num_seqs, stream);
  }
}

template <bool E4M3>
int sc_context_by_size(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  return block_size == 8    ? sc_context_by_head<E4M3, 8>(a, num_seqs, stream)
         : block_size == 16 ? sc_context_by_head<E4M3, 16>(a, num_seqs, stream)
                            : sc_context_by_head<E4M3, 32>(a, num_seqs, stream);
}

}  // namespace sw
