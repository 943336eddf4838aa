// Attention of many rows over the 8-bit cache with one scale for each (block, kv head) (included by scaled_context_*.hip).
//
// The mathematics of scaled_decode.cuh, for prompts: rows (new tokens times the query heads of a kv head) in tiles of 128 or 256, 32 a wave,
// bound by the matrix products and the vector work beside them, 4 head_size operations a (row, token) on the one and some 8
// instructions a (row, token) / 64 on the other.  So what can be done once for the workgroup is done once:
//   * a stage of 64 tokens goes global -> registers (one stage ahead) -> halves -> LDS, where all waves read it as operands of
//     v_mfma_f32_32x32x16_f16: S^T = K . Q^T [32 tokens x 32 rows], O^T += V^T . P^T [32 dims x 32 rows].  A row is a lane's column in both;
//   * the accumulator of S^T is P^T's operand as it stands: lane half h has tokens 8 b + 4 h + j, so values are laid down with the tokens of
//     a run of 16 in the order 0-3, 8-11, 4-7, 12-15;
//   * scales come as three numbers for each 8 tokens, made by 8 threads for all: the key scale; log2 of the value scale, which goes into
//     the weight's exponent; and its reciprocal, which takes it out of the weights' sum again.  A score costs one product-and-sum, one
//     exp2, one addition, half a maximum and half a packing;
//   * sums are rescaled only where a row's maximum or its reference may have grown by more than 2^8: the largest score and the largest
//     value scale of a stage say so, and only then is looked for the largest of both together.
// Measured: 2041 tokens of 64 heads of 128 on 8 behind 14003, bf16, int8, 1001 to 1027 us from card to card (under a profiler 1071 to 1203), 1.0
// PFLOP/s, where a plain product of large matrices reaches 1.2: matrix cores busy 47 % of the cycles and vector units 57 %, at a clock that
// the power lets down to 2 GHz.  (So what takes vector instructions out counts, not what moves them: two halves of the waves half a stage
// apart, with a barrier more, 1135; all products of a stage together and its weights behind them 1125.)  8 x 1024 of 32 heads on 8 behind
// 1000 324 us.
#pragma once

#include "scaled_attention.cuh"

namespace sw {

using sc_f32x16 = __attribute__((ext_vector_type(16))) float;

constexpr int kScRows = 32;                                   // of a wave
constexpr float kScLazy = 8.f;                                // powers of two by which a row's maximum may pass what its sums are to
constexpr float kScRaised = 7.f;                              // and that its largest weight then stands above 1: 2^15 at most fits a half

constexpr float kScApart = 90.f;                              // powers of two by which that reference and the scores' maximum may be apart

constexpr int kScSteps = 8;                                   // dwords of codes of a key's piece and a value's

__host__ __device__ constexpr int sc_stage(int head) { return head <= 128 ? 64 : 32; }
__host__ __device__ constexpr int sc_padded(int head) { return (head + 31) / 32 * 32; }
__host__ __device__ constexpr int sc_kstride(int head) { return head * 2 + 16; }            // bytes; 16 rows on 64 banks
__host__ __device__ constexpr int sc_vstride(int head) { return sc_stage(head) * 2 + 16; }
__host__ __device__ constexpr int sc_buffer(int head) {
  return sc_stage(head) * sc_kstride(head) + sc_padded(head) * sc_vstride(head) + 128;      // and the scales
}

// The larger one; a NaN, if one of them is one.  (One instruction for three, and none to quiet a NaN first.)
__device__ __forceinline__ float sc_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The larger and the smaller of a lane's number and another lane's (a register's lanes crossed as CTRL says).
template <int CTRL>
__device__ __forceinline__ void sc_most_least(float& most, float& least) {
  most = fmaxf(most, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(most), CTRL, 0xf, 0xf, true)));
  least = fminf(least, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(least), CTRL, 0xf, 0xf, true)));
}

// Waves of a SIMD that the registers are shared out for.  (Two for heads of 256 leave some 50 of a lane's numbers in memory: 2 x 1000 tokens of
// 4 heads behind 1500 115 us, 81 with one.  Heads of 64 need 2 registers more than three waves have: 8 x 1024 tokens of 32 heads on 8 behind
// 1000 265 us with two waves, 220 with three and those 2 in memory.)
__host__ __device__ constexpr int sc_waves(int head) { return head > 128 ? 1 : head == 64 ? 3 : 2; }

template <bool E4M3, int HEAD, int BS, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, sc_waves(HEAD)) scaled_context_kernel(const ScAttention a) {
  using C = ScCode<E4M3>;
  constexpr int TILE = WAVES * kScRows;
  constexpr int KT = sc_stage(HEAD), NT = KT / 32, KS = HEAD / 16, DB = sc_padded(HEAD) / 32;
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
  if (tile * TILE >= rows) return;

  const int row0 = tile * TILE;
  const int pos_low = s.first + row0 / a.group, pos_high = s.first + min(rows - 1, row0 + TILE - 1) / a.group;
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

  // ---- staging: a wave brings one run of 16 tokens (half of one, where there are fewer runs than waves), so that its blocks are the same
  // for all its lanes; a lane's pieces are 16 dims of one token's key and 16 tokens of one dim's values
  const int64_t head_bytes = (int64_t)HEAD * BS, block_bytes = head_bytes * a.kv_heads;
  const uint8_t* const k_base = a.key_cache + kv_head * head_bytes;
  const uint8_t* const v_base = a.value_cache + kv_head * head_bytes;
  const int32_t* table = a.tables + (int64_t)seq * a.table_stride;
  const int last_block = (s.len - 1) / BS;
  constexpr int RUNS = KT / 16, SHARE = WAVES / RUNS, NP = (HEAD + 64 * SHARE - 1) / (64 * SHARE);
  const int run = wave / SHARE, u0 = (wave % SHARE) * 64 + lane;
  auto mine = [&](int i) { return HEAD % (64 * SHARE) == 0 || u0 + i * 64 * SHARE < HEAD; };
  // (stages behind the last one bring the last block again: what they lay down is not read)
  auto entry = [&](int t) -> int { return table[min(t / BS, last_block)]; };
  int runblock[PB], sblock = 0;                               // one stage further ahead than the pieces
  sc_u32x4 kraw[NP], vraw[NP], keep = {0u, 0u, 0u, 0u};
  float kscale = 0.f, vscale = 0.f;
  bool sgood = false;
  auto look = [&](int t0) {
#pragma unroll
    for (int b = 0; b < PB; ++b) runblock[b] = entry(t0 + 16 * run + 8 * b);
    if (tid < SB) sblock = entry(t0 + 8 * tid);
  };
  auto fetch = [&](int t0) {
    const int off = (t0 + 16 * run) % BS;                     // of the run in its block
    bool good[PB];
    int64_t at[PB];
#pragma unroll
    for (int b = 0; b < PB; ++b) {
      good[b] = runblock[b] >= 0 && runblock[b] < a.num_blocks;
      at[b] = (good[b] ? runblock[b] : 0) * block_bytes;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (!mine(i)) continue;
      const int u = u0 + i * 64 * SHARE, t = u & 15, c = u >> 4;
      if constexpr (PB == 2) {
        kraw[i] = *reinterpret_cast<const sc_u32x4*>(k_base + (t < 8 ? at[0] : at[1]) + (c * BS + (t & 7)) * 16);
        vraw[i] = sc_join(*reinterpret_cast<const sc_u32x2*>(v_base + at[0] + u * BS), *reinterpret_cast<const sc_u32x2*>(v_base + at[1] + u * BS));
      } else {
        kraw[i] = *reinterpret_cast<const sc_u32x4*>(k_base + at[0] + off * 16 + (c * BS + t) * 16);
        vraw[i] = *reinterpret_cast<const sc_u32x4*>(v_base + at[0] + off + u * BS);
      }
    }
    if (tid < SB) {
      sgood = sblock >= 0 && sblock < a.num_blocks;
      kscale = sgood ? a.key_scales[(int64_t)sblock * a.kv_heads + kv_head] : 0.f;
      vscale = sgood ? a.value_scales[(int64_t)sblock * a.kv_heads + kv_head] : 0.f;
    }
    // slots that hold no token may hold a NaN's code: which of the run's values are kept
    if constexpr (E4M3) {
      const int left = s.len - t0 - 16 * run;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n = left - 4 * w;
        keep[w] = !good[PB == 2 ? w >> 1 : 0] || n <= 0 ? 0u : n >= 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
      }
    }
  };
  // widening and laying down, one of kScSteps * NP steps: a dword of codes each, 16 bytes stored with every second one
  sc_u32x2 held;
  auto lay_step = [&](auto K, int buf) {
    constexpr int i = decltype(K)::value / kScSteps, j = decltype(K)::value % kScSteps, w = j < 4 ? j : j == 5 ? 2 : j == 6 ? 1 : j & 3;
    if (!mine(i)) return;
    char* k_img = smem + buf * BUFFER;
    char* v_img = k_img + KT * KSTRIDE;
    const int u = u0 + i * 64 * SHARE;
    uint32_t code = j < 4 ? kraw[i][w] : vraw[i][w];
    if constexpr (E4M3 && j >= 4) code &= keep[w];
    const sc_u32x2 wide = C::widen(code);
    if constexpr (j % 2 == 0) {
      held = wide;
    } else {
      char* to = j < 4 ? k_img + (16 * run + (u & 15)) * KSTRIDE + (u >> 4) * 32 : v_img + u * VSTRIDE + run * 32;
      *reinterpret_cast<sc_u32x4*>(to + (j & 2) * 8) = sc_join(held, wide);
    }
  };
  auto lay = [&](int buf) { static_for<kScSteps * NP>([&](auto K) { lay_step(K, buf); }); };
  // eight tokens' key scale, log2 of the value scale, its reciprocal (finite, and of no use where the scale is that of zeros); which eights
  // do not exist, the largest and the least logarithm
  auto lay_scales = [&](int buf) {
    if (tid < SB) {
      float* f = reinterpret_cast<float*>(smem + buf * BUFFER + KT * KSTRIDE + sc_padded(HEAD) * VSTRIDE);
      f[tid] = kscale;
      float most = sc_log_scale(vscale), least = most;
      f[8 + tid] = most;
      f[16 + tid] = __builtin_amdgcn_rcpf(fmaxf(vscale, kScLeast));
      const uint64_t missing = __ballot(!sgood);
      sc_most_least<0xB1>(most, least);                        // of the neighbour, of the next two, of the other four
      sc_most_least<0x4E>(most, least);
      if constexpr (SB == 8) sc_most_least<0x141>(most, least);
      if (tid == 0) reinterpret_cast<uint32_t*>(f)[24] = (uint32_t)(missing & ((1u << SB) - 1u)), f[25] = most, f[26] = least;
    }
  };

  float m_run = -INFINITY, l_run = 0.f;
  float y_run = -INFINITY, unit = 0.f;                         // what the row's sums are powers of two to; 2^(it - m_run)
  float low = -INFINITY;                                       // a value scale that is none of the weights' sum as it stands
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
    look(first + KT);
    lay(0);
    lay_scales(0);
    fetch(first + KT);
    look(first + 2 * KT);
    __syncthreads();
  }
  int buf = 0;
  for (int st = 0; st < stages; ++st, buf ^= 1) {
    const int t0 = first + st * KT;
    lay_scales(buf ^ 1);
    if (!(active && t0 <= wave_high && t0 + KT > wave_from)) {
      lay(buf ^ 1);
      fetch(t0 + 2 * KT);
      look(t0 + 3 * KT);
    } else {
      const char* k_img = smem + buf * BUFFER;
      const char* v_img = k_img + KT * KSTRIDE;
      const float* f = reinterpret_cast<const float*>(v_img + sc_padded(HEAD) * VSTRIDE);
      const char* kp = k_img + col * KSTRIDE + half * 16;
      sc_f32x16 x[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
      float fs[SB], log_v[SB];
#pragma unroll
      for (int b = 0; b < SB; ++b) fs[b] = f[b] * row_scale, log_v[b] = f[8 + b];
      const float most_v = f[25], least_v = f[26];
      const uint32_t missing = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t*>(f)[24]);
      auto top_of = [&](int b) {
        const int u = b >> 2, i = (b & 3) * 4;
        return sc_max(sc_max(x[u][i], x[u][i + 1]), sc_max(x[u][i + 2], x[u][i + 3])) * fs[b];
      };
      float top = -INFINITY;
      __builtin_amdgcn_s_setprio(1);
      // The scores' products, their operands read ahead; between them the next stage's widening and the maximum of the scores that
      // are there: the order is held.
      {
        auto operand = [&](int n) { return *reinterpret_cast<const sc_f16x8*>(kp + n / KS * 32 * KSTRIDE + n % KS * 32); };
        // (heads of 256 have no registers for more than one ahead: 166 us for 2 x 1000 tokens of 4 heads behind 1500, 214 with three and two)
        constexpr int N = NT * KS, AHEAD = HEAD > 128 ? 1 : 3, STEPS = kScSteps * NP;
        sc_f16x8 ring[AHEAD + 1];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) ring[n] = operand(n);
        static_for<N>([&](auto I) {
          constexpr int n = decltype(I)::value, u = n / KS;
          if constexpr (n + AHEAD < N) ring[(n + AHEAD) % (AHEAD + 1)] = operand(n + AHEAD);
          x[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[n % (AHEAD + 1)], __builtin_bit_cast(sc_f16x8, qf[n % KS]), x[u], 0, 0, 0);
          static_for<STEPS*(n + 1) / N - STEPS * n / N>(
              [&](auto K) { lay_step(std::integral_constant<int, STEPS * n / N + decltype(K)::value>{}, buf ^ 1); });
          if constexpr (u > 0 && n % KS >= KS - 4) top = sc_max(top, top_of(4 * u - 4 + n % KS - KS + 4));
          __builtin_amdgcn_sched_barrier(0);
        });
      }
      __builtin_amdgcn_s_setprio(0);
      fetch(t0 + 2 * KT);
      look(t0 + 3 * KT);

      // scores in powers of two: x fs, where no row has anything to hide or to add
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
        top = -INFINITY;
#pragma unroll
        for (int b = 0; b < SB; ++b) {
          fs[b] = 1.f;
          const float t = top_of(b);
          if (t == -INFINITY) log_v[b] = 0.f;                  // (of a block that the row sees nothing of not even a NaN counts)
          top = sc_max(top, t);
        }
      } else {
#pragma unroll
        for (int b = SB - 4; b < SB; ++b) top = sc_max(top, top_of(b));
      }
      auto of_both = [](float v) {
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return sc_max(__uint_as_float(both[0]), __uint_as_float(both[1]));
      };
      top = of_both(top);
      if (__any(top > m_run + kScLazy || top + most_v > y_run + (kScLazy + kScRaised))) {
        float y_top = -INFINITY;
#pragma unroll
        for (int b = 0; b < SB; ++b) y_top = sc_max(y_top, top_of(b) + log_v[b]);
        const float m_new = fmaxf(m_run, top), y_new = fmaxf(y_run, of_both(y_top) - kScRaised);
        l_run *= __builtin_amdgcn_exp2f(m_run - sc_base(m_new));
        const float shrink = __builtin_amdgcn_exp2f(y_run - sc_base(y_new)), gap = sc_base(y_new) - sc_base(m_new);
        m_run = m_new, y_run = y_new;
        unit = __builtin_amdgcn_exp2f(gap);
        low = fabsf(gap) <= kScApart ? fmaxf(gap - kScDeep, kScNone + 1.f) : INFINITY;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[b][i] *= shrink;
      }
      // Scales far below the row's largest, or all of them far from 1: the weights' sum is the scores', and what is far below is no weight.
      const bool apart = __any(least_v < low);
      float direct = 0.f;
      if (apart) {
        const float m_base = sc_base(m_run), deep = sc_base(y_run) - m_base - kScDeep;
#pragma unroll
        for (int b = 0; b < SB; ++b) {
#pragma unroll
          for (int i = 0; i < 4; ++i) direct += __builtin_amdgcn_exp2f(fmaf(x[b >> 2][(b & 3) * 4 + i], fs[b], -m_base));
          if (log_v[b] < deep) log_v[b] = -INFINITY;
        }
      }
      float undo[SB], sum = 0.f;
#pragma unroll
      for (int b = 0; b < SB; ++b) undo[b] = f[16 + b];
      const float base = sc_base(y_run);
      // Weights of a run of 16 tokens, a few between each two products of the run before.
      const char* vp = v_img + col * VSTRIDE + half * 16;
      constexpr int RN = 2 * NT;
      float p[8], shift = 0.f;
      sc_u32x4 pf;
      auto weigh = [&](auto N_, auto E) {
        constexpr int n = decltype(N_)::value, e = decltype(E)::value, b = 2 * n + e / 4;
        if constexpr (e % 4 == 0) shift = log_v[b] - base;
        p[e] = __builtin_amdgcn_exp2f(fmaf(x[b >> 2][(b & 3) * 4 + e % 4], fs[b], shift));
      };
      auto pack = [&](auto N_) {
        constexpr int n = decltype(N_)::value;
        sum = fmaf((p[0] + p[1]) + (p[2] + p[3]), undo[2 * n], sum);
        sum = fmaf((p[4] + p[5]) + (p[6] + p[7]), undo[2 * n + 1], sum);
#pragma unroll
        for (int w = 0; w < 4; ++w) pf[w] = sc_pack_f16(p[2 * w], p[2 * w + 1]);
      };
      auto operand = [&](int n) { return *reinterpret_cast<const sc_f16x8*>(vp + n % DB * 32 * VSTRIDE + n / DB * 32); };
      constexpr int AHEAD = HEAD > 128 ? 1 : 2;
      sc_f16x8 ring[AHEAD + 1];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) ring[n] = operand(n);
      static_for<8>([&](auto E) { weigh(std::integral_constant<int, 0>{}, E); });
      pack(std::integral_constant<int, 0>{});
      static_for<RN * DB>([&](auto I) {
        constexpr int i = decltype(I)::value, n = i / DB, b = i % DB;
        if constexpr (i + AHEAD < RN * DB) ring[(i + AHEAD) % (AHEAD + 1)] = operand(i + AHEAD);
        o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % (AHEAD + 1)], __builtin_bit_cast(sc_f16x8, pf), o[b], 0, 0, 0);
        if constexpr (n + 1 < RN) {
          static_for<8 * (b + 1) / DB - 8 * b / DB>([&](auto E) {
            weigh(std::integral_constant<int, n + 1>{}, std::integral_constant<int, 8 * b / DB + decltype(E)::value>{});
          });
          if constexpr (b == DB - 1) pack(std::integral_constant<int, n + 1>{});
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      l_run = apart ? l_run + direct : fmaf(sum, unit, l_run);
    }
    __syncthreads();
  }

  l_run += __shfl_xor(l_run, 32, 64);
  if (!real) return;
  // (the two factors one after the other: their product may be below the smallest number)
  const float inv = a.partial ? 1.f : l_run > 0.f ? 1.f / l_run : l_run != l_run ? l_run : 0.f;   // a row that sees nothing gives zeros
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
      const float v0 = o[b][4 * q] * unit * inv, v1 = o[b][4 * q + 1] * unit * inv, v2 = o[b][4 * q + 2] * unit * inv,
                  v3 = o[b][4 * q + 3] * unit * inv;
      if (a.partial) *reinterpret_cast<sc_f32x4*>(to + d) = sc_f32x4{v0, v1, v2, v3};
      else *reinterpret_cast<sc_u32x2*>(out + d) = sc_u32x2{sc_pack16(v0, v1, a.bf16), sc_pack16(v2, v3, a.bf16)};
    }
}

template <bool E4M3, int HEAD, int BS, int WAVES>
int sc_launch_context(const ScAttention& a, int num_seqs, hipStream_t stream) {
  constexpr int lds = 2 * sc_buffer(HEAD);
  static_assert(lds <= 160 * 1024, "two stages must fit a compute unit's LDS");
  auto kernel = scaled_context_kernel<E4M3, HEAD, BS, WAVES>;
  if (lds > 64 * 1024)
    SW_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  kernel<<<dim3(a.kv_heads * a.tiles, num_seqs, a.parts), WAVES * 64, lds, stream>>>(a);
  SW_CHECK_LAUNCH();
  return SW_OK;
}

// (eight waves are for heads of 80 to 128: sc_plan)
template <bool E4M3, int BS, int WAVES>
int sc_context_by_head(const ScAttention& a, int num_seqs, hipStream_t stream) {
  if constexpr (WAVES == 4) {
    if (a.head_size == 64) return sc_launch_context<E4M3, 64, BS, WAVES>(a, num_seqs, stream);
    if (a.head_size == 256) return sc_launch_context<E4M3, 256, BS, WAVES>(a, num_seqs, stream);
  }
  switch (a.head_size) {
    case 80: return sc_launch_context<E4M3, 80, BS, WAVES>(a, num_seqs, stream);
    case 96: return sc_launch_context<E4M3, 96, BS, WAVES>(a, num_seqs, stream);
    case 112: return sc_launch_context<E4M3, 112, BS, WAVES>(a, num_seqs, stream);
    default: return sc_launch_context<E4M3, 128, BS, WAVES>(a, num_seqs, stream);
  }
}

template <bool E4M3, int WAVES>
int sc_context_by_size(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  return block_size == 8    ? sc_context_by_head<E4M3, 8, WAVES>(a, num_seqs, stream)
         : block_size == 16 ? sc_context_by_head<E4M3, 16, WAVES>(a, num_seqs, stream)
                            : sc_context_by_head<E4M3, 32, WAVES>(a, num_seqs, stream);
}

}  // namespace sw
