// Attention of few rows over the 8-bit cache with one scale for each (block, kv head) (included by scaled_decode_*.hip).
//
//     o = sum_t p_t sv_t v_t / sum_t p_t,    p_t = exp(scale * sk_t q.k_t + slope * (t - position) - m)
// over the codes k_t, v_t with the scales sk, sv of their blocks.  Bound by the cache's bytes: one per element, read once for up to 16
// rows (query heads of the kv head, and new tokens), so the products run on the matrix cores however few rows there are, and nothing
// but the codes is fetched for an element.
//
// A wave takes 64 tokens at a time, four runs of 16, and forms
//     S [16 tokens x 16 rows]  = K tile . Q^T             (v_mfma_f32_16x16x32_f16, four tiles)
//     O^T [16 dims x 16 rows] += V^T tile . P^T
// Codes are widened to halves exactly (integers up to 127; e4m3), after the load, in registers: 16 bytes of a lane are 16 dims of a
// key or 16 tokens of a dim's values, as the caches lie.  Both products may take their contraction in any order that their two operands
// share, and S's tokens any place among its rows, so that nothing changes hands between them:
//     K tile j, row r            <->  token 4 j + (r & 3) of run r >> 2
//     Q.K  slot (kq, e) of step 2 m + h  <->  dim 64 m + 16 kq + 8 h + e
//     S tile j of lane (kq, row), i      <->  token 4 j + i of run kq: 16 weights, which are
//     P.V  slot (kq, e) of step h        <->  token 8 h + e of run kq
// Scales are a factor of the score and, as powers of two, a summand of the weight's exponent, both fp32:
//     w_t = 2^(x_t + log2 sv_t - y),   sum_t p_t = sum_t w_t 2^(y - log2 sv_t),     x_t the score in powers of two
// w_t goes to the second product as a half, rounded by at most 2^-11 of it (f16's own step, an eighth of bf16's), where y is kept 14 below
// the largest exponent that the ROW has met: its largest weight is 2^14 whatever blocks without a token for it hold, and what a half cannot
// hold as a normal number is 2^-28 of that.  (A reference of scores and one of scales apart would let a large scale that has no weight take
// the bits of all others.)  bf16 queries go into halves by a power of two for each row that brings their largest to 2^14 .. 2^15, which goes
// into the row's scale.
//
// Measured (heads of 128): 61 sequences of some 1090 tokens, 32 heads, e4m3, 544 MB, 106 us, 5.2 TB/s, what a large copy reads and
// writes (a reading stream reaches 6.2); 201 of some 2000, 64 heads on 8, int8, 820 MB, 170 us, 4.8 TB/s (of one length 5.4: the longest
// sequences' workgroups run on alone); 3 of 34000 to 90000, 64 on 8, e4m3 in ten parts and their join, 431 MB, 84 us, 5.1 TB/s; one sequence of 500
// 8.8 us, a chain of loads.  Two to four tiles of rows a wave, loads a group ahead and pairs of waves that share a group's dims were no faster.
#pragma once

#include "scaled_attention.cuh"

namespace sw {

constexpr float kScUp = 14.f, kScDown = 0x1p-14f;             // powers of two that a row's largest weight stands above 1, and back

// NW waves take the groups of 64 tokens of one (sequence, kv head, tile of 16 rows, part) in turn and join at the end.
// EXACT: head_size == HEAD; else it is a smaller multiple of 16 (dims behind it count as zeros).
template <bool E4M3, int HEAD, bool EXACT, int BS, int NW>
__global__ void __launch_bounds__(NW * 64, HEAD <= 128 ? 2 : 1) scaled_decode_kernel(const ScAttention a) {
  using C = ScCode<E4M3>;
  constexpr int KM = HEAD / 64, DT = HEAD / 16;
  constexpr int PB = BS == 8 ? 2 : 1;                        // blocks of a run of 16 tokens
  extern __shared__ __attribute__((aligned(16))) float smem[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, kq = lane >> 4;
  const int seq = blockIdx.y, part = blockIdx.z;
  // (all tiles of a kv head on one XCD where the number of heads is a multiple of 8)
  const int tile = blockIdx.x / a.kv_heads, kv_head = blockIdx.x - tile * a.kv_heads;
  const ScSequence s = sc_sequence<BS>(a, seq);
  const int rows = s.fresh * a.group;
  if (tile * 16 >= rows) return;
  const int head_size = EXACT ? HEAD : a.head_size;

  // this lane's row: a new token and a query head of the kv head
  const int my = tile * 16 + r;
  const bool real = my < rows;
  const int row_tok = real ? my / a.group : 0, head = kv_head * a.group + (real ? my - row_tok * a.group : 0);
  const int pos = s.first + row_tok;                 // sees tokens up to its own
  // what the tile's rows see, of which this part
  const int last_tok = min(rows - 1, tile * 16 + 15) / a.group;
  const int pos_low = s.first + tile * 16 / a.group, pos_high = s.first + last_tok;
  const int seen_from = sc_seen_from(a, pos_low);            // a multiple of 64, as the parts' borders are
  const int begin = max(part * a.part_tokens, seen_from), end = sc_part_end(a, s, part, pos_high);
  if (a.partial && begin >= end) return;                     // (the join knows)
  // rows that all see a token: from here on the mask is to be looked at
  const int all_see = pos_low + 1, none_hidden = a.window > 0 ? pos_high - a.window + 1 : 0;

  sc_u32x4 qf[KM][2];
  float row_scale = a.scale2;
  {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.query) + (s.row0 + row_tok) * a.q_stride + (int64_t)head * head_size;
    float largest = 0.f;
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int d = 64 * m + 16 * kq + 8 * h;
        qf[m][h] = real && (EXACT || d < head_size) ? *reinterpret_cast<const sc_u32x4*>(q + d) : sc_u32x4{0u, 0u, 0u, 0u};
        if (a.bf16) {
#pragma unroll
          for (int w = 0; w < 4; ++w)
            largest = fmaxf(largest, fmaxf(fabsf(bf16_bits_to_float((uint16_t)(qf[m][h][w] & 0xffffu))),
                                           fabsf(bf16_bits_to_float((uint16_t)(qf[m][h][w] >> 16)))));
        }
      }
    if (a.bf16) {
      largest = fmaxf(largest, __shfl_xor(largest, 16, 64));
      largest = fmaxf(largest, __shfl_xor(largest, 32, 64));
      float up = 1.f;
      if (largest > 0.f && largest < INFINITY) {
        const int e = min(15 - (int)__builtin_amdgcn_frexp_expf(largest), 126);
        up = ldexpf(1.f, e);
        row_scale = ldexpf(row_scale, -e);
      }
#pragma unroll
      for (int m = 0; m < KM; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int w = 0; w < 4; ++w)
            qf[m][h][w] = sc_pack_f16(bf16_bits_to_float((uint16_t)(qf[m][h][w] & 0xffffu)) * up,
                                      bf16_bits_to_float((uint16_t)(qf[m][h][w] >> 16)) * up);
    }
  }
  const float slope = a.slopes ? a.slopes[head] * 1.44269504088896340736f : 0.f;

  const int64_t head_bytes = (int64_t)head_size * BS;
  const int32_t* table = a.tables + (int64_t)seq * a.table_stride;

  float m_run = -INFINITY, l_run = 0.f;                       // the scores' maximum, the sum of 2^(score - it)
  float y_run = -INFINITY;                                    // and what the sums `acc` are powers of two to
  sc_f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = sc_f32x4{0.f, 0.f, 0.f, 0.f};

  const int first_group = begin >> 6, groups = (end + 63) >> 6;
  for (int g = first_group + wave; g < groups; g += NW) {
    const int tok0 = g << 6;
    // blocks of the run whose keys this lane loads (r >> 2) and of the one whose values it loads and scores it gets (kq)
    int kb[PB], vb[PB];
    uint32_t good = 0xffffu;                                  // tokens of run kq that there are
    sc_u32x4 kraw[4][KM], vraw[DT];
    float ks[PB], vs[PB];
    const int last_block = (s.len - 1) / BS;
#pragma unroll
    for (int b = 0; b < PB; ++b) {
      kb[b] = table[min((tok0 + 16 * (r >> 2) + 8 * b) / BS, last_block)];
      vb[b] = table[min((tok0 + 16 * kq + 8 * b) / BS, last_block)];
      if (kb[b] < 0 || kb[b] >= a.num_blocks) kb[b] = 0;
      if (vb[b] < 0 || vb[b] >= a.num_blocks) {
        vb[b] = 0;
        good &= PB == 1 ? 0u : b == 0 ? 0xff00u : 0x00ffu;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = 4 * j + (r & 3);                          // token of the run
      const int b = PB == 2 ? j >> 1 : 0;
      const int off = BS == 8 ? o & 7 : BS == 16 ? o : ((r >> 2) & 1) * 16 + o;
      const uint8_t* p = a.key_cache + ((int64_t)kb[b] * a.kv_heads + kv_head) * head_bytes + off * 16;
#pragma unroll
      for (int m = 0; m < KM; ++m)
        kraw[j][m] = EXACT || 64 * m + 16 * kq < head_size ? *reinterpret_cast<const sc_u32x4*>(p + (4 * m + kq) * (BS * 16))
                                                           : sc_u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int b = 0; b < PB; ++b) {
      ks[b] = a.key_scales[(int64_t)vb[b] * a.kv_heads + kv_head];
      vs[b] = a.value_scales[(int64_t)vb[b] * a.kv_heads + kv_head];
    }
    {
      const uint8_t* p[PB];
#pragma unroll
      for (int b = 0; b < PB; ++b)
        p[b] = a.value_cache + ((int64_t)vb[b] * a.kv_heads + kv_head) * head_bytes + r * BS + (BS == 32 ? (kq & 1) * 16 : 0);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        if (!EXACT && 16 * dt >= head_size) {
          vraw[dt] = sc_u32x4{0u, 0u, 0u, 0u};
        } else if constexpr (PB == 2) {
          vraw[dt] = sc_join(*reinterpret_cast<const sc_u32x2*>(p[0] + 16 * dt * BS), *reinterpret_cast<const sc_u32x2*>(p[1] + 16 * dt * BS));
        } else {
          vraw[dt] = *reinterpret_cast<const sc_u32x4*>(p[0] + 16 * dt * BS);
        }
      }
    }

    // ---- scores: lane (kq, row r), tokens tok0 + 16 kq + 4 j + i
    sc_f32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = sc_f32x4{0.f, 0.f, 0.f, 0.f};
    // (products into one accumulator lie four apart)
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = sc_mfma(sc_join(C::widen(kraw[j][m][2 * h]), C::widen(kraw[j][m][2 * h + 1])), qf[m][h], x[j]);
    const int run0 = tok0 + 16 * kq;
    const int left = end - run0;
    good &= left >= 16 ? 0xffffu : left <= 0 ? 0u : (1u << left) - 1u;
    // (wave-uniform) all 64 tokens are there and every row sees all of them
    const bool masked = tok0 + 64 > all_see || tok0 < none_hidden || __any(good != 0xffffu);
    float top[PB];
#pragma unroll
    for (int b = 0; b < PB; ++b) top[b] = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = PB == 2 ? j >> 1 : 0;
      const float f = row_scale * ks[b];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = run0 + 4 * j + i;
        float v = x[j][i] * f;
        if (a.slopes) v += slope * (float)(t - pos);
        if (masked) {
          const bool see = (good >> (4 * j + i) & 1u) && t <= pos && (a.window <= 0 || t > pos - a.window);
          v = see ? v : -INFINITY;
        }
        x[j][i] = v;
        top[b] = fmaxf(top[b], v);
      }
    }
    float gmax = -INFINITY, ymax = -INFINITY, lv[PB];
#pragma unroll
    for (int b = 0; b < PB; ++b) {
      // (of a block that the row sees nothing of not even a NaN counts)
      lv[b] = top[b] == -INFINITY ? 0.f : sc_log_scale(vs[b]);
      gmax = fmaxf(gmax, top[b]);
      ymax = fmaxf(ymax, top[b] + lv[b]);
    }
    gmax = fmaxf(gmax, __shfl_xor(gmax, 16, 64));
    gmax = fmaxf(gmax, __shfl_xor(gmax, 32, 64));
    ymax = fmaxf(ymax, __shfl_xor(ymax, 16, 64));
    ymax = fmaxf(ymax, __shfl_xor(ymax, 32, 64));
    const float m_new = fmaxf(m_run, gmax), base = sc_base(m_new);
    const float y_new = fmaxf(y_run, ymax - kScUp), y_base = sc_base(y_new), gap = y_base - base;
    const float alpha = __builtin_amdgcn_exp2f(m_run - base), shrink = __builtin_amdgcn_exp2f(y_run - y_base);
    m_run = m_new;
    y_run = y_new;

    // ---- weights: their sum, and as the second product takes them
    sc_u32x4 pf[2];
    float sum = 0.f, shift[PB], undo[PB];
#pragma unroll
    for (int b = 0; b < PB; ++b) {
      const float low = gap - kScDeep;                        // (a weight of that is 0 as a half, and in `sum` it still counts)
      const float l = lv[b] < low ? low : lv[b];
      shift[b] = l - gap;
      undo[b] = __builtin_amdgcn_exp2f(gap - l);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = PB == 2 ? j >> 1 : 0;
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f((x[j][i] - base) + shift[b]);
      sum = fmaf((p[0] + p[1]) + (p[2] + p[3]), undo[b], sum);
      pf[j >> 1][2 * (j & 1)] = sc_pack_f16(p[0], p[1]);
      pf[j >> 1][2 * (j & 1) + 1] = sc_pack_f16(p[2], p[3]);
    }
    l_run = l_run * alpha + sum;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] *= shrink;

    // ---- values.  Slots that hold no token may hold anything, an e4m3 NaN included, and 0 x NaN is NaN: cleared.
    if (E4M3 && masked) {
      sc_u32x4 keep;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t some = good >> (4 * w) & 15u;
        keep[w] = (some & 1u ? 0xffu : 0u) | (some & 2u ? 0xff00u : 0u) | (some & 4u ? 0xff0000u : 0u) | (some & 8u ? 0xff000000u : 0u);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vraw[dt] &= keep;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      acc[dt] = sc_mfma(sc_join(C::widen(vraw[dt][0]), C::widen(vraw[dt][1])), pf[0], acc[dt]);
      acc[dt] = sc_mfma(sc_join(C::widen(vraw[dt][2]), C::widen(vraw[dt][3])), pf[1], acc[dt]);
    }
  }

  // ---- the waves join: a common maximum, then pairs of waves by halves
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  float* stat = smem;                                         // [NW][2][16]
  float* pass = smem + NW * 32;                               // [NW / 2][DT][64 lanes][4]
  if (kq == 0) {
    stat[wave * 32 + r] = m_run;
    stat[wave * 32 + 16 + r] = l_run;
  }
  __syncthreads();
  float m_all = -INFINITY, l_all = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) m_all = fmaxf(m_all, stat[w * 32 + r]);
  const float base = sc_base(m_all);
#pragma unroll
  for (int w = 0; w < NW; ++w) l_all += stat[w * 32 + 16 + r] * __builtin_amdgcn_exp2f(stat[w * 32 + r] - base);
  // (in steps: all in one may be below the smallest number)
  const float mine = __builtin_amdgcn_exp2f(m_run - base) * __builtin_amdgcn_exp2f(y_run + kScUp - sc_base(m_run));
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = acc[dt] * kScDown * mine;
#pragma unroll
  for (int half = NW / 2; half >= 1; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<sc_f32x4*>(pass + (((wave - half) * DT + dt) * 64 + lane) * 4) = acc[dt];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] += *reinterpret_cast<const sc_f32x4*>(pass + ((wave * DT + dt) * 64 + lane) * 4);
    }
    __syncthreads();
  }
  if (wave != 0 || !real) return;
  if (a.partial) {
    float* to = a.partial + (((s.row0 + row_tok) * a.heads + head) * a.parts + part) * (head_size + 4);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      if (EXACT || 16 * dt < head_size) *reinterpret_cast<sc_f32x4*>(to + 16 * dt + 4 * kq) = acc[dt];
    if (kq == 0) {
      to[head_size] = m_all;
      to[head_size + 1] = l_all;
    }
    return;
  }
  const float inv = l_all > 0.f ? 1.f / l_all : l_all != l_all ? l_all : 0.f;   // a row that sees nothing gives zeros
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (s.row0 + row_tok) * a.out_stride + (int64_t)head * head_size;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    if (EXACT || 16 * dt < head_size)
      *reinterpret_cast<sc_u32x2*>(out + 16 * dt + 4 * kq) =
          sc_u32x2{sc_pack16(acc[dt][0] * inv, acc[dt][1] * inv, a.bf16), sc_pack16(acc[dt][2] * inv, acc[dt][3] * inv, a.bf16)};
}

template <bool E4M3, int HEAD, bool EXACT, int BS, int NW>
int sc_launch_decode(const ScAttention& a, int num_seqs, hipStream_t stream) {
  constexpr int lds = (NW * 32 + (NW / 2) * (HEAD / 16) * 256) * 4;
  static_assert(lds <= 64 * 1024, "the waves' sums must fit a launch's plain LDS");
  scaled_decode_kernel<E4M3, HEAD, EXACT, BS, NW><<<dim3(a.kv_heads * a.tiles, num_seqs, a.parts), NW * 64, lds, stream>>>(a);
  SW_CHECK_LAUNCH();
  return SW_OK;
}

template <bool E4M3, int NW>
int sc_decode_by_size(const ScAttention& a, int block_size, int num_seqs, hipStream_t stream) {
  auto by_block = [&](auto head, auto exact, auto waves) {
    constexpr int H = decltype(head)::value, W = decltype(waves)::value;
    constexpr bool X = decltype(exact)::value;
    return block_size == 8    ? sc_launch_decode<E4M3, H, X, 8, W>(a, num_seqs, stream)
           : block_size == 16 ? sc_launch_decode<E4M3, H, X, 16, W>(a, num_seqs, stream)
                              : sc_launch_decode<E4M3, H, X, 32, W>(a, num_seqs, stream);
  };
  const std::integral_constant<int, NW> waves{};
  switch (a.head_size) {
    case 64: return by_block(std::integral_constant<int, 64>{}, std::true_type{}, waves);
    case 128: return by_block(std::integral_constant<int, 128>{}, std::true_type{}, waves);
    // (eight waves of such heads would have half the registers that they need)
    case 256: return by_block(std::integral_constant<int, 256>{}, std::true_type{}, std::integral_constant<int, 4>{});
    default: return by_block(std::integral_constant<int, 128>{}, std::false_type{}, waves);
  }
}

}  // namespace sw
