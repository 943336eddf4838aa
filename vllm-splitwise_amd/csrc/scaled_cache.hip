// Writing and reading back the 8-bit cache with one scale for each (block, kv head).
//
// Write: for the tokens of a call that go to block b, head h
//     a = max |x| over finite x,   s' = a / top (0 where a < 2^-100),   s = max(s_old, s'),   code = round(x / s), clipped to +-top
// where s_old is 0 if one of them goes to the block's first slot (the block then starts over, whatever it held) and the block's
// scale otherwise; codes that were there become round(code * s_old / s).  x / s is taken as x * (1 / s): the quotient of two
// roundings, so that a value next to the middle of two codes may go to the other one.
//
// One workgroup does all tokens of a block for two heads, a wave each for K and V of a head, because the scale is one for all of
// them and what was there has to be read, rescaled and written by the same hands.  The slots' list has no order that one could rely
// on.  A workgroup looks at `window` entries of it; those whose predecessor is in another block are heads of runs.  A run that
// covers its whole block in order needs no look at the rest of the list; for any other one the workgroup goes through the whole list,
// leaves if an earlier entry has the same block, and otherwise gathers the entries of that block, wherever they stand.
#include "scaled_cache.cuh"

#include <algorithm>

namespace sw {

namespace {

struct ScWrite {
  const void* x[2];            // keys, values [tokens, heads, head_size]
  uint8_t* cache[2];
  float* scales[2];
  const int64_t* slots;
  int64_t stride[2];           // elements from token to token
  int64_t num_slots;           // blocks * block size
  int num_tokens, heads, head_size, window;
};

struct ScRead {
  void* x[2];
  const uint8_t* cache[2];
  const float* scales[2];
  const int32_t *tables, *starts, *lens;
  int64_t stride[2], num_rows, table_stride;
  int num_blocks, width, heads, head_size;
};

template <typename act_t> struct ScAct {
  using S = typename Conv<act_t>::store_t;
  static constexpr int kWords = sizeof(S) * 16 / 4;            // dwords of 16 elements
  // element `i` of the dwords at w
  __device__ static __forceinline__ float get(const uint32_t* w, int i) {
    if constexpr (sizeof(S) == 4) return __uint_as_float(w[i]);
    else return Conv<act_t>::to_float((S)(w[i >> 1] >> (16 * (i & 1))));
  }
  __device__ static __forceinline__ uint32_t pair(float a, float b) {
    static_assert(sizeof(S) == 2 || sizeof(S) == 4, "");
    return (uint32_t)Conv<act_t>::from_float(a) | ((uint32_t)Conv<act_t>::from_float(b) << 16);
  }
};

__device__ __forceinline__ float sc_magnitude(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;                               // neither infinities nor NaN count
}

struct ScScale { float now, inverse, ratio; };

template <bool E4M3>
__device__ __forceinline__ ScScale sc_scale(float largest, float old) {
  ScScale s;
  s.now = fmaxf(old, largest < kScTiny ? 0.f : largest * ScCode<E4M3>::kUnit);
  s.inverse = s.now > 0.f ? 1.f / s.now : 0.f;
  s.ratio = s.now > 0.f ? old / s.now : 0.f;
  return s;
}

template <bool E4M3>
__device__ __forceinline__ uint32_t sc_rescale(uint32_t w, float ratio) {
  float o[4];
  ScCode<E4M3>::decode(w, o);
  return ScCode<E4M3>::encode(o[0] * ratio, o[1] * ratio, o[2] * ratio, o[3] * ratio);
}

// token of the call that goes to offset o of the block, -1: none
struct ScTokens {
  const int* map;              // LDS, or null: first + o
  int first;
  __device__ __forceinline__ int operator()(int o) const { return map ? map[o] : first + o; }
};

// A lane's pieces are 16 elements of one token's key: 32 bytes in, one 16-byte store.
template <typename act_t, bool E4M3, int BS, int DMAX>
__device__ __forceinline__ void sc_write_keys(const ScWrite& w, int64_t block, int head, const ScTokens& token, int lane) {
  using A = ScAct<act_t>;
  constexpr int NU = (BS * DMAX / 16 + 63) / 64;
  const int chunks = w.head_size >> 4, units = BS * chunks;
  const int64_t bh = block * w.heads + head;
  uint8_t* out = w.cache[0] + bh * w.head_size * BS;
  const float stored = w.scales[0][bh];
  uint32_t x[NU][A::kWords];
  int tok[NU], at[NU];
  float largest = 0.f;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = lane + 64 * i, t = u / chunks, c = u - t * chunks;
    tok[i] = u < units ? token(t) : -1;
    at[i] = u < units ? (c * BS + t) * 16 : -1;
    if (tok[i] >= 0) {
      const sc_u32x4* p = reinterpret_cast<const sc_u32x4*>(reinterpret_cast<const typename A::S*>(w.x[0]) + tok[i] * w.stride[0] +
                                                            (int64_t)head * w.head_size + 16 * c);
#pragma unroll
      for (int k = 0; k < A::kWords / 4; ++k) *reinterpret_cast<sc_u32x4*>(&x[i][4 * k]) = p[k];
#pragma unroll
      for (int e = 0; e < 16; ++e) largest = fmaxf(largest, sc_magnitude(A::get(x[i], e)));
    }
  }
  const bool fresh = token(0) >= 0;
  const ScScale s = sc_scale<E4M3>(wave_max(largest), fresh ? 0.f : sc_old_scale(stored));
  if (lane == 0) w.scales[0][bh] = s.now;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if (at[i] < 0) continue;
    sc_u32x4* p = reinterpret_cast<sc_u32x4*>(out + at[i]);
    if (tok[i] >= 0) {
      sc_u32x4 q;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        q[k] = ScCode<E4M3>::encode(A::get(x[i], 4 * k) * s.inverse, A::get(x[i], 4 * k + 1) * s.inverse,
                                    A::get(x[i], 4 * k + 2) * s.inverse, A::get(x[i], 4 * k + 3) * s.inverse);
      *p = q;
    } else if (fresh) {
      *p = sc_u32x4{0u, 0u, 0u, 0u};
    } else if (s.ratio != 1.f) {
      sc_u32x4 q = *p;
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = sc_rescale<E4M3>(q[k], s.ratio);
      *p = q;
    }
  }
}

// A lane's pieces are two elements of every token's value: 4 bytes a token in (a wave's load is a whole row of 128), two rows of the
// block's tokens out, 2 * BS bytes side by side.
template <typename act_t, bool E4M3, int BS, int DMAX>
__device__ __forceinline__ void sc_write_values(const ScWrite& w, int64_t block, int head, const ScTokens& token, int lane) {
  using A = ScAct<act_t>;
  constexpr int NP = DMAX / 128, W2 = sizeof(typename A::S) / 2;      // W2: dwords of two elements
  const int pairs = w.head_size >> 1;
  const int64_t bh = block * w.heads + head;
  uint8_t* out = w.cache[1] + bh * w.head_size * BS;
  const float stored = w.scales[1][bh];
  uint32_t x[NP][BS][W2];
  float largest = 0.f;
  uint32_t there = 0;                                                   // bit o: a token goes to offset o
#pragma unroll
  for (int o = 0; o < BS; ++o) there |= (token(o) >= 0 ? 1u : 0u) << o;
  there = __builtin_amdgcn_readfirstlane(there);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int p = lane + 64 * i;
#pragma unroll
    for (int o = 0; o < BS; ++o) {
#pragma unroll
      for (int k = 0; k < W2; ++k) x[i][o][k] = 0;
      if ((there >> o & 1u) && p < pairs) {
        const typename A::S* src = reinterpret_cast<const typename A::S*>(w.x[1]) + token(o) * w.stride[1] +
                                   (int64_t)head * w.head_size + 2 * p;
        if constexpr (W2 == 1) x[i][o][0] = *reinterpret_cast<const uint32_t*>(src);
        else *reinterpret_cast<sc_u32x2*>(x[i][o]) = *reinterpret_cast<const sc_u32x2*>(src);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int o = 0; o < BS; ++o)
      largest = fmaxf(largest, fmaxf(sc_magnitude(A::get(x[i][o], 0)), sc_magnitude(A::get(x[i][o], 1))));
  const bool fresh = there & 1u;
  const ScScale s = sc_scale<E4M3>(wave_max(largest), fresh ? 0.f : sc_old_scale(stored));
  if (lane == 0) w.scales[1][bh] = s.now;
  const bool merge = !fresh && there != (BS == 32 ? 0xffffffffu : (1u << (BS & 31)) - 1u);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int p = lane + 64 * i;
    if (p >= pairs) continue;
    uint32_t* row = reinterpret_cast<uint32_t*>(out + (int64_t)2 * p * BS);
    uint32_t q[2][BS / 4];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int k = 0; k < BS / 4; ++k) {
        const uint32_t some = there >> (4 * k) & 15u;
        uint32_t was = 0;
        if (merge && some != 15u) {
          was = row[e * (BS / 4) + k];
          if (s.ratio != 1.f) was = sc_rescale<E4M3>(was, s.ratio);
        }
        const uint32_t now = ScCode<E4M3>::encode(A::get(x[i][4 * k], e) * s.inverse, A::get(x[i][4 * k + 1], e) * s.inverse,
                                                  A::get(x[i][4 * k + 2], e) * s.inverse, A::get(x[i][4 * k + 3], e) * s.inverse);
        const uint32_t mask = (some & 1u ? 0xffu : 0u) | (some & 2u ? 0xff00u : 0u) | (some & 4u ? 0xff0000u : 0u) |
                              (some & 8u ? 0xff000000u : 0u);
        q[e][k] = (now & mask) | (was & ~mask);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if constexpr (BS >= 16) {
#pragma unroll
        for (int k = 0; k < BS / 16; ++k)
          reinterpret_cast<sc_u32x4*>(row)[e * (BS / 16) + k] = *reinterpret_cast<const sc_u32x4*>(&q[e][4 * k]);
      } else {
        reinterpret_cast<sc_u32x2*>(row)[e] = sc_u32x2{q[e][0], q[e][1]};
      }
    }
  }
}

template <typename act_t, bool E4M3, int BS, int DMAX>
__global__ void __launch_bounds__(256) scaled_write_kernel(const ScWrite w) {
  __shared__ int map[BS], earlier;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.y * 2 + (wave >> 1);
  const int t0 = blockIdx.x * w.window;
  auto block_of = [&](int64_t slot) -> int64_t { return slot >= 0 && slot < w.num_slots ? slot / BS : -1; };
  auto slot_of = [&](int t) -> int64_t { return t < w.num_tokens ? w.slots[t] : -1; };

  // heads of runs among this workgroup's entries (every wave finds the same ones)
  uint64_t heads;
  {
    const int t = t0 + lane;
    const int64_t mine = lane < w.window ? block_of(slot_of(t)) : -1;
    const int64_t before = lane < w.window && t > 0 ? block_of(slot_of(t - 1)) : -1;
    heads = __ballot(mine >= 0 && mine != before);
  }
  while (heads) {
    const int t = t0 + __builtin_ctzll(heads);
    heads &= heads - 1;
    const int64_t first = w.slots[t], block = first / BS;
    // the whole block in order, and nothing of it right behind
    const int64_t next = lane <= BS ? slot_of(t + lane) : -1;
    const bool as_run = lane < BS ? next == first + lane : lane > BS || block_of(next) != block;
    ScTokens token{nullptr, t};
    if (first % BS != 0 || __ballot(as_run) != ~0ull) {
      __syncthreads();                                          // the last run's map has been read
      if (threadIdx.x < BS) map[threadIdx.x] = -1;
      if (threadIdx.x == BS) earlier = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < w.num_tokens; i += 256) {
        const int64_t s = w.slots[i];
        if (block_of(s) != block) continue;
        if (i < t) earlier = 1;
        else atomicMax(&map[s % BS], i);                        // of two tokens for one slot the later one
      }
      __syncthreads();
      if (earlier) continue;                                    // that entry's workgroup does the block
      token.map = map;
    }
    if (head < w.heads) {
      if (wave & 1) sc_write_values<act_t, E4M3, BS, DMAX>(w, block, head, token, lane);
      else sc_write_keys<act_t, E4M3, BS, DMAX>(w, block, head, token, lane);
    }
  }
}

// One wave: K or V of one (block, head) of one sequence.
template <typename act_t, bool E4M3, int BS, int DMAX>
__global__ void __launch_bounds__(256) scaled_read_kernel(const ScRead w) {
  using A = ScAct<act_t>;
  using S = typename A::S;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.y * 2 + (wave >> 1), seq = blockIdx.z;
  const int64_t first = w.starts[seq];
  const int64_t len = min((int64_t)w.lens[seq], (int64_t)w.width * BS);
  const int at0 = blockIdx.x * BS;
  if (head >= w.heads || at0 >= len || first < 0) return;
  // rows behind the end of the output are not written
  const int count = (int)min((int64_t)min((int64_t)BS, len - at0), w.num_rows - first - at0);
  const int block = w.tables[(int64_t)seq * w.table_stride + blockIdx.x];
  const bool good = block >= 0 && block < w.num_blocks;        // tokens of blocks that do not exist are zeros
  const int64_t bh = (int64_t)(good ? block : 0) * w.heads + head;
  const int kv = wave & 1;
  const float scale = good ? w.scales[kv][bh] : 0.f;
  const uint8_t* in = w.cache[kv] + bh * w.head_size * BS;
  S* out = reinterpret_cast<S*>(w.x[kv]) + (first + at0) * w.stride[kv] + (int64_t)head * w.head_size;
  if (kv == 0) {
    constexpr int NU = (BS * DMAX / 16 + 63) / 64;
    const int chunks = w.head_size >> 4;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = lane + 64 * i, t = u / chunks, c = u - t * chunks;
      if (t >= count) continue;
      const sc_u32x4 q = good ? *reinterpret_cast<const sc_u32x4*>(in + (c * BS + t) * 16) : sc_u32x4{0u, 0u, 0u, 0u};
      float o[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) ScCode<E4M3>::decode(q[k], o + 4 * k);
      sc_u32x4* p = reinterpret_cast<sc_u32x4*>(out + t * w.stride[0] + 16 * c);
#pragma unroll
      for (int k = 0; k < A::kWords / 4; ++k) {
        sc_u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(S) == 2) v[e] = A::pair(o[8 * k + 2 * e] * scale, o[8 * k + 2 * e + 1] * scale);
          else v[e] = __float_as_uint(o[4 * k + e] * scale);
        }
        p[k] = v;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < DMAX / 128; ++i) {
      const int p = lane + 64 * i;
      if (p >= w.head_size >> 1) continue;
      const uint32_t* row = reinterpret_cast<const uint32_t*>(in + (int64_t)2 * p * BS);
      uint32_t q[2][BS / 4];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < BS / 4; ++k) q[e][k] = good ? row[e * (BS / 4) + k] : 0u;
#pragma unroll
      for (int k = 0; k < BS / 4; ++k) {
        float a[4], b[4];
        ScCode<E4M3>::decode(q[0][k], a);
        ScCode<E4M3>::decode(q[1][k], b);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (4 * k + e >= count) continue;
          S* to = out + (4 * k + e) * w.stride[1] + 2 * p;
          if constexpr (sizeof(S) == 2) *reinterpret_cast<uint32_t*>(to) = A::pair(a[e] * scale, b[e] * scale);
          else *reinterpret_cast<sc_u32x2*>(to) = sc_u32x2{__float_as_uint(a[e] * scale), __float_as_uint(b[e] * scale)};
        }
      }
    }
  }
}

template <typename F>
int sc_by_size(int head_size, int block_size, F&& f) {
  const bool wide = head_size > 128;
  switch (block_size) {
    case 8: return wide ? f(std::integral_constant<int, 8>{}, std::integral_constant<int, 256>{})
                        : f(std::integral_constant<int, 8>{}, std::integral_constant<int, 128>{});
    case 16: return wide ? f(std::integral_constant<int, 16>{}, std::integral_constant<int, 256>{})
                         : f(std::integral_constant<int, 16>{}, std::integral_constant<int, 128>{});
    default: return wide ? f(std::integral_constant<int, 32>{}, std::integral_constant<int, 256>{})
                         : f(std::integral_constant<int, 32>{}, std::integral_constant<int, 128>{});
  }
}

template <typename F>
int sc_by_type(int act, int cache, F&& f) {
  const bool e = cache == SW_E4M3_SCALED;
  switch (act) {
    case SW_F32: return e ? f(float{}, std::true_type{}) : f(float{}, std::false_type{});
    case SW_F16: return e ? f(f16_t{}, std::true_type{}) : f(f16_t{}, std::false_type{});
    default: return e ? f(bf16_t{}, std::true_type{}) : f(bf16_t{}, std::false_type{});
  }
}

int sc_check(const char* what, int heads, int head_size, int block_size, int64_t num_blocks, int act, int cache) {
  SW_CHECK_ARG(cache == SW_I8_SCALED || cache == SW_E4M3_SCALED, "%s: the cache type must be scaled int8 or e4m3", what);
  SW_CHECK_ARG(act == SW_F32 || act == SW_F16 || act == SW_BF16, "%s: unsupported activation type %d", what, act);
  SW_CHECK_ARG(sc_head_size(head_size), "%s: Unsupported head size: %d", what, head_size);
  SW_CHECK_ARG(block_size == 8 || block_size == 16 || block_size == 32, "%s: Unsupported block size: %d", what, block_size);
  SW_CHECK_ARG(heads > 0 && heads <= 65535 * 2, "%s: %d heads", what, heads);
  SW_CHECK_ARG(num_blocks > 0 && num_blocks <= INT32_MAX, "%s: %lld blocks", what, (long long)num_blocks);
  return SW_OK;
}

bool sc_aligned(const void* p, int64_t stride, int size) { return (uintptr_t)p % 16 == 0 && stride * size % 16 == 0; }

}  // namespace

}  // namespace sw

extern "C" {

int sw_reshape_and_cache_scaled(const void* key, const void* value, void* key_cache, void* value_cache, float* key_scales,
                                float* value_scales, const int64_t* slot_mapping, int num_tokens, int num_heads, int head_size,
                                int block_size, int64_t num_blocks, int64_t key_stride, int64_t value_stride, int act_dtype,
                                int cache_dtype, void* stream) {
  using namespace sw;
  const int bad = sc_check("reshape_and_cache_scaled", num_heads, head_size, block_size, num_blocks, act_dtype, cache_dtype);
  if (bad) return bad;
  SW_CHECK_ARG(num_tokens >= 0, "reshape_and_cache_scaled: %d tokens", num_tokens);
  const int es = dtype_size(act_dtype);
  SW_CHECK_ARG(sc_aligned(key, key_stride, es) && sc_aligned(value, value_stride, es) && (uintptr_t)key_cache % 16 == 0 &&
                   (uintptr_t)value_cache % 16 == 0,
               "reshape_and_cache_scaled: rows of keys and values, and the caches, must begin on multiples of 16 bytes");
  if (num_tokens == 0) return SW_OK;
  ScWrite w;
  w.x[0] = key, w.x[1] = value;
  w.cache[0] = (uint8_t*)key_cache, w.cache[1] = (uint8_t*)value_cache;
  w.scales[0] = key_scales, w.scales[1] = value_scales;
  w.slots = slot_mapping;
  w.stride[0] = key_stride, w.stride[1] = value_stride;
  w.num_slots = num_blocks * block_size;
  w.num_tokens = num_tokens, w.heads = num_heads, w.head_size = head_size;
  // a decode step's entries each begin a run, a prompt's only every block_size-th
  w.window = num_tokens <= 1024 ? 1 : block_size;
  const dim3 grid((num_tokens + w.window - 1) / w.window, (num_heads + 1) / 2);
  return sc_by_type(act_dtype, cache_dtype, [&](auto a, auto e) {
    return sc_by_size(head_size, block_size, [&](auto bs, auto d) -> int {
      scaled_write_kernel<decltype(a), decltype(e)::value, decltype(bs)::value, decltype(d)::value>
          <<<grid, 256, 0, (hipStream_t)stream>>>(w);
      SW_CHECK_LAUNCH();
      return SW_OK;
    });
  });
}

int sw_gather_cache_scaled(void* key, void* value, const void* key_cache, const void* value_cache, const float* key_scales,
                           const float* value_scales, const int32_t* block_tables, const int32_t* seq_starts,
                           const int32_t* seq_lens, int num_seqs, int max_seq_len, int64_t num_rows, int num_heads, int head_size,
                           int block_size, int64_t num_blocks, int max_blocks_per_seq, int64_t table_stride, int64_t key_stride,
                           int64_t value_stride, int act_dtype, int cache_dtype, void* stream) {
  using namespace sw;
  const int bad = sc_check("gather_cache_scaled", num_heads, head_size, block_size, num_blocks, act_dtype, cache_dtype);
  if (bad) return bad;
  SW_CHECK_ARG(num_seqs >= 0 && num_seqs <= 65535, "gather_cache_scaled: %d sequences, at most 65535 in a call", num_seqs);
  SW_CHECK_ARG(max_seq_len >= 0 && max_blocks_per_seq >= 0, "gather_cache_scaled: negative sizes");
  const int es = dtype_size(act_dtype);
  SW_CHECK_ARG(sc_aligned(key, key_stride, es) && sc_aligned(value, value_stride, es) && (uintptr_t)key_cache % 16 == 0 &&
                   (uintptr_t)value_cache % 16 == 0,
               "gather_cache_scaled: rows of keys and values, and the caches, must begin on multiples of 16 bytes");
  ScRead w;
  w.x[0] = key, w.x[1] = value;
  w.cache[0] = (const uint8_t*)key_cache, w.cache[1] = (const uint8_t*)value_cache;
  w.scales[0] = key_scales, w.scales[1] = value_scales;
  w.tables = block_tables, w.starts = seq_starts, w.lens = seq_lens;
  w.stride[0] = key_stride, w.stride[1] = value_stride;
  w.num_rows = num_rows, w.table_stride = table_stride;
  w.num_blocks = (int)num_blocks, w.width = max_blocks_per_seq, w.heads = num_heads, w.head_size = head_size;
  const int blocks = std::min((int)(((int64_t)max_seq_len + block_size - 1) / block_size), max_blocks_per_seq);
  if (num_seqs == 0 || blocks == 0 || num_rows == 0) return SW_OK;
  const dim3 grid(blocks, (num_heads + 1) / 2, num_seqs);
  return sc_by_type(act_dtype, cache_dtype, [&](auto a, auto e) {
    return sc_by_size(head_size, block_size, [&](auto bs, auto d) -> int {
      scaled_read_kernel<decltype(a), decltype(e)::value, decltype(bs)::value, decltype(d)::value>
          <<<grid, 256, 0, (hipStream_t)stream>>>(w);
      SW_CHECK_LAUNCH();
      return SW_OK;
    });
  });
}

}  // extern "C"
