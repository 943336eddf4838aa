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
// on, and may name blocks and slots more than once.  A workgroup looks at `window` entries of it; those whose predecessor is in another
// block are heads of runs.  For a run's head the workgroup goes through the whole list, leaves if an earlier entry has the same block, and
// otherwise gathers the entries of that block, wherever they stand.  In a long list that costs more than the blocks, and is for nothing
// where each block has one run, as in a list of whole sequences: so where there is a workspace, two small launches find that out first.
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
  const int* repeated;         // 0: no block has two runs, and no run more entries than its block slots; null: not known
  int num_tokens, heads, head_size, window, head_pairs;
};

struct ScRead {
  void* x[2];
  const uint8_t* cache[2];
  const float* scales[2];
  const int32_t *tables, *starts, *lens;
  int64_t stride[2], num_rows, table_stride;
  int num_blocks, width, heads, head_size, head_pairs;
};

template <typename act_t> struct ScAct {
  using S = typename Conv<act_t>::store_t;
  static constexpr int kWords = sizeof(S) * 16 / 4;            // dwords of 16 elements
  static constexpr uint32_t kInf = std::is_same<act_t, f16_t>::value ? 0x7c00u : std::is_same<act_t, bf16_t>::value ? 0x7f80u : 0x7f800000u;
  // element `i` of the dwords at w
  __device__ static __forceinline__ float get(const uint32_t* w, int i) {
    if constexpr (sizeof(S) == 4) return __uint_as_float(w[i]);
    else return Conv<act_t>::to_float((S)(w[i >> 1] >> (16 * (i & 1))));
  }
  __device__ static __forceinline__ uint32_t pair(float a, float b) {
    static_assert(sizeof(S) == 2 || sizeof(S) == 4, "");
    using f32x2 = __attribute__((ext_vector_type(2))) float;
    using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
    if constexpr (std::is_same<act_t, f16_t>::value) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), sc_f16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
  }
  // Magnitudes are compared as the integers that their bits are (16-bit ones two at a time): infinities and NaN are the largest.
  using u16x2 = __attribute__((ext_vector_type(2))) uint16_t;
  __device__ static __forceinline__ void larger(uint32_t& most, uint32_t w) {
    if constexpr (sizeof(S) == 4) most = max(most, w & 0x7fffffffu);
    else most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
  }
  // a wave's largest magnitude, as its bits
  __device__ static __forceinline__ uint32_t largest(uint32_t most) {
    if constexpr (sizeof(S) == 2) most = max(most & 0xffffu, most >> 16);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m, 64));
    return __builtin_amdgcn_readfirstlane(most);
  }
  __device__ static __forceinline__ float value(uint32_t bits) { return get(&bits, 0); }
};

__device__ __forceinline__ float sc_magnitude(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;                               // neither infinities nor NaN count
}

// Of four lanes 16 apart, r[k] of lane q becomes r[q] of lane k: two swaps of halves, two of 16 lanes.
__device__ __forceinline__ void sc_transpose(uint32_t (&r)[4]) {
  auto swap32 = [](uint32_t& a, uint32_t& b) {
    const auto t = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = t[0], b = t[1];
  };
  auto swap16 = [](uint32_t& a, uint32_t& b) {
    const auto t = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = t[0], b = t[1];
  };
  swap32(r[0], r[2]);
  swap32(r[1], r[3]);
  swap16(r[0], r[1]);
  swap16(r[2], r[3]);
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

constexpr int kScWindow = 16;        // entries of a workgroup; they, one before them and a block behind them are a wave's lanes
constexpr int kScLook = 16;          // entries that a thread asks for at a time as it goes through the list
// Entries of a list that is gone through for each of its runs.  (us, gone through / looked at first, in two launches: 2444 tokens of 32 heads
// 17.7 / 17.6, 3840 of 8 heads 11.6 / 11.7, 14293 44.5 / 22.4, 60000 443 / 78.)
constexpr int kScShort = 1024;

// Bound by vector instructions as much as by memory (an element is 2 bytes in and 1 out), so: a lane's addresses are one number and what
// the compiler can put into the instructions; magnitudes two at a time; codes of finite values, the rule, in 4 instructions an element; and
// blocks that the call fills look at no single token.  5 prompts of some 400 tokens, 32 heads of 128, f16 to e4m3 17.6 us, 16384 tokens of 8 heads
// in whole blocks 23 us, 4.4 TB/s, of which the look at the list is 3.5; 64 single tokens of 32 heads 6.5 us, of which the kernel's own chain of
// loads (list, list, token) is most.  (Asking for a short list and for what a block holds earlier made the chain shorter and the rest slower:
// 0.1 us more there, 1 us more for prompts.  The look at a long list in one launch of one workgroup: 16 us more for 16384 entries; at every
// block_size-th entry by each workgroup of a run that fills its block, the other runs in a launch of their own: 11 us more.)

// A lane's pieces are 16 elements of the key of one token, the same for all its pieces: 32 bytes in (64 of fp32), 16 out, where a wave's lie
// side by side.  FULL: tokens first, first + 1, ... fill the block.
template <typename act_t, bool E4M3, int BS, int DMAX, bool FULL>
__device__ __forceinline__ void sc_write_keys(const ScWrite& w, int64_t block, int head, const int* map, int first, int lane) {
  using A = ScAct<act_t>;
  constexpr int NU = (BS * DMAX / 16 + 63) / 64, STEP = 64 / BS;
  const int chunks = w.head_size >> 4, t = lane % BS, c0 = lane / BS;
  const int64_t bh = block * w.heads + head;
  uint8_t* out = w.cache[0] + bh * w.head_size * BS + lane * 16;
  const float stored = w.scales[0][bh];
  const int tok = FULL ? first + t : map[t];
  const typename A::S* in = reinterpret_cast<const typename A::S*>(w.x[0]) + tok * w.stride[0] + (int64_t)head * w.head_size + 16 * c0;
  uint32_t x[NU][A::kWords], most = 0;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
#pragma unroll
    for (int k = 0; k < A::kWords; ++k) x[i][k] = 0;
    if (c0 + i * STEP < chunks && (FULL || tok >= 0)) {
#pragma unroll
      for (int k = 0; k < A::kWords / 4; ++k)
        *reinterpret_cast<sc_u32x4*>(&x[i][4 * k]) = reinterpret_cast<const sc_u32x4*>(in + 16 * STEP * i)[k];
    }
  }
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int k = 0; k < A::kWords; ++k) A::larger(most, x[i][k]);
  most = A::largest(most);
  const bool finite = most < A::kInf;
  float largest = A::value(most);
  if (!finite) {
    largest = 0.f;
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) largest = fmaxf(largest, sc_magnitude(A::get(x[i], e)));
    largest = wave_max(largest);
  }
  const bool fresh = FULL || map[0] >= 0;
  const ScScale s = sc_scale<E4M3>(largest, fresh ? 0.f : sc_old_scale(stored));
  if (lane == 0) w.scales[0][bh] = s.now;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if (c0 + i * STEP >= chunks) continue;
    sc_u32x4* p = reinterpret_cast<sc_u32x4*>(out + i * 64 * 16);
    sc_u32x4 q;
    if (finite) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        q[k] = ScCode<E4M3>::encode_fitting(A::get(x[i], 4 * k), A::get(x[i], 4 * k + 1), A::get(x[i], 4 * k + 2), A::get(x[i], 4 * k + 3),
                                            s.inverse);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        q[k] = ScCode<E4M3>::encode(A::get(x[i], 4 * k) * s.inverse, A::get(x[i], 4 * k + 1) * s.inverse,
                                    A::get(x[i], 4 * k + 2) * s.inverse, A::get(x[i], 4 * k + 3) * s.inverse);
    }
    if (FULL || tok >= 0 || fresh) {                           // (slots without a token are zeros: x is)
      *p = q;
    } else if (s.ratio != 1.f) {
      q = *p;
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = sc_rescale<E4M3>(q[k], s.ratio);
      *p = q;
    }
  }
}

// A lane's pieces are two elements of every token's value: 4 bytes a token in (a wave's load is a whole row of 128, where the token's row
// begins is a scalar), two rows of the block's tokens out, 2 * BS bytes side by side.
template <typename act_t, bool E4M3, int BS, int DMAX, bool FULL>
__device__ __forceinline__ void sc_write_values(const ScWrite& w, int64_t block, int head, const int* map, int first, int lane) {
  using A = ScAct<act_t>;
  using S = typename A::S;
  constexpr int NP = DMAX / 128, W2 = sizeof(S) / 2;                   // W2: dwords of two elements
  const int pairs = w.head_size >> 1;
  const int64_t bh = block * w.heads + head;
  uint8_t* out = w.cache[1] + bh * w.head_size * BS;
  const float stored = w.scales[1][bh];
  const S* in = reinterpret_cast<const S*>(w.x[1]) + (int64_t)head * w.head_size;
  uint32_t x[NP][BS][W2], most = 0;
  uint32_t there = 0;                                                   // bit o: a token goes to offset o
#pragma unroll
  for (int o = 0; o < BS; ++o) {
    const int tok = FULL ? first + o : __builtin_amdgcn_readfirstlane(map[o]);
    there |= (FULL || tok >= 0 ? 1u : 0u) << o;
    const char* row = reinterpret_cast<const char*>(in + tok * w.stride[1]);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t p = lane + 64 * i;
#pragma unroll
      for (int k = 0; k < W2; ++k) x[i][o][k] = 0;
      if ((FULL || tok >= 0) && (int)p < pairs) {
        if constexpr (W2 == 1) x[i][o][0] = *reinterpret_cast<const uint32_t*>(row + p * 4);
        else *reinterpret_cast<sc_u32x2*>(x[i][o]) = *reinterpret_cast<const sc_u32x2*>(row + p * 8);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int o = 0; o < BS; ++o)
#pragma unroll
      for (int k = 0; k < W2; ++k) A::larger(most, x[i][o][k]);
  most = A::largest(most);
  const bool finite = most < A::kInf;
  float largest = A::value(most);
  if (!finite) {
    largest = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int o = 0; o < BS; ++o)
        largest = fmaxf(largest, fmaxf(sc_magnitude(A::get(x[i][o], 0)), sc_magnitude(A::get(x[i][o], 1))));
    largest = wave_max(largest);
  }
  const bool fresh = there & 1u;
  const ScScale s = sc_scale<E4M3>(largest, fresh ? 0.f : sc_old_scale(stored));
  if (lane == 0) w.scales[1][bh] = s.now;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int p = lane + 64 * i;
    if (p >= pairs) continue;
    uint32_t* row = reinterpret_cast<uint32_t*>(out + (uint32_t)(2 * p * BS));
    uint32_t q[2][BS / 4];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int k = 0; k < BS / 4; ++k) {
        const float v0 = A::get(x[i][4 * k], e), v1 = A::get(x[i][4 * k + 1], e), v2 = A::get(x[i][4 * k + 2], e), v3 = A::get(x[i][4 * k + 3], e);
        q[e][k] = finite ? ScCode<E4M3>::encode_fitting(v0, v1, v2, v3, s.inverse)
                         : ScCode<E4M3>::encode(v0 * s.inverse, v1 * s.inverse, v2 * s.inverse, v3 * s.inverse);
      }
    if (!FULL && !fresh) {                                      // what the call does not write is kept
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < BS / 4; ++k) {
          const uint32_t some = there >> (4 * k) & 15u;
          if (some == 15u) continue;
          uint32_t was = row[e * (BS / 4) + k];
          if (s.ratio != 1.f) was = sc_rescale<E4M3>(was, s.ratio);
          const uint32_t mask = (some & 1u ? 0xffu : 0u) | (some & 2u ? 0xff00u : 0u) | (some & 4u ? 0xff0000u : 0u) |
                                (some & 8u ? 0xff000000u : 0u);
          q[e][k] = (q[e][k] & mask) | (was & ~mask);
        }
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

__device__ __forceinline__ int64_t sc_slot(const ScWrite& w, int64_t t) { return t >= 0 && t < w.num_tokens ? w.slots[t] : -1; }
template <int BS>
__device__ __forceinline__ int64_t sc_block(const ScWrite& w, int64_t slot) { return slot >= 0 && slot < w.num_slots ? slot / BS : -1; }

// Whether the list names blocks in more than one run, or in one of more than BS entries, in two launches.  The heads of all runs enter
// themselves in `owner` (an entry for each block, whose contents before do not matter); then each looks whether it is still there.
template <int BS, bool ENTER>
__global__ void __launch_bounds__(256) scaled_index_kernel(const ScWrite w, int* owner, int* repeated) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t block = sc_block<BS>(w, sc_slot(w, i)), before = sc_block<BS>(w, sc_slot(w, i - 1));
  const bool head = block >= 0 && block != before;
  if constexpr (ENTER) {
    if (i == 0) *repeated = 0;
    if (head) owner[block] = (int)i;
  } else {
    if ((head && owner[block] != (int)i) || (block >= 0 && sc_block<BS>(w, sc_slot(w, i - BS)) == block)) *repeated = 1;
  }
}

template <typename act_t, bool E4M3, int BS, int DMAX>
__global__ void __launch_bounds__(256) scaled_write_kernel(const ScWrite w) {
  __shared__ int map[BS], leave, more;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (all heads of a stretch of the list side by side in time: a token's row, and a block, are whole then)
  const int stretch = blockIdx.x / w.head_pairs, head = (blockIdx.x - stretch * w.head_pairs) * 2 + (wave >> 1);
  const int t0 = stretch * w.window;

  // lane l: entry t0 - 1 + l (its block), of which `window` are this workgroup's; those whose predecessor is in another block are heads
  // of runs (every wave finds the same ones)
  const int64_t near = sc_slot(w, t0 - 1 + lane), near_block = sc_block<BS>(w, near), before = __shfl_up(near_block, 1, 64);
  const bool alone = w.repeated != nullptr && *w.repeated == 0;
  uint64_t heads = __ballot(lane >= 1 && lane <= w.window && near_block >= 0 && near_block != before);
  while (heads) {
    const int at = __builtin_ctzll(heads), t = t0 - 1 + at;
    heads &= heads - 1;
    const int64_t first = __shfl(near, at, 64), block = first / BS;
    // the run, and whether it is the whole block in order (a window and a block behind it are lanes of the wave)
    const uint64_t others = ~(__ballot(near_block == block) >> at);
    const int entries = others ? __builtin_ctzll(others) : 64;
    const bool in_order = lane < at || lane >= at + BS || near == first + (lane - at);
    bool full = first % BS == 0 && entries == BS && __ballot(in_order) == ~0ull;
    if (!(alone && full)) {
      __syncthreads();                                          // the last run's map and flags have been read
      if (threadIdx.x < BS) map[threadIdx.x] = -1;
      if (threadIdx.x == BS) leave = more = 0;
      __syncthreads();
      if (alone) {
        if (wave == 0 && lane >= at && lane < at + entries) atomicMax(&map[near % BS], t0 - 1 + lane);
      } else {
        for (int i0 = threadIdx.x; i0 < w.num_tokens; i0 += 256 * kScLook) {
          int64_t s[kScLook];
#pragma unroll
          for (int k = 0; k < kScLook; ++k) s[k] = sc_slot(w, i0 + 256 * k);
#pragma unroll
          for (int k = 0; k < kScLook; ++k) {
            const int i = i0 + 256 * k;
            if (sc_block<BS>(w, s[k]) != block) continue;
            if (i < t) leave = 1;
            else atomicMax(&map[s[k] % BS], i);                 // of two tokens for one slot the later one
            if (i >= t + BS) more = 1;
          }
        }
      }
      __syncthreads();
      if (leave) continue;                                      // that entry's workgroup does the block
      full = full && !more;
    }
    if (head >= w.heads) continue;
    if (full) {
      if (wave & 1) sc_write_values<act_t, E4M3, BS, DMAX, true>(w, block, head, nullptr, t, lane);
      else sc_write_keys<act_t, E4M3, BS, DMAX, true>(w, block, head, nullptr, t, lane);
    } else {
      if (wave & 1) sc_write_values<act_t, E4M3, BS, DMAX, false>(w, block, head, map, 0, lane);
      else sc_write_keys<act_t, E4M3, BS, DMAX, false>(w, block, head, map, 0, lane);
    }
  }
}

// One wave: K or V of one (block, head) of one sequence.  A lane's 16 bytes of a key block are 16 dims of a token, written as they are.
// Of a value block they are 16 tokens of two dims: lane (c, q) = (lane & 15, lane >> 4) takes dims 8 c + 2 q and the next, and has, in
// exchange with the three lanes 16 apart, 4 tokens of dims 8 c .. 8 c + 7, a token's 16 bytes each.  Bound by memory, whose writes are
// hurt by too many of them under way: 5 workgroups of a compute unit (kScReadLds) and stores past the caches.  9 sequences of some 6000
// tokens, 8 heads of 128, 353 MB: 80 us (8 workgroups 87; 4-byte stores of values 84 / 91; two and four blocks a wave 86 and 91 where one
// took 84).
constexpr int kScReadLds = 32 * 1000;                          // bytes that a launch asks for and does not use

template <typename act_t, bool E4M3, int BS, int DMAX>
__global__ void __launch_bounds__(256) scaled_read_kernel(const ScRead w) {
  using A = ScAct<act_t>;
  using S = typename A::S;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int page = blockIdx.x / w.head_pairs, head = (blockIdx.x - page * w.head_pairs) * 2 + (wave >> 1), seq = blockIdx.y;
  const int64_t first = w.starts[seq];
  const int64_t len = min((int64_t)w.lens[seq], (int64_t)w.width * BS);
  const int at0 = page * BS;
  if (head >= w.heads || at0 >= len || first < 0) return;
  // rows behind the end of the output are not written
  const int count = (int)min(min((int64_t)BS, len - at0), w.num_rows - first - at0);
  const int block = w.tables[(int64_t)seq * w.table_stride + page];
  const bool good = block >= 0 && block < w.num_blocks;        // tokens of blocks that do not exist are zeros
  const int64_t bh = (int64_t)(good ? block : 0) * w.heads + head;
  const int kv = wave & 1;
  const float scale = good ? w.scales[kv][bh] : 0.f;
  const uint8_t* in = w.cache[kv] + bh * w.head_size * BS;
  S* out = reinterpret_cast<S*>(w.x[kv]) + (first + at0) * w.stride[kv] + (int64_t)head * w.head_size;
  if (kv == 0) {
    constexpr int NU = (BS * DMAX / 16 + 63) / 64, STEP = 64 / BS;
    const int chunks = w.head_size >> 4, t = lane % BS, c0 = lane / BS;
    sc_u32x4 q[NU];
#pragma unroll
    for (int i = 0; i < NU; ++i)
      q[i] = good && c0 + i * STEP < chunks ? reinterpret_cast<const sc_u32x4*>(in)[lane + 64 * i] : sc_u32x4{0u, 0u, 0u, 0u};
    if (t >= count) return;
    S* row = out + t * w.stride[0] + 16 * c0;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (c0 + i * STEP >= chunks) continue;
      float o[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) ScCode<E4M3>::scaled(q[i][k], scale, o + 4 * k);
      sc_u32x4* p = reinterpret_cast<sc_u32x4*>(row + 16 * STEP * i);
#pragma unroll
      for (int k = 0; k < A::kWords / 4; ++k) {
        sc_u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(S) == 2) v[e] = A::pair(o[8 * k + 2 * e], o[8 * k + 2 * e + 1]);
          else v[e] = __float_as_uint(o[4 * k + e]);
        }
        __builtin_nontemporal_store(v, p + k);
      }
    }
  } else {
    constexpr int NP = DMAX / 128, H = BS == 32 ? 2 : 1, RW = BS < 16 ? BS / 4 : 4;
    const int c0 = lane & 15, q0 = lane >> 4;
    uint32_t r[NP][H][2][4];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t d = 8 * (c0 + 16 * i) + 2 * q0;
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            r[i][h][e][k] = k < RW && good && (int)d < w.head_size ? reinterpret_cast<const uint32_t*>(in + ((d + e) * BS + 16 * h))[k] : 0u;
    }
    const uint32_t lane_off = (uint32_t)(4 * q0 * w.stride[1] + 8 * c0) * sizeof(S);
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        sc_transpose(r[i][h][0]);
        sc_transpose(r[i][h][1]);
        float o[8][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) ScCode<E4M3>::scaled(r[i][h][e & 1][e >> 1], scale, o[e]);
        if (8 * (c0 + 16 * i) >= w.head_size) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (16 * h + 4 * q0 + j >= count) continue;
          char* to = reinterpret_cast<char*>(out + (16 * h + j) * w.stride[1] + 128 * i) + lane_off;
          if constexpr (sizeof(S) == 2) {
            const sc_u32x4 v = {A::pair(o[0][j], o[1][j]), A::pair(o[2][j], o[3][j]), A::pair(o[4][j], o[5][j]), A::pair(o[6][j], o[7][j])};
            __builtin_nontemporal_store(v, reinterpret_cast<sc_u32x4*>(to));
          } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const sc_u32x4 v = {__float_as_uint(o[4 * k][j]), __float_as_uint(o[4 * k + 1][j]), __float_as_uint(o[4 * k + 2][j]), __float_as_uint(o[4 * k + 3][j])};
              __builtin_nontemporal_store(v, reinterpret_cast<sc_u32x4*>(to) + k);
            }
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

int64_t sw_reshape_and_cache_scaled_indexed_workspace_bytes(int num_tokens, int64_t num_blocks) {
  return num_tokens <= sw::kScShort || num_blocks <= 0 ? 0 : (num_blocks + 1) * 4;
}

int sw_reshape_and_cache_scaled_indexed(const void* key, const void* value, void* key_cache, void* value_cache, float* key_scales,
                                        float* value_scales, const int64_t* slot_mapping, int num_tokens, int num_heads, int head_size,
                                        int block_size, int64_t num_blocks, int64_t key_stride, int64_t value_stride, int act_dtype,
                                        int cache_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace sw;
  const int bad = sc_check("reshape_and_cache_scaled", num_heads, head_size, block_size, num_blocks, act_dtype, cache_dtype);
  if (bad) return bad;
  SW_CHECK_ARG(num_tokens >= 0, "reshape_and_cache_scaled: %d tokens", num_tokens);
  const int es = dtype_size(act_dtype);
  SW_CHECK_ARG(sc_aligned(key, key_stride, es) && sc_aligned(value, value_stride, es) && (uintptr_t)key_cache % 16 == 0 &&
                   (uintptr_t)value_cache % 16 == 0,
               "reshape_and_cache_scaled: rows of keys and values, and the caches, must begin on multiples of 16 bytes");
  SW_CHECK_ARG(workspace == nullptr || ((uintptr_t)workspace % 4 == 0 &&
                                        workspace_bytes >= sw_reshape_and_cache_scaled_indexed_workspace_bytes(num_tokens, num_blocks)),
               "reshape_and_cache_scaled: the workspace for %d tokens is too small or not aligned", num_tokens);
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
  static_assert(1 + kScWindow + 32 <= 64, "");
  w.window = num_tokens <= kScShort ? 1 : kScWindow;
  w.head_pairs = (num_heads + 1) / 2;
  const int64_t workgroups = ((int64_t)num_tokens + w.window - 1) / w.window * w.head_pairs;
  SW_CHECK_ARG(workgroups <= kScMostWorkgroups, "reshape_and_cache_scaled: %d tokens of %d heads are too many for a call", num_tokens, num_heads);
  w.repeated = nullptr;
  if (workspace && num_tokens > kScShort) {
    int* const repeated = (int*)workspace;
    w.repeated = repeated;
    auto index = [&](auto bs) {
      const unsigned groups = ((unsigned)num_tokens + 255) / 256;
      scaled_index_kernel<decltype(bs)::value, true><<<groups, 256, 0, (hipStream_t)stream>>>(w, repeated + 1, repeated);
      scaled_index_kernel<decltype(bs)::value, false><<<groups, 256, 0, (hipStream_t)stream>>>(w, repeated + 1, repeated);
    };
    block_size == 8    ? index(std::integral_constant<int, 8>{})
    : block_size == 16 ? index(std::integral_constant<int, 16>{})
                       : index(std::integral_constant<int, 32>{});
    SW_CHECK_LAUNCH();
  }
  const dim3 grid((unsigned)workgroups);
  return sc_by_type(act_dtype, cache_dtype, [&](auto a, auto e) {
    return sc_by_size(head_size, block_size, [&](auto bs, auto d) -> int {
      scaled_write_kernel<decltype(a), decltype(e)::value, decltype(bs)::value, decltype(d)::value>
          <<<grid, 256, 0, (hipStream_t)stream>>>(w);
      SW_CHECK_LAUNCH();
      return SW_OK;
    });
  });
}

int sw_reshape_and_cache_scaled(const void* key, const void* value, void* key_cache, void* value_cache, float* key_scales,
                                float* value_scales, const int64_t* slot_mapping, int num_tokens, int num_heads, int head_size,
                                int block_size, int64_t num_blocks, int64_t key_stride, int64_t value_stride, int act_dtype,
                                int cache_dtype, void* stream) {
  return sw_reshape_and_cache_scaled_indexed(key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping, num_tokens,
                                             num_heads, head_size, block_size, num_blocks, key_stride, value_stride, act_dtype, cache_dtype,
                                             nullptr, 0, stream);
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
  // (a lane's place in a value's row counts 12 rows in 32 bits)
  SW_CHECK_ARG(num_rows == 1 || value_stride * es < 1 << 28, "gather_cache_scaled: rows of values must lie less than 2^28 bytes apart");
  w.head_pairs = (num_heads + 1) / 2;
  SW_CHECK_ARG((int64_t)blocks * w.head_pairs <= kScMostWorkgroups, "gather_cache_scaled: sequences of %d blocks of %d heads are too long for a call",
               blocks, num_heads);
  const dim3 grid(blocks * w.head_pairs, num_seqs);
  return sc_by_type(act_dtype, cache_dtype, [&](auto a, auto e) {
    return sc_by_size(head_size, block_size, [&](auto bs, auto d) -> int {
      scaled_read_kernel<decltype(a), decltype(e)::value, decltype(bs)::value, decltype(d)::value>
          <<<grid, 256, kScReadLds, (hipStream_t)stream>>>(w);
      SW_CHECK_LAUNCH();
      return SW_OK;
    });
  });
}

}  // extern "C"
