// The 8-bit cache with one scale for each (block, kv head): what its kernels share.
//
// A block's codes lie as the unscaled 8-bit cache's do, keys [blocks, heads, head_size / 16, block, 16] and values
// [blocks, heads, head_size, block], one byte each; scales are fp32 [blocks, heads], one tensor for keys and one for values.
// A code stands for code * scale.  Codes are int8 in -127 .. 127 or e4m3 (OCP, largest 448; the codes of NaN are not written).
#pragma once

#include "common.cuh"

namespace sw {

using sc_f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using sc_u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using sc_u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

// Workgroups of up to 512 threads that a launch's first dimension can have: it counts threads in 32 bits.
constexpr int64_t kScMostWorkgroups = UINT32_MAX / 512;

// Blocks whose largest magnitude is below this are held as zeros: its reciprocal, and that of a 448th of it, are finite.
constexpr float kScTiny = 0x1p-100f;

template <bool E4M3> struct ScCode;

template <> struct ScCode<false> {
  static constexpr float kTop = 127.f, kUnit = 1.f / 127.f;
  // four values in units of the scale -> four codes; a NaN is held as 0
  __device__ static __forceinline__ uint32_t encode(float a, float b, float c, float d) {
    return byte(a) | (byte(b) << 8) | (byte(c) << 16) | (byte(d) << 24);
  }
  // the same of finite values that a scale of theirs has brought to +-127: 1.5 x 2^23 + v has v's nearest integer in its low byte.  (Two
  // roundings: the product's takes what lies on the middle of two codes but for the reciprocal's rounding back there, and so to the even one.)
  __device__ static __forceinline__ uint32_t encode_fitting(float a, float b, float c, float d, float inverse) {
#pragma clang fp contract(off)
    constexpr float at = 12582912.f;
    const float pa = a * inverse, pb = b * inverse, pc = c * inverse, pd = d * inverse;
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(pb + at), __float_as_uint(pa + at), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(pd + at), __float_as_uint(pc + at), 0x04000c0cu);
    return lo | hi;
  }
  __device__ static __forceinline__ uint32_t byte(float x) {
    const float y = rintf(__builtin_amdgcn_fmed3f(x, -kTop, kTop));
    return (uint32_t)(int)(x != x ? 0.f : y) & 0xffu;
  }
  __device__ static __forceinline__ void decode(uint32_t w, float* o) {
    o[0] = (float)(int)(int8_t)(w & 0xffu);
    o[1] = (float)(int)(int8_t)((w >> 8) & 0xffu);
    o[2] = (float)(int)(int8_t)((w >> 16) & 0xffu);
    o[3] = (float)((int)w >> 24);
  }
  // four codes times a scale, each rounded once: (code + 128) scale - 128 scale in one operation
  __device__ static __forceinline__ void scaled(uint32_t w, float scale, float* o) {
    const uint32_t u = w ^ 0x80808080u;
    const float off = -128.f * scale;
    o[0] = fmaf((float)(u & 0xffu), scale, off);
    o[1] = fmaf((float)((u >> 8) & 0xffu), scale, off);
    o[2] = fmaf((float)((u >> 16) & 0xffu), scale, off);
    o[3] = fmaf((float)(u >> 24), scale, off);
  }
  // four codes as four halves, exactly: 0x6400 | u is 1024 + u, u = code + 128
  __device__ static __forceinline__ sc_u32x2 widen(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const sc_f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
    const sc_f16x2 lo = __builtin_bit_cast(sc_f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
    const sc_f16x2 hi = __builtin_bit_cast(sc_f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
    return sc_u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  }
};

template <> struct ScCode<true> {
  static constexpr float kTop = 448.f, kUnit = 1.f / 448.f;
  __device__ static __forceinline__ float clip(float x) {
    const float y = __builtin_amdgcn_fmed3f(x, -kTop, kTop);
    return x != x ? 0.f : y;
  }
  __device__ static __forceinline__ uint32_t encode(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(clip(a), clip(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(clip(c), clip(d), w, true);
    return (uint32_t)w;
  }
  __device__ static __forceinline__ void decode(uint32_t w, float* o) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    o[0] = lo[0];
    o[1] = lo[1];
    o[2] = hi[0];
    o[3] = hi[1];
  }
  // (the conversion takes what is a rounding above 448 to 448)
  __device__ static __forceinline__ uint32_t encode_fitting(float a, float b, float c, float d, float inverse) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inverse, b * inverse, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inverse, d * inverse, w, true);
    return (uint32_t)w;
  }
  __device__ static __forceinline__ void scaled(uint32_t w, float scale, float* o) {
    decode(w, o);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] *= scale;
  }
  // (e4m3's 4 bits of magnitude and powers down to 2^-9 fit a half exactly)
  __device__ static __forceinline__ sc_u32x2 widen(uint32_t w) {
    return sc_u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, true))};
  }
};

// A scale as an earlier write left it: 0, or at least kScTiny / 448.  A block that was never written may hold anything, also what has no
// finite reciprocal.
constexpr float kScLeast = 0x1p-110f;
__device__ __forceinline__ float sc_old_scale(float s) { return s >= kScLeast && s < INFINITY ? s : 0.f; }

inline bool sc_head_size(int d) { return d == 64 || d == 80 || d == 96 || d == 112 || d == 128 || d == 256; }

}  // namespace sw
