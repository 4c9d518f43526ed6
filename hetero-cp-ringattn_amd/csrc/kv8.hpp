// The 8-bit paged cache: codes [2, num_blocks, bs, Hkv, D] (plane 0 = K, 1 = V) and a scale
// for each plane, block and head [2, num_blocks, Hkv] fp32; a code stands for scale * code.
#pragma once

#include "kernels.hpp"

namespace hcp {

enum Kv8Format : int32_t { kE4M3 = 1, kInt8 = 2 };

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// The smallest power of two, 2^-100 at least, under which a block whose largest magnitude is
// `amax` (finite, >= 0) fits the format: 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.  A power of
// two makes x / scale exact, so a value is rounded once, and raising a block's scale later
// moves an e4m3 code's exponent only (codes that fall below 2^-6 round again; an int8 code
// each time, by at most 1/2 + 1/4 + ... < 1 step in all).  The floor keeps 1 / scale and the
// products of two scales normal; it quantises what is below 2^-109 to 0.
template <int F>
__device__ __forceinline__ float kv8_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127 - (F == kE4M3 ? 8 : 6) + ((u & 0x7fffffu) > (F == kE4M3 ? 0x600000u : 0x7e0000u));
  return __uint_as_float(static_cast<uint32_t>(max(e, -100) + 127) << 23);
}

// Four values, at most the format's largest in magnitude, to codes (nearest, ties to even).
template <int F>
__device__ __forceinline__ uint32_t kv8_encode4(float a, float b, float c, float d) {
  if constexpr (F == kE4M3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
  } else {
    auto code = [](float x) { return static_cast<uint32_t>(static_cast<int>(__builtin_rintf(x))) & 0xffu; };
    return code(a) | code(b) << 8 | code(c) << 16 | code(d) << 24;
  }
}

// A word of codes to four fp32 values.
template <int F>
__device__ __forceinline__ void kv8_decode4(uint32_t w, float* x) {
  if constexpr (F == kE4M3) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = lo[0]; x[1] = lo[1]; x[2] = hi[0]; x[3] = hi[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  }
}

// Eight consecutive values of a row in DT as they are stored, to fp32 and back.  VEC: 16-byte
// accesses.
template <int DT, bool VEC>
struct Row8 {
  float x[8];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = load_elem<DT>(p, at + i);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
  }
  __device__ __forceinline__ void get(float* y) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
  }
};
template <>
struct Row8<kF32, true> {
  float4 lo, hi;
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    lo = q[0];
    hi = q[1];
  }
  __device__ __forceinline__ void clear() { lo = hi = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float* y) const {
    y[0] = lo.x; y[1] = lo.y; y[2] = lo.z; y[3] = lo.w; y[4] = hi.x; y[5] = hi.y; y[6] = hi.z; y[7] = hi.w;
  }
};
template <int DT>
struct Row8<DT, true> {
  u32x4 w;
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
  }
  __device__ __forceinline__ void clear() { w = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void get(float* y) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = DT == kBF16 ? __uint_as_float(w[i] << 16) : f16_bits_to_f32(static_cast<uint16_t>(w[i] & 0xffffu));
      y[2 * i + 1] = DT == kBF16 ? __uint_as_float(w[i] & 0xffff0000u) : f16_bits_to_f32(static_cast<uint16_t>(w[i] >> 16));
    }
  }
};
template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* p, int64_t at, const float* x) {
  if constexpr (VEC && DT == kF32) {
    float* const q = static_cast<float*>(p) + at;
    store16_nt_sc1(q, __builtin_bit_cast(u32x4, make_float4(x[0], x[1], x[2], x[3])));
    store16_nt_sc1(q + 4, __builtin_bit_cast(u32x4, make_float4(x[4], x[5], x[6], x[7])));
  } else if constexpr (VEC) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = DT == kBF16 ? f32x2_to_bf16x2_bits(x[2 * i], x[2 * i + 1])
                         : static_cast<uint32_t>(f32_to_f16_bits(x[2 * i])) | static_cast<uint32_t>(f32_to_f16_bits(x[2 * i + 1])) << 16;
    store16_nt_sc1(static_cast<uint16_t*>(p) + at, w);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) store_elem<DT>(p, at + i, x[i]);
  }
}

}  // namespace hcp
