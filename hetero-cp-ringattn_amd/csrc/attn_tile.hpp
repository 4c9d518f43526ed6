// Pieces of the matrix-core attention kernels on 32-row query blocks: the 32x32x16 MFMAs, the
// key order that makes a score accumulator the next product's operand, and row epilogues.
#pragma once

#include "hcp_common.hpp"

namespace hcp {

constexpr float kInitMax = -1.0e30f;
constexpr float kGrowSum = 256.0f;  // 2^8: largest partial row sum kept without a max pass

// C-row r of a 32x32 S^T block holds key kperm(r) of that block:
// r = j*8 + h*4 + i  ->  16*(j/2) + 8*h + 4*(j%2) + i.
__device__ __forceinline__ int kperm(int r) {
  const int j = r >> 3, h = (r >> 2) & 1, i = r & 3;
  return 16 * (j >> 1) + 8 * h + 4 * (j & 1) + i;
}

template <int DT>
struct MfmaOps;

template <>
struct MfmaOps<kBF16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag pack(const float* p) {
    frag r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = static_cast<__bf16>(p[i]);
    return r;
  }
};

template <>
struct MfmaOps<kF16> {
  typedef f16x8 frag;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag pack(const float* p) {
    frag r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = static_cast<_Float16>(p[i]);
    return r;
  }
};

template <typename F>
__device__ __forceinline__ F as_frag(u32x4 v) {
  return __builtin_bit_cast(F, v);
}

// {x[lane], x[lane ^ 32]} in some order, on the VALU (no LDS round trip).
__device__ __forceinline__ float max_xor32(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_xor32(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 4 fp32 values as 16-bit `dtype` (bf16 or f16), packed in element order.
__device__ __forceinline__ u32x2 pack4(int dtype, float x0, float x1, float x2, float x3) {
  u32x2 w;
  if (dtype == kBF16) {
    w[0] = f32x2_to_bf16x2_bits(x0, x1);
    w[1] = f32x2_to_bf16x2_bits(x2, x3);
  } else {
    w[0] = static_cast<uint32_t>(f32_to_f16_bits(x0)) | (static_cast<uint32_t>(f32_to_f16_bits(x1)) << 16);
    w[1] = static_cast<uint32_t>(f32_to_f16_bits(x2)) | (static_cast<uint32_t>(f32_to_f16_bits(x3)) << 16);
  }
  return w;
}

// Stores 4 consecutive fp32 values as `dtype` at element offset `off` of `base`.
__device__ __forceinline__ void store4(void* base, int dtype, int64_t off, float x0, float x1, float x2, float x3) {
  if (dtype == kF32) {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + off) = make_float4(x0, x1, x2, x3);
  } else {
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(base) + off) = pack4(dtype, x0, x1, x2, x3);
  }
}

// Epilogue of one (head, query row): normalised output row
// in `dtype` at element offset `off` of `out`, natural-log LSE to *lse (if non-null);
// lanes l and l + 32 hold the two interleaved 4-wide d slices of each 8-wide group.
template <int D>
__device__ __forceinline__ void write_final_row(void* out, int dtype, int64_t off, float* lse, int lhalf,
                                                const f32x16 (&oacc)[D / 32], float m_run, float l_tot, int dn) {
  constexpr int DB = D / 32;
  const bool any = l_tot > 0.f;
  const float inv = any ? 1.f / l_tot : 0.f;
  // 16-bit rows whose starts are 16-byte aligned across the wave: lanes l and l + 32 hold
  // the two 4-wide halves of each 8-wide group, so swapping groups (j, j + 1) with
  // v_permlane32_swap hands each lane one whole group, stored as 16 bytes (half the store
  // instructions of 8-byte stores).  Lanes l and l + 32 share their row, so both are
  // active or neither.  The fused schedule's launcher admits only 16-byte aligned
  // outputs; the 8-byte path below is the fallback for any other caller.
  const bool st16 = dtype != kF32 && __all(((reinterpret_cast<uintptr_t>(out) + static_cast<uintptr_t>(off) * 2) & 15) == 0);
  if (st16) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        if (32 * b + 8 * j >= dn) continue;  // zero-padded columns
        const u32x2 lo = pack4(dtype, inv * oacc[b][4 * j], inv * oacc[b][4 * j + 1], inv * oacc[b][4 * j + 2],
                               inv * oacc[b][4 * j + 3]);
        const u32x2 hi = pack4(dtype, inv * oacc[b][4 * j + 4], inv * oacc[b][4 * j + 5], inv * oacc[b][4 * j + 6],
                               inv * oacc[b][4 * j + 7]);
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const auto r = __builtin_amdgcn_permlane32_swap(hi[k], lo[k], false, false);
          w[k] = r[0];
          w[2 + k] = r[1];
        }
        const int dcol = 32 * b + 8 * (j + 1 - lhalf);
        if (dcol < dn) *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + off + dcol) = w;
      }
  } else {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int dcol = 32 * b + 8 * j + 4 * lhalf;
        if (dcol >= dn) continue;  // zero-padded columns
        store4(out, dtype, off + dcol, inv * oacc[b][4 * j], inv * oacc[b][4 * j + 1], inv * oacc[b][4 * j + 2],
               inv * oacc[b][4 * j + 3]);
      }
  }
  if (lhalf == 0 && lse != nullptr) *lse = any ? (m_run + __log2f(l_tot)) * kLn2 : -INFINITY;
}

// Empty asm that uses x: keeps the code producing x on this side of the next barrier
// (the compiler may otherwise move register-only work across s_barrier).
template <typename T>
__device__ __forceinline__ void pin(const T& x) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass only parses device code; its asm has no "v" registers
  asm volatile("" : : "v"(x));
#else
  (void)x;
#endif
}

__device__ __forceinline__ int simd_id() {
  int r;
  asm volatile("s_getreg_b32 %0, hwreg(HW_REG_HW_ID, 4, 2)" : "=s"(r));
  return r;
}

}  // namespace hcp
