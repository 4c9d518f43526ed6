// Norms of the queries and keys of each head, the position rotation in the same pass, and
// the append of K / V to the paged cache through a slot map.
//
// A row x of D elements (one head of one token) becomes y = x * rsqrt(mean(x^2) + eps) * w,
// and of its first r dims every plane (i, j) is turned by its position's angle:
// (y_i cos - y_j sin, y_j cos + y_i sin), with (i, j) = (p, p + r/2) (halves) or (2p, 2p + 1)
// (pairs).  The arithmetic is fp32 from the loads on and rounds once, at the store.
//
// Bound by HBM: a row is read once and written once, ~10 flops an element.  A lane holds two
// chunks of C elements r/2 apart (16 bytes each), so that in the halves form both ends of a
// plane are in one lane and nothing is exchanged but the sum of squares; a row takes
// D / (2 C) lanes, a wave 64 / that rows of one token at a time.  Its lanes hold the token's cos and
// sin for all of them and load the weights for every run (from the L1: q's and k's differ); the next
// run's rows load while one is turned.  Stores
// stream (nt): 32768 tokens of 32/8 heads of 128 dims take 189 us so, 198 with plain ones (805 MB
// of rows and 17 MB of angles: 4.35 TB/s; a copy of 2 GiB reaches 4.97), 2048 tokens 12 and 14.5.
// Streaming loads as well: 184 and 11-14 (what the projection wrote last is still in the caches).
#include <algorithm>

#include "kernels.hpp"

namespace hcp {

namespace {

// C consecutive elements to fp32, in one load of C elements (VEC) or one each.
template <int DT, int C, bool VEC>
struct Chunk {
  static constexpr int kBytes = DT == kF32 ? 4 : 2;
  uint32_t w[C * kBytes / 4];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    if constexpr (VEC) {
      if constexpr (sizeof(w) == 16) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const char*>(base) + at * kBytes);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = x[i];
      } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(static_cast<const char*>(base) + at * kBytes);
        w[0] = x[0];
        w[1] = x[1];
      }
    } else if constexpr (DT == kF32) {
#pragma unroll
      for (int i = 0; i < C; ++i) w[i] = static_cast<const uint32_t*>(base)[at + i];
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(base) + at;
#pragma unroll
      for (int i = 0; i < C / 2; ++i) w[i] = static_cast<uint32_t>(p[2 * i]) | static_cast<uint32_t>(p[2 * i + 1]) << 16;
    }
  }
  __device__ __forceinline__ void store(void* base, int64_t at) const {
    if constexpr (VEC) {
      if constexpr (sizeof(w) == 16)
        __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]},
                                    reinterpret_cast<u32x4*>(static_cast<char*>(base) + at * kBytes));
      else
        *reinterpret_cast<u32x2*>(static_cast<char*>(base) + at * kBytes) = u32x2{w[0], w[1]};
    } else if constexpr (DT == kF32) {
#pragma unroll
      for (int i = 0; i < C; ++i) static_cast<uint32_t*>(base)[at + i] = w[i];
    } else {
      uint16_t* p = static_cast<uint16_t*>(base) + at;
#pragma unroll
      for (int i = 0; i < C / 2; ++i) {
        p[2 * i] = static_cast<uint16_t>(w[i]);
        p[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
      }
    }
  }
  __device__ __forceinline__ void unpack(float* x) const {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if constexpr (DT == kF32) x[i] = __uint_as_float(w[i]);
      else if constexpr (DT == kBF16) x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
      else x[i] = f16_bits_to_f32(static_cast<uint16_t>(i & 1 ? w[i / 2] >> 16 : w[i / 2]));
    }
  }
  __device__ __forceinline__ void pack(const float* x) {
    if constexpr (DT == kF32) {
#pragma unroll
      for (int i = 0; i < C; ++i) w[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < C / 2; ++i)
        w[i] = DT == kBF16 ? f32x2_to_bf16x2_bits(x[2 * i], x[2 * i + 1])
                           : static_cast<uint32_t>(f32_to_f16_bits(x[2 * i])) |
                                 static_cast<uint32_t>(f32_to_f16_bits(x[2 * i + 1])) << 16;
    }
  }
};

template <int N>
__device__ __forceinline__ void load_f32(const float* p, float* x) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = p[i];
}

}  // namespace

// A wave takes `groups` runs of 64 / lanes rows of one token: its q heads, k heads and, in
// the append, v heads in that order.
template <int DT, int C, bool VEC, bool PAIRS>
__global__ __launch_bounds__(256) void qk_norm_kernel(QkNorm a) {
  using Ch = Chunk<DT, C, VEC>;
  const int lane = threadIdx.x & 63;
  const int sub = lane & (a.lanes - 1), in_wave = lane >> a.lanes_log2, per_wave = 64 >> a.lanes_log2;
  const int rows = a.hq + a.hkv * (a.pool != nullptr ? 2 : 1);
  const int half = a.rot >> 1;
  // this lane's two chunks of a row
  const bool turns = sub * C < half;
  const int lo = turns ? sub * C : a.rot + (sub * C - half);
  const int hi = turns ? lo + half : lo + ((a.d - a.rot) >> 1);
  const bool in = sub * 2 * C < a.d;
  const int64_t items = a.tokens * a.splits;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); item < items;
       item += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t t = a.splits == 1 ? item : item / a.splits;
    const int part = static_cast<int>(item - t * a.splits);
    const int r1 = min(rows, (part + 1) * a.groups * per_wave);
    // the rows of one pass over the lanes: kind 0, 1, 2 = q, k, v
    auto kind_of = [&](int r) __attribute__((always_inline)) { return r < a.hq ? 0 : r < a.hq + a.hkv ? 1 : 2; };
    auto head_of = [&](int r, int kind) __attribute__((always_inline)) { return r - (kind > 0 ? a.hq : 0) - (kind > 1 ? a.hkv : 0); };
    auto load = [&](int r, Ch& c0, Ch& c1) __attribute__((always_inline)) {
      if (r >= r1 || !in) return;
      const int kind = kind_of(r);
      const int64_t at = head_of(r, kind) * a.hs[kind] + t * a.ss[kind];
      c0.load(a.src[kind], at + lo);
      c1.load(a.src[kind], at + hi);
    };
    int r = part * a.groups * per_wave + in_wave;
    Ch c0{}, c1{}, n0{}, n1{};
    load(r, c0, c1);
    // angles of the token: C of them in the halves form, C / 2 for each chunk in the pairs form
    float cs[C], sn[C];
    bool turn = a.rot > 0;
    if (turn) {
      const int64_t p = a.pos[t];
      if (p < 0 || p >= a.rope_rows) {
        turn = false;
        if (lane == 0 && part == 0) atomicOr(a.err, 4);
      } else if (turns && in) {
        const float* crow = a.rope_cos + p * half;
        const float* srow = a.rope_sin + p * half;
        if constexpr (PAIRS) {
          load_f32<C / 2>(crow + lo / 2, cs);
          load_f32<C / 2>(crow + hi / 2, cs + C / 2);
          load_f32<C / 2>(srow + lo / 2, sn);
          load_f32<C / 2>(srow + hi / 2, sn + C / 2);
        } else {
          load_f32<C>(crow + lo, cs);
          load_f32<C>(srow + lo, sn);
        }
      }
    }
    int64_t slot = -1;
    if (a.pool != nullptr) {
      slot = a.slots[t];
      if (slot >= a.pool_slots) {
        slot = -1;
        if (lane == 0 && part == 0) atomicOr(a.err, 1);
      }
    }
    for (; r - in_wave < r1; r += per_wave) {
      load(r + per_wave, n0, n1);  // the next pass's rows are on their way while this one's are turned
      const int kind = kind_of(r), head = head_of(r, kind);
      const bool keep = r < r1 && in && (kind == 0 || a.pool == nullptr || slot >= 0);
      float x0[C], x1[C];
      c0.unpack(x0);
      c1.unpack(x1);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < C; ++i) sum += x0[i] * x0[i] + x1[i] * x1[i];
      for (int off = 1; off < a.lanes; off <<= 1) sum += __shfl_xor(sum, off);
      if (kind < 2 && in) {
        const float f = rsqrtf(sum * a.inv_d + a.eps);
        if (a.w[kind] != nullptr) {
          Ch w0, w1;
          float v0[C], v1[C];
          w0.load(a.w[kind], lo);
          w1.load(a.w[kind], hi);
          w0.unpack(v0);
          w1.unpack(v1);
#pragma unroll
          for (int i = 0; i < C; ++i) {
            x0[i] = x0[i] * f * v0[i];
            x1[i] = x1[i] * f * v1[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < C; ++i) {
            x0[i] *= f;
            x1[i] *= f;
          }
        }
        if (turn && turns) {
          if constexpr (PAIRS) {
#pragma unroll
            for (int i = 0; i < C; i += 2) {
              const float a0 = x0[i], b0 = x0[i + 1], a1 = x1[i], b1 = x1[i + 1];
              x0[i] = a0 * cs[i / 2] - b0 * sn[i / 2];
              x0[i + 1] = b0 * cs[i / 2] + a0 * sn[i / 2];
              x1[i] = a1 * cs[C / 2 + i / 2] - b1 * sn[C / 2 + i / 2];
              x1[i + 1] = b1 * cs[C / 2 + i / 2] + a1 * sn[C / 2 + i / 2];
            }
          } else {
#pragma unroll
            for (int i = 0; i < C; ++i) {
              const float y0 = x0[i], y1 = x1[i];
              x0[i] = y0 * cs[i] - y1 * sn[i];
              x1[i] = y1 * cs[i] + y0 * sn[i];
            }
          }
        }
        c0.pack(x0);
        c1.pack(x1);
      }
      void* dst;
      int64_t at;
      if (kind == 0 || a.pool == nullptr) {
        dst = a.out[kind];
        at = head * a.out_hs[kind] + t * a.out_ss[kind];
      } else {
        dst = a.pool;
        at = (kind == 2 ? a.plane_elems : 0) + (slot * a.hkv + head) * a.d;
      }
      if (keep) {
        c0.store(dst, at + lo);
        c1.store(dst, at + hi);
      }
      c0 = n0;
      c1 = n1;
    }
  }
}

template <int DT, int C, bool VEC>
static void launch_qk_norm_p(const QkNorm& a, bool pairs, unsigned grid, hipStream_t stream) {
  if (pairs) qk_norm_kernel<DT, C, VEC, true><<<grid, 256, 0, stream>>>(a);
  else qk_norm_kernel<DT, C, VEC, false><<<grid, 256, 0, stream>>>(a);
}

void launch_qk_norm(int dtype, bool pairs, QkNorm a, hipStream_t stream) {
  const int es = dtype == kF32 ? 4 : 2;
  // 16-byte chunks where both parts of a row hold whole pairs of them, else of 4 elements
  const int c = es == 2 && a.d % 16 == 0 && a.rot % 16 == 0 ? 8 : 4;
  // one load of a chunk where every chunk starts on a multiple of its bytes
  bool vec = true;
  auto whole = [&](const void* p, int64_t hs, int64_t ss) {
    vec = vec && reinterpret_cast<uintptr_t>(p) % (c * es) == 0 && hs % c == 0 && ss % c == 0;
  };
  for (int i = 0; i < (a.pool != nullptr ? 3 : 2); ++i) whole(a.src[i], a.hs[i], a.ss[i]);
  for (int i = 0; i < (a.pool != nullptr ? 1 : 2); ++i) whole(a.out[i], a.out_hs[i], a.out_ss[i]);
  for (int i = 0; i < 2; ++i)
    if (a.w[i] != nullptr) whole(a.w[i], 0, 0);
  if (a.pool != nullptr) whole(a.pool, 0, 0);
  a.lanes = 1;
  a.lanes_log2 = 0;
  while (a.lanes * 2 * c < a.d) {
    a.lanes *= 2;
    ++a.lanes_log2;
  }
  // Runs of rows a wave takes: one each while the waves are no more than the GPU holds (64
  // tokens, 16/2 heads of 128 dims: 3.7 us with one, 5.8 with three), else so many that the
  // token's angles are loaded once for all of them (32768 tokens, 32/8 heads: 205 us with one,
  // 189 with all six; 8192 tokens, 14/2 heads of 64: 13.2 with one, 10.8 with both).
  constexpr int64_t kResident = 256 * 32;
  const int per_wave = 64 / a.lanes, rows = a.hq + a.hkv * (a.pool != nullptr ? 2 : 1);
  const int64_t runs = ceil_div(rows, per_wave);
  a.groups = static_cast<int32_t>(std::max<int64_t>(1, std::min(runs, a.tokens * runs / kResident)));
  a.splits = static_cast<int32_t>(ceil_div(runs, a.groups));
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(a.tokens * a.splits, 4), 1 << 20));
  if (dtype == kF32) {
    if (vec) launch_qk_norm_p<kF32, 4, true>(a, pairs, grid, stream);
    else launch_qk_norm_p<kF32, 4, false>(a, pairs, grid, stream);
  } else if (dtype == kBF16) {
    if (c == 8 && vec) launch_qk_norm_p<kBF16, 8, true>(a, pairs, grid, stream);
    else if (vec) launch_qk_norm_p<kBF16, 4, true>(a, pairs, grid, stream);
    else if (c == 8) launch_qk_norm_p<kBF16, 8, false>(a, pairs, grid, stream);
    else launch_qk_norm_p<kBF16, 4, false>(a, pairs, grid, stream);
  } else {
    if (c == 8 && vec) launch_qk_norm_p<kF16, 8, true>(a, pairs, grid, stream);
    else if (vec) launch_qk_norm_p<kF16, 4, true>(a, pairs, grid, stream);
    else if (c == 8) launch_qk_norm_p<kF16, 8, false>(a, pairs, grid, stream);
    else launch_qk_norm_p<kF16, 4, false>(a, pairs, grid, stream);
  }
  HCP_HIP(hipGetLastError());
}

}  // namespace hcp
