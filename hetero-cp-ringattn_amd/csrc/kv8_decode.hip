// Single-query attention over the 8-bit paged cache (layout in kv8.hpp): per sequence and
// query head S = scale * s_K (q . c_K) over its tokens, shard after shard; O = sum P s_V c_V,
// lse = ln sum e^S; no token: O = 0, lse = -inf.
//
// HBM-bound: every code is read once, half the bytes of the 16-bit decode for the same
// products, so the work beside the loads has to be half as large, too.  Both products run on
// the matrix cores and no value passes through LDS on the way:
//   * One launch covers all shards.  Where the sequences alone fill the chip, or are short, a
//     workgroup has one of them (direct): `heads` kv heads x `subs` waves that share its
//     tokens and meet in LDS.  Otherwise the 16-token groups of all sequences stand in one row
//     and every worker takes the same length of it (balanced), so ragged lengths leave no
//     CU behind: a worker that crosses a sequence's end writes one partial of each side, at
//     place (worker + sequence) of the workspace -- a pair moves on in one or the other, so no
//     two share a place -- and kv8_join_kernel merges a sequence's places, which are neighbours.
//   * A step is 32 tokens.  S^T = K Q^T (16x16x32, f16): A = 16 key rows, their codes converted
//     in registers (exact: a code has at most 8 significant bits), B = the rep <= 16 query
//     heads.  16-bit q times a power of two that brings its largest value to 2^14 is exact in
//     f16, too (what falls below f16 is 2^-38 of the largest), so bf16 and fp16 share the
//     kernel.  Scales are applied to S in fp32.
//   * O^T = V^T P^T: lane (col, grp) of S^T holds the scores of query col and keys 4 grp + i of
//     both groups, which is the B operand of keys {4 grp + i, 16 + 4 grp + i} as it stands.  A =
//     V^T for the same keys: lane (m, grp) loads D/16 neighbouring dims of those 8 keys, so
//     tile j of the product holds dims m D/16 + j and pairs of keys are put together by byte
//     permutes.  O^T stays in the lane whose query it is: max, rescale and sum need two
//     cross-lane steps each and no broadcast.
//   * Weights w = p s_V 2^(14 + m - a) with `a` the running maximum of log2(p s_V), which is
//     tracked like m, over each 16-token group's own scores and scale: w <= 2^14 whatever the
//     scales, and split into two f16 of 11 bits each, w = hi + lo, so P carries 22 bits (one f16
//     alone would put 2^-12 on every weight, against the fp32 weights of the 16-bit decode).
//     Sums and statistics are fp32.
//
// Measured, 32/8 heads of 128, e4m3, blocks of 16: 64 sequences of 8-16k tokens 267 us (1.63 GB at
// 6.1 TB/s, each byte fetched once; the 16-bit decode of 64 x 16k 635 us for 4.3 GB), 6 x 2085 of
// 16/2 heads 12.0 us, one sequence of 130 tokens 6.6 us.  What bounds the short ones is the chain of
// lengths, table, q and codes, one latency each (2.5-4 us), then 0.95 us a step of a lone wave, whose
// instructions no other wave hides.  Two steps of codes under way instead of one cost more in
// registers and instructions than they hid (64 sequences 263 -> 270 us, one of 130 tokens 6.6 -> 8.3).
#include <algorithm>
#include <type_traits>

#include "kv8.hpp"

namespace hcp {

struct Kv8DecodeArgs {
  const uint16_t* q;
  int64_t q_bs, q_hs;  // elements
  const uint8_t* pool;
  const float* scales;
  int64_t plane_bytes, plane_scales;  // from K's to V's
  int64_t num_blocks;
  int32_t bs, hkv, hq, rep;
  DecodeSpan span[kMaxDomains];
  int32_t n_spans, heads, subs;
  int32_t gpb, gpb_shift;  // 16-token groups per block, its log2 or -1
  int32_t q_bf16, out_dtype, dn;
  float scale_log2;
  int32_t workers, min_len;  // balanced: workers per head group (0: direct), least groups of one
  float *ws_o, *ws_lse;      // [workers + batch][hq][dn]
  int2* range;               // [batch] first place and places of a sequence
  void* out;
  int64_t out_rs;
  float* lse;
  int32_t batch;
  int* err;
};
static_assert(sizeof(Kv8DecodeArgs) <= 4096, "kernel arguments are limited to 4 KiB");

constexpr float kNoMax = -1.0e30f;
// V scales count as 2^-110 at least in the running maximum a (not in the product): a >= m - 110, so
// 2^(m - a + 14) and the 2^(a - m - 14) that takes it out again are normal numbers, for scales of 0,
// too.  The weights of smaller scales are below 2^14 by their distance; of 2^-126 they keep 22 bits.
constexpr float kLeastVScale = 0x1p-110f;
// Most waves per workgroup: four to a SIMD, which 128 registers allow; the padded form needs more.
constexpr int kv8_waves(bool pad) { return pad ? 8 : 16; }

// A word of codes to two pairs of f16: codes 0, 1 and 2, 3.  int8: u = code + 128 as the low
// byte of 1024 + u, then - 1152.
template <int F>
__device__ __forceinline__ void to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (F == kE4M3) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  } else {
    const f16x2 bias = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
    auto f = [&](uint32_t sel) {
      return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)) + bias);
    };
    w ^= 0x80808080u;
    lo = f(0x04010400u);
    hi = f(0x04030402u);
  }
}

__device__ __forceinline__ f32x4 mma_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The four lanes with the same lane & 15.
template <typename Op>
__device__ __forceinline__ float over_groups(float v, Op op) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2));
}

// N consecutive outputs (4 or 8) in the output type; rows start on 4-element boundaries.
template <int N>
__device__ __forceinline__ void store_out(void* out, int dtype, int64_t at, const float* x) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    if (dtype == kF32) {
      *reinterpret_cast<float4*>(static_cast<float*>(out) + at + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
    } else if (dtype == kBF16) {
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + at + e) =
          u32x2{f32x2_to_bf16x2_bits(x[e], x[e + 1]), f32x2_to_bf16x2_bits(x[e + 2], x[e + 3])};
    } else {
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + at + e) = u32x2{pack_f16(x[e], x[e + 1]), pack_f16(x[e + 2], x[e + 3])};
    }
  }
}

// PAD: head dim a.dn < D (a multiple of 8); 8-byte pieces past it are not loaded (zeros) nor
// stored.
template <int F, int D, bool PAD>
__global__ __launch_bounds__(64 * kv8_waves(PAD)) void kv8_decode_kernel(Kv8DecodeArgs a) {
  const int dn = PAD ? a.dn : D;
  constexpr int KL = D / 64;  // 16-byte loads of a key row per lane
  constexpr int KS = D / 32;  // k-steps of S
  constexpr int VB = D / 16;  // dims of V per lane, and tiles of O
  constexpr int VW = VB / 4;
  constexpr int OS = D + 4;   // LDS row of the meeting, 4 floats apart from a bank's multiple
  extern __shared__ __attribute__((aligned(16))) float meet_lds[];  // subs > 1: [wave][rep][OS], then lse [wave][16]

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sub = wave / a.heads;
  const int kvh = blockIdx.z * a.heads + wave - sub * a.heads;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  int b = blockIdx.y;

  auto span_end = [&](int s) __attribute__((always_inline)) -> int64_t {
    const DecodeSpan& sp = a.span[s];
    if (sp.seq_lens == nullptr) return sp.t1;
    return min(sp.t1, static_cast<int64_t>(__builtin_amdgcn_readfirstlane(sp.seq_lens[b])) - sp.len_off);
  };
  auto span_groups = [&](int s, int64_t t_end) __attribute__((always_inline)) {
    const int64_t t0 = a.span[s].t0;
    return t_end > t0 ? static_cast<int>((t_end + 15) / 16 - t0 / 16) : 0;
  };
  auto seq_groups = [&]() __attribute__((always_inline)) {
    int n = 0;
    for (int s = 0; s < a.n_spans; ++s) n += span_groups(s, span_end(s));
    return n;
  };
  int total, begin = 0, end_all;  // groups of sequence b; the workgroup's: [begin, end_all)
  int left = 0;                   // groups of the worker after those
  if (a.workers == 0) {
    total = end_all = seq_groups();
  } else {
    // The row of all sequences' groups, each rounded to whole steps: lane i has sequence i of 64.
    auto lane_groups = [&](int i) __attribute__((always_inline)) {
      int n = 0;
      if (i < a.batch)
        for (int s = 0; s < a.n_spans; ++s) {
          const DecodeSpan& sp = a.span[s];
          const int64_t t_end = sp.seq_lens == nullptr ? sp.t1 : min(sp.t1, static_cast<int64_t>(sp.seq_lens[i]) - sp.len_off);
          n += span_groups(s, t_end);
        }
      return (n + 1) & ~1;
    };
    auto scan = [&](int n) __attribute__((always_inline)) {  // inclusive, over the wave
      for (int off = 1; off < 64; off *= 2) {
        const int v = __shfl_up(n, off);
        if (lane >= off) n += v;
      }
      return n;
    };
    int all = 0;
    for (int i = 0; i < a.batch; i += 64) all += __builtin_amdgcn_readlane(scan(lane_groups(i + lane)), 63);
    const int len = max((all + 2 * a.workers - 1) / (2 * a.workers) * 2, a.min_len);
    const int w = blockIdx.x;
    const int64_t from = static_cast<int64_t>(w) * len;
    if (w == 0 && blockIdx.z == 0 && wave == 0) {  // where the join finds every sequence
      int start = 0;
      for (int i = 0; i < a.batch; i += 64) {
        const int n = lane_groups(i + lane), sum = scan(n), at = start + sum - n;
        if (i + lane < a.batch) a.range[i + lane] = n == 0 ? make_int2(0, 0) : make_int2(at / len + i + lane, (at + n - 1) / len - at / len + 1);
        start += __builtin_amdgcn_readlane(sum, 63);
      }
    }
    if (from >= all) return;  // the whole workgroup
    int start = 0;
    b = 0;
    for (int i = 0; i < a.batch; i += 64) {
      const int n = lane_groups(i + lane), sum = scan(n);
      const uint64_t past = __ballot(start + sum > from);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        b = i + at;
        begin = static_cast<int>(from) - (start + __builtin_amdgcn_readlane(sum - n, at));
        break;
      }
      start += __builtin_amdgcn_readlane(sum, 63);
    }
    total = seq_groups();
    const int mine = min(len, all - static_cast<int>(from));
    end_all = min(begin + mine, (total + 1) & ~1);
    left = mine - (end_all - begin);
  }

  for (;;) {  // one sequence's share
    const int run_len = (end_all - begin + 2 * a.subs - 1) / (2 * a.subs) * 2;  // whole steps
    const int g0 = min(begin + sub * run_len, total);
    const int g1 = min(min(g0 + run_len, end_all), total);

    // Q^T in f16, times a power of two that brings the row's largest value to 2^14 .. 2^15.
    // k-step 2 h + e holds dims 16 grp + 64 h + 8 e + i, as the 16-byte loads of K bring them.
    u32x4 qf[KS];
    float c_log2;
    {
      float x[KS][8];
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d0 = grp * 16 + 64 * (s / 2) + 8 * (s % 2);
        u32x4 v = {0, 0, 0, 0};
        if (col < a.rep && (!PAD || d0 < dn))
          v = *reinterpret_cast<const u32x4*>(a.q + b * a.q_bs + (kvh * a.rep + col) * a.q_hs + d0);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          x[s][2 * w] = a.q_bf16 ? __uint_as_float(v[w] << 16) : f16_bits_to_f32(static_cast<uint16_t>(v[w] & 0xffffu));
          x[s][2 * w + 1] = a.q_bf16 ? __uint_as_float(v[w] & 0xffff0000u) : f16_bits_to_f32(static_cast<uint16_t>(v[w] >> 16));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[s][i]) & 0x7fffffffu);
      }
      // as floats the bits of |x| keep their order (NaN: dropped by the maximum, kept in x)
      const float m = over_groups(__uint_as_float(top), [](float u, float v) { return fmaxf(u, v); });
      const bool plain = m > 0.f && m < INFINITY;
      const int k = plain ? max(static_cast<int>(__float_as_uint(m) >> 23) - 127, -100) : 14;
      const float up = __uint_as_float(static_cast<uint32_t>(14 - k + 127) << 23);
      c_log2 = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(k - 14 + 127) << 23);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int w = 0; w < 4; ++w) qf[s][w] = pack_f16(x[s][2 * w] * up, x[s][2 * w + 1] * up);
    }

    f32x4 acc[VB];
#pragma unroll
    for (int j = 0; j < VB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = kNoMax, a_run = kNoMax, l_run = 0.f;

    const uint32_t row = static_cast<uint32_t>(a.hkv) * dn;  // bytes of a slot, all heads
    const int64_t block_bytes = static_cast<int64_t>(a.bs) * row;
    const uint8_t* const k_head = a.pool + kvh * dn;
    const uint8_t* const v_head = k_head + a.plane_bytes;
    const uint32_t k_at = col * row + grp * 16, v_at = grp * 4 * row + col * VB;  // of a group's first row
    u32x4 kx[2][KL];         // the step's codes
    uint32_t vx[2][4][VW];
    // Groups of the shard, 64 at a time: lane i holds the place in the pool and the scales of
    // group `batch` + i (place 0 and scales 0 for one that is not there: always in the pool, of
    // no weight), and the block id of group batch + 64 + i.
    int batch = 0, next_id = -1;
    int64_t place = 0;
    float ks_l = 0.f, vs_l = 0.f;
    uint64_t absent = 0;  // groups of the batch with a bad block id
    auto load_k = [&](int h, int64_t at) __attribute__((always_inline)) {
      const uint8_t* const p = k_head + at;
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        if constexpr (PAD) {  // rows of 8-byte multiples
          u32x2 x = {0, 0}, y = {0, 0};
          if (grp * 16 + 64 * i < dn) x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p + k_at + 64 * i));
          if (grp * 16 + 64 * i + 8 < dn) y = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p + k_at + 64 * i + 8));
          kx[h][i] = u32x4{x[0], x[1], y[0], y[1]};
        } else {
          kx[h][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + k_at + 64 * i));
        }
      }
    };
    auto load_v = [&](int h, int64_t at) __attribute__((always_inline)) {
      const uint8_t* const p = v_head + at;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (VW == 2) {
          u32x2 x = {0, 0};
          if (!PAD || col * VB < dn) x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p + v_at + j * row));
          vx[h][j][0] = x[0];
          vx[h][j][1] = x[1];
        } else {
          vx[h][j][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p + v_at + j * row));
        }
      }
    };
    auto place_of = [&](int i) __attribute__((always_inline)) -> int64_t {
      return static_cast<int64_t>(
          static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(place >> 32), i))) << 32 |
          static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(place), i)));
    };
    auto scale_of = [&](float v, int i) __attribute__((always_inline)) {
      return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
    };

    int before = 0;  // groups of the shards before
    for (int s = 0; s < a.n_spans; ++s) {
      const DecodeSpan& sp = a.span[s];
      const int64_t t_beg = sp.t0, t_end = span_end(s);
      const int here = span_groups(s, t_end), g_first = static_cast<int>(t_beg / 16);
      // the run's groups of this shard, counted from the table's start
      const int lo = max(g0 - before, 0) + g_first, end = min(g1 - before, here) + g_first;
      before += here;
      if (lo >= end) continue;
      const int32_t* const table = sp.tables + static_cast<int64_t>(b) * sp.table_stride;
      auto id_of = [&](int g) __attribute__((always_inline)) {
        const int e = a.gpb_shift >= 0 ? g >> a.gpb_shift : g / a.gpb;
        return g < end && e < sp.table_len ? table[e] : -1;
      };
      auto take_batch = [&](int first) __attribute__((always_inline)) {
        batch = first;
        const int g = first + lane, blk = next_id;
        const bool in = g < end, ok = in && blk >= 0 && blk < a.num_blocks;
        const int slot = 16 * (a.gpb_shift >= 0 ? g & (a.gpb - 1) : g % a.gpb);
        place = ok ? blk * block_bytes + static_cast<int64_t>(slot) * row : 0;
        ks_l = vs_l = 0.f;
        if (ok) {
          const float* const sc = a.scales + static_cast<int64_t>(blk) * a.hkv + kvh;
          ks_l = sc[0];
          vs_l = sc[a.plane_scales];
        }
        absent = __ballot(in && !ok);
        if (in && !ok) atomicOr(a.err, 1);
        next_id = id_of(g + 64);
      };
      const int full_lo = static_cast<int>((t_beg + 15) / 16);
      const int full_end = min(end, static_cast<int>(min(t_end / 16, static_cast<int64_t>(INT32_MAX))));

      // 32 tokens: groups g, g + 1.  The next step's K takes the registers of this one's once S
      // is known, its V those of this one's at the end: loads are always under way, and none
      // stands in a branch (where it would make every wait one for all loads).
      auto step = [&](int g, auto more) __attribute__((always_inline)) {
        constexpr bool kMore = decltype(more)::value;
        const int at = g - batch;
        const float ks[2] = {scale_of(ks_l, at), scale_of(ks_l, at + 1)}, vs[2] = {scale_of(vs_l, at), scale_of(vs_l, at + 1)};
        const bool full = g >= full_lo && g + 1 < full_end && (absent >> at & 3) == 0;
        const uint64_t gone = absent >> at;
        // ---- scores: s4[h][i] is key 4 grp + i of group h ----
        f32x4 s4[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          s4[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t w[4];
            to_f16<F>(kx[h][k / 2][2 * (k % 2)], w[0], w[1]);
            to_f16<F>(kx[h][k / 2][2 * (k % 2) + 1], w[2], w[3]);
            s4[h] = mma_f16(u32x4{w[0], w[1], w[2], w[3]}, qf[k], s4[h]);
          }
        }
        int64_t next[2] = {0, 0};
        if constexpr (kMore) {
          if (g + 2 - batch >= 64) take_batch(g + 2);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            next[h] = place_of(g + 2 + h - batch);
            load_k(h, next[h]);
          }
        }
        // ---- log2 domain; keys outside the range and groups that are not there weigh nothing ----
        bool ok[2][4];
        float c[2] = {c_log2 * ks[0], c_log2 * ks[1]};  // >= 0: the maximum may come first
        if (!full) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int64_t tok = static_cast<int64_t>(g + h) * 16 + grp * 4 + i;
              ok[h][i] = g + h < end && tok >= t_beg && tok < t_end && (gone >> h & 1) == 0;
              s4[h][i] = ok[h][i] ? s4[h][i] * c[h] : -INFINITY;
            }
            c[h] = 1.f;
          }
        }
        // ---- running maxima of the scores and of weight times scale, the latter from each group's own ----
        float tmax = -INFINITY, atop = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float t = c[h] * fmaxf(fmaxf(s4[h][0], s4[h][1]), fmaxf(s4[h][2], s4[h][3]));
          tmax = fmaxf(tmax, t);
          atop = fmaxf(atop, t + __builtin_amdgcn_logf(fmaxf(vs[h], kLeastVScale)));
        }
        tmax = over_groups(tmax, [](float u, float v) { return fmaxf(u, v); });
        atop = over_groups(atop, [](float u, float v) { return fmaxf(u, v); });
        const float m_new = fmaxf(m_run, tmax), a_new = fmaxf(a_run, atop);
        l_run *= __builtin_amdgcn_exp2f(m_run - m_new);
        if (__any(a_new > a_run)) {
          const float f = __builtin_amdgcn_exp2f(a_run - a_new);
#pragma unroll
          for (int j = 0; j < VB; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] *= f;
        }
        m_run = m_new;
        a_run = a_new;
        const float f = __builtin_amdgcn_exp2f(m_new - a_new + 14.f);
        // ---- weights: hi + lo ----
        u32x4 ph, pl;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s4[h][i], c[h], -m_new));
            l_run += p;
            w[i] = p * f * vs[h];  // f * vs alone may overflow
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t u = pack_f16(w[2 * i], w[2 * i + 1]);
            const f16x2 x = __builtin_bit_cast(f16x2, u);
            ph[2 * h + i] = u;
            pl[2 * h + i] = pack_f16(__builtin_fmaf(static_cast<float>(x[0]), -1.f, w[2 * i]),
                                     __builtin_fmaf(static_cast<float>(x[1]), -1.f, w[2 * i + 1]));
          }
        }
        // ---- O^T += V^T P^T ----
        if (F == kE4M3 && !full) {  // a NaN code times a weight of 0
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int w = 0; w < VW; ++w) vx[h][i][w] = ok[h][i] ? vx[h][i][w] : 0;
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // tiles 4 w + 2 half, + 1
            uint32_t va[2][4];
#pragma unroll
            for (int p = 0; p < 4; ++p)  // keys 2 p, 2 p + 1 of the lane's eight
              to_f16<F>(__builtin_amdgcn_perm(vx[p / 2][2 * (p % 2) + 1][w], vx[p / 2][2 * (p % 2)][w], half ? 0x07030602u : 0x05010400u),
                        va[0][p], va[1][p]);
            f32x4* const o = acc + 4 * w + 2 * half;
#pragma unroll
            for (int j = 0; j < 2; ++j) o[j] = mma_f16(u32x4{va[j][0], va[j][1], va[j][2], va[j][3]}, ph, o[j]);
#pragma unroll
            for (int j = 0; j < 2; ++j) o[j] = mma_f16(u32x4{va[j][0], va[j][1], va[j][2], va[j][3]}, pl, o[j]);
          }
        if constexpr (kMore) {
#pragma unroll
          for (int h = 0; h < 2; ++h) load_v(h, next[h]);
        }
      };
      next_id = id_of(lo + lane);
      take_batch(lo);
#pragma unroll
      for (int h = 0; h < 2; ++h) load_k(h, place_of(h));
#pragma unroll
      for (int h = 0; h < 2; ++h) load_v(h, place_of(h));
      int g = lo;
      for (; g + 2 < end; g += 2) step(g, std::true_type{});
      step(g, std::false_type{});
    }

    // ---- epilogue: dims (4 grp + i) VB + j of query col are acc[j][i] ----
    const float l = over_groups(l_run, [](float u, float v) { return u + v; });
    const float inv = l == 0.f ? 0.f : 1.f / l;  // NaN stays
    const float down = __builtin_amdgcn_exp2f(a_run - m_run - 14.f);  // applied last: it may be 2^-124
    const float lse2 = l == 0.f ? -INFINITY : m_run + __log2f(l);
    // Addresses below are made from a lane number of their own: hoisted out of the loop over
    // sequences they would cost registers all the way through it.
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int col = ln & 15, grp = ln >> 4;
    // rows of the output, or of the workspace
    const bool last = a.workers == 0;
    const int64_t row0 = (last ? b : blockIdx.x + b) * static_cast<int64_t>(a.hq) + kvh * a.rep;
    void* const o_to = last ? a.out : a.ws_o;
    float* const lse_to = last ? a.lse : a.ws_lse;
    const int64_t o_rs = last ? a.out_rs : dn;
    const int o_dt = last ? a.out_dtype : kF32;
    if (a.subs == 1) {
      if (col < a.rep) {
        const int64_t r = row0 + col;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d0 = (4 * grp + i) * VB;
          float x[VB];
#pragma unroll
          for (int j = 0; j < VB; ++j) x[j] = acc[j][i] * inv * down;
          if (!PAD || d0 < dn) store_out<VB>(o_to, o_dt, r * o_rs + d0, x);
        }
        if (grp == 0 && lse_to != nullptr) lse_to[r] = lse2 * kLn2;
      }
    } else {
      // The waves of a kv head meet in LDS; wave `sub` finishes its query heads sub, sub + subs, ...
      float* const o_lds = meet_lds;
      float* const lse_lds = meet_lds + a.heads * a.subs * a.rep * OS;
      if (col < a.rep) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < VB; j += 4)
            *reinterpret_cast<float4*>(o_lds + (wave * a.rep + col) * OS + (4 * grp + i) * VB + j) =
                make_float4(acc[j][i] * inv * down, acc[j + 1][i] * inv * down, acc[j + 2][i] * inv * down, acc[j + 3][i] * inv * down);
        if (grp == 0) lse_lds[wave * 16 + col] = lse2;
      }
      __syncthreads();
      const int w0 = wave - sub * a.heads;
      for (int c = sub; c < a.rep; c += a.subs) {
        float m = -INFINITY;
        for (int i = 0; i < a.subs; ++i) m = fmaxf(m, lse_lds[(w0 + i * a.heads) * 16 + c]);
        const float ref = m == -INFINITY ? 0.f : m;  // no finite one: 0, or NaN with a NaN one
        float o[D / 64] = {}, den = 0.f;
        for (int i = 0; i < a.subs; ++i) {
          const int w = w0 + i * a.heads;
          const float f = __builtin_amdgcn_exp2f(lse_lds[w * 16 + c] - ref);
          den += f;
#pragma unroll
          for (int k = 0; k < D / 64; ++k) o[k] += f * o_lds[(w * a.rep + c) * OS + ln + 64 * k];
        }
        const float inv_den = den == 0.f ? 0.f : 1.f / den;
        const int64_t r = row0 + c;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
          const int d0 = ln + 64 * k;
          if (!PAD || d0 < dn) store_elem_rt(o_to, o_dt, r * o_rs + d0, o[k] * inv_den);
        }
        if (ln == 0 && lse_to != nullptr) lse_to[r] = den == 0.f ? -INFINITY : (ref + __log2f(den)) * kLn2;
      }
    }
    if (left == 0) return;
    if (a.subs > 1) __syncthreads();  // LDS is read
    do {  // the next sequence that holds tokens
      if (++b >= a.batch) return;
      total = seq_groups();
    } while (total == 0);
    begin = 0;
    end_all = min(left, (total + 1) & ~1);
    left -= end_all;
  }
}

// Merge of a sequence's neighbouring places, one (sequence, query head) per workgroup:
// 256 / lpr slots take every so-manieth place with kU loads in flight each, and meet in LDS.
template <int OUT_DT>
__global__ __launch_bounds__(256) void kv8_join_kernel(const float* ws_o, const float* ws_lse, const int2* range, int hq, int dn,
                                                       int lpr, void* out, int64_t out_rs, float* lse) {
  constexpr int kU = 4;
  __shared__ float4 acc_l[256];
  __shared__ float m_l[256], den_l[256];
  const int h = blockIdx.x, b = blockIdx.y;
  const int2 where = range[b];
  const int slots = 256 / lpr, slot = threadIdx.x / lpr, c = threadIdx.x % lpr * 4;
  const bool active = c < dn;
  float m = -INFINITY, den = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = slot; base < where.y; base += kU * slots) {
    float l[kU];
    float4 v[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = base + u * slots;
      const int64_t r = static_cast<int64_t>(where.x + i) * hq + h;
      l[u] = i < where.y ? ws_lse[r] : -INFINITY;
      v[u] = i < where.y && active ? *reinterpret_cast<const float4*>(ws_o + r * dn + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < kU; ++u) mn = fmaxf(mn, l[u]);
    const float ref = mn == -INFINITY ? 0.f : mn;  // all empty so far: they add 0, a NaN stays
    const float sc = __expf(m - ref);
    den *= sc;
    acc.x *= sc; acc.y *= sc; acc.z *= sc; acc.w *= sc;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const float w = __expf(l[u] - ref);
      den += w;
      acc.x += w * v[u].x; acc.y += w * v[u].y; acc.z += w * v[u].z; acc.w += w * v[u].w;
    }
    m = mn;
  }
  acc_l[threadIdx.x] = acc;
  m_l[threadIdx.x] = m;
  den_l[threadIdx.x] = den;
  __syncthreads();
  if (slot != 0) return;
  const int used = max(min(slots, where.y), 1);
  float mt = -INFINITY;
  for (int s = 0; s < used; ++s) mt = fmaxf(mt, m_l[threadIdx.x + s * lpr]);
  const float ref = mt == -INFINITY ? 0.f : mt;
  float dt = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < used; ++s) {
    const float ms = m_l[threadIdx.x + s * lpr];
    const float w = ms == -INFINITY ? 1.f : __expf(ms - ref);  // no finite place: its sum is 0 or NaN as it stands
    const float4 x = acc_l[threadIdx.x + s * lpr];
    dt += w * den_l[threadIdx.x + s * lpr];
    o.x += w * x.x; o.y += w * x.y; o.z += w * x.z; o.w += w * x.w;
  }
  const float inv = dt == 0.f ? 0.f : 1.f / dt;
  const float x[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  const int64_t r = static_cast<int64_t>(b) * hq + h;
  if (active) store_out<4>(out, OUT_DT, r * out_rs + c, x);
  if (lse != nullptr && threadIdx.x == 0) lse[r] = dt == 0.f ? -INFINITY : ref + __logf(dt);
}

struct Kv8Plan {
  int workers, heads, subs, min_len;  // workers 0: direct
};

// Waves that take a head's share alone, of all sequences: one for every step while that is at
// most two a SIMD, so that no worker crosses a sequence's end (2.5-4 us each time: lengths,
// table, q and the first codes one after another), else one a SIMD -- it reaches 6.1 TB/s, more
// of them no more.
static int64_t lone_workers(int batch, int hkv, int64_t steps) {
  const int64_t cus = device_cus();
  return batch * steps * hkv <= 8 * cus ? batch * steps : std::max<int64_t>(4 * cus / hkv, 1);
}

// Direct or balanced, by modelled time (us, fitted on MI355X).  Over 38 calls (1-2000 sequences of
// 64-100000 tokens, 1 to 12 kv heads of 128, 64 and 96 dims) what it takes is 1.4% in the mean behind
// the fastest of up to 75 splits tried, 16% at most (one sequence of 32000 tokens, 16/2 heads, below):
//   direct:   6 + the longest sequence's steps over four waves, 0.95 each, times the workgroups a
//             CU has, or the bytes at 6 TB/s -- of sequences as long as the longest, as long as a
//             CU has no more than two; past that the lengths even out.
//   balanced: 11 (the join is a launch of its own) + its waves' steps, or three quarters of those
//             bytes (lengths between half the longest and the longest, as a serving batch's), +
//             2.5 for every sequence that a worker meets.
// e.g. 4 x 700 tokens, 32/8 heads: 9.9 direct, 10.7 balanced; 64 x 1000: 26.3 / 29.1; 64 x 2000:
// 50.0 / 45.2; 64 x 16384: 362 / 267; 6 x 2085, 16/2 heads: 19.2 / 12.0; 200 x 500, 14/2 heads of 64
// dims: 10.1 / 21.0.  A direct workgroup is one kv head and four waves, one a SIMD: eight take as
// long (4 x 700: 10.3), two longer (14.4).
static Kv8Plan plan_kv8(int batch, int hq, int hkv, int d, int n, const DecodeSpan* spans) {
  const int64_t groups = span_groups(n, spans), steps = ceil_div(groups, 2);
  const int most = kv8_waves(d != 128 && d != 64);
  const Kv8Plan direct{0, 1, static_cast<int>(std::min<int64_t>(4, steps)), 0};
  // the lanes that lay out the row count groups in 32 bits and take 64 sequences at a time
  if (batch > 1024 || batch * (groups + 1) > INT32_MAX / 2 || steps <= 4) return direct;
  const int64_t lone = lone_workers(batch, hkv, steps);
  const double cus = device_cus(), all = static_cast<double>(batch) * hkv * steps;  // steps of a wave
  const double bytes = all * 64 * d / 6e6, per_cu = batch * hkv / cus;
  const double run = std::max(all / (static_cast<double>(lone) * hkv), all / (4 * cus));
  const double t_direct = 6.0 + std::max(bytes * (0.75 + 0.25 * std::min(1.0, 2.0 / per_cu)), 0.95 * steps / 4 * std::max(1.0, per_cu));
  const double t_balanced = 11.0 + std::max(0.75 * bytes, 0.95 * run) + (run > 1.0 ? 2.5 * (1.0 + static_cast<double>(batch) / lone) : 0.0);
  if (t_direct <= t_balanced) return direct;
  // Up to 100 places a sequence and head for the join, 200 where runs are long: else waves of a
  // workgroup meet first, four at least (one sequence of 4096 tokens, 32/8 heads: 11.3 us as 32
  // workers of four waves a head, 13.3 as 128 lone ones or as 64 of two; of 100000: 53.3 as 32 of
  // four, 44.4 lone).  Where the rule loses: 32000 tokens, 16/2 heads, 17.4 us as 63 workers of 16
  // waves, 15.1 as 128 of four; it is as fast at 16000 (13.6, 14.2).
  // Lone waves of four heads share a workgroup (1% faster, they read whole rows), never those of
  // two: workgroups of two waves leave half of the SIMDs without one (64 x 16384 tokens, 14/2
  // heads of 64 dims: 63.4 us, single waves 52.5).
  int subs = 1;
  const int64_t places = (run < 16.0 ? 100 : 200) * static_cast<int64_t>(batch);
  if (lone > places)
    for (subs = 4; subs < most && lone > places * subs;) subs *= 2;
  const int heads = subs == 1 && hkv % 4 == 0 ? 4 : 1;
  return Kv8Plan{static_cast<int>(ceil_div(lone, subs)), heads, subs, 2 * subs};
}

static size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }
static size_t workers_bytes(int64_t workers, int batch, int hq, int d) {
  const size_t rows = static_cast<size_t>(workers + batch) * hq;
  return align256(rows * d * sizeof(float)) + align256(rows * sizeof(float)) + align256(sizeof(int2) * batch);
}

// Covers these spans and any shorter ones.
size_t kv8_decode_workspace_bytes(int batch, int hq, int hkv, int d, int n, const DecodeSpan* spans) {
  const int64_t steps = ceil_div(span_groups(n, spans), 2), cus = device_cus();
  return workers_bytes(std::min<int64_t>(batch * steps, std::max<int64_t>(8 * cus / hkv, 1)), batch, hq, d);
}

template <int F, int D, bool PAD>
static void launch_kv8_typed(const Kv8DecodeArgs& a, dim3 grid, hipStream_t stream) {
  const int waves = a.heads * a.subs;
  const size_t lds = a.subs > 1 ? sizeof(float) * waves * (static_cast<size_t>(a.rep) * (D + 4) + 16) : 0;
  kv8_decode_kernel<F, D, PAD><<<grid, 64 * waves, lds, stream>>>(a);
}

void launch_kv8_decode(const Kv8Pool& pool, int dtype, int batch, int hq, const void* q, int64_t q_bs, int64_t q_hs, int n,
                       const DecodeSpan* spans, float scale, int out_dtype, void* out, int64_t out_rs, float* lse, void* ws,
                       size_t ws_bytes, int* err, hipStream_t stream) {
  const int hkv = pool.hkv, d = pool.d;
  require(batch <= 65535, "kv8_decode: batch must be at most 65535");  // grid y
  require(16ll * hkv * d < (1ll << 31), "kv8_decode: too many heads");   // 32-bit offsets in a group
  for (int i = 0; i < n; ++i) require(spans[i].t0 >= 0 && spans[i].t0 < pool.bs, "kv8_decode: a span starts in its first block");
  require(span_groups(n, spans) <= INT32_MAX / 4, "kv8_decode: too many tokens");  // a sequence's groups are counted in 32 bits
  const Kv8Plan p = plan_kv8(batch, hq, hkv, d, n, spans);
  require(hkv % p.heads == 0, "kv8_decode: a workgroup's heads divide the kv heads");
  Kv8DecodeArgs a;
  a.ws_o = a.ws_lse = nullptr;
  a.range = nullptr;
  if (p.workers > 0) {
    const size_t rows = static_cast<size_t>(p.workers + batch) * hq;
    const size_t need = workers_bytes(p.workers, batch, hq, d);
    if (ws == nullptr || ws_bytes < need) throw Error(-6, "workspace too small: need " + std::to_string(need) + " bytes");
    require(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "workspace must be 16-byte aligned");
    char* at = static_cast<char*>(ws);
    a.ws_o = reinterpret_cast<float*>(at);
    at += align256(rows * d * sizeof(float));
    a.ws_lse = reinterpret_cast<float*>(at);
    at += align256(rows * sizeof(float));
    a.range = reinterpret_cast<int2*>(at);
  }
  a.workers = p.workers;
  a.min_len = p.min_len;
  a.q = static_cast<const uint16_t*>(q);
  a.q_bs = q_bs;
  a.q_hs = q_hs;
  a.pool = pool.codes;
  a.scales = pool.scales;
  a.plane_bytes = pool.num_blocks * pool.bs * hkv * static_cast<int64_t>(d);
  a.plane_scales = pool.num_blocks * hkv;
  a.num_blocks = pool.num_blocks;
  a.bs = pool.bs;
  a.hkv = hkv;
  a.hq = hq;
  a.rep = hq / hkv;
  a.n_spans = n;
  for (int i = 0; i < n; ++i) a.span[i] = spans[i];
  a.heads = p.heads;
  a.subs = p.subs;
  a.gpb = pool.bs / 16;
  a.gpb_shift = (a.gpb & (a.gpb - 1)) == 0 ? __builtin_ctz(a.gpb) : -1;
  a.q_bf16 = dtype == kBF16;
  a.out_dtype = out_dtype;
  a.dn = d;
  a.scale_log2 = scale * kLog2e;
  a.out = out;
  a.out_rs = out_rs;
  a.lse = lse;
  a.batch = batch;
  a.err = err;
  const dim3 grid(std::max(p.workers, 1), p.workers > 0 ? 1 : batch, static_cast<unsigned>(hkv / p.heads));
  // head dim 64: its own kernel; other multiples of 8 up to 128: 128 with the dims past it zero
  if (pool.format == kE4M3) {
    if (d == 128) launch_kv8_typed<kE4M3, 128, false>(a, grid, stream);
    else if (d == 64) launch_kv8_typed<kE4M3, 64, false>(a, grid, stream);
    else launch_kv8_typed<kE4M3, 128, true>(a, grid, stream);
  } else {
    if (d == 128) launch_kv8_typed<kInt8, 128, false>(a, grid, stream);
    else if (d == 64) launch_kv8_typed<kInt8, 64, false>(a, grid, stream);
    else launch_kv8_typed<kInt8, 128, true>(a, grid, stream);
  }
  HCP_HIP(hipGetLastError());
  if (p.workers == 0) return;
  int lpr = 1;
  while (lpr * 4 < d) lpr *= 2;
  const dim3 rows(hq, batch);
  switch (out_dtype) {
    case kBF16: kv8_join_kernel<kBF16><<<rows, 256, 0, stream>>>(a.ws_o, a.ws_lse, a.range, hq, d, lpr, out, out_rs, lse); break;
    case kF16: kv8_join_kernel<kF16><<<rows, 256, 0, stream>>>(a.ws_o, a.ws_lse, a.range, hq, d, lpr, out, out_rs, lse); break;
    default: kv8_join_kernel<kF32><<<rows, 256, 0, stream>>>(a.ws_o, a.ws_lse, a.range, hq, d, lpr, out, out_rs, lse); break;
  }
  HCP_HIP(hipGetLastError());
}

}  // namespace hcp
