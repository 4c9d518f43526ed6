// Rows into and out of the 8-bit paged cache (layout in kv8.hpp).
//
// Append: the tokens of a step go to the slots of a slot map.  A run is a stretch of tokens
// whose slots follow each other inside one block; it starts at slot `a`, so rows < a of the
// block are held already.  Per plane and head
//   s' = max(s, need) if a > 0, need otherwise;  need = the least power of two that holds
//   the run's largest magnitude;  new codes = rne(x / s');  where s' > s the held codes
//   become rne(c * s / s').  Products with the fp32 factors 1 / s' and s / s' stand for both:
//   exact where the scales are powers of two, else within 2^-23, which is seen next to a tie only
//   (divisions corrected to odd cost grown blocks 11% and prompts 2-6%, for no nearer code).
// One wave has one run of one head and plane: it alone reads and writes that scale and those
// rows, so nothing is shared and no result depends on an order.  A value that is not finite
// makes the scale NaN (every score and output row that meets the block is then NaN, in both
// formats, though only e4m3 has a NaN code).
//
// Gather: out = scale * code, rounded to the output type (exact in bf16 and fp16 where the
// scale is a power of two within the type's range).
//
// Both are bound by HBM where the tokens are many, else by the latency of a launch and two
// loads in line (slot, then row and scale).  32768 tokens of 8 heads of 128, bf16, blocks of 16:
// append 46 us (202 MB, 4.4 TB/s), gather 39.5 us (201 MB, 5.1 TB/s), the bytes of both read and
// written once by the counters; a 2 GiB copy 4.8-4.9 TB/s.  64 tokens 4.1 us, 1027 (2 heads of 64,
// gather) 3.6 us.
#include <algorithm>
#include <type_traits>

#include "kv8.hpp"

namespace hcp {

// Largest magnitude over the n lanes of a group, as the bits of |x| (NaN above infinity above finite).
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int n) {
  for (int off = n / 2; off > 0; off /= 2) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), off)));
  return v;
}
__device__ __forceinline__ uint32_t top_of(const float* x, uint32_t top) {
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  return top;
}

// A block's scale after a run whose largest magnitude is `top` (bits), `old` held rows' (0: none).
struct BlockScale {
  float s;   // what divides
  bool bad;  // a value that is not finite: the scale is NaN, codes 0
};
template <int F>
__device__ __forceinline__ BlockScale block_scale(uint32_t top, float old) {
  const bool bad = top >= 0x7f800000u || !(old >= 0.f && old < INFINITY);
  return BlockScale{fmaxf(old, kv8_scale<F>(__uint_as_float(bad ? 0u : top))), bad};
}
template <int F>
__device__ __forceinline__ void put_codes(uint8_t* at, const float* x, float inv, bool bad) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = bad ? 0.f : x[i] * inv;
  *reinterpret_cast<u32x2*>(at) = u32x2{kv8_encode4<F>(y[0], y[1], y[2], y[3]), kv8_encode4<F>(y[4], y[5], y[6], y[7])};
}
// Codes of the held rows from, from + step, ... to a scale grown by 1 / f, eight of them under way (the
// 63 before a token of 64 sequences, 8 heads of 128: 8.3 us, one after another 13.7).
template <int F>
__device__ __forceinline__ void scale_rows(uint8_t* at, int64_t row, int from, int to, int step, float f) {
  constexpr int kU = 8;
  for (int r0 = from; r0 < to; r0 += kU * step) {
    u32x2 w[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (r0 + u * step < to) w[u] = *reinterpret_cast<const u32x2*>(at + (r0 + u * step) * row);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (r0 + u * step >= to) continue;
      float y[8];
      kv8_decode4<F>(w[u][0], y);
      kv8_decode4<F>(w[u][1], y + 4);
      put_codes<F>(at + (r0 + u * step) * row, y, f, false);
    }
  }
}

// One run of n tokens (rows tok0 .. of the view) into slots a .. a + n of block blk, by a wave.
// A pass is 64 chunks of 8 values; KEEP passes stay in registers from the maximum to the codes
// (4: a block of 16 tokens of 128 dims; 16: of 64), later ones are read again, from the L2.  Four
// passes at a time, so that a short run in a long block does not go through all of them (4 tokens
// of 64 sequences, blocks of 64: 7.3 us, 9.7 with sixteen passes each).
template <int F, int DT, bool VEC, int KEEP>
__device__ __forceinline__ void append_run(const Kv8Append& p, int plane, int head, int64_t blk, int a, int n, int64_t tok0) {
  const int lane = threadIdx.x & 63;
  const int lpr = p.lanes_per_row, rpp = 64 / lpr;  // lanes per row, rows per pass
  const int c = lane % lpr * 8, r0 = lane / lpr;
  const bool in = c < p.d;
  const void* src = p.src[plane];
  const int64_t ss = p.ss[plane], src0 = head * p.hs[plane] + tok0 * ss + c;
  float* const scale_at = p.scales + (plane * p.num_blocks + blk) * p.hkv + head;
  const float old = a > 0 ? *scale_at : 0.f;
  uint8_t* const dst = p.pool + ((plane * p.num_blocks + blk) * p.bs * p.hkv + head) * p.d + c;
  const int64_t row = static_cast<int64_t>(p.hkv) * p.d;
  uint32_t top = 0;
  Row8<DT, VEC> x[KEEP];
#pragma unroll
  for (int k0 = 0; k0 < KEEP; k0 += 4) {
    if (k0 * rpp >= n) break;
#pragma unroll
    for (int k = k0; k < k0 + 4; ++k) {
      const int r = r0 + k * rpp;
      if (in && r < n) x[k].load(src, src0 + r * ss);
      else x[k].clear();
    }
  }
  float y[8];
#pragma unroll
  for (int k0 = 0; k0 < KEEP; k0 += 4) {
    if (k0 * rpp >= n) break;
#pragma unroll
    for (int k = k0; k < k0 + 4; ++k) {
      x[k].get(y);
      top = top_of(y, top);
    }
  }
  for (int r = r0 + KEEP * rpp; r < n; r += rpp)
    if (in) {
      Row8<DT, VEC> z;
      z.load(src, src0 + r * ss);
      z.get(y);
      top = top_of(y, top);
    }
  const BlockScale b = block_scale<F>(lanes_max(top, 64), old);
  if (lane == 0) *scale_at = b.bad ? __uint_as_float(0x7fc00000u) : b.s;
  const float inv = 1.f / b.s;
#pragma unroll
  for (int k0 = 0; k0 < KEEP; k0 += 4) {
    if (k0 * rpp >= n) break;
#pragma unroll
    for (int k = k0; k < k0 + 4; ++k)
      if (in && r0 + k * rpp < n) {
        x[k].get(y);
        put_codes<F>(dst + (a + r0 + k * rpp) * row, y, inv, b.bad);
      }
  }
  for (int r = r0 + KEEP * rpp; r < n; r += rpp)
    if (in) {
      Row8<DT, VEC> z;
      z.load(src, src0 + r * ss);
      z.get(y);
      put_codes<F>(dst + (a + r) * row, y, inv, b.bad);
    }
  if (b.bad || b.s == old || a == 0) return;
  if (in) scale_rows<F>(dst, row, r0, a, rpp, old / b.s);
}

// Block of a slot: a shift where bs is a power of two (a 64-bit division takes some 150
// instructions: 1000 decode tokens, 32/8 heads, 11.7 us with three of them a wave).
__device__ __forceinline__ int64_t block_of(const Kv8Append& p, int64_t slot) {
  return p.bs_shift >= 0 ? slot >> p.bs_shift : slot / p.bs;
}

// N runs of one token (a decode step's), by the lanes_per_row lanes of a group: 64 / lpr
// heads and planes a wave, where a wave for each would have most of its lanes idle, and the N
// runs' rows and scales under way together.  slot[u] < 0: none.
template <int F, int DT, bool VEC, int N>
__device__ __forceinline__ void append_singles(const Kv8Append& p, int plane, int head, const int64_t* slot, const int64_t* tok) {
  const int lpr = p.lanes_per_row, c = (threadIdx.x & 63) % lpr * 8;
  const int64_t row = static_cast<int64_t>(p.hkv) * p.d;
  Row8<DT, VEC> x[N];
  float old[N];
  float* scale_at[N];
  uint8_t* block[N];
  int a[N];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int64_t blk = slot[u] < 0 ? 0 : block_of(p, slot[u]);
    a[u] = slot[u] < 0 ? -1 : static_cast<int>(slot[u] - blk * p.bs);
    scale_at[u] = p.scales + (plane * p.num_blocks + blk) * p.hkv + head;
    block[u] = p.pool + ((plane * p.num_blocks + blk) * p.bs * p.hkv + head) * p.d + c;
    old[u] = a[u] > 0 ? *scale_at[u] : 0.f;
    if (c < p.d && a[u] >= 0) x[u].load(p.src[plane], head * p.hs[plane] + tok[u] * p.ss[plane] + c);
    else x[u].clear();
  }
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float y[8];
    x[u].get(y);
    const BlockScale b = block_scale<F>(lanes_max(top_of(y, 0), lpr), old[u]);
    if (a[u] < 0) continue;
    if (c == 0) *scale_at[u] = b.bad ? __uint_as_float(0x7fc00000u) : b.s;
    if (c >= p.d) continue;
    put_codes<F>(block[u] + a[u] * row, y, 1.f / b.s, b.bad);
    if (b.bad || b.s == old[u]) continue;
    scale_rows<F>(block[u], row, 0, a[u], 1, old[u] / b.s);
  }
}

// One wave per window of tokens, head and plane; it has the runs that begin in the window, those of
// one token for as many heads and planes of its workgroup as it has groups of lanes.
template <int F, int DT, bool VEC, int KEEP>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8Append p) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), task = blockIdx.y * 4 + wave;
  if (task >= 2 * p.hkv) return;
  const int lane = threadIdx.x & 63;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.window;
  // lane i: does token first + i begin a run, and of more than itself?
  bool begins = false, longer = false;
  const int64_t t = first + lane;
  int64_t slot = -1;
  if (lane < p.window && t < p.tokens) {
    slot = p.slots[t];
    const int64_t before = t > 0 ? p.slots[t - 1] : -2, after = t + 1 < p.tokens ? p.slots[t + 1] : -2;
    const int64_t blk = block_of(p, slot);
    begins = slot >= 0 && (before != slot - 1 || blk * p.bs == slot);
    longer = after == slot + 1 && after != (blk + 1) * p.bs;
    if (begins && blk >= p.num_blocks) {
      begins = false;
      if (task == 0) atomicOr(p.err, 1);
    }
  }
  auto slot_at = [&](int i) __attribute__((always_inline)) {
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(slot >> 32), i))) << 32 |
                                static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(slot), i)));
  };
  uint64_t singles = __ballot(begins && !longer), runs = __ballot(begins && longer);
  const int groups = min(64 / p.lanes_per_row, 4), mine = task + lane / p.lanes_per_row;
  const bool lanes_used = lane / p.lanes_per_row < groups && mine < 2 * p.hkv;
  if (wave % groups != 0) singles = 0;
  if (singles != 0 && (singles & (singles - 1)) == 0) {
    const int i = __builtin_ctzll(singles);
    const int64_t at[1] = {slot_at(i)}, tok[1] = {first + i};
    if (lanes_used) append_singles<F, DT, VEC, 1>(p, mine / p.hkv, mine % p.hkv, at, tok);
    singles = 0;
  }
  while (singles != 0) {
    int64_t at[4], tok[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      at[u] = -1;
      tok[u] = 0;
      if (singles == 0) continue;
      const int i = __builtin_ctzll(singles);
      singles &= singles - 1;
      at[u] = slot_at(i);
      tok[u] = first + i;
    }
    if (lanes_used) append_singles<F, DT, VEC, 4>(p, mine / p.hkv, mine % p.hkv, at, tok);
  }
  for (; runs != 0; runs &= runs - 1) {
    const int i0 = __builtin_ctzll(runs);
    const int64_t t0 = first + i0, s0 = slot_at(i0), blk = block_of(p, s0);
    const int a = static_cast<int>(s0 - blk * p.bs);
    int n = 1;
    for (;;) {  // 64 followers at a time
      const int64_t i = t0 + n + lane;
      const bool follows = a + n + lane < p.bs && i < p.tokens && p.slots[i] == s0 + n + lane;
      const uint64_t stop = __ballot(!follows);
      n += stop == 0 ? 64 : __builtin_ctzll(stop);
      if (stop != 0) break;
    }
    append_run<F, DT, VEC, KEEP>(p, task / p.hkv, task % p.hkv, blk, a, n, t0);
  }
}

template <int F, int DT>
static void append_typed(const Kv8Append& p, bool vec, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(ceil_div(p.tokens, p.window)), static_cast<unsigned>(ceil_div(2 * p.hkv, 4)));
  const bool large = static_cast<int64_t>(p.bs) * p.lanes_per_row > 4 * 64;  // a block is more than four passes
  if (vec && large) kv8_append_kernel<F, DT, true, 16><<<grid, 256, 0, stream>>>(p);
  else if (vec) kv8_append_kernel<F, DT, true, 4><<<grid, 256, 0, stream>>>(p);
  else kv8_append_kernel<F, DT, false, 4><<<grid, 256, 0, stream>>>(p);
}

// 8-element chunks of every row start on a 16-byte boundary.
static bool rows_aligned(const void* p, int64_t hs, int64_t ss, int es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && hs * es % 16 == 0 && ss * es % 16 == 0;
}

static int lanes_for(int d) {
  int l = 1;
  while (l * 8 < d) l *= 2;
  return l;
}

void launch_kv8_append(int format, int dtype, Kv8Append p, hipStream_t stream) {
  if (p.tokens == 0) return;
  require(p.tokens < (1ll << 32) / 256, "kv8_append: too many tokens");  // threads of a launch
  const int es = dtype == kF32 ? 4 : 2;
  const bool vec = rows_aligned(p.src[0], p.hs[0], p.ss[0], es) && rows_aligned(p.src[1], p.hs[1], p.ss[1], es);
  p.lanes_per_row = lanes_for(p.d);
  p.bs_shift = (p.bs & (p.bs - 1)) == 0 ? __builtin_ctz(p.bs) : -1;
  // The smallest window that leaves at most 4096 waves, 16 at most: most waves of a prompt find that
  // no run begins at their token, and a wave goes through its window's runs in turn.  bf16, 8 heads of
  // 128, us at a window of 1 / 4 / 16: a prompt of 500 tokens 7.6 / 4.8 / 5.5, of 1000 16.6 / 5.9 / 5.7,
  // of 4000 63 / 21 / 8.6; tokens of 64 sequences 4.3 / 6.5 / 17, of 1000 9.2 / 7.6 / 17.
  p.window = 1;
  while (p.window < 16 && p.tokens * 2 * p.hkv > 4096ll * p.window) p.window *= 2;
  auto typed = [&](auto f) {
    constexpr int F = decltype(f)::value;
    if (dtype == kBF16) append_typed<F, kBF16>(p, vec, stream);
    else if (dtype == kF16) append_typed<F, kF16>(p, vec, stream);
    else append_typed<F, kF32>(p, vec, stream);
  };
  if (format == kE4M3) typed(std::integral_constant<int, kE4M3>{});
  else typed(std::integral_constant<int, kInt8>{});
  HCP_HIP(hipGetLastError());
}

// One wave per 16 consecutive slots of a table entry, head and plane: its block id and scale
// are read once, all its codes are under way before the first row is written.
constexpr int kRows = 16;
template <int F, int DT, bool VEC>
__global__ __launch_bounds__(256) void kv8_gather_kernel(Kv8Gather p) {
  const int task = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (task >= 2 * p.hkv) return;
  const int plane = task / p.hkv, head = task - plane * p.hkv;
  int ri = 0;
  while (ri + 1 < p.n && static_cast<int>(blockIdx.x) >= p.begin[ri + 1]) ++ri;
  const Kv8Range& R = p.r[ri];
  const int item = blockIdx.x - p.begin[ri];
  const int e = item / p.per_block, part = item - e * p.per_block;
  const int64_t entry = R.entry0 + e;
  const int32_t blk = R.table[entry];
  if (blk < 0 || blk >= p.num_blocks) {
    if (threadIdx.x == 0 && blockIdx.y == 0 && part == 0) atomicOr(p.err, 1);
    return;
  }
  const int64_t block = plane * p.num_blocks + blk;
  const float s = p.scales[block * p.hkv + head];
  const int lane = threadIdx.x & 63, lpr = p.lanes_per_row, rpp = 64 / lpr;
  const int c = lane % lpr * 8;
  if (c >= p.d) return;
  const int64_t row = static_cast<int64_t>(p.hkv) * p.d;
  const uint8_t* const src = p.pool + (block * p.bs * p.hkv + head) * p.d + c;
  void* const dst = plane ? R.v : R.k;
  const int64_t tok0 = entry * p.bs - R.at0;  // of the range, at slot 0
  const int end = min(p.bs, (part + 1) * kRows);
  constexpr int kU = 4;  // loads in flight: all of a 16-row item of 128 dims
  for (int r0 = part * kRows + lane / lpr; r0 < end; r0 += kU * rpp) {
    u32x2 w[kU];
#pragma unroll
    for (int k = 0; k < kU; ++k)
      if (r0 + k * rpp < end) w[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(src + (r0 + k * rpp) * row));
#pragma unroll
    for (int k = 0; k < kU; ++k) {
      const int64_t t = tok0 + r0 + k * rpp;
      if (r0 + k * rpp >= end || t < 0 || t >= R.tokens) continue;
      float x[8];
      kv8_decode4<F>(w[k][0], x);
      kv8_decode4<F>(w[k][1], x + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= s;
      store8<DT, VEC>(dst, head * R.hs + t * R.ss + c, x);
    }
  }
}

template <int F, int DT>
static void gather_typed(const Kv8Gather& p, bool vec, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.begin[p.n]), static_cast<unsigned>(ceil_div(2 * p.hkv, 4)));
  if (vec) kv8_gather_kernel<F, DT, true><<<grid, 256, 0, stream>>>(p);
  else kv8_gather_kernel<F, DT, false><<<grid, 256, 0, stream>>>(p);
}

void launch_kv8_gather(const Kv8Pool& pool, int dtype, int n, const PagedRangeDesc* ranges, int* err, hipStream_t stream) {
  const int es = dtype == kF32 ? 4 : 2;
  for (int next = 0; next < n;) {
    Kv8Gather p;
    p.pool = pool.codes;
    p.scales = pool.scales;
    p.num_blocks = pool.num_blocks;
    p.bs = pool.bs;
    p.hkv = pool.hkv;
    p.d = pool.d;
    p.lanes_per_row = lanes_for(pool.d);
    p.err = err;
    p.per_block = static_cast<int32_t>(ceil_div(pool.bs, kRows));
    p.n = 0;
    int64_t items = 0;
    bool vec = true;
    for (; next < n && p.n < kKv8Ranges; ++next) {
      const PagedRangeDesc& d = ranges[next];
      if (d.t1 <= d.t0) continue;
      const int64_t at0 = d.t0 - d.table_seq_offset, last = (d.t1 - 1 - d.table_seq_offset) / pool.bs;
      p.begin[p.n] = static_cast<int32_t>(items);
      items += (last - at0 / pool.bs + 1) * p.per_block;
      require(items < (1 << 24), "kv8_gather: too many tokens");  // threads of a launch: 2^32
      p.r[p.n++] = Kv8Range{d.table, at0 / pool.bs, at0, d.t1 - d.t0, d.k_buf, d.v_buf, d.head_stride, d.seq_stride};
      vec = vec && rows_aligned(d.k_buf, d.head_stride, d.seq_stride, es) && rows_aligned(d.v_buf, d.head_stride, d.seq_stride, es);
    }
    if (p.n == 0) continue;
    p.begin[p.n] = static_cast<int32_t>(items);
    auto typed = [&](auto f) {
      constexpr int F = decltype(f)::value;
      if (dtype == kBF16) gather_typed<F, kBF16>(p, vec, stream);
      else if (dtype == kF16) gather_typed<F, kF16>(p, vec, stream);
      else gather_typed<F, kF32>(p, vec, stream);
    };
    if (pool.format == kE4M3) typed(std::integral_constant<int, kE4M3>{});
    else typed(std::integral_constant<int, kInt8>{});
    HCP_HIP(hipGetLastError());
  }
}

}  // namespace hcp
