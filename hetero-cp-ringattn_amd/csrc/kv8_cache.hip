// Rows into and out of the 8-bit paged cache (layout in kv8.hpp).
//
// Append: the tokens of a step go to the slots of a slot map.  A run is a stretch of tokens
// whose slots follow each other inside one block; it starts at slot `a`, so rows < a of the
// block are held already.  Per plane and head
//   s' = max(s, need) if a > 0, need otherwise;  need = the least power of two that holds
//   the run's largest magnitude;  new codes = rne(x / s');  where s' > s the held codes
//   become rne(c * s / s').
// One wave has one run of one head and plane: it alone reads and writes that scale and those
// rows, so nothing is shared and no result depends on an order.  A value that is not finite
// makes the scale NaN (every score and output row that meets the block is then NaN, in both
// formats, though only e4m3 has a NaN code).
//
// Gather: out = scale * code, rounded to the output type (exact in bf16 and fp16 where the
// scale is a power of two within the type's range).
#include <algorithm>
#include <type_traits>

#include "kv8.hpp"

namespace hcp {

// Largest magnitude over the wave, as the bits of |x| (NaN above infinity above finite).
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  for (int off = 32; off > 0; off /= 2) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), off)));
  return v;
}

// One run of n tokens (rows tok0 .. of the view) into slots a .. a + n of block blk.  A pass
// is 64 chunks of 8 values; kKeep passes stay in registers from the maximum to the codes
// (a block of 16 tokens of 128 dims: 4), later ones are read again, from the L2.
constexpr int kKeep = 4;
template <int F, int DT, bool VEC>
__device__ void append_run(const Kv8Append& p, int plane, int head, int64_t blk, int a, int n, int64_t tok0) {
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
  float x[kKeep][8];
#pragma unroll
  for (int k = 0; k < kKeep; ++k) {
    const int r = r0 + k * rpp;
    if (in && r < n) load8<DT, VEC>(src, src0 + r * ss, x[k]);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k][i] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < kKeep; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[k][i]) & 0x7fffffffu);
  for (int r = r0 + kKeep * rpp; r < n; r += rpp)
    if (in) {
      float y[8];
      load8<DT, VEC>(src, src0 + r * ss, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
    }
  top = wave_max(top);
  const bool bad = top >= 0x7f800000u || !(old >= 0.f && old < INFINITY);
  const float need = kv8_scale<F>(__uint_as_float(bad ? 0u : top));
  const float s = fmaxf(old, need);
  if (lane == 0) *scale_at = bad ? __uint_as_float(0x7fc00000u) : s;
  const float inv = 1.f / s;
  auto put = [&](int r, const float* v) __attribute__((always_inline)) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = bad ? 0.f : v[i] * inv;
    *reinterpret_cast<u32x2*>(dst + (a + r) * row) = u32x2{kv8_encode4<F>(y[0], y[1], y[2], y[3]), kv8_encode4<F>(y[4], y[5], y[6], y[7])};
  };
#pragma unroll
  for (int k = 0; k < kKeep; ++k)
    if (in && r0 + k * rpp < n) put(r0 + k * rpp, x[k]);
  for (int r = r0 + kKeep * rpp; r < n; r += rpp)
    if (in) {
      float y[8];
      load8<DT, VEC>(src, src0 + r * ss, y);
      put(r, y);
    }
  if (bad || s == old || a == 0) return;
  const float f = old / s;
  for (int r = r0; r < a; r += rpp)
    if (in) {
      u32x2* const at = reinterpret_cast<u32x2*>(dst + r * row);
      const u32x2 w = *at;
      float y[8];
      kv8_decode4<F>(w[0], y);
      kv8_decode4<F>(w[1], y + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= f;
      *at = u32x2{kv8_encode4<F>(y[0], y[1], y[2], y[3]), kv8_encode4<F>(y[4], y[5], y[6], y[7])};
    }
}

// One wave per window of tokens, head and plane; it has the runs that begin in the window.
template <int F, int DT, bool VEC>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8Append p) {
  const int task = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (task >= 2 * p.hkv) return;
  const int plane = task / p.hkv, head = task - plane * p.hkv;
  const int lane = threadIdx.x & 63;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.window;
  // lane i: does token first + i begin a run?
  bool begins = false;
  const int64_t t = first + lane;
  if (lane < p.window && t < p.tokens) {
    const int64_t slot = p.slots[t];
    begins = slot >= 0 && (slot % p.bs == 0 || t == 0 || p.slots[t - 1] != slot - 1);
  }
  for (uint64_t todo = __ballot(begins); todo != 0; todo &= todo - 1) {
    const int64_t t0 = first + __builtin_ctzll(todo), slot = p.slots[t0];
    const int64_t blk = slot / p.bs;
    if (blk >= p.num_blocks) {
      if (lane == 0 && task == 0) atomicOr(p.err, 1);
      continue;
    }
    const int a = static_cast<int>(slot - blk * p.bs);
    int n = 1;
    for (;;) {  // 64 followers at a time
      const int64_t i = t0 + n + lane;
      const bool follows = a + n + lane < p.bs && i < p.tokens && p.slots[i] == slot + n + lane;
      const uint64_t stop = __ballot(!follows);
      n += stop == 0 ? 64 : __builtin_ctzll(stop);
      if (stop != 0) break;
    }
    append_run<F, DT, VEC>(p, plane, head, blk, a, n, t0);
  }
}

template <int F, int DT>
static void append_typed(const Kv8Append& p, bool vec, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(ceil_div(p.tokens, p.window)), static_cast<unsigned>(ceil_div(2 * p.hkv, 4)));
  if (vec) kv8_append_kernel<F, DT, true><<<grid, 256, 0, stream>>>(p);
  else kv8_append_kernel<F, DT, false><<<grid, 256, 0, stream>>>(p);
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
  p.window = p.tokens > 2048 ? 16 : 1;
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
