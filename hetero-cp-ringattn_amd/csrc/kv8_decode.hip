// Single-query attention over the 8-bit paged cache (layout in kv8.hpp): per sequence and
// query head S = scale * s_K (q . c_K) over its tokens, shard after shard; O = sum P s_V c_V,
// lse = ln sum e^S; no token: O = 0, lse = -inf.
#include "kv8.hpp"

namespace hcp {

struct Kv8DecodeArgs {
  const void* q;
  int64_t q_bs, q_hs;
  const uint8_t* pool;
  const float* scales;
  int64_t num_blocks;
  int32_t bs, hkv, hq, d;
  DecodeSpan span[kMaxDomains];
  int32_t n_spans, out_dtype;
  float scale;
  void* out;
  int64_t out_rs;
  float* lse;
  int* err;
};
static_assert(sizeof(Kv8DecodeArgs) <= 4096, "kernel arguments are limited to 4 KiB");

// One wave per sequence and query head; lane l has dims 2l, 2l + 1.
template <int F, int DT>
__global__ __launch_bounds__(64) void kv8_decode_kernel(Kv8DecodeArgs a) {
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x, kvh = h / (a.hq / a.hkv);
  const int c = lane * 2;
  const bool in = c < a.d;
  float q0 = 0.f, q1 = 0.f;
  if (in) {
    q0 = load_elem<DT>(a.q, b * a.q_bs + h * a.q_hs + c) * a.scale;
    q1 = load_elem<DT>(a.q, b * a.q_bs + h * a.q_hs + c + 1) * a.scale;
  }
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  const int64_t row = static_cast<int64_t>(a.hkv) * a.d;
  for (int s = 0; s < a.n_spans; ++s) {
    const DecodeSpan& sp = a.span[s];
    const int64_t end = sp.seq_lens == nullptr ? sp.t1 : min(sp.t1, static_cast<int64_t>(sp.seq_lens[b]) - sp.len_off);
    const int32_t* table = sp.tables + b * sp.table_stride;
    for (int64_t t = sp.t0; t < end; ++t) {
      const int64_t entry = t / a.bs;
      const int32_t blk = table[entry];
      if (blk < 0 || blk >= a.num_blocks) {
        if (lane == 0) atomicOr(a.err, 1);
        continue;
      }
      const int64_t at = (static_cast<int64_t>(blk) * a.bs + (t - entry * a.bs)) * row + kvh * a.d + c;
      const uint8_t* k = a.pool + at;
      const uint8_t* v = k + a.num_blocks * a.bs * row;
      float kx[4] = {}, vx[4] = {};
      if (in) {
        kv8_decode4<F>(*reinterpret_cast<const uint16_t*>(k), kx);
        kv8_decode4<F>(*reinterpret_cast<const uint16_t*>(v), vx);
      }
      float sc = q0 * kx[0] + q1 * kx[1];
      for (int off = 32; off > 0; off /= 2) sc += __shfl_xor(sc, off);
      sc *= a.scales[static_cast<int64_t>(blk) * a.hkv + kvh];
      const float vs = a.scales[(a.num_blocks + blk) * a.hkv + kvh];
      const float mn = fmaxf(m, sc), f = m == -INFINITY ? 0.f : __expf(m - mn), p = __expf(sc - mn);
      m = mn;
      l = l * f + p;
      o0 = o0 * f + p * vs * vx[0];
      o1 = o1 * f + p * vs * vx[1];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t r = static_cast<int64_t>(b) * a.hq + h;
  if (in) {
    store_elem_rt(a.out, a.out_dtype, r * a.out_rs + c, o0 * inv);
    store_elem_rt(a.out, a.out_dtype, r * a.out_rs + c + 1, o1 * inv);
  }
  if (lane == 0 && a.lse != nullptr) a.lse[r] = l == 0.f ? -INFINITY : m + __logf(l);
}

size_t kv8_decode_workspace_bytes(int batch, int hq, int hkv, int d, int n, const DecodeSpan* spans) { return 0; }

void launch_kv8_decode(const Kv8Pool& pool, int dtype, int batch, int hq, const void* q, int64_t q_bs, int64_t q_hs, int n,
                       const DecodeSpan* spans, float scale, int out_dtype, void* out, int64_t out_rs, float* lse, void* ws,
                       size_t ws_bytes, int* err, hipStream_t stream) {
  (void)ws;
  (void)ws_bytes;
  Kv8DecodeArgs a;
  a.q = q;
  a.q_bs = q_bs;
  a.q_hs = q_hs;
  a.pool = pool.codes;
  a.scales = pool.scales;
  a.num_blocks = pool.num_blocks;
  a.bs = pool.bs;
  a.hkv = pool.hkv;
  a.hq = hq;
  a.d = pool.d;
  a.n_spans = n;
  for (int i = 0; i < n; ++i) a.span[i] = spans[i];
  a.out_dtype = out_dtype;
  a.scale = scale;
  a.out = out;
  a.out_rs = out_rs;
  a.lse = lse;
  a.err = err;
  const dim3 grid(hq, batch);
  if (pool.format == kE4M3) {
    if (dtype == kBF16) kv8_decode_kernel<kE4M3, kBF16><<<grid, 64, 0, stream>>>(a);
    else kv8_decode_kernel<kE4M3, kF16><<<grid, 64, 0, stream>>>(a);
  } else {
    if (dtype == kBF16) kv8_decode_kernel<kInt8, kBF16><<<grid, 64, 0, stream>>>(a);
    else kv8_decode_kernel<kInt8, kF16><<<grid, 64, 0, stream>>>(a);
  }
  HCP_HIP(hipGetLastError());
}

}  // namespace hcp
