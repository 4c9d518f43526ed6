// The step plan of a paged cache, from request lengths alone: block tables, the slot and the
// position of every new token, and the free-block stack, without a host read (a captured
// graph replays it as the lengths change).
//
//   used = ceil(len / bs);  need = ceil((len + new) / bs) - used;  new < 0: the sequence
//   ended.  The ended ones' blocks lie on the stack first, in order of b and of their table;
//   blocks are then taken from its top in order of b.  A sequence is served if its table and
//   the token list have room for it and either need = 0 or the needs up to it fit the stack
//   (an inclusive sum, so no decision waits on another one).
//
// The stack is never built: place p of it is free[p] below the old count, and above it the
// (p - count)-th block of the ended sequences, found by binary search over their running
// sum.  So the pushes, the table entries and the slots are all computed side by side, and
// the entries that are read (below the old count) and written (from it on) never meet.
//
// Bound by latency: a batch of 256 reads and writes some 20 KB.  The running sums need all
// sequences, so one workgroup takes them; where it can hold them in LDS and the tokens are few
// it fills everything, too, in one launch (kv_plan_one_kernel), else the whole grid fills in a
// second one (kv_plan_fill_kernel).  Decode steps of 16 sequences 3.5 us, of 256 with five that
// ended 7.4 (4.8 without: their 800 blocks go on the stack); 1000 sequences, 60000 places 12.
#include <algorithm>

#include "kernels.hpp"

namespace hcp {

// Per sequence, from scan to fill: the old length (seq_lens_out may be seq_lens), what
// happens to it and where its blocks lie in the order of all blocks taken or given back.
struct PlanInfo {
  int32_t len, state, first, need;  // state: kIdle, kServed or kEnded
};
enum { kIdle = 0, kServed = 1, kEnded = 2 };
struct PlanHead {
  int32_t count, top, left, pad;  // old stack height, with the ended blocks, after the step
};

struct PlanArgs {
  KvPlan p;
  PlanHead* head;
  PlanInfo* info;     // [batch]
  int32_t* back_end;  // [batch] blocks given back by sequences 0 .. b
};

// What the scan leaves for the filling, in LDS or in the workspace.
struct PlanSums {
  const PlanInfo* info;
  const int32_t *starts, *back_end;  // starts as token_starts
  PlanHead head;
};

constexpr int kScan = 1024;       // threads of the scan's workgroup, and most sequences of the one-launch form
// Most tokens of the one-launch form, where each token's three loads in line are one CU's: 2000 tokens
// of 1000 sequences take it 9.3 us, two launches 10.4, of 16 8.1 and 8.9; 4000 of 1000 12.5 and 10.9.
constexpr int kOneTokens = 2048;

// Inclusive sums over the T threads of the workgroup of two counts each, and their totals.
struct Pair {
  int64_t x, y;
};
template <int T>
__device__ Pair scan_pair(Pair v, Pair* part, Pair& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int off = 1; off < 64; off *= 2) {
    const int64_t x = __shfl_up(v.x, off), y = __shfl_up(v.y, off);
    if (lane >= off) {
      v.x += x;
      v.y += y;
    }
  }
  __syncthreads();  // the last scan's totals are read
  if (lane == 63) part[wave] = v;
  __syncthreads();
  Pair before{0, 0};
  total = Pair{0, 0};
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    if (w == wave) before = total;
    total.x += part[w].x;
    total.y += part[w].y;
  }
  return Pair{v.x + before.x, v.y + before.y};
}

__device__ __forceinline__ int32_t sat32(int64_t v) { return static_cast<int32_t>(min(v, static_cast<int64_t>(INT32_MAX))); }

// x / bs: by a shift where bs is a power of two (a 64-bit division takes some 150 instructions).
__device__ __forceinline__ uint32_t plan_div(const KvPlan& p, uint32_t x) { return p.bs_shift >= 0 ? x >> p.bs_shift : x / p.bs; }
__device__ __forceinline__ uint32_t plan_ceil(const KvPlan& p, uint32_t x) {
  const uint32_t q = plan_div(p, x);
  return q + (q * p.bs != x);
}

// One sequence's lengths and what they ask for.
struct PlanSeq {
  int64_t len, add, used;
  bool sane, ended;
};
__device__ __forceinline__ PlanSeq plan_seq(const KvPlan& p, int b) {
  PlanSeq s;
  s.len = p.seq_lens[b];
  s.add = p.new_lens[b];
  s.used = plan_ceil(p, max(p.seq_lens[b], 0));
  s.sane = s.len >= 0 && s.used <= p.table_len;
  s.ended = s.sane && s.add < 0;
  return s;
}
// New blocks of a sequence with room for them, its tokens ending at `end`; -1 without.
__device__ __forceinline__ int64_t plan_need(const KvPlan& p, const PlanSeq& s, int32_t end) {
  const int64_t blocks = plan_ceil(p, static_cast<uint32_t>(max(s.len, static_cast<int64_t>(0)) + max(s.add, static_cast<int64_t>(0))));
  const bool fits = s.sane && s.add >= 0 && blocks <= p.table_len && s.len + s.add <= INT32_MAX && end <= p.capacity;
  return fits ? blocks - s.used : -1;
}
// What happens to it: `end` is the running sum of the needs, its own included.
__device__ __forceinline__ PlanInfo plan_info(const PlanSeq& s, int64_t need, int64_t end, int64_t top, int32_t back_end) {
  const bool served = need == 0 || (need > 0 && end <= top);
  return PlanInfo{static_cast<int32_t>(s.len), s.ended ? kEnded : served ? kServed : kIdle,
                  sat32(s.ended ? back_end - s.used : end - max(need, static_cast<int64_t>(0))),
                  static_cast<int32_t>(s.ended ? s.used : served ? need : 0)};
}
__device__ __forceinline__ int32_t plan_len_out(const PlanSeq& s, const PlanInfo& i) {
  return static_cast<int32_t>(i.state == kEnded ? 0 : i.state == kServed ? s.len + s.add : s.len);
}
// Height of the stack, and with the ended sequences' blocks on it; flags of what is wrong with them.
__device__ __forceinline__ int64_t plan_count(const KvPlan& p, int& flags) {
  const int64_t count = *p.free_count;
  if (count < 0 || count > p.num_blocks) flags |= 8;
  return min(max(count, static_cast<int64_t>(0)), p.num_blocks);
}
__device__ __forceinline__ int64_t plan_top(const KvPlan& p, int64_t count, int64_t back, int& flags) {
  if (count + back > p.num_blocks) flags |= 8;  // given back twice: what has no place is dropped
  return min(count + back, p.num_blocks);
}

// Place `at` of the stack with the ended sequences' blocks on it.
__device__ __forceinline__ int32_t stack_block(const KvPlan& p, const PlanSums& s, int64_t at) {
  if (at < s.head.count) return p.free_blocks[at];
  const int32_t i = static_cast<int32_t>(at) - s.head.count;
  int lo = 0, hi = p.batch - 1;  // first sequence whose running sum is past i
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (s.back_end[mid] > i) hi = mid;
    else lo = mid + 1;
  }
  return p.block_tables[lo * p.table_stride + i - s.info[lo].first];
}

// The sequence of token i among lo .. hi: the first that ends past it.
__device__ __forceinline__ int plan_seq_of(const int32_t* starts, int lo, int hi, int64_t i) {
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (starts[mid + 1] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Slot and position of token i, which is one of sequences lo .. hi's or lies past all tokens.
__device__ __forceinline__ void plan_token(const KvPlan& p, const PlanSums& s, int64_t i, int lo, int hi) {
  int64_t slot = -1, pos = 0;
  if (i < s.starts[p.batch]) {
    const int b = plan_seq_of(s.starts, lo, hi, i);
    const PlanInfo q = s.info[b];
    pos = q.len < 0 ? 0 : static_cast<int64_t>(q.len) + i - s.starts[b];
    if (q.state == kServed) {
      const int32_t entry = plan_div(p, static_cast<uint32_t>(pos)), used = plan_ceil(p, q.len);
      const int32_t blk = entry < used ? p.block_tables[b * p.table_stride + entry]
                                       : stack_block(p, s, s.head.top - 1 - (static_cast<int64_t>(q.first) + entry - used));
      if (blk >= 0 && blk < p.num_blocks) slot = static_cast<int64_t>(blk) * p.bs + (pos - static_cast<int64_t>(entry) * p.bs);
      else atomicOr(p.err, 1);
    }
  }
  p.slots[i] = slot;
  p.positions[i] = pos;
}

// Entries from .. , from + step, ... that sequence b gets or gives back.
__device__ __forceinline__ void plan_blocks(const KvPlan& p, const PlanSums& s, int64_t b, int from, int to, int step) {
  const PlanInfo q = s.info[b];
  int32_t* const row = p.block_tables + b * p.table_stride;
  if (q.state == kServed) {
    const int32_t used = plan_ceil(p, q.len);
    for (int32_t i = from; i < min(q.need, to); i += step)
      row[used + i] = stack_block(p, s, s.head.top - 1 - (static_cast<int64_t>(q.first) + i));
  } else if (q.state == kEnded) {
    uint32_t most = 0;  // a negative id is past every block, too
    for (int32_t i = from; i < min(q.need, to); i += step) {
      const int64_t at = static_cast<int64_t>(s.head.count) + q.first + i;
      if (at >= s.head.left) continue;  // taken again in this step, and looked at by its token
      const int32_t blk = row[i];
      most = max(most, static_cast<uint32_t>(blk));
      p.free_blocks[at] = blk;
    }
    if (most >= p.num_blocks) atomicOr(p.err, 1);
  }
}

// Up to T sequences, one a thread, their sums in registers and LDS.  kFill: tokens and blocks,
// too; else the sums go to the workspace for the fill kernel.
template <int T, bool kFill>
__global__ __launch_bounds__(T) void kv_plan_one_kernel(PlanArgs a) {
  const KvPlan& p = a.p;
  __shared__ Pair part[T / 64];
  __shared__ PlanInfo info[T];
  __shared__ int32_t starts[T + 1], back_end[T], many[T];
  __shared__ int32_t taken, n_many;
  const int b = threadIdx.x;
  int flags = 0;
  PlanSeq s{0, 0, 0, true, false};
  if (b < p.batch) s = plan_seq(p, b);
  if (!s.sane) flags |= 8;
  const int64_t count = plan_count(p, flags);
  if (b == 0) taken = n_many = 0;
  Pair total;
  const Pair sum = scan_pair<T>(Pair{max(s.add, static_cast<int64_t>(0)), s.ended ? s.used : 0}, part, total);
  const int64_t top = plan_top(p, count, total.y, flags);
  starts[b + 1] = sat32(sum.x);
  if (b == 0) starts[0] = 0;
  back_end[b] = sat32(sum.y);
  const int64_t need = b < p.batch ? plan_need(p, s, starts[b + 1]) : -1;
  const int64_t end = scan_pair<T>(Pair{max(need, static_cast<int64_t>(0)), 0}, part, total).x;
  const PlanInfo mine = plan_info(s, need, end, top, back_end[b]);
  info[b] = mine;
  // the served ones that need blocks come before those that get none: the last one's end is what is taken
  if (mine.state == kServed && mine.need > 0) atomicMax(&taken, static_cast<int32_t>(end));
  if (flags != 0) atomicOr(p.err, flags);
  __syncthreads();
  const PlanSums sums{info, starts, back_end,
                      PlanHead{static_cast<int32_t>(count), static_cast<int32_t>(top), static_cast<int32_t>(top - taken), 0}};
  if (b < p.batch) {
    p.seq_lens_out[b] = plan_len_out(s, mine);
    p.token_starts[b + 1] = starts[b + 1];
  }
  if (b == 0) {
    p.token_starts[0] = 0;
    *p.free_count_out = sums.head.left;
  }
  if constexpr (!kFill) {
    if (b < p.batch) {
      a.info[b] = mine;
      a.back_end[b] = back_end[b];
    }
    if (b == 0) *a.head = sums.head;
    return;
  }
  for (int64_t i = b; i < p.capacity; i += T) plan_token(p, sums, i, 0, p.batch - 1);
  if (b < p.batch) plan_blocks(p, sums, b, 0, 2, 1);  // a decode step's sequence gets one at most
  // long rows (a prompt's, an ended sequence's): one a wave, from a list whose order is of no matter
  if (mine.need > 2) many[atomicAdd(&n_many, 1)] = b;
  __syncthreads();
  for (int w = b >> 6; w < n_many; w += T / 64) plan_blocks(p, sums, many[w], 2 + (b & 63), INT32_MAX, 64);
}

// Any number of sequences.
__global__ __launch_bounds__(kScan) void kv_plan_scan_kernel(PlanArgs a) {
  __shared__ Pair part[kScan / 64];
  __shared__ int32_t taken;
  const KvPlan& p = a.p;
  int flags = 0;
  const int64_t count = plan_count(p, flags);
  if (threadIdx.x == 0) taken = 0;
  // tokens and blocks given back first: the stack's height decides who is served
  Pair sum{0, 0}, total;
  for (int base = 0; base < p.batch; base += kScan) {
    const int b = base + threadIdx.x;
    PlanSeq s{0, 0, 0, true, false};
    if (b < p.batch) s = plan_seq(p, b);
    if (!s.sane) flags |= 8;
    const Pair inc = scan_pair<kScan>(Pair{max(s.add, static_cast<int64_t>(0)), s.ended ? s.used : 0}, part, total);
    if (b < p.batch) {
      p.token_starts[b + 1] = sat32(sum.x + inc.x);
      a.back_end[b] = sat32(sum.y + inc.y);
    }
    sum.x += total.x;
    sum.y += total.y;
  }
  const int64_t top = plan_top(p, count, sum.y, flags);
  int64_t asked = 0;
  for (int base = 0; base < p.batch; base += kScan) {
    const int b = base + threadIdx.x;
    PlanSeq s{0, 0, 0, true, false};
    int64_t need = -1;
    if (b < p.batch) {
      s = plan_seq(p, b);
      need = plan_need(p, s, p.token_starts[b + 1]);
    }
    const int64_t end = asked + scan_pair<kScan>(Pair{max(need, static_cast<int64_t>(0)), 0}, part, total).x;
    asked += total.x;
    if (b < p.batch) {
      const PlanInfo mine = plan_info(s, need, end, top, a.back_end[b]);
      a.info[b] = mine;
      if (mine.state == kServed && mine.need > 0) atomicMax(&taken, static_cast<int32_t>(end));
      p.seq_lens_out[b] = plan_len_out(s, mine);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    p.token_starts[0] = 0;
    const int32_t left = static_cast<int32_t>(top) - taken;
    *a.head = PlanHead{static_cast<int32_t>(count), static_cast<int32_t>(top), left, 0};
    *p.free_count_out = left;
  }
  if (flags != 0) atomicOr(p.err, flags);
}

// As plan_seq_of by a whole wave: 64 probes at a time (1000 sequences: two loads in line, not ten).
__device__ __forceinline__ int plan_seq_of_wave(const int32_t* starts, int lo, int hi, int64_t i) {
  const int lane = threadIdx.x & 63;
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64;
    const int64_t mid = static_cast<int64_t>(lo) + (lane + 1ll) * step - 1;
    const uint64_t past = __ballot(mid >= hi || starts[mid + 1] > i);
    if (past == 0) return hi;
    const int f = __builtin_ctzll(past);
    hi = static_cast<int>(min(static_cast<int64_t>(lo) + (f + 1ll) * step - 1, static_cast<int64_t>(hi)));
    lo = lo + f * step;
  }
  return lo;
}

// The first workgroups: 256 tokens each, whose sequences lie between its first and its last token's;
// where those are few their starts are searched in LDS.  The others: a sequence's blocks a wave.
constexpr int kStarts = 512;
__global__ __launch_bounds__(256) void kv_plan_fill_kernel(PlanArgs a, int token_groups) {
  __shared__ int ends[2];
  __shared__ int32_t near[kStarts + 1];
  const KvPlan& p = a.p;
  const PlanSums sums{a.info, p.token_starts, a.back_end, *a.head};
  if (static_cast<int>(blockIdx.x) >= token_groups) {
    const int64_t b = static_cast<int64_t>(blockIdx.x - token_groups) * 4 + (threadIdx.x >> 6);
    if (b < p.batch) plan_blocks(p, sums, b, threadIdx.x & 63, INT32_MAX, 64);
    return;
  }
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256, i = first + threadIdx.x;
  const int32_t all = p.token_starts[p.batch];
  if (first >= all) {  // past all tokens
    if (i < p.capacity) {
      p.slots[i] = -1;
      p.positions[i] = 0;
    }
    return;
  }
  if (threadIdx.x < 128) {
    const int e = plan_seq_of_wave(p.token_starts, 0, p.batch - 1, threadIdx.x < 64 ? first : first + 255);
    if ((threadIdx.x & 63) == 0) ends[threadIdx.x >> 6] = e;
  }
  __syncthreads();
  const int lo = ends[0], n = ends[1] - lo + 1;
  int b = lo;
  if (n <= kStarts) {
    for (int k = threadIdx.x; k <= n; k += 256) near[k] = p.token_starts[lo + k];
    __syncthreads();
    b = lo + plan_seq_of(near, 0, n - 1, i);
  } else {
    b = plan_seq_of(p.token_starts, lo, ends[1], i);
  }
  if (i < p.capacity) plan_token(p, sums, i, b, b);
}

static size_t plan_align(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

size_t kv_plan_workspace_bytes(int batch) {
  return plan_align(sizeof(PlanHead)) + plan_align(sizeof(PlanInfo) * batch) + plan_align(sizeof(int32_t) * batch);
}

void launch_kv_plan(const KvPlan& p, void* ws, hipStream_t stream) {
  PlanArgs a;
  a.p = p;
  char* at = static_cast<char*>(ws);
  a.head = reinterpret_cast<PlanHead*>(at);
  at += plan_align(sizeof(PlanHead));
  a.info = reinterpret_cast<PlanInfo*>(at);
  at += plan_align(sizeof(PlanInfo) * p.batch);
  a.back_end = reinterpret_cast<int32_t*>(at);
  if (p.batch <= kScan && p.capacity <= kOneTokens) {
    // four waves for a decode step (256 tokens 4.8 us); 1024 tokens 8.3 us with four, 7.1 with sixteen
    if (p.batch <= 256 && p.capacity <= 512) kv_plan_one_kernel<256, true><<<1, 256, 0, stream>>>(a);
    else kv_plan_one_kernel<kScan, true><<<1, kScan, 0, stream>>>(a);
    HCP_HIP(hipGetLastError());
    return;
  }
  const int64_t token_groups = ceil_div(p.capacity, 256), grid = token_groups + ceil_div(p.batch, 4);
  require(grid < (1 << 24), "kv_plan: too many tokens or sequences");  // threads of a launch: 2^32
  if (p.batch <= kScan) kv_plan_one_kernel<kScan, false><<<1, kScan, 0, stream>>>(a);
  else kv_plan_scan_kernel<<<1, kScan, 0, stream>>>(a);
  HCP_HIP(hipGetLastError());
  kv_plan_fill_kernel<<<static_cast<unsigned>(grid), 256, 0, stream>>>(a, static_cast<int>(token_groups));
  HCP_HIP(hipGetLastError());
}

}  // namespace hcp
