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
// sequences, so one workgroup takes them (scan), then the whole grid fills (fill).
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

constexpr int kScan = 1024;  // threads of the scan's workgroup

// Inclusive sums over the workgroup of two counts per thread, and their totals.
struct Pair {
  int64_t x, y;
};
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
  for (int w = 0; w < kScan / 64; ++w) {
    if (w == wave) before = total;
    total.x += part[w].x;
    total.y += part[w].y;
  }
  return Pair{v.x + before.x, v.y + before.y};
}

__device__ __forceinline__ int32_t sat32(int64_t v) { return static_cast<int32_t>(min(v, static_cast<int64_t>(INT32_MAX))); }

__device__ void plan_scan(const PlanArgs& a) {
  __shared__ Pair part[kScan / 64];
  const KvPlan& p = a.p;
  int flags = 0;
  int64_t count = *p.free_count;
  if (count < 0 || count > p.num_blocks) flags |= 8;
  count = min(max(count, static_cast<int64_t>(0)), p.num_blocks);
  // tokens and blocks given back first: the stack's height decides who is served
  Pair sum{0, 0}, total;
  for (int base = 0; base < p.batch; base += kScan) {
    const int b = base + threadIdx.x;
    Pair v{0, 0};
    if (b < p.batch) {
      const int64_t len = p.seq_lens[b], add = p.new_lens[b];
      const int64_t used = (max(len, static_cast<int64_t>(0)) + p.bs - 1) / p.bs;
      const bool sane = len >= 0 && used <= p.table_len;
      if (!sane) flags |= 8;
      v.x = max(add, static_cast<int64_t>(0));
      v.y = sane && add < 0 ? used : 0;
    }
    const Pair inc = scan_pair(v, part, total);
    if (b < p.batch) {
      p.token_starts[b + 1] = sat32(sum.x + inc.x);
      a.back_end[b] = sat32(sum.y + inc.y);
    }
    sum.x += total.x;
    sum.y += total.y;
  }
  int64_t top = count + sum.y;
  if (top > p.num_blocks) {  // blocks given back twice: what has no place is dropped
    flags |= 8;
    top = p.num_blocks;
  }
  Pair taken{0, 0};  // needs of all, and of the served
  int64_t tokens = 0;
  for (int base = 0; base < p.batch; base += kScan) {
    const int b = base + threadIdx.x;
    Pair v{0, 0};
    int64_t len = 0, add = 0, used = 0;
    bool fits = false, ended = false;
    if (b < p.batch) {
      len = p.seq_lens[b];
      add = p.new_lens[b];
      used = (max(len, static_cast<int64_t>(0)) + p.bs - 1) / p.bs;
      const bool sane = len >= 0 && used <= p.table_len;
      ended = sane && add < 0;
      const int64_t blocks = (len + max(add, static_cast<int64_t>(0)) + p.bs - 1) / p.bs;
      fits = sane && add >= 0 && blocks <= p.table_len && len + add <= INT32_MAX &&
             p.token_starts[b + 1] <= p.capacity;
      if (fits) v.x = blocks - used;
    }
    const Pair inc = scan_pair(v, part, total);
    const int64_t end = taken.x + inc.x;
    const bool served = fits && (v.x == 0 || end <= top);
    if (b < p.batch) {
      PlanInfo i;
      i.len = static_cast<int32_t>(len);
      i.state = ended ? kEnded : served ? kServed : kIdle;
      i.first = sat32(ended ? a.back_end[b] - used : end - v.x);
      i.need = static_cast<int32_t>(ended ? used : served ? v.x : 0);
      a.info[b] = i;
      p.seq_lens_out[b] = static_cast<int32_t>(ended ? 0 : served ? len + add : len);
    }
    // the served ones that need blocks are a prefix of those that ask: the last one's end is
    // what is taken
    const Pair most = Pair{0, served ? v.x : 0};
    taken.x += total.x;
    scan_pair(most, part, total);
    tokens += total.y;
  }
  if (threadIdx.x == 0) {
    p.token_starts[0] = 0;
    *a.head = PlanHead{static_cast<int32_t>(count), static_cast<int32_t>(top), static_cast<int32_t>(top - tokens), 0};
    *p.free_count_out = static_cast<int32_t>(top - tokens);
  }
  if (flags != 0) atomicOr(p.err, flags);
}

// Place `at` of the stack with the ended sequences' blocks on it.
__device__ __forceinline__ int32_t stack_block(const PlanArgs& a, const PlanHead& h, int64_t at) {
  if (at < h.count) return a.p.free_blocks[at];
  const int32_t i = static_cast<int32_t>(at) - h.count;
  int lo = 0, hi = a.p.batch - 1;  // first sequence whose running sum is past i
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.back_end[mid] > i) hi = mid;
    else lo = mid + 1;
  }
  return a.p.block_tables[lo * a.p.table_stride + i - a.info[lo].first];
}

__device__ void plan_fill(const PlanArgs& a, int64_t thread, int64_t threads) {
  const KvPlan& p = a.p;
  const PlanHead h = *a.head;
  const int64_t total = p.token_starts[p.batch];
  for (int64_t i = thread; i < p.capacity; i += threads) {
    int64_t slot = -1, pos = 0;
    if (i < total) {
      int lo = 0, hi = p.batch - 1;  // the sequence of token i
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (p.token_starts[mid + 1] > i) hi = mid;
        else lo = mid + 1;
      }
      const PlanInfo s = a.info[lo];
      pos = s.len < 0 ? 0 : static_cast<int64_t>(s.len) + i - p.token_starts[lo];
      if (s.state == kServed) {
        const int64_t entry = pos / p.bs, used = (s.len + p.bs - 1) / p.bs;
        const int32_t blk = entry < used ? p.block_tables[lo * p.table_stride + entry]
                                         : stack_block(a, h, h.top - 1 - (s.first + entry - used));
        if (blk >= 0 && blk < p.num_blocks) slot = static_cast<int64_t>(blk) * p.bs + (pos - entry * p.bs);
        else atomicOr(p.err, 1);
      }
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
  }
}

// Entries that a sequence gets or gives back, by one wave.
__device__ void plan_blocks(const PlanArgs& a, int64_t wave, int64_t waves) {
  const KvPlan& p = a.p;
  const PlanHead h = *a.head;
  for (int64_t b = wave; b < p.batch; b += waves) {
    const PlanInfo s = a.info[b];
    int32_t* const row = p.block_tables + b * p.table_stride;
    if (s.state == kServed) {
      const int32_t used = (s.len + p.bs - 1) / p.bs;
      for (int32_t i = threadIdx.x & 63; i < s.need; i += 64) row[used + i] = stack_block(a, h, h.top - 1 - (int64_t(s.first) + i));
    } else if (s.state == kEnded) {
      for (int32_t i = threadIdx.x & 63; i < s.need; i += 64) {
        const int64_t at = int64_t(h.count) + s.first + i;
        if (at < h.left) p.free_blocks[at] = row[i];
      }
    }
  }
}

__global__ __launch_bounds__(kScan) void kv_plan_scan_kernel(PlanArgs a) { plan_scan(a); }

__global__ __launch_bounds__(256) void kv_plan_fill_kernel(PlanArgs a) {
  const int64_t thread = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  plan_fill(a, thread, static_cast<int64_t>(gridDim.x) * 256);
  plan_blocks(a, thread >> 6, static_cast<int64_t>(gridDim.x) * 4);
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
  kv_plan_scan_kernel<<<1, kScan, 0, stream>>>(a);
  HCP_HIP(hipGetLastError());
  const int64_t items = std::max<int64_t>(p.capacity, static_cast<int64_t>(p.batch) * 64);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(ceil_div(items, 256), 1), 2048));
  kv_plan_fill_kernel<<<grid, 256, 0, stream>>>(a);
  HCP_HIP(hipGetLastError());
}

}  // namespace hcp
