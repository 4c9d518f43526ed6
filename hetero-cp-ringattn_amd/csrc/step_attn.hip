// Attention of one serving step over the paged cache: a batch of sequences with one or many
// new tokens each, behind what the cache holds of each and behind prefixes that several share.
//
//   o = softmax(q K^T scale) V over a sequence's prefix keys and those of its own keys that a
//   token sees; a prefix's K and V are read once for all of the step's tokens behind it.
//
// Rows.  The query heads of a kv head are packed token-major: row r of a source (a sequence's new
// tokens, or all the tokens behind one prefix) is token r / rep, head r % rep of the group.  A long
// source is cut into wide tiles of 256 rows, 32 a wave, whose K and V tiles of 128 keys are shared
// through LDS: the ping-pong of the ring kernels, with the rows of a tile fetched block by block,
// bound by the MFMA rate and the softmax's VALU work beside it (16384 tokens of 32/8 heads of 128
// dims: 1.90 ms, 1157 TFLOP/s; the ring kernel on contiguous K and V 1240-1280).  A short one is cut
// into narrow tiles of 32 rows: 8 waves hold the same rows and take 32 keys each in turn, out of
// LDS of their own, with no barrier until their results meet, bound by HBM reads (64 sequences of
// up to 16384 tokens, 32/8 heads: 592 us, 5.7 TB/s) or, in short steps, by the chain of loads that
// leads to the keys.  64 sequences behind one prefix of 16384 tokens: 67 us (54 where the pass before
// has read the same keys), where every one reading it for itself would take some 700.
//
// Work.  The (tile, kv head) units of each kind are laid end to end on an axis of modelled time,
// the wide ones by kv head first (workgroups of one XCD then read one head's K and V).  Every XCD
// gets an eighth of both, and its workgroups, one a CU, equal parts of that: a unit that falls to
// several is joined afterwards (step_join_kernel), as is a row's part behind a shared prefix with
// its own part.  The plan (step_plan_kernel) lays both axes out once a step for the calls of all
// layers.
//
// Rounding.  Scores, statistics, sums and joins are fp32.  A weight enters the product with V in 16
// bits: one term in wide tiles of 16-bit output (its rounding is as large as the output's own;
// errors add to 1.4 times that), two in narrow ones, whose matrix cores wait for HBM anyway, and for
// fp32 output as many as hold 22 bits or more (two of f16, three of bf16: the prompt above takes 2.9
// and 3.5 ms so, 2.0 and 1.9 with one).
#include <algorithm>

#include "kernels.hpp"
#include "lds_dma.hpp"
#include "attn_tile.hpp"

namespace hcp {

namespace {

constexpr int kStepWaves = 8;
constexpr int kStepThreads = 64 * kStepWaves;
constexpr int kWideRows = 32 * kStepWaves;  // rows of a wide tile
constexpr int kWideKeys = 128;              // keys of its steps
constexpr int kNarrowRows = 32;
constexpr int kNarrowMost = 128;            // most rows of a source that is cut into narrow tiles in any step
constexpr int kPlanThreads = 1024;
constexpr int kPlanMagic = 0x53544550;

// Modelled time in 0.1 us: of a unit beside its steps, and of a step of 128 (wide) or up to
// 8 x 32 keys (narrow).  Measured with all CUs busy: wide 60-130 and 33-43, narrow 30-45 and 16-51
// (keys in the L2; HBM reads at their limit).
constexpr int kWideFixed = 70, kWideStep = 40;
constexpr int kNarrowFixed = 32, kNarrowStep = 26;
// Of a worker: less is not worth another part to join.
constexpr int kLeastShare = 50;
// Sources of more rows are narrow tiles too where that is this much longer at most per worker: a
// step of few wide units cuts them among many workers, each of which leaves 256 rows to join.  512
// queries x 2085 keys, 8/1 heads of 96 dims, fp32 rows: 32 us as 16 wide units, 22.6 as 128 narrow
// ones; 1500-token prefixes behind 16 sequences of 5 tokens, 14/2 heads of 64: 24.5 and 23.3.
constexpr int kNarrowMore = 150;
constexpr int kXcds = 8;

// Where a unit's rows go when it is not cut.
enum { kToOut = 0, kToOwn = 1, kToPrefix = 2 };

struct StepTile {
  int32_t tok0;        // query token of row 0 of the source, or its first list entry (list)
  int32_t row0, rows;  // rows of the source in this tile
  int32_t p_row, p_len;     // prefix table's row and keys (0: none)
  int32_t s_row, s_len;     // own table's row and the keys that some row of the tile sees
  int32_t vis0, vis_step;   // token i of the source sees own keys j < vis0 + i * vis_step
  int32_t steps;
  int32_t dest, list0;      // kTo*, list entry of token 0 of the source
  int32_t list;             // tokens through the list
  int32_t pad[3];
};
static_assert(sizeof(StepTile) == 64, "read_tile counts 16 words");

// A token behind a shared prefix: its own narrow tile, and its rows in the prefix's tiles.
struct StepShared {
  int32_t token;
  int32_t own_tile, own_row;           // the sequence's first narrow tile (counted from 0), row of the token's first head
  int32_t pre_tile, pre_row, pre_wide; // the same of the prefix's tiles, wide or narrow
  int32_t pad[2];
};

// A cut unit whose rows go to the output: where they are, and its entry of cuts.
struct StepCut {
  int32_t cut, row0, rows, tok0, head0, pad[3];
};

struct StepHead {
  int32_t magic, batch, tokens, hq, hkv, d, bs, causal, prefixes, max_own, max_prefix, workers;
  int32_t n_wide, n_narrow, n_shared, cut_wide, cut_narrow, pad[3];
};
// Whether the plan was made for this shape and number of workers.
template <typename P>
__device__ bool plan_fits(P head, const StepShape& s, int workers) {
  const int want[12] = {kPlanMagic, s.batch, static_cast<int>(s.tokens), s.hq, s.hkv, s.d, s.bs, s.causal, s.prefixes,
                        static_cast<int>(s.max_own), static_cast<int>(s.max_prefix), workers};
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 12; ++i) ok = ok && head[i] == want[i];
  return ok;
}

// Offsets of the plan's arrays, from host-known bounds alone.
struct PlanLayout {
  int64_t max_wide, max_narrow, max_shared, max_units;
  size_t tiles, cum_wide, cum_narrow, shared, starts, cuts, cut_wide, cut_narrow, bytes;
};

size_t up256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

PlanLayout plan_layout(const StepShape& s) {
  const int64_t rep = s.hq / s.hkv, live = std::min<int64_t>(s.batch, s.tokens);
  PlanLayout l;
  l.max_shared = s.prefixes > 0 ? std::min<int64_t>(s.tokens, live * (kNarrowMost / rep)) : 0;
  l.max_wide = s.tokens * rep / kWideRows + live + (s.prefixes > 0 ? l.max_shared * rep / kWideRows + std::min<int64_t>(s.prefixes, live) : 0);
  l.max_narrow = s.tokens * rep / kNarrowRows + live + (s.prefixes > 0 ? l.max_shared * rep / kNarrowRows + std::min<int64_t>(s.prefixes, live) : 0);
  l.max_units = (l.max_wide + l.max_narrow) * s.hkv;
  size_t at = up256(sizeof(StepHead));
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += up256(bytes);
    return here;
  };
  l.tiles = take((l.max_wide + l.max_narrow) * sizeof(StepTile));
  l.cum_wide = take((l.max_wide + 1) * sizeof(int64_t));
  l.cum_narrow = take((l.max_narrow + 1) * sizeof(int64_t));
  l.shared = take(l.max_shared * sizeof(StepShared));
  l.starts = take(2 * (kStepMaxWorkers + 1) * 2 * sizeof(int32_t));
  l.cuts = take(l.max_units * sizeof(int32_t));
  l.cut_wide = take(kStepMaxWorkers * sizeof(StepCut));
  l.cut_narrow = take(kStepMaxWorkers * sizeof(StepCut));
  l.bytes = at;
  return l;
}

// The workspace: two slots of partial rows a worker of either kind (its first and its last unit, where cut),
// then the rows of tokens behind shared prefixes, their own part and the prefix's.
struct WorkLayout {
  int32_t slot_rows;
  size_t slot_o, slot_lse, own_o, own_lse, pre_o, pre_lse, bytes;
};
WorkLayout work_layout(const StepShape& s, int workers) {
  const int64_t rep = s.hq / s.hkv;
  WorkLayout w;
  w.slot_rows = static_cast<int32_t>(std::min<int64_t>(kWideRows, (s.tokens * rep + 31) / 32 * 32));
  size_t at = 0;
  auto take = [&](size_t floats) {
    const size_t here = at;
    at += up256(floats * sizeof(float));
    return here;
  };
  const size_t slots = 4 * static_cast<size_t>(workers + 1) * w.slot_rows;  // by the worker's place in the plan's starts
  const size_t rows = static_cast<size_t>(plan_layout(s).max_shared) * s.hq;
  w.slot_o = take(slots * s.d);
  w.slot_lse = take(slots);
  w.own_o = take(rows * s.d);
  w.own_lse = take(rows);
  w.pre_o = take(rows * s.d);
  w.pre_lse = take(rows);
  w.bytes = std::max<size_t>(at, 256);  // without tokens too: a size of 0 says that the shape is bad
  return w;
}

}  // namespace

size_t step_plan_bytes(const StepShape& s) { return plan_layout(s).bytes; }
size_t step_work_bytes(const StepShape& s) { return work_layout(s, step_workers()).bytes; }
int step_workers() { return std::min(device_cus(), kStepMaxWorkers); }

// ----------------------------------------------------------------------------------
// Plan: one workgroup.
// ----------------------------------------------------------------------------------
struct PlanKernelArgs {
  StepShape s;
  int32_t workers;
  const int32_t *token_starts, *seq_lens, *prefix_ids, *prefix_lens;
  char* plan;
  PlanLayout l;
  int* err;
};

namespace {

// Exclusive running sum of a[0 .. n) in LDS in place, by the whole workgroup; the total.
__device__ int scan_lds(int* a, int n, int* tmp) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (n + kPlanThreads - 1) / kPlanThreads, b = min(tid * per, n), e = min(b + per, n);
  int sum = 0;
  for (int i = b; i < e; ++i) sum += a[i];
  int x = sum;
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int before = x - sum, total = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += tmp[w];
    total += tmp[w];
  }
  for (int i = b; i < e; ++i) {
    const int v = a[i];
    a[i] = before;
    before += v;
  }
  __syncthreads();
  return total;
}

// cum[0 .. n] = running sums of cost(i), by the whole workgroup.
template <typename F>
__device__ int64_t scan_costs(int64_t* cum, int n, F&& cost, int64_t* tmp) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t base = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const int64_t c = i < n ? cost(i) : 0;
    int64_t x = c;
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t y = __shfl_up(x, off);
      if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    int64_t before = base + x - c, total = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      if (w < wave) before += tmp[w];
      total += tmp[w];
    }
    if (i < n) cum[i] = before;
    base += total;
  }
  if (tid == 0) cum[n] = base;
  __syncthreads();
  return base;
}

// The last i of a[0 .. n) (non-decreasing, a[0] <= x) with a[i] <= x.
template <typename T>
__device__ int last_at_most(const T* a, int n, T x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

}  // namespace

__global__ __launch_bounds__(kPlanThreads) void step_plan_kernel(PlanKernelArgs a) {
  __shared__ int s_tok[kStepMaxBatch], s_n[kStepMaxBatch], s_vis[kStepMaxBatch], s_len[kStepMaxBatch];
  __shared__ int s_pid[kStepMaxBatch], s_wide[kStepMaxBatch], s_nar[kStepMaxBatch], s_list[kStepMaxBatch];
  __shared__ int g_seq[kStepMaxPrefixes], g_tok[kStepMaxPrefixes], g_list[kStepMaxPrefixes], g_wide[kStepMaxPrefixes],
      g_nar[kStepMaxPrefixes];
  __shared__ int64_t tmp64[kPlanThreads / 64];
  __shared__ int tmp[kPlanThreads / 64];
  __shared__ int st_unit[2 * (kStepMaxWorkers + 1)], st_step[2 * (kStepMaxWorkers + 1)];
  __shared__ int n_cut[2];
  __shared__ unsigned long long more[2];  // modelled time of the sources above kNarrowMost rows: wide, narrow

  const int tid = threadIdx.x;
  const int B = a.s.batch, NP = a.s.prefixes, rep = a.s.hq / a.s.hkv, hkv = a.s.hkv;
  const int tokens = static_cast<int>(a.s.tokens);
  StepHead* head = reinterpret_cast<StepHead*>(a.plan);
  StepTile* tiles = reinterpret_cast<StepTile*>(a.plan + a.l.tiles);
  int64_t* cum_w = reinterpret_cast<int64_t*>(a.plan + a.l.cum_wide);
  int64_t* cum_n = reinterpret_cast<int64_t*>(a.plan + a.l.cum_narrow);
  StepShared* shared = reinterpret_cast<StepShared*>(a.plan + a.l.shared);
  int32_t* starts = reinterpret_cast<int32_t*>(a.plan + a.l.starts);
  int32_t* cuts = reinterpret_cast<int32_t*>(a.plan + a.l.cuts);
  StepCut* cut_wide = reinterpret_cast<StepCut*>(a.plan + a.l.cut_wide);
  StepCut* cut_narrow = reinterpret_cast<StepCut*>(a.plan + a.l.cut_narrow);
  auto flag = [&] { atomicOr(a.err, 8); };
  auto prefix_len = [&](int p) {  // of prefix p, within its table
    const int64_t n = a.prefix_lens[p];
    return static_cast<int>(n < 0 ? 0 : n > a.s.max_prefix ? a.s.max_prefix : n);
  };

  // ---- sequences: tokens within the query, lengths within their tables ----
  for (int p = tid; p < NP; p += kPlanThreads) {
    g_seq[p] = g_tok[p] = 0;
    const int n = a.prefix_lens[p];
    if (n < 0 || n > a.s.max_prefix) flag();
  }
  if (tid < 2) n_cut[tid] = more[tid] = 0;
  int falls = 0;
  for (int b = tid; b < B; b += kPlanThreads) falls |= a.token_starts[b + 1] < a.token_starts[b];
  falls = __syncthreads_or(falls);
  for (int b = tid; b < B; b += kPlanThreads) {
    int t0 = a.token_starts[b], t1 = a.token_starts[b + 1];
    if (t0 < 0 || t1 < t0) {
      flag();
      t0 = t1 = 0;
    }
    // Where the starts fall somewhere, a later sequence may name the tokens of an earlier one again: it
    // keeps those behind all earlier starts, since the plan has room for every token once.
    if (falls) {
      for (int c = 0; c < b; ++c) t0 = max(t0, a.token_starts[c]);
      t1 = max(t0, t1);
    }
    int64_t len = a.seq_lens[b];
    if (len < 0 || len > a.s.max_own) {
      flag();
      len = len < 0 ? 0 : a.s.max_own;
    }
    const int n = min(t1, tokens) - min(t0, tokens);
    int pid = NP > 0 && a.prefix_ids != nullptr ? a.prefix_ids[b] : -1;
    if (pid < -1 || pid >= NP) {
      flag();
      pid = -1;
    }
    if (pid >= 0 && prefix_len(pid) == 0) pid = -1;
    s_tok[b] = min(t0, tokens);
    s_n[b] = n;
    s_len[b] = static_cast<int>(len);
    // own keys that the sequence's first token sees (its last one sees all)
    s_vis[b] = a.s.causal ? static_cast<int>(max(len - (static_cast<int64_t>(t1) - t0) + 1, static_cast<int64_t>(INT32_MIN / 2)))
                          : static_cast<int>(len);
    s_pid[b] = pid;
    const bool narrow = n > 0 && static_cast<int64_t>(n) * rep <= kNarrowMost;
    if (narrow && pid >= 0) {
      atomicAdd(&g_seq[pid], 1);
      atomicAdd(&g_tok[pid], n);
    }
  }
  __syncthreads();
  // ---- prefixes with tokens of several sequences behind them; which sources are wide ----
  auto weigh = [&](int64_t rows, int64_t keys) {
    if (rows <= kNarrowMost) return;
    atomicAdd(&more[0], static_cast<unsigned long long>((rows + kWideRows - 1) / kWideRows * (kWideFixed + (keys + kWideKeys - 1) / kWideKeys * kWideStep)));
    atomicAdd(&more[1], static_cast<unsigned long long>((rows + kNarrowRows - 1) / kNarrowRows * (kNarrowFixed + (keys + 255) / 256 * kNarrowStep)));
  };
  for (int p = tid; p < NP; p += kPlanThreads) {
    const bool on = g_seq[p] >= 2;
    if (!on) g_seq[p] = 0;
    else weigh(static_cast<int64_t>(g_tok[p]) * rep, prefix_len(p));
    g_list[p] = on ? g_tok[p] : 0;
  }
  for (int b = tid; b < B; b += kPlanThreads)
    if (s_n[b] > 0)
      weigh(static_cast<int64_t>(s_n[b]) * rep,
            (s_pid[b] >= 0 ? prefix_len(s_pid[b]) : 0) + max(s_len[b] - (a.s.causal ? s_n[b] / 2 : 0), 0));
  __syncthreads();
  const int64_t narrow_more = static_cast<int64_t>(more[1] - more[0]) * hkv / a.workers;
  const int64_t most = narrow_more <= kNarrowMore ? INT64_MAX : kNarrowMost;  // rows of a source in narrow tiles
  for (int p = tid; p < NP; p += kPlanThreads) {
    const int rows = g_list[p] * rep;
    g_wide[p] = rows > most ? (rows + kWideRows - 1) / kWideRows : 0;
    g_nar[p] = rows <= most ? (rows + kNarrowRows - 1) / kNarrowRows : 0;
  }
  __syncthreads();
  const int n_shared = NP > 0 ? scan_lds(g_list, NP, tmp) : 0;
  const int pre_wide = NP > 0 ? scan_lds(g_wide, NP, tmp) : 0;
  const int pre_nar = NP > 0 ? scan_lds(g_nar, NP, tmp) : 0;
  for (int b = tid; b < B; b += kPlanThreads) {
    const int64_t rows = static_cast<int64_t>(s_n[b]) * rep;
    s_wide[b] = rows > most ? static_cast<int>((rows + kWideRows - 1) / kWideRows) : 0;
    s_nar[b] = rows <= most ? static_cast<int>((rows + kNarrowRows - 1) / kNarrowRows) : 0;
  }
  __syncthreads();
  const int n_wide = pre_wide + scan_lds(s_wide, B, tmp);
  const int n_nar = pre_nar + scan_lds(s_nar, B, tmp);

  // ---- the list of tokens behind shared prefixes ----
  for (int b = tid; b < B; b += kPlanThreads) {
    const int n = s_n[b], p = s_pid[b];
    s_list[b] = -1;
    if (n == 0 || p < 0 || g_seq[p] == 0 || static_cast<int64_t>(n) * rep > kNarrowMost) continue;
    int at = g_list[p];  // behind the earlier sequences of the same prefix
#pragma unroll 8
    for (int c = 0; c < b; ++c) {
      const int there = s_pid[c], k = s_n[c];
      at += there == p && k <= kNarrowMost / rep ? k : 0;
    }
    const int wide = static_cast<int64_t>(g_tok[p]) * rep > most;
    for (int i = 0; i < n; ++i)
      shared[at + i] = StepShared{s_tok[b] + i, pre_nar + s_nar[b], i * rep, wide ? g_wide[p] : g_nar[p], (at + i - g_list[p]) * rep, wide, {0, 0}};
    s_list[b] = at;
  }
  __syncthreads();
  const int vstep = a.s.causal ? 1 : 0;
  // rows row0 .. of a sequence or of a prefix's tokens as a tile of up to `size` rows
  auto own_tile = [&](int b, int row0, int size) {
    StepTile t{};
    const int p = s_pid[b];
    const bool shares = s_list[b] >= 0;
    t.tok0 = s_tok[b];
    t.row0 = row0;
    t.rows = min(size, s_n[b] * rep - row0);
    t.p_row = max(p, 0);
    t.p_len = p >= 0 && !shares ? prefix_len(p) : 0;
    t.s_row = b;
    t.s_len = max(0, min(s_len[b], s_vis[b] + (row0 + t.rows - 1) / rep * vstep));
    t.vis0 = s_vis[b];
    t.vis_step = vstep;
    t.dest = shares ? kToOwn : kToOut;
    t.list0 = max(s_list[b], 0);
    return t;
  };
  auto prefix_tile = [&](int p, int row0, int size) {
    StepTile t{};
    t.tok0 = t.list0 = g_list[p];
    t.list = 1;
    t.row0 = row0;
    t.rows = min(size, g_tok[p] * rep - row0);
    t.p_row = p;
    t.p_len = prefix_len(p);
    t.dest = kToPrefix;
    return t;
  };
  // ---- narrow tiles, one a thread ----
  for (int i = tid; i < n_nar; i += kPlanThreads) {
    StepTile t;
    if (i < pre_nar) {
      const int p = last_at_most(g_nar, NP, i);
      t = prefix_tile(p, (i - g_nar[p]) * kNarrowRows, kNarrowRows);
    } else {
      const int b = last_at_most(s_nar, B, i - pre_nar);
      t = own_tile(b, (i - pre_nar - s_nar[b]) * kNarrowRows, kNarrowRows);
    }
    t.steps = max(1, ((t.p_len + 31) / 32 + (t.s_len + 31) / 32 + kStepWaves - 1) / kStepWaves);
    tiles[n_wide + i] = t;
  }
  // ---- wide tiles, one a thread.  Those of sequences are laid out column by column: dealt to the
  // columns (the workers of a kv head) to and fro, the last of a sequence first, so that a worker
  // starts with a long tile and all get about as much; the workgroups of an XCD then go through
  // the keys side by side and find them in its L2 (a prompt of 16384 tokens, 32/8 heads: 2.16 ms in
  // the order of the rows, 2.04 so). ----
  const int own_wide = n_wide - pre_wide, cols = max(1, min(own_wide, a.workers / hkv)), rounds = (own_wide + cols - 1) / cols;
  const int rest = own_wide - (rounds - 1) * cols;  // tiles of the last round
  for (int i = tid; i < n_wide; i += kPlanThreads) {
    StepTile t;
    if (i < pre_wide) {
      const int p = last_at_most(g_wide, NP, i);
      t = prefix_tile(p, (i - g_wide[p]) * kWideRows, kWideRows);
    } else {
      const int b = last_at_most(s_wide, B, i - pre_wide);
      t = own_tile(b, (i - pre_wide - s_wide[b]) * kWideRows, kWideRows);
    }
    t.steps = max(1, (t.p_len + kWideKeys - 1) / kWideKeys + (t.s_len + kWideKeys - 1) / kWideKeys);
    int to = i;
    if (i >= pre_wide) {
      const int k = n_wide - 1 - i, r = k / cols, c = r & 1 ? cols - 1 - k % cols : k % cols;
      to = pre_wide + c * (rounds - 1) + (rounds & 1 ? min(c, rest) : max(0, c - (cols - rest))) + r;
    }
    tiles[to] = t;
  }
  const int units_w = n_wide * hkv, units = units_w + n_nar * hkv;
  for (int i = tid; i < units; i += kPlanThreads) cuts[i] = 0;
  __syncthreads();

  // ---- the two axes, and every worker's start on them: worker w of the wide ones at w, of the
  // narrow ones at W + 1 + w, the ends behind each ----
  const int64_t all_w = scan_costs(cum_w, n_wide, [&](int i) { return static_cast<int64_t>(kWideFixed + tiles[i].steps * kWideStep); }, tmp64);
  const int64_t all_n = scan_costs(cum_n, n_nar, [&](int i) { return static_cast<int64_t>(kNarrowFixed + tiles[n_wide + i].steps * kNarrowStep); }, tmp64);
  const int W = a.workers;
  // Each XCD's workers (a run of W / 8) take an eighth of both axes: the wide part first, so that
  // all but one of them have units of one kind.
  const int slices = W % kXcds == 0 ? kXcds : 1, per = W / slices;
  const int64_t share = max(((all_w + all_n) * hkv + W - 1) / W, static_cast<int64_t>(kLeastShare));
  const int64_t slack = share / 64;
  for (int i = tid; i < 2 * (W + 1); i += kPlanThreads) {
    const bool narrow = i > W;
    const int w = narrow ? i - W - 1 : i;
    const int64_t all = narrow ? all_n : all_w, total = all * hkv;
    const int xcd = w / per;
    const int64_t w0 = all_w * hkv * xcd / slices, w1 = all_w * hkv * (xcd + 1) / slices;
    const int64_t n0 = all_n * hkv * xcd / slices, n1 = all_n * hkv * (xcd + 1) / slices, p = share * (w - xcd * per);
    const int64_t x = narrow ? min(n1, n0 + max(p - (w1 - w0), static_cast<int64_t>(0))) : min(w1, w0 + p);
    int unit = narrow ? units : units_w, step = 0;
    if (w < W && x < total) {
      int t, fixed, each;
      int64_t off;
      if (!narrow) {
        const int kvh = static_cast<int>(x / all_w);
        const int64_t y = x - kvh * all_w;
        t = last_at_most(cum_w, n_wide, y);
        off = y - cum_w[t];
        unit = kvh * n_wide + t;
        fixed = kWideFixed;
        each = kWideStep;
      } else {
        const int k = last_at_most(cum_n, n_nar, x / hkv);
        const int64_t cost = cum_n[k + 1] - cum_n[k], z = x - cum_n[k] * hkv;
        const int kvh = static_cast<int>(z / cost);
        t = n_wide + k;
        off = z - kvh * cost;
        unit = units_w + k * hkv + kvh;
        fixed = kNarrowFixed;
        each = kNarrowStep;
      }
      // a cut so near a unit's end that it costs more than it evens out is moved there
      step = off <= fixed + slack ? 0 : static_cast<int>((off - fixed + each / 2) / each);
      if (step > 0 && static_cast<int64_t>(tiles[t].steps - step) * each <= slack) {
        ++unit;
        step = 0;
      }
    }
    st_unit[i] = unit;
    st_step[i] = step;
    starts[2 * i] = unit;
    starts[2 * i + 1] = step;
  }
  __syncthreads();
  // ---- units that several workers share: the first of them and their number ----
  for (int i = tid; i < 2 * (W + 1); i += kPlanThreads) {
    const int unit = st_unit[i];
    if (st_step[i] == 0 || (st_unit[i - 1] == unit && st_step[i - 1] > 0)) continue;  // an axis starts at step 0
    int k = i + 1;
    while (st_unit[k] == unit) ++k;
    const int cut = i | (k - i + 1) << 16;  // first worker's place + 1, workers
    cuts[unit] = cut;
    const bool wide = unit < units_w;
    const int ti = wide ? unit % n_wide : n_wide + (unit - units_w) / hkv, kvh = wide ? unit / n_wide : (unit - units_w) % hkv;
    const StepTile& t = tiles[ti];
    if (t.dest == kToOut)
      (wide ? cut_wide : cut_narrow)[atomicAdd(&n_cut[wide ? 0 : 1], 1)] = StepCut{cut, t.row0, t.rows, t.tok0, kvh * rep, {0, 0, 0}};
  }
  __syncthreads();
  if (tid == 0)
    *head = StepHead{kPlanMagic, B, tokens, a.s.hq, hkv, a.s.d, a.s.bs, a.s.causal, NP, static_cast<int>(a.s.max_own),
                     static_cast<int>(a.s.max_prefix), W, n_wide, n_nar, n_shared, n_cut[0], n_cut[1], {0, 0, 0}};
}

void launch_step_plan(const StepShape& s, const int32_t* token_starts, const int32_t* seq_lens, const int32_t* prefix_ids,
                      const int32_t* prefix_lens, void* plan, int* err, hipStream_t stream) {
  const PlanKernelArgs a{s, step_workers(), token_starts, seq_lens, prefix_ids, prefix_lens, static_cast<char*>(plan), plan_layout(s), err};
  step_plan_kernel<<<1, kPlanThreads, 0, stream>>>(a);
  HCP_HIP(hipGetLastError());
}

// ----------------------------------------------------------------------------------
// Attention
// ----------------------------------------------------------------------------------
struct StepArgs {
  const char* plan;
  size_t p_tiles, p_shared, p_starts, p_cuts, p_cut_wide, p_cut_narrow;
  StepShape s;
  int32_t workers;
  const uint16_t* q;
  int64_t q_hs, q_ss;
  const uint16_t* pool;
  int64_t plane_bytes, num_blocks;
  int32_t rep;
  uint32_t gpb, gpb_inv, block_bytes;  // 16-token groups of a block, (2^32 - 1) / gpb, bytes of a block in a plane
  const int32_t *tables, *prefix_tables;
  int64_t table_stride, prefix_stride;
  float scale_log2;
  void* out;
  int64_t out_hs, out_ss;
  int32_t out_dtype;
  float* lse;  // [hq, tokens] or null
  float *slot_o, *slot_lse, *own_o, *own_lse, *pre_o, *pre_lse;
  int32_t slot_rows;
  int* err;
};

namespace {

// Wave-uniform reads through scalar loads: they wait on a counter of their own, not on the
// K / V loads in flight.
typedef const __attribute__((address_space(4))) int32_t* scalar_i32;
__device__ __forceinline__ scalar_i32 scalar_ptr(const void* p) {
  return (scalar_i32)(reinterpret_cast<uintptr_t>(p));
}

__device__ __forceinline__ void wait_dma(int left) {  // at most `left` (0 or one K or V part) still in flight
  if (left == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  else if (left == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else if (left == 2) asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Bytes of LDS: the wide tiles' rings (2 K + 3 V of 128 rows); the narrow tiles' 8 x 64 rows,
// then their 8 results of 32 rows, fit within.
template <int DW>
constexpr int kStepLds = 5 * kWideKeys * DW * 2;

// A group of 16 keys of the paged cache: its block's id as the table has it, its first token's
// place in the block and how many of its tokens count.
struct KeyGroup {
  int id, slot, rows;
};

// The kernel's arguments as they lie in memory.  Read through `again`, a value is loaded where
// it is used, not kept in scalar registers across a unit's loop.
typedef const __attribute__((address_space(4))) StepArgs* args_ptr;
__device__ __forceinline__ args_ptr again(args_ptr a) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+s"(a));
#endif
  return a;
}

// What the loads of a unit go by.  All of it is the same for a wave's lanes: some 30 scalar
// instructions a 16-key group, which the wide tiles' loop has to fit beside its softmax.
struct StepKeys {
  scalar_i32 p_tab, s_tab;  // table rows of the tile
  int p_len, s_len;
  uint64_t base;            // the kv head's first K row of block 0
  int64_t plane_bytes;
  uint32_t num_blocks, gpb, gpb_inv, block_bytes;
  int row_bytes, span_bytes;  // span_bytes: of a row's head
  bool bad;                   // a block id outside the pool was met
  StepKeys() = default;
  __device__ __forceinline__ StepKeys(args_ptr a, const StepTile& t, int kvh)
      : p_tab(scalar_ptr(a->prefix_tables + t.p_row * a->prefix_stride)), s_tab(scalar_ptr(a->tables + t.s_row * a->table_stride)),
        p_len(t.p_len), s_len(t.s_len), base(reinterpret_cast<uint64_t>(a->pool) + static_cast<uint64_t>(kvh) * a->s.d * 2),
        plane_bytes(a->plane_bytes), num_blocks(static_cast<uint32_t>(a->num_blocks)), gpb(a->gpb), gpb_inv(a->gpb_inv),
        block_bytes(a->block_bytes), row_bytes(a->s.hkv * a->s.d * 2), span_bytes(a->s.d * 2), bad(false) {}
  // The group at key0 of the prefix or the own keys.  Its table entry is (key0 / 16) / gpb: the
  // product with floor((2^32 - 1) / gpb) is at most one too low.
  __device__ __forceinline__ KeyGroup fetch(bool pre, int key0) const {
    const uint32_t g = static_cast<uint32_t>(key0) >> 4;
    uint32_t e = __umulhi(g, gpb_inv), r = g - e * gpb;
    if (r >= gpb) {
      ++e;
      r -= gpb;
    }
    const int rows = min((pre ? p_len : s_len) - key0, 16);
    return {rows > 0 ? (pre ? p_tab : s_tab)[e] : 0, static_cast<int>(r << 4), max(rows, 0)};
  }
  // Buffer descriptors of its K and V rows; rows past the last that counts, and all of a bad
  // block, lie out of range and give zeros.
  __device__ __forceinline__ void srd(const KeyGroup& g, u32x4& k, u32x4& v) {
    const bool ok = static_cast<uint32_t>(g.id) < num_blocks;
    bad = bad || !ok;
    const uint64_t at = base + static_cast<uint64_t>(static_cast<uint32_t>(g.id)) * block_bytes + static_cast<uint32_t>(g.slot * row_bytes);
    const uint32_t bytes = ok && g.rows > 0 ? static_cast<uint32_t>((g.rows - 1) * row_bytes + span_bytes) : 0u;
    const uint64_t vat = at + plane_bytes;
    k[0] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
    k[1] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32) & 0xffffu);
    v[0] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(vat));
    v[1] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(vat >> 32) & 0xffffu);
    k[2] = v[2] = __builtin_amdgcn_readfirstlane(bytes);
    k[3] = v[3] = 0x00020000u;
  }
  __device__ __forceinline__ void report(args_ptr a) const {
    if (bad && (threadIdx.x & 63) == 0) atomicOr(again(a)->err, 1);
  }
};

// Destination of row r of a unit: element offsets of its output row and its LSE.
struct RowDest {
  void* o;
  int dtype;
  int64_t o_off;
  float* lse;
};
__device__ __forceinline__ RowDest row_dest(args_ptr a, const StepTile& t, int kvh, int slot, int row, int token, int i, int h) {
  const int head = kvh * a->rep + h, d = a->s.d;
  if (slot >= 0) {
    const int64_t at = static_cast<int64_t>(slot) * a->slot_rows + row;
    return {a->slot_o, kF32, at * d, a->slot_lse + at};
  }
  if (t.dest == kToOut)
    return {a->out, a->out_dtype, head * a->out_hs + token * a->out_ss, a->lse != nullptr ? a->lse + head * a->s.tokens + token : nullptr};
  const int64_t at = static_cast<int64_t>(t.list0 + i) * a->s.hq + head;
  return t.dest == kToOwn ? RowDest{a->own_o, kF32, at * d, a->own_lse + at} : RowDest{a->pre_o, kF32, at * d, a->pre_lse + at};
}

// Row `row` of a tile: token i of its source and query head h of the group, and the token's row
// of the query.
struct RowOf {
  int i, h, token;
};
__device__ __forceinline__ RowOf row_of(args_ptr a, const StepTile& t, int row) {
  const int r = t.row0 + min(row, t.rows - 1), i = r / a->rep;
  int token = t.tok0 + i;
  if (t.list) token = reinterpret_cast<const StepShared*>(a->plan + a->p_shared)[token].token;
  return {i, r - i * a->rep, token};
}

__device__ __forceinline__ StepTile read_tile(args_ptr a, int ti) {
  const scalar_i32 tp = scalar_ptr(a->plan + a->p_tiles) + ti * 16;
  StepTile t;
  t.tok0 = tp[0]; t.row0 = tp[1]; t.rows = tp[2]; t.p_row = tp[3]; t.p_len = tp[4]; t.s_row = tp[5]; t.s_len = tp[6];
  t.vis0 = tp[7]; t.vis_step = tp[8]; t.steps = tp[9]; t.dest = tp[10]; t.list0 = tp[11]; t.list = tp[12];
  return t;
}

// Own keys that token i of the tile's source sees.
__device__ __forceinline__ int sees(const StepTile& t, int i) { return min(max(t.vis0 + i * t.vis_step, 0), t.s_len); }

// An opaque copy: what is worked out from it stays where it is used.  Hoisted out of the loops, the
// lane constants of a unit's loads and stores are registers that the wide tiles do not have: they
// went through scratch memory, whose loads wait for the K and V loads before them (a prompt of
// 16384 tokens, 32/8 heads, 4.4 ms so).
template <typename T>
__device__ __forceinline__ T fresh(T x) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(x));
#endif
  return x;
}
__device__ __forceinline__ uint32_t fresh_lane() {
  return fresh(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)));
}

// Where a lane reads and writes K and V rows in LDS: the swizzles and fragment addresses of the
// ring kernels (rows of 256 or 128 bytes).  A group of 16 keys takes NJ loads of RPI rows
// (1 KiB); load j holds row j RPI + r0 in lane r0 CPR + p, whose chunk is p ^ swizzle(row).
template <int DW>
struct StepLanes {
  static constexpr int PW = DW * 2, CPR = PW / 16, RPI = 1024 / PW, NJ = 16 / RPI, DB = DW / 32;
  uint32_t k_rd, v_rd0;
  __device__ __forceinline__ explicit StepLanes(int lane) {
    const int krow = kperm(lane & 31), g16 = lane >> 4, sl = lane & 15;
    k_rd = krow * PW + (((lane >> 5) ^ (PW == 256 ? (krow & 15) : ((krow >> 1) & 7))) << 4);
    const int vs = PW == 256 ? (sl >> 2) : ((sl >> 3) & 1);
    v_rd0 = (8 * (g16 >> 1) + (sl >> 2)) * PW + ((4 * vs + 2 * (g16 & 1) + ((sl & 3) >> 1)) << 4) + 8 * (sl & 1);
  }
  // The NJ loads of a group's K or V rows to LDS at `to`: the K swizzle of row j RPI + r0 is that
  // of r0 with bits 2 and 3 of the chunk flipped by j, the V swizzle the same for all j.  With
  // PAD (a head dim below DW) chunks past span_bytes lie out of range and give zeros.
  template <bool PAD>
  static __device__ __forceinline__ void load_k(u32x4 srd, uint32_t to, uint32_t row_bytes, uint32_t span_bytes) {
    const uint32_t lane = fresh_lane(), r0 = lane / CPR, c0 = ((lane % CPR) ^ (PW == 256 ? r0 : r0 >> 1)) << 4, row0 = r0 * row_bytes;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint32_t ch = c0 ^ (j << 6);
      dma16(srd, !PAD || ch < span_bytes ? ch + row0 + j * RPI * row_bytes : 0x80000000u, to + j * 1024);
    }
  }
  template <bool PAD>
  static __device__ __forceinline__ void load_v(u32x4 srd, uint32_t to, uint32_t row_bytes, uint32_t span_bytes) {
    const uint32_t lane = fresh_lane(), r0 = lane / CPR, ch = ((lane % CPR) ^ (PW == 256 ? 4 * r0 : 4 * ((r0 >> 1) & 1))) << 4;
    const uint32_t v0 = !PAD || ch < span_bytes ? ch + r0 * row_bytes : 0x80000000u;
#pragma unroll
    for (int j = 0; j < NJ; ++j) dma16(srd, v0 + j * RPI * row_bytes, to + j * 1024);
  }
  // LDS byte of this lane's half of the V^T fragment of dims 32 b .. + 31, key step 0
  static __device__ __forceinline__ uint32_t v_rd(uint32_t rd0, int b) { return rd0 ^ (b << 6); }
};

// Q fragments of a row: dims 16 s + 8 (lane / 32) .. + 7 of step s, zeros past the head dim.
template <int DT, int DW, bool PAD>
__device__ __forceinline__ void load_q(args_ptr a, const RowOf& r, int kvh, int lhalf, typename MfmaOps<DT>::frag (&qf)[DW / 16]) {
  const int dn = a->s.d;
  const uint16_t* qrow = a->q + (kvh * a->rep + r.h) * a->q_hs + r.token * a->q_ss;
  u32x4 x[DW / 16];
#pragma unroll
  for (int s = 0; s < DW / 16; ++s) {
    const int at = 16 * s + 8 * lhalf;
    x[s] = *reinterpret_cast<const u32x4*>(qrow + (!PAD || at < dn ? at : 0));
  }
#pragma unroll
  for (int s = 0; s < DW / 16; ++s)
    qf[s] = as_frag<typename MfmaOps<DT>::frag>(!PAD || 16 * s + 8 * lhalf < dn ? x[s] : u32x4{0u, 0u, 0u, 0u});
}

// The largest weight of a row is 2^kBias where its maximum was last taken, and no sum of a lane's
// weights passes kMostSum: f16 holds weights down to 2^-31 of the largest so, whose sum over a long
// row is still within fp32's needs (with the largest at 1 all below 2^-24 were lost).
template <int DT>
constexpr float kBias = DT == kF16 ? 7.f : 0.f;
template <int DT>
constexpr float kMostSum = kGrowSum * (DT == kF16 ? 128.f : 1.f);

template <int DT>
__device__ __forceinline__ float frag_value(typename MfmaOps<DT>::frag f, int i) {
  return static_cast<float>(f[i]);
}

}  // namespace

// Where a worker's units of one kind start and end.
struct StepRun {
  int n_wide, unit, step, end_unit, end_step;
  __device__ __forceinline__ StepRun(args_ptr a, int place) {
    const scalar_i32 s = scalar_ptr(a->plan + a->p_starts) + 2 * place;
    n_wide = scalar_ptr(a->plan)[12];
    unit = s[0];
    step = s[1];
    end_unit = s[2];
    end_step = s[3];
  }
};

// The narrow units of the worker at `place` of the plan's starts.  TN: terms of 16 bits in which
// a softmax weight enters the product with V.
template <int DT, int DW, bool PAD, int TN>
__device__ __forceinline__ void step_narrow(args_ptr a, const StepRun& run, int place, char* lds) {
  using Ops = MfmaOps<DT>;
  using frag = typename Ops::frag;
  using Lanes = StepLanes<DW>;
  constexpr int KS = DW / 16, DB = Lanes::DB, PW = Lanes::PW, NJ = Lanes::NJ;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lcol = lane & 31, lhalf = lane >> 5;
  const int n_wide = run.n_wide, end_unit = run.end_unit, end_step = run.end_step;
  const Lanes at(lane);
  const uint32_t lds0 = lds_offset(lds);
  const float c = a->scale_log2;
  auto some = [&](int unit, int step) __attribute__((always_inline)) { return unit < end_unit || (unit == end_unit && step < end_step); };
  int unit = run.unit;
  if (!some(unit, run.step)) return;
  constexpr int kDma = 2 * NJ;
  constexpr int kStage = kStepWaves * 64 * PW;  // LDS: 32 K and 32 V rows of each wave, then the small results
  const uint32_t kbuf = lds0 + wave * (64 * PW), vbuf = kbuf + 32 * PW;

  // ---- the unit being worked on ----
  StepTile t;
  int kvh, slot, np, ng, g;       // this wave's groups of 32 keys: g, g + 8, ..., the first np of the unit's of the prefix
  int vis, vis_min;               // own keys that this lane's row and the tile's first row see
  StepKeys keys;
  frag qf[KS];
  KeyGroup n0, n1;                // the two 16-key groups to load next
  u32x4 ks0, ks1, vs0, vs1;       // descriptors of those being loaded
  auto key_of = [&](int g) __attribute__((always_inline)) { return 32 * (g < np ? g : g - np); };
  auto fetch = [&](int g) __attribute__((always_inline)) {
    if (g >= ng) return;
    n0 = keys.fetch(g < np, key_of(g));
    n1 = keys.fetch(g < np, key_of(g) + 16);
  };
  auto locate = [&] __attribute__((always_inline)) {
    keys.srd(n0, ks0, vs0);
    keys.srd(n1, ks1, vs1);
  };
  auto load_k = [&] __attribute__((always_inline)) {
    Lanes::template load_k<PAD>(ks0, kbuf, keys.row_bytes, keys.span_bytes);
    Lanes::template load_k<PAD>(ks1, kbuf + NJ * 1024, keys.row_bytes, keys.span_bytes);
  };
  auto load_v = [&] __attribute__((always_inline)) {
    Lanes::template load_v<PAD>(vs0, vbuf, keys.row_bytes, keys.span_bytes);
    Lanes::template load_v<PAD>(vs1, vbuf + NJ * 1024, keys.row_bytes, keys.span_bytes);
  };
  // Takes up a unit from step s0 on: its first keys are on their way when this returns.
  auto begin = [&](int u, int s0) __attribute__((always_inline)) {
    const args_ptr b0 = again(a);
    const int un = u - n_wide * b0->s.hkv, ti = un / b0->s.hkv;
    kvh = un - ti * b0->s.hkv;
    t = read_tile(b0, n_wide + ti);
    const int s1 = u == end_unit ? min(end_step, t.steps) : t.steps;
    slot = s0 > 0 ? 2 * place : s1 < t.steps ? 2 * place + 1 : -1;
    np = (t.p_len + 31) >> 5;
    ng = min(np + ((t.s_len + 31) >> 5), s1 * kStepWaves);
    g = s0 * kStepWaves + wave;
    keys = StepKeys(b0, t, kvh);
    fetch(g);
    const RowOf mine = row_of(b0, t, lcol);
    load_q<DT, DW, PAD>(b0, mine, kvh, lhalf, qf);
    vis = sees(t, mine.i);
    vis_min = sees(t, t.row0 / b0->rep);
    if (g < ng) {
      locate();
      load_k();
      load_v();
      fetch(g + kStepWaves);
    }
  };
  __syncthreads();  // the wide units' reads of LDS are over
  begin(unit, run.step);
  while (true) {
    f32x16 oacc[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[b][r] = 0.f;
    float m_run = kInitMax, l_run = 0.f;
    bool first = true;
    for (; g < ng; g += kStepWaves) {
      const bool more = g + kStepWaves < ng;
      const bool own = g >= np;
      const int key0 = key_of(g), end = own ? t.s_len : t.p_len;
      wait_dma(kDma);  // K is there, V may still be on its way
      f32x16 sacc;
#pragma unroll
      for (int r = 0; r < 16; ++r) sacc[r] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const frag kf = as_frag<frag>(*reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
            static_cast<uintptr_t>((kbuf + at.k_rd) ^ static_cast<uint32_t>(s << 5))));
        sacc = Ops::mma(kf, qf[s], sacc);
      }
      pin(sacc);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K's last reads are done
      if (more) {
        locate();
        load_k();
        fetch(g + 2 * kStepWaves);
      }
      if (end - key0 < 32 || (own && vis_min < key0 + 32)) {
        const int lim = min(end - key0, own ? vis - key0 : 32) - 1 - 8 * lhalf;
#pragma unroll
        for (int r = 0; r < 16; ++r) sacc[r] = 16 * (r >> 3) + 4 * ((r >> 2) & 1) + (r & 3) <= lim ? sacc[r] : -INFINITY;
      }
      float p[16];
      auto weigh = [&] __attribute__((always_inline)) {
        float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[r], c, -m_run));
          l4[r & 3] += p[r];
        }
        return (l4[0] + l4[1]) + (l4[2] + l4[3]);
      };
      float lsum = 0.f;
      bool redo = first;
      if (!redo) {
        lsum = weigh();
        redo = __any(!(lsum <= kMostSum<DT>));
      }
      if (redo) {
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, sacc[r]);
        const float m_new = fmaxf(m_run, max_xor32(top) * c - kBias<DT>);
        const float alpha = exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[b][r] *= alpha;
        m_run = m_new;
        lsum = weigh();
      }
      l_run += lsum;
      first = false;
      wait_dma(more ? kDma : 0);  // V is there
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        frag pf[TN];
        float rest[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] = p[8 * s + i];
#pragma unroll
        for (int k = 0; k < TN; ++k) {
          pf[k] = Ops::pack(rest);
#pragma unroll
          for (int i = 0; i < 8; ++i) rest[i] -= frag_value<DT>(pf[k], i);
        }
#pragma unroll
        for (int b = 0; b < DB; ++b) {
          const char* p0 = lds + (vbuf - lds0) + Lanes::v_rd(at.v_rd0, b) + s * 16 * PW;
          const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p0));
          const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p0 + 4 * PW));
          const u32x2 lo2 = __builtin_bit_cast(u32x2, lo), hi2 = __builtin_bit_cast(u32x2, hi);
          const frag vf = as_frag<frag>(u32x4{lo2[0], lo2[1], hi2[0], hi2[1]});
#pragma unroll
          for (int k = 0; k < TN; ++k) oacc[b] = Ops::mma(vf, pf[k], oacc[b]);
        }
      }
#pragma unroll
      for (int b = 0; b < DB; ++b) pin(oacc[b]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) load_v();
    }
    keys.report(a);
    // ---- the waves' results meet in LDS: [wave][row][DW + 4] and m, l of every row.  Few rows
    // meet behind the waves' K and V, up to kFew at a time, while the next unit's first keys load
    // there; more take the place of K and V, all at once ----
    constexpr int OS = DW + 4, kFew = 7;
    static_assert(kStage + kStepWaves * kFew * (OS + 2) * 4 <= kStepLds<DW> && kStepWaves * kNarrowRows * (OS + 2) * 4 <= kStepLds<DW>,
                  "results fit");
    const StepTile et = t;
    const int ekvh = kvh, eslot = slot;
    const bool few = et.rows <= 2 * kFew, more_units = some(++unit, 0);
    if (few && more_units) begin(unit, 0);
    const int most = few ? kFew : kNarrowRows;
    float* const os = reinterpret_cast<float*>(lds + (few ? kStage : 0));
    float* const ml = os + kStepWaves * most * OS;
    const float l_tot = sum_xor32(l_run);
    const args_ptr e = again(a);
    for (int r0 = 0; r0 < et.rows; r0 += most) {
      const int n_rows = min(most, et.rows - r0);
      __syncthreads();  // earlier reads of this place are over
      const int lr = lcol - r0;
      if (lr >= 0 && lr < n_rows) {
        if (lhalf == 0) {
          ml[(wave * most + lr) * 2] = m_run;
          ml[(wave * most + lr) * 2 + 1] = l_tot;
        }
        if (l_tot != 0.f) {
#pragma unroll
          for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<f32x4*>(os + (wave * most + lr) * OS + 32 * b + 8 * j + 4 * lhalf) =
                  f32x4{oacc[b][4 * j], oacc[b][4 * j + 1], oacc[b][4 * j + 2], oacc[b][4 * j + 3]};
        }
      }
      __syncthreads();
      for (int i = tid; i < n_rows * (DW / 4); i += kStepThreads) {
        const int r = i / (DW / 4), d = i - r * (DW / 4);
        if (PAD && 4 * d >= e->s.d) continue;
        float m = kInitMax;
#pragma unroll
        for (int w = 0; w < kStepWaves; ++w) m = fmaxf(m, ml[(w * most + r) * 2]);
        float den = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kStepWaves; ++w) {
          const float lw = ml[(w * most + r) * 2 + 1];
          if (lw == 0.f) continue;  // took no key
          const float f = exp2f(ml[(w * most + r) * 2] - m);
          den += f * lw;
          const f32x4 o = *reinterpret_cast<const f32x4*>(os + (w * most + r) * OS + 4 * d);
#pragma unroll
          for (int k = 0; k < 4; ++k) x[k] += f * o[k];
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const RowOf ro = row_of(e, et, r0 + r);
        const RowDest dst = row_dest(e, et, ekvh, eslot, r0 + r, ro.token, ro.i, ro.h);
        store4(dst.o, dst.dtype, dst.o_off + 4 * d, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        if (d == 0 && dst.lse != nullptr) *dst.lse = den == 0.f ? -INFINITY : (m + __log2f(den)) * kLn2;
      }
    }
    if (!more_units) return;
    if (!few) {
      __syncthreads();
      begin(unit, 0);
    }
  }
}

// The wide units of the worker at `place`.  TW: as TN.
template <int DT, int DW, bool PAD, int TW>
__device__ __forceinline__ void step_wide(args_ptr a, const StepRun& run, int place, char* lds) {
  using Ops = MfmaOps<DT>;
  using frag = typename Ops::frag;
  using Lanes = StepLanes<DW>;
  constexpr int KS = DW / 16, DB = Lanes::DB, PW = Lanes::PW, NJ = Lanes::NJ;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lcol = lane & 31, lhalf = lane >> 5;
  const int n_wide = run.n_wide, end_unit = run.end_unit, end_step = run.end_step;
  const Lanes at(lane);
  const uint32_t lds0 = lds_offset(lds);
  const float c = a->scale_log2;
  for (int unit = run.unit, s0 = run.step; unit < end_unit || (unit == end_unit && s0 < end_step); ++unit, s0 = 0) {
    const args_ptr b0 = again(a);
    const int kvh = unit / n_wide;
    const StepTile t = read_tile(b0, unit - kvh * n_wide);
    const int s1 = unit == end_unit ? min(end_step, t.steps) : t.steps;
    const int slot = s0 > 0 ? 2 * place : s1 < t.steps ? 2 * place + 1 : -1;
    StepKeys keys(b0, t, kvh);
    frag qf[KS];
    const RowOf mine = row_of(b0, t, wave * 32 + lcol);
    load_q<DT, DW, PAD>(b0, mine, kvh, lhalf, qf);
    // own keys that this row and the wave's first one see
    const int vis = sees(t, mine.i), vis_min = sees(t, (t.row0 + min(wave * 32, t.rows - 1)) / b0->rep);
    f32x16 oacc[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[b][r] = 0.f;
    float m_run = kInitMax, l_run = 0.f;
    __syncthreads();  // the previous unit's reads of LDS are over

    // ---- wide: tiles of 128 keys, [0, np) of the prefix, then the sequence's own ----
    constexpr int BK = kWideKeys, NKB = BK / 32, NPS = BK / 16;
    constexpr int kTile = BK * PW, NBK = 2, NBV = 3;
    const int np = (t.p_len + BK - 1) / BK;
    const int n_tiles = s1 - s0;
    const uint32_t k_lds0 = lds0, v_lds0 = lds0 + NBK * kTile;
    const char* v_lds_c = lds + NBK * kTile;
    int* const simd_of = reinterpret_cast<int*>(lds + (NBK + NBV - 1) * kTile);  // in the last V buffer, first written in super-step 1
    auto key_of = [&](int u) __attribute__((always_inline)) { return BK * (s0 + u < np ? s0 + u : s0 + u - np); };
    KeyGroup nx;  // wave w loads rows 16 w .. 16 w + 15 of a tile: one 16-key group
    auto fetch = [&](int u) __attribute__((always_inline)) {
      if (u < n_tiles) nx = keys.fetch(s0 + u < np, key_of(u) + 16 * wave);
    };
    auto issue_tile = [&](int u) __attribute__((always_inline)) {
      u32x4 ks, vs;
      keys.srd(nx, ks, vs);
      Lanes::template load_k<PAD>(ks, k_lds0 + (u % NBK) * kTile + wave * 16 * PW, keys.row_bytes, keys.span_bytes);
      Lanes::template load_v<PAD>(vs, v_lds0 + (u % NBV) * kTile + wave * 16 * PW, keys.row_bytes, keys.span_bytes);
      fetch(u + 1);
    };
    fetch(0);
    issue_tile(0);
    if (lane == 0) simd_of[wave] = simd_id();
    f32x16 sacc[NKB];
    frag pf[TW == 1 ? NPS : 1];  // several terms are made from P, left in place of S, as V is read

    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    bool lead = true;
    {
      const int mine = simd_of[wave];
#pragma unroll
      for (int w = 0; w < kStepWaves; ++w) lead = lead && !(w < wave && simd_of[w] == mine);
    }
    lead = __builtin_amdgcn_readfirstlane(static_cast<int>(lead)) != 0;
    // last tile with a key that some row of this wave sees
    int last_live = -1;
    if (wave * 32 < t.rows) {
      const int most = sees(t, (t.row0 + min(wave * 32 + 31, t.rows - 1)) / a->rep);
      last_live = min(n_tiles, np + (most + BK - 1) / BK - s0) - 1;
    }
    auto live = [&](int u) __attribute__((always_inline)) { return u >= 0 && u <= last_live; };

    auto pv_part = [&](int vb) __attribute__((always_inline)) {
      const char* vl = v_lds_c + vb * kTile;
      const uint32_t rd0 = fresh(at.v_rd0);
#pragma unroll
      for (int s = 0; s < NPS; ++s) {
        frag pk[TW];
        if constexpr (TW == 1) {
          pk[0] = pf[s];
        } else {
          float rest[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) rest[i] = sacc[s >> 1][8 * (s & 1) + i];
#pragma unroll
          for (int k = 0; k < TW; ++k) {
            pk[k] = Ops::pack(rest);
#pragma unroll
            for (int i = 0; i < 8; ++i) rest[i] -= frag_value<DT>(pk[k], i);
          }
        }
#pragma unroll
        for (int b = 0; b < DB; ++b) {
          const char* p0 = vl + Lanes::v_rd(rd0, b) + s * 16 * PW;
          const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p0));
          const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p0 + 4 * PW));
          const u32x2 lo2 = __builtin_bit_cast(u32x2, lo), hi2 = __builtin_bit_cast(u32x2, hi);
          const frag vf = as_frag<frag>(u32x4{lo2[0], lo2[1], hi2[0], hi2[1]});
#pragma unroll
          for (int k = 0; k < TW; ++k) oacc[b] = Ops::mma(vf, pk[k], oacc[b]);
        }
      }
    };
    auto s_part = [&](int kb) __attribute__((always_inline)) {
      const uint32_t kl = k_lds0 + kb * kTile + at.k_rd;
#pragma unroll
      for (int b = 0; b < NKB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) sacc[b][r] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint32_t ks = kl ^ static_cast<uint32_t>(s << 5);
#pragma unroll
        for (int b = 0; b < NKB; ++b) {
          const frag kf = as_frag<frag>(*reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
              static_cast<uintptr_t>(ks + b * 32 * PW)));
          sacc[b] = Ops::mma(kf, qf[s], sacc[b]);
        }
      }
    };
    auto m_full = [&](int kb, int vb) __attribute__((always_inline)) {
      __builtin_amdgcn_s_setprio(1);
      pv_part(vb);
      s_part(kb);
      if constexpr (TW == 1) {
        constexpr int A = 8, NPV = NPS * DB, NS = NKB * KS;
        __builtin_amdgcn_sched_group_barrier(0x100, A, 0);
#pragma unroll
        for (int i = 0; i < NPV - A / 2; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, A / 2, 0);
      }
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int b = 0; b < DB; ++b) pin(oacc[b]);
#pragma unroll
      for (int b = 0; b < NKB; ++b) pin(sacc[b]);
    };
    auto xphase = [&](int u) __attribute__((always_inline)) {
      const bool own = s0 + u >= np;
      const int key0 = key_of(u), end = own ? t.s_len : t.p_len;
      if (end - key0 < BK || (own && vis_min < key0 + BK)) {
        const int lim = min(min(end - key0, BK), own ? vis - key0 : BK) - 1 - 8 * static_cast<int>(fresh_lane() >> 5);
#pragma unroll
        for (int b = 0; b < NKB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            sacc[b][r] = 32 * b + 16 * (r >> 3) + 4 * ((r >> 2) & 1) + (r & 3) <= lim ? sacc[b][r] : -INFINITY;
      }
      float lsum = 0.f;
      auto weigh = [&] __attribute__((always_inline)) {  // P = 2^(s c - m)
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NKB; ++b) {
          float p[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[b][r], c, -m_run));
            ls[r & 3] += p[r];
          }
          if constexpr (TW == 1) {
            pf[2 * b] = Ops::pack(p);
            pf[2 * b + 1] = Ops::pack(p + 8);
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) sacc[b][r] = p[r];
          }
        }
        lsum = (ls[0] + ls[1]) + (ls[2] + ls[3]);
      };
      auto highest = [&] __attribute__((always_inline)) {
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < NKB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, sacc[b][r]);
        return max_xor32(top) * c;
      };
      // The maximum moves where it has to: seen from the sums of the weights where S outlives
      // them, from S itself where P takes its place.
      bool redo = u == 0;
      if constexpr (TW == 1) {
        if (!redo) {
          weigh();
          redo = __any(!(lsum <= kMostSum<DT>));
        }
      }
      const float top = TW > 1 || redo ? highest() : 0.f;
      if (TW > 1) redo = redo || __any(!(top <= m_run + 8.f + kBias<DT>));
      if (redo) {
        const float m_new = fmaxf(m_run, top - kBias<DT>);
        const float alpha = exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[b][r] *= alpha;
        m_run = m_new;
      }
      if (redo || TW > 1) weigh();
      l_run += lsum;
      if constexpr (TW == 1) {
#pragma unroll
        for (int s = 0; s < NPS; ++s) pin(pf[s]);
      } else {
#pragma unroll
        for (int b = 0; b < NKB; ++b) pin(sacc[b]);
      }
      pin(l_run);
    };
    auto issue = [&](int u) __attribute__((always_inline)) {
      if (u + 1 < n_tiles) issue_tile(u + 1);
    };
    auto settle = [&](int u) __attribute__((always_inline)) {
      if (u < n_tiles) {
        // K_{u+1} and V_u have to be there; V_{u+1}, issued after K_{u+1}, may be on its way
        wait_dma(u + 1 < n_tiles ? NJ : 0);
        __syncthreads();
      }
    };
    const int hot = max(last_live, 0);
    auto next = [](int r, int nb) __attribute__((always_inline)) { return r + 1 == nb ? 0 : r + 1; };
    if (lead) {
      if (live(0)) s_part(0);
      issue(0);
      if (live(0)) xphase(0);
      settle(0);
    } else {
      issue(0);
      if (live(0)) s_part(0);
      settle(0);
      issue(1);
      if (live(0)) xphase(0);
    }
    const int lag = lead ? 0 : 1;
    int u = 1, rk = 1 % NBK, rv = 0;
    for (; u <= hot; ++u, rk = next(rk, NBK), rv = next(rv, NBV)) {
      m_full(rk, rv);
      if (!lead) settle(u);
      issue(u + lag);
      xphase(u);
      if (lead) settle(u);
    }
    for (; u <= n_tiles; ++u, rv = next(rv, NBV)) {
      if (live(u - 1)) pv_part(rv);
      if (lead) issue(u);
      settle(u);
      if (!lead) issue(u + 1);
    }
    keys.report(a);
    const args_ptr e = again(a);
    const int row = wave * 32 + (static_cast<int>(fresh_lane()) & 31);
    if (row < t.rows) {
      const RowOf ro = row_of(e, t, row);
      const RowDest dst = row_dest(e, t, kvh, slot, row, ro.token, ro.i, ro.h);
      const float l_tot = sum_xor32(l_run);
      const int half = static_cast<int>(fresh_lane() >> 5);
      write_final_row<DW>(dst.o, dst.dtype, dst.o_off, dst.lse, half, oacc, m_run, l_tot, e->s.d);
      // a row that met a NaN key says so, or a join would take it for one without keys
      if (half == 0 && dst.lse != nullptr && l_tot != l_tot) *dst.lse = l_tot;
    }
  }
}

// A workgroup takes its share of the wide units, then of the narrow ones (mostly one of the two).
template <int DT, int DW, bool PAD, int TN, int TW>
__global__ __launch_bounds__(kStepThreads, 1) void step_attn_kernel(StepArgs args) {
  __shared__ __attribute__((aligned(1024))) char lds[kStepLds<DW>];
  const args_ptr a = (args_ptr)__builtin_amdgcn_kernarg_segment_ptr();
  const int workers = a->workers, worker = xcd_remap(blockIdx.x, workers), narrow = workers + 1 + worker;
  const StepRun wide_run(a, worker), narrow_run(a, narrow);  // loaded beside the head
  if (!plan_fits(scalar_ptr(a->plan), args.s, args.workers)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(args.err, 8);
    return;
  }
  step_wide<DT, DW, PAD, TW>(a, wide_run, worker, lds);
  step_narrow<DT, DW, PAD, TN>(a, narrow_run, narrow, lds);
}

// ----------------------------------------------------------------------------------
// Join: 32 lanes a row, 16 for every other part of it.  The rows of tokens behind shared prefixes
// (own part and prefix part), then those of cut units; a part is a unit's rows as one worker left
// them.  Bound by the chain of loads that finds a row's parts (three or four, some 0.7 us each).
// ----------------------------------------------------------------------------------
constexpr int kJoinLanes = 32, kJoinRows = 256 / kJoinLanes;

__global__ __launch_bounds__(256) void step_join_kernel(StepArgs a) {
  const int32_t* head = reinterpret_cast<const int32_t*>(a.plan);
  const int n_wide = head[12], n_shared = head[14], cut_wide = head[15], cut_narrow = head[16];
  if (!plan_fits(head, a.s, a.workers)) return;  // the attention kernel has said so
  const int units_w = n_wide * a.s.hkv, hkv = a.s.hkv, hq = a.s.hq, d = a.s.d;
  const int2* starts = reinterpret_cast<const int2*>(a.plan + a.p_starts);
  const int sub = threadIdx.x % kJoinLanes, col = sub % 16 * 8 < d ? sub % 16 * 8 : 0;
  const int64_t shared_rows = static_cast<int64_t>(n_shared) * hq;
  const int64_t rows = shared_rows + cut_wide * kWideRows + cut_narrow * kNarrowRows;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kJoinRows + threadIdx.x / kJoinLanes; i < rows;
       i += static_cast<int64_t>(gridDim.x) * kJoinRows) {
    // up to two sources of parts: a cut unit's slots or one row
    const float *o1 = nullptr, *l1 = nullptr;  // an uncut row
    const float *o2 = nullptr, *l2 = nullptr;
    int c1 = 0, r1 = 0, c2 = 0, r2 = 0;        // cuts entry and row in the slots
    int token, hd;
    if (i < shared_rows) {
      const int32_t* cuts = reinterpret_cast<const int32_t*>(a.plan + a.p_cuts);
      const int li = static_cast<int>(i / hq);
      hd = static_cast<int>(i - static_cast<int64_t>(li) * hq);
      const StepShared s = reinterpret_cast<const StepShared*>(a.plan + a.p_shared)[li];
      token = s.token;
      const int kvh = hd / a.rep, h = hd - kvh * a.rep, own = s.own_row + h, pre = s.pre_row + h;
      c1 = cuts[units_w + (s.own_tile + own / kNarrowRows) * hkv + kvh];
      r1 = own % kNarrowRows;
      o1 = a.own_o + i * d;
      l1 = a.own_lse + i;
      c2 = s.pre_wide ? cuts[kvh * n_wide + s.pre_tile + pre / kWideRows] : cuts[units_w + (s.pre_tile + pre / kNarrowRows) * hkv + kvh];
      r2 = s.pre_wide ? pre % kWideRows : pre % kNarrowRows;
      o2 = a.pre_o + i * d;
      l2 = a.pre_lse + i;
    } else {
      int x = static_cast<int>(i - shared_rows);
      const bool wide = x < cut_wide * kWideRows;
      if (!wide) x -= cut_wide * kWideRows;
      const StepCut t = reinterpret_cast<const StepCut*>(a.plan + (wide ? a.p_cut_wide : a.p_cut_narrow))[wide ? x / kWideRows : x / kNarrowRows];
      r1 = wide ? x % kWideRows : x % kNarrowRows;
      if (r1 >= t.rows) continue;  // for all of a row's lanes
      c1 = t.cut;
      const int sr = t.row0 + r1, ri = sr / a.rep;
      token = t.tok0 + ri;
      hd = t.head0 + sr - ri * a.rep;
    }
    const int w1 = (c1 & 0xffff) - 1, w2 = (c2 & 0xffff) - 1;  // place of the first worker
    const int n1 = c1 != 0 ? c1 >> 16 : 1, n2 = o2 == nullptr ? 0 : c2 != 0 ? c2 >> 16 : 1, n = n1 + n2;
    float m = -INFINITY, den = 0.f, x[8] = {};
    for (int k0 = 0; k0 < n; k0 += kJoinLanes) {
      // part k0 + sub: its row and LSE; a worker without steps left nothing
      const float* o = nullptr;
      float l = -INFINITY;
      if (k0 + sub < n) {
        const bool one = k0 + sub < n1;
        const int j = one ? k0 + sub : k0 + sub - n1;
        if ((one ? c1 : c2) == 0) {
          o = one ? o1 : o2;
          l = *(one ? l1 : l2);
        } else {
          const int worker = (one ? w1 : w2) + j;
          const int64_t row = static_cast<int64_t>(2 * worker + (j == 0 ? 1 : 0)) * a.slot_rows + (one ? r1 : r2);
          const int2 from = starts[worker], to = starts[worker + 1];
          const float got = a.slot_lse[row];
          o = a.slot_o + row * d;
          if (from.x != to.x || from.y != to.y) l = got;
        }
      }
      float top = l;
      for (int off = 1; off < kJoinLanes; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
      const float m_new = fmaxf(m, top);
      const float keep = m == -INFINITY ? 0.f : __expf(m - m_new);
      const float f = l == -INFINITY ? 0.f : __expf(l - m_new);  // a NaN part (a NaN key) stays one
      m = m_new;
      float fs = f;
      for (int off = 1; off < kJoinLanes; off <<= 1) fs += __shfl_xor(fs, off);
      den = den * keep + fs;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= keep;
      // A lane loads four parts at a time; one without weight from where its address would be (the
      // slots' start where it has none), to be left out.
      const uint64_t ptr = reinterpret_cast<uint64_t>(o != nullptr ? o : a.slot_o);
      const int parts = min(kJoinLanes, n - k0), lane0 = (threadIdx.x & 63) - sub;
      // The same number of rounds for all of a row's lanes: they read each other's addresses.
      for (int round = 0; round < parts; round += 8) {
        const int k = round + sub / 16;
        f32x4 v[4][2];
        float fk[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int src = lane0 + min(k + 2 * e, parts - 1);
          fk[e] = __shfl(f, src);
          if (k + 2 * e >= parts) fk[e] = 0.f;
          const uint64_t pk = static_cast<uint64_t>(__shfl(static_cast<uint32_t>(ptr), src)) |
                              static_cast<uint64_t>(__shfl(static_cast<uint32_t>(ptr >> 32), src)) << 32;
          const f32x4* ok = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(pk) + col);
          v[e][0] = ok[0];
          v[e][1] = ok[1];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (fk[e] != 0.f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x[i] += fk[e] * v[e][0][i];
              x[4 + i] += fk[e] * v[e][1][i];
            }
          }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += __shfl_xor(x[e], 16);
    const float inv = den == 0.f ? 0.f : 1.f / den;
    if (sub < 16 && 8 * sub < d) {
      const int64_t off = hd * a.out_hs + token * a.out_ss + 8 * sub;
      store4(a.out, a.out_dtype, off, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
      store4(a.out, a.out_dtype, off + 4, x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    }
    if (sub == 0 && a.lse != nullptr) a.lse[hd * a.s.tokens + token] = den == 0.f ? -INFINITY : m + __logf(den);
  }
}

template <int DT, int DW, bool PAD>
static void launch_step_d(const StepArgs& a, hipStream_t stream) {
  if (a.out_dtype == kF32) step_attn_kernel<DT, DW, PAD, DT == kBF16 ? 3 : 2, DT == kBF16 ? 3 : 2><<<a.workers, kStepThreads, 0, stream>>>(a);
  else step_attn_kernel<DT, DW, PAD, 2, 1><<<a.workers, kStepThreads, 0, stream>>>(a);
}
template <int DT>
static void launch_step(const StepArgs& a, hipStream_t stream) {
  if (a.s.d == 128) launch_step_d<DT, 128, false>(a, stream);
  else if (a.s.d == 64) launch_step_d<DT, 64, false>(a, stream);
  else if (a.s.d < 64) launch_step_d<DT, 64, true>(a, stream);
  else launch_step_d<DT, 128, true>(a, stream);
}

void launch_step_attn(const StepLaunch& L, hipStream_t stream) {
  const PlanLayout l = plan_layout(L.s);
  const int workers = step_workers();
  const WorkLayout w = work_layout(L.s, workers);
  StepArgs a;
  a.plan = static_cast<const char*>(L.plan);
  a.p_tiles = l.tiles; a.p_shared = l.shared; a.p_starts = l.starts; a.p_cuts = l.cuts; a.p_cut_wide = l.cut_wide; a.p_cut_narrow = l.cut_narrow;
  a.s = L.s;
  a.workers = workers;
  a.q = static_cast<const uint16_t*>(L.q);
  a.q_hs = L.q_hs; a.q_ss = L.q_ss;
  a.pool = static_cast<const uint16_t*>(L.pool);
  a.num_blocks = L.num_blocks;
  a.plane_bytes = L.num_blocks * L.s.bs * L.s.hkv * static_cast<int64_t>(L.s.d) * 2;
  a.rep = L.s.hq / L.s.hkv;
  a.gpb = L.s.bs / 16;
  a.gpb_inv = 0xffffffffu / a.gpb;
  a.block_bytes = static_cast<uint32_t>(L.s.bs) * L.s.hkv * L.s.d * 2;
  a.tables = L.tables; a.prefix_tables = L.prefix_tables;
  a.table_stride = L.table_stride; a.prefix_stride = L.prefix_stride;
  a.scale_log2 = L.scale * kLog2e;
  a.out = L.out; a.out_hs = L.out_hs; a.out_ss = L.out_ss; a.out_dtype = L.out_dtype;
  a.lse = L.lse;
  char* ws = static_cast<char*>(L.ws);
  auto f = [&](size_t at) { return reinterpret_cast<float*>(ws + at); };
  a.slot_o = f(w.slot_o); a.slot_lse = f(w.slot_lse); a.own_o = f(w.own_o); a.own_lse = f(w.own_lse);
  a.pre_o = f(w.pre_o); a.pre_lse = f(w.pre_lse);
  a.slot_rows = w.slot_rows;
  a.err = L.err;
  if (L.dtype == kBF16) launch_step<kBF16>(a, stream);
  else launch_step<kF16>(a, stream);
  HCP_HIP(hipGetLastError());
  // no more rows are joined than the query has, nor than shared ones and two cut units a worker
  const int64_t rows = std::min(L.s.tokens * L.s.hq, l.max_shared * L.s.hq + 2 * static_cast<int64_t>(workers) * w.slot_rows);
  const int64_t grid = std::min<int64_t>(ceil_div(rows, kJoinRows) + 1, 32 * workers);
  step_join_kernel<<<static_cast<unsigned>(grid), 256, 0, stream>>>(a);
  HCP_HIP(hipGetLastError());
}

}  // namespace hcp
