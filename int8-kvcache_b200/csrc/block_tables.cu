// Block tables and slot maps from request lengths, on the device: growth of the tables from a free list, the slots of
// the tokens that a step adds, and the way back of finished requests' blocks.
//
// With c cached and n new tokens of a request, S tokens per block, W table columns and the free list's cursor f:
//   old = ceil(c / S), want = ceil((c + n) / S) - old (0 and refused when c + n > W * S),
//   first = exclusive prefix sum of want over the requests, granted = want == 0 or first + want <= free entries,
//   table[old + j] = free[f + first + j],  slot of token i = block(pos / S) * S + pos % S with pos = c + i.
// Everything hangs on two prefix sums over the requests.  A CTA makes them in about a microsecond out of L2, so every
// CTA of the launch makes them for itself and then writes its share of slots and blocks: one launch, no workspace, no
// pass over intermediate records.  Small calls are one CTA, bound by launch latency and one chain of dependent
// loads (length -> block id -> slot); a decode step, where every request adds a few tokens, goes thread by thread with
// the block id requested ahead of the sums.  Large ones are bound by the 8 bytes per slot that they write.
// With many requests, or when a large call's new lengths or cursor are to be written over the old ones (which other
// CTAs may still be reading), one CTA makes the sums, leaves 24 bytes per request in the workspace, and a second kernel,
// launched with programmatic dependent launch, writes slots and blocks.
// The CTA that writes the new lengths and the cursor has read the old ones by then, so they may be the same memory: a
// captured step then advances its own state.
#include <algorithm>

#include "common.cuh"

namespace int8kv {

constexpr uint32_t kTabSat = 0x7fffffffu;  // prefix sums saturate here: an absurd length is refused, never wrapped

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kTabSat); }

__device__ __forceinline__ void store_index(void* base, int is_i64, int64_t idx, int64_t v) {
  if (is_i64) reinterpret_cast<int64_t*>(base)[idx] = v;
  else reinterpret_cast<int32_t*>(base)[idx] = static_cast<int32_t>(v);
}
// Index load from a buffer that this launch also writes (at other places): not through the read-only path.
__device__ __forceinline__ int64_t load_index_rw(const void* base, int is_i64, int64_t idx) {
  return is_i64 ? reinterpret_cast<int64_t*>(const_cast<void*>(base))[idx]
                : static_cast<int64_t>(reinterpret_cast<int32_t*>(const_cast<void*>(base))[idx]);
}

// x / S for a position: 32-bit division wherever it fits (a 64-bit one costs several times as much)
__device__ __forceinline__ int64_t div_block(int64_t x, int S) {
  if (static_cast<uint64_t>(x) <= 0xffffffffull) return static_cast<uint32_t>(x) / static_cast<uint32_t>(S);
  return x / S;
}

// One request: how many tokens and blocks it asks for.
__device__ __forceinline__ void tab_request(const TableParams& p, int b, int64_t& c, uint32_t& n, uint32_t& want,
                                            bool& fits) {
  c = load_index_rw(p.lens, p.lens_is_i64, b);
  const int64_t cap = p.width * p.block_size;
  n = 0;
  want = 0;
  fits = true;
  if (p.mode == kTabRelease) {
    const int64_t len = c < 0 ? 0 : (c > cap ? cap : c);
    if (p.finished[b]) want = static_cast<uint32_t>(min(div_block(len + p.block_size - 1, p.block_size), static_cast<int64_t>(kTabSat)));
    return;
  }
  c = c < 0 ? 0 : min(c, static_cast<int64_t>(1) << 60);  // positions stay inside 64 bits
  int64_t nn = load_index_rw(p.new_lens, p.new_is_i64, b);
  nn = nn < 0 ? 0 : (nn > kTabSat ? kTabSat : nn);
  n = static_cast<uint32_t>(nn);
  if (p.mode == kTabGrow) {
    fits = c + nn <= cap && (p.lens_is_i64 || c + nn <= 0x7fffffffll);
    if (fits)
      want = static_cast<uint32_t>(min(div_block(c + nn + p.block_size - 1, p.block_size) -
                                           div_block(c + p.block_size - 1, p.block_size), static_cast<int64_t>(kTabSat)));
  }
}

// Exclusive saturating prefix sums of (x, y) over the CTA's threads, in place; totals in `all`.  (Exclusive by shifting,
// not by subtraction: a sum that has saturated cannot be undone.)
// Returns whether `vote` held on any thread.
__device__ __forceinline__ bool tab_scan(uint32_t& x, uint32_t& y, uint32_t* warp_x, uint32_t* warp_y, uint2& all, bool vote) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  auto warp_scan = [lane](uint32_t& a, uint32_t& b) {
    for (int o = 1; o < kWarp; o <<= 1) {
      const uint32_t u = __shfl_up_sync(kFull, a, o), v = __shfl_up_sync(kFull, b, o);
      if (lane >= o) {
        a = sat_add(a, u);
        b = sat_add(b, v);
      }
    }
  };
  warp_scan(x, y);
  if (lane == kWarp - 1) {
    warp_x[warp] = x;
    warp_y[warp] = y;
  }
  x = __shfl_up_sync(kFull, x, 1);
  y = __shfl_up_sync(kFull, y, 1);
  if (lane == 0) x = y = 0u;
  const bool any = __syncthreads_or(vote);
  uint32_t a = lane < warps ? warp_x[lane] : 0u, b = lane < warps ? warp_y[lane] : 0u;  // every warp scans the sums
  warp_scan(a, b);
  all = make_uint2(__shfl_sync(kFull, a, kWarp - 1), __shfl_sync(kFull, b, kWarp - 1));
  const int before = warp == 0 ? 0 : warp - 1;
  a = __shfl_sync(kFull, a, before);
  b = __shfl_sync(kFull, b, before);
  if (warp > 0) {
    x = sat_add(x, a);
    y = sat_add(y, b);
  }
  return any;
}

template <bool BY_TOKEN>
__device__ __forceinline__ uint32_t tab_key(const TabRecord& r) { return BY_TOKEN ? r.start : r.first; }

// Last request b in [lo, hi) with key(b) <= k, where key(lo) <= k.
template <bool BY_TOKEN>
__device__ __forceinline__ int tab_owner(const TabRecord* rec, int lo, int hi, uint32_t k) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab_key<BY_TOKEN>(rec[mid]) <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The same by a whole warp: 32 probes per round, two rounds for up to 1024 requests.
template <bool BY_TOKEN>
__device__ __forceinline__ int tab_owner_warp(const TabRecord* rec, int R, uint32_t k, int lane) {
  int lo = 0, len = R;
  while (len > 1) {
    const int step = (len + kWarp - 1) / kWarp, at = lane * step;
    const unsigned hit = __ballot_sync(kFull, at < len && (lane == 0 || tab_key<BY_TOKEN>(rec[lo + min(at, len - 1)]) <= k));
    const int skip = (__popc(hit) - 1) * step;  // the hits are a prefix of the lanes
    lo += skip;
    len = min(step, len - skip);
  }
  return lo;
}

// Free entries ahead of the cursor, below the saturation value.
__device__ __forceinline__ uint32_t tab_room(const TableParams& p, int64_t cursor) {
  const int64_t room = p.num_free - cursor;
  return room <= 0 ? 0u : static_cast<uint32_t>(min(room, static_cast<int64_t>(kTabSat - 1)));
}

__device__ __forceinline__ int64_t tab_table(const TableParams& p, int b, int64_t j) {
  return load_index_rw(p.bt, p.bt_is_i64, b * p.bt_st[0] + j * p.bt_st[1]);
}

// Slot of token `tok` of the packed order, which belongs to request b.
__device__ __forceinline__ int64_t tab_slot(const TableParams& p, const TabRecord* rec, const TabTotals& tot, int b, uint32_t tok) {
  const TabRecord r = rec[b];
  if (r.cached < 0) return -1;
  const int64_t pos = r.cached + (tok - r.start);
  const int64_t j = div_block(pos, p.block_size);
  const int64_t begin = j * p.block_size;
  int64_t blk = -1;
  if (p.mode == kTabGrow && begin >= r.cached) blk = load_index(p.free_blocks, p.free_is_i64, tot.cursor + j + r.shift);
  else if (j < p.width) blk = tab_table(p, b, j);
  return blk < 0 ? -1 : blk * p.block_size + (pos - begin);
}

// One block that moves: number k in the order of all blocks, of request b.
__device__ __forceinline__ void tab_move(const TableParams& p, const TabRecord* rec, const TabTotals& tot, int b, uint32_t k) {
  const TabRecord r = rec[b];
  if (r.cached < 0) return;
  const int64_t j = static_cast<int64_t>(k) - r.shift;
  if (p.mode == kTabGrow) {
    store_index(p.bt, p.bt_is_i64, b * p.bt_st[0] + j * p.bt_st[1], load_index(p.free_blocks, p.free_is_i64, tot.cursor + k));
  } else {
    const int64_t at = tot.cursor - tot.blocks + k;
    if (at >= 0 && at < p.num_free) store_index(p.free_out, p.free_is_i64, at, tab_table(p, b, j));
  }
}

// Blocks that can move at all: of a growth the ones the free list has, of a release all.
__device__ __forceinline__ uint32_t tab_moves(const TableParams& p, const TabTotals& tot) {
  if (p.mode == kTabSlots) return 0u;
  return p.mode == kTabGrow ? min(tot.blocks, tab_room(p, tot.cursor)) : tot.blocks;
}

// The write phase of warp `me` of `warps`: a run of consecutive tokens, then one of blocks that move.  The warp finds the
// requests of the run's first and last item together.  Runs of few requests (prompts) go request by request, with
// everything but the position uniform; in the others each lane searches between the two, five steps where every token is
// another request's.
__device__ __forceinline__ void tab_run(uint32_t items, uint32_t me, uint32_t warps, uint32_t& lo, uint32_t& hi) {
  const uint32_t rows = (items >> 5) + 1, per = (rows + warps - 1) / warps;  // rows of 32 items, per warp
  const uint64_t a = static_cast<uint64_t>(me) * per * 32u, b = a + per * 32ull;
  lo = static_cast<uint32_t>(a < items ? a : items);
  hi = static_cast<uint32_t>(b < items ? b : items);
}

// Slots of tokens lo + lane, lo + lane + 32, ... below hi, at positions p0 + token, through block ids ids[j * stride] of
// logical blocks j < blocks: four loads in flight per lane.
template <typename T>
__device__ __forceinline__ void tab_span(int64_t* slots, uint32_t lo, uint32_t hi, uint32_t p0, int S, int shift, const T* ids,
                                         int64_t stride, uint32_t blocks, int lane) {
  constexpr int kAhead = 4;
  for (uint32_t tok = lo + lane; tok < hi; tok += kAhead * kWarp) {
    int64_t blk[kAhead];
    uint32_t off[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t pos = p0 + tok + u * kWarp;
      const uint32_t j = shift >= 0 ? pos >> shift : pos / static_cast<uint32_t>(S);
      off[u] = pos - j * S;
      blk[u] = tok + u * kWarp < hi && j < blocks ? static_cast<int64_t>(ids[j * stride]) : -1;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (tok + u * kWarp < hi) slots[tok + u * kWarp] = blk[u] < 0 ? -1 : blk[u] * S + off[u];
  }
}

// Slots of tokens [lo, hi) of the packed order, all of request b, by one warp.
__device__ __forceinline__ void tab_request_slots(const TableParams& p, const TabRecord* rec, const TabTotals& tot, int b,
                                                  uint32_t lo, uint32_t hi, int lane) {
  const TabRecord r = rec[b];
  if (r.cached < 0 || r.cached + hi > 0x7fffffffll) {  // refused, or positions beyond 31 bits
    for (uint32_t tok = lo + lane; tok < hi; tok += kWarp) p.slots[tok] = tab_slot(p, rec, tot, b, tok);
    return;
  }
  const uint32_t p0 = static_cast<uint32_t>(r.cached) - r.start;
  uint32_t known = hi;  // tokens below this one lie in blocks that the table has
  if (p.mode == kTabGrow) {
    const uint32_t left = static_cast<uint32_t>(r.cached) % static_cast<uint32_t>(p.block_size);
    known = left == 0u ? r.start : r.start + (p.block_size - left);
    known = max(lo, min(hi, known));
  }
  const uint32_t width = static_cast<uint32_t>(p.width);
  auto span = [&](uint32_t from, uint32_t to, const void* ids, int is_i64, int64_t first, int64_t stride, uint32_t blocks) {
    if (is_i64) tab_span(p.slots, from, to, p0, p.block_size, p.block_shift, static_cast<const int64_t*>(ids) + first, stride, blocks, lane);
    else tab_span(p.slots, from, to, p0, p.block_size, p.block_shift, static_cast<const int32_t*>(ids) + first, stride, blocks, lane);
  };
  if (lo < known) span(lo, known, p.bt, p.bt_is_i64, b * p.bt_st[0], p.bt_st[1], width);
  if (known < hi) span(known, hi, p.free_blocks, p.free_is_i64, tot.cursor + r.shift, 1, width);
}

__device__ __forceinline__ void tab_write_slots(const TableParams& p, const TabRecord* rec, const TabTotals& tot, uint32_t me,
                                                uint32_t warps, int lane) {
  uint32_t lo, hi;
  tab_run(static_cast<uint32_t>(p.num_tokens), me, warps, lo, hi);
  const uint32_t live = min(hi, tot.tokens);
  if (lo < live) {
    const int b0 = tab_owner_warp<true>(rec, p.R, lo, lane);
    const int b1 = tab_owner_warp<true>(rec, p.R, live - 1, lane);
    if (static_cast<uint32_t>(b1 - b0) <= (live - lo) / kWarp) {
      for (int b = b0; b <= b1; ++b) tab_request_slots(p, rec, tot, b, max(lo, rec[b].start), b < b1 ? min(live, rec[b + 1].start) : live, lane);
    } else {
      for (uint32_t tok = lo + lane; tok < live; tok += kWarp)
        p.slots[tok] = tab_slot(p, rec, tot, tab_owner<true>(rec, b0, b1 + 1, tok), tok);
    }
  }
  for (uint32_t tok = max(lo, live) + lane; tok < hi; tok += kWarp) p.slots[tok] = -1;
}

__device__ __forceinline__ void tab_write_moves(const TableParams& p, const TabRecord* rec, const TabTotals& tot, uint32_t me,
                                                uint32_t warps, int lane) {
  uint32_t lo, hi;
  tab_run(tab_moves(p, tot), me, warps, lo, hi);
  if (lo >= hi) return;
  const int b0 = tab_owner_warp<false>(rec, p.R, lo, lane);
  const int b1 = tab_owner_warp<false>(rec, p.R, hi - 1, lane);
  for (uint32_t k = lo + lane; k < hi; k += kWarp)
    tab_move(p, rec, tot, b0 == b1 ? b0 : tab_owner<false>(rec, b0, b1 + 1, k), k);
}

constexpr int kTabThreads = 1024;
constexpr uint32_t kTabFew = 4;  // new tokens of a request that one thread places by itself

// The prefix sums, the outputs of one value per request (CTA 0), and, when FUSED, this CTA's share of the write phase.
// More than one CTA only when no output is an input.
template <bool FUSED>
__global__ void __launch_bounds__(kTabThreads) table_plan_kernel(const __grid_constant__ TableParams p) {
  extern __shared__ __align__(16) uint8_t tab_smem[];
  __shared__ uint32_t warp_x[kWarp], warp_y[kWarp];
  __shared__ unsigned int taken_s;
  grid_dependency_wait();
  grid_launch_dependents();
  TabRecord* rec = FUSED ? reinterpret_cast<TabRecord*>(tab_smem) : p.records;
  const bool first_cta = blockIdx.x == 0;
  TabTotals tot;
  tot.cursor = p.mode == kTabSlots ? 0 : *p.cursor;
  if (threadIdx.x == 0) taken_s = 0u;
  const int run = (p.R + static_cast<int>(blockDim.x) - 1) / static_cast<int>(blockDim.x);
  const int lo = min(static_cast<int>(threadIdx.x) * run, p.R), hi = min(lo + run, p.R);
  uint32_t x = 0, y = 0;
  int64_t c0 = 0;  // this thread's first request stays in registers
  uint32_t n0 = 0, want0 = 0;
  bool fits0 = false;
  for (int b = lo; b < hi; ++b) {
    int64_t c;
    uint32_t n, want;
    bool fits;
    tab_request(p, b, c, n, want, fits);
    if (b == lo) {
      c0 = c; n0 = n; want0 = want; fits0 = fits;
    }
    x = sat_add(x, n);
    y = sat_add(y, want);
  }
  // A thread's only request with few new tokens: its first block, if the table has it, is requested ahead of the sums.
  const bool few = FUSED && p.mode != kTabRelease && run <= 1 && n0 <= kTabFew;
  int64_t j0 = 0, known = -1;
  int off0 = 0;
  if (few && lo < hi && n0 > 0) {
    j0 = div_block(c0, p.block_size);
    off0 = static_cast<int>(c0 - j0 * p.block_size);
    if (j0 < p.width && (off0 > 0 || p.mode == kTabSlots)) known = tab_table(p, lo, j0);
  }
  uint2 all;
  const bool some_many = tab_scan(x, y, warp_x, warp_y, all, !few);
  if (tot.cursor < 0) tot.cursor = 0;
  if (p.mode == kTabRelease && tot.cursor > p.num_free) tot.cursor = p.num_free;
  tot.tokens = all.x;
  tot.blocks = all.y;
  const uint32_t room = p.mode == kTabGrow ? tab_room(p, tot.cursor) : kTabSat;
  uint32_t at_x = x, at_y = y, taken = 0;
  for (int b = lo; b < hi; ++b) {
    int64_t c = c0;
    uint32_t n = n0, want = want0;
    bool fits = fits0;
    if (b != lo) tab_request(p, b, c, n, want, fits);
    const uint32_t end = sat_add(at_y, want);
    TabRecord r;
    r.cached = c;
    r.start = at_x;
    r.first = at_y;
    r.shift = static_cast<int32_t>(at_y);  // release: from the row's first block on
    if (p.mode == kTabGrow) {
      const bool granted = fits && (want == 0u || end <= room);
      if (granted && want > 0u) taken = max(taken, end);
      if (!granted) r.cached = -1;
      // (a refused request's shift is never used; a granted one has c <= width * S, so its block count fits 32 bits)
      r.shift = static_cast<int32_t>(at_y - static_cast<uint32_t>(div_block(c + p.block_size - 1, p.block_size)));
      if (first_cta) store_index(p.lens_out, p.lens_is_i64, b, granted ? c + n : c);
    } else if (p.mode == kTabRelease) {
      r.cached = 0;
      if (first_cta) store_index(p.lens_out, p.lens_is_i64, b, p.finished[b] ? 0 : c);
    }
    if (!FUSED || some_many) {
      rec[b] = r;
    } else if (first_cta) {  // every request of the call has few tokens: each thread places its own
      int64_t j = j0, blk = known;
      int off = off0;
      for (uint32_t i = 0; i < n; ++i) {
        if (p.mode == kTabGrow && off == 0 && r.cached >= 0) {
          blk = load_index(p.free_blocks, p.free_is_i64, tot.cursor + j + r.shift);
          store_index(p.bt, p.bt_is_i64, b * p.bt_st[0] + j * p.bt_st[1], blk);
        } else if (p.mode == kTabSlots && off == 0 && i > 0) {
          blk = j < p.width ? tab_table(p, b, j) : -1;
        }
        const uint32_t tok = at_x + i;
        if (tok < static_cast<uint32_t>(p.num_tokens)) p.slots[tok] = r.cached < 0 || blk < 0 ? -1 : blk * p.block_size + off;
        if (++off == p.block_size) {
          off = 0;
          ++j;
        }
      }
    }
    if (first_cta && p.query_start != nullptr) p.query_start[b] = static_cast<int32_t>(at_x);
    at_x = sat_add(at_x, n);
    at_y = end;
  }
  if (first_cta && p.query_start != nullptr && threadIdx.x == 0) p.query_start[p.R] = static_cast<int32_t>(tot.tokens);
  if (p.mode == kTabGrow && taken > 0u) atomicMax(&taken_s, taken);
  __syncthreads();
  if (first_cta && threadIdx.x == 0) {
    if (p.mode != kTabSlots) {
      const int64_t next = p.mode == kTabGrow ? tot.cursor + taken_s : tot.cursor - static_cast<int64_t>(tot.blocks);
      *p.cursor_out = next < 0 ? 0 : next;
    }
    if (!FUSED) *p.totals = tot;
  }
  if constexpr (FUSED) {
    const int lane = threadIdx.x & 31;
    const uint32_t warps = gridDim.x * (blockDim.x >> 5), me = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (some_many) {
      tab_write_moves(p, rec, tot, me, warps, lane);
      tab_write_slots(p, rec, tot, me, warps, lane);
    } else {
      const uint32_t tokens = static_cast<uint32_t>(p.num_tokens);
      for (uint32_t tok = min(tot.tokens, tokens) + me * kWarp + lane; tok < tokens; tok += warps * kWarp) p.slots[tok] = -1;
    }
  }
}

constexpr int kTabWriteThreads = 256;

// The write phase of a call whose sums another kernel has left in the workspace.
__global__ void __launch_bounds__(kTabWriteThreads) table_write_kernel(const __grid_constant__ TableParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const TabTotals tot = *p.totals;
  const int lane = threadIdx.x & 31;
  const uint32_t warps = gridDim.x * (kTabWriteThreads / kWarp);
  const uint32_t me = blockIdx.x * (kTabWriteThreads / kWarp) + (threadIdx.x >> 5);
  tab_write_moves(p, p.records, tot, me, warps, lane);
  tab_write_slots(p, p.records, tot, me, warps, lane);
}

int64_t table_workspace_bytes(int R) { return static_cast<int64_t>(R) * sizeof(TabRecord) + 32; }

constexpr int kFusedRequests = kTabThreads;  // one request per thread, 24 KB of records in shared memory
constexpr int64_t kOneCtaItems = 4096;       // slots and blocks that one CTA writes faster than a second launch starts

bool table_single_launch(const TableParams& p, int64_t items) {
  if (p.R > kFusedRequests) return false;
  return items <= kOneCtaItems || p.mode == kTabSlots || (p.lens_out != p.lens && p.lens_out != p.new_lens && p.cursor_out != p.cursor);
}

int launch_tables(TableParams p, void* workspace, int64_t items, int sm_count, cudaStream_t stream) {
  p.block_shift = (p.block_size & (p.block_size - 1)) == 0 ? 31 - __builtin_clz(static_cast<unsigned>(p.block_size)) : -1;
  const unsigned threads = p.R <= 256 && items <= 1024 ? 256u : static_cast<unsigned>(kTabThreads);
  if (table_single_launch(p, items)) {
    // the registers hold one such CTA per SM
    const int64_t ctas = items <= kOneCtaItems ? 1 : std::min<int64_t>((items + kTabThreads - 1) / kTabThreads, sm_count);
    return launch_pdl(table_plan_kernel<true>, static_cast<unsigned>(ctas), threads, p.R * sizeof(TabRecord), stream, p);
  }
  p.totals = reinterpret_cast<TabTotals*>(workspace);
  p.records = reinterpret_cast<TabRecord*>(static_cast<char*>(workspace) + 32);
  const int rc = launch_pdl(table_plan_kernel<false>, 1u, threads, 0, stream, p);
  if (rc != INT8KV_OK) return rc;
  const int64_t want = (items + kTabWriteThreads - 1) / kTabWriteThreads;
  const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(want, sm_count * 8)));
  return launch_pdl(table_write_kernel, grid, kTabWriteThreads, 0, stream, p);
}

}  // namespace int8kv
