// Block tables and slot maps from request lengths, on the device: growth of the tables from a free list, the slots of
// the tokens that a step adds, and the way back of finished requests' blocks.
//
// With c cached and n new tokens of a request, S tokens per block, W table columns and the free list's cursor f:
//   old = ceil(c / S), want = ceil((c + n) / S) - old (0 and refused when c + n > W * S),
//   first = exclusive prefix sum of want over the requests, granted = want == 0 or first + want <= free entries,
//   table[old + j] = free[f + first + j],  slot of token i = block(pos / S) * S + pos % S with pos = c + i.
// Everything hangs on two prefix sums over the requests, so one CTA makes them (plan).  Small calls are bound by launch
// latency and finish in that CTA, out of its shared memory; larger ones leave 16 bytes per request in the workspace
// and a second kernel, launched with programmatic dependent launch, writes tables and slots with the whole machine,
// one 8-byte slot per token being what it cannot do without.
// All inputs are read before any output is written by the one CTA that reads them, so the new lengths and the cursor
// may be written over the old ones: a captured step then advances its own state.
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
__device__ __forceinline__ void tab_scan(uint32_t& x, uint32_t& y, uint32_t* warp_x, uint32_t* warp_y, uint2& all) {
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
  __syncthreads();
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
}

// Last request b in [0, R) with key(b) <= k (key(0) = 0 <= k always).
template <bool BY_TOKEN>
__device__ __forceinline__ int tab_owner(const TabRecord* rec, int R, uint32_t k) {
  int lo = 0, hi = R;  // key(lo) <= k, key(hi) > k or hi == R
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const uint32_t key = BY_TOKEN ? rec[mid].start : rec[mid].first;
    if (key <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Free entries ahead of the cursor, below the saturation value.
__device__ __forceinline__ uint32_t tab_room(const TableParams& p, int64_t cursor) {
  const int64_t room = p.num_free - cursor;
  return room <= 0 ? 0u : static_cast<uint32_t>(min(room, static_cast<int64_t>(kTabSat - 1)));
}

__device__ __forceinline__ int64_t tab_slot(const TableParams& p, const TabRecord* rec, const TabTotals& tot, uint32_t tok) {
  if (tok >= tot.tokens) return -1;
  const int b = tab_owner<true>(rec, p.R, tok);
  const TabRecord r = rec[b];
  if (r.cached < 0) return -1;
  const int64_t pos = r.cached + (tok - r.start);
  const int64_t j = div_block(pos, p.block_size);
  int64_t blk = -1;
  const int64_t old = p.mode == kTabGrow ? div_block(r.cached + p.block_size - 1, p.block_size) : p.width;
  if (j < old) blk = load_index_rw(p.bt, p.bt_is_i64, b * p.bt_st[0] + j * p.bt_st[1]);
  else if (p.mode == kTabGrow) blk = load_index(p.free_blocks, p.free_is_i64, tot.cursor + r.first + (j - old));
  return blk < 0 ? -1 : blk * p.block_size + (pos - j * p.block_size);
}

// One block that moves: number k in the order of all blocks.
__device__ __forceinline__ void tab_move(const TableParams& p, const TabRecord* rec, const TabTotals& tot, uint32_t k) {
  const int b = tab_owner<false>(rec, p.R, k);
  const TabRecord r = rec[b];
  if (r.cached < 0) return;
  if (p.mode == kTabGrow) {
    const int64_t j = div_block(r.cached + p.block_size - 1, p.block_size) + (k - r.first);
    store_index(p.bt, p.bt_is_i64, b * p.bt_st[0] + j * p.bt_st[1],
                load_index(p.free_blocks, p.free_is_i64, tot.cursor + k));
  } else {
    const int64_t at = tot.cursor - tot.blocks + k;
    if (at >= 0 && at < p.num_free)
      store_index(p.free_out, p.free_is_i64, at,
                  load_index_rw(p.bt, p.bt_is_i64, b * p.bt_st[0] + static_cast<int64_t>(k - r.first) * p.bt_st[1]));
  }
}

// Blocks that can move at all: of a growth the ones the free list has, of a release all.
__device__ __forceinline__ uint32_t tab_moves(const TableParams& p, const TabTotals& tot) {
  if (p.mode == kTabSlots) return 0u;
  return p.mode == kTabGrow ? min(tot.blocks, tab_room(p, tot.cursor)) : tot.blocks;
}

constexpr int kTabThreads = 1024;

// The prefix sums, the outputs of one value per request, and, when FUSED, the whole write phase.
template <bool FUSED>
__global__ void __launch_bounds__(kTabThreads) table_plan_kernel(const TableParams p) {
  extern __shared__ __align__(16) uint8_t tab_smem[];
  __shared__ uint32_t warp_x[kWarp], warp_y[kWarp];
  __shared__ unsigned int taken_s;
  grid_dependency_wait();
  grid_launch_dependents();
  TabRecord* rec = FUSED ? reinterpret_cast<TabRecord*>(tab_smem) : p.records;
  TabTotals tot;
  tot.cursor = p.mode == kTabSlots ? 0 : *p.cursor;
  if (tot.cursor < 0) tot.cursor = 0;
  if (p.mode == kTabRelease && tot.cursor > p.num_free) tot.cursor = p.num_free;
  if (threadIdx.x == 0) taken_s = 0u;
  const int run = (p.R + static_cast<int>(blockDim.x) - 1) / static_cast<int>(blockDim.x);
  const int lo = min(static_cast<int>(threadIdx.x) * run, p.R), hi = min(lo + run, p.R);
  uint32_t x = 0, y = 0;
  for (int b = lo; b < hi; ++b) {
    int64_t c;
    uint32_t n, want;
    bool fits;
    tab_request(p, b, c, n, want, fits);
    x = sat_add(x, n);
    y = sat_add(y, want);
  }
  uint2 all;
  tab_scan(x, y, warp_x, warp_y, all);
  tot.tokens = all.x;
  tot.blocks = all.y;
  const uint32_t room = p.mode == kTabGrow ? tab_room(p, tot.cursor) : kTabSat;
  uint32_t at_x = x, at_y = y;
  uint32_t taken = 0;
  for (int b = lo; b < hi; ++b) {
    int64_t c;
    uint32_t n, want;
    bool fits;
    tab_request(p, b, c, n, want, fits);
    const uint32_t end = sat_add(at_y, want);
    TabRecord r;
    r.start = at_x;
    r.first = at_y;
    if (p.mode == kTabGrow) {
      const bool granted = fits && (want == 0u || end <= room);
      if (granted && want > 0u) taken = max(taken, end);
      r.cached = granted ? c : -1;
      store_index(p.lens_out, p.lens_is_i64, b, granted ? c + n : c);
    } else if (p.mode == kTabRelease) {
      r.cached = 0;
      store_index(p.lens_out, p.lens_is_i64, b, p.finished[b] ? 0 : c);
    } else {
      r.cached = c;
    }
    rec[b] = r;
    if (p.query_start != nullptr) p.query_start[b] = static_cast<int32_t>(at_x);
    at_x = sat_add(at_x, n);
    at_y = end;
  }
  if (p.query_start != nullptr && threadIdx.x == 0) p.query_start[p.R] = static_cast<int32_t>(tot.tokens);
  if (p.mode == kTabGrow && taken > 0u) atomicMax(&taken_s, taken);
  __syncthreads();
  if (threadIdx.x == 0 && p.mode != kTabSlots) {
    const int64_t next = p.mode == kTabGrow ? tot.cursor + taken_s : tot.cursor - static_cast<int64_t>(tot.blocks);
    *p.cursor_out = next < 0 ? 0 : next;
  }
  if (!FUSED && threadIdx.x == 0) *p.totals = tot;
  if constexpr (FUSED) {
    const uint32_t moves = tab_moves(p, tot);
    for (uint32_t k = threadIdx.x; k < moves; k += blockDim.x) tab_move(p, rec, tot, k);
    for (uint32_t tok = threadIdx.x; tok < static_cast<uint32_t>(p.num_tokens); tok += blockDim.x)
      p.slots[tok] = tab_slot(p, rec, tot, tok);
  }
}

constexpr int kTabWriteThreads = 256;

// The write phase with the whole machine: grid-stride over the tokens, then over the blocks that move.
__global__ void __launch_bounds__(kTabWriteThreads) table_write_kernel(const TableParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const TabTotals tot = *p.totals;
  const uint32_t step = gridDim.x * kTabWriteThreads;
  const uint32_t me = blockIdx.x * kTabWriteThreads + threadIdx.x;
  for (uint32_t tok = me; tok < static_cast<uint32_t>(p.num_tokens); tok += step) p.slots[tok] = tab_slot(p, p.records, tot, tok);
  const uint32_t moves = tab_moves(p, tot);
  for (uint32_t k = me; k < moves; k += step) tab_move(p, p.records, tot, k);
}

int64_t table_workspace_bytes(int R) { return static_cast<int64_t>(R) * sizeof(TabRecord) + 32; }

constexpr int kFusedRequests = 2048;  // 32 KB of records in shared memory
constexpr int64_t kFusedItems = 8192;

bool table_single_launch(int R, int64_t items) { return R <= kFusedRequests && items <= kFusedItems; }

int launch_tables(TableParams p, void* workspace, int64_t items, int sm_count, cudaStream_t stream) {
  const unsigned threads = p.R <= 256 ? 256u : static_cast<unsigned>(kTabThreads);
  if (table_single_launch(p.R, items))
    return launch_pdl(table_plan_kernel<true>, 1u, threads, p.R * sizeof(TabRecord), stream, p);
  p.totals = reinterpret_cast<TabTotals*>(workspace);
  p.records = reinterpret_cast<TabRecord*>(static_cast<char*>(workspace) + 32);
  const int rc = launch_pdl(table_plan_kernel<false>, 1u, threads, 0, stream, p);
  if (rc != INT8KV_OK) return rc;
  const int64_t want = (items + kTabWriteThreads - 1) / kTabWriteThreads;
  const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(want, sm_count * 8)));
  return launch_pdl(table_write_kernel, grid, kTabWriteThreads, 0, stream, p);
}

}  // namespace int8kv
