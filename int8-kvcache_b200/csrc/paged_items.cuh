// What the TMA-tiled paged-attention kernels share: the per-warp ring of staged tiles, the numbering of work items
// (arithmetic or planned on the device), and the tensor-core steps on 16-token tiles.
#pragma once

#include "common.cuh"

namespace int8kv {

constexpr int kTile = 16;  // tokens per tile

// ---------------------------------------------------------------------------------------------
// Per-warp TMA ring over the tiles [t0, t1) of one (sequence, kv head).
// ---------------------------------------------------------------------------------------------
// With DYN each stage also carries the tile's 16 K scales and 16 V scales (fp32, one per token) in a 128-byte
// slot: every lane copies one of them with cp.async, whose completion arrives on the stage's mbarrier next to
// the TMA bytes.
template <int NST, int STAGE_BYTES, int LOADS_PER_TENSOR, bool DYN = false>
struct TileRing {
  static constexpr int PIECE = STAGE_BYTES / 2 / LOADS_PER_TENSOR;  // bytes one load brings: the tensor map's box
  uint32_t stage0;  // shared address of stage 0 (1024-byte aligned)
  uint32_t bar0;    // shared address of the first mbarrier
  const CUtensorMap* tmK;
  const CUtensorMap* tmV;
  const void* bt_row;  // block table row of this sequence
  int bt_is_i64;
  int64_t bt_stride;
  int64_t bt_limit;  // number of valid entries in the row
  int tpb;           // tiles per cache block
  int head;
  int t0;   // first tile
  int lb0;  // logical block of tile t0
  int cur_win;
  int bt_cur, bt_next;
  int lane;
  uint64_t kv_policy;  // L2 policy of the tile loads: every page is read once
  // DYN only
  uint32_t scale0;        // shared address of the first 128-byte scale slot
  const float* sc_src;    // this lane's scale cache (lanes 0-15: K, 16-31: V), offset to the lane's head
  int64_t sc_blk_stride;  // strides in elements of that cache: per block, per token
  int64_t sc_tok_stride;
  int64_t sc_blocks;      // number of blocks in the scale caches: ids outside are not read
  int seq_len;

  __device__ __forceinline__ int load_window(int win) const {
    const int64_t lb = static_cast<int64_t>(lb0) + static_cast<int64_t>(win) * 32 + lane;
    if (lb >= bt_limit) return -1;  // out-of-range ids make TMA zero-fill; such tiles are never consumed
    return static_cast<int>(load_index(bt_row, bt_is_i64, lb * bt_stride));
  }

  // Barrier set-up: touches shared memory only, so it may run before the grid dependency is resolved.
  __device__ __forceinline__ void init_barriers(int lane_) {
    lane = lane_;
    kv_policy = l2_evict_first_policy();
    if (lane == 0) {
#pragma unroll
      for (int s = 0; s < NST; ++s) mbar_init(bar0 + 8 * s, DYN ? 1 + kWarp : 1);
      mbar_fence_init();
    }
    __syncwarp();
  }

  // Speculative load of the first two block-id windows at `guess_lb0`, so that the block-table read overlaps
  // the seq_lens read that the true range depends on.
  __device__ __forceinline__ void prefetch_tables(int guess_lb0) {
    lb0 = guess_lb0;
    cur_win = 0;
    bt_cur = load_window(0);
    bt_next = load_window(1);
  }

  // Fix the range once it is known; the windows are reloaded only when the guess was wrong.
  __device__ __forceinline__ void set_range(int t0_, int tpb_) {
    t0 = t0_;
    const int real_lb0 = t0_ / tpb_;
    if (real_lb0 != lb0) {
      lb0 = real_lb0;
      bt_cur = load_window(0);
      bt_next = load_window(1);
    }
  }

  // Issue the loads of tile ordinal i (tile t0 + i) into stage i % NST.  Called by all lanes, in order of i.
  __device__ __forceinline__ void issue(int i) {
    const int tau = t0 + i;
    const int lb = tau / tpb;
    const int sub = tau - lb * tpb;
    const int idx = lb - lb0;
    const int win = idx >> 5;
    if (win != cur_win) {
      bt_cur = bt_next;
      cur_win = win;
      bt_next = load_window(win + 1);
    }
    const int blk = __shfl_sync(kFull, bt_cur, idx & 31);
    if constexpr (DYN) {
      const int st = i % NST;
      const int tok = lane & 15;
      const bool live = blk >= 0 && blk < sc_blocks && tau * kTile + tok < seq_len;  // others get scale 0
      const float* src = live ? sc_src + blk * sc_blk_stride + (sub * kTile + tok) * sc_tok_stride : sc_src;
      cp_async_4(scale0 + st * 128 + lane * 4, src, live ? 4u : 0u);
      cp_async_mbar_arrive_noinc(bar0 + 8 * st);
    }
    if (lane == 0) {
      const int st = i % NST;
      const uint32_t bar = bar0 + 8 * st;
      const uint32_t dst = stage0 + st * STAGE_BYTES;
      mbar_expect_tx(bar, STAGE_BYTES);
#pragma unroll
      for (int x = 0; x < LOADS_PER_TENSOR; ++x)
        tma_load_4d(dst + x * PIECE, tmK, bar, x * 128, sub * kTile, head, blk, kv_policy);
#pragma unroll
      for (int x = 0; x < LOADS_PER_TENSOR; ++x)
        tma_load_4d(dst + (LOADS_PER_TENSOR + x) * PIECE, tmV, bar, x * 128, sub * kTile, head, blk, kv_policy);
    }
  }

  // Wait for tile ordinal i; false if the bounded wait ran out on any lane.
  __device__ __forceinline__ bool wait(int i, uint32_t limit = kWaitSpinLimit) const {
    const bool ok = mbar_wait_bounded(bar0 + 8 * (i % NST), (i / NST) & 1, limit);
    return __all_sync(kFull, ok);
  }

  __device__ __forceinline__ uint32_t stage(int i) const { return stage0 + (i % NST) * STAGE_BYTES; }
  __device__ __forceinline__ uint32_t scales(int i) const { return scale0 + (i % NST) * 128; }
};

struct ItemCoord {
  int b, h, c;       // sequence, kv head, split
  int seq_len;       // tokens of the sequence (clamped to what the table can address)
  int t0, t1;        // tile range of this split
};

// Which (sequence, kv head, split) a work item is: arithmetic only.
__device__ __forceinline__ bool item_coords(const AttnParams& p, int64_t item, ItemCoord& it) {
  const int64_t total = static_cast<int64_t>(p.B) * p.num_splits * p.Hkv;
  if (item >= total) return false;
  // a grid has fewer than 2^31 CTAs, so the item number fits 32 bits: unsigned 32-bit divisions cost a fraction of
  // the 64-bit ones, and this runs in every warp's prologue
  const uint32_t i = static_cast<uint32_t>(item);
  const uint32_t r = i / static_cast<uint32_t>(p.Hkv);
  it.h = static_cast<int>(i - r * static_cast<uint32_t>(p.Hkv));
  const uint32_t b = r / static_cast<uint32_t>(p.num_splits);
  it.c = static_cast<int>(r - b * static_cast<uint32_t>(p.num_splits));
  it.b = static_cast<int>(b);
  return true;
}

// First logical block of split c if the sequence had the hinted maximum length (the guess used to start the
// block-table read early; exact for batches of full-length sequences).
__device__ __forceinline__ int guessed_first_block(const AttnParams& p, int c) {
  return static_cast<int>(static_cast<uint32_t>(c * p.per_longest) / static_cast<uint32_t>(p.tiles_per_block));
}

// The tile range of the item: reads seq_lens[b]; every sequence splits its own tiles evenly over the parts it uses.
__device__ __forceinline__ void item_range(const AttnParams& p, ItemCoord& it) {
  int64_t sl = load_index(p.sl, p.sl_is_i64, it.b);
  const int64_t cap = p.bt_width * p.block_size;
  if (sl > cap) sl = cap;
  if (sl < 0) sl = 0;
  it.seq_len = static_cast<int>(sl);
  const int ntiles = (it.seq_len + kTile - 1) / kTile;
  // A sequence uses as many of the num_splits parts as it takes to give each about the tile count that the
  // longest sequence's parts have, and leaves the rest empty: in a ragged batch every working warp then has
  // a similar amount to read, and short sequences write few partial rows.
  const uint32_t per_longest = static_cast<uint32_t>(p.per_longest);  // ceil(hint_tiles / num_splits), at least 1
  const int used = min(p.num_splits, max(1, static_cast<int>((static_cast<uint32_t>(ntiles) + per_longest - 1) / per_longest)));
  const int per = static_cast<int>(static_cast<uint32_t>(ntiles + used - 1) / static_cast<uint32_t>(used));
  it.t0 = it.c * per;
  it.t1 = it.c < used ? min(it.t0 + per, ntiles) : it.t0;
}

// Device-planned splits.  Every sequence is cut into parts of one common length P (in 16-token tiles), the smallest
// for which the parts of all sequences, W(P) = Hkv * sum_b max(1, ceil(tiles_b / P)), fit k resident waves of
// warps, for the largest k <= plan_k_max whose parts are still plan_min_part tiles long.  P comes from the actual
// lengths, so a ragged batch fills its waves as exactly as a batch of equal lengths.  There is no planning kernel
// and no item list: every warp reads seq_lens (B values, L1-resident after the first pass), computes the same P
// with the same integer arithmetic, and locates its own item in the order (sequence, part, kv head).  Returns
// false for an item number past the end.  row0 = first partial row of the item's query-head group, or -1 when
// the sequence has a single part and the result goes straight to `out`.
// Length of sequence b clamped to what its table row can address (the host admits a plan only when that bound
// is below 2^25 tokens).
__device__ __forceinline__ int plan_len(const AttnParams& p, int b, int cap) {
  if (p.sl_is_i64) {
    const long long v = __ldg(reinterpret_cast<const long long*>(p.sl) + b);
    return v > cap ? cap : (v < 0 ? 0 : static_cast<int>(v));
  }
  return min(max(__ldg(reinterpret_cast<const int*>(p.sl) + b), 0), cap);
}

// Parts of a sequence of `len` tokens cut into parts of P tiles: max(1, ceil(tiles / P)), 0 for len < 0 (no
// sequence).  No integer division: tiles + P < 2^22 is exact in fp32, rP and the product are rounded down, so the
// product can only fall short of the quotient, and by less than one.
__device__ __forceinline__ int plan_parts(int len, int P, float rP) {
  if (len < 0) return 0;
  const int n = ((len + kTile - 1) >> 4) + P - 1;
  int q = __float2int_rz(__fmul_rd(__int2float_rz(n), rP));
  if ((q + 1) * P <= n) ++q;
  return q < 1 ? 1 : q;
}

constexpr int kPlanRun = 16;  // sequences per lane: a plan covers up to 32 * 16 sequences
constexpr int kPlanShortestPart = 8;
constexpr int kPlanHeaderTag = 0x504c414e;  // marks the 16 bytes before the status word as a plan header

// What a planning warp has to leave in the workspace: the plan header (item 0) and its sequence's {first part, parts}
// entry (the warp of part 0, head 0).  The stores are made by plan_commit, which the kernels call once the grid
// dependency is resolved: with a deferred wait the preceding call's merge may still be reading the same bytes.
struct PlanNote {
  int count, part_tiles, waves;  // header, written when count >= 0
  int table_b;                   // sequence whose table entry this warp writes, or -1
  int2 table_entry;
};

__device__ __forceinline__ void plan_commit(const AttnParams& p, const PlanNote& note, int lane) {
  if (lane != 0) return;
  if (note.count >= 0 && p.plan_header != nullptr) {
    p.plan_header[0] = note.count;
    p.plan_header[1] = note.part_tiles;
    p.plan_header[2] = note.waves;
    p.plan_header[3] = kPlanHeaderTag;
  }
  if (note.table_b >= 0) p.plan_table[note.table_b] = note.table_entry;
}

__device__ __forceinline__ bool plan_in_warp(const AttnParams& p, int64_t item, int lane, ItemCoord& it, int64_t& row0,
                                             PlanNote& note) {
  // lane l holds the lengths of sequences [l * run, (l + 1) * run) in registers; every pass below works on them
  const int cap = static_cast<int>(p.bt_width * p.block_size);
  const int run = (p.B + kWarp - 1) / kWarp;
  const int b_lo = lane * run;
  int len[kPlanRun];
#pragma unroll
  for (int j = 0; j < kPlanRun; ++j) {
    len[j] = -1;
    if (j < run && b_lo + j < p.B) len[j] = plan_len(p, b_lo + j, cap);
  }
  long long total = 0;
  int longest = 0;
#pragma unroll
  for (int j = 0; j < kPlanRun; ++j) {
    if (j >= run) break;
    const int t = len[j] < 0 ? 0 : (len[j] + kTile - 1) >> 4;
    total += t;
    longest = max(longest, t);
  }
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(kFull, total, o);
    longest = max(longest, __shfl_xor_sync(kFull, longest, o));
  }
  // estimate from W(P) ~ Hkv * (total / P + B / 2), then correct with the exact count
  const long long work = total * p.Hkv;
  const int floor_p = max(1, (longest + kMaxSplits - 1) / kMaxSplits);  // at most kMaxSplits parts per sequence
  int k = p.plan_k_max < 1 ? 1 : p.plan_k_max;
  int P = 1;
  for (; k >= 1; --k) {
    const long long room = static_cast<long long>(k) * p.plan_slots - static_cast<long long>(p.Hkv) * p.B / 2;
    if (room <= 0) continue;
    P = static_cast<int>((work + room - 1) / room);
    if (P >= p.plan_min_part || k == 1) break;
  }
  if (k < 1) k = 1;
  P = max(max(P, floor_p), kPlanShortestPart);  // below 8 tiles a part is mostly prologue and partial rows
  const long long target = min(static_cast<long long>(k) * p.plan_slots, static_cast<long long>(p.plan_grid_items));
  float rP = 1.f;
  int mine = 0, upto = 0;
  for (int round = 0; round < 64; ++round) {
    rP = __frcp_rd(__int2float_rz(P));
    mine = 0;
#pragma unroll
    for (int j = 0; j < kPlanRun; ++j) {
      if (j >= run) break;
      mine += plan_parts(len[j], P, rP);
    }
    upto = mine;  // inclusive scan over the lanes: lane 31 ends up with the number of parts
    for (int o = 1; o < kWarp; o <<= 1) {
      const int v = __shfl_up_sync(kFull, upto, o);
      if (lane >= o) upto += v;
    }
    const int parts = __shfl_sync(kFull, upto, kWarp - 1);
    // one part per sequence always fits: the launch covers at least B * Hkv items
    if (static_cast<long long>(parts) * p.Hkv <= target || P >= longest) break;
    P += round < 16 ? max(1, P >> 4) : P;
  }
  const int all_parts = __shfl_sync(kFull, upto, kWarp - 1);
  const long long count = static_cast<long long>(all_parts) * p.Hkv;
  note.count = item == 0 ? static_cast<int>(count) : -1;
  note.part_tiles = P;
  note.waves = k;
  note.table_b = -1;
  if (item >= count) return false;

  // the item in the order (sequence, part, kv head): its part index falls into exactly one lane's run
  const int part = static_cast<int>(item / p.Hkv);
  it.h = static_cast<int>(item - static_cast<int64_t>(part) * p.Hkv);
  const bool owner = part >= upto - mine && part < upto;
  int fb = 0, fc = 0, fused = 1, flen = 0;
  if (owner) {
    int first = upto - mine;
#pragma unroll
    for (int j = 0; j < kPlanRun; ++j) {
      if (j >= run) break;
      const int u = plan_parts(len[j], P, rP);
      if (part >= first && part < first + u) {
        fb = b_lo + j; fc = part - first; fused = u; flen = len[j];
      }
      first += u;
    }
  }
  const int src = __ffs(__ballot_sync(kFull, owner)) - 1;
  it.b = __shfl_sync(kFull, fb, src);
  it.c = __shfl_sync(kFull, fc, src);
  const int used = __shfl_sync(kFull, fused, src);
  it.seq_len = __shfl_sync(kFull, flen, src);
  const int tiles = (it.seq_len + kTile - 1) >> 4;
  const int per = (tiles + used - 1) / used;
  it.t0 = min(it.c * per, tiles);
  it.t1 = min(it.t0 + per, tiles);
  row0 = used == 1 ? -1 : static_cast<int64_t>(part) * p.Hq + it.h * p.G;
  if (it.c == 0 && it.h == 0) {
    note.table_b = it.b;
    note.table_entry = make_int2(part, used);
  }
  return true;
}

// First partial row of the item's query-head group when items are numbered arithmetically.
__device__ __forceinline__ int64_t arithmetic_row0(const AttnParams& p, const ItemCoord& it) {
  if (p.part == nullptr) return -1;
  return (static_cast<int64_t>(it.c) * p.B + it.b) * p.Hq + it.h * p.G;
}

// Where the item's result goes: the partial row of the group's first query head (the others follow), or null
// for `out`.  A planned sequence with a single part has no workspace row (row0 < 0): its result is final and
// goes to `out`, or to the caller's partial rows when those were asked for.
__device__ __forceinline__ float* result_row(const AttnParams& p, const ItemCoord& it, int64_t row0) {
  if (row0 >= 0) return p.part + row0 * p.row_floats;
  if (p.direct_part != nullptr) return p.direct_part + (static_cast<int64_t>(it.b) * p.Hq + it.h * p.G) * p.row_floats;
  return nullptr;
}

// Result of an empty tile range: zeros to `out` (direct mode) or lse = -inf (partial mode).
__device__ __forceinline__ void write_empty(const AttnParams& p, const ItemCoord& it, int lane, const float* prow) {
  if (prow == nullptr) {
    for (int hg = 0; hg < p.G; ++hg) {
      const int hq = it.h * p.G + hg;
      for (int d = lane; d < p.D; d += kWarp)
        store_from_float(p.out, p.out_dtype, it.b * p.o_st[0] + hq * p.o_st[1] + d * p.o_st[2], 0.f);
    }
  } else if (lane < p.G) {
    const_cast<float*>(prow)[lane * p.row_floats + p.D] = -INFINITY;
  }
}

// ---------------------------------------------------------------------------------------------
// Tensor-core steps on one 16-token tile
// ---------------------------------------------------------------------------------------------
// One V tile (16 tokens x 128 dims of one head, swizzled in shared memory) times P^T (two B registers):
// acc[j] += V^T[dims 16g+2j, 16g+2j+1 | tokens] . P^T.  `vx` are the lane's four 16-byte row pieces
// (tokens 2t, 2t+1, 2t+8, 2t+9; dims 16g..16g+15).
__device__ __forceinline__ void pv_tile(float (&acc)[8][4], const uint4 (&vx)[4], uint32_t pb0, uint32_t pb1) {
  const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&vx[0]);
  const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&vx[1]);
  const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&vx[2]);
  const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&vx[3]);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t x0 = w0[c] ^ 0x80808080u, x1 = w1[c] ^ 0x80808080u;
    const uint32_t x2 = w2[c] ^ 0x80808080u, x3 = w3[c] ^ 0x80808080u;
    const uint32_t lo01 = prmt(x0, x1, 0x5140u), hi01 = prmt(x0, x1, 0x7362u);
    const uint32_t lo23 = prmt(x2, x3, 0x5140u), hi23 = prmt(x2, x3, 0x7362u);
    mma_f16(acc[2 * c], u8pair_to_half2(lo01, 0x4140u), u8pair_to_half2(lo01, 0x4342u),
            u8pair_to_half2(lo23, 0x4140u), u8pair_to_half2(lo23, 0x4342u), pb0, pb1);
    mma_f16(acc[2 * c + 1], u8pair_to_half2(hi01, 0x4140u), u8pair_to_half2(hi01, 0x4342u),
            u8pair_to_half2(hi23, 0x4140u), u8pair_to_half2(hi23, 0x4342u), pb0, pb1);
  }
}

// Raw integer scores of one K tile: s[0..3] = 256 * (K . Qhi^T) + (K . Qlo^T) on the C fragment
// (rows = tokens g / g+8, cols = heads 2t / 2t+1).  The K bytes go to the tensor core as they are.
__device__ __forceinline__ void qk_tile(int (&s)[4], uint32_t kbase, const uint32_t (&koff)[4], const uint32_t (&qh)[8],
                                        const uint32_t (&ql)[8], bool two_limbs) {
  const uint4 a0 = lds128(kbase + koff[0]), a1 = lds128(kbase + koff[1]);
  const uint4 c0 = lds128(kbase + koff[2]), c1 = lds128(kbase + koff[3]);
  const uint32_t ka[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
  const uint32_t kc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
  int lo[4] = {0, 0, 0, 0}, hi[4] = {0, 0, 0, 0};
#pragma unroll
  for (int st = 0; st < 4; ++st) mma_s8(lo, ka[2 * st], kc[2 * st], ka[2 * st + 1], kc[2 * st + 1], ql[2 * st], ql[2 * st + 1]);
  if (two_limbs) {
#pragma unroll
    for (int st = 0; st < 4; ++st) mma_s8(hi, ka[2 * st], kc[2 * st], ka[2 * st + 1], kc[2 * st + 1], qh[2 * st], qh[2 * st + 1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = (hi[i] << 8) + lo[i];
}

template <bool IS_BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return IS_BF16 ? pack_bf162(lo, hi) : pack_half2(lo, hi);
}
template <bool IS_BF16>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (IS_BF16) mma_bf16(d, a[0], a[1], a[2], a[3], b0, b1);
  else mma_f16(d, a[0], a[1], a[2], a[3], b0, b1);
}

}  // namespace int8kv
