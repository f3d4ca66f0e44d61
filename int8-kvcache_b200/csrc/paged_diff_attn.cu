// Differential paged decode attention for sm_100a: for every query pair h and the KV pair g = h / group that serves it,
//   o = (softmax(q_{2h} K_{2g}^T / sqrt(D)) - lam_h * softmax(q_{2h+1} K_{2g+1}^T / sqrt(D))) [V_{2g} | V_{2g+1}],
// optionally followed by a root-mean-square norm over the 2 D values of o, a weight per value and a constant factor.
// The caches are the ordinary ones, [num_blocks, BS, 2 * pairs, D]: a pair's two K heads and its V row of 2 D values
// (heads 2g and 2g+1 side by side) are neighbours in every token.
//
// What it has to read is the pair's K and V rows once, 4 D values per token, for both maps and all query pairs of the
// group: HBM traffic bounds it, as it does ordinary decode attention.  Both maps therefore run in one pass over the
// pages, each with its own running maximum and sum, and both are kept unnormalised until the end, because the
// subtraction needs the two sums.  Every part of a sequence leaves one fp32 row per map in the workspace (row 2h + map of
// the part): [2 D sums of p v, before 1 / l and the V scales | m | l], with p = 2^(score - m) in log2 units and l the sum of
// p; m = -inf marks an empty part, whose other values are not written.  diff_merge_kernel joins the parts, subtracts,
// norms and writes.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "paged_items.cuh"

namespace int8kv {


// Reference of a softmax that has seen no score.  Finite, so that a score of -inf (a token that a -inf in its key masks)
// gives p = 0 even ahead of the first finite one, and a part of nothing but such tokens, or of NaN, is no empty part.
constexpr float kNoRef = -3.402823466e38f;

// ---------------------------------------------------------------------------------------------
// Every shape: one warp per (sequence, query pair, split), lanes over the dims, four tokens per step, plain loads.
// ---------------------------------------------------------------------------------------------
template <int KIND>
__device__ __forceinline__ float diff_elem(const void* base, int64_t idx) {
  if constexpr (KIND == kCacheInt8) return static_cast<float>(__ldg(reinterpret_cast<const int8_t*>(base) + idx));
  else if constexpr (KIND == kCacheBf16) return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(base) + idx));
  else return __half2float(__ldg(reinterpret_cast<const __half*>(base) + idx));
}

template <int KIND, int SLOTS>
__global__ void __launch_bounds__(128) diff_generic_kernel(const DiffParams d) {
  const AttnParams& p = d.a;
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (item >= static_cast<int64_t>(p.B) * p.num_splits * d.heads) return;
  const int h = static_cast<int>(item % d.heads);
  const int64_t rr = item / d.heads;
  const int c = static_cast<int>(rr % p.num_splits);
  const int b = static_cast<int>(rr / p.num_splits);
  const int pair = h / d.group, D = d.Dk;
  int64_t sl = load_index(p.sl, p.sl_is_i64, b);
  const int64_t cap = p.bt_width * p.block_size;
  sl = sl > cap ? cap : (sl < 0 ? 0 : sl);
  const int64_t nblk = (sl + p.block_size - 1) / p.block_size;
  const int64_t per = (nblk + p.num_splits - 1) / p.num_splits;
  const int64_t tok_lo = c * per * p.block_size;
  int64_t tok_hi = (c + 1) * per * p.block_size;
  if (tok_hi > sl) tok_hi = sl;

  float q[2][SLOTS], acc[2][2][SLOTS];  // acc[map][half of the V row]
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int dd = lane + kWarp * s;
      q[m][s] = dd < D ? load_as_float(p.q, p.q_dtype, b * p.q_st[0] + (2 * h + m) * p.q_st[1] + dd * p.q_st[2]) : 0.f;
      acc[m][0][s] = acc[m][1][s] = 0.f;
    }
  float ksc[2], mx[2] = {kNoRef, kNoRef}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    ksc[m] = (p.k_scale ? fmaxf(__ldg(p.k_scale + 2 * pair + m), 1e-6f) : 1.f) * p.sm_scale_log2;
  }
  constexpr int kTok = 4;
  for (int64_t tok = tok_lo; tok < tok_hi; tok += kTok) {
    bool ok[kTok];
    int64_t kof[kTok], vof[kTok];
    int64_t lb = tok / p.block_size;
    int off = static_cast<int>(tok - lb * p.block_size);
#pragma unroll
    for (int u = 0; u < kTok; ++u) {
      if (u > 0 && ++off >= p.block_size) {
        off = 0;
        ++lb;
      }
      ok[u] = tok + u < tok_hi;
      kof[u] = vof[u] = 0;
      if (ok[u]) {
        const int64_t blk = load_index(p.bt, p.bt_is_i64, b * p.bt_st[0] + lb * p.bt_st[1]);
        ok[u] = blk >= 0 && blk < p.num_blocks;  // never read outside the cache
        if (ok[u]) {
          kof[u] = blk * p.kc_st[0] + off * p.kc_st[1] + 2 * pair * p.kc_st[2];
          vof[u] = blk * p.vc_st[0] + off * p.vc_st[1] + 2 * pair * p.vc_st[2];
        }
      }
    }
    float pe[2][kTok];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float dot[kTok] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const int dd = lane + kWarp * s;
        if (dd < D) {
#pragma unroll
          for (int u = 0; u < kTok; ++u)
            if (ok[u]) dot[u] += q[m][s] * diff_elem<KIND>(p.kc, kof[u] + m * p.kc_st[2] + dd);
        }
      }
      for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
        for (int u = 0; u < kTok; ++u) dot[u] += __shfl_xor_sync(kFull, dot[u], o);
      }
      float mn = mx[m];
#pragma unroll
      for (int u = 0; u < kTok; ++u) {
        dot[u] = ok[u] ? dot[u] * ksc[m] : -INFINITY;
        mn = fmaxf(mn, dot[u]);
      }
      const float al = exp2f(mx[m] - mn);
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < kTok; ++u) {
        pe[m][u] = ok[u] ? exp2f(dot[u] - mn) : 0.f;
        sum += pe[m][u];
      }
      l[m] = l[m] * al + sum;
      mx[m] = mn;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        acc[m][0][s] *= al;
        acc[m][1][s] *= al;
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const int dd = lane + kWarp * s;
        if (dd < D) {
#pragma unroll
          for (int u = 0; u < kTok; ++u)
            if (ok[u]) {
              const float v = diff_elem<KIND>(p.vc, vof[u] + half * p.vc_st[2] + dd);
              acc[0][half][s] += pe[0][u] * v;
              acc[1][half][s] += pe[1][u] * v;
            }
        }
      }
  }
  const int64_t row = (static_cast<int64_t>(c) * p.B + b) * p.Hq + 2 * h;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    float* out = p.part + (row + m) * p.row_floats;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const int dd = lane + kWarp * s;
        if (dd < D) out[half * D + dd] = acc[m][half][s];
      }
    if (lane == 0) {
      out[p.D] = mx[m];
      out[p.D + 1] = l[m];
    }
  }
}

// ---------------------------------------------------------------------------------------------
// TMA-tiled kernels: D = 64 or 128, block size a multiple of 16, up to 8 query pairs per KV pair.
//
// One warp, a CTA of its own, serves one (sequence, KV pair, split) with the ring of the ordinary tiled kernels; a stage holds a 16-token
// tile of both K heads and both halves of V, so every page byte is read once for both maps and the whole group.
// Columns of the tensor-core tile (8 per block) are (map, query pair): up to 4 pairs share one block, columns 0-3 for
// the first map and 4-7 for the second (NB = 1), larger groups use a block per map (NB = 2).  From the scores on the two
// maps are just columns: one softmax step and one P.V step serve both, V is converted once.
//   D = 128: a stage is {K head 2g, K head 2g+1, V head 2g, V head 2g+1} of 16 x 128 elements; the scores of a column
//            come from its map's K tile.
//   D = 64 (INT8): the pair's two K rows are 128 consecutive bytes, one tile row; a column's query is zero in the
//            other map's half of the row, so the tile step for 128 dims gives its map's score as it is.
// ---------------------------------------------------------------------------------------------
// Column c of block nb -> map and query pair of the group.
template <int NB>
__device__ __forceinline__ int col_map(int nb, int c) { return NB == 1 ? c >> 2 : nb; }
template <int NB>
__device__ __forceinline__ int col_pair(int c) { return NB == 1 ? c & 3 : c; }

// Running softmax of the columns of one block: reference m of columns 2t (index 0) and 2t+1, in log2 units, p =
// 2^(score - m).  m is set to OFFSET below a column's maximum, so that the maximum has p = 2^OFFSET, and is set again only
// when a score reaches more than SLACK above that maximum.
//  * OFFSET + SLACK = 15 keeps p inside fp16 (65504) and uses its range: what fp16 P loses starts 2^-32 below the maximum,
//    not 2^-25, which a crowd of many tokens far below one that dominates would feel.
//  * A step needs no reduction across the token lanes, just a vote, and with SLACK = 8 the accumulators are rescaled a few
//    times per part instead of in every other tile (INT8, 32 x 32k tokens, groups of eight: 324 -> 309 us).
//  * SLACK = 0 keeps the largest probability a power of two, which is exact however few bits P has: of use where P has
//    the 8 bits of bf16 (8 x 4096 tokens: error against 64 bits 0.0019 of the output's norm instead of 0.0023, of which the
//    output's own rounding is 0.0017; 22.1 us instead of 21.8).
//
// One step over NV / 2 score rows per lane and NB column blocks at once.  x: scores before the factors sc, x[nb][2k] and
// x[nb][2k+1] being columns 2t and 2t+1 of token row g + 8k, of which the first `valid` count.  x becomes the
// probabilities; returns whether m moved, and with it the accumulators, by f[nb][0], f[nb][1].
template <int SLACK, int NB, int NV>
__device__ __forceinline__ bool softmax_step(float (&m)[NB][2], float (&x)[NB][NV], const float (&sc)[NB][2], float (&f)[NB][2],
                                             int valid, int g) {
  constexpr float kTop = 15.f, kOffset = kTop - SLACK;
  float y[NB][NV];
  float top = -INFINITY;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int k = 0; k < NV; ++k) y[nb][k] = fmaf(x[nb][k], sc[nb][k & 1], -m[nb][k & 1]);
  if (valid < 4 * NV) {  // the sequence's last tile (NV / 2 rows of 8 tokens)
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (g + 8 * (k >> 1) >= valid) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) y[nb][k] = -INFINITY;
      }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int k = 0; k < NV; ++k) top = fmaxf(top, y[nb][k]);
  const bool moved = __any_sync(kFull, top > kTop);  // also while m is kNoRef: y is huge then
  if (moved) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float z = -INFINITY;
#pragma unroll
        for (int k = e; k < NV; k += 2) {
          y[nb][k] = g + 8 * (k >> 1) < valid ? x[nb][k] * sc[nb][e] : -INFINITY;
          z = fmaxf(z, y[nb][k]);
        }
        z = fmaxf(z, __shfl_xor_sync(kFull, z, 4));
        z = fmaxf(z, __shfl_xor_sync(kFull, z, 8));
        z = fmaxf(z, __shfl_xor_sync(kFull, z, 16));
        z = fmaxf(z - kOffset, m[nb][e]);
        f[nb][e] = z == m[nb][e] ? 1.f : exp2_fast(m[nb][e] - z);  // 0 for the first score: kNoRef is that far below
        m[nb][e] = z;
#pragma unroll
        for (int k = e; k < NV; k += 2) y[nb][k] -= z;
      }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int k = 0; k < NV; ++k) x[nb][k] = exp2_fast(y[nb][k]);
  return moved;
}

// The ring of one item: tiles are issued and consumed in order, so stage, phase, block and tile-in-block are counters
// instead of divisions of the tile number.
template <int NST, int STAGE, int LOADS>
struct DiffRing : TileRing<NST, STAGE, LOADS> {
  int left;                 // tiles not issued yet
  int in_stage, in_idx, in_sub;  // next tile to issue: stage, block relative to lb0, tile inside the block
  int out_stage;            // next tile to consume
  uint32_t out_phase;

  __device__ __forceinline__ void start(const ItemCoord& it) {
    left = it.t1 - it.t0;
    in_stage = in_idx = out_stage = 0;
    out_phase = 0u;
    in_sub = it.t0 - this->lb0 * this->tpb;
  }
  __device__ __forceinline__ void issue_next() {  // called by all lanes
    if (left <= 0) return;
    --left;
    const int win = in_idx >> 5;
    if (win != this->cur_win) {
      this->bt_cur = this->bt_next;
      this->cur_win = win;
      this->bt_next = this->load_window(win + 1);
    }
    const int blk = __shfl_sync(kFull, this->bt_cur, in_idx & 31);
    if (this->lane == 0) {
      const uint32_t bar = this->bar0 + 8 * in_stage, dst = this->stage0 + in_stage * STAGE;
      mbar_expect_tx(bar, STAGE);
#pragma unroll
      for (int x = 0; x < LOADS; ++x)
        tma_load_4d(dst + x * this->PIECE, this->tmK, bar, x * 128, in_sub * kTile, this->head, blk, this->kv_policy);
#pragma unroll
      for (int x = 0; x < LOADS; ++x)
        tma_load_4d(dst + (LOADS + x) * this->PIECE, this->tmV, bar, x * 128, in_sub * kTile, this->head, blk, this->kv_policy);
    }
    in_stage = in_stage + 1 == NST ? 0 : in_stage + 1;
    if (++in_sub == this->tpb) {
      in_sub = 0;
      ++in_idx;
    }
  }
  __device__ __forceinline__ void fill() {
#pragma unroll 1
    for (int i = 0; i < NST; ++i) issue_next();
  }
  // Stage of tile u of this trip (u = 0, 1).
  __device__ __forceinline__ int stage_index(int u) const {
    const int x = out_stage + u;
    return x >= NST ? x - NST : x;
  }
  __device__ __forceinline__ uint32_t stage_addr(int u) const { return this->stage0 + stage_index(u) * STAGE; }
  // Wait for tile u of this trip; false if the bounded wait ran out on any lane.
  __device__ __forceinline__ bool wait_tile(int u, uint32_t limit = kWaitSpinLimit) const {
    const int x = out_stage + u;
    const bool ok = mbar_wait_bounded(this->bar0 + 8 * stage_index(u), x >= NST ? out_phase ^ 1u : out_phase, limit);
    return __all_sync(kFull, ok);
  }
  // The trip's `count` tiles are consumed: their stages are refilled.
  __device__ __forceinline__ void advance(int count) {
    out_stage += count;
    if (out_stage >= NST) {
      out_stage -= NST;
      out_phase ^= 1u;
    }
    __syncwarp();  // every lane has read the stages
    for (int k = 0; k < count; ++k) issue_next();
  }
  // A wait ran out: report it, and wait, again with a limit, for the `flying` tiles that were issued and not consumed.
  __device__ __forceinline__ void give_up(const AttnParams& p, int flying) {
    if (this->lane == 0 && p.status != nullptr) atomicOr(p.status, INT8KV_DEV_WAIT_TIMEOUT);
    for (int u = 0; u < flying; ++u) {
      wait_tile(0, 1u << 12);
      if (++out_stage == NST) {
        out_stage = 0;
        out_phase ^= 1u;
      }
    }
  }
};

// Whether the queries are rows that 16-byte loads can read: then nothing is staged through the idle ring.
__device__ __forceinline__ bool direct_queries(const AttnParams& p) {
  const int64_t unit = p.q_dtype == INT8KV_FP32 ? 4 : 8;  // elements per 16 bytes
  return p.q_st[2] == 1 && (reinterpret_cast<uintptr_t>(p.q) & 15u) == 0 && p.q_st[0] % unit == 0 && p.q_st[1] % unit == 0;
}

// The work item of a one-warp CTA, first half: coordinates; everything up to the first global read.
template <typename Ring>
__device__ __forceinline__ void diff_item(const DiffParams& d, Ring& ring, ItemCoord& it, int lane, int heads_per_box) {
  const AttnParams& p = d.a;
  ring.bt_is_i64 = p.bt_is_i64;
  ring.bt_stride = p.bt_st[1];
  ring.bt_limit = p.bt_width;
  ring.tpb = p.tiles_per_block;
  if (lane == 0) {
    tma_prefetch_desc(ring.tmK);
    tma_prefetch_desc(ring.tmV);
  }
  ring.init_barriers(lane);
  grid_dependency_wait();  // from here on global memory is read
  grid_launch_dependents();
  item_coords(p, blockIdx.x, it);  // the grid is exactly the items
  ring.bt_row = reinterpret_cast<const char*>(p.bt) + it.b * p.bt_st[0] * (p.bt_is_i64 ? 8 : 4);
  ring.head = it.h * heads_per_box;
}

// Second half: tile range, the first of the item's 2 * group partial rows, and the first tiles under way (unless `hold`).
// Returns false when the part is empty.
template <typename Ring>
__device__ __forceinline__ bool diff_range(const DiffParams& d, Ring& ring, ItemCoord& it, float*& prow, int lane, bool hold) {
  const AttnParams& p = d.a;
  ring.prefetch_tables(guessed_first_block(p, it.c));
  item_range(p, it);
  prow = p.part + arithmetic_row0(p, it) * p.row_floats;
  if (it.t0 >= it.t1) {  // rows that the join skips
    if (lane < p.G) prow[lane * p.row_floats + p.D] = -INFINITY;
    return false;
  }
  ring.set_range(it.t0, p.tiles_per_block);
  ring.start(it);
  if (!hold) ring.fill();
  return true;
}

// 16 bytes of a query, requested at this place in the program (the values are used much later).
__device__ __forceinline__ uint4 ldg_early(const void* ptr) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(ptr));
  return v;
}

// Two 16-bit floats -> floats.
__device__ __forceinline__ float2 unpack16(uint32_t w, int dtype) {
  if (dtype == INT8KV_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Queries of a column as two INT8 limbs, q ~= q_mul * (256 hi + lo) with |256 hi + lo| <= 32000: 16-bit fixed point per
// head, so that the K bytes go to the INT8 tensor cores as they lie in the cache.  The 1.5 * 2^23 addition of the
// FMA rounds and leaves the integer in the low mantissa bits.  `abits`: bits of the largest magnitude of this lane's
// elements.  A NaN or infinity in a head makes q_mul NaN, and with it the
// head's output.
struct QueryScale {
  float inv, mul;
};
template <int LANES>  // lanes that share a head: the column's four, or two (D = 64 with a block per map)
__device__ __forceinline__ QueryScale query_scale(uint32_t abits) {
  abits = max(abits, __shfl_xor_sync(kFull, abits, 1));
  if (LANES == 4) abits = max(abits, __shfl_xor_sync(kFull, abits, 2));
  const float amax = __uint_as_float(abits);
  QueryScale s;
  const bool live = amax > 1e-20f;
  s.inv = live ? __fdividef(32000.f, amax) : 0.f;
  s.mul = live ? __fdividef(1.f, s.inv) : 0.f;
  if (abits >= 0x7f800000u) s.mul = __uint_as_float(0x7fffffffu);
  return s;
}
__device__ __forceinline__ void query_limbs(float a, float b, float c, float e, float inv, uint32_t& lo, uint32_t& hi) {
  const float t0 = fmaf(a, inv, kRoundMagic), t1 = fmaf(b, inv, kRoundMagic), t2 = fmaf(c, inv, kRoundMagic), t3 = fmaf(e, inv, kRoundMagic);
  lo = prmt(prmt(__float_as_uint(t0), __float_as_uint(t1), 0x0040u), prmt(__float_as_uint(t2), __float_as_uint(t3), 0x0040u), 0x5410u);
  // the second byte of v + 128 is round(v / 256): adding 128 to the float is exact
  hi = prmt(prmt(__float_as_uint(t0 + 128.f), __float_as_uint(t1 + 128.f), 0x0051u),
            prmt(__float_as_uint(t2 + 128.f), __float_as_uint(t3 + 128.f), 0x0051u), 0x5410u);
}

// The item's partial rows go through shared memory (the ring's stages, free by then) and leave as whole lines: written from
// the fragments (16 bytes per lane, 64 bytes apart) they would reach the workspace as 1024 half-written sectors per
// warp, 2.2 us at the end of every item.  Lane t's rows lie in slots t, t + 4, ..., a row (a multiple of 128 bytes plus
// 16) apart, so that a warp's 16-byte stores spread over all banks.
template <int NB>
__device__ __forceinline__ int row_slot(int nb, int e, int t) { return t + 4 * (e + 2 * nb); }

template <int NB, int VALUES>
__device__ __forceinline__ void store_rows(float* prow, uint32_t slots, int group, int lane) {
  constexpr int kRow = VALUES + 4;  // floats
  __syncwarp();
#pragma unroll 4
  for (int slot = 0; slot < 8 * NB; ++slot) {
    const int t = slot & 3, e = (slot >> 2) & 1, nb = slot >> 3;
    const int hg = col_pair<NB>(2 * t + e), m = col_map<NB>(nb, 2 * t + e);
    if (hg >= group) continue;
    float* dst = prow + (2 * hg + m) * kRow;
#pragma unroll
    for (int i = 0; i < VALUES; i += 128) {
      const uint4 x = lds128(slots + (slot * kRow + i + 4 * lane) * 4);
      *reinterpret_cast<uint4*>(dst + i + 4 * lane) = x;
    }
    if (lane == 0) *reinterpret_cast<uint4*>(dst + VALUES) = lds128(slots + (slot * kRow + VALUES) * 4);
  }
}
__device__ __forceinline__ void sts128(uint32_t addr, float a, float b, float c, float e) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(e) : "memory");
}
__device__ __forceinline__ void sts64(uint32_t addr, float a, float b) {
  asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t addr, float a) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(a) : "memory");
}

// One V tile (16 tokens x 128 values, INT8) times P^T of NB column blocks.  ldmatrix transposes 16-bit units: lane (g, t)
// receives the bytes of values 2g, 2g+1 of a 16-value chunk for tokens 2t and 2t+1 in one register, from which one byte
// permute each makes the two rows of the MMA's A operand (row g = value 2g, row g + 8 = value 2g + 1), as 1024 + (v + 128)
// in fp16; the subtraction of 1152 is exact.
template <int NB>
__device__ __forceinline__ void pv_blocks(float (&acc)[NB][8][4], uint32_t tile, const uint32_t (&voff)[4], const uint32_t (&pb)[NB][2]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {  // two chunks
    uint32_t w[4];
    ldmatrix_x4_trans(w, tile + voff[c]);  // {tokens 0-7, 8-15} of chunk 2c, then of chunk 2c + 1
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] ^= 0x80808080u;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t f0 = u8pair_to_half2(w[2 * s], 0x4240u), f1 = u8pair_to_half2(w[2 * s], 0x4341u);
      const uint32_t f2 = u8pair_to_half2(w[2 * s + 1], 0x4240u), f3 = u8pair_to_half2(w[2 * s + 1], 0x4341u);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) mma_f16(acc[nb][2 * c + s], f0, f1, f2, f3, pb[nb][0], pb[nb][1]);
    }
  }
}

// Scores of one 16-token tile against every column, as integers: s[nb] = 256 (K . Qhi) + (K . Qlo) on the C fragment.
// The limbs' and blocks' chains of MMAs run side by side.
template <int DK, int NB>
__device__ __forceinline__ void diff_scores(int (&s)[NB][4], uint32_t kb, const uint32_t (&koff)[4], const uint32_t (&qh)[NB][8],
                                            const uint32_t (&ql)[NB][8], int t) {
  constexpr int KT = DK / 64;                 // K tiles: the two heads' (D = 128), or one of both (D = 64)
  constexpr int CH = NB > KT ? NB : KT;       // chains: block nb against its map's tile; NB = 1, D = 128: both tiles
  uint32_t ka[KT][8], kc[KT][8];
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    const uint4 a0 = lds128(kb + k * 2048 + koff[0]), a1 = lds128(kb + k * 2048 + koff[1]);
    const uint4 c0 = lds128(kb + k * 2048 + koff[2]), c1 = lds128(kb + k * 2048 + koff[3]);
    ka[k][0] = a0.x; ka[k][1] = a0.y; ka[k][2] = a0.z; ka[k][3] = a0.w; ka[k][4] = a1.x; ka[k][5] = a1.y; ka[k][6] = a1.z; ka[k][7] = a1.w;
    kc[k][0] = c0.x; kc[k][1] = c0.y; kc[k][2] = c0.z; kc[k][3] = c0.w; kc[k][4] = c1.x; kc[k][5] = c1.y; kc[k][6] = c1.z; kc[k][7] = c1.w;
  }
  int lo[CH][4], hi[CH][4];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) lo[c][r] = hi[c][r] = 0;
#pragma unroll
  for (int st = 0; st < 4; ++st)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int k = KT == 1 ? 0 : c, nb = NB == 1 ? 0 : c;
      mma_s8(lo[c], ka[k][2 * st], kc[k][2 * st], ka[k][2 * st + 1], kc[k][2 * st + 1], ql[nb][2 * st], ql[nb][2 * st + 1]);
      mma_s8(hi[c], ka[k][2 * st], kc[k][2 * st], ka[k][2 * st + 1], kc[k][2 * st + 1], qh[nb][2 * st], qh[nb][2 * st + 1]);
    }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (CH > NB) s[nb][r] = t < 2 ? (hi[0][r] << 8) + lo[0][r] : (hi[CH - 1][r] << 8) + lo[CH - 1][r];  // own map's tile
      else s[nb][r] = (hi[nb][r] << 8) + lo[nb][r];
    }
}

// Items resident per SM and ring depth: 192 KB of ring per SM (the bytes in flight that keep HBM busy); a stage is 8 KB
// for D = 128 and 4 KB for D = 64.  kTrip tiles are consumed per trip: with 4 KB tiles two, for which one softmax step
// serves both.  The accumulators, 32 floats per lane and (column block, 128 values of V), set how many warps the register
// file carries; more, shallower rings win as long as two trips fit (61 ragged sequences of up to 8191 tokens, D = 64, no
// groups: 12 / 16 per SM 87.6 / 85.4 us; 16 x 4096, D = 128, groups of four: 8 / 10 per SM 20.0 / 22.0 us).
template <int DK, int NB>
struct DiffInt8Shape {
  static constexpr int kHalves = DK / 64;
  static constexpr int kStage = kHalves * 4096;
  static constexpr int kTrip = DK == 128 ? 1 : 2;
  static constexpr int kPerSm = DK == 64 && NB == 1 ? 16 : 8;
  static constexpr int kStages = 192 * 1024 / (kPerSm * kStage);
  static constexpr int kSmem = kStages * (kStage + 8) + 1024;
};

template <int DK, int NB>
__global__ void __launch_bounds__(kWarp, DiffInt8Shape<DK, NB>::kPerSm)
diff_int8_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ DiffParams d) {
  using Shape = DiffInt8Shape<DK, NB>;
  constexpr int NST = Shape::kStages, STAGE = Shape::kStage, TRIP = Shape::kTrip, HV = Shape::kHalves;
  constexpr int QB = DK == 64 ? 1 : NB;  // rows of 32 query values per lane (D = 64: a lane's half row is one map's)
  extern __shared__ uint8_t smem_raw[];
  const AttnParams& p = d.a;
  const int lane = threadIdx.x, g = lane >> 2, t = lane & 3;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  DiffRing<NST, STAGE, 1> ring;
  ring.stage0 = smem_base;
  ring.bar0 = smem_base + NST * STAGE;
  ring.tmK = &tmK;
  ring.tmV = &tmV;
  ItemCoord it;
  float* prow;
  diff_item(d, ring, it, lane, HV);

  // Lane (g, t) holds column g's dims [32t, 32t+32) of the 128-value tile row.  Rows of 16-bit values that 16-byte loads
  // can read (the usual case) are requested ahead of lengths, tables and tiles, and converted while the tiles are in
  // flight; any other layout is staged through the ring's first stage, ahead of the tiles.
  const bool direct = direct_queries(p), raw16 = direct && p.q_dtype != INT8KV_FP32;
  int64_t q_at[QB];
  bool q_live[QB];
#pragma unroll
  for (int k = 0; k < QB; ++k) {
    const int m = DK == 64 ? t >> 1 : col_map<NB>(k, g), hg = col_pair<NB>(g);
    q_live[k] = hg < d.group && (DK == 128 || NB == 2 || m == col_map<NB>(0, g));
    q_at[k] = it.b * p.q_st[0] + (2 * (it.h * d.group + hg) + m) * p.q_st[1] + (DK == 128 ? 32 * t : 32 * (t & 1)) * p.q_st[2];
  }
  uint4 raw[QB][4];
#pragma unroll
  for (int k = 0; k < QB; ++k)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      raw[k][w] = make_uint4(0u, 0u, 0u, 0u);
      if (raw16 && q_live[k]) raw[k][w] = ldg_early(reinterpret_cast<const uint16_t*>(p.q) + q_at[k] + 8 * w);
    }
  const float ks0 = __ldg(p.k_scale + 2 * it.h), ks1 = __ldg(p.k_scale + 2 * it.h + 1);
  if (!diff_range(d, ring, it, prow, lane, !direct)) return;
  const int n = it.t1 - it.t0;

  uint32_t qh[NB][8], ql[NB][8];
  float q_mul[QB];
  if (raw16) {
#pragma unroll
    for (int k = 0; k < QB; ++k) {
      uint32_t top = 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = __vmaxu2(top, reinterpret_cast<const uint32_t*>(&raw[k][i >> 2])[i & 3] & 0x7fff7fffu);
      top = max(top & 0xffffu, top >> 16);  // magnitudes of 16-bit floats order like their bits
      const float2 amax = unpack16(top, p.q_dtype);
      const QueryScale sc = query_scale<DK == 64 && NB == 2 ? 2 : 4>(__float_as_uint(amax.x));
      q_mul[k] = sc.mul;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4& r = raw[k][i >> 1];
        const float2 x = unpack16(i & 1 ? r.z : r.x, p.q_dtype), y = unpack16(i & 1 ? r.w : r.y, p.q_dtype);
        query_limbs(x.x, x.y, y.x, y.y, sc.inv, ql[k][i], qh[k][i]);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < QB; ++k) {
      float x[32];
      if (q_live[k]) {
        load32_as_float(p.q, p.q_dtype, q_at[k], p.q_st[2], x, ring.stage0, lane);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = 0.f;
      }
      uint32_t abits = 0u;
#pragma unroll
      for (int i = 0; i < 32; ++i) abits = max(abits, __float_as_uint(x[i]) & 0x7fffffffu);
      const QueryScale sc = query_scale<DK == 64 && NB == 2 ? 2 : 4>(abits);
      q_mul[k] = sc.mul;
#pragma unroll
      for (int i = 0; i < 8; ++i) query_limbs(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], sc.inv, ql[k][i], qh[k][i]);
    }
    if (!direct) {
      fence_proxy_async_smem();  // the queries were staged by the lanes; the first tile is written by the TMA unit
      __syncwarp();
      ring.fill();
    }
  }
  if constexpr (DK == 64 && NB == 2) {  // the row belongs to one map, that is to one block; zero in the other
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ql[1][i] = t >= 2 ? ql[0][i] : 0u;
      qh[1][i] = t >= 2 ? qh[0][i] : 0u;
      ql[0][i] = t < 2 ? ql[0][i] : 0u;
      qh[0][i] = t < 2 ? qh[0][i] : 0u;
    }
  }
  // score multipliers of columns 2t and 2t+1, which belong to the same map; D = 64, NB = 2: lanes 0, 1 of a column hold
  // the first map's scale, lanes 2, 3 the second's
  float sc[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float mul = q_mul[QB == 1 ? 0 : nb];
    const int holder = DK == 64 && NB == 2 ? 2 * nb : 0;
    const float kmul = fmaxf(col_map<NB>(nb, 2 * t) ? ks1 : ks0, 1e-6f) * p.sm_scale_log2;
    sc[nb][0] = kmul * __shfl_sync(kFull, mul, (2 * t) * 4 + holder);
    sc[nb][1] = kmul * __shfl_sync(kFull, mul, (2 * t + 1) * 4 + holder);
  }

  const uint32_t koff[4] = {swz128(g, 2 * t), swz128(g, 2 * t + 1), swz128(g + 8, 2 * t), swz128(g + 8, 2 * t + 1)};
  // ldmatrix lane roles in a V tile: matrix lane / 8 = (tokens 0-7 / 8-15, chunk 2c / 2c + 1), row lane % 8
  uint32_t voff[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) voff[c] = swz128((lane & 7) + 8 * ((lane >> 3) & 1), 2 * c + (lane >> 4));
  // The columns' sums are a row of the P.V product too, with ones for V: they then hold what was multiplied, P as rounded
  // to fp16, whose error cancels where one token carries the softmax, and need no reduction at the end.
  constexpr uint32_t kOnes = 0x3c003c00u;
  float acc[HV][NB][8][4], sum[NB][4], m[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb][0] = m[nb][1] = kNoRef;
    sum[nb][0] = sum[nb][1] = sum[nb][2] = sum[nb][3] = 0.f;
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[h][nb][j][0] = acc[h][nb][j][1] = acc[h][nb][j][2] = acc[h][nb][j][3] = 0.f;
  }
  const int limit = min(it.seq_len, it.t1 * kTile) - it.t0 * kTile;  // tokens of the range

  // When the range holds an odd number of tiles the last trip of two has one all masked tile; its stage holds finite
  // integers, stale or fresh, that meet p = 0.
  for (int i = 0; i < n; i += TRIP) {
    bool ok = ring.wait_tile(0);
    if (TRIP == 2 && ok && i + 1 < n) ok = ring.wait_tile(1);
    if (!ok) {
      ring.give_up(p, min(NST, n - i));
      return;
    }
    float x[NB][4 * TRIP], f[NB][2];
#pragma unroll
    for (int u = 0; u < TRIP; ++u) {
      int raw[NB][4];
      diff_scores<DK, NB>(raw, ring.stage_addr(u), koff, qh, ql, t);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[nb][4 * u + r] = static_cast<float>(raw[nb][r]);
    }
    if (softmax_step<8>(m, x, sc, f, limit - i * kTile, g)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        sum[nb][0] *= f[nb][0]; sum[nb][1] *= f[nb][1];
#pragma unroll
        for (int h = 0; h < HV; ++h)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            acc[h][nb][j][0] *= f[nb][0]; acc[h][nb][j][1] *= f[nb][1]; acc[h][nb][j][2] *= f[nb][0]; acc[h][nb][j][3] *= f[nb][1];
          }
      }
    }
#pragma unroll
    for (int u = 0; u < TRIP; ++u) {
      uint32_t pb[NB][2];  // P^T as B operands
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        pb[nb][0] = movmatrix_trans(pack_half2(x[nb][4 * u], x[nb][4 * u + 1]));
        pb[nb][1] = movmatrix_trans(pack_half2(x[nb][4 * u + 2], x[nb][4 * u + 3]));
        mma_f16(sum[nb], kOnes, kOnes, kOnes, kOnes, pb[nb][0], pb[nb][1]);
      }
#pragma unroll
      for (int h = 0; h < HV; ++h) pv_blocks<NB>(acc[h], ring.stage_addr(u) + STAGE / 2 + h * 2048, voff, pb);
    }
    ring.advance(TRIP);
  }

  // ---- epilogue: lane (g, t) holds values 128 h + 16 j + 2g, + 1 of columns 2t and 2t+1 ---------------------------
  constexpr int kRow = (2 * DK + 4) * 4;  // bytes of a partial row
  static_assert(8 * NB * kRow <= NST * STAGE, "the rows of a group fit the ring");
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // (columns without a query pair write slots that are not copied out)
      const uint32_t row = ring.stage0 + row_slot<NB>(nb, e, t) * kRow;
#pragma unroll
      for (int h = 0; h < HV; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) sts64(row + (128 * h + 16 * j + 2 * g) * 4, acc[h][nb][j][e], acc[h][nb][j][e + 2]);
      if (g == 0) sts128(row + 2 * DK * 4, m[nb][e], sum[nb][e], 0.f, 0.f);
    }
  store_rows<NB, 2 * DK>(prow, ring.stage0, d.group, lane);
}

// ---------------------------------------------------------------------------------------------
// bf16 / fp16 caches: same ring and columns, fragments straight from shared memory with ldmatrix
// ---------------------------------------------------------------------------------------------
// A stage is 16 KB for D = 128 and 8 KB for D = 64 (45 ragged fp16 sequences of up to 8191 tokens, D = 128, groups of four:
// 4 items of 3 stages / 6 of 2 per SM 120 / 115 us).
template <int DK>
struct DiffF16Shape {
  static constexpr int kStage = DK * 128;  // 2 tensors x 2 heads x 16 tokens x 2 DK bytes
  static constexpr int kPerSm = DK == 128 ? 6 : 12;
  static constexpr int kStages = 192 * 1024 / (kPerSm * kStage);
  static constexpr int kSmem = kStages * (kStage + 8) + 1024;
};

template <int DK, int NB, bool IS_BF16>
__global__ void __launch_bounds__(kWarp, DiffF16Shape<DK>::kPerSm)
diff_f16_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ DiffParams d) {
  using Shape = DiffF16Shape<DK>;
  constexpr int NST = Shape::kStages, STAGE = Shape::kStage;
  constexpr int STEPS = DK / 16;          // 16-dim steps of a score, 16-dim rows of a half of the output
  constexpr int PIECE = 4096;             // one load: 128 bytes x 16 tokens x 2 heads
  extern __shared__ uint8_t smem_raw[];
  const AttnParams& p = d.a;
  const int lane = threadIdx.x, g = lane >> 2, t = lane & 3;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  DiffRing<NST, STAGE, DK / 64> ring;
  static_assert(TileRing<NST, STAGE, DK / 64>::PIECE == PIECE, "box of the tensor map");
  ring.stage0 = smem_base;
  ring.bar0 = smem_base + NST * STAGE;
  ring.tmK = &tmK;
  ring.tmV = &tmV;
  ItemCoord it;
  float* prow;
  diff_item(d, ring, it, lane, 2);
  if (!diff_range(d, ring, it, prow, lane, false)) return;
  const int n = it.t1 - it.t0;

  // Queries as B fragments, rounded to the cache's type: step s covers dims 16s..16s+15; lane (g, t) holds column g,
  // dims 16s+2t, +1 and 16s+8+2t, +1
  uint32_t qf[NB][2 * STEPS];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int map = col_map<NB>(nb, g), hg = col_pair<NB>(g);
    const int64_t base = it.b * p.q_st[0] + (2 * (it.h * d.group + hg) + map) * p.q_st[1];
    const bool same_type = p.q_dtype == (IS_BF16 ? INT8KV_BF16 : INT8KV_FP16) && p.q_st[2] == 1 &&
                           ((reinterpret_cast<uintptr_t>(p.q) + 2 * base) & 3u) == 0;
    if (hg >= d.group) {
#pragma unroll
      for (int s = 0; s < 2 * STEPS; ++s) qf[nb][s] = 0u;
    } else if (same_type) {
      const uint32_t* words = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(p.q) + base);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        qf[nb][2 * s] = __ldg(words + 8 * s + t);
        qf[nb][2 * s + 1] = __ldg(words + 8 * s + 4 + t);
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2 * STEPS; ++s) {
        const int dim = 8 * s + 2 * t;
        qf[nb][s] = pack16<IS_BF16>(load_as_float(p.q, p.q_dtype, base + dim * p.q_st[2]),
                                    load_as_float(p.q, p.q_dtype, base + (dim + 1) * p.q_st[2]));
      }
    }
  }

  constexpr uint32_t kOnes = IS_BF16 ? 0x3f803f80u : 0x3c003c00u;  // the columns' sums as a row of the product, see above
  float acc[2][NB][STEPS][4], sum[NB][4], m[NB][2], sc[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb][0] = m[nb][1] = kNoRef;
    sc[nb][0] = sc[nb][1] = p.sm_scale_log2;
    sum[nb][0] = sum[nb][1] = sum[nb][2] = sum[nb][3] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < STEPS; ++j) acc[h][nb][j][0] = acc[h][nb][j][1] = acc[h][nb][j][2] = acc[h][nb][j][3] = 0.f;
  }
  // ldmatrix lane roles: matrix mi = lane / 8, row r = lane % 8
  const int mi = lane >> 3, r8 = lane & 7;
  const int k_tok = r8 + 8 * (mi & 1), k_chunk = mi >> 1;   // K (non-transposed): matrices (tok lo/hi, chunk +0/+1)
  const int v_tok = r8 + 8 * (mi >> 1), v_chunk = mi & 1;   // V (transposed)

  for (int i = 0; i < n; ++i) {
    if (!ring.wait_tile(0)) {
      ring.give_up(p, min(NST, n - i));
      return;
    }
    const uint32_t kb = ring.stage_addr(0), vb = kb + STAGE / 2;
    float sm[2][2][4];  // [map's K head][even / odd step]: two chains per head
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sm[k][0][r] = sm[k][1][r] = 0.f;
      const int nb = NB == 1 ? 0 : k;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int ch = 2 * s + k_chunk;  // 16-byte chunk of the row
        uint32_t a[4];
        ldmatrix_x4(a, kb + (ch >> 3) * PIECE + k * 2048 + swz128(k_tok, ch & 7));
        mma16<IS_BF16>(sm[k][s & 1], a, qf[nb][2 * s], qf[nb][2 * s + 1]);
      }
    }
    const int nvalid = it.seq_len - (it.t0 + i) * kTile;  // >= 1
    float x[NB][4], f[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 4; ++r)  // NB = 1: both K heads met all columns, each column keeps its own map's score
        x[nb][r] = NB == 1 ? (t < 2 ? sm[0][0][r] + sm[0][1][r] : sm[1][0][r] + sm[1][1][r]) : sm[nb][0][r] + sm[nb][1][r];
    if (softmax_step<0>(m, x, sc, f, nvalid, g)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        sum[nb][0] *= f[nb][0]; sum[nb][1] *= f[nb][1];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < STEPS; ++j) {
            acc[h][nb][j][0] *= f[nb][0]; acc[h][nb][j][1] *= f[nb][1]; acc[h][nb][j][2] *= f[nb][0]; acc[h][nb][j][3] *= f[nb][1];
          }
      }
    }
    uint32_t pb[NB][2];  // P^T as B operands, rounded to the cache's type
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      pb[nb][0] = movmatrix_trans(pack16<IS_BF16>(x[nb][0], x[nb][1]));
      pb[nb][1] = movmatrix_trans(pack16<IS_BF16>(x[nb][2], x[nb][3]));
      const uint32_t ones[4] = {kOnes, kOnes, kOnes, kOnes};
      mma16<IS_BF16>(sum[nb], ones, pb[nb][0], pb[nb][1]);
    }
    // A float cache may hold NaN or infinities behind the last token, and 0 * NaN would poison the sums: those V values
    // are zeroed (their scores were replaced above).
    uint32_t keep_lo = 0xffffffffu, keep_hi = 0xffffffffu;  // masks for (tokens 2t, 2t+1) and (2t+8, 2t+9)
    if (nvalid < kTile) {
      keep_lo = (2 * t < nvalid ? 0x0000ffffu : 0u) | (2 * t + 1 < nvalid ? 0xffff0000u : 0u);
      keep_hi = (2 * t + 8 < nvalid ? 0x0000ffffu : 0u) | (2 * t + 9 < nvalid ? 0xffff0000u : 0u);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const int ch = 2 * j + v_chunk;
        uint32_t a[4];
        ldmatrix_x4_trans(a, vb + (ch >> 3) * PIECE + h * 2048 + swz128(v_tok, ch & 7));
        a[0] &= keep_lo; a[1] &= keep_lo; a[2] &= keep_hi; a[3] &= keep_hi;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma16<IS_BF16>(acc[h][nb][j], a, pb[nb][0], pb[nb][1]);
      }
    ring.advance(1);
  }

  constexpr int kRow = (2 * DK + 4) * 4;  // bytes of a partial row
  static_assert(8 * NB * kRow <= NST * STAGE, "the rows of a group fit the ring");
  // ---- epilogue: values DK h + 16 j + g (registers 0, 1) and + 8 (2, 3) of columns 2t and 2t+1 --------------------
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t row = ring.stage0 + row_slot<NB>(nb, e, t) * kRow;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
          sts32(row + (DK * h + 16 * j + g) * 4, acc[h][nb][j][e]);
          sts32(row + (DK * h + 16 * j + g + 8) * 4, acc[h][nb][j][e + 2]);
        }
      if (g == 0) sts128(row + 2 * DK * 4, m[nb][e], sum[nb][e], 0.f, 0.f);
    }
  store_rows<NB, 2 * DK>(prow, ring.stage0, d.group, lane);
}

// ---------------------------------------------------------------------------------------------
// Join of the parts, subtraction, norm: one CTA per (sequence, query pair), grid (sequence, pair).
// ---------------------------------------------------------------------------------------------
// A short kernel on the critical path of a small call.  The two rows of a part lie side by side and arrive by one bulk copy
// per part, all parts of a batch in flight at once: ordinary loads, 1024 lines from as many 16-byte pieces, ran at
// 9 bytes per cycle and SM, limited by the misses that an SM keeps outstanding.  A warp then owns 128 bytes of the row:
// lane (sub, c) takes 16-byte piece c of the parts sub, sub + 4, ... of both maps; maximum, sum and weighted rows meet
// in two shuffle steps, and the only CTA barrier is the norm's.  Rows of empty parts (m = -inf) were never
// written: what is read of them meets no weight.
constexpr int kMergeBatch = 32;  // parts in shared memory at a time, at most

__global__ void __launch_bounds__(512) diff_merge_kernel(const __grid_constant__ DiffParams d, const int batch) {
  extern __shared__ __align__(16) uint8_t merge_smem[];  // [batch] pairs of rows
  __shared__ __align__(8) uint64_t bar_s;
  __shared__ float sq_s[16];
  const AttnParams& p = d.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane >> 3;
  const int b = blockIdx.x, h = blockIdx.y;
  const int dim = 32 * warp + 4 * (lane & 7);  // first of this lane's four values
  const bool live = dim < p.row_floats;
  const uint32_t rows_s = smem_u32(merge_smem), bar = smem_u32(&bar_s), pair_bytes = 8u * p.row_floats;
  if (tid == 0) {
    mbar_init(bar, 1);
    mbar_fence_init();
  }
  // lam, the norm's weights and the scales are inputs of the call: whatever wrote them was complete before the attention kernel let
  // this one be scheduled
  const float lam = load_as_float(d.lam, d.lam_dtype, h * d.lam_st);
  float nw[4] = {1.f, 1.f, 1.f, 1.f};
  if (d.norm_w != nullptr && sub == 0) {
    if (dim + 3 < p.D) {
      load4_as_float(d.norm_w, d.norm_dtype, dim, 1, nw);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (dim + u < p.D) nw[u] = load_as_float(d.norm_w, d.norm_dtype, dim + u);
    }
  }
  // V scale of this lane's values, which may straddle the two halves of the row (head dims that are no multiple of 4)
  float vs[4];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    vs[u] = p.v_scale != nullptr && dim + u < p.D ? fmaxf(p.v_scale[2 * (h / d.group) + (dim + u >= d.Dk)], 1e-6f) : 1.f;
  __syncthreads();  // the barrier is initialised
  grid_dependency_wait();
  grid_launch_dependents();
  const int R = p.num_splits;
  const int64_t stride_r = static_cast<int64_t>(p.B) * p.Hq * p.row_floats;
  const float* base = p.part + (static_cast<int64_t>(b) * p.Hq + 2 * h) * p.row_floats;
  float4 acc[2];
  float top[2] = {-INFINITY, -INFINITY}, den[2] = {0.f, 0.f};
  acc[0] = acc[1] = make_float4(0.f, 0.f, 0.f, 0.f);
  uint32_t phase = 0u;
  for (int r0 = 0; r0 < R; r0 += batch) {
    const int count = min(batch, R - r0);
    if (warp == 0) {
      if (lane == 0) mbar_expect_tx(bar, count * pair_bytes);
      __syncwarp();
      for (int r = lane; r < count; r += kWarp)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(rows_s + r * pair_bytes), "l"(base + (r0 + r) * stride_r), "r"(pair_bytes), "r"(bar) : "memory");
    }
    if (!__syncthreads_and(mbar_wait_bounded(bar, phase))) {
      if (tid == 0 && p.status != nullptr) atomicOr(p.status, INT8KV_DEV_WAIT_TIMEOUT);
      return;
    }
    phase ^= 1u;
    // this lane's (at most eight) parts, both maps side by side
    float ref[kMergeBatch / 4][2];
    float t[2] = {top[0], top[1]};
#pragma unroll
    for (int u = 0; u < kMergeBatch / 4; ++u)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int r = sub + 4 * u;
        ref[u][m] = r < count ? lds32f(rows_s + r * pair_bytes + 4u * (m * p.row_floats + p.D)) : -INFINITY;
        t[m] = fmaxf(t[m], ref[u][m]);
      }
#pragma unroll
    for (int o = 8; o <= 16; o <<= 1) {  // the four sub-rows of parts share the reference
      const float a0 = __shfl_xor_sync(kFull, t[0], o), a1 = __shfl_xor_sync(kFull, t[1], o);
      t[0] = fmaxf(t[0], a0);
      t[1] = fmaxf(t[1], a1);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (r0 > 0) {
        const float f = top[m] == -INFINITY ? 1.f : exp2_fast(top[m] - t[m]);
        den[m] *= f;
        acc[m].x *= f; acc[m].y *= f; acc[m].z *= f; acc[m].w *= f;
      }
      top[m] = t[m];
    }
#pragma unroll
    for (int u = 0; u < kMergeBatch / 4; ++u) {
      if (4 * u >= count) break;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (ref[u][m] != -INFINITY && live) {
          const uint32_t row = rows_s + (sub + 4 * u) * pair_bytes + 4u * m * p.row_floats;
          const float w = exp2_fast(ref[u][m] - t[m]);
          const uint4 q = lds128(row + 4u * dim);
          den[m] = fmaf(w, lds32f(row + 4u * p.D + 4u), den[m]);
          acc[m].x = fmaf(w, __uint_as_float(q.x), acc[m].x); acc[m].y = fmaf(w, __uint_as_float(q.y), acc[m].y);
          acc[m].z = fmaf(w, __uint_as_float(q.z), acc[m].z); acc[m].w = fmaf(w, __uint_as_float(q.w), acc[m].w);
        }
      }
    }
    if (r0 + batch < R) __syncthreads();  // the rows are consumed before the next batch lands on them
  }
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    float y[5] = {acc[m].x, acc[m].y, acc[m].z, acc[m].w, den[m]};
#pragma unroll
    for (int u = 0; u < 5; ++u) y[u] += __shfl_xor_sync(kFull, y[u], 8);
#pragma unroll
    for (int u = 0; u < 5; ++u) y[u] += __shfl_xor_sync(kFull, y[u], 16);
    const float f = y[4] == 0.f ? 0.f : (m == 0 ? 1.f : -lam) / y[4];  // a NaN sum stays one
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = fmaf(f, y[u], v[u]);
  }
  // what lies behind the row's values (m, l, padding) is not part of the norm
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] = dim + u < p.D ? v[u] * vs[u] : 0.f;
  float f = d.out_scale;
  if (d.norm_w != nullptr) {
    float sq = (v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3]);
    sq += __shfl_xor_sync(kFull, sq, 1);  // over the eight pieces
    sq += __shfl_xor_sync(kFull, sq, 2);
    sq += __shfl_xor_sync(kFull, sq, 4);
    if (lane == 0) sq_s[warp] = sq;
    __syncthreads();
    sq = 0.f;
    for (int u = 0; u < static_cast<int>(blockDim.x) / kWarp; ++u) sq += sq_s[u];
    f *= rsqrtf(sq / static_cast<float>(p.D) + d.norm_eps);
  }
  if (sub != 0 || dim >= p.D) return;
#pragma unroll
  for (int u = 0; u < 4; ++u) v[u] *= f * nw[u];
  const int64_t ob = b * p.o_st[0] + h * p.o_st[1], at = ob + dim;
  if (p.out_dtype != INT8KV_FP32 && p.o_st[2] == 1 && dim + 3 < p.D &&
      ((reinterpret_cast<uintptr_t>(p.out) + 2 * at) & 7u) == 0) {
    uint2 word;
    word.x = p.out_dtype == INT8KV_BF16 ? pack_bf162(v[0], v[1]) : pack_half2(v[0], v[1]);
    word.y = p.out_dtype == INT8KV_BF16 ? pack_bf162(v[2], v[3]) : pack_half2(v[2], v[3]);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) = word;
    return;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (dim + u < p.D) store_from_float(p.out, p.out_dtype, ob + (dim + u) * p.o_st[2], v[u]);
}

// ---------------------------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------------------------
int launch_diff_generic(const DiffParams& d, cudaStream_t stream) {
  if (d.Dk > kDiffMaxD) return INT8KV_E_UNSUPPORTED;
  const int64_t items = static_cast<int64_t>(d.a.B) * d.a.num_splits * d.heads;
  if (items >= (int64_t(1) << 31)) return INT8KV_E_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>((items + 3) / 4);
  auto by_slots = [&](auto kind) {
    constexpr int K = decltype(kind)::value;
    if (d.Dk <= 64) return launch_pdl(diff_generic_kernel<K, 2>, grid, 128, 0, stream, d);
    if (d.Dk <= 128) return launch_pdl(diff_generic_kernel<K, 4>, grid, 128, 0, stream, d);
    return launch_pdl(diff_generic_kernel<K, 8>, grid, 128, 0, stream, d);
  };
  if (d.a.cache_kind == kCacheInt8) return by_slots(std::integral_constant<int, kCacheInt8>{});
  if (d.a.cache_kind == kCacheBf16) return by_slots(std::integral_constant<int, kCacheBf16>{});
  return by_slots(std::integral_constant<int, kCacheFp16>{});
}

// The dynamic shared-memory limit is raised once per (kernel, device); later calls, which may sit inside a stream capture,
// launch without touching function attributes.
template <auto KERNEL>
static bool raise_smem(size_t bytes) {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const bool track = dev >= 0 && dev < 64;
  if (track && done[dev].load(std::memory_order_acquire)) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != cudaSuccess)
    return false;
  if (track) done[dev].store(true, std::memory_order_release);
  return true;
}

template <auto KERNEL, typename Shape>
static int launch_diff_shape(const DiffParams& d, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t stream) {
  if (!raise_smem<KERNEL>(Shape::kSmem)) return INT8KV_E_LAUNCH;
  const AttnParams& p = d.a;
  const int64_t items = static_cast<int64_t>(p.B) * p.num_splits * p.Hkv;
  if (items >= (int64_t(1) << 31)) return INT8KV_E_UNSUPPORTED;  // the kernels number their items in 32 bits
  return launch_pdl(KERNEL, static_cast<unsigned>(items), kWarp, Shape::kSmem, stream, tmK, tmV, d);
}

template <int DK, int NB>
static int launch_diff_tiled_shape(const DiffParams& d, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t stream) {
  if (d.a.cache_kind == kCacheInt8)
    return launch_diff_shape<diff_int8_kernel<DK, NB>, DiffInt8Shape<DK, NB>>(d, tmK, tmV, stream);
  if (d.a.cache_kind == kCacheBf16)
    return launch_diff_shape<diff_f16_kernel<DK, NB, true>, DiffF16Shape<DK>>(d, tmK, tmV, stream);
  return launch_diff_shape<diff_f16_kernel<DK, NB, false>, DiffF16Shape<DK>>(d, tmK, tmV, stream);
}

int diff_items_per_sm(int cache_kind, int D, int group) {
  if (cache_kind != kCacheInt8) return D == 128 ? DiffF16Shape<128>::kPerSm : DiffF16Shape<64>::kPerSm;
  if (D == 128) return group <= 4 ? DiffInt8Shape<128, 1>::kPerSm : DiffInt8Shape<128, 2>::kPerSm;
  return group <= 4 ? DiffInt8Shape<64, 1>::kPerSm : DiffInt8Shape<64, 2>::kPerSm;
}

int launch_diff_tiled(const DiffParams& d, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t stream) {
  if (d.Dk == 128)
    return d.group <= 4 ? launch_diff_tiled_shape<128, 1>(d, tmK, tmV, stream)
                        : launch_diff_tiled_shape<128, 2>(d, tmK, tmV, stream);
  return d.group <= 4 ? launch_diff_tiled_shape<64, 1>(d, tmK, tmV, stream)
                      : launch_diff_tiled_shape<64, 2>(d, tmK, tmV, stream);
}

int launch_diff_merge(const DiffParams& d, cudaStream_t stream) {
  const AttnParams& p = d.a;
  const int batch = std::min(kMergeBatch, p.num_splits);
  if (!raise_smem<diff_merge_kernel>(kMergeBatch * 8 * (2 * kDiffMaxD + 4))) return INT8KV_E_LAUNCH;
  const unsigned warps = static_cast<unsigned>((p.D + 31) / 32);  // at most 16
  return launch_pdl(diff_merge_kernel, dim3(static_cast<unsigned>(p.B), static_cast<unsigned>(d.heads), 1), warps * kWarp,
                    static_cast<size_t>(batch) * 8 * p.row_floats, stream, d, batch);
}

}  // namespace int8kv
