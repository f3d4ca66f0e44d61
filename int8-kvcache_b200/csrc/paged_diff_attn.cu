// Differential paged decode attention for sm_100a: for every query pair h and the KV pair g = h / group that serves it,
//   o = (softmax(q_{2h} K_{2g}^T / sqrt(D)) - lam_h * softmax(q_{2h+1} K_{2g+1}^T / sqrt(D))) [V_{2g} | V_{2g+1}],
// optionally followed by a root-mean-square norm over the 2 D values of o, a weight per value and a constant factor.
// The caches are the ordinary ones, [num_blocks, BS, 2 * pairs, D]: a pair's two K heads and its V row of 2 D values
// (heads 2g and 2g+1 side by side) are neighbours in every token.
//
// What it has to read is the pair's K and V rows once, 4 D values per token, for both maps and all query pairs of the
// group: HBM traffic bounds it, as it does ordinary decode attention.  Both maps therefore run in one pass over the
// pages, each with its own running maximum and sum, and both are kept unnormalised until the end, because the
// subtraction needs the two sums.  The parts of a split sequence leave one fp32 row [2 D values | log-sum-exp] per map
// in the workspace (row 2h + map of the part); diff_merge_kernel joins the parts, subtracts, norms and writes.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "paged_items.cuh"

namespace int8kv {

constexpr float kLn2 = 0.6931471805599453f;

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
  float ksc[2], vsc[2], mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    ksc[m] = (p.k_scale ? fmaxf(__ldg(p.k_scale + 2 * pair + m), 1e-6f) : 1.f) * p.sm_scale_log2;
    vsc[m] = p.v_scale ? fmaxf(__ldg(p.v_scale + 2 * pair + m), 1e-6f) : 1.f;
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
      const float al = mx[m] == -INFINITY ? 0.f : exp2f(mx[m] - mn);
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
    const float inv = l[m] == 0.f ? 0.f : 1.f / l[m];  // a NaN sum stays one
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const int dd = lane + kWarp * s;
        if (dd < D) out[half * D + dd] = acc[m][half][s] * inv * vsc[half];
      }
    if (lane == 0) out[p.D] = l[m] == 0.f ? -INFINITY : (mx[m] + log2f(l[m])) * kLn2;
  }
}

// ---------------------------------------------------------------------------------------------
// TMA-tiled kernels: D = 64 or 128, block size a multiple of 16, up to 8 query pairs per KV pair.
//
// One warp serves one (sequence, KV pair, split) with the ring of the ordinary tiled kernels; a stage holds a 16-token
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

// Running softmax of the columns of one block: maximum and sum of columns 2t (index 0) and 2t+1.
struct ColStats {
  float m[2], l[2];
};

// One online-softmax step on a 16-token tile's C fragment v (log2 units, rows g / g+8, columns 2t / 2t+1): v becomes the
// probabilities relative to the running maximum; returns whether the accumulators have to follow, by f[0], f[1].
__device__ __forceinline__ bool softmax_step(ColStats& s, float (&v)[4], float (&f)[2]) {
  float mx0 = fmaxf(v[0], v[2]), mx1 = fmaxf(v[1], v[3]);
  mx0 = fmaxf(mx0, __shfl_xor_sync(kFull, mx0, 4));
  mx1 = fmaxf(mx1, __shfl_xor_sync(kFull, mx1, 4));
  mx0 = fmaxf(mx0, __shfl_xor_sync(kFull, mx0, 8));
  mx1 = fmaxf(mx1, __shfl_xor_sync(kFull, mx1, 8));
  mx0 = fmaxf(mx0, __shfl_xor_sync(kFull, mx0, 16));
  mx1 = fmaxf(mx1, __shfl_xor_sync(kFull, mx1, 16));
  const float mn0 = fmaxf(s.m[0], mx0), mn1 = fmaxf(s.m[1], mx1);
  const bool moved = __any_sync(kFull, (mn0 != s.m[0]) || (mn1 != s.m[1]));
  if (moved) {
    f[0] = exp2_fast(s.m[0] - mn0);
    f[1] = exp2_fast(s.m[1] - mn1);
    s.l[0] *= f[0];
    s.l[1] *= f[1];
    s.m[0] = mn0;
    s.m[1] = mn1;
  }
  v[0] = exp2_fast(v[0] - s.m[0]);
  v[1] = exp2_fast(v[1] - s.m[1]);
  v[2] = exp2_fast(v[2] - s.m[0]);
  v[3] = exp2_fast(v[3] - s.m[1]);
  s.l[0] += v[0] + v[2];
  s.l[1] += v[1] + v[3];
  return moved;
}

// Row sums over the token lanes.
__device__ __forceinline__ void reduce_sums(ColStats& s) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    s.l[e] += __shfl_xor_sync(kFull, s.l[e], 4);
    s.l[e] += __shfl_xor_sync(kFull, s.l[e], 8);
    s.l[e] += __shfl_xor_sync(kFull, s.l[e], 16);
  }
}

__device__ __forceinline__ float inv_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }  // a NaN sum stays one
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

// Result of an empty tile range.
__device__ __forceinline__ void diff_write_empty(const DiffParams& d, const ItemCoord& it, int lane, float* prow) {
  const AttnParams& p = d.a;
  if (prow != nullptr) {
    if (lane < p.G) prow[lane * p.row_floats + p.D] = -INFINITY;
    return;
  }
  for (int hg = 0; hg < d.group; ++hg) {
    const int64_t base = it.b * p.o_st[0] + (it.h * d.group + hg) * p.o_st[1];
    for (int i = lane; i < p.D; i += kWarp) store_from_float(p.out, p.out_dtype, base + i * p.o_st[2], 0.f);
  }
}

// The work item of a warp: coordinates, tile range, first partial row (null: the result goes to `out`), and the ring
// ready to issue.  Returns false when the warp has nothing (more) to do.
template <bool PLANNED, typename Ring>
__device__ __forceinline__ bool diff_begin(const DiffParams& d, Ring& ring, ItemCoord& it, float*& prow, int64_t item,
                                           int heads_per_box, int lane) {
  const AttnParams& p = d.a;
  int64_t row0;
  if constexpr (PLANNED) {
    if (item >= p.plan_grid_items) return false;
  } else {
    if (!item_coords(p, item, it)) return false;
  }
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
  if constexpr (PLANNED) {
    PlanNote note;
    const bool live = plan_in_warp(p, item, lane, it, row0, note);
    plan_commit(p, note, lane);
    if (!live) return false;
  }
  ring.bt_row = reinterpret_cast<const char*>(p.bt) + it.b * p.bt_st[0] * (p.bt_is_i64 ? 8 : 4);
  ring.head = it.h * heads_per_box;
  if constexpr (PLANNED) {
    ring.prefetch_tables(it.t0 / p.tiles_per_block);
  } else {
    ring.prefetch_tables(guessed_first_block(p, it.c));
    item_range(p, it);
    row0 = arithmetic_row0(p, it);
  }
  prow = result_row(p, it, row0);
  if (it.t0 >= it.t1) {
    diff_write_empty(d, it, lane, prow);
    return false;
  }
  ring.set_range(it.t0, p.tiles_per_block);
  return true;
}

// A wait ran out at tile i of n: report it, and wait (again with a limit) for the loads that are still in flight.
template <int NST, typename Ring>
__device__ __forceinline__ void diff_timed_out(const AttnParams& p, const Ring& ring, int i, int n, int lane) {
  if (lane == 0 && p.status != nullptr) atomicOr(p.status, INT8KV_DEV_WAIT_TIMEOUT);
  const int issued = (i + NST < n) ? i + NST : n;
  for (int j = i; j < issued; ++j) ring.wait(j, 1u << 12);
}

// Eight dims x 16 tokens of V^T per step, INT8 -> fp16 on the way (see pv_tile), times P^T of NB column blocks.
template <int NB>
__device__ __forceinline__ void pv_blocks(float (&acc)[NB][8][4], const uint4 (&vx)[4], const uint32_t (&pb)[NB][2]) {
  const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&vx[0]);
  const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&vx[1]);
  const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&vx[2]);
  const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&vx[3]);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t x0 = w0[c] ^ 0x80808080u, x1 = w1[c] ^ 0x80808080u;
    const uint32_t x2 = w2[c] ^ 0x80808080u, x3 = w3[c] ^ 0x80808080u;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t a01 = prmt(x0, x1, s == 0 ? 0x5140u : 0x7362u), a23 = prmt(x2, x3, s == 0 ? 0x5140u : 0x7362u);
      const uint32_t f0 = u8pair_to_half2(a01, 0x4140u), f1 = u8pair_to_half2(a01, 0x4342u);
      const uint32_t f2 = u8pair_to_half2(a23, 0x4140u), f3 = u8pair_to_half2(a23, 0x4342u);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) mma_f16(acc[nb][2 * c + s], f0, f1, f2, f3, pb[nb][0], pb[nb][1]);
    }
  }
}

// Resident warps per SM and ring depth: 192 KB of ring per SM in every variant (the bytes in flight that keep HBM busy);
// a stage is 8 KB for D = 128 and 4 KB for D = 64.  The accumulators, 32 floats per lane and (column block, 128 values
// of V), set how many warps the register file carries.
template <int DK, int NB>
struct DiffInt8Shape {
  static constexpr int kHalves = DK / 64;
  static constexpr int kStage = kHalves * 4096;
  static constexpr int kWarpsPerSm = kHalves * NB == 1 ? 12 : 8;
  static constexpr int kStages = 192 * 1024 / (kWarpsPerSm * kStage);
};

template <int DK, int NB, bool PLANNED>
__global__ void __launch_bounds__(kDiffWarpsPerCta * kWarp, DiffInt8Shape<DK, NB>::kWarpsPerSm / kDiffWarpsPerCta)
diff_int8_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ DiffParams d) {
  using Shape = DiffInt8Shape<DK, NB>;
  constexpr int HV = Shape::kHalves, NST = Shape::kStages, STAGE = Shape::kStage;
  extern __shared__ uint8_t smem_raw[];
  const AttnParams& p = d.a;
  const int wpc = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  TileRing<NST, STAGE, 1> ring;
  ring.stage0 = smem_base + warp * (NST * STAGE);
  ring.bar0 = smem_base + wpc * NST * STAGE + warp * (NST * 8);
  ring.tmK = &tmK;
  ring.tmV = &tmV;
  ItemCoord it;
  float* prow;
  if (!diff_begin<PLANNED>(d, ring, it, prow, static_cast<int64_t>(blockIdx.x) * wpc + warp, HV, lane)) return;

  const float ks0 = __ldg(p.k_scale + 2 * it.h), ks1 = __ldg(p.k_scale + 2 * it.h + 1);
  const float vs0 = __ldg(p.v_scale + 2 * it.h), vs1 = __ldg(p.v_scale + 2 * it.h + 1);
  // The queries are requested first (a strided or unaligned one is staged through the idle ring), then the tiles; the
  // queries' arithmetic runs while the tiles are in flight.  Lane (g, t) holds column g's dims [32t, 32t+32) of the
  // 128-value tile row.
  float qv[NB][32];
  auto load_query = [&](int m, int hg, int dim, float (&x)[32]) {
    load32_as_float(p.q, p.q_dtype, it.b * p.q_st[0] + (2 * (it.h * d.group + hg) + m) * p.q_st[1] + dim * p.q_st[2],
                    p.q_st[2], x, ring.stage0, lane);
  };
  if constexpr (DK == 64 && NB == 2) {  // the lane's half of the row belongs to one map, that is to one block
    float x[32];
    const bool live = g < d.group;
    if (live) load_query(t >> 1, g, 32 * (t & 1), x);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      qv[0][i] = live && t < 2 ? x[i] : 0.f;
      qv[1][i] = live && t >= 2 ? x[i] : 0.f;
    }
  } else {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int m = col_map<NB>(nb, g), hg = col_pair<NB>(g);
      if (hg < d.group && (DK == 128 || (t >> 1) == m)) {
        load_query(m, hg, DK == 128 ? 32 * t : 32 * (t & 1), qv[nb]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) qv[nb][i] = 0.f;
      }
    }
  }
  fence_proxy_async_smem();  // a staged query was written by the lanes; the first tile is written by the TMA unit
  __syncwarp();
  const int n = it.t1 - it.t0;
  const int pre = n < NST ? n : NST;
  for (int i = 0; i < pre; ++i) ring.issue(i);

  // Queries as two INT8 limbs, q ~= q_mul * (256 hi + lo) with |256 hi + lo| <= 32000: 16-bit fixed point per head, so
  // that the K bytes go to the INT8 tensor cores as they lie in the cache.  A NaN or infinity in a head makes its
  // multiplier NaN, and with it the head's output.
  uint32_t qh[NB][8], ql[NB][8];
  float sc[NB][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    uint32_t abits = 0u;
#pragma unroll
    for (int i = 0; i < 32; ++i) abits = max(abits, __float_as_uint(qv[nb][i]) & 0x7fffffffu);
    abits = max(abits, __shfl_xor_sync(kFull, abits, 1));
    abits = max(abits, __shfl_xor_sync(kFull, abits, 2));
    const float amax = __uint_as_float(abits);
    const bool live_q = amax > 1e-20f;
    const float inv = live_q ? __fdividef(32000.f, amax) : 0.f;
    float q_mul = live_q ? __fdividef(1.f, inv) : 0.f;
    if (abits >= 0x7f800000u) q_mul = __uint_as_float(0x7fffffffu);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      uint32_t v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = static_cast<uint32_t>(__float_as_int(fmaf(qv[nb][4 * w + k], inv, kRoundMagic)) - kRoundMagicBits);
      ql[nb][w] = prmt(prmt(v[0], v[1], 0x0040u), prmt(v[2], v[3], 0x0040u), 0x5410u);
      qh[nb][w] = prmt(prmt(v[0] + 128u, v[1] + 128u, 0x0051u), prmt(v[2] + 128u, v[3] + 128u, 0x0051u), 0x5410u);
    }
    // score multipliers of columns 2t and 2t+1, which belong to the same map
    const float kmul = fmaxf(col_map<NB>(nb, 2 * t) ? ks1 : ks0, 1e-6f) * p.sm_scale_log2;
    sc[nb][0] = kmul * __shfl_sync(kFull, q_mul, (2 * t) * 4);
    sc[nb][1] = kmul * __shfl_sync(kFull, q_mul, (2 * t + 1) * 4);
  }

  const uint32_t koff[4] = {swz128(g, 2 * t), swz128(g, 2 * t + 1), swz128(g + 8, 2 * t), swz128(g + 8, 2 * t + 1)};
  const uint32_t voff[4] = {swz128(2 * t, g), swz128(2 * t + 1, g), swz128(2 * t + 8, g), swz128(2 * t + 9, g)};
  float acc[HV][NB][8][4];
  ColStats st[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    st[nb].m[0] = st[nb].m[1] = -INFINITY;
    st[nb].l[0] = st[nb].l[1] = 0.f;
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[h][nb][j][0] = acc[h][nb][j][1] = acc[h][nb][j][2] = acc[h][nb][j][3] = 0.f;
  }

  for (int i = 0; i < n; ++i) {
    if (!ring.wait(i)) {
      diff_timed_out<NST>(p, ring, i, n, lane);
      return;
    }
    const uint32_t kb = ring.stage(i), vb = kb + STAGE / 2;
    int raw[NB][4];
    if constexpr (DK == 128 && NB == 1) {  // both K tiles against all columns; each column keeps its own map's score
      int second[4];
      qk_tile(raw[0], kb, koff, qh[0], ql[0], true);
      qk_tile(second, kb + 2048, koff, qh[0], ql[0], true);
#pragma unroll
      for (int r = 0; r < 4; ++r) raw[0][r] = t < 2 ? raw[0][r] : second[r];
    } else {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) qk_tile(raw[nb], DK == 128 ? kb + nb * 2048 : kb, koff, qh[nb], ql[nb], true);
    }
    uint4 vx[HV][4];
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) vx[h][r] = lds128(vb + h * 2048 + voff[r]);

    const int tok0 = (it.t0 + i) * kTile + g;
    uint32_t pb[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float v[4], f[2];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = static_cast<float>(raw[nb][r]) * sc[nb][r & 1];
      if (tok0 >= it.seq_len) v[0] = v[1] = -INFINITY;
      if (tok0 + 8 >= it.seq_len) v[2] = v[3] = -INFINITY;
      if (softmax_step(st[nb], v, f)) {
#pragma unroll
        for (int h = 0; h < HV; ++h)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            acc[h][nb][j][0] *= f[0]; acc[h][nb][j][1] *= f[1]; acc[h][nb][j][2] *= f[0]; acc[h][nb][j][3] *= f[1];
          }
      }
      // P^T as B operands, rounded to fp16 (the sum keeps the unrounded values)
      pb[nb][0] = movmatrix_trans(pack_half2(v[0], v[1]));
      pb[nb][1] = movmatrix_trans(pack_half2(v[2], v[3]));
    }
#pragma unroll
    for (int h = 0; h < HV; ++h) pv_blocks<NB>(acc[h], vx[h], pb);

    __syncwarp();  // every lane has consumed the stage before lane 0 refills it
    if (i + NST < n) ring.issue(i + NST);
  }

  // ---- epilogue: lane (g, t) holds dims 128 h + 16 g .. + 15 of columns 2t and 2t+1 ----------------------
  const float v0 = fmaxf(vs0, 1e-6f), v1 = fmaxf(vs1, 1e-6f);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    reduce_sums(st[nb]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float inv = inv_sum(st[nb].l[e]);
#pragma unroll
      for (int h = 0; h < HV; ++h) {
        const float f = inv * (DK == 128 ? (h ? v1 : v0) : (g >= 4 ? v1 : v0));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          acc[h][nb][j][e] *= f;
          acc[h][nb][j][e + 2] *= f;
        }
      }
    }
  }
  if (prow != nullptr) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int hg = col_pair<NB>(2 * t + e), m = col_map<NB>(nb, 2 * t + e);
        if (hg >= d.group) continue;
        float* row = prow + (2 * hg + m) * p.row_floats;
#pragma unroll
        for (int h = 0; h < HV; ++h) {
          float4* dst = reinterpret_cast<float4*>(row + 128 * h + 16 * g);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            dst[k] = make_float4(acc[h][nb][2 * k][e], acc[h][nb][2 * k][e + 2], acc[h][nb][2 * k + 1][e], acc[h][nb][2 * k + 1][e + 2]);
        }
        if (g == 0) row[p.D] = lse_of(st[nb].m[e], st[nb].l[e]);
      }
    return;
  }
  // a sequence in one part: subtract, norm and write here.  The second map's column sits two lanes on (NB = 1) or in
  // the second block.
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int hg = col_pair<NB>(2 * t + e);
    const bool mine = hg < d.group && (NB == 2 || t < 2);
    const int head = it.h * d.group + (mine ? hg : 0);
    const float lam = load_as_float(d.lam, d.lam_dtype, head * d.lam_st);
    float o[HV][16], sq = 0.f;
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float a = acc[h][0][k >> 1][e + 2 * (k & 1)];
        const float b = NB == 2 ? acc[h][NB - 1][k >> 1][e + 2 * (k & 1)] : __shfl_xor_sync(kFull, a, 2);
        o[h][k] = a - lam * b;
        sq = fmaf(o[h][k], o[h][k], sq);
      }
    float f = d.out_scale;
    if (d.norm_w != nullptr) {
      sq += __shfl_xor_sync(kFull, sq, 4);
      sq += __shfl_xor_sync(kFull, sq, 8);
      sq += __shfl_xor_sync(kFull, sq, 16);
      f *= rsqrtf(sq / static_cast<float>(2 * DK) + d.norm_eps);
    }
    if (!mine) continue;
#pragma unroll
    for (int h = 0; h < HV; ++h) {
      const int dim = 128 * h + 16 * g;
#pragma unroll
      for (int k = 0; k < 16; ++k) o[h][k] *= f;
      if (d.norm_w != nullptr) {
#pragma unroll
        for (int k = 0; k < 16; ++k) o[h][k] *= load_as_float(d.norm_w, d.norm_dtype, dim + k);
      }
      store16_from_float(p.out, p.out_dtype, it.b * p.o_st[0] + head * p.o_st[1] + dim * p.o_st[2], p.o_st[2], o[h],
                         ring.stage0, lane);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// bf16 / fp16 caches: same ring and columns, fragments straight from shared memory with ldmatrix
// ---------------------------------------------------------------------------------------------
template <int DK>
struct DiffF16Shape {
  static constexpr int kStage = DK * 128;  // 2 tensors x 2 heads x 16 tokens x 2 DK bytes
  static constexpr int kWarpsPerSm = DK == 128 ? 4 : 8;
  static constexpr int kStages = 192 * 1024 / (kWarpsPerSm * kStage);
};

template <int DK, int NB, bool IS_BF16, bool PLANNED>
__global__ void __launch_bounds__(kDiffWarpsPerCta * kWarp, DiffF16Shape<DK>::kWarpsPerSm / kDiffWarpsPerCta)
diff_f16_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ DiffParams d) {
  using Shape = DiffF16Shape<DK>;
  constexpr int NST = Shape::kStages, STAGE = Shape::kStage;
  constexpr int STEPS = DK / 16;          // 16-dim steps of a score, 16-dim rows of a half of the output
  constexpr int PIECE = 4096;             // one load: 128 bytes x 16 tokens x 2 heads
  extern __shared__ uint8_t smem_raw[];
  const AttnParams& p = d.a;
  const int wpc = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  TileRing<NST, STAGE, DK / 64> ring;
  static_assert(TileRing<NST, STAGE, DK / 64>::PIECE == PIECE, "box of the tensor map");
  ring.stage0 = smem_base + warp * (NST * STAGE);
  ring.bar0 = smem_base + wpc * NST * STAGE + warp * (NST * 8);
  ring.tmK = &tmK;
  ring.tmV = &tmV;
  ItemCoord it;
  float* prow;
  if (!diff_begin<PLANNED>(d, ring, it, prow, static_cast<int64_t>(blockIdx.x) * wpc + warp, 2, lane)) return;
  const int n = it.t1 - it.t0;
  const int pre = n < NST ? n : NST;
  for (int i = 0; i < pre; ++i) ring.issue(i);

  // Queries as B fragments, rounded to the cache's type: step s covers dims 16s..16s+15; lane (g, t) holds column g,
  // dims 16s+2t, +1 and 16s+8+2t, +1
  uint32_t qf[NB][2 * STEPS];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int m = col_map<NB>(nb, g), hg = col_pair<NB>(g);
    const int64_t base = it.b * p.q_st[0] + (2 * (it.h * d.group + hg) + m) * p.q_st[1];
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

  float acc[2][NB][STEPS][4];
  ColStats st[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    st[nb].m[0] = st[nb].m[1] = -INFINITY;
    st[nb].l[0] = st[nb].l[1] = 0.f;
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
    if (!ring.wait(i)) {
      diff_timed_out<NST>(p, ring, i, n, lane);
      return;
    }
    const uint32_t kb = ring.stage(i), vb = kb + STAGE / 2;
    float sm[2][2][4];  // [map's K head][even / odd step]: two chains per head
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sm[m][0][r] = sm[m][1][r] = 0.f;
      const int nb = NB == 1 ? 0 : m;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int ch = 2 * s + k_chunk;  // 16-byte chunk of the row
        uint32_t a[4];
        ldmatrix_x4(a, kb + (ch >> 3) * PIECE + m * 2048 + swz128(k_tok, ch & 7));
        mma16<IS_BF16>(sm[m][s & 1], a, qf[nb][2 * s], qf[nb][2 * s + 1]);
      }
    }
    const int tile_tok = (it.t0 + i) * kTile;
    const int tok0 = tile_tok + g;
    uint32_t pb[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float v[4], f[2];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // NB = 1: both K heads met all columns, each column keeps its own map's score
        const float own = NB == 1 ? (t < 2 ? sm[0][0][r] + sm[0][1][r] : sm[1][0][r] + sm[1][1][r])
                                  : sm[nb][0][r] + sm[nb][1][r];
        v[r] = own * p.sm_scale_log2;
      }
      if (tok0 >= it.seq_len) v[0] = v[1] = -INFINITY;
      if (tok0 + 8 >= it.seq_len) v[2] = v[3] = -INFINITY;
      if (softmax_step(st[nb], v, f)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < STEPS; ++j) {
            acc[h][nb][j][0] *= f[0]; acc[h][nb][j][1] *= f[1]; acc[h][nb][j][2] *= f[0]; acc[h][nb][j][3] *= f[1];
          }
      }
      // P^T as B operands, rounded to the cache's type (the sum keeps the unrounded values)
      pb[nb][0] = movmatrix_trans(pack16<IS_BF16>(v[0], v[1]));
      pb[nb][1] = movmatrix_trans(pack16<IS_BF16>(v[2], v[3]));
    }
    // A float cache may hold NaN or infinities behind the last token, and 0 * NaN would poison the sums: those V values
    // are zeroed (their scores were replaced above).
    const int nvalid = it.seq_len - tile_tok;  // >= 1
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
    __syncwarp();
    if (i + NST < n) ring.issue(i + NST);
  }

  // ---- epilogue: dims DK h + 16 j + g (registers 0, 1) and + 8 (2, 3) of columns 2t and 2t+1 --------------------
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    reduce_sums(st[nb]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float inv = inv_sum(st[nb].l[e]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
          acc[h][nb][j][e] *= inv;
          acc[h][nb][j][e + 2] *= inv;
        }
    }
  }
  if (prow != nullptr) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int hg = col_pair<NB>(2 * t + e), m = col_map<NB>(nb, 2 * t + e);
        if (hg >= d.group) continue;
        float* row = prow + (2 * hg + m) * p.row_floats;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < STEPS; ++j) {
            row[DK * h + 16 * j + g] = acc[h][nb][j][e];
            row[DK * h + 16 * j + g + 8] = acc[h][nb][j][e + 2];
          }
        if (g == 0) row[p.D] = lse_of(st[nb].m[e], st[nb].l[e]);
      }
    return;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int hg = col_pair<NB>(2 * t + e);
    const bool mine = hg < d.group && (NB == 2 || t < 2);
    const int head = it.h * d.group + (mine ? hg : 0);
    const float lam = load_as_float(d.lam, d.lam_dtype, head * d.lam_st);
    float o[2][STEPS][2], sq = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < STEPS; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float a = acc[h][0][j][e + 2 * k];
          const float b = NB == 2 ? acc[h][NB - 1][j][e + 2 * k] : __shfl_xor_sync(kFull, a, 2);
          o[h][j][k] = a - lam * b;
          sq = fmaf(o[h][j][k], o[h][j][k], sq);
        }
    float f = d.out_scale;
    if (d.norm_w != nullptr) {
      sq += __shfl_xor_sync(kFull, sq, 4);
      sq += __shfl_xor_sync(kFull, sq, 8);
      sq += __shfl_xor_sync(kFull, sq, 16);
      f *= rsqrtf(sq / static_cast<float>(2 * DK) + d.norm_eps);
    }
    if (!mine) continue;
    const int64_t base = it.b * p.o_st[0] + head * p.o_st[1];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < STEPS; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int dim = DK * h + 16 * j + g + 8 * k;
          const float nw = d.norm_w != nullptr ? load_as_float(d.norm_w, d.norm_dtype, dim) : 1.f;
          store_from_float(p.out, p.out_dtype, base + dim * p.o_st[2], o[h][j][k] * f * nw);
        }
  }
}

// ---------------------------------------------------------------------------------------------
// Join of the parts, subtraction, norm: one CTA per (sequence, query pair).
// ---------------------------------------------------------------------------------------------
// Thread (group, col) sums 16-byte piece col of the parts group, group + groups, ... of both maps, already weighted
// with w / den and with -lam for the second map; the groups are added in a fixed order.  Empty parts (log-sum-exp
// -inf) were never written and are not read.
constexpr int kDiffMergeThreads = 128;
static_assert(kDiffMergeThreads >= kMaxSplits, "one thread per part");

__global__ void __launch_bounds__(kDiffMergeThreads) diff_merge_kernel(const DiffParams d) {
  __shared__ float w_s[2][kMaxSplits];
  __shared__ float4 red_s[kDiffMergeThreads];
  __shared__ float warp_s[4][2];
  const AttnParams& p = d.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = static_cast<int>(blockIdx.x / d.heads), h = static_cast<int>(blockIdx.x - static_cast<unsigned>(b) * d.heads);
  const float lam = load_as_float(d.lam, d.lam_dtype, h * d.lam_st);
  grid_dependency_wait();
  grid_launch_dependents();
  int R = p.num_splits;
  int64_t stride_r = static_cast<int64_t>(p.B) * p.Hq * p.row_floats;
  const float* base = p.part + (static_cast<int64_t>(b) * p.Hq + 2 * h) * p.row_floats;
  if (p.plan_table != nullptr) {  // device-planned parts: consecutive part numbers; a single one went to `out` itself
    const int2 e = __ldcg(p.plan_table + b);
    if (e.y <= 1) return;
    R = e.y < kMaxSplits ? e.y : kMaxSplits;
    stride_r = static_cast<int64_t>(p.Hq) * p.row_floats;
    base = p.part + (static_cast<int64_t>(e.x) * p.Hq + 2 * h) * p.row_floats;
  }

  float lse[2] = {-INFINITY, -INFINITY};
  if (tid < R) {
    lse[0] = __ldcg(base + tid * stride_r + p.D);
    lse[1] = __ldcg(base + tid * stride_r + p.row_floats + p.D);
  }
  // block maximum, then block sum, of both maps
  float top[2], den[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    float t = lse[m];
    for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(kFull, t, o));
    if (lane == 0) warp_s[warp][m] = t;
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 2; ++m) top[m] = fmaxf(fmaxf(warp_s[0][m], warp_s[1][m]), fmaxf(warp_s[2][m], warp_s[3][m]));
  __syncthreads();
  float w[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    w[m] = lse[m] == -INFINITY ? 0.f : __expf(lse[m] - top[m]);
    float t = w[m];
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(kFull, t, o);
    if (lane == 0) warp_s[warp][m] = t;
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    den[m] = (warp_s[0][m] + warp_s[1][m]) + (warp_s[2][m] + warp_s[3][m]);
    const float f = den[m] == 0.f ? 0.f : (m == 0 ? 1.f : -lam) / den[m];
    if (tid < R) w_s[m][tid] = lse[m] == -INFINITY ? 0.f : w[m] * f;
  }
  __syncthreads();

  const int cols = (p.D + 3) / 4;  // at most 128
  const int groups = kDiffMergeThreads / cols;
  const int group = tid / cols, col = tid - group * cols;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (group < groups) {
#pragma unroll 4
    for (int r = group; r < R; r += groups) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float wr = w_s[m][r];
        // a part that weighs nothing is not read; lam = 0 switches the second map off (a NaN weight is not zero)
        if (wr != 0.f) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(base + r * stride_r + m * p.row_floats) + col);
          a.x += wr * x.x; a.y += wr * x.y; a.z += wr * x.z; a.w += wr * x.w;
        }
      }
    }
  }
  red_s[tid] = a;
  __syncthreads();
  float sq = 0.f;
  if (group == 0) {
    for (int u = 1; u < groups; ++u) {
      const float4 x = red_s[u * cols + col];
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    }
    // the last piece of a row whose length is not a multiple of four ends in the log-sum-exp and padding
    if (4 * col + 1 >= p.D) a.y = 0.f;
    if (4 * col + 2 >= p.D) a.z = 0.f;
    if (4 * col + 3 >= p.D) a.w = 0.f;
    sq = (a.x * a.x + a.y * a.y) + (a.z * a.z + a.w * a.w);
  }
  float f = d.out_scale;
  if (d.norm_w != nullptr) {
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(kFull, sq, o);
    if (lane == 0) warp_s[warp][0] = sq;
    __syncthreads();
    sq = (warp_s[0][0] + warp_s[1][0]) + (warp_s[2][0] + warp_s[3][0]);
    f *= rsqrtf(sq / static_cast<float>(p.D) + d.norm_eps);
  }
  if (group != 0) return;
  const float v[4] = {a.x, a.y, a.z, a.w};
  const int64_t ob = b * p.o_st[0] + h * p.o_st[1];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int dd = 4 * col + u;
    if (dd >= p.D) break;
    const float nw = d.norm_w != nullptr ? load_as_float(d.norm_w, d.norm_dtype, dd) : 1.f;
    store_from_float(p.out, p.out_dtype, ob + dd * p.o_st[2], v[u] * f * nw);
  }
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
static int launch_diff_shape(const DiffParams& d, const CUtensorMap& tmK, const CUtensorMap& tmV, int sm_count, cudaStream_t stream) {
  constexpr int per_warp = Shape::kStages * (Shape::kStage + 8);
  if (!raise_smem<KERNEL>(kDiffWarpsPerCta * per_warp + 1024)) return INT8KV_E_LAUNCH;
  const AttnParams& p = d.a;
  const int64_t items = p.plan_table != nullptr ? p.plan_grid_items : static_cast<int64_t>(p.B) * p.num_splits * p.Hkv;
  if (items >= (int64_t(1) << 31)) return INT8KV_E_UNSUPPORTED;  // the kernels number their items in 32 bits
  // a grid that does not fill the machine with four-warp CTAs runs as one-warp CTAs, spread over all SMs
  const int wpc = items <= static_cast<int64_t>(sm_count) * Shape::kWarpsPerSm ? 1 : kDiffWarpsPerCta;
  return launch_pdl(KERNEL, static_cast<unsigned>((items + wpc - 1) / wpc), wpc * kWarp,
                    static_cast<size_t>(wpc) * per_warp + 1024, stream, tmK, tmV, d);
}

template <int DK, int NB>
static int launch_diff_tiled_shape(const DiffParams& d, const CUtensorMap& tmK, const CUtensorMap& tmV, int sm_count,
                                   cudaStream_t stream) {
  const bool planned = d.a.plan_table != nullptr;
  if (d.a.cache_kind == kCacheInt8)
    return planned ? launch_diff_shape<diff_int8_kernel<DK, NB, true>, DiffInt8Shape<DK, NB>>(d, tmK, tmV, sm_count, stream)
                   : launch_diff_shape<diff_int8_kernel<DK, NB, false>, DiffInt8Shape<DK, NB>>(d, tmK, tmV, sm_count, stream);
  if (d.a.cache_kind == kCacheBf16)
    return planned ? launch_diff_shape<diff_f16_kernel<DK, NB, true, true>, DiffF16Shape<DK>>(d, tmK, tmV, sm_count, stream)
                   : launch_diff_shape<diff_f16_kernel<DK, NB, true, false>, DiffF16Shape<DK>>(d, tmK, tmV, sm_count, stream);
  return planned ? launch_diff_shape<diff_f16_kernel<DK, NB, false, true>, DiffF16Shape<DK>>(d, tmK, tmV, sm_count, stream)
                 : launch_diff_shape<diff_f16_kernel<DK, NB, false, false>, DiffF16Shape<DK>>(d, tmK, tmV, sm_count, stream);
}

int diff_warps_per_sm(int cache_kind, int D, int group) {
  if (cache_kind != kCacheInt8) return D == 128 ? DiffF16Shape<128>::kWarpsPerSm : DiffF16Shape<64>::kWarpsPerSm;
  if (D == 128) return group <= 4 ? DiffInt8Shape<128, 1>::kWarpsPerSm : DiffInt8Shape<128, 2>::kWarpsPerSm;
  return group <= 4 ? DiffInt8Shape<64, 1>::kWarpsPerSm : DiffInt8Shape<64, 2>::kWarpsPerSm;
}

int launch_diff_tiled(const DiffParams& d, const CUtensorMap& tmK, const CUtensorMap& tmV, int sm_count, cudaStream_t stream) {
  if (d.Dk == 128)
    return d.group <= 4 ? launch_diff_tiled_shape<128, 1>(d, tmK, tmV, sm_count, stream)
                        : launch_diff_tiled_shape<128, 2>(d, tmK, tmV, sm_count, stream);
  return d.group <= 4 ? launch_diff_tiled_shape<64, 1>(d, tmK, tmV, sm_count, stream)
                      : launch_diff_tiled_shape<64, 2>(d, tmK, tmV, sm_count, stream);
}

int launch_diff_merge(const DiffParams& d, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(d.a.B) * d.heads;
  if (rows >= (int64_t(1) << 31)) return INT8KV_E_UNSUPPORTED;
  return launch_pdl(diff_merge_kernel, static_cast<unsigned>(rows), kDiffMergeThreads, 0, stream, d);
}

}  // namespace int8kv
