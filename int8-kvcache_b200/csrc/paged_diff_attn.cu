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
#include <cstring>
#include <type_traits>

#include "common.cuh"

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

int launch_diff_merge(const DiffParams& d, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(d.a.B) * d.heads;
  if (rows >= (int64_t(1) << 31)) return INT8KV_E_UNSUPPORTED;
  return launch_pdl(diff_merge_kernel, static_cast<unsigned>(rows), kDiffMergeThreads, 0, stream, d);
}

}  // namespace int8kv
