// Router of the expert layer: the k largest logits of every token, their
// gates, and the plan that groups the (token, choice) pairs by expert.
//
//   experts[t][j] = argmax of the row without the j chosen before (lowest index
//                   among equals; -inf and NaN are masked: never chosen)
//   gates[t][j]   = exp(l_j - m) / sum exp(l - m)   m = the row's maximum; the
//                   sum runs over the chosen experts or over the whole row
//   slot(t, j)    = offsets[e] + #{(t', j') of expert e with t' < t}
//
// A token holds its E logits as 8 consecutive ones in each of L lanes (L = the
// power of two with 8 L >= E), so a row of 64 bf16 logits is one 16-B load a
// lane, and every maximum is a short lane reduction.  A token chooses an expert
// at most once, so the choices of 256 consecutive tokens are one 256-bit mask
// an expert in LDS (set by OR: order-free), and the rank of a choice inside its
// expert is a population count of the bits below its token: no sort, no ordered
// atomics, the same plan every time.
//
// Block b owns `tiles` consecutive 256-token tiles (at most 256 blocks, so the
// count table stays small); with one block it finishes alone, else a second
// launch adds what the blocks before counted.
//
// 65536 tokens, 64 experts, k = 4, bf16: 13.8 us (12.6 MB: 2.7 us at the rate of a
// copy): 9.1 in the first kernel, half of them instructions of the selection, 4.7 in
// the second, two waits for memory and a launch.  4 tokens: 4 us on the GPU; the
// host needs 6.8 to call.  The gradient of 32768 tokens, 128 experts, k = 8: 9.4 us
// (3.9 TB/s).
#include "common.h"
#include "../dsml.h"
#include "../experts.h"

namespace dsml {
namespace {

constexpr int kRtThreads = 1024;
constexpr int kRtTile = 256;    // tokens of one mask pass
constexpr int kRtBlocks = 256;  // blocks at most

template <int DT>
__device__ __forceinline__ float rt_load(const void* p, int64_t i) {
  if constexpr (DT == kF32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == kBF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  else return __half2float(static_cast<const __half*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ uint16_t rt_h16(float v) {
  if constexpr (DT == kBF16) return f32_to_bf16(v);
  else return __half_as_ushort(__float2half(v));
}

// The 8 logits of this lane; columns >= E and NaN read as masked (-inf).
template <int DT>
__device__ __forceinline__ void rt_row(const void* logits, int64_t row, int E, int c0, bool vec, float (&v)[8]) {
  if (vec) {  // E % 8 == 0 and 16-B rows: a lane's 8 columns are whole or absent
    if (c0 < E) {
      if constexpr (DT == kF32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(logits) + row + c0);
        const float4 x = p[0], y = p[1];
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(logits) + row + c0);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t h = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
          if constexpr (DT == kBF16) v[i] = bf16_to_f32(h);
          else v[i] = __half2float(__ushort_as_half(h));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = -INFINITY;
    }
  } else {  // no load under a condition: a column past the end is read as the last
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = rt_load<DT>(logits, row + (c0 + i < E ? c0 + i : E - 1));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < E ? v[i] : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = v[i] == v[i] ? v[i] : -INFINITY;
}

// Reductions over a token's L lanes (every lane gets the result): by DPP within a row
// of 16, then across the two rows of each half (FAR: the two halves) of a wave.
template <bool FAR, class T, class Op>
__device__ __forceinline__ T rt_rows(T x, Op op) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if constexpr (FAR) {
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return op(__builtin_bit_cast(T, (uint32_t)s[0]), __builtin_bit_cast(T, (uint32_t)s[1]));
  } else {
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return op(__builtin_bit_cast(T, (uint32_t)s[0]), __builtin_bit_cast(T, (uint32_t)s[1]));
  }
}
template <int L>
__device__ __forceinline__ float rt_max(float x) {
  if constexpr (L >= 2) x = fmaxf(x, dpp_f<kDppQuadXor1>(x));
  if constexpr (L >= 4) x = fmaxf(x, dpp_f<kDppQuadXor2>(x));
  if constexpr (L >= 8) x = fmaxf(x, dpp_f<kDppRowHalfMirror>(x));
  if constexpr (L >= 16) x = fmaxf(x, dpp_f<kDppRowMirror>(x));
  if constexpr (L >= 32) x = rt_rows<false>(x, [](float p, float q) { return fmaxf(p, q); });
  if constexpr (L >= 64) x = rt_rows<true>(x, [](float p, float q) { return fmaxf(p, q); });
  return x;
}
template <int L>
__device__ __forceinline__ float rt_sum(float x) {
  if constexpr (L >= 2) x += dpp_f<kDppQuadXor1>(x);
  if constexpr (L >= 4) x += dpp_f<kDppQuadXor2>(x);
  if constexpr (L >= 8) x += dpp_f<kDppRowHalfMirror>(x);
  if constexpr (L >= 16) x += dpp_f<kDppRowMirror>(x);
  if constexpr (L >= 32) x = rt_rows<false>(x, [](float p, float q) { return p + q; });
  if constexpr (L >= 64) x = rt_rows<true>(x, [](float p, float q) { return p + q; });
  return x;
}
template <int L>
__device__ __forceinline__ uint32_t rt_max_u(uint32_t x) {
  if constexpr (L >= 2) x = max(x, (uint32_t)dpp_i<kDppQuadXor1>((int)x));
  if constexpr (L >= 4) x = max(x, (uint32_t)dpp_i<kDppQuadXor2>((int)x));
  if constexpr (L >= 8) x = max(x, (uint32_t)dpp_i<kDppRowHalfMirror>((int)x));
  if constexpr (L >= 16) x = max(x, (uint32_t)dpp_i<kDppRowMirror>((int)x));
  if constexpr (L >= 32) x = rt_rows<false>(x, [](uint32_t p, uint32_t q) { return max(p, q); });
  if constexpr (L >= 64) x = rt_rows<true>(x, [](uint32_t p, uint32_t q) { return max(p, q); });
  return x;
}
template <int L>
__device__ __forceinline__ int rt_min(int x) {
  if constexpr (L >= 2) x = min(x, dpp_i<kDppQuadXor1>(x));
  if constexpr (L >= 4) x = min(x, dpp_i<kDppQuadXor2>(x));
  if constexpr (L >= 8) x = min(x, dpp_i<kDppRowHalfMirror>(x));
  if constexpr (L >= 16) x = min(x, dpp_i<kDppRowMirror>(x));
  if constexpr (L >= 32) x = rt_rows<false>(x, [](int p, int q) { return min(p, q); });
  if constexpr (L >= 64) x = rt_rows<true>(x, [](int p, int q) { return min(p, q); });
  return x;
}

// A lane's logits that were not chosen yet.  take() finds the token's largest
// (m; -inf: none left) and its lowest column, and removes it.
//
// 16-bit types leave at least 13 low bits of their fp32 form zero: value (its bits
// in an order that unsigned comparison keeps) and column go into one word, and one
// maximum finds both.
template <int DT, int L>
struct RtRow {
  uint32_t key[8];  // 0: masked
  __device__ __forceinline__ RtRow(const float (&v)[8], int c0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(v[i] + 0.f);  // -0 is 0
      const uint32_t o = u ^ (uint32_t)(((int)u >> 31) | (int)0x80000000);
      key[i] = v[i] > -INFINITY ? (o & ~0x1fffu) | (uint32_t)(0x1fff - (c0 + i)) : 0u;
    }
  }
  __device__ __forceinline__ void take(int, float& m, int& at) {
    uint32_t k = key[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) k = max(k, key[i]);
    k = rt_max_u<L>(k);
#pragma unroll
    for (int i = 0; i < 8; ++i) key[i] = key[i] == k ? 0u : key[i];
    at = 0x1fff - (int)(k & 0x1fffu);
    const uint32_t u = k >> 31 ? (k & 0x7fffe000u) : ~(k | 0x1fffu);
    m = k ? __uint_as_float(u) : -INFINITY;
  }
};
template <int L>
struct RtRow<kF32, L> {
  float v[8];
  __device__ __forceinline__ RtRow(const float (&x)[8], int) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i];
  }
  __device__ __forceinline__ void take(int c0, float& m, int& at) {
    m = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, v[i]);
    m = rt_max<L>(m);
    at = 0x7fffffff;
#pragma unroll
    for (int i = 7; i >= 0; --i) at = v[i] == m ? c0 + i : at;
    at = rt_min<L>(at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i == at ? -INFINITY : v[i];
  }
};

// Slots of the experts' first choices: exclusive sums of cnt[E] into base[E + 1]
// (and offsets, by the block that writes them).  One wave.
__device__ __forceinline__ void rt_offsets(const int* cnt, int* base, int32_t* offsets, int E, bool write) {
  const int lane = threadIdx.x;
  int acc = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int e = e0 + lane, n = e < E ? cnt[e] : 0;
    int inc = n;
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x112, 0xf, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x114, 0xf, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x118, 0xf, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x143, 0xc, 0xf, false);
    if (e < E) {
      base[e] = acc + inc - n;
      if (write) offsets[e] = acc + inc - n;
    }
    acc += __builtin_amdgcn_readlane(inc, 63);
  }
  if (lane == 0) {
    base[E] = acc;
    if (write) offsets[E] = acc;
  }
}

// Choices of expert e by the tile's tokens before tl (all of them: tl = 256).
__device__ __forceinline__ int rt_rank(const uint32_t* mask, int e, int tl) {
  const uint4* m = reinterpret_cast<const uint4*>(mask + 8 * e);
  const uint4 x = m[0], y = m[1];
  const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  int r = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int left = tl - 32 * i;
    r += __popc(left >= 32 ? w[i] : (left > 0 ? w[i] & ((1u << left) - 1u) : 0u));
  }
  return r;
}

// LDS: mask[E][8] words (one bit a token of the tile), run[E] (this block's
// choices before the tile), base[E + 1], pick[256 k] (the tile's choices).
template <int DT, int L>
__global__ __launch_bounds__(kRtThreads) void route_topk_k(RouteArgs a, int tiles, int vec) {
  extern __shared__ __attribute__((aligned(16))) uint32_t rt_lds[];
  uint32_t* mask = rt_lds;
  int* run = reinterpret_cast<int*>(rt_lds + 8 * a.E);
  int* base = run + a.E;
  int* pick = base + a.E + 1;
  const int tid = threadIdx.x;
  constexpr int kPer = kRtThreads / L;                                  // tokens of one pass of the block
  constexpr int kPasses = kRtTile > kPer ? kRtTile / kPer : 1;
  constexpr int kAhead = kPasses < 4 ? kPasses : 4;                     // rows a lane loads before the first is used
  const int sub = tid % L, c0 = 8 * sub;
  for (int e = tid; e < a.E; e += kRtThreads) run[e] = 0;
  const int64_t t_first = (int64_t)blockIdx.x * tiles * kRtTile;
  const bool only = gridDim.x == 1;
  for (int tile = 0; tile < tiles; ++tile) {
    const int64_t t0 = t_first + (int64_t)tile * kRtTile;
    if (t0 >= a.T) break;
    const int nt = (int)(a.T - t0 < kRtTile ? a.T - t0 : kRtTile);
    for (int p0 = 0; p0 < kPasses; p0 += kAhead) {
      float v[kAhead][8];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {  // a token past the end: the last one's row, not used
        const int tl = (p0 + q) * kPer + tid / L;
        rt_row<DT>(a.logits, (t0 + (tl < nt ? tl : nt - 1)) * a.ldl, a.E, c0, vec, v[q]);
      }
      if (p0 == 0) {
        for (int i = tid; i < 8 * a.E; i += kRtThreads) mask[i] = 0u;
        __syncthreads();
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int tl = (p0 + q) * kPer + tid / L;
        if (tl >= nt) continue;  // whole L-lane groups leave together
        const int64_t t = t0 + tl;
        // lane j % L keeps choice j: one exponential, one division, one store each
        constexpr int KM = (kRouteMaxK + L - 1) / L;
        float mine[KM], num[KM], top = -INFINITY, sum = 0.f;
        int pk[KM];
#pragma unroll
        for (int i = 0; i < KM; ++i) {
          mine[i] = 0.f;
          pk[i] = -1;
        }
        RtRow<DT, L> left(v[q], c0);
#pragma unroll
        for (int j = 0; j < kRouteMaxK; ++j) {
          if (j >= a.k) break;
          float m;
          int at;
          left.take(c0, m, at);
          if (j == 0) top = m;
          if (sub == j % L) {
            mine[j / L] = m;
            pk[j / L] = m > -INFINITY ? at : -1;
          }
        }
#pragma unroll
        for (int i = 0; i < KM; ++i) {
          if (L * i >= a.k) break;
          num[i] = pk[i] >= 0 ? expf(mine[i] - top) : 0.f;
          sum += num[i];
        }
        if (a.all) {
          sum = 0.f;
          if (top > -INFINITY) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += expf(v[q][i] - top);
          }
        }
        sum = rt_sum<L>(sum);
#pragma unroll
        for (int i = 0; i < KM; ++i) {
          if (L * i >= a.k) break;
          const int j = sub + L * i;
          if (j < a.k) {
            a.experts[t * a.k + j] = pk[i];
            a.gates[t * a.k + j] = pk[i] >= 0 ? num[i] / sum : 0.f;
            pick[tl * a.k + j] = pk[i];
            if (pk[i] >= 0) atomicOr(&mask[pk[i] * 8 + (tl >> 5)], 1u << (tl & 31));
          }
        }
      }
    }
    __syncthreads();
    if (only) {  // one block, one tile: its counts are the plan
      for (int e = tid; e < a.E; e += kRtThreads) run[e] = rt_rank(mask, e, kRtTile);
      __syncthreads();
      if (tid < 64) rt_offsets(run, base, a.offsets, a.E, true);
      __syncthreads();
      const int total = base[a.E];
      for (int i = tid; i < nt * a.k; i += kRtThreads) {
        const int e = pick[i], tl = i / a.k;
        const int s = e >= 0 ? base[e] + rt_rank(mask, e, tl) : -1;
        a.slots[i] = s;
        if (s >= 0) a.rows[s] = tl;
        if (i >= total) a.rows[i] = -1;
      }
      return;
    }
    // rank of every choice in its expert, among this block's choices so far
    for (int i = tid; i < nt * a.k; i += kRtThreads) {
      const int e = pick[i];
      a.slots[t0 * a.k + i] = e >= 0 ? run[e] + rt_rank(mask, e, i / a.k) : -1;
    }
    __syncthreads();
    for (int e = tid; e < a.E; e += kRtThreads) run[e] += rt_rank(mask, e, kRtTile);
    __syncthreads();
  }
  if (!only) {
    for (int e = tid; e < a.E; e += kRtThreads) a.counts[(int64_t)blockIdx.x * a.E + e] = run[e];
  } else if (a.T == 0) {
    for (int e = tid; e <= a.E; e += kRtThreads) a.offsets[e] = 0;
  }
}

// Second launch: block b adds the choices of the blocks before it and of the
// experts before each, from the whole count table (it is a few KB to 512 KB).
__global__ __launch_bounds__(kRtThreads) void route_place_k(RouteArgs a, int tiles, int blocks) {
  extern __shared__ __attribute__((aligned(16))) uint32_t rt_lds[];
  int* before = reinterpret_cast<int*>(rt_lds);  // choices of the blocks before, per expert
  int* total = before + a.E;                     // all choices, per expert
  int* base = total + a.E;                       // [E + 1]
  const int tid = threadIdx.x;
  const int64_t i0 = (int64_t)blockIdx.x * tiles * kRtTile * a.k;
  int64_t i1 = i0 + (int64_t)tiles * kRtTile * a.k;
  if (i1 > a.T * a.k) i1 = a.T * a.k;
  const int64_t first = i0 + tid < i1 ? i0 + tid : i1 - 1;
  int e = a.experts[first], r = a.slots[first];  // in flight while the table is summed
  for (int x = tid; x < a.E; x += kRtThreads) before[x] = total[x] = 0;
  __syncthreads();
  // thread = (expert, slice of the blocks): coalesced over experts
  const int per = kRtThreads / a.E;
  for (int x = tid; x < a.E * per; x += kRtThreads) {
    const int ex = x % a.E, q = x / a.E;
    int sum = 0, bef = 0;
#pragma unroll 8
    for (int b = q; b < blocks; b += per) {
      const int n = a.counts[(int64_t)b * a.E + ex];
      sum += n;
      bef += b < (int)blockIdx.x ? n : 0;
    }
    atomicAdd(&total[ex], sum);  // integers: any order gives the same sum
    atomicAdd(&before[ex], bef);
  }
  __syncthreads();
  if (tid < 64) rt_offsets(total, base, a.offsets, a.E, blockIdx.x == 0);
  __syncthreads();
  const int64_t all = base[a.E];
  for (int64_t i = i0 + tid; i < i1; i += kRtThreads) {
    if (i != first) {
      e = a.experts[i];
      r = a.slots[i];
    }
    if (e >= 0) {
      const int s = base[e] + before[e] + r;
      a.slots[i] = s;
      a.rows[s] = (int32_t)(i / a.k);
    }
    if (i >= all) a.rows[i] = -1;
  }
}

// dlogits: one token in L lanes, as above.
//   chosen-normalised: dl_j = g_j (dg_j - sum_i g_i dg_i) at the chosen experts, else 0
//   row-normalised:    dl_e = [chosen] g_e dg_e - p_e sum_i g_i dg_i,  p = softmax(row)
// K: at least k; every load of the token is requested before the first is used.
template <int DT, int L, int K>
__global__ __launch_bounds__(256) void route_bwd_k(RouteBwdArgs a, int vec, int ovec) {
  const int sub = threadIdx.x % L, c0 = 8 * sub;
  const int64_t t = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (t >= a.T) return;  // whole L-lane groups leave together
  int e[K];
  float g[K], u[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const int64_t at = t * a.k + (j < a.k ? j : 0);
    e[j] = a.experts[at];
    g[j] = a.gates[at];
    u[j] = a.dgates[at];
  }
  float v[8];
  if (a.all) rt_row<DT>(a.logits, t * a.ldl, a.E, c0, vec, v);
  float inner = 0.f;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (j >= a.k) e[j] = -1;
    if (e[j] >= 0) inner += g[j] * u[j];
  }
  float d[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] = 0.f;
  if (a.all) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, v[i]);
    m = rt_max<L>(m);
    if (m > -INFINITY) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = expf(v[i] - m);
        s += v[i];
      }
      s = rt_sum<L>(s);
      const float f = inner / s;
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = -v[i] * f;
    }
  }
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const float w = g[j] * (a.all ? u[j] : u[j] - inner);
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] += e[j] == c0 + i ? w : 0.f;
  }
  if (c0 >= a.E) return;
  const int64_t o = t * a.E + c0;
  if constexpr (DT == kF32) {
    float* p = static_cast<float*>(a.dlogits) + o;
    if (ovec) {
      reinterpret_cast<float4*>(p)[0] = make_float4(d[0], d[1], d[2], d[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(d[4], d[5], d[6], d[7]);
    } else {
      for (int i = 0; i < 8 && c0 + i < a.E; ++i) p[i] = d[i];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(a.dlogits) + o;
    if (ovec) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = rt_h16<DT>(d[2 * i]) | ((uint32_t)rt_h16<DT>(d[2 * i + 1]) << 16);
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int i = 0; i < 8 && c0 + i < a.E; ++i) p[i] = rt_h16<DT>(d[i]);
    }
  }
}

int rt_tiles(int64_t T) {  // 256-token tiles of one block
  const int64_t n = (T + kRtTile - 1) / kRtTile;
  return (int)((n + kRtBlocks - 1) / kRtBlocks);
}
int rt_blocks(int64_t T) {
  const int64_t per = (int64_t)rt_tiles(T) * kRtTile;
  return (int)((T + per - 1) / per);
}
int rt_lanes(int E) {
  int L = 1;
  while (8 * L < E) L *= 2;
  return L;
}
size_t esize(int dt) { return dt == kF32 ? 4 : 2; }

template <int DT>
hipError_t launch_topk(const RouteArgs& a, int L, int blocks, int tiles, int vec, hipStream_t s) {
  const size_t lds = (size_t)(8 * a.E + a.E + a.E + 1 + kRtTile * a.k) * 4;
#define DSML_RT(LL) \
  case LL: hipLaunchKernelGGL((route_topk_k<DT, LL>), dim3(blocks), dim3(kRtThreads), lds, s, a, tiles, vec); break
  switch (L) {
    DSML_RT(1); DSML_RT(2); DSML_RT(4); DSML_RT(8); DSML_RT(16); DSML_RT(32); DSML_RT(64);
    default: return hipErrorInvalidValue;
  }
#undef DSML_RT
  return hipGetLastError();
}
template <int DT, int K>
hipError_t launch_bwd(const RouteBwdArgs& a, int L, int vec, int ovec, hipStream_t s) {
  const int64_t per = 256 / L, blocks = (a.T + per - 1) / per;
  if (blocks * 256 > kMaxThreads) return hipErrorInvalidValue;
#define DSML_RT(LL) \
  case LL: hipLaunchKernelGGL((route_bwd_k<DT, LL, K>), dim3((uint32_t)blocks), dim3(256), 0, s, a, vec, ovec); break
  switch (L) {
    DSML_RT(1); DSML_RT(2); DSML_RT(4); DSML_RT(8); DSML_RT(16); DSML_RT(32); DSML_RT(64);
    default: return hipErrorInvalidValue;
  }
#undef DSML_RT
  return hipGetLastError();
}

template <int DT>
hipError_t launch_bwd_k(const RouteBwdArgs& a, int L, int vec, int ovec, hipStream_t s) {
  if (a.k <= 2) return launch_bwd<DT, 2>(a, L, vec, ovec, s);
  if (a.k <= 8) return launch_bwd<DT, 8>(a, L, vec, ovec, s);
  return launch_bwd<DT, kRouteMaxK>(a, L, vec, ovec, s);
}

bool route_ok(int64_t T, int E, int k) {
  return T >= 0 && E >= 1 && E <= kRouteMaxExperts && k >= 1 && k <= kRouteMaxK && k <= E && T <= 0x7fffffffLL / k;
}

}  // namespace

int64_t route_ws_words(int64_t T, int E) { return T > 0 ? (int64_t)rt_blocks(T) * E : 0; }

hipError_t route_topk(const RouteArgs& a, hipStream_t s) {
  if (!route_ok(a.T, a.E, a.k)) return hipErrorInvalidValue;
  const int blocks = a.T > 0 ? rt_blocks(a.T) : 1, tiles = a.T > 0 ? rt_tiles(a.T) : 0;
  const size_t es = esize(a.dtype);
  const int vec = a.E % 8 == 0 && (a.ldl * es) % 16 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
  const int L = rt_lanes(a.E);
  hipError_t e;
  switch (a.dtype) {
    case kF32: e = launch_topk<kF32>(a, L, blocks, tiles, vec, s); break;
    case kBF16: e = launch_topk<kBF16>(a, L, blocks, tiles, vec, s); break;
    case kF16: e = launch_topk<kF16>(a, L, blocks, tiles, vec, s); break;
    default: return hipErrorInvalidValue;
  }
  if (e != hipSuccess || blocks == 1) return e;
  hipLaunchKernelGGL(route_place_k, dim3(blocks), dim3(kRtThreads), (size_t)(3 * a.E + 1) * 4, s, a, tiles, blocks);
  return hipGetLastError();
}

hipError_t route_topk_backward(const RouteBwdArgs& a, hipStream_t s) {
  if (!route_ok(a.T, a.E, a.k)) return hipErrorInvalidValue;
  if (a.T == 0) return hipSuccess;
  const size_t es = esize(a.dtype);
  const int vec = a.E % 8 == 0 && (a.ldl * es) % 16 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
  const int ovec = a.E % 8 == 0 && (reinterpret_cast<uintptr_t>(a.dlogits) & 15) == 0;
  const int L = rt_lanes(a.E);
  switch (a.dtype) {
    case kF32: return launch_bwd_k<kF32>(a, L, vec, ovec, s);
    case kBF16: return launch_bwd_k<kBF16>(a, L, vec, ovec, s);
    case kF16: return launch_bwd_k<kF16>(a, L, vec, ovec, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace dsml
