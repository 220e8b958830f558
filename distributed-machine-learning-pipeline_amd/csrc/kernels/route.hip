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
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < E ? rt_load<DT>(logits, row + c0 + i) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = v[i] == v[i] ? v[i] : -INFINITY;
}

// Reductions over a token's L lanes (every lane gets the result).
template <int L>
__device__ __forceinline__ float rt_max(float x) {
  if constexpr (L >= 2) x = fmaxf(x, dpp_f<kDppQuadXor1>(x));
  if constexpr (L >= 4) x = fmaxf(x, dpp_f<kDppQuadXor2>(x));
  if constexpr (L >= 8) x = fmaxf(x, dpp_f<kDppRowHalfMirror>(x));
  if constexpr (L >= 16) x = fmaxf(x, dpp_f<kDppRowMirror>(x));
  if constexpr (L >= 32) x = fmaxf(x, __shfl_xor(x, 16));
  if constexpr (L >= 64) x = fmaxf(x, __shfl_xor(x, 32));
  return x;
}
template <int L>
__device__ __forceinline__ float rt_sum(float x) {
  if constexpr (L >= 2) x += dpp_f<kDppQuadXor1>(x);
  if constexpr (L >= 4) x += dpp_f<kDppQuadXor2>(x);
  if constexpr (L >= 8) x += dpp_f<kDppRowHalfMirror>(x);
  if constexpr (L >= 16) x += dpp_f<kDppRowMirror>(x);
  if constexpr (L >= 32) x += __shfl_xor(x, 16);
  if constexpr (L >= 64) x += __shfl_xor(x, 32);
  return x;
}
template <int L>
__device__ __forceinline__ int rt_min(int x) {
  if constexpr (L >= 2) x = min(x, dpp_i<kDppQuadXor1>(x));
  if constexpr (L >= 4) x = min(x, dpp_i<kDppQuadXor2>(x));
  if constexpr (L >= 8) x = min(x, dpp_i<kDppRowHalfMirror>(x));
  if constexpr (L >= 16) x = min(x, dpp_i<kDppRowMirror>(x));
  if constexpr (L >= 32) x = min(x, __shfl_xor(x, 16));
  if constexpr (L >= 64) x = min(x, __shfl_xor(x, 32));
  return x;
}

// LDS: mask[E][8] words (one bit a token of the tile), run[E] (this block's
// choices before the tile), base[E] (slot of the block's first choice).
template <int DT, int L>
__global__ __launch_bounds__(kRtThreads) void route_topk_k(RouteArgs a, int tiles, int vec) {
  extern __shared__ uint32_t rt_lds[];
  uint32_t* mask = rt_lds;
  int* run = reinterpret_cast<int*>(rt_lds + 8 * a.E);
  int* base = run + a.E;
  const int tid = threadIdx.x;
  constexpr int kPer = kRtThreads / L;  // tokens of one pass of the block
  const int sub = tid % L, c0 = 8 * sub;
  for (int e = tid; e < a.E; e += kRtThreads) run[e] = 0;
  const int64_t t_first = (int64_t)blockIdx.x * tiles * kRtTile;
  for (int tile = 0; tile < tiles; ++tile) {
    const int64_t t0 = t_first + (int64_t)tile * kRtTile;
    if (t0 >= a.T) break;
    const int nt = (int)(a.T - t0 < kRtTile ? a.T - t0 : kRtTile);
    for (int i = tid; i < 8 * a.E; i += kRtThreads) mask[i] = 0u;
    __syncthreads();
    for (int p = 0; p < nt; p += kPer) {
      const int tl = p + tid / L;
      if (tl >= nt || tl >= kRtTile) continue;  // whole L-lane groups leave together
      const int64_t t = t0 + tl;
      float v[8];
      rt_row<DT>(a.logits, t * a.ldl, a.E, c0, vec, v);
      float m = v[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) m = fmaxf(m, v[i]);
      m = rt_max<L>(m);
      const float top = m;
      float all = 0.f;
      if (a.all && top > -INFINITY) {
#pragma unroll
        for (int i = 0; i < 8; ++i) all += expf(v[i] - top);
        all = rt_sum<L>(all);
      }
      float den = 0.f;
      float mine = 0.f;  // lane j of the token keeps choice j's numerator (k > L: in turns)
      (void)mine;
      float num[kRouteMaxK];
      int pick[kRouteMaxK];
#pragma unroll
      for (int j = 0; j < kRouteMaxK; ++j) {
        if (j >= a.k) break;
        if (j) {
          m = v[0];
#pragma unroll
          for (int i = 1; i < 8; ++i) m = fmaxf(m, v[i]);
          m = rt_max<L>(m);
        }
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 7; i >= 0; --i) at = v[i] == m ? c0 + i : at;
        at = rt_min<L>(at);
        const bool live = m > -INFINITY;
        pick[j] = live ? at : -1;
        num[j] = live ? expf(m - top) : 0.f;
        den += num[j];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c0 + i == at ? -INFINITY : v[i];
      }
      const float d = a.all ? all : den;
#pragma unroll
      for (int j = 0; j < kRouteMaxK; ++j) {
        if (j >= a.k) break;
        if (sub == j % L) {
          a.experts[t * a.k + j] = pick[j];
          a.gates[t * a.k + j] = pick[j] >= 0 ? num[j] / d : 0.f;
          if (pick[j] >= 0) atomicOr(&mask[pick[j] * 8 + (tl >> 5)], 1u << (tl & 31));
        }
      }
    }
    __syncthreads();
    // rank of every choice in its expert, among this block's choices so far
    for (int i = tid; i < nt * a.k; i += kRtThreads) {
      const int tl = i / a.k;
      const int e = a.experts[t0 * a.k + i];
      int r = -1;
      if (e >= 0) {
        r = run[e];
        const uint32_t* mk = mask + e * 8;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          const uint32_t bits = w < (tl >> 5) ? mk[w] : (w == (tl >> 5) ? mk[w] & ((1u << (tl & 31)) - 1u) : 0u);
          r += __popc(bits);
        }
      }
      a.slots[t0 * a.k + i] = r;
    }
    __syncthreads();
    for (int e = tid; e < a.E; e += kRtThreads) {
      int n = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) n += __popc(mask[e * 8 + w]);
      run[e] += n;
    }
    __syncthreads();
  }
  if (gridDim.x > 1) {
    for (int e = tid; e < a.E; e += kRtThreads) a.counts[(int64_t)blockIdx.x * a.E + e] = run[e];
    return;
  }
  // the only block: offsets, then slots and rows
  if (tid < 64) {
    int acc = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int e = e0 + tid;
      const int n = e < a.E ? run[e] : 0;
      int inc = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o);
        if (tid >= o) inc += u;
      }
      if (e < a.E) {
        base[e] = acc + inc - n;
        a.offsets[e] = acc + inc - n;
      }
      acc += __shfl(inc, 63);
    }
    if (tid == 0) {
      a.offsets[a.E] = acc;
      base[a.E] = acc;
    }
  }
  __syncthreads();
  const int total = base[a.E];
  const int n = (int)(a.T * a.k);
  for (int i = tid; i < n; i += kRtThreads) {
    const int e = a.experts[i];
    if (e >= 0) {
      const int s = base[e] + a.slots[i];
      a.slots[i] = s;
      a.rows[s] = i / a.k;
    }
    if (i >= total) a.rows[i] = -1;
  }
}

// Second launch: block b adds the choices of the blocks before it and of the
// experts before each, from the whole count table (it is a few KB to 128 KB).
__global__ __launch_bounds__(kRtThreads) void route_place_k(RouteArgs a, int tiles, int blocks) {
  extern __shared__ uint32_t rt_lds[];
  int* before = reinterpret_cast<int*>(rt_lds);  // choices of the blocks before, per expert
  int* total = before + a.E;                     // all choices, per expert
  int* base = total + a.E;                       // [E + 1]
  const int tid = threadIdx.x;
  for (int e = tid; e < a.E; e += kRtThreads) before[e] = total[e] = 0;
  __syncthreads();
  // thread = (expert, slice of the blocks): coalesced over experts
  const int per = kRtThreads / a.E > 0 ? kRtThreads / a.E : 1;
  for (int i = tid; i < a.E * per; i += kRtThreads) {
    const int e = i % a.E, q = i / a.E;
    int sum = 0, bef = 0;
    for (int b = q; b < blocks; b += per) {
      const int n = a.counts[(int64_t)b * a.E + e];
      sum += n;
      bef += b < (int)blockIdx.x ? n : 0;
    }
    atomicAdd(&total[e], sum);  // integers: any order gives the same sum
    atomicAdd(&before[e], bef);
  }
  __syncthreads();
  if (tid < 64) {
    int acc = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int e = e0 + tid;
      const int n = e < a.E ? total[e] : 0;
      int inc = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o);
        if (tid >= o) inc += u;
      }
      if (e < a.E) {
        base[e] = acc + inc - n + before[e];
        if (blockIdx.x == 0) a.offsets[e] = acc + inc - n;
      }
      acc += __shfl(inc, 63);
    }
    if (tid == 0) {
      base[a.E] = acc;
      if (blockIdx.x == 0) a.offsets[a.E] = acc;
    }
  }
  __syncthreads();
  const int64_t total_n = base[a.E];
  const int64_t i0 = (int64_t)blockIdx.x * tiles * kRtTile * a.k;
  int64_t i1 = i0 + (int64_t)tiles * kRtTile * a.k;
  if (i1 > a.T * a.k) i1 = a.T * a.k;
  for (int64_t i = i0 + tid; i < i1; i += kRtThreads) {
    const int e = a.experts[i];
    if (e >= 0) {
      const int s = base[e] + a.slots[i];
      a.slots[i] = s;
      a.rows[s] = (int32_t)(i / a.k);
    }
    if (i >= total_n) a.rows[i] = -1;
  }
}

// dlogits: one token in L lanes, as above.
//   chosen-normalised: dl_j = g_j (dg_j - sum_i g_i dg_i) at the chosen experts, else 0
//   row-normalised:    dl_e = [chosen] g_e dg_e - p_e sum_i g_i dg_i,  p = softmax(row)
template <int DT, int L>
__global__ __launch_bounds__(256) void route_bwd_k(RouteBwdArgs a, int vec, int ovec) {
  const int sub = threadIdx.x % L, c0 = 8 * sub;
  const int64_t t = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (t >= a.T) return;  // whole L-lane groups leave together
  float inner = 0.f;
  for (int j = 0; j < a.k; ++j)
    if (a.experts[t * a.k + j] >= 0) inner += a.gates[t * a.k + j] * a.dgates[t * a.k + j];
  float d[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] = 0.f;
  if (a.all) {
    float v[8];
    rt_row<DT>(a.logits, t * a.ldl, a.E, c0, vec, v);
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
  for (int j = 0; j < a.k; ++j) {
    const int e = a.experts[t * a.k + j];
    const float g = a.gates[t * a.k + j], dg = a.dgates[t * a.k + j];
    const float u = a.all ? g * dg : g * (dg - inner);
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] += e == c0 + i ? u : 0.f;
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
  const size_t lds = (size_t)(8 * a.E + a.E + a.E + 1) * 4;
#define DSML_RT(LL) \
  case LL: hipLaunchKernelGGL((route_topk_k<DT, LL>), dim3(blocks), dim3(kRtThreads), lds, s, a, tiles, vec); break
  switch (L) {
    DSML_RT(1); DSML_RT(2); DSML_RT(4); DSML_RT(8); DSML_RT(16); DSML_RT(32); DSML_RT(64);
    default: return hipErrorInvalidValue;
  }
#undef DSML_RT
  return hipGetLastError();
}
template <int DT>
hipError_t launch_bwd(const RouteBwdArgs& a, int L, int vec, int ovec, hipStream_t s) {
  const int64_t per = 256 / L, blocks = (a.T + per - 1) / per;
#define DSML_RT(LL) \
  case LL: hipLaunchKernelGGL((route_bwd_k<DT, LL>), dim3((uint32_t)blocks), dim3(256), 0, s, a, vec, ovec); break
  switch (L) {
    DSML_RT(1); DSML_RT(2); DSML_RT(4); DSML_RT(8); DSML_RT(16); DSML_RT(32); DSML_RT(64);
    default: return hipErrorInvalidValue;
  }
#undef DSML_RT
  return hipGetLastError();
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
    case kF32: return launch_bwd<kF32>(a, L, vec, ovec, s);
    case kBF16: return launch_bwd<kBF16>(a, L, vec, ovec, s);
    case kF16: return launch_bwd<kF16>(a, L, vec, ovec, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace dsml
