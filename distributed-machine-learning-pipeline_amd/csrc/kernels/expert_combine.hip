// Gated sum of a token's expert rows, and its gradient:
//
//   out[t]     = sum_j gate[t][j] y[slot[t][j]]          (gates null: 1)
//   dy[s]      = gate[t][j] dout[t]  for s = slot[t][j]
//   dgate[t][j] = sum_n dout[t][n] y[slot[t][j]][n]
//
// Sums in fp32, one rounding at the store.  Slot -1 (or any slot outside
// [0, S)) contributes nothing.  The kernels only move bytes: a row takes LPR
// lanes of 8 columns each (16-B accesses), several rows share a wave when rows
// are short, and all of a token's rows are requested before the first is used.
// 16384 tokens of 2 rows of 4096 columns: 70 us (5.75 TB/s); the gradient of 8191 of
// 4 rows of 1000: 29.6 us (5.0 TB/s).
#include "common.h"
#include "../dsml.h"
#include "../experts.h"

namespace dsml {
namespace {

constexpr int kCbThreads = 256;

template <int DT>
__device__ __forceinline__ float cb_f(uint16_t h) {
  if constexpr (DT == kBF16) return bf16_to_f32(h);
  else return __half2float(__ushort_as_half(h));
}
template <int DT>
__device__ __forceinline__ uint16_t cb_h(float v) {
  if constexpr (DT == kBF16) return f32_to_bf16(v);
  else return __half_as_ushort(__float2half(v));
}
// How a row's 8-column chunks move: whole 16-B words (kWords), words of any
// alignment, the last one moved back into the row (kMoved, N >= 8), or one by one
// (8191 tokens of 4 rows of 1001: 44 us, the gradient 80; moved 17 and 29).
enum CbForm { kSingle, kMoved, kWords };
// 8 columns from c on; columns >= N read 0.
template <CbForm F>
__device__ __forceinline__ uint4 cb_load(const uint16_t* p, int c, int N) {
  if constexpr (F == kWords) return *reinterpret_cast<const uint4*>(p + c);
  if constexpr (F == kMoved) {
    const int at = c < N - 8 ? c : N - 8;
    uint4 u;
    __builtin_memcpy(&u, p + at, 16);
    return drop_front8(u, c - at);
  }
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < N) w[i >> 1] |= (uint32_t)p[c + i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int DT, CbForm F>
__device__ __forceinline__ void cb_store(uint16_t* p, int c, int N, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = cb_h<DT>(v[2 * i]) | ((uint32_t)cb_h<DT>(v[2 * i + 1]) << 16);
  if constexpr (F == kWords) {
    *reinterpret_cast<uint4*>(p + c) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if (F == kMoved && c + 8 <= N) {
    __builtin_memcpy(p + c, w, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < N) p[c + i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  }
}
template <int DT>
__device__ __forceinline__ void cb_unpack(uint4 u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = cb_f<DT>((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
}

// K: choices held at once (k <= K: one round).  Workgroups next to each other
// take a row's column chunks in turn: whole rows are read and written together.
template <int DT, CbForm F, int LPR, int K>
__global__ __launch_bounds__(kCbThreads) void combine_k(CombineArgs a, int chunks) {
  const int sub = threadIdx.x % LPR, chunk = blockIdx.x % chunks;
  const int64_t t = (int64_t)(blockIdx.x / chunks) * (kCbThreads / LPR) + threadIdx.x / LPR;
  if (t >= a.T) return;
  const int c = 8 * (chunk * LPR + sub);
  if (c >= a.N) return;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  for (int j0 = 0; j0 < a.k; j0 += K) {
    int s[K];
    float g[K];
    uint4 u[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const bool in = j0 + j < a.k;
      s[j] = in ? a.slots[t * a.k + j0 + j] : -1;
      g[j] = in ? (a.gates ? a.gates[t * a.k + j0 + j] : 1.f) : 0.f;
    }
    const uint16_t* y = static_cast<const uint16_t*>(a.y);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      u[j] = make_uint4(0u, 0u, 0u, 0u);
      if (s[j] >= 0 && s[j] < a.S) u[j] = cb_load<F>(y + (int64_t)s[j] * a.ldy, c, a.N);
      else g[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      float f[8];
      cb_unpack<DT>(u[j], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += g[j] * f[i];
    }
  }
  cb_store<DT, F>(static_cast<uint16_t*>(a.out) + t * a.ldo, c, a.N, acc);
}

// One token a wave part of LPR lanes; its row in chunks of 8 LPR columns.
template <int LPR>
__device__ __forceinline__ float cb_row_sum(float x) {
  if constexpr (LPR >= 2) x += dpp_f<kDppQuadXor1>(x);
  if constexpr (LPR >= 4) x += dpp_f<kDppQuadXor2>(x);
  if constexpr (LPR >= 8) x += dpp_f<kDppRowHalfMirror>(x);
  if constexpr (LPR >= 16) x += dpp_f<kDppRowMirror>(x);
  if constexpr (LPR >= 32) x += __shfl_xor(x, 16);
  if constexpr (LPR >= 64) x += __shfl_xor(x, 32);
  return x;
}

// LPR kCbThreads: a token a workgroup, its waves' dot products joined in their order
// (few tokens, where a row's chunks one after another would be the time).
template <int DT, CbForm F, int LPR, int K>
__global__ __launch_bounds__(kCbThreads) void combine_bwd_k(CombineBwdArgs a) {
  constexpr bool kWhole = LPR == kCbThreads;
  __shared__ float part[kWhole ? kCbThreads / 64 : 1][K];
  const int sub = threadIdx.x % LPR;
  const int64_t t = (int64_t)blockIdx.x * (kCbThreads / LPR) + threadIdx.x / LPR;
  if (t >= a.T) return;
  const uint16_t* dout = static_cast<const uint16_t*>(a.dout) + t * a.ldd;
  const uint16_t* y = static_cast<const uint16_t*>(a.y);
  uint16_t* dy = static_cast<uint16_t*>(a.dy);
  // slots in no group: there are as many as choices without a slot, all behind
  // *offsets; pair (t, j) zeroes slot t k + j when that is one of them
  const int64_t used = *a.offsets;
  for (int j0 = 0; j0 < a.k; j0 += K) {
    int s[K];
    float g[K], dot[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const bool in = j0 + j < a.k;
      s[j] = in ? a.slots[t * a.k + j0 + j] : -1;
      if (s[j] >= a.S) s[j] = -1;
      g[j] = in ? a.gates[t * a.k + j0 + j] : 0.f;
      dot[j] = 0.f;
    }
    for (int c = 8 * sub; c < a.N; c += 8 * LPR) {
      float d[8];
      cb_unpack<DT>(cb_load<F>(dout, c, a.N), d);
      uint4 u[K];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        u[j] = make_uint4(0u, 0u, 0u, 0u);
        if (s[j] >= 0) u[j] = cb_load<F>(y + (int64_t)s[j] * a.ldy, c, a.N);
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (s[j] < 0) continue;
        float f[8], o[8];
        cb_unpack<DT>(u[j], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dot[j] += d[i] * f[i];
          o[i] = g[j] * d[i];
        }
        cb_store<DT, F>(dy + (int64_t)s[j] * a.N, c, a.N, o);
      }
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      float r = cb_row_sum<kWhole ? 64 : LPR>(dot[j]);
      if constexpr (kWhole) {
        if (sub % 64 == 0) part[sub / 64][j] = r;
        __syncthreads();
        r = 0.f;
#pragma unroll
        for (int q = 0; q < kCbThreads / 64; ++q) r += part[q][j];
      }
      if (sub == 0 && j0 + j < a.k) a.dgates[t * a.k + j0 + j] = r;
    }
    if constexpr (kWhole) __syncthreads();
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int64_t z = t * a.k + j0 + j;
      if (j0 + j < a.k && z >= used && z < a.S) {
        const float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int c = 8 * sub; c < a.N; c += 8 * LPR) cb_store<DT, F>(dy + z * a.N, c, a.N, o);
      }
    }
  }
}

int cb_lpr(int N) {
  int l = 8;
  while (l < 64 && 8 * l < N) l *= 2;
  return l;
}
bool al16(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

template <int DT, CbForm F, int LPR>
hipError_t launch_combine(const CombineArgs& a, hipStream_t s) {
  const int per = kCbThreads / LPR, chunks = (a.N + 8 * LPR - 1) / (8 * LPR);
  const int64_t blocks = (a.T + per - 1) / per * chunks;
  if (blocks * kCbThreads > kMaxThreads) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)blocks);
  if (a.k == 1) hipLaunchKernelGGL((combine_k<DT, F, LPR, 1>), grid, dim3(kCbThreads), 0, s, a, chunks);
  else if (a.k == 2) hipLaunchKernelGGL((combine_k<DT, F, LPR, 2>), grid, dim3(kCbThreads), 0, s, a, chunks);
  else hipLaunchKernelGGL((combine_k<DT, F, LPR, 4>), grid, dim3(kCbThreads), 0, s, a, chunks);
  return hipGetLastError();
}
template <int DT, CbForm F, int LPR>
hipError_t launch_combine_bwd(const CombineBwdArgs& a, hipStream_t s) {
  // (512 tokens of 2 rows of 4096: 5.4 us, 9.7 with a wave a token; 1024: 8.5 and 11.6;
  // 1024 of 4 rows of 1000: 6.2 and 6.5)
  if constexpr (LPR == 64) {
    if (a.T <= 1024) return launch_combine_bwd<DT, F, kCbThreads>(a, s);
  }
  const int per = kCbThreads / LPR;
  const int64_t blocks = (a.T + per - 1) / per;
  if (blocks * kCbThreads > kMaxThreads) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)blocks);
  if (a.k == 1) hipLaunchKernelGGL((combine_bwd_k<DT, F, LPR, 1>), grid, dim3(kCbThreads), 0, s, a);
  else if (a.k == 2) hipLaunchKernelGGL((combine_bwd_k<DT, F, LPR, 2>), grid, dim3(kCbThreads), 0, s, a);
  else hipLaunchKernelGGL((combine_bwd_k<DT, F, LPR, 4>), grid, dim3(kCbThreads), 0, s, a);
  return hipGetLastError();
}
#define DSML_CB_LPR(FN, F, a, s)                    \
  switch (cb_lpr(a.N)) {                            \
    case 8: return FN<DT, F, 8>(a, s);              \
    case 16: return FN<DT, F, 16>(a, s);            \
    case 32: return FN<DT, F, 32>(a, s);            \
    default: return FN<DT, F, 64>(a, s);            \
  }
#define DSML_CB_DISPATCH(FN, a, words, s)           \
  if (words) DSML_CB_LPR(FN, kWords, a, s)          \
  if (a.N >= 8) DSML_CB_LPR(FN, kMoved, a, s)       \
  return FN<DT, kSingle, 8>(a, s);
template <int DT>
hipError_t combine_dt(const CombineArgs& a, bool words, hipStream_t s) {
  DSML_CB_DISPATCH(launch_combine, a, words, s)
}
template <int DT>
hipError_t combine_bwd_dt(const CombineBwdArgs& a, bool words, hipStream_t s) {
  DSML_CB_DISPATCH(launch_combine_bwd, a, words, s)
}
#undef DSML_CB_DISPATCH
#undef DSML_CB_LPR

bool cb_ok(int64_t T, int N, int k) {
  return T >= 0 && N >= 1 && k >= 1 && k <= kCombineMaxK && T <= 0x7fffffffLL / k && N <= 65535 * 64;
}

}  // namespace

hipError_t expert_combine(const CombineArgs& a, hipStream_t s) {
  if (!cb_ok(a.T, a.N, a.k)) return hipErrorInvalidValue;
  if (a.T == 0) return hipSuccess;
  const bool words = a.N % 8 == 0 && al16(a.y, a.ldy) && al16(a.out, a.ldo);
  if (a.dtype == kBF16) return combine_dt<kBF16>(a, words, s);
  if (a.dtype == kF16) return combine_dt<kF16>(a, words, s);
  return hipErrorInvalidValue;
}

hipError_t expert_combine_backward(const CombineBwdArgs& a, hipStream_t s) {
  if (!cb_ok(a.T, a.N, a.k)) return hipErrorInvalidValue;
  if (a.T == 0) return hipSuccess;
  const bool words = a.N % 8 == 0 && al16(a.y, a.ldy) && al16(a.dout, a.ldd) && al16(a.dy, a.N);
  if (a.dtype == kBF16) return combine_bwd_dt<kBF16>(a, words, s);
  if (a.dtype == kF16) return combine_bwd_dt<kF16>(a, words, s);
  return hipErrorInvalidValue;
}

}  // namespace dsml
