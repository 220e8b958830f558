// Global norm of many gradient tensors, and clipping by it:
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   out  = g * min(1, max_norm / (norm + eps))       (out may be g itself)
//
// Squares are summed in fp64 (any finite fp32 gradient's square is finite
// there, and the sum loses nothing that matters over 1e9 elements; the kernel
// waits for bytes, not for arithmetic).  Two passes: the first leaves one fp64
// partial per workgroup, every workgroup of the second sums all of them in
// the same order -- no atomics, so the result does not depend on timing -- and
// scales its share.  Tensors are cut into pieces of 256 to 4096 16-B words: about
// 1024 pieces in all while 4096 words are enough for that (400 M fp32 gradients are
// some 24400 of them), of which a workgroup takes every gridDim-th, 8 words a thread in
// flight.  The tensor table travels in the kernel arguments, so a call keeps
// nothing on the device and can be captured.  Tensors that do not start at a
// multiple of 16 B go element by element.
//
// 400 M fp32 gradients in 60 tensors, clipped into others: 899 us, 290 for the norm
// (5.5 TB/s) and 600 for the scaling (5.3 TB/s, read and write).  109386 in 6: 7.7 us
// in the two kernels; the host needs 10 to call.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "../dsml.h"
#include "../experts.h"

namespace dsml {
namespace {

constexpr int kGnThreads = 256;
constexpr int kGnMax = 128;            // tensors of one launch (3.6 KB of arguments)
constexpr int kGnBlocks = 1024;        // workgroups over all launches, about

struct GnTable {
  const void* g[kGnMax];
  void* out[kGnMax];
  int64_t n[kGnMax];
  uint32_t start[kGnMax + 1];  // first piece of each tensor
  int count;
  int piece;  // 16-B words
};

template <int DT>
constexpr int gn_per() { return DT == kF32 ? 4 : 8; }

template <int DT>
__device__ __forceinline__ float gn_ld(const void* p, int64_t i) {
  if constexpr (DT == kF32) return static_cast<const float*>(p)[i];
  else if constexpr (DT == kBF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  else return __half2float(static_cast<const __half*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void gn_st(void* p, int64_t i, float v) {
  if constexpr (DT == kF32) static_cast<float*>(p)[i] = v;
  else if constexpr (DT == kBF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  else static_cast<__half*>(p)[i] = __float2half(v);
}
template <int DT>
__device__ __forceinline__ void gn_unpack(uint4 u, float (&f)[gn_per<DT>()]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < gn_per<DT>(); ++i) {
    if constexpr (DT == kF32) f[i] = __uint_as_float(w[i]);
    else if constexpr (DT == kBF16) f[i] = bf16_to_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
    else f[i] = __half2float(__ushort_as_half((uint16_t)(w[i >> 1] >> (16 * (i & 1)))));
  }
}
template <int DT>
__device__ __forceinline__ uint4 gn_pack(const float (&f)[gn_per<DT>()]) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < gn_per<DT>(); ++i) {
    if constexpr (DT == kF32) w[i] = __float_as_uint(f[i]);
    else if constexpr (DT == kBF16) w[i >> 1] |= (uint32_t)f32_to_bf16(f[i]) << (16 * (i & 1));
    else w[i >> 1] |= (uint32_t)__half_as_ushort(__float2half(f[i])) << (16 * (i & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Tensor of piece p.  The lanes look at all the starts at once: the arguments
// lie in memory, and a search would wait for them once a halving.
__device__ __forceinline__ int gn_find(const GnTable& t, uint32_t p) {
  const int lane = threadIdx.x & 63;
  const GnTable* k = (const GnTable*)__builtin_amdgcn_kernarg_segment_ptr();  // t is the first argument
  int at = 0;
#pragma unroll
  for (int i = 0; i < kGnMax; i += 64) {
    const bool before = i + lane < t.count && k->start[i + lane] <= p;
    at += __popcll(__ballot(before));
  }
  return __builtin_amdgcn_readfirstlane(at - 1);
}

// f(k) for this thread's 16-B words k of a piece, [first, last) in elements of
// which whole words are [k0, k1); U words in flight.
template <int U, class Load, class Use>
__device__ __forceinline__ void gn_words(int64_t k0, int64_t k1, Load load, Use use) {
  int64_t k = k0 + threadIdx.x;
  for (; k + (U - 1) * kGnThreads < k1; k += U * kGnThreads) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load(k + u * kGnThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) use(k + u * kGnThreads, v[u]);
  }
  for (; k < k1; k += kGnThreads) use(k, load(k));
}

__device__ __forceinline__ double gn_block_sum(double v, double* lds) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  const int w = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[w] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kGnThreads / 64; ++i) s += lds[i];
  return s;
}

template <int DT>
__global__ __launch_bounds__(kGnThreads) void grad_sq_k(GnTable t, double* part) {
  __shared__ double lds[kGnThreads / 64];
  constexpr int P = gn_per<DT>();
  double acc = 0.0;
  const uint32_t pieces = t.start[t.count];
  for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
    const int i = gn_find(t, p);
    const void* g = t.g[i];
    const int64_t n = t.n[i], first = (int64_t)(p - t.start[i]) * t.piece * P;
    const int64_t last = first + (int64_t)t.piece * P < n ? first + (int64_t)t.piece * P : n;
    if ((reinterpret_cast<uintptr_t>(g) & 15) == 0) {
      const uint4* v = reinterpret_cast<const uint4*>(g);
      const int64_t v1 = last / P;
      gn_words<8>(first / P, v1, [&](int64_t k) { return v[k]; }, [&](int64_t, uint4 u) {
        float f[P];
        gn_unpack<DT>(u, f);
#pragma unroll
        for (int j = 0; j < P; ++j) acc = fma((double)f[j], (double)f[j], acc);
      });
      for (int64_t k = v1 * P + threadIdx.x; k < last; k += kGnThreads) {
        const double x = gn_ld<DT>(g, k);
        acc = fma(x, x, acc);
      }
    } else {
      for (int64_t k = first + threadIdx.x; k < last; k += kGnThreads) {
        const double x = gn_ld<DT>(g, k);
        acc = fma(x, x, acc);
      }
    }
  }
  const double s = gn_block_sum(acc, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double gn_total(const double* part, int parts, double* lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kGnThreads) s += part[i];
  return gn_block_sum(s, lds);
}

__global__ __launch_bounds__(kGnThreads) void grad_norm_k(const double* part, int parts, float* norm) {
  __shared__ double lds[kGnThreads / 64];
  const double s = gn_total(part, parts, lds);
  if (threadIdx.x == 0) norm[0] = (float)sqrt(s);
}

// g * factor over this workgroup's pieces: one fp32 product, or (FINE) one in fp64,
// where fp32 would not hold the factor's bits.
template <int DT, bool FINE>
__device__ __forceinline__ void gn_scale(const GnTable& t, double factor) {
  constexpr int P = gn_per<DT>();
  const float c = (float)factor;
  auto scaled = [&](float g) { return FINE ? (float)((double)g * factor) : g * c; };
  const uint32_t pieces = t.start[t.count];
  for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
    const int i = gn_find(t, p);
    const void* g = t.g[i];
    void* o = t.out[i];
    if (!FINE && c == 1.f && o == g) continue;  // nothing changes
    const int64_t n = t.n[i], first = (int64_t)(p - t.start[i]) * t.piece * P;
    const int64_t last = first + (int64_t)t.piece * P < n ? first + (int64_t)t.piece * P : n;
    if (((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(o)) & 15) == 0) {
      const uint4* v = reinterpret_cast<const uint4*>(g);
      uint4* w = reinterpret_cast<uint4*>(o);
      const int64_t v1 = last / P;
      gn_words<FINE ? 1 : 8>(first / P, v1, [&](int64_t k) { return v[k]; }, [&](int64_t k, uint4 u) {
        float f[P];
        gn_unpack<DT>(u, f);
#pragma unroll
        for (int j = 0; j < P; ++j) f[j] = scaled(f[j]);
        w[k] = gn_pack<DT>(f);
      });
      for (int64_t k = v1 * P + threadIdx.x; k < last; k += kGnThreads) gn_st<DT>(o, k, scaled(gn_ld<DT>(g, k)));
    } else {
      for (int64_t k = first + threadIdx.x; k < last; k += kGnThreads) gn_st<DT>(o, k, scaled(gn_ld<DT>(g, k)));
    }
  }
}

// Every workgroup sums the partials in the same order, so all scale by the same value.
template <int DT>
__global__ __launch_bounds__(kGnThreads) void grad_scale_k(GnTable t, const double* part, int parts, float* norm,
                                                           double max_norm, double eps) {
  __shared__ double lds[kGnThreads / 64];
  const double nrm = sqrt(gn_total(part, parts, lds));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)nrm;
  double cd = nrm + eps == 0.0 ? 1.0 : max_norm / (nrm + eps);  // nothing but zeros: not 0 / 0
  cd = cd > 1.0 ? 1.0 : cd;  // NaN stays NaN: a broken gradient is not hidden
  // below 2^-126 (a norm past 1e38 times the limit) fp32 drops bits of the factor;
  // fp16 results are zeros by then
  if constexpr (DT != kF16) {
    if (cd > 0.0 && cd < 0x1p-126) return gn_scale<DT, true>(t, cd);
  }
  gn_scale<DT, false>(t, cd);
}

// gn_find reads the table where the first argument lies.
template <class F>
struct GnFirst;
template <class A, class... R>
struct GnFirst<void (*)(A, R...)> {
  using type = A;
};
static_assert(std::is_same_v<GnFirst<decltype(&grad_sq_k<kF32>)>::type, GnTable>, "the table comes first");
static_assert(std::is_same_v<GnFirst<decltype(&grad_scale_k<kF32>)>::type, GnTable>, "the table comes first");

int64_t gn_pieces(int64_t n, int P, int piece) {
  const int64_t per = (int64_t)piece * P;
  return (n + per - 1) / per;
}
// 16-B words of a piece: about 1024 pieces, whole rounds of the threads.
int gn_piece(int64_t words) {
  const int64_t w = (words / kGnBlocks + kGnThreads - 1) / kGnThreads * kGnThreads;
  return (int)std::min<int64_t>(4096, std::max<int64_t>(kGnThreads, w));
}
// Workgroups of one launch: its share of the pieces of the whole call.
int gn_grid(int64_t pieces, int64_t all) {
  if (pieces <= 0) return 1;
  int64_t g = all <= kGnBlocks ? pieces : (pieces * kGnBlocks + all - 1) / all;
  return (int)std::max<int64_t>(1, g);
}

}  // namespace

int64_t grad_norm_ws_doubles(int count) {
  // every launch rounds its share up by at most one workgroup
  return kGnBlocks + (count + kGnMax - 1) / kGnMax + 1;
}

template <int DT>
static hipError_t run_norm(const ClipTensor* t, int count, double* ws, float* norm, bool clip, double max_norm,
                           double eps, hipStream_t s) {
  constexpr int P = gn_per<DT>();
  int64_t all = 0, words = 0;
  for (int i = 0; i < count; ++i) words += t[i].n / P;
  const int piece = gn_piece(words);
  for (int i = 0; i < count; ++i) {
    if (t[i].n < 0 || gn_pieces(t[i].n, P, piece) > 0x3fffffffLL) return hipErrorInvalidValue;
    all += gn_pieces(t[i].n, P, piece);
  }
  int parts = 0;
  for (int pass = 0; pass < (clip ? 2 : 1); ++pass) {
    for (int i0 = 0; i0 < count; i0 += kGnMax) {
      GnTable tb;
      tb.count = std::min(kGnMax, count - i0);
      tb.piece = piece;
      int64_t pieces = 0;
      for (int i = 0; i < tb.count; ++i) {
        tb.g[i] = t[i0 + i].g;
        tb.out[i] = t[i0 + i].out;
        tb.n[i] = t[i0 + i].n;
        tb.start[i] = (uint32_t)pieces;
        pieces += gn_pieces(t[i0 + i].n, P, piece);
        if (pieces > 0x7fffffffLL) return hipErrorInvalidValue;
      }
      tb.start[tb.count] = (uint32_t)pieces;
      const int grid = gn_grid(pieces, all);
      if (pass == 0) {
        hipLaunchKernelGGL((grad_sq_k<DT>), dim3(grid), dim3(kGnThreads), 0, s, tb, ws + parts);
        parts += grid;
      } else {
        hipLaunchKernelGGL((grad_scale_k<DT>), dim3(grid), dim3(kGnThreads), 0, s, tb, ws, parts,
                           i0 == 0 ? norm : nullptr, max_norm, eps);
      }
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  if (!clip || count == 0) {
    hipLaunchKernelGGL(grad_norm_k, dim3(1), dim3(kGnThreads), 0, s, ws, parts, norm);
    return hipGetLastError();
  }
  return hipSuccess;
}

hipError_t grad_norm(const ClipTensor* t, int count, int dtype, double* ws, float* norm, bool clip, double max_norm,
                     double eps, hipStream_t s) {
  switch (dtype) {
    case kF32: return run_norm<kF32>(t, count, ws, norm, clip, max_norm, eps, s);
    case kBF16: return run_norm<kBF16>(t, count, ws, norm, clip, max_norm, eps, s);
    case kF16: return run_norm<kF16>(t, count, ws, norm, clip, max_norm, eps, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace dsml
