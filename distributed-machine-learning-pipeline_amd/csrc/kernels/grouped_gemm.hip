// Matrix products grouped by expert: group e owns the rows [off[e], off[e + 1])
// of the slot axis, of any length, zero and one included.
//
//   linear : y[s][n]   = act(sum_k x[row(s)][k] w[e][n][k] + b[e][n])
//   dgrad  : dx[s][k]  = (sum_n dz[s][n] w[e][n][k]) * (mask[s][k] > 0)
//   wgrad  : dw[e][n][k] = sum_s dz[s][n] x[row(s)][k]   (fp32),  db[e][n] = sum_s dz[s][n]
//
// The offsets live on the GPU (the router writes them), so the host sizes the
// grid by what they can be at most -- ceil(S / BM) + E row tiles -- and every
// workgroup finds its expert by a wave scan over the groups' tile counts.
// Offsets and rows are clamped to the buffers they index: a wrong plan gives
// wrong numbers, never an access outside the operands.
#include "common.h"
#include "../dsml.h"
#include "../experts.h"

namespace dsml {
namespace {

typedef __bf16 gg_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gg_f16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x4 gg_mfma16(uint4 a, uint4 b, f32x4 c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gg_bf16x8, a), __builtin_bit_cast(gg_bf16x8, b),
                                                    c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gg_f16x8, a), __builtin_bit_cast(gg_f16x8, b), c,
                                                   0, 0, 0);
}
template <int DT>
__device__ __forceinline__ float gg_f(uint16_t h) {
  if constexpr (DT == kBF16) return bf16_to_f32(h);
  else return __half2float(__ushort_as_half(h));
}
template <int DT>
__device__ __forceinline__ uint16_t gg_h(float v) {
  if constexpr (DT == kBF16) return f32_to_bf16(v);
  else return __half_as_ushort(__float2half(v));
}

struct GgTile {
  int e;          // expert, -1: rows to zero, -2: nothing
  int64_t s0, s1; // rows of this tile
};

__device__ __forceinline__ int64_t gg_clamp(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Row tile `mt` in the order: the experts' tiles, then (zero_rest) the tiles of
// the rows before the first group and behind the last.  One wave scan per 64
// experts; every wave does it for itself (no LDS, no barrier).
__device__ __forceinline__ GgTile gg_find(const int32_t* off, int E, int64_t S, int BM, int64_t mt, bool zero_rest) {
  const int lane = threadIdx.x & 63;
  int64_t base = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int e = e0 + lane;
    int64_t a = 0, b = 0;
    if (e < E) {
      a = gg_clamp(off[e], 0, S);
      b = gg_clamp(off[e + 1], a, S);
    }
    const int n = (int)((b - a + BM - 1) / BM);
    int inc = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(inc, o);
      if (lane >= o) inc += u;
    }
    const int tot = __shfl(inc, 63);
    if (mt < base + tot) {
      const uint64_t hit = __ballot(base + inc > mt);
      const int l = __ffsll((unsigned long long)hit) - 1;
      const int64_t first = base + __shfl(inc, l) - __shfl(n, l);
      const int64_t a0 = __shfl((int)a, l), b0 = __shfl((int)b, l);
      GgTile t;
      t.e = e0 + l;
      t.s0 = a0 + (mt - first) * BM;
      t.s1 = t.s0 + BM < b0 ? t.s0 + BM : b0;
      return t;
    }
    base += tot;
  }
  GgTile t{-2, 0, 0};
  if (!zero_rest) return t;
  const int64_t head = gg_clamp(off[0], 0, S), tail = gg_clamp(off[E], head, S);
  int64_t r = mt - base;
  const int64_t hn = (head + BM - 1) / BM;
  if (r < hn) {
    t.e = -1; t.s0 = r * BM; t.s1 = t.s0 + BM < head ? t.s0 + BM : head;
  } else {
    r -= hn;
    const int64_t s = tail + r * BM;
    if (s < S) { t.e = -1; t.s0 = s; t.s1 = s + BM < S ? s + BM : S; }
  }
  return t;
}

// ---------------------------------------------------------------------------
// Any size, stride and alignment: 64 x 64 output tile, 4 waves of 32 x 32,
// operands loaded element by element into LDS as [row][reduction].
// ---------------------------------------------------------------------------
constexpr int kGgBk = 32;
constexpr int kGgPitch = 40;  // elements of an LDS row (80 B: 16-B aligned fragments)

template <int DT, int OP>
__global__ __launch_bounds__(256) void grouped_any_k(GroupedArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t la[64 * kGgPitch], lb[64 * kGgPitch];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const uint16_t* A = static_cast<const uint16_t*>(a.a);
  const uint16_t* B = static_cast<const uint16_t*>(a.b);
  int e, n0 = 64 * blockIdx.y;
  int64_t m0, m1, r0, r1;  // output rows [m0, m1), reduction [r0, r1)
  const int ncols = OP == kLinear ? a.N : a.K;
  if constexpr (OP == kWgrad) {
    e = blockIdx.z;
    m0 = 64 * (int64_t)blockIdx.x;
    m1 = m0 + 64 < a.N ? m0 + 64 : a.N;
    r0 = gg_clamp(a.offsets[e], 0, a.S);
    r1 = gg_clamp(a.offsets[e + 1], r0, a.S);
  } else {
    const GgTile t = gg_find(a.offsets, a.E, a.S, 64, blockIdx.x, a.zero_rest);
    if (t.e == -2) return;
    e = t.e; m0 = t.s0; m1 = t.s1;
    r0 = 0;
    r1 = e < 0 ? 0 : (OP == kLinear ? a.K : a.N);
  }
  f32x4 acc[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) acc[x][y] = {0.f, 0.f, 0.f, 0.f};
  float dbias = 0.f;
  const int wm = 32 * (w >> 1), wn = 32 * (w & 1), i = lane & 15, g = lane >> 4;
  for (int64_t r = r0; r < r1; r += kGgBk) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      // consecutive threads walk the operand's contiguous axis
      uint16_t va = 0, vb = 0;
      int ra, ka, rb, kb;
      if constexpr (OP == kWgrad) {
        ra = tid & 63; ka = (tid >> 6) + 4 * q;
        rb = ra; kb = ka;
        const int64_t s = r + ka;
        if (s < r1) {
          if (m0 + ra < m1) va = A[s * a.lda + m0 + ra];
          const int64_t row = a.rows ? a.rows[s] : s;
          if (row >= 0 && row < a.T && n0 + rb < ncols) vb = B[row * a.ldb + n0 + rb];
        }
      } else {
        ka = tid & 31; ra = (tid >> 5) + 8 * q;
        const int64_t s = m0 + ra;
        if (s < m1 && r + ka < r1) {
          const int64_t row = OP == kLinear && a.rows ? a.rows[s] : s;
          if (OP != kLinear || (row >= 0 && row < a.T)) va = A[row * a.lda + r + ka];
        }
        if constexpr (OP == kLinear) {
          kb = ka; rb = ra;
          if (n0 + rb < ncols && r + kb < r1) vb = B[e * a.strb + (int64_t)(n0 + rb) * a.ldb + r + kb];
        } else {
          rb = tid & 63; kb = (tid >> 6) + 4 * q;
          if (n0 + rb < ncols && r + kb < r1) vb = B[e * a.strb + (r + kb) * a.ldb + n0 + rb];
        }
      }
      la[ra * kGgPitch + ka] = va;
      lb[rb * kGgPitch + kb] = vb;
    }
    __syncthreads();
    uint4 fa[2], fb[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      fa[x] = *reinterpret_cast<const uint4*>(la + (wm + 16 * x + i) * kGgPitch + 8 * g);
      fb[x] = *reinterpret_cast<const uint4*>(lb + (wn + 16 * x + i) * kGgPitch + 8 * g);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) acc[x][y] = gg_mfma16<DT>(fa[x], fb[y], acc[x][y]);
    if constexpr (OP == kWgrad) {
      if (a.db && blockIdx.y == 0 && tid < 64)
        for (int k = 0; k < kGgBk; ++k) dbias += gg_f<DT>(la[tid * kGgPitch + k]);
    }
    __syncthreads();
  }
  if constexpr (OP == kWgrad) {
    if (a.db && blockIdx.y == 0 && tid < 64 && m0 + tid < m1) a.db[(int64_t)e * a.N + m0 + tid] = dbias;
  }
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int n = n0 + wn + 16 * y + i;
      if (n >= ncols) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t m = m0 + wm + 16 * x + 4 * g + q;
        if (m >= m1) continue;
        float v = acc[x][y][q];
        if constexpr (OP == kLinear) {
          if (e >= 0) {
            if (a.bias) v += a.bias[(int64_t)e * a.ldbias + n];
            if (a.relu) v = v < 0.f ? 0.f : v;  // NaN stays NaN
          }
        } else if constexpr (OP == kDgrad) {
          if (e >= 0 && a.mask && !(gg_f<DT>(static_cast<const uint16_t*>(a.mask)[m * a.ldmask + n]) > 0.f)) v = 0.f;
        }
        if constexpr (OP == kWgrad) static_cast<float*>(a.out)[e * a.stro + m * a.ldo + n] = v;
        else static_cast<uint16_t*>(a.out)[m * a.ldo + n] = gg_h<DT>(v);
      }
    }
}

template <int DT>
hipError_t launch_any(GroupedOp op, const GroupedArgs& a, hipStream_t s) {
  const int64_t tiles = (a.S + 63) / 64 + a.E + (a.zero_rest ? 2 : 0);
  if (op == kWgrad) {
    const dim3 grid((a.N + 63) / 64, (a.K + 63) / 64, a.E);
    hipLaunchKernelGGL((grouped_any_k<DT, kWgrad>), grid, dim3(256), 0, s, a);
  } else {
    const int cols = op == kLinear ? a.N : a.K;
    const dim3 grid((uint32_t)(tiles < a.S ? tiles : a.S), (cols + 63) / 64);
    if (op == kLinear) hipLaunchKernelGGL((grouped_any_k<DT, kLinear>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((grouped_any_k<DT, kDgrad>), grid, dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace

int64_t grouped_ws_floats(GroupedOp op, const GroupedArgs& a) {
  (void)op; (void)a;
  return 0;
}

hipError_t grouped_gemm(GroupedOp op, const GroupedArgs& a, hipStream_t s) {
  if (a.E < 1 || a.N < 1 || a.K < 1 || a.S < 0 || a.T < 0 || a.S > 0x7fffffffLL || a.T > 0x7fffffffLL ||
      (a.dtype != kBF16 && a.dtype != kF16))
    return hipErrorInvalidValue;
  if (op != kWgrad && a.S == 0) return hipSuccess;
  return a.dtype == kBF16 ? launch_any<kBF16>(op, a, s) : launch_any<kF16>(op, a, s);
}

}  // namespace dsml
