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
#include <type_traits>

#include "common.h"
#include "../dsml.h"
#include "../experts.h"

// The LDS-DMA below sets M0 by itself; the compiler keeps nothing there.
#pragma clang diagnostic ignored "-Winline-asm"

namespace dsml {

typedef int gg_i4 __attribute__((ext_vector_type(4)));
// A scalar load behind a buffer descriptor (0 past its end).
__device__ int gg_sload(gg_i4 rsrc, int offset, int policy) __asm("llvm.amdgcn.s.buffer.load.i32");

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

// The groups' row tiles, experts first, then (zero_rest) the tiles of the rows
// before the first group and behind the last.  `pick` maps the number of tiles
// to the one wanted (< 0 or too large: nothing).  One wave scan per 64 experts,
// done by every wave for itself: no LDS, no barrier.
template <class Pick>
__device__ __forceinline__ GgTile gg_find(const int32_t* off, int E, int64_t S, int BM, bool zero_rest, Pick pick) {
  const int lane = threadIdx.x & 63;
  int a = 0, b = 0, n = 0, inc = 0, tot = 0;
  auto scan = [&](int e0) {
    const int e = e0 + lane;
    a = b = 0;
    if (e < E) {
      a = (int)gg_clamp(off[e], 0, S);
      b = (int)gg_clamp(off[e + 1], a, S);
    }
    n = (int)(((int64_t)b - a + BM - 1) / BM);
    inc = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(inc, o);
      if (lane >= o) inc += u;
    }
    tot = __builtin_amdgcn_readlane(inc, 63);
  };
  int total = 0;
  for (int e0 = (E - 1) & ~63; e0 >= 0; e0 -= 64) {  // the first 64 stay in registers
    scan(e0);
    total += tot;
  }
  int64_t head = 0, tail = 0;
  int hn = 0, tn = 0;
  if (zero_rest) {
    head = gg_clamp(off[0], 0, S);
    tail = gg_clamp(off[E], head, S);
    hn = (int)((head + BM - 1) / BM);
    tn = (int)((S - tail + BM - 1) / BM);
  }
  GgTile t{-2, 0, 0};
  int mt = pick(total + hn + tn);
  if (mt < 0) return t;
  if (mt < total) {
    int e0 = 0;
    while (mt >= tot) {
      mt -= tot;
      e0 += 64;
      if (e0 >= E) return t;
      scan(e0);
    }
    const int l = __ffsll((unsigned long long)__ballot(inc > mt)) - 1;
    const int first = __builtin_amdgcn_readlane(inc, l) - __builtin_amdgcn_readlane(n, l);
    const int64_t a0 = __builtin_amdgcn_readlane(a, l), b0 = __builtin_amdgcn_readlane(b, l);
    t.e = e0 + l;
    t.s0 = a0 + (int64_t)(mt - first) * BM;
    t.s1 = t.s0 + BM < b0 ? t.s0 + BM : b0;
    return t;
  }
  mt -= total;
  if (mt < hn) {
    t.e = -1; t.s0 = (int64_t)mt * BM; t.s1 = t.s0 + BM < head ? t.s0 + BM : head;
  } else if (mt - hn < tn) {
    t.e = -1; t.s0 = tail + (int64_t)(mt - hn) * BM; t.s1 = t.s0 + BM < S ? t.s0 + BM : S;
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
    const GgTile t = gg_find(a.offsets, a.E, a.S, 64, a.zero_rest, [](int) { return (int)blockIdx.x; });
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

// ---------------------------------------------------------------------------
// Fast path: widths and row strides of whole 16-B words.  256 x 256 output
// tile, 64-deep steps, 8 waves of 128 x 64 (16x16x32 MFMA), operands by LDS-DMA
// into two buffers.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void* gg_lptr;
typedef short gg_i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) gg_i16x4* gg_lv4;
typedef uint32_t gg_u4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kGgOob = 0xfffffff0u;    // past every buffer: reads 0
constexpr int64_t kGgSpan = 0xffffff00LL;   // bytes a buffer descriptor may span

__device__ __forceinline__ __amdgpu_buffer_rsrc_t gg_rsrc(const void* base, int64_t bytes) {
  const uint32_t n = bytes <= 0 ? 0u : (bytes > kGgSpan ? (uint32_t)kGgSpan : (uint32_t)bytes);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, n, 0x00020000);
}
// A value every lane holds, in scalar registers.
__device__ __forceinline__ int64_t gg_uni(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ const char* gg_uni(const char* v) { return reinterpret_cast<const char*>(gg_uni((int64_t)v)); }
template <int IMM>
__device__ __forceinline__ void gg_dma(__amdgpu_buffer_rsrc_t r, char* lds, uint32_t vo, uint32_t so) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (gg_lptr)lds, 16, vo, so, IMM, 0);
}
// LDS image of one 64-deep step of an operand, 1-KiB pieces of 8 rows x 128 B:
//   row-major   rows of 64 reduction elements; row r lies at 64 (r / 64) + 8 (r % 8) + r / 8 % 8
//   transposed  per 64 columns, 64 reduction rows of them; row r lies at 8 (r % 8) + r / 8
// so the 8 rows of one LDS-DMA instruction are 8 rows apart in memory: adjacent
// rows of some power-of-two strides (8 KiB among them) fall on one cache channel,
// 35 B/clk a CU instead of 52.  16-B chunks are XORed with a function of the LDS
// row, so fragment reads touch every bank once.
__device__ __forceinline__ int gg_swz(int pos) { return (pos >> 3) & 7; }
__device__ __forceinline__ int gg_swz_tr(int pos) { return 2 * (((pos >> 1) & 1) | (((pos >> 3) & 1) << 1)); }

// One operand of the product as a stream of 64-deep steps.  GATHER (transposed
// only): reduction row k is row ids[k] of base; a step's 8 ids of a wave are
// scalar loads made a step ahead.
template <int R, int WAVES, bool TR, bool GATHER = false>
struct GgOperand {
  static constexpr int kPieces = R / 8 / WAVES;  // 1-KiB pieces of a step, a wave
  const char* base;
  int64_t bytes;   // behind base, all rows
  int64_t step;    // bytes the base moves a step (TR)
  uint32_t vo[kPieces];
  int c8;          // !TR: this lane's first element in a step
  gg_u4 rs;
  uint32_t so;
  // GATHER
  gg_i4 irs;        // the group's ids
  uint32_t iat;     // byte offset of this wave's first id of the step to fetch
  int id[8];
  uint32_t ld2, rows, rowoff;
  int k, rr;        // this lane's reduction row in a step: w + 8 rr

  __device__ __forceinline__ void fetch_ids() {
#pragma unroll
    for (int q = 0; q < 8; ++q) id[q] = gg_sload(irs, (int)(iat + 32 * q), 0);
    iat += 256;
  }
  // Row offset of the step whose ids were fetched (left: its reduction rows); fetches the next ids.
  __device__ __forceinline__ void take_ids(int left) {
    int v = id[0];
#pragma unroll
    for (int q = 1; q < 8; ++q) v = rr == q ? id[q] : v;
    rowoff = (uint32_t)v < rows && k < left ? (uint32_t)v * ld2 : kGgOob;
    fetch_ids();
  }

  __device__ __forceinline__ void first() {
    const int64_t b = reinterpret_cast<int64_t>(base);
    const int64_t n = bytes < 0 ? 0 : (bytes > kGgSpan ? kGgSpan : bytes);
    rs = gg_u4{(uint32_t)b, (uint32_t)((uint64_t)b >> 32) & 0xffffu, (uint32_t)n, 0x00020000u};
    so = 0;
  }
  __device__ __forceinline__ void next() {
    if constexpr (!TR) {
      so += 128;
    } else {
      base += step;
      bytes -= step;
      first();
    }
  }
  __device__ __forceinline__ void tail(int left) {  // a row-major step that ends inside, or is none: zeros
    if constexpr (!TR) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) vo[j] = (c8 ^ (8 * (WAVES * j & 7))) < left ? vo[j] : kGgOob;
    }
  }
  // On to the next step, which has `left` reduction rows or elements (or fewer than none).
  __device__ __forceinline__ void advance(int left) {
    if constexpr (GATHER) {
      take_ids(left);
    } else {
      next();
      if (left < 64) tail(left);
    }
  }
  // The LDS-DMA is opaque to the compiler: it would wait for every one in
  // flight before any LDS read.  Arrival is waited for by count (arrived()).
  __device__ __forceinline__ void issue(uint32_t lds, int j) {
    uint32_t v = vo[j];
    if constexpr (GATHER) v = __builtin_elementwise_add_sat(v, rowoff);  // kGgOob stays past the end
    asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(v), "s"(rs),
                 "s"(so), "i"(WAVES * j * 1024)
                 : "m0", "scc");
  }
};

// Fragments of 16 rows (columns when TR): lane (i, g) holds reduction elements
// 32 h + 8 g .. + 7 of row i.  Lane part of the address; the rest is constant.
template <bool TR>
struct GgReader {
  uint32_t p[TR ? 4 : 2];
  __device__ __forceinline__ void init(int wbase, int lane) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (!TR) {
      const int pos = 64 * (wbase >> 6) + 8 * (i & 7) + ((wbase & 63) >> 3) + (i >> 3);
#pragma unroll
      for (int h = 0; h < 2; ++h) p[h] = pos * 128 + 16 * ((4 * h + g) ^ gg_swz(pos));
    } else {
      const int q = i >> 2, pp = i & 3, pos = 8 * q + g;  // + 4 h, + 32 for elements 4 .. 7
#pragma unroll
      for (int x = 0; x < 4; ++x)
        p[x] = (wbase >> 6) * 8192 + pos * 128 + 16 * ((2 * (((wbase & 63) >> 4) ^ x) + (pp >> 1)) ^ gg_swz_tr(pos)) + 8 * (pp & 1);
    }
  }
};
typedef __attribute__((address_space(3))) const gg_u4* gg_lu4;
template <bool TR>
__device__ __forceinline__ gg_u4 gg_frag(const GgReader<TR>& rd, uint32_t img, int h, int x) {
  if constexpr (!TR) return *(gg_lu4)(uintptr_t)(rd.p[h] + img + (x >> 2) * 8192 + (x & 3) * 256);
  const uint32_t a = rd.p[x & 3] + img + (x >> 2) * 8192 + h * 512;
  const gg_i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gg_lv4)(uintptr_t)(a));
  const gg_i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gg_lv4)(uintptr_t)(a + 4096));
  const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
  return gg_u4{l2.x, l2.y, h2.x, h2.y};
}

template <int DT>
__device__ __forceinline__ f32x4 gg_mfma(gg_u4 a, gg_u4 b, f32x4 c) {
  return gg_mfma16<DT>(__builtin_bit_cast(uint4, a), __builtin_bit_cast(uint4, b), c);
}

// This wave's LDS reads are done, and its vector-memory operations but the last N.
template <int N>
__device__ __forceinline__ void gg_wait() {
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
}

template <int DT>
__device__ __forceinline__ uint32_t gg_pack2(float a, float b) {  // round to nearest even
  if constexpr (DT == kBF16) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, v2{(__bf16)a, (__bf16)b});
  } else {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, v2{(_Float16)a, (_Float16)b});
  }
}

// Order of an mt x nt grid of tiles.  Workgroups are dealt to the 8 XCDs in
// turn, 32 CUs each, so 256 run at once: 32 consecutive positions are one XCD's
// share of that (4 x 8 tiles: 12 operand panels into its L2 instead of 64), and
// 8 such shares lie together (16 x 16 tiles), so panels that several XCDs read
// come out of the last-level cache.
__device__ __forceinline__ int gg_pos(int b, int all) {
  const int x = b & 7, j = b >> 3, round = j >> 5, in = j & 31;
  const int left = all - 256 * round;
  if (left >= 256) return 256 * round + 32 * x + in;
  const int share = (left + 7) >> 3;  // the last round: as even as can be
  const int pos = share * x + in;
  return in < share && pos < left ? 256 * round + pos : -1;
}
__device__ __forceinline__ void gg_order(int pos, int mt, int nt, int& mi, int& ni) {
  const int strip = pos / (16 * nt);
  int r = pos - strip * 16 * nt;
  const int h = mt - 16 * strip < 16 ? mt - 16 * strip : 16;
  const int nb = r / (8 * h), wd = nt - 8 * nb < 8 ? nt - 8 * nb : 8;
  r -= nb * 8 * h;
  const int ms = r / (4 * wd), hm = h - 4 * ms < 4 ? h - 4 * ms : 4;
  r -= ms * 4 * wd;
  ni = r / hm;
  mi = 16 * strip + 4 * ms + (r - ni * hm);
  ni += 8 * nb;
}

// BM x BN tile, WM x WN waves.
template <int DT, int OP, int BM, int BN, int WM, int WN, bool GATHER>
__global__ __launch_bounds__(64 * WM * WN, WM * WN / 4) void grouped_fast_k(GroupedArgs a, int mt_max, int nt) {
  constexpr int W = WM * WN, XF = BM / WM / 16, YF = BN / WN / 16;
  constexpr bool TA = OP == kWgrad, TB = OP != kLinear;
  // units of 256 rows x 64: A of step t, B of step t, A of step t + 1, ...
  static_assert(BM == BN, "one unit size");
  constexpr uint32_t kUnit = BM * 128, kUnits = 5;
  __shared__ __attribute__((aligned(1024))) char lds[kUnits * kUnit];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rr = lane >> 3, p = lane & 7;
  const char* A = static_cast<const char*>(a.a);
  const char* B = static_cast<const char*>(a.b);
  const int cols = OP == kLinear ? a.N : a.K;

  // ---- which tile ----
  int e, mrows;           // expert (-1: rows to zero), rows of this tile
  int64_t m0, red0 = 0;   // first output row; first reduction row (wgrad)
  int red;                // reduction length
  int n0;
  if constexpr (OP == kWgrad) {
    const int per = mt_max * nt, pos = gg_pos(blockIdx.x, per * a.E);
    if (pos < 0) return;
    e = pos / per;
    int mi, ni;
    gg_order(pos - e * per, mt_max, nt, mi, ni);
    m0 = (int64_t)mi * BM;
    n0 = ni * BN;
    mrows = (int)(a.N - m0 < BM ? a.N - m0 : BM);
    red0 = __builtin_amdgcn_readfirstlane((int)gg_clamp(a.offsets[e], 0, a.S));
    red = __builtin_amdgcn_readfirstlane((int)(gg_clamp(a.offsets[e + 1], red0, a.S) - red0));
  } else {
    int ni = 0;
    const GgTile t = gg_find(a.offsets, a.E, a.S, BM, a.zero_rest, [&](int mts) {
      const int pos = gg_pos(blockIdx.x, mts * nt);
      if (pos < 0) return -1;
      int mi;
      gg_order(pos, mts, nt, mi, ni);
      return mi;
    });
    if (t.e == -2) return;
    n0 = ni * BN;
    e = __builtin_amdgcn_readfirstlane(t.e);
    m0 = __builtin_amdgcn_readfirstlane((int)t.s0);
    mrows = __builtin_amdgcn_readfirstlane((int)(t.s1 - t.s0));
    red = e < 0 ? 0 : (OP == kLinear ? a.K : a.N);
  }
  const int ncols = cols - n0 < BN ? cols - n0 : BN;

  // ---- operand streams ----
  GgOperand<BM, W, TA> oa;
  GgOperand<BN, W, TB, GATHER> ob;
  if constexpr (!TA) {
    oa.c8 = 8 * (p ^ gg_swz(8 * w));
    const bool gather = OP == kLinear && a.rows;
    oa.base = gather ? A : A + m0 * a.lda * 2;
    oa.bytes = gather ? ((a.T - 1) * a.lda + a.K) * 2 : ((int64_t)(mrows - 1) * a.lda + red) * 2;
#pragma unroll
    for (int j = 0; j < oa.kPieces; ++j) {
      const int r = 64 * (W * j / 8) + (w + W * j % 8) + 8 * rr, c = oa.c8 ^ (8 * (W * j % 8));
      int64_t row = r;
      bool ok = r < mrows;
      if (gather) {
        row = ok && e >= 0 ? a.rows[m0 + r] : 0;
        ok = ok && row >= 0 && row < a.T;
      }
      oa.vo[j] = ok ? (uint32_t)((row * a.lda + c) * 2) : kGgOob;
    }
  } else {
    oa.base = A + (red0 * a.lda + m0) * 2;
    oa.bytes = ((int64_t)(red - 1) * a.lda + mrows) * 2;
    oa.step = 64 * a.lda * 2;
#pragma unroll
    for (int j = 0; j < oa.kPieces; ++j) {
      const int r = (w + W * j % 8) + 8 * rr, c = 64 * (W * j / 8) + 8 * (p ^ gg_swz_tr(8 * w + rr));
      oa.vo[j] = c < mrows ? (uint32_t)((r * a.lda + c) * 2) : kGgOob;
    }
  }
  if constexpr (!TB) {
    ob.c8 = 8 * (p ^ gg_swz(8 * w));
    ob.base = B + ((int64_t)e * a.strb + (int64_t)n0 * a.ldb) * 2;
    ob.bytes = ((int64_t)(ncols - 1) * a.ldb + red) * 2;
#pragma unroll
    for (int j = 0; j < ob.kPieces; ++j) {
      const int r = 64 * (W * j / 8) + (w + W * j % 8) + 8 * rr, c = ob.c8 ^ (8 * (W * j % 8));
      ob.vo[j] = r < ncols ? (uint32_t)((r * a.ldb + c) * 2) : kGgOob;
    }
  } else {
    ob.base = OP == kDgrad ? B + ((int64_t)e * a.strb + n0) * 2 : B + ((GATHER ? 0 : red0 * a.ldb) + n0) * 2;
    ob.bytes = ((GATHER ? a.T - 1 : (int64_t)(red - 1)) * a.ldb + ncols) * 2;
    ob.step = 64 * a.ldb * 2;
    if constexpr (GATHER) {
      const int64_t ip = gg_uni(reinterpret_cast<int64_t>(a.rows + red0));
      ob.irs = gg_i4{(int)ip, (int)(ip >> 32) & 0xffff, 4 * red, 0x00020000};
      ob.iat = 4 * w;
      ob.ld2 = (uint32_t)a.ldb * 2;
      ob.rows = (uint32_t)a.T;
      ob.rr = rr;
      ob.k = w + 8 * rr;
    }
#pragma unroll
    for (int j = 0; j < ob.kPieces; ++j) {
      const int r = GATHER ? 0 : (w + W * j % 8) + 8 * rr, c = 64 * (W * j / 8) + 8 * (p ^ gg_swz_tr(8 * w + rr));
      ob.vo[j] = c < ncols ? (uint32_t)((r * a.ldb + c) * 2) : kGgOob;
    }
  }

  oa.base = gg_uni(oa.base);
  oa.bytes = gg_uni(oa.bytes);
  ob.base = gg_uni(ob.base);
  ob.bytes = gg_uni(ob.bytes);
  red = __builtin_amdgcn_readfirstlane(red);
  f32x4 acc[XF][YF];
#pragma unroll
  for (int x = 0; x < XF; ++x)
#pragma unroll
    for (int y = 0; y < YF; ++y) acc[x][y] = {0.f, 0.f, 0.f, 0.f};
  const int wm = (w / WN) * (BM / WM), wn = (w % WN) * (BN / WN);

  // A step has two halves of 32 deep.  A half's MFMAs run on fragments in
  // registers while the next half's are read from LDS and 32 KiB of a later step
  // arrive (first half: A of step t + 2, second: B), all spread over the half so
  // that nothing queues: LDS-DMA moves 52 B/clk a CU, half of what the step takes.
  // One barrier a step, between its halves: everybody has read all of step t, so
  // its units may be filled, and step t + 1 is in LDS.
  static_assert(W == 8 || W == 4, "piece maps");
  const int steps = (red + 63) / 64;
  constexpr int kPA = GgOperand<BM, W, TA>::kPieces, kPB = GgOperand<BN, W, TB, GATHER>::kPieces;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(gg_lptr)lds;
  asm volatile("" ::"v"(lds0) : "memory");
  GgReader<TA> ra;
  GgReader<TB> rb;
  ra.init(wm, lane);
  rb.init(wn, lane);
  const uint32_t dma0 = lds0 + w * 1024;
  gg_u4 fa[2][XF], fb[2][YF];
  const bool sums = OP == kWgrad && a.db && n0 == 0;
  constexpr uint32_t kOnes = DT == kBF16 ? 0x3f803f80u : 0x3c003c00u;
  const gg_u4 ones = {kOnes, kOnes, kOnes, kOnes};
  f32x4 accs[XF / WN > 0 ? XF / WN : 1];
#pragma unroll
  for (int u = 0; u < XF / WN; ++u) accs[u] = {0.f, 0.f, 0.f, 0.f};
  auto turn = [&](uint32_t u) {  // unit offset, wrapped
    const uint32_t v = u - kUnits * kUnit;
    return u < v ? u : v;
  };
  auto sync = [&]() {
    asm volatile("" ::: "memory");
    gg_wait<kPA>();  // all but the newest unit
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // MFMAs on (ac, bc); read half h of images (ia, ib) into (an, bn)
  auto half = [&](auto& op, uint32_t dst, int h, uint32_t ia, uint32_t ib, gg_u4 (&ac)[XF], gg_u4 (&bc)[YF], gg_u4 (&an)[XF],
                  gg_u4 (&bn)[YF], int left) {
    constexpr int kR = XF + YF, kOver = XF - 2;
    if constexpr (GATHER) {  // before this half's LDS reads: the scalar loads share their counter
      if constexpr (std::is_same_v<std::decay_t<decltype(op)>, GgOperand<BN, W, TB, true>>) op.advance(left);
    }
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      if (x == 1) {
        if constexpr (!GATHER || !std::is_same_v<std::decay_t<decltype(op)>, GgOperand<BN, W, TB, true>>) op.advance(left);
      }
#pragma unroll
      for (int q = 0; q < kR; ++q)
        if (q * kOver / kR == x) {
          if (q < YF) bn[q] = gg_frag<TB>(rb, ib, h, q);
          else an[q - YF] = gg_frag<TA>(ra, ia, h, q - YF);
        }
#pragma unroll
      for (int j = 0; j < kPA; ++j)  // all after next()
        if (1 + j * (XF - 1) / kPA == x) op.issue(dst, j);
#pragma unroll
      for (int y = 0; y < YF; ++y) acc[x][y] = gg_mfma<DT>(bc[y], ac[x], acc[x][y]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (OP == kWgrad) {
      if (sums) {  // column sums of dz: a product with ones, each wave of a row its part
#pragma unroll
        for (int c = 0; c < WN; ++c)
          if (w % WN == c) {
#pragma unroll
            for (int u = 0; u < XF / WN; ++u) accs[u] = gg_mfma<DT>(ones, ac[XF / WN * c + u], accs[u]);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  static_assert(kPA == kPB, "one count for both operands");
  if (steps > 0) {
    oa.first();
    ob.first();
    if (red < 64) oa.tail(red);
    if constexpr (GATHER) {
      ob.fetch_ids();
      ob.take_ids(red);
    } else if (red < 64) {
      ob.tail(red);
    }
#pragma unroll
    for (int j = 0; j < kPA; ++j) oa.issue(dma0, j);
#pragma unroll
    for (int j = 0; j < kPB; ++j) ob.issue(dma0 + kUnit, j);
    oa.advance(red - 64);
    ob.advance(red - 64);
#pragma unroll
    for (int j = 0; j < kPA; ++j) oa.issue(dma0 + 2 * kUnit, j);
#pragma unroll
    for (int j = 0; j < kPB; ++j) ob.issue(dma0 + 3 * kUnit, j);
    asm volatile("" ::: "memory");
    gg_wait<kPA + kPB>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int y = 0; y < YF; ++y) fb[0][y] = gg_frag<TB>(rb, lds0 + kUnit, 0, y);
#pragma unroll
    for (int x = 0; x < XF; ++x) fa[0][x] = gg_frag<TA>(ra, lds0, 0, x);
    uint32_t ua = 0;
    for (int t = 0; t < steps; ++t) {
      const int left = red - 64 * (t + 2);
      const uint32_t ub = turn(ua + kUnit), va = turn(ua + 2 * kUnit), vb = turn(va + kUnit), fr = turn(vb + kUnit);
      half(oa, dma0 + fr, 1, lds0 + ua, lds0 + ub, fa[0], fb[0], fa[1], fb[1], left);
      sync();
      half(ob, dma0 + ua, 0, lds0 + va, lds0 + vb, fa[1], fb[1], fa[0], fb[0], left);
      ua = va;
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // no LDS-DMA outlives the workgroup
  }

  // ---- epilogue: lane (i, g) holds columns 4 g .. 4 g + 3 of row i of every 16 x 16 tile ----
  const int i = lane & 15, g = lane >> 4;
  if constexpr (OP == kWgrad) {
    float* out = static_cast<float*>(a.out) + (int64_t)e * a.stro;
    if (sums && g == 0) {
#pragma unroll
      for (int u = 0; u < XF / WN; ++u) {
        const int m = wm + 16 * (XF / WN * (w % WN) + u) + i;
        if (m < mrows) a.db[(int64_t)e * a.N + m0 + m] = accs[u][0];
      }
    }
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      const int m = wm + 16 * x + i;
      if (m >= mrows) continue;
      float* o = out + (m0 + m) * a.ldo + n0;
#pragma unroll
      for (int y = 0; y < YF; ++y) {
        const int n = wn + 16 * y + 4 * g;
        if (n < ncols) *reinterpret_cast<f32x4*>(o + n) = acc[x][y];
      }
    }
  } else {
    if constexpr (OP == kLinear) {
      if (e >= 0 && a.bias) {
#pragma unroll
        for (int y = 0; y < YF; ++y) {
          const int n = wn + 16 * y + 4 * g;
          f32x4 b = {0.f, 0.f, 0.f, 0.f};
          if (n < ncols) {
            const float* bp = a.bias + (int64_t)e * a.ldbias + n0 + n;
            b = f32x4{bp[0], bp[1], bp[2], bp[3]};
          }
#pragma unroll
          for (int x = 0; x < XF; ++x) acc[x][y] += b;
        }
      }
      if (a.relu) {
#pragma unroll
        for (int x = 0; x < XF; ++x)
#pragma unroll
          for (int y = 0; y < YF; ++y)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[x][y][q] = acc[x][y][q] < 0.f ? 0.f : acc[x][y][q];
      }
    }
    uint16_t* out = static_cast<uint16_t*>(a.out);
    const uint16_t* mk = OP == kDgrad && e >= 0 ? static_cast<const uint16_t*>(a.mask) : nullptr;
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      const int m = wm + 16 * x + i;
#pragma unroll
      for (int y = 0; y < YF; y += 2) {
        // two neighbouring tiles: lanes of even g take the first, of odd g the
        // second, 8 columns each
        uint32_t u0 = gg_pack2<DT>(acc[x][y][0], acc[x][y][1]), u1 = gg_pack2<DT>(acc[x][y][2], acc[x][y][3]);
        uint32_t v0 = gg_pack2<DT>(acc[x][y + 1][0], acc[x][y + 1][1]);
        uint32_t v1 = gg_pack2<DT>(acc[x][y + 1][2], acc[x][y + 1][3]);
        const auto s0 = __builtin_amdgcn_permlane16_swap(u0, v0, false, false);
        const auto s1 = __builtin_amdgcn_permlane16_swap(u1, v1, false, false);
        gg_u4 o = {s0[0], s1[0], s0[1], s1[1]};
        const int n = wn + 16 * (y + (g & 1)) + 8 * (g >> 1);
        if (m < mrows && n < ncols) {
          if (mk) {
            const gg_u4 k = *reinterpret_cast<const gg_u4*>(mk + (m0 + m) * a.ldmask + n0 + n);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t lo = gg_f<DT>((uint16_t)k[q]) > 0.f ? 0x0000ffffu : 0u;
              const uint32_t hi = gg_f<DT>((uint16_t)(k[q] >> 16)) > 0.f ? 0xffff0000u : 0u;
              o[q] &= lo | hi;
            }
          }
          *reinterpret_cast<gg_u4*>(out + (m0 + m) * a.ldo + n0 + n) = o;
        }
      }
    }
  }
}

bool gg_al(const void* p, int64_t ld, int64_t need) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && ld >= need;
}
// Whole 16-B words everywhere, rows that do not overlap, and offsets of 32 bits
// from each stream's base.
bool fast_ok(GroupedOp op, const GroupedArgs& a) {
  if (a.K % 8 || a.N % 8) return false;
  if (!gg_al(a.a, a.lda, op == kLinear ? a.K : a.N) || !gg_al(a.b, a.ldb, a.K)) return false;
  if (op != kWgrad && a.E > 1 && a.strb % 8) return false;
  if (a.lda > 0x7fffff || a.ldb > 0x7fffff) return false;
  if (op == kLinear && a.rows && (a.T * a.lda + a.K) * 2 > kGgSpan) return false;
  if (op == kWgrad)
    return (!a.rows || (a.T * a.ldb + a.K) * 2 <= kGgSpan) && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 &&
           a.ldo % 4 == 0 && (a.E <= 1 || a.stro % 4 == 0);
  if (!gg_al(a.out, a.ldo, 0)) return false;
  return op != kDgrad || !a.mask || gg_al(a.mask, a.ldmask, 0);
}

template <int DT, int OP, int BM, int BN, int WM, int WN, bool GATHER = false>
hipError_t launch_fast(const GroupedArgs& a, hipStream_t s) {
  const int cols = OP == kLinear ? a.N : a.K;
  const int nt = (cols + BN - 1) / BN;
  int64_t mt;
  if (OP == kWgrad) mt = (a.N + BM - 1) / BM;
  else {
    mt = (a.S + BM - 1) / BM + a.E + (a.zero_rest ? 2 : 0);
    mt = mt < a.S ? mt : a.S;
  }
  const int64_t tiles = mt * nt * (OP == kWgrad ? a.E : 1), blocks = (tiles + 7) / 8 * 8;  // the XCDs in turn
  if (blocks > 0x7fffff00LL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((grouped_fast_k<DT, OP, BM, BN, WM, WN, GATHER>), dim3((uint32_t)blocks), dim3(64 * WM * WN), 0, s, a,
                     (int)mt, nt);
  return hipGetLastError();
}
template <int DT>
hipError_t launch_fast_op(GroupedOp op, const GroupedArgs& a, hipStream_t s) {
  switch (op) {
    case kLinear: return launch_fast<DT, kLinear, 256, 256, 2, 4>(a, s);
    case kDgrad: return launch_fast<DT, kDgrad, 256, 256, 2, 4>(a, s);
    default:
      return a.rows ? launch_fast<DT, kWgrad, 256, 256, 2, 4, true>(a, s) : launch_fast<DT, kWgrad, 256, 256, 2, 4>(a, s);
  }
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
  if (fast_ok(op, a)) return a.dtype == kBF16 ? launch_fast_op<kBF16>(op, a, s) : launch_fast_op<kF16>(op, a, s);
  return a.dtype == kBF16 ? launch_any<kBF16>(op, a, s) : launch_any<kF16>(op, a, s);
}

}  // namespace dsml
