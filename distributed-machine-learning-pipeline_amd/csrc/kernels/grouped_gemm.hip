// Matrix products grouped by expert: group e owns the rows [off[e], off[e + 1])
// of the slot axis, of any length, zero and one included.
//
//   linear : y[s][n]   = act(sum_k x[row(s)][k] w[e][n][k] + b[e][n])
//   dgrad  : dx[s][k]  = (sum_n dz[s][n] w[e][n][k]) * (mask[s][k] > 0)
//   wgrad  : dw[e][n][k] = sum_s dz[s][n] x[row(s)][k]   (fp32),  db[e][n] = sum_s dz[s][n]
//
// Three kernels: grouped_fast_k (operands of whole 16-B words, by LDS-DMA; 256 x 256
// and 128 x 128 tiles), grouped_skinny_k (few rows: the waves of a workgroup share
// the reduction) and grouped_any_k (any width, stride and alignment).
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

struct GgTile {
  int e;          // expert, -1: rows to zero, -2: nothing
  int64_t s0, s1; // rows of this tile
};

__device__ __forceinline__ int64_t gg_clamp(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Inclusive sums over the lanes of a wave: within rows of 16, then across them.
__device__ __forceinline__ int gg_scan64(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31 into rows 2 and 3
  return v;
}

constexpr int kGgZero = 128;  // workgroups that clear rows of no group

// The groups, cut into tiles on the GPU: count(rows) is what a group of that
// many rows holds of some kind of tile.  One wave scan per 64 experts, done by
// every wave for itself: no LDS, no barrier.
struct GgGroups {
  const int32_t* off;
  int E;
  int64_t S;
  int a0, b0;  // the first 64 groups', in the lanes

  __device__ __forceinline__ GgGroups(const int32_t* o, int e, int64_t s) : off(o), E(e), S(s) { bounds(0, a0, b0); }
  __device__ __forceinline__ void bounds(int e0, int& a, int& b) const {
    const int e = e0 + (threadIdx.x & 63);
    a = b = 0;
    if (e < E) {
      a = (int)gg_clamp(off[e], 0, S);
      b = (int)gg_clamp(off[e + 1], a, S);
    }
  }
  template <class Count>
  __device__ __forceinline__ void scan(int e0, Count count, int& a, int& b, int& n, int& inc) const {
    if (e0 == 0) {
      a = a0;
      b = b0;
    } else {
      bounds(e0, a, b);
    }
    n = count((int64_t)b - a);
    inc = gg_scan64(n);
  }
  // All tiles, `most` at most: more only if the offsets are no plan.
  template <class Count>
  __device__ __forceinline__ int total(Count count, int64_t most) const {
    int64_t t = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
      int a, b, n, inc;
      scan(e0, count, a, b, n, inc);
      t += __builtin_amdgcn_readlane(inc, 63);
    }
    return (int)(t < most ? t : most);
  }
  // The group that holds tile t, its rows and the tile's number in it.
  template <class Count>
  __device__ __forceinline__ bool find(int t, Count count, int& e, int64_t& lo, int64_t& hi, int& in) const {
    for (int e0 = 0; e0 < E; e0 += 64) {
      int a, b, n, inc;
      scan(e0, count, a, b, n, inc);
      const int tot = __builtin_amdgcn_readlane(inc, 63);
      if (t < tot) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(inc > t)) - 1);
        in = t - (__builtin_amdgcn_readlane(inc, l) - __builtin_amdgcn_readlane(n, l));
        lo = __builtin_amdgcn_readlane(a, l);
        hi = __builtin_amdgcn_readlane(b, l);
        e = e0 + l;
        return true;
      }
      t -= tot;
    }
    return false;
  }
  // Tiles of BM rows that lie in no group: before the first, behind the last.
  __device__ __forceinline__ void rest(int& head, int& tail, int BM) const {
    const int64_t h = gg_clamp(off[0], 0, S), t = gg_clamp(off[E], h, S);
    head = (int)((h + BM - 1) / BM);
    tail = (int)((S - t + BM - 1) / BM);
  }
  __device__ __forceinline__ bool find_rest(int t, int BM, int64_t& lo, int64_t& hi) const {
    const int64_t h = gg_clamp(off[0], 0, S), u = gg_clamp(off[E], h, S), hn = (h + BM - 1) / BM;
    lo = t < hn ? (int64_t)t * BM : u + (t - hn) * BM;
    hi = t < hn ? h : S;
    hi = lo + BM < hi ? lo + BM : hi;
    return lo < hi;
  }
  // All of them at once, by kGgZero workgroups of 256 (whole 16-B words): a row
  // tile each would be S / 128 column strips of workgroups that mostly end at
  // once (27 us at 32768 rows of 4096 columns).
  __device__ __forceinline__ void zero_rest(const GroupedArgs& a, int cols, int part) const {
    const int64_t h = gg_clamp(off[0], 0, S), n = h + S - gg_clamp(off[E], h, S);
    const int words = cols / 8, step = kGgZero * 256 / 64, lane = threadIdx.x & 63;
    for (int64_t r = part * 4 + (threadIdx.x >> 6); r < n; r += step) {
      uint16_t* o = static_cast<uint16_t*>(a.out) + (r < h ? r : S - n + r) * a.ldo;
      for (int c = lane; c < words; c += 64) reinterpret_cast<uint4*>(o)[c] = make_uint4(0, 0, 0, 0);
    }
  }
};

// Row tile of BM rows number pick(how many there are): the experts' tiles, then
// (zero_rest) those of the rows in no group.
template <class Pick>
__device__ __forceinline__ GgTile gg_find(const int32_t* off, int E, int64_t S, int BM, bool zero_rest, Pick pick) {
  const GgGroups gr(off, E, S);
  auto count = [BM](int64_t rows) { return (int)((rows + BM - 1) / BM); };
  const int total = gr.total(count, S / BM + E);
  int head = 0, tail = 0;
  if (zero_rest) gr.rest(head, tail, BM);
  GgTile t{-2, 0, 0};
  const int mt = pick(total + head + tail);
  if (mt < 0) return t;
  if (mt < total) {
    int64_t lo, hi;
    int in;
    if (!gr.find(mt, count, t.e, lo, hi, in)) return t;
    t.s0 = lo + (int64_t)in * BM;
    t.s1 = t.s0 + BM < hi ? t.s0 + BM : hi;
  } else if (mt - total < head + tail && gr.find_rest(mt - total, BM, t.s0, t.s1)) {
    t.e = -1;
  }
  return t;
}

// ---------------------------------------------------------------------------
// Fast path: widths and row strides of whole 16-B words.  256 x 256 output
// tile, 64-deep steps, 8 waves of 128 x 64 (16x16x32 MFMA), operands by LDS-DMA
// into a ring of five 32-KiB units: all 160 KiB of LDS, one workgroup a CU.  The
// 128 x 128 tile (4 waves of 64 x 64, five units of 16 KiB, two workgroups a CU)
// has the same loop.
//
// bf16, 8 experts: 32768 rows x 4096 x 4096 851 us (1292 TFLOP/s; 1535 for a plain
// library product of that size), the input gradient of 16384 rows 493 (1115), the
// weight gradient 493 (1116); up to 4 % more on some cards.  With random data the
// first runs at the power limit (1.73 GHz, matrix units 64 % busy; 788 us of a step
// count alike on zeros), the gradients do not (2.04 and 2.09 GHz, 56 and 47 %);
// outside of the products a tile costs about 8 us: its stores, its search, its
// first loads.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void* gg_lptr;
typedef short gg_i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) gg_i16x4* gg_lv4;
typedef uint32_t gg_u4 __attribute__((ext_vector_type(4)));

// Past every buffer: reads 0, also behind a scalar offset that is past the end by
// itself (sizes and offsets are multiples of 16, so "size - offset" never wraps
// into the last 16 bytes).
constexpr uint32_t kGgOob = 0xfffffff0u;
constexpr int64_t kGgSpan = 0xffffff00LL;   // bytes a buffer descriptor may span
constexpr int64_t kGgIds = 1LL << 29;       // ids a scalar stream can't hold any more

__device__ __forceinline__ gg_u4 gg_desc(const char* base, int64_t bytes) {
  const int64_t b = reinterpret_cast<int64_t>(base);
  const int64_t n = bytes < 0 ? 0 : (bytes > kGgSpan ? kGgSpan : bytes);
  return gg_u4{(uint32_t)b, (uint32_t)((uint64_t)b >> 32) & 0xffffu, (uint32_t)n, 0x00020000u};
}
// 1 KiB straight into LDS at `lds`, 16 B a lane.  Opaque to the compiler, which
// would wait for every one in flight before any LDS read; arrival is waited for
// by count (gg_wait).
__device__ __forceinline__ void gg_dma(uint32_t lds, uint32_t vo, gg_u4 rs, uint32_t so) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(vo), "s"(rs), "s"(so)
               : "m0");
}
// A value every lane holds, in scalar registers.
__device__ __forceinline__ int64_t gg_uni(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ const char* gg_uni(const char* v) { return reinterpret_cast<const char*>(gg_uni((int64_t)v)); }
// LDS image of one 64-deep step of an operand, 1-KiB pieces of 8 rows x 128 B:
//   row-major   rows of 64 reduction elements; row r lies at 64 (r / 64) + 8 (r % 8) + r / 8 % 8
//   transposed  per 64 columns, 64 reduction rows of them; row r lies at 8 (r % 8) + r / 8
// so the 8 rows of one LDS-DMA instruction are 8 rows apart in memory: adjacent
// rows of some power-of-two strides (8 KiB among them) fall on one cache channel,
// 35 B/clk a CU instead of 52.  16-B chunks are XORed with a function of the LDS
// row, so fragment reads touch every bank once.
__device__ __forceinline__ int gg_swz(int pos) { return (pos >> 3) & 7; }
// Transposing reads take 32 lanes a turn, 8 reduction rows of 2 x 4 positions: with
// this swizzle they cover every bank once (wgrad of 16384 rows x 4096 x 4096, 8
// experts: 512 -> 507 us).
__device__ __forceinline__ int gg_swz_tr(int pos) { return 2 * ((pos >> 3) & 3); }

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
  static constexpr int kSets = 8 / WAVES;  // rows w + 8 rr, or those and w + 4 + 8 rr
  int id[kSets][8];
  uint32_t ld2, rows, rowoff[kSets];
  int k, rr;        // this lane's reduction row in a step: w + 8 rr

  __device__ __forceinline__ void fetch_ids() {
#pragma unroll
    for (int u = 0; u < kSets; ++u)
#pragma unroll
      for (int q = 0; q < 8; ++q) id[u][q] = gg_sload(irs, (int)(iat + 4 * WAVES * u + 32 * q), 0);
    iat += 256;
  }
  // Row offsets of the step whose ids were fetched (left: its reduction rows); fetches the next ids.
  __device__ __forceinline__ void take_ids(int left) {
#pragma unroll
    for (int u = 0; u < kSets; ++u) {
      int v = id[u][0];
#pragma unroll
      for (int q = 1; q < 8; ++q) {
        int t = id[u][q];
        asm("" : "+s"(t));  // a select, not an indexed array in scratch memory
        v = rr == q ? t : v;
      }
      rowoff[u] = (uint32_t)v < rows && k + WAVES * u < left ? (uint32_t)v * ld2 : kGgOob;
    }
    fetch_ids();
  }

  __device__ __forceinline__ void first() {
    rs = gg_desc(base, bytes);
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
  __device__ __forceinline__ void issue(uint32_t lds, int j) {
    uint32_t v = vo[j];
    if constexpr (GATHER) v = __builtin_elementwise_add_sat(v, rowoff[j % kSets]);  // kGgOob stays past the end
    gg_dma(lds + WAVES * j * 1024, v, rs, so);
  }
};

// Fragments of 16 rows (columns when TR): lane (i, g) holds reduction elements
// 32 h + 8 g .. + 7 of row i.  A wave's x-th is the image's block X0 + SKIP x of
// 16 rows (SKIP 1: X0 a multiple of 4; SKIP 2: X0 0 or 1).  Lane part of the
// address here, the rest is constant.
template <bool TR, int SKIP>
struct GgReader {
  static_assert(SKIP == 1 || SKIP == 2, "block maps");
  uint32_t p[TR ? 4 / SKIP : 2];
  __device__ __forceinline__ void init(int X0, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const int at = SKIP == 1 ? (X0 >> 2) * 8192 : 0, x0 = SKIP == 1 ? 0 : X0;
    if constexpr (!TR) {
      const int pos = 8 * (i & 7) + 2 * x0 + (i >> 3);
#pragma unroll
      for (int h = 0; h < 2; ++h) p[h] = at + pos * 128 + 16 * ((4 * h + g) ^ gg_swz(pos));
    } else {
      const int q = i >> 2, pp = i & 3, pos = 8 * q + g;  // + 4 h, + 32 for elements 4 .. 7
#pragma unroll
      for (int x = 0; x < 4 / SKIP; ++x)
        p[x] = at + pos * 128 + 16 * ((2 * (x0 + SKIP * x) + (pp >> 1)) ^ gg_swz_tr(pos)) + 8 * (pp & 1);
    }
  }
};
typedef __attribute__((address_space(3))) const gg_u4* gg_lu4;
template <bool TR, int SKIP>
__device__ __forceinline__ gg_u4 gg_frag(const GgReader<TR, SKIP>& rd, uint32_t img, int h, int x) {
  constexpr int kIn = 4 / SKIP;  // blocks of one 64-row group (64-column image)
  if constexpr (!TR) return *(gg_lu4)(uintptr_t)(rd.p[h] + img + (x / kIn) * 8192 + (x % kIn) * 256 * SKIP);
  const uint32_t a = rd.p[x % kIn] + img + (x / kIn) * 8192 + h * 512;
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

// Which tiles run as 256 x 256 and which as 128 x 128, from what is known on the
// GPU only: both kernels make the same choice.  A round of 256 x 256 tiles over
// the CUs takes as long as about 540 tiles of 128 x 128 (which move twice the
// bytes a product: 1250 against 700 TFLOP/s), and a launch of few of those as long
// as 190; a round that is not full costs a whole one.  So the last round, and the
// groups' last rows that fill no 256, go where they are done sooner.
constexpr int kGgCus = 256, kGgRound = 540, kGgSmallMin = 190, kGgGap = 1300;
// (a second launch costs about 4 us: kGgGap tiles at one step each.  Measured with
// the plan against whole rounds of 256 x 256: 4096 rows, 8 experts of 4096 x 4096,
// 183 us against 224; 5003 rows, 16 experts of 1000 x 784, 20.5 against 23.8)
__host__ __device__ __forceinline__ int64_t gg_small_cost(int64_t tiles, int steps) {
  return tiles == 0 ? 0 : (tiles > kGgSmallMin ? tiles : kGgSmallMin) + kGgGap / (steps > 0 ? steps : 1);
}
struct GgPlan {
  int whole, mt;   // row tiles of 256: full ones, all of this plan (the others have fewer rows)
  int big;         // tiles of the mt x ntb grid run as 256 x 256, in gg_order; the rest in quarters
  int halves;      // 128-row tiles of the rows that fill no 256, when the plan leaves those out
};
__device__ __forceinline__ GgPlan gg_plan(const GgGroups& gr, int ntb, int nts, int steps, bool only_small) {
  const int f = gr.total([](int64_t r) { return (int)(r / 256); }, gr.S / 256);
  const int p = gr.total([](int64_t r) { return r % 256 ? 1 : 0; }, gr.E);
  const int h = gr.total([](int64_t r) { return (int)((r % 256 + 127) / 128); }, 2 * (int64_t)gr.E);
  GgPlan best{f, f, 0, h};
  if (only_small) return best;
  int64_t least = -1;
#pragma unroll
  for (int o = 0; o < 4; ++o) {
    const bool part = o & 1, up = !(o & 2);
    const int mt = part ? f + p : f;
    const int64_t q = (int64_t)mt * ntb, last = q % kGgCus, whole = q - last;
    const int64_t extra = part ? 0 : (int64_t)h * nts;
    const int64_t lp = part ? (last < (int64_t)p * ntb ? last : (int64_t)p * ntb) : 0;  // not full: these come last
    const int64_t tail = 4 * (last - lp) + (lp ? 2 * lp * h / p : 0);
    const int64_t cost = up ? (q + kGgCus - 1) / kGgCus * kGgRound + gg_small_cost(extra, steps)
                            : q / kGgCus * kGgRound + gg_small_cost(tail + extra, steps);
    if (least < 0 || cost < least) {
      least = cost;
      best.mt = mt;
      best.big = (int)(up ? q : whole);
      best.halves = part ? 0 : h;
    }
  }
  return best;
}
// Rows of row tile mi of a plan's grid.
__device__ __forceinline__ bool gg_rows(const GgGroups& gr, const GgPlan& pl, int mi, int& e, int64_t& m0, int& rows) {
  int64_t lo, hi;
  int in;
  if (mi < pl.whole) {
    if (!gr.find(mi, [](int64_t r) { return (int)(r / 256); }, e, lo, hi, in)) return false;
    m0 = lo + 256 * in;
    rows = 256;
  } else {
    if (!gr.find(mi - pl.whole, [](int64_t r) { return r % 256 ? 1 : 0; }, e, lo, hi, in)) return false;
    rows = (int)((hi - lo) % 256);
    m0 = hi - rows;
  }
  return true;
}

// wgrad: the rows of group e, or (split) part `part` of them: whole 64-row steps,
// the first parts full.  A part's sums go to the workspace, [parts][E][N][K] and
// [parts][E][N].
__device__ __forceinline__ void gg_part(GroupedArgs& a, int e, int part, int64_t& red0, int& red) {
  const int64_t lo = gg_clamp(a.offsets[e], 0, a.S), hi = gg_clamp(a.offsets[e + 1], lo, a.S);
  red0 = lo;
  red = (int)(hi - lo);
  if (a.split > 1) {
    const int64_t rows = ((int64_t)red + 64 * a.split - 1) / (64 * a.split) * 64;
    red0 = lo + part * rows < hi ? lo + part * rows : hi;
    red = (int)(hi - red0 < rows ? hi - red0 : rows);
    a.stro = (int64_t)a.N * a.K;
    a.ldo = a.K;
    a.out = a.ws + part * a.E * a.stro;
    if (a.db) a.db = a.ws + a.split * a.E * a.stro + (int64_t)part * a.E * a.N;
  }
  red0 = __builtin_amdgcn_readfirstlane((int)red0);
  red = __builtin_amdgcn_readfirstlane(red);
}

// BM x BN tile, WM x WN waves.
template <int DT, int OP, int BM, int BN, int WM, int WN, bool GATHER>
__global__ __launch_bounds__(64 * WM * WN, 2) void grouped_fast_k(GroupedArgs a, int big) {
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
  int e, mrows;           // expert, rows of this tile
  int64_t m0, red0 = 0;   // first output row; first reduction row (wgrad)
  int red;                // reduction length
  int n0;
  // The grid in 256 x 256 tiles; the 128 x 128 kernel takes the last of them
  // (big <= tile, four workgroups each) and the rows that fill no 256.
  constexpr bool kSmall = BM == 128;
  const int ntb = (cols + 255) / 256;
  int sub_m = 0, sub_n = 0;  // kSmall: 128-row (column) half of the tile
  if constexpr (OP == kWgrad) {
    const int mtb = (a.N + 255) / 256, per = mtb * ntb;
    int pos, part = 0;
    if constexpr (kSmall) {
      const int tiles = 4 * (per * a.E - big);
      pos = gg_pos(blockIdx.x, tiles * a.split);
      if (pos < 0) return;
      part = pos / tiles;
      pos -= part * tiles;
      sub_m = (pos >> 1) & 1;
      sub_n = pos & 1;
      pos = big + (pos >> 2);
    } else {
      pos = gg_pos(blockIdx.x, big);
      if (pos < 0) return;
    }
    e = pos / per;
    int mi, ni;
    gg_order(pos - e * per, mtb, ntb, mi, ni);
    m0 = (int64_t)mi * 256 + 128 * sub_m;
    n0 = ni * 256 + 128 * sub_n;
    if (m0 >= a.N || n0 >= cols) return;
    mrows = (int)(a.N - m0 < BM ? a.N - m0 : BM);
    gg_part(a, e, part, red0, red);
  } else {
    const GgGroups gr(a.offsets, a.E, a.S);
    if (kSmall && a.zero_rest && blockIdx.x >= gridDim.x - kGgZero) {
      gr.zero_rest(a, cols, blockIdx.x - (gridDim.x - kGgZero));
      return;
    }
    const int nts = (cols + 127) / 128;
    const GgPlan pl = gg_plan(gr, ntb, nts, ((OP == kLinear ? a.K : a.N) + 63) / 64, big < 0);
    int mi, ni;
    if constexpr (!kSmall) {
      const int pos = gg_pos(blockIdx.x, pl.big);
      if (pos < 0) return;
      gg_order(pos, pl.mt, ntb, mi, ni);
      if (!gg_rows(gr, pl, mi, e, m0, mrows)) return;
      n0 = ni * 256;
    } else {
      const int quarters = 4 * (pl.mt * ntb - pl.big), mts = pl.halves;
      int pos = gg_pos(blockIdx.x, quarters + mts * nts);
      if (pos < 0) return;
      if (pos < quarters) {
        gg_order(pl.big + (pos >> 2), pl.mt, ntb, mi, ni);
        if (!gg_rows(gr, pl, mi, e, m0, mrows)) return;
        const int sub = 128 * ((pos >> 1) & 1);
        m0 += sub;
        mrows = mrows - sub < 128 ? mrows - sub : 128;
        n0 = 256 * ni + 128 * (pos & 1);
        if (mrows <= 0 || n0 >= cols) return;
      } else {
        pos -= quarters;  // strips of 8 row tiles
        const int strip = pos / (8 * nts), r = pos - strip * 8 * nts, h = mts - 8 * strip < 8 ? mts - 8 * strip : 8;
        ni = r / h;
        mi = 8 * strip + (r - ni * h);
        n0 = 128 * ni;
        int64_t lo, hi;
        int in;
        if (!gr.find(mi, [](int64_t x) { return (int)((x % 256 + 127) / 128); }, e, lo, hi, in)) return;
        m0 = lo + (hi - lo) / 256 * 256 + 128 * in;
        mrows = (int)(hi - m0 < 128 ? hi - m0 : 128);
      }
    }
    e = __builtin_amdgcn_readfirstlane(e);
    m0 = __builtin_amdgcn_readfirstlane((int)m0);
    n0 = __builtin_amdgcn_readfirstlane(n0);
    mrows = __builtin_amdgcn_readfirstlane(mrows);
    red = OP == kLinear ? a.K : a.N;
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
        row = ok ? a.rows[m0 + r] : 0;
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
  // wave (wr, wc): row blocks wr, wr + 2, ... of 16 (a tile that is not full keeps
  // both wave rows busy, and blocks without rows are skipped), columns 64 wc ..
  const int wr = w / WN, wc = w % WN, wn = wc * (BN / WN);
  const bool sums = OP == kWgrad && a.db && n0 == 0;  // every wave column sums a part of dz
  const int xn = wn < ncols || sums ? ((mrows + 15) / 16 - wr + 1) / 2 : 0;

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
  static_assert(WM == 2 && YF == 4, "block maps");
  GgReader<TA, 2> ra;
  GgReader<TB, 1> rb;
  ra.init(wr, lane);
  rb.init(YF * wc, lane);
  const uint32_t dma0 = lds0 + w * 1024;
  gg_u4 fa[2][XF], fb[2][YF];
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
  auto half = [&](auto full, auto& op, uint32_t dst, int h, uint32_t ia, uint32_t ib, gg_u4 (&ac)[XF], gg_u4 (&bc)[YF], gg_u4 (&an)[XF],
                  gg_u4 (&bn)[YF], int left) {
    if constexpr (GATHER) {  // before this half's LDS reads: the scalar loads share their counter
      if constexpr (std::is_same_v<std::decay_t<decltype(op)>, GgOperand<BN, W, TB, true>>) op.advance(left);
    }
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      if (x == 1) {
        if constexpr (!GATHER || !std::is_same_v<std::decay_t<decltype(op)>, GgOperand<BN, W, TB, true>>) op.advance(left);
      }
#pragma unroll
      for (int j = 0; j < kPA; ++j)  // all after advance()
        if (1 + j * (XF - 1) / kPA == x) op.issue(dst, j);
      if (decltype(full)::value || x < xn) {
        if (x == 0) {
#pragma unroll
          for (int y = 0; y < YF; ++y) bn[y] = gg_frag(rb, ib, h, y);
          an[0] = gg_frag(ra, ia, h, 0);
        }
        if (x + 1 < XF) an[x + 1] = gg_frag(ra, ia, h, x + 1);
#pragma unroll
        for (int y = 0; y < YF; ++y) acc[x][y] = gg_mfma<DT>(bc[y], ac[x], acc[x][y]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (OP == kWgrad) {
      if (sums) {  // column sums of dz: a product with ones, each wave of a row its part
#pragma unroll
        for (int c = 0; c < WN; ++c)
          if (wc == c) {
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
    for (int y = 0; y < YF; ++y) fb[0][y] = gg_frag(rb, lds0 + kUnit, 0, y);
#pragma unroll
    for (int x = 0; x < XF; ++x) fa[0][x] = gg_frag(ra, lds0, 0, x);
    auto run = [&](auto full) {
      uint32_t ua = 0;
      for (int t = 0; t < steps; ++t) {
        const int left = red - 64 * (t + 2);
        const uint32_t ub = turn(ua + kUnit), va = turn(ua + 2 * kUnit), vb = turn(va + kUnit), fr = turn(vb + kUnit);
        half(full, oa, dma0 + fr, 1, lds0 + ua, lds0 + ub, fa[0], fb[0], fa[1], fb[1], left);
        sync();
        half(full, ob, dma0 + ua, 0, lds0 + va, lds0 + vb, fa[1], fb[1], fa[0], fb[0], left);
        ua = va;
      }
    };
    if (!kSmall || xn == XF) run(std::true_type{});
    else run(std::false_type{});
    __builtin_amdgcn_s_waitcnt(0x0f70);  // no LDS-DMA outlives the workgroup
  }

  // ---- epilogue: lane (i, g) holds columns 4 g .. 4 g + 3 of row i of every 16 x 16 tile ----
  const int i = lane & 15, g = lane >> 4;
  if constexpr (OP == kWgrad) {
    float* out = static_cast<float*>(a.out) + (int64_t)e * a.stro;
    if (sums && g == 0) {
#pragma unroll
      for (int u = 0; u < XF / WN; ++u) {
        const int m = 16 * (2 * (XF / WN * wc + u) + wr) + i;
        if (m < mrows) a.db[(int64_t)e * a.N + m0 + m] = accs[u][0];
      }
    }
    const int64_t bytes = ((int64_t)(mrows - 1) * a.ldo + ncols) * 4;
    const char* base = gg_uni(reinterpret_cast<const char*>(out + m0 * a.ldo + n0));
    const auto od = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, (int)(uint32_t)gg_uni(bytes), 0x00020000);
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      const int m = 16 * (2 * x + wr) + i;
#pragma unroll
      for (int y = 0; y < YF; ++y) {
        const int n = wn + 16 * y + 4 * g;
        const uint32_t at = m < mrows && n < ncols ? ((uint32_t)m * (uint32_t)a.ldo + (uint32_t)n) * 4u : kGgOob;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(gg_i4, acc[x][y]), od, (int)at, 0, 0);
      }
    }
  } else {
    if constexpr (OP == kLinear) {
      if (a.bias) {
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
    // Through buffer descriptors, so that nothing stands under a condition: all mask
    // loads go out first, and no store is waited for (32768 rows of 4096, 8 experts, a
    // reduction of 64, with a mask: 145 us; under bounds checks 171).
    const auto desc = [&](const void* p, int64_t ld) {
      const int64_t bytes = ((int64_t)(mrows - 1) * ld + ncols) * 2;
      const char* q = gg_uni(static_cast<const char*>(p) + (m0 * ld + n0) * 2);
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(q), 0, (int)(uint32_t)gg_uni(bytes), 0x00020000);
    };
    const auto at = [&](int x, int y, int64_t ld) {  // lanes of even g the first of two tiles, of odd g the second
      const int m = 16 * (2 * x + wr) + i, n = wn + 16 * (y + (g & 1)) + 8 * (g >> 1);
      return (int)(m < mrows && n < ncols ? ((uint32_t)m * (uint32_t)ld + (uint32_t)n) * 2u : kGgOob);
    };
    const auto od = desc(a.out, a.ldo);
    gg_i4 keep[XF][YF / 2];
    const bool mask = OP == kDgrad && a.mask;
    if (mask) {
      const auto md = desc(a.mask, a.ldmask);
#pragma unroll
      for (int x = 0; x < XF; ++x)
#pragma unroll
        for (int y = 0; y < YF; y += 2)
          keep[x][y / 2] = __builtin_amdgcn_raw_buffer_load_b128(md, at(x, y, a.ldmask), 0, 0);
    } else {
#pragma unroll
      for (int x = 0; x < XF; ++x)
#pragma unroll
        for (int y = 0; y < YF / 2; ++y) keep[x][y] = {0, 0, 0, 0};
    }
#pragma unroll
    for (int x = 0; x < XF; ++x) {
#pragma unroll
      for (int y = 0; y < YF; y += 2) {
        uint32_t u0 = gg_pack2<DT>(acc[x][y][0], acc[x][y][1]), u1 = gg_pack2<DT>(acc[x][y][2], acc[x][y][3]);
        uint32_t v0 = gg_pack2<DT>(acc[x][y + 1][0], acc[x][y + 1][1]);
        uint32_t v1 = gg_pack2<DT>(acc[x][y + 1][2], acc[x][y + 1][3]);
        const auto s0 = __builtin_amdgcn_permlane16_swap(u0, v0, false, false);
        const auto s1 = __builtin_amdgcn_permlane16_swap(u1, v1, false, false);
        gg_u4 o = {s0[0], s1[0], s0[1], s1[1]};
        if (mask) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t k = (uint32_t)keep[x][y / 2][q];
            const uint32_t lo = gg_f<DT>((uint16_t)k) > 0.f ? 0x0000ffffu : 0u;
            const uint32_t hi = gg_f<DT>((uint16_t)(k >> 16)) > 0.f ? 0xffff0000u : 0u;
            o[q] &= lo | hi;
          }
        }
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(gg_i4, o), od, at(x, y, a.ldo), 0, 0);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Few rows an expert (single tokens): the weights are read once and that is
// the time.  A workgroup owns 64 output columns of up to 16 MX rows; its 4 waves
// take the 64-deep steps in turn, each with a ring of its own (2 slots of 64
// weight rows and 16 MX operand rows), so the loop has no barrier and 4 x 2 slots
// a workgroup are in flight, of two workgroups a CU (MX 1: 80 KiB of LDS) or one
// (MX 2: 96 KiB).  The waves' partial tiles are
// summed in wave order through LDS.  16 rows, 8 experts of 4096 x 4096: 54 us with
// cold weights (4.9 TB/s), 92 with 128 x 128 tiles.
// ---------------------------------------------------------------------------
template <int DT, int OP, int MX>
__global__ __launch_bounds__(256, 2) void grouped_skinny_k(GroupedArgs a, int nt) {
  constexpr int BM = 16 * MX, BN = 64;
  constexpr bool TB = OP == kDgrad;
  constexpr int kW = 8192, kX = BM * 128, kStage = kW + kX, kPX = BM / 8;  // bytes and pieces of a stage
  __shared__ __attribute__((aligned(1024))) char lds[4 * 2 * kStage];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rr = lane >> 3, p = lane & 7, i = lane & 15, g = lane >> 4;
  const int cols = OP == kLinear ? a.N : a.K;
  // An XCD takes every 8th column tile, all its row tiles together; with fewer than
  // 8 columns an eighth of the tiles.  (An eighth each with more: neighbouring rows
  // of the weights are no longer read at once, 16 rows, 8 experts of 4096 x 4096: 54 us become 65.)
  int ni = 0;
  const GgTile t = gg_find(a.offsets, a.E, a.S, BM, a.zero_rest, [&](int mts) {
    const int x = blockIdx.x & 7, in = blockIdx.x >> 3;
    if (mts == 0) return -1;
    if (nt >= 8) {
      ni = x + 8 * (in / mts);
      return ni < nt ? in % mts : -1;
    }
    const int all = mts * nt, share = (all + 7) >> 3, u = x * share + in;
    if (in >= share || u >= all) return -1;
    ni = u / mts;
    return u - ni * mts;
  });
  if (t.e == -2) return;
  const int e = __builtin_amdgcn_readfirstlane(t.e);
  const int64_t m0 = __builtin_amdgcn_readfirstlane((int)t.s0);
  const int mrows = __builtin_amdgcn_readfirstlane((int)(t.s1 - t.s0));
  const int red = e < 0 ? 0 : (OP == kLinear ? a.K : a.N);
  const int n0 = ni * BN, ncols = cols - n0 < BN ? cols - n0 : BN;

  // weights: as one operand of 64 rows (columns)
  GgOperand<64, 1, TB> ob;
  const char* B = static_cast<const char*>(a.b);
  if constexpr (!TB) {
    ob.c8 = 8 * p;
    ob.base = gg_uni(B + ((int64_t)e * a.strb + (int64_t)n0 * a.ldb) * 2);
    ob.bytes = gg_uni(((int64_t)(ncols - 1) * a.ldb + red) * 2);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = j + 8 * rr;
      ob.vo[j] = r < ncols ? (uint32_t)((r * a.ldb + (ob.c8 ^ (8 * j))) * 2) : kGgOob;
    }
  } else {
    ob.base = gg_uni(B + ((int64_t)e * a.strb + n0) * 2);
    ob.bytes = gg_uni(((int64_t)(red - 1) * a.ldb + ncols) * 2);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = j + 8 * rr, c = 8 * (p ^ gg_swz_tr(8 * j + rr));
      ob.vo[j] = c < ncols ? (uint32_t)((r * a.ldb + c) * 2) : kGgOob;
    }
  }
  // operand rows in their order, chunk c of row r at c ^ ((r >> 1) & 7)
  const bool gather = OP == kLinear && a.rows;
  const char* A = static_cast<const char*>(a.a);
  const gg_u4 ars = gg_desc(gg_uni(gather ? A : A + m0 * a.lda * 2),
                            gg_uni(gather ? ((a.T - 1) * a.lda + red) * 2 : ((int64_t)(mrows - 1) * a.lda + red) * 2));
  uint32_t av[kPX];
  int ac[kPX];
#pragma unroll
  for (int j = 0; j < kPX; ++j) {
    const int r = 8 * j + rr;
    ac[j] = 8 * (p ^ ((r >> 1) & 7));
    int64_t row = r;
    bool ok = r < mrows && e >= 0;
    if (gather) {
      row = ok ? a.rows[m0 + r] : 0;
      ok = ok && row >= 0 && row < a.T;
    }
    av[j] = ok ? (uint32_t)((row * a.lda + ac[j]) * 2) : kGgOob;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(gg_lptr)lds;
  asm volatile("" ::"v"(lds0) : "memory");
  const uint32_t ring = lds0 + w * 2 * kStage;
  const int steps = (red + 63) / 64;
  const int mine = steps > w ? (steps - w + 3) / 4 : 0;  // steps w, w + 4, ...
  auto stage = [&](int j, uint32_t at) {
    const int st = w + 4 * j, left = red - 64 * st;
    const uint32_t so = (uint32_t)st * 128u;
    gg_u4 rs;
    if constexpr (!TB) rs = gg_desc(ob.base, ob.bytes);
    else rs = gg_desc(ob.base + (int64_t)st * 64 * a.ldb * 2, ob.bytes - (int64_t)st * 64 * a.ldb * 2);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      uint32_t v = ob.vo[q];
      if constexpr (!TB) v = (ob.c8 ^ (8 * q)) < left ? v : kGgOob;
      gg_dma(at + 1024 * q, v, rs, TB ? 0u : so);
    }
#pragma unroll
    for (int q = 0; q < kPX; ++q) gg_dma(at + kW + 1024 * q, ac[q] < left ? av[q] : kGgOob, ars, so);
  };
  GgReader<TB, 1> rb;
  rb.init(0, lane);
  uint32_t rx[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) rx[h] = i * 128 + 16 * ((4 * h + g) ^ ((i >> 1) & 7));
  f32x4 acc[MX][4];
#pragma unroll
  for (int x = 0; x < MX; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[x][y] = {0.f, 0.f, 0.f, 0.f};
  if (mine > 0) stage(0, ring);
  if (mine > 1) stage(1, ring + kStage);
  for (int j = 0; j < mine; ++j) {
    asm volatile("" ::: "memory");
    if (j + 1 < mine) gg_wait<8 + kPX>();
    else gg_wait<0>();
    asm volatile("" ::: "memory");
    const uint32_t at = ring + (j & 1) * kStage;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      gg_u4 fa[MX], fb[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) fb[y] = gg_frag(rb, at, h, y);
#pragma unroll
      for (int x = 0; x < MX; ++x) fa[x] = *(gg_lu4)(uintptr_t)(at + kW + rx[h] + x * 2048);
#pragma unroll
      for (int x = 0; x < MX; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = gg_mfma<DT>(fb[y], fa[x], acc[x][y]);
    }
    asm volatile("" ::: "memory");
    if (j + 2 < mine) {
      gg_wait<8 + kPX>();  // this slot has been read
      asm volatile("" ::: "memory");
      stage(j + 2, at);
    }
  }
  __syncthreads();  // every wave is out of its ring
  constexpr int kPitch = 68;
  float* red_t = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int x = 0; x < MX; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y)
      *reinterpret_cast<f32x4*>(red_t + (w * BM + 16 * x + i) * kPitch + 16 * y + 4 * g) = acc[x][y];
  __syncthreads();
  const int c = 4 * (tid & 15), n = n0 + c;
#pragma unroll
  for (int x = 0; x < MX; ++x) {
    const int m = 16 * x + (tid >> 4);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q) v += *reinterpret_cast<const f32x4*>(red_t + (q * BM + m) * kPitch + c);
    if (m >= mrows || c >= ncols) continue;
    if constexpr (OP == kLinear) {
      if (e >= 0 && a.bias) {
        const float* bp = a.bias + (int64_t)e * a.ldbias + n;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += bp[q];
      }
      if (a.relu) {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = v[q] < 0.f ? 0.f : v[q];
      }
    } else {
      if (e >= 0 && a.mask) {
        const uint2 k = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.mask) + (m0 + m) * a.ldmask + n);
        const uint16_t mk[4] = {(uint16_t)k.x, (uint16_t)(k.x >> 16), (uint16_t)k.y, (uint16_t)(k.y >> 16)};
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = gg_f<DT>(mk[q]) > 0.f ? v[q] : 0.f;
      }
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (m0 + m) * a.ldo + n) =
        make_uint2(gg_pack2<DT>(v[0], v[1]), gg_pack2<DT>(v[2], v[3]));
  }
}

// ---------------------------------------------------------------------------
// Any width, stride and alignment (rows of odd length start at any 2 bytes, so
// nothing can go straight to LDS): 128 x 128 tile, 4 waves of 64 x 64, the same
// LDS images; a thread loads 16-B chunks of a step into registers while the
// step before is multiplied, and stores them into the other buffer after.  On
// operands that the fast path takes too it needs 51 us against 37 (8192 rows, 8
// experts of 1000 x 1000) and 1415 against 980 (32768 of 4096 x 4096); 8192 rows of
// 1003 x 1001 with a bias: 36 (44 with the bias loaded at its use; backward with a
// mask 46 and 52).  Against the same sizes rounded up to whole words: 5003 rows, 4
// experts of 301 x 2003, 29 us against 18; 2000 rows of 1001 x 1003 27 and 14; 16 rows,
// 8 experts of 4001 x 4095, 92 and 49; the weight gradient of 8192 rows of 127 x 783
// 23 and 16.
// ---------------------------------------------------------------------------
// Loads are never under a condition (the compiler waits for such a load at the
// end of its branch: 115 us against 58 at 8192 rows, 8 experts of 1003 x 1001):
// a chunk that does not fit its row is the row's last 8 elements, shifted when
// it is stored, and one that has no row is some other, zeroed then.
struct GgChunk {
  gg_u4 v;
  int shift;  // elements to drop at the front; 8 or more: all of them
};
template <bool NARROW>
__device__ __forceinline__ void gg_load8(GgChunk& u, const uint16_t* row, int c, int width, bool ok) {
  if constexpr (!NARROW) {
    const int at = c < width - 8 ? c : width - 8;
    __builtin_memcpy(&u.v, row + at, 16);
    u.shift = ok ? c - at : 8;
  } else {  // rows that may have fewer than 8
    uint64_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < width) (i < 4 ? lo : hi) |= (uint64_t)row[c + i] << (16 * (i & 3));
    u.v = gg_u4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    u.shift = ok ? 0 : 8;
  }
}
__device__ __forceinline__ gg_u4 gg_settle(const GgChunk& u) {
  return __builtin_bit_cast(gg_u4, drop_front8(__builtin_bit_cast(uint4, u.v), u.shift));
}

template <int DT, int OP, bool NARROW>
__global__ __launch_bounds__(256, 2) void grouped_any_k(GroupedArgs a) {
  constexpr int BM = 128, BN = 128, XF = 4, YF = 4;
  constexpr bool TA = OP == kWgrad, TB = OP != kLinear;
  constexpr uint32_t kImg = BM * 128;
  __shared__ __attribute__((aligned(1024))) char lds[4 * kImg];  // A, B, and again
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, wr = w >> 1, wc = w & 1, wn = 64 * wc;
  const int cols = OP == kLinear ? a.N : a.K, nt = (cols + BN - 1) / BN;
  const uint16_t* A = static_cast<const uint16_t*>(a.a);
  const uint16_t* B = static_cast<const uint16_t*>(a.b);
  int e, mrows, red, ni = 0, part = 0;
  int64_t m0, red0 = 0;
  if constexpr (OP == kWgrad) {
    const int mtb = (a.N + BM - 1) / BM, per = mtb * nt;
    int pos = gg_pos(blockIdx.x, per * a.E * a.split);
    if (pos < 0) return;
    part = pos / (per * a.E);
    pos -= part * per * a.E;
    e = pos / per;
    int mi;
    gg_order(pos - e * per, mtb, nt, mi, ni);
    m0 = (int64_t)mi * BM;
    mrows = (int)(a.N - m0 < BM ? a.N - m0 : BM);
    gg_part(a, e, part, red0, red);
  } else {
    const GgTile t = gg_find(a.offsets, a.E, a.S, BM, a.zero_rest, [&](int mts) {
      const int pos = gg_pos(blockIdx.x, mts * nt * a.split);
      if (pos < 0) return -1;
      part = pos / (mts * nt);
      int mi;
      gg_order(pos - part * mts * nt, mts, nt, mi, ni);
      return mi;
    });
    if (t.e == -2 || (t.e < 0 && a.split > 1)) return;  // (the join clears rows of no group)
    e = __builtin_amdgcn_readfirstlane(t.e);
    m0 = __builtin_amdgcn_readfirstlane((int)t.s0);
    mrows = __builtin_amdgcn_readfirstlane((int)(t.s1 - t.s0));
    red = e < 0 ? 0 : (OP == kLinear ? a.K : a.N);
  }
  const int n0 = __builtin_amdgcn_readfirstlane(ni * BN), ncols = cols - n0 < BN ? cols - n0 : BN;

  // chunk q = tid + 256 j of a step: row-major operands row q / 8, chunk q % 8;
  // transposed ones reduction row q / 16, column chunk q % 16
  struct Set {
    GgChunk a[4], b[4];
  };
  const uint16_t *ap[4], *bp[4];  // row-major: this thread's rows
  bool ao[4], bo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = (tid >> 3) + 32 * j;
    if constexpr (!TA) {
      ao[j] = r < mrows;
      int64_t row = m0 + (ao[j] ? r : 0);
      if (OP == kLinear && a.rows && e >= 0) {
        row = a.rows[row];
        ao[j] = ao[j] && row >= 0 && row < a.T;
        row = ao[j] ? row : 0;
      }
      ap[j] = A + row * a.lda;
    }
    if constexpr (!TB) {
      bo[j] = r < ncols;
      bp[j] = B + (int64_t)(e < 0 ? 0 : e) * a.strb + (int64_t)(n0 + (bo[j] ? r : 0)) * a.ldb;
    }
  }
  const bool empty = OP != kDgrad && a.rows && a.T == 0;  // a gather from nothing
  auto load = [&](int t, Set& u) {
    const int k0 = 64 * t;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 8 * (tid & 7), k = k0 + (tid >> 4) + 16 * j, kk = k < red ? k : red - 1, m = 8 * (tid & 15);
      if constexpr (!TA) gg_load8<NARROW>(u.a[j], empty ? B : ap[j], k0 + c, red, ao[j] && !empty);
      else gg_load8<NARROW>(u.a[j], A + (red0 + kk) * a.lda, (int)m0 + m, a.N, k < red && m < mrows);
      if constexpr (!TB) {
        gg_load8<NARROW>(u.b[j], bp[j], k0 + c, red, bo[j]);
      } else if constexpr (OP == kDgrad) {
        gg_load8<NARROW>(u.b[j], B + (int64_t)e * a.strb + (int64_t)kk * a.ldb, n0 + m, cols, k < red && m < ncols);
      } else {
        int64_t row = red0 + kk;
        bool ok = k < red && m < ncols && !empty;
        if (a.rows) {
          row = a.rows[row];
          ok = ok && row >= 0 && row < a.T;
          row = ok ? row : 0;
        }
        gg_load8<NARROW>(u.b[j], empty ? A : B + row * a.ldb, empty ? 0 : n0 + m, empty ? a.N : cols, ok);
      }
    }
  };
  auto put = [&](char* img, bool tr, bool settle, const GgChunk (&u)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const gg_u4 v = settle ? gg_settle(u[j]) : u[j].v;
      if (!tr) {
        const int r = (tid >> 3) + 32 * j, pos = 64 * (r >> 6) + 8 * (r & 7) + ((r >> 3) & 7);
        *reinterpret_cast<gg_u4*>(img + pos * 128 + 16 * ((tid & 7) ^ gg_swz(pos))) = v;
      } else {
        const int k = (tid >> 4) + 16 * j, pos = 8 * (k & 7) + (k >> 3), c = tid & 15;
        *reinterpret_cast<gg_u4*>(img + (c >> 3) * 8192 + pos * 128 + 16 * ((c & 7) ^ gg_swz_tr(pos))) = v;
      }
    }
  };
  f32x4 acc[XF][YF], accs[2];
#pragma unroll
  for (int x = 0; x < XF; ++x)
#pragma unroll
    for (int y = 0; y < YF; ++y) acc[x][y] = {0.f, 0.f, 0.f, 0.f};
  accs[0] = accs[1] = {0.f, 0.f, 0.f, 0.f};
  const bool sums = OP == kWgrad && a.db && n0 == 0;
  constexpr uint32_t kOnes = DT == kBF16 ? 0x3f803f80u : 0x3c003c00u;
  const gg_u4 ones = {kOnes, kOnes, kOnes, kOnes};
  GgReader<TA, 2> ra;
  GgReader<TB, 1> rb;
  ra.init(wr, lane);
  rb.init(YF * wc, lane);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(gg_lptr)lds;
  // steps [first, steps): all, or a part of the reduction
  int steps = (red + 63) / 64, first = 0;
  if (OP != kWgrad && a.split > 1) {
    const int per = (steps + a.split - 1) / a.split;
    first = part * per < steps ? part * per : steps;
    steps = steps - first < per ? steps : first + per;
  }
  // whole chunks need no shifting: full tiles of rows that exist, but a last step
  const bool whole = !NARROW && mrows == BM && ncols == BN && !(OP != kDgrad && a.rows);
  auto store = [&](int t, const Set& u) {
    char* to = lds + (t & 1) * 2 * kImg;
    if (whole && 64 * t + 64 <= red) {
      put(to, TA, false, u.a);
      put(to + kImg, TB, false, u.b);
    } else {
      put(to, TA, true, u.a);
      put(to + kImg, TB, true, u.b);
    }
  };
  auto multiply = [&](int t) {
    const uint32_t at = lds0 + (t & 1) * 2 * kImg;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      gg_u4 fa[XF], fb[YF];
#pragma unroll
      for (int y = 0; y < YF; ++y) fb[y] = gg_frag(rb, at + kImg, h, y);
#pragma unroll
      for (int x = 0; x < XF; ++x) fa[x] = gg_frag(ra, at, h, x);
#pragma unroll
      for (int x = 0; x < XF; ++x)
#pragma unroll
        for (int y = 0; y < YF; ++y) acc[x][y] = gg_mfma<DT>(fb[y], fa[x], acc[x][y]);
      if (sums) {
#pragma unroll
        for (int u = 0; u < 2; ++u) accs[u] = gg_mfma<DT>(ones, wc ? fa[2 + u] : fa[u], accs[u]);
      }
    }
  };
  // step t is multiplied while steps t + 1 (stored after it) and t + 2 are in flight
  Set u0, u1;
  if (steps > first) {
    load(first, u0);
    load(steps > first + 1 ? first + 1 : first, u1);
    store(first, u0);
    load(steps > first + 2 ? first + 2 : first, u0);
    __syncthreads();
    for (int t = first; t < steps; t += 2) {
      multiply(t);
      if (t + 1 < steps) {
        store(t + 1, u1);
        if (t + 3 < steps) load(t + 3, u1);
        __syncthreads();
        multiply(t + 1);
        if (t + 2 < steps) {
          store(t + 2, u0);
          if (t + 4 < steps) load(t + 4, u0);
          __syncthreads();
        }
      }
    }
  }

  if constexpr (OP == kWgrad) {
    float* out = static_cast<float*>(a.out) + (int64_t)e * a.stro;
    if (sums && g == 0) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int m = 16 * (2 * (2 * wc + u) + wr) + i;
        if (m < mrows) a.db[(int64_t)e * a.N + m0 + m] = accs[u][0];
      }
    }
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      const int m = 16 * (2 * x + wr) + i;
      if (m >= mrows) continue;
      float* o = out + (m0 + m) * a.ldo + n0;
#pragma unroll
      for (int y = 0; y < YF; ++y) {
        const int n = wn + 16 * y + 4 * g;
        if (n + 4 <= ncols) {
          __builtin_memcpy(o + n, &acc[x][y], 16);
        } else {
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (n + q < ncols) o[n + q] = acc[x][y][q];
        }
      }
    }
  } else if (a.split > 1) {  // [parts][S][columns]
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      const int m = 16 * (2 * x + wr) + i;
      if (m >= mrows) continue;
      float* o = a.ws + ((int64_t)part * a.S + m0 + m) * cols + n0;
#pragma unroll
      for (int y = 0; y < YF; ++y) {
        const int n = wn + 16 * y + 4 * g;
        if (n + 4 <= ncols) {
          __builtin_memcpy(o + n, &acc[x][y], 16);
        } else {
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (n + q < ncols) o[n + q] = acc[x][y][q];
        }
      }
    }
  } else {
    uint16_t* out = static_cast<uint16_t*>(a.out);
    const uint16_t* mk = OP == kDgrad && e >= 0 ? static_cast<const uint16_t*>(a.mask) : nullptr;
    // bias and mask: all loads first and none under a condition, from the nearest
    // column (row) that exists
    f32x4 bias[YF];
    if (OP == kLinear && e >= 0 && a.bias) {
#pragma unroll
      for (int y = 0; y < YF; ++y)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + wn + 16 * y + 4 * g + q;
          bias[y][q] = a.bias[(int64_t)e * a.ldbias + (n < cols ? n : cols - 1)];
        }
    } else {
#pragma unroll
      for (int y = 0; y < YF; ++y) bias[y] = {0.f, 0.f, 0.f, 0.f};
    }
    uint64_t keep[XF][YF];  // 4 mask values each
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      const int m = 16 * (2 * x + wr) + i;
      const uint16_t* row = mk ? mk + (m0 + (m < mrows ? m : mrows - 1)) * a.ldmask : nullptr;
#pragma unroll
      for (int y = 0; y < YF; ++y) {
        const int n = n0 + wn + 16 * y + 4 * g;
        keep[x][y] = 0;
        if (mk) {
          if constexpr (!NARROW) {
            __builtin_memcpy(&keep[x][y], row + (n < cols - 4 ? n : cols - 4), 8);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (n + q < cols) keep[x][y] |= (uint64_t)row[n + q] << (16 * q);
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < XF; ++x) {
      const int m = 16 * (2 * x + wr) + i;
      if (m >= mrows) continue;
      uint16_t* o = out + (m0 + m) * a.ldo + n0;
#pragma unroll
      for (int y = 0; y < YF; ++y) {
        const int n = wn + 16 * y + 4 * g;
        f32x4 v = acc[x][y];
        if constexpr (OP == kLinear) {
          v += bias[y];
          if (a.relu) {
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = v[q] < 0.f ? 0.f : v[q];
          }
        } else if (mk) {
          const int past = NARROW ? 0 : n0 + n - (cols - 4);  // columns the load was moved back by
          const uint64_t k = keep[x][y] >> (past < 1 ? 0 : (past < 4 ? 16 * past : 63));
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = gg_f<DT>((uint16_t)(k >> (16 * q))) > 0.f ? v[q] : 0.f;
        }
        const uint2 u = make_uint2(gg_pack2<DT>(v[0], v[1]), gg_pack2<DT>(v[2], v[3]));
        if (n + 4 <= ncols) {
          __builtin_memcpy(o + n, &u, 8);
        } else {
          if (n < ncols) o[n] = (uint16_t)u.x;
          if (n + 1 < ncols) o[n + 1] = (uint16_t)(u.x >> 16);
          if (n + 2 < ncols) o[n + 2] = (uint16_t)u.y;
        }
      }
    }
  }
}

// The parts' sums, in order: 4 columns a thread (V), or 1.
template <bool V>
__global__ __launch_bounds__(256) void grouped_join_k(GroupedArgs a) {
  const int64_t n = (int64_t)a.E * a.N * a.K, nb = a.db ? (int64_t)a.E * a.N : 0, step = (int64_t)gridDim.x * 256;
  constexpr int W = V ? 4 : 1;
  const float* bias = a.ws + a.split * n;
  for (int64_t t = blockIdx.x * 256 + threadIdx.x; t * W < n; t += step) {
    const int64_t i = t * W, row = i / a.K, c = i - row * a.K, e = row / a.N;
    float v[W];
#pragma unroll
    for (int q = 0; q < W; ++q) v[q] = 0.f;
#pragma unroll 8
    for (int p = 0; p < a.split; ++p) {
      float u[W];
      if constexpr (V) __builtin_memcpy(u, __builtin_assume_aligned(a.ws + p * n + i, 16), 16);
      else u[0] = a.ws[p * n + i];
#pragma unroll
      for (int q = 0; q < W; ++q) v[q] += u[q];
    }
    float* o = static_cast<float*>(a.out) + e * a.stro + (row - e * a.N) * a.ldo + c;
#pragma unroll
    for (int q = 0; q < W; ++q) o[q] = v[q];
  }
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < nb; i += step) {
    float v = 0.f;
#pragma unroll 8
    for (int p = 0; p < a.split; ++p) v += bias[p * nb + i];
    a.db[i] = v;
  }
}
hipError_t launch_join(const GroupedArgs& a, hipStream_t s) {
  const bool v = a.K % 4 == 0 && (reinterpret_cast<uintptr_t>(a.ws) & 15) == 0;
  const int64_t threads = (int64_t)a.E * a.N * a.K / (v ? 4 : 1), blocks = (threads + 255) / 256;
  const dim3 grid((uint32_t)(blocks < 2048 ? blocks : 2048));
  if (v) hipLaunchKernelGGL((grouped_join_k<true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((grouped_join_k<false>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

// The same for rows of an output: a wave 256 columns of a row, which it finds the
// expert of for the bias; rows of no group are cleared or left.
template <int DT, int OP>
__global__ __launch_bounds__(256) void grouped_join_rows_k(GroupedArgs a) {
  const int lane = threadIdx.x & 63, cols = OP == kLinear ? a.N : a.K;
  const int64_t r = blockIdx.x * 4 + (threadIdx.x >> 6), n = a.S * cols;
  if (r >= a.S) return;
  int e = -1;
  for (int e0 = 0; e0 < a.E && e < 0; e0 += 64) {
    bool in = false;
    if (e0 + lane < a.E) {
      const int64_t lo = gg_clamp(a.offsets[e0 + lane], 0, a.S), hi = gg_clamp(a.offsets[e0 + lane + 1], lo, a.S);
      in = r >= lo && r < hi;
    }
    const unsigned long long hit = __ballot(in);
    if (hit) e = e0 + __ffsll(hit) - 1;
  }
  if (e < 0 && !a.zero_rest) return;
  const int c0 = 256 * blockIdx.y + lane;  // and c0 + 64, + 128, + 192; past the end: the last column's loads
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (e >= 0) {
    for (int q0 = 0; q0 < a.split; q0 += 8) {  // 8 parts in flight; past the last: the last's, not added
      float t[8][4];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float* p = a.ws + (q0 + q < a.split ? q0 + q : a.split - 1) * n + r * cols;
#pragma unroll
        for (int u = 0; u < 4; ++u) t[q][u] = p[c0 + 64 * u < cols ? c0 + 64 * u : cols - 1];
      }
#pragma unroll
      for (int q = 0; q < 8; ++q)
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] += q0 + q < a.split ? t[q][u] : 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int c = c0 + 64 * u;
    if (c >= cols) continue;
    float x = v[u];
    if (e >= 0) {
      if constexpr (OP == kLinear) {
        if (a.bias) x += a.bias[(int64_t)e * a.ldbias + c];
        if (a.relu) x = x < 0.f ? 0.f : x;
      } else if (a.mask) {
        x = gg_f<DT>(static_cast<const uint16_t*>(a.mask)[r * a.ldmask + c]) > 0.f ? x : 0.f;
      }
    }
    static_cast<uint16_t*>(a.out)[r * a.ldo + c] = (uint16_t)gg_pack2<DT>(x, x);
  }
}

template <int DT, int OP>
hipError_t launch_any(const GroupedArgs& a, hipStream_t s) {
  const int64_t nt = ((OP == kLinear ? a.N : a.K) + 127) / 128, some = a.E < a.S ? a.E : a.S;
  const int64_t mt = OP == kWgrad ? (int64_t)a.E * ((a.N + 127) / 128) * a.split : ((a.S + 127) / 128 + some + (a.zero_rest ? 2 : 0)) * a.split;
  const int64_t blocks = (mt * nt + 7) / 8 * 8;
  if (blocks * 256 > kMaxThreads) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)blocks);
  if (a.N < 8 || a.K < 8) hipLaunchKernelGGL((grouped_any_k<DT, OP, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((grouped_any_k<DT, OP, false>), grid, dim3(256), 0, s, a);
  if constexpr (OP != kWgrad) {
    if (a.split > 1)
      hipLaunchKernelGGL((grouped_join_rows_k<DT, OP>), dim3((uint32_t)((a.S + 3) / 4), (uint32_t)((nt + 1) / 2)), dim3(256),
                         0, s, a);
  }
  return hipGetLastError();
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
  // a group's ids: 4 bytes each behind offsets and a length of 32 bits
  if (op == kWgrad && a.rows && a.S >= kGgIds) return false;
  if (op == kWgrad)
    return (!a.rows || (a.T * a.ldb + a.K) * 2 <= kGgSpan) && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 &&
           a.ldo % 4 == 0 && a.ldo <= 0x3fffff && (a.E <= 1 || a.stro % 4 == 0);
  if (!gg_al(a.out, a.ldo, 0) || a.ldo > 0x7fffff) return false;
  return op != kDgrad || !a.mask || (gg_al(a.mask, a.ldmask, 0) && a.ldmask <= 0x7fffff);
}

template <int DT, int OP, bool GATHER = false>
hipError_t launch_fast(const GroupedArgs& a, hipStream_t s) {
  const int cols = OP == kLinear ? a.N : a.K;
  const int64_t ntb = (cols + 255) / 256, nts = (cols + 127) / 128;
  int64_t big, small;  // workgroups at most
  int keep = 0;
  if (OP == kWgrad) {
    const int64_t all = (a.N + 255) / 256 * ntb * a.E;
    if (all > 0x3fffffffLL) return hipErrorInvalidValue;
    const int64_t last = all % kGgCus;  // a last round in quarters where that is sooner
    keep = (int)(gg_small_cost(4 * last, (int)(a.S / a.E / 64)) < kGgRound ? all - last : all);
    if (a.split > 1) keep = 0;
    big = keep;
    small = 4 * (all - keep) * a.split;
  } else {
    // Too few tiles for a round of 256 x 256, if half the groups end inside one, or a
    // reduction so short that a tile is mostly its first loads and its stores, which
    // two workgroups a CU hide from each other (with 256 x 256 / 128 x 128 only: 13424
    // rows of 568, reduction 1024, 36 / 29 us; 8192 rows of 4096, 256 53 / 41, 512 64 /
    // 67; 32768 of 4096, 64 104 / 103, 256 146 / 156).
    const int64_t some = a.E < a.S ? a.E : a.S;
    if (4 * (a.S / 256 + some / 2) * ntb <= 700 || (OP == kLinear ? a.K : a.N) <= 256) keep = -1;
    big = keep < 0 ? 0 : (a.S / 256 + some) * ntb;
    // quarters, halves of the groups' last rows, rows in no group
    const int64_t quarters = keep < 0 ? a.S / 256 * ntb : kGgCus;
    small = 4 * quarters + 2 * some * nts;
    const int64_t most = (a.S / 128 + 2 * some) * 2 * ntb;
    small = ((small < most ? small : most) + 7) / 8 * 8 + (a.zero_rest ? kGgZero : 0);
  }
  big = (big + 7) / 8 * 8;
  small = (small + 7) / 8 * 8;
  if (big * 512 > kMaxThreads || small * 256 > kMaxThreads) return hipErrorInvalidValue;
  if (big)
    hipLaunchKernelGGL((grouped_fast_k<DT, OP, 256, 256, 2, 4, GATHER>), dim3((uint32_t)big), dim3(512), 0, s, a, keep);
  if (small)
    hipLaunchKernelGGL((grouped_fast_k<DT, OP, 128, 128, 2, 2, GATHER>), dim3((uint32_t)small), dim3(256), 0, s, a, keep);
  return hipGetLastError();
}

template <int DT, int OP, int MX>
hipError_t launch_skinny(const GroupedArgs& a, hipStream_t s) {
  const int cols = OP == kLinear ? a.N : a.K;
  const int nt = (cols + 63) / 64;
  int64_t mt = (a.S + 16 * MX - 1) / (16 * MX) + a.E + (a.zero_rest ? 2 : 0);
  mt = mt < a.S ? mt : a.S;
  const int64_t blocks = nt >= 8 ? (int64_t)(nt + 7) / 8 * 8 * mt : (nt * mt + 7) / 8 * 8;
  if (blocks * 256 > kMaxThreads) return hipErrorInvalidValue;
  hipLaunchKernelGGL((grouped_skinny_k<DT, OP, MX>), dim3((uint32_t)blocks), dim3(256), 0, s, a, nt);
  return hipGetLastError();
}
template <int DT>
hipError_t launch_skinny_op(GroupedOp op, const GroupedArgs& a, int mx, hipStream_t s) {
  if (op == kLinear) {
    if (mx == 1) return launch_skinny<DT, kLinear, 1>(a, s);
    return launch_skinny<DT, kLinear, 2>(a, s);
  }
  if (mx == 1) return launch_skinny<DT, kDgrad, 1>(a, s);
  return launch_skinny<DT, kDgrad, 2>(a, s);
}

template <int DT>
hipError_t launch_any_op(GroupedOp op, const GroupedArgs& a, hipStream_t s) {
  if (op == kLinear) return launch_any<DT, kLinear>(a, s);
  return op == kDgrad ? launch_any<DT, kDgrad>(a, s) : launch_any<DT, kWgrad>(a, s);
}
template <int DT>
hipError_t launch_fast_op(GroupedOp op, const GroupedArgs& a, hipStream_t s) {
  if (op == kWgrad) return a.rows ? launch_fast<DT, kWgrad, true>(a, s) : launch_fast<DT, kWgrad>(a, s);
  // Few rows.  The kernel that shares the reduction among its waves wins where the
  // 128 x 128 tiles are fewer than the CUs, each of them a long chain of steps (8
  // experts of 1024 x 4096, microseconds, 128 x 128 after the slash: 32 rows an
  // expert 16 / 36, 96 29 / 38, 128 40 / 39; of 1024 x 1024: 32 6 / 12, 96 11 / 13,
  // 128 15 / 14).  32 rows a tile leave one workgroup a CU: the limits, two rounds of
  // the chip and two and a half, lie between those sizes.
  // With 16 rows a tile while experts have no more (4096 x 4096: 8 rows 44 / 52, 16
  // 46 / 55; backward 45 / 42 and 52 / 47), else 32 (24 rows: 47 against 50, and 55).
  const int red = op == kLinear ? a.K : a.N, cols = op == kLinear ? a.N : a.K;
  const int64_t wgs = (a.S / 32 + (a.E + 1) / 2) * ((cols + 63) / 64);
  if (a.S / a.E <= 16) return launch_skinny_op<DT>(op, a, 1, s);
  if (wgs <= (red >= 2048 ? 640 : 512)) return launch_skinny_op<DT>(op, a, 2, s);
  return op == kLinear ? launch_fast<DT, kLinear>(a, s) : launch_fast<DT, kDgrad>(a, s);
}

}  // namespace

// Parts of a reduction whose 128 x 128 tiles leave CUs idle: a group's rows (weight
// gradients), or all of it (the kernel for any width).  A step of 64 takes about
// 0.57 us (1.4 in the kernel for any width), as long as a CU has one tile; parts
// shorten that chain and cost their sums' way through the workspace and a launch.
// Microseconds without parts and with the number taken here: weight gradients of 20000
// rows of 304 x 200 178 / 18 (32), of 301 x 201 437 / 26 (32), of 32768 of 1024 x 1024
// 293 / 95 (8), 8 experts, 32768 of 128 x 784 53 / 31 (4); products of 75 rows, 21 experts
// of 248 x 3154, 59 / 21, backward of 101 rows, 2 experts, 1788 to 159, 44 / 12.
int parts_of(GroupedOp op, const GroupedArgs& a) {
  const bool fast = fast_ok(op, a);
  if (a.S == 0 || (op != kWgrad && fast)) return 1;
  const int cols = op == kLinear ? a.N : a.K, red = op == kLinear ? a.K : a.N;
  const int64_t nt = (cols + 127) / 128, some = a.E < a.S ? a.E : a.S;
  const int64_t tiles = nt * (op == kWgrad ? (int64_t)a.E * ((a.N + 127) / 128) : a.S / 128 + some);
  if (tiles > kGgCus) return 1;
  const int64_t steps = ((op == kWgrad ? a.S / a.E : red) + 63) / 64, step = fast ? 570 : 1400;  // step: ns
  const int64_t bytes = (op == kWgrad ? (int64_t)a.E * a.N : a.S) * cols * 4;
  const int64_t weights = op == kWgrad ? 0 : some * a.N * a.K * 2 / 3000;  // ns to read them
  int best = 1;
  int64_t least = -1;
  for (int p = 1; p <= 32; p *= 2) {
    const int64_t on_cu = (tiles * p + kGgCus - 1) / kGgCus;
    // two tiles on a CU share its fetch: no gain in the kernel for any width
    int64_t chain = (steps + p - 1) / p * step * (on_cu > 1 ? (fast ? 85 : 100) * on_cu : 100) / 100;
    chain = chain > weights ? chain : weights;
    const int64_t cost = chain + (p > 1 ? 5000 + (2 * p + 1) * bytes / 4000 : 0);  // 4 TB/s
    if (least < 0 || cost < least) {
      least = cost;
      best = p;
    }
  }
  return best;
}

bool grouped_whole_words(GroupedOp op, const GroupedArgs& a) { return fast_ok(op, a); }

int64_t grouped_ws_floats(GroupedOp op, const GroupedArgs& a) {
  const int parts = parts_of(op, a);
  if (parts == 1) return 0;
  if (op == kWgrad) return (int64_t)parts * a.E * a.N * (a.K + (a.db ? 1 : 0));
  return parts * a.S * (op == kLinear ? a.N : a.K);
}

hipError_t grouped_gemm(GroupedOp op, const GroupedArgs& args, hipStream_t s) {
  GroupedArgs a = args;
  if (a.E < 1 || a.N < 1 || a.K < 1 || a.S < 0 || a.T < 0 || a.S > 0x7fffffffLL - (op == kWgrad ? 255 : 0) ||
      a.T > 0x7fffffffLL || (a.dtype != kBF16 && a.dtype != kF16))
    return hipErrorInvalidValue;
  if (op != kWgrad && a.S == 0) return hipSuccess;
  a.split = parts_of(op, a);
  if (a.split > 1 && !a.ws) return hipErrorInvalidValue;
  const hipError_t e = fast_ok(op, a)
                           ? (a.dtype == kBF16 ? launch_fast_op<kBF16>(op, a, s) : launch_fast_op<kF16>(op, a, s))
                           : (a.dtype == kBF16 ? launch_any_op<kBF16>(op, a, s) : launch_any_op<kF16>(op, a, s));
  return e == hipSuccess && op == kWgrad && a.split > 1 ? launch_join(a, s) : e;
}

}  // namespace dsml
