// Expert-layer operators and gradient clipping: host entry points of
// kernels/route.hip, kernels/grouped_gemm.hip, kernels/expert_combine.hip and
// kernels/grad_clip.hip.  All pointers are device pointers; every launch goes
// to the stream given and none synchronises.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dsml {

constexpr int64_t kMaxThreads = 0xffffffffLL;  // of a launch, along one axis

// ---- router -------------------------------------------------------------
constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxK = 16;
struct RouteArgs {
  const void* logits;  // [T][ldl], dtype
  int64_t ldl;
  int64_t T;
  int E, k;
  int dtype;
  int all;          // gates normalised over the whole row (else over the chosen experts)
  float* gates;     // [T][k]
  int32_t* experts; // [T][k], -1: none
  int32_t* offsets; // [E + 1]
  int32_t* rows;    // [T k], slot -> token, -1 behind offsets[E]
  int32_t* slots;   // [T][k], -1: none
  int32_t* counts;  // workspace, route_ws_words(T, E) words
};
int64_t route_ws_words(int64_t T, int E);
hipError_t route_topk(const RouteArgs& a, hipStream_t s);

struct RouteBwdArgs {
  const void* logits;  // [T][ldl]
  int64_t ldl;
  const float* gates;      // [T][k]
  const int32_t* experts;  // [T][k]
  const float* dgates;     // [T][k]
  void* dlogits;           // [T][E] contiguous, dtype of the logits
  int64_t T;
  int E, k;
  int dtype;
  int all;
};
hipError_t route_topk_backward(const RouteBwdArgs& a, hipStream_t s);

// ---- products grouped by expert -------------------------------------------
// Group e owns rows [offsets[e], offsets[e + 1]) (clamped to [0, S] on the GPU).
struct GroupedArgs {
  const void* a;  // linear: x [T][lda]; dgrad, wgrad: dz [S][lda]
  int64_t lda;
  const void* b;  // linear, dgrad: w [E][N][K] (ldb a row, strb an expert); wgrad: x [T][ldb]
  int64_t ldb, strb;
  const int32_t* offsets;  // [E + 1]
  const int32_t* rows;     // row of x for every slot, or null: slot s reads row s
  const float* bias;       // linear: [E][ldbias]
  int64_t ldbias;
  const void* mask;  // dgrad: [S][ldmask], outputs kept where > 0
  int64_t ldmask;
  void* out;  // linear: [S][ldo] (N columns); dgrad: [S][ldo] (K columns); wgrad: fp32 [E][N][K]
  int64_t ldo, stro;
  float* ws;  // grouped_ws_floats() of workspace, if any
  int split;  // parts of the reduction (set by grouped_gemm)
  float* db;  // wgrad: fp32 [E][N], or null
  int64_t S, T;  // slots, rows of x
  int E, N, K;
  int dtype;  // kBF16 or kF16
  int relu;
  int zero_rest;  // rows of out in no group are zeroed (else left as they were)
};
enum GroupedOp : int { kLinear = 0, kDgrad = 1, kWgrad = 2 };
int64_t grouped_ws_floats(GroupedOp op, const GroupedArgs& a);  // 0: none
// The kernels for whole 16-B words take the call (else the one for any width).
bool grouped_whole_words(GroupedOp op, const GroupedArgs& a);
hipError_t grouped_gemm(GroupedOp op, const GroupedArgs& a, hipStream_t s);

// ---- gated sum of a token's expert rows -------------------------------------
constexpr int kCombineMaxK = 16;
struct CombineArgs {
  const void* y;  // [S][ldy]
  int64_t ldy;
  const int32_t* slots;  // [T][k]
  const float* gates;    // [T][k], or null: 1
  void* out;             // [T][ldo]
  int64_t ldo;
  int64_t T, S;
  int N, k;
  int dtype;
};
hipError_t expert_combine(const CombineArgs& a, hipStream_t s);
struct CombineBwdArgs {
  const void* dout;  // [T][ldd]
  int64_t ldd;
  const void* y;  // [S][ldy]
  int64_t ldy;
  const int32_t* slots;    // [T][k]
  const int32_t* offsets;  // &offsets[E]: the slots in use
  const float* gates;      // [T][k]
  void* dy;                // [S][N] contiguous; slots behind *offsets are zeroed
  float* dgates;           // [T][k]
  int64_t T, S;
  int N, k;
  int dtype;
};
hipError_t expert_combine_backward(const CombineBwdArgs& a, hipStream_t s);

// ---- global gradient norm and clipping ----------------------------------------
struct ClipTensor {
  const void* g;
  void* out;  // == g: in place
  int64_t n;
};
// Doubles of workspace: the partial sums of `count` tensors.
int64_t grad_norm_ws_doubles(int count);
// norm[0] = sqrt(sum g^2); clip: out = g * min(1, max_norm / (norm + eps)).
hipError_t grad_norm(const ClipTensor* t, int count, int dtype, double* ws, float* norm, bool clip, double max_norm,
                     double eps, hipStream_t s);

}  // namespace dsml
