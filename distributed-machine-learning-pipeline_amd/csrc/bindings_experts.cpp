// Bindings of the expert-layer operators and gradient clipping.
//
// Shapes, types and strides are checked before the device, so the refusals can
// be exercised on host tensors; nothing is launched unless every check passed.
// A call runs on its tensors' device and that device's current stream, with
// workspaces from the caching allocator of that stream.
#include <ATen/hip/HIPContext.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <algorithm>

#include "dsml.h"
#include "experts.h"

namespace py = pybind11;
using namespace dsml;

namespace {

using Opt = c10::optional<torch::Tensor>;

void ex_hip_ok(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

// The call's device made current, and its current stream.
struct OnDevice {
  int prev = -1;
  hipStream_t stream;
  explicit OnDevice(const torch::Tensor& t) {
    const int d = t.get_device();
    ex_hip_ok(hipGetDevice(&prev), "hipGetDevice");
    if (d == prev) prev = -1;
    else ex_hip_ok(hipSetDevice(d), "hipSetDevice");
    stream = at::hip::getCurrentHIPStream((c10::DeviceIndex)d).stream();
  }
  ~OnDevice() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
};

void check_gpu(std::initializer_list<const torch::Tensor*> ts) {
  const torch::Tensor* first = *ts.begin();
  for (const torch::Tensor* t : ts) {
    if (!t) continue;
    TORCH_CHECK(t->is_cuda(), "operands must be GPU tensors");
    TORCH_CHECK(t->get_device() == first->get_device(), "operands must be on one GPU");
  }
}

// No call here is recorded by autograd: an operand that requires a gradient would
// lose it without a word.
void check_unrecorded(std::initializer_list<const torch::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return;
  for (const torch::Tensor* t : ts)
    TORCH_CHECK(!t || !t->requires_grad(),
                "an operand requires a gradient, and autograd does not record this call: make it under "
                "torch.no_grad(), with the explicit gradient calls, or detach the operand");
}

int32_t half_type(const torch::Tensor& t, const char* name) {
  if (t.scalar_type() == torch::kBFloat16) return kBF16;
  TORCH_CHECK(t.scalar_type() == torch::kFloat16, name, " must be bfloat16 or float16");
  return kF16;
}
int32_t float_type(const torch::Tensor& t, const char* name) {
  if (t.scalar_type() == torch::kFloat32) return kF32;
  if (t.scalar_type() == torch::kBFloat16) return kBF16;
  TORCH_CHECK(t.scalar_type() == torch::kFloat16, name, " must be float32, bfloat16 or float16");
  return kF16;
}
// Rows of `dim` axes with a contiguous last axis.
void check_rows(const torch::Tensor& t, int64_t dim, const char* name) {
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " axes, got ", t.dim());
  TORCH_CHECK(t.size(dim - 1) <= 1 || t.stride(dim - 1) == 1, name, ": the last axis must be contiguous");
}
void check_i32(const torch::Tensor& t, int64_t n, const char* name) {
  TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.numel() == n, name, " must hold ", n, " values, got ", t.numel());
}
void check_f32_plain(const torch::Tensor& t, int64_t n, const char* name) {
  TORCH_CHECK(t.scalar_type() == torch::kFloat32, name, " must be float32");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.numel() == n, name, " must hold ", n, " values, got ", t.numel());
}
// An output written by many lanes: no two of its elements share memory.
void check_out_rows(const torch::Tensor& t, int64_t rows, int64_t cols, const char* name) {
  check_rows(t, 2, name);
  TORCH_CHECK(t.size(0) == rows && t.size(1) == cols, name, " must be [", rows, ", ", cols, "]");
  TORCH_CHECK(rows <= 1 || t.stride(0) >= cols, name, ": rows must not overlap");
}
struct Span { const char* lo; const char* hi; };
Span span_of(const torch::Tensor& t) {
  const char* p = static_cast<const char*>(t.data_ptr());
  if (t.numel() == 0) return {p, p};
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {p, p + (last + 1) * t.element_size()};
}
bool meets(const torch::Tensor& a, const torch::Tensor& b) {
  const Span x = span_of(a), y = span_of(b);
  if (x.lo >= y.hi || y.lo >= x.hi) return false;
  // column ranges of one buffer lie apart though their spans do not
  if (a.dim() != 2 || b.dim() != 2) return true;
  const int64_t ea = a.element_size(), eb = b.element_size();
  const int64_t ld = a.size(0) > 1 ? a.stride(0) * ea : b.stride(0) * eb;
  if (ld <= 0 || (b.size(0) > 1 && b.stride(0) * eb != ld)) return true;
  const int64_t wa = a.size(1) * ea, wb = b.size(1) * eb;
  const int64_t at = ((y.lo - x.lo) % ld + ld) % ld;  // b's first column, from a's
  return at < wa || at + wb > ld;
}
void check_apart(const torch::Tensor& out, std::initializer_list<const torch::Tensor*> ins, const char* name) {
  for (const torch::Tensor* t : ins) TORCH_CHECK(!t || !meets(out, *t), name, " must not overlap an input");
}
const torch::Tensor* opt(const Opt& t) { return t ? &*t : nullptr; }
int64_t row_stride(const torch::Tensor& t, int64_t axis) { return t.size(axis) > 1 ? t.stride(axis) : t.size(axis + 1); }
void check_count(int64_t n, const char* name) {
  TORCH_CHECK(n <= 0x7fffffffLL, name, ": more than 2^31 - 1 rows");
}

bool whole_row(const std::string& normalize) {
  TORCH_CHECK(normalize == "topk" || normalize == "all", "normalize must be 'topk' or 'all', got '", normalize, "'");
  return normalize == "all";
}

// ---- router -------------------------------------------------------------
py::tuple py_route_topk(const torch::Tensor& logits, int64_t k, const std::string& normalize) {
  check_unrecorded({&logits});
  check_rows(logits, 2, "logits");
  const int64_t T = logits.size(0), E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= kRouteMaxExperts, "route_topk: 1..", kRouteMaxExperts, " experts, got ", E);
  TORCH_CHECK(k >= 1 && k <= std::min<int64_t>(E, kRouteMaxK), "route_topk: k must be 1..min(", kRouteMaxK,
              ", experts), got ", k);
  check_count(T * k, "route_topk");
  RouteArgs a{};
  a.all = whole_row(normalize);
  a.dtype = float_type(logits, "logits");
  check_gpu({&logits});
  OnDevice on(logits);
  const auto i32 = logits.options().dtype(torch::kInt32);
  torch::Tensor gates = torch::empty({T, k}, logits.options().dtype(torch::kFloat32));
  torch::Tensor experts = torch::empty({T, k}, i32), offsets = torch::empty({E + 1}, i32);
  torch::Tensor rows = torch::empty({T * k}, i32), slots = torch::empty({T, k}, i32);
  const int64_t words = T > 256 ? route_ws_words(T, (int)E) : 0;
  torch::Tensor ws;
  if (words) ws = torch::empty({words}, i32);
  a.logits = logits.data_ptr(); a.ldl = row_stride(logits, 0); a.T = T; a.E = (int)E; a.k = (int)k;
  a.gates = gates.data_ptr<float>(); a.experts = experts.data_ptr<int32_t>();
  a.offsets = offsets.data_ptr<int32_t>(); a.rows = rows.data_ptr<int32_t>(); a.slots = slots.data_ptr<int32_t>();
  a.counts = words ? ws.data_ptr<int32_t>() : nullptr;
  ex_hip_ok(route_topk(a, on.stream), "route_topk");
  return py::make_tuple(gates, experts, offsets, rows, slots);
}

torch::Tensor py_route_backward(const torch::Tensor& dgates, const torch::Tensor& logits, const torch::Tensor& gates,
                                const torch::Tensor& experts, const std::string& normalize) {
  check_unrecorded({&logits, &dgates, &gates});
  check_rows(logits, 2, "logits");
  TORCH_CHECK(dgates.dim() == 2, "dgates must have 2 axes, got ", dgates.dim());
  const int64_t T = logits.size(0), E = logits.size(1), k = dgates.size(1);
  TORCH_CHECK(E >= 1 && E <= kRouteMaxExperts, "route_topk_backward: 1..", kRouteMaxExperts, " experts, got ", E);
  TORCH_CHECK(k >= 1 && k <= std::min<int64_t>(E, kRouteMaxK), "route_topk_backward: k must be 1..min(", kRouteMaxK,
              ", experts), got ", k);
  check_count(T * k, "route_topk_backward");
  check_f32_plain(dgates, T * k, "dgates");
  check_f32_plain(gates, T * k, "gates");
  check_i32(experts, T * k, "experts");
  RouteBwdArgs a{};
  a.all = whole_row(normalize);
  a.dtype = float_type(logits, "logits");
  check_gpu({&logits, &dgates, &gates, &experts});
  OnDevice on(logits);
  torch::Tensor out = torch::empty({T, E}, logits.options());
  a.logits = logits.data_ptr(); a.ldl = row_stride(logits, 0); a.gates = gates.data_ptr<float>();
  a.experts = experts.data_ptr<int32_t>(); a.dgates = dgates.data_ptr<float>(); a.dlogits = out.data_ptr();
  a.T = T; a.E = (int)E; a.k = (int)k;
  ex_hip_ok(route_topk_backward(a, on.stream), "route_topk_backward");
  return out;
}

// ---- products grouped by expert -------------------------------------------
void check_weights(const torch::Tensor& w) {
  check_rows(w, 3, "w");
  TORCH_CHECK(w.size(0) >= 1 && w.size(1) >= 1 && w.size(2) >= 1, "w must be [experts, out, in], none of them 0");
  TORCH_CHECK(w.size(1) <= 0xffffff && w.size(2) <= 0xffffff && w.size(0) <= 0xffff, "w is too large in one axis");
}

void run_grouped(GroupedOp op, GroupedArgs& a, const torch::Tensor& like, const char* what) {
  OnDevice on(like);
  torch::Tensor ws;
  if (const int64_t words = grouped_ws_floats(op, a)) {
    ws = torch::empty({words}, like.options().dtype(torch::kFloat32));
    a.ws = ws.data_ptr<float>();
  }
  ex_hip_ok(grouped_gemm(op, a, on.stream), what);
}

torch::Tensor py_grouped_linear(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& offsets,
                                const Opt& bias, bool relu, const Opt& rows, const Opt& out) {
  check_unrecorded({&x, &w, opt(bias), opt(out)});
  check_rows(x, 2, "x");
  check_weights(w);
  const int64_t E = w.size(0), N = w.size(1), K = w.size(2);
  GroupedArgs a{};
  a.dtype = half_type(x, "x");
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), "w must have x's type");
  TORCH_CHECK(x.size(1) == K, "x has ", x.size(1), " columns, w takes ", K);
  check_i32(offsets, E + 1, "offsets");
  if (rows) {
    TORCH_CHECK(rows->dim() == 1, "rows must have 1 axis");
    check_i32(*rows, rows->numel(), "rows");
  }
  const int64_t S = rows ? rows->numel() : x.size(0);
  check_count(S, "grouped_linear");
  check_count(x.size(0), "grouped_linear");
  if (bias) {
    check_rows(*bias, 2, "bias");
    TORCH_CHECK(bias->scalar_type() == torch::kFloat32, "bias must be float32");
    TORCH_CHECK(bias->size(0) == E && bias->size(1) == N, "bias must be [", E, ", ", N, "]");
  }
  if (out) {
    TORCH_CHECK(out->scalar_type() == x.scalar_type(), "out must have x's type");
    check_out_rows(*out, S, N, "out");
    check_apart(*out, {&x, &w, &offsets, opt(bias), opt(rows)}, "out");
  }
  check_gpu({&x, &w, &offsets, opt(bias), opt(rows), opt(out)});
  torch::Tensor y = out ? *out : torch::empty({S, N}, x.options());
  a.a = x.data_ptr(); a.lda = row_stride(x, 0); a.T = x.size(0);
  a.b = w.data_ptr(); a.ldb = row_stride(w, 1); a.strb = E > 1 ? w.stride(0) : 0;
  a.offsets = offsets.data_ptr<int32_t>();
  a.rows = rows ? rows->data_ptr<int32_t>() : nullptr;
  if (bias) { a.bias = bias->data_ptr<float>(); a.ldbias = row_stride(*bias, 0); }
  a.relu = relu; a.out = y.data_ptr(); a.ldo = row_stride(y, 0);
  a.S = S; a.E = (int)E; a.N = (int)N; a.K = (int)K; a.zero_rest = out ? 0 : 1;
  run_grouped(kLinear, a, x, "grouped_linear");
  return y;
}

torch::Tensor py_grouped_dgrad(const torch::Tensor& dz, const torch::Tensor& w, const torch::Tensor& offsets,
                               const Opt& mask, const Opt& out) {
  check_unrecorded({&dz, &w, opt(mask), opt(out)});
  check_rows(dz, 2, "dz");
  check_weights(w);
  const int64_t E = w.size(0), N = w.size(1), K = w.size(2), S = dz.size(0);
  GroupedArgs a{};
  a.dtype = half_type(dz, "dz");
  TORCH_CHECK(w.scalar_type() == dz.scalar_type(), "w must have dz's type");
  TORCH_CHECK(dz.size(1) == N, "dz has ", dz.size(1), " columns, w gives ", N);
  check_i32(offsets, E + 1, "offsets");
  check_count(S, "grouped_dgrad");
  if (mask) {
    check_rows(*mask, 2, "mask");
    TORCH_CHECK(mask->scalar_type() == dz.scalar_type(), "mask must have dz's type");
    TORCH_CHECK(mask->size(0) == S && mask->size(1) == K, "mask must be [", S, ", ", K, "]");
  }
  if (out) {
    TORCH_CHECK(out->scalar_type() == dz.scalar_type(), "out must have dz's type");
    check_out_rows(*out, S, K, "out");
    check_apart(*out, {&dz, &w, &offsets, opt(mask)}, "out");
  }
  check_gpu({&dz, &w, &offsets, opt(mask), opt(out)});
  torch::Tensor dx = out ? *out : torch::empty({S, K}, dz.options());
  a.a = dz.data_ptr(); a.lda = row_stride(dz, 0); a.T = S;
  a.b = w.data_ptr(); a.ldb = row_stride(w, 1); a.strb = E > 1 ? w.stride(0) : 0;
  a.offsets = offsets.data_ptr<int32_t>();
  if (mask) { a.mask = mask->data_ptr(); a.ldmask = row_stride(*mask, 0); }
  a.out = dx.data_ptr(); a.ldo = row_stride(dx, 0);
  a.S = S; a.E = (int)E; a.N = (int)N; a.K = (int)K; a.zero_rest = out ? 0 : 1;
  run_grouped(kDgrad, a, dz, "grouped_dgrad");
  return dx;
}

py::tuple py_grouped_wgrad(const torch::Tensor& dz, const torch::Tensor& x, const torch::Tensor& offsets,
                           const Opt& rows, bool bias, const Opt& dw_out, const Opt& db_out) {
  check_unrecorded({&dz, &x, opt(dw_out), opt(db_out)});
  check_rows(dz, 2, "dz");
  check_rows(x, 2, "x");
  GroupedArgs a{};
  a.dtype = half_type(dz, "dz");
  TORCH_CHECK(x.scalar_type() == dz.scalar_type(), "x must have dz's type");
  TORCH_CHECK(offsets.dim() == 1 && offsets.numel() >= 2, "offsets must have 1 axis and hold experts + 1 values");
  const int64_t E = offsets.numel() - 1, S = dz.size(0), N = dz.size(1), K = x.size(1);
  check_i32(offsets, E + 1, "offsets");
  TORCH_CHECK(N >= 1 && K >= 1 && N <= 0xffffff && K <= 0xffffff && E <= 0xffff, "grouped_wgrad: bad sizes");
  if (rows) {
    TORCH_CHECK(rows->dim() == 1, "rows must have 1 axis");
    check_i32(*rows, S, "rows");
  } else {
    TORCH_CHECK(x.size(0) == S, "x has ", x.size(0), " rows, dz ", S);
  }
  // the reduction's steps of 64, two ahead of the last, are counted in 32 bits
  TORCH_CHECK(S <= 0x7fffffffLL - 255, "grouped_wgrad: more than 2^31 - 256 rows");
  check_count(x.size(0), "grouped_wgrad");
  TORCH_CHECK(bias || !db_out, "a bias gradient buffer was given with bias=False");
  if (dw_out) {
    check_rows(*dw_out, 3, "dw");
    TORCH_CHECK(dw_out->scalar_type() == torch::kFloat32, "dw must be float32");
    TORCH_CHECK(dw_out->size(0) == E && dw_out->size(1) == N && dw_out->size(2) == K, "dw must be [", E, ", ", N, ", ",
                K, "]");
    TORCH_CHECK((N <= 1 || dw_out->stride(1) >= K) && (E <= 1 || dw_out->stride(0) >= (N - 1) * row_stride(*dw_out, 1) + K),
                "dw: rows must not overlap");
    check_apart(*dw_out, {&dz, &x, &offsets, opt(rows), opt(db_out)}, "dw");
  }
  if (db_out) {
    check_f32_plain(*db_out, E * N, "db");
    check_apart(*db_out, {&dz, &x, &offsets, opt(rows)}, "db");
  }
  check_gpu({&dz, &x, &offsets, opt(rows), opt(dw_out), opt(db_out)});
  const auto f32 = dz.options().dtype(torch::kFloat32);
  torch::Tensor dw = dw_out ? *dw_out : torch::empty({E, N, K}, f32);
  Opt db;
  if (bias) db = db_out ? *db_out : torch::empty({E, N}, f32);
  a.a = dz.data_ptr(); a.lda = row_stride(dz, 0); a.b = x.data_ptr(); a.ldb = row_stride(x, 0);
  a.offsets = offsets.data_ptr<int32_t>();
  a.rows = rows ? rows->data_ptr<int32_t>() : nullptr;
  a.out = dw.data_ptr(); a.ldo = row_stride(dw, 1); a.stro = E > 1 ? dw.stride(0) : 0;
  a.db = db ? db->data_ptr<float>() : nullptr;
  a.S = S; a.T = x.size(0); a.E = (int)E; a.N = (int)N; a.K = (int)K;
  run_grouped(kWgrad, a, dz, "grouped_wgrad");
  return py::make_tuple(dw, db);
}

// Which kernels contiguous, aligned operands of these sizes go to.
bool py_grouped_whole_words(const std::string& op, int64_t S, int64_t T, int E, int N, int K, bool gathered) {
  TORCH_CHECK(op == "linear" || op == "dgrad" || op == "wgrad", "op must be 'linear', 'dgrad' or 'wgrad', got '", op, "'");
  const GroupedOp o = op == "linear" ? kLinear : op == "dgrad" ? kDgrad : kWgrad;
  const int32_t id = 0;
  GroupedArgs a{};
  a.lda = o == kLinear ? K : N;
  a.ldb = K;
  a.strb = (int64_t)N * K;
  a.rows = gathered ? &id : nullptr;
  a.ldo = o == kLinear ? N : K;
  a.stro = (int64_t)N * K;
  a.S = S; a.T = T; a.E = E; a.N = N; a.K = K; a.dtype = kBF16;
  return grouped_whole_words(o, a);
}

// ---- combine ---------------------------------------------------------------
void check_slots(const torch::Tensor& slots, int64_t* T, int64_t* k, const char* what) {
  TORCH_CHECK(slots.dim() == 2, "slots must have 2 axes, got ", slots.dim());
  *T = slots.size(0);
  *k = slots.size(1);
  TORCH_CHECK(*k >= 1 && *k <= kCombineMaxK, what, ": k must be 1..", kCombineMaxK, ", got ", *k);
  check_count(*T * *k, what);
  check_i32(slots, *T * *k, "slots");
}

torch::Tensor py_combine(const torch::Tensor& y, const torch::Tensor& slots, const Opt& gates, const Opt& out) {
  check_unrecorded({&y, opt(gates), opt(out)});
  check_rows(y, 2, "y");
  CombineArgs a{};
  a.dtype = half_type(y, "y");
  int64_t T, k;
  check_slots(slots, &T, &k, "expert_combine");
  const int64_t N = y.size(1);
  TORCH_CHECK(N >= 1 && N <= 0x3fffff, "expert_combine: 1..4194303 columns");
  check_count(y.size(0), "expert_combine");
  if (gates) check_f32_plain(*gates, T * k, "gates");
  if (out) {
    TORCH_CHECK(out->scalar_type() == y.scalar_type(), "out must have y's type");
    check_out_rows(*out, T, N, "out");
    check_apart(*out, {&y, &slots, opt(gates)}, "out");
  }
  check_gpu({&y, &slots, opt(gates), opt(out)});
  OnDevice on(y);
  torch::Tensor o = out ? *out : torch::empty({T, N}, y.options());
  a.y = y.data_ptr(); a.ldy = row_stride(y, 0); a.slots = slots.data_ptr<int32_t>();
  a.gates = gates ? gates->data_ptr<float>() : nullptr;
  a.out = o.data_ptr(); a.ldo = row_stride(o, 0);
  a.T = T; a.S = y.size(0); a.N = (int)N; a.k = (int)k;
  ex_hip_ok(expert_combine(a, on.stream), "expert_combine");
  return o;
}

py::tuple py_combine_backward(const torch::Tensor& dout, const torch::Tensor& y, const torch::Tensor& slots,
                              const torch::Tensor& gates, const torch::Tensor& offsets) {
  check_unrecorded({&dout, &y, &gates});
  check_rows(dout, 2, "dout");
  check_rows(y, 2, "y");
  CombineBwdArgs a{};
  a.dtype = half_type(y, "y");
  TORCH_CHECK(dout.scalar_type() == y.scalar_type(), "dout must have y's type");
  int64_t T, k;
  check_slots(slots, &T, &k, "expert_combine_backward");
  const int64_t N = y.size(1), S = y.size(0);
  TORCH_CHECK(N >= 1 && N <= 0x3fffff, "expert_combine_backward: 1..4194303 columns");
  TORCH_CHECK(dout.size(0) == T && dout.size(1) == N, "dout must be [", T, ", ", N, "]");
  TORCH_CHECK(S == T * k, "y must have one row a slot: ", T * k, ", got ", S);
  check_f32_plain(gates, T * k, "gates");
  TORCH_CHECK(offsets.dim() == 1 && offsets.numel() >= 2, "offsets must have 1 axis and hold experts + 1 values");
  check_i32(offsets, offsets.numel(), "offsets");
  check_gpu({&y, &dout, &slots, &gates, &offsets});
  OnDevice on(y);
  torch::Tensor dy = torch::empty({S, N}, y.options()), dg = torch::empty({T, k}, gates.options());
  a.dout = dout.data_ptr(); a.ldd = row_stride(dout, 0); a.y = y.data_ptr(); a.ldy = row_stride(y, 0);
  a.slots = slots.data_ptr<int32_t>(); a.offsets = offsets.data_ptr<int32_t>() + offsets.numel() - 1;
  a.gates = gates.data_ptr<float>(); a.dy = dy.data_ptr(); a.dgates = dg.data_ptr<float>();
  a.T = T; a.S = S; a.N = (int)N; a.k = (int)k;
  ex_hip_ok(expert_combine_backward(a, on.stream), "expert_combine_backward");
  return py::make_tuple(dy, dg);
}

// ---- gradient norm -----------------------------------------------------------
torch::Tensor py_grad_norm(const std::vector<torch::Tensor>& grads, bool clip, double max_norm, double eps,
                           const c10::optional<std::vector<torch::Tensor>>& out) {
  TORCH_CHECK(!grads.empty(), "no gradients given");
  TORCH_CHECK(!clip || max_norm >= 0.0, "max_norm must not be negative, got ", max_norm);
  TORCH_CHECK(!clip || eps >= 0.0, "eps must not be negative, got ", eps);
  const int32_t dt = float_type(grads[0], "gradients");
  TORCH_CHECK(!out || out->size() == grads.size(), "out must hold one tensor a gradient");
  std::vector<ClipTensor> t(grads.size());
  bool gpu = true;
  for (size_t i = 0; i < grads.size(); ++i) {
    const torch::Tensor& g = grads[i];
    check_unrecorded({&g, out ? &(*out)[i] : nullptr});
    TORCH_CHECK(g.scalar_type() == grads[0].scalar_type(), "gradients must have one type");
    TORCH_CHECK(g.is_contiguous(), "gradients must be contiguous");
    const torch::Tensor& o = out ? (*out)[i] : g;
    if (out) {
      TORCH_CHECK(o.scalar_type() == g.scalar_type(), "out must have the gradients' type");
      TORCH_CHECK(o.is_contiguous() && o.sizes() == g.sizes(), "out must be contiguous and of the gradients' shapes");
    }
    gpu = gpu && g.is_cuda() && o.is_cuda() && g.get_device() == grads[0].get_device() &&
          o.get_device() == grads[0].get_device();
    t[i] = ClipTensor{g.data_ptr(), o.data_ptr(), g.numel()};
  }
  if (clip) {
    // what is written must be written once, and not read as another gradient
    struct Iv { const char* lo; const char* hi; size_t i; bool w; };
    std::vector<Iv> iv;
    const int64_t es = grads[0].element_size();
    for (size_t i = 0; i < t.size(); ++i) {
      if (t[i].n == 0) continue;
      const char* o = static_cast<const char*>(t[i].out);
      iv.push_back({o, o + t[i].n * es, i, true});
      if (t[i].out != t[i].g) {
        const char* g = static_cast<const char*>(t[i].g);
        iv.push_back({g, g + t[i].n * es, i, false});
      }
    }
    std::sort(iv.begin(), iv.end(), [](const Iv& x, const Iv& y) { return x.lo < y.lo; });
    const char *end_w = nullptr, *end_r = nullptr;
    for (const Iv& v : iv) {
      TORCH_CHECK(v.lo >= end_w && (!v.w || v.lo >= end_r), "clipped gradients must not overlap");
      if (v.w) end_w = std::max(end_w, v.hi);
      else end_r = std::max(end_r, v.hi);
    }
  }
  TORCH_CHECK(gpu, "gradients must be on one GPU");
  OnDevice on(grads[0]);
  const int64_t words = grad_norm_ws_doubles((int)t.size());
  torch::Tensor ws = torch::empty({words}, grads[0].options().dtype(torch::kFloat64));
  torch::Tensor norm = torch::empty({}, grads[0].options().dtype(torch::kFloat32));
  ex_hip_ok(grad_norm(t.data(), (int)t.size(), dt, ws.data_ptr<double>(), norm.data_ptr<float>(), clip, max_norm, eps,
                      on.stream),
            "grad_norm");
  return norm;
}

}  // namespace

void bind_experts(py::module_& m) {
  m.def("route_topk", &py_route_topk, py::arg("logits"), py::arg("k"), py::arg("normalize") = "topk",
        "(gates, experts, offsets, rows, slots) of the k largest logits of every row (kernels/route.hip)");
  m.def("route_topk_backward", &py_route_backward, py::arg("dgates"), py::arg("logits"), py::arg("gates"),
        py::arg("experts"), py::arg("normalize") = "topk");
  m.def("grouped_linear", &py_grouped_linear, py::arg("x"), py::arg("w"), py::arg("offsets"),
        py::arg("bias") = py::none(), py::arg("relu") = false, py::arg("rows") = py::none(),
        py::arg("out") = py::none(), "products grouped by expert (kernels/grouped_gemm.hip)");
  m.def("grouped_dgrad", &py_grouped_dgrad, py::arg("dz"), py::arg("w"), py::arg("offsets"),
        py::arg("mask") = py::none(), py::arg("out") = py::none());
  m.def("grouped_wgrad", &py_grouped_wgrad, py::arg("dz"), py::arg("x"), py::arg("offsets"),
        py::arg("rows") = py::none(), py::arg("bias") = true, py::arg("dw") = py::none(), py::arg("db") = py::none());
  m.def("grouped_whole_words", &py_grouped_whole_words, py::arg("op"), py::arg("S"), py::arg("T"), py::arg("E"),
        py::arg("N"), py::arg("K"), py::arg("gathered") = false,
        "whether contiguous operands of these sizes go to the kernels for whole 16-B words");
  m.def("expert_combine", &py_combine, py::arg("y"), py::arg("slots"), py::arg("gates") = py::none(),
        py::arg("out") = py::none());
  m.def("expert_combine_backward", &py_combine_backward, py::arg("dout"), py::arg("y"), py::arg("slots"),
        py::arg("gates"), py::arg("offsets"));
  m.def("grad_norm", &py_grad_norm, py::arg("grads"), py::arg("clip") = false, py::arg("max_norm") = 0.0,
        py::arg("eps") = 1e-6, py::arg("out") = py::none(),
        "global norm of the gradients; clip: scaled by min(1, max_norm / (norm + eps)) (kernels/grad_clip.hip)");
}
