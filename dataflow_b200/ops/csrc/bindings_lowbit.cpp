// Torch-facing bindings of the narrow-format operators.  Every shape, type, stride and overlap check stands in front of the
// device check, so that a refusal can be tested on host tensors; a call that passes launches on the device of its operands and
// on that device's current stream.  Refused arguments raise ValueError.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>

#include "lowbit.h"

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

namespace {

#define REFUSE_UNLESS(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

bool aligned(const Tensor& t, size_t bytes) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & (bytes - 1)) == 0; }

// Two row-major matrices (rows of `width` elements, `pitch` apart) over common memory: the same matrix, or no common element?
struct Span {
  uintptr_t p;
  int64_t rows, width, pitch;      // bytes
};
Span span2d(const Tensor& t, int64_t rows, int64_t cols, int64_t ld) {
  const int64_t e = t.element_size();
  return {reinterpret_cast<uintptr_t>(t.const_data_ptr()), rows, cols * e, (rows > 1 ? ld : cols) * e};
}
bool same(const Span& a, const Span& b) { return a.p == b.p && a.rows == b.rows && a.width == b.width && (a.rows <= 1 || a.pitch == b.pitch); }
bool disjoint(const Span& a, const Span& b) {
  if (!a.rows || !b.rows || !a.width || !b.width) return true;
  const uintptr_t ae = a.p + (a.rows - 1) * a.pitch + a.width, be = b.p + (b.rows - 1) * b.pitch + b.width;
  if (ae <= b.p || be <= a.p) return true;
  if (a.pitch == b.pitch && a.rows > 1 && b.rows > 1) {      // column ranges of one buffer
    const Span &lo = a.p <= b.p ? a : b, &hi = a.p <= b.p ? b : a;
    const int64_t d = static_cast<int64_t>((hi.p - lo.p) % lo.pitch);
    return d >= lo.width && d + hi.width <= lo.pitch;
  }
  return false;
}

void on_device(const char* op, std::initializer_list<const Tensor*> ts) {
  const Tensor* first = *ts.begin();
  for (const Tensor* t : ts) REFUSE_UNLESS(t->device() == first->device(), op, ": operands are on different devices");
  REFUSE_UNLESS(first->is_cuda(), op, ": operands must be CUDA tensors");
}
Tensor empty_like_device(at::IntArrayRef sizes, at::ScalarType dt, const Tensor& t) {      // at::empty without the dispatcher
  return at::detail::empty_cuda(sizes, dt, t.device(), c10::nullopt);
}
int sms(const Tensor& t) { return at::cuda::getDeviceProperties(t.device().index())->multiProcessorCount; }
cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void launched(int rc, const char* op) { TORCH_CHECK(rc == 0, op, " failed to launch (code ", rc, ")"); }

// x as `rows` rows of its last axis: the common pitch of the rows, or a refusal
int64_t row_pitch(const char* op, const char* name, const Tensor& t, int64_t cols) {
  REFUSE_UNLESS(t.dim() >= 1 && t.size(-1) == cols, op, ": ", name, " has another width");
  if (t.numel() == 0) return cols;
  REFUSE_UNLESS(cols == 1 || t.stride(-1) == 1, op, ": the last axis of ", name, " must be contiguous");
  if (t.is_contiguous()) return cols;
  REFUSE_UNLESS(t.dim() == 2 && t.stride(0) >= cols, op, ": ", name, " is contiguous, or a matrix whose rows are strided");
  return t.stride(0);
}

int64_t tile_cols(int64_t K) { return 2 * ((K + 255) / 256); }
void check_mx(const char* op, const char* what, const Tensor& q, const Tensor& s) {
  REFUSE_UNLESS(q.dim() == 2 && q.scalar_type() == at::kByte && q.is_contiguous(), op, ": ", what, "codes are a contiguous (rows, K / 2) uint8 matrix");
  REFUSE_UNLESS(q.size(1) > 0 && q.size(1) % 16 == 0 && q.size(1) <= 65535 * 128, op, ": ", what, "codes cover a positive multiple of 32 elements per row");
  REFUSE_UNLESS(s.scalar_type() == at::kByte && s.is_contiguous() && s.dim() == 3 && s.size(0) == (q.size(0) + 127) / 128 &&
                    s.size(1) == tile_cols(2 * q.size(1)) && s.size(2) == 512,
                op, ": ", what, "scales are a contiguous uint8 tensor of shape (ceil(rows / 128), 2 ceil(K / 256), 512)");
  REFUSE_UNLESS(aligned(q, 16) && aligned(s, 16), op, ": ", what, "codes and scales must be 16-byte aligned");
}

// ---------------------------------------------------------------- 4-bit format
std::tuple<Tensor, Tensor> quant_mxfp4(const Tensor& x, bool transpose) {
  REFUSE_UNLESS(x.dim() == 2, "quant_mxfp4: x is a matrix");
  const bool f32 = x.scalar_type() == at::kFloat;
  REFUSE_UNLESS(f32 || x.scalar_type() == at::kBFloat16, "quant_mxfp4: x is bf16 or fp32");
  REFUSE_UNLESS(x.stride(1) == 1 || x.size(1) <= 1,
                "quant_mxfp4: the last axis of x must be contiguous (transpose=True takes a weight as it is stored)");
  const int64_t rows = transpose ? x.size(1) : x.size(0), K = transpose ? x.size(0) : x.size(1);
  REFUSE_UNLESS(K > 0 && K % 32 == 0, "quant_mxfp4: the contraction length must be a positive multiple of 32");
  REFUSE_UNLESS(K <= 65535 * 256, "quant_mxfp4: the contraction is too long (at most 16776960)");
  const int64_t ld = x.size(0) > 1 ? x.stride(0) : x.size(1);
  REFUSE_UNLESS(ld >= x.size(1), "quant_mxfp4: rows of x must not overlap");
  on_device("quant_mxfp4", {&x});
  c10::cuda::CUDAGuard guard(x.device());
  Tensor q = empty_like_device({rows, K / 2}, at::kByte, x), s = empty_like_device({(rows + 127) / 128, tile_cols(K), 512}, at::kByte, x);
  launched(dfb::quant_mxfp4(x.const_data_ptr(), ld, f32, transpose, q.data_ptr(), s.data_ptr(), rows, (int)K, stream_of(x)), "quant_mxfp4");
  return {q, s};
}

Tensor dequant_mxfp4(const Tensor& q, const Tensor& scale, at::ScalarType dt) {
  check_mx("dequant_mxfp4", "", q, scale);
  REFUSE_UNLESS(dt == at::kBFloat16 || dt == at::kFloat, "dequant_mxfp4: values are bf16 or fp32");
  on_device("dequant_mxfp4", {&q, &scale});
  c10::cuda::CUDAGuard guard(q.device());
  Tensor y = empty_like_device({q.size(0), q.size(1) * 2}, dt, q);
  launched(dfb::dequant_mxfp4(q.const_data_ptr(), scale.const_data_ptr(), y.data_ptr(), dt == at::kFloat, q.size(0), (int)q.size(1) * 2, stream_of(q)),
           "dequant_mxfp4");
  return y;
}

Tensor linear_mxfp4(const Tensor& xq, const Tensor& xs, const Tensor& wq, const Tensor& ws, const OptTensor& out, const OptTensor& add,
                    const OptTensor& bias, at::ScalarType out_dtype) {
  check_mx("linear_mxfp4", "x ", xq, xs);
  check_mx("linear_mxfp4", "w ", wq, ws);
  REFUSE_UNLESS(xq.size(1) == wq.size(1), "linear_mxfp4: both operands have the same K");
  const int64_t M = xq.size(0), N = wq.size(0);
  REFUSE_UNLESS(M <= 0x7fffffff - 256 && N <= 0x7fffffff - 256, "linear_mxfp4: too many rows");
  const at::ScalarType dt = out.has_value() ? out->scalar_type() : out_dtype;
  REFUSE_UNLESS(dt == at::kBFloat16 || dt == at::kFloat, "linear_mxfp4: the result is bf16 or fp32");
  auto like = [&](const Tensor& t, const char* msg) {
    REFUSE_UNLESS(t.dim() == 2 && t.size(0) == M && t.size(1) == N && t.scalar_type() == dt && (N <= 1 || t.stride(1) == 1) &&
                      (M <= 1 || t.stride(0) >= N), "linear_mxfp4: ", msg);
  };
  if (out.has_value()) like(*out, "out is (M, N) with contiguous rows");
  if (add.has_value()) like(*add, "add is like the result");
  if (bias.has_value())
    REFUSE_UNLESS(bias->dim() == 1 && bias->size(0) == N && bias->scalar_type() == at::kBFloat16 && bias->is_contiguous(), "linear_mxfp4: bias is (N,) bf16");
  auto ld = [&](const Tensor& t) { return M > 1 ? t.stride(0) : N; };
  if (out.has_value()) {
    const Span o = span2d(*out, M, N, ld(*out));
    if (add.has_value()) {
      const Span a = span2d(*add, M, N, ld(*add));
      REFUSE_UNLESS(same(o, a) || disjoint(o, a), "linear_mxfp4: out and add overlap without being the same matrix");
    }
    for (const Tensor* t : {&xq, &xs, &wq, &ws}) REFUSE_UNLESS(disjoint(o, span2d(*t, 1, t->numel(), t->numel())), "linear_mxfp4: out overlaps an operand");
    if (bias.has_value()) REFUSE_UNLESS(disjoint(o, span2d(*bias, 1, N, N)), "linear_mxfp4: out overlaps the bias");
  }
  on_device("linear_mxfp4", {&xq, &xs, &wq, &ws, out.has_value() ? &*out : &xq, add.has_value() ? &*add : &xq, bias.has_value() ? &*bias : &xq});
  c10::cuda::CUDAGuard guard(xq.device());
  Tensor d = out.has_value() ? *out : empty_like_device({M, N}, dt, xq);
  launched(dfb::gemm_mxfp4(xq.const_data_ptr(), xs.const_data_ptr(), wq.const_data_ptr(), ws.const_data_ptr(), d.data_ptr(), ld(d), dt == at::kFloat,
                           add.has_value() ? add->const_data_ptr() : nullptr, add.has_value() ? ld(*add) : 0,
                           bias.has_value() ? bias->const_data_ptr() : nullptr, M, N, (int)xq.size(1) * 2, sms(xq), stream_of(xq)),
           "linear_mxfp4");
  return d;
}

// ---------------------------------------------------------------- norm with a narrow output
std::tuple<Tensor, Tensor, Tensor, Tensor> rmsnorm_narrow(bool mx, const Tensor& x, const Tensor& w, double eps, const OptTensor& residual,
                                                          const OptTensor& rstd_in, const OptTensor& h_out) {
  const char* op = mx ? "rmsnorm_mxfp4" : "rmsnorm_fp8";
  const int64_t mult = mx ? 32 : 8, cols = x.dim() ? x.size(-1) : 0;
  REFUSE_UNLESS(cols > 0 && cols % mult == 0 && cols <= (1 << 30), op, ": the width must be a positive multiple of ", mult);
  const int64_t rows = x.numel() / cols;
  REFUSE_UNLESS(x.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16, op, ": x and w are bf16");
  REFUSE_UNLESS(w.dim() == 1 && w.size(0) == cols && w.is_contiguous(), op, ": w has one entry per column");
  auto operand = [&](const char* name, const Tensor& t) {
    REFUSE_UNLESS(t.sizes() == x.sizes() && t.scalar_type() == at::kBFloat16, op, ": ", name, " is like x");
    const int64_t ld = row_pitch(op, name, t, cols);
    REFUSE_UNLESS(aligned(t, 16) && (rows <= 1 || ld % 8 == 0), op, ": rows of ", name, " must be 16-byte aligned");
    return ld;
  };
  const int64_t ldx = operand("x", x);
  const int64_t ldr = residual.has_value() ? operand("residual", *residual) : 0;
  REFUSE_UNLESS(aligned(w, 16), op, ": w must be 16-byte aligned");
  REFUSE_UNLESS(!h_out.has_value() || residual.has_value(), op, ": h_out comes with a residual");
  if (rstd_in.has_value())
    REFUSE_UNLESS(rstd_in->scalar_type() == at::kFloat && rstd_in->numel() == rows && rstd_in->is_contiguous(), op, ": rstd has one fp32 entry per row");
  int64_t ldh = cols;
  if (h_out.has_value()) {
    ldh = operand("h_out", *h_out);
    const Span h = span2d(*h_out, rows, cols, ldh);
    for (const auto& [t, ld] : {std::make_pair(&x, ldx), std::make_pair(&*residual, ldr)}) {
      const Span s = span2d(*t, rows, cols, ld);
      REFUSE_UNLESS(same(h, s) || disjoint(h, s), op, ": h_out overlaps x or the residual without being the same matrix");
    }
    REFUSE_UNLESS(disjoint(h, span2d(w, 1, cols, cols)), op, ": h_out overlaps w");
    if (rstd_in.has_value()) REFUSE_UNLESS(disjoint(h, span2d(*rstd_in, 1, rows, rows)), op, ": h_out overlaps rstd");
  }
  on_device(op, {&x, &w, residual.has_value() ? &*residual : &x, rstd_in.has_value() ? &*rstd_in : &x, h_out.has_value() ? &*h_out : &x});
  c10::cuda::CUDAGuard guard(x.device());
  Tensor h = !residual.has_value() ? x : h_out.has_value() ? *h_out : empty_like_device(x.sizes(), at::kBFloat16, x);
  Tensor rstd = rstd_in.has_value() ? rstd_in->view({rows}) : empty_like_device({rows}, at::kFloat, x);
  float* rstd_out = rstd_in.has_value() ? nullptr : rstd.data_ptr<float>();
  const float* given = rstd_in.has_value() ? rstd_in->const_data_ptr<float>() : nullptr;
  const void* rp = residual.has_value() ? residual->const_data_ptr() : nullptr;
  void* hp = residual.has_value() ? h.data_ptr() : nullptr;
  if (mx) {
    Tensor q = empty_like_device({rows, cols / 2}, at::kByte, x), s = empty_like_device({(rows + 127) / 128, tile_cols(cols), 512}, at::kByte, x);
    launched(dfb::rmsnorm_mxfp4(x.const_data_ptr(), ldx, rp, ldr, w.const_data_ptr(), given, (float)eps, hp, ldh, q.data_ptr(), s.data_ptr(), rstd_out,
                                rows, (int)cols, sms(x), stream_of(x)), op);
    return {q, s, h, rstd};
  }
  Tensor q = empty_like_device(x.sizes(), at::kFloat8_e4m3fn, x), s = empty_like_device({rows}, at::kFloat, x);
  launched(dfb::rmsnorm_fp8(x.const_data_ptr(), ldx, rp, ldr, w.const_data_ptr(), given, (float)eps, hp, ldh, q.data_ptr(), s.data_ptr<float>(), rstd_out,
                            rows, (int)cols, sms(x), stream_of(x)), op);
  return {q, s, h, rstd};
}

// ---------------------------------------------------------------- AdamW over many tensors
void adamw_multi(const std::vector<Tensor>& ws, const std::vector<Tensor>& gs, const std::vector<Tensor>& ms, const std::vector<Tensor>& vs,
                 double lr, double b1, double b2, double eps, const std::vector<double>& wds, int64_t step,
                 const c10::optional<std::vector<Tensor>>& masters, const c10::optional<std::vector<Tensor>>& los,
                 const c10::optional<std::vector<Tensor>>& m_scales, const c10::optional<std::vector<Tensor>>& v_scales, double gscale,
                 int64_t seed, const c10::optional<std::vector<int64_t>>& seeds) {
  const char* op = "adamw_multi_step";
  const size_t n = ws.size();
  auto len = [&](const char* name, size_t k) { REFUSE_UNLESS(k == n, op, ": ", name, " has one entry per tensor"); };
  len("gs", gs.size()); len("ms", ms.size()); len("vs", vs.size()); len("wds", wds.size());
  if (masters.has_value()) len("masters", masters->size());
  if (los.has_value()) len("los", los->size());
  if (m_scales.has_value()) len("m_scales", m_scales->size());
  if (v_scales.has_value()) len("v_scales", v_scales->size());
  if (seeds.has_value()) len("seed", seeds->size());
  REFUSE_UNLESS(!(masters.has_value() && los.has_value()), op, ": masters and los exclude each other");
  REFUSE_UNLESS(step >= 1, op, ": step counts from 1");
  if (!n) return;
  const bool bits8 = ms[0].scalar_type() == at::kFloat8_e4m3fn;
  REFUSE_UNLESS(!bits8 || (m_scales.has_value() && v_scales.has_value()), op, ": 8-bit moments come with m_scales and v_scales");
  REFUSE_UNLESS(bits8 || !(m_scales.has_value() || v_scales.has_value()), op, ": scales belong to 8-bit moments");
  const at::ScalarType wt = ws[0].scalar_type(), gt = gs[0].scalar_type(), st = bits8 ? at::kFloat8_e4m3fn : at::kFloat;
  REFUSE_UNLESS(wt == at::kBFloat16 || wt == at::kFloat, op, ": weights are all bf16 or all fp32");
  REFUSE_UNLESS(gt == at::kBFloat16 || gt == at::kFloat, op, ": gradients are all bf16 or all fp32");
  REFUSE_UNLESS(!(masters.has_value() || los.has_value()) || wt == at::kBFloat16, op, ": masters and los go with bf16 weights");
  std::vector<dfb::AdamTensor> table;
  table.reserve(n);
  struct Range { uintptr_t lo, hi; bool written; };
  std::vector<Range> ranges;
  ranges.reserve(7 * n);
  const c10::Device dev = ws[0].device();
  auto take = [&](const Tensor& t, at::ScalarType dt, int64_t numel, const char* msg, bool written) {
    REFUSE_UNLESS(t.scalar_type() == dt, op, ": ", msg);
    REFUSE_UNLESS(t.numel() == numel, op, ": every operand of a tensor has its element count (scales: one per 128 elements)");
    REFUSE_UNLESS(t.is_contiguous(), op, ": operands are contiguous");
    REFUSE_UNLESS(t.device() == dev, op, ": operands are on different devices");
    void* p = const_cast<void*>(t.const_data_ptr());
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    if (numel) ranges.push_back({lo, lo + t.nbytes(), written});
    return p;
  };
  for (size_t i = 0; i < n; ++i) {
    const int64_t k = ws[i].numel(), nb = (k + 127) / 128;
    dfb::AdamTensor t{};
    t.n = k;
    t.wd = (float)wds[i];
    t.seed = static_cast<uint32_t>(seeds.has_value() ? (*seeds)[i] : seed);
    t.w = take(ws[i], wt, k, "weights are all bf16 or all fp32", true);
    t.g = take(gs[i], gt, k, "gradients are all bf16 or all fp32", false);
    t.m = take(ms[i], st, k, "moments are all fp32 or all float8_e4m3fn", true);
    t.v = take(vs[i], st, k, "moments are all fp32 or all float8_e4m3fn", true);
    if (masters.has_value()) t.extra = take((*masters)[i], at::kFloat, k, "masters are fp32", true);
    if (los.has_value()) t.extra = take((*los)[i], at::kShort, k, "los are int16", true);
    if (bits8) {
      t.m_scale = static_cast<float*>(take((*m_scales)[i], at::kFloat, nb, "scales are fp32, one per 128 elements", true));
      t.v_scale = static_cast<float*>(take((*v_scales)[i], at::kFloat, nb, "scales are fp32, one per 128 elements", true));
    }
    if (k) table.push_back(t);
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  uintptr_t end_written = 0, end_any = 0;
  for (const Range& r : ranges) {
    REFUSE_UNLESS(r.lo >= end_written && (!r.written || r.lo >= end_any), op, ": a tensor that is written appears twice or overlaps another");
    if (r.written) end_written = std::max(end_written, r.hi);
    end_any = std::max(end_any, r.hi);
  }
  REFUSE_UNLESS(dev.is_cuda(), op, ": operands must be CUDA tensors");
  if (table.empty()) return;
  c10::cuda::CUDAGuard guard(dev);
  dfb::AdamHyper h;
  h.lr = (float)lr;
  h.b1 = (float)b1; h.c1 = (float)(1.0 - b1);
  h.b2 = (float)b2; h.c2 = (float)(1.0 - b2);
  h.eps = (float)eps;
  h.inv_bc1 = (float)(1.0 / (1.0 - std::pow(b1, (double)step)));
  h.inv_sqrt_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(b2, (double)step)));
  h.gscale = (float)gscale;
  const int weights = masters.has_value() ? dfb::kAdamMaster : los.has_value() ? dfb::kAdamSplit : wt == at::kFloat ? dfb::kAdamF32 : dfb::kAdamBf16;
  launched(dfb::adamw_multi(table.data(), (int)table.size(), weights, gt == at::kFloat, bits8, h, sms(ws[0]), stream_of(ws[0])), op);
}

at::ScalarType dtype_of(const py::object& o) { return torch::python::detail::py_object_to_dtype(o); }

}  // namespace

void bind_lowbit(py::module& m) {
  m.def("quant_mxfp4", &quant_mxfp4);
  m.def("dequant_mxfp4", [](const Tensor& q, const Tensor& s, const py::object& dt) { return dequant_mxfp4(q, s, dtype_of(dt)); });
  m.def("linear_mxfp4", [](const Tensor& xq, const Tensor& xs, const Tensor& wq, const Tensor& ws, const OptTensor& out, const OptTensor& add,
                           const OptTensor& bias, const py::object& dt) { return linear_mxfp4(xq, xs, wq, ws, out, add, bias, dtype_of(dt)); });
  m.def("rmsnorm_fp8", [](const Tensor& x, const Tensor& w, double eps, const OptTensor& res, const OptTensor& rstd, const OptTensor& h) {
    return rmsnorm_narrow(false, x, w, eps, res, rstd, h);
  });
  m.def("rmsnorm_mxfp4", [](const Tensor& x, const Tensor& w, double eps, const OptTensor& res, const OptTensor& rstd, const OptTensor& h) {
    return rmsnorm_narrow(true, x, w, eps, res, rstd, h);
  });
  m.def("adamw_multi", &adamw_multi);
  m.def("gemm_mxfp4_last_error", []() { return (int64_t)dfb::gemm_mxfp4_last_error(); });
}
