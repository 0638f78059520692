// torch glue for fp8_ops.cu and fp8_gemm_sm100.cu: checks and stream selection.  Outputs are allocated
// by the caller (elf_b200/ops/fp8.py), which knows the row pitches the products need.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "fp8_ops.h"

namespace {

cudaStream_t cur() { return at::cuda::getCurrentCUDAStream(); }

void check(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, "elf_b200 ", what, ": ", cudaGetErrorString(e)); }

elfb::Elem elem_of(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return elfb::Elem::kBf16;
  if (t.scalar_type() == at::kHalf) return elfb::Elem::kF16;
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be bf16, fp16 or fp32, got ", t.scalar_type());
  return elfb::Elem::kF32;
}

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

void need_matrix(const at::Tensor& t, const char* name, const at::Device& dev) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, name, " must be a CUDA tensor on ", dev);
  TORCH_CHECK(t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1), name, " must be a matrix with a contiguous last dimension");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " must not overlap itself");
  TORCH_CHECK(t.size(0) <= INT_MAX - 1024 && t.size(1) <= INT_MAX - 1024, name, " is too large");
}

void need_scaled(const at::Tensor& data, const at::Tensor& scale, int64_t row_shift, const char* name, const at::Device& dev) {
  need_matrix(data, name, dev);
  need_matrix(scale, "scale", dev);
  TORCH_CHECK(data.element_size() == 1 && scale.element_size() == 1, name, " must hold 8-bit values and exponents");
  TORCH_CHECK(row_shift == 0 || row_shift == 7, "scales belong to rows or to tiles of 128 rows");
  const int64_t rows = row_shift ? blocks_of(data.size(0)) : data.size(0);
  TORCH_CHECK(scale.size(0) == rows && scale.size(1) == blocks_of(data.size(1)), name, ": expected scales [", rows, ", ", blocks_of(data.size(1)), "], got ",
              scale.sizes());
}

uint8_t* bytes(const at::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }
int64_t pitch(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.stride(0), t.size(1)); }

void quantize(const at::Tensor& x, at::Tensor& data, at::Tensor& scale, bool tiles) {
  const auto dev = data.device();
  need_matrix(x, "x", dev);
  need_scaled(data, scale, tiles ? 7 : 0, "data", dev);
  TORCH_CHECK(x.sizes() == data.sizes(), "x and data must have the same shape");
  c10::cuda::CUDAGuard g(dev);
  auto* fn = tiles ? elfb::fp8_quantize_tiles : elfb::fp8_quantize_rows;
  check(fn(x.data_ptr(), elem_of(x, "x"), pitch(x), bytes(data), pitch(data), bytes(scale), pitch(scale), x.size(0), int(x.size(1)), cur()), "fp8_quantize");
}

void dequantize(const at::Tensor& data, const at::Tensor& scale, int64_t row_shift, at::Tensor& out) {
  const auto dev = data.device();
  need_scaled(data, scale, row_shift, "data", dev);
  need_matrix(out, "out", dev);
  TORCH_CHECK(out.sizes() == data.sizes(), "out and data must have the same shape");
  c10::cuda::CUDAGuard g(dev);
  check(elfb::fp8_dequantize(bytes(data), pitch(data), bytes(scale), pitch(scale), int(row_shift), out.data_ptr(), elem_of(out, "out"), pitch(out),
                             data.size(0), int(data.size(1)), cur()),
        "fp8_dequantize");
}

void need_dense_bf16(const at::Tensor& t, const char* name, const at::Device& dev) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev && t.scalar_type() == at::kBFloat16 && t.is_contiguous(), name, " must be a contiguous bf16 tensor on ", dev);
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, name, " must be 16-byte aligned");
}

// returns (rstd, h): h = x + residual, or x itself without one
std::tuple<at::Tensor, at::Tensor> rmsnorm(const at::Tensor& x, const at::Tensor& w, double eps, const c10::optional<at::Tensor>& residual, at::Tensor& data,
                                           at::Tensor& scale) {
  const auto dev = x.device();
  TORCH_CHECK(x.dim() == 2, "x must be a matrix");
  need_dense_bf16(x, "x", dev);
  need_dense_bf16(w, "weight", dev);
  need_scaled(data, scale, 0, "data", dev);
  TORCH_CHECK(x.sizes() == data.sizes() && w.numel() == x.size(1), "x, data and weight do not match");
  TORCH_CHECK(x.size(1) % 8 == 0 && x.size(1) <= 8192, "the norm's width must be a multiple of 8, at most 8192");
  TORCH_CHECK(pitch(data) % 8 == 0 && (reinterpret_cast<uintptr_t>(data.data_ptr()) & 7) == 0, "data must have 8-byte aligned rows");
  c10::cuda::CUDAGuard g(dev);
  at::Tensor h = x;
  const void* res = nullptr;
  if (residual.has_value() && residual->defined()) {
    need_dense_bf16(*residual, "residual", dev);
    TORCH_CHECK(residual->sizes() == x.sizes(), "residual must match x");
    h = at::empty_like(x);
    res = residual->data_ptr();
  }
  auto rstd = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  check(elfb::fp8_rmsnorm(x.data_ptr(), res, w.data_ptr(), res ? h.data_ptr() : nullptr, rstd.data_ptr<float>(), bytes(data), pitch(data), bytes(scale),
                          pitch(scale), x.size(0), int(x.size(1)), float(eps), cur()),
        "fp8_rmsnorm");
  return {rstd, h};
}

void swiglu_bwd(const at::Tensor& dact, const at::Tensor& gu, const at::Tensor& gu_scale, at::Tensor& dgu, at::Tensor& dgu_scale) {
  const auto dev = dact.device();
  need_matrix(dact, "dact", dev);
  need_scaled(gu, gu_scale, 0, "gate_up", dev);
  need_scaled(dgu, dgu_scale, 0, "d_gate_up", dev);
  const int64_t f = dact.size(1);
  TORCH_CHECK(dact.scalar_type() == at::kFloat && f % 128 == 0, "dact must be fp32, its width a multiple of 128");
  TORCH_CHECK(gu.size(0) == dact.size(0) && gu.size(1) == 2 * f && gu.sizes() == dgu.sizes(), "gate_up does not match dact");
  for (const at::Tensor* t : {&dact, &gu, &static_cast<const at::Tensor&>(dgu)})
    TORCH_CHECK((pitch(*t) * t->element_size()) % 16 == 0 && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0, "rows must be 16-byte aligned");
  c10::cuda::CUDAGuard g(dev);
  check(elfb::fp8_swiglu_backward(dact.data_ptr<float>(), pitch(dact), bytes(gu), pitch(gu), bytes(gu_scale), pitch(gu_scale), bytes(dgu), pitch(dgu),
                                  bytes(dgu_scale), pitch(dgu_scale), dact.size(0), int(f), cur()),
        "fp8_swiglu_backward");
}

elfb::Fp8Operand operand(const at::Tensor& data, const at::Tensor& scale, int64_t row_shift, bool mn_major, const char* name, const at::Device& dev) {
  need_scaled(data, scale, row_shift, name, dev);
  elfb::Fp8Operand o;
  o.data = bytes(data);
  o.ld = pitch(data);
  TORCH_CHECK(o.ld % 16 == 0 && (reinterpret_cast<uintptr_t>(o.data) & 15) == 0, name, " must have 16-byte aligned rows");
  o.scale = bytes(scale);
  o.mn_major = mn_major;
  if (mn_major) {
    // stored [K][MN]: a row of the product is a column of the matrix, so scales of single rows would
    // change inside a block of the reduction
    TORCH_CHECK(row_shift == 7, name, " must be scaled in tiles of 128 x 128 to be used transposed");
    o.row_shift = 7;
    o.row_stride = 1;
    o.block_stride = pitch(scale);
  } else {
    o.row_shift = int(row_shift);
    o.row_stride = pitch(scale);
    o.block_stride = 1;
  }
  return o;
}

int sm_count(const at::Device& dev) { return at::cuda::getDeviceProperties(dev.index())->multiProcessorCount; }

int* status_ptr(const at::Tensor& status, const at::Device& dev) {
  TORCH_CHECK(status.is_cuda() && status.device() == dev && status.scalar_type() == at::kInt && status.numel() >= 4, "status must be an int32[4] tensor on ", dev);
  return status.data_ptr<int>();
}

// d = a . b^T (b [N, K]), or a . b (b_mn_major, b [K, N])
void gemm(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale, int64_t b_row_shift, bool b_mn_major, at::Tensor& d,
          const c10::optional<at::Tensor>& bias, const at::Tensor& status) {
  const auto dev = d.device();
  c10::cuda::CUDAGuard guard(dev);
  need_matrix(d, "out", dev);
  elfb::Fp8GemmArgs g;
  g.a = operand(a, a_scale, 0, false, "a", dev);
  g.b = operand(b, b_scale, b_row_shift, b_mn_major, "b", dev);
  g.M = int(d.size(0));
  g.N = int(d.size(1));
  g.K = int(a.size(1));
  TORCH_CHECK(a.size(0) == g.M && b.size(b_mn_major ? 1 : 0) == g.N && b.size(b_mn_major ? 0 : 1) == g.K, "shapes do not match");
  g.d = d.data_ptr();
  g.ldd = pitch(d);
  g.out = elem_of(d, "out");
  if (bias.has_value() && bias->defined()) {
    TORCH_CHECK(bias->device() == dev && bias->scalar_type() == d.scalar_type() && bias->dim() == 1 && bias->numel() == g.N && bias->is_contiguous(),
                "bias must be a contiguous [N] tensor of the output's dtype");
    g.bias = bias->data_ptr();
  }
  g.status = status_ptr(status, dev);
  const char* err = elfb::fp8_gemm(g, sm_count(dev), cur());
  TORCH_CHECK(err == nullptr, "elf_b200 fp8_gemm: ", err);
}

// act [M, F] = silu(gate) * up for gate | up = a . b^T (b [2F, K]); gu (and its scales) may be None
void gated(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale, int64_t b_row_shift, at::Tensor& act,
           at::Tensor& act_scale, const c10::optional<at::Tensor>& gu, const c10::optional<at::Tensor>& gu_scale, const at::Tensor& status) {
  const auto dev = act.device();
  c10::cuda::CUDAGuard guard(dev);
  need_scaled(act, act_scale, 0, "act", dev);
  elfb::Fp8GemmArgs g;
  g.a = operand(a, a_scale, 0, false, "a", dev);
  g.b = operand(b, b_scale, b_row_shift, false, "b", dev);
  g.M = int(act.size(0));
  g.N = int(b.size(0));
  g.K = int(a.size(1));
  TORCH_CHECK(a.size(0) == g.M && b.size(1) == g.K && 2 * act.size(1) == g.N, "shapes do not match");
  g.gated = true;
  g.act = bytes(act);
  g.ld_act = pitch(act);
  g.act_scale = bytes(act_scale);
  g.ld_act_scale = pitch(act_scale);
  if (gu.has_value() && gu->defined()) {
    TORCH_CHECK(gu_scale.has_value(), "gate_up needs its scales");
    need_scaled(*gu, *gu_scale, 0, "gate_up", dev);
    TORCH_CHECK(gu->size(0) == g.M && gu->size(1) == g.N, "gate_up does not match the weights");
    g.gu = bytes(*gu);
    g.ld_gu = pitch(*gu);
    g.gu_scale = bytes(*gu_scale);
    g.ld_gu_scale = pitch(*gu_scale);
  }
  g.status = status_ptr(status, dev);
  const char* err = elfb::fp8_gemm(g, sm_count(dev), cur());
  TORCH_CHECK(err == nullptr, "elf_b200 fp8_gated: ", err);
}

}  // namespace

void register_fp8(pybind11::module_& m) {
  m.def("fp8_quantize", &quantize, py::arg("x"), py::arg("data"), py::arg("scale"), py::arg("tiles"));
  m.def("fp8_dequantize", &dequantize, py::arg("data"), py::arg("scale"), py::arg("row_shift"), py::arg("out"));
  m.def("fp8_rmsnorm", &rmsnorm, py::arg("x"), py::arg("w"), py::arg("eps"), py::arg("residual"), py::arg("data"), py::arg("scale"));
  m.def("fp8_swiglu_bwd", &swiglu_bwd, py::arg("dact"), py::arg("gu"), py::arg("gu_scale"), py::arg("dgu"), py::arg("dgu_scale"));
  m.def("fp8_gemm", &gemm, py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"), py::arg("b_row_shift"), py::arg("b_mn_major"), py::arg("d"),
        py::arg("bias"), py::arg("status"));
  m.def("fp8_gated", &gated, py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"), py::arg("b_row_shift"), py::arg("act"), py::arg("act_scale"),
        py::arg("gu"), py::arg("gu_scale"), py::arg("status"));
}
