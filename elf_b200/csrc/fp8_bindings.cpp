// torch glue for fp8_ops.cu and fp8_gemm_sm100.cu: checks, output allocation, stream selection.  The small
// calls of these operators are bound by what the host does per call, so shapes are taken apart here
// and not in Python.
#include <torch/extension.h>
#include <climits>
#include <tuple>
#include <utility>
#include <vector>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include "fp8_ops.h"
#include "gemm_sm100.h"

namespace {

cudaStream_t cur() { return at::cuda::getCurrentCUDAStream(); }

void check(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, "elf_b200 ", what, ": ", cudaGetErrorString(e)); }

elfb::Elem elem_of(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return elfb::Elem::kBf16;
  if (t.scalar_type() == at::kHalf) return elfb::Elem::kF16;
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be bf16, fp16 or fp32, got ", t.scalar_type());
  return elfb::Elem::kF32;
}

int sm_count(const at::Device& dev) { return at::cuda::getDeviceProperties(dev.index())->multiProcessorCount; }
int* status_ptr(const at::Tensor& status, const at::Device& dev) {
  TORCH_CHECK(status.is_cuda() && status.device() == dev && status.scalar_type() == at::kInt && status.numel() >= 4, "status must be an int32[4] tensor on ", dev);
  return status.data_ptr<int>();
}

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }
int64_t round_up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// A tensor [..., cols] seen as a matrix with a contiguous last dimension; a copy only where strides force one.
struct Mat {
  at::Tensor t;
  int64_t rows, cols, pitch;  // pitch in elements
  uint8_t* bytes() const { return static_cast<uint8_t*>(t.data_ptr()); }
  bool aligned(int64_t to) const { return (reinterpret_cast<uintptr_t>(t.data_ptr()) | uintptr_t(pitch * t.element_size())) % to == 0; }
};

bool row_pitch(const at::Tensor& t, int64_t* pitch) {
  const int64_t d = t.dim(), cols = t.size(d - 1);
  if (cols > 1 && t.stride(d - 1) != 1) return false;
  *pitch = cols;
  int64_t expected = 0;  // stride the next dimension outwards must have
  for (int64_t i = d - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (expected == 0) {
      if (t.stride(i) < cols) return false;
      *pitch = t.stride(i);
    } else if (t.stride(i) != expected) {
      return false;
    }
    expected = t.stride(i) * t.size(i);
  }
  if (expected == 0 && d >= 2 && t.stride(d - 2) > cols) *pitch = t.stride(d - 2);  // a single row
  return true;
}

Mat matrix(const at::Tensor& t, const char* name, const at::Device& dev, bool may_copy = true) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, name, " must be a CUDA tensor on ", dev);
  TORCH_CHECK(t.dim() >= 1, name, " must have at least one dimension");
  Mat m{t, 0, t.size(-1), 0};
  m.rows = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) m.rows *= t.size(i);
  TORCH_CHECK(m.cols <= INT_MAX - 1024, name, " is too wide");
  if (t.numel() == 0) {
    m.pitch = m.cols;
  } else if (!row_pitch(t, &m.pitch)) {
    TORCH_CHECK(may_copy, name, " must have a contiguous last dimension and rows that do not overlap");
    m.t = t.contiguous();
    m.pitch = m.cols;
  }
  return m;
}

// Block-scaled matrix; scales of rows (row_shift 0) or of tiles of 128 rows (7).
struct Scaled {
  Mat data, scale;
};

Scaled scaled(const at::Tensor& data, const at::Tensor& scale, int64_t row_shift, const char* name, const at::Device& dev, bool may_copy = true) {
  TORCH_CHECK(data.element_size() == 1 && scale.element_size() == 1, name, " must hold 8-bit values and exponents");
  TORCH_CHECK(row_shift == 0 || row_shift == 7, "scales belong to rows or to tiles of 128 rows");
  Scaled s{matrix(data, name, dev, may_copy), matrix(scale, "the scales", dev, may_copy)};
  const int64_t rows = row_shift ? blocks_of(s.data.rows) : s.data.rows;
  TORCH_CHECK(s.scale.rows == rows && s.scale.cols == blocks_of(s.data.cols), name, ": expected scales [", rows, ", ", blocks_of(s.data.cols), "], got [",
              s.scale.rows, ", ", s.scale.cols, "]");
  return s;
}

// New tensor whose rows are `pitch` elements apart.
at::Tensor new_rows(at::IntArrayRef lead, int64_t cols, int64_t pitch, at::ScalarType dtype, const at::Device& dev) {
  c10::SmallVector<int64_t, 6> sizes(lead.begin(), lead.end()), strides(lead.size() + 1);
  sizes.push_back(cols);
  strides.back() = 1;
  int64_t step = pitch;
  for (int64_t i = int64_t(lead.size()) - 1; i >= 0; --i) {
    strides[i] = step;
    step *= std::max<int64_t>(sizes[i], 1);
  }
  return at::detail::empty_strided_cuda(sizes, strides, dtype, dev);  // past the dispatcher
}

at::Tensor dense(at::IntArrayRef sizes, at::ScalarType dtype, const at::Device& dev) { return at::detail::empty_cuda(sizes, dtype, dev, c10::nullopt); }

// Block-scaled tensor [*lead, cols] with the row pitches the products want.
std::pair<at::Tensor, at::Tensor> new_scaled(at::IntArrayRef lead, int64_t cols, bool tiles, const at::Device& dev) {
  const int64_t tile_rows[1] = {tiles ? blocks_of(lead[0]) : 0};
  return {new_rows(lead, cols, round_up(cols, 16), at::kFloat8_e4m3fn, dev),
          new_rows(tiles ? at::IntArrayRef(tile_rows, 1) : lead, blocks_of(cols), round_up(blocks_of(cols), 4), at::kByte, dev)};
}

at::IntArrayRef lead_of(const at::Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }

std::pair<at::Tensor, at::Tensor> quantize(const at::Tensor& x, bool tiles, const c10::optional<at::Tensor>& data_out, const c10::optional<at::Tensor>& scale_out) {
  const auto dev = x.device();
  const Mat m = matrix(x, "x", dev);
  TORCH_CHECK(!tiles || x.dim() == 2, "only matrices have tiles");
  c10::cuda::CUDAGuard g(dev);
  std::pair<at::Tensor, at::Tensor> q;
  if (data_out.has_value()) {
    TORCH_CHECK(scale_out.has_value() && data_out->sizes() == x.sizes(), "data must have the shape of x and come with its scales");
    q = {*data_out, *scale_out};
  } else {
    q = new_scaled(lead_of(x), m.cols, tiles, dev);
  }
  const Scaled s = scaled(q.first, q.second, tiles ? 7 : 0, "data", dev, false);
  auto* fn = tiles ? elfb::fp8_quantize_tiles : elfb::fp8_quantize_rows;
  check(fn(m.t.data_ptr(), elem_of(x, "x"), m.pitch, s.data.bytes(), s.data.pitch, s.scale.bytes(), s.scale.pitch, m.rows, int(m.cols), cur()), "fp8_quantize");
  return q;
}

at::Tensor dequantize(const at::Tensor& data, const at::Tensor& scale, int64_t row_shift, at::ScalarType dtype, const c10::optional<at::Tensor>& out) {
  const auto dev = data.device();
  const Scaled s = scaled(data, scale, row_shift, "data", dev);
  c10::cuda::CUDAGuard g(dev);
  at::Tensor y = out.has_value() ? *out : dense(data.sizes(), dtype, dev);
  TORCH_CHECK(y.sizes() == data.sizes(), "out must have the shape of data");
  const Mat m = matrix(y, "out", dev, false);
  check(elfb::fp8_dequantize(s.data.bytes(), s.data.pitch, s.scale.bytes(), s.scale.pitch, int(row_shift), y.data_ptr(), elem_of(y, "out"), m.pitch,
                             s.data.rows, int(s.data.cols), cur()),
        "fp8_dequantize");
  return y;
}

at::Tensor dense_bf16(const at::Tensor& t, const char* name, const at::Device& dev) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev && t.scalar_type() == at::kBFloat16, name, " must be a bf16 tensor on ", dev);
  const at::Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone();
}

// returns (data, scale, rstd, h): h = x + residual, or x itself without one
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> rmsnorm(const at::Tensor& x_in, const at::Tensor& w_in, double eps,
                                                                   const c10::optional<at::Tensor>& residual) {
  const auto dev = x_in.device();
  c10::cuda::CUDAGuard g(dev);
  TORCH_CHECK(x_in.dim() >= 1, "x must have at least one dimension");
  const at::Tensor x = dense_bf16(x_in, "x", dev), w = dense_bf16(w_in, "weight", dev);
  const int64_t dim = x.size(-1);
  TORCH_CHECK(w.numel() == dim && dim % 8 == 0 && dim > 0 && dim <= 8192, "the norm's width must match the weight's and be a multiple of 8, at most 8192");
  const int64_t rows = x.numel() / dim;
  at::Tensor h = x_in, res;
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == x.sizes(), "residual must match x");
    res = dense_bf16(*residual, "residual", dev);
    h = dense(x.sizes(), at::kBFloat16, dev);
  }
  auto q = new_scaled(lead_of(x), dim, false, dev);
  auto rstd = dense(lead_of(x), at::kFloat, dev);
  const Scaled s = scaled(q.first, q.second, 0, "data", dev, false);
  check(elfb::fp8_rmsnorm(x.data_ptr(), res.defined() ? res.data_ptr() : nullptr, w.data_ptr(), res.defined() ? h.data_ptr() : nullptr, rstd.data_ptr<float>(),
                          s.data.bytes(), s.data.pitch, s.scale.bytes(), s.scale.pitch, rows, int(dim), eps, sm_count(dev), cur()),
        "fp8_rmsnorm");
  return {q.first, q.second, rstd, h};
}

// the rows of `m` in new memory, `pitch` elements apart
at::Tensor repacked(const Mat& m, int64_t pitch, const at::Device& dev) {
  const int64_t lead[1] = {m.rows}, size = m.t.element_size();
  TORCH_CHECK(m.cols * size <= INT_MAX - 1024, "rows are too wide to be copied");
  at::Tensor out = new_rows(at::IntArrayRef(lead, 1), m.cols, pitch, m.t.scalar_type(), dev);
  check(elfb::fp8_repack(m.t.data_ptr(), m.pitch * size, out.data_ptr(), pitch * size, m.rows, int(m.cols * size), cur()), "fp8_repack");
  return out;
}

// An operand of a product and the tensors that keep its memory alive until the launch is queued.
struct Operand {
  Scaled s;
  elfb::Fp8Operand o;
};

Operand operand(const at::Tensor& data, const at::Tensor& scale, int64_t row_shift, bool mn_major, const char* name, const at::Device& dev, int64_t align = 16) {
  Operand r{scaled(data, scale, row_shift, name, dev), {}};
  TORCH_CHECK(r.s.data.rows <= INT_MAX - 1024, name, " has too many rows");
  if (!r.s.data.aligned(align)) {  // TMA wants rows on 16-byte boundaries: a copy with padded rows
    const at::Tensor padded = repacked(r.s.data, round_up(r.s.data.cols, align), dev);
    r.s.data = matrix(padded, name, dev, false);
  }
  r.o.data = r.s.data.bytes();
  r.o.ld = round_up(r.s.data.pitch, align);  // (a single row may have any pitch)
  r.o.scale = r.s.scale.bytes();
  r.o.mn_major = mn_major;
  if (mn_major) {
    // stored [K][MN]: a row of the product is a column of the matrix, so scales of single rows would
    // change inside a block of the reduction
    TORCH_CHECK(row_shift == 7, name, " must be scaled in tiles of 128 x 128 to be used transposed");
    r.o.row_shift = 7;
    r.o.row_stride = 1;
    r.o.block_stride = r.s.scale.pitch;
  } else {
    r.o.row_shift = int(row_shift);
    r.o.row_stride = r.s.scale.pitch;
    r.o.block_stride = 1;
  }
  return r;
}

void launch(elfb::Fp8GemmArgs& g, const at::Tensor& status, const at::Device& dev, const char* what) {
  g.status = status_ptr(status, dev);
  // from the caching allocator, call by call: two streams or two captured graphs never share it
  at::Tensor workspace;
  if (const size_t bytes = elfb::fp8_gemm_workspace(g, sm_count(dev))) {
    workspace = dense({int64_t(bytes)}, at::kByte, dev);
    g.workspace = workspace.data_ptr();
  }
  const char* err = elfb::fp8_gemm(g, sm_count(dev), cur());
  TORCH_CHECK(err == nullptr, "elf_b200 ", what, ": ", err);
}

// a . b^T (b [N, K]), or a . b (b_mn_major, b [K, N]); a [..., K]
at::Tensor gemm(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale, int64_t b_row_shift, bool b_mn_major,
                at::ScalarType dtype, const c10::optional<at::Tensor>& bias, const at::Tensor& status) {
  const auto dev = a.device();
  c10::cuda::CUDAGuard guard(dev);
  const Operand oa = operand(a, a_scale, 0, false, "the activation", dev), ob = operand(b, b_scale, b_row_shift, b_mn_major, "the weight", dev);
  elfb::Fp8GemmArgs g;
  g.a = oa.o;
  g.b = ob.o;
  g.M = int(oa.s.data.rows);
  g.K = int(oa.s.data.cols);
  g.N = int(b_mn_major ? ob.s.data.cols : ob.s.data.rows);
  TORCH_CHECK(g.K == (b_mn_major ? ob.s.data.rows : ob.s.data.cols), "the operands disagree on the reduction length");
  auto sizes = a.sizes().vec();
  sizes.back() = g.N;
  at::Tensor d = dense(sizes, dtype, dev);
  g.d = d.data_ptr();
  g.ldd = g.N;
  g.out = elem_of(d, "the product");
  if (bias.has_value()) {
    TORCH_CHECK(bias->device() == dev && bias->scalar_type() == dtype && bias->dim() == 1 && bias->numel() == g.N && bias->is_contiguous(),
                "the bias must be a contiguous [N] tensor of the product's dtype");
    g.bias = bias->data_ptr();
  }
  launch(g, status, dev, "fp8_gemm");
  return d;
}

// act [..., F] = silu(gate) * up for gate | up = a . b^T (b [2F, K]); returns (act, act_scale, gate_up, its scales), the last two undefined unless `keep`
std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>> gated(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b,
                                                                                               const at::Tensor& b_scale, int64_t b_row_shift, bool keep,
                                                                                               const at::Tensor& status) {
  const auto dev = a.device();
  c10::cuda::CUDAGuard guard(dev);
  const Operand oa = operand(a, a_scale, 0, false, "the activation", dev), ob = operand(b, b_scale, b_row_shift, false, "the weight", dev);
  elfb::Fp8GemmArgs g;
  g.a = oa.o;
  g.b = ob.o;
  g.M = int(oa.s.data.rows);
  g.K = int(oa.s.data.cols);
  g.N = int(ob.s.data.rows);
  TORCH_CHECK(g.K == ob.s.data.cols, "the operands disagree on the reduction length");
  TORCH_CHECK(g.N % 256 == 0, "the width of gate and of up must be a multiple of 128");
  auto act = new_scaled(lead_of(a), g.N / 2, false, dev);
  const Scaled sa = scaled(act.first, act.second, 0, "act", dev, false);
  g.form = elfb::Fp8Form::kGated;
  g.act = sa.data.bytes();
  g.ld_act = sa.data.pitch;
  g.act_scale = sa.scale.bytes();
  g.ld_act_scale = sa.scale.pitch;
  c10::optional<at::Tensor> gu_data, gu_scale;
  if (keep) {
    auto gu = new_scaled(lead_of(a), g.N, false, dev);
    const Scaled sg = scaled(gu.first, gu.second, 0, "gate_up", dev, false);
    g.gu = sg.data.bytes();
    g.ld_gu = sg.data.pitch;
    g.gu_scale = sg.scale.bytes();
    g.ld_gu_scale = sg.scale.pitch;
    gu_data = gu.first;
    gu_scale = gu.second;
  }
  launch(g, status, dev, "fp8_gated");
  return {act.first, act.second, gu_data, gu_scale};
}

// gradient [..., 2F] of gate | up for the gradient dy [..., D] of the block's output, w_down [D, F] and gate | up from their checkpoint
std::pair<at::Tensor, at::Tensor> gated_bwd(const at::Tensor& dy, const at::Tensor& dy_scale, const at::Tensor& w, const at::Tensor& w_scale,
                                            const at::Tensor& gu, const at::Tensor& gu_scale, const at::Tensor& status) {
  const auto dev = dy.device();
  c10::cuda::CUDAGuard guard(dev);
  const Operand oa = operand(dy, dy_scale, 0, false, "the gradient", dev), ob = operand(w, w_scale, 7, true, "the weight", dev),
                og = operand(gu, gu_scale, 0, false, "gate_up", dev, 32);
  elfb::Fp8GemmArgs g;
  g.form = elfb::Fp8Form::kGatedBackward;
  g.a = oa.o;
  g.b = ob.o;
  g.M = int(oa.s.data.rows);
  g.K = int(oa.s.data.cols);
  g.N = int(ob.s.data.cols);
  TORCH_CHECK(g.K == ob.s.data.rows, "the operands disagree on the reduction length");
  TORCH_CHECK(g.N % 128 == 0 && og.s.data.rows == g.M && og.s.data.cols == 2 * int64_t(g.N), "gate_up does not match the gradient and the weight");
  auto dgu = new_scaled(lead_of(gu), 2 * int64_t(g.N), false, dev);
  const Scaled sd = scaled(dgu.first, dgu.second, 0, "d_gate_up", dev, false);
  g.act = sd.data.bytes();
  g.ld_act = sd.data.pitch;
  g.act_scale = sd.scale.bytes();
  g.ld_act_scale = sd.scale.pitch;
  g.gu = og.s.data.bytes();
  g.ld_gu = og.s.data.pitch;
  g.gu_scale = og.s.scale.bytes();
  g.ld_gu_scale = og.s.scale.pitch;
  launch(g, status, dev, "fp8_gated_bwd");
  return dgu;
}

// The gated feed-forward block: x to 8 bits, act = silu(gate) * up, y = act . w_down^T, one call for its three kernels.
// With `keep` also what its backward pass works from: (y, x, act, gate_up), each block-scaled tensor as values and scales.
std::vector<c10::optional<at::Tensor>> ffn(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wg_scale, const at::Tensor& wd, const at::Tensor& wd_scale,
                                           bool keep, const at::Tensor& status) {
  const auto xq = quantize(x, false, c10::nullopt, c10::nullopt);
  auto [act, act_scale, gu, gu_scale] = gated(xq.first, xq.second, wg, wg_scale, 7, keep, status);
  at::Tensor y = gemm(act, act_scale, wd, wd_scale, 7, false, x.scalar_type(), c10::nullopt, status);
  if (!keep) return {y};
  return {y, xq.first, xq.second, act, act_scale, gu, gu_scale};
}

// One operand of the 16-bit product, rows on 16-byte boundaries.  An operand is the sum of `parts` bf16 matrices (block-scaled and
// bf16 tensors of one, see split_into_bf16_parts), and each pair of parts of the two has its stretch of the reduction: the
// matrices lie one behind the other, part p (0: the largest) at stretch (parts - 1 - p) * part_step and, for the other
// operand's parts, `copies` times copy_step further on.
Mat stacked(const at::Tensor& t, const c10::optional<at::Tensor>& scale, int parts, int64_t part_step, int copies, int64_t copy_step, const char* name,
            const at::Device& dev) {
  const Mat m = matrix(t, name, dev);
  if (parts * copies == 1 && !scale.has_value() && m.aligned(16)) return m;
  const int64_t pitch = round_up(m.cols, 8), stretch = m.rows * pitch, lead[1] = {m.rows * parts * copies};
  const at::Tensor out = new_rows(at::IntArrayRef(lead, 1), m.cols, pitch, at::kBFloat16, dev);
  for (int c = 0; c < copies; ++c) {
    at::BFloat16* first = out.data_ptr<at::BFloat16>() + c * copy_step * stretch;
    if (scale.has_value()) {
      const Scaled s = scaled(t, *scale, 0, name, dev);
      check(elfb::fp8_dequantize(s.data.bytes(), s.data.pitch, s.scale.bytes(), s.scale.pitch, 0, first, elfb::Elem::kBf16, pitch, m.rows, int(m.cols), cur()),
            "fp8_dequantize");
    } else if (parts == 1) {
      TORCH_CHECK(m.cols * 2 <= INT_MAX - 1024, "rows are too wide to be copied");
      check(elfb::fp8_repack(m.t.data_ptr(), m.pitch * 2, first, pitch * 2, m.rows, int(m.cols * 2), cur()), "fp8_repack");
    } else {
      check(elfb::split_into_bf16_parts(m.t.data_ptr(), elem_of(t, name), m.pitch, first + (parts - 1) * part_step * stretch, pitch, -part_step * stretch, m.rows,
                                        int(m.cols), cur()),
            "split_into_bf16_parts");
    }
  }
  return {out, lead[0], m.cols, pitch};
}

// dy^T x over all leading dimensions, on the 16-bit tensor path; added to `out` when it is given.  Either operand block-scaled
// (with its scales) or plain.  The reduction runs over all pairs of bf16 parts of the operands, the small ones first, so that the
// large ones' sum is rounded no more often than alone.
at::Tensor weight_grad(const at::Tensor& dy, const c10::optional<at::Tensor>& dy_scale, const at::Tensor& x, const c10::optional<at::Tensor>& x_scale,
                       const c10::optional<at::Tensor>& out, at::ScalarType dtype, const at::Tensor& status, int64_t variant, bool split_tail) {
  const auto dev = x.device();
  c10::cuda::CUDAGuard guard(dev);
  auto parts_of = [](const at::Tensor& t, const c10::optional<at::Tensor>& scale, const char* name) { return scale.has_value() ? 1 : elfb::bf16_parts(elem_of(t, name)); };
  const int dy_parts = parts_of(dy, dy_scale, "dy"), x_parts = parts_of(x, x_scale, "x");
  const Mat a = stacked(dy, dy_scale, dy_parts, x_parts, x_parts, 1, "dy", dev), b = stacked(x, x_scale, x_parts, 1, dy_parts, x_parts, "x", dev);
  TORCH_CHECK(a.rows == b.rows && a.rows <= INT_MAX, "dy and x must have the same number of rows");
  // fp16 results, whole operands' sums with a bf16 gradient, and widths whose rows are not on 16-byte boundaries, go through a
  // buffer
  const bool direct = out.has_value() && (dy_parts * x_parts == 1 || out->scalar_type() == at::kFloat) && b.cols % 8 == 0 && out->is_contiguous() && reinterpret_cast<uintptr_t>(out->data_ptr()) % 16 == 0;
  const int64_t lead[1] = {a.cols};
  const at::ScalarType held = !out.has_value() && dtype == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
  at::Tensor dw = direct ? *out : new_rows(at::IntArrayRef(lead, 1), b.cols, round_up(b.cols, 8), held, dev);
  elfb::GemmArgs g;
  g.fmt = 1;
  g.M = int(a.cols);
  g.N = int(b.cols);
  g.K = int(a.rows);
  g.a = a.t.data_ptr();
  g.b = b.t.data_ptr();
  g.d = dw.data_ptr();
  g.lda = a.pitch;
  g.ldb = b.pitch;
  g.ldd = direct ? b.cols : round_up(b.cols, 8);
  g.a_mn_major = g.b_mn_major = true;
  g.out_f32 = dw.scalar_type() == at::kFloat;
  g.accumulate = direct;
  g.variant = int(variant);
  g.split_tail = split_tail;
  g.status = status_ptr(status, dev);
  // tiles that are split along the tokens: parts in fp32, one order of sums
  at::Tensor workspace;
  if (const size_t bytes = elfb::gemm_pair_workspace(g, sm_count(dev))) {
    workspace = dense({int64_t(bytes)}, at::kByte, dev);
    g.workspace = workspace.data_ptr();
  }
  const char* err = elfb::gemm_tcgen05(g, sm_count(dev), cur());
  TORCH_CHECK(err == nullptr, "elf_b200 fp8_weight_grad: ", err);
  if (direct) return dw;
  if (out.has_value()) {
    at::Tensor sum = *out;
    return sum.add_(dw);
  }
  if (dw.scalar_type() != dtype) return dw.to(dtype).contiguous();
  return dw.is_contiguous() ? dw : repacked(matrix(dw, "the gradient", dev, false), b.cols, dev);
}

// Backward of `ffn` from what it kept: (dx, dw_gate_up, dw_down), each only on request.
std::vector<c10::optional<at::Tensor>> ffn_bwd(const at::Tensor& dy, const std::vector<at::Tensor>& kept, const at::Tensor& wg, const at::Tensor& wg_scale,
                                               const at::Tensor& wd, const at::Tensor& wd_scale, const std::vector<bool>& need,
                                               const std::vector<at::ScalarType>& dtypes, const at::Tensor& status, int64_t variant, bool split_tail) {
  TORCH_CHECK(kept.size() == 6 && need.size() == 3 && dtypes.size() == 3, "fp8_ffn_bwd: bad arguments");
  std::vector<c10::optional<at::Tensor>> grads(3);
  if (need[2]) grads[2] = weight_grad(dy, c10::nullopt, kept[2], kept[3], c10::nullopt, dtypes[2], status, variant, split_tail);
  if (need[0] || need[1]) {
    const auto dyq = quantize(dy, false, c10::nullopt, c10::nullopt);
    const auto dgu = gated_bwd(dyq.first, dyq.second, wd, wd_scale, kept[4], kept[5], status);
    if (need[0]) grads[0] = gemm(dgu.first, dgu.second, wg, wg_scale, 7, true, dtypes[0], c10::nullopt, status);
    if (need[1]) grads[1] = weight_grad(dgu.first, dgu.second, kept[0], kept[1], c10::nullopt, dtypes[1], status, variant, split_tail);
  }
  return grads;
}

}  // namespace

void register_fp8(pybind11::module_& m) {
  m.def("fp8_quantize", &quantize, py::arg("x"), py::arg("tiles"), py::arg("data") = c10::nullopt, py::arg("scale") = c10::nullopt);
  m.def("fp8_dequantize", &dequantize, py::arg("data"), py::arg("scale"), py::arg("row_shift"), py::arg("dtype"), py::arg("out") = c10::nullopt);
  m.def("fp8_rmsnorm", &rmsnorm, py::arg("x"), py::arg("w"), py::arg("eps"), py::arg("residual"));
  m.def("fp8_gemm", &gemm, py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"), py::arg("b_row_shift"), py::arg("b_mn_major"), py::arg("dtype"),
        py::arg("bias"), py::arg("status"));
  m.def("fp8_gated", &gated, py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"), py::arg("b_row_shift"), py::arg("keep"), py::arg("status"));
  m.def("fp8_ffn", &ffn, py::arg("x"), py::arg("wg"), py::arg("wg_scale"), py::arg("wd"), py::arg("wd_scale"), py::arg("keep"), py::arg("status"));
  m.def("fp8_weight_grad", &weight_grad, py::arg("dy"), py::arg("dy_scale"), py::arg("x"), py::arg("x_scale"), py::arg("out"), py::arg("dtype"), py::arg("status"),
        py::arg("variant"), py::arg("split_tail"));
  m.def("fp8_ffn_bwd", &ffn_bwd, py::arg("dy"), py::arg("kept"), py::arg("wg"), py::arg("wg_scale"), py::arg("wd"), py::arg("wd_scale"), py::arg("need"),
        py::arg("dtypes"), py::arg("status"), py::arg("variant"), py::arg("split_tail"));
  m.def("fp8_gated_bwd", &gated_bwd, py::arg("dy"), py::arg("dy_scale"), py::arg("w"), py::arg("w_scale"), py::arg("gu"), py::arg("gu_scale"), py::arg("status"));
}
