// Host entry points of the block-scaled 8-bit kernels (fp8_ops.cu, fp8_gemm_sm100.cu).
//
// A block-scaled matrix holds e4m3 values and one biased exponent byte per block of 128 columns
// (and 1 or 128 rows): value = data * 2^(byte - 127).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace elfb {

enum class Elem : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

// x [rows][cols] (pitch ldx elements) -> data [rows][cols] (pitch ldq bytes), scale [rows][ceil(cols/128)] (pitch lds bytes)
cudaError_t fp8_quantize_rows(const void* x, Elem type, long long ldx, uint8_t* data, long long ldq, uint8_t* scale, long long lds, long long rows,
                              int cols, cudaStream_t stream);
// the same with one scale per 128 x 128 tile: scale [ceil(rows/128)][ceil(cols/128)]
cudaError_t fp8_quantize_tiles(const void* x, Elem type, long long ldx, uint8_t* data, long long ldq, uint8_t* scale, long long lds, long long rows,
                               int cols, cudaStream_t stream);
// scale row of matrix row r is r >> row_shift (0 or 7)
cudaError_t fp8_dequantize(const uint8_t* data, long long ldq, const uint8_t* scale, long long lds, int row_shift, void* y, Elem type, long long ldy,
                           long long rows, int cols, cudaStream_t stream);
// copies rows of bytes to another pitch (pitches in bytes)
cudaError_t fp8_repack(const void* src, long long ld_src, void* dst, long long ld_dst, long long rows, int row_bytes, cudaStream_t stream);
// x [rows][cols] (fp16 or fp32, pitch ldx elements) as bf16_parts(type) bf16 matrices whose sum it is, the largest first: part p
// begins p * part_step elements into `out`, whose rows are ldo elements apart (16-byte aligned, ldo a multiple of 8)
int bf16_parts(Elem type);
cudaError_t split_into_bf16_parts(const void* x, Elem type, long long ldx, void* out, long long ldo, long long part_step, long long rows, int cols,
                                  cudaStream_t stream);
// h = x + residual (bf16, written when residual is given); data/scale = blocks of h * rstd * w
cudaError_t fp8_rmsnorm(const void* x, const void* residual, const void* w, void* h, float* rstd, uint8_t* data, long long ldq, uint8_t* scale,
                        long long lds, long long rows, int dim, double eps, int num_sms, cudaStream_t stream);
// One operand of a block-scaled product.  Its scale for (row of the product, block of the
// reduction) is scale[(row >> row_shift) * row_stride + block * block_stride].
struct Fp8Operand {
  const uint8_t* data = nullptr;
  long long ld = 0;  // bytes between consecutive rows in memory, a multiple of 16
  const uint8_t* scale = nullptr;
  long long row_stride = 0, block_stride = 0;
  int row_shift = 0;
  bool mn_major = false;  // stored [K][MN] instead of [MN][K]
};

enum class Fp8Form {
  kPlain,
  kGated,          // b is [2F][K] (gate rows, up rows): silu(gate) * up and, on request, gate | up leave in 8 bits
  kGatedBackward,  // b is [K][F] mn_major: the product is the gradient of the activation, that of gate | up leaves in 8 bits
};

struct Fp8GemmArgs {
  Fp8Form form = Fp8Form::kPlain;
  Fp8Operand a, b;             // a: [M][K]; b: [N][K], or [K][N] when mn_major
  void* d = nullptr;           // plain: [M][N], pitch ldd elements
  Elem out = Elem::kBf16;
  long long ldd = 0;
  const void* bias = nullptr;  // plain, optional: [N], type of d
  int M = 0, N = 0, K = 0;
  uint8_t* act = nullptr;      // gated: the activation [M][F]; gated backward: the gradient of gate | up [M][2F]
  long long ld_act = 0;
  uint8_t* act_scale = nullptr;
  long long ld_act_scale = 0;
  uint8_t* gu = nullptr;       // gate | up [M][2F]: written by the gated form (nullptr when no backward pass follows), read by its backward
  long long ld_gu = 0;
  uint8_t* gu_scale = nullptr;
  long long ld_gu_scale = 0;
  void* workspace = nullptr;   // fp8_gemm_workspace() bytes, used by this launch alone
  int* status = nullptr;
};
size_t fp8_gemm_workspace(const Fp8GemmArgs& args, int num_sms);
// Returns nullptr on success, otherwise a description of the failure.
const char* fp8_gemm(const Fp8GemmArgs& args, int num_sms, cudaStream_t stream);

}  // namespace elfb
