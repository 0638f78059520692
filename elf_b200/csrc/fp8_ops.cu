// Bandwidth-bound kernels that write or read block-scaled 8-bit tensors: quantise, restore, RMSNorm
// with an 8-bit output.  Each reads its inputs once and writes its outputs once; all arithmetic is
// fp32.
#include "fp8_ops.h"

#include <algorithm>

#include "fp8_block.cuh"

namespace elfb {

namespace {

constexpr int BLOCK = 128;  // columns that share a scale
constexpr int UNIT = 16;    // consecutive values a thread holds: 8 lanes make up a block
constexpr int THREADS = 256;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __uint_as_float(uint32_t(__bfloat16_as_ushort(v)) << 16); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// N consecutive values as fp32.  VEC: the address is a multiple of 16 bytes and all N exist.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_values(const T* p, int have, float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < N / PER; ++i) {
      const uint4 q = reinterpret_cast<const uint4*>(p)[i];
      const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int j = 0; j < PER; ++j) v[i * PER + j] = to_float(e[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < have ? to_float(p[j]) : 0.f;
  }
}
template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_values(T* p, int have, const float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < N / PER; ++i) {
      uint4 q;
      T* e = reinterpret_cast<T*>(&q);
#pragma unroll
      for (int j = 0; j < PER; ++j) e[j] = from_float<T>(v[i * PER + j]);
      reinterpret_cast<uint4*>(p)[i] = q;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < have) p[j] = from_float<T>(v[j]);
  }
}
__device__ __forceinline__ void store_bytes_ragged(uint8_t* p, int have, const uint32_t (&q)[UNIT / 4]) {
#pragma unroll
  for (int j = 0; j < UNIT; ++j)
    if (j < have) p[j] = uint8_t(q[j / 4] >> (8 * (j % 4)));
}

// ------------------------------------------------------------------------------ quantise
// One thread per 16 values; the 8 lanes of a block find its maximum with three shuffles.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) quantize_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ data, long long ldq,
                                                                uint8_t* __restrict__ scale, long long lds, uint32_t total, uint32_t units_per_row,
                                                                int cols) {
  const uint32_t u = blockIdx.x * THREADS + threadIdx.x;
  const uint32_t row = u / units_per_row;
  const int col = int(u - row * units_per_row) * UNIT;
  const int have = u < total ? min(cols - col, UNIT) : 0;  // 0 or less: padding of a row's last block
  float v[UNIT];
  if (have > 0) {
    load_values<T, UNIT, VEC>(x + (long long)row * ldx + col, have, v);
  } else {
#pragma unroll
    for (int j = 0; j < UNIT; ++j) v[j] = 0.f;
  }
  uint32_t q[UNIT / 4];
  const uint32_t byte = quantize_block<UNIT, 8>(v, q);
  if (have > 0) {
    uint8_t* dst = data + (long long)row * ldq + col;
    if constexpr (VEC)
      *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
    else
      store_bytes_ragged(dst, have, q);
    if ((col & (BLOCK - 1)) == 0) scale[(long long)row * lds + col / BLOCK] = uint8_t(byte);
  }
}

// One block of threads per 128 x 128 tile: every thread holds four groups of 16 values (rows 32
// apart), so the tile is read once.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) quantize_tiles_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ data, long long ldq,
                                                                 uint8_t* __restrict__ scale, long long lds, long long rows, int cols) {
  __shared__ uint32_t warp_max[2][THREADS / 32];
  const int col = blockIdx.x * BLOCK + (threadIdx.x & 7) * UNIT;
  const long long row0 = (long long)blockIdx.y * BLOCK + (threadIdx.x >> 3);
  const int have_cols = min(cols - col, UNIT);
  float v[4][UNIT];
  uint32_t any = 0, finite = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = row0 + 32 * i;
    if (have_cols > 0 && row < rows) {
      load_values<T, UNIT, VEC>(x + row * ldx + col, have_cols, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < UNIT; ++j) v[i][j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < UNIT; ++j) {
      any = max(any, abs_bits(v[i][j]));
      finite = max(finite, finite_bits(v[i][j]));
    }
  }
  any = group_max<32>(any);
  finite = group_max<32>(finite);
  if ((threadIdx.x & 31) == 0) {
    warp_max[0][threadIdx.x >> 5] = any;
    warp_max[1][threadIdx.x >> 5] = finite;
  }
  __syncthreads();
  any = finite = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    any = max(any, warp_max[0][w]);
    finite = max(finite, warp_max[1][w]);
  }
  const uint32_t byte = block_exponent(finite);
  const float inv = inverse_exponent_value(byte);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = row0 + 32 * i;
    if (have_cols <= 0 || row >= rows) continue;
    float s[UNIT];
#pragma unroll
    for (int j = 0; j < UNIT; ++j) {
      s[j] = mul_exact(v[i][j], inv);
      if (any >= kInfBits) s[j] = nan_unless_finite(s[j], v[i][j]);
    }
    uint32_t q[UNIT / 4];
#pragma unroll
    for (int j = 0; j < UNIT / 4; ++j) q[j] = to_e4m3x4(s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]);
    uint8_t* dst = data + row * ldq + col;
    if constexpr (VEC)
      *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
    else
      store_bytes_ragged(dst, have_cols, q);
  }
  if (threadIdx.x == 0) scale[(long long)blockIdx.y * lds + blockIdx.x] = uint8_t(byte);
}

// ------------------------------------------------------------------------------ restore
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(const uint8_t* __restrict__ data, long long ldq, const uint8_t* __restrict__ scale,
                                                             long long lds, int row_shift, T* __restrict__ y, long long ldy, uint32_t total,
                                                             uint32_t units_per_row, long long first_row, int cols) {
  const uint32_t u = blockIdx.x * THREADS + threadIdx.x;
  if (u >= total) return;
  const uint32_t r = u / units_per_row;
  const int col = int(u - r * units_per_row) * UNIT;
  const long long row = first_row + r;
  const int have = min(cols - col, UNIT);
  const uint8_t* src = data + row * ldq + col;
  uint32_t q[UNIT / 4];
  if constexpr (VEC) {
    const uint4 t = *reinterpret_cast<const uint4*>(src);
    q[0] = t.x, q[1] = t.y, q[2] = t.z, q[3] = t.w;
  } else {
#pragma unroll
    for (int j = 0; j < UNIT / 4; ++j) q[j] = 0;
#pragma unroll
    for (int j = 0; j < UNIT; ++j)
      if (j < have) q[j / 4] |= uint32_t(src[j]) << (8 * (j % 4));
  }
  const float s = exponent_value(scale[(row >> row_shift) * lds + col / BLOCK]);
  float v[UNIT];
#pragma unroll
  for (int j = 0; j < UNIT / 4; ++j) {
    const float2 lo = from_e4m3x2(q[j] & 0xffffu), hi = from_e4m3x2(q[j] >> 16);
    v[4 * j] = mul_exact(lo.x, s);
    v[4 * j + 1] = mul_exact(lo.y, s);
    v[4 * j + 2] = mul_exact(hi.x, s);
    v[4 * j + 3] = mul_exact(hi.y, s);
  }
  store_values<T, UNIT, VEC>(y + row * ldy + col, have, v);
}

// ------------------------------------------------------------------------------ RMSNorm
// h = x + residual (rounded to bf16, as the next residual addition reads it), y = h * rstd * w, y in
// 8 bits.  TPR threads per row hold it in registers, 8 values (16 bytes) per thread and step; the 16
// lanes whose values make up a block scale it with four shuffles.
template <int TPR, int VPT, bool RESIDUAL>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) rmsnorm_fp8_kernel(const uint4* __restrict__ x, const uint4* __restrict__ res,
                                                                            const uint4* __restrict__ w, uint4* __restrict__ h, float* __restrict__ rstd,
                                                                            uint8_t* __restrict__ data, long long ldq, uint8_t* __restrict__ scale,
                                                                            long long lds, long long rows, int dim8, float inv_dim, float eps) {
  constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;  // rows per block
  __shared__ float red[TPR / 32 + 1];
  const int t = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool live = row < rows;
  float v[VPT][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = t + i * TPR;
    if (live && c < dim8) {
      load_values<__nv_bfloat16, 8, true>(reinterpret_cast<const __nv_bfloat16*>(x + row * dim8 + c), 8, v[i]);
      if (RESIDUAL) {
        float r[8];
        load_values<__nv_bfloat16, 8, true>(reinterpret_cast<const __nv_bfloat16*>(res + row * dim8 + c), 8, r);
        uint4 packed;
        __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(&packed);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = __float2bfloat16_rn(v[i][j] + r[j]);
          v[i][j] = to_float(e[j]);
        }
        h[row * dim8 + c] = packed;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) ss += red[i];
  }
  const float rs = rsqrtf(ss * inv_dim + eps);
  if (live && t == 0) rstd[row] = rs;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = t + i * TPR;
    if ((c & ~31) >= dim8) break;  // the whole warp is past the row
    float g[8], y[8];
    if (c < dim8) {
      load_values<__nv_bfloat16, 8, true>(reinterpret_cast<const __nv_bfloat16*>(w + c), 8, g);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = c < dim8 ? v[i][j] * rs * g[j] : 0.f;
    uint32_t q[2];
    const uint32_t byte = quantize_block<8, 16>(y, q);
    if (live && c < dim8) {
      *reinterpret_cast<uint2*>(data + row * ldq + c * 8) = make_uint2(q[0], q[1]);
      if ((c & 15) == 0) scale[row * lds + c / 16] = uint8_t(byte);
    }
  }
}

bool aligned16(const void* p, long long pitch_bytes) { return ((reinterpret_cast<uintptr_t>(p) | uintptr_t(pitch_bytes)) & 15) == 0; }

// rows per launch, so that a launch's units fit 31 bits
long long rows_per_launch(uint32_t units_per_row) { return std::max(1ll, (1ll << 30) / units_per_row); }

template <typename T>
cudaError_t quantize_rows_as(const void* x, long long ldx, uint8_t* data, long long ldq, uint8_t* scale, long long lds, long long rows, int cols,
                             cudaStream_t stream) {
  const bool vec = cols % UNIT == 0 && aligned16(x, ldx * sizeof(T)) && aligned16(data, ldq);
  const uint32_t upr = uint32_t((cols + BLOCK - 1) / BLOCK) * (BLOCK / UNIT);
  const long long step = rows_per_launch(upr);
  for (long long r = 0; r < rows; r += step) {
    const uint32_t total = uint32_t(std::min(step, rows - r)) * upr;
    auto* kern = vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>;
    kern<<<(total + THREADS - 1) / THREADS, THREADS, 0, stream>>>(static_cast<const T*>(x) + r * ldx, ldx, data + r * ldq, ldq, scale + r * lds, lds, total,
                                                                  upr, cols);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t quantize_tiles_as(const void* x, long long ldx, uint8_t* data, long long ldq, uint8_t* scale, long long lds, long long rows, int cols,
                              cudaStream_t stream) {
  const bool vec = cols % UNIT == 0 && aligned16(x, ldx * sizeof(T)) && aligned16(data, ldq);
  constexpr long long kGridY = 65535;
  const long long tiles = (rows + BLOCK - 1) / BLOCK;
  for (long long t = 0; t < tiles; t += kGridY) {
    const long long r = t * BLOCK;
    const dim3 grid((cols + BLOCK - 1) / BLOCK, unsigned(std::min(kGridY, tiles - t)));
    auto* kern = vec ? quantize_tiles_kernel<T, true> : quantize_tiles_kernel<T, false>;
    kern<<<grid, THREADS, 0, stream>>>(static_cast<const T*>(x) + r * ldx, ldx, data + r * ldq, ldq, scale + t * lds, lds, rows - r, cols);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize_as(const uint8_t* data, long long ldq, const uint8_t* scale, long long lds, int row_shift, void* y, long long ldy, long long rows,
                          int cols, cudaStream_t stream) {
  const bool vec = cols % UNIT == 0 && aligned16(y, ldy * sizeof(T)) && aligned16(data, ldq);
  const uint32_t upr = uint32_t((cols + UNIT - 1) / UNIT);
  const long long step = rows_per_launch(upr);
  for (long long r = 0; r < rows; r += step) {
    const uint32_t total = uint32_t(std::min(step, rows - r)) * upr;
    auto* kern = vec ? dequantize_kernel<T, true> : dequantize_kernel<T, false>;
    kern<<<(total + THREADS - 1) / THREADS, THREADS, 0, stream>>>(data, ldq, scale, lds, row_shift, static_cast<T*>(y), ldy, total, upr, r, cols);
  }
  return cudaGetLastError();
}

template <int TPR, int VPT>
cudaError_t rmsnorm_as(const void* x, const void* residual, const void* w, void* h, float* rstd, uint8_t* data, long long ldq, uint8_t* scale, long long lds,
                       long long rows, int dim, float eps, cudaStream_t stream) {
  constexpr int threads = TPR < 128 ? 128 : TPR;
  const long long blocks = (rows + threads / TPR - 1) / (threads / TPR);
  auto* kern = residual ? rmsnorm_fp8_kernel<TPR, VPT, true> : rmsnorm_fp8_kernel<TPR, VPT, false>;
  kern<<<unsigned(blocks), threads, 0, stream>>>(static_cast<const uint4*>(x), static_cast<const uint4*>(residual), static_cast<const uint4*>(w),
                                                 static_cast<uint4*>(h), rstd, data, ldq, scale, lds, rows, dim / 8, 1.f / float(dim), eps);
  return cudaGetLastError();
}

}  // namespace

cudaError_t fp8_quantize_rows(const void* x, Elem type, long long ldx, uint8_t* data, long long ldq, uint8_t* scale, long long lds, long long rows, int cols,
                              cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (type == Elem::kBf16) return quantize_rows_as<__nv_bfloat16>(x, ldx, data, ldq, scale, lds, rows, cols, stream);
  if (type == Elem::kF16) return quantize_rows_as<__half>(x, ldx, data, ldq, scale, lds, rows, cols, stream);
  return quantize_rows_as<float>(x, ldx, data, ldq, scale, lds, rows, cols, stream);
}

cudaError_t fp8_quantize_tiles(const void* x, Elem type, long long ldx, uint8_t* data, long long ldq, uint8_t* scale, long long lds, long long rows, int cols,
                               cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (type == Elem::kBf16) return quantize_tiles_as<__nv_bfloat16>(x, ldx, data, ldq, scale, lds, rows, cols, stream);
  if (type == Elem::kF16) return quantize_tiles_as<__half>(x, ldx, data, ldq, scale, lds, rows, cols, stream);
  return quantize_tiles_as<float>(x, ldx, data, ldq, scale, lds, rows, cols, stream);
}

cudaError_t fp8_dequantize(const uint8_t* data, long long ldq, const uint8_t* scale, long long lds, int row_shift, void* y, Elem type, long long ldy,
                           long long rows, int cols, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (type == Elem::kBf16) return dequantize_as<__nv_bfloat16>(data, ldq, scale, lds, row_shift, y, ldy, rows, cols, stream);
  if (type == Elem::kF16) return dequantize_as<__half>(data, ldq, scale, lds, row_shift, y, ldy, rows, cols, stream);
  return dequantize_as<float>(data, ldq, scale, lds, row_shift, y, ldy, rows, cols, stream);
}

cudaError_t fp8_rmsnorm(const void* x, const void* residual, const void* w, void* h, float* rstd, uint8_t* data, long long ldq, uint8_t* scale,
                        long long lds, long long rows, int dim, float eps, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  if (dim <= 0 || dim % 8 || dim > 8192 || rows > (1ll << 31) - 1) return cudaErrorInvalidValue;
  // the fewest threads per row that still hold it in at most four 16-byte steps each
#define ELFB_NORM(TPR, VPT) return rmsnorm_as<TPR, VPT>(x, residual, w, h, rstd, data, ldq, scale, lds, rows, dim, eps, stream)
  if (dim <= 256) ELFB_NORM(32, 1);
  if (dim <= 512) ELFB_NORM(32, 2);
  if (dim <= 1024) ELFB_NORM(32, 4);
  if (dim <= 2048) ELFB_NORM(128, 2);
  if (dim <= 4096) ELFB_NORM(128, 4);
  ELFB_NORM(256, 4);
#undef ELFB_NORM
}

}  // namespace elfb
