// What the two kernels of the block-scaled products (one CTA, CTA pair) share: scale words, epilogues.
#pragma once

#include <type_traits>

#include "fp8_block.cuh"
#include "fp8_ops.h"
#include "sm100_ptx.cuh"

namespace elfb {
namespace fp8 {

constexpr int BM = 128;  // rows per CTA
constexpr int BK = 128;  // bytes = values; one scale block
constexpr int UMMA_K = 32;
constexpr int BOX_BYTES = 128 * BK;  // 16 KiB: 128 rows of an operand
constexpr int TMEM_COLS = 512;
constexpr int SF_COL = 480;  // two 16-column scale slots: A's 4 columns, then B's

struct Scales {
  const uint8_t* p;
  long long row_stride, block_stride;
  int row_shift;
  bool words;  // the bytes of four consecutive blocks can be read as one aligned word
  explicit Scales(const Fp8Operand& o)
      : p(o.scale), row_stride(o.row_stride), block_stride(o.block_stride), row_shift(o.row_shift),
        words(o.block_stride == 1 && o.row_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(o.scale) & 3) == 0) {}
};

struct Params {
  int M, N, K;
  Scales sa, sb;
  void* d;
  long long ldd;
  const void* bias;
  bool vec;  // D may be stored in 16-byte pieces
  // gated form
  uint8_t *act, *act_scale, *gu, *gu_scale;
  long long ld_act, ld_act_scale, ld_gu, ld_gu_scale;
  int* status;
};

// Exponent bytes of blocks 4g .. 4g+3 for rows row0 + lane, + 32, + 64, + 96 of an operand, as they come from
// memory: nothing here looks at a loaded value, so a warp issues the loads of all operands and goes on; they are
// combined one group of blocks later, when they have long arrived.
struct RawScales {
  uint32_t v[4][4];  // [row][byte]; aligned words: [row][0]; one scale for all 128 rows: [0]
};
// Rows and blocks that do not exist read the last that does: what they scale is zero, or never used.
__device__ __forceinline__ void load_scales(const Scales& s, int row0, int rows, int g, int blocks, int lane, RawScales& r) {
  const bool word = s.words && 4 * g + 4 <= blocks;
  const int n = s.row_shift ? 1 : 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j < n) {
      const int row = s.row_shift ? min(row0, rows - 1) >> 7 : min(row0 + 32 * j + lane, rows - 1);
      const uint8_t* p = s.p + (long long)row * s.row_stride;
      if (word) {
        r.v[j][0] = *reinterpret_cast<const uint32_t*>(p + 4 * g);
      } else {
#pragma unroll
        for (int b = 0; b < 4; ++b) r.v[j][b] = p[(long long)min(4 * g + b, blocks - 1) * s.block_stride];
      }
    }
  }
}
__device__ __forceinline__ void combine_scales(const Scales& s, int g, int blocks, const RawScales& r, uint32_t (&w)[4]) {
  const bool word = s.words && 4 * g + 4 <= blocks;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t v[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) v[b] = s.row_shift ? r.v[0][b] : r.v[j][b];
    w[j] = word ? v[0] : v[0] | v[1] << 8 | v[2] << 16 | v[3] << 24;
  }
}

template <typename T>
__device__ __forceinline__ float bias_at(const void* bias, int col) {
  const T v = static_cast<const T*>(bias)[col];
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T rounded(float f) {
  if constexpr (sizeof(T) == 4) return f;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(f);
  else return __float2bfloat16_rn(f);
}
// v[i] of lane l becomes v[l] of lane i
__device__ __forceinline__ void transpose_32x32(uint32_t (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1)
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if ((i & s) == 0) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & s ? v[i] : v[i | s], s);
        if (lane & s) v[i] = got;
        else v[i | s] = got;
      }
}
// D[row, col .. col+32) = v (+ bias) for the 32 rows of a warp, all of whose lanes call this.  Where D's rows or its last
// columns do not allow 16-byte pieces the warp turns the block over and writes row by row, lanes side by side: stores of
// single values down a column touched 32 sectors each (4069 x 5803 from 58: 241 us).
template <typename T>
__device__ __forceinline__ void store_chunk(uint32_t (&v)[32], int row, int col, const Params& p) {
  if (!p.vec || col + 32 > p.N) {
    const int lane = threadIdx.x & 31, row0 = row - lane;
    transpose_32x32(v);
    const bool live = col + lane < p.N;
    const float bias = p.bias != nullptr && live ? bias_at<T>(p.bias, col + lane) : 0.f;
    T* dst = static_cast<T*>(p.d) + (long long)row0 * p.ldd + col + lane;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (live && row0 + i < p.M) dst[i * p.ldd] = rounded<T>(p.bias != nullptr ? __uint_as_float(v[i]) + bias : __uint_as_float(v[i]));
    return;
  }
  if (row >= p.M) return;
  T* dst = static_cast<T*>(p.d) + (long long)row * p.ldd + col;
  float f[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
  if (p.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] += bias_at<T>(p.bias, col + j);
  }
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(dst + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      uint4 o;
      if constexpr (std::is_same<T, __half>::value)
        o = make_uint4(pack_f16x2(f[j], f[j + 1]), pack_f16x2(f[j + 2], f[j + 3]), pack_f16x2(f[j + 4], f[j + 5]), pack_f16x2(f[j + 6], f[j + 7]));
      else
        o = make_uint4(pack_bf16x2(f[j], f[j + 1]), pack_bf16x2(f[j + 2], f[j + 3]), pack_bf16x2(f[j + 4], f[j + 5]), pack_bf16x2(f[j + 6], f[j + 7]));
      *reinterpret_cast<uint4*>(dst + j) = o;
    }
  }
}

// D[row, col .. col+4) = s (+ bias); row < M
template <typename T>
__device__ __forceinline__ void store_quad(float (&s)[4], int row, int col, const Params& p) {
  T* dst = static_cast<T*>(p.d) + (long long)row * p.ldd + col;
  alignas(16) T o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (p.bias != nullptr && col + j < p.N) s[j] += bias_at<T>(p.bias, col + j);
    o[j] = rounded<T>(s[j]);
  }
  if (p.vec && col + 4 <= p.N) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(o);
    else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < p.N) dst[j] = o[j];
  }
}

// 32-byte accesses (addresses 32-byte aligned): a lane whose row is its own moves whole sectors.
__device__ __forceinline__ void load_32_bytes(const uint8_t* p, uint32_t (&v)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void store_32_bytes(uint8_t* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
               "r"(v[6]), "r"(v[7])
               : "memory");
}
// N values times 2^(127 - byte) to e4m3.  ODD: some may not be finite and become NaN; without it that costs nothing.
template <int N, bool ODD>
__device__ __forceinline__ void to_scaled_e4m3(const float* v, float inv, uint32_t* q) {
  const uint64_t inv2 = pair_of(inv, inv);
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    float2 a = halves(mul2(pair_of(v[4 * j], v[4 * j + 1]), inv2)), b = halves(mul2(pair_of(v[4 * j + 2], v[4 * j + 3]), inv2));
    if (ODD) {
      a = make_float2(nan_unless_finite(a.x, v[4 * j]), nan_unless_finite(a.y, v[4 * j + 1]));
      b = make_float2(nan_unless_finite(b.x, v[4 * j + 2]), nan_unless_finite(b.y, v[4 * j + 3]));
    }
    q[j] = to_e4m3x4(a.x, a.y, b.x, b.y);
  }
}
template <int N, bool ODD>
__device__ __forceinline__ void scale_and_store(const float* v, float inv, uint8_t* dst) {
#pragma unroll
  for (int c = 0; c < N / 32; ++c) {
    uint32_t q[8];
    to_scaled_e4m3<32, ODD>(v + 32 * c, inv, q);
    store_32_bytes(dst + 32 * c, q);
  }
}
// largest magnitude as fp32 bits; ODD: of the values that are finite, otherwise infinity or more if one is not
template <int N, bool ODD>
__device__ __forceinline__ uint32_t magnitude(const float* v, uint32_t top = 0) {
  if constexpr (ODD) {
#pragma unroll
    for (int j = 0; j < N; ++j) top = max(top, finite_bits(v[j]));
    return top;
  } else {
    float m[4] = {__uint_as_float(top), 0.f, 0.f, 0.f};  // four short chains
#pragma unroll
    for (int j = 0; j < N; ++j) m[j % 4] = larger_magnitude(m[j % 4], v[j]);
    return abs_bits(larger_magnitude(larger_magnitude(m[0], m[1]), larger_magnitude(m[2], m[3])));
  }
}

// The layout tcgen05.cp wants: 16 bytes per lane, word j for row 32 j + lane.
__device__ __forceinline__ void store_scale_words(uint32_t smem, int lane, const uint32_t (&w)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem + lane * 16), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
}  // namespace fp8
}  // namespace elfb
