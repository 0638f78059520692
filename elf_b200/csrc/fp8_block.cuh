// Scaling and conversion of blocks of e4m3 values, and how their kernels are launched, shared by the kernels that write
// or read them.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace elfb {

// A kernel starts before the one in front of it in its stream has ended: barriers, TMEM and its blocks' places are ready
// by then.  `await_previous` comes before a kernel's first access to global memory; it returns when everything in front
// has ended and its writes are visible (a launch of another kind has ended before this one starts).  Saves 1 to 4 us a
// launch: quantise and restore 2047 x 5504 15.8 -> 12.2 us, 16 x 4096 x 14336 17.6 -> 15.9.
template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kern)(Params...), dim3 grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (cluster > 0) {  // 0: as the kernel says
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attrs;
  return cudaLaunchKernelEx(&cfg, kern, Params(args)...);
}
__device__ __forceinline__ void await_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Products by powers of two are exact as long as subnormal inputs and results survive, so they are
// written out: the library is built with flush-to-zero arithmetic.
__device__ __forceinline__ float mul_exact(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float add_exact(float a, float b) {
  float r;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two fp32 operations in one instruction, on a pair in a 64-bit register; subnormal numbers survive.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t fma2_towards_zero(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// larger magnitude of the two (the sign is arbitrary), NaN if either is
__device__ __forceinline__ float larger_magnitude(float a, float b) {
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr uint32_t kInfBits = 0x7f800000u;

// Exponent byte of a block whose largest finite magnitude has the bits `amax` (an fp32 pattern):
// the smallest power of two s with amax <= 448 s.  448 = 1.75 * 2^8, so with amax = m * 2^e the
// exponent is e - 8 where m <= 1.75 and e - 7 above; subnormal and zero blocks get the smallest
// scale that is itself a normal number.
__device__ __forceinline__ uint32_t block_exponent(uint32_t amax) {
  const int e = int(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return uint32_t(e < 1 ? 1 : e);
}
// 2^(byte - 127); bytes 0 and 255 (never written here, legal in a tensor from elsewhere) are 2^-127 and NaN
__device__ __forceinline__ float exponent_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}
// 2^(127 - byte) for bytes 1 to 253
__device__ __forceinline__ float inverse_exponent_value(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// two values to e4m3, round to nearest even: lo in bits 0-7, hi in bits 8-15
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) { return to_e4m3x2(a, b) | (to_e4m3x2(c, d) << 16); }
__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {  // exact
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(v)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// magnitude that counts towards a block's maximum: what is not finite does not
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = abs_bits(v);
  return b < kInfBits ? b : 0u;
}
// a value that is not finite becomes NaN (an infinity would otherwise saturate to a finite 448)
__device__ __forceinline__ float nan_unless_finite(float scaled, float v) { return abs_bits(v) < kInfBits ? scaled : __uint_as_float(0x7fc00000u); }

// maximum over groups of W consecutive lanes
template <int W>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <int N>
__device__ __forceinline__ void scaled_to_e4m3(const float (&v)[N], float inv, uint32_t (&out)[N / 4]) {
  const uint64_t inv2 = pair_of(inv, inv);
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    const float2 a = halves(mul2(pair_of(v[4 * j], v[4 * j + 1]), inv2)), b = halves(mul2(pair_of(v[4 * j + 2], v[4 * j + 3]), inv2));
    out[j] = to_e4m3x4(a.x, a.y, b.x, b.y);
  }
}
template <int N>
__device__ __forceinline__ void scaled_to_e4m3_odd(const float (&v)[N], float inv, uint32_t (&out)[N / 4]) {  // with infinities or NaN
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    float s[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = nan_unless_finite(mul_exact(v[4 * j + k], inv), v[4 * j + k]);
    out[j] = to_e4m3x4(s[0], s[1], s[2], s[3]);
  }
}
// Scales and converts the N values a lane holds of a 128-column block shared by W consecutive lanes (all 32 lanes of
// the warp call this); `top` is the largest magnitude among the lane's values.  Returns the block's exponent byte.
// Blocks without infinities and NaN, practically all, take the branch without per-value tests.
template <int N, int W>
__device__ __forceinline__ uint32_t quantize_block(const float (&v)[N], uint32_t top, uint32_t (&out)[N / 4]) {
  top = group_max<W>(top);
  if (__any_sync(0xffffffffu, top >= kInfBits)) {
    uint32_t f = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) f = max(f, finite_bits(v[j]));
    const uint32_t byte = block_exponent(group_max<W>(f));
    scaled_to_e4m3_odd(v, inverse_exponent_value(byte), out);
    return byte;
  }
  const uint32_t byte = block_exponent(top);
  scaled_to_e4m3(v, inverse_exponent_value(byte), out);
  return byte;
}

}  // namespace elfb
