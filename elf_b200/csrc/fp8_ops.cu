// Bandwidth-bound kernels that write or read block-scaled 8-bit tensors: quantise, restore, RMSNorm
// with an 8-bit output, and bf16 parts of wider operands.  Each reads its inputs once and writes its outputs once; arithmetic is
// fp32, the norm's statistic 64 bits once a thread's squares are added.
#include "fp8_ops.h"

#include <algorithm>
#include <type_traits>

#include "fp8_block.cuh"
#include "sm100_ptx.cuh"

namespace elfb {

namespace {

constexpr int BLOCK = 128;  // columns that share a scale
constexpr int UNIT = 16;    // consecutive values a thread holds: 8 lanes make up a block
constexpr int THREADS = 256;
constexpr int NORM_THREADS = 256;
constexpr int TILE_THREADS = 512;
constexpr int UNITS = 2;    // groups of 16 values per thread of the streaming kernels

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

// How a thread's 16 values are moved: in pieces of 32 bytes where rows start on such addresses and hold whole units (the
// 8-bit rows in 16-byte pieces then), in pieces of 16 bytes, or in 16-byte pieces shifted into place.  Units that a row's
// end cuts off go one value at a time; kernels without that code are 3 to 5 % faster.
enum class Access { kShifted, kPieces16, kPieces32 };

__device__ __forceinline__ void load_piece(const void* p, uint4& a) { a = *static_cast<const uint4*>(p); }
__device__ __forceinline__ void load_piece(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p));
}
__device__ __forceinline__ void store_piece(void* p, uint4 a, uint4 b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// UNIT consecutive values as they lie in memory.
template <typename T>
struct Raw {
  uint4 q[UNIT * sizeof(T) / 16];
};
// N words of the stream w, from its byte `shift` (0 to 15) on
template <int N>
__device__ __forceinline__ void shifted(uint32_t (&w)[N + 4], uint32_t shift, uint32_t (&out)[N]) {
  if (shift & 8)
#pragma unroll
    for (int j = 0; j < N + 2; ++j) w[j] = w[j + 2];
  if (shift & 4)
#pragma unroll
    for (int j = 0; j < N + 1; ++j) w[j] = w[j + 1];
#pragma unroll
  for (int j = 0; j < N; ++j) out[j] = __funnelshift_r(w[j], w[j + 1], (shift & 3) * 8);
}
struct Span {  // of a matrix in memory: what may be read around a row
  uintptr_t begin, end;
};
// Units are loaded in two steps, whole ones of all groups first: a branch between two groups' loads would make the
// second wait for the first.
template <typename T, Access A>
__device__ __forceinline__ bool loads_whole(const T* p, int have, Span span) {
  if constexpr (A == Access::kPieces32) return have > 0;
  const uintptr_t base = reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15);
  return have >= UNIT && (A != Access::kShifted || (base >= span.begin && base + UNIT * sizeof(T) + 16 <= span.end));
}
template <typename T, Access A>
__device__ __forceinline__ void load_whole(const T* p, Raw<T>& r) {
  constexpr int N = UNIT * sizeof(T) / 16;
  if constexpr (A == Access::kPieces32) {
#pragma unroll
    for (int i = 0; i < N; i += 2) load_piece(reinterpret_cast<const uint4*>(p) + i, r.q[i], r.q[i + 1]);
  } else if constexpr (A == Access::kPieces16) {
#pragma unroll
    for (int i = 0; i < N; ++i) load_piece(reinterpret_cast<const uint4*>(p) + i, r.q[i]);
  } else {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), base = at & ~uintptr_t(15);
    uint32_t w[4 * N + 4], out[4 * N];
#pragma unroll
    for (int i = 0; i <= N; ++i) {
      const uint4 t = reinterpret_cast<const uint4*>(base)[i];
      w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
    }
    shifted<4 * N>(w, uint32_t(at & 15), out);
#pragma unroll
    for (int i = 0; i < N; ++i) r.q[i] = make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
  }
}
template <typename T>
__device__ __forceinline__ void load_part(const T* p, int have, Raw<T>& r) {
  T* e = reinterpret_cast<T*>(r.q);
#pragma unroll
  for (int j = 0; j < UNIT; ++j) e[j] = j < have ? p[j] : T{};
}
// units of `G` groups; nothing is there where have[i] <= 0
template <typename T, Access A, int G>
__device__ __forceinline__ void load_groups(const T* const (&p)[G], const int (&have)[G], Span span, Raw<T> (&r)[G]) {
#pragma unroll
  for (int i = 0; i < G; ++i) {
    if (loads_whole<T, A>(p[i], have[i], span)) {
      load_whole<T, A>(p[i], r[i]);
    } else {
#pragma unroll
      for (uint4& q : r[i].q) q = make_uint4(0, 0, 0, 0);
    }
  }
  if constexpr (A != Access::kPieces32) {
#pragma unroll
    for (int i = 0; i < G; ++i)
      if (have[i] > 0 && !loads_whole<T, A>(p[i], have[i], span)) load_part(p[i], have[i], r[i]);
  }
}
template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float (&v)[UNIT]) {
  const T* e = reinterpret_cast<const T*>(r.q);
#pragma unroll
  for (int j = 0; j < UNIT; ++j) v[j] = to_float(e[j]);
}
// Largest magnitude as the bits of an fp32 number, those of infinity or more if a value is not finite.  16-bit values are
// compared two at a time, as integers.
template <typename T>
__device__ __forceinline__ uint32_t largest(const Raw<T>& r) {
  uint32_t top = 0;
#pragma unroll
  for (const uint4& q : r.q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) top = max(top, w[j] & 0x7fffffffu);
      else top = __vmaxu2(top, w[j] & 0x7fff7fffu);
    }
  }
  if constexpr (sizeof(T) == 4) return top;
  const uint32_t m = max(top >> 16, top & 0xffffu);
  if constexpr (std::is_same<T, __half>::value) return m >= 0x7c00u ? kInfBits : __float_as_uint(__half2float(__ushort_as_half(uint16_t(m))));
  else return m << 16;
}
// Stores a lane's unit of a row; all 32 lanes of the warp call this, lanes with consecutive units.  kShifted: 16-byte
// pieces lie across two lanes' units; a lane stores those that begin in its own, with the start of the next lane's.
template <typename T, Access A>
__device__ __forceinline__ void store_raw(T* p, int col, int have, const Raw<T>& r) {
  constexpr int N = UNIT * sizeof(T) / 16;
  const T* e = reinterpret_cast<const T*>(r.q);
  int last = have;  // elements stored one by one
  if constexpr (A == Access::kPieces32) {
    if (have > 0) {
#pragma unroll
      for (int i = 0; i < N; i += 2) store_piece(reinterpret_cast<uint4*>(p) + i, r.q[i], r.q[i + 1]);
    }
    return;
  } else if constexpr (A == Access::kPieces16) {
    if (have >= UNIT) {
      last = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(p)[i] = r.q[i];
    }
  } else {
    const int lane = threadIdx.x & 31;
    const int next_col = __shfl_down_sync(0xffffffffu, col, 1), next_have = __shfl_down_sync(0xffffffffu, have, 1);
    uint32_t w[4 * N + 4], out[4 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[4 * i] = r.q[i].x, w[4 * i + 1] = r.q[i].y, w[4 * i + 2] = r.q[i].z, w[4 * i + 3] = r.q[i].w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[4 * N + j] = __shfl_down_sync(0xffffffffu, w[j], 1);
    if (have >= UNIT) {
      const uint32_t head = (16 - uint32_t(reinterpret_cast<uintptr_t>(p) & 15)) & 15;  // bytes before the first piece
      const bool joined = lane < 31 && next_col == col + UNIT && next_have >= UNIT;     // the next lane's start is at hand
      const bool taken = lane > 0 && col > 0;                                           // the lane before stores this one's start
      uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(p) + head);
      shifted<4 * N>(w, head, out);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i + 1 < N || head == 0 || joined) dst[i] = make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
      // what is left: a start that nobody takes, an end that nobody joins
      const int before = int(head / sizeof(T)), after = head == 0 ? UNIT : before + (N - 1) * int(16 / sizeof(T));
#pragma unroll
      for (int j = 0; j < UNIT; ++j)
        if ((j < before && !taken) || (j >= after && !joined)) p[j] = e[j];
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < UNIT; ++j)
    if (j < last) p[j] = e[j];
}
template <typename T, Access A>
__device__ __forceinline__ void store_values(T* p, int col, int have, const float (&v)[UNIT]) {
  Raw<T> r;
  T* e = reinterpret_cast<T*>(r.q);
#pragma unroll
  for (int j = 0; j < UNIT; ++j) e[j] = from_float<T>(v[j]);
  store_raw<T, A>(p, col, have, r);
}
__device__ __forceinline__ void store_bytes_ragged(uint8_t* p, int have, const uint32_t (&q)[UNIT / 4]) {
#pragma unroll
  for (int j = 0; j < UNIT; ++j)
    if (j < have) p[j] = uint8_t(q[j / 4] >> (8 * (j % 4)));
}

// ------------------------------------------------------------------------------ quantise
// A thread takes two groups of 16 values, 256 groups apart, and loads both before it looks at either; the 8 lanes
// of a block find its maximum with three shuffles.  Bound by memory: 4096 x 28672 bf16 (353 MB read and written)
// 51 us, 6.9 TB/s.
template <typename T, Access A>
__global__ void __launch_bounds__(THREADS) quantize_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ data, long long ldq,
                                                                uint8_t* __restrict__ scale, long long lds, uint32_t total, uint32_t units_per_row,
                                                                int cols, Span span, bool packed) {
  await_previous();
  Raw<T> raw[UNITS];
  const T* src[UNITS];
  uint32_t row[UNITS];
  int col[UNITS], have[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const uint32_t u = (blockIdx.x * UNITS + i) * THREADS + threadIdx.x;
    row[i] = u / units_per_row;
    col[i] = int(u - row[i] * units_per_row) * UNIT;
    have[i] = u < total ? min(cols - col[i], UNIT) : 0;  // 0 or less: padding of a row's last block
    src[i] = x + (long long)row[i] * ldx + col[i];
  }
  load_groups<T, A>(src, have, span, raw);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    float v[UNIT];
    unpack<T>(raw[i], v);
    uint32_t q[UNIT / 4];
    const uint32_t byte = quantize_block<UNIT, 8>(v, largest(raw[i]), q);
    if (have[i] > 0) {
      uint8_t* dst = data + (long long)row[i] * ldq + col[i];
      if (A == Access::kPieces32 || (packed && have[i] == UNIT)) *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
      else store_bytes_ragged(dst, have[i], q);
      if ((col[i] & (BLOCK - 1)) == 0) scale[(long long)row[i] * lds + col[i] / BLOCK] = uint8_t(byte);
    }
  }
}

// One block of threads per 128 x 128 tile: every thread holds two groups of 16 values (64 rows apart), so the tile is
// read once.  Bound by memory: 28672 x 4096 bf16 (353 MB) 65 us, 5.4 TB/s; with 256 threads of four groups, one block to an
// SM, 129.
template <typename T, Access A>
__global__ void __launch_bounds__(TILE_THREADS, 2) quantize_tiles_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ data, long long ldq,
                                                                 uint8_t* __restrict__ scale, long long lds, long long rows, int cols, Span span, bool packed) {
  __shared__ uint32_t warp_max[TILE_THREADS / 32];
  await_previous();
  const int col = blockIdx.x * BLOCK + (threadIdx.x & 7) * UNIT;
  const long long row0 = (long long)blockIdx.y * BLOCK + (threadIdx.x >> 3);
  const int have_cols = min(cols - col, UNIT);
  constexpr int GROUPS = BLOCK * BLOCK / UNIT / TILE_THREADS, STEP = BLOCK / GROUPS;
  Raw<T> raw[GROUPS];
  const T* src[GROUPS];
  int have[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const long long row = row0 + STEP * i;
    src[i] = x + row * ldx + col;
    have[i] = row < rows ? have_cols : 0;
  }
  load_groups<T, A>(src, have, span, raw);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) top = max(top, largest(raw[i]));
  auto tile_max = [&](uint32_t m) {
    m = group_max<32>(m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TILE_THREADS / 32; ++w) m = max(m, warp_max[w]);
    return m;
  };
  top = tile_max(top);
  const bool odd = top >= kInfBits;
  if (odd) {  // the largest of the finite values counts
    top = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      float v[UNIT];
      unpack<T>(raw[i], v);
#pragma unroll
      for (int j = 0; j < UNIT; ++j) top = max(top, finite_bits(v[j]));
    }
    __syncthreads();
    top = tile_max(top);
  }
  const uint32_t byte = block_exponent(top);
  const float inv = inverse_exponent_value(byte);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const long long row = row0 + STEP * i;
    if (have_cols <= 0 || row >= rows) continue;
    float v[UNIT];
    unpack<T>(raw[i], v);
    uint32_t q[UNIT / 4];
    if (odd) scaled_to_e4m3_odd(v, inv, q);
    else scaled_to_e4m3(v, inv, q);
    uint8_t* dst = data + row * ldq + col;
    if (A == Access::kPieces32 || (packed && have_cols == UNIT)) *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
    else store_bytes_ragged(dst, have_cols, q);
  }
  if (threadIdx.x == 0) scale[(long long)blockIdx.y * lds + blockIdx.x] = uint8_t(byte);
}

// ------------------------------------------------------------------------------ restore
// value = data 2^(byte - 127), exact in fp32, one rounding where the output has fewer bits.  Units as above.  Bound by
// memory: 4096 x 28672 to bf16 (353 MB) 53 us, 6.6 TB/s.
template <typename T, Access A>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(const uint8_t* __restrict__ data, long long ldq, const uint8_t* __restrict__ scale,
                                                             long long lds, int row_shift, T* __restrict__ y, long long ldy, uint32_t total,
                                                             uint32_t units_per_row, long long first_row, int cols, bool packed) {
  await_previous();
  uint32_t q[UNITS][UNIT / 4], byte[UNITS];
  long long row[UNITS];
  int col[UNITS], have[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const uint32_t u = (blockIdx.x * UNITS + i) * THREADS + threadIdx.x;
    const uint32_t r = u / units_per_row;
    row[i] = first_row + r;
    col[i] = int(u - r * units_per_row) * UNIT;
    have[i] = u < total ? min(cols - col[i], UNIT) : 0;
    const uint8_t* src = data + row[i] * ldq + col[i];
    q[i][0] = q[i][1] = q[i][2] = q[i][3] = byte[i] = 0;
    if (have[i] > 0) byte[i] = scale[(row[i] >> row_shift) * lds + col[i] / BLOCK];
    if (A == Access::kPieces32 ? have[i] > 0 : packed && have[i] >= UNIT) {
      const uint4 t = *reinterpret_cast<const uint4*>(src);
      q[i][0] = t.x, q[i][1] = t.y, q[i][2] = t.z, q[i][3] = t.w;
    }
  }
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {  // cut off by the row's end, or on no 16-byte boundary
    if (A == Access::kPieces32 || have[i] <= 0 || (packed && have[i] >= UNIT)) continue;
    const uint8_t* src = data + row[i] * ldq + col[i];
#pragma unroll
    for (int j = 0; j < UNIT; ++j)
      if (j < have[i]) q[i][j / 4] |= uint32_t(src[j]) << (8 * (j % 4));
  }
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const float s = exponent_value(byte[i]);
    float v[UNIT];
#pragma unroll
    for (int j = 0; j < UNIT / 4; ++j) {
      const float2 lo = from_e4m3x2(q[i][j] & 0xffffu), hi = from_e4m3x2(q[i][j] >> 16);
      v[4 * j] = mul_exact(lo.x, s);
      v[4 * j + 1] = mul_exact(lo.y, s);
      v[4 * j + 2] = mul_exact(hi.x, s);
      v[4 * j + 3] = mul_exact(hi.y, s);
    }
    store_values<T, A>(y + row[i] * ldy + col[i], col[i], have[i], v);
  }
}

// ------------------------------------------------------------------------------ rows moved to another pitch
// TMA wants rows on 16-byte boundaries, a caller's tensor or a dense result may have them anywhere: one pass over the bytes.
template <Access FROM, Access TO>
__global__ void __launch_bounds__(THREADS) repack_kernel(const uint8_t* __restrict__ src, long long ld_src, uint8_t* __restrict__ dst, long long ld_dst,
                                                         uint32_t total, uint32_t units_per_row, int row_bytes, Span span) {
  await_previous();
  Raw<uint8_t> raw[2 * UNITS];
  const uint8_t* from[2 * UNITS];
  uint32_t row[2 * UNITS];
  int col[2 * UNITS], have[2 * UNITS];
#pragma unroll
  for (int i = 0; i < 2 * UNITS; ++i) {
    const uint32_t u = (blockIdx.x * 2 * UNITS + i) * THREADS + threadIdx.x;
    row[i] = u / units_per_row;
    col[i] = int(u - row[i] * units_per_row) * UNIT;
    have[i] = u < total ? min(row_bytes - col[i], UNIT) : 0;
    from[i] = src + (long long)row[i] * ld_src + col[i];
  }
  load_groups<uint8_t, FROM>(from, have, span, raw);
#pragma unroll
  for (int i = 0; i < 2 * UNITS; ++i) store_raw<uint8_t, TO>(dst + (long long)row[i] * ld_dst + col[i], col[i], have[i], raw[i]);
}

// ------------------------------------------------------------------------------ 16- and 32-bit values as sums of bf16
// Operands of the 16-bit product that are not bf16: a value is cut off after 8 significant bits, what is left again.  fp16 has
// 11 bits and is the sum of two parts, fp32 has 24 and is that of three, both exactly (down to bf16's smallest step, 2^-133).
// Infinities and NaN are all in the first part.
template <typename T>
constexpr int BF16_PARTS = sizeof(T) == 2 ? 2 : 3;
template <typename T, Access A>
__global__ void __launch_bounds__(THREADS) bf16_parts_kernel(const T* __restrict__ x, long long ldx, __nv_bfloat16* __restrict__ out, long long ldo,
                                                             long long part_step, uint32_t total, uint32_t units_per_row, int cols, Span span) {
  await_previous();
  Raw<T> raw[UNITS];
  const T* src[UNITS];
  uint32_t row[UNITS];
  int col[UNITS], have[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const uint32_t u = (blockIdx.x * UNITS + i) * THREADS + threadIdx.x;
    row[i] = u / units_per_row;
    col[i] = int(u - row[i] * units_per_row) * UNIT;
    have[i] = u < total ? min(cols - col[i], UNIT) : 0;
    src[i] = x + (long long)row[i] * ldx + col[i];
  }
  load_groups<T, A>(src, have, span, raw);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    float v[UNIT];
    unpack<T>(raw[i], v);
#pragma unroll
    for (int p = 0; p < BF16_PARTS<T>; ++p) {
      Raw<__nv_bfloat16> part;
      __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(part.q);
#pragma unroll
      for (int j = 0; j < UNIT; ++j) {
        const uint32_t bits = __float_as_uint(v[j]);
        const bool finite = abs_bits(v[j]) < kInfBits;
        const uint32_t top = abs_bits(v[j]) > kInfBits ? 0x7fc00000u : bits & 0xffff0000u;  // NaN stays NaN without its low bits
        e[j] = __ushort_as_bfloat16(uint16_t(top >> 16));
        v[j] = finite ? add_exact(v[j], __uint_as_float(top ^ 0x80000000u)) : 0.f;
      }
      store_raw<__nv_bfloat16, Access::kPieces16>(out + p * part_step + (long long)row[i] * ldo + col[i], col[i], have[i], part);
    }
  }
}

// ------------------------------------------------------------------------------ RMSNorm
// h = x + residual (rounded to bf16, as the next residual addition reads it), y = h * rstd * w, y in
// 8 bits.  Each thread holds 8 values (16 bytes) of a row per step; the 16 lanes whose values make up a
// block scale it with four shuffles.
__device__ __forceinline__ void unpack8(uint4 q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
}
// v = x + r rounded to bf16; returns it packed
__device__ __forceinline__ uint4 add_rounded(uint4 x, uint4 r, float (&v)[8]) {
  float a[8], b[8];
  unpack8(x, a);
  unpack8(r, b);
  const uint4 h = make_uint4(pack_bf16x2(a[0] + b[0], a[1] + b[1]), pack_bf16x2(a[2] + b[2], a[3] + b[3]), pack_bf16x2(a[4] + b[4], a[5] + b[5]),
                             pack_bf16x2(a[6] + b[6], a[7] + b[7]));
  unpack8(h, v);
  return h;
}

struct NormArgs {
  const uint4 *x, *res, *w;
  uint4* h;
  float* rstd;
  uint8_t *data, *scale;
  long long ldq, lds, rows;
  int dim8;
  double inv_dim, eps;
};

// A value next to the middle between two e4m3 values goes to the wrong one when its fp32 error is larger than its
// distance, and is off by a whole step then.  So the sum of squares is compensated, the statistic (ss / dim + eps)^-1/2
// carried as two floats (one Newton step in 64 bits from the fp32 root), and the product rounded to odd: the last bit
// says that something was cut off, and the rounding to e4m3 is that of the exact product.
//
// The sum starts from a power of two B above all it will hold, so it stays in [B, 2B) and what an addition cuts off its
// square is exact: square - (new sum - old sum).  Those rests add up beside it.  (Kahan's sum rounds the next square
// together with the correction: errors of 1e-9, enough to move one value in 10^8.)
template <int N>
__device__ __forceinline__ double square_sum(const float (&v)[N][8]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = larger_magnitude(top, v[i][j]);
  // |v| < 2^(e + 1): each chain, of even or of odd columns, adds N * 4 squares below 2^(2 e + 2), less than its base 2^(2 e + 7)
  static_assert(N * 4 * 4 < 128, "a chain of squares must stay below its base");
  const int e = int(abs_bits(top) >> 23) - 127;
  if (e < -50 || e > 58) {  // far from everyday values: in 64 bits
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fma(double(v[i][j]), double(v[i][j]), sum);
    return sum;
  }
  const float base = __uint_as_float(uint32_t(2 * e + 7 + 127) << 23);
  uint64_t sum = pair_of(base, base), rest = pair_of(0.f, 0.f);  // of even and of odd columns
  const uint64_t minus_one = pair_of(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const uint64_t x = pair_of(v[i][j], v[i][j + 1]);
      const uint64_t t = fma2(x, x, sum);
      const uint64_t cut = fma2(x, x, fma2(t, minus_one, sum));
      rest = fma2(cut, pair_of(1.f, 1.f), rest);
      sum = t;
    }
  const float2 s = halves(sum), r = halves(rest);
  return (double(s.x - base) + double(s.y - base)) + double(r.x + r.y);
}
struct InverseRms {
  float hi, lo;
};
__device__ __forceinline__ InverseRms inverse_rms(double ss, const NormArgs& p) {
  const double m = fma(ss, p.inv_dim, p.eps);
  const double r0 = double(rsqrtf(float(m)));
  const double r = fma(0.5 * r0, fma(-m * r0, r0, 1.0), r0);
  // rows whose statistic fp32 cannot hold take the fp32 root: 0 for infinity, NaN for NaN
  const float hi = isfinite(r) ? float(r) : float(r0);
  return {hi, isfinite(r) ? float(r - double(hi)) : 0.f};
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 8 normalised values of column group c (zeros past the row) to 8 bits; all 32 lanes of the warp call this
__device__ __forceinline__ void store_normalised(const NormArgs& p, long long row, int c, const float (&v)[8], uint4 gain, InverseRms rs) {
  float g[8], y[8];
  unpack8(gain, g);
  const uint64_t hi = pair_of(rs.hi, rs.hi), lo = pair_of(rs.lo, rs.lo);
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint64_t t = mul2(pair_of(v[j], v[j + 1]), pair_of(g[j], g[j + 1]));  // exact: both have 8 significant bits
    float2 q;
    if (rs.lo != 0.f) {  // hi + lo has more than 24 bits, its product with any t but 0 as well
      q = halves(fma2_towards_zero(t, hi, mul2(t, lo)));
      q.x = __uint_as_float(__float_as_uint(q.x) | 1u);
      q.y = __uint_as_float(__float_as_uint(q.y) | 1u);
    } else {
      const float2 s = halves(t);
      q.x = __fmul_rz(s.x, rs.hi);
      q.y = __fmul_rz(s.y, rs.hi);
      if (fmaf(s.x, rs.hi, -q.x) != 0.f) q.x = __uint_as_float(__float_as_uint(q.x) | 1u);
      if (fmaf(s.y, rs.hi, -q.y) != 0.f) q.y = __uint_as_float(__float_as_uint(q.y) | 1u);
    }
    y[j] = q.x, y[j + 1] = q.y;
    top = larger_magnitude(top, larger_magnitude(q.x, q.y));
  }
  uint32_t q[2];
  const uint32_t byte = quantize_block<8, 16>(y, abs_bits(top), q);
  if (c < p.dim8) {
    *reinterpret_cast<uint2*>(p.data + row * p.ldq + c * 8) = make_uint2(q[0], q[1]);
    if ((c & 15) == 0) p.scale[row * p.lds + c / 16] = uint8_t(byte);
  }
}

// Rows of up to 1536 values: a warp per row.  15465 x 1304: 23 us, a block per row 33; 8192 x 2048 with residual 32 and 27,
// so wider rows take a block.
template <int VPT, bool RESIDUAL>
__global__ void __launch_bounds__(256) rmsnorm_fp8_warp_kernel(const __grid_constant__ NormArgs p) {
  await_previous();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  float v[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * 32;
    if (c < p.dim8) {
      const long long at = row * p.dim8 + c;
      if (RESIDUAL) p.h[at] = add_rounded(p.x[at], p.res[at], v[i]);
      else unpack8(p.x[at], v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  const InverseRms rs = inverse_rms(warp_sum(square_sum(v)), p);
  if (lane == 0) p.rstd[row] = rs.hi;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * 32;
    if (i * 32 >= p.dim8) break;
    store_normalised(p, row, c, v[i], c < p.dim8 ? p.w[c] : make_uint4(0, 0, 0, 0), rs);
  }
}

// Wider rows: a block per row, as many blocks as fit an SM, which walk the rows; the next row's loads are issued before
// the current one is reduced.  4096 x 4096 with residual (117 MB): 23 us, 78 % of the copy bandwidth, and 18 without (84 MB,
// 72 %).  What bounds it is instructions as much as bytes: one fp32 operation at a time instead of pairs 26 us; two or
// four blocks per SM (four spill registers) 24 and 29; 128 or 512 threads per row, or a ring of rows in shared memory
// filled by bulk copies, 3 us more when that was 24.
template <int VPT>
constexpr int NORM_BLOCKS = VPT == 1 ? 4 : VPT == 2 ? 3 : 2;  // of NORM_THREADS, per SM
template <int VPT, bool RESIDUAL, bool FULL>  // FULL: NORM_THREADS threads, otherwise fewer
__global__ void __launch_bounds__(NORM_THREADS, NORM_BLOCKS<VPT>) rmsnorm_fp8_block_kernel(const __grid_constant__ NormArgs p) {
  __shared__ double red[2][NORM_THREADS / 32];
  await_previous();
  const int t = threadIdx.x, threads = FULL ? NORM_THREADS : int(blockDim.x);
  uint4 nx[VPT], nr[VPT], gain[VPT];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * threads;
      if (row < p.rows && c < p.dim8) {
        nx[i] = p.x[row * p.dim8 + c];
        if (RESIDUAL) nr[i] = p.res[row * p.dim8 + c];
      }
    }
  };
  fetch(blockIdx.x);
#pragma unroll
  for (int i = 0; i < VPT; ++i) gain[i] = t + i * threads < p.dim8 ? p.w[t + i * threads] : make_uint4(0, 0, 0, 0);
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    float v[VPT][8];
  #pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * threads;
      if (c < p.dim8) {
        if (RESIDUAL) p.h[row * p.dim8 + c] = add_rounded(nx[i], nr[i], v[i]);
        else unpack8(nx[i], v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      }
    }
    fetch(row + gridDim.x);
    double sum = warp_sum(square_sum(v));
    if ((t & 31) == 0) red[turn][t >> 5] = sum;  // the other half may still be read by warps of the last round
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < NORM_THREADS / 32; ++i)
      if (i < threads / 32) sum += red[turn][i];
    const InverseRms rs = inverse_rms(sum, p);
    if (t == 0) p.rstd[row] = rs.hi;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * threads;
      if ((c & ~31) >= p.dim8) break;  // the whole warp is past the row
      store_normalised(p, row, c, v[i], gain[i], rs);
    }
  }
}

bool aligned(const void* p, long long pitch_bytes, int to) { return (reinterpret_cast<uintptr_t>(p) | uintptr_t(pitch_bytes)) % to == 0; }
Access access_for(const void* p, long long pitch_bytes, bool packed, int cols) {
  return packed && cols % UNIT == 0 && aligned(p, pitch_bytes, 32) ? Access::kPieces32 : aligned(p, pitch_bytes, 16) ? Access::kPieces16 : Access::kShifted;
}
#define ELFB_ACCESS(KERNEL, T, A) \
  (A == Access::kPieces32 ? KERNEL<T, Access::kPieces32> : A == Access::kPieces16 ? KERNEL<T, Access::kPieces16> : KERNEL<T, Access::kShifted>)
template <typename T>
Span span_of(const void* x, long long ldx, long long rows, int cols) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(x);
  return {at, at + uintptr_t((rows - 1) * ldx + cols) * sizeof(T)};
}

// rows per launch, so that a launch's units fit 31 bits
long long rows_per_launch(uint32_t units_per_row) { return std::max(1ll, (1ll << 30) / units_per_row); }

template <typename T>
cudaError_t quantize_rows_as(const void* x, long long ldx, uint8_t* data, long long ldq, uint8_t* scale, long long lds, long long rows, int cols,
                             cudaStream_t stream) {
  const bool packed = aligned(data, ldq, 16);
  const Access how = access_for(x, ldx * sizeof(T), packed, cols);
  const Span span = span_of<T>(x, ldx, rows, cols);
  const uint32_t upr = uint32_t((cols + BLOCK - 1) / BLOCK) * (BLOCK / UNIT);
  const long long step = rows_per_launch(upr);
  for (long long r = 0; r < rows; r += step) {
    const uint32_t total = uint32_t(std::min(step, rows - r)) * upr;
    auto* kern = ELFB_ACCESS(quantize_rows_kernel, T, how);
    if (cudaError_t e = launch_overlapped(kern, (total + UNITS * THREADS - 1) / (UNITS * THREADS), THREADS, 0, 0, stream, static_cast<const T*>(x) + r * ldx, ldx,
                                          data + r * ldq, ldq, scale + r * lds, lds, total, upr, cols, span, packed);
        e != cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t quantize_tiles_as(const void* x, long long ldx, uint8_t* data, long long ldq, uint8_t* scale, long long lds, long long rows, int cols,
                              cudaStream_t stream) {
  const bool packed = aligned(data, ldq, 16);
  const Access how = access_for(x, ldx * sizeof(T), packed, cols);
  const Span span = span_of<T>(x, ldx, rows, cols);
  constexpr long long kGridY = 65535;
  const long long tiles = (rows + BLOCK - 1) / BLOCK;
  for (long long t = 0; t < tiles; t += kGridY) {
    const long long r = t * BLOCK;
    const dim3 grid((cols + BLOCK - 1) / BLOCK, unsigned(std::min(kGridY, tiles - t)));
    auto* kern = ELFB_ACCESS(quantize_tiles_kernel, T, how);
    if (cudaError_t e = launch_overlapped(kern, grid, TILE_THREADS, 0, 0, stream, static_cast<const T*>(x) + r * ldx, ldx, data + r * ldq, ldq, scale + t * lds, lds,
                                          rows - r, cols, span, packed);
        e != cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t dequantize_as(const uint8_t* data, long long ldq, const uint8_t* scale, long long lds, int row_shift, void* y, long long ldy, long long rows,
                          int cols, cudaStream_t stream) {
  const bool packed = aligned(data, ldq, 16);
  const Access how = access_for(y, ldy * sizeof(T), packed, cols);
  const uint32_t upr = uint32_t((cols + UNIT - 1) / UNIT);
  const long long step = rows_per_launch(upr);
  for (long long r = 0; r < rows; r += step) {
    const uint32_t total = uint32_t(std::min(step, rows - r)) * upr;
    auto* kern = ELFB_ACCESS(dequantize_kernel, T, how);
    if (cudaError_t e = launch_overlapped(kern, (total + UNITS * THREADS - 1) / (UNITS * THREADS), THREADS, 0, 0, stream, data, ldq, scale, lds, row_shift,
                                          static_cast<T*>(y), ldy, total, upr, r, cols, packed);
        e != cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t bf16_parts_as(const void* x, long long ldx, void* out, long long ldo, long long part_step, long long rows, int cols, cudaStream_t stream) {
  const Span span = span_of<T>(x, ldx, rows, cols);
  const uint32_t upr = uint32_t((cols + UNIT - 1) / UNIT);
  const long long step = rows_per_launch(upr);
  auto* kern = aligned(x, ldx * sizeof(T), 16) ? bf16_parts_kernel<T, Access::kPieces16> : bf16_parts_kernel<T, Access::kShifted>;
  for (long long r = 0; r < rows; r += step) {
    const uint32_t total = uint32_t(std::min(step, rows - r)) * upr;
    if (cudaError_t e = launch_overlapped(kern, (total + UNITS * THREADS - 1) / (UNITS * THREADS), THREADS, 0, 0, stream, static_cast<const T*>(x) + r * ldx, ldx,
                                          static_cast<__nv_bfloat16*>(out) + r * ldo, ldo, part_step, total, upr, cols, span);
        e != cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

template <int VPT>
cudaError_t rmsnorm_warps(const NormArgs& p, cudaStream_t stream) {
  auto* kern = p.res ? rmsnorm_fp8_warp_kernel<VPT, true> : rmsnorm_fp8_warp_kernel<VPT, false>;
  constexpr long long kRows = 1ll << 33;  // of one launch: its blocks fit the grid
  for (long long r = 0; r < p.rows; r += kRows) {
    NormArgs q = p;
    q.rows = std::min(kRows, p.rows - r);
    q.x += r * p.dim8, q.rstd += r, q.data += r * p.ldq, q.scale += r * p.lds;
    if (p.res) q.res += r * p.dim8, q.h += r * p.dim8;
    if (cudaError_t e = launch_overlapped(kern, unsigned((q.rows + 7) / 8), 256, 0, 0, stream, q); e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int VPT>
cudaError_t rmsnorm_blocks(const NormArgs& p, int num_sms, cudaStream_t stream) {
  // whole warps, as many as the row fills: 1000 x 5120 on 160 threads instead of 256
  const int threads = ((p.dim8 + VPT - 1) / VPT + 31) / 32 * 32, per_sm = NORM_BLOCKS<VPT> * NORM_THREADS / threads;
  auto* kern = threads == NORM_THREADS ? (p.res ? rmsnorm_fp8_block_kernel<VPT, true, true> : rmsnorm_fp8_block_kernel<VPT, false, true>)
                                       : (p.res ? rmsnorm_fp8_block_kernel<VPT, true, false> : rmsnorm_fp8_block_kernel<VPT, false, false>);
  return launch_overlapped(kern, unsigned(std::min(p.rows, (long long)per_sm * num_sms)), unsigned(threads), 0, 0, stream, p);
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

cudaError_t fp8_repack(const void* src, long long ld_src, void* dst, long long ld_dst, long long rows, int row_bytes, cudaStream_t stream) {
  if (rows <= 0 || row_bytes <= 0) return cudaSuccess;
  const uint8_t* from = static_cast<const uint8_t*>(src);
  uint8_t* to = static_cast<uint8_t*>(dst);
  const Span span = span_of<uint8_t>(src, ld_src, rows, row_bytes);
  const uint32_t upr = uint32_t((row_bytes + UNIT - 1) / UNIT);
  const long long step = rows_per_launch(upr);
  constexpr Access P = Access::kPieces16, S = Access::kShifted;
  const bool from_pieces = aligned(src, ld_src, 16), to_pieces = aligned(dst, ld_dst, 16);
  auto* kern = from_pieces ? (to_pieces ? repack_kernel<P, P> : repack_kernel<P, S>) : to_pieces ? repack_kernel<S, P> : repack_kernel<S, S>;
  for (long long r = 0; r < rows; r += step) {
    const uint32_t total = uint32_t(std::min(step, rows - r)) * upr;
    if (cudaError_t e = launch_overlapped(kern, (total + 2 * UNITS * THREADS - 1) / (2 * UNITS * THREADS), THREADS, 0, 0, stream, from + r * ld_src, ld_src,
                                          to + r * ld_dst, ld_dst, total, upr, row_bytes, span);
        e != cudaSuccess)
      return e;
  }
  return cudaSuccess;
}

int bf16_parts(Elem type) { return type == Elem::kBf16 ? 1 : type == Elem::kF16 ? BF16_PARTS<__half> : BF16_PARTS<float>; }
cudaError_t split_into_bf16_parts(const void* x, Elem type, long long ldx, void* out, long long ldo, long long part_step, long long rows, int cols,
                                  cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  if (type == Elem::kBf16) return cudaErrorInvalidValue;
  if (type == Elem::kF16) return bf16_parts_as<__half>(x, ldx, out, ldo, part_step, rows, cols, stream);
  return bf16_parts_as<float>(x, ldx, out, ldo, part_step, rows, cols, stream);
}

cudaError_t fp8_rmsnorm(const void* x, const void* residual, const void* w, void* h, float* rstd, uint8_t* data, long long ldq, uint8_t* scale,
                        long long lds, long long rows, int dim, double eps, int num_sms, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  if (dim <= 0 || dim % 8 || dim > 8192) return cudaErrorInvalidValue;
  const NormArgs p{static_cast<const uint4*>(x), static_cast<const uint4*>(residual), static_cast<const uint4*>(w), static_cast<uint4*>(h), rstd, data, scale,
                   ldq, lds, rows, dim / 8, 1.0 / double(dim), eps};
  if (dim <= 256) return rmsnorm_warps<1>(p, stream);
  if (dim <= 512) return rmsnorm_warps<2>(p, stream);
  if (dim <= 1024) return rmsnorm_warps<4>(p, stream);
  if (dim <= 1536) return rmsnorm_warps<6>(p, stream);
  if (dim <= 2048) return rmsnorm_blocks<1>(p, num_sms, stream);
  if (dim <= 4096) return rmsnorm_blocks<2>(p, num_sms, stream);
  return rmsnorm_blocks<4>(p, num_sms, stream);
}

}  // namespace elfb
