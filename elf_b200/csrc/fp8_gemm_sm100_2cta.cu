// CTA-pair kernel of the block-scaled products: two CTAs on neighbouring SMs share a 256 x 256 tile
// through tcgen05.mma.cta_group::2.
//
// Why pairs: a 128 x 256 tile on one CTA fetches 48 KiB for 512 cycles of 8-bit MMA, 25 TB/s over the chip,
// which is more than L2 delivers; the pair fetches 32 KiB per CTA in the same time (each its own 128 rows
// of A and half of B).  4096 x 4096 x 14336: 181 us; a kernel of single CTAs with 128 x 256 tiles took 249.
// What bounds it: the tensor pipe, 76 % busy there and 83 % in the gradient's form (4096 x 4096 x 28672, 348 us); under a
// lasting load the chip's power, which takes the clock from 1.9 to 1.1 - 1.4 GHz.
//
// Roles per CTA as in fp8_gemm_sm100.cu.  The even CTA's MMA thread issues for both.  Barriers, each of a slot of two
// stages:
//   full[s]      even CTA: armed with both CTAs' bytes, both CTAs' copies complete on it, and both CTAs' scale warps
//                arrive when their words lie in shared memory
//   empty[s]     one per CTA, committed to both at once: a commit costs about as much as a step of MMA (two single
//                commits per stage instead: 218 us against 200 in the loop alone)
//   acc_full[a]  one per CTA, committed to both
//   acc_free     even CTA: the epilogue warps of both arrive once the columns the two accumulators share
//                have been read (16 arrivals per unit)
//
// The tiles of a last, partly filled wave are split along K into units on different pairs.  Every unit but
// the last to finish leaves its fp32 sums in a workspace; the last one adds all parts in their order, so
// results do not depend on who that is.  Nobody waits for another unit.
#include "fp8_gemm.cuh"

namespace elfb {
namespace fp8 {
namespace pair {

constexpr int BN = 256;
constexpr int STAGES = 6;
constexpr int STAGE_BYTES = 2 * BOX_BYTES;  // per CTA: 128 rows of A, 128 rows of B
constexpr int SLOTS = STAGES / 2;           // two consecutive stages are filled, waited for and freed together
constexpr int EPI_WARPS = 8;     // two per quarter of the TMEM lanes, each with one half of the columns
constexpr int EPI_THREADS = EPI_WARPS * 32;
constexpr int NUM_THREADS = 96 + EPI_THREADS;
constexpr int SF_BYTES = 3 * 512;           // scale words of a slot: 128 rows of A, 256 columns of B
// Tile rows (of 256) that are swept together before moving to the next columns: B is read from DRAM once for each group.
// In groups of 2, 4, 8 and 16 (us): 4096 x 4096 x 14336 180, 180, 178, 178; gated forward 4096 x 28672 x 4096 397, 375, 362,
// 355; its backward 266, 266, 262, 260; input gradient 4096 x 4096 x 28672 348, 347, 342, 339.
constexpr int GROUP_M = 4;
constexpr int ACC1 = 224;   // first column of the second accumulator: shares 32 with the first
constexpr int EXCHANGE_BYTES = 3 * 2 * BM * 4;  // block maxima that the two halves of a row tell each other (gated forms)
constexpr size_t SMEM_BYTES = size_t(STAGES) * STAGE_BYTES + SLOTS * SF_BYTES + EXCHANGE_BYTES + 1024 /*align slack*/ + 256 /*barriers*/;
constexpr int PART_FLOATS = BM * BN;  // one CTA's half of a tile in the workspace

struct Schedule {
  int tiles_m, tiles_n, full_tiles, ksplit, total_units;
};

struct Unit {
  int m0, n0;    // first row of this pair's tile; first column (gated: of gate)
  int kb0, kb1;  // blocks of the reduction
  int part;      // index among the parts of its tile
  int rest;      // index of its tile among the split tiles, -1 for a whole one
};

__device__ __forceinline__ Unit unit_at(int u, const Schedule& s, int k_blocks, int width) {
  Unit r;
  int tile = u;
  r.kb0 = 0, r.kb1 = k_blocks, r.part = 0, r.rest = -1;
  if (u >= s.full_tiles) {
    const int rem = (s.total_units - s.full_tiles) / s.ksplit;  // parts of one tile are `rem` units apart: other pairs
    const int v = u - s.full_tiles;
    r.rest = v % rem;
    r.part = v / rem;
    tile = s.full_tiles + r.rest;
    if (s.ksplit == 1) {
      r.rest = -1;
    } else {  // whole groups of four blocks, which share scale words
      const int groups = (k_blocks + 3) / 4;
      r.kb0 = 4 * int((long long)groups * r.part / s.ksplit);
      r.kb1 = min(k_blocks, 4 * int((long long)groups * (r.part + 1) / s.ksplit));
    }
  }
  const int per_group = GROUP_M * s.tiles_n;
  const int group = tile / per_group;
  const int first_m = group * GROUP_M;
  const int rows = min(GROUP_M, s.tiles_m - first_m);
  const int in_group = tile - group * per_group;
  r.m0 = (first_m + in_group % rows) * 2 * BM;
  r.n0 = (in_group / rows) * width;
  return r;
}

__device__ __forceinline__ void umma_ss_mxf8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
      "}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

// Arrival on a barrier that may live in the other CTA, after what this warp has written to this CTA's shared memory (each
// lane's proxy fence and a __syncwarp come before).  The release covers shared memory only: one that also waits for the
// warp's global accesses takes longer than the MMAs of a slot (4096 x 4096 x 14336: 287 us against 182).  The MMA thread
// tests the barrier without ordering anything and then acquires, likewise shared memory only (184 us with an acquiring test).
__device__ __forceinline__ void mbar_arrive_cluster_smem(uint32_t cluster_addr) {
  asm volatile("fence.release.sync_restrict::shared::cta.cluster;" ::: "memory");
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Four accumulating MMAs, a block of K apart by A_STEP and B_STEP in the descriptors' address units; returns whether the
// barrier's phase had completed when the test, issued before them, came up (the caller acquires what it stands for).
template <int A_STEP, int B_STEP>
__device__ __forceinline__ bool umma_x4_then_ready(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t sfa, uint32_t bar, uint32_t parity) {
  uint32_t ready;
  asm volatile(
      "{\n\t"
      ".reg .pred p, t;\n\t"
      ".reg .b64 a, b;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 t, [%7], %8;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%1], %2, %3, %4, [%5], [%6], p;\n\t"
      "add.s64 a, %2, %9;\n\t"
      "add.s64 b, %3, %10;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%1], a, b, %4, [%5], [%6], p;\n\t"
      "add.s64 a, a, %9;\n\t"
      "add.s64 b, b, %10;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%1], a, b, %4, [%5], [%6], p;\n\t"
      "add.s64 a, a, %9;\n\t"
      "add.s64 b, b, %10;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%1], a, b, %4, [%5], [%6], p;\n\t"
      "selp.u32 %0, 1, 0, t;\n\t"
      "}\n"
      : "=r"(ready)
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(sfa), "r"(sfa + 4), "r"(bar), "r"(parity), "n"(A_STEP), "n"(B_STEP)
      : "memory");
  return ready != 0;
}
constexpr float kLog2e = 1.4426950408889634f;
// sigmoid of two values given times -log2(e)
__device__ __forceinline__ uint64_t sigmoid2(uint64_t x) {
  const float2 a = halves(x);
  const float2 b = halves(fma2(pair_of(exp2f(a.x), exp2f(a.y)), pair_of(1.f, 1.f), pair_of(1.f, 1.f)));
  return pair_of(__fdividef(1.f, b.x), __fdividef(1.f, b.y));
}
// One tile of the gated form: columns 0..127 of the accumulator are gate, 128..255 up.  A thread takes 64 columns
// of gate and the same of up of one row into registers and gives the accumulator back at once; the maxima of the
// three blocks (gate, up, activation) are exchanged with the thread that has the row's other half.
// 4096 x 28672 x 4096: 375 to 383 us of 285 at the 8-bit peak (393 before its arithmetic went by fp32 pairs), tensor pipe 74 %
// busy: 32 blocks of K are about as long as this epilogue, and the last of 25 waves is a quarter full.
template <typename Release>
__device__ __forceinline__ void gated_tile(uint32_t taddr, int row, int half, int f0, int f, const Params& p, uint32_t* exchange, Release&& release) {
  uint32_t raw[4][32];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    tmem_ld_32x32b_x32(taddr + half * 64 + c * 32, raw[c]);
    tmem_ld_32x32b_x32(taddr + 128 + half * 64 + c * 32, raw[2 + c]);
  }
  tmem_ld_wait();
  release();
  float g[64], u[64];
#pragma unroll
  for (int j = 0; j < 64; ++j) g[j] = __uint_as_float(raw[j / 32][j % 32]), u[j] = __uint_as_float(raw[2 + j / 32][j % 32]);
  const bool live = row < p.M;
  const int col = f0 + half * 64;
  auto block_byte = [&](int which, uint32_t top) {  // exponent byte of the row's block, from both halves
    exchange[(which * 2 + half) * BM] = top;
    named_barrier_sync(1, EPI_THREADS);
    return block_exponent(max(top, exchange[(which * 2 + (half ^ 1)) * BM]));
  };
  // blocks without infinities and NaN, practically all, take the branches that do not look for them
  auto any = [](bool odd) { return __any_sync(0xffffffffu, odd) != 0; };
  if (p.gu != nullptr) {
    uint32_t top_g = magnitude<64, false>(g), top_u = magnitude<64, false>(u);
    const bool odd = any(top_g >= kInfBits || top_u >= kInfBits);
    if (odd) top_g = magnitude<64, true>(g), top_u = magnitude<64, true>(u);
    exchange[half * BM] = top_g;
    const uint32_t byte_u = block_byte(1, top_u);
    const uint32_t byte_g = block_exponent(max(top_g, exchange[(half ^ 1) * BM]));
    if (live) {
      uint8_t* dst = p.gu + (long long)row * p.ld_gu + col;
      const float inv_g = inverse_exponent_value(byte_g), inv_u = inverse_exponent_value(byte_u);
      if (odd) {
        scale_and_store<64, true>(g, inv_g, dst);
        scale_and_store<64, true>(u, inv_u, dst + f);
      } else {
        scale_and_store<64, false>(g, inv_g, dst);
        scale_and_store<64, false>(u, inv_u, dst + f);
      }
      if (half == 0) {
        uint8_t* s = p.gu_scale + (long long)row * p.ld_gu_scale;
        s[f0 / 128] = uint8_t(byte_g);
        s[(f + f0) / 128] = uint8_t(byte_u);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 64; j += 2) {
    const uint64_t g2 = pair_of(g[j], g[j + 1]);
    const float2 a = halves(mul2(mul2(g2, sigmoid2(mul2(g2, pair_of(-kLog2e, -kLog2e)))), pair_of(u[j], u[j + 1])));
    g[j] = a.x, g[j + 1] = a.y;
  }
  uint32_t top = magnitude<64, false>(g);
  const bool odd = any(top >= kInfBits);
  if (odd) top = magnitude<64, true>(g);
  const uint32_t byte = block_byte(2, top);
  if (live) {
    uint8_t* dst = p.act + (long long)row * p.ld_act + col;
    if (odd) scale_and_store<64, true>(g, inverse_exponent_value(byte), dst);
    else scale_and_store<64, false>(g, inverse_exponent_value(byte), dst);
    if (half == 0) p.act_scale[(long long)row * p.ld_act_scale + f0 / 128] = uint8_t(byte);
  }
}

// One tile of the gated form's backward: the accumulator holds the gradient d of the activation, the thread one row
// of one block of 128 columns.  gate and up come from their checkpoint.
//   dgate = d up s (1 + gate (1 - s)),  dup = d gate s,  s = sigmoid(gate)
// are formed twice, once for the maxima of their blocks and once to be scaled: a thread that has a row's block alone would
// hold 256 values.  (Two threads to a block, as above, would hold 128 each: not built.)  d stays in TMEM but for the 32 columns shared with the other accumulator, which half of the threads
// hold.  The checkpoint is read and the result written 32 bytes at a time, whole sectors of a row that is one
// thread's own: 16-byte accesses cost 40 us more.
//
// 4096 x 14336 x 4096: 264 to 268 us (180 without this epilogue, 142 at the 8-bit peak); the epilogue of a tile outlasts the
// next tile's MMAs.  Before its arithmetic went by pairs it took 283: arithmetic alone beside the MMAs 243, loads and
// stores with next to no arithmetic 273, one sweep 250.  Neither 16 epilogue warps (289) nor fetching the next tile's
// checkpoint into L2 (291) helped.
//
// With t = d s and the scales sg, su of gate and up taken out of the sums (powers of two: exact),
//   dup = sg (t gate_q),  dgate = su (up_q (t + t gate_q sg (1 - s))).
struct GateScales {
  float sg;       // gate = gate_q * sg
  float log2e;    // -log2(e) * sg
};
// dup / sg and dgate / su for 16 columns
__device__ __forceinline__ void gated_grad(const uint32_t* d, const uint32_t* gq, const uint32_t* uq, GateScales c, float (&dg)[16], float (&du)[16]) {
  const uint64_t sg = pair_of(c.sg, c.sg), minus_sg = pair_of(-c.sg, -c.sg), log2e = pair_of(c.log2e, c.log2e);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 g2 = from_e4m3x2((gq[j / 2] >> (16 * (j & 1))) & 0xffffu), u2 = from_e4m3x2((uq[j / 2] >> (16 * (j & 1))) & 0xffffu);
    const uint64_t g = pair_of(g2.x, g2.y), sig = sigmoid2(mul2(g, log2e));
    const uint64_t t = mul2(pair_of(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1])), sig), tg = mul2(t, g);
    const float2 a = halves(mul2(pair_of(u2.x, u2.y), fma2(tg, fma2(sig, minus_sg, sg), t))), b = halves(tg);
    dg[2 * j] = a.x, dg[2 * j + 1] = a.y;
    du[2 * j] = b.x, du[2 * j + 1] = b.y;
  }
}
template <typename Release>
__device__ __forceinline__ void gated_backward_tile(uint32_t taddr, int acc, int row, int half, int n0, int f, const Params& p, Release&& release) {
  taddr += half * 128;
  // chunks of 32 columns: of accumulator 0 the last is shared, of accumulator 1 the first
  const bool shares = half != acc;
  const int held_chunk = acc == 0 ? 3 : 0, from = shares && acc == 1 ? 1 : 0, to = shares && acc == 0 ? 3 : 4;
  uint32_t held[32];
  if (shares) {
    tmem_ld_32x32b_x32(taddr + held_chunk * 32, held);
    tmem_ld_wait();
  }
  release();
  const int col = n0 + half * 128;
  const bool live = row < p.M && col < f;  // (loads from TMEM are for the whole warp)
  const long long r = live ? row : 0;
  const int c0 = live ? col : 0;
  const uint8_t* gate = p.gu + r * p.ld_gu + c0;
  const uint8_t* scales = p.gu_scale + r * p.ld_gu_scale + c0 / 128;
  const float sg = exponent_value(scales[0]), su = exponent_value(scales[f / 128]);
  const GateScales gs{sg, -kLog2e * sg};
  uint8_t* dst = p.act + r * p.ld_act + c0;
  // calls handle(d, gate_q, up_q, chunk) for the row's four chunks, the checkpoint of the next one on its way
  auto sweep = [&](auto&& handle) {
    uint32_t g[8], u[8], next_g[8], next_u[8];
    load_32_bytes(gate + 32 * from, next_g);
    load_32_bytes(gate + f + 32 * from, next_u);
    if (shares) {
      load_32_bytes(gate + 32 * held_chunk, g);
      load_32_bytes(gate + f + 32 * held_chunk, u);
      handle(held, g, u, held_chunk);
    }
#pragma unroll 1
    for (int c = from; c < to; ++c) {
      uint32_t d[32];
      tmem_ld_32x32b_x32(taddr + c * 32, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = next_g[j], u[j] = next_u[j];
      if (c + 1 < to) {
        load_32_bytes(gate + 32 * (c + 1), next_g);
        load_32_bytes(gate + f + 32 * (c + 1), next_u);
      }
      tmem_ld_wait();
      handle(d, g, u, c);
    }
  };
  // Maxima of gradient / scale; multiplying by the scale keeps their order.  Infinite or NaN gradients, practically
  // never there, make the sweep run once more looking at finite ones only.
  uint32_t top_g = 0, top_u = 0;
  sweep([&](const uint32_t (&d)[32], const uint32_t (&g)[8], const uint32_t (&u)[8], int) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float dg[16], du[16];
      gated_grad(d + 16 * h, g + 4 * h, u + 4 * h, gs, dg, du);
      top_g = magnitude<16, false>(dg, top_g);
      top_u = magnitude<16, false>(du, top_u);
    }
  });
  auto odd_at = [&](uint32_t top, float scale) { return abs_bits(mul_exact(__uint_as_float(top), scale)) >= kInfBits; };
  const bool odd = __any_sync(0xffffffffu, odd_at(top_g, su) || odd_at(top_u, sg));
  if (odd) {
    top_g = top_u = 0;
    sweep([&](const uint32_t (&d)[32], const uint32_t (&g)[8], const uint32_t (&u)[8], int) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float dg[16], du[16];
        gated_grad(d + 16 * h, g + 4 * h, u + 4 * h, gs, dg, du);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          top_g = max(top_g, odd_at(__float_as_uint(dg[j]), su) ? 0u : abs_bits(dg[j]));
          top_u = max(top_u, odd_at(__float_as_uint(du[j]), sg) ? 0u : abs_bits(du[j]));
        }
      }
    });
  }
  const uint32_t byte_g = block_exponent(abs_bits(mul_exact(__uint_as_float(top_g), su))), byte_u = block_exponent(abs_bits(mul_exact(__uint_as_float(top_u), sg)));
  const float inv_g = inverse_exponent_value(byte_g), inv_u = inverse_exponent_value(byte_u);
  auto emit = [&](auto odd_tag) {
    constexpr bool ODD = decltype(odd_tag)::value;
    sweep([&](const uint32_t (&d)[32], const uint32_t (&g)[8], const uint32_t (&u)[8], int c) {
      uint32_t qg[8], qu[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float dg[16], du[16];
        gated_grad(d + 16 * h, g + 4 * h, u + 4 * h, gs, dg, du);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float2 a = halves(mul2(pair_of(dg[j], dg[j + 1]), pair_of(su, su))), b = halves(mul2(pair_of(du[j], du[j + 1]), pair_of(sg, sg)));
          dg[j] = a.x, dg[j + 1] = a.y;
          du[j] = b.x, du[j + 1] = b.y;
        }
        to_scaled_e4m3<16, ODD>(dg, inv_g, qg + 4 * h);
        to_scaled_e4m3<16, ODD>(du, inv_u, qu + 4 * h);
      }
      if (live) {
        store_32_bytes(dst + 32 * c, qg);
        store_32_bytes(dst + f + 32 * c, qu);
      }
    });
  };
  if (odd) emit(std::true_type());
  else emit(std::false_type());
  if (live) {
    uint8_t* s = p.act_scale + r * p.ld_act_scale + c0 / 128;
    s[0] = uint8_t(byte_g);
    s[f / 128] = uint8_t(byte_u);
  }
}

template <bool B_MN, Fp8Form FORM, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
fp8_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ Params p,
                     const __grid_constant__ Schedule sched, float* __restrict__ parts, unsigned int* __restrict__ parts_done) {
  constexpr bool GATED = FORM == Fp8Form::kGated;  // the tile's columns are 128 of gate and the same 128 of up
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_aligned = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t sf_base = smem_base + STAGES * STAGE_BYTES;
  uint32_t* exchange = reinterpret_cast<uint32_t*>(smem_aligned + size_t(STAGES) * STAGE_BYTES + SLOTS * SF_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_aligned + size_t(STAGES) * STAGE_BYTES + SLOTS * SF_BYTES + EXCHANGE_BYTES);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int slot) { return bar0 + 8u * slot; };
  auto empty_bar = [&](int slot) { return bar0 + 8u * (SLOTS + slot); };
  auto acc_full_bar = [&](int a) { return bar0 + 8u * (2 * SLOTS + a); };
  const uint32_t acc_free_bar = bar0 + 8u * (2 * SLOTS + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * SLOTS + 3);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile unsigned int* arrived = tmem_slot + 2;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();  // 0 = leader
  const bool leader = cta == 0;
  const int pair_id = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;
  const int f = GATED ? p.N / 2 : p.N;  // gated forms: width of the activation
  const int width = GATED ? 128 : BN;
  const int k_blocks = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(full_bar(s), 3);  // the leader's arrive.expect_tx and both scale warps
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(acc_free_bar, 2 * EPI_WARPS);
    for (int a = 0; a < 2; ++a) mbar_init(acc_full_bar(a), 1);
    fence_barrier_init();
    prefetch_tensormap(&tmap_a);
    prefetch_tensormap(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before anyone touches the peer's
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  await_previous();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = pair_id; u < sched.total_units && ok; u += num_pairs) {
        const Unit unit = unit_at(u, sched, k_blocks, width);
        const int m0 = unit.m0 + int(cta) * BM;
        // this CTA's 128 rows of B; gated: gate in the even CTA, up in the odd one.  Boxes behind the last row arrive as zeros.
        const int n0 = unit.n0 + int(cta) * (GATED ? f : 128);
        for (int kb2 = unit.kb0; kb2 < unit.kb1; kb2 += 2) {
          if (!mbar_wait(empty_bar(slot), phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const int blocks = min(2, unit.kb1 - kb2);
          const uint32_t bar = map_to_cta(full_bar(slot), 0);
          if (leader) mbar_arrive_expect_tx(full_bar(slot), blocks * 2 * STAGE_BYTES);
          for (int b = 0; b < blocks; ++b) {
            const uint32_t sa = smem_base + (2 * slot + b) * STAGE_BYTES, sb = sa + BOX_BYTES;
            const int k0 = (kb2 + b) * BK;
            tma_load_2d_pair(sa, &tmap_a, bar, k0, m0);
            if (B_MN) tma_load_2d_pair(sb, &tmap_b, bar, n0, k0);
            else tma_load_2d_pair(sb, &tmap_b, bar, k0, n0);
          }
          if (++slot == SLOTS) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader only)
    if (leader && lane == 0) {
      // A barrier test queues up behind the MMAs issued before it and its answer is late by then: one test per four MMAs
      // made the loop 730 cycles per block of K where the MMAs alone take 523 (512 at best).  So there is one test per
      // slot of eight, it is issued before the slot's last four and its answer read after them (`umma_x4_then_ready`);
      // descriptors are one addition each.
      constexpr uint32_t B_KSTEP = B_MN ? UMMA_K * 128 : UMMA_K;  // see fp8_gemm_sm100.cu; one 128-wide box per CTA
      constexpr uint32_t IDESC = make_idesc_mxf8(2 * BM, BN, 0u, B_MN ? 1u : 0u, 0), IDESC_STEP = (1u << 4) | (1u << 29);
      const uint64_t desc_a0 = make_smem_desc_sw128(smem_base, 0, 1024), desc_b0 = make_smem_desc_sw128(smem_base + BOX_BYTES, 0, 1024);
      const uint64_t desc_sf0 = make_smem_desc_rows16(sf_base);
      int slot = 0;
      uint32_t phase = 0, sf_count = 0;
      bool ok = true;
      int i = 0;  // units of this pair so far
      for (int u = pair_id; u < sched.total_units && ok; u += num_pairs, ++i) {
        const Unit unit = unit_at(u, sched, k_blocks, width);
        const int acc = i & 1;
        if (i > 0 && !mbar_wait<true>(acc_free_bar, uint32_t(i - 1) & 1u, abort_flag)) break;
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + acc * ACC1;
        bool ready = false;
        for (int kb = unit.kb0; kb < unit.kb1; kb += 2) {
          if (ready) {
            fence_acquire_cluster_smem();
          } else if (!mbar_wait<true>(full_bar(slot), phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const int next = slot + 1 == SLOTS ? 0 : slot + 1;
          const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
          const uint32_t sfa = tmem_base + SF_COL + (sf_count++ & 1) * 16;
          const uint64_t sf = desc_sf0 + uint32_t(slot * (SF_BYTES >> 4));
#pragma unroll
          for (int j = 0; j < 3; ++j) tmem_cp_32x128b_pair(sfa + 4 * j, sf + 32 * j);
          const uint64_t da = desc_a0 + uint32_t(slot * (2 * STAGE_BYTES >> 4)), db = desc_b0 + uint32_t(slot * (2 * STAGE_BYTES >> 4));
          const uint32_t idesc = IDESC + (kb & 3) * IDESC_STEP;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            umma_ss_mxf8_pair(tmem_d, da + ((k * UMMA_K) >> 4), db + ((k * B_KSTEP) >> 4), idesc, sfa, sfa + 4, (kb > unit.kb0 || k) ? 1u : 0u);
          ready = false;
          if (kb + 1 < unit.kb1)
            ready = umma_x4_then_ready<(UMMA_K >> 4), (B_KSTEP >> 4)>(tmem_d, da + (STAGE_BYTES >> 4), db + (STAGE_BYTES >> 4), idesc + IDESC_STEP, sfa,
                                                                      full_bar(next), next_phase) && kb + 2 < unit.kb1;
          umma_commit_both(empty_bar(slot));
          slot = next;
          phase = next_phase;
        }
        if (!ok) break;
        umma_commit_both(acc_full_bar(acc));
      }
    }
    __syncwarp();
  } else if (warp < 2 + EPI_WARPS) {
    // ------------------------------------------------------------------ epilogue (warps 2..9 of both CTAs)
    const int quarter = warp & 3;       // TMEM lanes [32*quarter, 32*quarter+32) belong to this warp
    const int half = (warp - 2) >> 2;   // plain forms: columns 128 * half onwards; gated: 64 of gate and of up
    const uint32_t free_bar = map_to_cta(acc_free_bar, 0);
    int i = 0;
    for (int u = pair_id; u < sched.total_units; u += num_pairs, ++i) {
      const Unit unit = unit_at(u, sched, k_blocks, width);
      const int acc = i & 1;
      const int row = unit.m0 + int(cta) * BM + quarter * 32 + lane;
      // all warps go on or none does: they meet at barriers below
      if (!named_barrier_all(1, EPI_THREADS, mbar_wait(acc_full_bar(acc), uint32_t(i >> 1) & 1u, abort_flag))) break;
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + acc * ACC1;
      auto release = [&] {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(free_bar);
      };
      if constexpr (GATED) {
        gated_tile(taddr, row, half, unit.n0, f, p, exchange + quarter * 32 + lane, release);
      } else if constexpr (FORM == Fp8Form::kGatedBackward) {
        gated_backward_tile(taddr, acc, row, half, unit.n0, f, p, release);
      } else {
        constexpr int CHUNKS = BN / 64;  // of 32 columns, for each half
        if (unit.rest < 0) {
#pragma unroll 1
          for (int j = 0; j < CHUNKS; ++j) {
            const int c = half * CHUNKS + (acc == 0 ? CHUNKS - 1 - j : j);  // the shared columns first
            uint32_t v[32];
            tmem_ld_32x32b_x32(taddr + c * 32, v);
            tmem_ld_wait();
            if (j == 0) release();
            const int col = unit.n0 + c * 32;
            if (col < p.N) store_chunk<T>(v, row, col, p);
          }
        } else {
          // A part of a split tile.  Workspace layout [part][CTA][chunk][4 columns][row]: a warp's access covers
          // 512 consecutive bytes.  The part that finds all others done keeps its own sums in TMEM.
          const int others = sched.ksplit - 1;
          unsigned int* done = parts_done + unit.rest * 2 + cta;
          float4* tile = reinterpret_cast<float4*>(parts) + ((long long)unit.rest * sched.ksplit * 2 + cta) * (PART_FLOATS / 4) + quarter * 32 + lane;
          constexpr long long PART_STEP = 2 * (PART_FLOATS / 4);
          if (threadIdx.x == 64) *arrived = *reinterpret_cast<volatile unsigned int*>(done);
          named_barrier_sync(1, EPI_THREADS);
          bool last = *arrived == unsigned(others);
          if (!last) {
            float4* mine = tile + unit.part * PART_STEP;
#pragma unroll 1
            for (int c = half * CHUNKS; c < (half + 1) * CHUNKS; ++c) {
              uint32_t v[32];
              tmem_ld_32x32b_x32(taddr + c * 32, v);
              tmem_ld_wait();
              if (unit.n0 + c * 32 < p.N && row < p.M) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                  mine[(c * 8 + q) * BM] = make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]), __uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3]));
              }
            }
            __threadfence();
            named_barrier_sync(1, EPI_THREADS);  // every thread has also read `arrived`
            if (threadIdx.x == 64) *arrived = atomicAdd(done, 1u);
            named_barrier_sync(1, EPI_THREADS);
            last = *arrived == unsigned(others);
          }
          if (last) {
            __threadfence();
#pragma unroll 1
            for (int c = half * CHUNKS; c < (half + 1) * CHUNKS; ++c) {
              uint32_t v[32];
              tmem_ld_32x32b_x32(taddr + c * 32, v);
              tmem_ld_wait();
              const int col = unit.n0 + c * 32;
              if (col >= p.N) continue;
              float s[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) s[j] = 0.f;
#pragma unroll 2
              for (int part = 0; part <= others; ++part) {  // in this order whoever is last
                if (part == unit.part) {
#pragma unroll
                  for (int j = 0; j < 32; ++j) s[j] += __uint_as_float(v[j]);
                } else {
                  float4 t[8];
#pragma unroll
                  for (int q = 0; q < 8; ++q) t[q] = row < p.M ? __ldcg(tile + part * PART_STEP + (c * 8 + q) * BM) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                  for (int q = 0; q < 8; ++q) s[4 * q] += t[q].x, s[4 * q + 1] += t[q].y, s[4 * q + 2] += t[q].z, s[4 * q + 3] += t[q].w;
                }
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(s[j]);
              store_chunk<T>(v, row, col, p);
            }
          }
          named_barrier_sync(1, EPI_THREADS);  // `arrived` may be written again
          release();
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ scale words (warp 10 of both CTAs)
    // A second producer of the ring: the words of a group of four blocks go to both slots of the group.  Those
    // of the next group are fetched from global memory before a slot is waited for.
    int u = pair_id, g = 0, slot = 0;
    uint32_t phase = 0;
    Unit unit{};
    RawScales ra, rb0, rb1;
    auto load = [&] {
      load_scales(p.sa, unit.m0 + int(cta) * BM, p.M, g, k_blocks, lane, ra);
      load_scales(p.sb, unit.n0, p.N, g, k_blocks, lane, rb0);
      load_scales(p.sb, unit.n0 + (GATED ? f : 128), p.N, g, k_blocks, lane, rb1);
    };
    auto begin = [&] {
      unit = unit_at(u, sched, k_blocks, width);
      g = unit.kb0 / 4;
    };
    if (u < sched.total_units) {
      begin();
      load();
    }
    bool ok = true;
    while (ok && u < sched.total_units) {
      uint32_t a[4], b0[4], b1[4];
      combine_scales(p.sa, g, k_blocks, ra, a);
      combine_scales(p.sb, g, k_blocks, rb0, b0);
      combine_scales(p.sb, g, k_blocks, rb1, b1);
      const int slots = unit.kb1 - 4 * g > 2 ? 2 : 1;
      if (4 * ++g >= unit.kb1) {
        u += num_pairs;
        if (u < sched.total_units) begin();
      }
      for (int i = 0; i < slots; ++i) {
        if (!mbar_wait(empty_bar(slot), phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        store_scale_words(sf_base + slot * SF_BYTES, lane, a);
        store_scale_words(sf_base + slot * SF_BYTES + 512, lane, b0);
        store_scale_words(sf_base + slot * SF_BYTES + 1024, lane, b1);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_smem(map_to_cta(full_bar(slot), 0));
        if (++slot == SLOTS) {
          slot = 0;
          phase ^= 1u;
        }
      }
      if (u < sched.total_units) load();
    }
  }

  // ------------------------------------------------------------------ common exit
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) {
      // let TMA copies that are still in flight land before the CTA's shared memory goes away
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) {
      }
      if (p.status != nullptr && atomicCAS(p.status, kOk, kErrBarrierTimeout) == kOk) {
        p.status[1] = 3000000 + blockIdx.x;
        p.status[2] = p.M;
        p.status[3] = p.N;
      }
    }
    __syncthreads();
  }
  cluster_sync_all();  // the peer may still be signalling barriers in this CTA's shared memory
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

Schedule make_schedule(int M, int N, int K, Fp8Form form, int num_pairs) {
  Schedule s;
  const int k_blocks = (K + BK - 1) / BK, groups = (k_blocks + 3) / 4;
  s.tiles_m = (M + 2 * BM - 1) / (2 * BM);
  s.tiles_n = (N + BN - 1) / BN;  // gated: N is a multiple of 256
  const long long tiles = (long long)s.tiles_m * s.tiles_n;
  const int rem = int(tiles % num_pairs);
  s.ksplit = 1;
  if (rem != 0 && form == Fp8Form::kPlain && k_blocks >= 48) {
    // Cycles of the last wave, fitted to rem = 16, 32, 34, 54, 64 tiles, K = 1024 .. 14336, split 1 to 8 ways: 600 per
    // block of K, and for split tiles 6000 to clear the counters and 200 for each part that is written and read back.
    // N = 4096, whole against split in two (us):  256 rows, K = 4096: 20.5 and 23.2; K = 14336: 45.1 and 35.5 (in four
    // 31.7); 2048 rows (54 of 128 tiles left over), K = 14336: 97 and 110; 4096 rows (34 left over): 188 and 184.
    // Shorter reductions, where a split would gain 3 us for a tile or two at best, stay whole: above 128 rows a row's
    // result does not depend on their number then (up to 128 another kernel splits K by a rule of its own).
    long long best = 600ll * k_blocks;
    for (int w = 2; w <= 8 && 2 * w <= groups; ++w) {
      const long long waves = ((long long)rem * w + num_pairs - 1) / num_pairs;
      const long long cost = waves * 2400 * ((groups + w - 1) / w) + 6000 + 200ll * rem * w;
      if (cost < best) {
        best = cost;
        s.ksplit = w;
      }
    }
  }
  s.full_tiles = int(s.ksplit == 1 ? tiles : tiles - rem);
  s.total_units = s.full_tiles + int(tiles - s.full_tiles) * s.ksplit;
  return s;
}

template <bool B_MN, Fp8Form FORM, typename T>
cudaError_t launch(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, const Schedule& s, void* workspace, int num_pairs, cudaStream_t stream) {
  auto kern = fp8_gemm_pair_kernel<B_MN, FORM, T>;
  // function attributes are per device: remember which devices of this process have been set up
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(SMEM_BYTES));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
  }
  const int rem = s.ksplit > 1 ? (s.total_units - s.full_tiles) / s.ksplit : 0;
  unsigned int* counters = static_cast<unsigned int*>(workspace);
  float* parts = rem ? reinterpret_cast<float*>(static_cast<char*>(workspace) + ((size_t(rem) * 2 * sizeof(unsigned int) + 255) & ~size_t(255))) : nullptr;
  if (rem) {
    if (cudaError_t e = cudaMemsetAsync(counters, 0, size_t(rem) * 2 * sizeof(unsigned int), stream); e != cudaSuccess) return e;
  }
  const int pairs = s.total_units < num_pairs ? s.total_units : num_pairs;
  if (cudaError_t e = launch_overlapped(kern, unsigned(2 * pairs), NUM_THREADS, SMEM_BYTES, 0, stream, ta, tb, p, s, parts, counters); e != cudaSuccess) return e;
  flush_bounds_record(p.status, stream);
  return cudaGetLastError();
}

}  // namespace pair

size_t pair_workspace(const Fp8GemmArgs& g, int num_sms) {
  const pair::Schedule s = pair::make_schedule(g.M, g.N, g.K, g.form, num_sms / 2);
  if (s.ksplit == 1) return 0;
  const size_t rem = size_t(s.total_units - s.full_tiles) / s.ksplit;
  return ((rem * 2 * sizeof(unsigned int) + 255) & ~size_t(255)) + rem * s.ksplit * 2 * pair::PART_FLOATS * sizeof(float);
}

cudaError_t launch_pair(const Fp8GemmArgs& g, const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int num_sms, cudaStream_t stream) {
  using namespace pair;
  const int num_pairs = num_sms / 2;
  const Schedule s = make_schedule(g.M, g.N, g.K, g.form, num_pairs);
#define ELFB_LAUNCH(MN, FORM, T) return launch<MN, Fp8Form::FORM, T>(ta, tb, p, s, g.workspace, num_pairs, stream)
  if (g.form == Fp8Form::kGated) ELFB_LAUNCH(false, kGated, float);
  if (g.form == Fp8Form::kGatedBackward) ELFB_LAUNCH(true, kGatedBackward, float);
  if (g.b.mn_major) {
    if (g.out == Elem::kBf16) ELFB_LAUNCH(true, kPlain, __nv_bfloat16);
    if (g.out == Elem::kF16) ELFB_LAUNCH(true, kPlain, __half);
    ELFB_LAUNCH(true, kPlain, float);
  }
  if (g.out == Elem::kBf16) ELFB_LAUNCH(false, kPlain, __nv_bfloat16);
  if (g.out == Elem::kF16) ELFB_LAUNCH(false, kPlain, __half);
  ELFB_LAUNCH(false, kPlain, float);
#undef ELFB_LAUNCH
}

}  // namespace fp8
}  // namespace elfb
