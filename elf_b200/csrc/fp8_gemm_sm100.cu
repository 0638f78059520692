// Products of block-scaled 8-bit matrices on the tcgen05 block-scaled tensor path.
//
//   D[m, n] = sum over blocks b of 128:  2^(sa[m, b] - 127) 2^(sb[n, b] - 127)  sum over k in b:  a[m, k] b[n, k]
//
// The scales are powers of two, so the tensor core applies them itself (kind::mxf8f6f4: exponent bytes
// read from TMEM) and the products run at the full 8-bit rate with one fp32 accumulation over all of
// K; no partial sum passes through registers.  The instruction takes one exponent per 32 values of K:
// the four steps of a block name the same byte.
//
//   forward     Y  = X . W^T   A = X  [M,K]   B = W [N,K]  K-major   (gated form: B = [gate | up])
//   input grad  dX = dY . W    A = dY [M,K]   B = W [K,N]  MN-major  (its 128 x 128 tiles scale either way)
//
// This file: the kernel for up to 128 rows, and the choice between it and the CTA-pair kernel
// (fp8_gemm_sm100_2cta.cu).  With few rows the time is that of reading B, so the work is spread over all
// SMs: one 128 x 128 tile per cluster of up to 8 CTAs that split K among them and add their fp32 sums,
// in rank order, through distributed shared memory.
//
// Roles per CTA (224 threads):
//   warp 0      TMA producer: ring of (A 128 x 128, B 128 x 128) byte tiles, 128B-swizzled.
//   warp 1      MMA issuer: 128 x 128 x 32 steps into one TMEM accumulator.
//   warps 2..5  epilogue, thread = row.
//   warp 6      scale words: exponent bytes of four blocks of K, from global to shared memory; the MMA thread
//               copies them to TMEM in order with its MMAs.
#include "fp8_gemm.cuh"

namespace elfb {

namespace fp8 {

namespace rows128 {

constexpr int BN = 128;
// A's box holds ROWS (32 or 128) rows.  The MMA always reads 128; behind a box of 32 lies B's, whose bytes end in
// accumulator rows that nobody looks at.  Up to 32 rows leave room for two CTAs per SM, one of which starts or ends
// while the other streams.  16 x 4096 x 14336, one launch after the other: 15.9 us (59 MB: 9.0 at the copy rate); a launch
// by itself spends 5.5 on the weights (in L2), 3.5 until the first bytes, most of it hidden behind the launch before, and
// 3.3 on adding the parts.  Without the split 45.5.
template <int ROWS>
constexpr int CTAS_PER_SM = ROWS == 32 ? 2 : 1;
template <int ROWS>
constexpr int STAGES = ROWS == 32 ? 4 : 6;
template <int ROWS>
constexpr int SLOTS = STAGES<ROWS> / 2;     // two consecutive stages share scale words and are freed together
template <int ROWS>
constexpr int A_BYTES = ROWS * BK;
template <int ROWS>
constexpr int STAGE_BYTES = A_BYTES<ROWS> + BOX_BYTES;
constexpr int SF_BYTES = 2 * 512;           // scale words of a slot: 128 rows of A, 128 columns of B
constexpr int NUM_THREADS = 224;
constexpr int TMEM_COLUMNS = 256;           // 128 of the accumulator, then two 8-column scale slots
constexpr int MAX_CLUSTER = 8;
template <int ROWS>
constexpr size_t SMEM_BYTES = size_t(STAGES<ROWS>) * STAGE_BYTES<ROWS> + SLOTS<ROWS> * SF_BYTES + 1024 /*align slack*/ + 256 /*barriers*/;
static_assert(STAGES<32> * STAGE_BYTES<32> >= 32 * BN * 4 && STAGES<128> * STAGE_BYTES<128> >= BM * BN * 4, "the sums are exchanged in the ring's memory");
static_assert(STAGE_BYTES<32> >= BM * BK, "an MMA reads 128 rows from where A begins: they end inside the stage");

__device__ __forceinline__ float4 load_cluster_f4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}

template <int ROWS, bool B_MN, typename T>
__global__ void __launch_bounds__(NUM_THREADS, CTAS_PER_SM<ROWS>)
fp8_gemm_rows128_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ Params p, int ksplit) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_aligned = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t sf_base = smem_base + STAGES<ROWS> * STAGE_BYTES<ROWS>;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_aligned + size_t(STAGES<ROWS>) * STAGE_BYTES<ROWS> + SLOTS<ROWS> * SF_BYTES);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int slot) { return bar0 + 8u * (STAGES<ROWS> + slot); };
  const uint32_t done_bar = bar0 + 8u * (STAGES<ROWS> + SLOTS<ROWS>);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + STAGES<ROWS> + SLOTS<ROWS> + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = ksplit > 1 ? int(cluster_ctarank()) : 0;
  const int n0 = int(blockIdx.x) / ksplit * BN;
  const int k_blocks = (p.K + BK - 1) / BK, groups = (k_blocks + 3) / 4;
  const int kb0 = 4 * int((long long)groups * rank / ksplit), kb1 = min(k_blocks, 4 * int((long long)groups * (rank + 1) / ksplit));

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES<ROWS>; ++s) mbar_init(full_bar(s), s & 1 ? 1 : 2);  // a slot's first stage also waits for the scale warp
    for (int s = 0; s < SLOTS<ROWS>; ++s) mbar_init(empty_bar(s), 1);
    mbar_init(done_bar, 1);
    fence_barrier_init();
    prefetch_tensormap(&tmap_a);
    prefetch_tensormap(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  await_previous();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb2 = kb0; kb2 < kb1 && ok; kb2 += 2) {
        if (!mbar_wait(empty_bar(slot), phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        for (int kb = kb2; kb < min(kb2 + 2, kb1); ++kb) {
          const int stage = 2 * slot + (kb - kb2);
          const uint32_t sa = smem_base + stage * STAGE_BYTES<ROWS>, sb = sa + A_BYTES<ROWS>, bar = full_bar(stage);
          mbar_arrive_expect_tx(bar, STAGE_BYTES<ROWS>);
          tma_load_2d(sa, &tmap_a, bar, kb * BK, 0);
          if (B_MN) tma_load_2d(sb, &tmap_b, bar, n0, kb * BK);
          else tma_load_2d(sb, &tmap_b, bar, kb * BK, n0);
        }
        if (++slot == SLOTS<ROWS>) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      // K-major: rows of 128 bytes, 8-row groups 1024 B apart, a step of 32 values = 32 B.
      // MN-major: 128-wide boxes of 128 k-rows, 8-row groups 1024 B apart, a step of 32 rows = 4096 B.
      constexpr uint32_t B_KSTEP = B_MN ? UMMA_K * 128 : UMMA_K;
      int slot = 0;
      uint32_t stage_phase = 0, sf_count = 0;
      bool ok = true;
      for (int kb2 = kb0; kb2 < kb1 && ok; kb2 += 2) {
        const uint32_t sfa = tmem_base + BN + (sf_count++ & 1) * 8, sfb = sfa + 4;
        for (int kb = kb2; kb < min(kb2 + 2, kb1); ++kb) {
          const int stage = 2 * slot + (kb - kb2);
          if (!mbar_wait(full_bar(stage), (stage_phase >> stage) & 1u, abort_flag)) {
            ok = false;
            break;
          }
          stage_phase ^= 1u << stage;
          tc_fence_after_sync();
          const uint32_t sa = smem_base + stage * STAGE_BYTES<ROWS>, sb = sa + A_BYTES<ROWS>;
          if (kb == kb2) {
            const uint32_t sf = sf_base + slot * SF_BYTES;
            tmem_cp_32x128b(sfa, make_smem_desc_rows16(sf));
            tmem_cp_32x128b(sfb, make_smem_desc_rows16(sf + 512));
          }
          const uint32_t idesc = make_idesc_mxf8(BM, BN, 0u, B_MN ? 1u : 0u, kb & 3);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t da = make_smem_desc_sw128(sa + k * UMMA_K, 0, 1024);
            const uint64_t db = make_smem_desc_sw128(sb + k * B_KSTEP, 0, 1024);
            umma_ss_mxf8(tmem_base, da, db, idesc, sfa, sfb, (kb > kb0 || k) ? 1u : 0u);
          }
        }
        if (!ok) break;
        umma_commit(empty_bar(slot));
        if (++slot == SLOTS<ROWS>) slot = 0;
      }
      if (ok) umma_commit(done_bar);
    }
    __syncwarp();
  } else if (warp < 6) {
    // ------------------------------------------------------------------ accumulator: to D, or to shared memory for the exchange
    const int quarter = warp & 3;  // TMEM lanes [32*quarter, 32*quarter+32) belong to this warp
    const int row = quarter * 32 + lane;
    if (mbar_wait(done_bar, 0, abort_flag)) {
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16);
      if (quarter * 32 < p.M) {
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          const int col = n0 + c * 32;
          if (col >= p.N) break;
          uint32_t v[32];
          tmem_ld_32x32b_x32(taddr + c * 32, v);
          tmem_ld_wait();
          if (ksplit == 1) {
            store_chunk<T>(v, row, col, p);
          } else if (row < p.M) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {  // 16-byte pieces of a row, exchanged so that the lanes' stores hit different banks
              const uint32_t dst = smem_base + uint32_t(row) * (BN * 4) + (uint32_t((c * 8 + q) ^ (row & 31)) << 4);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[4 * q]), "r"(v[4 * q + 1]), "r"(v[4 * q + 2]), "r"(v[4 * q + 3]) : "memory");
            }
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ scale words (warp 6)
    // A second producer of the ring: the words of a group of four blocks go to both slots of the group.  Those
    // of the next group are fetched from global memory before a slot is waited for.
    int g = kb0 / 4, slot = 0;
    uint32_t phase = 0;
    RawScales ra, rb;
    auto load = [&] {
      load_scales(p.sa, 0, p.M, g, k_blocks, lane, ra);
      load_scales(p.sb, n0, p.N, g, k_blocks, lane, rb);
    };
    if (kb0 < kb1) load();
    bool ok = true;
    while (ok && 4 * g < kb1) {
      uint32_t a[4], b[4];
      combine_scales(p.sa, g, k_blocks, ra, a);
      combine_scales(p.sb, g, k_blocks, rb, b);
      const int slots = kb1 - 4 * g > 2 ? 2 : 1;
      ++g;
      if (4 * g < kb1) load();
      for (int i = 0; i < slots; ++i) {
        if (!mbar_wait(empty_bar(slot), phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        store_scale_words(sf_base + slot * SF_BYTES, lane, a);
        store_scale_words(sf_base + slot * SF_BYTES + 512, lane, b);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar(2 * slot));
        if (++slot == SLOTS<ROWS>) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
  }

  // ------------------------------------------------------------------ sums of the cluster
  tc_fence_before_sync();
  __syncthreads();
  if (ksplit > 1) {
    cluster_sync_all();
    // a row's 32 pieces go to 32 consecutive threads; rows are dealt to the CTAs
    if (!*abort_flag && warp < 4) {
      const int q = lane;
      const int col = n0 + 4 * q;
      for (int row = rank + warp * ksplit; row < p.M; row += 4 * ksplit) {
        const uint32_t src = smem_base + uint32_t(row) * (BN * 4) + (uint32_t(q ^ (row & 31)) << 4);
        float4 part[MAX_CLUSTER];
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; ++r)
          if (r < ksplit) part[r] = load_cluster_f4(map_to_cta(src, r));
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; ++r)
          if (r < ksplit) s[0] += part[r].x, s[1] += part[r].y, s[2] += part[r].z, s[3] += part[r].w;
        store_quad<T>(s, row, col, p);
      }
    }
    cluster_sync_all();  // the peers may still be reading this CTA's shared memory
  }

  // ------------------------------------------------------------------ common exit
  if (*abort_flag) {
    if (threadIdx.x == 0) {
      // let TMA copies that are still in flight land before the CTA's shared memory goes away
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) {
      }
      if (p.status != nullptr && atomicCAS(p.status, kOk, kErrBarrierTimeout) == kOk) {
        p.status[1] = 2000000 + blockIdx.x;
        p.status[2] = p.M;
        p.status[3] = p.N;
      }
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLUMNS);
  }
}

template <int ROWS, bool B_MN, typename T>
cudaError_t launch(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int num_sms, cudaStream_t stream) {
  auto kern = fp8_gemm_rows128_kernel<ROWS, B_MN, T>;
  // function attributes are per device: remember which devices of this process have been set up
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(SMEM_BYTES<ROWS>));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
  }
  const int tiles = (p.N + BN - 1) / BN, groups = (p.K + 4 * BK - 1) / (4 * BK);
  int ksplit = 1;  // as many parts as there are SMs for, each at least four blocks of K long
  while (ksplit < MAX_CLUSTER && 2 * ksplit * tiles <= num_sms * CTAS_PER_SM<ROWS> && 2 * ksplit <= groups) ksplit *= 2;
  if (cudaError_t e = launch_overlapped(kern, unsigned(tiles) * ksplit, NUM_THREADS, SMEM_BYTES<ROWS>, unsigned(ksplit), stream, ta, tb, p, ksplit); e != cudaSuccess)
    return e;
  flush_bounds_record(p.status, stream);
  return cudaGetLastError();
}

}  // namespace rows128

cudaError_t launch_rows128(const Fp8GemmArgs& g, const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int num_sms, cudaStream_t s) {
  using namespace rows128;
#define ELFB_LAUNCH(MN, T) return g.M <= 32 ? launch<32, MN, T>(ta, tb, p, num_sms, s) : launch<128, MN, T>(ta, tb, p, num_sms, s)
  if (g.b.mn_major) {
    if (g.out == Elem::kBf16) ELFB_LAUNCH(true, __nv_bfloat16);
    if (g.out == Elem::kF16) ELFB_LAUNCH(true, __half);
    ELFB_LAUNCH(true, float);
  }
  if (g.out == Elem::kBf16) ELFB_LAUNCH(false, __nv_bfloat16);
  if (g.out == Elem::kF16) ELFB_LAUNCH(false, __half);
  ELFB_LAUNCH(false, float);
#undef ELFB_LAUNCH
}

cudaError_t launch_pair(const Fp8GemmArgs& g, const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int num_sms, cudaStream_t stream);
size_t pair_workspace(const Fp8GemmArgs& g, int num_sms);

// The gated forms, whose epilogues want whole blocks of 128 columns, have one kernel.
bool use_pair(const Fp8GemmArgs& g) { return g.form != Fp8Form::kPlain || g.M > 128; }

}  // namespace fp8

size_t fp8_gemm_workspace(const Fp8GemmArgs& g, int num_sms) {
  if (g.M <= 0 || g.N <= 0 || g.K <= 0 || !fp8::use_pair(g)) return 0;
  return fp8::pair_workspace(g, num_sms);
}

const char* make_tmap_bytes(CUtensorMap* out, const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols, uint32_t box_rows);

const char* fp8_gemm(const Fp8GemmArgs& g, int num_sms, cudaStream_t stream) {
  using namespace fp8;
  if (g.M <= 0 || g.N <= 0 || g.K <= 0) return nullptr;
  CUtensorMap ta, tb;
  const char* err = make_tmap_bytes(&ta, g.a.data, uint64_t(g.M), uint64_t(g.K), uint64_t(g.a.ld), BK, use_pair(g) || g.M > 32 ? BM : 32);
  if (err) return err;
  if (g.b.mn_major) err = make_tmap_bytes(&tb, g.b.data, uint64_t(g.K), uint64_t(g.N), uint64_t(g.b.ld), 128, BK);
  else              err = make_tmap_bytes(&tb, g.b.data, uint64_t(g.N), uint64_t(g.K), uint64_t(g.b.ld), BK, 128);
  if (err) return err;
  Params p{g.M, g.N, g.K, Scales(g.a), Scales(g.b)};
  p.status = g.status;
  cudaError_t e;
  if (g.form != Fp8Form::kPlain) {
    auto aligned = [](const void* q, long long pitch) { return ((reinterpret_cast<uintptr_t>(q) | uintptr_t(pitch)) & 31) == 0; };
    const bool backward = g.form == Fp8Form::kGatedBackward;
    if (g.b.mn_major != backward || g.N % (backward ? 128 : 256) != 0) return "the gated product's width must be a multiple of 128";
    if (!aligned(g.act, g.ld_act) || (g.gu && !aligned(g.gu, g.ld_gu))) return "8-bit matrices of the gated forms must be 32-byte aligned with a 32-byte multiple row pitch";
    p.act = g.act, p.act_scale = g.act_scale, p.gu = g.gu, p.gu_scale = g.gu_scale;
    p.ld_act = g.ld_act, p.ld_act_scale = g.ld_act_scale, p.ld_gu = g.ld_gu, p.ld_gu_scale = g.ld_gu_scale;
    e = launch_pair(g, ta, tb, p, num_sms, stream);
  } else {
    const long long esz = g.out == Elem::kF32 ? 4 : 2;
    p.d = g.d, p.ldd = g.ldd, p.bias = g.bias;
    p.vec = ((reinterpret_cast<uintptr_t>(g.d) | uintptr_t(g.ldd * esz)) & 15) == 0;
    e = use_pair(g) ? launch_pair(g, ta, tb, p, num_sms, stream) : launch_rows128(g, ta, tb, p, num_sms, stream);
  }
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace elfb
