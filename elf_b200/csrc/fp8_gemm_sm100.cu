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
// Structure per CTA (320 threads, one CTA per SM, persistent over 128 x BN tiles):
//   warp 0      TMA producer: ring of (A 128 x 128, B BN x 128) byte tiles, 128B-swizzled.
//   warp 1      MMA issuer: 128 x BN x 32 steps into one of two TMEM accumulators.
//   warps 2..5  epilogue, thread = row.
//   warps 6..9  scale writers: read the exponent bytes of the next four blocks of K (512 values) from
//               global memory and store them to one of two TMEM slots, each warp its own quarter of
//               the lanes.  4 + BN/32 words per lane and 512 values of K: negligible traffic.
//
// TMEM has 512 columns; two 256-column accumulators would leave none for the scales.  The second one
// therefore starts 32 columns early and shares them with the first; the epilogue reads the shared
// columns first and the next tile's products start as soon as it has.
#include "fp8_gemm.cuh"

namespace elfb {

namespace fp8 {

constexpr int STAGES = 4;
constexpr int NUM_THREADS = 320;
constexpr int GROUP_M = 8;  // tiles of GROUP_M consecutive M-blocks share B panels in L2

template <int BN>
constexpr int kStageBytes = BOX_BYTES * (1 + BN / 128);
template <int BN>
constexpr size_t kSmemBytes = size_t(STAGES) * kStageBytes<BN> + 1024 /*align slack*/ + 256 /*barriers*/;

struct Tile {
  int m0, n0, n1;  // first row of A; first rows of B's two 128-row halves
};

template <int BN, bool GATED>
__device__ __forceinline__ Tile tile_at(int t, int tiles_m, int tiles_n, int f) {
  const int per_group = GROUP_M * tiles_n;
  const int group = t / per_group;
  const int first_m = group * GROUP_M;
  const int rows = min(GROUP_M, tiles_m - first_m);
  const int in_group = t - group * per_group;
  Tile r;
  r.m0 = (first_m + in_group % rows) * BM;
  if (GATED) {
    r.n0 = (in_group / rows) * 128;
    r.n1 = f + r.n0;
  } else {
    r.n0 = (in_group / rows) * BN;
    r.n1 = r.n0 + 128;
  }
  return r;
}

template <int BN, bool B_MN, bool GATED, typename T>
__global__ void __launch_bounds__(NUM_THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ Params p) {
  constexpr int STAGE = kStageBytes<BN>;
  constexpr bool OVERLAP = BN == 256;           // the accumulators share 32 columns
  constexpr int ACC1 = OVERLAP ? 224 : 256;     // first column of the second one
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_aligned = smem_raw + (smem_base - smem_u32(smem_raw));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_aligned + size_t(STAGES) * STAGE);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto acc_full_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
  auto acc_empty_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };  // OVERLAP: only [0], one completion per tile
  auto sf_full_bar = [&](int s) { return bar0 + 8u * (2 * STAGES + 4 + s); };
  auto sf_empty_bar = [&](int s) { return bar0 + 8u * (2 * STAGES + 6 + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int f = p.N / 2;  // gated: width of the activation
  const int tiles_m = (p.M + BM - 1) / BM;
  const int tiles_n = GATED ? f / 128 : (p.N + BN - 1) / BN;
  const int tiles = tiles_m * tiles_n;
  const int k_blocks = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full_bar(a), 1);
      mbar_init(acc_empty_bar(a), 4);  // one arrival per epilogue warp
      mbar_init(sf_full_bar(a), 4);    // one arrival per scale warp
      mbar_init(sf_empty_bar(a), 1);
    }
    fence_barrier_init();
    prefetch_tensormap(&tmap_a);
    prefetch_tensormap(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const Tile tile = tile_at<BN, GATED>(t, tiles_m, tiles_n, f);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t sa = smem_base + stage * STAGE, sb = sa + BOX_BYTES, bar = full_bar(stage);
          mbar_arrive_expect_tx(bar, STAGE);
          const int k0 = kb * BK;
          tma_load_2d(sa, &tmap_a, bar, k0, tile.m0);
          // a box that lies behind B's last row arrives as zeros
          if (B_MN) {
            tma_load_2d(sb, &tmap_b, bar, tile.n0, k0);
            if (BN == 256) tma_load_2d(sb + BOX_BYTES, &tmap_b, bar, tile.n1, k0);
          } else {
            tma_load_2d(sb, &tmap_b, bar, k0, tile.n0);
            if (BN == 256) tma_load_2d(sb + BOX_BYTES, &tmap_b, bar, k0, tile.n1);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      // K-major: rows of 128 bytes, 8-row groups 1024 B apart, a step of 32 values = 32 B.
      // MN-major: 128-wide boxes of 128 k-rows, 8-row groups 1024 B apart, a step of 32 rows = 4096 B.
      constexpr uint32_t B_LBO = B_MN ? BOX_BYTES : 0;
      constexpr uint32_t B_KSTEP = B_MN ? UMMA_K * 128 : UMMA_K;
      int stage = 0;
      uint32_t phase = 0, sf_count = 0;
      bool ok = true;
      int i = 0;  // tiles of this CTA so far
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++i) {
        const int acc = i & 1;
        if (OVERLAP) {
          if (i > 0 && !mbar_wait(acc_empty_bar(0), uint32_t(i - 1) & 1u, abort_flag)) break;
        } else {
          if (!mbar_wait(acc_empty_bar(acc), (uint32_t(i >> 1) & 1u) ^ 1u, abort_flag)) break;
        }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + acc * ACC1;
        for (int kb = 0; kb < k_blocks; ++kb) {
          const int slot = sf_count & 1;
          if ((kb & 3) == 0 && !mbar_wait(sf_full_bar(slot), (sf_count >> 1) & 1u, abort_flag)) {
            ok = false;
            break;
          }
          if (!mbar_wait(full_bar(stage), phase, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sa = smem_base + stage * STAGE, sb = sa + BOX_BYTES;
          const uint32_t sfa = tmem_base + SF_COL + slot * 16, sfb = sfa + 4;
          const uint32_t idesc = make_idesc_mxf8(BM, BN, 0u, B_MN ? 1u : 0u, kb & 3);
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t da = make_smem_desc_sw128(sa + k * UMMA_K, 0, 1024);
            const uint64_t db = make_smem_desc_sw128(sb + k * B_KSTEP, B_LBO, 1024);
            umma_ss_mxf8(tmem_d, da, db, idesc, sfa, sfb, (kb | k) ? 1u : 0u);
          }
          umma_commit(empty_bar(stage));
          if ((kb & 3) == 3 || kb + 1 == k_blocks) {
            umma_commit(sf_empty_bar(slot));
            ++sf_count;
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit(acc_full_bar(acc));
      }
    }
    __syncwarp();
  } else if (warp < 6) {
    // ------------------------------------------------------------------ epilogue (warps 2..5)
    const int quarter = warp & 3;  // TMEM lanes [32*quarter, 32*quarter+32) belong to this warp
    int i = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
      const Tile tile = tile_at<BN, GATED>(t, tiles_m, tiles_n, f);
      const int acc = i & 1;
      const int row = tile.m0 + quarter * 32 + lane;
      if (!mbar_wait(acc_full_bar(acc), uint32_t(i >> 1) & 1u, abort_flag)) break;
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + acc * ACC1;
      auto release = [&](int bar) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty_bar(bar));
      };
      if constexpr (GATED) {
        if (acc == 0) gated_tile<0>(taddr, row, tile.n0, f, p, [&] { release(0); });
        else gated_tile<1>(taddr, row, tile.n0, f, p, [&] { release(0); });
      } else {
        constexpr int CHUNKS = BN / 32;
#pragma unroll 1
        for (int j = 0; j < CHUNKS; ++j) {
          const int c = OVERLAP && acc == 0 ? CHUNKS - 1 - j : j;  // the shared columns first
          uint32_t v[32];
          tmem_ld_32x32b_x32(taddr + c * 32, v);
          tmem_ld_wait();
          if (OVERLAP && j == 0) release(0);
          const int col = tile.n0 + c * 32;
          if (col < p.N) store_chunk<T>(v, row, col, p);
        }
        if (!OVERLAP) release(acc);
      }
    }
  } else {
    // ------------------------------------------------------------------ scale writers (warps 6..9)
    // The words of the next group are fetched before the slot of this one is waited for.
    const int quarter = warp & 3;
    int t = blockIdx.x, g = 0;
    Tile tile = tile_at<BN, GATED>(t, tiles_m, tiles_n, f);
    RawScales ra, rb0, rb1;
    auto load = [&] {
      load_scales(p.sa, tile.m0, p.M, g, k_blocks, lane, ra);
      load_scales(p.sb, tile.n0, p.N, g, k_blocks, lane, rb0);
      if (BN == 256) load_scales(p.sb, tile.n1, p.N, g, k_blocks, lane, rb1);
    };
    if (t < tiles) load();
    for (uint32_t count = 0; t < tiles; ++count) {
      uint32_t a[4], b0[4], b1[4];
      combine_scales(p.sa, g, k_blocks, ra, a);
      combine_scales(p.sb, g, k_blocks, rb0, b0);
      if (BN == 256) combine_scales(p.sb, g, k_blocks, rb1, b1);
      if (4 * ++g >= k_blocks) {
        g = 0;
        t += gridDim.x;
        if (t < tiles) tile = tile_at<BN, GATED>(t, tiles_m, tiles_n, f);
      }
      if (t < tiles) load();
      const int slot = count & 1;
      if (!mbar_wait(sf_empty_bar(slot), ((count >> 1) & 1u) ^ 1u, abort_flag)) break;
      tc_fence_after_sync();
      const uint32_t dst = tmem_base + (uint32_t(quarter) * 32u << 16) + SF_COL + slot * 16;
      tmem_st_32x32b_x4(dst, a);
      tmem_st_32x32b_x4(dst + 4, b0);
      if (BN == 256) tmem_st_32x32b_x4(dst + 8, b1);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(sf_full_bar(slot));
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
        p.status[1] = 2000000 + blockIdx.x;
        p.status[2] = p.M;
        p.status[3] = p.N;
      }
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int BN, bool B_MN, bool GATED, typename T>
cudaError_t launch(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int num_sms, cudaStream_t stream) {
  auto kern = fp8_gemm_kernel<BN, B_MN, GATED, T>;
  constexpr size_t smem = kSmemBytes<BN>;
  // function attributes are per device: remember which devices of this process have been set up
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
  }
  const int tiles = ((p.M + BM - 1) / BM) * (GATED ? p.N / 256 : (p.N + BN - 1) / BN);
  kern<<<tiles < num_sms ? tiles : num_sms, NUM_THREADS, smem, stream>>>(ta, tb, p);
  flush_bounds_record(p.status, stream);
  return cudaGetLastError();
}

template <int BN>
cudaError_t dispatch(const Fp8GemmArgs& g, const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int num_sms, cudaStream_t s) {
  if (g.b.mn_major) {
    if (g.out == Elem::kBf16) return launch<BN, true, false, __nv_bfloat16>(ta, tb, p, num_sms, s);
    if (g.out == Elem::kF16) return launch<BN, true, false, __half>(ta, tb, p, num_sms, s);
    return launch<BN, true, false, float>(ta, tb, p, num_sms, s);
  }
  if (g.out == Elem::kBf16) return launch<BN, false, false, __nv_bfloat16>(ta, tb, p, num_sms, s);
  if (g.out == Elem::kF16) return launch<BN, false, false, __half>(ta, tb, p, num_sms, s);
  return launch<BN, false, false, float>(ta, tb, p, num_sms, s);
}

cudaError_t launch_pair(const Fp8GemmArgs& g, const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int num_sms, cudaStream_t stream);
size_t pair_workspace(int M, int N, int K, bool gated, int num_sms);

// Few rows leave most of a 256-row tile empty.
bool use_pair(const Fp8GemmArgs& g, int num_sms) { return num_sms >= 2 && g.M > 128; }

}  // namespace fp8

size_t fp8_gemm_workspace(const Fp8GemmArgs& g, int num_sms) {
  if (g.M <= 0 || g.N <= 0 || g.K <= 0 || !fp8::use_pair(g, num_sms)) return 0;
  return fp8::pair_workspace(g.M, g.N, g.K, g.gated, num_sms);
}

const char* make_tmap_bytes(CUtensorMap* out, const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols, uint32_t box_rows);

const char* fp8_gemm(const Fp8GemmArgs& g, int num_sms, cudaStream_t stream) {
  using namespace fp8;
  if (g.M <= 0 || g.N <= 0 || g.K <= 0) return nullptr;
  CUtensorMap ta, tb;
  const char* err = make_tmap_bytes(&ta, g.a.data, uint64_t(g.M), uint64_t(g.K), uint64_t(g.a.ld), BK, BM);
  if (err) return err;
  if (g.b.mn_major) err = make_tmap_bytes(&tb, g.b.data, uint64_t(g.K), uint64_t(g.N), uint64_t(g.b.ld), 128, BK);
  else              err = make_tmap_bytes(&tb, g.b.data, uint64_t(g.N), uint64_t(g.K), uint64_t(g.b.ld), BK, 128);
  if (err) return err;
  Params p{g.M, g.N, g.K, Scales(g.a), Scales(g.b)};
  p.status = g.status;
  cudaError_t e;
  if (g.gated) {
    auto aligned = [](const void* q, long long pitch) { return ((reinterpret_cast<uintptr_t>(q) | uintptr_t(pitch)) & 15) == 0; };
    if (g.b.mn_major || g.N % 256 != 0) return "the gated product needs K-major weights and a width that is a multiple of 128";
    if (!aligned(g.act, g.ld_act) || (g.gu && !aligned(g.gu, g.ld_gu))) return "8-bit outputs must be 16-byte aligned with a 16-byte multiple row pitch";
    p.act = g.act, p.act_scale = g.act_scale, p.gu = g.gu, p.gu_scale = g.gu_scale;
    p.ld_act = g.ld_act, p.ld_act_scale = g.ld_act_scale, p.ld_gu = g.ld_gu, p.ld_gu_scale = g.ld_gu_scale;
    e = use_pair(g, num_sms) ? launch_pair(g, ta, tb, p, num_sms, stream) : launch<256, false, true, __nv_bfloat16>(ta, tb, p, num_sms, stream);
  } else {
    const long long esz = g.out == Elem::kF32 ? 4 : 2;
    p.d = g.d, p.ldd = g.ldd, p.bias = g.bias;
    p.vec = ((reinterpret_cast<uintptr_t>(g.d) | uintptr_t(g.ldd * esz)) & 15) == 0;
    if (use_pair(g, num_sms)) e = launch_pair(g, ta, tb, p, num_sms, stream);
    else e = g.N > 128 ? dispatch<256>(g, ta, tb, p, num_sms, stream) : dispatch<128>(g, ta, tb, p, num_sms, stream);
  }
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace elfb
