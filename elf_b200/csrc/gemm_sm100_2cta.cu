// CTA-pair variant of the tcgen05 GEMM: two CTAs on neighbouring SMs (a cluster of 2) share
// one 256x256 output tile through `tcgen05.mma.cta_group::2`.
//
// Each CTA owns 128 of the tile's 256 rows: it TMA-loads its own A slab (128 x 64) and HALF
// of the B slab (128 of the 256 B rows) into its own shared memory and receives its 128
// accumulator rows in its own TMEM.  Per flop, each SM therefore reads half as much B from
// shared memory as in the single-CTA kernel (and fetches half as much from L2), which is
// what lets the tensor pipe run closer to its peak under the power cap.
//
// Synchronisation (every wait bounded, see sm100_ptx.cuh):
//   full[s]      (one per slot of two stages) lives in the EVEN CTA (the leader).  The leader's producer arms it with the
//                byte count of both CTAs' loads; both CTAs' TMA copies complete on it
//                (the odd CTA addresses it through the cluster window; no multicast).
//   empty[s]     one per CTA; the leader's MMA thread commits to both after the MMAs that
//                read the two stages of slot s.
//   acc_full[a]  one per CTA; committed by the leader after the last MMA of a tile.
//   acc_empty[a] in the leader; the epilogue warps of both CTAs arrive on it (8 arrivals).
// Only the leader's MMA thread issues MMAs.  TMEM is allocated and freed with the
// cta_group::2 forms by warp 1 of both CTAs.

#include <algorithm>
#include <cstdio>
#include <cstdlib>

#include "sm100_ptx.cuh"
#include "gemm_epilogue.cuh"
#include "dp_signal.cuh"
#include "gemm_sm100.h"

namespace elfb {

namespace pair {

constexpr int BM = 128;          // rows per CTA (256 per pair)
constexpr int BN = 256;          // columns per pair tile
constexpr int BK = 64;
constexpr int STAGES = 6;
constexpr int SLOTS = STAGES / 2;  // two consecutive stages are filled, waited for and freed together
constexpr int UMMA_K = 16;
constexpr int A_BYTES = BM * BK * 2;        // 16 KiB
constexpr int B_BYTES = (BN / 2) * BK * 2;  // 16 KiB: this CTA's half of the B slab
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int NUM_THREADS = 192;
constexpr int TMEM_COLS = 512;
constexpr int DEFAULT_GROUP_M = 4;  // tile rows (of 256) that are swept together before moving to the next columns
constexpr int PART_FLOATS = BM * BN;  // one CTA's half of a tile in the workspace
constexpr int STAGING_BYTES = 2 * 16384;  // two 128-row x 128-byte chunks for the TMA-store epilogue
constexpr size_t SMEM_BYTES = size_t(STAGES) * STAGE_BYTES + STAGING_BYTES + 1024 + 256;

// Tensor maps over the peers' copies of D (same shape and pitch as the local D), used when the
// epilogue also pushes its tiles to other GPUs.
struct alignas(64) PeerMaps {
  CUtensorMap m[kMaxPeers];
};

struct WorkUnit {
  int m, n0;      // tile row (in 256-row units) and first output column
  int kb0, kb1;   // range of 64-wide k-blocks this unit contracts over
  int part;       // index of this unit among the k-parts of its tile (0 when the tile is whole)
  bool partial;   // true: the unit holds a partial sum and must add it to D
};
// Tiles are dealt round-robin to the CTA pairs.  When the tile count is not a multiple of
// the pair count the last, partly filled wave would cost a whole tile time with most SMs
// idle; instead each tile of that wave is split along K into `ksplit` units that run on
// different pairs and add their partial sums to D (TMA add-reduce in L2), or leave them in fp32 in a
// workspace for the last one to add in their order (2048 x 5504 from 2047 tokens, with the operands'
// restores: 51 and 55 us).  Unlike a split
// along N this keeps the 256x256 tile's ratio of MMA work to bytes loaded.
struct Schedule {
  int tiles_m, tiles_n, full_tiles, ksplit, total_units, group_m;
};

__host__ __device__ inline Schedule make_schedule(int M, int N, int k_blocks, int num_pairs, int max_split, int group_m) {
  Schedule s;
  s.group_m = group_m;
  s.tiles_m = (M + 2 * BM - 1) / (2 * BM);
  s.tiles_n = (N + BN - 1) / BN;
  const int tiles = s.tiles_m * s.tiles_n;
  const int rem = tiles % num_pairs;
  s.ksplit = 1;
  if (rem != 0 && tiles > rem) {
    // cost of the last wave in 1/840 tile times, plus a charge per extra part for its exposed epilogue
    int best = 840;
    for (int f = 2; f <= max_split && f * 4 <= k_blocks; ++f) {
      const int waves = (rem * f + num_pairs - 1) / num_pairs;
      const int cost = waves * 840 / f + 30 * (f - 1);
      if (cost < best) {
        best = cost;
        s.ksplit = f;
      }
    }
  }
  s.full_tiles = s.ksplit == 1 ? tiles : tiles - rem;
  s.total_units = s.full_tiles + (tiles - s.full_tiles) * s.ksplit;
  return s;
}

__host__ __device__ inline void tile_coords(int tile, const Schedule& s, int* m, int* n) {
  const int per_group = s.group_m * s.tiles_n;
  const int group = tile / per_group;
  const int first_m = group * s.group_m;
  const int rows = (s.tiles_m - first_m) < s.group_m ? (s.tiles_m - first_m) : s.group_m;
  const int in_group = tile - group * per_group;
  *m = first_m + in_group % rows;
  *n = in_group / rows;
}

__device__ __forceinline__ WorkUnit work_unit(int unit, const Schedule& s, int k_blocks) {
  WorkUnit wu;
  int tile = unit;
  wu.kb0 = 0;
  wu.kb1 = k_blocks;
  wu.part = 0;
  wu.partial = false;
  if (unit >= s.full_tiles) {
    // parts of one tile are `rem` units apart, so they land on different pairs
    const int rem = (s.total_units - s.full_tiles) / s.ksplit;
    const int u = unit - s.full_tiles;
    tile = s.full_tiles + u % rem;
    wu.part = u / rem;
    wu.kb0 = int((long long)k_blocks * wu.part / s.ksplit);
    wu.kb1 = int((long long)k_blocks * (wu.part + 1) / s.ksplit);
    wu.partial = true;
  }
  int n;
  tile_coords(tile, s, &wu.m, &n);
  wu.n0 = n * BN;
  return wu;
}

// Four accumulating MMAs, k-steps of A_STEP and B_STEP descriptor address units; returns whether the barrier's phase had
// completed when the test, issued before them, came up.
template <int A_STEP, int B_STEP>
__device__ __forceinline__ bool umma_x4_then_ready(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t bar, uint32_t parity) {
  uint32_t ready;
  asm volatile(
      "{\n\t"
      ".reg .pred p, t;\n\t"
      ".reg .b64 a, b;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 t, [%5], %6;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%1], %2, %3, %4, p;\n\t"
      "add.s64 a, %2, %7;\n\t"
      "add.s64 b, %3, %8;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%1], a, b, %4, p;\n\t"
      "add.s64 a, a, %7;\n\t"
      "add.s64 b, b, %8;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%1], a, b, %4, p;\n\t"
      "add.s64 a, a, %7;\n\t"
      "add.s64 b, b, %8;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%1], a, b, %4, p;\n\t"
      "selp.u32 %0, 1, 0, t;\n\t"
      "}\n"
      : "=r"(ready)
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(bar), "r"(parity), "n"(A_STEP), "n"(B_STEP)
      : "memory");
  return ready != 0;
}

template <bool A_MN, bool B_MN, bool OUT_F32, bool ACCUM, bool BIAS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
gemm_tcgen05_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                         const __grid_constant__ CUtensorMap tmap_d, void* __restrict__ d_ptr, const void* __restrict__ bias_ptr, int M, int N, int K, long long ldd,
                         uint32_t fmt, float alpha, int max_split, int group_m, int* __restrict__ status, const __grid_constant__ PushTarget push,
                         const __grid_constant__ PeerMaps peer_maps, float* __restrict__ parts, unsigned int* __restrict__ parts_done) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_aligned = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t staging_base = smem_base + STAGES * STAGE_BYTES;  // 1024-byte aligned
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_aligned + size_t(STAGES) * STAGE_BYTES + STAGING_BYTES);
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int slot) { return bar0 + 8u * slot; };
  auto empty_bar = [&](int slot) { return bar0 + 8u * (SLOTS + slot); };
  auto acc_full_bar = [&](int a) { return bar0 + 8u * (2 * SLOTS + a); };
  auto acc_empty_bar = [&](int a) { return bar0 + 8u * (2 * SLOTS + 2 + a); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * SLOTS + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile unsigned int* arrived = tmem_slot + 2;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();  // 0 = leader, 1 = peer
  const bool leader = cta == 0;
  const int pair_id = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;
  const int k_blocks = (K + BK - 1) / BK;
  const Schedule sched = make_schedule(M, N, k_blocks, num_pairs, max_split, group_m);
  const int num_units = sched.total_units;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(full_bar(s), 1);   // used in the leader only: its producer's arrive.expect_tx
      mbar_init(empty_bar(s), 1);  // one commit per use
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full_bar(a), 1);
      mbar_init(acc_empty_bar(a), 8);  // used in the leader only: 4 epilogue warps of each CTA
    }
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

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int unit = pair_id; unit < num_units && ok; unit += num_pairs) {
        const WorkUnit wu = work_unit(unit, sched, k_blocks);
        const int m0 = wu.m * (2 * BM) + int(cta) * BM;  // this CTA's 128 rows
        constexpr int half = BN / 2;
        const int n0 = wu.n0 + int(cta) * half;          // this CTA's half of the B rows
        for (int kb2 = wu.kb0; kb2 < wu.kb1; kb2 += 2) {
          if (!mbar_wait(empty_bar(slot), phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const int blocks = min(2, wu.kb1 - kb2);
          const uint32_t bar = map_to_cta(full_bar(slot), 0);  // the leader's barrier
          if (leader) mbar_arrive_expect_tx(full_bar(slot), uint32_t(blocks) * 2u * STAGE_BYTES);
          for (int i = 0; i < blocks; ++i) {
            const uint32_t sa = smem_base + (2 * slot + i) * STAGE_BYTES;
            const uint32_t sb = sa + A_BYTES;
            const int k0 = (kb2 + i) * BK;
            if (A_MN) {
#pragma unroll
              for (int j = 0; j < BM / 64; ++j) tma_load_2d_pair(sa + j * (BK * 128), &tmap_a, bar, m0 + 64 * j, k0);
            } else {
              tma_load_2d_pair(sa, &tmap_a, bar, k0, m0);
            }
            if (B_MN) {
#pragma unroll
              for (int j = 0; j < half / 64; ++j) tma_load_2d_pair(sb + j * (BK * 128), &tmap_b, bar, n0 + 64 * j, k0);
            } else {
              tma_load_2d_pair(sb, &tmap_b, bar, k0, n0);
            }
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
      constexpr uint32_t A_LBO = A_MN ? BK * 128 : 0, B_LBO = B_MN ? BK * 128 : 0;
      constexpr uint32_t A_KSTEP = A_MN ? UMMA_K * 128 : UMMA_K * 2, B_KSTEP = B_MN ? UMMA_K * 128 : UMMA_K * 2;
      // A barrier test queues up behind the MMAs issued before it, so its answer comes when the tensor pipe has nearly
      // run dry.  There is one test per slot of eight MMAs, issued before the slot's last four and read after them.
      int slot = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      const uint32_t idesc = make_idesc_f16(fmt, 2 * BM, BN, A_MN ? 1u : 0u, B_MN ? 1u : 0u);
      const uint64_t desc_a0 = make_smem_desc_sw128(smem_base, A_LBO, 1024), desc_b0 = make_smem_desc_sw128(smem_base + A_BYTES, B_LBO, 1024);
      for (int unit = pair_id; unit < num_units && ok; unit += num_pairs) {
        const WorkUnit wu = work_unit(unit, sched, k_blocks);
        if (!mbar_wait(acc_empty_bar(acc), acc_phase ^ 1u, abort_flag)) break;
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + acc * BN;
        bool ready = false;
        for (int kb = wu.kb0; kb < wu.kb1; kb += 2) {
          if (!ready && !mbar_wait(full_bar(slot), phase, abort_flag)) {
            ok = false;
            break;
          }
          const int next = slot + 1 == SLOTS ? 0 : slot + 1;
          const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
          const uint64_t da = desc_a0 + uint32_t(slot * (2 * STAGE_BYTES >> 4)), db = desc_b0 + uint32_t(slot * (2 * STAGE_BYTES >> 4));
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            umma_ss_pair(tmem_d, da + ((k * A_KSTEP) >> 4), db + ((k * B_KSTEP) >> 4), idesc, (kb > wu.kb0 || k) ? 1u : 0u);
          ready = false;
          if (kb + 1 < wu.kb1)
            ready = umma_x4_then_ready<int(A_KSTEP >> 4), int(B_KSTEP >> 4)>(tmem_d, da + (STAGE_BYTES >> 4), db + (STAGE_BYTES >> 4), idesc, full_bar(next), next_phase) &&
                    kb + 2 < wu.kb1;
          umma_commit_both(empty_bar(slot));
          slot = next;
          phase = next_phase;
        }
        if (!ok) break;
        umma_commit_both(acc_full_bar(acc));
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue (both CTAs)
    // The tile leaves through shared memory: each thread converts its row of a 128-byte-wide
    // column chunk into a swizzled staging buffer and one thread hands the chunk to TMA (store,
    // or add-reduce in L2 when accumulating), so the LSU issues no global stores and D is
    // written in full lines.  With a push target (once per step and matrix) the same staged
    // chunk is also TMA-stored into every peer's copy of D over NVLink; when that launch
    // accumulates, the threads read the old values of their rows themselves and the finished
    // sum is stored (locally and remotely) instead of being add-reduced.
    const int quarter = warp & 3;
    const int ep_tid = threadIdx.x - 64;  // 0..127 over the four epilogue warps
    int acc = 0;
    uint32_t acc_phase = 0;
    const uint32_t leader_acc_empty[2] = {map_to_cta(acc_empty_bar(0), 0), map_to_cta(acc_empty_bar(1), 0)};
    const bool pushing = push.n_peers > 0;
    constexpr int CHUNK_COLS = OUT_F32 ? 32 : 64;  // 128 bytes of output per row
    int chunk_counter = 0;
    for (int unit = pair_id; unit < num_units; unit += num_pairs) {
      const WorkUnit wu = work_unit(unit, sched, k_blocks);
      const int row0 = wu.m * (2 * BM) + int(cta) * BM;
      const int row = row0 + quarter * 32 + lane;
      const bool joined = wu.partial && parts != nullptr;  // fp32 parts in the workspace, added by the last to finish
      const bool add_bias = BIAS && (wu.part == 0 || joined);
      const int n0 = wu.n0;
      if (!named_barrier_all(1, 128, mbar_wait(acc_full_bar(acc), acc_phase, abort_flag))) break;
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + acc * BN;
      bool finish = true;  // this unit's sums are D's
      const float4* tile = nullptr;
      constexpr long long PART_STEP = 2 * (PART_FLOATS / 4);
      if (joined) {
        // Workspace layout [tile][part][CTA][4 columns][row]: a warp's access covers 512 consecutive bytes.
        const int rest = (unit - sched.full_tiles) % ((sched.total_units - sched.full_tiles) / sched.ksplit);
        const unsigned others = unsigned(sched.ksplit - 1);
        unsigned int* done = parts_done + rest * 2 + cta;
        float4* first = reinterpret_cast<float4*>(parts) + ((long long)rest * sched.ksplit * 2 + cta) * (PART_FLOATS / 4) + quarter * 32 + lane;
        tile = first;
        if (ep_tid == 0) *arrived = *reinterpret_cast<volatile unsigned int*>(done);
        named_barrier_sync(1, 128);
        finish = *arrived == others;
        if (!finish) {
          float4* mine = first + wu.part * PART_STEP;
#pragma unroll 1
          for (int c = 0; c < BN / 32; ++c) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(taddr + c * 32, v);
            tmem_ld_wait();
            if (n0 + c * 32 < N && row < M) {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                mine[(c * 8 + q) * BM] = make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]), __uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3]));
            }
          }
          __threadfence();
          named_barrier_sync(1, 128);  // every thread has also read `arrived`
          if (ep_tid == 0) *arrived = atomicAdd(done, 1u);
          named_barrier_sync(1, 128);
          finish = *arrived == others;
        }
        __threadfence();
        named_barrier_sync(1, 128);  // `arrived` may be written again
      }
      if (finish) {
        const int r_local = quarter * 32 + lane;          // row inside this CTA's 128-row slab
        const uint32_t swz = uint32_t(r_local & 7);
#pragma unroll 1
        for (int c = 0; c < BN / CHUNK_COLS; ++c) {
          const int col = n0 + c * CHUNK_COLS;
          if (col >= N) break;
          const uint32_t buf = staging_base + uint32_t(chunk_counter & 1) * 16384u;
          // the chunk that used this buffer two chunks ago must have been read out by TMA
          if (ep_tid == 0) tma_store_wait_read<1>();
          named_barrier_sync(1, 128);
          const uint32_t row_base = buf + uint32_t(r_local) * 128u;
#pragma unroll
          for (int h = 0; h < CHUNK_COLS / 32; ++h) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(taddr + c * CHUNK_COLS + h * 32, v);
            tmem_ld_wait();
            if (joined && row < M && col + h * 32 < N) {  // the parts in their order, whoever is last
              float s[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) s[j] = 0.f;
#pragma unroll 1
              for (int part = 0; part < sched.ksplit; ++part) {
                if (part == wu.part) {
#pragma unroll
                  for (int j = 0; j < 32; ++j) s[j] += __uint_as_float(v[j]);
                } else {
                  float4 t[8];
#pragma unroll
                  for (int q = 0; q < 8; ++q) t[q] = __ldcg(tile + part * PART_STEP + ((c * (CHUNK_COLS / 32) + h) * 8 + q) * BM);
#pragma unroll
                  for (int q = 0; q < 8; ++q) s[4 * q] += t[q].x, s[4 * q + 1] += t[q].y, s[4 * q + 2] += t[q].z, s[4 * q + 3] += t[q].w;
                }
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(s[j]);
            }
            float f[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]) * alpha;
            if (add_bias) {
              if (OUT_F32) {
                const float* b = reinterpret_cast<const float*>(bias_ptr) + col + h * 32;
#pragma unroll
                for (int j = 0; j < 32; ++j) f[j] += (col + h * 32 + j < N) ? b[j] : 0.f;
              } else {
                const uint16_t* b = reinterpret_cast<const uint16_t*>(bias_ptr) + col + h * 32;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  const uint16_t hb = (col + h * 32 + j < N) ? b[j] : uint16_t(0);
                  f[j] += fmt == 1u ? __bfloat162float(__ushort_as_bfloat16(hb)) : __half2float(__ushort_as_half(hb));
                }
              }
            }
            if (ACCUM && pushing && row < M) {  // the sum itself is stored: fetch what D holds
              const int c0 = col + h * 32;
              if (OUT_F32) {
                const float* old = reinterpret_cast<const float*>(d_ptr) + (long long)row * ldd + c0;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                  if (c0 + 4 * q + 4 <= N) {
                    const float4 o4 = *reinterpret_cast<const float4*>(old + 4 * q);
                    f[4 * q] += o4.x; f[4 * q + 1] += o4.y; f[4 * q + 2] += o4.z; f[4 * q + 3] += o4.w;
                  } else {
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                      if (c0 + 4 * q + t < N) f[4 * q + t] += old[4 * q + t];
                  }
                }
              } else {
                const uint16_t* old = reinterpret_cast<const uint16_t*>(d_ptr) + (long long)row * ldd + c0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  if (c0 + 8 * q + 8 <= N) {
                    const uint4 o4 = *reinterpret_cast<const uint4*>(old + 8 * q);
                    const uint32_t w[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                      const uint16_t lo = uint16_t(w[t] & 0xffffu), hi = uint16_t(w[t] >> 16);
                      f[8 * q + 2 * t] += fmt == 1u ? __bfloat162float(__ushort_as_bfloat16(lo)) : __half2float(__ushort_as_half(lo));
                      f[8 * q + 2 * t + 1] += fmt == 1u ? __bfloat162float(__ushort_as_bfloat16(hi)) : __half2float(__ushort_as_half(hi));
                    }
                  } else {
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                      if (c0 + 8 * q + t < N) f[8 * q + t] += fmt == 1u ? __bfloat162float(__ushort_as_bfloat16(old[8 * q + t])) : __half2float(__ushort_as_half(old[8 * q + t]));
                  }
                }
              }
            }
            if (OUT_F32) {
#pragma unroll
              for (int q = 0; q < 8; ++q) {  // eight 16-byte vectors = the whole 128-byte row
                const uint32_t dst = row_base + ((uint32_t(q) ^ swz) << 4);
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(f[4 * q]), "f"(f[4 * q + 1]), "f"(f[4 * q + 2]), "f"(f[4 * q + 3]) : "memory");
              }
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q) {  // four 16-byte vectors = this half of the row
                uint32_t p0, p1, p2, p3;
                if (fmt == 1u) {
                  p0 = pack_bf16x2(f[8 * q], f[8 * q + 1]); p1 = pack_bf16x2(f[8 * q + 2], f[8 * q + 3]);
                  p2 = pack_bf16x2(f[8 * q + 4], f[8 * q + 5]); p3 = pack_bf16x2(f[8 * q + 6], f[8 * q + 7]);
                } else {
                  p0 = pack_f16x2(f[8 * q], f[8 * q + 1]); p1 = pack_f16x2(f[8 * q + 2], f[8 * q + 3]);
                  p2 = pack_f16x2(f[8 * q + 4], f[8 * q + 5]); p3 = pack_f16x2(f[8 * q + 6], f[8 * q + 7]);
                }
                const uint32_t dst = row_base + ((uint32_t(h * 4 + q) ^ swz) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(p0), "r"(p1), "r"(p2), "r"(p3) : "memory");
              }
            }
          }
          fence_proxy_async_smem();
          named_barrier_sync(1, 128);
          if (ep_tid == 0) {
            if ((ACCUM && !pushing) || (wu.partial && !joined)) tma_reduce_add_2d(&tmap_d, buf, col, row0);
            else tma_store_2d(&tmap_d, buf, col, row0);
            for (int p = 0; p < push.n_peers; ++p) tma_store_2d(&peer_maps.m[p], buf, col, row0);
            tma_store_commit();
          }
          ++chunk_counter;
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_acc_empty[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (ep_tid == 0) tma_store_wait_all();  // every store of this CTA has been performed, the remote ones included
  }

  // ------------------------------------------------------------------ common exit
  if (push.n_peers > 0) signal_peers_when_last(push.done_counter, push.peer_flag, push.n_peers, push.flag_value);
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) {
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) {
      }
      if (status != nullptr && atomicCAS(status, kOk, kErrBarrierTimeout) == kOk) {
        status[1] = 1000000 + blockIdx.x;
        status[2] = M;
        status[3] = N;
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

}  // namespace pair

const char* make_tmap_2d(CUtensorMap* out, const void* ptr, int fmt, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols,
                         uint32_t box_rows);
const char* make_tmap_out(CUtensorMap* out, const void* ptr, int fmt, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols,
                          uint32_t box_rows);

// the workspace begins with two arrival counters per split tile
static size_t parts_offset(int split_tiles) { return (size_t(split_tiles) * 2 * sizeof(unsigned int) + 255) & ~size_t(255); }
static int split_limit(const GemmArgs& g) {  // a pushing launch stores finished sums; partial sums of a K-split tile cannot be pushed
  return !g.split_tail || g.push.n_peers > 0 ? 1 : 4;
}
size_t gemm_pair_workspace(const GemmArgs& g, int num_sms) {
  using namespace pair;
  if (g.variant != 1 || num_sms < 2 || g.M <= 0 || g.N <= 0 || g.K <= 0) return 0;
  const int tiles = ((g.M + 2 * BM - 1) / (2 * BM)) * ((g.N + BN - 1) / BN);
  const Schedule s = make_schedule(g.M, g.N, (g.K + BK - 1) / BK, std::min(tiles, num_sms / 2), split_limit(g), DEFAULT_GROUP_M);
  if (s.ksplit == 1) return 0;
  const int rem = (s.total_units - s.full_tiles) / s.ksplit;
  return parts_offset(rem) + size_t(rem) * s.ksplit * 2 * PART_FLOATS * sizeof(float);
}

template <bool A_MN, bool B_MN, bool OUT_F32, bool ACCUM, bool BIAS>
static cudaError_t launch_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& td, const GemmArgs& g, int num_sms, cudaStream_t stream) {
  using namespace pair;
  auto kern = gemm_tcgen05_pair_kernel<A_MN, B_MN, OUT_F32, ACCUM, BIAS>;
  // function attributes are per device: remember which devices of this process have been set up
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
  }
  const int tiles = ((g.M + 2 * BM - 1) / (2 * BM)) * ((g.N + BN - 1) / BN);
  int pairs = num_sms / 2;
  if (tiles < pairs) pairs = tiles;
  const int max_split = split_limit(g);
  static const int group_m = [] {
    const char* e = getenv("ELF_B200_GEMM_GROUP_M");
    const int v = e ? atoi(e) : DEFAULT_GROUP_M;
    return v >= 1 && v <= 64 ? v : DEFAULT_GROUP_M;
  }();
  const Schedule sched = make_schedule(g.M, g.N, (g.K + BK - 1) / BK, pairs, max_split, group_m);
  float* parts = nullptr;
  if (sched.ksplit > 1 && g.workspace != nullptr) {
    const size_t counters = parts_offset((sched.total_units - sched.full_tiles) / sched.ksplit);
    parts = reinterpret_cast<float*>(static_cast<char*>(g.workspace) + counters);
    if (cudaError_t e = cudaMemsetAsync(g.workspace, 0, counters, stream); e != cudaSuccess) return e;
  } else if (sched.ksplit > 1 && !g.accumulate) {
    // K-split tiles add their partial sums to D, so D must start at zero there.  The split
    // tiles are the last ones of the tile order, all inside the row band that starts at the
    // first row of the group holding the first of them: one memset clears that band (the
    // whole tiles that share it are stored afterwards and simply overwrite the zeros).
    int m, n;
    tile_coords(sched.full_tiles, sched, &m, &n);
    const long long row_start = (long long)(m / group_m) * group_m * 2 * BM;
    const size_t esz = g.out_f32 ? 4 : 2;
    char* base = static_cast<char*>(g.d) + size_t(row_start) * size_t(g.ldd) * esz;
    const size_t rows = size_t(g.M - row_start);
    cudaError_t e = g.ldd == g.N ? cudaMemsetAsync(base, 0, rows * size_t(g.N) * esz, stream)
                                 : cudaMemset2DAsync(base, size_t(g.ldd) * esz, 0, size_t(g.N) * esz, rows, stream);
    if (e != cudaSuccess) return e;
  }
  PeerMaps peers;
  for (int p = 0; p < kMaxPeers; ++p) peers.m[p] = td;  // unused entries stay valid maps
  for (int p = 0; p < g.push.n_peers; ++p) {
    if (make_tmap_out(&peers.m[p], g.push.peer_out[p], g.out_f32 ? 2 : g.fmt, (uint64_t)g.M, (uint64_t)g.N, (uint64_t)g.ldd, g.out_f32 ? 32 : 64, BM) != nullptr)
      return cudaErrorInvalidValue;
  }
  kern<<<2 * pairs, NUM_THREADS, SMEM_BYTES, stream>>>(ta, tb, td, g.d, g.bias, g.M, g.N, g.K, g.ldd, (uint32_t)g.fmt, g.alpha, max_split, group_m, g.status, g.push, peers, parts, static_cast<unsigned int*>(g.workspace));
  flush_bounds_record(g.status, stream);
  return cudaGetLastError();
}

template <bool A_MN, bool B_MN>
static cudaError_t dispatch_pair(const GemmArgs& g, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& td, int num_sms, cudaStream_t s) {
#define ELFB_LAUNCH(F32, ACC, BI) return launch_pair<A_MN, B_MN, F32, ACC, BI>(ta, tb, td, g, num_sms, s)
  if (g.out_f32) {
    if (g.accumulate) { if (g.bias) ELFB_LAUNCH(true, true, true); else ELFB_LAUNCH(true, true, false); }
    else              { if (g.bias) ELFB_LAUNCH(true, false, true); else ELFB_LAUNCH(true, false, false); }
  } else {
    if (g.accumulate) { if (g.bias) ELFB_LAUNCH(false, true, true); else ELFB_LAUNCH(false, true, false); }
    else              { if (g.bias) ELFB_LAUNCH(false, false, true); else ELFB_LAUNCH(false, false, false); }
  }
#undef ELFB_LAUNCH
}

const char* gemm_tcgen05_pair(const GemmArgs& g, int num_sms, cudaStream_t stream) {
  using namespace pair;
  if (g.M <= 0 || g.N <= 0 || g.K <= 0) return nullptr;
  CUtensorMap ta, tb;
  const char* err;
  if (g.a_mn_major) err = make_tmap_2d(&ta, g.a, g.fmt, (uint64_t)g.K, (uint64_t)g.M, (uint64_t)g.lda, 64, BK);
  else              err = make_tmap_2d(&ta, g.a, g.fmt, (uint64_t)g.M, (uint64_t)g.K, (uint64_t)g.lda, BK, BM);
  if (err) return err;
  // each CTA fetches half of the tile's B rows: one 128-row box (K-major) or two 64-wide boxes (MN-major)
  if (g.b_mn_major) err = make_tmap_2d(&tb, g.b, g.fmt, (uint64_t)g.K, (uint64_t)g.N, (uint64_t)g.ldb, 64, BK);
  else              err = make_tmap_2d(&tb, g.b, g.fmt, (uint64_t)g.N, (uint64_t)g.K, (uint64_t)g.ldb, BK, BN / 2);
  if (err) return err;
  const int esz = g.out_f32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(g.d) & 15) != 0 || (g.ldd * esz) % 16 != 0) return "GEMM output must be 16-byte aligned with a 16-byte multiple row pitch";
  // output map for the TMA-store epilogue: 128-byte-wide, 128-row boxes
  CUtensorMap td;
  err = make_tmap_out(&td, g.d, g.out_f32 ? 2 : g.fmt, (uint64_t)g.M, (uint64_t)g.N, (uint64_t)g.ldd, g.out_f32 ? 32 : 64, BM);
  if (err) return err;
  cudaError_t e;
  if (g.a_mn_major && g.b_mn_major) e = dispatch_pair<true, true>(g, ta, tb, td, num_sms, stream);
  else if (!g.a_mn_major && g.b_mn_major) e = dispatch_pair<false, true>(g, ta, tb, td, num_sms, stream);
  else if (!g.a_mn_major && !g.b_mn_major) e = dispatch_pair<false, false>(g, ta, tb, td, num_sms, stream);
  else e = dispatch_pair<true, false>(g, ta, tb, td, num_sms, stream);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace elfb
