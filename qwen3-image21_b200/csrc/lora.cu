// lora.cu — per-request low-rank adapters beside a shared projection (include/b200_lora.h):
//   out = y + scale * (x A^T) B^T
// in one launch.  At ranks of 8 to 128 the operator is bound by HBM: x, y and out are read
// or written once (the adapters are small), so the inner product u = x A^T must not leave
// the chip.
//
// One cluster of C CTAs per 128-row tile of a request.
//   1. CTA c multiplies its part of K: x tiles [128 x 64] and A tiles [rank x 64] arrive by
//      TMA, u_c accumulates in TMEM (tcgen05.mma M128 N=rank).
//   2. The partial sums meet through distributed shared memory: CTA c adds the C partials of
//      its share of the rows in rank order, scales, rounds to bf16, and fetches the other rows
//      (of few rows, each CTA adds up all).
//   3. CTA c walks its part of N in 64-column steps: B tiles and y tiles by TMA, u B^T in
//      TMEM (two accumulators), the epilogue adds y in shared memory and writes whole
//      128-byte row segments.  Rows of another request in the tile are not written.
// C grows as the tiles get fewer, so that small calls still use the whole GPU; the loads of
// step 3 start while step 2 runs.
//
// u is rounded to bf16 because the second product's operands are bf16, as B is.  That is one
// rounding more than the sums need (in all 0.0021 off the 64-bit result where the output's own
// rounding makes 0.0017); the same product as two bf16 GEMMs rounds u in the same place.  Two
// bf16 parts of u would avoid it for twice the second product and 16 or 32 KB of shared memory.
//
// On the GPU: 4 requests of 4096 rows, 4096 -> 12288, rank 64: 177 us, 5.3 TB/s (190 in a
// series of calls on changing inputs); step 1 runs at 4.8 TB/s, step 2 takes 5 us, step 3 runs
// at 6.3 TB/s.  16 ragged requests of 4600 rows in all: 37 us, of which 15 go into set-up,
// first loads and step 2.  4 single rows: 12.9 us, all latency.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "../../include/b200_lora.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kTM = 128;                 // rows of a tile
constexpr int kTK = 64;                  // K per step (one 128-byte swizzle span)
constexpr int kTN = 64;                  // output columns per step
constexpr int kXBytes = kTM * kTK * 2;   // x tile, or y tile: 16 KiB
constexpr int kLThreads = 256;
constexpr uint32_t kLTmemCols = 256;     // u: 128 columns, two accumulators of 64
constexpr uint32_t kAccCol = 128;
constexpr int kMaxStages = 8;
constexpr int kMaxC = 16;
constexpr int kMaxExtent = 1 << 30;      // of K and N
constexpr int kBarBytes = 768;
constexpr int kMaxSmem = 227 * 1024;
// Columns times groups of 4 rows of u up to which every CTA of a cluster adds the partials up
// for itself, which saves one exchange between the CTAs.
constexpr int kDirect = 256;

struct LoraParams {
  const __nv_bfloat16* y;
  __nv_bfloat16* out;
  int64_t ldy, ldo;
  const int32_t* seg_start;
  const int32_t* seg_adapter;
  const float* scale;
  int32_t rows, segments, adapters, n, k, rank;
  int32_t rp;            // rank rounded up to 16
  int32_t stages, stage_bytes;
  int32_t C;             // CTAs of a cluster
  int32_t* status;
};

__device__ __forceinline__ uint32_t lora_rank_in_cluster() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void lora_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
  return r;
}

__device__ __forceinline__ float4 peer_ld_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ uint4 peer_ld_16b(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Arrive on the barrier at this offset in CTA `cta`, releasing at cluster scope.
__device__ __forceinline__ void peer_arrive(uint64_t* bar, uint32_t cta) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(peer_addr(bar, cta))
               : "memory");
}

__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// mbar_wait for barriers that other CTAs of the cluster arrive on.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const uint64_t t0 = global_timer_ns();
  for (uint32_t i = 1; !try_wait_cluster(bar, parity); ++i)
    if ((i & 255u) == 0 && (*abort_flag || global_timer_ns() - t0 > kWaitLimitNs)) return false;
  return true;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int32_t c0,
                                            int32_t c1, int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

__device__ __forceinline__ uint32_t lora_pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// The barrier of the four epilogue warps.  It has no limit, so every path of theirs passes the
// same ones: whether a wait of theirs ran out decides about the work between, never about a
// barrier.
__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// The same barrier; true if `ok` holds in all of its threads.
__device__ __forceinline__ bool epi_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(ok ? 1u : 0u)
      : "memory");
  return all != 0;
}

// The adapter and rows of tile `tile`; all lanes of one warp call it.  Returns the number of
// rows, 0 when there is no such tile.
__device__ __forceinline__ int find_tile(const LoraParams& p, int tile, int lane, int& adapter, int& row0) {
  int before = 0;
  for (int s0 = 0; s0 < p.segments; s0 += 32) {
    const int s = s0 + lane;
    int lo = 0, len = 0, mine_adapter = -1;
    if (s < p.segments) {
      mine_adapter = p.seg_adapter[s];
      lo = min(max(p.seg_start[s], 0), p.rows);
      len = max(min(p.seg_start[s + 1], p.rows) - lo, 0);
    }
    const int mine = (len + kTM - 1) / kTM;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const int all = __shfl_sync(0xffffffffu, sum, 31);
    if (tile < before + all) {
      const unsigned hit = __ballot_sync(0xffffffffu, tile < before + sum);
      const int who = __ffs(hit) - 1;
      const int skip = tile - before - (__shfl_sync(0xffffffffu, sum - mine, who));
      const int base = __shfl_sync(0xffffffffu, lo, who), rows = __shfl_sync(0xffffffffu, len, who);
      adapter = __shfl_sync(0xffffffffu, mine_adapter, who);
      row0 = base + skip * kTM;
      return min(kTM, rows - skip * kTM);
    }
    before += all;
  }
  return 0;
}

// Rows [row, row + 4) of one column of u: the C partials, loaded together (a remote load takes
// about half a microsecond) and added in rank order.
template <int kMost>
__device__ __forceinline__ float4 sum_partials(const uint32_t (&at)[kMost], int C) {
  float4 v[kMost];
#pragma unroll
  for (int c = 0; c < kMost; ++c) v[c] = peer_ld_f32x4(at[c]);
  float4 sum = v[0];
#pragma unroll
  for (int c = 1; c < kMost; ++c)
    if (c < C) {
      sum.x += v[c].x;
      sum.y += v[c].y;
      sum.z += v[c].z;
      sum.w += v[c].w;
    }
  return sum;
}

__global__ void __launch_bounds__(kLThreads, 2)
    lora_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_a,
                const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_y,
                const LoraParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* u_buf = ring + p.stages * p.stage_bytes;  // bf16 u, K-major, 128-byte swizzle
  const int u_regions = p.rp > 64 ? 2 : 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(u_buf + u_regions * kXBytes);
  uint64_t* full = bars;                      // [kMaxStages]
  uint64_t* empty = bars + kMaxStages;        // [kMaxStages] step 1: the MMAs are done
  uint64_t* empty2 = bars + 2 * kMaxStages;   // [kMaxStages] step 3: the epilogue is done
  uint64_t* u_full = bars + 3 * kMaxStages;   // partial u in TMEM
  uint64_t* u_ready = u_full + 1;             // bf16 u in u_buf
  uint64_t* acc_full = u_full + 2;            // [2]
  uint64_t* acc_empty = u_full + 4;           // [2]
  uint64_t* part_ready = u_full + 6;          // every CTA's partials are written
  uint64_t* slice_ready = u_full + 7;         // every CTA's rows are reduced (and partials read)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(u_full + 8);
  int* tile_word = reinterpret_cast<int*>(u_full + 9);  // [3]: rows, adapter, first row
  volatile int* abort_flag = tile_word + 3;
  int* k_from = tile_word + 4;        // [C + 1]: first step of K of each CTA
  int* quad_from = k_from + kMaxC + 1;   // [C + 1]: first group of 4 rows that each CTA adds up
  int* quad_of = quad_from + kMaxC + 1;  // [32]: the CTA of each group

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = p.C;
  const int rank = C > 1 ? static_cast<int>(lora_rank_in_cluster()) : 0;
  const int NS = p.stages;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
      mbar_init(empty2 + s, 4);
    }
    mbar_init(u_full, 1);
    mbar_init(u_ready, 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, 4);
    }
    mbar_init(part_ready, C);
    mbar_init(slice_ready, C);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  const int nkb = (p.k + kTK - 1) / kTK, nnb = (p.n + kTN - 1) / kTN;  // steps (K, N <= 2^30: 16
  if (threadIdx.x >= 128 && threadIdx.x <= 128 + C) {                  // times them fit 32 bits)
    const int c = threadIdx.x - 128, q0 = kTM / 4 * c / C;
    k_from[c] = nkb * c / C;
    quad_from[c] = q0;
    if (c < C)
      for (int q = q0; q < kTM / 4 * (c + 1) / C; ++q) quad_of[q] = c;
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, kLTmemCols);
    tmem_relinquish();
  }
  if (warp == 3) {
    int of = -1, first = 0;
    const int n = find_tile(p, blockIdx.x / C, lane, of, first);
    if (lane == 0) {
      tile_word[0] = n;
      tile_word[1] = of;
      tile_word[2] = first;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int rows = tile_word[0], row0 = tile_word[2];
  int adapter = rows > 0 ? tile_word[1] : -1;
  if (adapter >= p.adapters) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, B200_LORA_STATUS_BAD_ADAPTER);
    adapter = -1;
  }
  // This CTA's part of K and of N (the same for every tile)
  const int nk = k_from[rank + 1] - k_from[rank];
  const int n_first = nnb * rank / C;
  const int nb = nnb * (rank + 1) / C - n_first;

  if (adapter < 0) {  // the whole cluster: nothing to add (rows of y are copied to out)
    if (rows > 0 && p.out != p.y) {
      const int c0 = n_first * kTN, c1 = min((n_first + nb) * kTN, p.n);
      for (int r = warp; r < rows; r += kLThreads / 32) {
        const __nv_bfloat16* from = p.y + static_cast<int64_t>(row0 + r) * p.ldy;
        __nv_bfloat16* to = p.out + static_cast<int64_t>(row0 + r) * p.ldo;
#pragma unroll 4
        for (int c = c0 + lane * 8; c < c1; c += 256)
          *reinterpret_cast<uint4*>(to + c) = *reinterpret_cast<const uint4*>(from + c);
      }
    }
    __syncthreads();
    if (warp == 2) tmem_dealloc(tmem_base, kLTmemCols);
    return;
  }
  if (C > 1) lora_cluster_sync();  // every CTA's barriers are ready for remote arrivals

  const uint32_t a_bytes = p.rp * kTK * 2;
  const uint32_t b_bytes = u_regions * kTN * kTK * 2;
  // The partial sums, f32 [rp][128 rows], lie in the one or two ring stages that step 3
  // fills last in its first round: stages (nk + NS - nx + i) % NS of a CTA with nk steps, with
  // per_stage columns in each.
  const int per_stage = p.stage_bytes / (kTM * 4);
  const int nx = C == 1 ? 0 : p.rp > per_stage ? 2 : 1;
  const int steps0 = nkb / C, stage0 = (steps0 + NS - nx) % NS;  // of a CTA with steps0
  auto part_at = [&](int steps, int col) {  // this CTA's address of a column of partials
    const int second = col >= per_stage ? 1 : 0;
    int st = stage0 + (steps - steps0) + second;  // steps is steps0 or one more
    if (st >= NS) st -= NS;
    return reinterpret_cast<float*>(ring + st * p.stage_bytes) + (col - second * per_stage) * kTM;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_x);
      tma_prefetch_desc(&tm_a);
      tma_prefetch_desc(&tm_b);
      tma_prefetch_desc(&tm_y);
      int it = 0;
      bool ok = true;
      const int kb0 = k_from[rank];
      for (; it < nk; ++it) {
        const int s = it % NS;
        if (!mbar_wait(empty + s, ((it / NS) & 1) ^ 1, abort_flag)) {
          ok = false;
          break;
        }
        uint8_t* dst = ring + s * p.stage_bytes;
        mbar_expect_tx(full + s, kXBytes + a_bytes);
        tma_load_2d(dst, &tm_x, full + s, (kb0 + it) * kTK, row0);
        tma_load_3d(dst + kXBytes, &tm_a, full + s, (kb0 + it) * kTK, 0, adapter);
      }
      for (int i = 0; i < nb && ok; ++i, ++it) {
        const int s = it % NS;
        // first round: the stage's last use was in step 1; later: the epilogue has left it
        ok = i < NS ? mbar_wait(empty + s, ((it / NS) & 1) ^ 1, abort_flag)
                    : mbar_wait(empty2 + s, ((i / NS) & 1) ^ 1, abort_flag);
        if (ok && i < NS && i >= NS - nx) ok = wait_cluster(slice_ready, 0, abort_flag);
        if (!ok) break;
        uint8_t* dst = ring + s * p.stage_bytes;
        const int n0 = (n_first + i) * kTN;
        mbar_expect_tx(full + s, kXBytes + b_bytes);
        for (int r = 0; r < u_regions; ++r)
          tma_load_3d(dst + kXBytes + r * kTN * kTK * 2, &tm_b, full + s, r * kTK, n0, adapter);
        tma_load_2d(dst, &tm_y, full + s, n0, row0);
      }
      if (!ok) {
        *abort_flag = 1;
        if (p.status) atomicCAS(p.status, 0, 1);
        for (int j = max(it - NS, 0); j < it; ++j)  // copies in flight land first
          mbar_wait(full + j % NS, (j / NS) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t idesc_u = idesc_bf16_f32(kTM, p.rp, 0, 0);
      constexpr uint32_t idesc_y = idesc_bf16_f32(kTM, kTN, 0, 0);
      const uint64_t d0 = smem_desc(smem_addr(ring), 16, 1024);
      const uint32_t hi = static_cast<uint32_t>(d0 >> 32), lo0 = static_cast<uint32_t>(d0);
      const uint32_t lo_u = static_cast<uint32_t>(smem_desc(smem_addr(u_buf), 16, 1024));
      bool ok = true;
      int it = 0;
      for (; it < nk; ++it) {
        const int s = it % NS;
        if (!mbar_wait(full + s, (it / NS) & 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = lo0 + ((s * p.stage_bytes) >> 4), b = a + (kXBytes >> 4);
        mma_ss_off<0, 0>(tmem_base, a, hi, b, hi, idesc_u, it > 0 ? 1u : 0u);
        mma_ss_off<2, 2>(tmem_base, a, hi, b, hi, idesc_u, 1u);
        mma_ss_off<4, 4>(tmem_base, a, hi, b, hi, idesc_u, 1u);
        mma_ss_off<6, 6>(tmem_base, a, hi, b, hi, idesc_u, 1u);
        mma_commit(empty + s);
      }
      if (ok) mma_commit(u_full);
      if (ok) ok = mbar_wait(u_ready, 0, abort_flag);
      tc_fence_after();
      for (int i = 0; i < nb && ok; ++i, ++it) {
        const int s = it % NS;
        if (!mbar_wait(full + s, (it / NS) & 1, abort_flag) ||
            !mbar_wait(acc_empty + (i & 1), ((i >> 1) & 1) ^ 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + kAccCol + (i & 1) * kTN;
        const uint32_t b = lo0 + ((s * p.stage_bytes + kXBytes) >> 4);
        for (int kk = 0; kk < p.rp / 16; ++kk) {  // 16 of the rank: 32 bytes of the span
          const uint32_t in = (kk & 3) * 2;
          const uint32_t ao = lo_u + (kk >> 2) * (kXBytes >> 4) + in;
          const uint32_t bo = b + (kk >> 2) * ((kTN * kTK * 2) >> 4) + in;
          mma_ss_off<0, 0>(d, ao, hi, bo, hi, idesc_y, kk > 0 ? 1u : 0u);
        }
        mma_commit(acc_full + (i & 1));
      }
      if (!ok) {
        *abort_flag = 1;
        if (p.status) atomicCAS(p.status, 0, 2);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3;
    const int tr = q * 32 + lane;  // row of the tile = TMEM lane
    const int mine = rows - q * 32;  // rows of this warp; <= 0: it only keeps the barriers going
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    const float scale = p.scale ? p.scale[adapter] : 1.f;
    bool ok = mbar_wait(u_full, 0, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    // u, 16 columns at a time; a CTA without any part of K has zeros.  Columns from the rank on
    // are made zeros below: A has zeros there, but an infinity in x makes them NaN.
    auto u_cols = [&](int c, uint32_t (&r)[16]) {
      if (nk > 0) {
        tmem_ld16(tmem_base + lane_off + c, r);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = 0;
      }
    };
    // 16-byte chunk j (8 of the rank) of row r in u_buf
    auto u_chunk = [&](int r, int j) { return u_buf + (j >> 3) * kXBytes + r * 128 + (((j & 7) ^ (r & 7)) << 4); };
    if (C == 1) {
      for (int c = 0; c < p.rp && mine > 0 && ok; c += 16) {
        uint32_t r[16];
        u_cols(c, r);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = lora_pack(__uint_as_float(r[8 * j + 2 * e]) * scale, __uint_as_float(r[8 * j + 2 * e + 1]) * scale);
          *reinterpret_cast<uint4*>(u_chunk(tr, c / 8 + j)) =
              c + 8 * j < p.rank ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(0, 0, 0, 0);
        }
      }
    } else {
      for (int c = 0; c < p.rp && mine > 0 && ok; c += 16) {
        uint32_t r[16];
        u_cols(c, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) part_at(nk, c + i)[tr] = __uint_as_float(r[i]);
      }
      fence_proxy_async();  // the ring stages under the partials are TMA targets again later
      ok = epi_all(ok);
      const int e = threadIdx.x - 128;
      if (ok) {  // else the other CTAs' waits for this one's partials run out too
        if (e < C) peer_arrive(part_ready, e);
        ok = __all_sync(0xffffffffu, wait_cluster(part_ready, 0, abort_flag));
      }
      // Sums of `quads` groups of 4 rows from row `from` on, one column of one group at a
      // time: U of them in flight.
      auto reduce = [&](auto c_tag, int from, int quads) {
        constexpr int CC = decltype(c_tag)::value, U = CC >= 8 ? 1 : 8 / CC;
        const int units = p.rp * quads;
        for (int i0 = e; ok && i0 < units; i0 += 128 * U) {
          float4 sum[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int i = min(i0 + 128 * u, units - 1), col = i / quads, r = from + (i % quads) * 4;
            uint32_t at[CC];
#pragma unroll
            for (int c = 0; c < CC; ++c) {
              const int from_c = c < C ? c : 0;  // past the last CTA: read, not added
              at[c] = peer_addr(part_at(k_from[from_c + 1] - k_from[from_c], col) + r, from_c);
            }
            sum[u] = sum_partials<CC>(at, C);
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int i = i0 + 128 * u, col = i / quads, r = from + (i % quads) * 4;
            if (i >= units) break;
            const float s4[4] = {sum[u].x, sum[u].y, sum[u].z, sum[u].w};
#pragma unroll
            for (int z = 0; z < 4; ++z)
              reinterpret_cast<__nv_bfloat16*>(u_chunk(r + z, col >> 3))[col & 7] =
                  __float2bfloat16_rn(col < p.rank ? s4[z] * scale : 0.f);
          }
        }
      };
      auto reduce_rows = [&](int from, int quads) {
        if (C <= 2) reduce(std::integral_constant<int, 2>(), from, quads);
        else if (C <= 4) reduce(std::integral_constant<int, 4>(), from, quads);
        else if (C <= 8) reduce(std::integral_constant<int, 8>(), from, quads);
        else reduce(std::integral_constant<int, 16>(), from, quads);
      };
      const int quads = (rows + 3) / 4;
      if (quads * p.rp <= kDirect) {  // few rows: every CTA adds them all up for itself
        reduce_rows(0, quads);
        epi_sync();
        if (e < C) peer_arrive(slice_ready, e);
      } else {                        // its own share, then the others' from them
        reduce_rows(quad_from[rank] * 4, min(quad_from[rank + 1], quads) - quad_from[rank]);
        epi_sync();
        if (e < C) peer_arrive(slice_ready, e);
        ok = __all_sync(0xffffffffu, ok && wait_cluster(slice_ready, 0, abort_flag));
        const int chunks = p.rp / 8, all = rows * chunks;
        for (int i0 = e; ok && i0 < all; i0 += 128 * 4) {
          uint4 v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int i = min(i0 + 128 * u, all - 1), r = i / chunks;
            v[u] = peer_ld_16b(peer_addr(u_chunk(r, i % chunks), quad_of[r / 4]));
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int i = i0 + 128 * u, r = i / chunks;
            if (i < all && quad_of[r / 4] != rank) *reinterpret_cast<uint4*>(u_chunk(r, i % chunks)) = v[u];
          }
        }
      }
    }
    fence_proxy_async();
    tc_fence_before();
    mbar_arrive(u_ready);
    int it = nk;
    for (int i = 0; i < nb && ok; ++i, ++it) {
      const int s = it % NS;
      ok = mbar_wait(full + s, (it / NS) & 1, abort_flag) &&
           mbar_wait(acc_full + (i & 1), (i >> 1) & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint8_t* yt = ring + s * p.stage_bytes;
      uint4* yrow = reinterpret_cast<uint4*>(yt + tr * 128);
      if (mine > 0) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t r[32];
          tmem_ld32(tmem_base + kAccCol + lane_off + (i & 1) * kTN + half * 32, r);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4* at = yrow + ((half * 4 + j) ^ (tr & 7));
            const uint4 v = *at;
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            uint32_t o[4];
#pragma unroll
            for (int z = 0; z < 4; ++z)
              o[z] = lora_pack(__uint_as_float(w[z] << 16) + __uint_as_float(r[8 * j + 2 * z]),
                               __uint_as_float(w[z] & 0xffff0000u) + __uint_as_float(r[8 * j + 2 * z + 1]));
            *at = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty + (i & 1));
      // this warp's rows: 4 rows of 128 bytes per pass
      const int col = (n_first + i) * kTN + (lane & 7) * 8;
      auto store4 = [&](int pass) {
        const int rr = q * 32 + pass * 4 + (lane >> 3);
        const uint4 v = reinterpret_cast<const uint4*>(yt)[rr * 8 + ((lane & 7) ^ (rr & 7))];
        if (rr < rows && col < p.n)
          *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(row0 + rr) * p.ldo + col) = v;
      };
      if (mine >= 32) {
#pragma unroll
        for (int pass = 0; pass < 8; ++pass) store4(pass);
      } else {
        for (int pass = 0; pass * 4 < mine; ++pass) store4(pass);
      }
      if (i + NS < nb) {  // the stage takes another tile: after this warp's plain accesses to it
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(empty2 + s);
      }
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      if (p.status) atomicCAS(p.status, 0, 3);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (C > 1) lora_cluster_sync();  // peers may still read this CTA's rows of u
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kLTmemCols);
  }
}

// ------------------------------------------------------------------ host
PFN_cuTensorMapEncodeTiled_v12000 lora_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// bf16 map of [d2][d1][d0] (d0 dense, rows ld1 elements apart, planes ld2) with a box of
// 64 x box1, 128-byte swizzle, zeros outside.  dims 2 or 3.
int lora_map(CUtensorMap* map, const void* base, int dims, int64_t d0, int64_t d1, int64_t d2, int64_t ld1,
             int64_t ld2, uint32_t box1) {
  auto fn = lora_encode_fn();
  if (!fn) return B200_ERR_CUDA;
  const cuuint64_t size[3] = {static_cast<cuuint64_t>(d0), static_cast<cuuint64_t>(d1),
                              static_cast<cuuint64_t>(d2)};
  const cuuint64_t stride[2] = {static_cast<cuuint64_t>(ld1) * 2, static_cast<cuuint64_t>(ld2) * 2};
  const cuuint32_t box[3] = {kTK, box1, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, const_cast<void*>(base), size, stride, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? B200_OK
             : B200_ERR_CUDA;
}

// The same values on every call: threads that launch at the same time do not disturb each
// other.
int lora_attributes() {
  if (cudaFuncSetAttribute(lora_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) == cudaSuccess &&
      cudaFuncSetAttribute(lora_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess)
    return B200_OK;
  cudaGetLastError();
  return B200_ERR_CUDA;
}

// Clusters of C CTAs that the current device runs at once (clusters do not straddle its GPU
// clusters, so this is less than the CTAs that fit / C).  The occupancy query counts one CTA
// per SM for a kernel with tensor memory; with its 256 of the SM's 512 columns, two run
// wherever shared memory holds two.  A property of the kernel and the device, asked for once.
constexpr int kTwoPerSm = 113 * 1024;  // dynamic shared memory of which an SM holds two
int active_clusters(int C, int smem) {
  static std::mutex lock;
  static int known[64][2][kMaxC + 1] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> hold(lock);
  int& n = known[dev][smem > kTwoPerSm ? 1 : 0][C];
  if (n == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(C);
    cfg.blockDim = dim3(kLThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, lora_kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    if (smem <= kTwoPerSm) n *= 2;
  }
  return n;
}

bool lora_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether writing `out` (rows of n, ldo apart) can disturb reads of `in` (rows of cols, ldi
// apart) that are still to come.  Column ranges of one buffer that keep apart do not.  With
// same_row, a row's own writes may hit its own reads: the whole cluster has read its rows of x
// before any of it writes.
bool lora_disturbs(const void* out, int64_t ldo, int64_t n, const void* in, int64_t ldi, int64_t cols,
                   int64_t rows, bool same_row) {
  using wide = __int128;
  const wide o = reinterpret_cast<uintptr_t>(out) / 2, i = reinterpret_cast<uintptr_t>(in) / 2;
  if (o + wide(rows - 1) * ldo + n <= i || i + wide(rows - 1) * ldi + cols <= o) return false;
  if (rows == 1) return !same_row;
  if (ldo != ldi) return true;
  // row r of out starts m elements behind the start of row r + q of in
  const wide d = o - i;
  const wide q = d >= 0 ? d / ldi : -((-d + ldi - 1) / ldi);
  const wide m = d - q * ldi;
  const bool meets = m < cols, meets_next = m + n > ldi;  // row r + q, row r + q + 1
  return same_row ? (meets && q != 0) || (meets_next && q != -1) : meets || meets_next;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_lora_add(const void* x, int64_t ldx, const void* a, const void* b, const void* y,
                             int64_t ldy, void* out, int64_t ldo, const int32_t* seg_start,
                             const int32_t* seg_adapter, const float* scale, int32_t rows,
                             int32_t segments, int32_t adapters, int32_t n, int32_t k, int32_t rank,
                             int32_t* status, b200_stream_t stream) {
  if (rows < 0 || segments < 0 || adapters < 0 || n < 0) return B200_ERR_INVALID;
  if (k <= 0 || k > kMaxExtent || n > kMaxExtent || k % 8 != 0 || n % 8 != 0 || rank <= 0 || rank % 8 != 0 || rank > B200_LORA_MAX_RANK)
    return B200_ERR_INVALID;
  if (rows == 0 || segments == 0 || n == 0) return B200_OK;
  if (!x || !y || !out || !seg_start || !seg_adapter || (adapters > 0 && (!a || !b)))
    return B200_ERR_INVALID;
  const void* ptrs[] = {x, a, b, y, out};
  for (const void* ptr : ptrs)
    if (!lora_al16(ptr)) return B200_ERR_INVALID;
  if (ldx < k || ldy < n || ldo < n || ldx % 8 != 0 || ldy % 8 != 0 || ldo % 8 != 0) return B200_ERR_INVALID;
  if (out == y && ldo != ldy) return B200_ERR_INVALID;
  if (out != y && lora_disturbs(out, ldo, n, y, ldy, n, rows, false)) return B200_ERR_INVALID;
  if (lora_disturbs(out, ldo, n, x, ldx, k, rows, true)) return B200_ERR_INVALID;
  LoraParams p{};
  p.y = static_cast<const __nv_bfloat16*>(y);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldy = ldy;
  p.ldo = ldo;
  p.seg_start = seg_start;
  p.seg_adapter = seg_adapter;
  p.scale = scale;
  p.rows = rows;
  p.segments = segments;
  p.adapters = adapters;
  p.n = n;
  p.k = k;
  p.rank = rank;
  p.rp = (rank + 15) / 16 * 16;
  p.status = status;
  const int regions = p.rp > 64 ? 2 : 1;
  p.stage_bytes = kXBytes + regions * kTN * kTK * 2;
  const auto smem_of = [&](int stages) { return stages * p.stage_bytes + regions * kXBytes + kBarBytes + 1024; };
  // Every request ends in a tile of its own: rows / 128 + segments tiles at most.  The
  // cluster is the largest whose tiles are expected to run all at once, with every request's
  // last tile half full on average.  (16 ragged requests of 4600 rows: 44 expected, and 44
  // clusters of 6 run at once, 30 of 8; 72 us in clusters of 2, 43 of 4, 37 of 6.)
  const int64_t tiles = static_cast<int64_t>(rows) / kTM + std::min(segments, rows);
  const int64_t expect = std::min<int64_t>(tiles, (rows + kTM - 1) / kTM + segments / 2);
  const int steps = std::max((k + kTK - 1) / kTK, (n + kTN - 1) / kTN);
  int rc;
  if ((rc = lora_attributes()) != B200_OK) return rc;
  // The ring: 3 stages with two CTAs per SM, or (rank over 64) 4 with one; where one CTA per
  // SM holds all tiles in clusters as large, the rest of its shared memory too.
  p.stages = regions == 1 ? 3 : 4;
  p.C = std::min(kMaxC, steps);
  while (p.C > 1 && expect > active_clusters(p.C, smem_of(p.stages))) --p.C;
  const int deep = regions == 1 ? 7 : 6;
  if (expect <= active_clusters(p.C, smem_of(deep))) p.stages = deep;
  const int C = p.C, smem = smem_of(p.stages);
  if (tiles * C > 0x7fffffff) return B200_ERR_INVALID;
  CUtensorMap mx{}, ma{}, mb{}, my{};
  if ((rc = lora_map(&mx, x, 2, k, rows, 1, ldx, 0, kTM)) != B200_OK) return rc;
  if ((rc = lora_map(&my, y, 2, n, rows, 1, ldy, 0, kTM)) != B200_OK) return rc;
  if (adapters > 0) {
    if ((rc = lora_map(&ma, a, 3, k, rank, adapters, k, static_cast<int64_t>(rank) * k, p.rp)) != B200_OK) return rc;
    if ((rc = lora_map(&mb, b, 3, rank, n, adapters, rank, static_cast<int64_t>(rank) * n, kTN)) != B200_OK) return rc;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * C));
  cfg.blockDim = dim3(kLThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, lora_kernel, mx, ma, mb, my, p) != cudaSuccess) {
    cudaGetLastError();
    return B200_ERR_CUDA;
  }
  return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}
