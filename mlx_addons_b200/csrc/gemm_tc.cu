// Products with an epilogue on the tensor cores: D[i, j] = sum_k P[i, k]
// Q[j, k] with 16-bit factors and 32-bit sums (tcgen05.mma kind::f16, operands
// by TMA, accumulators in tensor memory).
//
// A pair of CTAs (two SMs) computes a 256 x 256 tile (cta_group::2): each CTA
// holds 128 rows of P and 128 of Q's 256 in shared memory and 128 x 256 of D
// in its tensor memory. The pairs are persistent, one CTA an SM, and tensor
// memory holds two accumulators, so the epilogue of a tile runs under the MMAs
// of the next. Where D is too small for that, single CTAs compute 128 x BN
// tiles, several to an SM, and k may be split over a cluster of up to 4 of
// them, whose partial sums are joined in order through distributed shared
// memory.
//
// Roles in a CTA: one thread issues the TMA loads (a ring of 64-deep slices),
// one thread (of the leading CTA) issues the MMAs, four or eight warps take
// finished accumulators from tensor memory through the epilogue.
//
// Both axis orders of an operand are read as they lie: with unit stride along
// k ("K-major") and along the rows ("MN-major"), both with 128-byte swizzle.
//
// Split operands: a float32 value is three bf16 planes or, where its range is
// known, two f16 planes; the product is then the sum of the plane pairs whose
// weight is 2^-24 or more (6 of 9, or 3 of 4), smallest first. The tensor
// cores truncate when they add to an accumulator, so such a product's
// accumulator is joined in float32 registers after every slice (JOIN):
// without that the truncations, all towards zero, add up along k. A slice in
// shared memory holds all planes, each loaded once for all its products. One
// plane is joined too, but rarely and over a long k alone (kJoinAfter).
#include <cmath>

#include "b2c_kernels.cuh"
#include "gemm_tile.cuh"

namespace b2c {

__device__ unsigned int g_gemm_fault;

namespace {

// The tensor cores cut off what they add to an accumulator: a sum of terms of one sign loses 9e-8 of itself with every
// 16 products (all-positive bf16 and f16, k = 131,072 in one accumulator: 7.2e-4, more than half a step of f16). So
// one plane, too, is joined in float32 registers every kJoinSlices where an accumulator would take more than kJoinAfter
// slices (8,192 k, up to which it loses 5e-5 at the most, a tenth of half a step of f16). Joining every product takes
// up to 1.1 times as long (8192 x 4096 x 16384 bf16: 695 and 767 us).
constexpr int kJoinAfter = 128, kJoinSlices = 32;

// Warps of a pair's CTA: its epilogue warps, then a warpgroup of loads,
// products and two idle warps. Joined sums stay in registers, 64 a thread with
// sixteen epilogue warps (eight, with 128, took 1.3 times as long over a tile).
template <bool JOIN>
struct Pair {
  static constexpr int EPI = JOIN ? 16 : 8;
  static constexpr int NT = (EPI + 4) * 32;
  // registers where JOIN: 640 x 96 at launch = 128 x 64 + 512 x 104 after the split
  static constexpr int FEW = 64, MANY = 104;
};
// Blocks of staging: one for each epilogue warp, or, with one plane joined over a long k, one for two of them, which take turns
// at the end of a tile, so that the ring holds six slices instead of four (4096 x 32768 x 4096 bf16: 815 and 915 us; 785 without joining).
__host__ __device__ constexpr int pair_staging(int planes) { return planes > 1 ? 16 : 8; }

// ---------------------------------------------------------------------------
// pairs of CTAs
// ---------------------------------------------------------------------------

template <int PLANES, bool JOIN, typename OUT>
__global__ void __launch_bounds__(Pair<JOIN>::NT, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ TcParams p) {
  extern __shared__ unsigned char raw[];
  next_may_launch();
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 5];  // the last: nothing arrives on it
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  constexpr int STAGES = pair_staging(PLANES);
  constexpr int EPI = Pair<JOIN>::EPI, GROUPS = EPI / 4, SLICES = 8 / GROUPS;  // slices: 32 columns of a warp's rows
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  unsigned char* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  float* staging = reinterpret_cast<float*>(ring + p.stages * p.stage_bytes);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, tfull0 = empty0 + 8 * kMaxStages,
                 tempty0 = tfull0 + 16, never = tempty0 + 16;
  const uint64_t limit = p.inject ? 1000000ull : kWaitNs;

  if (tid == 0) {
    gave_up = 0;
    for (int s = 0; s < p.stages; ++s) {
      bar_init(full0 + 8 * s, 1);
      bar_init(empty0 + 8 * s, 1);
    }
    bar_init(never, 1);
    for (int s = 0; s < 2; ++s) {
      bar_init(tfull0 + 8 * s, 1);
      bar_init(tempty0 + 8 * s, EPI * 2);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == EPI) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    fence_before();
  }
  __syncthreads();
  cluster_sync();
  fence_after();
  const uint32_t tmem = tmem_slot;
  previous_done();
  const int64_t first = blockIdx.x / 2, step = gridDim.x / 2;
  volatile int* gu = &gave_up;
  const int per = PLANES > 1 ? 1 : JOIN ? kJoinSlices : p.kblocks;  // slices of one accumulator

  if (warp < EPI) {
    if constexpr (JOIN) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Pair<JOIN>::MANY));
    // ---- epilogue: warps w, w + 4, ... share the rows 32 (w % 4).. and deal out the columns ----
    const int quad = warp & 3, group = warp >> 2;
    const uint32_t lead_tempty0 = map_rank(tempty0, 0);
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    float* stage = staging + warp % STAGES * kStageFloats;
    uint32_t buf = 0, tphase = 0;
    bool ok = true;
    const float bad = __int_as_float(0x7fffffff);
    if (p.inject && blockIdx.x == 0) ok = __all_sync(kFull, bar_wait(never, 0, gu, limit, &g_gemm_fault));
    for (int64_t t = first; t < p.tiles; t += step) {
      const Tile o = tile_at<2>(p, t);
      const int64_t i = o.i + rank * BM + quad * 32;
#pragma unroll
      for (int q = 0; q < SLICES; ++q) prefetch_res(p, o.b, i + lane, o.j + (GROUPS * q + group) * 32);
      if constexpr (JOIN) {
        float acc[SLICES][32];
#pragma unroll
        for (int q = 0; q < SLICES; ++q)
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[q][c] = 0.f;
        for (int kb = 0; kb < p.kblocks; kb += per) {
          ok = __all_sync(kFull, ok && bar_wait(tfull0 + 8 * buf, tphase, gu, limit, &g_gemm_fault));
          fence_after();
#pragma unroll
          for (int q = 0; q < SLICES; ++q) {
            float v[32];
            tmem_row32(lanes + buf * 256 + (GROUPS * q + group) * 32, v);
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[q][c] += v[c];
          }
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive_cluster(lead_tempty0 + 8 * buf);
          if (++buf == 2) buf = 0, tphase ^= 1;
        }
        if (STAGES < EPI && warp >= STAGES) asm volatile("bar.sync 1, %0;" ::"n"(EPI * 32) : "memory");
        // one copy of the epilogue's code: the sums move up instead of the index
#pragma unroll 1
        for (int q = 0; q < SLICES; ++q) {
          if (!ok) {
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[0][c] = bad;
          }
          finish32<OUT>(p, acc[0], o.b, i, o.j + (GROUPS * q + group) * 32, o.mirror, stage, lane);
#pragma unroll
          for (int c = 0; c < 32; ++c)
#pragma unroll
            for (int m = 1; m < SLICES; ++m) acc[m - 1][c] = acc[m][c];
        }
        // the first half of the warps lets the second one in, and stays out until that is done
        if (STAGES < EPI && warp < STAGES) asm volatile("bar.sync 1, %0;" ::"n"(EPI * 32) : "memory");
        if (STAGES < EPI) asm volatile("bar.sync 2, %0;" ::"n"(EPI * 32) : "memory");
      } else {
        ok = __all_sync(kFull, ok && bar_wait(tfull0 + 8 * buf, tphase, gu, limit, &g_gemm_fault));
        fence_after();
        for (int col = group * 32; col < 256; col += GROUPS * 32) {
          float v[32];
          tmem_row32(lanes + buf * 256 + col, v);
          if (col + GROUPS * 32 >= 256) {  // the last of this warp's columns: the accumulator is free
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_cluster(lead_tempty0 + 8 * buf);
          }
          if (!ok) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = bad;
          }
          finish_row32<OUT>(v, p, o.b, i, o.j + col, clamp32(p.I - i), clamp32(p.J - o.j - col), o.mirror,
                            reinterpret_cast<unsigned char*>(stage), lane);
        }
        if (++buf == 2) buf = 0, tphase ^= 1;
      }
    }
  } else {
    if constexpr (JOIN) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Pair<JOIN>::FEW));
    if (warp == EPI) {
      // ---- loads ----
      const bool lead = elect_one();
      const uint32_t lead_full0 = map_rank(full0, 0);
      uint32_t s = 0, phase = 0;
      for (int64_t t = first; t < p.tiles && !*gu; t += step) {
        const Tile o = tile_at<2>(p, t);
        const int i0 = (int)(o.i + rank * BM), j0 = (int)(o.j + rank * p.share);
        const int bp = p.p_bcast ? 0 : (int)o.b, bq = p.q_bcast ? 0 : (int)o.b;
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!bar_wait(empty0 + 8 * s, phase ^ 1, gu, limit, &g_gemm_fault)) break;
          if (lead) {
            if (rank == 0) bar_expect(full0 + 8 * s, 2 * p.stage_bytes);
            load_slice<2, PLANES>(p, &map_p, &map_q, smem_u32(ring + s * p.stage_bytes), i0, j0, kb, bp, bq, lead_full0 + 8 * s);
          }
          if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
        }
      }
    } else if (warp == EPI + 1 && rank == 0) {
      // ---- products ----
      const bool lead = elect_one();
      const Multiplier<2, PLANES> mul(p, smem_u32(ring));
      uint32_t s = 0, phase = 0, buf = 0, tphase = 0;
      for (int64_t t = first; t < p.tiles && !*gu; t += step) {
        for (int k0 = 0; k0 < p.kblocks; k0 += per) {
          if (!bar_wait(tempty0 + 8 * buf, tphase ^ 1, gu, limit, &g_gemm_fault)) break;
          fence_after();
          const int n = p.kblocks - k0 < per ? p.kblocks - k0 : per;
          for (int kb = 0; kb < n; ++kb) {
            if (!bar_wait(full0 + 8 * s, phase, gu, limit, &g_gemm_fault)) break;
            fence_after();
            if (lead) {
              mul.slice(s, tmem + buf * 256, kb == 0);
              commit<2>(empty0 + 8 * s);
            }
            if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
          }
          if (*gu) break;
          if (lead) commit<2>(tfull0 + 8 * buf);
          if (++buf == 2) buf = 0, tphase ^= 1;
        }
      }
    }
  }
  __syncthreads();
  if (gave_up) settle();
  fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == EPI) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---------------------------------------------------------------------------
// single CTAs, one tile each, k split over a cluster
// ---------------------------------------------------------------------------

// JOIN: one CTA an SM with eight epilogue warps, so that a slice's planes fit
// twice; otherwise two CTAs with four.
template <bool JOIN>
struct Solo {
  static constexpr int EPI = JOIN ? 8 : 4;
  static constexpr int NT = (EPI + 2) * 32;
  static constexpr int CTAS = JOIN ? 1 : 2;
  static constexpr int SMEM = JOIN ? kSmemMax - 1024 : 113 * 1024;
};

template <int PLANES, bool JOIN, typename OUT>
__global__ void __launch_bounds__(Solo<JOIN>::NT, Solo<JOIN>::CTAS)
    gemm_solo_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ TcParams p) {
  extern __shared__ unsigned char raw[];
  next_may_launch();
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 5];  // the last: nothing arrives on it
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  constexpr int EPI = Solo<JOIN>::EPI, GROUPS = EPI / 4, SLICES = JOIN ? 4 / GROUPS : 1;
  constexpr int per = PLANES > 1 ? 1 : kJoinSlices;  // slices of one accumulator where JOIN
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = p.split, rank = split > 1 ? (int)cluster_rank() : 0;
  unsigned char* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, tfull0 = empty0 + 8 * kMaxStages,
                 tempty0 = tfull0 + 16, never = tempty0 + 16;
  const uint64_t limit = p.inject ? 1000000ull : kWaitNs;
  const Tile o = tile_at<1>(p, blockIdx.x / split);
  // this CTA's slices of k
  const int kb0 = (int)((int64_t)p.kblocks * rank / split), kb1 = (int)((int64_t)p.kblocks * (rank + 1) / split);

  if (tid == 0) {
    gave_up = 0;
    for (int s = 0; s < p.stages; ++s) {
      bar_init(full0 + 8 * s, 1);
      bar_init(empty0 + 8 * s, 1);
    }
    bar_init(never, 1);
    for (int s = 0; s < 2; ++s) {
      bar_init(tfull0 + 8 * s, 1);
      bar_init(tempty0 + 8 * s, EPI);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == EPI) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(p.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    fence_before();
  }
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  previous_done();
  volatile int* gu = &gave_up;
  const int quad = warp & 3, group = warp >> 2;
  const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
  const int pitch = p.BN + 4;
  float* partial = reinterpret_cast<float*>(ring);  // this CTA's sums of the tile, once the ring is free

  if (warp < EPI) {
    for (int col = group * 32; col < p.BN; col += GROUPS * 32) prefetch_res(p, o.b, o.i + quad * 32 + lane, o.j + col);
    bool ok = true;
    if (p.inject && blockIdx.x == 0) ok = __all_sync(kFull, bar_wait(never, 0, gu, limit, &g_gemm_fault));
    float acc[SLICES][32];
    if constexpr (JOIN) {
#pragma unroll
      for (int q = 0; q < SLICES; ++q)
#pragma unroll
        for (int c = 0; c < 32; ++c) acc[q][c] = 0.f;
      uint32_t buf = 0, tphase = 0;
      for (int kb = kb0; kb < kb1; kb += per) {
        ok = __all_sync(kFull, ok && bar_wait(tfull0 + 8 * buf, tphase, gu, limit, &g_gemm_fault));
        fence_after();
#pragma unroll
        for (int q = 0; q < SLICES; ++q) {
          const int col = (GROUPS * q + group) * 32;
          if (col < p.BN) {
            float v[32];
            tmem_row32(lanes + buf * p.BN + col, v);
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[q][c] += v[c];
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_cluster(tempty0 + 8 * buf);
        if (++buf == 2) buf = 0, tphase ^= 1;
      }
    } else {
      ok = __all_sync(kFull, ok && bar_wait(tfull0, 0, gu, limit, &g_gemm_fault));
      fence_after();
    }
    // every product is done, so the ring is free (after a wait that ran out, once what is
    // still in flight has landed)
    if (!ok) settle();
#pragma unroll
    for (int q = 0; q < (JOIN ? SLICES : 4); ++q) {
      const int col = (GROUPS * q + group) * 32;
      if (col < p.BN) {
        float(&v)[32] = acc[JOIN ? q : 0];
        if constexpr (!JOIN) tmem_row32(lanes + col, v);
        if (!ok) {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = __int_as_float(0x7fffffff);
        }
        float4* at = reinterpret_cast<float4*>(partial + (quad * 32 + lane) * pitch + col);
#pragma unroll
        for (int c = 0; c < 8; ++c) at[c] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
      }
    }
  } else if (warp == EPI) {
    // ---- loads ----
    const bool lead = elect_one();
    uint32_t s = 0, phase = 0;
    const int bp = p.p_bcast ? 0 : (int)o.b, bq = p.q_bcast ? 0 : (int)o.b;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!bar_wait(empty0 + 8 * s, phase ^ 1, gu, limit, &g_gemm_fault)) break;
      if (lead) {
        bar_expect(full0 + 8 * s, p.stage_bytes);
        load_slice<1, PLANES>(p, &map_p, &map_q, smem_u32(ring + s * p.stage_bytes), (int)o.i, (int)o.j, kb, bp, bq,
                              full0 + 8 * s);
      }
      if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
    }
  } else if (warp == EPI + 1) {
    // ---- products ----
    const bool lead = elect_one();
    const Multiplier<1, PLANES> mul(p, smem_u32(ring));
    uint32_t s = 0, phase = 0, buf = 0, tphase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      // an accumulator's first and last slice
      const bool fresh = JOIN ? (kb - kb0) % per == 0 : kb == kb0, done = kb == kb1 - 1 || (JOIN && (kb - kb0) % per == per - 1);
      if (JOIN && fresh && !bar_wait(tempty0 + 8 * buf, tphase ^ 1, gu, limit, &g_gemm_fault)) break;
      if (!bar_wait(full0 + 8 * s, phase, gu, limit, &g_gemm_fault)) break;
      fence_after();
      if (lead) {
        mul.slice(s, tmem + buf * p.BN, fresh);
        commit<1>(empty0 + 8 * s);
        if (done) commit<1>(tfull0 + 8 * buf);
      }
      if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
      if (JOIN && done && ++buf == 2) buf = 0, tphase ^= 1;
    }
  }
  __syncwarp();
  if (split > 1) cluster_sync();
  else __syncthreads();
  // each CTA of the cluster finishes its share of the rows
  const int nrows = BM / split, r0 = rank * nrows;
  const Block mine{o.b, o.i + r0, o.j, partial + r0 * pitch, pitch, 31 - __clz(nrows), 31 - __clz(p.BN)};
  finish<OUT, true, 1>(p, mine, o.mirror, tid, Solo<JOIN>::NT);
  if (o.mirror) {
    __syncthreads();
    mirror_units<OUT>(p, mine, tid, Solo<JOIN>::NT);
  }
  __syncwarp();
  if (split > 1) cluster_sync();  // peers' sums stay until they have been read
  __syncthreads();
  if (gave_up) settle();
  fence_before();
  __syncthreads();
  if (warp == EPI) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols));
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int slices_of_cta(int kblocks, int split) { return (kblocks + split - 1) / split; }

template <typename Kern>
cudaError_t launch_in_clusters(Kern kern, int64_t ctas, int cluster, int threads, size_t smem, cudaStream_t s,
                               const CUtensorMap& mp, const CUtensorMap& mq, const TcParams& p) {
  if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (p.chained) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, mp, mq, p);
}

template <int PLANES, bool JOIN, typename OUT>
cudaError_t launch_pair(const CUtensorMap& mp, const CUtensorMap& mq, TcParams p, int sms, cudaStream_t s) {
  constexpr int NT = Pair<JOIN>::NT;
  const int staging = pair_staging(PLANES) * kStageFloats * 4;
  const int stages = (kSmemMax - 1024 - 512 - staging) / p.stage_bytes;
  p.stages = stages > kMaxStages ? kMaxStages : stages;
  const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + staging;
  auto kern = gemm_pair_kernel<PLANES, JOIN, OUT>;
  static int cache[64];
  int occ = 0;
  cudaError_t e = kernel_occupancy(kern, NT, smem, cache, &occ);
  if (e != cudaSuccess) return e;
  const int64_t want = p.tiles * 2, cap = sms / 2 * 2;
  return launch_in_clusters(kern, want < cap ? want : cap, 2, NT, smem, s, mp, mq, p);
}

template <int PLANES, bool JOIN, typename OUT>
cudaError_t launch_solo(const CUtensorMap& mp, const CUtensorMap& mq, TcParams p, int sms, cudaStream_t s) {
  constexpr int NT = Solo<JOIN>::NT;
  const int sums = BM * (p.BN + 4) * 4;
  const int per = (p.kblocks + p.split - 1) / p.split;
  // all of an SM's shared memory where it gets one CTA anyway: a slice takes about 2,000 clocks to arrive
  const int room = p.tiles * p.split <= sms ? kSmemMax - 1024 : Solo<JOIN>::SMEM;
  int stages = (room - 1024 - 512) / p.stage_bytes;
  if (stages > kMaxStages) stages = kMaxStages;
  p.stages = stages > per ? per : stages;
  size_t smem = (size_t)p.stages * p.stage_bytes;
  if (smem < (size_t)sums) smem = sums;
  smem += 1024;
  p.tmem_cols = 32;
  while (p.tmem_cols < (JOIN ? 2 : 1) * p.BN) p.tmem_cols *= 2;
  auto kern = gemm_solo_kernel<PLANES, JOIN, OUT>;
  static int cache[64];
  int occ = 0;
  cudaError_t e = kernel_occupancy(kern, NT, smem, cache, &occ);
  if (e != cudaSuccess) return e;
  return launch_in_clusters(kern, p.tiles * p.split, p.split, NT, smem, s, mp, mq, p);
}

template <bool PAIR, int PLANES, typename OUT>
cudaError_t launch_form(const CUtensorMap& mp, const CUtensorMap& mq, const TcParams& p, int sms, cudaStream_t s) {
  if (PLANES > 1 || slices_of_cta(p.kblocks, p.split) > kJoinAfter) {
    if constexpr (PAIR) return launch_pair<PLANES, true, OUT>(mp, mq, p, sms, s);
    else return launch_solo<PLANES, true, OUT>(mp, mq, p, sms, s);
  }
  if constexpr (PLANES == 1) {
    if constexpr (PAIR) return launch_pair<PLANES, false, OUT>(mp, mq, p, sms, s);
    else return launch_solo<PLANES, false, OUT>(mp, mq, p, sms, s);
  }
  return cudaErrorInvalidValue;
}

template <bool PAIR>
cudaError_t launch_out(const TcProblem& t, const CUtensorMap& mp, const CUtensorMap& mq, const TcParams& p, int sms,
                       cudaStream_t s) {
  if (t.kind == kOne) {
    if (t.out == B2C_BF16) return launch_form<PAIR, 1, __nv_bfloat16>(mp, mq, p, sms, s);
    if (t.out == B2C_F16) return launch_form<PAIR, 1, __half>(mp, mq, p, sms, s);
    return cudaErrorInvalidValue;
  }
  if (t.kind == kThirds && t.out == B2C_F32) return launch_form<PAIR, 3, float>(mp, mq, p, sms, s);
  if (t.kind == kHalves && t.out == B2C_F32) return launch_form<PAIR, 2, float>(mp, mq, p, sms, s);
  if (t.kind == kHalves && t.out == B2C_F16) return launch_form<PAIR, 2, __half>(mp, mq, p, sms, s);
  if (t.kind == kHalves && t.out == kOutHalves) return launch_form<PAIR, 2, Halves>(mp, mq, p, sms, s);
  return cudaErrorInvalidValue;
}

// The form of a product: pairs, or single CTAs with BN columns and k split
// over `split` of them.
struct Form {
  int pair, BN, split;
  double clocks;
};

// Estimated clocks: waves of CTAs times their slices of k, each the longest of
// its arrival (500 clocks with a full ring), its load (L2 gives an SM up to
// 100 bytes a clock and all of them 6,000) and its products (4096 a clock, and
// 128 bytes of shared memory a clock), plus what a CTA costs beside them. Fitted to
// sweeps of these forms; measured, us, the first of each the choice:
//   16 x 4096 x 16384 f16       32 columns 37, split 2 38, 4 48, 64 columns 39
//   16 x 8192 x 8192 bf16       32 columns split 2 36, 1 51, 4 39, 8 48
//   512 x 2048 x 512 bf16       64 columns split 4 11, 2 13, 1 17, pairs 20
//   1000 x 777 x 1301 float32   128 columns 28, split 2 38, 64 columns 46, pairs 69
//   2048 x 2048 x 2048 bf16     pairs 22, 128 columns 25, 64 columns 37
Form choose_form(const TcProblem& t, int kblocks, int planes, int nseg, int sms) {
  Form best{0, 0, 0, 1e300};
  const int64_t ti = (t.I + BM - 1) / BM;
  auto rate = [&](double ctas) { return fmin(100.0, 6000.0 / fmin(ctas, (double)sms)); };
  for (int BN = t.sym ? 128 : 32; BN <= 128; BN *= 2) {
    if (!t.sym && BN > 32 && BN / 2 >= t.J) break;
    const int64_t tj = (t.J + BN - 1) / BN, tiles = t.batch * (t.sym ? ti * (ti + 1) / 2 : ti * tj);
    for (int split = 1; split <= 4 && split <= kblocks; split *= 2) {
      const double ctas = (double)tiles * split, on_sm = ceil(ctas / sms), at_once = fmin(on_sm, planes > 1 || slices_of_cta(kblocks, split) > kJoinAfter ? 1.0 : 2.0);
      const double load = planes * (16384.0 + BN * 128.0) / rate(ctas), mul = nseg * 4.0 * fmax(BN / 2.0, (128 + BN) / 4.0);
      const double slice = fmax(500.0, at_once * fmax(load, mul));
      const double c = ceil(on_sm / at_once) * ((kblocks + split - 1) / split * slice + 8000 + BN * 20) +
                       (split > 2 ? 4000 : split > 1 ? 1500 : 0);
      if (c < best.clocks) best = Form{0, BN, split, c};
    }
  }
  if (t.I > BM && t.J > 128) {
    const int64_t ti2 = (t.I + 255) / 256, tj2 = (t.J + 255) / 256;
    const int64_t tiles = t.batch * (t.sym ? ti2 * (ti2 + 1) / 2 : ti2 * tj2);
    // with two planes the ring holds two slices, with three one: their arrival is hardly hidden
    const double slice = planes > 1 ? planes * 2000.0 : fmax(32768.0 / rate(2.0 * tiles), 4.0 * 128);
    const double c = ceil(2.0 * tiles / sms) * kblocks * slice + 11000;
    if (c < best.clocks) best = Form{1, 256, 1, c};
  }
  return best;
}

}  // namespace

bool tc_direct(const GemmOperand& o, int64_t batch, int64_t rows, int64_t K, TcOperand* out) {
  if ((reinterpret_cast<uintptr_t>(o.p) & 15) != 0) return false;
  TcOperand r{};
  r.p = o.p;
  r.bcast = batch == 1 || o.bs == 0;
  r.batch_stride = o.bs;
  if (!r.bcast && (o.bs % 8 != 0 || o.bs >= ((int64_t)1 << 38))) return false;
  // an axis of one element has no stride of its own
  const int64_t rs = rows == 1 ? 0 : o.rs, ks = K == 1 ? 0 : o.ks;
  auto pitch_ok = [](int64_t n, int64_t p) { return n == 1 || (p > 0 && p % 8 == 0 && p < ((int64_t)1 << 38)); };
  if ((K == 1 || ks == 1) && pitch_ok(rows, rs)) {
    r.rows_inner = 0;
    r.pitch = rows == 1 ? (K + 7) / 8 * 8 : rs;
  } else if ((rows == 1 || rs == 1) && pitch_ok(K, ks)) {
    r.rows_inner = 1;
    r.pitch = K == 1 ? (rows + 7) / 8 * 8 : ks;
  } else {
    return false;
  }
  *out = r;
  return true;
}

cudaError_t launch_gemm_tc(const TcProblem& t, cudaStream_t s) {
  int sms = 0;
  const cudaError_t e = device_sms(&sms);
  if (e != cudaSuccess) return e;
  TcParams p{};
  p.I = t.I;
  p.J = t.J;
  p.kblocks = (int)((t.K + BK - 1) / BK);
  const int planes = t.kind == kOne ? 1 : t.kind == kHalves ? 2 : 3;
  const Form f = choose_form(t, p.kblocks, planes, planes == 1 ? 1 : planes == 2 ? 3 : 6, sms);
  const int CG = f.pair ? 2 : 1;
  p.BN = f.BN;
  p.split = f.split;
  p.share = p.BN / CG;
  p.tiles_i = (int)((t.I + BM * CG - 1) / (BM * CG));
  p.tiles_j = (int)((t.J + p.BN - 1) / p.BN);
  p.tiles = t.batch * (t.sym ? (int64_t)p.tiles_i * (p.tiles_i + 1) / 2 : (int64_t)p.tiles_i * p.tiles_j);
  p.band = 8;
  p.p_inner = t.P.rows_inner;
  p.q_inner = t.Q.rows_inner;
  p.p_bcast = t.P.bcast;
  p.q_bcast = t.Q.bcast;
  p.sym = t.sym;
  p.b_bytes = (p.q_inner ? (p.share + 63) / 64 * 64 : p.share) * BK * 2;
  p.stage_bytes = planes * (kABytes + p.b_bytes);
  p.idesc = mma_idesc(t.f16, p.p_inner, p.q_inner, BM * CG, p.BN);
  p.e = t.e;
  p.polar = t.polar;
  p.res_kind = t.res;
  p.y_plane = t.y_plane;
  p.res_plane = t.res_plane;
  const int64_t osize = t.out == B2C_F32 ? 4 : 2, rsize = t.res == B2C_F32 ? 4 : 2;
  const bool along_i = t.e.y.js != 1;
  p.y_vec = vec16(t.e.y, along_i, osize, t.y_plane);
  p.pre_vec = vec16(t.e.pre, along_i, osize, 0);
  p.res_vec = vec16(t.e.res, along_i, rsize, t.res_plane);
  p.bias_vec = (reinterpret_cast<uintptr_t>(t.e.bias) & 15) == 0;
  p.inject = injected_timeout() == 1;
  p.chained = t.chained;
  CUtensorMap mp, mq;
  if (!encode(&mp, t.P, t.f16, planes, t.batch, t.I, t.K, BM) ||
      !encode(&mq, t.Q, t.f16, planes, t.batch, t.J, t.K, p.share))
    return cudaErrorInvalidValue;
  return f.pair ? launch_out<true>(t, mp, mq, p, sms, s) : launch_out<false>(t, mp, mq, p, sms, s);
}

cudaError_t gemm_take_fault(unsigned int* fault) {
  unsigned int f = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&f, g_gemm_fault, sizeof(unsigned int));
  if (e != cudaSuccess) return e;
  *fault |= f;
  return cudaMemcpyToSymbol(g_gemm_fault, &zero, sizeof(unsigned int));
}

}  // namespace b2c
