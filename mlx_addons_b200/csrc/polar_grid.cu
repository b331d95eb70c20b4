// Newton-Schulz orthogonalisation of matrices of middle size, every step in
// one launch: a cooperative grid of one CTA an SM walks the three products of
// each step (S, P, X'), with a barrier of the grid between them.
//
// With a launch for each product, 17 launches take about 10 us each however
// small they are: about 3 for the launch and its set-up and 5 for an epilogue whose
// instructions all come from memory, since a kernel runs its epilogue once. Here
// both are paid once (256 x 256 bf16: 115 us against 182, 8 x 256 x 1024 bf16: 148 against 231).
//
// Roles in a CTA as in gemm_tc.cu: a thread of loads, one of products, eight
// epilogue warps, which also meet the barrier: their stores, then a fence that
// orders them before the other CTAs' TMA loads, a counter in memory, and the
// word to the loading thread.
//
// Every wait is bounded. A CTA whose wait runs out leaves NaN in its own tiles of
// the result, whichever product it was in; the tiles of a CTA that finished stand.
#include <cmath>

#include "b2c_kernels.cuh"
#include "gemm_tile.cuh"
#include "polar.cuh"

namespace b2c {

__device__ unsigned int g_grid_fault;

namespace {

constexpr int kEpi = 8;
constexpr int kThreadsG = (kEpi + 4) * 32;
constexpr int kMaxStepsG = 64;
constexpr uint64_t kBarrierNs = 2000000000ull;

// One of the three products of a step.
struct GridPhase : SliceLayout {
  int64_t I, J, tiles;
  int tiles_i, tiles_j, kblocks, BN, sym;
};

struct GridStep {
  float s_alpha, s_k;
  float p_alpha, p_beta, p_k, p_k2, p_k3, p_k4;
  float x_alpha, x_beta, x_k;
};

struct GridParams {
  GridPhase phase[3];
  int steps, stages, stage_bytes, bcast, wide, inject, last_vec;
  int64_t batch, side, mn, xx, ss, pitch_x, pitch_s, x_plane, s_plane;
  __half *X[2], *S, *P;
  float *ds, *dp;
  const float* r;
  void* out;
  int64_t out_rs, out_cs;
  unsigned int* counter;  // zero at the start
  GridStep step[kMaxStepsG];
};

struct GridMaps {
  CUtensorMap s_p[2], s_q[2];  // S = X X^T on either X
  CUtensorMap p_p, p_q;        // P = S S
  CUtensorMap x_p[2], x_q[2];  // X' = P X or X P
};

// What the general epilogue needs for the last product, whose outputs have the
// caller's type and layout.
template <int PLANES>
__device__ __forceinline__ void set_last(TcParams& c, const GridParams& p) {
  const GridStep& k = p.step[p.steps - 1];
  const int inner = PLANES == 2 ? kOutHalves : B2C_F16, cur = (p.steps - 1) & 1;
  c = TcParams{};
  c.I = p.phase[2].I, c.J = p.phase[2].J;
  c.split = 1;
  c.res_kind = inner;
  c.y_vec = p.last_vec;
  c.res_vec = p.out_cs == 1;
  c.e.y = GemmView{p.out, p.mn, p.out_rs, p.out_cs};
  c.e.res = GemmView{p.X[cur], p.xx, p.pitch_x, 1};
  c.res_plane = p.x_plane;
  c.e.alpha = k.x_alpha, c.e.beta = k.x_beta;
  c.polar.mode = p.wide ? kPolarXi : kPolarXj;
  c.polar.r = p.steps > 1 ? nullptr : p.r;
  c.polar.d_in = c.polar.d_out = p.dp;
  c.polar.side = p.pitch_s;
  c.polar.k = k.x_k;
}

// The tile order of a phase alone.
__device__ __forceinline__ Tile phase_tile(const GridPhase& g, int64_t t) {
  TcParams c;
  c.tiles_i = g.tiles_i, c.tiles_j = g.tiles_j, c.BN = g.BN, c.sym = g.sym, c.band = 8;
  return tile_at<1>(c, t);
}

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kEpi * 32) : "memory"); }
// The same, and whether any of the epilogue's threads says yes: they leave a
// phase together or not at all.
__device__ __forceinline__ bool epi_any(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred.aligned q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"((uint32_t)x), "n"(kEpi * 32)
      : "memory");
  return r != 0;
}

template <int PLANES>
__device__ __forceinline__ void load_x(float (&x)[8], const __half* at, int64_t plane) {
  const uint4 h = *reinterpret_cast<const uint4*>(at);
  const __half2* q = reinterpret_cast<const __half2*>(&h);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = __half22float2(q[k]);
    x[2 * k] = f.x, x[2 * k + 1] = f.y;
  }
  if constexpr (PLANES == 2) {
    const uint4 l = *reinterpret_cast<const uint4*>(at + plane);
    const __half2* m = reinterpret_cast<const __half2*>(&l);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __half22float2(m[k]);
      x[2 * k] += f.x, x[2 * k + 1] += f.y;
    }
  }
}

template <int PLANES>
__device__ __forceinline__ void store_x(const float (&v)[8], __half* at, int64_t plane) {
  __align__(16) __half2 h[4], l[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    h[k] = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
    if constexpr (PLANES == 2) {
      const float2 f = __half22float2(h[k]);
      l[k] = __floats2half2_rn(v[2 * k] - f.x, v[2 * k + 1] - f.y);
    }
  }
  *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(h);
  if constexpr (PLANES == 2) *reinterpret_cast<uint4*>(at + plane) = *reinterpret_cast<const uint4*>(l);
}

// The epilogue of a 32 x 32 block of S, P or an X that is not the last: the
// formulas of TcPolarMode. Everything that it reads from memory is asked for at
// once, before anything else, and rows are padded to units of 8, which needs no
// edges inside a unit (the general epilogue took 5,000 clocks a block, this one 1,500).
template <int PLANES>
__device__ __forceinline__ void polar_block(const GridParams& p, const GridStep& k, int ph, int x, float f, const float (&acc)[32],
                                            int64_t b, int64_t i, int64_t j, bool mirror, float* stage, int lane) {
  const int64_t I = p.phase[ph].I, J = p.phase[ph].J;
  const int c8 = (lane & 3) * 8, r0 = lane >> 2;
  const int64_t pitch = ph == 2 ? p.pitch_x : p.pitch_s, plane = ph == 2 ? p.x_plane : p.s_plane;
  __half* y = ph == 0 ? p.S + b * p.ss : ph == 1 ? p.P + b * p.ss : p.X[x ^ 1] + b * p.xx;
  const __half* res = ph == 1 ? p.S + b * p.ss : p.X[x] + b * p.xx;
  const float* d = (ph == 1 ? p.ds : p.dp) + b * p.pitch_s;
  const bool cols = j + c8 < J, by_row = ph == 1 || p.wide, by_col = ph == 1 || !p.wide;
  float xr[4][8], di[4] = {}, dj[8] = {};
  if (ph) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (cols && i + r0 + 8 * t < I) {
        load_x<PLANES>(xr[t], res + (i + r0 + 8 * t) * pitch + j + c8, plane);
        if (by_row) di[t] = d[i + r0 + 8 * t];
      }
    if (by_col && cols) {
      const float4 a = *reinterpret_cast<const float4*>(d + j + c8), c = *reinterpret_cast<const float4*>(d + j + c8 + 4);
      dj[0] = a.x, dj[1] = a.y, dj[2] = a.z, dj[3] = a.w, dj[4] = c.x, dj[5] = c.y, dj[6] = c.z, dj[7] = c.w;
    }
  }
#pragma unroll
  for (int c = 0; c < 32; ++c) stage[lane * kStagePitch + c] = acc[c];
  __syncwarp();
  float* d_out = (ph == 0 ? p.ds : p.dp) + b * p.pitch_s;
  const float alpha = ph == 0 ? k.s_alpha * f * f : ph == 1 ? k.p_alpha : f * k.x_alpha;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int r = r0 + 8 * t;
    float* at = stage + r * kStagePitch + c8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at[e] * alpha;
    if (ph < 2) {
      float w = 0.f;  // this row's diagonal element, where it is among the eight
      const int here = i == j ? r - c8 : -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w = e == here ? v[e] : w;
        if (ph == 1) v[e] = fmaf(fmaf(k.p_k, di[t] + dj[e], k.p_beta), xr[t][e], v[e]);
        v[e] = e == here ? 0.f : v[e];
      }
      if (here >= 0 && here < 8 && i + r < I)
        d_out[i + r] = ph == 0 ? w * k.s_k : fmaf(k.p_k2, w, di[t] * fmaf(k.p_k3, di[t], k.p_k4));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(f * k.x_beta * (k.x_k + di[t] + dj[e]), xr[t][e], v[e]);
    }
    if (cols && i + r < I) store_x<PLANES>(v, y + (i + r) * pitch + j + c8, plane);
    if (mirror) {
#pragma unroll
      for (int e = 0; e < 8; ++e) at[e] = v[e];
    }
  }
  __syncwarp();
  if (!mirror) return;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int c = r0 + 8 * t;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = stage[(c8 + e) * kStagePitch + c];
    if (j + c < I && i + c8 < J) store_x<PLANES>(v, y + (j + c) * pitch + i + c8, plane);
  }
  __syncwarp();
}

template <int PLANES, typename T>
__global__ void __launch_bounds__(kThreadsG, 1)
    polar_grid_kernel(const __grid_constant__ GridMaps maps, const __grid_constant__ GridParams p) {
  constexpr bool JOIN = PLANES > 1;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 6];
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  __shared__ TcParams cur;
  __shared__ volatile int heard;  // the phase that the loading thread is in
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  float* staging = reinterpret_cast<float*>(ring + p.stages * p.stage_bytes);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, tfull0 = empty0 + 8 * kMaxStages,
                 tempty0 = tfull0 + 16, go = tempty0 + 16, never = go + 8;
  const uint64_t limit = p.inject == 1 ? 1000000ull : kWaitNs;
  volatile int* gu = &gave_up;
  if (tid == 0) {
    gave_up = 0;
    heard = 0;
    for (int s = 0; s < p.stages; ++s) {
      bar_init(full0 + 8 * s, 1);
      bar_init(empty0 + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      bar_init(tfull0 + 8 * s, 1);
      bar_init(tempty0 + 8 * s, kEpi);
    }
    bar_init(go, 1);
    bar_init(never, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kEpi) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    fence_before();
  }
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  const int phases = 3 * p.steps;

  if (warp < kEpi) {
    const int quad = warp & 3, group = warp >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    float* stage = staging + warp * kStageFloats;
    uint32_t buf = 0, tphase = 0;
    if (p.inject == 1 && blockIdx.x == 0) bar_wait(never, 0, gu, limit, &g_grid_fault);
    for (int f = 0; f < phases; ++f) {
      const int st = f / 3, ph = f - 3 * st;
      if (f == phases - 1 && tid == 0) set_last<PLANES>(cur, p);
      if (epi_any(*gu != 0)) break;
      const int kblocks = p.phase[ph].kblocks, BN = p.phase[ph].BN;
      const bool last = f == phases - 1;
      if (p.inject == 2 && last && blockIdx.x == 0) bar_wait(never, 0, gu, 1000000ull, &g_grid_fault);
      for (int64_t t = blockIdx.x; t < p.phase[ph].tiles; t += gridDim.x) {
        const Tile o = phase_tile(p.phase[ph], t);
        float acc[2][32];
        bool ok = true;
        for (int kb = 0; kb < (JOIN ? kblocks : 1); ++kb) {
          ok = __all_sync(kFull, ok && bar_wait(tfull0 + 8 * buf, tphase, gu, limit, &g_grid_fault));
          fence_after();
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int col = (2 * q + group) * 32;
            if (col < BN) {
              float v[32];
              tmem_row32(lanes + buf * 128 + col, v);
#pragma unroll
              for (int c = 0; c < 32; ++c) acc[q][c] = kb ? acc[q][c] + v[c] : v[c];
            }
          }
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive_cluster(tempty0 + 8 * buf);
          if (++buf == 2) buf = 0, tphase ^= 1;
        }
        if (!ok) break;
        // one copy of the epilogue's code: the sums move up instead of the index
#pragma unroll 1
        for (int q = 0; q < BN / 64; ++q) {
          const int64_t i = o.i + quad * 32, j = o.j + (2 * q + group) * 32;
          if (last) finish32<T>(cur, acc[0], o.b, i, j, o.mirror, stage, lane);
          else polar_block<PLANES>(p, p.step[st], ph, st & 1, st ? 1.f : p.r[o.b], acc[0], o.b, i, j, o.mirror, stage, lane);
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[0][c] = acc[1][c];
        }
      }
      if (last || epi_any(*gu != 0)) break;
      // ---- barrier of the grid ----
      __threadfence();
      asm volatile("fence.proxy.async;" ::: "memory");
      epi_sync();
      if (tid == 0) {
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p.counter) : "memory");
        const unsigned int target = (unsigned int)(f + 1) * gridDim.x;
        const uint64_t t0 = now_ns();
        for (;;) {
          unsigned int seen;
          asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(p.counter) : "memory");
          if (seen >= target) break;
          if (now_ns() - t0 > (p.inject == 1 ? 3000000ull : kBarrierNs) || (p.inject == 3 && blockIdx.x == 0 && f == phases - 2)) {
            *gu = 1;
            atomicOr(&g_grid_fault, 1u);
            break;
          }
        }
        asm volatile("fence.proxy.async;" ::: "memory");
        // the loading thread has taken the word before (its CTA may have had no tile, and nothing else keeps it in step)
        while (heard < f && !*gu)
          if (now_ns() - t0 > 2 * kBarrierNs) *gu = 1, atomicOr(&g_grid_fault, 1u);
        bar_arrive_cluster(go);
      }
    }
  } else if (warp == kEpi) {
    // ---- loads ----
    const bool lead = elect_one();
    uint32_t s = 0, phase = 0;
    for (int f = 0; f < phases && !*gu; ++f) {
      const int st = f / 3, ph = f - 3 * st, x = st & 1;
      const GridPhase& g = p.phase[ph];
      const CUtensorMap* mp = ph == 0 ? &maps.s_p[x] : ph == 1 ? &maps.p_p : &maps.x_p[x];
      const CUtensorMap* mq = ph == 0 ? &maps.s_q[x] : ph == 1 ? &maps.p_q : &maps.x_q[x];
      if (f && !bar_wait(go, (f - 1) & 1, gu, 2 * kBarrierNs, &g_grid_fault)) break;
      __syncwarp();
      if (lead) heard = f;
      asm volatile("fence.proxy.async;" ::: "memory");
      for (int64_t t = blockIdx.x; t < g.tiles && !*gu; t += gridDim.x) {
        const Tile o = phase_tile(g, t);
        const int b = p.bcast ? 0 : (int)o.b;
        for (int kb = 0; kb < g.kblocks; ++kb) {
          if (!bar_wait(empty0 + 8 * s, phase ^ 1, gu, limit, &g_grid_fault)) break;
          if (lead) {
            bar_expect(full0 + 8 * s, g.stage_bytes);
            load_slice<1, PLANES>(g, mp, mq, smem_u32(ring + s * p.stage_bytes), (int)o.i, (int)o.j, kb, b, b, full0 + 8 * s);
          }
          if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == kEpi + 1) {
    // ---- products ----
    const bool lead = elect_one();
    uint32_t s = 0, phase = 0, buf = 0, tphase = 0;
    for (int f = 0; f < phases && !*gu; ++f) {
      const GridPhase& g = p.phase[f % 3];
      Multiplier<1, PLANES> mul(g, smem_u32(ring));
      mul.stage = p.stage_bytes >> 4;
      const int per = JOIN ? 1 : g.kblocks;  // slices of one accumulator
      for (int64_t t = blockIdx.x; t < g.tiles && !*gu; t += gridDim.x) {
        for (int k0 = 0; k0 < g.kblocks; k0 += per) {
          // nothing of the next phase arrives before this CTA's epilogue has met the grid: its wait may be long
          if (!bar_wait(tempty0 + 8 * buf, tphase ^ 1, gu, 2 * kBarrierNs, &g_grid_fault)) break;
          fence_after();
          for (int kb = 0; kb < per; ++kb) {
            if (!bar_wait(full0 + 8 * s, phase, gu, 2 * kBarrierNs, &g_grid_fault)) break;
            fence_after();
            if (lead) {
              mul.slice(s, tmem + buf * 128, kb == 0);
              commit<1>(empty0 + 8 * s);
            }
            if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
          }
          if (*gu) break;
          if (lead) commit<1>(tfull0 + 8 * buf);
          if (++buf == 2) buf = 0, tphase ^= 1;
        }
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (gave_up) {
    settle();
    __syncthreads();
    // NaN for this CTA's tiles of the last product, which no other CTA writes: the others either give up at the next
    // barrier, where this one is missed, and do the same for theirs, or finish theirs without it
    const GridPhase& g = p.phase[2];
    for (int64_t t = blockIdx.x; t < g.tiles; t += gridDim.x) {
      const Tile o = phase_tile(g, t);
      for (int e = tid; e < BM * g.BN; e += kThreadsG) {
        const int64_t i = o.i + e / g.BN, j = o.j + e % g.BN;
        if (i < g.I && j < g.J) static_cast<T*>(p.out)[o.b * p.mn + i * p.out_rs + j * p.out_cs] = from_f32<T>(__int_as_float(0x7fffffff));
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kEpi) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem));
  }
}

template <int PLANES, typename T>
cudaError_t launch_g(const GridMaps& maps, const GridParams& p, int grid, size_t smem, cudaStream_t s) {
  auto kern = polar_grid_kernel<PLANES, T>;
  static int cache[64];
  int occ = 0;
  cudaError_t e = kernel_occupancy(kern, kThreadsG, smem, cache, &occ);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreadsG);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, maps, p);
}

}  // namespace

// Where the launches cost more than what their pairs of CTAs save, whose tiles
// read half as much. With one plane (bf16) that is up to two rounds of 128 x 128
// tiles of X (2048 x 2048: 328 us against 396 as launches), and eight of a side
// up to 1024 (64 x 512 x 512: 651 against 757; but 2 x 2048 x 2048: 540 against 482).
// With two planes the products take three times as long: up to one round of a
// side up to 256 (256 x 256: 149 against 166, 8 x 200 x 260: 160 against 184; but
// 1000 x 517: 238 against 216, 64 x 256 x 256: 421 against 338). A long side makes few
// and long products of S, which only launches of their own split.
bool polar_grid_fits(const PolarParams& p, int sms) {
  const int64_t tiles = p.batch * ((p.m + 127) / 128) * ((p.n + 127) / 128);
  const int64_t side = p.m < p.n ? p.m : p.n, along = p.m < p.n ? p.n : p.m;
  const bool one = p.dtype == B2C_BF16;
  const int rounds = one ? (side <= 1024 ? 8 : 2) : side <= 256 ? 1 : 0;
  return tiles <= rounds * (int64_t)sms && along <= (one ? 4096 : 1024) && p.steps <= kMaxStepsG;
}

cudaError_t launch_polar_grid(const PolarParams& in, const PolarScratch& w, int sms, cudaStream_t s) {
  GridParams p{};
  GridMaps maps;
  const int planes = in.dtype == B2C_BF16 ? 1 : 2;
  const bool wide = in.m <= in.n;
  p.steps = in.steps;
  p.batch = in.batch;
  p.bcast = in.batch == 1;
  p.wide = wide;
  p.side = w.side;
  p.mn = in.m * in.n;
  p.pitch_x = w.pitch_x, p.pitch_s = w.pitch_s;
  p.xx = in.m * w.pitch_x, p.ss = w.side * w.pitch_s;
  p.x_plane = w.x_plane, p.s_plane = w.s_plane;
  p.X[0] = w.X0, p.X[1] = w.X1, p.S = w.S, p.P = w.P;
  p.ds = w.ds, p.dp = w.dp, p.r = w.r;
  p.out = in.out;
  p.out_rs = in.out_rs, p.out_cs = in.out_cs;
  p.counter = w.counter;
  p.inject = injected_timeout();
  const int64_t elt = in.dtype == B2C_F32 ? 4 : 2, other = in.out_cs == 1 ? in.out_rs : in.out_cs;
  p.last_vec = (reinterpret_cast<uintptr_t>(in.out) & 15) == 0 && p.mn * elt % 16 == 0 && other * elt % 16 == 0;
  for (int ph = 0; ph < 3; ++ph) {
    GridPhase& g = p.phase[ph];
    g.sym = ph < 2;
    g.I = ph < 2 ? w.side : in.m;
    g.J = ph < 2 ? w.side : in.n;
    const int64_t K = ph == 0 ? (wide ? in.n : in.m) : w.side;
    g.kblocks = (int)((K + BK - 1) / BK);
    g.p_inner = ph == 0 && !wide;
    g.q_inner = ph == 0 ? !wide : ph == 2 && wide;
    g.tiles_i = (int)((g.I + BM - 1) / BM);
    // 64 columns where that is less work for the busiest SM: loads of 16 KB + 128 BN a plane and slice, about 2,000 clocks
    // a tile beside them
    double best = 1e300;
    for (int BN = 64; BN <= 128; BN *= 2) {
      const int64_t tj = (g.J + BN - 1) / BN;
      const int64_t tiles = in.batch * (g.sym ? (int64_t)(BM / BN) * g.tiles_i * (g.tiles_i + 1) / 2 : g.tiles_i * tj);
      const double rate = fmin(100.0, 6000.0 / fmin((double)tiles, (double)sms));
      const double clocks = ceil((double)tiles / sms) *
                            (g.kblocks * fmax(planes * (16384.0 + BN * 128.0) / rate, planes == 2 ? 900.0 : 400.0) + 2000);
      if (clocks < best) best = clocks, g.BN = BN, g.tiles_j = (int)tj, g.tiles = tiles;
    }
    g.b_bytes = g.BN * BK * 2;
    g.stage_bytes = planes * (kABytes + g.b_bytes);
    g.idesc = mma_idesc(1, g.p_inner, g.q_inner, BM, g.BN);
    if (g.stage_bytes > p.stage_bytes) p.stage_bytes = g.stage_bytes;
  }
  const int staging = kEpi * kStageFloats * 4;
  p.stages = (kSmemMax - 1024 - 1024 - staging) / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + staging;

  auto x_op = [&](int x, int inner) { return TcOperand{p.X[x], p.xx, p.pitch_x, p.x_plane, inner, p.bcast}; };
  const TcOperand s_op{p.S, p.ss, p.pitch_s, p.s_plane, 0, p.bcast}, p_op{p.P, p.ss, p.pitch_s, p.s_plane, 0, p.bcast};
  const int64_t side = w.side, L = wide ? in.n : in.m;
  bool ok = true;
  for (int x = 0; x < 2; ++x) {
    // S: rows are the smaller side, k the longer
    ok = ok && encode(&maps.s_p[x], x_op(x, !wide), 1, planes, in.batch, side, L, BM);
    ok = ok && encode(&maps.s_q[x], x_op(x, !wide), 1, planes, in.batch, side, L, p.phase[0].BN);
    ok = ok && (wide ? encode(&maps.x_p[x], p_op, 1, planes, in.batch, side, side, BM)
                     : encode(&maps.x_p[x], x_op(x, 0), 1, planes, in.batch, in.m, in.n, BM));
    ok = ok && (wide ? encode(&maps.x_q[x], x_op(x, 1), 1, planes, in.batch, in.n, side, p.phase[2].BN)
                     : encode(&maps.x_q[x], p_op, 1, planes, in.batch, side, side, p.phase[2].BN));
  }
  ok = ok && encode(&maps.p_p, s_op, 1, planes, in.batch, side, side, BM);
  ok = ok && encode(&maps.p_q, s_op, 1, planes, in.batch, side, side, p.phase[1].BN);
  if (!ok) return cudaErrorInvalidValue;

  double hi = 1.0;
  for (int t = 0; t < in.steps; ++t) {
    const double a = in.coef[3 * t], b = in.coef[3 * t + 1], c = in.coef[3 * t + 2], t2 = hi * hi, sx = kPolarScale;
    const double ss = polar_scale_for(t2), sp = polar_scale_for(fabs(b) * t2 + fabs(c) * t2 * t2);
    const double so = t == in.steps - 1 ? 1.0 : sx;
    p.step[t] = GridStep{(float)(ss / (sx * sx)), (float)(1 / ss),
                         (float)(c * sp / (ss * ss)), (float)(b * sp / ss), (float)(c * sp / ss), (float)(1 / sp), (float)c,
                         (float)b,
                         (float)(so / (sp * sx)), (float)(so / sx), (float)a};
    hi = polar_poly_bound(a, b, c, hi);
  }
  int64_t most = 0;
  for (const GridPhase& g : p.phase) most = g.tiles > most ? g.tiles : most;
  const int grid = (int)(most < sms ? most : sms);
  switch (in.dtype) {
    case B2C_F32: return launch_g<2, float>(maps, p, grid, smem, s);
    case B2C_BF16: return launch_g<1, __nv_bfloat16>(maps, p, grid, smem, s);
    default: return launch_g<2, __half>(maps, p, grid, smem, s);
  }
}

cudaError_t polar_grid_take_fault(unsigned int* fault) {
  unsigned int f = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&f, g_grid_fault, sizeof(unsigned int));
  if (e != cudaSuccess) return e;
  *fault |= f;
  return cudaMemcpyToSymbol(g_grid_fault, &zero, sizeof(unsigned int));
}

}  // namespace b2c
