// Products with an epilogue on the tensor cores: D[i, j] = sum_k P[i, k]
// Q[j, k] with 16-bit factors and 32-bit sums (tcgen05.mma kind::f16, operands
// by TMA, accumulators in tensor memory).
//
// A pair of CTAs (two SMs) computes a 256 x 256 tile (cta_group::2): each CTA
// holds 128 rows of P and 128 of Q's 256 in shared memory and 128 x 256 of D
// in its tensor memory. Where D has fewer rows or columns than that pays for,
// single CTAs compute 128 x BN tiles. Both forms are persistent: the grid is
// one CTA per SM, tiles are dealt in order.
//
// Roles in a CTA: one thread issues the TMA loads (a ring of 64-deep slices),
// one thread of the leading CTA issues the MMAs, eight warps take finished
// accumulators from tensor memory through the epilogue. Tensor memory holds
// two accumulators, so the epilogue of a tile runs under the MMAs of the next.
//
// Both axis orders of an operand are read as they lie: with unit stride along
// k ("K-major") and along the rows ("MN-major"), both with 128-byte swizzle.
//
// Split operands: a float32 value is three bf16 planes or, where its range is
// known, two f16 planes; the product is then the sum of the plane pairs whose
// weight is 2^-24 or more (6 of 9, or 3 of 4), smallest first. The tensor
// cores truncate when they add to an accumulator, so such a product's
// accumulator is joined in float32 registers every kChunk values of k
// (JOIN): without that the truncations, all towards zero, add up along k.
#include <cstdlib>
#include <cstring>
#include <type_traits>

#include "b2c_kernels.cuh"
#include "gemm_tc.cuh"
#include "tcgen05.cuh"

namespace b2c {

__device__ unsigned int g_gemm_fault;

namespace {

constexpr int BM = 128;          // rows of D per CTA
constexpr int BK = 64;           // depth of a slice: 128 bytes
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarps + 4) * 32;  // the last warpgroup: loads, products, two idle warps
// Registers: 384 x 168 at launch = 128 x 72 + 256 x 216 after the split.
constexpr int kRegsFew = 72, kRegsMany = 216;
constexpr int kMaxStages = 8;
constexpr int kChunk = 2;        // slices of k per joined accumulator
constexpr int kMaxSeg = 6;
constexpr int kSmemMax = 232448;

struct TcParams {
  int64_t I, J, tiles;
  int tiles_i, tiles_j, band;
  int kblocks, nseg, chunk;
  int seg_p[kMaxSeg], seg_q[kMaxSeg];
  int BN, share, stages, a_bytes, b_bytes;
  int p_inner, q_inner, p_bcast, q_bcast, sym;
  uint32_t idesc;
  GemmEpilogue e;
  TcPolar polar;
  int res_kind, y_vec, pre_vec, res_vec;
  int64_t y_plane, res_plane;
  int inject;
};

// ---------------------------------------------------------------------------
// epilogue of one lane's 32 columns
// ---------------------------------------------------------------------------

struct Halves {};  // output tag: two f16 planes

template <typename OUT>
struct OutOf { typedef OUT T; };
template <>
struct OutOf<Halves> { typedef __half T; };

__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 a, __nv_bfloat16 b) {
  const __nv_bfloat162 v = __halves2bfloat162(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(__half a, __half b) {
  const __half2 v = __halves2half2(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Writes 32 x 32 values, one row per lane, to rows of unit stride: through
// shared memory, so that every store is 16 bytes of a full sector.
template <typename T>
__device__ __forceinline__ void store_rows(const float (&v)[32], T* base, int64_t row_stride, int rows, int cols,
                                           int vec, unsigned char* stage, int lane) {
  constexpr int PITCH = 32 * sizeof(T) + 16, PER = 16 / sizeof(T), U = 32 / PER;
  uint4* mine = reinterpret_cast<uint4*>(stage + lane * PITCH);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint4 w;
    if constexpr (sizeof(T) == 4) {
      w = make_uint4(__float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]), __float_as_uint(v[4 * u + 2]),
                     __float_as_uint(v[4 * u + 3]));
    } else {
      const float* q = &v[8 * u];
      w = make_uint4(pack2(from_f32<T>(q[0]), from_f32<T>(q[1])), pack2(from_f32<T>(q[2]), from_f32<T>(q[3])),
                     pack2(from_f32<T>(q[4]), from_f32<T>(q[5])), pack2(from_f32<T>(q[6]), from_f32<T>(q[7])));
    }
    mine[u] = w;
  }
  __syncwarp();
#pragma unroll
  for (int t = 0; t < U; ++t) {
    const int r = t * (32 / U) + lane / U, u = lane % U;
    if (r < rows) {
      const unsigned char* src = stage + r * PITCH + u * 16;
      T* dst = base + (int64_t)r * row_stride + u * PER;
      if (vec && (u + 1) * PER <= cols) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
      } else {
#pragma unroll
        for (int c = 0; c < PER; ++c)
          if (u * PER + c < cols) dst[c] = reinterpret_cast<const T*>(src)[c];
      }
    }
  }
  __syncwarp();
}

// The same where the row index has unit stride: lanes lie next to each other.
template <typename T>
__device__ __forceinline__ void store_cols(const float (&v)[32], T* base, int64_t col_stride, int rows, int cols, int lane) {
  if (lane >= rows) return;
#pragma unroll
  for (int c = 0; c < 32; ++c)
    if (c < cols) base[lane + (int64_t)c * col_stride] = from_f32<T>(v[c]);
}

template <typename T>
__device__ __forceinline__ void store_tile(const float (&v)[32], const GemmView& o, int64_t b, int64_t i, int64_t j,
                                           int rows, int cols, int vec, unsigned char* stage, int lane) {
  T* base = static_cast<T*>(o.p) + b * o.bs + i * o.is + j * o.js;
  if (o.js == 1) store_rows<T>(v, base, o.is, rows, cols, vec, stage, lane);
  else store_cols<T>(v, base, o.js, rows, cols, lane);
}

// r[c] += 32 columns of an addend's row.
template <typename T>
__device__ __forceinline__ void load_res(float (&r)[32], const T* base, int64_t js, int cols, int vec) {
  if (vec && cols >= 32) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < 32 / PER; ++u) {
      const uint4 w = *reinterpret_cast<const uint4*>(base + u * PER);
      const T* q = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int c = 0; c < PER; ++c) r[u * PER + c] += to_f32(q[c]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 32; ++c)
      if (c < cols) r[c] += to_f32(base[(int64_t)c * js]);
  }
}

template <bool FAST>
__device__ __forceinline__ void apply_act(float (&v)[32], int act) {
  switch (act) {
    case B2C_ACT_RELU:
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = act_f32<FAST>(v[c], B2C_ACT_RELU);
      break;
    case B2C_ACT_GELU:
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = act_f32<FAST>(v[c], B2C_ACT_GELU);
      break;
    case B2C_ACT_GELU_TANH:
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = act_f32<FAST>(v[c], B2C_ACT_GELU_TANH);
      break;
    case B2C_ACT_SILU:
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = act_f32<FAST>(v[c], B2C_ACT_SILU);
      break;
    default: break;
  }
}

// v = alpha D, r = the addend; see TcPolarMode.
__device__ __forceinline__ void polar_epilogue(float (&v)[32], const float (&r)[32], const TcPolar& q, const GemmEpilogue& e,
                                               int64_t b, int64_t i, int64_t j, int rows, int cols, int lane) {
  const float f = q.r ? q.r[b] : 1.f;
  const float* d = q.d_in + b * q.side;
  const int64_t diag = i + lane - j;  // the column of this row's diagonal element
  if (q.mode == kPolarS) {
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] *= f * f;
    if (diag >= 0 && diag < 32 && lane < rows) {
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (c == diag) {
          q.d_out[b * q.side + i + lane] = v[c] * q.k;
          v[c] = 0.f;
        }
    }
    return;
  }
  const float di = q.mode != kPolarXj && lane < rows ? d[i + lane] : 0.f;
  const float dj = q.mode != kPolarXi && lane < cols ? d[j + lane] : 0.f;
  if (q.mode == kPolarP) {
    const float w = fmaf(q.k, di, e.beta);
    const bool here = diag >= 0 && diag < 32 && lane < rows;
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      const float x = fmaf(q.k, __shfl_sync(kFull, dj, c), w);
      if (here && c == diag) {
        q.d_out[b * q.side + i + lane] = fmaf(q.k2, v[c], di * fmaf(q.k3, di, q.k4));
        v[c] = 0.f;
      } else {
        v[c] = fmaf(x, r[c], v[c]);
      }
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const float x = q.k + (q.mode == kPolarXi ? di : __shfl_sync(kFull, dj, c));
    v[c] = f * fmaf(e.beta * x, r[c], v[c]);
  }
}

// v: 32 columns j.. of row i + lane. rows / cols: how many of the 32 x 32
// exist (either may be <= 0).
template <typename OUT>
__device__ __forceinline__ void epilogue32(float (&v)[32], const TcParams& p, int64_t b, int64_t i, int64_t j, int rows,
                                           int cols, bool mirror, unsigned char* stage, int lane) {
  typedef typename OutOf<OUT>::T T;
  const GemmEpilogue& e = p.e;
  if (rows <= 0 || cols <= 0) return;
#pragma unroll
  for (int c = 0; c < 32; ++c) v[c] *= e.alpha;
  if constexpr (!std::is_same<OUT, Halves>::value) {
    if (e.bias) {
      const T* bias = static_cast<const T*>(e.bias);
      if (e.bias_on_i) {
        const float x = lane < rows ? to_f32(bias[i + lane]) : 0.f;
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] += x;
      } else {
        const float x = lane < cols ? to_f32(bias[j + lane]) : 0.f;
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] += __shfl_sync(kFull, x, c);
      }
    }
    if (e.pre.p) store_tile<T>(v, e.pre, b, i, j, rows, cols, p.pre_vec, stage, lane);
    apply_act<sizeof(T) == 2>(v, e.act);
  }
  float r[32] = {};
  if (e.res.p && lane < rows) {
    const int64_t off = b * e.res.bs + (i + lane) * e.res.is + j * e.res.js;
    switch (p.res_kind) {
      case B2C_F32: load_res(r, static_cast<const float*>(e.res.p) + off, e.res.js, cols, p.res_vec); break;
      case B2C_BF16: load_res(r, static_cast<const __nv_bfloat16*>(e.res.p) + off, e.res.js, cols, p.res_vec); break;
      default:
        if (p.res_kind == kOutHalves)
          load_res(r, static_cast<const __half*>(e.res.p) + p.res_plane + off, e.res.js, cols, p.res_vec);
        load_res(r, static_cast<const __half*>(e.res.p) + off, e.res.js, cols, p.res_vec);
    }
  }
  if (p.polar.mode == kPolarNone) {
    if (e.res.p) {
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = fmaf(e.beta, r[c], v[c]);
    }
  } else {
    polar_epilogue(v, r, p.polar, e, b, i, j, rows, cols, lane);
  }
  const GemmView flip{e.y.p, e.y.bs, e.y.js, e.y.is};
  if constexpr (std::is_same<OUT, Halves>::value) {
    float lo[32];
#pragma unroll
    for (int c = 0; c < 32; ++c) lo[c] = v[c] - __half2float(__float2half_rn(v[c]));
    store_tile<__half>(v, e.y, b, i, j, rows, cols, p.y_vec, stage, lane);
    if (mirror) store_tile<__half>(v, flip, b, i, j, rows, cols, p.y_vec, stage, lane);
    const GemmView y2{static_cast<__half*>(e.y.p) + p.y_plane, e.y.bs, e.y.is, e.y.js};
    const GemmView f2{y2.p, e.y.bs, e.y.js, e.y.is};
    store_tile<__half>(lo, y2, b, i, j, rows, cols, p.y_vec, stage, lane);
    if (mirror) store_tile<__half>(lo, f2, b, i, j, rows, cols, p.y_vec, stage, lane);
  } else {
    store_tile<T>(v, e.y, b, i, j, rows, cols, p.y_vec, stage, lane);
    if (mirror) store_tile<T>(v, flip, b, i, j, rows, cols, p.y_vec, stage, lane);
  }
}

struct Tile {
  int64_t b, i, j;  // batch, first row and column (of the pair's tile)
  bool mirror;
};

// The t-th tile. Bands of `band` tile rows are walked column by column, so
// that the tiles in flight at a time share rows and columns in L2. With sym,
// the lower triangle of square tiles, row by row.
template <int CG>
__device__ __forceinline__ Tile tile_at(const TcParams& p, int64_t t) {
  Tile o;
  if (p.sym) {
    const int64_t per = (int64_t)p.tiles_i * (p.tiles_i + 1) / 2;
    o.b = t / per;
    const int64_t u = t - o.b * per;
    int64_t r = (int64_t)((sqrt(8.0 * (double)u + 1.0) - 1.0) * 0.5);
    while (r * (r + 1) / 2 > u) --r;
    while ((r + 1) * (r + 2) / 2 <= u) ++r;
    const int64_t c = u - r * (r + 1) / 2;
    o.i = r * (BM * CG);
    o.j = c * p.BN;
    o.mirror = r != c;
    return o;
  }
  const int64_t per = (int64_t)p.tiles_i * p.tiles_j;
  o.b = t / per;
  const int64_t u = t - o.b * per, band = u / ((int64_t)p.band * p.tiles_j), r0 = band * p.band;
  const int64_t w = p.tiles_i - r0 < p.band ? p.tiles_i - r0 : p.band, v = u - r0 * p.tiles_j;
  o.i = (r0 + v % w) * (BM * CG);
  o.j = v / w * p.BN;
  o.mirror = false;
  return o;
}

__device__ __forceinline__ int clamp32(int64_t n) { return n > 32 ? 32 : (int)n; }

template <int CG, bool JOIN, typename OUT>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_tc_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ TcParams p) {
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 5];  // the last: nothing arrives on it
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  typedef typename OutOf<OUT>::T T;
  constexpr int kStage = 32 * (32 * sizeof(T) + 16);  // one warp's staging rows
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  unsigned char* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  const int stage_bytes = p.a_bytes + p.b_bytes;
  unsigned char* staging = ring + p.stages * stage_bytes;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, tfull0 = empty0 + 8 * kMaxStages,
                 tempty0 = tfull0 + 16;
  const uint32_t never = tempty0 + 16;
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
      bar_init(tempty0 + 8 * s, kEpiWarps * CG);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kEpiWarps) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
  }
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  fence_after();
  const uint32_t tmem = tmem_slot;
  const int64_t first = blockIdx.x / CG, step = gridDim.x / CG;
  volatile int* gu = &gave_up;

  if (warp < kEpiWarps) {
    if constexpr (JOIN) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMany));
    // ---- epilogue: warps w and w + 4 share the rows 32 (w % 4).., and take every other 32 columns ----
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t lead_tempty0 = CG == 2 ? map_rank(tempty0, 0) : tempty0;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    unsigned char* stage = staging + warp * kStage;
    uint32_t buf = 0, tphase = 0;
    bool ok = true;
    const float bad = __int_as_float(0x7fffffff);
    if (p.inject && blockIdx.x == 0) ok = __all_sync(kFull, bar_wait(never, 0, gu, limit, &g_gemm_fault));
    for (int64_t t = first; t < p.tiles; t += step) {
      const Tile o = tile_at<CG>(p, t);
      const int64_t i = o.i + rank * BM + quad * 32;
      const int rows = clamp32(p.I - i);
      if constexpr (JOIN) {
        float acc[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[q][c] = 0.f;
        for (int c0 = 0; c0 < p.kblocks; c0 += p.chunk) {
          ok = __all_sync(kFull, ok && bar_wait(tfull0 + 8 * buf, tphase, gu, limit, &g_gemm_fault));
          fence_after();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int col = (2 * q + half) * 32;
            if (col < p.BN) {
              float v[32];
              tmem_row32(lanes + buf * 256 + col, v);
#pragma unroll
              for (int c = 0; c < 32; ++c) acc[q][c] += v[c];
            }
          }
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive_cluster(lead_tempty0 + 8 * buf);
          if (++buf == 2) buf = 0, tphase ^= 1;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = (2 * q + half) * 32;
          if (col < p.BN) {
            if (!ok) {
#pragma unroll
              for (int c = 0; c < 32; ++c) acc[q][c] = bad;
            }
            epilogue32<OUT>(acc[q], p, o.b, i, o.j + col, rows, clamp32(p.J - o.j - col), o.mirror, stage, lane);
          }
        }
      } else {
        ok = __all_sync(kFull, ok && bar_wait(tfull0 + 8 * buf, tphase, gu, limit, &g_gemm_fault));
        fence_after();
        for (int col = half * 32; col < p.BN; col += 64) {
          float v[32];
          tmem_row32(lanes + buf * 256 + col, v);
          if (col + 64 >= p.BN) {  // the last of this warp's columns: the accumulator is free
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_cluster(lead_tempty0 + 8 * buf);
          }
          if (!ok) {
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = bad;
          }
          epilogue32<OUT>(v, p, o.b, i, o.j + col, rows, clamp32(p.J - o.j - col), o.mirror, stage, lane);
        }
        if (half * 32 >= p.BN && lane == 0) bar_arrive_cluster(lead_tempty0 + 8 * buf);
        if (++buf == 2) buf = 0, tphase ^= 1;
      }
    }
  } else {
    if constexpr (JOIN) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
    if (warp == kEpiWarps && lane == 0) {
      // ---- loads ----
      const uint32_t lead_full0 = CG == 2 ? map_rank(full0, 0) : full0;
      uint32_t s = 0, phase = 0;
      for (int64_t t = first; t < p.tiles && !*gu; t += step) {
        const Tile o = tile_at<CG>(p, t);
        const int i0 = (int)(o.i + rank * BM), j0 = (int)(o.j + rank * p.share);
        const int bp = p.p_bcast ? 0 : (int)o.b, bq = p.q_bcast ? 0 : (int)o.b;
        for (int c0 = 0; c0 < p.kblocks && !*gu; c0 += p.chunk) {
          const int c1 = min(c0 + p.chunk, p.kblocks);
          for (int g = 0; g < p.nseg; ++g) {
            for (int kb = c0; kb < c1; ++kb) {
              if (!bar_wait(empty0 + 8 * s, phase ^ 1, gu, limit, &g_gemm_fault)) break;
              if (rank == 0) bar_expect(full0 + 8 * s, CG * stage_bytes);
              const uint32_t bar = lead_full0 + 8 * s, a = smem_u32(ring + s * stage_bytes), q = a + p.a_bytes;
              if (p.p_inner) {
                tma_load<CG>(a, &map_p, i0, kb * BK, bp, p.seg_p[g], bar);
                tma_load<CG>(a + 8192, &map_p, i0 + 64, kb * BK, bp, p.seg_p[g], bar);
              } else {
                tma_load<CG>(a, &map_p, kb * BK, i0, bp, p.seg_p[g], bar);
              }
              if (p.q_inner) {
                for (int h = 0; h < p.b_bytes / 8192; ++h)
                  tma_load<CG>(q + h * 8192, &map_q, j0 + 64 * h, kb * BK, bq, p.seg_q[g], bar);
              } else {
                tma_load<CG>(q, &map_q, kb * BK, j0, bq, p.seg_q[g], bar);
              }
              if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
            }
          }
        }
      }
    } else if (warp == kEpiWarps + 1 && rank == 0 && lane == 0) {
      // ---- products ----
      uint32_t s = 0, phase = 0, buf = 0, tphase = 0;
      const uint32_t step_p = p.p_inner ? 2048 >> 4 : 32 >> 4, step_q = p.q_inner ? 2048 >> 4 : 32 >> 4;
      for (int64_t t = first; t < p.tiles && !*gu; t += step) {
        for (int c0 = 0; c0 < p.kblocks && !*gu; c0 += p.chunk) {
          const int n = (min(c0 + p.chunk, p.kblocks) - c0) * p.nseg;
          if (!bar_wait(tempty0 + 8 * buf, tphase ^ 1, gu, limit, &g_gemm_fault)) break;
          fence_after();
          const uint32_t d = tmem + buf * 256;
          for (int it = 0; it < n; ++it) {
            if (!bar_wait(full0 + 8 * s, phase, gu, limit, &g_gemm_fault)) break;
            fence_after();
            const uint32_t a = smem_u32(ring + s * stage_bytes);
            const uint64_t da = tile_desc(a, p.p_inner), dq = tile_desc(a + p.a_bytes, p.q_inner);
  #pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk)
              mma<CG>(d, da + kk * step_p, dq + kk * step_q, p.idesc, it > 0 || kk > 0);
            commit<CG>(empty0 + 8 * s);
            if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
          }
          if (*gu) break;
          commit<CG>(tfull0 + 8 * buf);
          if (++buf == 2) buf = 0, tphase ^= 1;
        }
      }
    }
  }
  __syncthreads();
  if (gave_up) {
    // copies and MMAs of this CTA that are still in flight end within microseconds
    const uint64_t t0 = now_ns();
    while (now_ns() - t0 < 20000000ull) {
    }
  }
  fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  if (warp == kEpiWarps) {
    fence_after();
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (EncodeTiledFn) nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// Boxes of 64 k x `box_rows` rows (K-major) or 64 rows x 64 k (MN-major).
bool encode(CUtensorMap* m, const TcOperand& o, int f16, int planes, int64_t batch, int64_t rows, int64_t K, int box_rows) {
  const EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const int64_t inner = o.rows_inner ? rows : K, outer = o.rows_inner ? K : rows;
  const int64_t nb = o.bcast ? 1 : batch;
  const cuuint64_t dims[4] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)nb, (cuuint64_t)planes};
  // an axis of one element may carry any stride: give it a legal one
  const cuuint64_t s1 = (cuuint64_t)o.pitch * 2, s2 = nb > 1 ? (cuuint64_t)o.batch_stride * 2 : s1,
                   s3 = planes > 1 ? (cuuint64_t)o.plane_stride * 2 : s1;
  const cuuint64_t strides[3] = {s1, s2, s3};
  const cuuint32_t box[4] = {64, (cuuint32_t)(o.rows_inner ? 64 : box_rows), 1, 1}, ones[4] = {1, 1, 1, 1};
  return fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(o.p), dims,
            strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool vec16(const void* p, int64_t elt, int64_t bs, int64_t is, int64_t js, int64_t plane) {
  return js == 1 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && bs * elt % 16 == 0 && is * elt % 16 == 0 &&
         plane * elt % 16 == 0;
}

template <int CG, bool JOIN, typename OUT>
cudaError_t launch_t(const CUtensorMap& mp, const CUtensorMap& mq, TcParams p, int sms, cudaStream_t s) {
  typedef typename OutOf<OUT>::T T;
  const int staging = kEpiWarps * 32 * (32 * (int)sizeof(T) + 16), stage = p.a_bytes + p.b_bytes;
  int stages = (kSmemMax - 1024 - 512 - staging) / stage;
  p.stages = stages > kMaxStages ? kMaxStages : stages;
  const size_t smem = 1024 + (size_t)p.stages * stage + staging;
  auto kern = gemm_tc_kernel<CG, JOIN, OUT>;
  static int cache[64];
  int occ = 0;
  cudaError_t e = kernel_occupancy(kern, kThreads, smem, cache, &occ);
  if (e != cudaSuccess) return e;
  const int64_t want = p.tiles * CG, cap = sms / CG * CG;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(want < cap ? want : cap));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, mp, mq, p);
}

template <int CG>
cudaError_t launch_cg(const TcProblem& t, const CUtensorMap& mp, const CUtensorMap& mq, const TcParams& p, int sms,
                      cudaStream_t s) {
  if (t.kind == kOne) {
    if (t.out == B2C_BF16) return launch_t<CG, false, __nv_bfloat16>(mp, mq, p, sms, s);
    if (t.out == B2C_F16) return launch_t<CG, false, __half>(mp, mq, p, sms, s);
    return cudaErrorInvalidValue;
  }
  if (t.out == B2C_F32) return launch_t<CG, true, float>(mp, mq, p, sms, s);
  if (t.out == B2C_F16) return launch_t<CG, true, __half>(mp, mq, p, sms, s);
  if (t.out == kOutHalves) return launch_t<CG, true, Halves>(mp, mq, p, sms, s);
  return cudaErrorInvalidValue;
}

bool inject_timeout() {
  const char* t = getenv("B2C_GEMM_INJECT_TIMEOUT");
  return t && strcmp(t, "1") == 0;
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
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  TcParams p{};
  p.I = t.I;
  p.J = t.J;
  p.kblocks = (int)((t.K + BK - 1) / BK);
  const int planes = t.kind == kOne ? 1 : t.kind == kHalves ? 2 : 3;
  static const int seg2[3][2] = {{1, 0}, {0, 1}, {0, 0}};
  static const int seg3[6][2] = {{2, 0}, {1, 1}, {0, 2}, {1, 0}, {0, 1}, {0, 0}};
  p.nseg = t.kind == kOne ? 1 : t.kind == kHalves ? 3 : 6;
  for (int g = 0; g < p.nseg; ++g) {
    p.seg_p[g] = t.kind == kOne ? 0 : t.kind == kHalves ? seg2[g][0] : seg3[g][0];
    p.seg_q[g] = t.kind == kOne ? 0 : t.kind == kHalves ? seg2[g][1] : seg3[g][1];
  }
  p.chunk = t.kind == kOne ? p.kblocks : kChunk;
  // a pair's 256 x 256 tile where there is at least half a wave of them
  const int64_t big = ((t.I + 255) / 256) * ((t.J + 255) / 256) * t.batch;
  const bool pair = t.I > 128 && t.J > 128 && big * 4 >= sms;
  const int CG = pair ? 2 : 1;
  if (pair) {
    p.BN = 256;
  } else if (t.sym) {
    p.BN = 128;
  } else {
    const int64_t ti = (t.I + 127) / 128;
    p.BN = 256;
    while (p.BN > 32 && (p.BN / 2 >= t.J || ti * ((t.J + p.BN - 1) / p.BN) * t.batch < sms)) p.BN /= 2;
  }
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
  p.a_bytes = BM * BK * 2;
  p.b_bytes = (p.q_inner ? (p.share + 63) / 64 * 64 : p.share) * BK * 2;
  p.idesc = mma_idesc(t.f16, p.p_inner, p.q_inner, BM * CG, p.BN);
  p.e = t.e;
  p.polar = t.polar;
  p.res_kind = t.res;
  p.y_plane = t.y_plane;
  p.res_plane = t.res_plane;
  const int64_t osize = t.out == B2C_F32 ? 4 : 2, rsize = t.res == B2C_F32 ? 4 : 2;
  p.y_vec = vec16(t.e.y.p, osize, t.e.y.bs, t.e.y.is, t.e.y.js, t.y_plane);
  p.pre_vec = vec16(t.e.pre.p, osize, t.e.pre.bs, t.e.pre.is, t.e.pre.js, 0);
  p.res_vec = t.e.res.p && vec16(t.e.res.p, rsize, t.e.res.bs, t.e.res.is, t.e.res.js, t.res_plane);
  p.inject = inject_timeout();
  CUtensorMap mp, mq;
  if (!encode(&mp, t.P, t.f16, planes, t.batch, t.I, t.K, BM) ||
      !encode(&mq, t.Q, t.f16, planes, t.batch, t.J, t.K, p.share))
    return cudaErrorInvalidValue;
  return pair ? launch_cg<2>(t, mp, mq, p, sms, s) : launch_cg<1>(t, mp, mq, p, sms, s);
}

cudaError_t gemm_take_fault(unsigned int* fault) {
  unsigned int f = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&f, g_gemm_fault, sizeof(unsigned int));
  if (e != cudaSuccess) return e;
  *fault |= f;
  return cudaMemcpyToSymbol(g_gemm_fault, &zero, sizeof(unsigned int));
}

}  // namespace b2c
