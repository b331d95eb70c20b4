// Products with an epilogue on the tensor cores: D[i, j] = sum_k P[i, k]
// Q[j, k] with 16-bit factors and 32-bit sums (tcgen05.mma kind::f16, operands
// by TMA, accumulators in tensor memory).
//
// A pair of CTAs (two SMs) computes a 256 x 256 tile (cta_group::2): each CTA
// holds 128 rows of P and 128 of Q's 256 in shared memory and 128 x 256 of D
// in its tensor memory. The pairs are persistent, one CTA an SM, and tensor
// memory holds two accumulators, so the epilogue of a tile runs under the MMAs
// of the next. Where D is too small for that, single CTAs compute 128 x BN
// tiles, several to an SM, and k may be split over a cluster of up to 8 of
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
// shared memory holds all planes, each loaded once for all its products.
#include <cmath>
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
constexpr int kEpiWarps = 8;      // of a pair's CTA
constexpr int kThreads = (kEpiWarps + 4) * 32;  // the last warpgroup: loads, products, two idle warps
// Registers: 384 x 168 at launch = 128 x 72 + 256 x 216 after the split.
constexpr int kRegsFew = 72, kRegsMany = 216;
constexpr int kMaxStages = 8;
constexpr int kABytes = BM * BK * 2;  // one plane of P's rows in a slice
constexpr int kSmemMax = 232448;

struct TcParams {
  int64_t I, J, tiles;
  int tiles_i, tiles_j, band;
  int kblocks;
  int BN, share, split, stages, b_bytes, stage_bytes, tmem_cols;
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

// After a wait that ran out: copies and MMAs still in flight end within microseconds.
__device__ __forceinline__ void settle() {
  const uint64_t t0 = now_ns();
  while (now_ns() - t0 < 20000000ull) {
  }
}

// The plane pairs of a product, smallest first.
template <int PLANES>
struct Segs;
template <>
struct Segs<1> {
  static constexpr int N = 1;
  static __host__ __device__ constexpr int p(int) { return 0; }
  static __host__ __device__ constexpr int q(int) { return 0; }
};
template <>
struct Segs<2> {  // lo hi, hi lo, hi hi
  static constexpr int N = 3;
  static __host__ __device__ constexpr int p(int g) { return g == 0; }
  static __host__ __device__ constexpr int q(int g) { return g == 1; }
};
template <>
struct Segs<3> {  // lo hi, mid mid, hi lo, mid hi, hi mid, hi hi
  static constexpr int N = 6;
  static __host__ __device__ constexpr int p(int g) { return g == 0 ? 2 : g == 1 || g == 3 ? 1 : 0; }
  static __host__ __device__ constexpr int q(int g) { return g == 2 ? 2 : g == 1 || g == 4 ? 1 : 0; }
};

// One slice: every plane of this CTA's rows of P, then of Q.
template <int CG, int PLANES>
__device__ __forceinline__ void load_slice(const TcParams& p, const CUtensorMap* map_p, const CUtensorMap* map_q, uint32_t at,
                                           int i0, int j0, int kb, int bp, int bq, uint32_t bar) {
#pragma unroll
  for (int g = 0; g < PLANES; ++g, at += kABytes) {
    if (p.p_inner) {
      tma_load<CG>(at, map_p, i0, kb * BK, bp, g, bar);
      tma_load<CG>(at + 8192, map_p, i0 + 64, kb * BK, bp, g, bar);
    } else {
      tma_load<CG>(at, map_p, kb * BK, i0, bp, g, bar);
    }
  }
#pragma unroll
  for (int g = 0; g < PLANES; ++g, at += p.b_bytes) {
    if (p.q_inner) {
      for (int h = 0; h < p.b_bytes / 8192; ++h) tma_load<CG>(at + h * 8192, map_q, j0 + 64 * h, kb * BK, bq, g, bar);
    } else {
      tma_load<CG>(at, map_q, kb * BK, j0, bq, g, bar);
    }
  }
}

// What the issuing thread needs of every slice: descriptors of stage 0 and the
// steps to the next 16 values of k, kept in registers (the thread must not be
// slower than 4 MMAs of 32 clocks).
template <int CG, int PLANES>
struct Multiplier {
  uint64_t dp, dq;
  uint32_t step_p, step_q, plane_q, stage, idesc;
  __device__ __forceinline__ Multiplier(const TcParams& p, uint32_t ring) {
    dp = tile_desc(ring, p.p_inner);
    dq = tile_desc(ring + PLANES * kABytes, p.q_inner);
    step_p = p.p_inner ? 2048 >> 4 : 32 >> 4;
    step_q = p.q_inner ? 2048 >> 4 : 32 >> 4;
    plane_q = p.b_bytes >> 4;
    stage = p.stage_bytes >> 4;
    idesc = p.idesc;
  }
  // The products of stage s into the accumulator at d; fresh: its first ones.
  __device__ __forceinline__ void slice(uint32_t s, uint32_t d, bool fresh) const {
    typedef Segs<PLANES> S;
#pragma unroll
    for (int g = 0; g < S::N; ++g) {
      const uint64_t a = dp + s * stage + S::p(g) * (kABytes >> 4), q = dq + s * stage + S::q(g) * plane_q;
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) mma<CG>(d, a + kk * step_p, q + kk * step_q, idesc, g || kk ? 1u : !fresh);
    }
  }
};

// ---------------------------------------------------------------------------
// pairs of CTAs
// ---------------------------------------------------------------------------

template <int PLANES, typename OUT>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ TcParams p) {
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 5];  // the last: nothing arrives on it
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  typedef typename OutOf<OUT>::T T;
  constexpr bool JOIN = PLANES > 1;
  constexpr int kStage = 32 * (32 * sizeof(T) + 16);  // one warp's staging rows
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  unsigned char* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  unsigned char* staging = ring + p.stages * p.stage_bytes;
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
      bar_init(tempty0 + 8 * s, kEpiWarps * 2);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kEpiWarps) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    fence_before();
  }
  __syncthreads();
  cluster_sync();
  fence_after();
  const uint32_t tmem = tmem_slot;
  const int64_t first = blockIdx.x / 2, step = gridDim.x / 2;
  volatile int* gu = &gave_up;
  const int per = JOIN ? 1 : p.kblocks;  // slices of one accumulator

  if (warp < kEpiWarps) {
    if constexpr (JOIN) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMany));
    // ---- epilogue: warps w and w + 4 share the rows 32 (w % 4).., and take every other 32 columns ----
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t lead_tempty0 = map_rank(tempty0, 0);
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    unsigned char* stage = staging + warp * kStage;
    uint32_t buf = 0, tphase = 0;
    bool ok = true;
    const float bad = __int_as_float(0x7fffffff);
    if (p.inject && blockIdx.x == 0) ok = __all_sync(kFull, bar_wait(never, 0, gu, limit, &g_gemm_fault));
    for (int64_t t = first; t < p.tiles; t += step) {
      const Tile o = tile_at<2>(p, t);
      const int64_t i = o.i + rank * BM + quad * 32;
      const int rows = clamp32(p.I - i);
      if constexpr (JOIN) {
        float acc[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[q][c] = 0.f;
        for (int kb = 0; kb < p.kblocks; ++kb) {
          ok = __all_sync(kFull, ok && bar_wait(tfull0 + 8 * buf, tphase, gu, limit, &g_gemm_fault));
          fence_after();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[32];
            tmem_row32(lanes + buf * 256 + (2 * q + half) * 32, v);
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[q][c] += v[c];
          }
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive_cluster(lead_tempty0 + 8 * buf);
          if (++buf == 2) buf = 0, tphase ^= 1;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = (2 * q + half) * 32;
          if (!ok) {
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[q][c] = bad;
          }
          epilogue32<OUT>(acc[q], p, o.b, i, o.j + col, rows, clamp32(p.J - o.j - col), o.mirror, stage, lane);
        }
      } else {
        ok = __all_sync(kFull, ok && bar_wait(tfull0 + 8 * buf, tphase, gu, limit, &g_gemm_fault));
        fence_after();
        for (int col = half * 32; col < 256; col += 64) {
          float v[32];
          tmem_row32(lanes + buf * 256 + col, v);
          if (col + 64 >= 256) {  // the last of this warp's columns: the accumulator is free
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
        if (++buf == 2) buf = 0, tphase ^= 1;
      }
    }
  } else {
    if constexpr (JOIN) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
    if (warp == kEpiWarps && lane == 0) {
      // ---- loads ----
      const uint32_t lead_full0 = map_rank(full0, 0);
      uint32_t s = 0, phase = 0;
      for (int64_t t = first; t < p.tiles && !*gu; t += step) {
        const Tile o = tile_at<2>(p, t);
        const int i0 = (int)(o.i + rank * BM), j0 = (int)(o.j + rank * p.share);
        const int bp = p.p_bcast ? 0 : (int)o.b, bq = p.q_bcast ? 0 : (int)o.b;
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!bar_wait(empty0 + 8 * s, phase ^ 1, gu, limit, &g_gemm_fault)) break;
          if (rank == 0) bar_expect(full0 + 8 * s, 2 * p.stage_bytes);
          load_slice<2, PLANES>(p, &map_p, &map_q, smem_u32(ring + s * p.stage_bytes), i0, j0, kb, bp, bq, lead_full0 + 8 * s);
          if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
        }
      }
    } else if (warp == kEpiWarps + 1 && rank == 0 && lane == 0) {
      // ---- products ----
      const Multiplier<2, PLANES> mul(p, smem_u32(ring));
      uint32_t s = 0, phase = 0, buf = 0, tphase = 0;
      for (int64_t t = first; t < p.tiles && !*gu; t += step) {
        for (int k0 = 0; k0 < p.kblocks; k0 += per) {
          if (!bar_wait(tempty0 + 8 * buf, tphase ^ 1, gu, limit, &g_gemm_fault)) break;
          fence_after();
          for (int kb = 0; kb < per; ++kb) {
            if (!bar_wait(full0 + 8 * s, phase, gu, limit, &g_gemm_fault)) break;
            fence_after();
            mul.slice(s, tmem + buf * 256, kb == 0);
            commit<2>(empty0 + 8 * s);
            if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
          }
          if (*gu) break;
          commit<2>(tfull0 + 8 * buf);
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
  if (warp == kEpiWarps) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---------------------------------------------------------------------------
// single CTAs, one tile each, k split over a cluster
// ---------------------------------------------------------------------------

// JOIN: one CTA an SM with eight epilogue warps, so that a slice's planes fit
// twice; otherwise two CTAs with four.
template <int PLANES>
struct Solo {
  static constexpr bool JOIN = PLANES > 1;
  static constexpr int EPI = JOIN ? 8 : 4;
  static constexpr int NT = (EPI + 2) * 32;
  static constexpr int CTAS = JOIN ? 1 : 2;
  static constexpr int SMEM = JOIN ? kSmemMax - 1024 : 113 * 1024;
};

template <int PLANES, typename OUT>
__global__ void __launch_bounds__(Solo<PLANES>::NT, Solo<PLANES>::CTAS)
    gemm_solo_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ TcParams p) {
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 5];  // the last: nothing arrives on it
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  typedef typename OutOf<OUT>::T T;
  constexpr bool JOIN = PLANES > 1;
  constexpr int EPI = Solo<PLANES>::EPI, GROUPS = EPI / 4, SLICES = JOIN ? 4 / GROUPS : 1;
  constexpr int kStage = 32 * (32 * sizeof(T) + 16);
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
  volatile int* gu = &gave_up;
  const int quad = warp & 3, group = warp >> 2;
  const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
  const int64_t i = o.i + quad * 32;
  const int rows = clamp32(p.I - i), pitch = p.BN + 4;
  float* partial = reinterpret_cast<float*>(ring);
  unsigned char* stage = ring + (split > 1 ? BM * pitch * 4 : 0) + warp * kStage;

  if (warp < EPI) {
    bool ok = true;
    if (p.inject && blockIdx.x == 0) ok = __all_sync(kFull, bar_wait(never, 0, gu, limit, &g_gemm_fault));
    float acc[SLICES][32];
    if constexpr (JOIN) {
#pragma unroll
      for (int q = 0; q < SLICES; ++q)
#pragma unroll
        for (int c = 0; c < 32; ++c) acc[q][c] = 0.f;
      uint32_t buf = 0, tphase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
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
    // every product is done: the ring is free for partial sums and staging (after a wait that ran out, once what is
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
        if (split > 1) {
          float4* at = reinterpret_cast<float4*>(partial + (quad * 32 + lane) * pitch + col);
#pragma unroll
          for (int c = 0; c < 8; ++c) at[c] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
        } else {
          epilogue32<OUT>(v, p, o.b, i, o.j + col, rows, clamp32(p.J - o.j - col), o.mirror, stage, lane);
        }
      }
    }
  } else if (warp == EPI && lane == 0) {
    // ---- loads ----
    uint32_t s = 0, phase = 0;
    const int bp = p.p_bcast ? 0 : (int)o.b, bq = p.q_bcast ? 0 : (int)o.b;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!bar_wait(empty0 + 8 * s, phase ^ 1, gu, limit, &g_gemm_fault)) break;
      bar_expect(full0 + 8 * s, p.stage_bytes);
      load_slice<1, PLANES>(p, &map_p, &map_q, smem_u32(ring + s * p.stage_bytes), (int)o.i, (int)o.j, kb, bp, bq, full0 + 8 * s);
      if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
    }
  } else if (warp == EPI + 1 && lane == 0) {
    // ---- products ----
    const Multiplier<1, PLANES> mul(p, smem_u32(ring));
    uint32_t s = 0, phase = 0, buf = 0, tphase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (JOIN && !bar_wait(tempty0 + 8 * buf, tphase ^ 1, gu, limit, &g_gemm_fault)) break;
      if (!bar_wait(full0 + 8 * s, phase, gu, limit, &g_gemm_fault)) break;
      fence_after();
      mul.slice(s, tmem + buf * p.BN, JOIN || kb == kb0);
      commit<1>(empty0 + 8 * s);
      if (++s == (uint32_t)p.stages) s = 0, phase ^= 1;
      if (JOIN || kb == kb1 - 1) commit<1>(tfull0 + 8 * buf);
      if (JOIN && ++buf == 2) buf = 0, tphase ^= 1;
    }
  }
  if (split > 1) {
    __syncwarp();
    cluster_sync();
    // the tile's 32 x 32 pieces are dealt over the cluster's epilogue warps
    if (warp < EPI) {
      for (int u = rank * EPI + warp; u < 4 * (p.BN / 32); u += split * EPI) {
        const int pq = u & 3, col = (u >> 2) * 32;
        const uint32_t at = smem_u32(partial + (pq * 32 + lane) * pitch + col);
        float v[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = 0.f;
        for (int q = 0; q < split; ++q) {
          const uint32_t peer = map_rank(at, q);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            float x, y, z, w;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x), "=f"(y), "=f"(z), "=f"(w) : "r"(peer + c * 4) : "memory");
            v[c] += x, v[c + 1] += y, v[c + 2] += z, v[c + 3] += w;
          }
        }
        const int64_t ii = o.i + pq * 32;
        epilogue32<OUT>(v, p, o.b, ii, o.j + col, clamp32(p.I - ii), clamp32(p.J - o.j - col), o.mirror, stage, lane);
      }
    }
    __syncwarp();
    cluster_sync();  // peers' partial sums stay until they have been read
  }
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

template <typename Kern>
cudaError_t launch_in_clusters(Kern kern, int64_t ctas, int cluster, int threads, size_t smem, cudaStream_t s,
                               const CUtensorMap& mp, const CUtensorMap& mq, const TcParams& p) {
  if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, mp, mq, p);
}

template <int PLANES, typename OUT>
cudaError_t launch_pair(const CUtensorMap& mp, const CUtensorMap& mq, TcParams p, int sms, cudaStream_t s) {
  typedef typename OutOf<OUT>::T T;
  const int staging = kEpiWarps * 32 * (32 * (int)sizeof(T) + 16);
  const int stages = (kSmemMax - 1024 - 512 - staging) / p.stage_bytes;
  p.stages = stages > kMaxStages ? kMaxStages : stages;
  const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + staging;
  auto kern = gemm_pair_kernel<PLANES, OUT>;
  static int cache[64];
  int occ = 0;
  cudaError_t e = kernel_occupancy(kern, kThreads, smem, cache, &occ);
  if (e != cudaSuccess) return e;
  const int64_t want = p.tiles * 2, cap = sms / 2 * 2;
  return launch_in_clusters(kern, want < cap ? want : cap, 2, kThreads, smem, s, mp, mq, p);
}

template <int PLANES, typename OUT>
cudaError_t launch_solo(const CUtensorMap& mp, const CUtensorMap& mq, TcParams p, int, cudaStream_t s) {
  typedef typename OutOf<OUT>::T T;
  constexpr int NT = Solo<PLANES>::NT;
  const int staging = Solo<PLANES>::EPI * 32 * (32 * (int)sizeof(T) + 16) + (p.split > 1 ? BM * (p.BN + 4) * 4 : 0);
  const int per = (p.kblocks + p.split - 1) / p.split;
  int stages = (Solo<PLANES>::SMEM - 1024 - 512) / p.stage_bytes;
  if (stages > kMaxStages) stages = kMaxStages;
  p.stages = stages > per ? per : stages;
  size_t smem = (size_t)p.stages * p.stage_bytes;
  if (smem < (size_t)staging) smem = staging;
  smem += 1024;
  p.tmem_cols = 32;
  while (p.tmem_cols < (PLANES > 1 ? 2 : 1) * p.BN) p.tmem_cols *= 2;
  auto kern = gemm_solo_kernel<PLANES, OUT>;
  static int cache[64];
  int occ = 0;
  cudaError_t e = kernel_occupancy(kern, NT, smem, cache, &occ);
  if (e != cudaSuccess) return e;
  return launch_in_clusters(kern, p.tiles * p.split, p.split, NT, smem, s, mp, mq, p);
}

template <bool PAIR, int PLANES, typename OUT>
cudaError_t launch_form(const CUtensorMap& mp, const CUtensorMap& mq, const TcParams& p, int sms, cudaStream_t s) {
  if constexpr (PAIR) return launch_pair<PLANES, OUT>(mp, mq, p, sms, s);
  else return launch_solo<PLANES, OUT>(mp, mq, p, sms, s);
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

// Estimated clocks of an SM: its share of tiles times the longer of loading a
// slice (about 40 bytes a clock and SM from L2) and multiplying it (128 x 16 x
// 16 values a clock, and 128 bytes of shared memory a clock), plus what a
// launch, a join over a cluster and an epilogue cost. Only the order of these
// estimates matters: on 1000 x 777 x 1301 float32 the forms take 26 to 80 us, on
// 16 x 4096 x 16384 f16 29 to 44 us, and the estimate's choice is the first.
Form choose_form(const TcProblem& t, int kblocks, int planes, int nseg, int sms) {
  Form best{0, 0, 0, 1e300};
  const int64_t ti = (t.I + BM - 1) / BM;
  for (int BN = t.sym ? 128 : 32; BN <= 128; BN *= 2) {
    if (!t.sym && BN > 32 && BN / 2 >= t.J) break;
    const int64_t tj = (t.J + BN - 1) / BN, tiles = t.batch * (t.sym ? ti * (ti + 1) / 2 : ti * tj);
    for (int split = 1; split <= 8 && split <= kblocks; split *= 2) {
      const double load = planes * (16384.0 + BN * 128.0) / 40, mul = nseg * 4.0 * fmax(BN / 2.0, (128 + BN) / 4.0);
      const double slice = fmax(load, mul), ctas = ceil((double)tiles * split / sms);
      const double c = ctas * ((kblocks + split - 1) / split * slice + BN * 12.0) + 3000 + (split > 1 ? 1500 : 0);
      if (c < best.clocks) best = Form{0, BN, split, c};
    }
  }
  if (t.I > BM && t.J > 128) {
    const int64_t ti2 = (t.I + 255) / 256, tj2 = (t.J + 255) / 256;
    const int64_t tiles = t.batch * (t.sym ? ti2 * (ti2 + 1) / 2 : ti2 * tj2);
    const double slice = fmax(planes * 32768.0 / 40, nseg * 4.0 * 128);
    const double c = ceil(2.0 * tiles / sms) * kblocks * slice + 4000 + 3000;
    if (c < best.clocks) best = Form{1, 256, 1, c};
  }
  return best;
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
  p.y_vec = vec16(t.e.y.p, osize, t.e.y.bs, t.e.y.is, t.e.y.js, t.y_plane);
  p.pre_vec = vec16(t.e.pre.p, osize, t.e.pre.bs, t.e.pre.is, t.e.pre.js, 0);
  p.res_vec = t.e.res.p && vec16(t.e.res.p, rsize, t.e.res.bs, t.e.res.is, t.e.res.js, t.res_plane);
  p.inject = inject_timeout();
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
