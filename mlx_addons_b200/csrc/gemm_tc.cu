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
// Warps of a pair's CTA: its epilogue warps, then a warpgroup of loads,
// products and two idle warps. Joined sums stay in registers, 64 a thread with
// sixteen epilogue warps (eight, with 128, took 1.3 times as long over a tile).
template <int PLANES>
struct Pair {
  static constexpr bool JOIN = PLANES > 1;
  static constexpr int EPI = JOIN ? 16 : 8;
  static constexpr int NT = (EPI + 4) * 32;
  // registers where JOIN: 640 x 96 at launch = 128 x 64 + 512 x 104 after the split
  static constexpr int FEW = 64, MANY = 104;
};
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
  int res_kind, y_vec, pre_vec, res_vec, bias_vec;
  int64_t y_plane, res_plane;
  int inject, chained;
};

// ---------------------------------------------------------------------------
// epilogue
// ---------------------------------------------------------------------------

struct Halves {};  // output tag: two f16 planes

template <typename OUT>
struct OutOf { typedef OUT T; };
template <>
struct OutOf<Halves> { typedef __half T; };

// Eight neighbours along i or j: v = alpha D, r = the addends; see TcPolarMode.
template <bool ALONG_I>
__device__ __forceinline__ void polar8(float (&v)[8], const float (&r)[8], const TcPolar& q, float beta, int64_t b, int64_t i,
                                       int64_t j, int n) {
  const float f = q.r ? q.r[b] : 1.f;
  const float* d = q.d_in + b * q.side;
  float* out = q.d_out + b * q.side;
  const int64_t along = ALONG_I ? i : j, across = ALONG_I ? j : i, diag = across - along;  // which of them is diagonal
  if (q.mode == kPolarS) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] *= f * f;
      if (k == diag && k < n) out[across] = v[k] * q.k, v[k] = 0.f;
    }
    return;
  }
  // the diagonal enters by the row, the column or both
  const bool by_along = q.mode == kPolarP || q.mode == (ALONG_I ? kPolarXi : kPolarXj);
  const bool by_across = q.mode == kPolarP || q.mode == (ALONG_I ? kPolarXj : kPolarXi);
  const float da = by_across ? d[across] : 0.f;
  float w[8] = {};
  if (by_along) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) w[k] = d[along + k];
  }
  if (q.mode == kPolarP) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k == diag && k < n) out[across] = fmaf(q.k2, v[k], da * fmaf(q.k3, da, q.k4)), v[k] = 0.f;
      else v[k] = fmaf(fmaf(q.k, da + w[k], beta), r[k], v[k]);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = f * fmaf(beta * (q.k + da + w[k]), r[k], v[k]);
}

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
__device__ __forceinline__ void polar_row32(float (&v)[32], const float (&r)[32], const TcPolar& q, const GemmEpilogue& e,
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

// The epilogue of a pair's 16-bit outputs, 32 columns (v) of row i + lane in
// every lane. The main loop of a pair takes all of its shared memory's
// bandwidth (64 bytes a clock arriving, 64 read by the tensor cores), so what
// passes through shared memory here is the rounded outputs alone; with the
// sums staged in float32 (finish32) four 4096 x 4096 orthogonalisation steps take 1.28
// times as long.
// rows / cols: how many of the 32 x 32 exist (either may be <= 0).
template <typename T>
__device__ __forceinline__ void finish_row32(float (&v)[32], const TcParams& p, int64_t b, int64_t i, int64_t j, int rows,
                                             int cols, bool mirror, unsigned char* stage, int lane) {
  static_assert(sizeof(T) == 2, "16-bit outputs");
  const GemmEpilogue& e = p.e;
  if (rows <= 0 || cols <= 0) return;
#pragma unroll
  for (int c = 0; c < 32; ++c) v[c] *= e.alpha;
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
  apply_act<true>(v, e.act);
  float r[32] = {};
  if (e.res.p && lane < rows) {
    const int64_t off = b * e.res.bs + (i + lane) * e.res.is + j * e.res.js;
    const int vec = p.res_vec && e.res.js == 1;
    if (p.res_kind == B2C_BF16) load_res(r, static_cast<const __nv_bfloat16*>(e.res.p) + off, e.res.js, cols, vec);
    else load_res(r, static_cast<const __half*>(e.res.p) + off, e.res.js, cols, vec);
  }
  if (p.polar.mode != kPolarNone) {
    polar_row32(v, r, p.polar, e, b, i, j, rows, cols, lane);
  } else if (e.res.p) {
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] = fmaf(e.beta, r[c], v[c]);
  }
  store_tile<T>(v, e.y, b, i, j, rows, cols, p.y_vec, stage, lane);
  if (mirror) store_tile<T>(v, GemmView{e.y.p, e.y.bs, e.y.js, e.y.is}, b, i, j, rows, cols, 0, stage, lane);
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


// The epilogue of a block of D whose sums lie in shared memory, row by row:
// the sums leave tensor memory with a row in every lane, but addends and outputs are
// read and written along their rows. Kept small on purpose, since a kernel
// that runs once over a tile fetches every instruction from memory (with 32 columns a
// lane, unrolled, 32 x 32 values took 2,600 clocks, 8,400 with an addend).

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* at, int64_t js, int n, bool vec) {
  if (vec) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < 8 / PER; ++u) {
      const uint4 w = *reinterpret_cast<const uint4*>(at + u * PER);
      const T* q = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int c = 0; c < PER; ++c) v[u * PER + c] += to_f32(q[c]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < n) v[c] += to_f32(at[c * js]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* at, const float (&v)[8], int n, bool vec) {
  if (vec) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < 8 / PER; ++u) {
      uint4 w;
      T* q = reinterpret_cast<T*>(&w);
#pragma unroll
      for (int c = 0; c < PER; ++c) q[c] = from_f32<T>(v[u * PER + c]);
      *reinterpret_cast<uint4*>(at + u * PER) = w;
    }
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < n) at[c] = from_f32<T>(v[c]);
  }
}

// n (up to 8) addends at stride js.
__device__ __forceinline__ void load_res8(float (&r)[8], const TcParams& p, int64_t at, int64_t js, int n, bool vec) {
  const void* base = p.e.res.p;
  if (p.res_kind == B2C_F32) load8(r, static_cast<const float*>(base) + at, js, n, vec);
  else if (p.res_kind == B2C_BF16) load8(r, static_cast<const __nv_bfloat16*>(base) + at, js, n, vec);
  else load8(r, static_cast<const __half*>(base) + at, js, n, vec);
  if (p.res_kind == kOutHalves) load8(r, static_cast<const __half*>(base) + p.res_plane + at, js, n, vec);
}

template <bool FAST>
__device__ __forceinline__ void act8(float (&v)[8], int act) {
  switch (act) {
    case B2C_ACT_RELU:
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = act_f32<FAST>(v[k], B2C_ACT_RELU);
      break;
    case B2C_ACT_GELU:
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = act_f32<FAST>(v[k], B2C_ACT_GELU);
      break;
    case B2C_ACT_GELU_TANH:
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = act_f32<FAST>(v[k], B2C_ACT_GELU_TANH);
      break;
    case B2C_ACT_SILU:
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = act_f32<FAST>(v[k], B2C_ACT_SILU);
      break;
    default: break;
  }
}

// The addends of 8 neighbours, zeros where there are none.
template <bool ALONG_I>
__device__ __forceinline__ void addends8(float (&x)[8], const TcParams& p, int64_t b, int64_t i, int64_t j, int n) {
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = 0.f;
  const GemmEpilogue& e = p.e;
  if (e.res.p)
    load_res8(x, p, b * e.res.bs + i * e.res.is + j * e.res.js, ALONG_I ? e.res.is : e.res.js, n, n == 8 && p.res_vec);
}

// The sums v (results on return) and addends x of n (up to 8) neighbours from
// (i, j) along the axis that has unit stride in y and pre: i (ALONG_I) or j.
template <typename OUT, bool ALONG_I>
__device__ __forceinline__ void finish8(const TcParams& p, int64_t b, int64_t i, int64_t j, int n, float (&v)[8],
                                        const float (&x)[8]) {
  typedef typename OutOf<OUT>::T T;
  const GemmEpilogue& e = p.e;
  const bool whole = n == 8;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] *= e.alpha;
  if constexpr (!std::is_same<OUT, Halves>::value) {
    if (e.bias) {
      const bool along = ALONG_I == (bool)e.bias_on_i;
      load8(v, static_cast<const T*>(e.bias) + (e.bias_on_i ? i : j), along ? 1 : 0, n, along && whole && p.bias_vec);
    }
    if (e.pre.p)
      store8(static_cast<T*>(e.pre.p) + b * e.pre.bs + i * e.pre.is + j * e.pre.js, v, n, whole && p.pre_vec);
    act8<sizeof(T) == 2>(v, e.act);
  }
  if (p.polar.mode != kPolarNone) {
    polar8<ALONG_I>(v, x, p.polar, e.beta, b, i, j, n);
  } else if (e.res.p) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = fmaf(e.beta, x[k], v[k]);
  }
  T* y = static_cast<T*>(e.y.p) + b * e.y.bs + i * e.y.is + j * e.y.js;
  store8(y, v, n, whole && p.y_vec);
  if constexpr (std::is_same<OUT, Halves>::value) {
    float lo[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) lo[k] = v[k] - __half2float(__float2half_rn(v[k]));
    store8(y + p.y_plane, lo, n, whole && p.y_vec);
  }
}

// The sum over the cluster, in order, of 8 values at distance `step` from `at`.
template <bool CLUSTER>
__device__ __forceinline__ void joined8(const float* at, int step, int split, float (&v)[8]) {
  if (!CLUSTER || split == 1) {
    if (CLUSTER && step == 1) {  // rows of the single CTAs' sums start on 16 bytes
      const float4 x = *reinterpret_cast<const float4*>(at), y = *reinterpret_cast<const float4*>(at + 4);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = at[k * step];
    }
    return;
  }
  const uint32_t a = smem_u32(at);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.f;
  for (int q = 0; q < split; ++q) {
    const uint32_t peer = map_rank(a, q);
    if (step == 1) {
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        float x, y, z, w;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(x), "=f"(y), "=f"(z), "=f"(w)
                     : "r"(peer + k * 4)
                     : "memory");
        v[k] += x, v[k + 1] += y, v[k + 2] += z, v[k + 3] += w;
      }
      continue;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(peer + k * step * 4) : "memory");
      v[k] += x;
    }
  }
}

// A block of sums: 2^lg_rows x 2^lg_cols of them, from row i and column j of D.
struct Block {
  int64_t b, i, j;
  float* sums;
  int pitch, lg_rows, lg_cols;
};

// Threads t0, t0 + nt, ... take a block's units of 8 neighbours along the axis
// of unit stride in y (i with ALONG_I), BATCH at a time: their addends are asked
// for together, since each is a trip to memory. With KEEP the results replace the sums.
template <typename OUT, bool CLUSTER, int BATCH, bool ALONG_I>
__device__ __forceinline__ void finish_units(const TcParams& p, const Block& o, bool keep, int t0, int nt) {
  const int total = 1 << (o.lg_rows + o.lg_cols - 3), lg = (ALONG_I ? o.lg_rows : o.lg_cols) - 3;
  const int64_t end_i = p.I, end_j = p.J;
#pragma unroll 1
  for (int u0 = t0; u0 < total; u0 += nt * BATCH) {
    float x[BATCH][8];
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const int u = u0 + q * nt, across = u >> lg, along = (u & ((1 << lg) - 1)) * 8;
      const int64_t i = o.i + (ALONG_I ? along : across), j = o.j + (ALONG_I ? across : along);
      const int64_t left = ALONG_I ? end_i - i : end_j - j;
      if (u < total && i < end_i && j < end_j) addends8<ALONG_I>(x[q], p, o.b, i, j, left < 8 ? (int)left : 8);
    }
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const int u = u0 + q * nt, across = u >> lg, along = (u & ((1 << lg) - 1)) * 8;
      const int64_t i = o.i + (ALONG_I ? along : across), j = o.j + (ALONG_I ? across : along);
      const int64_t left = ALONG_I ? end_i - i : end_j - j;
      if (u >= total || i >= end_i || j >= end_j) continue;
      float* at = o.sums + (ALONG_I ? along : across) * o.pitch + (ALONG_I ? across : along);
      float v[8];
      joined8<CLUSTER>(at, ALONG_I ? o.pitch : 1, p.split, v);
      finish8<OUT, ALONG_I>(p, o.b, i, j, left < 8 ? (int)left : 8, v, x[q]);
      if (keep) {
#pragma unroll
        for (int k = 0; k < 8; ++k) at[k * (ALONG_I ? o.pitch : 1)] = v[k];
      }
    }
  }
}

// Writes a finished block's results once more, as its transpose: the other
// half of a symmetric product. Lanes run along 16 columns and two units of rows, so
// that shared memory is read without conflicts and stores fill 32-byte sectors.
template <typename OUT>
__device__ __forceinline__ void mirror_units(const TcParams& p, const Block& o, int t0, int nt) {
  typedef typename OutOf<OUT>::T T;
  const int total = 1 << (o.lg_rows + o.lg_cols - 3);
#pragma unroll 1
  for (int u = t0; u < total; u += nt) {
    const int c = (u & 15) | (u >> 5 << 4 & ((1 << o.lg_cols) - 1));
    const int r = ((u >> 4 & 1) | (u >> (o.lg_cols + 1) << 1)) * 8;
    const int64_t i = o.j + c, j = o.i + r;
    if (i >= p.I || j >= p.J) continue;
    const int n = p.J - j < 8 ? (int)(p.J - j) : 8;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = o.sums[(r + k) * o.pitch + c];
    T* y = static_cast<T*>(p.e.y.p) + o.b * p.e.y.bs + i * p.e.y.is + j;
    store8(y, v, n, n == 8 && p.y_vec);
    if constexpr (std::is_same<OUT, Halves>::value) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] -= __half2float(__float2half_rn(v[k]));
      store8(y + p.y_plane, v, n, n == 8 && p.y_vec);
    }
  }
}

// Thread t0 of nt finishes its share of the block; with keep, for
// mirror_units, which needs a barrier in between.
template <typename OUT, bool CLUSTER, int BATCH>
__device__ __forceinline__ void finish(const TcParams& p, const Block& o, bool keep, int t0, int nt) {
  if (p.e.y.js == 1) finish_units<OUT, CLUSTER, BATCH, false>(p, o, keep, t0, nt);
  else finish_units<OUT, CLUSTER, BATCH, true>(p, o, keep, t0, nt);
}

// Asks for 32 addends of a row, to be in L2 when the epilogue reads them: a
// trip to HBM there is not hidden by anything (1000 products of 256 x 256 x 256, float32, with
// an addend: 421 us without this).
__device__ __forceinline__ void prefetch_res(const TcParams& p, int64_t b, int64_t i, int64_t j) {
  const GemmView& r = p.e.res;
  if (!r.p || r.js != 1 || i >= p.I || j >= p.J) return;
  const int64_t at = b * r.bs + i * r.is + j, size = p.res_kind == B2C_F32 ? 4 : 2;
  const char* q = static_cast<const char*>(r.p) + at * size;
  asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
  if (p.res_kind == kOutHalves) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + p.res_plane * 2));
}

// A warp's 32 x 32 values, one row a lane, through its own staging rows.
// With 33 floats a row both ways of reading it touch every bank once.
constexpr int kStagePitch = 33;
constexpr int kStageFloats = 32 * kStagePitch;  // a multiple of 4, for 16-byte units in other layouts
template <typename OUT>
__device__ __forceinline__ void finish32(const TcParams& p, const float (&v)[32], int64_t b, int64_t i, int64_t j, bool mirror,
                                         float* stage, int lane) {
#pragma unroll
  for (int c = 0; c < 32; ++c) stage[lane * kStagePitch + c] = v[c];
  __syncwarp();
  const Block o{b, i, j, stage, kStagePitch, 5, 5};
  finish<OUT, false, 1>(p, o, mirror, lane, 32);
  __syncwarp();
  if (mirror) {
    mirror_units<OUT>(p, o, lane, 32);
    __syncwarp();
  }
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
__global__ void __launch_bounds__(Pair<PLANES>::NT, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ TcParams p) {
  extern __shared__ unsigned char raw[];
  next_may_launch();
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 5];  // the last: nothing arrives on it
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  constexpr bool JOIN = PLANES > 1;
  constexpr int EPI = Pair<PLANES>::EPI, GROUPS = EPI / 4, SLICES = 8 / GROUPS;  // slices: 32 columns of a warp's rows
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
  const int per = JOIN ? 1 : p.kblocks;  // slices of one accumulator

  if (warp < EPI) {
    if constexpr (JOIN) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Pair<PLANES>::MANY));
    // ---- epilogue: warps w, w + 4, ... share the rows 32 (w % 4).. and deal out the columns ----
    const int quad = warp & 3, group = warp >> 2;
    const uint32_t lead_tempty0 = map_rank(tempty0, 0);
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    float* stage = staging + warp * kStageFloats;
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
        for (int kb = 0; kb < p.kblocks; ++kb) {
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
    if constexpr (JOIN) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Pair<PLANES>::FEW));
    if (warp == EPI && lane == 0) {
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
    } else if (warp == EPI + 1 && rank == 0 && lane == 0) {
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
  next_may_launch();
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 5];  // the last: nothing arrives on it
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  constexpr bool JOIN = PLANES > 1;
  constexpr int EPI = Solo<PLANES>::EPI, GROUPS = EPI / 4, SLICES = JOIN ? 4 / GROUPS : 1;
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
  __syncwarp();
  if (split > 1) cluster_sync();
  else __syncthreads();
  // each CTA of the cluster finishes its share of the rows
  const int nrows = BM / split, r0 = rank * nrows;
  const Block mine{o.b, o.i + r0, o.j, partial + r0 * pitch, pitch, 31 - __clz(nrows), 31 - __clz(p.BN)};
  finish<OUT, true, 1>(p, mine, o.mirror, tid, Solo<PLANES>::NT);
  if (o.mirror) {
    __syncthreads();
    mirror_units<OUT>(p, mine, tid, Solo<PLANES>::NT);
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

// Whether 8 neighbours along j (or i) can be read and written as 16-byte units.
bool vec16(const GemmView& v, bool along_i, int64_t elt, int64_t plane) {
  const int64_t unit = along_i ? v.is : v.js, other = along_i ? v.js : v.is;
  return v.p && unit == 1 && (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.bs * elt % 16 == 0 && other * elt % 16 == 0 &&
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

template <int PLANES, typename OUT>
cudaError_t launch_pair(const CUtensorMap& mp, const CUtensorMap& mq, TcParams p, int sms, cudaStream_t s) {
  constexpr int NT = Pair<PLANES>::NT;
  const int staging = Pair<PLANES>::EPI * kStageFloats * 4;
  const int stages = (kSmemMax - 1024 - 512 - staging) / p.stage_bytes;
  p.stages = stages > kMaxStages ? kMaxStages : stages;
  const size_t smem = 1024 + (size_t)p.stages * p.stage_bytes + staging;
  auto kern = gemm_pair_kernel<PLANES, OUT>;
  static int cache[64];
  int occ = 0;
  cudaError_t e = kernel_occupancy(kern, NT, smem, cache, &occ);
  if (e != cudaSuccess) return e;
  const int64_t want = p.tiles * 2, cap = sms / 2 * 2;
  return launch_in_clusters(kern, want < cap ? want : cap, 2, NT, smem, s, mp, mq, p);
}

template <int PLANES, typename OUT>
cudaError_t launch_solo(const CUtensorMap& mp, const CUtensorMap& mq, TcParams p, int sms, cudaStream_t s) {
  constexpr int NT = Solo<PLANES>::NT;
  const int sums = BM * (p.BN + 4) * 4;
  const int per = (p.kblocks + p.split - 1) / p.split;
  // all of an SM's shared memory where it gets one CTA anyway: a slice takes about 2,000 clocks to arrive
  const int room = p.tiles * p.split <= sms ? kSmemMax - 1024 : Solo<PLANES>::SMEM;
  int stages = (room - 1024 - 512) / p.stage_bytes;
  if (stages > kMaxStages) stages = kMaxStages;
  p.stages = stages > per ? per : stages;
  size_t smem = (size_t)p.stages * p.stage_bytes;
  if (smem < (size_t)sums) smem = sums;
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
      const double ctas = (double)tiles * split, on_sm = ceil(ctas / sms), at_once = fmin(on_sm, planes > 1 ? 1.0 : 2.0);
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
    // with several planes the ring holds two or three slices, and their arrival is not hidden
    const double slice = planes > 1 ? planes * 2000.0 : fmax(32768.0 / rate(2.0 * tiles), 4.0 * 128);
    const double c = ceil(2.0 * tiles / sms) * kblocks * slice + 11000;
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
  const bool along_i = t.e.y.js != 1;
  p.y_vec = vec16(t.e.y, along_i, osize, t.y_plane);
  p.pre_vec = vec16(t.e.pre, along_i, osize, 0);
  p.res_vec = vec16(t.e.res, along_i, rsize, t.res_plane);
  p.bias_vec = (reinterpret_cast<uintptr_t>(t.e.bias) & 15) == 0;
  p.inject = inject_timeout();
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
