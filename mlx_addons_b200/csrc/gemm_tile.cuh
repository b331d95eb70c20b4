// What the kernels that run products on tcgen05 share (gemm_tc.cu,
// polar_grid.cu): tiles, slices of k, epilogues, tensor maps.
#pragma once

#include <type_traits>

#include "gemm_tc.cuh"
#include "tcgen05.cuh"

namespace b2c {

namespace {

constexpr int BM = 128;          // rows of D per CTA
constexpr int BK = 64;           // depth of a slice: 128 bytes
constexpr int kMaxStages = 8;
constexpr int kABytes = BM * BK * 2;  // one plane of P's rows in a slice
constexpr int kSmemMax = 232448;

// How the operands of a product lie in a slice.
struct SliceLayout {
  int p_inner, q_inner;      // rows have unit stride (1) or k (0)
  int b_bytes, stage_bytes;  // one plane of Q's rows; all planes of both
  uint32_t idesc;
};

struct TcParams : SliceLayout {
  int64_t I, J, tiles;
  int tiles_i, tiles_j, band;
  int kblocks;
  int BN, share, split, stages, tmem_cols;
  int p_bcast, q_bcast, sym;
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
// the rows' tiles up to the one on the diagonal; those left of it are mirrored.
template <int CG>
__device__ __forceinline__ Tile tile_at(const TcParams& p, int64_t t) {
  Tile o;
  if (p.sym) {
    const int64_t w = BM * CG / p.BN, per = w * p.tiles_i * (p.tiles_i + 1) / 2;
    o.b = t / per;
    const int64_t u = t - o.b * per, h = u / w;
    int64_t r = (int64_t)((sqrt(8.0 * (double)h + 1.0) - 1.0) * 0.5);
    while (r * (r + 1) / 2 > h) --r;
    while ((r + 1) * (r + 2) / 2 <= h) ++r;
    const int64_t c = u - w * (r * (r + 1) / 2);
    o.i = r * (BM * CG);
    o.j = c * p.BN;
    o.mirror = o.j + p.BN <= o.i;
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

// The plane pairs of a product, smallest first; shift: by how many bits the sum
// so far goes down before the first product of a pair is added.
template <int PLANES>
struct Segs;
template <>
struct Segs<1> {
  static constexpr int N = 1;
  static __host__ __device__ constexpr int p(int) { return 0; }
  static __host__ __device__ constexpr int q(int) { return 0; }
  static __host__ __device__ constexpr int shift(int) { return 0; }
};
template <>
struct Segs<2> {  // lo hi, hi lo, hi hi
  static constexpr int N = 3;
  static __host__ __device__ constexpr int p(int g) { return g == 0; }
  static __host__ __device__ constexpr int q(int g) { return g == 1; }
  static __host__ __device__ constexpr int shift(int) { return 0; }
};
template <>
struct Segs<3> {  // lo hi, mid mid, hi lo, mid hi, hi mid, hi hi
  static constexpr int N = 6;
  static __host__ __device__ constexpr int p(int g) { return g == 0 ? 2 : g == 1 || g == 3 ? 1 : 0; }
  static __host__ __device__ constexpr int q(int g) { return g == 2 ? 2 : g == 1 || g == 4 ? 1 : 0; }
  // mid is held times 2^8, lo times 2^16: the first three products are 2^16 times what they stand for, the next two 2^8
  static __host__ __device__ constexpr int shift(int g) { return g == 3 || g == 5 ? 8 : 0; }
};

// One slice: every plane of this CTA's rows of P, then of Q.
template <int CG, int PLANES>
__device__ __forceinline__ void load_slice(const SliceLayout& p, const CUtensorMap* map_p, const CUtensorMap* map_q, uint32_t at,
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
  __device__ __forceinline__ Multiplier(const SliceLayout& p, uint32_t ring) {
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
      for (int kk = 0; kk < BK / 16; ++kk) {
        if (S::shift(g) && kk == 0) mma<CG, 8>(d, a, q, idesc, 1u);
        else mma<CG>(d, a + kk * step_p, q + kk * step_q, idesc, g || kk ? 1u : !fresh);
      }
    }
  }
};

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

}  // namespace

}  // namespace b2c
