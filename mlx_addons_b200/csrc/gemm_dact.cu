// Gradient of a product's epilogue: dP = dY act'(pre), its column sums (the
// bias gradient) and beta dY (the residual's), in one pass over dY and pre.
//
// Bound by HBM: it reads dY and pre and writes dP once. A CTA takes 256
// columns (8 per lane, as 16-byte accesses where alignment allows) of a band
// of rows; its 8 warps walk the band and their float32 column sums join in
// shared memory, one partial row per band.
// A second kernel adds the bands in a fixed order, so the sums do not depend
// on which CTA ran first. The sums take dP before it is rounded; dP itself is
// rounded once to the product's type, since it is an operand of the two
// products that follow.
#include "b2c_kernels.cuh"
#include "gemm.cuh"

namespace b2c {

namespace {

constexpr int kDactWarps = 8;
constexpr int kCols = 256;      // columns of a CTA: 8 per lane
constexpr int kMaxBands = 256;

// Rows of a band: one a warp, and more once that makes a thousand CTAs.
int64_t dact_band_rows(int64_t rows, int64_t N) {
  const int64_t blocks = (N + kCols - 1) / kCols;
  int64_t band = kDactWarps;
  while ((rows + band - 1) / band > kMaxBands || (rows + band - 1) / band * blocks > 1024) {
    if (band >= rows) break;
    band *= 2;
  }
  return band;
}

// VEC: every row of every array starts on 16 bytes and N is a multiple of 8;
// a lane takes 8 neighbouring columns. Otherwise it takes every 32nd.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const void* p, int64_t off, int64_t cs, int64_t c, int64_t N, float (&v)[8]) {
  const T* q = static_cast<const T*>(p) + off;
  if constexpr (VEC) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < 8 / PER; ++u) {
      const uint4 w = *reinterpret_cast<const uint4*>(q + c + u * PER);
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int k = 0; k < PER; ++k) v[u * PER + k] = to_f32(e[k]);
    }
  } else {
    // every load is issued, past the end that of c again: none waits for a branch
    T t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = q[(c + 32 * k < N ? c + 32 * k : c) * cs];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + 32 * k < N ? to_f32(t[k]) : 0.f;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(void* p, int64_t off, int64_t c, int64_t N, const float (&v)[8]) {
  T* q = static_cast<T*>(p) + off;
  if constexpr (VEC) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < 8 / PER; ++u) {
      uint4 w;
      T* e = reinterpret_cast<T*>(&w);
#pragma unroll
      for (int k = 0; k < PER; ++k) e[k] = from_f32<T>(v[u * PER + k]);
      *reinterpret_cast<uint4*>(q + c + u * PER) = w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + 32 * k < N) q[c + 32 * k] = from_f32<T>(v[k]);
  }
}

// d[k] = dy[k] act'(x[k]); one choice of act for the eight.
template <bool FAST>
__device__ __forceinline__ void slope8(float (&d)[8], const float (&dy)[8], const float (&x)[8], int act) {
  switch (act) {
    case B2C_ACT_RELU:
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] = x[k] > 0.f ? dy[k] : 0.f;
      break;
    case B2C_ACT_GELU:
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] = dy[k] * act_slope_f32<FAST>(x[k], B2C_ACT_GELU);
      break;
    case B2C_ACT_GELU_TANH:
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] = dy[k] * act_slope_f32<FAST>(x[k], B2C_ACT_GELU_TANH);
      break;
    default:
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] = dy[k] * act_slope_f32<FAST>(x[k], B2C_ACT_SILU);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kDactWarps * 32) gemm_dact_kernel(const DactParams p, int64_t band) {
  __shared__ float part[kDactWarps][kCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rows = p.batch * p.M, c0 = (int64_t)blockIdx.x * kCols, r0 = (int64_t)blockIdx.y * band;
  const int64_t c = c0 + (VEC ? lane * 8 : lane), r1 = r0 + band < rows ? r0 + band : rows;
  float sum[8] = {};
  if (c < p.N) {
    int64_t b = (r0 + warp) / p.M, i = (r0 + warp) - b * p.M;
    for (int64_t r = r0 + warp; r < r1; r += kDactWarps) {
      float dy[8], d[8];
      load8<T, VEC>(p.dY, b * p.dy_bs + i * p.dy_rs, p.dy_cs, c, p.N, dy);
      if (p.pre) {
        float x[8];
        load8<T, VEC>(p.pre, b * p.pre_bs + i * p.pre_rs, p.pre_cs, c, p.N, x);
        slope8<sizeof(T) == 2>(d, dy, x, p.act);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k] = dy[k];
      }
      if (p.dP) store8<T, VEC>(p.dP, r * p.N, c, p.N, d);
      if (p.dR) {
        float q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = p.beta * dy[k];
        store8<T, VEC>(p.dR, r * p.N, c, p.N, q);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += d[k];
      for (i += kDactWarps; i >= p.M; i -= p.M) ++b;
    }
  }
  if (!p.dbias) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) part[warp][VEC ? lane * 8 + k : lane + 32 * k] = sum[k];
  __syncthreads();
  if (c0 + threadIdx.x < p.N) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kDactWarps; ++w) t += part[w][threadIdx.x];
    p.ws[(int64_t)blockIdx.y * p.N + c0 + threadIdx.x] = t;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) gemm_dbias_kernel(const float* ws, void* dbias, int64_t N, int bands) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float t = 0.f;
  for (int b = 0; b < bands; ++b) t += ws[(int64_t)b * N + c];
  static_cast<T*>(dbias)[c] = from_f32<T>(t);
}

template <typename T>
bool rows_on_16(const void* p, int64_t bs, int64_t rs, int64_t cs) {
  constexpr int64_t PER = 16 / sizeof(T);
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && cs == 1 && bs % PER == 0 && rs % PER == 0;
}

template <typename T>
cudaError_t launch_t(const DactParams& p, cudaStream_t s) {
  const int64_t rows = p.batch * p.M, band = dact_band_rows(rows, p.N);
  const int bands = (int)((rows + band - 1) / band);
  if (bands > 0) {
    const dim3 grid((unsigned)((p.N + kCols - 1) / kCols), (unsigned)bands);
    const bool vec = p.N % 8 == 0 && rows_on_16<T>(p.dY, p.dy_bs, p.dy_rs, p.dy_cs) &&
                     rows_on_16<T>(p.pre, p.pre_bs, p.pre_rs, p.pre ? p.pre_cs : 1) && rows_on_16<T>(p.dP, 0, 0, 1) &&
                     rows_on_16<T>(p.dR, 0, 0, 1);
    if (vec) gemm_dact_kernel<T, true><<<grid, kDactWarps * 32, 0, s>>>(p, band);
    else gemm_dact_kernel<T, false><<<grid, kDactWarps * 32, 0, s>>>(p, band);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  if (p.dbias) gemm_dbias_kernel<T><<<(unsigned)((p.N + 255) / 256), 256, 0, s>>>(p.ws, p.dbias, p.N, bands);
  return cudaGetLastError();
}

}  // namespace

size_t dact_ws_floats(int64_t batch, int64_t M, int64_t N) {
  const int64_t rows = batch * M, band = dact_band_rows(rows, N);
  return (size_t)((rows + band - 1) / band) * (size_t)N;
}

cudaError_t launch_gemm_dact(const DactParams& p, cudaStream_t s) {
  switch (p.dtype) {
    case B2C_F32: return launch_t<float>(p, s);
    case B2C_BF16: return launch_t<__nv_bfloat16>(p, s);
    default: return launch_t<__half>(p, s);
  }
}

}  // namespace b2c
