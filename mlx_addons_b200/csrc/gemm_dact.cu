// Gradient of a product's epilogue: dP = dY act'(pre), its column sums (the
// bias gradient) and beta dY (the residual's), in one pass over dY and pre.
//
// Bound by HBM: it reads dY and pre and writes dP once. A CTA takes 32
// columns (one per lane) of a band of rows; its 8 warps walk the band and
// their float32 column sums join in shared memory, one partial row per band.
// A second kernel adds the bands in a fixed order, so the sums do not depend
// on which CTA ran first. The sums take dP before it is rounded; dP itself is
// rounded once to the product's type, since it is an operand of the two
// products that follow.
#include "b2c_kernels.cuh"
#include "gemm.cuh"

namespace b2c {

namespace {

constexpr int kDactWarps = 8;
constexpr int kMaxBands = 1024;

int64_t dact_band_rows(int64_t rows) {
  int64_t band = 64;
  while ((rows + band - 1) / band > kMaxBands) band *= 2;
  return band;
}

template <typename T>
__global__ void __launch_bounds__(kDactWarps * 32) gemm_dact_kernel(const DactParams p, int64_t band) {
  __shared__ float part[kDactWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rows = p.batch * p.M, c = (int64_t)blockIdx.x * 32 + lane, r0 = (int64_t)blockIdx.y * band;
  const int64_t r1 = r0 + band < rows ? r0 + band : rows;
  float sum = 0.f;
  if (c < p.N) {
    for (int64_t r = r0 + warp; r < r1; r += kDactWarps) {
      const int64_t b = r / p.M, i = r - b * p.M;
      const float dy = to_f32(static_cast<const T*>(p.dY)[b * p.dy_bs + i * p.dy_rs + c * p.dy_cs]);
      float d = dy;
      if (p.pre) {
        const float x = to_f32(static_cast<const T*>(p.pre)[b * p.pre_bs + i * p.pre_rs + c * p.pre_cs]);
        d = p.act == B2C_ACT_RELU ? (x > 0.f ? dy : 0.f) : dy * act_slope_f32(x, p.act);
      }
      if (p.dP) static_cast<T*>(p.dP)[r * p.N + c] = from_f32<T>(d);
      if (p.dR) static_cast<T*>(p.dR)[r * p.N + c] = from_f32<T>(p.beta * dy);
      sum += d;
    }
  }
  if (!p.dbias) return;
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < p.N) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kDactWarps; ++w) t += part[w][lane];
    p.ws[(int64_t)blockIdx.y * p.N + c] = t;
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
cudaError_t launch_t(const DactParams& p, cudaStream_t s) {
  const int64_t rows = p.batch * p.M, band = dact_band_rows(rows);
  const int bands = (int)((rows + band - 1) / band);
  if (bands > 0) {
    const dim3 grid((unsigned)((p.N + 31) / 32), (unsigned)bands);
    gemm_dact_kernel<T><<<grid, kDactWarps * 32, 0, s>>>(p, band);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  if (p.dbias) gemm_dbias_kernel<T><<<(unsigned)((p.N + 255) / 256), 256, 0, s>>>(p.ws, p.dbias, p.N, bands);
  return cudaGetLastError();
}

}  // namespace

size_t dact_ws_floats(int64_t batch, int64_t M, int64_t N) {
  const int64_t rows = batch * M, band = dact_band_rows(rows);
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
