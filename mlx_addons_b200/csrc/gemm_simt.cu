// Products with an epilogue on the FP32 units: any strides, any alignment,
// any of the three types.
//
// One CTA of 256 threads computes a 64 x 64 tile of D, a thread 4 x 4 of it,
// from 64 x 16 slices of both operands held in shared memory as float32
// (converted on the way in, so a product of 16-bit types is exact and every
// sum is held in 32 bits). The loads walk whichever of the two axes has the
// smaller stride, so both a matrix and its transposed view are read in whole
// sectors.
#include "b2c_kernels.cuh"
#include "gemm.cuh"

namespace b2c {

namespace {

constexpr int TS = 64;   // tile side
constexpr int TK = 16;   // slice depth
constexpr int TP = TS + 4;

template <typename T>
__device__ __forceinline__ void load_slice(float (*s)[TP], const GemmOperand& o, int64_t b, int64_t r0, int64_t rows,
                                           int64_t k0, int64_t K) {
  const T* base = static_cast<const T*>(o.p) + b * o.bs;
  const bool along_k = o.ks <= o.rs;
#pragma unroll
  for (int t = 0; t < TS * TK / 256; ++t) {
    const int e = threadIdx.x + t * 256;
    const int r = along_k ? e / TK : e % TS, k = along_k ? e % TK : e / TS;
    const bool in = r0 + r < rows && k0 + k < K;
    s[k][r] = in ? to_f32(base[(r0 + r) * o.rs + (k0 + k) * o.ks]) : 0.f;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) gemm_simt_kernel(const GemmProblem g, int64_t tiles_i, int64_t tiles_j) {
  __shared__ float sp[TK][TP], sq[TK][TP];
  const int64_t per = tiles_i * tiles_j, b = blockIdx.x / per, t = blockIdx.x - b * per;
  const int64_t i0 = (t / tiles_j) * TS, j0 = (t % tiles_j) * TS;
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < g.K; k0 += TK) {
    load_slice<T>(sp, g.P, b, i0, g.I, k0, g.K);
    load_slice<T>(sq, g.Q, b, j0, g.J, k0, g.K);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TK; ++k) {
      const float4 a = *reinterpret_cast<const float4*>(&sp[k][ti * 4]);
      const float4 q = *reinterpret_cast<const float4*>(&sq[k][tj * 4]);
      const float av[4] = {a.x, a.y, a.z, a.w}, qv[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], qv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = i0 + ti * 4 + i, c = j0 + tj * 4 + j;
      if (r < g.I && c < g.J) epilogue_store<T>(g.e, b, r, c, acc[i][j]);
    }
}

}  // namespace

cudaError_t launch_gemm_simt(const GemmProblem& g, cudaStream_t s) {
  const int64_t ti = (g.I + TS - 1) / TS, tj = (g.J + TS - 1) / TS, total = g.batch * ti * tj;
  if (total > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const unsigned grid = (unsigned)total;
  switch (g.dtype) {
    case B2C_F32: gemm_simt_kernel<float><<<grid, 256, 0, s>>>(g, ti, tj); break;
    case B2C_BF16: gemm_simt_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(g, ti, tj); break;
    default: gemm_simt_kernel<__half><<<grid, 256, 0, s>>>(g, ti, tj); break;
  }
  return cudaGetLastError();
}

}  // namespace b2c
