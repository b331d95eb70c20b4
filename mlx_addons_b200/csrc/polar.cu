// Newton-Schulz orthogonalisation of a batch of matrices:
//
//   X = G / (|G|_F + eps);  steps times:  S = X X^T,  X <- a X + (b S + c S S) X
//
// taken on the smaller side (for a tall G, S = X^T X and X <- a X + X (b S +
// c S S)), so S has min(m, n) rows. Each step is three products with an
// epilogue: S; P = c S S + b S; X' = P X + a X.
#include "b2c_kernels.cuh"
#include "gemm.cuh"

namespace b2c {

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormParts = 64;  // partial sums of a matrix, added in a fixed order

struct PolarIn {
  const void* G;
  int64_t bs, rs, cs, batch, m, n;
};

// Sum of squares of one slice of one matrix, held in 64 bits: squares of any
// float32 neither overflow nor vanish there.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) polar_norm_kernel(const PolarIn in, double* part) {
  __shared__ double red[kNormThreads / 32];
  const int64_t total = in.m * in.n;
  for (int64_t b = blockIdx.y; b < in.batch; b += gridDim.y) {
  const T* base = static_cast<const T*>(in.G) + b * in.bs;
  double s = 0.0;
  for (int64_t e = (int64_t)blockIdx.x * kNormThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kNormThreads) {
    const int64_t r = e / in.n, c = e - r * in.n;
    const double v = (double)to_f32(base[r * in.rs + c * in.cs]);
    s += v * v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kNormThreads / 32; ++w) t += red[w];
    part[b * kNormParts + blockIdx.x] = t;
  }
  __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) polar_scale_kernel(const PolarIn in, const double* part, int parts,
                                                                   double eps, float* X) {
  const int64_t total = in.m * in.n;
  for (int64_t b = blockIdx.y; b < in.batch; b += gridDim.y) {
  const T* base = static_cast<const T*>(in.G) + b * in.bs;
  double s = 0.0;
  for (int i = 0; i < parts; ++i) s += part[b * kNormParts + i];
  const double inv = 1.0 / (sqrt(s) + eps);
  for (int64_t e = (int64_t)blockIdx.x * kNormThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kNormThreads) {
    const int64_t r = e / in.n, c = e - r * in.n;
    X[b * total + e] = (float)((double)to_f32(base[r * in.rs + c * in.cs]) * inv);
  }
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) polar_round_kernel(const float* X, void* out, int64_t total) {
  for (int64_t e = (int64_t)blockIdx.x * kNormThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kNormThreads)
    static_cast<T*>(out)[e] = from_f32<T>(X[e]);
}

template <typename T>
cudaError_t launch_t(const PolarParams& p, cudaStream_t s) {
  const int64_t mn = p.m * p.n, side = p.m < p.n ? p.m : p.n, ss = side * side;
  char* w = static_cast<char*>(p.ws);
  double* part = reinterpret_cast<double*>(w);
  float* X0 = reinterpret_cast<float*>(w + p.batch * kNormParts * sizeof(double));
  float *X1 = X0 + p.batch * mn, *S = X1 + p.batch * mn, *P = S + p.batch * ss;
  const PolarIn in{p.G, p.bs, p.rs, p.cs, p.batch, p.m, p.n};
  int64_t blocks = (mn + kNormThreads - 1) / kNormThreads;
  const int parts = (int)(blocks < kNormParts ? blocks : kNormParts);
  if (blocks > 4096) blocks = 4096;
  const unsigned by = (unsigned)(p.batch < 65535 ? p.batch : 65535);
  const dim3 gn((unsigned)parts, by), gs((unsigned)blocks, by);
  polar_norm_kernel<T><<<gn, kNormThreads, 0, s>>>(in, part);
  polar_scale_kernel<T><<<gs, kNormThreads, 0, s>>>(in, part, parts, p.eps, X0);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const bool wide = p.m <= p.n;
  const int64_t n = p.n;
  for (int t = 0; t < p.steps; ++t) {
    const float a = p.coef[3 * t], b = p.coef[3 * t + 1], c = p.coef[3 * t + 2];
    GemmProblem g{};
    g.dtype = B2C_F32;
    g.batch = p.batch;
    g.I = g.J = side;
    g.K = wide ? p.n : p.m;
    g.P = wide ? GemmOperand{X0, mn, n, 1} : GemmOperand{X0, mn, 1, n};
    g.Q = g.P;
    g.e.y = GemmView{S, ss, side, 1};
    g.e.alpha = 1.f;
    if ((e = launch_gemm_simt(g, s)) != cudaSuccess) return e;
    g.K = side;
    g.P = g.Q = GemmOperand{S, ss, side, 1};
    g.e.y = GemmView{P, ss, side, 1};
    g.e.res = GemmView{S, ss, side, 1};
    g.e.alpha = c;
    g.e.beta = b;
    if ((e = launch_gemm_simt(g, s)) != cudaSuccess) return e;
    g.I = p.m;
    g.J = p.n;
    // P is symmetric: either index may be the contracted one
    if (wide) {
      g.P = GemmOperand{P, ss, side, 1};
      g.Q = GemmOperand{X0, mn, 1, n};
    } else {
      g.P = GemmOperand{X0, mn, n, 1};
      g.Q = GemmOperand{P, ss, side, 1};
    }
    g.e.y = GemmView{X1, mn, n, 1};
    g.e.res = GemmView{X0, mn, n, 1};
    g.e.alpha = 1.f;
    g.e.beta = a;
    if ((e = launch_gemm_simt(g, s)) != cudaSuccess) return e;
    float* sw = X0;
    X0 = X1;
    X1 = sw;
  }
  const int64_t total = p.batch * mn, rb = (total + kNormThreads - 1) / kNormThreads;
  polar_round_kernel<T><<<(unsigned)(rb < 8192 ? rb : 8192), kNormThreads, 0, s>>>(X0, p.out, total);
  return cudaGetLastError();
}

}  // namespace

size_t polar_ws_bytes(const PolarParams& p) {
  const int64_t mn = p.m * p.n, side = p.m < p.n ? p.m : p.n;
  return (size_t)p.batch * kNormParts * sizeof(double) + (size_t)p.batch * (2 * mn + 2 * side * side) * sizeof(float);
}

cudaError_t launch_polar(const PolarParams& p, cudaStream_t s) {
  switch (p.dtype) {
    case B2C_F32: return launch_t<float>(p, s);
    case B2C_BF16: return launch_t<__nv_bfloat16>(p, s);
    default: return launch_t<__half>(p, s);
  }
}

}  // namespace b2c
