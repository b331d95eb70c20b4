// Newton-Schulz orthogonalisation of a batch of matrices:
//
//   X = G / (|G|_F + eps);  steps times:  S = X X^T,  X <- a X + (b S + c S S) X
//
// taken on the smaller side (for a tall G, S = X^T X and X <- a X + X (b S +
// c S S)), so S has min(m, n) rows. Each step is three products with an
// epilogue: S; P = c S S + b S; X' = P X + a X.
#include <cmath>

#include "b2c_kernels.cuh"
#include "gemm_tc.cuh"
#include "polar.cuh"

namespace b2c {

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormParts = kNormThreads;  // most partial sums of a matrix

struct PolarIn {
  const void* G;
  int64_t bs, rs, cs, batch, m, n;
  int vec;  // rows of unit stride on 16-byte boundaries
};

// Sum of a block's values in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double s, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < kNormThreads / 32; ++w) s += red[w];
  return s;
}

// Walks a matrix in units of 8 neighbouring elements of a row: this thread's
// next one is `blocks` blocks of threads further. One division at the start.
struct Walk {
  int64_t r, u, units, dr, du;
  __device__ __forceinline__ Walk(int64_t n, int64_t blocks, int64_t block) {
    units = (n + 7) / 8;
    const int64_t first = block * kNormThreads + threadIdx.x, step = blocks * kNormThreads;
    r = first / units, u = first - r * units;
    dr = step / units, du = step - dr * units;
  }
  __device__ __forceinline__ void next() {
    r += dr, u += du;
    if (u >= units) u -= units, ++r;
  }
};

template <typename T>
__device__ __forceinline__ void load_unit(const PolarIn& in, const T* row, int64_t c, float (&v)[8]) {
  if (in.vec && c + 8 <= in.n) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < 8 / PER; ++q) {
      const uint4 w = *reinterpret_cast<const uint4*>(row + c + q * PER);
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int k = 0; k < PER; ++k) v[q * PER + k] = to_f32(e[k]);
    }
  } else {
    // every load is issued, past the end that of c again: none waits for a branch
    T t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = row[(c + k < in.n ? c + k : c) * in.cs];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < in.n ? to_f32(t[k]) : 0.f;
  }
}

// Sum of squares of one slice of one matrix, held in 64 bits: squares of any
// float32 neither overflow nor vanish there. Bound by HBM (2 or 4 bytes an
// element; the 64-bit additions take about as long).
template <typename T>
__global__ void __launch_bounds__(kNormThreads) polar_norm_kernel(const PolarIn in, double* part, unsigned int* counter) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *counter = 0;
  __shared__ double red[kNormThreads / 32];
  for (int64_t b = blockIdx.y; b < in.batch; b += gridDim.y) {
    const T* base = static_cast<const T*>(in.G) + b * in.bs;
    double s = 0.0;
    for (Walk w(in.n, gridDim.x, blockIdx.x); w.r < in.m; w.next()) {
      float v[8];
      load_unit<T>(in, base + w.r * in.rs, w.u * 8, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += (double)v[k] * (double)v[k];
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[b * kNormParts + blockIdx.x] = s;
  }
}

// G times the power of two that puts |G|_F + eps in [2^13, 2^14), as one or two
// f16 planes, rows padded to units of 8; r = 2^14 X / that, in [1, 2], is left
// to the first step. So a bfloat16 G is held without a rounding, which the
// iteration would amplify by up to 3.4445^steps in its smallest directions.
template <typename T, bool HALVES>
__global__ void __launch_bounds__(kNormThreads) polar_scale_kernel(const PolarIn in, const double* part, int parts,
                                                                   double eps, __half* X, int64_t pitch, int64_t plane,
                                                                   float* r) {
  __shared__ double red[kNormThreads / 32];
  for (int64_t b = blockIdx.y; b < in.batch; b += gridDim.y) {
    const T* base = static_cast<const T*>(in.G) + b * in.bs;
    const double sum = block_sum((int)threadIdx.x < parts ? part[b * kNormParts + threadIdx.x] : 0.0, red);
    const PolarNorm norm = polar_norm(sqrt(sum) + eps);
    if (blockIdx.x == 0 && threadIdx.x == 0) r[b] = norm.r;
    for (Walk w(in.n, gridDim.x, blockIdx.x); w.r < in.m; w.next()) {
      float v[8];
      load_unit<T>(in, base + w.r * in.rs, w.u * 8, v);
      __align__(16) __half hi[8], lo[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = (float)((double)v[k] * norm.scale);
        hi[k] = __float2half_rn(x);
        lo[k] = __float2half_rn(x - __half2float(hi[k]));
      }
      const int64_t at = (b * in.m + w.r) * pitch + w.u * 8;
      *reinterpret_cast<uint4*>(X + at) = *reinterpret_cast<const uint4*>(hi);
      if constexpr (HALVES) *reinterpret_cast<uint4*>(X + plane + at) = *reinterpret_cast<const uint4*>(lo);
    }
  }
}

// The iteration on G^T gives the transposed result: a matrix whose columns lie
// closer together than its rows is taken as its transpose, so that reads run
// along memory.
PolarParams along_rows(const PolarParams& in) {
  PolarParams p = in;
  p.out_rs = p.n;
  p.out_cs = 1;
  if (p.m > 1 && p.n > 1 ? p.rs < p.cs : p.n == 1) {
    p.m = in.n, p.n = in.m;
    p.rs = in.cs, p.cs = in.rs;
    p.out_rs = 1, p.out_cs = in.n;
  }
  return p;
}

// Scratch of the product form: norms, two X, S and P.
struct PolarLayout {
  int64_t side, pitch_x, pitch_s, x_plane, s_plane, x_bytes, s_bytes, part_bytes, vec_bytes;
  int planes;
};

PolarLayout polar_layout(const PolarParams& p) {
  PolarLayout l;
  l.side = p.m < p.n ? p.m : p.n;
  l.planes = p.dtype == B2C_BF16 ? 1 : 2;
  l.pitch_x = (p.n + 7) / 8 * 8;
  l.pitch_s = (l.side + 7) / 8 * 8;
  l.x_plane = p.batch * p.m * l.pitch_x;
  l.s_plane = p.batch * l.side * l.pitch_s;
  l.x_bytes = (l.x_plane * l.planes * 2 + 255) / 256 * 256;
  l.s_bytes = (l.s_plane * l.planes * 2 + 255) / 256 * 256;
  l.part_bytes = (p.batch * kNormParts * (int64_t)sizeof(double) + 255) / 256 * 256;
  l.vec_bytes = (p.batch * l.pitch_s * (int64_t)sizeof(float) + 255) / 256 * 256;
  return l;
}

template <typename T>
cudaError_t launch_t(const PolarParams& p, int sms, cudaStream_t s) {
  const PolarLayout l = polar_layout(p);
  const int64_t mn = p.m * p.n, side = l.side;
  char* w = static_cast<char*>(p.ws);
  double* part = reinterpret_cast<double*>(w);
  w += l.part_bytes;
  __half* X0 = reinterpret_cast<__half*>(w);
  __half* X1 = reinterpret_cast<__half*>(w + l.x_bytes);
  __half* S = reinterpret_cast<__half*>(w + 2 * l.x_bytes);
  __half* P = reinterpret_cast<__half*>(w + 2 * l.x_bytes + l.s_bytes);
  constexpr int64_t PER = 16 / sizeof(T);
  w += 2 * l.x_bytes + 2 * l.s_bytes;
  float* ds = reinterpret_cast<float*>(w);  // diagonals of S and P
  float* dp = reinterpret_cast<float*>(w + l.vec_bytes);
  float* r = reinterpret_cast<float*>(w + 2 * l.vec_bytes);
  unsigned int* counter = reinterpret_cast<unsigned int*>(w + 3 * l.vec_bytes);
  const PolarIn in{p.G, p.bs, p.rs, p.cs, p.batch, p.m, p.n,
                   (reinterpret_cast<uintptr_t>(p.G) & 15) == 0 && p.cs == 1 && p.rs % PER == 0 && p.bs % PER == 0};
  const int64_t units = p.m * ((p.n + 7) / 8);
  int64_t blocks = (units + 4 * kNormThreads - 1) / (4 * kNormThreads);
  if (blocks > kNormParts) blocks = kNormParts;
  const int parts = (int)blocks;
  const dim3 grid((unsigned)blocks, (unsigned)(p.batch < 65535 ? p.batch : 65535));
  polar_norm_kernel<T><<<grid, kNormThreads, 0, s>>>(in, part, counter);
  constexpr bool kTwo = !std::is_same<T, __nv_bfloat16>::value;
  polar_scale_kernel<T, kTwo><<<grid, kNormThreads, 0, s>>>(in, part, parts, p.eps, X0, l.pitch_x, l.x_plane, r);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;

  if (polar_grid_fits(p, sms))
    return launch_polar_grid(p, PolarScratch{side, l.pitch_x, l.pitch_s, l.x_plane, l.s_plane, X0, X1, S, P, ds, dp, r, counter},
                             sms, s);
  const bool wide = p.m <= p.n;
  const int inner = kTwo ? kOutHalves : B2C_F16;
  TcProblem t{};
  t.kind = kTwo ? kHalves : kOne;
  t.f16 = 1;
  t.chained = 1;
  t.batch = p.batch;
  const int bcast = p.batch == 1;
  const int64_t sx = side * l.pitch_s, xx = p.m * l.pitch_x;
  const TcOperand s_op{S, sx, l.pitch_s, l.s_plane, 0, bcast}, p_op{P, sx, l.pitch_s, l.s_plane, 0, bcast};
  double hi = 1.0;
  for (int step = 0; step < p.steps; ++step) {
    const double a = p.coef[3 * step], b = p.coef[3 * step + 1], c = p.coef[3 * step + 2], t2 = hi * hi;
    const float ss = polar_scale_for(t2), sp = polar_scale_for(fabs(b) * t2 + fabs(c) * t2 * t2);
    const TcOperand x_rows{X0, xx, l.pitch_x, l.x_plane, 0, bcast}, x_cols{X0, xx, l.pitch_x, l.x_plane, 1, bcast};
    // S = X X^T (X^T X), the lower half of its tiles
    t.I = t.J = side;
    t.K = wide ? p.n : p.m;
    t.P = t.Q = wide ? x_rows : x_cols;
    t.sym = 1;
    t.e = GemmEpilogue{};
    t.e.y = GemmView{S, sx, l.pitch_s, 1};
    t.e.alpha = ss / (kPolarScale * kPolarScale);
    t.polar = TcPolar{};
    t.polar.mode = kPolarS;
    t.polar.r = step ? nullptr : r;
    t.polar.d_in = t.polar.d_out = ds;
    t.polar.side = l.pitch_s;
    t.polar.k = 1.f / ss;
    t.out = t.res = inner;
    t.y_plane = t.res_plane = l.s_plane;
    if ((e = launch_gemm_tc(t, s)) != cudaSuccess) return e;
    // P = c S S + b S
    t.K = side;
    t.P = t.Q = s_op;
    t.e.y.p = P;
    t.e.res = GemmView{S, sx, l.pitch_s, 1};
    t.e.alpha = (float)(c * sp / ((double)ss * ss));
    t.e.beta = (float)(b * sp / ss);
    t.polar.mode = kPolarP;
    t.polar.r = nullptr;
    t.polar.d_out = dp;
    t.polar.k = (float)(c * sp / ss);
    t.polar.k2 = 1.f / sp;
    t.polar.k3 = (float)c;
    t.polar.k4 = (float)b;
    if ((e = launch_gemm_tc(t, s)) != cudaSuccess) return e;
    // X' = P X + a X (X P + a X); P is symmetric, so either of its indices may be contracted
    const bool last = step == p.steps - 1;
    const float so = last ? 1.f : kPolarScale;
    t.I = p.m;
    t.J = p.n;
    t.P = wide ? p_op : x_rows;
    t.Q = wide ? x_cols : p_op;
    t.sym = 0;
    t.e.y = last ? GemmView{p.out, mn, p.out_rs, p.out_cs} : GemmView{X1, xx, l.pitch_x, 1};
    t.e.res = GemmView{X0, xx, l.pitch_x, 1};
    t.e.alpha = so / (sp * kPolarScale);
    t.e.beta = so / kPolarScale;
    t.polar.mode = wide ? kPolarXi : kPolarXj;
    t.polar.r = step ? nullptr : r;
    t.polar.d_in = dp;
    t.polar.k = (float)a;
    t.out = last ? p.dtype : inner;
    t.y_plane = last ? 0 : l.x_plane;
    t.res_plane = l.x_plane;
    if ((e = launch_gemm_tc(t, s)) != cudaSuccess) return e;
    __half* sw = X0;
    X0 = X1;
    X1 = sw;
    hi = polar_poly_bound(a, b, c, hi);
  }
  return cudaSuccess;
}

}  // namespace

double polar_poly_bound(double a, double b, double c, double hi) {
  auto at = [&](double v) { return fabs(v * (a + v * v * (b + c * v * v))); };
  double best = at(hi);
  // stationary points: a + 3 b t + 5 c t^2 = 0 with t = v^2
  double roots[2];
  int n = 0;
  if (c != 0.0) {
    const double disc = 9 * b * b - 20 * a * c;
    if (disc >= 0) {
      const double q = sqrt(disc);
      roots[n++] = (-3 * b + q) / (10 * c);
      roots[n++] = (-3 * b - q) / (10 * c);
    }
  } else if (b != 0.0) {
    roots[n++] = -a / (3 * b);
  }
  for (int i = 0; i < n; ++i)
    if (roots[i] > 0 && sqrt(roots[i]) < hi) best = fmax(best, at(sqrt(roots[i])));
  return best;
}

size_t polar_ws_bytes(const PolarParams& in) {
  const PolarParams p = along_rows(in);
  if (polar_cta_fits(p)) return 0;
  const PolarLayout l = polar_layout(p);
  return (size_t)(l.part_bytes + 2 * l.x_bytes + 2 * l.s_bytes + 3 * l.vec_bytes + 256);
}

cudaError_t launch_polar(const PolarParams& in, cudaStream_t s) {
  const PolarParams p = along_rows(in);
  int sms = 0;
  const cudaError_t e = device_sms(&sms);
  if (e != cudaSuccess) return e;
  if (polar_cta_fits(p)) return launch_polar_cta(p, sms, s);
  switch (p.dtype) {
    case B2C_F32: return launch_t<float>(p, sms, s);
    case B2C_BF16: return launch_t<__nv_bfloat16>(p, sms, s);
    default: return launch_t<__half>(p, sms, s);
  }
}

}  // namespace b2c
