// Products with an epilogue on the FP32 units: any strides, any alignment,
// any of the three types. For products too small or too shallow for the tensor
// cores to pay for their set-up (and for float32 its split operands).
//
// One CTA of 128 threads computes a 64 x 64 tile of D, a thread 8 x 4 of it,
// from 64 x 16 slices of both operands held in shared memory as float32
// (converted on the way in, so a product of 16-bit types is exact and every
// sum is held in 32 bits); the next slice is on its way in registers
// meanwhile. The loads walk whichever of the two axes has the smaller stride,
// so both a matrix and its transposed view are read in whole sectors. A
// shallow product is bound by writing D: the 4 columns of a thread are
// neighbours and stored as one unit where alignment allows, and 16 apart
// otherwise, so that a half warp's stores lie together.
#include "b2c_kernels.cuh"
#include "gemm.cuh"

namespace b2c {

namespace {

constexpr int TS = 64;   // tile side
constexpr int TK = 16;   // slice depth
constexpr int TP = TS + 4;
constexpr int kSimtThreads = 128;
constexpr int kLoads = TS * TK / kSimtThreads;

// This thread's 8 elements of a slice: every 8th row at one k, or every 2nd k of
// one row.
template <typename T>
struct SliceLoader {
  const T* at;       // element 0
  int64_t step, kstep, left_r, left_k, dr, dk;
  int r, k;
  __device__ __forceinline__ SliceLoader(const GemmOperand& o, int64_t b, int64_t r0, int64_t rows, int64_t K) {
    const bool along_k = o.ks <= o.rs;
    r = along_k ? threadIdx.x / TK : threadIdx.x % TS;
    k = along_k ? threadIdx.x % TK : threadIdx.x / TS;
    dr = along_k ? kSimtThreads / TK : 0;
    dk = along_k ? 0 : kSimtThreads / TS;
    at = static_cast<const T*>(o.p) + b * o.bs + (r0 + r) * o.rs + k * o.ks;
    step = dr * o.rs + dk * o.ks;
    kstep = TK * o.ks;
    left_r = rows - r0 - r;
    left_k = K - k;
  }
  __device__ __forceinline__ void load(float (&v)[kLoads]) {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) v[t] = t * dr < left_r && t * dk < left_k ? to_f32(at[t * step]) : 0.f;
    at += kstep;
    left_k -= TK;
  }
  __device__ __forceinline__ void store(float (*s)[TP], const float (&v)[kLoads]) const {
#pragma unroll
    for (int t = 0; t < kLoads; ++t) s[k + t * (int)dk][r + t * (int)dr] = v[t];
  }
};

// Four neighbours along j, as one 16- or 8-byte unit.
template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

// VEC: every row of y, pre and the addend starts on a unit of four.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kSimtThreads) gemm_simt_kernel(const GemmProblem g, int64_t tiles_i, int64_t tiles_j) {
  __shared__ __align__(16) float sp[TK][TP], sq[TK][TP];
  const int64_t per = tiles_i * tiles_j, b = blockIdx.x / per, t = blockIdx.x - b * per;
  const int64_t i0 = (t / tiles_j) * TS, j0 = (t % tiles_j) * TS;
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
  SliceLoader<T> lp(g.P, b, i0, g.I, g.K), lq(g.Q, b, j0, g.J, g.K);
  float acc[8][4] = {}, vp[kLoads], vq[kLoads];
  lp.load(vp);
  lq.load(vq);
  for (int64_t k0 = 0; k0 < g.K; k0 += TK) {
    lp.store(sp, vp);
    lq.store(sq, vq);
    __syncthreads();
    if (k0 + TK < g.K) {
      lp.load(vp);
      lq.load(vq);
    }
    const int n = g.K - k0 < TK ? (int)(g.K - k0) : TK;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float4 a = *reinterpret_cast<const float4*>(&sp[k][ti * 8]), c = *reinterpret_cast<const float4*>(&sp[k][ti * 8 + 4]);
      const float av[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
      float qv[4];
      if constexpr (VEC) {
        const float4 q = *reinterpret_cast<const float4*>(&sq[k][tj * 4]);
        qv[0] = q.x, qv[1] = q.y, qv[2] = q.z, qv[3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) qv[j] = sq[k][tj + 16 * j];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], qv[j], acc[i][j]);
    }
    __syncthreads();
  }
  const int64_t i = i0 + ti * 8, j = j0 + (VEC ? tj * 4 : tj);
  constexpr int JS = VEC ? 1 : 16;  // columns between a thread's four
  if (VEC && j + 4 <= g.J) {
    const GemmEpilogue& e = g.e;
    float bias[4] = {};
    if (e.bias && !e.bias_on_i)
#pragma unroll
      for (int c = 0; c < 4; ++c) bias[c] = to_f32(static_cast<const T*>(e.bias)[j + c]);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (i + r >= g.I) break;
      if (e.bias && e.bias_on_i) bias[0] = bias[1] = bias[2] = bias[3] = to_f32(static_cast<const T*>(e.bias)[i + r]);
      float v[4];
      Four<T> u;
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = fmaf(e.alpha, acc[r][c], bias[c]);
      if (e.pre.p) {
#pragma unroll
        for (int c = 0; c < 4; ++c) u.v[c] = from_f32<T>(v[c]);
        *reinterpret_cast<Four<T>*>(static_cast<T*>(e.pre.p) + b * e.pre.bs + (i + r) * e.pre.is + j) = u;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = act_f32<sizeof(T) == 2>(v[c], e.act);
      if (e.res.p) {
        u = *reinterpret_cast<const Four<T>*>(static_cast<const T*>(e.res.p) + b * e.res.bs + (i + r) * e.res.is + j);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = fmaf(e.beta, to_f32(u.v[c]), v[c]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) u.v[c] = from_f32<T>(v[c]);
      *reinterpret_cast<Four<T>*>(static_cast<T*>(e.y.p) + b * e.y.bs + (i + r) * e.y.is + j) = u;
    }
    return;
  }
  const GemmEpilogue& e = g.e;
#pragma unroll 2
  for (int r = 0; r < 8; ++r) {
    if (i + r >= g.I) break;
    T* y = static_cast<T*>(e.y.p) + b * e.y.bs + (i + r) * e.y.is + j * e.y.js;
    T* pre = static_cast<T*>(e.pre.p) + b * e.pre.bs + (i + r) * e.pre.is + j * e.pre.js;
    const T* res = static_cast<const T*>(e.res.p) + b * e.res.bs + (i + r) * e.res.is + j * e.res.js;
    const T* bias = static_cast<const T*>(e.bias) + (e.bias_on_i ? i + r : j);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (j + c * JS >= g.J) break;
      float v = e.alpha * acc[0][c];
      if (e.bias) v += to_f32(bias[e.bias_on_i ? 0 : c * JS]);
      if (e.pre.p) pre[c * JS * e.pre.js] = from_f32<T>(v);
      v = act_f32<sizeof(T) == 2>(v, e.act);
      if (e.res.p) v = fmaf(e.beta, to_f32(res[c * JS * e.res.js]), v);
      y[c * JS * e.y.js] = from_f32<T>(v);
    }
    // the sums move up instead of the index, for a loop that stays short
#pragma unroll
    for (int m = 1; m < 8; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[m - 1][c] = acc[m][c];
  }
}

template <typename T>
cudaError_t launch_t(const GemmProblem& g, cudaStream_t s) {
  const int64_t ti = (g.I + TS - 1) / TS, tj = (g.J + TS - 1) / TS, total = g.batch * ti * tj;
  if (total > 0x7fffffff) return cudaErrorInvalidConfiguration;
  auto fours = [](const GemmView& v) {
    return !v.p || (v.js == 1 && reinterpret_cast<uintptr_t>(v.p) % (4 * sizeof(T)) == 0 && v.is % 4 == 0 && v.bs % 4 == 0);
  };
  const unsigned grid = (unsigned)total;
  if (fours(g.e.y) && fours(g.e.pre) && fours(g.e.res)) gemm_simt_kernel<T, true><<<grid, kSimtThreads, 0, s>>>(g, ti, tj);
  else gemm_simt_kernel<T, false><<<grid, kSimtThreads, 0, s>>>(g, ti, tj);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gemm_simt(const GemmProblem& g, cudaStream_t s) {
  switch (g.dtype) {
    case B2C_F32: return launch_t<float>(g, s);
    case B2C_BF16: return launch_t<__nv_bfloat16>(g, s);
    default: return launch_t<__half>(g, s);
  }
}

}  // namespace b2c
