// Matrix products with an epilogue: types and device helpers shared by
// the gemm_*.cu and polar*.cu files.
//
// Every product is written as D[i, j] = sum_k P[i, k] Q[j, k] on two operands
// with free strides; the caller of b2c_gemm has P = A, Q = B^T, or the other
// way round where B's columns are the longer side.
#pragma once

#include <cstdlib>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "b2c.h"
#include "b2c_common.cuh"

namespace b2c {

// One operand: element (b, r, k) at p[b * bs + r * rs + k * ks].
struct GemmOperand {
  const void* p;
  int64_t bs, rs, ks;
};

// An addend or output in the coordinates of D.
struct GemmView {
  void* p;
  int64_t bs, is, js;
};

// out = act(alpha * D + bias) + beta * res; pre = alpha * D + bias.
struct GemmEpilogue {
  GemmView y, pre, res;  // pre.p / res.p null where absent; all of the product's type
  const void* bias;      // null where absent
  int bias_on_i;         // bias[i] (1) or bias[j] (0)
  int act;               // B2C_ACT_*
  float alpha, beta;
};

struct GemmProblem {
  int dtype;             // B2C_F32, B2C_BF16 or B2C_F16: operands, addends and outputs
  GemmOperand P, Q;
  int64_t batch;
  int64_t I, J, K;
  GemmEpilogue e;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// Rounds to nearest even; a half result past the type's range becomes inf.
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

constexpr float kGeluC = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float kGeluK = 0.044715f;
constexpr float kRsqrt2 = 0.7071067811865476f;
constexpr float kRsqrt2Pi = 0.3989422804014327f;  // 1 / sqrt(2 pi)

// Activations come in two forms: FAST for 16-bit results, on the exponential
// and reciprocal units, and one on the accurate functions for float32. The fast
// ones are within 2^-16 of their value wherever it is a normal number (most of it the exponent's
// rounding far out), a thirtieth of half a step of f16.
template <bool FAST>
__device__ __forceinline__ float exp_f32(float x) {
  return FAST ? __expf(x) : expf(x);
}
// By exp(-|x|), which leaves the divisor in [1, 2] and the lower tail its relative accuracy.
template <bool FAST>
__device__ __forceinline__ float sigmoid_f32(float x) {
  const float t = exp_f32<FAST>(-fabsf(x)), r = FAST ? __fdividef(1.f, 1.f + t) : 1.f / (1.f + t);
  return x < 0.f ? t * r : r;
}

// Normal distribution function; bell receives exp(-x^2 / 2). The fast form is
// Phi(-|x|) = bell t (c0 + c1 t + ... + c6 t^6) with t = 1 / (1 + p |x|): the c are the
// minimax fit of the relative error over |x| <= 14 (a linear programme on 1,400 points),
// p the one that makes it smallest; 7e-7 of the value, 1.0e-6 as evaluated in 32 bits.
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float x, float& bell) {
  bell = exp_f32<FAST>(-0.5f * x * x);
  if constexpr (!FAST) return 0.5f * (1.f + erff(x * kRsqrt2));
  const float t = __fdividef(1.f, fmaf(0.362480336f, fabsf(x), 1.f));
  float q = fmaf(0.0481144309f, t, -0.179940585f);
  q = fmaf(q, t, 0.175411849f);
  q = fmaf(q, t, 0.0294815642f);
  q = fmaf(q, t, 0.139324177f);
  q = fmaf(q, t, 0.142915497f);
  q = fmaf(q, t, 0.144693461f);
  const float tail = q * t * bell;
  return x < 0.f ? tail : 1.f - tail;
}

// act(x). NaN stays NaN.
template <bool FAST>
__device__ __forceinline__ float act_f32(float x, int act) {
  switch (act) {
    case B2C_ACT_RELU: return x < 0.f ? 0.f : x;
    case B2C_ACT_GELU: {
      float bell;
      return x * normal_cdf<FAST>(x, bell);
    }
    // 0.5 x (1 + tanh u) = x sigmoid(2 u)
    case B2C_ACT_GELU_TANH: return x * sigmoid_f32<FAST>(2.f * kGeluC * (x + kGeluK * x * x * x));
    case B2C_ACT_SILU: return x * sigmoid_f32<FAST>(x);
    default: return x;
  }
}

// d act(x) / dx, given the pre-activation.
template <bool FAST>
__device__ __forceinline__ float act_slope_f32(float x, int act) {
  switch (act) {
    case B2C_ACT_RELU: return x > 0.f ? 1.f : 0.f;
    case B2C_ACT_GELU: {
      float bell;
      const float cdf = normal_cdf<FAST>(x, bell);
      return fmaf(x * kRsqrt2Pi, bell, cdf);
    }
    case B2C_ACT_GELU_TANH: {
      const float s = sigmoid_f32<FAST>(2.f * kGeluC * (x + kGeluK * x * x * x));
      // beyond 16 the second term is zero in 32 bits, but its factors overflow there
      const float c = fminf(fmaxf(x, -16.f), 16.f);
      return s + c * s * (1.f - s) * 2.f * kGeluC * (1.f + 3.f * kGeluK * c * c);
    }
    case B2C_ACT_SILU: {
      const float s = sigmoid_f32<FAST>(x);
      return s * (1.f + x * (1.f - s));
    }
    default: return 1.f;
  }
}

// One element of the epilogue.
template <typename T>
__device__ __forceinline__ void epilogue_store(const GemmEpilogue& e, int64_t b, int64_t i, int64_t j, float acc) {
  float v = e.alpha * acc;
  if (e.bias) v += to_f32(static_cast<const T*>(e.bias)[e.bias_on_i ? i : j]);
  if (e.pre.p) static_cast<T*>(e.pre.p)[b * e.pre.bs + i * e.pre.is + j * e.pre.js] = from_f32<T>(v);
  v = act_f32<sizeof(T) == 2>(v, e.act);
  if (e.res.p) v = fmaf(e.beta, to_f32(static_cast<const T*>(e.res.p)[b * e.res.bs + i * e.res.is + j * e.res.js]), v);
  static_cast<T*>(e.y.p)[b * e.y.bs + i * e.y.is + j * e.y.js] = from_f32<T>(v);
}

// Launchers. gemm_simt.cu
cudaError_t launch_gemm_simt(const GemmProblem& g, cudaStream_t s);
int simt_split(const GemmProblem& g, int sms);

// gemm_skinny.cu: g.J columns in passes of up to 8
cudaError_t launch_gemm_skinny(const GemmProblem& g, int sms, cudaStream_t s);

// SM count of the current device.
inline cudaError_t device_sms(int* sms) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  return e == cudaSuccess ? cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) : e;
}

// Test only: which wait runs out (read per call). 1: one before the first product; in the
// grid-wide orthogonalisation also 2: one in its last product, 3: the last barrier of its grid.
inline int injected_timeout() {
  const char* t = getenv("B2C_GEMM_INJECT_TIMEOUT");
  return t ? atoi(t) : 0;
}

// dP = dY act'(pre) (rounded to the type once), and the column sums of the
// unrounded dP. gemm_dact.cu
struct DactParams {
  int dtype, act;
  const void* dY;      // (batch, M, N), strides below
  int64_t dy_bs, dy_rs, dy_cs;
  const void* pre;     // null where act is none
  int64_t pre_bs, pre_rs, pre_cs;
  void* dP;            // (batch, M, N) contiguous, null where only the sums are wanted
  void* dbias;         // (N,), null where unwanted
  void* dR;            // beta dY, contiguous, null where unwanted
  float beta;
  int64_t batch, M, N;
  float* ws;           // dact_ws_floats() floats where dbias is wanted
};
size_t dact_ws_floats(int64_t batch, int64_t M, int64_t N);
cudaError_t launch_gemm_dact(const DactParams& p, cudaStream_t s);

// polar.cu
struct PolarParams {
  int dtype;
  const void* G;       // (batch, m, n), strides below
  int64_t bs, rs, cs;
  void* out;           // (batch, m, n), contiguous for the caller's m and n
  int64_t out_rs, out_cs;  // set by launch_polar, which may take G as its transpose
  int64_t batch, m, n;
  const float* coef;   // host, steps x 3
  int steps;
  double eps;
  void* ws;
};
// The largest |a v + b v^3 + c v^5| over v in [0, hi].
double polar_poly_bound(double a, double b, double c, double hi);
size_t polar_ws_bytes(const PolarParams& p);
cudaError_t launch_polar(const PolarParams& p, cudaStream_t s);

}  // namespace b2c
