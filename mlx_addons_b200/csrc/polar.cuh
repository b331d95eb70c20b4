// Newton-Schulz orthogonalisation: what polar.cu and polar_cta.cu share.
#pragma once

#include <cmath>

#include "gemm.cuh"

namespace b2c {

// X is held times 2^14: singular values up to 3.5 stay below f16's 65504.
constexpr float kPolarScale = 16384.f;

// The largest power of two that keeps values up to `bound` within 2^15.
inline float polar_scale_for(double bound) {
  const double b = bound < 1e-3 ? 1e-3 : bound;
  return (float)exp2(floor(log2(32768.0 / b)));
}

// How a matrix of this norm (|G|_F + eps) is held: G * scale, scale a power of
// two that puts the norm into [2^13, 2^14), and r = 2^14 / (norm * scale) in
// (1, 2]. A norm of zero (0 / 0) or one that is not finite gives r = NaN.
struct PolarNorm {
  double scale;
  float r;
  int e;  // scale = 2^e
  // The scale as two float powers of two, neither beyond float's range.
  __device__ __forceinline__ float2 half_scale() const {
    return scale == 0.0 ? make_float2(0.f, 0.f) : make_float2(scalbnf(1.f, e / 2), scalbnf(1.f, e - e / 2));
  }
};
__device__ __forceinline__ PolarNorm polar_norm(double norm) {
  if (!isfinite(norm) || norm == 0.0) return PolarNorm{0.0, __int_as_float(0x7fffffff), 0};
  int q;
  const double f = frexp(norm, &q);
  return PolarNorm{scalbn(16384.0, -q), (float)(1.0 / f), 14 - q};
}

// Scratch of the forms that keep X, S and P in memory (polar.cu).
struct PolarScratch {
  int64_t side, pitch_x, pitch_s, x_plane, s_plane;
  __half *X0, *X1, *S, *P;  // X0 holds G, scaled
  float *ds, *dp, *r;       // diagonals of S and P, (batch, side); the first step's factors, (batch,)
  unsigned int* counter;    // zero
};
bool polar_grid_fits(const PolarParams& p, int sms);
cudaError_t launch_polar_grid(const PolarParams& p, const PolarScratch& w, int sms, cudaStream_t s);

// Both take a problem whose rows lie no closer together than its columns.
bool polar_cta_fits(const PolarParams& p);
cudaError_t launch_polar_cta(const PolarParams& p, int sms, cudaStream_t s);

}  // namespace b2c
