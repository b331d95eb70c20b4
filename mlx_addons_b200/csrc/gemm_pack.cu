// Copies of operands for the tensor-core products: rows padded to a multiple
// of 8 elements, so that every row starts on 16 bytes, and float32 values as
// three bf16 planes.
//
// Bound by HBM: 1000 x 256 x 256 float32 in 100 us, 6.5 TB/s. The axis with the
// smaller stride stays the inner one (the product reads either order), so reads
// and writes both run along it; a thread takes 8 neighbouring elements and
// writes each plane's as 16 bytes.
#include "b2c_kernels.cuh"
#include "gemm_tc.cuh"

namespace b2c {

namespace {

struct PackParams {
  const void* src;
  int64_t bs, os, is;            // strides of batch, outer, inner
  int64_t batch, outer, inner, pitch, plane;
  uint16_t* dst;
};

// Rounds to bf16; a finite value whose nearest is infinite is cut off instead.
__device__ __forceinline__ uint16_t bf16_finite(float x) {
  const uint16_t r = __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return (r & 0x7fff) == 0x7f80 ? (uint16_t)(__float_as_uint(x) >> 16) : r;
}
__device__ __forceinline__ float bf16_value(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

// x as hi + 2^-8 mid + 2^-16 lo, each bf16: the remainders are exact, so the three
// hold all 24 bits. Without the powers of two the last bits of a small x (below 2^-110)
// would fall under 2^-133, bf16's smallest value; with them float32's own smallest,
// 2^-149, is 2^-133 in lo. |mid| and |lo| stay within |hi|, so nothing overflows that hi
// would not.
//
// An infinity or a NaN lies in lo, which meets the other operand's hi alone, with a
// 1 of its sign in hi: in hi it would meet planes that are zero, and infinity times 0
// is NaN. hi is zero for a zero alone, so that an infinity makes NaN of that and of nothing else.
__device__ __noinline__ void thirds(float x, uint16_t& hi, uint16_t& mid, uint16_t& lo) {
  if (isfinite(x)) {
    hi = bf16_finite(x);
    if ((hi & 0x7fff) == 0 && x != 0.f) hi |= 1;
    const float r = (x - bf16_value(hi)) * 256.f;
    mid = bf16_finite(r);
    lo = bf16_finite((r - bf16_value(mid)) * 256.f);
  } else {
    lo = __bfloat16_as_ushort(__float2bfloat16_rn(x));
    hi = (lo & 0x8000) | 0x3f80;
    mid = 0;
  }
}
// Zeros, and values whose bf16 is neither zero nor infinite, go two at a time and without the cases above (an
// operand of 300 x 256 x 256: 28 us; with those cases for every value 37).
__device__ __forceinline__ bool common(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u == 0 || u - 0x8001u < 0x7f7f8000u - 0x8001u;
}
__device__ __forceinline__ uint32_t bf16x2(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void thirds2(float a, float b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = bf16x2(a, b);
  const float ra = (a - __uint_as_float(hi << 16)) * 256.f, rb = (b - __uint_as_float(hi & 0xffff0000u)) * 256.f;
  mid = bf16x2(ra, rb);
  lo = bf16x2((ra - __uint_as_float(mid << 16)) * 256.f, (rb - __uint_as_float(mid & 0xffff0000u)) * 256.f);
}

// VEC: rows of unit stride that start on 16 bytes, whole units of 8 in two or
// one loads of 16 bytes.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) gemm_pack_kernel(const PackParams p) {
  const int64_t units = (p.inner + 7) / 8, rows = p.batch * p.outer, total = rows * units;
  const bool narrow = total < ((int64_t)1 << 32);  // 64-bit divisions take as long as a unit's loads
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    int64_t row = 0, b = 0;
    if (rows > 1) {
      row = narrow ? (int64_t)((uint32_t)t / (uint32_t)units) : t / units;
      if (p.batch > 1) b = narrow ? (int64_t)((uint32_t)row / (uint32_t)p.outer) : row / p.outer;
    }
    const int64_t u = t - row * units, o = row - b * p.outer;
    const int64_t src = b * p.bs + o * p.os + u * 8 * p.is, dst = row * p.pitch + u * 8;
    const int n = (int)(p.inner - u * 8 < 8 ? p.inner - u * 8 : 8);
    if constexpr (F32) {
      const float* s = static_cast<const float*>(p.src) + src;
      __align__(16) float x[8];
      if (VEC && n == 8) {
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(s);
        *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(s + 4);
      } else {
        // every load is issued, past the end that of the first again: none waits for a branch
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = s[c < n ? c * p.is : 0];
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = c < n ? x[c] : 0.f;
      }
      __align__(16) uint32_t h[4], m[4], l[4];
      bool all = true;
#pragma unroll
      for (int c = 0; c < 8; ++c) all &= common(x[c]);
      if (all) {
#pragma unroll
        for (int c = 0; c < 4; ++c) thirds2(x[2 * c], x[2 * c + 1], h[c], m[c], l[c]);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint16_t p0, p1, p2, q0, q1, q2;
          thirds(x[2 * c], p0, p1, p2);
          thirds(x[2 * c + 1], q0, q1, q2);
          h[c] = p0 | (uint32_t)q0 << 16, m[c] = p1 | (uint32_t)q1 << 16, l[c] = p2 | (uint32_t)q2 << 16;
        }
      }
      *reinterpret_cast<uint4*>(p.dst + dst) = *reinterpret_cast<const uint4*>(h);
      *reinterpret_cast<uint4*>(p.dst + p.plane + dst) = *reinterpret_cast<const uint4*>(m);
      *reinterpret_cast<uint4*>(p.dst + 2 * p.plane + dst) = *reinterpret_cast<const uint4*>(l);
    } else {
      const uint16_t* s = static_cast<const uint16_t*>(p.src) + src;
      __align__(16) uint16_t h[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) h[c] = s[c < n ? c * p.is : 0];
#pragma unroll
      for (int c = 0; c < 8; ++c) h[c] = c < n ? h[c] : (uint16_t)0;
      *reinterpret_cast<uint4*>(p.dst + dst) = *reinterpret_cast<const uint4*>(h);
    }
  }
}

}  // namespace

PackPlan plan_pack(int dtype, const GemmOperand& o, int64_t batch, int64_t rows, int64_t K) {
  PackPlan r{};
  TcOperand direct;
  r.needed = dtype == B2C_F32 || !tc_direct(o, batch, rows, K, &direct);
  if (!r.needed) return r;
  const int64_t rs = rows == 1 ? INT64_MAX : o.rs, ks = K == 1 ? INT64_MAX : o.ks;
  r.rows_inner = rs < ks || (rs == ks && rows > K);
  r.batch = o.bs == 0 ? 1 : batch;
  r.outer = r.rows_inner ? K : rows;
  r.inner = r.rows_inner ? rows : K;
  r.pitch = (r.inner + 7) / 8 * 8;
  r.plane = r.batch * r.outer * r.pitch;
  r.bytes = (r.plane * 2 * (dtype == B2C_F32 ? 3 : 1) + 255) / 256 * 256;
  return r;
}

cudaError_t launch_pack(int dtype, const GemmOperand& o, const PackPlan& plan, void* dst, TcOperand* out, cudaStream_t s) {
  PackParams p{o.p, o.bs, plan.rows_inner ? o.ks : o.rs, plan.rows_inner ? o.rs : o.ks, plan.batch, plan.outer,
                     plan.inner, plan.pitch, plan.plane, static_cast<uint16_t*>(dst)};
  const int64_t total = plan.batch * plan.outer * ((plan.inner + 7) / 8), blocks = (total + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16);
  const bool vec = p.is == 1 && (reinterpret_cast<uintptr_t>(p.src) & 15) == 0 && p.os % 4 == 0 && p.bs % 4 == 0;
  // rows that follow one another without a gap are one row
  if (p.is == 1 && p.pitch == p.inner) {
    if (p.os == p.inner) p.inner *= p.outer, p.pitch = p.inner, p.outer = 1;
    if (p.outer == 1 && p.bs == p.inner) p.inner *= p.batch, p.pitch = p.inner, p.batch = 1;
  }
  if (dtype != B2C_F32) gemm_pack_kernel<false, false><<<grid, 256, 0, s>>>(p);
  else if (vec) gemm_pack_kernel<true, true><<<grid, 256, 0, s>>>(p);
  else gemm_pack_kernel<true, false><<<grid, 256, 0, s>>>(p);
  *out = TcOperand{dst, plan.outer * plan.pitch, plan.pitch, plan.plane, plan.rows_inner, plan.batch == 1};
  return cudaGetLastError();
}

}  // namespace b2c
