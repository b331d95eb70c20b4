// Newton-Schulz orthogonalisation of small matrices, the whole iteration in
// one CTA: X (smaller side `side` <= 128, longer side L) stays in shared
// memory as f16 planes, S and P share a second buffer, the sums are in tensor
// memory, and the matrix is read and written once.
//
// A CTA stacks g = 128 / side matrices (fewer where that would leave SMs
// idle) into the 128 rows of the tensor-core tile. S of the stack is block
// diagonal: only the diagonal blocks are written to shared memory, the rest of
// that buffer stays zero, and so P and P X keep the matrices apart. A matrix
// with a non-finite entry is left out (zeros) and written as NaN, since 0 * NaN
// would reach its neighbours.
//
// The buffer of X serves as three operands without a copy. Its layout, blocks
// of 64 columns with 128-byte swizzled rows, is K-major for S = X X^T and, read
// the other way, MN-major for P X.
//
// A matrix whose longer side does not fit is shared by a cluster of 2 to 8
// CTAs, each with some of the columns of X: S is then the sum of their parts,
// taken through distributed shared memory, and P X stays local (16 x 128 x 512
// float32: 82 us, with a grid for each product 173; a step costs 4 to 6 us more
// than one CTA's). Idle SMs join in the same way.
//
// The sums of S, P and P X stay in one accumulator: at most 192 additions of 16 products, each cut off at the
// accumulator's last place, the 128 of the small planes before the 64 that matter (10,000 x 64 x 64 float32: 8e-7 from
// the 64-bit iteration, float32 products 1.0e-6).
//
// Bound by the phases of a step in turn (product, conversion of the sums to
// the next operand, barrier): two CTAs share an SM and fill each other's gaps.

#include "b2c_kernels.cuh"
#include "gemm_tc.cuh"
#include "polar.cuh"
#include "tcgen05.cuh"

namespace b2c {

__device__ unsigned int g_polar_fault;

namespace {

constexpr int kBlockBytes = 16384;  // 128 rows x 64 columns of f16
constexpr int kMaxStepsC = 64;
constexpr int kRowsInFlight = 4;  // rows that a warp loads at a time
constexpr int kSmemMaxC = 232448 - 4096;

// S is stored times ss, P times sp; the sums of S are 2^28 S, of P ss^2 S S,
// of P X 2^14 sp P X.
struct CtaStep {
  float k1, k2, k3, k4, kp;  // ss / 2^28, c sp / ss^2, b sp / 2^28, 1 / sp, sp / 2^28
  float a, b, c;
};
constexpr float kUnitS = 1.f / (kPolarScale * kPolarScale);

struct CtaParams {
  const void* G;
  int64_t bs, sr, sl;     // strides of batch, small index, long index
  void* out;
  int64_t obs, orr, ol;
  int64_t batch;
  int cl, chunk, ppitch;  // CTAs of a cluster, columns of X each, pitch of a part of S
  int side, L, g, xblocks, sblocks, kk, steps, along_l, lanes_per_row, blockwise, vec_in, vec_out, inject;
  double eps;
  CtaStep step[kMaxStepsC];
};

// Byte offset of 8 columns (16 bytes) of a row in a 128-byte swizzled buffer
// of 64-column blocks.
__device__ __forceinline__ int unit_off(int row, int col8) {
  return (col8 >> 3) * kBlockBytes + row * 128 + (((col8 & 7) ^ (row & 7)) << 4);
}

__device__ __forceinline__ uint64_t block_desc(uint32_t addr, int inner) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(inner ? (kBlockBytes >> 4) : 1) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <int PLANES>
__device__ __forceinline__ void halves(const float (&v)[8], __half2 (&h)[PLANES][4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    h[0][k] = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
    if constexpr (PLANES == 2) {
      const float2 f = __half22float2(h[0][k]);
      h[1][k] = __floats2half2_rn(v[2 * k] - f.x, v[2 * k + 1] - f.y);
    }
  }
}
template <int PLANES>
__device__ __forceinline__ void store_unit(unsigned char* buf, int plane_bytes, int off, const float (&v)[8]) {
  __align__(16) __half2 h[PLANES][4];
  halves<PLANES>(v, h);
#pragma unroll
  for (int pl = 0; pl < PLANES; ++pl)
    *reinterpret_cast<uint4*>(buf + pl * plane_bytes + off) = *reinterpret_cast<const uint4*>(h[pl]);
}

// hi + lo of 8 columns.
template <int PLANES>
__device__ __forceinline__ void load_halves(const unsigned char* buf, int plane_bytes, int off, float (&v)[8]) {
  const uint4 h = *reinterpret_cast<const uint4*>(buf + off);
  const __half2* a = reinterpret_cast<const __half2*>(&h);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = __half22float2(a[k]);
    v[2 * k] = f.x, v[2 * k + 1] = f.y;
  }
  if constexpr (PLANES == 2) {
    const uint4 l = *reinterpret_cast<const uint4*>(buf + plane_bytes + off);
    const __half2* c = reinterpret_cast<const __half2*>(&l);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __half22float2(c[k]);
      v[2 * k] += f.x, v[2 * k + 1] += f.y;
    }
  }
}

// Shared memory of the q-th CTA of the cluster, at the place of a pointer of this one.
__device__ __forceinline__ double peer_double(const double* p, int q) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(map_rank(smem_u32(p), q)) : "memory");
  return v;
}
__device__ __forceinline__ void peer_load8(const float* p, int q, float (&v)[8]) {
  const uint32_t a = map_rank(smem_u32(p), q);
#pragma unroll
  for (int k = 0; k < 8; k += 4)
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[k]), "=f"(v[k + 1]), "=f"(v[k + 2]), "=f"(v[k + 3])
                 : "r"(a + k * 4)
                 : "memory");
}
__device__ __forceinline__ void peer_store_float(float* p, int q, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_rank(smem_u32(p), q)), "f"(v) : "memory");
}
__device__ __forceinline__ void peer_store16(unsigned char* p, int q, const void* v) {
  const uint4 w = *reinterpret_cast<const uint4*>(v);
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(map_rank(smem_u32(p), q)), "r"(w.x), "r"(w.y),
               "r"(w.z), "r"(w.w)
               : "memory");
}

// 8 elements of a row, zeros past its end.
template <typename T>
__device__ __forceinline__ void load_unit8(const T* row, int64_t stride, int c, int n, int vec, float (&v)[8]) {
  if (vec && c + 8 <= n) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < 8 / PER; ++q) {
      const uint4 w = *reinterpret_cast<const uint4*>(row + c + q * PER);
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int k = 0; k < PER; ++k) v[q * PER + k] = to_f32(e[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < n ? to_f32(row[(c + k) * stride]) : 0.f;
  }
}

// CL: a cluster of p.cl CTAs shares a stack, `chunk` columns of X each.
template <typename T, int PLANES, int NT, bool CL>
__global__ void __launch_bounds__(NT, 512 / NT) polar_cta_kernel(const __grid_constant__ CtaParams p) {
  extern __shared__ unsigned char raw[];
  __shared__ double rowsum[NT];
  __shared__ float2 factor[128];  // the scale of a matrix as two powers of two, 0 for a broken one
  __shared__ float first_r[128], sdiag[128], pdiag[128];
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  constexpr int NW = NT / 32, NG = NT / 128;  // warps; threads that share a row of X
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* X = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  const int x_plane = p.xblocks * kBlockBytes, s_plane = p.sblocks * kBlockBytes;
  unsigned char* S = X + PLANES * x_plane;
  const int rank = CL ? (int)cluster_rank() : 0, base = rank * p.chunk, L = CL ? max(0, min(p.chunk, p.L - base)) : p.L;
  float* partial = reinterpret_cast<float*>(S + PLANES * s_plane);  // CL: this CTA's part of S, rows of ppitch floats
  const uint32_t done = smem_u32(bars), never = done + 8;
  const uint64_t limit = p.inject ? 1000000ull : kWaitNs;
  volatile int* gu = &gave_up;

  if (tid == 0) {
    gave_up = 0;
    bar_init(done, 1);
    bar_init(never, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    fence_before();
  }
  // ---- norms ----
  const int64_t m0 = (int64_t)(blockIdx.x / (CL ? p.cl : 1)) * p.g;
  const int have = (int)(p.batch - m0 < p.g ? p.batch - m0 : p.g), rows = have * p.side;
  const T* G = static_cast<const T*>(p.G) + m0 * p.bs + base * p.sl;
  for (int e = tid * 16; e < PLANES * (x_plane + s_plane); e += NT * 16)
    *reinterpret_cast<uint4*>(X + e) = make_uint4(0, 0, 0, 0);
  // rows of X: `lpr` lanes take the 8-element units of a row in turn (its neighbours lie along the lanes), or, where the
  // small index has the smaller stride, NG threads share a row and the lanes run along the rows
  const int units = (L + 7) / 8, lpr = p.lanes_per_row;
  if (p.along_l) {
    const int per = 32 / lpr, sub = lane / lpr, u0 = lane % lpr;
    for (int r0 = warp * per; r0 < rows; r0 += NW * per * kRowsInFlight) {
      double s[kRowsInFlight] = {};
      for (int u = u0; u < units; u += lpr) {
        float v[kRowsInFlight][8];
#pragma unroll
        for (int k = 0; k < kRowsInFlight; ++k) {
          const int r = r0 + sub + k * NW * per, m = r / p.side;
          load_unit8<T>(G + m * p.bs + (r - m * p.side) * p.sr, p.sl, u * 8, r < rows ? L : 0, p.vec_in, v[k]);
        }
#pragma unroll
        for (int k = 0; k < kRowsInFlight; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) s[k] += (double)v[k][e] * (double)v[k][e];
      }
      for (int o = lpr / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < kRowsInFlight; ++k) s[k] += __shfl_xor_sync(kFull, s[k], o);
#pragma unroll
      for (int k = 0; k < kRowsInFlight; ++k) {
        const int r = r0 + sub + k * NW * per;
        if (u0 == 0 && r < rows) {
#pragma unroll
          for (int g = 0; g < NG; ++g) rowsum[r + 128 * g] = g ? 0.0 : s[k];
        }
      }
    }
  } else {
    const int r = tid & 127, m = r / p.side;
    const T* row = G + m * p.bs + (r - m * p.side) * p.sr;
    double s = 0.0;
    if (r < rows) {
      for (int u = tid >> 7; u < units; u += NG) {
        float v[8];
        load_unit8<T>(row, p.sl, u * 8, L, 0, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += (double)v[e] * (double)v[e];
      }
    }
    rowsum[tid] = s;
  }
  __syncthreads();
  for (int m = warp; m < have; m += NW) {
    double s = 0.0;
    for (int r = lane; r < p.side; r += 32)
#pragma unroll
      for (int g = 0; g < NG; ++g) s += rowsum[m * p.side + r + 128 * g];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
    if (CL) {
      if (lane == 0) rowsum[m * p.side] = s;  // this matrix's own entries have been read
    } else if (lane == 0) {
      const PolarNorm n = polar_norm(sqrt(s) + p.eps);
      factor[m] = n.half_scale();
      first_r[m] = n.r;
    }
  }
  if constexpr (CL) {
    __syncwarp();
    cluster_sync();
    if (tid < have) {
      double s = 0.0;
      for (int q = 0; q < p.cl; ++q) s += peer_double(&rowsum[tid * p.side], q);
      const PolarNorm n = polar_norm(sqrt(s) + p.eps);
      factor[tid] = n.half_scale();
      first_r[tid] = n.r;
    }
  }
  __syncthreads();
  // ---- X = G / (|G| + eps), up to the factor r ----
  if (p.along_l) {
    const int per = 32 / lpr, sub = lane / lpr, u0 = lane % lpr;
    for (int r0 = warp * per + sub; r0 < rows; r0 += NW * per * kRowsInFlight) {
      for (int u = u0; u < units; u += lpr) {
        float v[kRowsInFlight][8];
#pragma unroll
        for (int k = 0; k < kRowsInFlight; ++k) {
          const int r = r0 + k * NW * per, m = r / p.side;
          load_unit8<T>(G + m * p.bs + (r - m * p.side) * p.sr, p.sl, u * 8, r < rows ? L : 0, p.vec_in, v[k]);
        }
#pragma unroll
        for (int k = 0; k < kRowsInFlight; ++k) {
          const int r = r0 + k * NW * per;
          const float2 f = r < rows ? factor[r / p.side] : make_float2(0.f, 0.f);
          if (f.x == 0.f) continue;  // no such row, or a broken matrix
#pragma unroll
          for (int e = 0; e < 8; ++e) v[k][e] = v[k][e] * f.x * f.y;
          store_unit<PLANES>(X, x_plane, unit_off(r, u), v[k]);
        }
      }
    }
  } else {
    const int r = tid & 127, m = r / p.side;
    const float2 f = r < rows ? factor[m] : make_float2(0.f, 0.f);
    if (f.x != 0.f) {
      const T* row = G + m * p.bs + (r - m * p.side) * p.sr;
      for (int u = tid >> 7; u < units; u += NG) {
        float v[8];
        load_unit8<T>(row, p.sl, u * 8, L, 0, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * f.x * f.y;
        store_unit<PLANES>(X, x_plane, unit_off(r, u), v);
      }
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot, xa = smem_u32(X), sa = smem_u32(S);
  const uint32_t idesc_s = mma_idesc(1, 0, 0, 128, p.kk);
  constexpr int SEGS = PLANES == 2 ? 3 : 1;  // lo hi, hi lo, hi hi
  auto seg_p = [](int s) { return PLANES == 2 && s == 0 ? 1 : 0; };
  auto seg_q = [](int s) { return s == 1 ? 1 : 0; };
  uint32_t phase = 0;
  if (p.inject && blockIdx.x == 0) bar_wait(never, 0, gu, limit, &g_polar_fault);
  auto wait = [&] {
    bar_wait(done, phase, gu, limit, &g_polar_fault);
    phase ^= 1;
    fence_after();
  };

  // this lane's row, its matrix and where that matrix lies among the columns of S
  const int quad = warp & 3, group = warp >> 2, row = quad * 32 + lane;
  const int mine = row / p.side, lo = mine * p.side, hi = mine < p.g ? lo + p.side : lo;
  const int first = quad * 32 / p.side * p.side, last = min((quad * 32 + 31) / p.side * p.side + p.side, p.kk);
  const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);

  const float r0 = row < rows && factor[mine].x != 0.f ? first_r[mine] : 1.f;
  // with one plane, S and P are held without their diagonals, which stay in float32 (see polar.cu)
  constexpr bool kSplitDiag = PLANES == 1;
  for (int t = 0; t < p.steps; ++t) {
    const CtaStep k = p.step[t];
    const float f1 = t ? 1.f : r0, f2 = f1 * f1, k3 = CL ? k.k3 / k.k1 : k.k3 * f2, kp = CL ? k.kp / k.k1 : k.kp * f2;
    // ---- S = X X^T ----
    if (warp == 0) {
      if (elect_one()) {
#pragma unroll
        for (int s = 0; s < SEGS; ++s) {
          const uint64_t dp = block_desc(xa + seg_p(s) * x_plane, 0), dq = block_desc(xa + seg_q(s) * x_plane, 0);
          for (int b = 0; b < p.xblocks; ++b)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mma<1>(tmem, dp + b * (kBlockBytes >> 4) + q * 2, dq + b * (kBlockBytes >> 4) + q * 2, idesc_s, s + b + q > 0);
        }
        commit<1>(done);
      }
      __syncwarp();  // a warp that sleeps on the barrier sleeps as a whole
    }
    wait();
    if constexpr (CL) {
      // the sum over the cluster: every CTA puts its part into its own shared memory, takes a share of the rows of all
      // parts, in order, and gives the result to all. One that has given up spreads NaN.
      const float f = *gu ? __int_as_float(0x7fffffff) : k.k1 * f2;
      for (int c0 = first / 32 * 32; c0 < last; c0 += 32) {
        if (((c0 - first / 32 * 32) >> 5) % NG != group) continue;
        float v[32];
        tmem_row32(lanes + c0, v);
        float4* at = reinterpret_cast<float4*>(partial + row * p.ppitch + c0);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = (unsigned)(c0 + 4 * q + e - lo) < (unsigned)(hi - lo) ? v[4 * q + e] * f : 0.f;
          if (c0 + 4 * q < p.kk) at[q] = make_float4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
      cluster_sync();
      const int share = 128 / p.cl, per_row = p.kk / 8;
      for (int u = tid; u < share * per_row; u += NT) {
        const int r = rank * share + u / per_row, c8 = u % per_row, m = r / p.side;
        // blocks off the diagonal stay zero
        if (r >= p.kk || c8 * 8 + 8 <= m * p.side || c8 * 8 >= m * p.side + p.side) continue;
        float v[8] = {};
        const float* at = partial + r * p.ppitch + c8 * 8;
        // from this CTA's own part on, so that the CTAs read from different ones, two at a time
        for (int q = 0; q < p.cl; q += 2) {
          float w[2][8];
          peer_load8(at, (rank + q) & (p.cl - 1), w[0]);
          peer_load8(at, (rank + q + 1) & (p.cl - 1), w[1]);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += w[0][e] + w[1][e];
        }
        float d = 0.f;
        if constexpr (kSplitDiag) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c8 * 8 + e == r) d = v[e] * (kUnitS / k.k1), v[e] = 0.f;
        }
        const bool diag = kSplitDiag && r - c8 * 8 >= 0 && r - c8 * 8 < 8;
        __align__(16) __half2 h[PLANES][4];
        halves<PLANES>(v, h);
        for (int i = 0; i < p.cl; ++i) {
          const int q = (rank + i) & (p.cl - 1);
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) peer_store16(S + pl * s_plane + unit_off(r, c8), q, h[pl]);
          if (diag) peer_store_float(&sdiag[r], q, d);
        }
      }
      asm volatile("fence.proxy.async.shared::cluster;" ::: "memory");
      __syncwarp();
      cluster_sync();
    } else {
      for (int c0 = first / 32 * 32; c0 < last; c0 += 32) {
        if (((c0 - first / 32 * 32) >> 5) % NG != group) continue;
        float v[32];
        tmem_row32(lanes + c0, v);
  #pragma unroll
        for (int u = 0; u < 4; ++u) {
          float w[8];
          const float f = k.k1 * f2;
  #pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int c = c0 + u * 8 + e;
            if (kSplitDiag && c == row) sdiag[row] = v[u * 8 + e] * f2 * kUnitS;
            w[e] = (unsigned)(c - lo) < (unsigned)(hi - lo) && !(kSplitDiag && c == row) ? v[u * 8 + e] * f : 0.f;
          }
          if (c0 + u * 8 < p.kk) store_unit<PLANES>(S, s_plane, unit_off(row, (c0 >> 3) + u), w);
        }
      }
    }
    fence_before();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    fence_after();
    // ---- P = c S S + b S ----
    if (warp == 0) {
      // a matrix's columns of S S take its own rows of S alone: the rest are zeros
      const int width = p.blockwise ? p.side : p.kk;
      const uint32_t idesc_p = mma_idesc(1, 0, 0, 128, width);
      if (elect_one()) {
        for (int c0 = 0; c0 < p.kk; c0 += width)
#pragma unroll
          for (int s = 0; s < SEGS; ++s) {
            const uint64_t dp = block_desc(sa + seg_p(s) * s_plane, 0), dq = block_desc(sa + seg_q(s) * s_plane + c0 * 128, 0);
            for (int c = c0; c < c0 + width; c += 16) {
              const int off = (c >> 6) * (kBlockBytes >> 4) + (c & 63) / 8;
              mma<1>(tmem + 128 + c0, dp + off, dq + off, idesc_p, s + (c - c0) > 0);
            }
          }
        commit<1>(done);
      }
      __syncwarp();
    }
    wait();
    const float di = kSplitDiag && row < p.kk ? sdiag[row] : 0.f;
    for (int c0 = first / 32 * 32; c0 < last; c0 += 32) {
      if (((c0 - first / 32 * 32) >> 5) % NG != group) continue;
      float v[32], w[32];
      if constexpr (CL) {  // the whole S is in shared memory alone
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float x[8] = {};
          if (c0 + u * 8 < p.kk) load_halves<PLANES>(S, s_plane, unit_off(row, (c0 >> 3) + u), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[u * 8 + e] = x[e];
        }
      } else {
        tmem_row32(lanes + c0, v);
      }
      tmem_row32(lanes + 128 + c0, w);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = c0 + u * 8 + e;
          const bool in = (unsigned)(c - lo) < (unsigned)(hi - lo);
          const float o = v[u * 8 + e], oo = w[u * 8 + e] * k.k2;
          if constexpr (kSplitDiag) {
            const float b = fmaf(k.c, di + sdiag[c], k.b) * kp;
            x[e] = in && c != row ? fmaf(o, b, oo) : 0.f;
            if (c == row) pdiag[row] = fmaf(oo, k.k4, di * fmaf(k.c, di, k.b));
          } else {
            x[e] = in ? fmaf(o, k3, oo) : 0.f;
          }
        }
        if (c0 + u * 8 < p.kk) store_unit<PLANES>(S, s_plane, unit_off(row, (c0 >> 3) + u), x);
      }
    }
    fence_before();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    fence_after();
    const float ka = kSplitDiag ? k.a + (row < p.kk ? pdiag[row] : 0.f) : k.a;
    // ---- X <- P X + a X, up to 256 columns at a time ----
    for (int b0 = 0; b0 < p.xblocks; b0 += 4) {
      const int nb = min(4, p.xblocks - b0);
      if (warp == 0) {
        const uint32_t idesc_x = mma_idesc(1, 0, 1, 128, nb * 64);
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < SEGS; ++s) {
            const uint64_t dp = block_desc(sa + seg_p(s) * s_plane, 0),
                           dq = block_desc(xa + seg_q(s) * x_plane + b0 * kBlockBytes, 1);
            for (int q = 0; q < p.kk / 16; ++q)
              mma<1>(tmem, dp + (q >> 2) * (kBlockBytes >> 4) + (q & 3) * 2, dq + q * (2048 >> 4), idesc_x, s + q > 0);
          }
          commit<1>(done);
        }
        __syncwarp();
      }
      wait();
      for (int c0 = group * 32; c0 < nb * 64; c0 += NG * 32) {
        float v[32];
        tmem_row32(lanes + c0, v);
        const int c = b0 * 64 + c0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int off = unit_off(row, (c >> 3) + u);
          const uint4 xh = *reinterpret_cast<const uint4*>(X + off);
          const __half* h = reinterpret_cast<const __half*>(&xh);
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = __half2float(h[e]);
          if constexpr (PLANES == 2) {
            const uint4 xl = *reinterpret_cast<const uint4*>(X + x_plane + off);
            const __half* l = reinterpret_cast<const __half*>(&xl);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] += __half2float(l[e]);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[u * 8 + e] = f1 * fmaf(ka, w[e], v[u * 8 + e] * k.k4);
          if (t < p.steps - 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = v[u * 8 + e];
            store_unit<PLANES>(X, x_plane, off, w);
          }
        }
        if (t == p.steps - 1 && row < rows) {
          const float nan = __int_as_float(0x7fffffff);
          const float f = factor[mine].x == 0.f || *gu ? nan : 1.f / kPolarScale;
          T* o = static_cast<T*>(p.out) + (m0 + mine) * p.obs + (row - lo) * p.orr + (base + c) * p.ol;
          constexpr int PER = 16 / sizeof(T);
          if (p.vec_out && c + 32 <= L) {
#pragma unroll
            for (int u = 0; u < 32 / PER; ++u) {
              uint4 w;
              T* q = reinterpret_cast<T*>(&w);
#pragma unroll
              for (int e = 0; e < PER; ++e) q[e] = from_f32<T>(v[u * PER + e] * f);
              *reinterpret_cast<uint4*>(o + u * PER) = w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c + e < L) o[e * p.ol] = from_f32<T>(v[e] * f);
          }
        }
      }
      fence_before();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();
      fence_after();
    }
  }
  if (gave_up) {
    // MMAs still in flight end within microseconds
    const uint64_t t0 = now_ns();
    while (now_ns() - t0 < 20000000ull) {
    }
    __syncthreads();
  }
  if constexpr (CL) cluster_sync();  // no CTA ends while another may write to it
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem));
}

template <typename T, int PLANES, int NT, bool CL>
cudaError_t launch_n(const CtaParams& p, size_t smem, unsigned grid, cudaStream_t s) {
  auto kern = polar_cta_kernel<T, PLANES, NT, CL>;
  static int cache[64];
  int occ = 0;
  const cudaError_t e = kernel_occupancy(kern, NT, smem, cache, &occ);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)p.cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CL ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

// 16 warps where one CTA has an SM to itself, by its shared memory or because
// there are no more CTAs than SMs; otherwise two CTAs of 8.
template <typename T, int PLANES>
cudaError_t launch_c(const CtaParams& p, size_t smem, unsigned grid, int sms, cudaStream_t s) {
  if (p.cl > 1) return launch_n<T, PLANES, 512, true>(p, smem, grid, s);
  if (smem > 113 * 1024 || grid <= (unsigned)sms) return launch_n<T, PLANES, 512, false>(p, smem, grid, s);
  return launch_n<T, PLANES, 256, false>(p, smem, grid, s);
}

// How a problem is laid out over CTAs.
struct CtaPlan {
  int planes, cl, g, xblocks, kk;  // planes 0: does not fit
  size_t smem;
};

int rounded(int64_t rows) { return (int)((rows + 15) / 16 * 16); }

size_t plan_smem(int planes, int cl, int xblocks, int kk) {
  return 1024 + (size_t)planes * (xblocks + (kk + 63) / 64) * kBlockBytes + (cl > 1 ? (size_t)128 * (kk + 4) * 4 : 0);
}

// Two planes, or one for bfloat16 results where two do not fit: they cost three
// products instead of one, which these sizes hide, and leave a bfloat16
// result its own rounding alone. As few CTAs a matrix as hold it, and more, up to
// 8 of at least 128 columns, where that leaves SMs idle; as many matrices a CTA
// as keep two CTAs on every SM.
CtaPlan plan_cta(const PolarParams& p, int sms) {
  const int64_t side = p.m < p.n ? p.m : p.n, L = p.m < p.n ? p.n : p.m;
  CtaPlan r{};
  if (side > 128 || L > 64 * 8 * 16) return r;
  const int blocks = (int)((L + 63) / 64);
  for (int planes = 2; planes >= (p.dtype == B2C_BF16 ? 1 : 2) && !r.planes; --planes)
    for (int cl = 1; cl <= 8 && !r.planes; cl *= 2)
      if (plan_smem(planes, cl, (blocks + cl - 1) / cl, rounded(side)) <= (size_t)kSmemMaxC) r.planes = planes, r.cl = cl;
  if (!r.planes) return r;
  while (r.cl < 8 && (int64_t)p.batch * r.cl * 2 <= sms && (blocks + 2 * r.cl - 1) / (2 * r.cl) >= 2 &&
         plan_smem(r.planes, r.cl * 2, (blocks + 2 * r.cl - 1) / (2 * r.cl), rounded(side)) <= (size_t)kSmemMaxC)
    r.cl *= 2;
  r.xblocks = (blocks + r.cl - 1) / r.cl;
  const int64_t slots = (r.cl > 1 ? 1 : 2) * (int64_t)sms;
  int64_t g = (p.batch * r.cl + slots - 1) / slots;
  if (g > 128 / side) g = 128 / side;
  while (g > 1 && plan_smem(r.planes, r.cl, r.xblocks, rounded(g * side)) > (size_t)kSmemMaxC) --g;
  r.g = (int)g;
  r.kk = rounded(g * side);
  r.smem = plan_smem(r.planes, r.cl, r.xblocks, r.kk);
  return r;
}

}  // namespace

bool polar_cta_fits(const PolarParams& p) { return plan_cta(p, 148).planes > 0; }

cudaError_t launch_polar_cta(const PolarParams& in, int sms, cudaStream_t s) {
  CtaParams p{};
  const bool wide = in.m <= in.n;
  const CtaPlan plan = plan_cta(in, sms);
  p.G = in.G;
  p.bs = in.bs, p.sr = wide ? in.rs : in.cs, p.sl = wide ? in.cs : in.rs;
  p.out = in.out;
  p.obs = in.m * in.n, p.orr = wide ? in.out_rs : in.out_cs, p.ol = wide ? in.out_cs : in.out_rs;
  p.batch = in.batch;
  p.side = (int)(wide ? in.m : in.n);
  p.L = (int)(wide ? in.n : in.m);
  p.cl = plan.cl;
  p.xblocks = plan.xblocks;
  p.chunk = plan.xblocks * 64;
  p.g = plan.g;
  p.kk = plan.kk;
  p.ppitch = p.kk + 4;
  p.sblocks = (p.kk + 63) / 64;
  p.blockwise = p.side % 16 == 0;
  p.along_l = p.sl <= p.sr || p.side == 1;
  p.steps = in.steps;
  p.eps = in.eps;
  p.inject = injected_timeout() == 1;
  p.lanes_per_row = 1;
  while (p.lanes_per_row < 32 && p.lanes_per_row * 8 < (p.L < p.chunk ? p.L : p.chunk)) p.lanes_per_row *= 2;
  const int64_t per = in.dtype == B2C_F32 ? 4 : 8;
  p.vec_in = p.sl == 1 && (reinterpret_cast<uintptr_t>(in.G) & 15) == 0 && p.sr % per == 0 && p.bs % per == 0;
  const int64_t elt = in.dtype == B2C_F32 ? 4 : 2;
  p.vec_out = p.ol == 1 && (reinterpret_cast<uintptr_t>(in.out) & 15) == 0 && p.orr * elt % 16 == 0 && p.obs * elt % 16 == 0;
  double hi = 1.0;
  for (int t = 0; t < in.steps; ++t) {
    const double a = in.coef[3 * t], b = in.coef[3 * t + 1], c = in.coef[3 * t + 2], t2 = hi * hi, sx = kPolarScale;
    const double ss = polar_scale_for(t2), sp = polar_scale_for(fabs(b) * t2 + fabs(c) * t2 * t2);
    p.step[t] = CtaStep{(float)(ss / (sx * sx)), (float)(c * sp / (ss * ss)), (float)(b * sp / (sx * sx)), (float)(1 / sp),
                        (float)(sp / (sx * sx)), (float)a, (float)b, (float)c};
    hi = polar_poly_bound(a, b, c, hi);
  }
  size_t smem = plan.smem;
  if (smem < 77 * 1024) smem = 77 * 1024;  // two CTAs at most: each holds half of the tensor memory
  const int64_t ctas = (in.batch + p.g - 1) / p.g * p.cl;
  if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const unsigned grid = (unsigned)ctas;
  switch (in.dtype) {
    case B2C_F32: return launch_c<float, 2>(p, smem, grid, sms, s);
    case B2C_BF16:
      return plan.planes == 2 ? launch_c<__nv_bfloat16, 2>(p, smem, grid, sms, s)
                              : launch_c<__nv_bfloat16, 1>(p, smem, grid, sms, s);
    default: return launch_c<__half, 2>(p, smem, grid, sms, s);
  }
}

cudaError_t polar_take_fault(unsigned int* fault) {
  unsigned int f = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&f, g_polar_fault, sizeof(unsigned int));
  if (e != cudaSuccess) return e;
  *fault |= f;
  return cudaMemcpyToSymbol(g_polar_fault, &zero, sizeof(unsigned int));
}

}  // namespace b2c
