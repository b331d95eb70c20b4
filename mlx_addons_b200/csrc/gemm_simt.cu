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
//
// Too few tiles for the GPU: k is split over a cluster of up to 8 CTAs, which
// leave their sums in shared memory; each then joins, in order, and finishes its
// share of the tile's rows.
#include "b2c_kernels.cuh"
#include "gemm.cuh"
#include "tcgen05.cuh"

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
  __device__ __forceinline__ SliceLoader(const GemmOperand& o, int64_t b, int64_t r0, int64_t rows, int64_t k0, int64_t K) {
    const bool along_k = o.ks <= o.rs;
    r = along_k ? threadIdx.x / TK : threadIdx.x % TS;
    k = along_k ? threadIdx.x % TK : threadIdx.x / TS;
    dr = along_k ? kSimtThreads / TK : 0;
    dk = along_k ? 0 : kSimtThreads / TS;
    at = static_cast<const T*>(o.p) + b * o.bs + (r0 + r) * o.rs + (k0 + k) * o.ks;
    step = dr * o.rs + dk * o.ks;
    kstep = TK * o.ks;
    left_r = rows - r0 - r;
    left_k = K - k0 - k;
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

struct SimtParams {
  GemmProblem g;
  int64_t tiles_i, tiles_j;
  int64_t k_per;  // k of one CTA of a cluster
  int split;      // CTAs of a cluster
};

// What a thread finishes: single elements, units of four (every row of y, pre
// and the addend starts on one), or its share of a sum over a cluster.
enum SimtForm { kElements, kUnits, kSplit };

template <typename T, int FORM>
__global__ void __launch_bounds__(kSimtThreads) gemm_simt_kernel(const __grid_constant__ SimtParams p) {
  constexpr bool VEC = FORM != kElements;
  __shared__ __align__(16) float sp[TK][TP], sq[TK][TP];
  __shared__ __align__(16) float part[FORM == kSplit ? TS : 1][TP];
  const GemmProblem& g = p.g;
  const int64_t tiles_j = p.tiles_j, per = p.tiles_i * tiles_j, blk = FORM == kSplit ? blockIdx.x / p.split : blockIdx.x;
  const int rank = FORM == kSplit ? (int)cluster_rank() : 0;
  const int64_t kb = rank * p.k_per, ke = FORM == kSplit && kb + p.k_per < g.K ? kb + p.k_per : g.K;
  const int64_t b = blk / per, t = blk - b * per;
  const int64_t i0 = (t / tiles_j) * TS, j0 = (t % tiles_j) * TS;
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
  SliceLoader<T> lp(g.P, b, i0, g.I, kb, ke), lq(g.Q, b, j0, g.J, kb, ke);
  float acc[8][4] = {}, vp[kLoads], vq[kLoads];
  lp.load(vp);
  lq.load(vq);
  for (int64_t k0 = kb; k0 < ke; k0 += TK) {
    lp.store(sp, vp);
    lq.store(sq, vq);
    __syncthreads();
    if (k0 + TK < ke) {
      lp.load(vp);
      lq.load(vq);
    }
    const int n = ke - k0 < TK ? (int)(ke - k0) : TK;
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
  if constexpr (FORM == kSplit) {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      *reinterpret_cast<float4*>(&part[ti * 8 + r][tj * 4]) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
    __syncwarp();
    cluster_sync();
    const int share = TS / p.split;
    for (int u = threadIdx.x; u < share * (TS / 4); u += kSimtThreads) {
      const int r = rank * share + u / (TS / 4), c = u % (TS / 4) * 4;
      if (i0 + r >= g.I || j0 + c >= g.J) continue;
      const uint32_t at = smem_u32(&part[r][c]);
      float s[4] = {};
      for (int q = 0; q < p.split; q += 2) {
        float v[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[h][0]), "=f"(v[h][1]), "=f"(v[h][2]), "=f"(v[h][3])
                       : "r"(map_rank(at, q + h))
                       : "memory");
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[0][e], s[e] += v[1][e];
      }
      for (int e = 0; e < 4 && j0 + c + e < g.J; ++e) epilogue_store<T>(g.e, b, i0 + r, j0 + c + e, s[e]);
    }
    __syncwarp();
    cluster_sync();  // a CTA's sums stay until they have been read
    return;
  }
  const int64_t i = i0 + ti * 8, j = j0 + (VEC ? tj * 4 : tj);
  constexpr int JS = VEC ? 1 : 16;  // columns between a thread's four
  const GemmEpilogue& e = g.e;
  const bool alone = !e.bias && !e.pre.p && !e.res.p && e.act == B2C_ACT_NONE;
  const int rows = g.I - i < 8 ? (int)(g.I - i) : 8;
  if (VEC && j + 4 <= g.J) {
    T* y = static_cast<T*>(e.y.p) + b * e.y.bs + i * e.y.is + j;
    Four<T> u;
    if (alone) {
#pragma unroll
      for (int r = 0; r < 8; ++r, y += e.y.is) {
#pragma unroll
        for (int c = 0; c < 4; ++c) u.v[c] = from_f32<T>(e.alpha * acc[r][c]);
        if (r < rows) *reinterpret_cast<Four<T>*>(y) = u;
      }
      return;
    }
    T* pre = static_cast<T*>(e.pre.p) + b * e.pre.bs + i * e.pre.is + j;
    const T* res = static_cast<const T*>(e.res.p) + b * e.res.bs + i * e.res.is + j;
    float bias[4] = {};
    if (e.bias && !e.bias_on_i)
#pragma unroll
      for (int c = 0; c < 4; ++c) bias[c] = to_f32(static_cast<const T*>(e.bias)[j + c]);
    // all addends are asked for before anything is stored
    Four<T> x[8];
    if (e.res.p)
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < rows) x[r] = *reinterpret_cast<const Four<T>*>(res + r * e.res.is);
#pragma unroll
    for (int r = 0; r < 8; ++r, y += e.y.is, pre += e.pre.is) {
      if (r >= rows) break;
      if (e.bias && e.bias_on_i) bias[0] = bias[1] = bias[2] = bias[3] = to_f32(static_cast<const T*>(e.bias)[i + r]);
      float v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = fmaf(e.alpha, acc[r][c], bias[c]);
      if (e.pre.p) {
#pragma unroll
        for (int c = 0; c < 4; ++c) u.v[c] = from_f32<T>(v[c]);
        *reinterpret_cast<Four<T>*>(pre) = u;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = act_f32<sizeof(T) == 2>(v[c], e.act);
      if (e.res.p) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = fmaf(e.beta, to_f32(x[r].v[c]), v[c]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) u.v[c] = from_f32<T>(v[c]);
      *reinterpret_cast<Four<T>*>(y) = u;
    }
    return;
  }
  if (!VEC && alone && e.y.js == 1) {
    // a product alone: nothing but the stores (350 MB of rows of 10755 float32, k = 3: 115 us, 254 by the loop below)
    T* y = static_cast<T*>(e.y.p) + b * e.y.bs + i * e.y.is + j;
#pragma unroll
    for (int r = 0; r < 8; ++r, y += e.y.is)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (i + r < g.I && j + c * JS < g.J) y[c * JS] = from_f32<T>(e.alpha * acc[r][c]);
    return;
  }
  // a row's addends are asked for before the row above is stored
  const int cols = j >= g.J ? 0 : (int)((g.J - j + JS - 1) / JS < 4 ? (g.J - j + JS - 1) / JS : 4);
  if (cols == 0) return;
  const T* res = static_cast<const T*>(e.res.p) + b * e.res.bs + i * e.res.is + j * e.res.js;
  T* y = static_cast<T*>(e.y.p) + b * e.y.bs + i * e.y.is + j * e.y.js;
  T* pre = static_cast<T*>(e.pre.p) + b * e.pre.bs + i * e.pre.is + j * e.pre.js;
  T x[4] = {};
  float on_j[4] = {};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (e.res.p && rows > 0) x[c] = res[(c < cols ? c : 0) * JS * e.res.js];
    if (e.bias && !e.bias_on_i) on_j[c] = to_f32(static_cast<const T*>(e.bias)[j + (c < cols ? c : 0) * JS]);
  }
#pragma unroll 1
  for (int r = 0; r < rows; ++r) {
    T next[4] = {};
    res += e.res.is;
    if (e.res.p && r + 1 < rows)
#pragma unroll
      for (int c = 0; c < 4; ++c) next[c] = res[(c < cols ? c : 0) * JS * e.res.js];
    const float on_i = e.bias && e.bias_on_i ? to_f32(static_cast<const T*>(e.bias)[i + r]) : 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float v = e.alpha * acc[0][c];
      if (e.bias) v += e.bias_on_i ? on_i : on_j[c];
      if (e.pre.p && c < cols) pre[c * JS * e.pre.js] = from_f32<T>(v);
      v = act_f32<sizeof(T) == 2>(v, e.act);
      if (e.res.p) v = fmaf(e.beta, to_f32(x[c]), v);
      if (c < cols) y[c * JS * e.y.js] = from_f32<T>(v);
    }
    y += e.y.is, pre += e.pre.is;
    // the sums move up instead of the index, for a loop that stays short
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int m = 1; m < 8; ++m) acc[m - 1][c] = acc[m][c];
      x[c] = next[c];
    }
  }
}

template <typename T>
cudaError_t launch_t(const GemmProblem& g, int sms, cudaStream_t s) {
  SimtParams p{};
  p.g = g;
  p.tiles_i = (g.I + TS - 1) / TS, p.tiles_j = (g.J + TS - 1) / TS;
  const int64_t tiles = g.batch * p.tiles_i * p.tiles_j;
  p.split = simt_split(g, sms);
  p.k_per = (g.K + p.split - 1) / p.split;
  if (tiles * p.split > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const unsigned grid = (unsigned)(tiles * p.split);
  if (p.split > 1) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kSimtThreads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, gemm_simt_kernel<T, kSplit>, p);
  }
  auto fours = [](const GemmView& v) {
    return !v.p || (v.js == 1 && reinterpret_cast<uintptr_t>(v.p) % (4 * sizeof(T)) == 0 && v.is % 4 == 0 && v.bs % 4 == 0);
  };
  if (fours(g.e.y) && fours(g.e.pre) && fours(g.e.res)) gemm_simt_kernel<T, kUnits><<<grid, kSimtThreads, 0, s>>>(p);
  else gemm_simt_kernel<T, kElements><<<grid, kSimtThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

// CTAs that share a tile's k: up to 8, of at least 64 each, while they all fit at once.
int simt_split(const GemmProblem& g, int sms) {
  const int64_t tiles = g.batch * ((g.I + TS - 1) / TS) * ((g.J + TS - 1) / TS);
  int split = 1;
  while (split < 8 && tiles * split <= sms && g.K >= split * 128) split *= 2;
  return split;
}

cudaError_t launch_gemm_simt(const GemmProblem& g, cudaStream_t s) {
  int sms = 0;
  const cudaError_t e = device_sms(&sms);
  if (e != cudaSuccess) return e;
  switch (g.dtype) {
    case B2C_F32: return launch_t<float>(g, sms, s);
    case B2C_BF16: return launch_t<__nv_bfloat16>(g, sms, s);
    default: return launch_t<__half>(g, sms, s);
  }
}

}  // namespace b2c
