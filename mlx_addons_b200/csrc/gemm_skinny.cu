// Products with at most 8 columns of Q a pass (the weights of a layer against
// one or a few tokens): bound by one pass over P at HBM speed, so the sums run
// on the FP32 units and nothing is staged for the tensor cores. Any strides,
// alignment and type.
//
// P with unit stride along k: a warp takes 4 rows, its lanes run along k (16
// bytes a lane where alignment allows), so Q's values, read through L1, serve
// 4 rows. P with unit stride along the rows: a lane takes 8 rows, the 8 warps
// of a CTA take every 8th k (with 64 rows a CTA instead of 256, a quarter of a
// warp does), and Q's slice is staged in shared memory as float32 for broadcasts.
//
// Where there are too few rows to fill the GPU, k is split over the warps of
// a CTA and over a cluster of up to 8 CTAs; the partial sums are joined in
// order through (distributed) shared memory, in the same launch and without
// scratch.
#include "b2c_kernels.cuh"
#include "gemm.cuh"

namespace b2c {

namespace {

constexpr int kWarps = 8;
constexpr int kSkinnyThreads = kWarps * 32;
constexpr int kRows = 4;        // rows of a warp, unit stride along k
constexpr int kSlice = 256;     // k staged at a time there

struct SkinnyParams {
  GemmProblem g;
  int64_t row_blocks;  // CTAs (times cluster) along I
  int64_t k_per;       // k of one CTA of the cluster, a multiple of 8
  int split;           // CTAs of a cluster
  int warps, warp_split;  // warps of a CTA, and those of them that share rows (unit stride along k)
  int j0;              // first column of this pass
};

__device__ __forceinline__ uint32_t ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_float(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// How P's rows are read: any way, in 16-byte units, or units that stay out of L1,
// which then holds Q (533 MB of P with 9 columns: 178 us a pass of 8 against 245;
// where L2 holds P, 64 MB, units that go through L1 are faster, 34 us against 41).
enum SkinnyLoads { kAny, kUnits, kStream };
template <bool STREAM>
__device__ __forceinline__ uint4 load16(const void* p) {
  if constexpr (STREAM) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
  }
  return __ldg(reinterpret_cast<const uint4*>(p));
}

// Eight k of one row: neighbours (VEC, whole 16-byte units) or every 32nd.
template <typename T, bool VEC, bool STREAM>
__device__ __forceinline__ void load_k8(const T* row, int64_t ks, int64_t k, int64_t end, bool in, float (&v)[8]) {
  if constexpr (VEC) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < 8 / PER; ++q) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (in && k + q * PER < end) w = load16<STREAM>(row + k + q * PER);
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int c = 0; c < PER; ++c) v[q * PER + c] = to_f32(e[c]);
    }
  } else {
    // every load is issued, past the end that of the first k again: none waits for a branch
    const T* at = row + k * ks;
    const int left = (int)min((end - k + 31) / 32, (int64_t)8);
    T t[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) t[c] = at[c < left ? c * 32 * ks : 0];
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = in && c < left ? to_f32(t[c]) : 0.f;
  }
}

template <typename T, int JT, int LOADS>
__global__ void __launch_bounds__(kSkinnyThreads) skinny_k_kernel(const __grid_constant__ SkinnyParams p) {
  constexpr bool VEC = LOADS != kAny;
  __shared__ float part[kWarps * kRows * JT];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = p.split > 1 ? ctarank() : 0;
  const int64_t blk = blockIdx.x / p.split, b = blk / p.row_blocks;
  const int ws = p.warp_split, mine = warp / ws, sub = warp % ws;
  const int rows = kRows * (p.warps / ws);
  const int64_t i0 = (blk - b * p.row_blocks) * rows + mine * kRows;
  const int64_t k0 = rank * p.k_per, k1 = min(k0 + p.k_per, p.g.K);
  const T* P = static_cast<const T*>(p.g.P.p) + b * p.g.P.bs;
  const T* Q = static_cast<const T*>(p.g.Q.p) + b * p.g.Q.bs + p.j0 * p.g.Q.rs;
  const int nj = (int)min((int64_t)JT, p.g.J - p.j0);
  float acc[kRows][JT] = {};
  constexpr int kUnroll = JT <= 2 ? 4 : 2;
#pragma unroll kUnroll
  for (int64_t k = k0 + sub * 256 + (VEC ? lane * 8 : lane); k < k1; k += ws * 256) {
    float w[kRows][8];
#pragma unroll
    for (int r = 0; r < kRows; ++r) load_k8<T, VEC, LOADS == kStream>(P + (i0 + r < p.g.I ? i0 + r : 0) * p.g.P.rs, p.g.P.ks, k, k1, i0 + r < p.g.I, w[r]);
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      float x[8];
      load_k8<T, VEC, false>(Q + (j < nj ? j : 0) * p.g.Q.rs, p.g.Q.ks, k, k1, j < nj, x);
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[r][j] = fmaf(w[r][c], x[c], acc[r][j]);
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      const float t = warp_sum(acc[r][j]);
      if (lane == 0) part[(warp * kRows + r) * JT + j] = t;
    }
  if (p.split > 1) cluster_barrier();
  else __syncthreads();
  if (rank == 0) {
    for (int t = threadIdx.x; t < rows * JT; t += blockDim.x) {
      const int r = t / JT, j = t % JT;
      const int64_t i = (blk - b * p.row_blocks) * rows + r;
      if (i < p.g.I && j < nj) {
        float s = 0.f;
        for (int q = 0; q < p.split; ++q)
          for (int u = 0; u < ws; ++u) {
            const float* at = &part[((r / kRows * ws + u) * kRows + r % kRows) * JT + j];
            s += q == 0 ? *at : peer_float(at, q);
          }
        epilogue_store<T>(p.g.e, b, i, p.j0 + j, s);
      }
    }
  }
  if (p.split > 1) cluster_barrier();  // peers' shared memory stays until it has been read
}

// ROWS: rows of a CTA, 8 a lane.
template <typename T, int JT, bool VEC, int ROWS>
__global__ void __launch_bounds__(kSkinnyThreads) skinny_row_kernel(const __grid_constant__ SkinnyParams p) {
  __shared__ __align__(16) float xs[kSlice][JT];
  constexpr int LR = ROWS / 8, KG = 32 / LR;  // lanes along the rows, k of a warp at a time
  __shared__ float red[kWarps * KG][ROWS];
  __shared__ float part[JT][ROWS];
  const int lane = threadIdx.x % LR, kg = threadIdx.x / LR;  // lane of a row group, row group
  const uint32_t rank = p.split > 1 ? ctarank() : 0;
  const int64_t blk = blockIdx.x / p.split, b = blk / p.row_blocks, i0 = (blk - b * p.row_blocks) * ROWS;
  const int64_t k0 = rank * p.k_per, k1 = min(k0 + p.k_per, p.g.K);
  const int64_t il = i0 + (VEC ? lane * 8 : lane);  // this lane's rows: 8 neighbours, or every LR-th
  const T* P = static_cast<const T*>(p.g.P.p) + b * p.g.P.bs;
  const T* Q = static_cast<const T*>(p.g.Q.p) + b * p.g.Q.bs + p.j0 * p.g.Q.rs;
  const int nj = (int)min((int64_t)JT, p.g.J - p.j0);
  float acc[8][JT] = {};
  for (int64_t ks = k0; ks < k1; ks += kSlice) {
    const int n = (int)min((int64_t)kSlice, k1 - ks);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < JT; ++j)
      for (int k = threadIdx.x; k < kSlice; k += kSkinnyThreads)
        xs[k][j] = k < n && j < nj ? to_f32(Q[j * p.g.Q.rs + (ks + k) * p.g.Q.ks]) : 0.f;
    __syncthreads();
#pragma unroll 4
    for (int k = kg; k < n; k += kWarps * KG) {
      const T* at = P + (ks + k) * p.g.P.ks;
      float w[8];
      if constexpr (VEC) {
        constexpr int PER = 16 / sizeof(T);
#pragma unroll
        for (int q = 0; q < 8 / PER; ++q) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (il + q * PER < p.g.I) v = __ldg(reinterpret_cast<const uint4*>(at + il + q * PER));
          const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int c = 0; c < PER; ++c) w[q * PER + c] = to_f32(e[c]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c) w[c] = il + LR * c < p.g.I ? to_f32(at[(il + LR * c) * p.g.P.rs]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < JT; ++j) {
        const float x = xs[k][j];
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c][j] = fmaf(w[c], x, acc[c][j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < JT; ++j) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 8; ++c) red[kg][VEC ? lane * 8 + c : lane + LR * c] = acc[c][j];
    __syncthreads();
    if (threadIdx.x < ROWS) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps * KG; ++w) t += red[w][threadIdx.x];
      part[j][threadIdx.x] = t;
    }
  }
  if (p.split > 1) cluster_barrier();
  else __syncthreads();
  // each CTA of the cluster finishes its share of the rows
  const int share = ROWS / p.split;
  for (int t = threadIdx.x; t < share * JT; t += kSkinnyThreads) {
    const int j = t / share, r = rank * share + t % share;
    if (i0 + r < p.g.I && j < nj) {
      float s = 0.f;
      for (int q = 0; q < p.split; ++q) s += p.split > 1 ? peer_float(&part[j][r], q) : part[j][r];
      epilogue_store<T>(p.g.e, b, i0 + r, p.j0 + j, s);
    }
  }
  if (p.split > 1) cluster_barrier();
}

template <typename Kern>
cudaError_t launch_cluster(Kern kern, const SkinnyParams& p, int64_t ctas, int warps, cudaStream_t s) {
  if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(warps * 32);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)p.split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T, int JT>
cudaError_t launch_j(SkinnyParams p, int sms, cudaStream_t s) {
  constexpr int64_t PER = 16 / sizeof(T);
  const GemmProblem& g = p.g;
  auto on16 = [](const GemmOperand& o, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(o.p) & 15) == 0 && o.bs % PER == 0 && stride % PER == 0;
  };
  const bool rows_inner = g.P.rs < g.P.ks && g.I > 1;
  p.split = 1;
  if (!rows_inner) {
    // A dozen warps an SM, in CTAs as small as that allows: rows are shared by more warps until there are that many,
    // then k by a cluster.
    const int64_t groups = g.batch * ((g.I + kRows - 1) / kRows), want = 12 * (int64_t)sms;
    p.warp_split = 1;
    while (p.warp_split < kWarps && groups * p.warp_split < want && g.K > p.warp_split * 256) p.warp_split *= 2;
    while (p.split < 8 && groups * p.warp_split * p.split < want && g.K > p.split * p.warp_split * 256) p.split *= 2;
    p.warps = p.warp_split > 2 ? p.warp_split : 2;
    const int rows = kRows * (p.warps / p.warp_split);
    p.k_per = ((g.K + p.split - 1) / p.split + 255) / 256 * 256;
    p.row_blocks = (g.I + rows - 1) / rows;
    const int64_t ctas = g.batch * p.row_blocks * p.split;
    const bool vec = g.P.ks == 1 && g.Q.ks == 1 && on16(g.P, g.P.rs) && on16(g.Q, g.Q.rs) && g.K % PER == 0;
    if constexpr (sizeof(T) == 4 && JT > 1)  // 16-bit products of this form are small
      if (vec && g.batch * g.I * g.K * 4 > (96 << 20))
        return launch_cluster(skinny_k_kernel<T, JT, kStream>, p, ctas, p.warps, s);
    return vec ? launch_cluster(skinny_k_kernel<T, JT, kUnits>, p, ctas, p.warps, s)
               : launch_cluster(skinny_k_kernel<T, JT, kAny>, p, ctas, p.warps, s);
  }
  // 256 rows a CTA, or 64 where that leaves SMs idle
  const int rows = g.batch * ((g.I + 255) / 256) * 8 < sms ? 64 : 256;
  p.row_blocks = (g.I + rows - 1) / rows;
  const int64_t blocks = g.batch * p.row_blocks;
  while (p.split < 8 && blocks * p.split < 2 * (int64_t)sms && g.K > p.split * 64) p.split *= 2;
  p.k_per = ((g.K + p.split - 1) / p.split + 7) / 8 * 8;
  const bool vec = g.P.rs == 1 && on16(g.P, g.P.ks) && g.I % PER == 0;
  const int64_t ctas = blocks * p.split;
  if (rows == 64)
    return vec ? launch_cluster(skinny_row_kernel<T, JT, true, 64>, p, ctas, kWarps, s)
               : launch_cluster(skinny_row_kernel<T, JT, false, 64>, p, ctas, kWarps, s);
  return vec ? launch_cluster(skinny_row_kernel<T, JT, true, 256>, p, ctas, kWarps, s)
             : launch_cluster(skinny_row_kernel<T, JT, false, 256>, p, ctas, kWarps, s);
}

template <typename T>
cudaError_t launch_t(const GemmProblem& g, int sms, cudaStream_t s) {
  SkinnyParams p{};
  p.g = g;
  for (p.j0 = 0; p.j0 < g.J;) {
    const int64_t left = g.J - p.j0;
    const int jt = left > 4 ? 8 : left > 2 ? 4 : left == 2 ? 2 : 1;
    const cudaError_t e = jt == 8   ? launch_j<T, 8>(p, sms, s)
                          : jt == 4 ? launch_j<T, 4>(p, sms, s)
                          : jt == 2 ? launch_j<T, 2>(p, sms, s)
                                    : launch_j<T, 1>(p, sms, s);
    if (e != cudaSuccess) return e;
    p.j0 += jt;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_gemm_skinny(const GemmProblem& g, int sms, cudaStream_t s) {
  switch (g.dtype) {
    case B2C_F32: return launch_t<float>(g, sms, s);
    case B2C_BF16: return launch_t<__nv_bfloat16>(g, sms, s);
    default: return launch_t<__half>(g, sms, s);
  }
}

}  // namespace b2c
