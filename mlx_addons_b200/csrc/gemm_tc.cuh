// Tensor-core products: the launcher's interface (gemm_tc.cu), used by
// b2c_gemm and by the orthogonalisation (polar.cu).
#pragma once

#include "gemm.cuh"

namespace b2c {

// How a 16-bit array stands for the values of an operand, addend or output.
//   kOne      one array of bf16 or f16
//   kHalves   two f16 planes, value = hi + lo (22 bits and the sign of lo)
//   kThirds   three bf16 planes, value = hi + 2^-8 mid + 2^-16 lo (all 24 bits)
enum TcKind { kOne = 0, kHalves = 1, kThirds = 2 };

// One operand, as the tensor cores read it: 16-bit, one of its axes with unit
// stride, everything else in multiples of 16 bytes.
struct TcOperand {
  const void* p;
  int64_t batch_stride;  // elements; ignored where bcast
  int64_t pitch;         // stride of the other axis, elements
  int64_t plane_stride;  // elements; kHalves / kThirds
  int rows_inner;        // 1: the row axis has unit stride, 0: the k axis
  int bcast;             // one matrix for the whole batch
};

// The epilogues of an orthogonalisation step (polar.cu). S and P are stored
// without their diagonals, which are kept as float32 vectors: near the end of
// the iteration the diagonal is most of them, and so most of what f16 would
// round away.
//   kPolarS     y = alpha r^2 D off the diagonal, d_out = k r^2 D on it
//   kPolarP     y = alpha D + (beta + k (d_i + d_j)) res off it,
//               d_out = k2 D + k3 d^2 + k4 d on it
//   kPolarXi/j  y = r (alpha D + beta (k + d_i or d_j) res)
enum TcPolarMode { kPolarNone = 0, kPolarS, kPolarP, kPolarXi, kPolarXj };
struct TcPolar {
  int mode;
  const float* r;     // one factor a matrix, or null (1)
  const float* d_in;  // (batch, side)
  float* d_out;       // (batch, side)
  int64_t side;
  float k, k2, k3, k4;
};

struct TcProblem {
  TcOperand P, Q;
  int kind;              // TcKind of both operands
  int f16;               // operands f16 (1) or bf16 (0)
  int64_t batch, I, J, K;
  GemmEpilogue e;
  int out;               // B2C_F32 / B2C_BF16 / B2C_F16 with e.y, e.pre and e.bias of that type, or kOutHalves
  int res;               // the type of e.res, or kOutHalves
  int64_t y_plane, res_plane;  // plane strides, elements, where kOutHalves
  TcPolar polar;
  int chained;           // follows a kernel of the same chain: may be set up while that one ends
  int sym;               // D is symmetric (P and Q the same, or commuting symmetric): compute the lower tiles, mirror them
};
constexpr int kOutHalves = 3;

// Whether one batch of strided matrices can be read as it lies; rows / ks / bs
// are the strides of element (batch, row, k).
bool tc_direct(const GemmOperand& o, int64_t batch, int64_t rows, int64_t K, TcOperand* out);
cudaError_t launch_gemm_tc(const TcProblem& t, cudaStream_t s);

// Copies an operand to rows of a multiple of 8 elements: 16-bit as it is,
// float32 as three bf16 planes. gemm_pack.cu
struct PackPlan {
  int needed;
  int rows_inner;
  int64_t batch, outer, inner, pitch, plane, bytes;  // bytes: all planes
};
PackPlan plan_pack(int dtype, const GemmOperand& o, int64_t batch, int64_t rows, int64_t K);
cudaError_t launch_pack(int dtype, const GemmOperand& o, const PackPlan& plan, void* dst, TcOperand* out,
                        cudaStream_t s);

}  // namespace b2c
