// extern "C" boundary of the products with an epilogue and of the
// Newton-Schulz orthogonalisation (declared in include/b2c.h).
#include <cmath>
#include <cstdio>
#include <initializer_list>

#include "b2c_kernels.cuh"
#include "gemm_tc.cuh"

namespace {

using namespace b2c;

constexpr int64_t kMaxDim = (int64_t)1 << 30;
constexpr int64_t kMaxPolarDim = (int64_t)1 << 20;
constexpr double kSkinny16 = 2097152.0;  // largest 16-bit P of the FP32-unit form
constexpr int kMaxSteps = 64;
constexpr double kMaxSigma = 3.5;

int err(int code, const char* name, const char* what) {
  char buf[400];
  snprintf(buf, sizeof(buf), "%s: %s", name, what);
  return set_error(code, buf);
}

int cuda_err(cudaError_t e, const char* name) {
  if (e == cudaErrorInvalidConfiguration) return err(B2C_ERR_UNSUPPORTED, name, "more tiles than one launch holds");
  char buf[256];
  snprintf(buf, sizeof(buf), "%s (%s)", cudaGetErrorName(e), cudaGetErrorString(e));
  return err(B2C_ERR_CUDA, name, buf);
}

bool dtype_ok(int dtype) { return dtype >= B2C_F32 && dtype <= B2C_F16; }
bool on(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// Whether all of these addresses are multiples of an element's size.
bool aligned(int dtype, std::initializer_list<const void*> all) {
  for (const void* p : all)
    if (!on(p, dtype == B2C_F32 ? 4 : 2)) return false;
  return true;
}
bool strides_ok(const b2c_matrix& m) { return m.batch_stride >= 0 && m.row_stride >= 0 && m.col_stride >= 0; }

GemmProblem problem(int dtype, const b2c_matrix* A, const b2c_matrix* B, int64_t batch, int64_t M, int64_t K, int64_t N) {
  GemmProblem g{};
  g.dtype = dtype;
  g.batch = batch;
  g.I = M;
  g.J = N;
  g.K = K;
  g.P = GemmOperand{A->ptr, A->batch_stride, A->row_stride, A->col_stride};
  g.Q = GemmOperand{B->ptr, B->batch_stride, B->col_stride, B->row_stride};
  return g;
}

// Which kernel takes a product, and what has to be copied for it.
struct GemmChoice {
  GemmProblem g;
  enum { kSimt, kSkinny, kTc } tier;
  PackPlan pack_p, pack_q;
  size_t ws() const { return tier == kTc ? (size_t)(pack_p.bytes + pack_q.bytes) : 0; }
};

// Time of a product on the FP32 units, us: a launch, and 0.05 a k of a CTA that has an SM
// to itself, 0.03 more for each that it shares it with.
double simt_us(const GemmProblem& g, int sms) {
  const int split = simt_split(g, sms);
  const double ctas = (double)g.batch * (double)((g.I + 63) / 64) * (double)((g.J + 63) / 64) * split;
  return 6.0 + (double)((g.K + split - 1) / split) * (0.02 + 0.03 * ceil(ctas / sms));
}

GemmChoice choose(const GemmProblem& in) {
  constexpr int sms = 148;  // of a B200: the choice, and with it the workspace, depends on the sizes alone
  GemmChoice c{};
  c.g = in;
  const double macs = (double)in.I * (double)in.J * (double)in.K * (double)in.batch;
  const int64_t shorter = in.I < in.J ? in.I : in.J, longer = in.I < in.J ? in.J : in.I;
  const bool f32 = in.dtype == B2C_F32;
  // one to eight (float32: sixteen) columns: one pass over the other operand
  const bool thin = in.K > 0 && (f32 ? shorter <= 16 : shorter <= 8 && (double)longer * in.K * in.batch <= kSkinny16);
  // The tensor cores' set-up, and for float32 the pass that splits the operands, cost as much as this: float32 17 us at
  // the least, which the FP32 units need for about 200 k of a CTA (us on the FP32 units and on the tensor cores: 145 x 449 x 148
  // 13 and 19, 256 x 256 x 256 11 and 17, 512 x 512 x 512 19 and 19, 64 x 4096 x 64 32 and 25); 16-bit types 8 us.
  const bool shallow = f32 ? in.K < 40 || (in.K < 96 && macs <= 1e8) || macs <= 1e6 || simt_us(in, sms) <= 17
                           : in.K < 32 || macs <= 1048576.0;
  c.tier = thin ? GemmChoice::kSkinny : shallow ? GemmChoice::kSimt : GemmChoice::kTc;
  if (c.tier != GemmChoice::kSimt && in.I <= 64 && in.J > in.I) {  // the longer side takes the 128 rows of a tile
    GemmProblem& g = c.g;
    g.P = in.Q, g.Q = in.P;
    g.I = in.J, g.J = in.I;
    for (GemmView* v : {&g.e.y, &g.e.pre, &g.e.res}) {
      const int64_t t = v->is;
      v->is = v->js, v->js = t;
    }
    g.e.bias_on_i = !in.e.bias_on_i;
  }
  if (c.tier == GemmChoice::kTc) {
    c.pack_p = plan_pack(in.dtype, c.g.P, in.batch, c.g.I, in.K);
    c.pack_q = plan_pack(in.dtype, c.g.Q, in.batch, c.g.J, in.K);
  }
  return c;
}

cudaError_t launch_gemm(const GemmChoice& c, void* ws, cudaStream_t s) {
  const GemmProblem& g = c.g;
  cudaError_t e;
  if (c.tier == GemmChoice::kSimt) return launch_gemm_simt(g, s);
  if (c.tier == GemmChoice::kSkinny) {
    int sms = 0;
    return (e = device_sms(&sms)) == cudaSuccess ? launch_gemm_skinny(g, sms, s) : e;
  }
  TcProblem t{};
  char* w = static_cast<char*>(ws);
  if (!c.pack_p.needed) tc_direct(g.P, g.batch, g.I, g.K, &t.P);
  else if ((e = launch_pack(g.dtype, g.P, c.pack_p, w, &t.P, s)) != cudaSuccess) return e;
  if (!c.pack_q.needed) tc_direct(g.Q, g.batch, g.J, g.K, &t.Q);
  else if ((e = launch_pack(g.dtype, g.Q, c.pack_q, w + c.pack_p.bytes, &t.Q, s)) != cudaSuccess) return e;
  t.kind = g.dtype == B2C_F32 ? kThirds : kOne;
  t.f16 = g.dtype == B2C_F16;
  t.batch = g.batch;
  t.I = g.I, t.J = g.J, t.K = g.K;
  t.e = g.e;
  t.out = t.res = g.dtype;
  return launch_gemm_tc(t, s);
}

}  // namespace

extern "C" {

size_t b2c_gemm_workspace_size(int dtype, const b2c_matrix* A, const b2c_matrix* B, int64_t batch, int64_t M,
                               int64_t K, int64_t N) {
  if (!dtype_ok(dtype) || !A || !B || !strides_ok(*A) || !strides_ok(*B) || batch <= 0 || M <= 0 || K <= 0 || N <= 0 ||
      M > kMaxDim || K > kMaxDim || N > kMaxDim)
    return 0;
  // an operand without an address may get one that TMA cannot read, and then needs a copy
  GemmProblem g = problem(dtype, A, B, batch, M, K, N);
  const void* odd = reinterpret_cast<const void*>((uintptr_t)1);
  if (!g.P.p) g.P.p = odd;
  if (!g.Q.p) g.Q.p = odd;
  return choose(g).ws();
}

int b2c_gemm(int dtype, const b2c_matrix* A, const b2c_matrix* B, const void* bias, const b2c_matrix* R, void* Y,
             void* pre, int64_t batch, int64_t M, int64_t K, int64_t N, float alpha, float beta, int activation,
             void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "b2c_gemm";
  if (!dtype_ok(dtype)) return err(B2C_ERR_INVALID_ARGUMENT, name, "unknown dtype");
  if (activation < B2C_ACT_NONE || activation > B2C_ACT_SILU)
    return err(B2C_ERR_INVALID_ARGUMENT, name, "unknown activation");
  if (batch < 0 || M < 0 || K < 0 || N < 0) return err(B2C_ERR_INVALID_ARGUMENT, name, "sizes must be >= 0");
  if (M > kMaxDim || K > kMaxDim || N > kMaxDim) return err(B2C_ERR_UNSUPPORTED, name, "M, K and N are limited to 2^30");
  if (!A || !B) return err(B2C_ERR_INVALID_ARGUMENT, name, "A and B must be non-NULL");
  if (!strides_ok(*A) || !strides_ok(*B) || (R && !strides_ok(*R)))
    return err(B2C_ERR_INVALID_ARGUMENT, name, "strides must be >= 0");
  if (batch == 0 || M == 0 || N == 0) return set_error(B2C_OK, "");
  if (!Y || (K > 0 && (!A->ptr || !B->ptr)) || (R && !R->ptr))
    return err(B2C_ERR_INVALID_ARGUMENT, name, "A, B, R and Y must point to data");
  if (!aligned(dtype, {A->ptr, B->ptr, bias, R ? R->ptr : nullptr, Y, pre}))
    return err(B2C_ERR_INVALID_ARGUMENT, name, "an address is not aligned to its elements");
  GemmProblem g = problem(dtype, A, B, batch, M, K, N);
  g.e.y = GemmView{Y, M * N, N, 1};
  g.e.pre = GemmView{pre, M * N, N, 1};
  if (R) g.e.res = GemmView{const_cast<void*>(R->ptr), R->batch_stride, R->row_stride, R->col_stride};
  g.e.bias = bias;
  g.e.alpha = alpha;
  g.e.beta = beta;
  g.e.act = activation;
  const GemmChoice c = choose(g);
  if (c.ws() && (!workspace || workspace_bytes < c.ws() || !on(workspace, 16)))
    return err(B2C_ERR_WORKSPACE, name, "workspace missing, too small or not on 16 bytes");
  const cudaError_t e = launch_gemm(c, workspace, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? set_error(B2C_OK, "") : cuda_err(e, name);
}

size_t b2c_gemm_dact_workspace_size(int64_t batch, int64_t M, int64_t N) {
  if (batch <= 0 || M <= 0 || N <= 0 || M > kMaxDim || N > kMaxDim) return 0;
  return dact_ws_floats(batch, M, N) * sizeof(float);
}

int b2c_gemm_dact(int dtype, const b2c_matrix* dY, const b2c_matrix* pre, int activation, float beta, void* dP,
                  void* dbias, void* dR, int64_t batch, int64_t M, int64_t N, void* workspace,
                  size_t workspace_bytes, void* stream) {
  const char* name = "b2c_gemm_dact";
  if (!dtype_ok(dtype)) return err(B2C_ERR_INVALID_ARGUMENT, name, "unknown dtype");
  if (activation < B2C_ACT_NONE || activation > B2C_ACT_SILU)
    return err(B2C_ERR_INVALID_ARGUMENT, name, "unknown activation");
  if (batch < 0 || M < 0 || N < 0) return err(B2C_ERR_INVALID_ARGUMENT, name, "sizes must be >= 0");
  if (M > kMaxDim || N > kMaxDim) return err(B2C_ERR_UNSUPPORTED, name, "M and N are limited to 2^30");
  if (!dY || !strides_ok(*dY) || (pre && !strides_ok(*pre)))
    return err(B2C_ERR_INVALID_ARGUMENT, name, "dY must be non-NULL and strides >= 0");
  if (activation != B2C_ACT_NONE && !pre)
    return err(B2C_ERR_INVALID_ARGUMENT, name, "an activation's gradient needs pre");
  if (N == 0 || (!dP && !dbias && !dR)) return set_error(B2C_OK, "");
  const bool empty = batch == 0 || M == 0;
  if (empty && !dbias) return set_error(B2C_OK, "");
  if (!empty && (!dY->ptr || (activation != B2C_ACT_NONE && !pre->ptr)))
    return err(B2C_ERR_INVALID_ARGUMENT, name, "dY and pre must point to data");
  if (!aligned(dtype, {dY->ptr, activation != B2C_ACT_NONE ? pre->ptr : nullptr, dP, dbias, dR}))
    return err(B2C_ERR_INVALID_ARGUMENT, name, "an address is not aligned to its elements");
  DactParams p{};
  p.dtype = dtype;
  p.act = activation;
  p.dY = dY->ptr;
  p.dy_bs = dY->batch_stride, p.dy_rs = dY->row_stride, p.dy_cs = dY->col_stride;
  if (activation != B2C_ACT_NONE) {
    p.pre = pre->ptr;
    p.pre_bs = pre->batch_stride, p.pre_rs = pre->row_stride, p.pre_cs = pre->col_stride;
  }
  p.dP = dP;
  p.dbias = dbias;
  p.dR = dR;
  p.beta = beta;
  p.batch = batch;
  p.M = M;
  p.N = N;
  p.ws = static_cast<float*>(workspace);
  const size_t need = dbias ? dact_ws_floats(batch, M, N) * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need || !on(workspace, 16)))
    return err(B2C_ERR_WORKSPACE, name, "workspace missing, too small or not on 16 bytes");
  const cudaError_t e = launch_gemm_dact(p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? set_error(B2C_OK, "") : cuda_err(e, name);
}

static PolarParams polar_params(int dtype, const b2c_matrix* G, int64_t batch, int64_t m, int64_t n) {
  PolarParams p{};
  p.dtype = dtype;
  p.G = G->ptr;
  p.bs = G->batch_stride, p.rs = G->row_stride, p.cs = G->col_stride;
  p.batch = batch;
  p.m = m;
  p.n = n;
  return p;
}

size_t b2c_orthogonalize_workspace_size(int dtype, const b2c_matrix* G, int64_t batch, int64_t m, int64_t n) {
  if (!dtype_ok(dtype) || !G || batch <= 0 || m <= 0 || n <= 0 || m > kMaxPolarDim || n > kMaxPolarDim) return 0;
  return polar_ws_bytes(polar_params(dtype, G, batch, m, n));
}

int b2c_orthogonalize(int dtype, const b2c_matrix* G, void* out, int64_t batch, int64_t m, int64_t n,
                      const double* coefficients, int steps, double eps, void* workspace, size_t workspace_bytes,
                      void* stream) {
  const char* name = "b2c_orthogonalize";
  if (!dtype_ok(dtype)) return err(B2C_ERR_INVALID_ARGUMENT, name, "unknown dtype");
  if (batch < 0 || m < 0 || n < 0) return err(B2C_ERR_INVALID_ARGUMENT, name, "sizes must be >= 0");
  if (m > kMaxPolarDim || n > kMaxPolarDim) return err(B2C_ERR_UNSUPPORTED, name, "m and n are limited to 2^20");
  if (steps < 1 || steps > kMaxSteps) return err(B2C_ERR_INVALID_ARGUMENT, name, "steps must be 1 to 64");
  if (!coefficients) return err(B2C_ERR_INVALID_ARGUMENT, name, "coefficients must be non-NULL");
  if (!(eps >= 0.0) || std::isinf(eps)) return err(B2C_ERR_INVALID_ARGUMENT, name, "eps must be finite and >= 0");
  if (!G || !strides_ok(*G)) return err(B2C_ERR_INVALID_ARGUMENT, name, "G must be non-NULL and its strides >= 0");
  float coef[3 * kMaxSteps];
  double hi = 1.0;
  for (int t = 0; t < steps; ++t) {
    const double *c = coefficients + 3 * t;
    for (int i = 0; i < 3; ++i) {
      coef[3 * t + i] = (float)c[i];
      if (!std::isfinite(coef[3 * t + i])) return err(B2C_ERR_INVALID_ARGUMENT, name, "coefficients must be finite float32 values");
    }
    hi = polar_poly_bound(c[0], c[1], c[2], hi);
    if (!(hi <= kMaxSigma))
      return err(B2C_ERR_INVALID_ARGUMENT, name, "the coefficients let singular values grow past 3.5");
  }
  if (batch == 0 || m == 0 || n == 0) return set_error(B2C_OK, "");
  if (!G->ptr || !out) return err(B2C_ERR_INVALID_ARGUMENT, name, "G and out must point to data");
  if (!aligned(dtype, {G->ptr, out})) return err(B2C_ERR_INVALID_ARGUMENT, name, "an address is not aligned to its elements");
  PolarParams p = polar_params(dtype, G, batch, m, n);
  p.out = out;
  p.coef = coef;
  p.steps = steps;
  p.eps = eps;
  p.ws = workspace;
  const size_t need = polar_ws_bytes(p);
  if (need && (!workspace || workspace_bytes < need || !on(workspace, 16)))
    return err(B2C_ERR_WORKSPACE, name, "workspace missing, too small or not on 16 bytes");
  const cudaError_t e = launch_polar(p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? set_error(B2C_OK, "") : cuda_err(e, name);
}

}  // extern "C"
