// Mixed-precision linear-layer routines on device-resident data: argument checks, scratch
// layout and launches. No counterpart in the reference, whose tile operations are FP64 and
// FP32 BLAS (Library_scheduler/src/Subkernel.cpp:168,228).
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>

#include "exec.hpp"
#include "gemm_act.cuh"
#include "regions.hpp"
#include "runtime.hpp"

namespace paralia {
namespace {

bool is_trans(char t) { return t == 'T' || t == 't' || t == 'C' || t == 'c'; }
bool is_flag(char t) { return is_trans(t) || t == 'N' || t == 'n'; }

// What the forward product and its gradient check alike.
int check_common(int type, char TransA, char TransB, int64_t M, int64_t N, int64_t K, float alpha,
                 int64_t ldA, int64_t ldB, int act) {
  if (type == PARALIA_F32)
    return fail(PARALIA_ERR_UNSUPPORTED, "FP32 operands: use PARALiA_tile_sgemm, this routine takes FP16 and BF16");
  if (type != PARALIA_F16 && type != PARALIA_BF16)
    return fail(PARALIA_ERR_INVALID_ARG, "element type %d is not PARALIA_F16 or PARALIA_BF16", type);
  if (!is_flag(TransA) || !is_flag(TransB)) return fail(PARALIA_ERR_INVALID_ARG, "transpose flag is not N or T");
  if (M < 0 || N < 0 || K < 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX)
    return fail(PARALIA_ERR_INVALID_ARG, "dimension out of range");
  if (M > GA_MAX_ROWS || N > GA_MAX_ROWS)
    return fail(PARALIA_ERR_UNSUPPORTED, "M = %lld, N = %lld: more than %d rows or columns", (long long)M, (long long)N,
                GA_MAX_ROWS);
  if (act < PARALIA_ACT_NONE || act > PARALIA_ACT_SILU)
    return fail(PARALIA_ERR_INVALID_ARG, "activation %d is not one of PARALIA_ACT_*", act);
  if (ldA < std::max<int64_t>(1, is_trans(TransA) ? K : M) || ldB < std::max<int64_t>(1, is_trans(TransB) ? N : K))
    return fail(PARALIA_ERR_INVALID_ARG, "leading dimension smaller than the stored row count");
  if (!std::isfinite(alpha)) return fail(PARALIA_ERR_INVALID_ARG, "alpha is not finite");
  return PARALIA_OK;
}

int check_scratch(const void* scratch, int64_t have, int64_t need) {
  if (!scratch || have < need)
    return fail(PARALIA_ERR_INVALID_ARG, "the call needs %lld bytes of scratch, %lld were given", (long long)need,
                (long long)(scratch ? have : 0));
  if (reinterpret_cast<uintptr_t>(scratch) & 15)
    return fail(PARALIA_ERR_INVALID_ARG, "scratch is not aligned to 16 bytes");
  return PARALIA_OK;
}

bool odd_address(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1) != 0; }

Region matrix(const void* p, int64_t rows, int64_t cols, int64_t ld) { return region(p, rows, cols, ld, 2); }

// Whether one of the n_w written regions shares memory with another of them or with one that is read.
bool written_overlap(const Region* w, int n_w, const Region* r, int n_r) {
  for (int i = 0; i < n_w; ++i) {
    for (int j = i + 1; j < n_w; ++j)
      if (regions_overlap(w[i], w[j])) return true;
    for (int j = 0; j < n_r; ++j)
      if (regions_overlap(w[i], r[j])) return true;
  }
  return false;
}

}  // namespace

namespace {

// What the operands of op(A) op(B) have in scratch: `bytes` with every copy that pays, `needed` with those
// alone without which TMA cannot read an operand. The gradient reads A for N columns of dB and B
// for M rows of dA, as the product itself does.
struct OperandCopies {
  GemmActCopy a, b;
  int64_t bytes, needed;
  // which copies are made with `room` bytes of scratch
  bool make(GemmActCopy c, int64_t room) const { return c == GA_COPY_NEEDED || (c == GA_COPY_PAYS && room >= bytes); }
};
OperandCopies operand_copies(int64_t M, int64_t N, int64_t K, bool ta, bool tb, const void* A, int64_t ldA,
                             const void* B, int64_t ldB) {
  OperandCopies c;
  const int64_t ra = ta ? K : M, ca = ta ? M : K, rb = tb ? N : K, cb = tb ? K : N;
  c.a = gemm_act_operand_copy(A, ldA, ra, ca, N);
  c.b = gemm_act_operand_copy(B, ldB, rb, cb, M);
  const int64_t bytes_a = gemm_act_copy_bytes(ra, ca), bytes_b = gemm_act_copy_bytes(rb, cb);
  c.bytes = (c.a != GA_COPY_NONE ? bytes_a : 0) + (c.b != GA_COPY_NONE ? bytes_b : 0);
  c.needed = (c.a == GA_COPY_NEEDED ? bytes_a : 0) + (c.b == GA_COPY_NEEDED ? bytes_b : 0);
  return c;
}

}  // namespace

int64_t gemm_act_scratch_bytes(int type, char TransA, char TransB, int64_t M, int64_t N, int64_t K,
                               const void* A, int64_t ldA, const void* B, int64_t ldB) {
  if (check_common(type, TransA, TransB, M, N, K, 1.0f, ldA, ldB, PARALIA_ACT_NONE) != PARALIA_OK) return 0;
  if (M == 0 || N == 0 || K == 0) return 0;
  return operand_copies(M, N, K, is_trans(TransA), is_trans(TransB), A, ldA, B, ldB).bytes;
}

int exec_tile_gemm_act(int dev, void* stream, int type, char TransA, char TransB, int64_t M, int64_t N,
                       int64_t K, float alpha, const void* A, int64_t ldA, const void* B, int64_t ldB,
                       const void* bias, int act, float beta, const void* C, int64_t ldC, void* D,
                       int64_t ldD, void* pre, int64_t ldPre, void* scratch, int64_t scratch_bytes) {
  PL_TRY(check_common(type, TransA, TransB, M, N, K, alpha, ldA, ldB, act));
  if (!std::isfinite(beta)) return fail(PARALIA_ERR_INVALID_ARG, "beta is not finite");
  const int64_t rows = std::max<int64_t>(1, M);
  if (ldD < rows || (beta != 0.0f && ldC < rows) || (pre && ldPre < rows))
    return fail(PARALIA_ERR_INVALID_ARG, "leading dimension smaller than the stored row count");
  if (M == 0 || N == 0) return PARALIA_OK;
  const bool product = K > 0 && alpha != 0.0f;
  if (!D || (product && (!A || !B)) || (beta != 0.0f && !C)) return fail(PARALIA_ERR_INVALID_ARG, "NULL operand");
  if (odd_address(A) || odd_address(B) || odd_address(C) || odd_address(D) || odd_address(bias) || odd_address(pre))
    return fail(PARALIA_ERR_INVALID_ARG, "operand address is not a multiple of the element size");
  OperandCopies copies = {GA_COPY_NONE, GA_COPY_NONE, 0, 0};
  if (product) copies = operand_copies(M, N, K, is_trans(TransA), is_trans(TransB), A, ldA, B, ldB);
  if (copies.needed > 0) PL_TRY(check_scratch(scratch, scratch_bytes, copies.needed));
  const int64_t room = scratch && !(reinterpret_cast<uintptr_t>(scratch) & 15) ? scratch_bytes : 0;
  {
    const bool ta = is_trans(TransA), tb = is_trans(TransB);
    // D may be C; a tile of C is read before the same tile of D is written
    const bool in_place = beta != 0.0f && D == C && (ldD == ldC || N == 1);
    const int64_t used = room >= copies.bytes ? copies.bytes : copies.needed;
    const Region w[] = {matrix(D, M, N, ldD), matrix(pre, M, N, ldPre), region(scratch, used, 1, used, 1)};
    const Region r[] = {matrix(A, ta ? K : M, ta ? M : K, ldA), matrix(B, tb ? N : K, tb ? K : N, ldB),
                        matrix(bias, M, 1, M), matrix(beta != 0.0f && !in_place ? C : nullptr, M, N, ldC)};
    if (written_overlap(w, 3, r, 4))
      return fail(PARALIA_ERR_INVALID_ARG,
                  "an output or scratch may share memory with no operand, but D with C at the same leading dimension");
  }
  DeviceGuard guard;
  Runtime& rt = Runtime::get();
  PL_TRY(rt.init());
  PL_TRY(rt.enter_tile_call(dev, static_cast<cudaStream_t>(stream)));
  GemmActProblem p;
  memset(&p, 0, sizeof(p));
  p.A = A; p.B = B; p.bias = bias; p.C = beta != 0.0f ? C : nullptr; p.D = D; p.pre = pre;
  p.ldA = ldA; p.ldB = ldB; p.ldC = ldC; p.ldD = ldD; p.ldPre = ldPre;
  p.M = (int32_t)M; p.N = (int32_t)N; p.K = product ? (int32_t)K : 0;
  p.ta = is_trans(TransA); p.tb = is_trans(TransB);
  p.copy_a = copies.make(copies.a, room); p.copy_b = copies.make(copies.b, room);
  p.act = act; p.bf16 = type == PARALIA_BF16;
  p.alpha = alpha; p.beta = beta;
  return launch_gemm_act(&p, 1, scratch, rt.dev(dev).status_dev, static_cast<cudaStream_t>(stream));
}

namespace {

// Scratch of the gradient: dZ (M x N in an aligned layout; without an activation the copy of dD where it
// has one), then the copies of A and of B.
struct GradScratch {
  int64_t ldZ, z_bytes;
  OperandCopies copies;
};
GradScratch grad_scratch(int64_t M, int64_t N, int64_t K, bool ta, bool tb, const void* A, int64_t ldA, const void* B,
                         int64_t ldB) {
  GradScratch g;
  g.ldZ = gemm_act_copy_ld(std::max<int64_t>(1, M));
  g.z_bytes = gemm_act_copy_bytes(std::max<int64_t>(1, M), N);
  g.copies = operand_copies(M, N, K, ta, tb, A, ldA, B, ldB);
  return g;
}

}  // namespace

int64_t gemm_act_grad_scratch_bytes(int type, char TransA, char TransB, int64_t M, int64_t N, int64_t K,
                                    const void* A, int64_t ldA, const void* B, int64_t ldB, int act) {
  if (check_common(type, TransA, TransB, M, N, K, 1.0f, ldA, ldB, act) != PARALIA_OK) return 0;
  const GradScratch g = grad_scratch(M, N, K, is_trans(TransA), is_trans(TransB), A, ldA, B, ldB);
  return g.z_bytes + g.copies.bytes;
}

int exec_tile_gemm_act_grad(int dev, void* stream, int type, char TransA, char TransB, int64_t M, int64_t N,
                            int64_t K, float alpha, const void* A, int64_t ldA, const void* B, int64_t ldB,
                            int act, const void* pre, int64_t ldPre, const void* dD, int64_t lddD,
                            float betaA, void* dA, int64_t lddA, float betaB, void* dB, int64_t lddB,
                            float betaBias, void* dbias, void* scratch, int64_t scratch_bytes) {
  PL_TRY(check_common(type, TransA, TransB, M, N, K, alpha, ldA, ldB, act));
  if (!std::isfinite(betaA) || !std::isfinite(betaB) || !std::isfinite(betaBias))
    return fail(PARALIA_ERR_INVALID_ARG, "beta is not finite");
  if (K > GA_MAX_ROWS)
    return fail(PARALIA_ERR_UNSUPPORTED, "K = %lld: more than %d rows or columns", (long long)K, GA_MAX_ROWS);
  const bool ta = is_trans(TransA), tb = is_trans(TransB);
  const bool uses_pre = act != PARALIA_ACT_NONE;
  const int64_t rows = std::max<int64_t>(1, M);
  if (lddD < rows || (uses_pre && ldPre < rows) || (dA && lddA < std::max<int64_t>(1, ta ? K : M)) ||
      (dB && lddB < std::max<int64_t>(1, tb ? N : K)))
    return fail(PARALIA_ERR_INVALID_ARG, "leading dimension smaller than the stored row count");
  const bool want_a = dA && M > 0 && K > 0, want_b = dB && N > 0 && K > 0, want_bias = dbias && M > 0;
  if (!want_a && !want_b && !want_bias) return PARALIA_OK;
  const bool entries = M > 0 && N > 0;
  if (entries && (!dD || (uses_pre && !pre))) return fail(PARALIA_ERR_INVALID_ARG, "NULL operand");
  if (entries && alpha != 0.0f && ((want_a && !B) || (want_b && !A))) return fail(PARALIA_ERR_INVALID_ARG, "NULL operand");
  if (odd_address(A) || odd_address(B) || odd_address(pre) || odd_address(dD) || odd_address(dA) ||
      odd_address(dB) || odd_address(dbias))
    return fail(PARALIA_ERR_INVALID_ARG, "operand address is not a multiple of the element size");
  // What this call touches of its scratch: nothing without a product; without an activation dZ is dD, in
  // place unless it is to be copied.
  const GradScratch g = grad_scratch(M, N, K, ta, tb, A, ldA, B, ldB);
  const bool products = entries && K > 0 && alpha != 0.0f && (want_a || want_b);
  const int64_t room = scratch && !(reinterpret_cast<uintptr_t>(scratch) & 15) ? scratch_bytes : 0;
  const GemmActCopy copy_z = uses_pre ? GA_COPY_NEEDED : gemm_act_operand_copy(dD, lddD, M, N, K);
  const bool need_z =
      products && (copy_z == GA_COPY_NEEDED || (copy_z == GA_COPY_PAYS && room >= g.z_bytes + g.copies.needed));
  const int64_t z_bytes = need_z ? g.z_bytes : 0, needed = products ? z_bytes + g.copies.needed : 0;
  if (needed > 0) PL_TRY(check_scratch(scratch, scratch_bytes, needed));
  const bool every_copy = room - z_bytes >= g.copies.bytes;
  const int64_t used = !products ? 0 : z_bytes + (every_copy ? g.copies.bytes : g.copies.needed);
  {
    const Region w[] = {matrix(want_a ? dA : nullptr, ta ? K : M, ta ? M : K, lddA),
                        matrix(want_b ? dB : nullptr, tb ? N : K, tb ? K : N, lddB),
                        matrix(want_bias ? dbias : nullptr, M, 1, M), region(scratch, used, 1, used, 1)};
    const Region r[] = {matrix(A, ta ? K : M, ta ? M : K, ldA), matrix(B, tb ? N : K, tb ? K : N, ldB),
                        matrix(uses_pre ? pre : nullptr, M, N, ldPre), matrix(dD, M, N, lddD)};
    if (written_overlap(w, 4, r, 4))
      return fail(PARALIA_ERR_INVALID_ARG, "a gradient or scratch may share memory with no operand and no other gradient");
  }
  DeviceGuard guard;
  Runtime& rt = Runtime::get();
  PL_TRY(rt.init());
  PL_TRY(rt.enter_tile_call(dev, static_cast<cudaStream_t>(stream)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = type == PARALIA_BF16;

  // dZ and the bias gradient in one pass over dD and pre
  char* base = static_cast<char*>(scratch);
  if (need_z || want_bias) {
    ActGradProblem a;
    memset(&a, 0, sizeof(a));
    a.pre = pre; a.dD = dD; a.dZ = need_z ? base : nullptr; a.dbias = want_bias ? dbias : nullptr;
    a.ldPre = ldPre; a.ldD = lddD; a.ldZ = g.ldZ;
    a.M = (int32_t)M; a.N = (int32_t)N; a.act = act; a.bf16 = bf16; a.beta_bias = betaBias;
    PL_CUDA(launch_act_grad(a, s));
  }
  const void* dZ = need_z ? base : dD;
  const int64_t ldZ = need_z ? g.ldZ : lddD;
  void* copies = base + z_bytes;
  int* status = rt.dev(dev).status_dev;

  const bool copy_a = g.copies.make(g.copies.a, room - z_bytes);
  const bool copy_b = g.copies.make(g.copies.b, room - z_bytes);

  GemmActProblem ps[2];
  memset(ps, 0, sizeof(ps));
  int count = 0;
  if (want_b) {
    // d op(B) = alpha op(A)^T dZ, stored as B is
    GemmActProblem& p = ps[count++];
    p.D = dB; p.ldD = lddB; p.C = betaB != 0.0f ? dB : nullptr; p.ldC = lddB; p.beta = betaB;
    p.K = alpha != 0.0f ? (int32_t)M : 0;
    if (!tb) {
      p.A = A; p.ldA = ldA; p.ta = !ta; p.copy_a = copy_a; p.B = dZ; p.ldB = ldZ; p.tb = 0;
      p.M = (int32_t)K; p.N = (int32_t)N;
    } else {
      p.A = dZ; p.ldA = ldZ; p.ta = 1; p.B = A; p.ldB = ldA; p.tb = ta; p.copy_b = copy_a;
      p.M = (int32_t)N; p.N = (int32_t)K;
    }
  }
  if (want_a) {
    // d op(A) = alpha dZ op(B)^T, stored as A is
    GemmActProblem& p = ps[count++];
    p.D = dA; p.ldD = lddA; p.C = betaA != 0.0f ? dA : nullptr; p.ldC = lddA; p.beta = betaA;
    p.K = alpha != 0.0f ? (int32_t)N : 0;
    if (!ta) {
      p.A = dZ; p.ldA = ldZ; p.ta = 0; p.B = B; p.ldB = ldB; p.tb = !tb; p.copy_b = copy_b;
      p.M = (int32_t)M; p.N = (int32_t)K;
    } else {
      p.A = B; p.ldA = ldB; p.ta = tb; p.copy_a = copy_b; p.B = dZ; p.ldB = ldZ; p.tb = 1;
      p.M = (int32_t)K; p.N = (int32_t)M;
    }
  }
  for (int i = 0; i < count; ++i) {
    ps[i].act = PARALIA_ACT_NONE;
    ps[i].bf16 = bf16;
    ps[i].alpha = alpha;
  }
  return launch_gemm_act(ps, count, copies, status, s);
}

}  // namespace paralia
