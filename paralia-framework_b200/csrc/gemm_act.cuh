// Launchers of the mixed-precision linear-layer kernels (FP16 / BF16 operands, FP32 sums).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace paralia {

// One product with its epilogue:
//   Z = alpha * op(A) op(B) + bias,  pre <- Z (optional),  D <- act(Z) + beta * C.
// Every matrix is column-major with 16-bit elements of one type.
struct GemmActProblem {
  const void* A;
  const void* B;
  const void* bias;    // M elements or null
  const void* C;       // null when beta == 0
  void* D;
  void* pre;           // null when the pre-activation is not kept
  int64_t ldA, ldB, ldC, ldD, ldPre;
  int32_t M, N, K;
  int32_t ta, tb;      // op is the transpose
  int32_t copy_a, copy_b;   // the operand goes to scratch first, in an aligned layout
  int32_t act;         // PARALIA_ACT_*
  int32_t bf16;        // 1: BF16, 0: FP16
  float alpha, beta;
};

// Rows and columns a result may have: tiles are numbered, with panels of up to 16 of them and clusters of
// up to 8 CTAs, in 32 bits, and loops over rows or columns step past the end in them.
constexpr int GA_MAX_ROWS = (1 << 30) - 128;

// Leading dimension of an aligned copy of columns of `rows` elements: whole lines of 128 bytes unless
// that were a large part of a column.
int64_t gemm_act_copy_ld(int64_t rows);
// The aligned copy of a stored rows x cols operand whose every element meets `reuse` rows or columns of
// the result: whether TMA cannot read the operand without it, whether the product is faster with it.
enum GemmActCopy : int { GA_COPY_NONE = 0, GA_COPY_PAYS = 1, GA_COPY_NEEDED = 2 };
GemmActCopy gemm_act_operand_copy(const void* p, int64_t ld, int64_t rows, int64_t cols, int64_t reuse);
int64_t gemm_act_copy_bytes(int64_t rows, int64_t cols);   // a multiple of 256
// One or two products that do not depend on each other, of the same element type, in as few launches as
// pay; `pre` only with the first. `scratch` (16-byte aligned) holds the copies of operands, at most two in all,
// one behind the other; `status` is the GPU's word for waits that gave up. Returns a PARALIA_* code.
int launch_gemm_act(const GemmActProblem* problems, int count, void* scratch, int* status, cudaStream_t stream);

// Makes every GPU's kernels be configured anew at their next launch (library shutdown).
void gemm_act_forget_configuration();

// dZ <- dD * act'(pre) (dZ may be null; pre is not read for PARALIA_ACT_NONE), and, where
// dbias is not null, dbias <- row sums of the unrounded product + beta_bias * dbias.
struct ActGradProblem {
  const void* pre;
  const void* dD;
  void* dZ;
  void* dbias;
  int64_t ldPre, ldD, ldZ;
  int32_t M, N;
  int32_t act, bf16;
  float beta_bias;
};
cudaError_t launch_act_grad(const ActGradProblem& p, cudaStream_t stream);

}  // namespace paralia
