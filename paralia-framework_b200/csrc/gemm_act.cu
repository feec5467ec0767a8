// Matrix product with bias, activation and residual in its epilogue, FP16 / BF16.
#include "gemm_act.cuh"

#include <algorithm>

#include "act_math.cuh"

namespace paralia {
namespace {

constexpr int GA_TILE = 64;
constexpr int GA_K = 16;

// 64 x 64 tile of D per block of 256 threads, 4 x 4 entries per thread, operands through
// shared memory as FP32.
__global__ void __launch_bounds__(256) gemm_act_kernel(const GemmActProblem p) {
  __shared__ float sa[GA_K][GA_TILE + 1], sb[GA_K][GA_TILE + 1];
  const int m0 = blockIdx.x * GA_TILE, n0 = blockIdx.y * GA_TILE;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const bool bf = p.bf16 != 0;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += GA_K) {
    for (int i = threadIdx.x; i < GA_TILE * GA_K; i += 256) {
      // walk the contiguous dimension of the stored operand first
      const int ka = p.ta ? i % GA_K : i / GA_TILE, ma = p.ta ? i / GA_K : i % GA_TILE;
      const int kb = p.tb ? i / GA_TILE : i % GA_K, nb = p.tb ? i % GA_TILE : i / GA_K;
      const int64_t m = m0 + ma, n = n0 + nb;
      sa[ka][ma] = (m < p.M && k0 + ka < p.K)
                       ? load16(p.A, p.ta ? (k0 + ka) + m * p.ldA : m + (int64_t)(k0 + ka) * p.ldA, bf)
                       : 0.0f;
      sb[kb][nb] = (n < p.N && k0 + kb < p.K)
                       ? load16(p.B, p.tb ? n + (int64_t)(k0 + kb) * p.ldB : (k0 + kb) + n * p.ldB, bf)
                       : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < GA_K; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = sa[k][tx + 16 * i];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = sb[k][ty + 16 * j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
  with_act(p.act, [&](auto a) {
    for (int i = 0; i < 4; ++i) {
      const int64_t m = m0 + tx + 16 * i;
      if (m >= p.M) continue;
      const float bias = p.bias ? load16(p.bias, m, bf) : 0.0f;
      for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + ty + 16 * j;
        if (n >= p.N) continue;
        const float z = fmaf(p.alpha, acc[i][j], bias);
        if (p.pre) store16(p.pre, m + n * p.ldPre, z, bf);
        float v = act_value<decltype(a)::value>(z);
        if (p.C) v = fmaf(p.beta, load16(p.C, m + n * p.ldC, bf), v);
        store16(p.D, m + n * p.ldD, v, bf);
      }
    }
  });
}

// ------------------------------------------------------------------ gradient of the epilogue
constexpr int AG_ROWS = 256;     // rows of a block: 32 lanes x 8
constexpr int AG_WARPS = 8;

// A block takes AG_ROWS rows and a run of columns; a warp walks every AG_WARPS-th column of
// the run, a lane holds eight rows, so the row sums of the bias gradient stay in registers.
// The sums of the eight warps meet in shared memory in warp order and leave as one partial
// per row and run; act_grad_bias_kernel adds the runs in order.
//
// Bound by memory: two reads and one write of two bytes per entry. VEC: rows come and go as
// 16-byte accesses (eight rows of a lane are neighbours); otherwise a lane's eight rows lie
// 32 apart and every access is of one element, coalesced over the warp at any alignment.
template <bool VEC>
__global__ void __launch_bounds__(AG_WARPS * 32) act_grad_kernel(const ActGradProblem p, int cols) {
  __shared__ float sums[AG_WARPS][AG_ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row0 = (int64_t)blockIdx.x * AG_ROWS;
  const int64_t n_begin = (int64_t)blockIdx.y * cols;
  const int64_t n_end = min((int64_t)p.N, n_begin + cols);
  const bool bf = p.bf16 != 0;
  float acc[8] = {};
  with_act(p.act, [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    for (int64_t n = n_begin + warp; n < n_end; n += AG_WARPS) {
      if (VEC) {
        const int64_t m = row0 + lane * 8;
        if (m + 8 <= p.M) {
          const uint4 d = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.dD) + m + n * p.ldD);
          uint4 z = make_uint4(0, 0, 0, 0);
          if (ACT != PARALIA_ACT_NONE)
            z = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.pre) + m + n * p.ldPre);
          const uint32_t dv[4] = {d.x, d.y, d.z, d.w}, zv[4] = {z.x, z.y, z.z, z.w};
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 g = unpack16(dv[i], bf), q = unpack16(zv[i], bf);
            // a select, so that an infinite dD in a place that relu has closed gives 0
            const float g0 = ACT == PARALIA_ACT_RELU ? (q.x > 0.0f ? g.x : 0.0f) : g.x * act_slope<ACT>(q.x);
            const float g1 = ACT == PARALIA_ACT_RELU ? (q.y > 0.0f ? g.y : 0.0f) : g.y * act_slope<ACT>(q.y);
            acc[2 * i] += g0;
            acc[2 * i + 1] += g1;
            o[i] = pack16(g0, g1, bf);
          }
          if (p.dZ)
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dZ) + m + n * p.ldZ) = make_uint4(o[0], o[1], o[2], o[3]);
          continue;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t m = VEC ? row0 + lane * 8 + i : row0 + lane + 32 * i;
        if (m >= p.M) continue;
        const float g = load16(p.dD, m + n * p.ldD, bf);
        const float q = ACT != PARALIA_ACT_NONE ? load16(p.pre, m + n * p.ldPre, bf) : 0.0f;
        const float v = ACT == PARALIA_ACT_RELU ? (q > 0.0f ? g : 0.0f) : g * act_slope<ACT>(q);
        acc[i] += v;
        if (p.dZ) store16(p.dZ, m + n * p.ldZ, v, bf);
      }
    }
  });
  if (!p.dbias) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[warp][VEC ? lane * 8 + i : lane + 32 * i] = acc[i];
  __syncthreads();
  const int64_t m = row0 + threadIdx.x;
  if (m < p.M) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < AG_WARPS; ++w) s += sums[w][threadIdx.x];
    p.partials[(int64_t)blockIdx.y * p.M + m] = s;
  }
}

__global__ void __launch_bounds__(256) act_grad_bias_kernel(const ActGradProblem p, int chunks) {
  const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (m >= p.M) return;
  float s = 0.0f;
  for (int c = 0; c < chunks; ++c) s += p.partials[(int64_t)c * p.M + m];
  if (p.beta_bias != 0.0f) s = fmaf(p.beta_bias, load16(p.dbias, m, p.bf16 != 0), s);
  store16(p.dbias, m, s, p.bf16 != 0);
}

inline bool vec16(const void* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld & 7) == 0;
}

}  // namespace

cudaError_t launch_gemm_act(const GemmActProblem& p, cudaStream_t stream) {
  if (p.M == 0 || p.N == 0) return cudaSuccess;
  const dim3 grid((p.M + GA_TILE - 1) / GA_TILE, (p.N + GA_TILE - 1) / GA_TILE);
  gemm_act_kernel<<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

int act_grad_chunks(int64_t M, int64_t N) {
  // a function of the sizes alone, so that the order of the row sums is too: about 1200
  // blocks, eight for each of 148 SMs, and no run shorter than one column per warp
  const int64_t row_blocks = (M + AG_ROWS - 1) / AG_ROWS;
  const int64_t want = row_blocks > 0 ? (1184 + row_blocks - 1) / row_blocks : 1;
  const int64_t most = std::max<int64_t>(1, (N + AG_WARPS - 1) / AG_WARPS);
  return (int)std::max<int64_t>(1, std::min(want, most));
}

cudaError_t launch_act_grad(const ActGradProblem& p, cudaStream_t stream) {
  if (p.M == 0) return cudaSuccess;
  int chunks = act_grad_chunks(p.M, p.N);
  const int cols = std::max(1, (p.N + chunks - 1) / chunks);
  chunks = (p.N + cols - 1) / cols;   // 0 when there are no columns: the sums are 0
  if (chunks > 0) {
    const dim3 grid((p.M + AG_ROWS - 1) / AG_ROWS, chunks);
    const bool vec = vec16(p.dD, p.ldD) && (!p.dZ || vec16(p.dZ, p.ldZ)) &&
                     (p.act == PARALIA_ACT_NONE || vec16(p.pre, p.ldPre));
    if (vec) act_grad_kernel<true><<<grid, AG_WARPS * 32, 0, stream>>>(p, cols);
    else act_grad_kernel<false><<<grid, AG_WARPS * 32, 0, stream>>>(p, cols);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  if (p.dbias) {
    act_grad_bias_kernel<<<(p.M + 255) / 256, 256, 0, stream>>>(p, chunks);
    return cudaGetLastError();
  }
  return cudaSuccess;
}

}  // namespace paralia
