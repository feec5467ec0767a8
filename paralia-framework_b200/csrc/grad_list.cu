// Global norm of a list of gradient tensors, and their scaling to a largest norm:
//   norm = sqrt(sum_i sum_j g_ij^2),   out_ij = g_ij * (norm > max_norm ? max_norm / norm : 1).
//
// Both kernels are bound by HBM: one read of the list for the norm, one read and one write for
// the scaling. The list travels in the kernel's parameters (no copy, nothing kept between
// calls, capturable); it is cut into chunks of equal length, block b takes chunks b, b + grid,
// ..., and a binary search over the tensors' first chunks finds the tensor of a chunk. The
// order of every sum is a function of the list alone.
//
// Squares: of FP32 elements they are summed in FP64 throughout (a conversion and an FMA an
// element, which the FP64 pipe keeps up with at HBM speed). Of 16-bit elements the eight of
// one 16-byte load are summed in FP32 (their squares are exact there) and the sum goes to
// FP64: one conversion for eight elements instead of eight, at a relative error of a few
// 2^-24 per group of eight. Where such a sum leaves the range in which FP32 is that exact, the group is
// summed again in FP64, so that gradients near the ends of BF16's range count in full.
#include "grad_list.cuh"

#include <algorithm>

#include "act_math.cuh"

namespace paralia {
namespace {

constexpr int GL_THREADS = 512;

template <int CAP>
struct GradTable {
  int32_t count;
  int32_t chunk;        // elements
  int32_t chunk_begin;  // first chunk of this launch (chunk0 of the entries counts from there)
  int32_t chunks;
  GradEntry e[CAP];
};

// Index of the tensor that holds chunk c.
template <int CAP>
__device__ __forceinline__ int find_tensor(const GradTable<CAP>& t, int c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].chunk0 <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int type) {
  if (type == PARALIA_F32) return static_cast<const float*>(p)[i];
  return load16(p, i, type == PARALIA_BF16);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int type) {
  if (type == PARALIA_F32) static_cast<float*>(p)[i] = v;
  else store16(p, i, v, type == PARALIA_BF16);
}

// Eight neighbouring elements on a 16-byte boundary as loaded.
template <bool F32>
struct Raw {
  uint4 a, b;
};
template <>
struct Raw<false> {
  uint4 a;
};
template <bool F32>
__device__ __forceinline__ Raw<F32> load_raw(const void* p, int64_t i) {
  Raw<F32> r;
  if constexpr (F32) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
    r.a = q[0];
    r.b = q[1];
  } else {
    r.a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
  }
  return r;
}
template <bool F32>
__device__ __forceinline__ void to_floats(const Raw<F32>& r, bool bf, float (&v)[8]) {
  if constexpr (F32) {
    v[0] = __uint_as_float(r.a.x); v[1] = __uint_as_float(r.a.y);
    v[2] = __uint_as_float(r.a.z); v[3] = __uint_as_float(r.a.w);
    v[4] = __uint_as_float(r.b.x); v[5] = __uint_as_float(r.b.y);
    v[6] = __uint_as_float(r.b.z); v[7] = __uint_as_float(r.b.w);
  } else {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack16(w[i], bf);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <bool F32>
__device__ __forceinline__ double group_sumsq(const Raw<F32>& r, bool bf) {
  float v[8];
  to_floats<F32>(r, bf, v);
  if constexpr (F32) {
    double s0 = 0.0, s1 = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      s0 = fma((double)v[i], (double)v[i], s0);
      s1 = fma((double)v[i + 1], (double)v[i + 1], s1);
    }
    return s0 + s1;
  } else {
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      s0 = fmaf(v[i], v[i], s0);
      s1 = fmaf(v[i + 1], v[i + 1], s1);
    }
    const float s = s0 + s1;
    // 1e-30: what squares below 2^-126 lose is then under 2^-24 of the sum
    if (s > 1e-30f && s < 1e30f) return (double)s;
    if ((r.a.x | r.a.y | r.a.z | r.a.w) == 0u) return 0.0;
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) d = fma((double)v[i], (double)v[i], d);
    return d;
  }
}

// Sum over the block in a fixed order; every thread gets it.
__device__ __forceinline__ double block_total(double v, double* warp_sums) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < GL_THREADS / 32; ++w) s += warp_sums[w];
  return s;
}

// The part of a tensor that chunk c covers: elements [lo, hi), whose groups of eight start at
// `vec` (lo, or lo + head in the tensor's first chunk).
struct Span {
  int64_t lo, vec, hi;
};
__device__ __forceinline__ Span chunk_span(const GradEntry& e, int c, int chunk) {
  Span s;
  const int64_t first = e.head + (int64_t)(c - e.chunk0) * chunk;
  s.lo = c == e.chunk0 ? 0 : first;
  s.vec = first < e.n ? first : e.n;
  s.hi = min(e.n, first + chunk);
  return s;
}

template <bool F32>
__device__ __forceinline__ double chunk_sumsq(const GradEntry& e, const Span& s) {
  constexpr int U = F32 ? 2 : 4;
  const bool bf = e.src_type == PARALIA_BF16;
  double acc = 0.0;
  const int64_t groups = (e.flags & GL_SRC_VEC) ? (s.hi - s.vec) / 8 : 0;
  int64_t g = threadIdx.x;
  for (; g + (U - 1) * GL_THREADS < groups; g += U * GL_THREADS) {
    Raw<F32> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = load_raw<F32>(e.src, s.vec + (g + u * GL_THREADS) * 8);
#pragma unroll
    for (int u = 0; u < U; ++u) acc += group_sumsq<F32>(r[u], bf);
  }
  for (; g < groups; g += GL_THREADS) acc += group_sumsq<F32>(load_raw<F32>(e.src, s.vec + g * 8), bf);
  for (int64_t i = s.lo + threadIdx.x; i < s.vec; i += GL_THREADS) {
    const double v = load_any(e.src, i, e.src_type);
    acc = fma(v, v, acc);
  }
  for (int64_t i = s.vec + groups * 8 + threadIdx.x; i < s.hi; i += GL_THREADS) {
    const double v = load_any(e.src, i, e.src_type);
    acc = fma(v, v, acc);
  }
  return acc;
}

template <int CAP>
__global__ void __launch_bounds__(GL_THREADS)
grad_sumsq_kernel(const __grid_constant__ GradTable<CAP> t, double* __restrict__ partials) {
  __shared__ double warp_sums[GL_THREADS / 32];
  double acc = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const GradEntry& e = t.e[find_tensor(t, c)];
    const Span s = chunk_span(e, c, t.chunk);
    acc += e.src_type == PARALIA_F32 ? chunk_sumsq<true>(e, s) : chunk_sumsq<false>(e, s);
  }
  const double total = block_total(acc, warp_sums);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

__device__ __forceinline__ double sum_partials(const double* partials, int used, double* warp_sums) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < used; i += GL_THREADS) acc += partials[i];
  return block_total(acc, warp_sums);
}

__global__ void __launch_bounds__(GL_THREADS)
grad_norm_final_kernel(const double* __restrict__ partials, int used, double* sumsq, float* norm) {
  __shared__ double warp_sums[GL_THREADS / 32];
  const double s = sum_partials(partials, used, warp_sums);
  if (threadIdx.x == 0) {
    if (sumsq) *sumsq = s;
    if (norm) *norm = (float)sqrt(s);
  }
}

template <bool F32>
__device__ __forceinline__ void chunk_scale(const GradEntry& e, const Span& s, float k0, float k) {
  constexpr int U = F32 ? 2 : 4;
  const bool bf = e.src_type == PARALIA_BF16, dbf = e.dst_type == PARALIA_BF16;
  const int64_t groups = (e.flags & GL_SRC_VEC) ? (s.hi - s.vec) / 8 : 0;
  auto put = [&](int64_t i, const Raw<F32>& r) {
    float v[8];
    to_floats<F32>(r, bf, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * k0 * k;
    if (!(e.flags & GL_DST_VEC)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) store_any(e.dst, i + j, v[j], e.dst_type);
    } else if (e.dst_type == PARALIA_F32) {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(e.dst) + i);
      q[0] = make_float4(v[0], v[1], v[2], v[3]);
      q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(e.dst) + i) =
          make_uint4(pack16(v[0], v[1], dbf), pack16(v[2], v[3], dbf), pack16(v[4], v[5], dbf),
                     pack16(v[6], v[7], dbf));
    }
  };
  int64_t g = threadIdx.x;
  for (; g + (U - 1) * GL_THREADS < groups; g += U * GL_THREADS) {
    Raw<F32> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = load_raw<F32>(e.src, s.vec + (g + u * GL_THREADS) * 8);
#pragma unroll
    for (int u = 0; u < U; ++u) put(s.vec + (g + u * GL_THREADS) * 8, r[u]);
  }
  for (; g < groups; g += GL_THREADS) put(s.vec + g * 8, load_raw<F32>(e.src, s.vec + g * 8));
  for (int64_t i = s.lo + threadIdx.x; i < s.vec; i += GL_THREADS)
    store_any(e.dst, i, load_any(e.src, i, e.src_type) * k0 * k, e.dst_type);
  for (int64_t i = s.vec + groups * 8 + threadIdx.x; i < s.hi; i += GL_THREADS)
    store_any(e.dst, i, load_any(e.src, i, e.src_type) * k0 * k, e.dst_type);
}

// Chunks are taken from the end of the list: what the norm kernel read last is what L2 still
// holds.
template <int CAP>
__global__ void __launch_bounds__(GL_THREADS)
grad_scale_kernel(const __grid_constant__ GradTable<CAP> t, const double* __restrict__ partials, int used,
                  float max_norm, double* sumsq, float* norm) {
  __shared__ double warp_sums[GL_THREADS / 32];
  const double total = sum_partials(partials, used, warp_sums);
  const double len = sqrt(total);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (sumsq) *sumsq = total;
    if (norm) *norm = (float)len;
  }
  // a norm that is not finite clips nothing: the comparison is false for a NaN
  double factor = len > (double)max_norm && len < INFINITY ? (double)max_norm / len : 1.0;
  // a factor near the end of FP32's range (a norm near it) goes in two steps, since a subnormal
  // one would have lost digits
  const float k0 = factor < 0x1p-90 ? 0x1p-64f : 1.0f;
  if (k0 != 1.0f) factor *= 0x1p64;
  const float k = (float)factor;
  for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const GradEntry& e = t.e[find_tensor(t, c)];
    if (k == 1.0f && k0 == 1.0f && (e.flags & GL_IN_PLACE)) continue;
    const Span s = chunk_span(e, c, t.chunk);
    if (e.src_type == PARALIA_F32) chunk_scale<true>(e, s, k0, k);
    else chunk_scale<false>(e, s, k0, k);
  }
}

// Calls f(table) for each run of the list that fits one launch; `last_first`: from the end.
template <typename F>
cudaError_t for_tables(const GradList& l, bool last_first, F f) {
  const int runs = (l.count + GL_MAX_TENSORS - 1) / GL_MAX_TENSORS;
  for (int r = 0; r < runs; ++r) {
    const int i0 = (last_first ? runs - 1 - r : r) * GL_MAX_TENSORS;
    const int n = std::min(GL_MAX_TENSORS, l.count - i0);
    const int64_t begin = l.entries[i0].chunk0;
    const int64_t end = i0 + n < l.count ? l.entries[i0 + n].chunk0 : l.chunks;
    auto fill = [&](auto& t) {
      t.count = n;
      t.chunk = l.chunk;
      t.chunk_begin = (int32_t)begin;
      t.chunks = (int32_t)(end - begin);
      for (int i = 0; i < n; ++i) {
        t.e[i] = l.entries[i0 + i];
        t.e[i].chunk0 -= (int32_t)begin;
      }
      return f(t);
    };
    cudaError_t e;
    if (n <= 32) {
      GradTable<32> t;
      e = fill(t);
    } else if (n <= 256) {
      GradTable<256> t;
      e = fill(t);
    } else {
      GradTable<GL_MAX_TENSORS> t;
      e = fill(t);
    }
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

int grad_chunk_elements(int64_t total) {
  // about four chunks for every block of a full grid, between two and eight groups of eight
  // elements for every thread of a block
  const int64_t want = total / (GL_MAX_BLOCKS * 4);
  int chunk = GL_THREADS * 8;
  while (chunk < want && chunk < GL_THREADS * 64) chunk *= 2;
  return chunk;
}

int64_t grad_partials(int64_t count) {
  const int64_t runs = (count + GL_MAX_TENSORS - 1) / GL_MAX_TENSORS;
  return std::max<int64_t>(1, runs) * GL_MAX_BLOCKS;
}

cudaError_t launch_grad_sumsq(const GradList& l, double* partials, int* used, cudaStream_t stream) {
  *used = 0;
  return for_tables(l, false, [&](const auto& t) {
    const int grid = std::min(t.chunks, GL_MAX_BLOCKS);
    grad_sumsq_kernel<<<grid, GL_THREADS, 0, stream>>>(t, partials + *used);
    *used += grid;
    return cudaGetLastError();
  });
}

cudaError_t launch_grad_norm_final(const double* partials, int used, double* sumsq, float* norm, cudaStream_t stream) {
  grad_norm_final_kernel<<<1, GL_THREADS, 0, stream>>>(partials, used, sumsq, norm);
  return cudaGetLastError();
}

cudaError_t launch_grad_scale(const GradList& l, const double* partials, int used, float max_norm, double* sumsq,
                              float* norm, cudaStream_t stream) {
  if (l.count == 0) return launch_grad_norm_final(partials, used, sumsq, norm, stream);
  return for_tables(l, true, [&](const auto& t) {
    const int grid = std::min(t.chunks, GL_MAX_BLOCKS);
    grad_scale_kernel<<<grid, GL_THREADS, 0, stream>>>(t, partials, used, max_norm, sumsq, norm);
    return cudaGetLastError();
  });
}

}  // namespace paralia
