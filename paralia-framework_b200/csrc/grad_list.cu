// Global norm of a list of gradient tensors, and their scaling to a largest norm:
//   norm = sqrt(sum_i sum_j g_ij^2),   out_ij = g_ij * (norm > max_norm ? max_norm / norm : 1).
//
// Both kernels are bound by HBM: one read of the list for the norm, one read and one write for
// the scaling. The list travels in the kernel's parameters (no copy, nothing kept between
// calls, capturable). It is cut into units of 2048 elements and block b of G takes the b-th of G
// equal runs of units, so what a block has of one tensor is one contiguous span (chunks dealt out
// in turn, with a search for the tensor of each, read 2 GB of BF16 in 365 us; this takes 302, 6.6
// TB/s). The order of every sum is a function of the list alone: sizes, types, addresses modulo 16 bytes.
//
// Squares: of FP32 elements they are summed in FP64 throughout (a conversion and an FMA an
// element, which the FP64 pipe keeps up with at HBM speed: 256 Mi elements 161 us, 6.67 TB/s). Of 16-bit elements the eight of
// one 16-byte load are summed in FP32 (their squares are exact there) and the sum goes to
// FP64: one conversion for eight elements instead of eight, at a relative error of a few
// 2^-24 per group of eight. Where such a sum leaves the range in which FP32 is that exact, the group is
// summed again in FP64, so that gradients near the ends of BF16's range count in full.
#include "grad_list.cuh"

#include <algorithm>
#include <cstring>
#include <utility>

#include "act_math.cuh"

namespace paralia {
namespace {

constexpr int GL_THREADS = 512;
constexpr int GL_CHUNK = 8;      // units a block scales at most: four groups of eight for every thread

template <int CAP>
struct GradTable {
  int32_t count;
  int32_t units;        // of this launch (unit0 of the entries counts within it)
  int32_t starts;       // first[s] = the tensor with unit  units * s / starts
  uint16_t first[GL_NORM_BLOCKS];
  GradEntry e[CAP];
};

// Programmatic dependent launch: wait until the kernels this one depends on have completed; let
// the next kernel be set up on free resources.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    r.a = q[0];
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

// Units [u0, u1) of the launch within tensor e: elements [lo, hi), whose groups of eight start at
// `vec` (lo, or behind the head at the tensor's beginning).
struct Span {
  int64_t lo, vec, hi;
};
__device__ __forceinline__ Span unit_span(const GradEntry& e, int u0, int u1) {
  Span s;
  const int64_t first = e.head + (int64_t)(u0 - e.unit0) * GL_UNIT;
  s.lo = u0 == e.unit0 ? 0 : min(first, e.n);
  s.vec = min(first, e.n);
  s.hi = min(e.n, e.head + (int64_t)(u1 - e.unit0) * GL_UNIT);
  return s;
}

// This block's run of units.
template <int CAP>
__device__ __forceinline__ int2 block_units(const GradTable<CAP>& t) {
  return make_int2((int)((int64_t)t.units * blockIdx.x / gridDim.x), (int)((int64_t)t.units * (blockIdx.x + 1) / gridDim.x));
}
template <int CAP>
__device__ __forceinline__ int tensor_end(const GradTable<CAP>& t, int i) {
  return i + 1 < t.count ? t.e[i + 1].unit0 : t.units;
}

// The one element outside the groups of eight that this thread has, if any: the first threads take
// those in front, the threads from 32 on those behind (seven at most each). -1: none.
__device__ __forceinline__ int64_t odd_element(const Span& s, int64_t groups) {
  const int t = threadIdx.x;
  if (t < s.vec - s.lo) return s.lo + t;
  const int64_t i = s.vec + groups * 8 + t - 32;
  return t >= 32 && i < s.hi ? i : -1;
}

template <bool F32>
__device__ __forceinline__ double span_sumsq(const GradEntry& e, const Span& s) {
  constexpr int U = F32 ? 2 : 4;
  const bool bf = e.src_type == PARALIA_BF16;
  double acc = 0.0;
  const int64_t groups = (s.hi - s.vec) / 8;
  const int64_t odd = odd_element(s, groups);
  const double x = odd >= 0 ? (double)load_any(e.src, odd, e.src_type) : 0.0;   // in flight with the first groups
  for (int64_t g = threadIdx.x; g < groups; g += U * GL_THREADS) {
    Raw<F32> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      r[u] = Raw<F32>{};
      if (g + u * GL_THREADS < groups) r[u] = load_raw<F32>(e.src, s.vec + (g + u * GL_THREADS) * 8);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) acc += group_sumsq<F32>(r[u], bf);
  }
  return fma(x, x, acc);
}

template <int CAP>
__global__ void __launch_bounds__(GL_THREADS, 3)
grad_sumsq_kernel(const __grid_constant__ GradTable<CAP> t, double* __restrict__ partials) {
  __shared__ double warp_sums[GL_THREADS / 32];
  const int2 run = block_units(t);
  double acc = 0.0;
  int i = t.first[blockIdx.x];
  pdl_wait();
  pdl_launch();
  for (int u = run.x; u < run.y; ++i) {
    const GradEntry& e = t.e[i];
    const int end = min(run.y, tensor_end(t, i));
    const Span s = unit_span(e, u, end);
    acc += e.src_type == PARALIA_F32 ? span_sumsq<true>(e, s) : span_sumsq<false>(e, s);
    u = end;
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
grad_norm_final_kernel(const double* partials, int used, double* sumsq, float* norm) {
  __shared__ double warp_sums[GL_THREADS / 32];
  pdl_wait();
  pdl_launch();
  const double s = sum_partials(partials, used, warp_sums);
  if (threadIdx.x == 0) {
    if (sumsq) *sumsq = s;
    if (norm) *norm = (float)sqrt(s);
  }
}

// Groups of eight from element `from` on: SRC and DST are PARALIA_* types, both sides on 16-byte
// boundaries.
template <int SRC, int DST>
__device__ __forceinline__ void scale_groups(const void* src, void* dst, int64_t from, int groups, float k0, float k) {
  constexpr bool F32 = SRC == PARALIA_F32;
  constexpr int U = F32 ? 2 : 4;
  if ((int)threadIdx.x >= groups) return;
  Raw<F32> r[U];
  auto fetch = [&](int g) {
#pragma unroll
    for (int u = 0; u < U; ++u)   // past the end the last group again
      r[u] = load_raw<F32>(src, from + (int64_t)min(g + u * GL_THREADS, groups - 1) * 8);
  };
  for (int g = threadIdx.x; g < groups; g += U * GL_THREADS) {
    fetch(g);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = from + (int64_t)(g + u * GL_THREADS) * 8;
      float v[8];
      to_floats<F32>(r[u], SRC == PARALIA_BF16, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] * k0 * k;
      if (g + u * GL_THREADS < groups) {
        if constexpr (DST == PARALIA_F32) {
          float4* q = reinterpret_cast<float4*>(static_cast<float*>(dst) + i);
          q[0] = make_float4(v[0], v[1], v[2], v[3]);
          q[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          constexpr bool bf = DST == PARALIA_BF16;
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + i) =
              make_uint4(pack16(v[0], v[1], bf), pack16(v[2], v[3], bf), pack16(v[4], v[5], bf), pack16(v[6], v[7], bf));
        }
      }
    }
  }
}
template <int SRC>
__device__ __forceinline__ void scale_groups_to(int dst_type, const void* src, void* dst, int64_t from, int groups,
                                                float k0, float k) {
  if (dst_type == PARALIA_F32) scale_groups<SRC, PARALIA_F32>(src, dst, from, groups, k0, k);
  else if (dst_type == PARALIA_F16) scale_groups<SRC, PARALIA_F16>(src, dst, from, groups, k0, k);
  else scale_groups<SRC, PARALIA_BF16>(src, dst, from, groups, k0, k);
}

// SRC, DST: the types of every tensor of the list, or -1 where they differ.
template <int SRC, int DST>
__device__ __forceinline__ void span_scale(const GradEntry& e, const Span& s, float k0, float k) {
  const int src_type = SRC >= 0 ? SRC : e.src_type, dst_type = SRC >= 0 ? DST : e.dst_type;
  if (!(e.flags & GL_DST_VEC)) {
    // source and destination are out of step: an element at a time, both sides coalesced
    constexpr int U = 4;
    for (int64_t i = s.lo + threadIdx.x; i < s.hi; i += U * GL_THREADS) {
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = load_any(e.src, min(i + u * GL_THREADS, s.hi - 1), src_type);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * GL_THREADS < s.hi) store_any(e.dst, i + u * GL_THREADS, x[u] * k0 * k, dst_type);
    }
    return;
  }
  const int groups = (int)((s.hi - s.vec) / 8);   // a chunk's at most
  const int64_t odd = odd_element(s, groups);
  const float x = odd >= 0 ? load_any(e.src, odd, src_type) : 0.0f;
  if constexpr (SRC >= 0) scale_groups<SRC, DST>(e.src, e.dst, s.vec, groups, k0, k);
  else if (src_type == PARALIA_F32) scale_groups_to<PARALIA_F32>(dst_type, e.src, e.dst, s.vec, groups, k0, k);
  else if (src_type == PARALIA_F16) scale_groups_to<PARALIA_F16>(dst_type, e.src, e.dst, s.vec, groups, k0, k);
  else scale_groups_to<PARALIA_BF16>(dst_type, e.src, e.dst, s.vec, groups, k0, k);
  if (odd >= 0) store_any(e.dst, odd, x * k0 * k, dst_type);
}

// A block takes `chunk` units, the last blocks of the list first: what the norm kernel read last is what
// L2 still holds. As many blocks as there are chunks, not one for every place on the SMs: 1.4 GB of BF16
// to as much took 400 us, 473 with blocks that stay and take chunk after chunk (they fall into step,
// all reading, then all writing).
template <int CAP, int SRC, int DST>
__global__ void __launch_bounds__(GL_THREADS, 3)
grad_scale_kernel(const __grid_constant__ GradTable<CAP> t, const double* __restrict__ partials, int used, int chunk,
                  float max_norm, double* sumsq, float* norm) {
  __shared__ double warp_sums[GL_THREADS / 32];
  const int u0 = (int)(gridDim.x - 1 - blockIdx.x) * chunk;
  int u = min(t.units, u0 + chunk);
  // the tensor with the last unit of the chunk: from the table of starts, a step or two further
  int i = t.first[(int64_t)(u - 1) * t.starts / t.units];
  while (i + 1 < t.count && t.e[i + 1].unit0 < u) ++i;
  pdl_wait();
  pdl_launch();
  const double total = used == 1 ? *partials : sum_partials(partials, used, warp_sums);
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
  const bool nothing = k == 1.0f && k0 == 1.0f;
  while (true) {
    const GradEntry& e = t.e[i];
    const int begin = max(u0, e.unit0);
    if (!(nothing && (e.flags & GL_IN_PLACE))) span_scale<SRC, DST>(e, unit_span(e, begin, u), k0, k);
    u = begin;
    if (u <= u0) break;
    --i;
  }
}

// Calls f(table) for each run of the list that fits one launch; `last_first`: from the end.
template <typename F>
cudaError_t for_tables(const GradList& l, bool last_first, F f) {
  const int runs = (l.count + GL_MAX_TENSORS - 1) / GL_MAX_TENSORS;
  for (int r = 0; r < runs; ++r) {
    const int i0 = (last_first ? runs - 1 - r : r) * GL_MAX_TENSORS;
    const int n = std::min(GL_MAX_TENSORS, l.count - i0);
    const int64_t begin = l.entries[i0].unit0;
    const int64_t end = i0 + n < l.count ? l.entries[i0 + n].unit0 : l.units;
    auto fill = [&](auto& t) {
      t.count = n;
      t.units = (int32_t)(end - begin);
      for (int i = 0; i < n; ++i) {
        t.e[i] = l.entries[i0 + i];
        t.e[i].unit0 -= (int32_t)begin;
      }
      t.starts = std::min(t.units, GL_NORM_BLOCKS);
      for (int b = 0, i = 0; b < t.starts; ++b) {
        const int64_t unit = ((int64_t)t.units * b) / t.starts;
        while (i + 1 < n && t.e[i + 1].unit0 <= unit) ++i;
        t.first[b] = (uint16_t)i;
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

int64_t grad_partials(int64_t count) {
  const int64_t runs = (count + GL_MAX_TENSORS - 1) / GL_MAX_TENSORS;
  return std::max<int64_t>(1, runs) * GL_NORM_BLOCKS;
}

namespace {

template <typename... P, typename... Q>
cudaError_t launch_after(void (*kernel)(P...), int grid, cudaStream_t stream, Q&&... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(GL_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Q>(args)...);
}

template <int CAP>
cudaError_t launch_sumsq(const GradTable<CAP>& t, double* partials, int* grid, cudaStream_t stream) {
  *grid = t.starts;
  return launch_after(grad_sumsq_kernel<CAP>, t.starts, stream, t, partials);
}
template <int CAP>
cudaError_t launch_scale(const GradTable<CAP>& t, const double* partials, int used, float max_norm, double* sumsq,
                         float* norm, cudaStream_t stream) {
  // at most what a block loads at once; a short list is spread over the SMs
  const int chunk = std::max(1, std::min(GL_CHUNK, t.units / GL_NORM_BLOCKS));
  const int grid = (t.units + chunk - 1) / chunk;
  // one pair of types for the whole list, as most lists have it, gets a kernel of its own: a third
  // fewer registers than the one that looks at every tensor's. FP16 to BF16 and back share that one, which
  // costs them nothing that shows: 256 Mi elements take 156 and 157 us, BF16 to BF16 157
  const int src = t.e[0].src_type, dst = t.e[0].dst_type;
  bool same = true;
  for (int i = 1; i < t.count && same; ++i) same = t.e[i].src_type == src && t.e[i].dst_type == dst;
#define GL_CASE(S, D)                                                                                             \
  if (same && src == S && dst == D)                                                                               \
    return launch_after(grad_scale_kernel<CAP, S, D>, grid, stream, t, partials, used, chunk, max_norm, sumsq, norm);
  GL_CASE(PARALIA_F32, PARALIA_F32)
  GL_CASE(PARALIA_F32, PARALIA_F16)
  GL_CASE(PARALIA_F32, PARALIA_BF16)
  GL_CASE(PARALIA_F16, PARALIA_F32)
  GL_CASE(PARALIA_F16, PARALIA_F16)
  GL_CASE(PARALIA_BF16, PARALIA_F32)
  GL_CASE(PARALIA_BF16, PARALIA_BF16)
#undef GL_CASE
  return launch_after(grad_scale_kernel<CAP, -1, -1>, grid, stream, t, partials, used, chunk, max_norm, sumsq, norm);
}

}  // namespace

cudaError_t launch_grad_sumsq(const GradList& l, double* partials, int* used, cudaStream_t stream) {
  *used = 0;
  return for_tables(l, false, [&](auto& t) {
    int grid = 0;
    const cudaError_t e = launch_sumsq(t, partials + *used, &grid, stream);
    *used += grid;
    return e;
  });
}

cudaError_t launch_grad_norm_final(const double* partials, int used, double* sumsq, float* norm, cudaStream_t stream) {
  return launch_after(grad_norm_final_kernel, 1, stream, partials, used, sumsq, norm);
}

cudaError_t launch_grad_scale(const GradList& l, double* partials, int used, float max_norm, double* sumsq,
                              float* norm, cudaStream_t stream) {
  if (l.count == 0) return launch_grad_norm_final(partials, used, sumsq, norm, stream);
  if (used > 1 && l.units > (int64_t)GL_CHUNK * GL_NORM_BLOCKS * 2) {
    // many blocks: the partial sums are added up once and not in each of them
    const cudaError_t e = launch_grad_norm_final(partials, used, partials, norm, stream);
    if (e != cudaSuccess) return e;
    used = 1;
  }
  return for_tables(l, true, [&](auto& t) {
    return launch_scale(t, partials, used, max_norm, sumsq, norm, stream);
  });
}

}  // namespace paralia
