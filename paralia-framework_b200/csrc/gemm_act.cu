// Matrix product with bias, activation and residual in its epilogue, FP16 / BF16:
//   Z = alpha * op(A) op(B) + bias,  pre <- Z,  D <- act(Z) + beta * C,   column-major,
// on the fifth-generation tensor cores, and the elementwise part of its gradient.
//
// The product as the tensor core sees it is acc[r, q] = sum_k X[r, k] Y[q, k]: r runs over the
// lanes of tensor memory (the MMA's M), q over its columns (the MMA's N). QC chooses which
// dimension of D lies on the columns:
//   QC = true   r = column of D, q = row of D: a thread holds a run of one column of D, which is
//               contiguous, and moves it 16 bytes at a time. For D with many rows and columns.
//   QC = false  r = row of D, q = column of D: neighbouring lanes hold neighbouring rows, so every
//               access of a warp is 64 contiguous bytes at any alignment. For few columns (a
//               token or a small batch: the MMA's N is as small as 16) and for unaligned D.
//
// Operand tiles are 64 k deep and come by TMA with 128-byte swizzle, in the storage order the
// operand has (idesc and descriptors tell the tensor core whether k or r / q is contiguous), so
// all four transpose combinations run without a repacking pass:
//   k contiguous        one box of 64 k x rows; eight rows of 128 bytes are one swizzle atom
//                       (stride byte offset 1024), 16 k further is 32 bytes further.
//   r / q contiguous    boxes of 64 rows x 64 k; eight k of 128 bytes are one atom (stride byte
//                       offset 1024), the next 64 rows are 8 KB away (leading byte offset), 16 k
//                       further is 2 KB further.
// TMA fills with zeros outside the matrix, so no size has to be a multiple of anything.
//
// Roles: warp 0 loads, warp 1 issues MMAs, the others are the epilogue, with two accumulators in
// tensor memory so that the epilogue of one tile runs under the MMAs of the next. CG = 2 pairs
// two CTAs on one 256 x BN tile: each loads its half of X and of Y, the leader issues the MMAs
// for both. Every wait is bounded; on a timeout the CTA records an error word, stops issuing
// work and exits.
//
// What bounds it: at large sizes the board's power. 8192^3 BF16 takes 737 us in a burst (1490
// TFLOP/s) and 850 in a loop of a quarter second, in every storage order alike, with the tensor pipe at
// 85 % of the cycles of a clock that has fallen to 1.43 GHz. With few columns HBM: 16384 x 16384 by one
// column 82 us (6.5 TB/s), 16384 x 4096 24 us, of which 3.5 are start and drain. In between the bytes an
// SM gets out of L2, about 66 a clock: 128 x 128 tiles of one CTA take 0.26 us for 64 k, their MMAs 0.14.
//
// Split k: with few tiles, the S CTAs of a cluster take a run of k each, put their FP32
// accumulators into their shared memory and each sums one S-th of the columns over the cluster
// through distributed shared memory, in rank order: one launch, no scratch, the same bits every
// time.
#include "gemm_act.cuh"

#include <algorithm>
#include <atomic>
#include <cstring>
#include <utility>

#include "act_math.cuh"
#include "gemm_act_plan.hpp"
#include "runtime.hpp"
#include "sm100_prims.cuh"

namespace paralia {
using namespace prims;

namespace {

constexpr int GA_MAX_STAGES = 12;
constexpr int GA_X_BYTES = 128 * GA_BK * 2;
constexpr int GA_SMEM = 224 * 1024;       // operand ring and staging buffers
constexpr int GA_SMEM_HALF = 108 * 1024;  // the same where two CTAs share an SM (BN = 64)

// How an operand lies in memory and comes: k contiguous; r / q contiguous, one box for 64 of
// them; r / q contiguous and a multiple of 64 of them, one box for all of a tile (the tensor map
// then has the blocks of 64 as a dimension of its own).
enum : int { GA_K_MAJOR = 0, GA_MN_BOXES = 1, GA_MN_BLOCKS = 2 };

// One product of a launch.
struct GaProb {
  const void* bias;
  const void* C;
  void* D;
  void* pre;
  int64_t ldC, ldD, ldPre;
  int32_t tile0;                 // number of its first tile in the launch
  int32_t M, N;
  int32_t r_tiles, q_tiles;
  int32_t panel;                 // q tiles per panel of the tile numbering
  int32_t kblocks;
  int32_t x_mn, y_mn;            // GA_K_MAJOR, GA_MN_BOXES or GA_MN_BLOCKS
  int32_t tx_bytes;              // what a CTA loads for a stage
  int32_t act, bf16;
  int32_t vec;                   // D, C, pre and bias allow 16-byte accesses along M
  float alpha, beta;
};

struct GaArgs {
  GaProb p[GA_MAX_PROBS];
  int32_t tiles;                 // of all products
  int32_t tiles0;                // of the first
  int32_t bn;                    // columns of a tile: BN, or for BN = 64 any multiple of 16 up to it
  int32_t stages, stage_bytes;   // per CTA
  int32_t split;                 // CTAs that share a tile's k (the cluster, CG == 1)
  int32_t stage_out;             // results leave through shared memory by TMA (QC, no split),
  int32_t out_bytes;             // this much of it for each epilogue warp
  int* status;
};
struct alignas(64) GaMaps {
  CUtensorMap x[GA_MAX_PROBS], y[GA_MAX_PROBS], d[GA_MAX_PROBS], pre;
};

template <int BN>
struct GaShape {
  static constexpr int EPILOGUE_WARPS = BN >= 128 ? 8 : 4;
  static constexpr int THREADS = 64 + 32 * EPILOGUE_WARPS;
};

struct GaCtl {
  uint64_t full[GA_MAX_STAGES];
  uint64_t empty[GA_MAX_STAGES];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int GA_CTL_BYTES = 256;
static_assert(sizeof(GaCtl) <= GA_CTL_BYTES, "control block");

// ------------------------------------------------------------------ instructions
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Programmatic dependent launch: wait until the kernels this one depends on have completed and
// their writes are visible; allow the next kernel to be set up on free resources.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// L2 keeps a line of the streamed operand no longer than it has to: it is read by the CTAs of one
// round of tiles at about the same time, while the panel of the other operand comes again.
__device__ __forceinline__ uint64_t ga_policy_stream() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t ga_policy_normal() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// A bounded wait by a whole warp, with one outcome.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag));
}
// Tiled TMA load without multicast; `bar` is a shared::cluster address. With CG == 2 it may lie in
// the other CTA of the pair.
template <int CG>
__device__ __forceinline__ void ga_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, uint64_t policy, int c0, int c1, int c2 = 0) {
  if (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint "
        "[%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0),
        "r"(c1), "r"(c2), "l"(policy)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0),
        "r"(c1), "r"(c2), "l"(policy)
        : "memory");
}

// Shared-memory operand descriptor with 128-byte swizzle.
__device__ __forceinline__ uint64_t ga_desc(uint32_t saddr, int mn_major) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)(mn_major ? (8192 >> 4) : 1) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

template <int CG>
__device__ __forceinline__ void ga_mma(uint32_t tmem_d, uint64_t xdesc, uint64_t ydesc, uint32_t idesc,
                                       uint32_t accumulate) {
  if (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(xdesc), "l"(ydesc),
        "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(xdesc), "l"(ydesc),
        "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrive at `bar` (in both CTAs of the pair with CG == 2) when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void ga_commit(uint64_t* bar) {
  if (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// TMA store of a 64-column x 32-row box from shared memory, and the waits for it.
__device__ __forceinline__ void ga_store(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1), "r"(0)
               : "memory");
}
__device__ __forceinline__ void ga_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void ga_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void ga_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void st_shared16(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}

__device__ __forceinline__ void ga_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ga_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Sixteen columns of this warp's 32 lanes of tensor memory, on their way; they are there after
// ga_tmem_wait16, which ties the registers to the wait.
__device__ __forceinline__ void ga_tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void ga_tmem_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// ------------------------------------------------------------------ epilogue
// Eight neighbouring rows of one column of D. First Z from sums and bias, then D and Z packed.
template <bool bf>
__device__ __forceinline__ void ga_z8(const GaProb& a, const float* v, const uint4& b, float* z) {
  const uint32_t bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 bb = unpack16(bv[i], bf);
    z[2 * i] = fmaf(a.alpha, v[2 * i], bb.x);
    z[2 * i + 1] = fmaf(a.alpha, v[2 * i + 1], bb.y);
  }
}
template <int ACT, bool bf>
__device__ __forceinline__ void ga_d8(const GaProb& a, const float* z, const uint4& c, uint32_t (&d)[4]) {
  const uint32_t cv[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float d0 = act_value<ACT>(z[2 * i]), d1 = act_value<ACT>(z[2 * i + 1]);
    if (a.C) {
      const float2 cc = unpack16(cv[i], bf);
      d0 = fmaf(a.beta, cc.x, d0);
      d1 = fmaf(a.beta, cc.y, d1);
    }
    d[i] = pack16(d0, d1, bf);
  }
}
template <bool bf>
__device__ __forceinline__ void ga_pack8(const float* z, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = pack16(z[2 * i], z[2 * i + 1], bf);
}
// Eight 16-bit elements of which `valid` exist; the others are 0 and not read.
__device__ __forceinline__ uint4 ga_load_any8(const uint16_t* p, int64_t valid) {
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < valid) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 ga_load8(const void* p, int64_t valid) {   // on a 16-byte boundary
  if (valid >= 8) return *static_cast<const uint4*>(p);
  return ga_load_any8(static_cast<const uint16_t*>(p), valid);
}
__device__ __forceinline__ uint4 ga_load_bias8(const GaProb& a, int64_t m) {
  if (!a.bias || m >= a.M) return make_uint4(0, 0, 0, 0);
  return ga_load8(static_cast<const uint16_t*>(a.bias) + m, a.M - m);
}
__device__ __forceinline__ uint4 ga_load_c8(const GaProb& a, int64_t m, int64_t n) {
  if (!a.C || m >= a.M) return make_uint4(0, 0, 0, 0);
  return ga_load8(static_cast<const uint16_t*>(a.C) + m + n * a.ldC, a.M - m);
}

// Rows m .. m+7 of column n of D (QC): acc -> D, pre.
template <int ACT, bool bf>
__device__ __forceinline__ void ga_finish8(const GaProb& a, int64_t m, int64_t n, float* v) {
  if (a.vec && m + 8 <= a.M) {
    float zf[8];
    uint32_t z[4], d[4];
    ga_z8<bf>(a, v, ga_load_bias8(a, m), zf);
    ga_d8<ACT, bf>(a, zf, ga_load_c8(a, m, n), d);
    ga_pack8<bf>(zf, z);
    if (a.pre) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.pre) + m + n * a.ldPre) = make_uint4(z[0], z[1], z[2], z[3]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.D) + m + n * a.ldD) = make_uint4(d[0], d[1], d[2], d[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (m + i >= a.M) break;
    const float z = fmaf(a.alpha, v[i], a.bias ? load16(a.bias, m + i, bf) : 0.0f);
    if (a.pre) store16(a.pre, m + i + n * a.ldPre, z, bf);
    float d = act_value<ACT>(z);
    if (a.C) d = fmaf(a.beta, load16(a.C, m + i + n * a.ldC, bf), d);
    store16(a.D, m + i + n * a.ldD, d, bf);
  }
}

// W accumulator columns q0 .. q0+W-1 of lane row r.
template <bool QC, int W>
__device__ __forceinline__ void ga_finish(const GaProb& a, int64_t r, int64_t q0, float (&v)[W]) {
  with_act_type(a.act, a.bf16 != 0, [&](auto t, auto y) {
    constexpr int ACT = decltype(t)::value;
    constexpr bool bf = decltype(y)::value != 0;
    if constexpr (QC) {
      if (r >= a.N) return;
#pragma unroll
      for (int g = 0; g < W / 8; ++g)
        if (q0 + 8 * g < a.M) ga_finish8<ACT, bf>(a, q0 + 8 * g, r, &v[8 * g]);
    } else {
      if (r >= a.M) return;
      const float b = a.bias ? load16(a.bias, r, bf) : 0.0f;
      uint16_t c[W];
      if (a.C) {
        // all on their way before the first is used; past the last column the last one again
#pragma unroll
        for (int j = 0; j < W; ++j)
          c[j] = static_cast<const uint16_t*>(a.C)[r + min(q0 + j, (int64_t)a.N - 1) * a.ldC];
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float z = fmaf(a.alpha, v[j], b);
        float d = act_value<ACT>(z);
        if (a.C) d = fmaf(a.beta, load16(&c[j], 0, bf), d);
        if (q0 + j < a.N) {
          if (a.pre) store16(a.pre, r + (q0 + j) * a.ldPre, z, bf);
          store16(a.D, r + (q0 + j) * a.ldD, d, bf);
        }
      }
    }
  });
}

// The first `count` of eight packed elements, one by one.
__device__ __forceinline__ void ga_store_some(uint16_t* p, const uint32_t (&v)[4], int count) {
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < count) p[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
}

// One warp's share of a tile (QC): 32 columns of D, `cols` rows from q on, a multiple of 64. Once Z has
// been made of the sums of 16 rows, the next 16 are fetched under the rest of the work on these. 64
// rows at a time leave through this warp's staging buffer (128-byte lines, swizzled as the tensor map
// says) by TMA: whole lines, edges clipped by the map, the store under the next arithmetic. A TMA store
// writes whole groups of 16 bytes, also where the matrix ends inside one: the map ends with the last whole
// group, and the one to seven rows behind it are stored one by one. The loop
// is not unrolled: with ten variants and eight warps out of step the instruction cache is what an
// unrolled one waits for (8192 x 8192 x 1024 with tanh-GELU: 174 us unrolled by four).
template <int ACT, bool bf>
__device__ __forceinline__ void ga_staged_tile(const GaProb& a, const CUtensorMap* map_d,
                                               const CUtensorMap* map_pre, uint32_t taddr, uint32_t out, int q,
                                               int r_first, int cols, int lane) {
  const uint32_t row = out + lane * 128;
  const int64_t n = min((int64_t)r_first + lane, (int64_t)a.N - 1);   // a column that exists; its copy is cut off
  const int left = a.M - q;
  const int last = left >= cols ? cols : (left + 63) / 64 * 64;        // 64 rows of which none exists are left out
  if (last <= 0) return;
  const int whole = a.M & ~7;                                          // rows that leave by TMA
  const int rest = r_first + lane < a.N ? a.M - whole : 0;             // rows of this lane's column that do not
  uint32_t v[16];
  uint4 c0 = ga_load_c8(a, q, n), c1 = ga_load_c8(a, (int64_t)q + 8, n);
  uint4 b0 = ga_load_bias8(a, q), b1 = ga_load_bias8(a, (int64_t)q + 8);
  ga_tmem_ld16(taddr, v);
#pragma unroll 1
  for (int at = 0; at < last; at += 16) {
    ga_tmem_wait16(v);
    float x[16], z[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = a.kblocks == 0 ? 0.0f : __uint_as_float(v[e]);
    ga_z8<bf>(a, x, b0, z);
    ga_z8<bf>(a, x + 8, b1, z + 8);
    const uint4 cx0 = c0, cx1 = c1;
    if (at + 16 < last) {
      ga_tmem_ld16(taddr + at + 16, v);
      const int64_t m = (int64_t)q + at + 16;
      c0 = ga_load_c8(a, m, n);
      c1 = ga_load_c8(a, m + 8, n);
      b0 = ga_load_bias8(a, m);
      b1 = ga_load_bias8(a, m + 8);
    }
    if ((at & 63) == 0) {
      if (lane == 0) ga_store_wait_read();
      __syncwarp();
    }
    uint32_t o[4];
    const uint32_t to0 = row + (((at & 63) >> 3) ^ (lane & 7)) * 16, to1 = row + ((((at & 63) >> 3) + 1) ^ (lane & 7)) * 16;
    const bool end0 = q + at == whole, end1 = q + at + 8 == whole;
    uint16_t* const tail = static_cast<uint16_t*>(a.D) + whole + n * a.ldD;
    ga_d8<ACT, bf>(a, z, cx0, o);
    st_shared16(to0, o);
    if (end0) ga_store_some(tail, o, rest);
    ga_d8<ACT, bf>(a, z + 8, cx1, o);
    st_shared16(to1, o);
    if (end1) ga_store_some(tail, o, rest);
    if (a.pre) {
      uint16_t* const tail_pre = static_cast<uint16_t*>(a.pre) + whole + n * a.ldPre;
      ga_pack8<bf>(z, o);
      st_shared16(to0 + 4096, o);
      if (end0) ga_store_some(tail_pre, o, rest);
      ga_pack8<bf>(z + 8, o);
      st_shared16(to1 + 4096, o);
      if (end1) ga_store_some(tail_pre, o, rest);
    }
    if ((at & 63) == 48) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0 && r_first < a.N && q + at - 48 < whole) {
        ga_store(map_d, out, q + at - 48, r_first);
        if (a.pre) ga_store(map_pre, out + 4096, q + at - 48, r_first);
        ga_store_commit();
      }
    }
  }
}

// The same for QC == false: row r of D in columns q .. q+cols-1. A warp's access to a column is 64
// contiguous bytes wherever it starts. C of the next 16 columns is fetched with their sums, each address
// computed for itself: a pointer stepped from column to column made the loads wait for one another
// (5003 x 1237 x 1365 with residual: 102 us instead of 47).
template <int ACT, bool bf>
__device__ __forceinline__ void ga_direct_tile(const GaProb& a, uint32_t taddr, int64_t r, int64_t q, int cols) {
  const int last = (int)min((int64_t)cols, a.N - q);
  if (last <= 0) return;
  const bool in = r < a.M;
  const int64_t m = min(r, (int64_t)a.M - 1);
  const float b = a.bias ? load16(a.bias, m, bf) : 0.0f;
  const uint16_t* cp = static_cast<const uint16_t*>(a.C) + m + q * a.ldC;
  uint16_t* dp = static_cast<uint16_t*>(a.D) + m + q * a.ldD;
  uint16_t* pp = static_cast<uint16_t*>(a.pre) + m + q * a.ldPre;
  uint32_t v[16], c[16] = {};
  auto fetch = [&](int at) {
    ga_tmem_ld16(taddr + at, v);
    if (a.C) {
#pragma unroll
      for (int j = 0; j < 16; ++j) c[j] = cp[(int64_t)min(at + j, last - 1) * a.ldC];
    }
  };
  fetch(0);
#pragma unroll 1
  for (int at = 0; at < last; at += 16) {
    ga_tmem_wait16(v);
    float z[16];
    uint32_t cx[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      z[j] = fmaf(a.alpha, a.kblocks == 0 ? 0.0f : __uint_as_float(v[j]), b);
      cx[j] = c[j];
    }
    if (at + 16 < last) fetch(at + 16);
    if (!a.C && !a.pre && at + 16 <= last) {
      // the common case without a question for every element
      uint16_t o[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) store16(&o[j], 0, act_value<ACT>(z[j]), bf);
      if (in) {
#pragma unroll
        for (int j = 0; j < 16; ++j) dp[j * a.ldD] = o[j];
      }
      dp += 16 * a.ldD;
      continue;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float d = act_value<ACT>(z[j]);
      if (a.C) d = fmaf(a.beta, unpack16(cx[j], bf).x, d);
      if (in && at + j < last) {
        store16(dp, 0, d, bf);
        if (a.pre) store16(pp, 0, z[j], bf);
      }
      dp += a.ldD;
      pp += a.ldPre;
    }
  }
}

// Asks L2 for the rows m0 .. m0+rows-1 of the bias and of `cols` columns of C from n0 on. The epilogue's
// own loads come late and few at a time, each with the latency of where the line then is.
template <int THREADS>
__device__ __forceinline__ void ga_prefetch_inputs(const GaProb& a, int64_t m0, int rows, int64_t n0, int cols) {
  const int e = threadIdx.x - 64, lines = (rows + 63) / 64;
  if (a.bias && e < lines && m0 + e * 64 < a.M)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint16_t*>(a.bias) + m0 + e * 64));
  if (!a.C) return;
  for (int i = e; i < lines * cols; i += THREADS) {
    const int64_t m = m0 + (i % lines) * 64, n = n0 + i / lines;
    if (m < a.M && n < a.N)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint16_t*>(a.C) + m + n * a.ldC));
  }
}

// ------------------------------------------------------------------ kernel
struct GaTile {
  int rt, qt;
};
// Tiles are numbered in panels of a few q tiles, inside a panel along q first: what runs at
// one time then shares few X and few Y tiles, which cuts what is pulled through L2.
__device__ __forceinline__ GaTile ga_tile(const GaProb& a, int tile) {
  const uint32_t per_panel = (uint32_t)a.r_tiles * (uint32_t)a.panel;
  const uint32_t number = (uint32_t)(tile - a.tile0), panel = number / per_panel, rest = number - panel * per_panel;
  const uint32_t width = min((uint32_t)a.panel, (uint32_t)a.q_tiles - panel * (uint32_t)a.panel);
  GaTile t;
  t.rt = (int)(rest / width);
  t.qt = (int)(panel * (uint32_t)a.panel + rest - (uint32_t)t.rt * width);
  return t;
}

// The tile of place `place` in the round that starts at tile `base`. The last, incomplete round is dealt
// out from the other end: of two products the one with more k comes first, so that the places at
// the end have had less to do.
__device__ __forceinline__ int ga_number(int base, int place, int step, int tiles) {
  return base + (base + step > tiles ? step - 1 - place : place);
}

// TWO: the launch has two products. With one its description is read from constant addresses.
template <int BN, int CG, bool QC, bool TWO>
__global__ void __launch_bounds__(GaShape<BN>::THREADS, BN == 64 ? 2 : 1)
gemm_act_kernel(const __grid_constant__ GaMaps maps, const __grid_constant__ GaArgs g) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ GaCtl ctl_mem;
  GaCtl* ctl = &ctl_mem;
  volatile int* abort_flag = &ctl->abort_flag;
  constexpr int EW = GaShape<BN>::EPILOGUE_WARPS;
  constexpr int YROWS = BN / CG;                       // rows of Y this CTA loads
  constexpr uint32_t TMEM_COLS = 2 * BN;
  const int bn = BN == 64 && !QC ? g.bn : BN;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = (CG == 2 || g.split > 1) ? cluster_rank() : 0;
  const int split = CG == 1 ? g.split : 1;
  const int group = CG * split;                        // CTAs that share a tile
  const int place = blockIdx.x / group, tile_step = gridDim.x / group;
  const int first_tile = ga_number(0, place, tile_step, g.tiles);
  // this CTA's run of a product's k blocks
  auto k_begin = [&](const GaProb& a) { return split > 1 ? (int)((int64_t)a.kblocks * rank / split) : 0; };
  auto k_end = [&](const GaProb& a) { return split > 1 ? (int)((int64_t)a.kblocks * (rank + 1) / split) : a.kblocks; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ctl->acc_full[b], 1);
      mbar_init(&ctl->acc_empty[b], EW * CG);
    }
    ctl->abort_flag = 0;
    ctl->tmem_base = 0;
    mbar_fence_init();
    if (g.p[0].kblocks > 0) {
      prefetch_tensormap(&maps.x[0]);
      prefetch_tensormap(&maps.y[0]);
    }
  }
  __syncthreads();
  if (warp == 1) {
    if (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)),
                   "r"(TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)),
                   "r"(TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  ga_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();     // the other CTA's barriers are initialised, its columns allocated
  ga_fence_after();
  const uint32_t tmem_base = ctl->tmem_base;
  // Everything above may run while the kernel before this one in the stream still does; nothing
  // below may, operands, results and the status word being global memory.
  pdl_wait();
  pdl_launch();

  // The two issuing warps run their loops whole and elect a lane for the instructions that one
  // thread has to issue: inside a branch on the lane number the compiler cannot keep descriptors
  // and addresses in uniform registers, and the four MMAs of a stage then took 350 clocks to issue.
  if (warp == 0) {
    // ------------------------------ producer ------------------------------
    const uint64_t pol_x = ga_policy_stream(), pol_y = ga_policy_normal();
    int s = 0, filled = 0;           // stage, and how many stages have been filled at all (capped)
    uint32_t phase = 0;              // parity of the ring's round
    bool ok = true;
    for (int base = 0, tile; ok && (tile = ga_number(base, place, tile_step, g.tiles)) < g.tiles; base += tile_step) {
      const int which = TWO && tile >= g.tiles0 ? 1 : 0;
      const GaProb& a = g.p[which];
      const CUtensorMap *map_x = &maps.x[which], *map_y = &maps.y[which];
      const int kb0 = k_begin(a), kb1 = k_end(a);
      // how far one k block moves the first two coordinates of a box
      const int xk0 = a.x_mn ? 0 : GA_BK, xk1 = a.x_mn ? GA_BK : 0;
      const int yk0 = a.y_mn ? 0 : GA_BK, yk1 = a.y_mn ? GA_BK : 0;
      const bool x_boxes = a.x_mn == GA_MN_BOXES, y_boxes = a.y_mn == GA_MN_BOXES;
      const uint32_t tx = a.tx_bytes * CG;
      const GaTile t = ga_tile(a, tile);
      const int r0 = t.rt * (128 * CG) + (CG == 2 ? (int)rank * 128 : 0);
      const int q0 = t.qt * bn + (CG == 2 ? (int)rank * YROWS : 0);
      int x0 = a.x_mn == GA_MN_BOXES ? r0 : a.x_mn ? 0 : kb0 * GA_BK, x1 = a.x_mn ? kb0 * GA_BK : r0;
      int y0 = a.y_mn == GA_MN_BOXES ? q0 : a.y_mn ? 0 : kb0 * GA_BK, y1 = a.y_mn ? kb0 * GA_BK : q0;
      const int x2 = a.x_mn == GA_MN_BLOCKS ? r0 / 64 : 0, y2 = a.y_mn == GA_MN_BLOCKS ? q0 / 64 : 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (filled == g.stages && !warp_wait(&ctl->empty[s], phase ^ 1u, abort_flag)) {
          if (!*abort_flag) { *abort_flag = 1; atomicExch(g.status, KERR_EMPTY_WAIT_TIMEOUT); }
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t x = smem_u32(smem) + s * g.stage_bytes, y = x + GA_X_BYTES;
          uint32_t bar = smem_u32(&ctl->full[s]);
          if (CG == 2) bar = map_rank(bar, 0);
          if (CG == 1 || rank == 0) mbar_expect_tx(&ctl->full[s], tx);
          ga_load<CG>(x, map_x, bar, pol_x, x0, x1, x2);
          if (x_boxes) ga_load<CG>(x + 8192, map_x, bar, pol_x, x0 + 64, x1, 0);
          ga_load<CG>(y, map_y, bar, pol_y, y0, y1, y2);
          if (y_boxes) {
#pragma unroll
            for (int j = 1; j < YROWS / 64; ++j) ga_load<CG>(y + j * 8192, map_y, bar, pol_y, y0 + j * 64, y1, 0);
          }
        }
        x0 += xk0; x1 += xk1; y0 += yk0; y1 += yk1;
        if (filled < g.stages) ++filled;
        if (++s == g.stages) { s = 0; phase ^= 1u; }
      }
    }
    // Before shared memory is given up: every stage has been read by its MMAs (with CG == 2 the
    // leader's commits arrive here too, so none may still be on its way), or, after an abort,
    // every copy has landed.
    for (int j = 0; j < filled; ++j) {
      // the oldest stage first; `s` and `phase` are those of the next fill
      int zero = 0;
      const int q = filled < g.stages ? j : (s + j < g.stages ? s + j : s + j - g.stages);
      const uint32_t parity = filled < g.stages || q < s ? phase : phase ^ 1u;
      const bool clean = __all_sync(0xffffffffu, ok && !*abort_flag);
      if (CG == 2 && rank != 0 && !clean) break;   // its copies signal the leader
      if (!warp_wait(clean ? &ctl->empty[q] : &ctl->full[q], parity, &zero)) {
        *abort_flag = 1;
        atomicExch(g.status, KERR_DRAIN_TIMEOUT);
        break;
      }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer ------------------------------
    if (CG == 1 || rank == 0) {
      int s = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int base = 0, tile; ok && (tile = ga_number(base, place, tile_step, g.tiles)) < g.tiles; base += tile_step, ++local) {
        const int buf = local & 1;
        if (local >= 2 && !warp_wait(&ctl->acc_empty[buf], (uint32_t)(((local >> 1) - 1) & 1), abort_flag)) {
          if (!*abort_flag) { *abort_flag = 1; atomicExch(g.status, KERR_TMEM_WAIT_TIMEOUT); }
          ok = false;
          break;
        }
        const GaProb& a = g.p[TWO && tile >= g.tiles0 ? 1 : 0];
        const int kb0 = k_begin(a), kb1 = k_end(a);
        const uint32_t fmt = a.bf16 ? 1u : 0u;
        const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (a.x_mn ? 1u << 15 : 0u) | (a.y_mn ? 1u << 16 : 0u) |
                               ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
        const uint32_t x_step = a.x_mn ? (2048 >> 4) : (32 >> 4), y_step = a.y_mn ? (2048 >> 4) : (32 >> 4);
        const uint64_t x_desc = ga_desc(smem_u32(smem), a.x_mn), y_desc = ga_desc(smem_u32(smem) + GA_X_BYTES, a.y_mn);
        ga_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(buf * BN);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!warp_wait(&ctl->full[s], phase, abort_flag)) {
            if (!*abort_flag) { *abort_flag = 1; atomicExch(g.status, KERR_FULL_WAIT_TIMEOUT); }
            ok = false;
            break;
          }
          ga_fence_after();
          if (elect_one()) {
            const uint64_t dx = x_desc + (uint32_t)(s * (g.stage_bytes >> 4)), dy = y_desc + (uint32_t)(s * (g.stage_bytes >> 4));
#pragma unroll
            for (int j = 0; j < GA_BK / 16; ++j)
              ga_mma<CG>(d, dx + j * x_step, dy + j * y_step, idesc, (kb > kb0 || j > 0) ? 1u : 0u);
            ga_commit<CG>(&ctl->empty[s]);
          }
          __syncwarp();
          if (++s == g.stages) { s = 0; phase ^= 1u; }
        }
        if (ok && elect_one()) ga_commit<CG>(&ctl->acc_full[buf]);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------ epilogue ------------------------------
    const int quad = warp & 3, part = (warp - 2) >> 2;   // lanes of tensor memory; share of the columns
    const int part_cols = bn / (EW / 4);
    int local = 0;
    bool ok = true;
    for (int base = 0, tile; ok && (tile = ga_number(base, place, tile_step, g.tiles)) < g.tiles; base += tile_step, ++local) {
      const int buf = local & 1;
      const int which = TWO && tile >= g.tiles0 ? 1 : 0;
      const GaProb& a = g.p[which];
      const GaTile t = ga_tile(a, tile);
      {
        // what the epilogue will read, into L2 while the product runs
        const int q_cols = bn / split;
        const int64_t r_first = (int64_t)t.rt * (128 * CG) + (CG == 2 ? (int)rank * 128 : 0);
        const int64_t q_first = (int64_t)t.qt * bn + (split > 1 ? (int)rank * q_cols : 0);
        ga_prefetch_inputs<EW * 32>(a, QC ? q_first : r_first, QC ? q_cols : 128, QC ? r_first : q_first,
                                    QC ? 128 : q_cols);
      }
      // every k block of the tile comes before it: 4096 clocks for each on top, three times what one
      // takes where all SMs wait for HBM
      if (!mbar_wait_bounded(&ctl->acc_full[buf], (uint32_t)((local >> 1) & 1), abort_flag,
                             WAIT_BUDGET_CLOCKS + (long long)a.kblocks * 4096)) {
        if (!*abort_flag) { *abort_flag = 1; atomicExch(g.status, KERR_TMEM_WAIT_TIMEOUT); }
        ok = false;
        break;
      }
      ga_fence_after();
      const int64_t r = (int64_t)t.rt * (128 * CG) + (CG == 2 ? (int)rank * 128 : 0) + quad * 32 + lane;
      const int64_t q = (int64_t)t.qt * bn + part * part_cols;
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + part * part_cols);
      if constexpr (QC) {
        if (g.stage_out) {
          const uint32_t out = smem_u32(smem) + g.stages * g.stage_bytes + (warp - 2) * g.out_bytes;
          const int r_first = t.rt * (128 * CG) + (CG == 2 ? (int)rank * 128 : 0) + quad * 32;
          with_act_type(a.act, a.bf16 != 0, [&](auto k, auto y) {
            ga_staged_tile<decltype(k)::value, decltype(y)::value != 0>(a, &maps.d[which], &maps.pre, taddr, out, (int)q, r_first,
                                                                        part_cols, lane);
          });
        }
      }
      if (split > 1) {
#pragma unroll 1
        for (int c = 0; c < part_cols; c += 16) {
          uint32_t v[16];
          ga_tmem_ld16(taddr + c, v);
          ga_tmem_wait16(v);
          // column-major FP32 in the operand ring, which nothing reads any more
          float* stage = reinterpret_cast<float*>(smem) + (part * part_cols + c) * 128 + quad * 32 + lane;
#pragma unroll
          for (int j = 0; j < 16; ++j) stage[j * 128] = __uint_as_float(v[j]);
        }
      } else if constexpr (!QC) {
        with_act_type(a.act, a.bf16 != 0, [&](auto k, auto y) {
          ga_direct_tile<decltype(k)::value, decltype(y)::value != 0>(a, taddr, r, q, part_cols);
        });
      }
      ga_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) arrive_cluster(map_rank(smem_u32(&ctl->acc_empty[buf]), 0));
        else mbar_arrive(&ctl->acc_empty[buf]);
      }
    }
    if (QC && lane == 0) ga_store_wait();
  }

  if (CG == 1 && split > 1) {
    // ------------------------------ sum over the cluster ------------------------------
    __syncwarp();
    cluster_sync();
    if (warp >= 2) {
      // A warp sums one column of this CTA's share at a time, a lane four rows of it: 512 contiguous
      // bytes from each CTA. The sums replace this CTA's own share, which nobody else reads.
      const int cols = bn / split;                    // columns of this CTA
      const GaProb& a = g.p[TWO && first_tile >= g.tiles0 ? 1 : 0];
      const GaTile t = ga_tile(a, first_tile);
      float* own = reinterpret_cast<float*>(smem) + (int)rank * cols * 128;
      // columns that exist (QC: all, the others are cut off later)
      const int used = QC ? cols : (int)min((int64_t)cols, max((int64_t)0, a.N - ((int64_t)t.qt * bn + rank * cols)));
      for (int c = warp - 2; c < used; c += EW) {
        const uint32_t at = smem_u32(own + c * 128 + lane * 4);
        float4 p[8];
#pragma unroll
        for (int s = 0; s < 8; ++s)
          if (s < split) p[s] = ld_cluster(map_rank(at, s));
        float4 v = p[0];
#pragma unroll
        for (int s = 1; s < 8; ++s)
          if (s < split) { v.x += p[s].x; v.y += p[s].y; v.z += p[s].z; v.w += p[s].w; }
        *reinterpret_cast<float4*>(own + c * 128 + lane * 4) = v;
      }
      named_bar_sync(1, EW * 32);
      const int row = (threadIdx.x - 64) & 127, part = (threadIdx.x - 64) >> 7;
      constexpr int W = QC ? 8 : 2;
      for (int c = part * W; c < used; c += W * (EW / 4)) {
        float v[W];
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = own[(c + j) * 128 + row];
        ga_finish<QC, W>(a, (int64_t)t.rt * 128 + row, (int64_t)t.qt * bn + (int)rank * cols + c, v);
      }
    }
    __syncwarp();
    cluster_sync();      // nobody leaves while its shared memory is still read
  }

  // ------------------------------ teardown ------------------------------
  ga_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  if (warp == 1) {
    if (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ------------------------------------------------------------------ copy to an aligned layout
// A len x cols matrix at any 2-byte address and leading dimension, copied to a buffer whose columns
// start on 16-byte boundaries or better, so that TMA can read it, and fast; up to two matrices in a launch.
// A thread makes one aligned group of eight from the two aligned 16-byte words that it straddles, shifted
// together, so both sides move at full width. Bound by HBM: two matrices of 8192 x 8200 take 93 to 100 us, 5.6
// TB/s; 5003 columns of 1365 and 1237 of 1365 take 10 from cold. Two groups of a thread in flight change
// nothing, four take 105 us; columns worked on to the end of their padding cost a quarter more.
struct AlignCopy {
  const uint16_t* src;
  uint16_t* dst;
  int64_t ld_src, ld_dst, len, cols;
};
struct AlignCopies {
  AlignCopy m[2];
  int64_t groups[2];   // of eight elements, in a matrix
};

__global__ void __launch_bounds__(256) align_copy_kernel(const __grid_constant__ AlignCopies c) {
  pdl_wait();
  pdl_launch();
  const int64_t total = c.groups[0] + c.groups[1];
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const bool second = i >= c.groups[0];
    const AlignCopy& m = c.m[second ? 1 : 0];
    const int64_t j = second ? i - c.groups[0] : i;
    const uint32_t groups = (uint32_t)((m.len + 7) >> 3);
    const int64_t col = j < INT32_MAX ? (int64_t)((uint32_t)j / groups) : j / groups;
    const int64_t at = (j - col * groups) * 8;
    const uint16_t* s = m.src + col * m.ld_src + at;
    const int shift = (int)(reinterpret_cast<uintptr_t>(s) & 15) * 8;   // bits
    // words inside the matrix; what they hold of a neighbouring column, or of the gap to it, ends up
    // behind the copied column, where nobody reads
    const int64_t left = col + 1 < m.cols ? m.ld_src + m.len - at : m.len - at;
    uint4 o;
    if (shift == 0 ? left >= 8 : at + col * m.ld_src >= 8 && left >= 16) {
      const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(s) & ~uintptr_t(15));
      const uint4 lo = p[0], hi = shift == 0 ? lo : p[1];
      const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const int word = shift >> 5, bits = shift & 31;
      uint32_t q[5];
#pragma unroll
      for (int k = 0; k < 5; ++k)
        q[k] = word == 0 ? w[k] : word == 1 ? w[k + 1] : word == 2 ? w[k + 2] : w[k + 3 < 8 ? k + 3 : 7];
      o.x = __funnelshift_r(q[0], q[1], bits);
      o.y = __funnelshift_r(q[1], q[2], bits);
      o.z = __funnelshift_r(q[2], q[3], bits);
      o.w = __funnelshift_r(q[3], q[4], bits);
    } else {
      o = ga_load_any8(s, m.len - at);
    }
    *reinterpret_cast<uint4*>(m.dst + col * m.ld_dst + at) = o;
  }
}

// ------------------------------------------------------------------ gradient of the epilogue
constexpr int AG_ROWS = 64;      // rows of a block: eight lanes x 8
constexpr int AG_WARPS = 8;
constexpr int AG_COLS = 4 * AG_WARPS;   // columns that a block works on at a time
constexpr int AG_U = 2;          // columns in flight per thread

// The `parts` blocks of a cluster take AG_ROWS rows, each a run of the columns; eight lanes hold a column's
// rows, eight each, a warp four columns and then every AG_COLS-th one, so the row sums of the bias
// gradient stay in registers. The sums of the lanes meet by shuffles, those of the warps in shared memory
// in warp order, those of the blocks through distributed shared memory in rank order: one launch, no
// scratch, the same bits every time (a second kernel that added up to 99 partial sums a row took 11 us
// beside 12 of this one).
//
// Bound by memory: two reads and one write of two bytes per entry. VEC: rows come and go as 16-byte
// accesses (eight rows of a lane are neighbours), AG_U columns of a lane in flight; otherwise a lane
// holds two rows 32 apart and every access is of one element, coalesced over the warp at any alignment.
// 16384 x 8192 BF16: 145 us, 5.6 TB/s (157 us with four columns in flight, 172 with rows of 256 a block
// and partial sums in memory).
template <bool VEC>
__global__ void __launch_bounds__(AG_WARPS * 32) act_grad_kernel(const __grid_constant__ ActGradProblem p, int parts) {
  __shared__ float sums[AG_WARPS][AG_ROWS];
  __shared__ float total[AG_ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = blockIdx.x % parts;
  const int64_t row0 = (int64_t)(blockIdx.x / parts) * AG_ROWS;
  const int n_begin = (int)((int64_t)p.N * part / parts), n_end = (int)((int64_t)p.N * (part + 1) / parts);
  float acc[8] = {};
  pdl_wait();
  pdl_launch();
  with_act_type(p.act, p.bf16 != 0, [&](auto a, auto y) {
    constexpr int ACT = decltype(a)::value;
    constexpr bool bf = decltype(y)::value != 0;
    const uint16_t* dd = static_cast<const uint16_t*>(p.dD);
    const uint16_t* pre = static_cast<const uint16_t*>(p.pre);
    uint16_t* dz = static_cast<uint16_t*>(p.dZ);
    // a select for relu, so that an infinite dD in a place that it has closed gives 0
    auto value = [&](float g, float q) { return ACT == PARALIA_ACT_RELU ? (q > 0.0f ? g : 0.0f) : g * act_slope<ACT>(q); };
    const int64_t m = row0 + (lane & 7) * 8;
    const int first = n_begin + warp * 4 + (lane >> 3);
    if (VEC && m + 8 <= p.M) {
      auto finish = [&](int n, const uint4& d, const uint4& z) {
        const uint32_t dv[4] = {d.x, d.y, d.z, d.w}, zv[4] = {z.x, z.y, z.z, z.w};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 g = unpack16(dv[i], bf), q = unpack16(zv[i], bf);
          const float g0 = value(g.x, q.x), g1 = value(g.y, q.y);
          acc[2 * i] += g0;
          acc[2 * i + 1] += g1;
          o[i] = pack16(g0, g1, bf);
        }
        if (dz) *reinterpret_cast<uint4*>(dz + m + n * p.ldZ) = make_uint4(o[0], o[1], o[2], o[3]);
      };
      for (int n = first; n < n_end; n += AG_U * AG_COLS) {
        uint4 d[AG_U], z[AG_U];
#pragma unroll
        for (int u = 0; u < AG_U; ++u) {
          const int64_t c = min(n + u * AG_COLS, n_end - 1);   // past the end the last column again
          d[u] = *reinterpret_cast<const uint4*>(dd + m + c * p.ldD);
          z[u] = ACT != PARALIA_ACT_NONE ? *reinterpret_cast<const uint4*>(pre + m + c * p.ldPre) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < AG_U; ++u)
          if (n + u * AG_COLS < n_end) finish(n + u * AG_COLS, d[u], z[u]);
      }
    } else {
      for (int n = VEC ? first : n_begin + warp; n < n_end; n += VEC ? AG_COLS : AG_WARPS) {
#pragma unroll
        for (int i = 0; i < (VEC ? 8 : 2); ++i) {
          const int64_t r = VEC ? m + i : row0 + lane + 32 * i;
          if (r >= p.M) continue;
          const float v = value(load16(dd, r + n * p.ldD, bf), ACT != PARALIA_ACT_NONE ? load16(pre, r + n * p.ldPre, bf) : 0.0f);
          acc[i] += v;
          if (dz) store16(dz, r + n * p.ldZ, v, bf);
        }
      }
    }
  });
  if (!p.dbias) return;
  if (VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 8);
      acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 16);
      if (lane < 8) sums[warp][lane * 8 + i] = acc[i];
    }
  } else {
    sums[warp][lane] = acc[0];
    sums[warp][lane + 32] = acc[1];
  }
  __syncthreads();
  if (threadIdx.x < AG_ROWS) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < AG_WARPS; ++w) s += sums[w][threadIdx.x];
    total[threadIdx.x] = s;
  }
  if (parts > 1) cluster_sync();
  else __syncthreads();
  const int rows = AG_ROWS / parts;      // rows that this block finishes
  const int64_t row = row0 + part * rows + threadIdx.x;
  if ((int)threadIdx.x < rows && row < p.M) {
    const uint32_t at = smem_u32(&total[part * rows + threadIdx.x]);
    float t = 0.0f;
    for (int b = 0; b < parts; ++b) {
      float x;
      if (parts > 1) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(map_rank(at, b)) : "memory");
      else x = total[part * rows + threadIdx.x];
      t += x;
    }
    if (p.beta_bias != 0.0f) t = fmaf(p.beta_bias, load16(p.dbias, row, p.bf16 != 0), t);
    store16(p.dbias, row, t, p.bf16 != 0);
  }
  if (parts > 1) cluster_sync();         // nobody leaves while its sums are still read
}

inline bool vec16(const void* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld & 7) == 0;
}

}  // namespace

// ------------------------------------------------------------------ launches
namespace {

// Launch with programmatic stream serialization (the kernel waits with pdl_wait before it touches
// global memory), in clusters of `cluster` blocks.
template <typename... P, typename... Q>
cudaError_t launch_dependent(void (*kernel)(P...), int grid, int threads, int smem, int cluster, cudaStream_t stream,
                             Q&&... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Q>(args)...);
}

std::atomic<unsigned> ga_generation{1};

template <int BN, int CG, bool QC, bool TWO>
cudaError_t ga_launch(const GaMaps& maps, GaArgs& g, int count, cudaStream_t stream) {
  constexpr int YROWS = BN / CG;
  g.stage_bytes = 0;
  g.out_bytes = 0;
  for (int i = 0; i < count; ++i) {
    g.p[i].tx_bytes = GA_X_BYTES + (g.p[i].y_mn || BN != 64 ? YROWS : g.bn) * 128;
    g.stage_bytes = std::max(g.stage_bytes, g.p[i].tx_bytes);
    if (g.stage_out) g.out_bytes = std::max(g.out_bytes, g.p[i].pre ? 8192 : 4096);
  }
  const int staging = GaShape<BN>::EPILOGUE_WARPS * g.out_bytes;
  const int budget = (BN == 64 ? GA_SMEM_HALF : GA_SMEM) - staging;
  g.stages = std::min(GA_MAX_STAGES, budget / g.stage_bytes);
  int smem = g.stages * g.stage_bytes + staging;
  if (g.split > 1) smem = std::max(smem, BN * 128 * 4);
  smem += 1024;
  auto kernel = gemm_act_kernel<BN, CG, QC, TWO>;
  // once per GPU, and again after the library has been shut down
  static std::atomic<unsigned> configured[PARALIA_MAX_UNITS] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned now = ga_generation;
  if (configured[dev] != now) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GA_SMEM + 1024);
    if (e != cudaSuccess) return e;
    configured[dev] = now;
  }
  const int group = CG * g.split;
  int64_t grid = (int64_t)g.tiles * group;
  if (g.split == 1) grid = std::min<int64_t>(grid, (BN == 64 ? 2 * GA_SMS : GA_SMS) / CG * CG);
  return launch_dependent(kernel, (int)grid, GaShape<BN>::THREADS, smem, group, stream, maps, g);
}

// Whether TMA can read a stored operand of `cols` columns in place.
bool ga_in_place(const void* p, int64_t ld, int64_t cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (cols <= 1 || (ld & 7) == 0);
}

}  // namespace

void gemm_act_forget_configuration() { ++ga_generation; }

int64_t gemm_act_copy_ld(int64_t rows) {
  const int64_t q = rows < 64 ? 8 : rows < 512 ? 16 : 64;
  return (rows + q - 1) / q * q;
}

int64_t gemm_act_copy_bytes(int64_t rows, int64_t cols) {
  return (gemm_act_copy_ld(rows) * cols * 2 + 255) / 256 * 256;
}

// Columns that do not start on 32-byte sectors cost TMA five sectors and two lines for every 128 bytes:
// 8192 x 8192 by k = 8200 takes 1161 us in place and 809 with copies (703 by k = 8192), 4096 x 4096 by 4104
// 191 and 133, 8192 x 4096 by 1032 81 and 66; about 50 us for a GB that the SMs load. An element is
// loaded once for 256 rows or columns of the result; the copy writes and reads it, 310 us for a GB, and
// has to be waited for: small ones lose (4096 x 656 by 9320 53 us in place, 56 with B copied).
GemmActCopy gemm_act_operand_copy(const void* p, int64_t ld, int64_t rows, int64_t cols, int64_t reuse) {
  if (rows <= 0 || cols <= 0) return GA_COPY_NONE;
  if (!ga_in_place(p, ld, cols)) return GA_COPY_NEEDED;
  const bool sectors = (reinterpret_cast<uintptr_t>(p) & 31) == 0 && (cols <= 1 || (ld & 15) == 0);
  const double gain = 50.0 * ((reuse + 255) / 256) - 310.0;   // us for a GB of operand
  return !sectors && gain * (2e-9 * (double)rows * (double)cols) > 7.0 ? GA_COPY_PAYS : GA_COPY_NONE;
}

namespace {

// One launch of one or two products by plan v; their operands are where TMA can read them.
int ga_launch_products(const GemmActProblem* ps, int n, const GaPlan& v, bool vec, int* status, cudaStream_t stream) {
  GaArgs g;
  GaMaps maps;
  memset(&g, 0, sizeof(g));
  memset(&maps, 0, sizeof(maps));
  g.bn = v.bn;
  g.split = v.split;
  g.status = status;
  g.stage_out = v.qc && v.split == 1;
  int64_t tiles = 0;
  for (int i = 0; i < n; ++i) {
    const GemmActProblem& p = ps[i];
    GaProb& a = g.p[i];
    a.bias = p.bias; a.C = p.C; a.D = p.D; a.pre = p.pre;
    a.ldC = p.ldC; a.ldD = p.ldD; a.ldPre = p.ldPre;
    a.M = p.M; a.N = p.N;
    a.act = p.act; a.bf16 = p.bf16; a.alpha = p.alpha; a.beta = p.beta;
    a.vec = vec;
    a.kblocks = (int32_t)ga_kblocks(p.K);
    a.tile0 = (int32_t)tiles;
    const int64_t R = v.qc ? p.N : p.M, Q = v.qc ? p.M : p.N;
    const int64_t r_tiles = (R + 128 * v.cg - 1) / (128 * v.cg), q_tiles = (Q + v.bn - 1) / v.bn;
    a.r_tiles = (int32_t)r_tiles;
    a.q_tiles = (int32_t)q_tiles;
    tiles += r_tiles * q_tiles;
    // A panel's share of Y is what L2 is to hold on to while X streams past: about 32 MB. At
    // 8192^3 8 tiles of 256 rows are 850 us, 4 or 16 of them 880; at k = 4096 16 are 850 and 8 865.
    a.panel = (int32_t)std::min<int64_t>(16, std::max<int64_t>(4, (32 << 20) / ((int64_t)v.bn * std::max(p.K, 1) * 2)));
    // op(A) is stored with k contiguous if it is a transpose, op(B) if it is not
    const bool a_k = p.ta != 0, b_k = p.tb == 0;
    const int yrows = v.bn / v.cg, xrows = 128;
    // `inner` x `outer` as stored; `k_major`: inner is k
    auto operand = [&](CUtensorMap* map, const void* q, int64_t ld, int64_t inner, int64_t outer, bool k_major, int rows,
                       int32_t* how) -> int {
      *how = k_major ? GA_K_MAJOR : inner % 64 == 0 && rows >= 64 ? GA_MN_BLOCKS : GA_MN_BOXES;
      if (p.K == 0) return PARALIA_OK;
      if (*how == GA_MN_BLOCKS)
        return make_tensor_map(map, q, 2, 64, outer, inner / 64, ld * 2, 128, 64, 64, rows / 64);
      return make_tensor_map(map, q, 2, inner, outer, 1, ld * 2, (uint64_t)ld * outer * 2, 64, k_major ? rows : 64);
    };
    PL_TRY(operand(v.qc ? &maps.y[i] : &maps.x[i], p.A, p.ldA, p.ta ? p.K : p.M, p.ta ? p.M : p.K, a_k,
                   v.qc ? yrows : xrows, v.qc ? &a.y_mn : &a.x_mn));
    PL_TRY(operand(v.qc ? &maps.x[i] : &maps.y[i], p.B, p.ldB, p.tb ? p.N : p.K, p.tb ? p.K : p.N, b_k,
                   v.qc ? xrows : yrows, v.qc ? &a.x_mn : &a.y_mn));
    if (g.stage_out && p.M >= 8) {
      // whole groups of eight rows; the kernel stores what is behind them
      // (the leading dimension of a single column has no meaning and any value)
      const int64_t ld1 = ((int64_t)p.M + 7) / 8 * 8, ldD = p.N > 1 ? p.ldD : ld1, ldPre = p.N > 1 ? p.ldPre : ld1;
      const uint64_t whole = p.M & ~7;
      PL_TRY(make_tensor_map(&maps.d[i], p.D, 2, whole, p.N, 1, ldD * 2, (uint64_t)ldD * p.N * 2, 64, 32));
      if (p.pre) PL_TRY(make_tensor_map(&maps.pre, p.pre, 2, whole, p.N, 1, ldPre * 2, (uint64_t)ldPre * p.N * 2, 64, 32));
    }
    if (i == 0) g.tiles0 = (int32_t)tiles;
  }
  g.tiles = (int32_t)tiles;
  cudaError_t e = cudaErrorInvalidValue;
#define GA_CASE(BN, CG, QC) \
  if ((BN == 64 ? v.bn <= 64 : v.bn == BN) && v.cg == CG && v.qc == QC)                                     \
    e = n == 2 ? ga_launch<BN, CG, QC, true>(maps, g, n, stream) : ga_launch<BN, CG, QC, false>(maps, g, n, stream);
  GA_CASE(64, 1, false)
  GA_CASE(128, 1, false)
  GA_CASE(256, 2, false)
  GA_CASE(64, 1, true)
  GA_CASE(128, 1, true)
  GA_CASE(256, 2, true)
#undef GA_CASE
  PL_CUDA(e);
  return PARALIA_OK;
}

}  // namespace

int launch_gemm_act(const GemmActProblem* problems, int count, void* scratch, int* status, cudaStream_t stream) {
  GemmActProblem ps[GA_MAX_PROBS];
  int n = 0;
  for (int i = 0; i < count; ++i)
    if (problems[i].M > 0 && problems[i].N > 0) ps[n++] = problems[i];
  if (n == 0) return PARALIA_OK;
  if (n == 2 && ps[1].K > ps[0].K && !ps[0].pre) std::swap(ps[0], ps[1]);

  // operands that TMA cannot address where they are
  AlignCopies copies;
  memset(&copies, 0, sizeof(copies));
  int copied = 0;
  char* room = static_cast<char*>(scratch);
  auto in_reach = [&](const void*& q, int64_t& ld, int64_t rows, int64_t cols, bool copy) {
    const int64_t ld_copy = gemm_act_copy_ld(rows);
    if (copy) {
      copies.m[copied] = {static_cast<const uint16_t*>(q), reinterpret_cast<uint16_t*>(room), ld, ld_copy, rows, cols};
      copies.groups[copied++] = (rows + 7) / 8 * cols;
      q = room;
      room += gemm_act_copy_bytes(rows, cols);
      ld = ld_copy;
    } else if (cols <= 1) {
      ld = ld_copy;   // of no meaning, but TMA wants a multiple of 16 bytes
    }
  };
  // Results leave as 16-byte groups only if everything that is read or written beside them can: D, C, pre and
  // the bias, of every product of the call. One of them off the grid, the bias too, leaves the variants with
  // two-byte stores.
  bool vec = true;
  for (int i = 0; i < n; ++i) {
    GemmActProblem& p = ps[i];
    vec = vec && vec16(p.D, p.ldD) && (!p.C || vec16(p.C, p.ldC)) && (!p.pre || vec16(p.pre, p.ldPre)) && vec16(p.bias, 0);
    if (p.K == 0) continue;
    in_reach(p.A, p.ldA, p.ta ? p.K : p.M, p.ta ? p.M : p.K, p.copy_a != 0);
    in_reach(p.B, p.ldB, p.tb ? p.N : p.K, p.tb ? p.K : p.N, p.copy_b != 0);
  }
  if (copied > 0) {
    const int64_t blocks = std::min<int64_t>((copies.groups[0] + copies.groups[1] + 255) / 256, GA_SMS * 32);
    PL_CUDA(launch_dependent(align_copy_kernel, (int)blocks, 256, 0, 1, stream, copies));
  }

  GaPlan plans[GA_MAX_PROBS];
  const int launches = ga_plan_launches(ps, n, vec, plans);
  if (launches == 1) return ga_launch_products(ps, n, plans[0], vec, status, stream);
  PL_TRY(ga_launch_products(ps, 1, plans[0], vec, status, stream));
  return ga_launch_products(ps + 1, 1, plans[1], vec, status, stream);
}

cudaError_t launch_act_grad(const ActGradProblem& p, cudaStream_t stream) {
  if (p.M == 0) return cudaSuccess;
  // a function of the sizes alone; with that of the two loads, the order of the row sums depends on the sizes
  // and on whether rows come as 16-byte groups. As many blocks to a cluster as there are columns for,
  // eight at most
  int parts = 1;
  while (parts < 8 && p.N >= parts * AG_COLS) parts *= 2;
  const int64_t grid = (p.M + AG_ROWS - 1) / AG_ROWS * (int64_t)parts;
  const bool vec = vec16(p.dD, p.ldD) && (!p.dZ || vec16(p.dZ, p.ldZ)) &&
                   (p.act == PARALIA_ACT_NONE || vec16(p.pre, p.ldPre));
  return launch_dependent(vec ? act_grad_kernel<true> : act_grad_kernel<false>, (int)grid, AG_WARPS * 32, 0, parts, stream,
                          p, parts);
}

}  // namespace paralia
