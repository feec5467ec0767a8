// Host side of the gradient-list routines: argument checks and the description of the list.
// No counterpart in the reference; they stand beside its level-1 tile operations
// (Library_scheduler/src/Functions/daxpy.cpp:53-69, ddot.cpp:54-70).
#include <algorithm>
#include <cmath>
#include <vector>

#include "exec.hpp"
#include "grad_list.cuh"
#include "runtime.hpp"

namespace paralia {
namespace {

int64_t type_bytes(int t) { return t == PARALIA_F32 ? 4 : (t == PARALIA_F16 || t == PARALIA_BF16) ? 2 : 0; }

struct Range {
  uintptr_t lo, hi;
  bool write;
};

// Refuses memory that is written and also read or written for another tensor: the order of
// those accesses would decide the result. A tensor scaled in place appears once, as written.
bool ranges_conflict(std::vector<Range>& r) {
  auto less = [](const Range& a, const Range& b) { return a.lo < b.lo; };
  if (!std::is_sorted(r.begin(), r.end(), less)) std::sort(r.begin(), r.end(), less);
  uintptr_t written = 0, used = 0;   // ends of what lies before, written and at all
  for (const Range& x : r) {
    if (x.lo < written || (x.write && x.lo < used)) return true;
    used = std::max(used, x.hi);
    if (x.write) written = std::max(written, x.hi);
  }
  return false;
}

// Scratch and results stand apart from one another and from every tensor: some blocks still read what
// another one has written its result over.
int check_apart(const GradList& l, const void* scratch, int64_t scratch_bytes, const void* sumsq, const void* norm) {
  const void* p[3] = {scratch, sumsq, norm};
  const int64_t bytes[3] = {scratch_bytes, (int64_t)sizeof(double), (int64_t)sizeof(float)};
  Range r[3];
  for (int i = 0; i < 3; ++i) {
    r[i].lo = reinterpret_cast<uintptr_t>(p[i]);
    r[i].hi = p[i] ? r[i].lo + bytes[i] : 0;
  }
  auto meet = [](const Range& a, uintptr_t lo, uintptr_t hi) { return a.lo < hi && lo < a.hi; };
  bool near = false, shared = false;
  for (int i = 0; i < 3; ++i) {
    for (int j = i + 1; j < 3; ++j) shared = shared || meet(r[i], r[j].lo, r[j].hi);
    near = near || meet(r[i], l.lo, l.hi);
  }
  for (int t = 0; near && t < l.count; ++t) {
    const GradEntry& e = l.entries[t];
    const uintptr_t s = reinterpret_cast<uintptr_t>(e.src), d = reinterpret_cast<uintptr_t>(e.dst);
    const uintptr_t s_end = s + e.n * type_bytes(e.src_type), d_end = d + e.n * type_bytes(e.dst_type);
    for (const Range& x : r) shared = shared || meet(x, s, s_end) || meet(x, d, d_end);
  }
  if (shared) return fail(PARALIA_ERR_INVALID_ARG, "scratch, sumsq and norm may share memory with nothing");
  return PARALIA_OK;
}

// Checks the list and describes its non-empty tensors. out == nullptr: in place.
int describe(int count, const void* const* g, const int64_t* n, const int32_t* type, void* const* out,
             const int32_t* out_type, bool writes, std::vector<GradEntry>* entries, GradList* l) {
  if (count < 0) return fail(PARALIA_ERR_INVALID_ARG, "negative number of tensors");
  if (count > 0 && (!g || !n || !type)) return fail(PARALIA_ERR_INVALID_ARG, "NULL tensor list");
  if (out && !out_type) return fail(PARALIA_ERR_INVALID_ARG, "outputs without their element types");
  for (int i = 0; i < count; ++i) {
    const int32_t dt = out ? out_type[i] : type[i];
    if (!type_bytes(type[i]) || !type_bytes(dt))
      return fail(PARALIA_ERR_INVALID_ARG, "tensor %d: element type is not PARALIA_F32, PARALIA_F16 or PARALIA_BF16", i);
    if (n[i] < 0 || n[i] > ((int64_t)1 << 48)) return fail(PARALIA_ERR_INVALID_ARG, "tensor %d: size out of range", i);
    if (n[i] == 0) continue;
    const void* d = out ? out[i] : g[i];
    if (!g[i] || !d) return fail(PARALIA_ERR_INVALID_ARG, "tensor %d: NULL pointer", i);
    if (reinterpret_cast<uintptr_t>(g[i]) % type_bytes(type[i]) || reinterpret_cast<uintptr_t>(d) % type_bytes(dt))
      return fail(PARALIA_ERR_INVALID_ARG, "tensor %d: address is not a multiple of the element size", i);
  }
  l->units = 0;
  l->lo = UINTPTR_MAX;
  l->hi = 0;
  entries->reserve(count);
  std::vector<Range> reads_writes;
  if (writes) reads_writes.reserve(2 * (size_t)count);
  for (int i = 0; i < count; ++i) {
    if (n[i] == 0) continue;
    GradEntry e;
    e.src = g[i];
    e.dst = out ? out[i] : const_cast<void*>(g[i]);
    e.n = n[i];
    e.src_type = (uint8_t)type[i];
    e.dst_type = (uint8_t)(out ? out_type[i] : type[i]);
    e.flags = 0;
    e.head = 0;
    const uintptr_t s = reinterpret_cast<uintptr_t>(e.src), d = reinterpret_cast<uintptr_t>(e.dst);
    const int64_t sb = type_bytes(e.src_type), db = type_bytes(e.dst_type);
    l->lo = std::min(l->lo, std::min(s, d));
    l->hi = std::max(l->hi, std::max(s + (uintptr_t)(e.n * sb), d + (uintptr_t)(e.n * db)));
    if (e.dst == e.src && e.dst_type == e.src_type) e.flags |= GL_IN_PLACE;
    // the first element from which groups of eight are aligned, and in dst too if that can be
    for (int h = 7; h >= 0; --h) {
      if (((s + h * sb) & 15) != 0) continue;
      const bool both = ((d + h * db) & 15) == 0;
      if (!both && (e.flags & GL_DST_VEC)) continue;
      e.head = (uint8_t)h;
      if (both) e.flags |= GL_DST_VEC;
    }
    const int64_t body = std::max<int64_t>(0, e.n - e.head);
    if (l->units > INT32_MAX - body / GL_UNIT - 1) return fail(PARALIA_ERR_UNSUPPORTED, "the list has too many elements");
    e.unit0 = (int32_t)l->units;
    l->units += std::max<int64_t>(1, (body + GL_UNIT - 1) / GL_UNIT);
    entries->push_back(e);
    if (writes) {
      if (!(e.flags & GL_IN_PLACE)) reads_writes.push_back({s, s + (uintptr_t)(e.n * sb), false});
      reads_writes.push_back({d, d + (uintptr_t)(e.n * db), true});
    }
  }
  if (writes && ranges_conflict(reads_writes))
    return fail(PARALIA_ERR_INVALID_ARG, "a tensor to be written overlaps another tensor of the list");
  l->count = (int)entries->size();
  l->entries = entries->data();
  return PARALIA_OK;
}

int enter(int dev, void* stream) {
  Runtime& rt = Runtime::get();
  PL_TRY(rt.init());
  PL_TRY(rt.enter_tile_call(dev, static_cast<cudaStream_t>(stream)));
  return PARALIA_OK;
}

int check_max_norm(float max_norm) {
  if (!(max_norm >= 0.0f)) return fail(PARALIA_ERR_INVALID_ARG, "max_norm is negative or not a number");
  return PARALIA_OK;
}

int check_results(const double* sumsq, const float* norm) {
  if ((reinterpret_cast<uintptr_t>(sumsq) & 7) || (reinterpret_cast<uintptr_t>(norm) & 3))
    return fail(PARALIA_ERR_INVALID_ARG, "sumsq or norm is not aligned to its type");
  return PARALIA_OK;
}

int check_scratch(const void* scratch) {
  if (!scratch) return fail(PARALIA_ERR_INVALID_ARG, "NULL scratch");
  if (reinterpret_cast<uintptr_t>(scratch) & 7) return fail(PARALIA_ERR_INVALID_ARG, "scratch is not aligned to 8 bytes");
  return PARALIA_OK;
}

}  // namespace

int64_t grad_norm_scratch_bytes(int count) {
  return grad_partials(std::max(count, 0)) * (int64_t)sizeof(double);
}

int exec_tile_grad_norm(int dev, void* stream, int count, const void* const* g, const int64_t* n, const int32_t* type,
                        void* scratch, double* sumsq, float* norm) {
  std::vector<GradEntry> entries;
  GradList l;
  PL_TRY(describe(count, g, n, type, nullptr, nullptr, false, &entries, &l));
  PL_TRY(check_scratch(scratch));
  PL_TRY(check_results(sumsq, norm));
  if (!sumsq && !norm) return fail(PARALIA_ERR_INVALID_ARG, "NULL sumsq and norm");
  PL_TRY(check_apart(l, scratch, grad_norm_scratch_bytes(count), sumsq, norm));
  DeviceGuard guard;
  PL_TRY(enter(dev, stream));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int used = 0;
  PL_CUDA(launch_grad_sumsq(l, static_cast<double*>(scratch), &used, s));
  PL_CUDA(launch_grad_norm_final(static_cast<double*>(scratch), used, sumsq, norm, s));
  return PARALIA_OK;
}

int exec_tile_grad_clip(int dev, void* stream, int count, const void* const* g, const int64_t* n, const int32_t* type,
                        void* const* out, const int32_t* out_type, float max_norm, void* scratch, double* sumsq,
                        float* norm) {
  std::vector<GradEntry> entries;
  GradList l;
  PL_TRY(check_max_norm(max_norm));
  PL_TRY(describe(count, g, n, type, out, out_type, true, &entries, &l));
  PL_TRY(check_scratch(scratch));
  PL_TRY(check_results(sumsq, norm));
  PL_TRY(check_apart(l, scratch, grad_norm_scratch_bytes(count), sumsq, norm));
  DeviceGuard guard;
  PL_TRY(enter(dev, stream));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int used = 0;
  PL_CUDA(launch_grad_sumsq(l, static_cast<double*>(scratch), &used, s));
  PL_CUDA(launch_grad_scale(l, static_cast<double*>(scratch), used, max_norm, sumsq, norm, s));
  return PARALIA_OK;
}

int exec_tile_grad_scale(int dev, void* stream, int count, const void* const* g, const int64_t* n,
                         const int32_t* type, void* const* out, const int32_t* out_type, const double* sumsq,
                         float max_norm, float* norm) {
  std::vector<GradEntry> entries;
  GradList l;
  PL_TRY(check_max_norm(max_norm));
  PL_TRY(describe(count, g, n, type, out, out_type, true, &entries, &l));
  if (!sumsq) return fail(PARALIA_ERR_INVALID_ARG, "NULL sumsq");
  PL_TRY(check_results(sumsq, norm));
  PL_TRY(check_apart(l, nullptr, 0, sumsq, norm));
  DeviceGuard guard;
  PL_TRY(enter(dev, stream));
  // one partial sum is only read
  PL_CUDA(launch_grad_scale(l, const_cast<double*>(sumsq), 1, max_norm, nullptr, norm, static_cast<cudaStream_t>(stream)));
  return PARALIA_OK;
}

}  // namespace paralia
