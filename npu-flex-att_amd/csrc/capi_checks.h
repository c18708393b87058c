// Argument checks and small host helpers shared by the extern "C" entry points
// (capi.hip, capi_cache.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/flexatt.h"
#include "flexatt_kernels.h"

namespace flexatt {

#define FLEXATT_TRY(x)             \
  do {                             \
    const int rc_ = (x);           \
    if (rc_ != FLEXATT_OK) return rc_; \
  } while (0)

inline size_t elt_size(int dt) {
  switch (dt) {
    case FLEXATT_F32: return 4;
    case FLEXATT_F16:
    case FLEXATT_BF16: return 2;
    default: return 0;
  }
}

inline int head_index(int d) {
  switch (d) {
    case 32: return 0;
    case 64: return 1;
    case 128: return 2;
    case 256: return 3;
    default: return -1;
  }
}

inline int check_view(const flexatt_tensor* t, int64_t es) {
  if (!t || !t->data) return FLEXATT_EINVAL;
  if (t->stride_d != 1) return FLEXATT_ELAYOUT;
  if (t->stride_b < 0 || t->stride_h < 0 || t->stride_s < 0) return FLEXATT_ELAYOUT;
  if (((uintptr_t)t->data) % 16 != 0) return FLEXATT_ELAYOUT;
  if ((t->stride_b * es) % 16 || (t->stride_h * es) % 16 || (t->stride_s * es) % 16) return FLEXATT_ELAYOUT;
  return FLEXATT_OK;
}
inline int check_tensor(const flexatt_tensor* t, int dt) { return check_view(t, (int64_t)elt_size(dt)); }

// No two elements of an index space of up to five dimensions share an address.
// Sufficient test: over the dimensions of extent > 1 sorted by stride, each stride
// exceeds the span of the smaller ones.
inline int check_nested(const int64_t* st, const int64_t* ext, int n_dims) {
  int order[5], n = 0;
  for (int i = 0; i < n_dims; ++i)
    if (ext[i] > 1) order[n++] = i;
  for (int i = 1; i < n; ++i)  // insertion sort by stride
    for (int j = i; j > 0 && st[order[j]] < st[order[j - 1]]; --j) {
      const int x = order[j];
      order[j] = order[j - 1];
      order[j - 1] = x;
    }
  int64_t span = 0;  // largest offset reachable with the dims sorted so far
  for (int i = 0; i < n; ++i) {
    const int d = order[i];
    if (st[d] <= span) return FLEXATT_ELAYOUT;
    span += (ext[d] - 1) * st[d];
  }
  return FLEXATT_OK;
}

// Output tensors: the input rules, and no two elements may share an address (several
// workgroups would store to it, and the results would depend on their order).
inline int check_out_view(const flexatt_tensor* t, int64_t es, int64_t n_b, int64_t n_h, int64_t n_s, int64_t n_d) {
  FLEXATT_TRY(check_view(t, es));
  const int64_t st[4] = {t->stride_b, t->stride_h, t->stride_s, 1}, ext[4] = {n_b, n_h, n_s, n_d};
  return check_nested(st, ext, 4);
}
inline int check_out_tensor(const flexatt_tensor* t, int dt, int64_t n_b, int64_t n_h, int64_t n_s, int64_t n_d) {
  return check_out_view(t, (int64_t)elt_size(dt), n_b, n_h, n_s, n_d);
}

// Two output tensors of one shape that pass check_out_tensor: apart, or, with the same
// strides, one layout in which the step from one to the other is a dimension of extent 2
// (keys and values side by side in one buffer).
inline int check_out_views(const flexatt_tensor* x, const flexatt_tensor* y, int64_t es, int64_t n_b, int64_t n_h,
                           int64_t n_s, int64_t n_d) {
  const int64_t ext[5] = {n_b, n_h, n_s, n_d, 2};
  if ((uintptr_t)x->data > (uintptr_t)y->data) {
    const flexatt_tensor* z = x;
    x = y;
    y = z;
  }
  const uintptr_t step = (uintptr_t)y->data - (uintptr_t)x->data;
  const int64_t last = (n_b - 1) * x->stride_b + (n_h - 1) * x->stride_h + (n_s - 1) * x->stride_s + n_d;
  if (step >= (uintptr_t)(last * es)) return FLEXATT_OK;
  const int64_t st[5] = {x->stride_b, x->stride_h, x->stride_s, 1, (int64_t)step / es};
  const int64_t other[3] = {y->stride_b, y->stride_h, y->stride_s};
  for (int i = 0; i < 3; ++i)
    if (ext[i] > 1 && st[i] != other[i]) return FLEXATT_ELAYOUT;
  return check_nested(st, ext, 5);
}
inline int check_out_pair(const flexatt_tensor* x, const flexatt_tensor* y, int dt, int64_t n_b, int64_t n_h, int64_t n_s,
                          int64_t n_d) {
  return check_out_views(x, y, (int64_t)elt_size(dt), n_b, n_h, n_s, n_d);
}

// A launch has at most 2^32 - 1 work-items.
inline int check_launch(int64_t workgroups, int threads) {
  return workgroups <= (((int64_t)1 << 32) - 1) / threads ? FLEXATT_OK : FLEXATT_ERANGE;
}

inline View view(const flexatt_tensor* t) { return View{t->data, t->stride_b, t->stride_h, t->stride_s}; }
inline MutView mview(const flexatt_tensor* t) { return MutView{t->data, t->stride_b, t->stride_h, t->stride_s}; }

constexpr int kMaxDevices = 64;

// CUs of the current device (cached per device), 0 if unknown.  Host threads
// may call the ABI concurrently: the cache is atomic (a racing first lookup
// stores the same value twice).
inline int cu_count() {
  static std::atomic<int> cache[kMaxDevices];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
    cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

inline int cus() {  // 256 if unknown
  const int n = cu_count();
  return n > 0 ? n : 256;
}

}  // namespace flexatt
