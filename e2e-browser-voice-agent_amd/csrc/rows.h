// rows.h -- what the operators on callers' device buffers share on the host: checks of rows and arrays, element types.
#pragma once
#include <stdint.h>

#include "host.h"

namespace q4 {

// Threads of a launch at most: HIP takes less than 2^32.
constexpr uint32_t kMostThreads = 1u << 31;

inline int elem_size(int type) { return type == Q4HIP_TYPE_F32 ? 4 : 2; }

inline int check_type(int type) {
  if (type != Q4HIP_TYPE_F32 && type != Q4HIP_TYPE_F16 && type != Q4HIP_TYPE_BF16)
    return fail(Q4HIP_ETYPE, "type %d: expected F32, F16 or BF16", type);
  return Q4HIP_OK;
}

// Whether 16 bytes of any row can be loaded at once.
inline bool aligned16(const void* p, int64_t stride, int type) {
  return ((uintptr_t)p | (uintptr_t)(stride * elem_size(type))) % 16 == 0;
}

// `rows` rows of `width` elements, `stride` elements apart.
inline int check_rows(int device, const void* p, int rows, int64_t width, int64_t stride, int type, const char* what) {
  const int es = elem_size(type);
  if ((uintptr_t)p % es) return fail(Q4HIP_EINVAL, "%s: not aligned to its type", what);
  if (stride < width) return fail(Q4HIP_EINVAL, "%s: rows of %lld values, %lld apart", what, (long long)width, (long long)stride);
  if (stride > ((int64_t)1 << 31)) return fail(Q4HIP_EINVAL, "%s: rows %lld values apart", what, (long long)stride);
  return check_device_span(p, ((size_t)(rows - 1) * stride + width) * es, device, what);
}

// Rows that one call reads and another buffer's that it writes must not share a byte.  Neighbouring columns of the same
// rows may: where the strides differ, the whole spans count.
inline int check_apart(const void* p, int64_t p_stride, const void* out, int64_t out_stride, int rows, int64_t width, int type,
                       const char* what) {
  const int es = elem_size(type);
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)out, w = (uintptr_t)width * es;
  const uintptr_t a_end = a + (uintptr_t)(rows - 1) * p_stride * es + w, b_end = b + (uintptr_t)(rows - 1) * out_stride * es + w;
  if (a_end <= b || b_end <= a) return Q4HIP_OK;
  if (p_stride == out_stride) {
    const uintptr_t s = (uintptr_t)p_stride * es, d = b >= a ? (b - a) % s : (s - (a - b) % s) % s;
    if (d >= w && s - d >= w) return Q4HIP_OK;
  }
  return fail(Q4HIP_EINVAL, "%s overlap", what);
}

// int32 arrays of n elements; NULL or an empty one is not looked at.
inline int check_ints(int device, const void* p, size_t n, const char* what) {
  if (!p || !n) return Q4HIP_OK;
  if ((uintptr_t)p % 4) return fail(Q4HIP_EINVAL, "%s: not aligned to its type", what);
  return check_device_span(p, n * 4, device, what);
}

// Whether n bytes at p and m at q share any.
inline bool overlap(const void* p, size_t n, const void* q, size_t m) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return n && m && a < b + m && b < a + n;
}

template <class F>
void by_type(int type, F f) {
  if (type == Q4HIP_TYPE_F32) f(float());
  else if (type == Q4HIP_TYPE_F16) f(_Float16());
  else f(__bf16());
}

}  // namespace q4
