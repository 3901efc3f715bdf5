// serve_check.hpp -- operand checks of the serving entry points (serve_abi.hip, mx_abi.hip):
// their operands may be strided rows and caches past 2^31 elements, which the
// group entry points' descriptor check refuses.  Included by a file that has them for its own.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/npu_amd.h"
#include "plans.hpp"

namespace {

npu_status fail(npu_status code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  npu::set_last_error(buf);
  return code;
}

#define NPU_TRY(expr)                 \
  do {                                \
    npu_status _s = (expr);           \
    if (_s != NPU_OK) return _s;      \
  } while (0)

// A launcher's result; what it throws (the plan list's allocation) ends here.
template <class F>
npu_status launched(const char *what, F launch) {
  try {
    const hipError_t e = launch();
    if (e != hipSuccess) return fail(NPU_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    npu::set_last_error("");
    return NPU_OK;
  } catch (...) {
    return fail(NPU_ERR_OOM, "%s: out of host memory", what);
  }
}

constexpr long long kMaxInt = (1LL << 31) - 1;

bool absent(const npu_memref *m) { return !m || !m->aligned; }

int elem_size(int32_t dt) { return dt == NPU_BF16 ? 2 : dt == NPU_I8 || dt == NPU_U8 || dt == NPU_E4M3 ? 1 : 4; }

// Rank, element type, positive sizes below 2^31 and the data pointer's
// alignment; *ptr: the first element.
npu_status check_base(const npu_memref *m, const char *name, int32_t rank, int32_t dtype, int align,
                      const void **ptr) {
  if (!m) return fail(NPU_ERR_INVALID_ARG, "%s: null descriptor", name);
  if (m->rank != rank) return fail(NPU_ERR_INVALID_ARG, "%s: rank %d, expected %d", name, m->rank, rank);
  if (m->dtype != dtype)
    return fail(NPU_ERR_INVALID_ARG, "%s: element type %d, expected %d", name, m->dtype, dtype);
  if (!m->aligned) return fail(NPU_ERR_INVALID_ARG, "%s: null data pointer", name);
  if (m->offset < 0) return fail(NPU_ERR_INVALID_ARG, "%s: negative offset", name);
  for (int d = 0; d < rank; ++d)
    if (m->sizes[d] <= 0 || m->sizes[d] > kMaxInt)
      return fail(NPU_ERR_INVALID_ARG, "%s: size[%d] = %lld must be positive and below 2^31", name, d,
                  (long long)m->sizes[d]);
  const char *base = static_cast<const char *>(m->aligned) + m->offset * elem_size(dtype);
  if (reinterpret_cast<uintptr_t>(base) % align != 0)
    return fail(NPU_ERR_UNSUPPORTED, "%s: data pointer is not %d-byte aligned", name, align);
  *ptr = base;
  return NPU_OK;
}

// [rows, cols] with contiguous rows at a stride that keeps them aligned.
npu_status check_rows(const npu_memref *m, const char *name, int32_t dtype, int align, const void **ptr,
                      long long *stride) {
  NPU_TRY(check_base(m, name, 2, dtype, align, ptr));
  if (m->sizes[1] > 1 && m->strides[1] != 1)
    return fail(NPU_ERR_UNSUPPORTED, "%s: stride[1] = %lld, rows must be contiguous", name, (long long)m->strides[1]);
  *stride = m->sizes[0] > 1 ? m->strides[0] : m->sizes[1];
  if (*stride < m->sizes[1])
    return fail(NPU_ERR_UNSUPPORTED, "%s: stride[0] = %lld, rows of %lld overlap", name, *stride,
                (long long)m->sizes[1]);
  if (m->sizes[0] > 1 && *stride * elem_size(dtype) % align != 0)
    return fail(NPU_ERR_UNSUPPORTED, "%s: rows at a stride of %lld are not %d-byte aligned", name, *stride, align);
  return NPU_OK;
}

npu_status check_vec(const npu_memref *m, const char *name, int32_t dtype, long long n, const void **ptr) {
  NPU_TRY(check_base(m, name, 1, dtype, 4, ptr));
  if (m->sizes[0] > 1 && m->strides[0] != 1)
    return fail(NPU_ERR_UNSUPPORTED, "%s: stride %lld, must be contiguous", name, (long long)m->strides[0]);
  if (n >= 0 && m->sizes[0] != n)
    return fail(NPU_ERR_INVALID_ARG, "%s: size %lld, expected %lld", name, (long long)m->sizes[0], n);
  return NPU_OK;
}

npu_status expect_cols(const npu_memref *m, const char *name, long long rows, long long cols) {
  if (m->sizes[0] != rows || m->sizes[1] != cols)
    return fail(NPU_ERR_INVALID_ARG, "%s: [%lld,%lld], expected [%lld,%lld]", name, (long long)m->sizes[0],
                (long long)m->sizes[1], rows, cols);
  return NPU_OK;
}

npu_status check_workspace(const npu_memref *m, long long need, void **ptr) {
  const void *p;
  NPU_TRY(check_base(m, "workspace", 1, NPU_F32, 16, &p));
  if (m->sizes[0] > 1 && m->strides[0] != 1) return fail(NPU_ERR_UNSUPPORTED, "workspace: must be contiguous");
  if (m->sizes[0] < need)
    return fail(NPU_ERR_INVALID_ARG, "workspace: %lld elements, %lld needed", (long long)m->sizes[0], need);
  *ptr = const_cast<void *>(p);
  return NPU_OK;
}

}  // namespace
