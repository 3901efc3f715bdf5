// mx_abi.hip -- the extern "C" boundary of the entry points in microscaled floats.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/npu_amd.h"
#include "kernels.hpp"
#include "mx_device.hpp"
#include "serve_check.hpp"

namespace {

// (a launch's lanes are counted in 32 bits: kMaxRows and kMaxOut keep every grid below that)
constexpr long long kMaxK = 1 << 20, kMaxEntries = 1LL << 34, kMaxStride = 1 << 23, kMaxRows = 1 << 23, kMaxOut = 1LL << 32;

npu_status check_rows_k(const char *name, long long rows, long long K) {
  if (K % 32 != 0 || K > kMaxK)
    return fail(NPU_ERR_UNSUPPORTED, "%s: rows of %lld, expected a multiple of 32 up to 2^20", name, K);
  if (rows * K >= kMaxEntries) return fail(NPU_ERR_UNSUPPORTED, "%s: 2^34 entries or more", name);
  return NPU_OK;
}

// Blocks [rows, K] (rows or K < 0: whatever q says): elements of either type, and their scales.
npu_status check_blocks(const npu_memref *q, const npu_memref *scale, const char *name, const char *scale_name,
                        long long rows, long long K, bool *e4m3, const void **pq, const void **ps, long long *q_stride,
                        long long *s_stride) {
  if (!q) return fail(NPU_ERR_INVALID_ARG, "%s: null descriptor", name);
  *e4m3 = q->dtype == NPU_E4M3;
  NPU_TRY(check_rows(q, name, *e4m3 ? NPU_E4M3 : NPU_U8, 16, pq, q_stride));
  const long long R = rows < 0 ? q->sizes[0] : rows, k = K < 0 ? q->sizes[1] * (*e4m3 ? 1 : 2) : K;
  NPU_TRY(check_rows_k(name, R, k));
  NPU_TRY(expect_cols(q, name, R, *e4m3 ? k : k / 2));
  NPU_TRY(check_rows(scale, scale_name, NPU_U8, 1, ps, s_stride));
  return expect_cols(scale, scale_name, R, k / 32);
}

const uint8_t *u8(const void *p) { return static_cast<const uint8_t *>(p); }
uint8_t *u8w(const void *p) { return const_cast<uint8_t *>(u8(p)); }
const uint16_t *u16(const void *p) { return static_cast<const uint16_t *>(p); }
uint16_t *u16w(const void *p) { return const_cast<uint16_t *>(u16(p)); }

}  // namespace

extern "C" {

npu_status fused_mx_quantize(const npu_memref *x, const npu_memref *gate, const npu_memref *q, const npu_memref *scale,
                             const npu_memref *values, npu_stream stream) {
  npu::plans_reset();
  npu::MxQuantizeArgs a{};
  if (!x) return fail(NPU_ERR_INVALID_ARG, "x: null descriptor");
  a.f32 = x->dtype == NPU_F32;
  const int32_t dt = a.f32 ? NPU_F32 : NPU_BF16;
  const void *px, *pq, *ps, *pg = nullptr, *pv = nullptr;
  NPU_TRY(check_base(x, "x", 2, dt, a.f32 ? 4 : 2, &px));
  const long long R = x->sizes[0], K = x->sizes[1];
  NPU_TRY(check_rows_k("x", R, K));
  // (K is at least 32: a stride of 1 along it means rows)
  a.columns = x->strides[1] != 1;
  if (a.columns) {
    if (R > 1 && x->strides[0] != 1)
      return fail(NPU_ERR_UNSUPPORTED, "x: strides [%lld, %lld], rows or columns must be contiguous",
                  (long long)x->strides[0], (long long)x->strides[1]);
    if (x->strides[1] < R)
      return fail(NPU_ERR_UNSUPPORTED, "x: stride[1] = %lld, columns of %lld overlap", (long long)x->strides[1], R);
    a.x_stride = x->strides[1];
  } else {
    NPU_TRY(check_rows(x, "x", dt, 16, &px, &a.x_stride));
  }
  if (!absent(gate)) {
    if (a.f32) return fail(NPU_ERR_UNSUPPORTED, "gate: given, x is f32");
    if (a.columns) return fail(NPU_ERR_UNSUPPORTED, "gate: given, x has contiguous columns");
    NPU_TRY(check_rows(gate, "gate", NPU_BF16, 16, &pg, &a.gate_stride));
    NPU_TRY(expect_cols(gate, "gate", R, K));
  }
  NPU_TRY(check_blocks(q, scale, "q", "scale", R, K, &a.e4m3, &pq, &ps, &a.q_stride, &a.scale_stride));
  if (!absent(values)) {
    NPU_TRY(check_rows(values, "values", NPU_BF16, 16, &pv, &a.values_stride));
    NPU_TRY(expect_cols(values, "values", R, K));
  }
  a.x = px;
  a.gate = u16(pg);
  a.q = u8w(pq);
  a.scale = u8w(ps);
  a.values = u16w(pv);
  a.R = (int)R;
  a.K = (int)K;
  return launched("fused_mx_quantize launch", [&] { return npu::launch_mx_quantize(a, static_cast<hipStream_t>(stream)); });
}

npu_status fused_llama_add_rmsnorm(const npu_memref *x, const npu_memref *delta, const npu_memref *g, const npu_memref *h,
                                   const npu_memref *q, const npu_memref *scale, float eps, npu_stream stream) {
  npu::plans_reset();
  npu::AddRmsnormArgs a{};
  const void *px, *pd = nullptr, *pg, *ph = nullptr, *pq, *ps = nullptr;
  NPU_TRY(check_rows(x, "x", NPU_BF16, 16, &px, &a.x_stride));
  const long long T = x->sizes[0], D = x->sizes[1];
  if (D % 32 != 0 || D > 32768)
    return fail(NPU_ERR_UNSUPPORTED, "x: rows of %lld, expected a multiple of 32 up to 32768", D);
  if (T > kMaxRows) return fail(NPU_ERR_UNSUPPORTED, "x: %lld rows, at most 2^23", T);
  NPU_TRY(check_rows_k("x", T, D));
  if (!absent(delta)) {
    NPU_TRY(check_rows(delta, "delta", NPU_BF16, 16, &pd, &a.delta_stride));
    NPU_TRY(expect_cols(delta, "delta", T, D));
  }
  NPU_TRY(check_base(g, "g", 1, NPU_F32, 16, &pg));
  NPU_TRY(check_vec(g, "g", NPU_F32, D, &pg));
  if (!absent(h)) {
    NPU_TRY(check_rows(h, "h", NPU_BF16, 16, &ph, &a.h_stride));
    NPU_TRY(expect_cols(h, "h", T, D));
  }
  if (!q) return fail(NPU_ERR_INVALID_ARG, "q: null descriptor");
  if (q->dtype == NPU_BF16) {
    NPU_TRY(check_rows(q, "q", NPU_BF16, 16, &pq, &a.q_stride));
    NPU_TRY(expect_cols(q, "q", T, D));
    if (!absent(scale)) return fail(NPU_ERR_INVALID_ARG, "scale: given, q is bf16");
    a.kind = npu::kToBf16;
  } else {
    bool e4m3;
    NPU_TRY(check_blocks(q, scale, "q", "scale", T, D, &e4m3, &pq, &ps, &a.q_stride, &a.scale_stride));
    a.kind = e4m3 ? npu::kToE4m3 : npu::kToE2m1;
  }
  if (!(eps >= 0.0f) || eps > 3e38f) return fail(NPU_ERR_INVALID_ARG, "eps must be finite and not negative");
  a.x = u16(px);
  a.delta = u16(pd);
  a.g = static_cast<const float *>(pg);
  a.h = u16w(ph);
  a.q = u8w(pq);
  a.scale = u8w(ps);
  a.T = (int)T;
  a.D = (int)D;
  a.eps = eps;
  a.inv_D = 1.0 / (double)D;
  return launched("fused_llama_add_rmsnorm launch",
                  [&] { return npu::launch_add_rmsnorm(a, static_cast<hipStream_t>(stream)); });
}

int64_t npu_mx_matmul_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > kMaxRows || N > kMaxRows || K % 32 != 0 || K > kMaxK || M * K >= kMaxEntries ||
      N * K >= kMaxEntries || M * N >= kMaxOut)
    return -1;
  return (int64_t)(npu::mx_matmul_workspace((int)M, (int)N, (int)K) / sizeof(float));
}

npu_status fused_mx_matmul(const npu_memref *a, const npu_memref *a_scale, const npu_memref *w, const npu_memref *w_scale,
                           const npu_memref *out, const npu_memref *workspace, npu_stream stream) {
  npu::plans_reset();
  npu::MxMatmulArgs m{};
  const void *pa, *pas, *pw, *pws, *po;
  bool w_e4m3;
  NPU_TRY(check_blocks(a, a_scale, "a", "a_scale", -1, -1, &m.e4m3, &pa, &pas, &m.a_stride, &m.as_stride));
  const long long M = a->sizes[0], K = a->sizes[1] * (m.e4m3 ? 1 : 2);
  if (w && w->dtype == NPU_E4M3) return fail(NPU_ERR_UNSUPPORTED, "w: e4m3, expected e2m1");
  const long long N = w ? w->sizes[0] : 0;
  NPU_TRY(check_blocks(w, w_scale, "w", "w_scale", N, K, &w_e4m3, &pw, &pws, &m.w_stride, &m.ws_stride));
  // (the kernels' offsets within a tile have 32 bits)
  const long long stride = std::max(std::max(m.a_stride, m.as_stride), std::max(m.w_stride, m.ws_stride));
  if (stride >= kMaxStride) return fail(NPU_ERR_UNSUPPORTED, "a, w: rows at a stride of %lld bytes, at most 2^23", stride);
  NPU_TRY(check_rows(out, "out", NPU_BF16, 2, &po, &m.out_stride));
  NPU_TRY(expect_cols(out, "out", M, N));
  if (M > kMaxRows || N > kMaxRows) return fail(NPU_ERR_UNSUPPORTED, "out: [%lld,%lld], at most 2^23 each", M, N);
  if (M * N >= kMaxOut) return fail(NPU_ERR_UNSUPPORTED, "out: 2^32 entries or more");
  NPU_TRY(check_workspace(workspace, npu_mx_matmul_workspace(M, N, K), &m.workspace));
  m.a = u8(pa);
  m.a_scale = u8(pas);
  m.w = u8(pw);
  m.w_scale = u8(pws);
  m.out = u16w(po);
  m.M = (int)M;
  m.N = (int)N;
  m.K = (int)K;
  return launched("fused_mx_matmul launch", [&] { return npu::launch_mx_matmul(m, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
