// serve_abi.hip -- the extern "C" boundary of the serving entry points: their
// operands may be strided rows and caches past 2^31 elements, which the group
// entry points' descriptor check refuses.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/npu_amd.h"
#include "kernels.hpp"
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

int elem_size(int32_t dt) { return dt == NPU_BF16 ? 2 : dt == NPU_I8 ? 1 : 4; }

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

// One half of the cache: bf16 [P, Hkv, page, Dh], each page contiguous.
npu_status check_pages(const npu_memref *m, const char *name, const void **ptr, long long *stride) {
  NPU_TRY(check_base(m, name, 4, NPU_BF16, 16, ptr));
  const long long hkv = m->sizes[1], page = m->sizes[2], dh = m->sizes[3];
  if (dh != 64 && dh != 128)
    return fail(NPU_ERR_UNSUPPORTED, "%s: head dim %lld, expected 64 or 128", name, dh);
  if (page < 16 || (page & (page - 1)) != 0)
    return fail(NPU_ERR_UNSUPPORTED, "%s: page of %lld, expected a power of two of at least 16", name, page);
  if (hkv > 1024) return fail(NPU_ERR_UNSUPPORTED, "%s: %lld heads, at most 1024", name, hkv);
  if (hkv * page * dh > kMaxInt) return fail(NPU_ERR_UNSUPPORTED, "%s: a page holds 2^31 elements or more", name);
  if (m->strides[3] != 1 || m->strides[2] != dh || (hkv > 1 && m->strides[1] != page * dh))
    return fail(NPU_ERR_UNSUPPORTED, "%s: each page must be contiguous [Hkv, page, Dh]", name);
  *stride = m->sizes[0] > 1 ? m->strides[0] : hkv * page * dh;
  if (*stride < hkv * page * dh || *stride % 8 != 0)
    return fail(NPU_ERR_UNSUPPORTED, "%s: stride[0] = %lld, pages of %lld must not overlap and be 16-byte aligned",
                name, *stride, hkv * page * dh);
  return NPU_OK;
}

struct Cache {
  const void *k, *v;
  long long k_stride, v_stride;
  int Hkv, dh;
};

// The cache and the batch that the serving calls of a layer share.
npu_status check_batch(const npu_memref *k_pages, const npu_memref *v_pages, const npu_memref *page_table,
                       const npu_memref *kv_len, const npu_memref *q_start, long long T, int32_t prefix_len,
                       Cache *c, npu::ServeBatch *b) {
  NPU_TRY(check_pages(k_pages, "k_pages", &c->k, &c->k_stride));
  NPU_TRY(check_pages(v_pages, "v_pages", &c->v, &c->v_stride));
  for (int d = 0; d < 4; ++d)
    if (v_pages->sizes[d] != k_pages->sizes[d])
      return fail(NPU_ERR_INVALID_ARG, "v_pages: size[%d] = %lld, expected k_pages' %lld", d,
                  (long long)v_pages->sizes[d], (long long)k_pages->sizes[d]);
  c->Hkv = (int)k_pages->sizes[1];
  c->dh = (int)k_pages->sizes[3];
  const long long page = k_pages->sizes[2];
  const void *pt, *kl, *qs = nullptr;
  NPU_TRY(check_rows(page_table, "page_table", NPU_I32, 4, &pt, &b->table_stride));
  const long long B = page_table->sizes[0];
  if (B > 1 << 24) return fail(NPU_ERR_UNSUPPORTED, "%lld sequences, at most 2^24", B);
  NPU_TRY(check_vec(kv_len, "kv_len", NPU_I32, B, &kl));
  if (!absent(q_start)) {
    NPU_TRY(check_vec(q_start, "q_start", NPU_I32, B + 1, &qs));
  } else if (T != B) {
    return fail(NPU_ERR_INVALID_ARG, "%lld rows for %lld sequences: without q_start each has one token", T, B);
  }
  if (prefix_len < 0) return fail(NPU_ERR_INVALID_ARG, "prefix_len = %d is negative", prefix_len);
  if (prefix_len + page_table->sizes[1] * page > kMaxInt)
    return fail(NPU_ERR_UNSUPPORTED, "prefix_len + max_pages * page is 2^31 or more");
  b->page_table = static_cast<const int *>(pt);
  b->kv_len = static_cast<const int *>(kl);
  b->q_start = static_cast<const int *>(qs);
  b->T = (int)T;
  b->B = (int)B;
  b->max_pages = (int)page_table->sizes[1];
  b->page_log2 = __builtin_ctzll((unsigned long long)page);
  b->n_pages = (int)k_pages->sizes[0];
  b->prefix_len = prefix_len;
  return NPU_OK;
}

// Query heads of rows of `cols` entries: a multiple of the cache's heads.
npu_status check_heads(const char *name, long long cols, const Cache &c, int *heads) {
  const long long h = cols / c.dh;
  if (cols % c.dh != 0 || h % c.Hkv != 0 || h > 1024)
    return fail(NPU_ERR_INVALID_ARG, "%s: rows of %lld, expected H * %d with H a multiple of %d, at most 1024", name,
                cols, c.dh, c.Hkv);
  *heads = (int)h;
  return NPU_OK;
}

const uint16_t *u16(const void *p) { return static_cast<const uint16_t *>(p); }
uint16_t *u16w(const void *p) { return const_cast<uint16_t *>(static_cast<const uint16_t *>(p)); }

}  // namespace

extern "C" {

npu_status fused_llama_rope_append(const npu_memref *Q, const npu_memref *K, const npu_memref *V,
                                   const npu_memref *cos_t, const npu_memref *sin_t, const npu_memref *k_pages,
                                   const npu_memref *v_pages, const npu_memref *page_table, const npu_memref *kv_len,
                                   const npu_memref *q_start, const npu_memref *Qo, int32_t prefix_len, int32_t pairs,
                                   npu_stream stream) {
  npu::plans_reset();
  npu::RopeAppendArgs a{};
  Cache c;
  const void *pq, *pk, *pv, *pc, *ps, *po;
  long long tab_stride;
  NPU_TRY(check_rows(Q, "Q", NPU_BF16, 16, &pq, &a.q_stride));
  const long long T = Q->sizes[0];
  NPU_TRY(check_batch(k_pages, v_pages, page_table, kv_len, q_start, T, prefix_len, &c, &a.b));
  NPU_TRY(check_heads("Q", Q->sizes[1], c, &a.H));
  NPU_TRY(check_rows(K, "K", NPU_BF16, 16, &pk, &a.k_stride));
  NPU_TRY(expect_cols(K, "K", T, (long long)c.Hkv * c.dh));
  NPU_TRY(check_rows(V, "V", NPU_BF16, 16, &pv, &a.v_stride));
  NPU_TRY(expect_cols(V, "V", T, (long long)c.Hkv * c.dh));
  NPU_TRY(check_rows(Qo, "Qo", NPU_BF16, 16, &po, &a.o_stride));
  NPU_TRY(expect_cols(Qo, "Qo", T, Q->sizes[1]));
  NPU_TRY(check_rows(cos_t, "cos_t", NPU_F32, 16, &pc, &tab_stride));
  const long long width = cos_t->sizes[1], positions = cos_t->sizes[0];
  if (width % 8 != 0 || width > c.dh / 2)
    return fail(NPU_ERR_UNSUPPORTED, "cos_t: %lld columns, expected a multiple of 8 up to %d", width, c.dh / 2);
  if (tab_stride != width) return fail(NPU_ERR_UNSUPPORTED, "cos_t: must be contiguous");
  const long long need = (long long)prefix_len + ((long long)a.b.max_pages << a.b.page_log2);
  if (positions < need)
    return fail(NPU_ERR_INVALID_ARG, "cos_t: %lld positions, the prefix and the page table reach %lld", positions,
                need);
  NPU_TRY(check_rows(sin_t, "sin_t", NPU_F32, 16, &ps, &tab_stride));
  NPU_TRY(expect_cols(sin_t, "sin_t", positions, width));
  if (tab_stride != width) return fail(NPU_ERR_UNSUPPORTED, "sin_t: must be contiguous");
  if (pairs != NPU_PAIRS_INTERLEAVED && pairs != NPU_PAIRS_HALVES)
    return fail(NPU_ERR_INVALID_ARG, "pairs %d is not one of INTERLEAVED/HALVES", pairs);
  a.Q = u16(pq); a.K = u16(pk); a.V = u16(pv); a.Qo = u16w(po);
  a.cos_t = static_cast<const float *>(pc);
  a.sin_t = static_cast<const float *>(ps);
  a.k_pages = u16w(c.k); a.v_pages = u16w(c.v);
  a.kpage_stride = c.k_stride; a.vpage_stride = c.v_stride;
  a.Hkv = c.Hkv; a.dh = c.dh; a.width = (int)width; a.pairs = pairs;
  return launched("fused_llama_rope_append launch",
                  [&] { return npu::launch_llama_rope_append(a, static_cast<hipStream_t>(stream)); });
}

int64_t npu_paged_attention_workspace(int64_t T, int64_t B, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                      int32_t prefix_len) {
  if (T <= 0 || B <= 0 || T > kMaxInt || B > 1 << 24 || n_heads <= 0 || n_heads > 1024 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads != 0 || (head_dim != 64 && head_dim != 128) || prefix_len < 0 || T * n_heads > kMaxInt)
    return -1;
  npu::ServeBatch b{};
  b.T = (int)T;
  b.B = (int)B;
  b.prefix_len = prefix_len;
  return (int64_t)(npu::paged_attention_workspace(b, n_heads, n_kv_heads, head_dim) / sizeof(float));
}

npu_status fused_llama_paged_attention(const npu_memref *Q, const npu_memref *k_pages, const npu_memref *v_pages,
                                       const npu_memref *page_table, const npu_memref *kv_len,
                                       const npu_memref *q_start, const npu_memref *prefix_table, const npu_memref *A,
                                       const npu_memref *workspace, int32_t prefix_len, float scale,
                                       npu_stream stream) {
  npu::plans_reset();
  npu::PagedAttentionArgs a{};
  Cache c;
  const void *pq, *po, *pp = nullptr;
  NPU_TRY(check_rows(Q, "Q", NPU_BF16, 16, &pq, &a.q_stride));
  const long long T = Q->sizes[0];
  NPU_TRY(check_batch(k_pages, v_pages, page_table, kv_len, q_start, T, prefix_len, &c, &a.b));
  NPU_TRY(check_heads("Q", Q->sizes[1], c, &a.H));
  NPU_TRY(check_rows(A, "A", NPU_BF16, 16, &po, &a.o_stride));
  NPU_TRY(expect_cols(A, "A", T, Q->sizes[1]));
  if (T * a.H > kMaxInt) return fail(NPU_ERR_UNSUPPORTED, "T * H = %lld is 2^31 or more", T * a.H);
  if (prefix_len > 0) {
    if (absent(prefix_table)) return fail(NPU_ERR_INVALID_ARG, "prefix_table: absent, prefix_len is %d", prefix_len);
    NPU_TRY(check_vec(prefix_table, "prefix_table", NPU_I32, -1, &pp));
    const long long page = k_pages->sizes[2], need = (prefix_len + page - 1) / page;
    if (prefix_table->sizes[0] < need)
      return fail(NPU_ERR_INVALID_ARG, "prefix_table: %lld pages, the prefix needs %lld",
                  (long long)prefix_table->sizes[0], need);
  } else if (!absent(prefix_table) && prefix_table->sizes[0] != 0) {  // (no pages are a prefix's of no keys)
    return fail(NPU_ERR_INVALID_ARG, "prefix_table: given, prefix_len is 0");
  }
  if (!(scale > 0.0f) || scale > 3e38f) return fail(NPU_ERR_INVALID_ARG, "scale must be positive and finite");
  NPU_TRY(check_workspace(workspace, npu_paged_attention_workspace(T, a.b.B, a.H, c.Hkv, c.dh, prefix_len),
                          &a.workspace));
  a.Q = u16(pq); a.k_pages = u16(c.k); a.v_pages = u16(c.v);
  a.prefix_table = static_cast<const int *>(pp);
  a.out = u16w(po);
  a.kpage_stride = c.k_stride; a.vpage_stride = c.v_stride;
  a.Hkv = c.Hkv; a.dh = c.dh; a.scale = scale;
  return launched("fused_llama_paged_attention launch",
                  [&] { return npu::launch_llama_paged_attention(a, static_cast<hipStream_t>(stream)); });
}

// (a row's state is in LDS: the workspace is checked, for kernels that share a row, and not used)
int64_t npu_sample_workspace(int64_t B, int64_t V) {
  if (B <= 0 || B > kMaxInt || V <= 0 || V > 1 << 20) return -1;
  return 4;
}

npu_status fused_sample_tokens(const npu_memref *logits, const npu_memref *u, const npu_memref *temperature,
                               const npu_memref *top_k, const npu_memref *top_p, const npu_memref *min_p,
                               const npu_memref *tokens, const npu_memref *probs, const npu_memref *workspace,
                               npu_stream stream) {
  npu::plans_reset();
  npu::SampleArgs a{};
  if (!logits) return fail(NPU_ERR_INVALID_ARG, "logits: null descriptor");
  a.bf16 = logits->dtype == NPU_BF16;
  const void *pl, *p[7] = {};
  void *ws;
  NPU_TRY(check_rows(logits, "logits", a.bf16 ? NPU_BF16 : NPU_F32, a.bf16 ? 2 : 4, &pl, &a.row_stride));
  const long long B = logits->sizes[0], V = logits->sizes[1];
  if (V > 1 << 20) return fail(NPU_ERR_UNSUPPORTED, "logits: %lld columns, at most 2^20", V);
  NPU_TRY(check_vec(u, "u", NPU_F32, B, &p[0]));
  if (!absent(temperature)) NPU_TRY(check_vec(temperature, "temperature", NPU_F32, B, &p[1]));
  if (!absent(top_k)) NPU_TRY(check_vec(top_k, "top_k", NPU_I32, B, &p[2]));
  if (!absent(top_p)) NPU_TRY(check_vec(top_p, "top_p", NPU_F32, B, &p[3]));
  if (!absent(min_p)) NPU_TRY(check_vec(min_p, "min_p", NPU_F32, B, &p[4]));
  NPU_TRY(check_vec(tokens, "tokens", NPU_I32, B, &p[5]));
  if (!absent(probs)) NPU_TRY(check_vec(probs, "probs", NPU_F32, B, &p[6]));
  NPU_TRY(check_workspace(workspace, npu_sample_workspace(B, V), &ws));
  a.logits = pl;
  a.B = (int)B;
  a.V = (int)V;
  a.u = static_cast<const float *>(p[0]);
  a.temperature = static_cast<const float *>(p[1]);
  a.top_k = static_cast<const int *>(p[2]);
  a.top_p = static_cast<const float *>(p[3]);
  a.min_p = static_cast<const float *>(p[4]);
  a.tokens = const_cast<int *>(static_cast<const int *>(p[5]));
  a.probs = const_cast<float *>(static_cast<const float *>(p[6]));
  return launched("fused_sample_tokens launch",
                  [&] { return npu::launch_sample_tokens(a, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
