// k_rope_append.hip -- new queries, keys and values of a batch: rotated, and
// the keys and values stored in the paged cache.
//
//   (a, b) -> (a cos p - b sin p, a sin p + b cos p) for each pair of a head's
//   first 2 width entries, p the token's position; f32, rounded once to bf16.
//
// Bound by its bytes: every row is read once and written once (four prompts of 2500 to
// 4100 tokens, 32 + 2 8 heads of 128, 328 MB: 65 us, 5.0 TB/s; a step of 48 tokens:
// 5.1 us, a call of nothing).  A lane takes
// sixteen entries of one head as two 16-byte runs that hold eight whole pairs
// (consecutive runs for interleaved pairs, one run of each half otherwise), so
// every access is 16 bytes wide and no pair crosses lanes.  A workgroup takes
// whole tokens: where a token's keys go depends on kv_len and the page table
// (two dependent loads, and a bisection of q_start for ragged batches), which one
// lane per token looks up for all.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kernels.hpp"
#include "npu_device.hpp"
#include "plans.hpp"

namespace npu {

namespace {

constexpr int RT = 256;       // lanes of a workgroup
constexpr int MAX_TOK = 64;   // tokens of a workgroup, at most

__device__ __forceinline__ void rotate8(Frag16 &x, Frag16 &y, const float *cs, const float *sn, bool halves) {
  float a[16], c[8], s[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[2 * i] = __uint_as_float(x.u[i] << 16);
    a[2 * i + 1] = __uint_as_float(x.u[i] & 0xffff0000u);
    a[8 + 2 * i] = __uint_as_float(y.u[i] << 16);
    a[8 + 2 * i + 1] = __uint_as_float(y.u[i] & 0xffff0000u);
  }
  const f32x4 c0 = *reinterpret_cast<const f32x4 *>(cs), c1 = *reinterpret_cast<const f32x4 *>(cs + 4);
  const f32x4 s0 = *reinterpret_cast<const f32x4 *>(sn), s1 = *reinterpret_cast<const f32x4 *>(sn + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = c0[i], c[4 + i] = c1[i], s[i] = s0[i], s[4 + i] = s1[i];
  if (halves) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = a[i], v = a[8 + i];
      a[i] = u * c[i] - v * s[i];
      a[8 + i] = u * s[i] + v * c[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = a[2 * i], v = a[2 * i + 1];
      a[2 * i] = u * c[i] - v * s[i];
      a[2 * i + 1] = u * s[i] + v * c[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.u[i] = cvt_pk_bf16(a[2 * i], a[2 * i + 1]);
    y.u[i] = cvt_pk_bf16(a[8 + 2 * i], a[8 + 2 * i + 1]);
  }
}

__global__ __launch_bounds__(RT) void llama_rope_append_kernel(RopeAppendArgs a, int toks, int items, FastDiv per_tok,
                                                               int piece_log2) {
  __shared__ Place place[MAX_TOK];
  const int t0 = blockIdx.x * toks, nt = min(toks, a.b.T - t0);
  if ((int)threadIdx.x < nt) place[threadIdx.x] = place_of_token(a.b, t0 + threadIdx.x);
  __syncthreads();
  const int rot = a.width >> 3;  // pieces of a head that are rotated
  for (int i = threadIdx.x; i < nt * items; i += RT) {
    const int tl = per_tok.div(i), r = i - tl * items, head = r >> piece_log2, piece = r & ((1 << piece_log2) - 1);
    const Place p = place[tl];
    const long long t = t0 + tl;
    const bool turned = piece < rot && head < a.H + a.Hkv;
    // the two runs of this piece within the head
    const bool halves = a.pairs == 1 && piece < rot;
    const int e0 = halves ? piece * 8 : piece * 16, e1 = halves ? a.width + piece * 8 : piece * 16 + 8;
    const uint16_t *src;
    uint16_t *dst = nullptr;
    if (head < a.H) {
      src = a.Q + t * a.q_stride + head * a.dh;
      dst = a.Qo + t * a.o_stride + head * a.dh;
    } else {
      const bool is_k = head < a.H + a.Hkv;
      const int kh = head - a.H - (is_k ? 0 : a.Hkv);
      src = is_k ? a.K + t * a.k_stride + kh * a.dh : a.V + t * a.v_stride + kh * a.dh;
      if (p.page >= 0)
        dst = (is_k ? a.k_pages + p.page * a.kpage_stride : a.v_pages + p.page * a.vpage_stride) +
              (((long long)kh << a.b.page_log2) + p.in_page) * a.dh;
    }
    if (!dst) continue;
    Frag16 x = load16(src + e0), y = load16(src + e1);
    if (!p.live) {
      x = frag_zero();
      y = frag_zero();
    } else if (turned) {
      const long long at = (long long)p.pos * a.width + piece * 8;
      rotate8(x, y, a.cos_t + at, a.sin_t + at, halves);
    }
    *reinterpret_cast<u32x4 *>(dst + e0) = x.u;
    *reinterpret_cast<u32x4 *>(dst + e1) = y.u;
  }
}

}  // namespace

hipError_t launch_llama_rope_append(const RopeAppendArgs &a, hipStream_t s) {
  auto kern = llama_rope_append_kernel;
  const int piece_log2 = a.dh == 128 ? 3 : 2, items = (a.H + 2 * a.Hkv) << piece_log2;
  // whole tokens, at least two rounds of the workgroup's lanes' worth
  const int toks = std::min(MAX_TOK, std::max(1, 2 * RT / items));
  const int grid = (a.b.T + toks - 1) / toks;
  {
    npu_launch_plan p = make_plan("llama_rope_append", grid, wg_per_cu(kern, RT), grid, 16);
    const double runs = (double)toks * items;  // of 32 bytes
    p.load_phases = 4;  // kv_len, the page, the tables, the rows
    p.tile_valu = std::ceil(runs / 64) * 140.0;
    p.tile_lds_bytes = runs * sizeof(Place);
    p.tile_load_bytes = runs * (32.0 + 64.0);
    p.tile_store_bytes = runs * 32.0;
    p.hbm_bytes = (double)a.b.T * (items * 64.0 + a.width * 8.0);
    plans_add(p);
  }
  hipLaunchKernelGGL(kern, dim3(grid), dim3(RT), 0, s, a, toks, items, FastDiv(items), piece_log2);
  return hipGetLastError();
}

}  // namespace npu
