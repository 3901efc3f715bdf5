// k_mx_matmul.hip -- products of microscaled blocks: out[m][n] = sum_k a[m][k] w[n][k],
// a in e4m3 or e2m1, w in e2m1, bf16 out.
//
// One instruction, v_mfma_scale_f32_16x16x128_f8f6f4, takes a step of 128 k with both operands'
// scales: of an e2m1 operand lane l holds row l % 16's block l / 16 (16 bytes), of an e4m3
// one the row's 16-byte runs l / 16 and 4 + l / 16, and of a scale operand that block's
// byte.  w goes first, so that a lane gets four neighbouring n of one m.
//
// Few rows: the weights' bytes bound it.  A workgroup takes 16 n and up to 64 m, its eight
// waves a share of k each, straight from memory to registers, and their sums meet in LDS.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "kernels.hpp"
#include "mx_device.hpp"
#include "plans.hpp"

namespace npu {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 operand(u32x4 lo, u32x4 hi) {
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
__device__ __forceinline__ i32x8 operand(u32x4 lo) { return operand(lo, u32x4{0, 0, 0, 0}); }
// acc += w a over a step; the scales' low bytes count.
template <bool E4M3>
__device__ __forceinline__ f32x4 mma(i32x8 w, i32x8 a, f32x4 acc, int ws, int as) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 4, E4M3 ? 0 : 4, 0, ws, 0, as);
}

__device__ __forceinline__ uint64_t pack_bf16x4(f32x4 v) {
  return (uint64_t)cvt_pk_bf16(v[2], v[3]) << 32 | cvt_pk_bf16(v[0], v[1]);
}
// out[0..3] = v, of which n exist.
__device__ __forceinline__ void store4(uint16_t *out, f32x4 v, int n) {
  const uint64_t b = pack_bf16x4(v);
  if (n >= 4 && ((uintptr_t)out & 7) == 0) {
    *reinterpret_cast<uint64_t *>(out) = b;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) out[e] = (uint16_t)(b >> (16 * e));
  }
}

constexpr int SW = 8;  // waves of a workgroup

template <bool E4M3, int MT>
__global__ __launch_bounds__(SW * 64) void mx_matmul_few_kernel(MxMatmulArgs a, int steps, int per_wave) {
  __shared__ f32x4 sums[SW][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const long long n0 = (long long)blockIdx.x * 16, m0 = (long long)blockIdx.y * (16 * MT);
  // (rows past the last: its own again, not stored)
  const long long wr = min(n0 + r, (long long)a.N - 1);
  const uint8_t *w = a.w + wr * a.w_stride, *ws = a.w_scale + wr * a.ws_stride;
  const uint8_t *x[MT], *xs[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const long long mr = min(m0 + 16 * t + r, (long long)a.M - 1);
    x[t] = a.a + mr * a.a_stride;
    xs[t] = a.a_scale + mr * a.as_stride;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int blocks = a.K / 32, s1 = min(steps, (wave + 1) * per_wave);
#pragma unroll 4
  for (int s = wave * per_wave; s < s1; ++s) {
    // block g of the step; past the row's end zeros of scale 2^-127
    const int b = 4 * s + g;
    const u32x4 zero = u32x4{0, 0, 0, 0};
    const bool in = b < blocks;
    const int bc = in ? b : 0;
    const u32x4 wv = masked(load16(w + 16LL * bc).u, in);
    const int wsc = in ? ws[bc] : 0;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      u32x4 lo, hi = zero;
      if constexpr (E4M3) {
        const int b0 = 4 * s + (g >> 1), b1 = b0 + 2;
        lo = masked(load16(x[t] + 32LL * (b0 < blocks ? b0 : 0) + 16 * (g & 1)).u, b0 < blocks);
        hi = masked(load16(x[t] + 32LL * (b1 < blocks ? b1 : 0) + 16 * (g & 1)).u, b1 < blocks);
      } else {
        lo = masked(load16(x[t] + 16LL * bc).u, in);
      }
      const int xsc = in ? xs[t][bc] : 0;
      acc[t] = mma<E4M3>(operand(wv), operand(lo, hi), acc[t], wsc, xsc);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < MT; t += SW) {
    f32x4 v = sums[0][t][lane];
#pragma unroll
    for (int i = 1; i < SW; ++i) v += sums[i][t][lane];
    const long long m = m0 + 16 * t + r, n = n0 + 4 * g;
    if (m < a.M && n < a.N) store4(a.out + m * a.out_stride + n, v, (int)min(4LL, a.N - n));
  }
}

template <bool E4M3>
hipError_t matmul_few(const MxMatmulArgs &a, hipStream_t s) {
  const int steps = (a.K + 127) / 128, per_wave = (steps + SW - 1) / SW;
  auto run = [&](auto kern, int mt) {
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 16 * mt - 1) / (16 * mt)));
    const int total = (int)std::min(2147483647.0, (double)grid.x * grid.y);
    npu_launch_plan p = make_plan("mx_matmul_few", total, wg_per_cu(kern, SW * 64), total, 8);
    p.unit_waves = SW;
    p.tile_macs = 256.0 * mt * a.K;
    p.tile_valu = steps * (8.0 + 12.0 * mt);
    p.tile_lds_bytes = 2.0 * SW * mt * 1024;
    p.tile_load_bytes = 16.0 * a.K * (0.53 + mt * (E4M3 ? 1.03 : 0.53));
    p.tile_store_bytes = 512.0 * mt;
    p.hbm_bytes = (double)a.K * (a.M * (E4M3 ? 1.03 : 0.53) + a.N * 0.53) + 2.0 * a.M * a.N;
    plans_add(p);
    hipLaunchKernelGGL(kern, grid, dim3(SW * 64), 0, s, a, steps, per_wave);
    return hipGetLastError();
  };
  if (a.M <= 16) return run(mx_matmul_few_kernel<E4M3, 1>, 1);
  if (a.M <= 32) return run(mx_matmul_few_kernel<E4M3, 2>, 2);
  return run(mx_matmul_few_kernel<E4M3, 4>, 4);
}

}  // namespace

size_t mx_matmul_workspace(int, int, int) { return 16; }

hipError_t launch_mx_matmul(const MxMatmulArgs &a, hipStream_t s) {
  return a.e4m3 ? matmul_few<true>(a, s) : matmul_few<false>(a, s);
}

}  // namespace npu
