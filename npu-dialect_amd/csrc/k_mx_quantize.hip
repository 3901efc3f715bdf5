// k_mx_quantize.hip -- rows to microscaled blocks: as they are, gated, or out of a
// weight's columns; and the residual's addition and norm with such an output.
//
//   quantise: x, or x g / (1 + exp(-g)), in blocks of 32 (mx_device.hpp);
//   norm: h = bf16(x + delta), y = h / sqrt(mean(h^2) + eps) g, in blocks or bf16.
//
// Everything is read once and written once.  A lane takes eight entries (16 bytes of
// bf16) and a quad a block, whose largest magnitude two DPP moves give.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kernels.hpp"
#include "mx_device.hpp"
#include "plans.hpp"

namespace npu {

namespace {

constexpr int QT = 256;  // lanes of a workgroup

// v / d for v below 2^31: (v m) >> (31 + l), l = ceil(log2 d), m = ceil(2^(31 + l) / d);
// m d - 2^(31 + l) < d <= 2^l keeps the quotient's error below v / 2^31 d < 1 / d.
struct Div31 {
  uint32_t d, m, sh;
  explicit Div31(uint32_t dv = 1) : d(dv), m(0), sh(0) {
    if (dv < 2) return;
    const uint32_t l = 32 - __builtin_clz(dv - 1);
    m = (uint32_t)(((1ULL << (31 + l)) + dv - 1) / dv);
    sh = l - 1;
  }
  __device__ __forceinline__ uint32_t div(uint32_t v) const { return d == 1 ? v : __umulhi(v, m) >> sh; }
};

// g / (1 + exp(-g)): exp(-g) = 2^p 2^r with p = -g log2 e rounded and r what the rounding
// (of the product and of log2 e) left, since 2^p alone would be off by |g| 2^-24; one
// reciprocal (1 ulp).  Below -87, where the reciprocal leaves f32's normal range, 0.
__device__ __forceinline__ float silu(float g) {
  constexpr float L = 1.44269502f, L_REST = 1.92596299e-8f, LN2 = 0.693147181f;
  const float c = __builtin_amdgcn_fmed3f(g, -87.0f, 87.0f), p = -c * L, r = fmaf(-c, L_REST, fmaf(-c, L, -p));
  const float e = __builtin_amdgcn_exp2f(p), d = fmaf(e, r * LN2, e);
  return g < -87.0f ? 0.0f : g * __builtin_amdgcn_rcpf(1.0f + d);
}

// Eight entries of a block from a lane, the block's other three lanes beside it.
template <int KIND>
__device__ __forceinline__ void store_block(const float (&y)[8], uint8_t *q, uint8_t *scale, uint16_t *values) {
  const uint32_t byte = scale_byte<KIND>(quad_max(magnitude(y)));
  const float inv = inverse_scale(byte);
  const bool bad = byte == 255;
  float v[8];
  if constexpr (KIND == kToE4m3) {
    const uint2 r = pack_e4m3x8(y, inv, bad);
    *reinterpret_cast<uint2 *>(q) = r;
    if (values) values_e4m3(r, scale_of(byte), v);
  } else {
    const uint32_t r = pack_e2m1(y, inv, bad);
    *reinterpret_cast<uint32_t *>(q) = r;
    if (values) values_e2m1(r, scale_of(byte), v);
  }
  if (values) *reinterpret_cast<u32x4 *>(values) = pack_bf16x8(v);
  if ((threadIdx.x & 3) == 0) *scale = (uint8_t)byte;
}

template <int KIND, bool F32, bool GATE>
__global__ __launch_bounds__(QT) void mx_quantize_kernel(MxQuantizeArgs a, Div31 per_row, uint32_t chunks) {
  const uint32_t row_chunks = (uint32_t)(a.K >> 3);
  for (uint32_t c = blockIdx.x * QT + threadIdx.x; c < chunks; c += gridDim.x * QT) {
    const uint32_t r = per_row.div(c), k = (c - r * row_chunks) * 8;
    float y[8];
    if constexpr (F32) {
      const float *p = static_cast<const float *>(a.x) + r * a.x_stride + k;
      const f32x4 u = *reinterpret_cast<const f32x4 *>(p), v = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = u[e], y[4 + e] = v[e];
    } else {
      const u32x4 u = load16(static_cast<const uint16_t *>(a.x) + r * a.x_stride + k).u;
      unpack_bf16x8(u, y);
    }
    if constexpr (GATE) {
      float g[8];
      unpack_bf16x8(load16(a.gate + r * a.gate_stride + k).u, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= silu(g[e]);
    }
    store_block<KIND>(y, a.q + r * a.q_stride + (KIND == kToE4m3 ? k : k >> 1), a.scale + r * a.scale_stride + (k >> 5),
                      a.values ? a.values + r * a.values_stride + k : nullptr);
  }
}

// x with contiguous columns: entry (r, k) at k x_stride + r.  A lane takes a block of a row,
// lanes side by side rows, and a wave one block place.
template <int KIND, bool F32>
__global__ __launch_bounds__(QT) void mx_quantize_columns_kernel(MxQuantizeArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long r = (long long)blockIdx.x * 64 + lane;
  const int b = blockIdx.y * (QT / 64) + wave;
  if (r >= a.R || b * 32 >= a.K) return;
  float y[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const long long at = (b * 32LL + j) * a.x_stride + r;
    y[j] = F32 ? static_cast<const float *>(a.x)[at] : bf16_to_f32(static_cast<const uint16_t *>(a.x)[at]);
  }
  const uint32_t byte = scale_byte<KIND>(magnitude(y));
  const float inv = inverse_scale(byte), s = scale_of(byte);
  const bool bad = byte == 255;
  uint8_t *q = a.q + r * a.q_stride + b * (KIND == kToE4m3 ? 32 : 16);
  a.scale[r * a.scale_stride + b] = (uint8_t)byte;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float z[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = y[8 * i + e];
    if constexpr (KIND == kToE4m3) {
      const uint2 p = pack_e4m3x8(z, inv, bad);
      *reinterpret_cast<uint2 *>(q + 8 * i) = p;
      if (a.values) values_e4m3(p, s, v);
    } else {
      const uint32_t p = pack_e2m1(z, inv, bad);
      *reinterpret_cast<uint32_t *>(q + 4 * i) = p;
      if (a.values) values_e2m1(p, s, v);
    }
    if (a.values) *reinterpret_cast<u32x4 *>(a.values + r * a.values_stride + b * 32 + 8 * i) = pack_bf16x8(v);
  }
}

// One row by LPR lanes, CH runs of eight entries a lane.
template <int KIND, int LPR, int CH>
__global__ __launch_bounds__(LPR < QT ? QT : LPR) void add_rmsnorm_kernel(AddRmsnormArgs a) {
  constexpr int WG = LPR < QT ? QT : LPR, ROWS = WG / LPR;
  __shared__ float part[LPR > 64 ? LPR / 64 : 1];
  const int t = threadIdx.x % LPR;
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / LPR;
  if (ROWS > 1 && row >= a.T) return;  // (whole waves, and no barrier below)
  float y[CH][8];
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = (c * LPR + t) * 8;
    if (k >= a.D) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[c][e] = 0.0f;
      continue;
    }
    u32x4 u = load16(a.x + row * a.x_stride + k).u;
    unpack_bf16x8(u, y[c]);
    if (a.delta) {
      float d[8];
      unpack_bf16x8(load16(a.delta + row * a.delta_stride + k).u, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[c][e] += d[e];
      u = pack_bf16x8(y[c]);  // the norm is of what the next layer adds to
      unpack_bf16x8(u, y[c]);
    }
    if (a.h) *reinterpret_cast<u32x4 *>(a.h + row * a.h_stride + k) = u;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(y[c][e], y[c][e], sum);
  }
  sum = wave_sum(sum);
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < LPR / 64; ++w) sum += part[w];
  }
  const float r = 1.0f / sqrtf(sum / (float)a.D + a.eps);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = (c * LPR + t) * 8;
    if (k >= a.D) continue;
    const f32x4 g0 = *reinterpret_cast<const f32x4 *>(a.g + k), g1 = *reinterpret_cast<const f32x4 *>(a.g + k + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[c][e] = y[c][e] * r * (e < 4 ? g0[e] : g1[e - 4]);
    if constexpr (KIND == kToBf16) {
      *reinterpret_cast<u32x4 *>(a.q + 2 * (row * a.q_stride + k)) = pack_bf16x8(y[c]);
    } else {
      store_block<KIND>(y[c], a.q + row * a.q_stride + (KIND == kToE4m3 ? k : k >> 1),
                        a.scale + row * a.scale_stride + (k >> 5), nullptr);
    }
  }
}

template <int KIND>
hipError_t add_rmsnorm(const AddRmsnormArgs &a, hipStream_t s) {
  // a wave for a row where it fits in one, then as many lanes as give each at most four runs
  auto run = [&](auto kern, int lpr) {
    const int wg = std::max(lpr, QT), rows = wg / lpr, grid = (int)(((long long)a.T + rows - 1) / rows);
    npu_launch_plan p = make_plan("llama_add_rmsnorm", grid, wg_per_cu(kern, wg), grid, 16);
    const double n = (double)rows * a.D, in = a.delta ? 4.0 : 2.0;
    p.unit_waves = wg / 64;
    p.load_phases = 2;
    p.tile_valu = n / 64 * 10.0;
    p.tile_lds_bytes = lpr > 64 ? wg / 16.0 : 0.0;
    p.tile_load_bytes = n * (in + 4.0);
    p.tile_store_bytes = n * ((a.h ? 2.0 : 0.0) + (KIND == kToBf16 ? 2.0 : KIND == kToE4m3 ? 1.03 : 0.53));
    p.hbm_bytes = (double)a.T * a.D * in + a.D * 4.0 + grid * p.tile_store_bytes;
    plans_add(p);
    hipLaunchKernelGGL(kern, dim3(grid), dim3(wg), 0, s, a);
    return hipGetLastError();
  };
  if (a.D <= 512) return run(add_rmsnorm_kernel<KIND, 64, 1>, 64);
  if (a.D <= 2048) return run(add_rmsnorm_kernel<KIND, 256, 1>, 256);
  if (a.D <= 4096) return run(add_rmsnorm_kernel<KIND, 256, 2>, 256);
  if (a.D <= 8192) return run(add_rmsnorm_kernel<KIND, 256, 4>, 256);
  if (a.D <= 16384) return run(add_rmsnorm_kernel<KIND, 512, 4>, 512);
  return run(add_rmsnorm_kernel<KIND, 1024, 4>, 1024);
}

}  // namespace

hipError_t launch_add_rmsnorm(const AddRmsnormArgs &a, hipStream_t s) {
  return a.kind == kToBf16 ? add_rmsnorm<kToBf16>(a, s) : a.kind == kToE4m3 ? add_rmsnorm<kToE4m3>(a, s) : add_rmsnorm<kToE2m1>(a, s);
}

hipError_t launch_mx_quantize(const MxQuantizeArgs &a, hipStream_t s) {
  const double n = (double)a.R * a.K, in = (a.f32 ? 4.0 : 2.0) + (a.gate ? 2.0 : 0.0);
  const double out = (a.e4m3 ? 1.0 : 0.5) + 1.0 / 32 + (a.values ? 2.0 : 0.0);
  auto plan = [&](const char *name, int grid, int per_cu, double valu) {
    npu_launch_plan p = make_plan(name, grid, per_cu, grid, 16);
    p.tile_valu = valu * n / 64 / grid;
    p.tile_load_bytes = n * in / grid;
    p.tile_store_bytes = n * out / grid;
    p.hbm_bytes = n * (in + out);
    plans_add(p);
  };
  if (a.columns) {
    const dim3 grid((unsigned)((a.R + 63) / 64), (unsigned)((a.K / 32 + QT / 64 - 1) / (QT / 64)));
    auto kern = a.e4m3 ? (a.f32 ? mx_quantize_columns_kernel<kToE4m3, true> : mx_quantize_columns_kernel<kToE4m3, false>)
                       : (a.f32 ? mx_quantize_columns_kernel<kToE2m1, true> : mx_quantize_columns_kernel<kToE2m1, false>);
    plan("mx_quantize_columns", (int)(grid.x * grid.y), wg_per_cu(kern, QT), 8.0);
    hipLaunchKernelGGL(kern, grid, dim3(QT), 0, s, a);
    return hipGetLastError();
  }
  const uint32_t chunks = (uint32_t)((long long)a.R * a.K / 8);
  auto kern = a.e4m3 ? (a.gate ? mx_quantize_kernel<kToE4m3, false, true>
                               : a.f32 ? mx_quantize_kernel<kToE4m3, true, false> : mx_quantize_kernel<kToE4m3, false, false>)
                     : (a.gate ? mx_quantize_kernel<kToE2m1, false, true>
                               : a.f32 ? mx_quantize_kernel<kToE2m1, true, false> : mx_quantize_kernel<kToE2m1, false, false>);
  const int grid = (int)std::min<long long>((chunks + QT - 1LL) / QT, 16LL * device_cus());
  plan("mx_quantize", grid, wg_per_cu(kern, QT), a.gate ? 14.0 : 5.0);
  hipLaunchKernelGGL(kern, dim3(grid), dim3(QT), 0, s, a, Div31((uint32_t)(a.K >> 3)), chunks);
  return hipGetLastError();
}

}  // namespace npu
