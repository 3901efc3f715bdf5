// k_mx_quantize.hip -- rows to microscaled blocks: as they are, gated, or out of a
// weight's columns; and the residual's addition and norm with such an output.
//
//   quantise: x, or x g / (1 + exp(-g)), in blocks of 32 (mx_device.hpp);
//   norm: h = bf16(x + delta), y = h / sqrt(mean(h^2) + eps) g, in blocks or bf16; the sum,
//   the root and the entries in 64 bits (whose range squares of bf16 and their roots do not leave).
//
// Everything is read once and written once.  A lane takes eight entries (16 bytes of
// bf16) and a quad a block, whose largest magnitude two DPP moves give.  The bytes bound
// them all where rows are many: 4099 rows of 14336 gated bf16 to e4m3 58.9 us, 5.0 TB/s.
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
// reciprocal (1 ulp).  Not below -87, where the reciprocal leaves f32's normal range: there a large x
// still makes numbers of it, in 64 bits.
constexpr float SILU_LEAST = -87.0f;
__device__ __forceinline__ float silu(float g) {
  constexpr float L = 1.44269502f, L_REST = 1.92596299e-8f, LN2 = 0.693147181f;
  const float c = __builtin_amdgcn_fmed3f(g, -87.0f, 87.0f), p = -c * L, r = fmaf(-c, L_REST, fmaf(-c, L, -p));
  const float e = __builtin_amdgcn_exp2f(p), d = fmaf(e, r * LN2, e);
  return g * __builtin_amdgcn_rcpf(1.0f + d);
}

// The same in 64 bits: exp(-g) = 2^n e^r, n = -g log2 e to the nearest, |r| < 0.347, by its Taylor
// series to r^13 (what is left is below 2^-56).  Below -700 no x makes a number of it, and -Inf is closed.
__device__ __forceinline__ double silu64(float gate) {
  if (gate < -700.0f) return -0.0;
  if (gate > 87.0f) return gate;
  const double g = gate, n = rint(-g * 1.4426950408889634), r = fma(-n, 0.6931471805599453, -g) - n * 2.3190468138462996e-17;
  double e = 1.0;
#pragma unroll
  for (int k = 13; k >= 1; --k) e = fma(e * (1.0 / k), r, 1.0);
  return g / (1.0 + ldexp(e, (int)n));
}

// Eight entries of a block from a lane, the block's other three lanes beside it.  upper(): the
// largest upper half of theirs in 64 bits (nullptr: they are exact).
template <int KIND, class Upper>
__device__ __forceinline__ void store_block(const float (&y)[8], Upper upper, uint8_t *q, uint8_t *scale, uint16_t *values) {
  uint32_t mag = quad_max(magnitude(y));
  if constexpr (!std::is_null_pointer_v<Upper>) {
    if (next_to_power(mag)) mag = from_upper(quad_max(upper()));
  }
  const uint32_t byte = scale_byte<KIND>(mag);
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
    auto gated64 = [&](int e) __attribute__((always_inline)) {
      return bf16_to_f32(static_cast<const uint16_t *>(a.x)[r * a.x_stride + k + e]) * silu64(bf16_to_f32(a.gate[r * a.gate_stride + k + e]));
    };
    if constexpr (GATE) {
      float g[8], least = 0.0f;
      unpack_bf16x8(load16(a.gate + r * a.gate_stride + k).u, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= silu(g[e]), least = fminf(least, g[e]);
      if (least < SILU_LEAST) {  // (4099 rows of 14336 where every wave has such a gate: 154 us, otherwise 49)
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const float v = (float)gated64(e);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = i == e ? v : y[i];
        }
      }
    }
    auto store = [&](auto upper) __attribute__((always_inline)) {
      store_block<KIND>(y, upper, a.q + r * a.q_stride + (KIND == kToE4m3 ? k : k >> 1), a.scale + r * a.scale_stride + (k >> 5),
                        a.values ? a.values + r * a.values_stride + k : nullptr);
    };
    if constexpr (GATE) {
      store([&]() __attribute__((always_inline)) {
        uint32_t m = 0;
#pragma unroll 1
        for (int e = 0; e < 8; ++e) m = max(m, upper_magnitude(gated64(e)));
        return m;
      });
    } else {
      store(nullptr);
    }
  }
}

// x with contiguous columns: entry (r, k) at k x_stride + r.  A workgroup takes 128 rows by 256
// k, a wave one block of k and a lane two neighbouring rows, so that its 32 loads are 256 bytes of a
// column each.  Elements and scales meet in LDS and leave as whole lines of rows, with the values
// made of them on the way out: 14336 x 4096 bf16 to e2m1 with values 60 us, 4.5 TB/s (from each lane's
// own block, 16 bytes of a line at a time, 145; a branch in each of the 32 loads 97; tiles in launch order
// 66).  A run's place in its row's LDS line turns with the row, which spreads both sides over the
// banks.
constexpr int CT = 512, CROWS = 128, CK = 256;

template <int KIND, bool F32>
__global__ __launch_bounds__(CT) void mx_quantize_columns_kernel(MxQuantizeArgs a, bool pairs, int tiles_k) {
  constexpr int RUNS = KIND == kToE4m3 ? 16 : 8, LINE = 16 * RUNS;  // runs of 16 bytes in a row's line
  __shared__ __attribute__((aligned(16))) uint8_t elements[CROWS * LINE];
  __shared__ __attribute__((aligned(8))) uint8_t scales[CROWS][CK / 32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // an XCD (every eighth workgroup) takes neighbours along k, whose lines of a row are neighbours
  const int all = gridDim.x, x = blockIdx.x & 7, pos = x * (all >> 3) + min(x, all & 7) + (blockIdx.x >> 3);
  const int tile_r = pos / tiles_k, k0 = (pos - tile_r * tiles_k) * CK, kb = k0 + 32 * wave;
  const long long r0 = (long long)tile_r * CROWS, r = r0 + 2 * lane;
  const int rows = (int)min((long long)CROWS, a.R - r0), width = min(CK, a.K - k0);
  if (kb < a.K && r < a.R) {
    float y[2][32];
    const bool both = r + 1 < a.R;
    const long long at = (long long)kb * a.x_stride + r;
    if constexpr (F32) {
      const float *p = static_cast<const float *>(a.x) + at;
      if (pairs && both) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float2 v = *reinterpret_cast<const float2 *>(p + j * a.x_stride);
          y[0][j] = v.x, y[1][j] = v.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) y[0][j] = p[j * a.x_stride], y[1][j] = p[j * a.x_stride + both];  // (the row itself again)
      }
    } else {
      const uint16_t *p = static_cast<const uint16_t *>(a.x) + at;
      uint32_t v[32];
      if (pairs && both) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = *reinterpret_cast<const uint32_t *>(p + j * a.x_stride);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = p[j * a.x_stride] | (uint32_t)p[j * a.x_stride + both] << 16;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) y[0][j] = __uint_as_float(v[j] << 16), y[1][j] = __uint_as_float(v[j] & 0xffff0000u);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 2 * lane + h;
      const uint32_t byte = scale_byte<KIND>(magnitude(y[h]));
      const float inv = inverse_scale(byte);
      const bool bad = byte == 255;
      scales[row][wave] = (uint8_t)byte;
#pragma unroll
      for (int q = 0; q < RUNS / 8; ++q) {  // runs of the block
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (KIND == kToE4m3) {
            const float *z = &y[h][16 * q + 4 * i];
            v[i] = pack_e4m3(z[0] * inv, z[1] * inv, z[2] * inv, z[3] * inv, bad);
          } else {
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = y[h][8 * i + e];
            v[i] = pack_e2m1(z, inv, bad);
          }
        }
        const int run = wave * (RUNS / 8) + q;
        *reinterpret_cast<u32x4 *>(elements + row * LINE + 16 * (run ^ (row & (RUNS - 1)))) = v;
      }
    }
  }
  __syncthreads();
  const int runs = width / (KIND == kToE4m3 ? 16 : 32), blocks = width / 32;
  for (int u = tid; u < CROWS * RUNS; u += CT) {
    const int row = u / RUNS, run = u % RUNS;
    if (row < rows && run < runs)
      *reinterpret_cast<u32x4 *>(a.q + (r0 + row) * a.q_stride + (KIND == kToE4m3 ? k0 : k0 / 2) + 16 * run) =
          *reinterpret_cast<const u32x4 *>(elements + row * LINE + 16 * (run ^ (row & (RUNS - 1))));
  }
  if (tid < rows) {
    uint8_t *to = a.scale + (r0 + tid) * a.scale_stride + k0 / 32;
    if (blocks == CK / 32 && ((uintptr_t)to & 7) == 0) {
      *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(scales[tid]);
    } else {
      for (int b = 0; b < blocks; ++b) to[b] = scales[tid][b];
    }
  }
  if (!a.values) return;
  for (int u = tid; u < CROWS * (CK / 8); u += CT) {
    const int row = u / (CK / 8), c = u % (CK / 8);  // eight entries
    if (row >= rows || 8 * c >= width) continue;
    const int bytes = KIND == kToE4m3 ? 8 : 4, run = c * bytes / 16;
    const uint8_t *from = elements + row * LINE + 16 * (run ^ (row & (RUNS - 1))) + c * bytes % 16;
    const float s = scale_of(scales[row][c / 4]);
    float v[8];
    if constexpr (KIND == kToE4m3)
      values_e4m3(*reinterpret_cast<const uint2 *>(from), s, v);
    else
      values_e2m1(*reinterpret_cast<const uint32_t *>(from), s, v);
    *reinterpret_cast<u32x4 *>(a.values + (r0 + row) * a.values_stride + k0 + 8 * c) = pack_bf16x8(v);
  }
}

__device__ __forceinline__ double wave_sum64(double v) {
  auto moved = [&](auto ctrl) __attribute__((always_inline)) {
    constexpr int C = decltype(ctrl)::value;
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), C, 0xf, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), C, 0xf, 0xf, false));
  };
  v += moved(std::integral_constant<int, 0xb1>{});   // lane ^ 1
  v += moved(std::integral_constant<int, 0x4e>{});   // lane ^ 2
  v += moved(std::integral_constant<int, 0x141>{});  // the other half of eight
  v += moved(std::integral_constant<int, 0x140>{});  // of sixteen
  auto of = [&](int l) __attribute__((always_inline)) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
  };
  return ((of(0) + of(16)) + of(32)) + of(48);
}

// h root g, rounded to odd: where it is no f32, that neighbour whose last bit is set, so that a
// further rounding to fewer bits gives what it would give of the exact value.  The products in 64 bits
// are off by some 2^-51 of it whatever the sizes of h, root and g; above f32's largest it is Inf.
__device__ __forceinline__ float scaled(float h, double root, float g) {
  const double y = (double)h * root * (double)g;
  const float z = (float)y;
  const double back = (double)z;
  const uint32_t cut = __float_as_uint(z) - (fabs(back) > fabs(y) ? 1u : 0u);
  return back == y || fabsf(z) == __builtin_inff() ? z : __uint_as_float(cut | 1u);
}

// One row by LPR lanes, CH runs of eight entries a lane, so that the row stays in registers between
// its sum and its scaling: 8191 rows of 4096 with h in and out and e4m3 48.6 us, 4.8 TB/s (46.8 with all in
// f32, and then now and then an element or a block's scale that is not the formula's; 48.2 with the entries in
// pairs of f32, which the ends of its range leave without their second half).
template <int KIND, int LPR, int CH>
__global__ __launch_bounds__(LPR < QT ? QT : LPR) void add_rmsnorm_kernel(AddRmsnormArgs a) {
  constexpr int WG = LPR < QT ? QT : LPR, ROWS = WG / LPR;
  __shared__ double part[LPR > 64 ? LPR / 64 : 1];
  const int t = threadIdx.x % LPR;
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / LPR;
  if (ROWS > 1 && row >= a.T) return;  // (whole waves, and no barrier below)
  float y[CH][8];
  double sum = 0.0;
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
    for (int e = 0; e < 8; ++e) sum = fma((double)y[c][e], (double)y[c][e], sum);
  }
  sum = wave_sum64(sum);
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < LPR / 64; ++w) sum += part[w];
  }
  // 1 / sqrt, the instruction's 24 bits and two of Newton's steps (0 and Inf as they are)
  const double mean = fma(sum, a.inv_D, (double)a.eps);
  double root = __builtin_amdgcn_rsq(mean);
  if (mean > 0.0 && mean < __builtin_inf()) {
#pragma unroll
    for (int i = 0; i < 2; ++i) root = root * fma(-0.5 * mean * root, root, 1.5);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = (c * LPR + t) * 8;
    if (k >= a.D) continue;
    const f32x4 g0 = *reinterpret_cast<const f32x4 *>(a.g + k), g1 = *reinterpret_cast<const f32x4 *>(a.g + k + 4);
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = scaled(y[c][e], root, e < 4 ? g0[e] : g1[e - 4]);
    if constexpr (KIND == kToBf16) {
      *reinterpret_cast<u32x4 *>(a.q + 2 * (row * a.q_stride + k)) = pack_bf16x8(z);
    } else {
      store_block<KIND>(z, nullptr, a.q + row * a.q_stride + (KIND == kToE4m3 ? k : k >> 1),
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
    const int tiles_k = (a.K + CK - 1) / CK, grid = (int)((a.R + (long long)CROWS - 1) / CROWS * tiles_k);
    auto kern = a.e4m3 ? (a.f32 ? mx_quantize_columns_kernel<kToE4m3, true> : mx_quantize_columns_kernel<kToE4m3, false>)
                       : (a.f32 ? mx_quantize_columns_kernel<kToE2m1, true> : mx_quantize_columns_kernel<kToE2m1, false>);
    const bool pairs = (uintptr_t)a.x % (a.f32 ? 8 : 4) == 0 && a.x_stride % 2 == 0;  // two rows' entries by one load
    plan("mx_quantize_columns", grid, wg_per_cu(kern, CT), 8.0);
    hipLaunchKernelGGL(kern, dim3(grid), dim3(CT), 0, s, a, pairs, tiles_k);
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
