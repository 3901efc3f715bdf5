// k_mx_matmul.hip -- products of microscaled blocks: out[m][n] = sum_k a[m][k] w[n][k],
// a in e4m3 or e2m1, w in e2m1, bf16 out.
//
// One instruction, v_mfma_scale_f32_16x16x128_f8f6f4, takes a step of 128 k with both operands'
// scales: of an e2m1 operand lane l holds row l % 16's block l / 16 (16 bytes), of an e4m3
// one the row's 16-byte runs l / 16 and 4 + l / 16, and of a scale operand that block's
// byte.  w goes first, so that a lane gets four neighbouring n of one m.  e2m1 by e2m1 is summed
// as f32 sums are; with an e4m3 operand the instruction lines the terms of each eight neighbouring k up to
// the largest of the eight and cuts off what is less than 2^-13 of it (the eights' sums are added in f32).
// That stays: 2e-5 of a result of usual rows, far below its rounding to bf16 and the elements' own 2^-4, and
// no other instruction takes e4m3 by e2m1 with the blocks' scales.
//
// Few rows are bound by w's bytes and by what a CU's L1 passes on: 48 rows of e4m3 by 14336 x 4096
// 10.7 us (1 row 6.9, 4.4 TB/s of w), one by 4096 x 4096 4.1, half of it launch.  These are of w in the last-level
// cache; where weights change by more than that holds, 14.9, 8.4 and 5.7.  Many rows: 8192^3 e2m1 267 us,
// 4.1 PFLOP/s, the matrix units busy in 51 % of the clocks, at 1.95 GHz, without any loads of its operands 228;
// 4099 rows of e4m3 by 4096 x 14336 177 us, 2.7 PFLOP/s, busy in 64 % at 2.1 GHz.  How much of the rest is waits for
// operands, and how much of the clock power, was not told apart.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "kernels.hpp"
#include "mx_columns.hpp"
#include "mx_device.hpp"
#include "plans.hpp"

namespace npu {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 operand(u32x4 lo, u32x4 hi) {
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
__device__ __forceinline__ i32x8 operand(u32x4 lo) { return operand(lo, u32x4{0, 0, 0, 0}); }
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

// Where K is divided over workgroups (blockIdx.y), each one's sums go to the workspace, f32
// [parts][M][N4], N4 = N up to a multiple of 4, and a last kernel adds them in order.
__device__ __forceinline__ void put(const MxMatmulArgs &a, float *parts, long long m, long long n, f32x4 v) {
  if (m >= a.M || n >= a.N) return;
  if (parts) {
    const long long width = ((long long)a.N + 3) & ~3LL;
    *reinterpret_cast<f32x4 *>(parts + (blockIdx.y * (long long)a.M + m) * width + n) = v;
  } else {
    store4(a.out + m * a.out_stride + n, v, (int)min(4LL, a.N - n));
  }
}
__global__ __launch_bounds__(256) void mx_join_kernel(MxMatmulArgs a, const float *parts, int n_parts) {
  const int width = (a.N + 3) >> 2;
  const long long all = (long long)a.M * width, i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= all) return;
  const f32x4 *p = reinterpret_cast<const f32x4 *>(parts) + i;
  f32x4 v = p[0];
  for (int q = 1; q < n_parts; ++q) v += p[q * all];
  const long long m = i / width, n = 4 * (i - m * width);
  store4(a.out + m * a.out_stride + n, v, (int)min(4LL, a.N - n));
}

// ---- few rows ---------------------------------------------------------------------------
constexpr int SW = 8;  // waves of a workgroup

// The scales of a row's blocks b .. b + 3 (0 past its end), b = 4 (first step) + 4 g for lane group
// g, to the byte of block 4j + g for step j: a 4 x 4 transpose of bytes over the lane groups.
__device__ __forceinline__ int scales_by_step(uint32_t x, uint32_t pick) {
  const LanePair h = lane_pair32(__uint_as_float(x));
  const LanePair a = lane_pair16(h.lo), b = lane_pair16(h.hi);
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(a.hi), __float_as_uint(a.lo), pick);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(b.hi), __float_as_uint(b.lo), pick);
  return (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
// Four bytes from b on of a row of `blocks`: a load at any address, of the row's last four where
// it would pass the end.
struct ScaleWord {
  int at, shift;
  uint32_t keep;
  __device__ __forceinline__ ScaleWord(int b, int blocks) {
    const int over = min(max(b + 4 - blocks, 0), 4);
    at = over < 4 ? b - over : blocks - 4;
    shift = over < 4 ? 8 * over : 0;
    keep = over < 4 ? ~0u : 0u;
  }
  __device__ __forceinline__ uint32_t load(const uint8_t *row) const {
    uint32_t v;
    __builtin_memcpy(&v, row + at, 4);
    return v;
  }
  __device__ __forceinline__ uint32_t of(uint32_t v) const { return (v & keep) >> shift; }
  __device__ __forceinline__ uint32_t of(const uint8_t *row) const { return of(load(row)); }
};
__device__ __forceinline__ uint32_t scale_bytes(const uint8_t *row, int b, int blocks) {  // rows of less than four
  uint32_t v = 0;
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (b + e < blocks) v |= (uint32_t)row[b + e] << (8 * e);
  return v;
}

// acc += w a over a step; of the scales' bytes that of STEP counts.
template <bool E4M3, int STEP>
__device__ __forceinline__ f32x4 mma_step(i32x8 w, i32x8 a, f32x4 acc, int ws, int as) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 4, E4M3 ? 0 : 4, STEP, ws, STEP, as);
}

template <bool E4M3, int MT, int NT>
__global__ __launch_bounds__(SW * 64, NT *MT >= 3 ? 2 : 4) void mx_matmul_few_kernel(MxMatmulArgs a, int groups_m, int steps, int per_wave, float *parts) {
  extern __shared__ f32x4 sums[];  // [SW][MT NT][64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int bn = blockIdx.x / groups_m, bm = blockIdx.x - bn * groups_m;
  const FewColumns columns(bn, NT, a.N);
  const long long n0 = columns.n0, m0 = (long long)bm * (16 * MT);
  const int blocks = a.K / 32, s0 = (blockIdx.y * SW + wave) * per_wave, s1 = min(steps, s0 + per_wave);
  // Rows past the last: its own again, not stored.  (offsets fit 32 bits: strides are below 2^23)
  const uint8_t *w = a.w + n0 * a.w_stride, *ws = a.w_scale + n0 * a.ws_stride, *x = a.a + m0 * a.a_stride, *xs = a.a_scale + m0 * a.as_stride;
  uint32_t w_at[NT], ws_at[NT], x_at[MT], xs_at[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = columns.row(t, r);
    w_at[t] = (uint32_t)row * (uint32_t)a.w_stride;
    ws_at[t] = (uint32_t)row * (uint32_t)a.ws_stride;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int row = (int)min((long long)(16 * t + r), a.M - 1 - m0);
    x_at[t] = (uint32_t)row * (uint32_t)a.a_stride;
    xs_at[t] = (uint32_t)row * (uint32_t)a.as_stride;
  }
  // A load takes 64 bytes of each of 16 rows, half a line.  All the same half costs the L1 as much as
  // whole lines, so of each two such loads odd rows' halves come in the other order (48 rows by
  // 14336 x 4096: a sixth less time; sixteen rows are a whole number of lines apart).
  const bool w_odd = (r ^ (int)(((uintptr_t)w + (uint32_t)r * (uint32_t)a.w_stride) >> 6)) & 1;
  const bool x_odd = (r ^ (int)(((uintptr_t)x + (uint32_t)r * (uint32_t)a.a_stride) >> 6)) & 1;
  auto load_line = [&](const uint8_t *rows, uint32_t row, int at, int end, bool odd, u32x4 &first, u32x4 &second) __attribute__((always_inline)) {
    // (past a row's end its first bytes again, whose scales are 2^-127: such a product is below 2^-200)
    const int p = at + 16 * g + (odd ? 64 : 0), q = p ^ 64;
    first = load16(rows + (row + (uint32_t)(p < end ? p : 0))).u;
    second = load16(rows + (row + (uint32_t)(q < end ? q : 0))).u;
  };
  auto in_order = [&](bool odd, u32x4 &first, u32x4 &second) __attribute__((always_inline)) {
    const u32x4 f = first;
#pragma unroll
    for (int e = 0; e < 4; ++e) first[e] = odd ? second[e] : f[e], second[e] = odd ? f[e] : second[e];
  };
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t pick = 0x0c0c0400u + 0x0101u * (uint32_t)g;  // byte g of each of two
#pragma unroll 1
  for (int s = s0; s < s1; s += 4) {
    // the scales first, since they have to change places, then four steps of w and two of a
    uint32_t was[NT], xas[MT];
    const int b = 4 * s + 4 * g;
    if (blocks >= 4) {
      const ScaleWord word(b, blocks);
#pragma unroll
      for (int t = 0; t < NT; ++t) was[t] = word.of(ws + ws_at[t]);
#pragma unroll
      for (int t = 0; t < MT; ++t) xas[t] = word.of(xs + xs_at[t]);
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) was[t] = scale_bytes(ws + ws_at[t], b, blocks);
#pragma unroll
      for (int t = 0; t < MT; ++t) xas[t] = scale_bytes(xs + xs_at[t], b, blocks);
    }
    const bool more = s + 2 < s1;  // (a wave has whole pairs of steps)
    u32x4 wv[4][NT], av[4][MT];    // av: of e4m3 the halves of two steps
    auto load_w = [&](auto j) __attribute__((always_inline)) {
      constexpr int J = decltype(j)::value;
#pragma unroll
      for (int t = 0; t < NT; ++t) load_line(w, w_at[t], 64 * (s + J), a.K / 2, w_odd, wv[J][t], wv[J + 1][t]);
    };
    auto load_a = [&](auto j) __attribute__((always_inline)) {
      constexpr int J = decltype(j)::value, AT = E4M3 ? 2 * (J & 1) : J;
      if constexpr (E4M3 || J % 2 == 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
          load_line(x, x_at[i], (E4M3 ? 128 : 64) * (s + J), E4M3 ? a.K : a.K / 2, x_odd, av[AT][i], av[AT + 1][i]);
      }
    };
    load_w(std::integral_constant<int, 0>{});
    if (more) load_w(std::integral_constant<int, 2>{});
    load_a(std::integral_constant<int, 0>{});
    load_a(std::integral_constant<int, 1>{});
    if constexpr (!E4M3) {
      if (more) load_a(std::integral_constant<int, 2>{});
    }
    __builtin_amdgcn_sched_barrier(0);
    int wsc[NT], xsc[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) wsc[t] = scales_by_step(was[t], pick);
#pragma unroll
    for (int t = 0; t < MT; ++t) xsc[t] = scales_by_step(xas[t], pick);
    auto products = [&](auto j) __attribute__((always_inline)) {
      constexpr int J = decltype(j)::value, AT = E4M3 ? 2 * (J & 1) : J;
      if constexpr (J % 2 == 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) in_order(w_odd, wv[J][t], wv[J + 1][t]);
      }
      if constexpr (E4M3 || J % 2 == 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i) in_order(x_odd, av[AT][i], av[E4M3 || AT < 3 ? AT + 1 : AT][i]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[i][t] = mma_step<E4M3, J>(operand(wv[J][t]), E4M3 ? operand(av[AT][i], av[E4M3 ? AT + 1 : AT][i]) : operand(av[AT][i]),
                                        acc[i][t], wsc[t], xsc[i]);
      __builtin_amdgcn_sched_barrier(0);
    };
    products(std::integral_constant<int, 0>{});
    if constexpr (E4M3) {
      if (more) load_a(std::integral_constant<int, 2>{});
    }
    products(std::integral_constant<int, 1>{});
    if (!more) break;
    if constexpr (E4M3) load_a(std::integral_constant<int, 3>{});
    products(std::integral_constant<int, 2>{});
    products(std::integral_constant<int, 3>{});
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[(wave * (MT * NT) + i * NT + t) * 64 + lane] = acc[i][t];
  __syncthreads();
  for (int it = wave; it < MT * NT; it += SW) {
    f32x4 v = sums[it * 64 + lane];
#pragma unroll
    for (int q = 1; q < SW; ++q) v += sums[(q * (MT * NT) + it) * 64 + lane];
    put(a, parts, m0 + 16 * (it / NT) + r, columns.first(it % NT, g), v);
  }
}

// ---- many rows: tiles through LDS -----------------------------------------------------
// The scales come in the order that the instructions take them from a first kernel: for a chunk
// of 512 k, lane group g and row a word with the scales of the row's blocks 4j + g, j = 0 .. 3, a
// byte each (0 past the row's end), rows filled up to whole tiles.  A wave's load of them is
// four runs of 64 bytes; from the rows themselves it was sixteen requests of 16 bytes, as
// many in all as the elements took, and the L2's rate of requests was the bound.  Small tiles, of
// which a call has few, make their own words in LDS, for OWN chunks at a time: the first kernel's 4 us
// are more.
constexpr int TILE = 256;  // rows are filled up to a multiple of this

__global__ __launch_bounds__(256) void mx_scales_kernel(MxMatmulArgs a, uint32_t *a_out, uint32_t *w_out, int a_rows, int w_rows, int chunks) {
  const int blocks = a.K / 32;
  int row = blockIdx.x * 256 + threadIdx.x;
  const bool is_a = row < a_rows;
  if (!is_a) row -= a_rows;
  const int rows = is_a ? a.M : a.N, padded = is_a ? a_rows : w_rows;
  const uint8_t *p = is_a ? a.a_scale + row * a.as_stride : a.w_scale + row * a.ws_stride;
  uint32_t *out = (is_a ? a_out : w_out) + row;
  for (int c = blockIdx.y * 8; c < min(chunks, (int)blockIdx.y * 8 + 8); ++c) {
    uint32_t x[4] = {0, 0, 0, 0};  // of step j
    if (row < rows) {
      if (16 * c + 16 <= blocks) {
        __builtin_memcpy(x, p + 16 * c, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (16 * c + e < blocks) x[e / 4] |= (uint32_t)p[16 * c + e] << (8 * (e % 4));
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t pick = 0x0c0c0400u + 0x0101u * g;  // byte g of each of two
      const uint32_t lo = __builtin_amdgcn_perm(x[1], x[0], pick), hi = __builtin_amdgcn_perm(x[3], x[2], pick);
      out[(long long)(4 * c + g) * padded] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
  }
}

// A stage is one step (e4m3) or two (e2m1) of a BM x BN tile, brought to LDS by loads that
// pass no registers, NBUF stages in turn.  Rows are 128 bytes long where they can be (whole
// lines: half of one costs the L2 as much), their 16-byte runs exchanged so that the 16 lanes that
// ds_read_b128 serves together ({0-3, 12-15, 20-23, 24-27} of each half wave, and the rest)
// read 16 different sixteenths of the banks.
__device__ __forceinline__ int swap64(int row) { return (-(row >> 2)) & 3; }
__device__ __forceinline__ int swap128(int row) { return (row & 2) | (row >> 1 & 4); }  // 2 (h & 1) + 4 (h >> 2), h = row / 2 % 8

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef const __attribute__((address_space(1))) uint8_t global_u8;

__device__ __forceinline__ u32x4 read_lds(const uint8_t *p) { return *reinterpret_cast<const u32x4 *>(p); }

// All but the N latest loads, and the reads of LDS before a barrier.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// Tiles in an order in which those that run at a time on an XCD (which takes every eighth
// workgroup) are neighbours: XCDs take runs of it, in groups of 8 tiles along m.
struct TileOrder {
  int tiles_m, tiles_n;
  __device__ __forceinline__ void at(int bid, int &tm, int &tn) const {
    const int all = tiles_m * tiles_n, x = bid & 7, i = bid >> 3, per = all >> 3, more = all & 7;
    const int pos = x * per + min(x, more) + i;
    const int group = pos / (8 * tiles_n), first = group * 8, wide = min(8, tiles_m - first), in = pos - first * tiles_n;
    tn = in / wide;
    tm = first + in - tn * wide;
  }
};

// Loads of a stage go out spread between the products of an earlier one: all at once they held up
// the wave (8192^3 e2m1 308 us, so 276; with stages of 64-byte rows and scales from the rows 422).
// The scales' words too come to LDS by such loads, a chunk ahead: taken through registers they
// had the compiler wait for every load under way, once a chunk (276 us; 267 so; 512 rows of e4m3 by
// 4096 x 4096 in tiles of 64 18.4, of 64 x 128 13.8 so).
template <bool E4M3, int BM, int BN, int WM, int WN, int NBUF, int OWN>
__global__ __launch_bounds__(WM *WN * 64) void mx_matmul_tile_kernel(MxMatmulArgs a, TileOrder order, const uint32_t *a_scales,
                                                                     const uint32_t *w_scales, int a_rows, int w_rows, int part_chunks,
                                                                     float *parts) {
  constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, SPS = E4M3 ? 1 : 2;
  constexpr int AROW = 128, WROW = E4M3 ? 64 : 128, ABYTES = BM * AROW, STAGE = ABYTES + BN * WROW;
  constexpr int PA = ABYTES / 1024, PIECES = STAGE / 1024 / NW;
  constexpr int EACH = (PIECES + TM - 1) / TM;  // loads of a row of tiles
  constexpr int ROWS = BM + BN, PITCH = OWN ? ROWS + 4 : ROWS;  // of the scales' words, a line for each lane group of a chunk
  static_assert(STAGE % (1024 * NW) == 0 && PA % NW == 0, "whole loads for every wave");
  static_assert(OWN || ROWS * 16 == NW * 1024, "a load of a chunk's words for every wave");
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int wm = wave % WM, wn = wave / WM;
  int tm, tn;
  order.at(blockIdx.x, tm, tn);
  const long long m0 = (long long)tm * BM, n0 = (long long)tn * BN;
  // this part's chunks of 512 k and stages, of which the row has `all`
  const int c0 = blockIdx.y * part_chunks, chunks = min(part_chunks, (a.K + 511) / 512 - c0), s0 = c0 * (4 / SPS);
  const int a_bytes = E4M3 ? a.K : a.K / 2, w_bytes = a.K / 2, all = (a.K + 128 * SPS - 1) / (128 * SPS), stages = min(all - s0, chunks * (4 / SPS));
  // (offsets within a tile fit 32 bits: the launcher sees to it)
  const int last_m = (int)min((long long)BM, a.M - m0) - 1, last_n = (int)min((long long)BN, a.N - n0) - 1;
  const uint8_t *a_tile = a.a + m0 * a.a_stride, *w_tile = a.w + n0 * a.w_stride;
  // this lane's part of each load: 16 bytes of a row, at bytes `off` of each stage's part
  uint32_t src[PIECES];
  int off[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int p = wave + i * NW;
    if (i < PA / NW) {
      const int row = p * 8 + (lane >> 3);
      off[i] = 16 * ((lane & 7) ^ swap128(row));
      src[i] = (uint32_t)min(row, last_m) * (uint32_t)a.a_stride;
    } else {
      const int row = E4M3 ? (p - PA) * 16 + (lane >> 2) : (p - PA) * 8 + (lane >> 3);
      off[i] = E4M3 ? 16 * ((lane & 3) ^ swap64(row)) : 16 * ((lane & 7) ^ swap128(row));
      src[i] = (uint32_t)min(row, last_n) * (uint32_t)a.w_stride;
    }
  }
  // (past a row's end its first bytes again, whose scales are 2^-127: such a product is below 2^-200)
  auto load = [&](int s, int buf, auto piece) __attribute__((always_inline)) {
    constexpr int i = decltype(piece)::value;
    constexpr bool of_a = i < PA / NW;
    int at = off[i] + (s0 + s) * (of_a ? AROW : WROW);
    at = at < (of_a ? a_bytes : w_bytes) ? at : 0;
    __builtin_amdgcn_global_load_lds((global_u8 *)((of_a ? a_tile : w_tile) + (src[i] + (uint32_t)at)),
                                     (lds_u8 *)(lds + buf * STAGE + (wave + i * NW) * 1024), 16, 0, 0);
  };
  uint32_t *words = reinterpret_cast<uint32_t *>(lds + NBUF * STAGE);  // of OWN chunks, or of two
  // chunk c's words from the first kernel's: four rows of a lane group a lane
  const int line = (wave * 256 + lane * 4) / ROWS, line_at = (wave * 256 + lane * 4) % ROWS;
  const uint32_t *words_at = line_at < BM ? a_scales + (4LL * c0 + line) * a_rows + m0 + line_at
                                          : w_scales + (4LL * c0 + line) * w_rows + n0 + (line_at - BM);
  const long long words_step = 4LL * (line_at < BM ? a_rows : w_rows);
  auto load_words = [&](int c) __attribute__((always_inline)) {
    __builtin_amdgcn_global_load_lds((global_u8 *)words_at, (lds_u8 *)(words + (c & 1) * 4 * ROWS + wave * 256), 16, 0, 0);
    words_at += words_step;
  };
  // or those of chunks c .. c + OWN - 1 from the rows: step j's four of a chunk a lane, to the word of lane group j
  auto make_words = [&](int c) __attribute__((always_inline)) {
    constexpr int A_ROW = OWN ? OWN * 4 : 4, EACH_LANE = ROWS * A_ROW / (NW * 64), AT_ONCE = NW * 64 / A_ROW;  // rows
    const int q = threadIdx.x % A_ROW, j = q & 3;
    const ScaleWord word(16 * (c0 + c) + 4 * q, a.K / 32);
    uint32_t x[EACH_LANE];
#pragma unroll
    for (int i = 0; i < EACH_LANE; ++i) {
      const int row = threadIdx.x / A_ROW + i * AT_ONCE;
      x[i] = word.load(row < BM ? a.a_scale + (m0 + min(row, last_m)) * a.as_stride : a.w_scale + (n0 + min(row - BM, last_n)) * a.ws_stride);
    }
    const uint32_t pick = 0x0c0c0400u + 0x0101u * (uint32_t)j;  // byte j of each of two
#pragma unroll
    for (int i = 0; i < EACH_LANE; ++i) {
      const int v = (int)word.of(x[i]);
      auto of = [&](auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, 0xf, 0xf, false); };  // a lane of the quad
      const uint32_t x0 = of(std::integral_constant<int, 0x00>{}), x1 = of(std::integral_constant<int, 0x55>{});
      const uint32_t x2 = of(std::integral_constant<int, 0xaa>{}), x3 = of(std::integral_constant<int, 0xff>{});
      words[q * PITCH + threadIdx.x / A_ROW + i * AT_ONCE] =
          __builtin_amdgcn_perm(__builtin_amdgcn_perm(x3, x2, pick), __builtin_amdgcn_perm(x1, x0, pick), 0x05040100u);
    }
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // (the waits count loads: their order stays)
  if constexpr (!OWN) load_words(0);
#pragma unroll
  for (int s = 0; s < NBUF - 1; ++s) {
    asm volatile("" ::: "memory");
    static_for<PIECES>([&](auto i) __attribute__((always_inline)) { load(min(s, stages - 1), s, i); });
  }
  // this lane's runs in a stage: k 0 .. 127 of e4m3 are its runs g and 4 + g, a step of e2m1 run g
  const int a_at = (wm * TM * 16 + r) * AROW + 16 * (g ^ swap128(r)), a_more = a_at ^ 64;
  const int w_at = ABYTES + (wn * TN * 16 + r) * WROW + 16 * (g ^ (E4M3 ? swap64(r) : swap128(r))), w_more = w_at ^ 64;
  const uint32_t *as_at = words + g * PITCH + wm * TM * 16 + r, *ws_at = words + g * PITCH + BM + wn * TN * 16 + r;
  int as[TM], ws[TN];
  int buf = 0;
  if constexpr (OWN) make_words(0);
  // A stage's products, a row of tiles at a time: the next row's operand is read ahead, and
  // the loads of a later stage go out one by one between them (all at once they hold up the wave).
  // MORE: the chunk has another behind it, whose words its first stage asks for.
  auto stage = [&](int c, int s, auto j, auto more) __attribute__((always_inline)) {
    constexpr int STEP = decltype(j)::value, TILE_ROWS = SPS * TM, AT = STEP / SPS;
    constexpr bool WORDS = !OWN && decltype(more)::value;
    // (the words are older than the loads of the stage that asked for them)
    wait_loads<(NBUF - 2) * PIECES + (WORDS && AT >= 1 && AT <= NBUF - 2)>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if constexpr (STEP == 0) {
      const int slot = 4 * PITCH * (OWN ? c % (OWN ? OWN : 1) : c & 1);
#pragma unroll
      for (int t = 0; t < TM; ++t) as[t] = (int)as_at[slot + t * 16];
#pragma unroll
      for (int t = 0; t < TN; ++t) ws[t] = (int)ws_at[slot + t * 16];
      if constexpr (WORDS) load_words(c + 1);
    }
    const int ahead = min(s + NBUF - 1, stages - 1), free = buf == 0 ? NBUF - 1 : buf - 1;
    const uint8_t *base = lds + buf * STAGE;
    buf = buf == NBUF - 1 ? 0 : buf + 1;
    u32x4 wv[2][TN], lo[2], hi[2];
    hi[0] = hi[1] = u32x4{0, 0, 0, 0};
    auto read_w = [&](auto h) __attribute__((always_inline)) {
      constexpr int H = decltype(h)::value;
#pragma unroll
      for (int t = 0; t < TN; ++t) wv[H][t] = read_lds(base + (H ? w_more : w_at) + t * 16 * WROW);
    };
    auto read_a = [&](auto row) __attribute__((always_inline)) {
      constexpr int R = decltype(row)::value;
      lo[R & 1] = read_lds(base + (R >= TM ? a_more : a_at) + R % TM * 16 * AROW);
      if constexpr (E4M3) hi[R & 1] = read_lds(base + a_more + R * 16 * AROW);
    };
    read_w(std::integral_constant<int, 0>{});
    read_a(std::integral_constant<int, 0>{});
    static_for<TILE_ROWS>([&](auto row) __attribute__((always_inline)) {
      constexpr int R = decltype(row)::value, H = R / TM;
      if constexpr (R + 1 < TILE_ROWS) read_a(std::integral_constant<int, R + 1>{});
      if constexpr (SPS == 2 && R == TM - 2) read_w(std::integral_constant<int, 1>{});
      constexpr int P0 = std::min(PIECES, R * EACH), P1 = std::min(PIECES, (R + 1) * EACH);
      static_for<P1 - P0>([&](auto i) __attribute__((always_inline)) { load(ahead, free, std::integral_constant<int, P0 + decltype(i)::value>{}); });
#pragma unroll
      for (int t = 0; t < TN; ++t)
        acc[R % TM][t] = mma_step<E4M3, STEP + H>(operand(wv[H][t]), operand(lo[R & 1], hi[R & 1]), acc[R % TM][t], ws[t], as[R % TM]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  int s = 0;
#pragma unroll 1
  for (int c = 0; c + 1 < chunks; ++c) {
    constexpr std::true_type MORE{};
    if constexpr (OWN) {
      if (c > 0 && c % OWN == 0) make_words(c);
    }
    stage(c, s++, std::integral_constant<int, 0>{}, MORE);
    if constexpr (E4M3) {
      stage(c, s++, std::integral_constant<int, 1>{}, MORE);
      stage(c, s++, std::integral_constant<int, 2>{}, MORE);
      stage(c, s++, std::integral_constant<int, 3>{}, MORE);
    } else {
      stage(c, s++, std::integral_constant<int, 2>{}, MORE);
    }
  }
  {
    constexpr std::false_type MORE{};
    const int c = chunks - 1;
    if constexpr (OWN) {
      if (c > 0 && c % OWN == 0) make_words(c);
    }
    stage(c, s++, std::integral_constant<int, 0>{}, MORE);
    if constexpr (E4M3) {
      if (s < stages) stage(c, s++, std::integral_constant<int, 1>{}, MORE);
      if (s < stages) stage(c, s++, std::integral_constant<int, 2>{}, MORE);
      if (s < stages) stage(c, s++, std::integral_constant<int, 3>{}, MORE);
    } else {
      if (s < stages) stage(c, s++, std::integral_constant<int, 2>{}, MORE);
    }
  }
  wait_loads<0>();  // (the loads of stages past the last one)
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int t = 0; t < TN; ++t) put(a, parts, m0 + (wm * TM + i) * 16 + r, n0 + (wn * TN + t) * 16 + 4 * g, acc[i][t]);
}

// The words of the scales in the workspace: of a, then of w.
struct ScaleWords {
  int a_rows, w_rows, chunks;
  size_t bytes;
};
ScaleWords scale_words(int M, int N, int K) {
  ScaleWords w;
  auto up = [](int n) { return (int)std::min(((long long)n + TILE - 1) / TILE * TILE, 0x7fffff00LL); };
  w.a_rows = up(M);
  w.w_rows = up(N);
  w.chunks = (K + 511) / 512;
  w.bytes = 16 * (size_t)w.chunks * ((size_t)w.a_rows + w.w_rows);
  return w;
}

// Parts of K lie behind the scales' words, of which few rows have none.
size_t part_bytes(int M, int N) { return 4 * (size_t)M * (((size_t)N + 3) & ~(size_t)3); }
float *parts_at(const MxMatmulArgs &a, int parts, size_t behind) {
  return parts > 1 ? reinterpret_cast<float *>(static_cast<char *>(a.workspace) + behind) : nullptr;
}
hipError_t join(const MxMatmulArgs &a, int parts, const float *sums, hipStream_t s) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || parts == 1) return e;
  const int grid = (int)(((long long)a.M * ((a.N + 3) / 4) + 255) / 256);
  npu_launch_plan p = make_plan("mx_join", grid, wg_per_cu(mx_join_kernel, 256), grid, 8);
  p.tile_valu = 4 * (4.0 * parts + 30.0);
  p.tile_load_bytes = 4096.0 * parts;
  p.tile_store_bytes = 2048.0;
  p.hbm_bytes = 0.0;
  plans_add(p);
  hipLaunchKernelGGL(mx_join_kernel, dim3((unsigned)grid), dim3(256), 0, s, a, sums, parts);
  return hipGetLastError();
}

// The dynamic LDS limit of a kernel, raised once per device.
bool lds_allowed(const void *kern, int lds) {
  return cached_per_kernel(kern, [&](int) {
    return hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess ? 1 : 0;
  });
}

template <bool E4M3, int MT, int NT>
hipError_t matmul_few(const MxMatmulArgs &a, int parts, hipStream_t s) {
  constexpr int LDS = SW * MT * NT * 1024;
  auto kern = mx_matmul_few_kernel<E4M3, MT, NT>;
  if (!lds_allowed(reinterpret_cast<const void *>(kern), LDS)) return hipErrorInvalidValue;
  const int steps = (a.K + 127) / 128, per_wave = 2 * ((steps + 2 * parts * SW - 1) / (2 * parts * SW));  // (whole lines)
  const long long groups_m = (a.M + 16LL * MT - 1) / (16 * MT), grid = (a.N + 16LL * NT - 1) / (16 * NT) * groups_m;
  npu_launch_plan p = make_plan("mx_matmul_few", (int)(grid * parts), wg_per_cu(kern, SW * 64, LDS), (int)(grid * parts), 8);
  p.unit_waves = SW;
  p.tile_macs = 256.0 * MT * NT * a.K / parts;
  p.tile_valu = steps / (double)parts * (10.0 * (MT + NT) + 4.0 * MT);
  p.tile_lds_bytes = 2.0 * LDS;
  p.tile_load_bytes = 16.0 * a.K / parts * (0.53 * NT + MT * (E4M3 ? 1.03 : 0.53));
  p.tile_store_bytes = (parts > 1 ? 1024.0 : 512.0) * MT * NT;
  p.hbm_bytes = (double)a.K * (a.M * (E4M3 ? 1.03 : 0.53) + a.N * 0.53) + 2.0 * a.M * a.N;
  plans_add(p);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid, (unsigned)parts), dim3(SW * 64), LDS, s, a, (int)groups_m, steps, per_wave, parts_at(a, parts, 0));
  return join(a, parts, parts_at(a, parts, 0), s);
}

template <bool E4M3, int BM, int BN, int WM, int WN, int NBUF, int OWN>
hipError_t matmul_tiles(const MxMatmulArgs &a, int want_parts, hipStream_t s) {
  constexpr int STAGE = BM * 128 + BN * (E4M3 ? 64 : 128), LDS = NBUF * STAGE + (OWN ? OWN * 16 * (BM + BN + 4) : 32 * (BM + BN));
  static_assert(LDS <= 160 * 1024 && TILE % BM == 0 && TILE % BN == 0, "a CU's LDS; whole tiles of scales");
  const ScaleWords w = scale_words(a.M, a.N, a.K);
  const int part_chunks = (w.chunks + want_parts - 1) / want_parts, parts = (w.chunks + part_chunks - 1) / part_chunks;  // (none empty)
  float *sums = parts_at(a, parts, OWN ? 0 : w.bytes);
  uint32_t *a_words = static_cast<uint32_t *>(a.workspace), *w_words = a_words + 4 * (size_t)w.chunks * w.a_rows;
  if (!OWN) {
    const dim3 grid((unsigned)((w.a_rows + w.w_rows) / 256), (unsigned)((w.chunks + 7) / 8));
    npu_launch_plan p = make_plan("mx_scales", (int)(grid.x * grid.y), wg_per_cu(mx_scales_kernel, 256), (int)(grid.x * grid.y), 8);
    p.tile_valu = 4 * 8 * 30.0;
    p.tile_load_bytes = p.tile_store_bytes = 256 * 128.0;
    p.hbm_bytes = (double)a.K / 32 * ((double)a.M + a.N);
    plans_add(p);
    hipLaunchKernelGGL(mx_scales_kernel, grid, dim3(256), 0, s, a, a_words, w_words, w.a_rows, w.w_rows, w.chunks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  auto kern = mx_matmul_tile_kernel<E4M3, BM, BN, WM, WN, NBUF, OWN>;
  const int tiles_m = (int)((a.M + (long long)BM - 1) / BM), tiles_n = (int)((a.N + (long long)BN - 1) / BN);
  if (!lds_allowed(reinterpret_cast<const void *>(kern), LDS)) return hipErrorInvalidValue;
  npu_launch_plan p = make_plan("mx_matmul_tile", tiles_m * tiles_n * parts, wg_per_cu(kern, WM * WN * 64, LDS), tiles_m * tiles_n * parts, 8);
  const double steps = (a.K + 127) / 128 / (double)parts;
  p.unit_waves = WM * WN;
  p.tile_macs = (double)BM * BN * a.K / parts;
  p.tile_valu = steps * WM * WN * 40.0;
  p.tile_lds_bytes = steps * (STAGE / (E4M3 ? 1 : 2) + WN * BM * (E4M3 ? 128.0 : 64.0) + WM * BN * 64.0);
  p.tile_load_bytes = steps * STAGE / (E4M3 ? 1 : 2) * 33.0 / 32;
  p.tile_store_bytes = (parts > 1 ? 4.0 : 2.0) * BM * BN;
  p.hbm_bytes = (double)a.K * (a.M * (E4M3 ? 1.03 : 0.53) + a.N * 0.53) + 2.0 * a.M * a.N;
  plans_add(p);
  hipLaunchKernelGGL(kern, dim3((unsigned)(tiles_m * tiles_n), (unsigned)parts), dim3(WM * WN * 64), LDS, s, a, TileOrder{tiles_m, tiles_n}, a_words,
                     w_words, w.a_rows, w.w_rows, part_chunks, sums);
  return join(a, parts, sums, s);
}

// ---- which kernel ------------------------------------------------------------------------
// A call is a few-rows kernel in groups of up to 48 rows by 16 or 32 columns, or tiles of 32 x 64, 64 x 128,
// 128 x 128 or 256 x 256, with K in one part or in up to eight, by the least of the times that these
// estimate, in us, from measurements of 480 shapes (M 1 .. 4096, N 512 .. 14336, K 512 .. 14336, both types;
// profiles/product_kernels_by_shape.txt).  The choice takes 4 % more than each shape's fastest of these on
// average, and these 1.3 % more than the fastest of 22 tried.  Past that range it extrapolates: 1, 48 and 128 rows of
// e4m3 by 128000 x 4096 54, 64 and 98 us with other weights each time, w's bytes 53 of them.
// In us, e4m3, parts after the slash:
//   rows      by                  16 cols  32 cols  32 x 64  64 x 128  128 x 128  256 x 256
//      1   4096 x 14336 (N x K)    9.9/1    10.1/4   10.6/4    12.6/8    14.9/8
//     48  14336 x 4096            21.2/1    14.5/1   10.8/1    13.3/2    15.1/2
//    512   4096 x 4096            54.9/1    39.8/1   19.4/1    13.8/1    18.9/1     49.6
//   1000   4096 x 4096             113/1    79.3/1   33.7/1    21.9/1    21.0/1     50.9
//   4096   4096 x 14336                                448/1     271/1     239/1      173
struct Choice {
  int tile;        // rows of a tile; 0: few rows
  int mt, nt;      // groups of 16 mt x 16 nt (few rows)
  int parts;
  double us;
};
constexpr int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// A group's time is its wave's steps, whose operands eight waves bring through one L1.
double few_us(bool e4m3, int M, int N, int K, int mt, int nt, int parts, int cus) {
  const int per_wave = 2 * ceil_div(ceil_div(K, 128), 2 * SW * parts);
  const double rounds = std::ceil((double)ceil_div(M, 16 * mt) * ceil_div(N, 16 * nt) * parts / cus);
  const double group = per_wave * (e4m3 ? 0.20 * nt + 0.33 * mt : 0.23 * nt + 0.21 * mt);
  return 2.1 + group * (1.0 + (e4m3 ? 0.92 : 0.81) * (rounds - 1.0)) + (parts > 1 ? 2.6 + 4.8e-6 * parts * M * N : 0.0);
}

// Rounds of as many workgroups as fit the CUs, then what is left, a step of which takes as long as
// that many workgroups on a CU have it take.
struct TileCost {
  int m, n, fit;
  double call, round, step[3];
};
const TileCost kTiles[2][4] = {{{32, 64, 2, 3.7, 1.5, {0.107, 0.163}},
                                {64, 128, 1, 4.0, 2.0, {0.212}},
                                {128, 128, 2, 4.3, 5.3, {0.403, 0.609}},
                                {256, 256, 1, 15.1, 9.8, {0.843}}},
                               {{32, 64, 3, 3.8, 2.0, {0.148, 0.244, 0.331}},
                                {64, 128, 2, 4.3, 3.5, {0.294, 0.505}},
                                {128, 128, 1, 5.4, 3.2, {0.488}},
                                {256, 256, 1, 15.3, 8.8, {1.374}}}};
double tile_us(bool e4m3, const TileCost &t, int M, int N, int K, int parts, int cus) {
  const int chunks = ceil_div(K, 512), per = ceil_div(chunks, parts), real = ceil_div(chunks, per);
  const double steps = std::min(ceil_div(K, 128), 4 * per), tiles = (double)ceil_div(M, t.m) * ceil_div(N, t.n) * real / cus;
  const double rounds = std::floor(tiles / t.fit), left = tiles - rounds * t.fit, full = t.step[t.fit - 1];
  // (one to a CU: the fewer CUs run, the faster)
  const double last = left <= 0 ? 0.0 : t.fit > 1 ? t.step[(int)std::ceil(left) - 1] : full * (0.73 + 0.27 * left);
  return t.call + rounds * (full * steps + t.round) + last * steps + (real > 1 ? 2.6 + 1.2e-6 * real * M * N : 0.0);
}

Choice choose(bool e4m3, int M, int N, int K, int cus) {
  Choice best{0, 1, 1, 1, 1e30};
  const int steps = ceil_div(K, 128);
  for (int parts = 1; parts <= 8; parts *= 2) {
    if (K >= 128 && parts <= ceil_div(K, 512))
      for (const TileCost &t : kTiles[e4m3]) {
        if (t.m == 256 && parts > 1) continue;  // (where K has to be divided, smaller tiles are the faster)
        const double us = tile_us(e4m3, t, M, N, K, parts, cus);
        if (us < best.us) best = Choice{t.m, 0, 0, parts, us};
      }
    // (a thousand rows are tiles' whatever N and K)
    if (M > 1024 && K >= 128) continue;
    if (parts > 1 && steps < SW * parts) continue;
    const int mt = std::min(3, ceil_div(M, 16));
    for (int nt : {1, 2}) {
      if (nt > 1 && N < 16 * nt) break;
      const double us = few_us(e4m3, M, N, K, mt, nt, parts, cus);
      if (us < best.us) best = Choice{0, mt, nt, parts, us};
    }
  }
  return best;
}

// Rows past the last whole tile of 256 are a call of their own where that is faster than a tile
// mostly of other rows' copies (4099 rows by 4096 x 14336: 16 rounds' worth of tiles in one and 3 rows).
struct Calls {
  Choice first, rest;
  int m;  // rows of the first
};
Calls choose_calls(bool e4m3, int M, int N, int K, int cus) {
  Calls c{choose(e4m3, M, N, K, cus), Choice{}, M};
  const int rest = M % 256;
  if (M < 256 || rest == 0) return c;
  const Choice a = choose(e4m3, M - rest, N, K, cus), b = choose(e4m3, rest, N, K, cus);
  if (a.us + b.us < c.first.us) c = Calls{a, b, M - rest};
  return c;
}

size_t call_bytes(const Choice &c, int M, int N, int K) {
  return (c.tile == 256 ? scale_words(M, N, K).bytes : 0) + (c.parts > 1 ? c.parts * part_bytes(M, N) : 0);
}

// Of a shape's calls by type, and what the larger needs of the workspace.  A thread keeps its latest 64 shapes':
// a call asks three times, and each time takes 0.2 to 0.7 us.
struct Decided {
  int M, N, K, cus;
  Calls calls[2];
  size_t bytes;
};
const Decided &decided(int M, int N, int K) {
  static thread_local Decided kept[64];
  const int cus = device_cus();
  Decided &d = kept[((uint32_t)M * 2654435761u ^ (uint32_t)N * 2246822519u ^ (uint32_t)K * 3266489917u) >> 26];
  if (d.M == M && d.N == N && d.K == K && d.cus == cus) return d;
  d = Decided{M, N, K, cus, {choose_calls(false, M, N, K, cus), choose_calls(true, M, N, K, cus)}, 16};
  for (const Calls &c : d.calls) {
    d.bytes = std::max(d.bytes, call_bytes(c.first, c.m, N, K));
    if (c.m < M) d.bytes = std::max(d.bytes, call_bytes(c.rest, M - c.m, N, K));
  }
  return d;
}

template <bool E4M3>
hipError_t call(const MxMatmulArgs &a, const Choice &c, hipStream_t s) {
  // (stages of e4m3 are shorter: eight waves of 64 x 128 are the faster there)
  if (c.tile == 256) return E4M3 ? matmul_tiles<E4M3, 256, 256, 4, 2, E4M3 ? 3 : 2, 0>(a, c.parts, s) : matmul_tiles<E4M3, 256, 256, 2, 4, 2, 0>(a, c.parts, s);
  if (c.tile == 128) return matmul_tiles<E4M3, 128, 128, 4, 2, E4M3 ? 3 : 2, E4M3 ? 4 : 2>(a, c.parts, s);
  if (c.tile == 64) return matmul_tiles<E4M3, 64, 128, 2, 4, 3, E4M3 ? 8 : 4>(a, c.parts, s);
  if (c.tile == 32) return matmul_tiles<E4M3, 32, 64, 1, 4, 4, 8>(a, c.parts, s);
  if (c.mt == 1) return c.nt == 1 ? matmul_few<E4M3, 1, 1>(a, c.parts, s) : matmul_few<E4M3, 1, 2>(a, c.parts, s);
  if (c.mt == 2) return c.nt == 1 ? matmul_few<E4M3, 2, 1>(a, c.parts, s) : matmul_few<E4M3, 2, 2>(a, c.parts, s);
  return c.nt == 1 ? matmul_few<E4M3, 3, 1>(a, c.parts, s) : matmul_few<E4M3, 3, 2>(a, c.parts, s);
}

}  // namespace

size_t mx_matmul_workspace(int M, int N, int K) { return decided(M, N, K).bytes; }

hipError_t launch_mx_matmul(const MxMatmulArgs &a, hipStream_t s) {
  const Calls c = decided(a.M, a.N, a.K).calls[a.e4m3];
  MxMatmulArgs b = a;
  b.M = c.m;
  const hipError_t e = a.e4m3 ? call<true>(b, c.first, s) : call<false>(b, c.first, s);
  if (e != hipSuccess || c.m == a.M) return e;
  b.M = a.M - c.m;
  b.a += c.m * a.a_stride;
  b.a_scale += c.m * a.as_stride;
  b.out += c.m * a.out_stride;
  return a.e4m3 ? call<true>(b, c.rest, s) : call<false>(b, c.rest, s);
}

}  // namespace npu
