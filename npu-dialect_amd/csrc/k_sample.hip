// k_sample.hip -- the next token of each row of logits, from a given random
// number: temperature, top-k, top-p, min-p.
//
// Entries are ordered by logit, descending, then by index.  With weights w =
// exp((x - max) / T), every setting keeps a prefix of that order: top-k a number of
// entries, top-p a mass, min-p a value; the token is the entry where the
// running mass passes u times the kept mass.  So each is the same search, for
// the first entry whose running count or mass exceeds a bound, and nothing is
// sorted: a histogram of counts and masses over the distance from the maximum
// gives the bin, and the bin's few entries the rest.
//
// Masses are whole numbers, w 2^42 rounded from f64: their sums are exact
// whatever the order of the atomic additions, and the answer is the same every
// time.  2^20 entries of weight 1 sum below 2^63, which bounds V.  f32 weights
// would not do: their rounding, 2^-24 of a mass, is of the order of the
// distance of u from the nearest of 10^5 borders.
//
// A workgroup takes a row.  A bin of more than LIST entries (equal logits, or
// all of them far below the maximum) is divided further by the order's own key,
// the logit's bits and then the index, eleven bits at a time.
#include <hip/hip_runtime.h>

#include <cmath>

#include "kernels.hpp"
#include "npu_device.hpp"
#include "plans.hpp"

namespace npu {

namespace {

constexpr int ST = 1024;     // lanes of a workgroup
constexpr int BINS = 2048;
constexpr int LIST = 2048;   // entries of a bin that are ranked at once
constexpr float BINS_PER_NAT = 64.0f;
constexpr double ONE = 4398046511104.0;  // 2^42: weight 1

typedef unsigned long long u64;

// A candidate's place in the order as a number: smaller comes first.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? b : ~b & 0x7fffffffu;  // descending, x never NaN or -0
}
__device__ __forceinline__ u64 order_key(float x, int i) { return (u64)order_bits(x) << 32 | (uint32_t)i; }

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ u64 uniform(u64 v) {
  return (u64)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ double uniform(double v) {
  return __longlong_as_double((long long)uniform((u64)__double_as_longlong(v)));
}

// 2^y for y <= 0: the nearest whole power times the Taylor polynomial of
// exp(f ln 2), |f| <= 1/2, to degree 11 (the next term is below 7e-15).
__device__ __forceinline__ double exp2_64(double y) {
  y = fmax(y, -1000.0);
  const double whole = rint(y), r = (y - whole) * 0.69314718055994530942;
  double p = 1.0 / 39916800;
  p = fma(p, r, 1.0 / 3628800);
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)whole);
}
// A weight's whole number, rounded to nearest: the significand of w 2^42 + 2^52.
__device__ __forceinline__ u64 fixed(double w) {
  const double big = 4503599627370496.0;  // 2^52
  return (u64)__double_as_longlong(fma(w, ONE, big)) - (u64)__double_as_longlong(big);
}

// The row's entries, each once, as f(x, index): 16-byte loads of the aligned part.
template <bool BF, class F>
__device__ __forceinline__ void each_entry(const void *row, int V, F f) {
  constexpr int PER = BF ? 8 : 4, ES = BF ? 2 : 4;
  const char *p = static_cast<const char *>(row);
  const int tid = threadIdx.x;
  auto one = [&](int i) {
    f(BF ? bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[i]) : reinterpret_cast<const float *>(p)[i], i);
  };
  const int head = min(V, (int)((16 - ((uintptr_t)p & 15)) & 15) / ES);
  if (tid < head) one(tid);
  const int chunks = (V - head) / PER;
  const u32x4 *body = reinterpret_cast<const u32x4 *>(p + head * ES);
#pragma unroll 1
  for (int c = tid; c < chunks; c += ST) {
    const u32x4 v = body[c];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = head + c * PER + e * (PER / 4);
      if constexpr (BF) {
        f(__uint_as_float(v[e] << 16), i);
        f(__uint_as_float(v[e] & 0xffff0000u), i + 1);
      } else {
        f(__uint_as_float(v[e]), i);
      }
    }
  }
  for (int i = head + chunks * PER + tid; i < V; i += ST) one(i);
}

struct Shared {
  u64 mass[BINS];
  uint32_t count[BINS];
  float lx[LIST];
  int li[LIST];
  u64 lw[LIST];
  u64 wave_m[ST / 64], wave_c[ST / 64];
  u64 key;               // the maximum's order key
  int n_list, bin, pos;
  u64 rank, cum, own;    // the entry found: entries and mass up to it (inclusive), its mass
};

// Exclusive prefix sums of the histogram in place; the totals to all lanes.
__device__ __forceinline__ void scan_bins(Shared &s, u64 &mass, u64 &count) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const u64 m0 = s.mass[2 * tid], m1 = s.mass[2 * tid + 1];
  const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
  u64 m = m0 + m1, c = (u64)c0 + c1;
  for (int off = 1; off < 64; off <<= 1) {
    const u64 pm = __shfl_up(m, off), pc = __shfl_up(c, off);
    if (lane >= off) m += pm, c += pc;
  }
  if (lane == 63) s.wave_m[wave] = m, s.wave_c[wave] = c;
  __syncthreads();
  u64 bm = 0, bc = 0;
  u64 am = 0, ac = 0;
#pragma unroll 2
  for (int v = 0; v < ST / 64; ++v) {
    if (v < wave) bm += s.wave_m[v], bc += s.wave_c[v];
    am += s.wave_m[v], ac += s.wave_c[v];
  }
  mass = uniform(am);
  count = uniform(ac);
  m += bm - m0 - m1;
  c += bc - c0 - c1;
  s.mass[2 * tid] = m;
  s.mass[2 * tid + 1] = m + m0;
  s.count[2 * tid] = (uint32_t)c;
  s.count[2 * tid + 1] = (uint32_t)c + c0;
  __syncthreads();
}
static_assert(BINS == 2 * ST, "two bins a lane");

__device__ __forceinline__ void clear_bins(Shared &s) {
  for (int b = threadIdx.x; b < BINS; b += ST) s.mass[b] = 0, s.count[b] = 0;
  __syncthreads();
}

// The bin whose running count (by_count) or mass passes t: t is below the total.
// Every lane gets the bin, its entries, and what comes before it.
struct Found {
  int bin, entries;
  u64 count, mass;
};
__device__ __forceinline__ Found find_bin(Shared &s, bool by_count, u64 t, u64 all_mass, u64 all_count) {
  for (int b = threadIdx.x; b < BINS; b += ST) {
    const u64 lo = by_count ? s.count[b] : s.mass[b];
    const u64 hi = b + 1 < BINS ? (by_count ? s.count[b + 1] : s.mass[b + 1]) : (by_count ? all_count : all_mass);
    if (lo <= t && t < hi) s.bin = b;
  }
  __syncthreads();
  const int b = uniform(s.bin);
  Found f;
  f.bin = b;
  f.count = (u64)(uint32_t)uniform((int)s.count[b]);
  f.mass = uniform(s.mass[b]);
  f.entries = uniform((int)((b + 1 < BINS ? s.count[b + 1] : (uint32_t)all_count) - (uint32_t)f.count));
  __syncthreads();
  return f;
}

template <bool BF>
__global__ __launch_bounds__(ST) void sample_tokens_kernel(SampleArgs a) {
  __shared__ Shared s;
  const int tid = threadIdx.x, row = blockIdx.x, V = a.V;
  const char *x0 = static_cast<const char *>(a.logits) + (long long)row * a.row_stride * (BF ? 2 : 4);
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;

  // the maximum and its first index
  if (tid == 0) s.key = ~0ull;
  __syncthreads();
  u64 best = ~0ull;
  each_entry<BF>(x0, V, [&](float x, int i) {
    x += 0.0f;  // -0 is 0
    if (x > -__builtin_inff()) best = min(best, order_key(x, i));
  });
  for (int off = 32; off; off >>= 1) best = min(best, (u64)__shfl_xor(best, off));
  if ((tid & 63) == 0) atomicMin(&s.key, best);
  __syncthreads();
  best = uniform(s.key);
  const int first = (int)(uint32_t)best;
  // no candidate, or one that every setting leaves
  const bool greedy = !(temp > 0.0f) || k == 1 || top_p <= 0.0f;
  if (best == ~0ull || greedy) {
    if (tid == 0) {
      a.tokens[row] = best == ~0ull ? -1 : first;
      if (a.probs) a.probs[row] = best == ~0ull ? 0.0f : 1.0f;
    }
    return;
  }
  const uint32_t ob = (uint32_t)(best >> 32);
  const float top = __uint_as_float(ob & 0x80000000u ? ob : ~ob & 0x7fffffffu);
  const bool infinite = top == __builtin_inff();  // then only the infinite logits are candidates
  const double rate = uniform(1.4426950408889634074 / (double)temp);
  auto weight = [&](float x) { return infinite ? 1.0 : exp2_64(((double)x - (double)top) * rate); };
  auto is_candidate = [&](float x) { return infinite ? x == top : x > -__builtin_inff(); };
  const float per = BINS_PER_NAT / temp;
  auto bin_of = [&](float x) {
    const float d = infinite ? 0.0f : (top - x) * per;
    return d < (float)(BINS - 1) ? (int)d : BINS - 1;
  };

  // The histogram's range: the whole row by bins, or, where a bin is divided, the
  // entries of bin `in_bin` whose key starts with `prefix`, by the key's next bits.
  int in_bin = -1, shift = 64, next = 64;
  u64 prefix = 0, base_m = 0, base_n = 0;
  auto inside = [&](float x, int i) {
    if (!is_candidate(x)) return false;
    if (in_bin < 0) return true;
    return bin_of(x) == in_bin && (shift == 64 || order_key(x, i) >> shift == prefix);
  };

  // The searches in turn: 0 for top-k's count, 1 for top-p's mass, 2 for the draw.
  u64 n = 0, m = 0, range_m = 0, range_n = 0, all_n = 0, all_m = 0, keep_n = 0, keep_m = 0, t = 0;
  bool by_count = false, have = false, known = false;
  for (int step = -1;;) {
    if (!have) {
      clear_bins(s);
      u64 kn = 0, km = 0;
      each_entry<BF>(x0, V, [&](float x, int i) {
        x += 0.0f;
        if (!inside(x, i)) return;
        const double w = weight(x);
        const u64 f = fixed(w);
        const int b = in_bin < 0 ? bin_of(x) : (int)(order_key(x, i) >> next & ((1ull << (shift - next)) - 1));
        atomicAdd(&s.mass[b], f);
        atomicAdd(&s.count[b], 1u);
        if (w >= (double)min_p) ++kn, km += f;
      });
      if (step < 0) {  // what min-p keeps, counted on the way
        if (tid == 0) s.rank = 0, s.cum = 0;
        __syncthreads();
        for (int off = 32; off; off >>= 1) kn += __shfl_xor(kn, off), km += __shfl_xor(km, off);
        if ((tid & 63) == 0) {
          atomicAdd(&s.rank, kn);
          atomicAdd(&s.cum, km);
        }
      }
      __syncthreads();
      scan_bins(s, range_m, range_n);
      have = true;
    }
    if (step < 0) {
      keep_n = uniform(s.rank);
      keep_m = uniform(s.cum);
      n = all_n = range_n;
      m = all_m = range_m;
      step = 0;
      __syncthreads();
    }
    if (!known) {  // the search's bound
      if (step == 0) {
        if (k > 0 && (u64)k < n) {
          by_count = true;
          t = (u64)k - 1;
          known = true;
        } else {
          step = 1;
        }
      }
      if (step == 1) {
        if (top_p < 1.0f) {
          const double v = uniform(ceil((double)top_p * (double)m));
          by_count = false;
          t = v >= 1.0 ? min((u64)v, m) - 1 : 0;
          known = true;
        } else {
          step = 2;
        }
      }
      if (step == 2) {
        if (min_p > 0.0f && keep_n < n) n = keep_n > 0 ? keep_n : 1, m = keep_n > 0 ? keep_m : (u64)ONE;
        const double v = uniform(floor((double)a.u[row] * (double)m));
        by_count = false;
        t = v >= 0.0 ? min((u64)v, m - 1) : 0;
        known = true;
      }
    }
    const Found f = find_bin(s, by_count, t - (by_count ? base_n : base_m), range_m, range_n);
    if (in_bin < 0) {
      in_bin = f.bin;
    } else {
      prefix = (shift == 64 ? 0 : prefix << (shift - next)) | (u64)f.bin;
      shift = next;
    }
    base_m += f.mass;
    base_n += f.count;
    if (f.entries > LIST) {
      next = shift > 11 ? shift - 11 : 0;
      have = false;
      continue;
    }
    // the entries that are left, ranked by comparing each with all
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    each_entry<BF>(x0, V, [&](float x, int i) {
      x += 0.0f;
      if (!inside(x, i)) return;
      const int at = atomicAdd(&s.n_list, 1);
      if (at < LIST) s.lx[at] = x, s.li[at] = i;
    });
    __syncthreads();
    const int listed = uniform(min(s.n_list, LIST));
    for (int e = tid; e < listed; e += ST) s.lw[e] = fixed(weight(s.lx[e]));
    __syncthreads();
    for (int e = tid; e < listed; e += ST) {
      const u64 key = order_key(s.lx[e], s.li[e]), w = s.lw[e];
      u64 rank = base_n, cum = base_m;
#pragma unroll 4
      for (int j = 0; j < listed; ++j)
        if (order_key(s.lx[j], s.li[j]) < key) ++rank, cum += s.lw[j];
      const u64 lo = by_count ? rank : cum, hi = by_count ? rank + 1 : cum + w;
      if (lo <= t && t < hi) s.rank = rank + 1, s.cum = cum + w, s.own = w, s.pos = s.li[e];
    }
    __syncthreads();
    if (step == 2) break;
    if (uniform(s.rank) < n) n = uniform(s.rank), m = uniform(s.cum);
    __syncthreads();
    // a divided bin's histogram is of no use for the next search
    if (shift != 64) have = false;
    if (have) range_m = all_m, range_n = all_n;
    in_bin = -1;
    shift = next = 64;
    prefix = base_m = base_n = 0;
    known = false;
    ++step;
  }
  if (tid == 0) {
    a.tokens[row] = s.pos;
    if (a.probs) a.probs[row] = (float)((double)s.own / (double)m);
  }
}

}  // namespace

size_t sample_workspace(int, int) { return 16; }

hipError_t launch_sample_tokens(const SampleArgs &a, hipStream_t s) {
  auto kern = a.bf16 ? sample_tokens_kernel<true> : sample_tokens_kernel<false>;
  {
    npu_launch_plan p = make_plan("sample_tokens", a.B, wg_per_cu(kern, ST), a.B, 16);
    const double rounds = std::ceil((double)a.V / ST) * (ST / 64);
    p.unit_waves = ST / 64;
    p.load_phases = 3;
    p.tile_valu = rounds * 60.0;
    p.tile_lds_bytes = a.V * 12.0;
    p.tile_load_bytes = 3.0 * a.V * (a.bf16 ? 2 : 4);
    p.tile_store_bytes = 8.0;
    p.hbm_bytes = (double)a.B * a.V * (a.bf16 ? 2 : 4);
    plans_add(p);
  }
  hipLaunchKernelGGL(kern, dim3(a.B), dim3(ST), 0, s, a);
  return hipGetLastError();
}

}  // namespace npu
