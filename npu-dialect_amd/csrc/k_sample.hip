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
// A workgroup takes a row.  What bounds it: each pass over a long row is at the rate
// of the memory behind the L2 (256 rows of 128000 f32, 131 MB: 18 us), and in the
// histogram's pass the f64 arithmetic and the LDS atomics (46 us of those rows' 126), so
// passes and work in them are saved:
//  - the maximum, always;
//  - with top-k, the entries that can be among the k: at least k of the lanes' own
//    maxima are in the bins up to the k-th's, so all entries up to that bin are
//    copied to LDS, and the rest of the row is not looked at again;
//  - else the histogram, with every entry's weight, and then the entries of the
//    bins that the searches end in, in one pass for all of them: the bin that one
//    search ends in bounds the mass that the next one starts from.
// A row alone (one of 32000: 19 us in the kernel) is a chain of
// such steps, each with a barrier and an LDS or memory latency.
// A bin of more than LIST entries (equal logits, say) is divided further by the
// order's own key, the logit's bits and then the index, eleven bits at a time.
#include <hip/hip_runtime.h>

#include <cmath>

#include "kernels.hpp"
#include "npu_device.hpp"
#include "plans.hpp"

namespace npu {

namespace {

constexpr int ST = 512;      // lanes of a workgroup: 1024 would leave a lane 128 registers
constexpr int BINS = 2048;
constexpr int LIST = 2048;   // entries of a bin that are ranked at once
constexpr int CAND = 4096;   // entries that are kept from one pass over the row
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
__device__ __forceinline__ float uniform(float v) { return __int_as_float(uniform(__float_as_int(v))); }
__device__ __forceinline__ double uniform(double v) {
  return __longlong_as_double((long long)uniform((u64)__double_as_longlong(v)));
}

// 2^y, |y| <= 1/2, by the Taylor polynomial of exp(y ln 2) to degree 11 (the next term
// is below 7e-15): for the table below.
__device__ __forceinline__ double exp2_small(double y) {
  const double r = y * 0.69314718055994530942;
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
  return fma(p, r, 1.0);
}

// The weights of a row: 2^42 2^y, y = (x - top) rate, as a whole power, a table of
// 64ths and the Taylor polynomial of what is left, |r| <= 1/128, to degree 4 (the next
// term is 4e-14, a third of the last bit of a weight's whole number).  A polynomial of
// degree 9 in place of the table took 133 us for 256 rows of 128000 f32 to this one's 126.
constexpr int TABLE = 64;
struct Weights {
  const double *table;  // 2^42 2^(j / 64), in LDS
  double top, rate;
  // (-Inf and NaN, which are no candidates, weigh 0)
  __device__ __forceinline__ double power(float x) const { return fmax(((double)x - top) * rate, -1000.0); }
  static constexpr double MAGIC = 6755399441055744.0;  // 1.5 2^52: a sum's low bits are the other's nearest whole number
  // The weight as a whole number, rounded to nearest (the significand of w + 2^52), and
  // -k, the 64ths of y.
  __device__ __forceinline__ u64 operator()(float x, int &bin) const {
    const double y = power(x), t = fma(y, 64.0, MAGIC);
    const int k = (int)__double_as_longlong(t);
    bin = -k;
    const double r = fma(t - MAGIC, -1.0 / 64, y);
    constexpr double L = 0.69314718055994530942;
    double p = L * L * L * L / 24;
    p = fma(p, r, L * L * L / 6);
    p = fma(p, r, L * L / 2);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    // (k is above -2^16: the exponent's field cannot underflow)
    const double big = 4503599627370496.0;  // 2^52
    const double scale = __longlong_as_double(__double_as_longlong(table[k & (TABLE - 1)]) + ((long long)(k & -TABLE) << 46));
    return (u64)__double_as_longlong(fma(scale, p, big)) - (u64)__double_as_longlong(big);
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    int bin;
    return (*this)(x, bin);
  }
  // -k alone, for any x that is not NaN.
  __device__ __forceinline__ int steps(float x) const {
    return -(int)__double_as_longlong(fma(fmin(power(x), 0.0), 64.0, MAGIC));
  }
};

// The row's entries, each once, as f(x, i): x four entries from index i on, in rising
// order for a lane, NaN past the row's ends.  After a round of n entries done(i0, n): the
// j-th of them has index i0 + j / PER ST PER + j % PER.  16-byte loads of the aligned
// part, UN of them together a round ahead (a longer queue costs a move each step for
// every register in it); the ends are chunks of their own.  f32 rows take 4 or 8 copies of f
// for 4 entries each, which hides the loads' latency; a bf16 row's load has 8 entries,
// and more copies only make the code longer (96 rows of 50257: 49 us, with 4 and 2 58).
template <bool BF>
constexpr int PER = BF ? 8 : 4;
template <bool BF, int UN, class F, class D>
__device__ __forceinline__ void each_four(const void *row, int V, F f, D done) {
  constexpr int PER = npu::PER<BF>, ES = BF ? 2 : 4;
  const char *p = static_cast<const char *>(row);
  const int head = min(V, (int)((16 - ((uintptr_t)p & 15)) & 15) / ES), chunks = (V - head) / PER;
  const u32x4 *body = reinterpret_cast<const u32x4 *>(p + head * ES);
  auto give = [&](const float (&x)[PER], int i) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < PER; e += 4) {
      const float y[4] = {x[e], x[e + 1], x[e + 2], x[e + 3]};
      f(y, i + e);
    }
  };
  u32x4 v[UN], next[UN] = {};
#pragma unroll 1
  for (int c0 = -1;; c0 = c0 < 0 ? 0 : c0 + UN * ST) {  // -1: the ends, a lane each
    if (c0 >= chunks) break;
#pragma unroll
    for (int d = 0; d < UN; ++d) {
      const int c = (c0 < 0 ? 0 : c0 + UN * ST) + d * ST + (int)threadIdx.x;
      v[d] = next[d];
      next[d] = u32x4{0, 0, 0, 0};
      if (c < chunks) next[d] = body[c];
    }
    int i0 = 0;
#pragma unroll
    for (int d = 0; d < UN; ++d) {
      const int c = c0 + d * ST + (int)threadIdx.x;
      float x[PER];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (BF) {
          x[2 * e] = __uint_as_float(v[d][e] << 16);
          x[2 * e + 1] = __uint_as_float(v[d][e] & 0xffff0000u);
        } else {
          x[e] = __uint_as_float(v[d][e]);
        }
      }
      int i = head + c * PER;
      if (c0 < 0 || c >= chunks) {
        // (the first two lanes of the first round: the head, the tail)
        const bool tail = threadIdx.x == 1;
        i = tail ? head + chunks * PER : 0;
        const int end = c0 < 0 && d == 0 && threadIdx.x < 2 ? (tail ? V : head) : 0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          x[e] = __builtin_nanf("");
          if (i + e < end)
            x[e] = BF ? bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[i + e]) : reinterpret_cast<const float *>(p)[i + e];
        }
        if (c0 < 0 && d > 0) break;
      }
      if (d == 0) i0 = i;
      give(x, i);
    }
    done(i0, c0 < 0 ? PER : UN * PER);
  }
}
template <bool BF, int UN, class F>
__device__ __forceinline__ void each_four(const void *row, int V, F f) {
  each_four<BF, UN>(row, V, f, [](int, int) {});
}

struct Shared {
  u64 mass[BINS];
  uint32_t count[BINS];
  double table[TABLE];
  float cx[CAND];        // candidates kept from a pass
  int ci[CAND];
  ulonglong2 list[LIST];  // a bin's order keys and weights
  u64 wave_m[ST / 64], wave_c[ST / 64];
  u64 key;               // the first index of the maximum
  u64 total;             // the mass of all
  int n_cand, n_list, pos, candidates;
  u64 cum, own;          // the entry found: the mass up to it (inclusive), its own
};

// Exclusive prefix sums of the histogram in place; the totals to all lanes.
__device__ __forceinline__ void scan_bins(Shared &s, u64 &mass, u64 &count) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int PL = BINS / ST;  // bins of a lane
  u64 bin_m[PL], m = 0;
  uint32_t bin_c[PL], c = 0;
#pragma unroll
  for (int i = 0; i < PL; ++i) m += bin_m[i] = s.mass[PL * tid + i], c += bin_c[i] = s.count[PL * tid + i];
  const u64 lane_m = m;
  const uint32_t lane_c = c;
  for (int off = 1; off < 64; off <<= 1) {
    const u64 pm = __shfl_up(m, off);
    const uint32_t pc = __shfl_up(c, off);
    if (lane >= off) m += pm, c += pc;
  }
  if (lane == 63) s.wave_m[wave] = m, s.wave_c[wave] = c;
  __syncthreads();
  // every wave scans the waves' totals
  constexpr int NW = ST / 64;
  u64 tm = lane < NW ? s.wave_m[lane] : 0;
  uint32_t tc = lane < NW ? s.wave_c[lane] : 0;
  for (int off = 1; off < NW; off <<= 1) {
    const u64 pm = __shfl_up(tm, off);
    const uint32_t pc = __shfl_up(tc, off);
    if (lane >= off) tm += pm, tc += pc;
  }
  const u64 bm = wave > 0 ? __shfl(tm, wave - 1) : 0;
  const uint32_t bc = wave > 0 ? __shfl(tc, wave - 1) : 0;
  mass = uniform(__shfl(tm, NW - 1));
  count = (u64)(uint32_t)uniform((int)__shfl(tc, NW - 1));
  m += bm - lane_m;
  c += bc - lane_c;
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    s.mass[PL * tid + i] = m;
    s.count[PL * tid + i] = c;
    m += bin_m[i];
    c += bin_c[i];
  }
  __syncthreads();
}
static_assert(BINS % ST == 0, "whole bins a lane");

__device__ __forceinline__ void clear_bins(Shared &s) {
  for (int b = threadIdx.x; b < BINS; b += ST) s.mass[b] = 0, s.count[b] = 0;
  __syncthreads();
}

// The bin whose running count (by_count) or mass passes t, which is below the total:
// the last one before which no more than t lies, of empty ones among it the last.
// Every wave looks for itself: one of 64 runs of bins, then one of its 32.
__device__ __forceinline__ int bin_of_total(const Shared &s, bool by_count, u64 t) {
  const int lane = threadIdx.x & 63;
  const u64 a = by_count ? (u64)s.count[lane * (BINS / 64)] : s.mass[lane * (BINS / 64)];
  const int run = 63 - __builtin_clzll(__ballot(a <= t));  // (bin 0's is 0)
  const int at = run * (BINS / 64) + (lane & (BINS / 64 - 1));
  const u64 b = by_count ? (u64)s.count[at] : s.mass[at];
  const uint32_t in = (uint32_t)__ballot(b <= t);
  return uniform(run * (BINS / 64) + 31 - __builtin_clz(in));
}
static_assert(BINS / 64 == 32, "a run's bins in half a wave");
// What comes before a bin.
__device__ __forceinline__ u64 mass_before(const Shared &s, int b, u64 all) { return b < BINS ? uniform(s.mass[b]) : all; }
__device__ __forceinline__ int count_before(const Shared &s, int b, u64 all) {
  return b < BINS ? uniform((int)s.count[b]) : (int)all;
}

// What a histogram divides: the row by the distance from the maximum (kNear: by 64ths of
// the weight's power of two, for 32 powers, the rest in the last bin; kFar: that bin, by
// 16ths), or a bin by the order key's bits from `shift` down to `next`.
enum { kNear = 0, kFar = 1, kKeys = 2 };
struct Range {
  int level, bin, shift, next;  // bin: of level `from`, that kKeys divides
  int from;
  u64 prefix, mass, count;      // mass, count: what comes before the range
};
// The smallest x whose bin is at most b, for a bin that does not rise with x: 64 lanes
// try 64 places of the order, six bits at a time.
template <class B>
__device__ __forceinline__ float least_in(B bin_of, int b) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t first = 0;  // the order's numbers up to `first` are in
  for (int shift = 26;; shift = shift > 6 ? shift - 6 : 0) {
    const u64 at = (u64)first + ((u64)lane << shift);
    const uint32_t o = at > 0xff800000ull ? 0xff800000u : (uint32_t)at;  // (past -Inf: NaN)
    const float x = __uint_as_float(o & 0x80000000u ? o : ~o & 0x7fffffffu);
    // the order begins with NaNs, which no entry is: they count as in
    const u64 in = __ballot(at <= 0xff800000ull && (x != x || bin_of(x) <= b));
    first += (uint32_t)(63 - __builtin_clzll(in | 1)) << shift;
    if (shift == 0) break;
  }
  return uniform(__uint_as_float(first & 0x80000000u ? first : ~first & 0x7fffffffu));
}

// The next float below a finite one.
__device__ __forceinline__ float below(float x) {
  const uint32_t b = __float_as_uint(x);
  return x == 0.0f ? __uint_as_float(0x80000001u) : __uint_as_float(x > 0.0f ? b - 1 : b + 1);
}

// A row with +Inf: its like weigh 1 and nothing else is a candidate, so each setting
// leaves a number of them, by index.
template <bool BF>
__device__ __forceinline__ void sample_infinite(const SampleArgs &a, Shared &s, const char *row, int r, int k, float top_p, float min_p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto is_inf = [&](int i) {
    return i < a.V && (BF ? bf16_to_f32(reinterpret_cast<const uint16_t *>(row)[i]) : reinterpret_cast<const float *>(row)[i]) ==
                          __builtin_inff();
  };
  if (tid == 0) s.n_list = 0;
  __syncthreads();
  int mine = 0;
  for (int i = tid; i < a.V; i += ST) mine += is_inf(i);
  atomicAdd(&s.n_list, mine);
  __syncthreads();
  int n = s.n_list;
  if (k > 0) n = min(n, k);
  if (top_p < 1.0f) n = min(n, max(1, (int)ceil((double)top_p * n)));
  if (min_p > 1.0f) n = 1;
  const double at = floor((double)a.u[r] * n);
  const int pick = at >= 0.0 ? min(n - 1, (int)fmin(at, 2e9)) : 0;
  // the pick-th of them, a tile of lanes at a time
  int before = 0;
  for (int i0 = 0; i0 < a.V; i0 += ST) {
    const bool in = is_inf(i0 + tid);
    const u64 votes = __ballot(in);
    if (lane == 0) s.wave_c[wave] = __popcll(votes);
    __syncthreads();
    int total = 0, place = before + __popcll(votes & ((1ull << lane) - 1));
    for (int v = 0; v < ST / 64; ++v) {
      if (v < wave) place += (int)s.wave_c[v];
      total += (int)s.wave_c[v];
    }
    if (in && place == pick) {
      a.tokens[r] = i0 + tid;
      if (a.probs) a.probs[r] = (float)(1.0 / n);
    }
    before += total;
    __syncthreads();
    if (before > pick) break;
  }
}

template <bool BF>
__global__ __launch_bounds__(ST, 1) void sample_tokens_kernel(SampleArgs a) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x, V = a.V;
  const char *x0 = static_cast<const char *>(a.logits) + (long long)row * a.row_stride * (BF ? 2 : 4);
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;

  // the maximum and its first index
  if (tid == 0) s.key = ~0ull, s.n_cand = 0, s.candidates = 0;
  if (tid < TABLE) s.table[tid] = ONE * (tid < TABLE / 2 ? exp2_small(tid / 64.0) : 2.0 * exp2_small(tid / 64.0 - 1.0));
  __syncthreads();
  float mine = -__builtin_inff();  // this lane's maximum
  int finite = 0;                  // its candidates
  each_four<BF, BF ? 1 : 8>(x0, V, [&](const float (&x)[4], int) __attribute__((always_inline)) {
    mine = fmaxf(fmaxf(fmaxf(mine, x[0]), fmaxf(x[1], x[2])), x[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) finite += x[e] > -__builtin_inff();
  });
  {
    float m = mine;
    for (int off = 32; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, off)), finite += __shfl_xor(finite, off);
    if (lane == 0) s.wave_m[tid >> 6] = (u64)__float_as_uint(m), atomicAdd(&s.candidates, finite);
  }
  clear_bins(s);
  float top = -__builtin_inff();
  for (int v = 0; v < ST / 64; ++v) top = fmaxf(top, __uint_as_float((uint32_t)s.wave_m[v]));
  top = uniform(top) + 0.0f;  // -0 is 0
  if (!(top > -__builtin_inff())) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.probs) a.probs[row] = 0.0f;
    }
    return;
  }
  if (!(temp > 0.0f) || k == 1 || top_p <= 0.0f) {  // the first of the largest
    each_four<BF, BF ? 1 : 8>(x0, V, [&](const float (&x)[4], int i) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x[e] == top) atomicMin(&s.key, (u64)(i + e));
    });
    __syncthreads();
    if (tid == 0) {
      a.tokens[row] = (int)s.key;
      if (a.probs) a.probs[row] = 1.0f;
    }
    return;
  }
  if (top == __builtin_inff()) {
    sample_infinite<BF>(a, s, x0, row, k, top_p, min_p);
    return;
  }
  Weights weight;
  weight.table = s.table;
  weight.rate = uniform(1.4426950408889634074 / (double)temp);
  weight.top = uniform((double)top);
  const int candidates = uniform(s.candidates);
  auto near_bin = [&](float x) { return min(weight.steps(x), BINS - 1); };
  auto far_bin = [&](float x) { return min((weight.steps(x) - (BINS - 1)) >> 2, BINS - 1); };  // of a last near bin's
  auto keep = [&](float x, int i) __attribute__((always_inline)) {  // to the list in LDS
    const int at = atomicAdd(&s.n_cand, 1);
    if (at < CAND) s.cx[at] = x + 0.0f, s.ci[at] = i;
  };

  // All entries of the row for which in(x) to the list: a round's are marked in a bit
  // each and then kept, by index, with one atomic addition a lane; their logits are read
  // again at the end.  (Kept one by one the atomic's latency was most of the pass.)
  auto keep_all = [&](auto in) __attribute__((always_inline)) {
    uint32_t hits = 0;
    auto mark = [&](const float (&x)[4], int) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) hits = hits * 2 + (in(x[e]) ? 1 : 0);
    };
    auto keep_marked = [&](int i0, int n) __attribute__((always_inline)) {
      if (hits == 0) return;
      int at = atomicAdd(&s.n_cand, __popc(hits));
      while (hits) {
        const int bit = 31 - __clz(hits), j = n - 1 - bit;
        hits ^= 1u << bit;
        if (at < CAND) s.ci[at] = i0 + j / PER<BF> * (ST * PER<BF>) + j % PER<BF>;
        ++at;
      }
    };
    each_four<BF, BF ? 1 : 8>(x0, V, mark, keep_marked);
    __syncthreads();
    const int kept = uniform(min(s.n_cand, CAND));
#pragma unroll 4
    for (int e = tid; e < kept; e += ST) {
      const int i = s.ci[e];
      s.cx[e] = (BF ? bf16_to_f32(reinterpret_cast<const uint16_t *>(x0)[i]) : reinterpret_cast<const float *>(x0)[i]) + 0.0f;
    }
    __syncthreads();
  };

  // The entries that the searches look at: the row's, or the list's where it holds
  // all that can be drawn.
  bool listed_all = false;
  u64 range_m = 0, range_n = 0;
  if (V <= CAND || (k > 0 && k <= ST / 2)) {
    float least = -3.402823466e38f;  // the list's last entry
    bool small = true;
    if (V > CAND) {
      if (mine > -__builtin_inff()) atomicAdd(&s.count[near_bin(mine)], 1u);
      __syncthreads();
      scan_bins(s, range_m, range_n);
      const int last = range_n >= (u64)k ? bin_of_total(s, true, (u64)k - 1) : BINS - 1;
      small = last < BINS - 1;
      if (small) least = least_in(near_bin, last);
    }
    if (small) {
      keep_all([&](float x) __attribute__((always_inline)) { return x >= least; });
      listed_all = uniform(s.n_cand) <= CAND;
    }
    __syncthreads();
    if (!listed_all && tid == 0) s.n_cand = 0;
  }
  const int n_all = listed_all ? uniform(s.n_cand) : 0;
  auto each = [&](auto f) __attribute__((always_inline)) {
    if (listed_all) {
#pragma unroll 1
      for (int e = tid; e < n_all; e += ST) f(s.cx[e], s.ci[e]);
    } else {
      each_four<BF, BF ? 1 : 4>(x0, V, [&](const float (&x)[4], int i) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x[e] > -__builtin_inff()) f(x[e] + 0.0f, i + e);
      });
    }
  };

  Range g{kNear, 0, 64, 64, kNear, 0, 0, 0};
  auto inside = [&](float x, int i) __attribute__((always_inline)) {  // of the range
    if (near_bin(x) != (g.from == kNear && g.level == kKeys ? g.bin : BINS - 1)) return false;
    if (g.level == kFar) return true;
    if (g.from == kFar && far_bin(x) != g.bin) return false;
    return g.shift == 64 || order_key(x, i) >> g.shift == g.prefix;
  };

  // The searches in turn: 0 for top-k's count, 1 for top-p's mass, 2 for the draw.
  u64 m = 0, keep_m = 0, t = 0;
  const double u = uniform((double)a.u[row]);
  auto bound_p = [&](u64 mass) {
    const double v = uniform(ceil((double)top_p * (double)mass));
    return v >= 1.0 ? min((u64)v, mass) - 1 : (u64)0;
  };
  auto bound_u = [&](u64 mass) {
    const double v = uniform(floor(u * (double)mass));
    return v >= 0.0 ? min((u64)v, mass - 1) : (u64)0;
  };
  // min-p's bound lies in the bin of its power of two or, by rounding, one next to it;
  // past the last bin but one, in any bin from there on
  const u64 min_mass = min_p > 0.0f ? (u64)uniform(ceil(fmin((double)min_p, 2.0) * ONE)) : 0;
  const int min_at = min_p > 0.0f ? (int)fminf(fmaxf(-64.0f * log2f(min_p), 0.0f), (float)(BINS - 2)) : 0;
  const int min_bin = uniform(max(min_at - 1, 0));
  const uint32_t min_bins = min_p > 0.0f ? (min_at < BINS - 2 ? 4u : 0x7fffffffu) : 0u;
  // The entries of bins are counted where top-k needs it.  Elsewhere the bins' masses
  // say it, from above, as all weights of a bin are alike: half of the atomics.
  const bool counted = listed_all || k > 0;
  bool by_count = false, have = false, known = false;
  int iv[3][2] = {{0, 0}, {0, 0}, {0, 0}};  // the near bins whose entries are in the list: [first, past the last)
  for (int step = -1;;) {
    if (!have) {
      if (tid == 0) s.cum = 0, s.total = 0;
      clear_bins(s);
      if (g.level == kNear) {
        // what min-p keeps of the bins that its bound can be in is counted on the way; the
        // last bin, which most entries may be in, is what the others leave of the total
        u64 km = 0, total = 0;
        auto add = [&](const float (&x)[4], int) __attribute__((always_inline)) {
          u64 f[4];
          int b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[e] = weight(x[e], b[e]);
            total += f[e];
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (b[e] < BINS - 1) {
              atomicAdd(&s.mass[b[e]], f[e]);
              if (counted) atomicAdd(&s.count[b[e]], 1u);
            }
            if ((uint32_t)(b[e] - min_bin) < min_bins && f[e] >= min_mass) km += f[e];
          }
        };
        if (listed_all) {
          const float none = __builtin_nanf("");
#pragma unroll 1
          for (int e = tid; e < n_all; e += ST) {
            const float x[4] = {s.cx[e], none, none, none};
            add(x, 0);
          }
        } else {
          each_four<BF, BF ? 1 : 4>(x0, V, add);
        }
        for (int off = 32; off; off >>= 1) {
          km += __shfl_xor(km, off);
          total += __shfl_xor(total, off);
        }
        if (lane == 0) {
          atomicAdd(&s.total, total);
          atomicAdd(&s.cum, km);
        }
      } else {
        each([&](float x, int i) __attribute__((always_inline)) {
          if (!inside(x, i)) return;
          const int b = g.level == kFar ? far_bin(x)
                                        : (int)(order_key(x, i) >> g.next & ((1ull << (g.shift - g.next)) - 1));
          atomicAdd(&s.mass[b], weight(x));
          atomicAdd(&s.count[b], 1u);
        });
      }
      __syncthreads();
      scan_bins(s, range_m, range_n);
      if (g.level == kNear) range_m = uniform(s.total), range_n = (u64)(listed_all ? n_all : candidates);
      have = true;
    }
    if (step < 0) {
      keep_m = uniform(s.cum) + mass_before(s, min_bin, range_m);
      m = range_m;
      step = 0;
      __syncthreads();
    }
    if (!known) {  // the search's bound
      if (step == 0) {
        if (k > 0 && (u64)k < range_n) {
          by_count = true;
          t = (u64)k - 1;
          known = true;
        } else {
          step = 1;
        }
      }
      if (step == 1) {
        if (top_p < 1.0f) {
          by_count = false;
          t = bound_p(m);
          known = true;
        } else {
          step = 2;
        }
      }
      if (step == 2) {
        if (min_p > 0.0f) m = min(m, keep_m > 0 ? keep_m : (u64)ONE);
        by_count = false;
        t = bound_u(m);
        known = true;
      }
    }
    auto entries_of = [&](int from, int to) {
      if (counted || g.level != kNear) return count_before(s, to, range_n) - count_before(s, from, range_n);
      if (to == BINS) return CAND + 1;
      const float least = exp2f(42.0f - ((float)to - 0.5f) / 64.0f);  // of a weight
      return uniform((int)fminf((float)(mass_before(s, to, range_m) - mass_before(s, from, range_m)) / least * 1.01f + 1.0f, CAND + 1.0f));
    };
    const int bin = bin_of_total(s, by_count, t - (by_count ? g.count : g.mass));
    const u64 before_m = mass_before(s, bin, range_m);
    const int before_n = count_before(s, bin, range_n);
    const int entries = entries_of(bin, bin + 1);
    g.mass += before_m;
    g.count += (u64)before_n;
    const bool near = g.level == kNear;
    if (g.level == kKeys) {
      g.prefix = (g.shift == 64 ? 0 : g.prefix << (g.shift - g.next)) | (u64)bin;
      g.shift = g.next;
    }
    if (entries > LIST) {  // divide the bin
      if (near && bin == BINS - 1) {
        g.level = kFar;
      } else {
        if (g.level != kKeys) g.from = g.level, g.bin = bin, g.level = kKeys;
        g.next = g.shift > 11 ? g.shift - 11 : 0;
      }
      __syncthreads();
      have = false;
      continue;
    }
    // The bin's entries, from the list or, to the list, from the row.
    const auto in_list = [&](int b) {
      return (b >= iv[0][0] && b < iv[0][1]) || (b >= iv[1][0] && b < iv[1][1]) || (b >= iv[2][0] && b < iv[2][1]);
    };
    if (!listed_all && !(near && in_list(bin))) {
      iv[0][0] = bin, iv[0][1] = bin + 1;
      iv[1][0] = iv[1][1] = iv[2][0] = iv[2][1] = 0;
      if (near) {
        // where the searches that follow can end, from the mass that this one leaves
        u64 lo = mass_before(s, bin, range_m), hi = mass_before(s, bin + 1, range_m);
        auto follow = [&](int w, u64 t_lo, u64 t_hi) __attribute__((always_inline)) {
          iv[w][0] = bin_of_total(s, false, t_lo);
          iv[w][1] = bin_of_total(s, false, t_hi) + 1;
          lo = mass_before(s, iv[w][0], range_m);
          hi = mass_before(s, iv[w][1], range_m);
        };
        if (lo == 0) lo = 1;  // (a search leaves at least an entry)
        if (step == 0 && top_p < 1.0f) follow(1, bound_p(lo), bound_p(hi));
        if (step < 2) {
          if (lo == 0) lo = 1;
          if (min_p > 0.0f && keep_m > 0) lo = min(lo, keep_m), hi = min(hi, keep_m);
          follow(2, bound_u(lo), bound_u(hi));
        }
        int total = entries;
#pragma unroll
        for (int w = 1; w < 3; ++w)
          if (iv[w][1] > iv[w][0]) total = min(total + entries_of(iv[w][0], iv[w][1]), CAND + 1);
        if (total > CAND || iv[1][1] >= BINS || iv[2][1] >= BINS || bin == BINS - 1)
          iv[1][0] = iv[1][1] = iv[2][0] = iv[2][1] = 0;
      }
      if (tid == 0) s.n_cand = 0;
      __syncthreads();
      if (near && bin < BINS - 1) {
        // the intervals as logits, [lo, hi]: an entry is in one that leaves it as it is
        float lo[3], hi[3];
#pragma unroll
        for (int w = 0; w < 3; ++w) {
          const int from = iv[w][0], to = iv[w][1];
          lo[w] = to > from ? least_in(near_bin, to - 1) : __builtin_inff();
          hi[w] = to > from && from > 0 ? below(least_in(near_bin, from - 1)) : __builtin_inff();
        }
        if (iv[1][1] == iv[1][0]) lo[1] = lo[0], hi[1] = hi[0];
        const bool three = iv[1][1] > iv[1][0] && iv[2][1] > iv[2][0];
        if (!three && iv[2][1] > iv[2][0]) lo[1] = lo[2], hi[1] = hi[2];
        keep_all([&](float x) __attribute__((always_inline)) {
          bool in = (__builtin_amdgcn_fmed3f(x, lo[0], hi[0]) == x) | (__builtin_amdgcn_fmed3f(x, lo[1], hi[1]) == x);
          if (three) in |= __builtin_amdgcn_fmed3f(x, lo[2], hi[2]) == x;
          return in;
        });
      } else {
        const int level = g.level;
        if (level != kKeys) g.from = level, g.bin = bin, g.level = kKeys;  // inside(): this bin
        each([&](float x, int i) __attribute__((always_inline)) {
          if (inside(x, i)) keep(x, i);
        });
        g.level = level;
      }
    }
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    const int kept = uniform(min(s.n_cand, CAND));
    {
      const int level = g.level;
      if (level != kKeys) g.from = level, g.bin = bin, g.level = kKeys;
      for (int e = tid; e < kept; e += ST) {
        const float x = s.cx[e];
        if (!inside(x, s.ci[e])) continue;
        const int at = atomicAdd(&s.n_list, 1);
        if (at < LIST) s.list[at] = make_ulonglong2(order_key(x, s.ci[e]), weight(x));
      }
      g.level = level;
    }
    __syncthreads();
    // ranked by comparing each with all
    const int listed = uniform(min(s.n_list, LIST));
    for (int e = tid; e < listed; e += ST) {
      const u64 key = s.list[e].x, w = s.list[e].y;
      uint32_t ahead = 0;
      u64 cum = g.mass;
#pragma unroll 8
      for (int j = 0; j < listed; ++j) {
        const ulonglong2 v = s.list[j];
        ahead += v.x < key;
        cum += v.x < key ? v.y : 0;
      }
      const u64 rank = g.count + ahead;
      const u64 lo = by_count ? rank : cum, hi = by_count ? rank + 1 : cum + w;
      if (lo <= t && t < hi) s.cum = cum + w, s.own = w, s.pos = (int)(uint32_t)key;
    }
    __syncthreads();
    if (step == 2) break;
    m = min(m, uniform(s.cum));
    __syncthreads();
    // a divided bin's histogram is of no use for the next search
    if (!near) {
      have = false;
      iv[0][1] = iv[1][1] = iv[2][1] = 0;
    }
    g = Range{kNear, 0, 64, 64, kNear, 0, 0, 0};
    known = false;
    ++step;
  }
  if (tid == 0) {
    a.tokens[row] = s.pos;
    if (a.probs) a.probs[row] = (float)((double)s.own / (double)m);
  }
}

}  // namespace

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
