// k_token_logprobs.hip -- of each row of logits: the log probability and rank of a given
// token, the entropy, and the k best entries.
//
//   m = max x, S = sum 2^d, W = sum 2^d d, d = (x - m) log2 e;
//   log p(x) = (x - m) - ln S, entropy = ln S - ln 2 W / S.
//
// A row is read once.  It is cut into parts, each of which a workgroup of four waves holds
// in registers (NCH runs of 16 bytes a lane), so that the maximum is known before the
// sums begin and an entry costs one exponential; a second kernel joins the parts where a row
// has several.  The exponent d is one fma, x log2 e - c, c = m log2 e rounded; what c's rounding
// left, the same for all entries, is taken off the sums' logarithm at the end.  It grows with m
// (2^-4 at 1e6, past the exponential's range from 2e9 on): from 1e6 on, which only masked rows and
// parts reach, d is (x - m) log2 e (2000 rows of 128000 all but masked at -1e30: 116 us, others 103).
//
// The k best: at least k of 64 groups of lanes have a maximum that is no less than the k-th largest
// of theirs, so that the part's k best are among the entries that reach it: little more
// than k, which go to a list in LDS and are ranked by comparing each with all.  One
// wave looks for that bound while the others sum.  A list that overflows (a row of equal
// logits, or one whose part is masked at one finite value) is searched for the k best one after the other instead,
// each time over the part in memory: 48 such rows of 50257 with 20 alternatives 70 us in place of 12, 2000 of 128000
// with five 1770 in place of 119 (masked with -Inf 118, which is no candidate).
//
// Where rows are many, their bytes and the vector instructions bound it alike: 2000 rows of 128000 bf16,
// 512 MB, 119 us with five alternatives, 4.3 TB/s, of which 6 are the join (some 900 instructions a
// wave for its 4096 entries, and 64 exponentials).  Where they are few, the chain of a part's steps and the join:
// 48 rows of 50257 with 20 alternatives 7.3 and 4.3, without 4.6 and 2.3.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kernels.hpp"
#include "npu_device.hpp"
#include "plans.hpp"

namespace npu {

namespace {

constexpr int LT = 256;      // lanes of a workgroup
constexpr int LIST = 1024;   // entries that are ranked at once (a multiple of 16)
constexpr int MAX_K = 32;
constexpr int MAX_PARTS = LT;  // of a row: 129 at most with 8 runs a lane (2^20 f32)
constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;

typedef unsigned long long u64;

// An entry's place in the order as a number, smaller first: by logit, descending, then index.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
  return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float from_order(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o : ~o & 0x7fffffffu); }
constexpr u64 NO_KEY = ~0ull;

// The next float below one that is not -Inf.
__device__ __forceinline__ float below(float x) {
  const uint32_t b = __float_as_uint(x);
  return x == 0.0f ? __uint_as_float(0x80000001u) : __uint_as_float(x > 0.0f ? b - 1 : b + 1);
}

// A part's result, and behind it the k keys.
struct Part {
  float m, S, W;  // m -Inf: no entry above -Inf (S, W 0)
  int before;     // entries before the token
};
__device__ __forceinline__ u64 *keys_of(Part *p) { return reinterpret_cast<u64 *>(p + 1); }
__host__ __device__ constexpr size_t part_bytes(int k) { return sizeof(Part) + 8 * (size_t)k; }

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_mov<0xb1>(v));   // lane ^ 1
  v = fmaxf(v, dpp_mov<0x4e>(v));   // lane ^ 2
  v = fmaxf(v, dpp_mov<0x141>(v));  // the other half of eight
  v = fmaxf(v, dpp_mov<0x140>(v));  // of sixteen
  auto of = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
  return fmaxf(fmaxf(of(0), of(16)), fmaxf(of(32), of(48)));
}

// The token's logit (-Inf: NaN, or none), read where the kernels begin.
struct Given {
  bool given;
  int token;
  float x;
  __device__ __forceinline__ Given(const TokenLogprobsArgs &a, long long row) {
    token = a.tokens[row];
    given = token >= 0 && token < a.V;
    x = -__builtin_inff();
    const long long at = row * a.row_stride + token;
    if (given) x = a.bf16 ? bf16_to_f32(static_cast<const uint16_t *>(a.logits)[at]) : static_cast<const float *>(a.logits)[at];
    if (!(x > -__builtin_inff())) x = -__builtin_inff();
  }
};

// What the joined sums give; lane `t` of the caller writes alternative t.
__device__ __forceinline__ void finish(const TokenLogprobsArgs &a, long long row, const Given &tok, const Part &p, const u64 *keys, int t) {
  const float inf = __builtin_inff(), lnS = p.S > 0.0f ? logf(p.S) : 0.0f;
  // ((x - m) is exact or far from 0)
  auto logp = [&](float x) { return !(x > -inf) ? -inf : x == p.m ? -lnS : (x - p.m) - lnS; };
  if (t == 0) {
    a.logprobs[row] = tok.given ? logp(tok.x) : 0.0f;
    if (a.ranks) a.ranks[row] = tok.given ? p.before : -1;
    if (a.entropy) a.entropy[row] = p.S > 0.0f ? lnS - LN2 * (p.W / p.S) : 0.0f;
  }
  if (t < a.k) {
    const u64 key = keys[t];
    const float x = from_order((uint32_t)(key >> 32));
    const bool in = key != NO_KEY && (p.m < inf || x == inf);
    a.top_tokens[row * a.toks_stride + t] = in ? (int)(uint32_t)key : -1;
    a.top_logprobs[row * a.tops_stride + t] = in ? logp(x) : -inf;
  }
}

// How many of n keys in LDS are smaller; NO_KEY lies behind them up to a multiple of 16 (read one by
// one, what a multiple leaves took most of the time).
__device__ __forceinline__ int keys_below(const u64 *list, int n, u64 key) {
  int ahead = 0;
#pragma unroll 1
  for (int j = 0; j < n; j += 16) {
    ulonglong2 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const ulonglong2 *>(list + j + 2 * i);
#pragma unroll
    for (int i = 0; i < 8; ++i) ahead += (int)(v[i].x < key) + (int)(v[i].y < key);
  }
  return ahead;
}
// The k smallest of n keys in LDS, in order, to `out`; called by all lanes of a workgroup.  (list's first
// LT entries were NO_KEY before)
__device__ __forceinline__ void rank_keys(u64 *list, int n, int k, u64 *out) {
  if (n > LT) {
    if (threadIdx.x < (-n & 15)) list[n + threadIdx.x] = NO_KEY;
    __syncthreads();
  }
  for (int e = threadIdx.x; e < n; e += blockDim.x) {
    const u64 key = list[e];
    const int ahead = keys_below(list, n, key);
    if (ahead < k) out[ahead] = key;
  }
}

template <bool BF, int NCH>
__global__ __launch_bounds__(LT) void token_logprobs_kernel(TokenLogprobsArgs a, int parts) {
  constexpr int PER = BF ? 8 : 4, ES = BF ? 2 : 4, NW = LT / 64;
  __shared__ __attribute__((aligned(16))) u64 list[LIST];
  __shared__ u64 best[MAX_K];
  __shared__ float wave_a[NW], wave_b[NW];
  __shared__ int wave_c[NW];
  __shared__ uint32_t ups[LT], bound;
  __shared__ u64 wave_k[NW];
  __shared__ int n_list;
  const float inf = __builtin_inff();
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long row = blockIdx.x / (unsigned)parts;
  const int part = blockIdx.x % (unsigned)parts;
  const char *p = static_cast<const char *>(a.logits) + row * a.row_stride * ES;
  // runs of 16 bytes at aligned places; what lies before the first whole one, and after the
  // last, at most PER - 1 entries each, goes to lanes of the part whose range has it
  const int skew = (int)((uintptr_t)p & 15) / ES;
  const u32x4 *body = reinterpret_cast<const u32x4 *>(p - skew * ES);
  const int whole0 = skew ? 1 : 0, whole1 = (a.V + skew) / PER;
  const int c0 = part * NCH * LT + tid;
  u32x4 v[NCH];
  constexpr uint32_t NONE = BF ? 0xff80ff80u : 0xff800000u;  // -Inf
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = c0 + i * LT;
    v[i] = u32x4{NONE, NONE, NONE, NONE};
    if (c >= whole0 && c < whole1) v[i] = body[c];
  }
  auto entry = [&](int j) __attribute__((always_inline)) {
    return BF ? bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[j]) : reinterpret_cast<const float *>(p)[j];
  };
  int edge_j = -1;
  if (part == 0 && tid < PER && tid < min(whole0 * PER - skew, a.V)) edge_j = tid;
  const int tail = max(whole1, whole0);
  if (part == tail / (NCH * LT) && tid >= PER && tid < 2 * PER) {
    const int j = tail * PER - skew + tid - PER;
    if (j < a.V) edge_j = j;
  }
  float edge = -inf;
  if (edge_j >= 0) edge = entry(edge_j);
  const Given tok(a, row);
  const int token = tok.token;
  const float xt = tok.x;
  if (tid == 0) n_list = 0;
  if (a.k > 0) list[tid] = NO_KEY;
  auto get = [&](u32x4 u, int e) __attribute__((always_inline)) {
    return BF ? __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16) : __uint_as_float(u[e]);
  };
  // (the entries are taken out of the runs again each time: all of them would not fit)
  auto packed = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) asm volatile("" : "+v"(v[i]));
  };
  // every entry of the part again, from memory: f(x, j)
  auto again = [&](auto f) __attribute__((always_inline)) {
    const int from = max(0, part * NCH * LT * PER - skew), to = min(a.V, (part + 1) * NCH * LT * PER - skew);
#pragma unroll 1
    for (int j = from + tid; j < to; j += LT) f(entry(j), j);
  };
  // the lane's maximum, the part's
  float mine = fmaxf(edge, -inf), run_max[NCH];  // (no NaN)
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    run_max[i] = -inf;
#pragma unroll
    for (int e = 0; e < PER; e += 2) run_max[i] = fmaxf(fmaxf(run_max[i], get(v[i], e)), get(v[i], e + 1));
    mine = fmaxf(mine, run_max[i]);
  }
  packed();
  {
    const float m = wave_max(mine);
    if (lane == 0) wave_a[wave] = m;
    if (a.k > 0) ups[tid] = ~order_bits(mine);  // (a number that rises with it)
  }
  __syncthreads();
  float m = wave_a[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) m = fmaxf(m, wave_a[w]);
  if (a.k > 0 && wave == 0) {
    // the k-th largest of the maxima of NW lanes each, two bits at a time down to the 16th (what is left
    // of f32 makes the bound a little lower)
    uint32_t up = 0, found = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) up = max(up, ups[64 * w + lane]);
    auto reach = [&](uint32_t at) __attribute__((always_inline)) { return __popcll(__ballot(up >= at)); };
#pragma unroll 1
    for (int b = 30; b >= 16; b -= 2) {
      const uint32_t at1 = found | 1u << b, at2 = found | 2u << b, at3 = found | 3u << b;
      const int n1 = reach(at1), n2 = reach(at2), n3 = reach(at3);
      found = n3 >= a.k ? at3 : n2 >= a.k ? at2 : n1 >= a.k ? at1 : found;
    }
    if (lane == 0) bound = found;
  }
  // sums, the rank, the list
  const bool far = !(fabsf(m) < 1e6f);  // summed from x - m below
  const float c = far ? 0.0f : m * LOG2E, rest = far ? 0.0f : fmaf(m, LOG2E, -c);
  float rest_off;  // 2^-rest, as 1 / what the exponential makes of rest (a step after the instruction's 1 ulp)
  {
    const float w = __builtin_amdgcn_exp2f(rest), near = __builtin_amdgcn_rcpf(w);
    rest_off = fmaf(near, fmaf(-w, near, 1.0f), near);
  }
  const float at_before = xt > -inf ? below(xt) : -inf;
  float S = 0.0f, W = 0.0f;
  int before = 0;
  auto add = [&](float x) __attribute__((always_inline)) {
    const float d = fmaxf(fmaf(x, LOG2E, -c), -1000.0f), w = __builtin_amdgcn_exp2f(d);
    S += w;
    W = fmaf(w, d, W);
  };
  auto keep = [&](int at, float x, int j) __attribute__((always_inline)) {
    if (at < LIST) list[at] = (u64)order_bits(x) << 32 | (uint32_t)j;
  };
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    // (runs of a wave without an entry before the token are most of them, where a model gave the token)
    if (__any(run_max[i] >= xt)) {
      const float over = (c0 + i * LT) * PER - skew + PER <= token ? at_before : xt;
#pragma unroll
      for (int e = 0; e < PER; ++e) before += get(v[i], e) > over;
    }
    asm volatile("" : "+v"(v[i]));
#pragma unroll
    for (int e = 0; e < PER; e += 4) {
      // (four at a time: a result of the exponential is not there for the next instruction)
      float x[4], d[4], w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = get(v[i], e + q);
#pragma unroll
      for (int q = 0; q < 4; ++q) d[q] = fmaxf(fmaf(x[q], LOG2E, -c), -1000.0f);
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = __builtin_amdgcn_exp2f(d[q]);
#pragma unroll
      for (int q = 0; q < 4; ++q) W = fmaf(w[q], d[q], W);
      S += (w[0] + w[1]) + (w[2] + w[3]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  add(edge);  // (-Inf: none)
  before += edge > (edge_j < token ? at_before : xt);
  packed();
  float least = __builtin_inff();
  if (a.k > 0) {
    __syncthreads();
    least = fmaxf(from_order(~bound), -3.402823466e38f);  // (-Inf is no candidate)
  }
  if (a.k > 0 && mine >= least) {
    uint32_t runs = 0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) runs |= (uint32_t)(run_max[i] >= least) << i;
    while (runs) {
      const int at = __builtin_ctz(runs);
      runs &= runs - 1;
      u32x4 u = v[0];
#pragma unroll
      for (int i = 1; i < NCH; ++i)
        if (at == i) u = v[i];
      int n = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) n += get(u, e) >= least;
      int to = atomicAdd(&n_list, n);  // (one for a run: its answer is a wait)
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (get(u, e) >= least) keep(to++, get(u, e), (c0 + at * LT) * PER - skew + e);
    }
    if (edge >= least) keep(atomicAdd(&n_list, 1), edge, edge_j);
  }
  if (!tok.given) {
    before = 0;
  } else if (!(xt > -inf)) {
    // behind all above -Inf, and those like it with a lower index
    before = 0;
    again([&](float x, int j) { before += j < token || x > -inf; });
  } else if (tid < PER) {
    // the run that holds the token: its equals before it, unless they were edges
    const int run = (token + skew) / PER, j = run * PER - skew + tid;
    if (run >= whole0 && run < whole1 && run / (NCH * LT) == part && j < token) before += entry(j) == xt;
  }
  if (far) {
    S = W = 0.0f;
    auto add_far = [&](float x) __attribute__((always_inline)) {
      const float d = x == m ? 0.0f : fmaxf((x - m) * LOG2E, -1000.0f), w = __builtin_amdgcn_exp2f(d);
      S += w;
      W = fmaf(w, d, W);
    };
    if (m > -inf) {  // (a run at a time: all at once cost every other row 2 %)
#pragma unroll 1
      for (int at = 0; at < NCH; ++at) {
        u32x4 u = v[0];
#pragma unroll
        for (int i = 1; i < NCH; ++i)
          if (at == i) u = v[i];
#pragma unroll
        for (int e = 0; e < PER; ++e) add_far(get(u, e));
      }
      add_far(edge);
    }
  }
  S = wave_sum(S);
  W = wave_sum(W);
  before = (int)wave_sum((float)before);  // (a row has at most 2^20)
  __syncthreads();  // (wave_a was read above)
  if (lane == 0) wave_a[wave] = S, wave_b[wave] = W, wave_c[wave] = before;
  __syncthreads();
  const int n = n_list;
  if (a.k > 0) {
    if (tid < a.k) best[tid] = NO_KEY;
    __syncthreads();
    if (n <= LIST) {
      rank_keys(list, n, a.k, best);
    } else {
      u64 last = 0;  // (no candidate's key: NaN's place in the order)
#pragma unroll 1
      for (int r = 0; r < a.k; ++r) {
        u64 next = NO_KEY;
        again([&](float x, int j) {
          const u64 key = (u64)order_bits(x) << 32 | (uint32_t)j;
          if (x >= least && key > last) next = min(next, key);
        });
        for (int off = 32; off; off >>= 1) next = min(next, (u64)__shfl_xor(next, off));
        if (lane == 0) wave_k[wave] = next;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) next = min(next, wave_k[w]);
        if (tid == 0) best[r] = next;
        last = next;
        __syncthreads();
      }
    }
    __syncthreads();
  }
  Part out{m, 0.0f, 0.0f, 0};
#pragma unroll
  for (int w = 0; w < NW; ++w) out.S += wave_a[w], out.W += wave_b[w], out.before += wave_c[w];
  // S and W of exact exponents: each is off by `rest`.  The largest entry is 1 of S and 0 of W: divided by
  // what the exponential makes of `rest`, so that it comes out as 1 (or the number below it), and S is 1 at
  // least and W 0 at most, no log probability is above 0 and no entropy below.
  if (out.S > 0.0f) {
#pragma clang fp contract(off)
    const float shift = rest * out.S;
    out.W = fminf((out.W - shift) * rest_off, 0.0f);
    out.S = fmaxf(out.S * rest_off, 1.0f);
  }
  if (parts == 1) {
    finish(a, row, tok, out, best, tid);
    return;
  }
  Part *to = reinterpret_cast<Part *>(static_cast<char *>(a.workspace) + (row * parts + part) * part_bytes(a.k));
  if (tid == 0) *to = out;
  if (tid < a.k) keys_of(to)[tid] = best[tid];
}

// A row's parts, one a lane; their sums in a fixed order (a wave's lanes, then the waves).  The k
// best come no later than the k-th of the lists' first keys (of so many of each that there are k):
// most of the keys need not be ranked.
__global__ __launch_bounds__(LT) void token_logprobs_join_kernel(TokenLogprobsArgs a, int parts) {
  constexpr int NW = LT / 64;
  __shared__ __attribute__((aligned(16))) u64 heads[MAX_PARTS], list[MAX_K * MAX_K];
  __shared__ u64 best[MAX_K];
  __shared__ float wave_m[NW], wave_s[NW], wave_w[NW];
  __shared__ int wave_b[NW];
  __shared__ u64 bound;
  __shared__ int n_list;
  const float inf = __builtin_inff();
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long row = blockIdx.x;
  const Given tok(a, row);
  const size_t step = part_bytes(a.k);
  char *from = static_cast<char *>(a.workspace) + row * parts * step;
  auto part = [&](int i) { return reinterpret_cast<Part *>(from + i * step); };
  Part p{-inf, 0.0f, 0.0f, 0};
  if (tid < parts) p = *part(tid);
  const int depth = parts >= a.k ? 1 : (a.k + parts - 1) / parts, n_heads = a.k > 0 ? parts * depth : 0;  // (below 2 MAX_K, or parts)
  const u64 head = tid < n_heads ? keys_of(part(tid / depth))[tid % depth] : NO_KEY;
  // (the first of the keys below, asked for now)
  const int n_keys = parts * a.k, at0 = tid < n_keys ? tid / a.k : 0;
  const u64 key0 = tid < n_keys ? keys_of(part(at0))[tid - at0 * a.k] : NO_KEY;
  heads[tid] = head;
  list[tid] = NO_KEY;
  if (tid < a.k) best[tid] = NO_KEY;
  if (tid == 0) n_list = 0, bound = NO_KEY;
  const float m = wave_max(p.m);
  const int before = (int)wave_sum((float)p.before);
  if (lane == 0) wave_m[wave] = m, wave_b[wave] = before;
  __syncthreads();
  Part out{wave_m[0], 0.0f, 0.0f, 0};
#pragma unroll
  for (int w = 1; w < NW; ++w) out.m = fmaxf(out.m, wave_m[w]);
  float S = 0.0f, W = 0.0f;
  if (p.S > 0.0f) {
    const float d = p.m == out.m ? 0.0f : fmaxf((p.m - out.m) * LOG2E, -1000.0f), f = __builtin_amdgcn_exp2f(d);
    S = f * p.S;
    W = f * fmaf(d, p.S, p.W);
  }
  S = wave_sum(S);
  W = wave_sum(W);
  if (lane == 0) wave_s[wave] = S, wave_w[wave] = W;
  if (head != NO_KEY && keys_below(heads, n_heads, head) == a.k - 1) bound = head;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) out.S += wave_s[w], out.W += wave_w[w], out.before += wave_b[w];
  if (a.k > 0) {
    const u64 last = bound;
    for (int e = tid; e < n_keys; e += LT) {
      const int i = e / a.k;
      if (heads[i * depth] > last || heads[i * depth] == NO_KEY) continue;
      const u64 key = e < LT ? key0 : keys_of(part(i))[e - i * a.k];
      if (key > last || key == NO_KEY) continue;
      list[atomicAdd(&n_list, 1)] = key;  // (of at most k lists: with fewer real heads than k, all there are)
    }
    __syncthreads();
    rank_keys(list, n_list, a.k, best);
    __syncthreads();
  }
  finish(a, row, tok, out, best, tid);
}

// Runs of 16 bytes a lane holds: the most (8: more would halve the workgroups on a CU), or fewer
// where that leaves CUs without two workgroups, as far as a join takes the parts.  us with 8, 4, 2
// and 1 runs: 48 rows of 50257 bf16 and 20 alternatives 14.2, 14.0, 13.1, 13.9; one of 128000 13.0,
// 12.2, 12.1, 12.7; 256 and 5 27, 29, 37, 55; 2000 124, 154, 215, 368.
struct Cut {
  int nch, parts;
};
Cut cut_rows(int T, int V, bool bf16) {
  const int per = bf16 ? 8 : 4;
  const long long chunks = (V + per - 1) / per + 1;  // (a row that begins and ends inside a run)
  auto parts = [&](int nch) { return (chunks + nch * LT - 1) / (nch * LT); };
  int nch = 8;
  while (nch > 2 && (long long)T * parts(nch) < 2LL * device_cus() && parts(nch / 2) <= MAX_PARTS) nch /= 2;
  return Cut{nch, (int)parts(nch)};
}

}  // namespace

size_t token_logprobs_workspace(int T, int V, int k) {
  size_t most = 16;
  for (bool bf16 : {false, true}) {
    const Cut c = cut_rows(T, V, bf16);
    if (c.parts > 1) most = std::max(most, (size_t)T * c.parts * part_bytes(k));
  }
  return most;
}

hipError_t launch_token_logprobs(const TokenLogprobsArgs &a, hipStream_t s) {
  const Cut cut = cut_rows(a.T, a.V, a.bf16);
  const long long grid = (long long)a.T * cut.parts;
  auto kern = a.bf16 ? (cut.nch == 8 ? token_logprobs_kernel<true, 8> : cut.nch == 4 ? token_logprobs_kernel<true, 4>
                        : token_logprobs_kernel<true, 2>)
                     : (cut.nch == 8 ? token_logprobs_kernel<false, 8> : cut.nch == 4 ? token_logprobs_kernel<false, 4>
                        : token_logprobs_kernel<false, 2>);
  const double es = a.bf16 ? 2.0 : 4.0;
  {
    npu_launch_plan p = make_plan("token_logprobs", (int)grid, wg_per_cu(kern, LT), (int)grid, 16);
    const double n = std::min((double)a.V, (double)cut.nch * LT * (a.bf16 ? 8 : 4));
    p.load_phases = 2;
    p.tile_valu = n / 64 * 12.0;
    p.tile_lds_bytes = 8.0 * a.k * a.k;
    p.tile_load_bytes = n * es;
    p.tile_store_bytes = (double)part_bytes(a.k);
    p.hbm_bytes = (double)a.T * a.V * es;
    plans_add(p);
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(LT), 0, s, a, cut.parts);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || cut.parts == 1) return e;
  {
    npu_launch_plan p = make_plan("token_logprobs_join", a.T, wg_per_cu(token_logprobs_join_kernel, LT), a.T, 16);
    p.load_phases = 3;
    p.tile_valu = 100.0 * (LT / 64) + std::ceil(cut.parts / 64.0) * cut.parts * 4.0 + 4.0 * a.k * a.k;
    p.tile_lds_bytes = 8.0 * cut.parts * cut.parts;
    p.tile_load_bytes = (double)cut.parts * part_bytes(a.k);
    p.tile_store_bytes = 12.0 + 8.0 * a.k;
    p.hbm_bytes = 0.0;
    plans_add(p);
  }
  hipLaunchKernelGGL(token_logprobs_join_kernel, dim3(a.T), dim3(LT), 0, s, a, cut.parts);
  return hipGetLastError();
}

}  // namespace npu
