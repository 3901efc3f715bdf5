// k_paged_attention.hip -- attention of new tokens over a paged cache.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),
//   m = max_j scale q.k_j, over the keys a token sees; no key: o = 0.
//
// One pass over keys and values with the running maximum and sum: a new maximum
// scales what was summed so far by exp(m_old - m_new).  Partial (o, m, l) of
// different keys join the same way, so keys can be divided anywhere.
//
// One token per sequence reads every key once for G query heads: bound by the
// cache's bytes.  The work is divided by serve_batch.hpp's units, equal shares of
// 128-key blocks for two workgroups per CU whatever the sequences' lengths; a
// group of blocks that a border cuts leaves partial sums in the workspace, joined
// by a second launch.
//
// A wave takes 32 of a block's 128 keys and all the tile's 16 rows, without LDS:
//  - S^T = K Q^T: a key is an MFMA row, so a lane's A operand is 16 bytes of one
//    key as they lie in the cache.
//  - The lane that holds S^T's keys 4 q + i of both 16-key halves (q its 16-lane
//    row) feeds them to O^T = V^T P^T as the eight k slots of its row: the
//    probabilities never leave their lane.
//  - V is loaded by whole keys, eight keys and Dh / 16 entries a lane, which a
//    v_perm per dword turns into the A operands of Dh / 16 MFMAs; MFMA e covers
//    entries n Dh/16 + e of row n, so the lane ends with Dh / 16 consecutive
//    entries of each of its four rows' outputs.
// The next block's 16 KB per wave are in flight while this one is computed.  Measured: 48
// sequences of up to 8000 keys, 8 key heads of 128, 776 MB: 138 us; one of 131 000, 537 MB:
// 96 us; 5.6 TB/s both, more than a copy's rate.
//
// The probabilities are rounded to bf16 for the second product (2^-8 of each
// term, as the prompt's attention does); sums, maxima and outputs are f32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kernels.hpp"
#include "npu_device.hpp"
#include "plans.hpp"

namespace npu {

namespace {

constexpr int NT = 256;      // lanes of a workgroup
constexpr int ROWS = 16;     // rows of a tile
constexpr int KEYS = 128;    // keys of a unit, 32 a wave

// A partial row in the workspace: Dh sums, then m (base-2 logits), l, and, in a
// group's first part, the workgroup and the number of the parts that follow.
template <int DH>
struct PartRow {
  float o[DH];
  float m, l;
  int first, more;
};
// What the join needs of the group whose first part workgroup w left.
struct PartInfo {
  int rows;        // 0: none
  int token, row0; // the sequence's first token, the tile's first row
  int head, more;
  int pad[3];
};

// The workspace's regions.  Plain: info[W], first parts [W][rows of a tile],
// later parts the same.  Stacked prefix, for the own keys and for the prefix:
// first parts [T][H], later parts [W][rows of a tile].
template <int DH>
struct Parts {
  PartInfo *info;
  PartRow<DH> *first, *later;
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes of the cache; ONCE: past the caches.
template <bool ONCE>
__device__ __forceinline__ Frag16 load_cache(const uint16_t *p) {
  if constexpr (!ONCE) return load16(p);
  Frag16 f;
  f.u = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
  return f;
}

// A later new token's values may be anything to the rows that do not see them, but in a
// tile's product they meet a weight of 0, and 0 Inf is NaN.  So in a block that some
// rows of a tile see more of than others, an Inf or NaN is taken out of the product
// and added to the rows that do see it, key by key; such values are not expected,
// and finite ones cost that block the look (four prompts of 800 to 2000 tokens: 147 ->
// 154 us before the shares had pauses).
// Bits 15 and 31: which of a pair is not finite.  (In whole numbers throughout: as
// conditions, a block's would take hundreds of scalar registers.)
__device__ __forceinline__ uint32_t not_finite(uint32_t pair) {
  return ((pair & 0x7fff7fffu) + 0x00800080u) & 0x80008000u;
}
// The larger magnitudes of two pairs, as bits.
__device__ __forceinline__ uint32_t max_magnitudes(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                               __builtin_bit_cast(u16x2, b & 0x7fff7fffu)));
}
__device__ __forceinline__ uint32_t finite_only(uint32_t pair) {
  const uint32_t out = not_finite(pair);
  return pair & ~((out << 1) - (out >> 15));
}
// An entry that is not finite, else 0.
__device__ __forceinline__ float not_finite_only(uint16_t v) {
  const uint32_t x = (uint32_t)v << 16;
  return __uint_as_float(x & (uint32_t)((int)not_finite(x) >> 31));
}
// A sequence's own key j in a head's pages; null: the table names no page.
__device__ __forceinline__ const uint16_t *value_of(const ServeBatch &b, const int *table, const uint16_t *head,
                                                    long long page_stride, int dh, int j) {
  const int page = checked_page(table[j >> b.page_log2], b.n_pages);
  return page < 0 ? nullptr : head + page * page_stride + (j & ((1 << b.page_log2) - 1)) * dh;
}

// One 32-key step's loads of a wave.
template <int DH>
struct KeyBlock {
  Frag16 k[2][DH / 32];
  uint32_t v[8][DH / 32];  // [key][dword]: DH / 16 bf16 of the lane's entries
};

template <int DH, bool ONCE>
__device__ __forceinline__ void load_block(KeyBlock<DH> &b, const uint16_t *k0, const uint16_t *k1,
                                           const uint16_t *v0, const uint16_t *v1, int lane) {
  const int r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int d = 0; d < DH / 32; ++d) {
    b.k[0][d] = load_cache<ONCE>(k0 + r * DH + d * 32 + q * 8);
    b.k[1][d] = load_cache<ONCE>(k1 + r * DH + d * 32 + q * 8);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint16_t *p = (e < 4 ? v0 : v1) + (q * 4 + (e & 3)) * DH + r * (DH / 16);
    if constexpr (DH == 128) {
      const Frag16 f = load_cache<ONCE>(p);
      for (int i = 0; i < 4; ++i) b.v[e][i] = f.u[i];
    } else {
      const uint2 f = *reinterpret_cast<const uint2 *>(p);
      b.v[e][0] = f.x;
      b.v[e][1] = f.y;
    }
  }
}

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ long long uniform(long long v) {
  return (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                     (unsigned)__builtin_amdgcn_readfirstlane((int)v));
}

// Inclusive sum over the lanes of a wave: within rows of 16 lanes, shifted by 1, 2, 4 and 8,
// then a row's last lane to the row after it, and the second row's to the last two.
template <int CTRL, int ROWS_TO>
__device__ __forceinline__ int from_lane(int v) {  // 0 where there is none
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS_TO, 0xf, false);
}
template <int CTRL, int ROWS_TO>
__device__ __forceinline__ long long from_lane(long long v) {
  return (long long)((unsigned long long)(unsigned)from_lane<CTRL, ROWS_TO>((int)(v >> 32)) << 32 |
                     (unsigned)from_lane<CTRL, ROWS_TO>((int)v));
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
  v += from_lane<0x111, 0xf>(v);
  v += from_lane<0x112, 0xf>(v);
  v += from_lane<0x114, 0xf>(v);
  v += from_lane<0x118, 0xf>(v);
  v += from_lane<0x142, 0xa>(v);
  v += from_lane<0x143, 0xc>(v);
  return v;
}

__device__ __forceinline__ long long lane_value(long long v, int lane) {
  return (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
                     (unsigned)__builtin_amdgcn_readlane((int)v, lane));
}

// serve_batch.hpp's wave.
struct Wave64 {
  using Ints = int;
  int lane;
  template <class F>
  __device__ __forceinline__ int each(F f) const {
    return f(lane);
  }
  template <class F>
  __device__ __forceinline__ long long sum(F f) const {
    return lane_value(wave_scan((long long)f(lane)), 63);
  }
  __device__ __forceinline__ int scan(int v) const { return wave_scan(v); }
  __device__ __forceinline__ int at(int v, int l) const { return __builtin_amdgcn_readlane(v, l); }
  __device__ __forceinline__ int above(int v, int x) const { return __builtin_ctzll(__ballot(v > x)); }
  __device__ __forceinline__ int same(int v) const { return __builtin_amdgcn_readfirstlane(v); }
  __device__ __forceinline__ long long same(long long v) const { return uniform(v); }
};

// A workgroup's number w in the division, its share of the units, [u0, u1) of U,
// and the group its first lies in; false: none (the launch has more workgroups
// than units, or the share is in a pause).  Every workgroup finds its own: the
// units of each sequence, a scan over the lanes, and in the sequence that holds u0 a
// scan over its tiles.
struct Share {
  long long sum[NT], wave[NT / 64];
  SeqUnits seq;  // the one that holds u0
};
__device__ __forceinline__ bool take_share(const AttnSplit &sp, Share &s, long long &U, int &W, long long &u0,
                                           long long &u1, UnitCursor &c, int &w, bool by_xcd) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int seqs = split_seqs(sp), per = seqs_per_lane(sp, NT);
  const Wave64 lanes{lane};
  long long mine = 0;
  if (sum_by_waves(sp, NT)) {
    for (int q = wave; q < seqs; q += NT / 64) {
      const long long units = head_units_by(lanes, sp, split_kv(sp, q), split_span(sp, q).n) * sp.Hkv;
      if (lane == 63) s.sum[q] = units;
    }
    __syncthreads();
    if (tid < seqs) mine = s.sum[tid];
  } else {
    mine = lane_units(sp, tid, per);
  }
  const long long in_wave = wave_scan(mine);
  if (lane == 63) s.wave[wave] = in_wave;
  __syncthreads();
  long long before = in_wave - mine;
  U = 0;
  for (int v = 0; v < NT / 64; ++v) {
    if (v < wave) before += s.wave[v];
    U += s.wave[v];
  }
  U = uniform(U);
  ShareRange r;
  const bool some = share_of(sp, U, gridDim.x, blockIdx.x, by_xcd, r);
  W = r.W;
  w = r.w;
  if (!some) return false;
  u0 = r.u0;
  u1 = r.u1;
  // one lane's sequences hold u0
  if (u0 >= before && u0 < before + mine) s.seq = seq_in_lane(sp, tid, per, before, mine, u0);
  __syncthreads();
  SeqUnits seq = s.seq;
  seq.seq = __builtin_amdgcn_readfirstlane(seq.seq);
  c = seek_in_seq(lanes, sp, seq, u0);
  skip_pause(c, u0);
  return u0 < u1;
}

// Rows of no sequence give zeros.
template <int DH>
__device__ __forceinline__ void zero_spare_rows(const PagedAttentionArgs &a, const AttnSplit &sp) {
  if (sp.stacked || !sp.b.q_start) return;
  const int lo = clamp_int(sp.b.q_start[0], 0, sp.b.T), hi = clamp_int(sp.b.q_start[sp.b.B], lo, sp.b.T);
  const int spare = lo + (sp.b.T - hi), cols = sp.Hkv * sp.G * DH / 8;
  for (long long i = (long long)blockIdx.x * NT + threadIdx.x; i < (long long)spare * cols; i += (long long)gridDim.x * NT) {
    const int t = (int)(i / cols), c = (int)(i - (long long)t * cols);
    *reinterpret_cast<u32x4 *>(a.out + (long long)(t < lo ? t : hi + t - lo) * a.o_stride + c * 8) = u32x4{0, 0, 0, 0};
  }
}

// The rows of one tile over the key blocks [b0, b1) of their group, 32 keys of
// each block a wave: this wave's sums o, maximum m (base 2) and l.  b1 < 0: to the
// group's last block; then the first block's loads do not wait for kv_len (a block
// past the end is read from what pages the table names there, and masked).
// ONCE: keys and values are loaded past the caches (48 sequences of up to 8000 keys
// 147 -> 137 us, one of 131 000 96 -> 91; not for the short ones below, 16.8 -> 21).
// MANY: a tile's rows may be of several tokens.
template <int DH, int NW, bool ONCE, bool MANY>
struct TileWalk {
  static constexpr int E = DH / 16;  // MFMAs of the second product, entries of a lane's output run
  f32x4 o[E];
  float m, l;

  __device__ __forceinline__ void run(const PagedAttentionArgs &a, const AttnSplit &sp, const UnitCursor &c, int b0,
                                      int b1) {
    constexpr int BLOCK = 32 * NW;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const float scale = a.scale * 1.44269504088896340736f;  // exponentials in base 2
    const int row0 = c.tile * ROWS, rows = min(ROWS, c.n * sp.G - row0);
    const int row = row0 + min(r, rows - 1), tok = row / sp.G;  // this lane's query
    Frag16 qf[DH / 32];
    {
      const uint16_t *p = a.Q + (long long)(c.start + tok) * a.q_stride + (c.head * sp.G + row - tok * sp.G) * DH + q * 8;
#pragma unroll
      for (int d = 0; d < DH / 32; ++d) qf[d] = load16(p + d * 32);
    }
    int lim = 0, first_lim = 0, tile_lim = 0;
    auto limits = [&]() __attribute__((always_inline)) {
      lim = visible_keys(sp, c.kv, c.n, tok);
      first_lim = visible_keys(sp, c.kv, c.n, row0 / sp.G);
      tile_lim = visible_keys(sp, c.kv, c.n, (row0 + rows - 1) / sp.G);
    };
    const int *table = sp.b.page_table + (sp.stacked ? 0 : c.seq * sp.b.table_stride);
    const uint16_t *kh = a.k_pages + ((long long)c.head << sp.b.page_log2) * DH;
    const uint16_t *vh = a.v_pages + ((long long)c.head << sp.b.page_log2) * DH;

#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -__builtin_inff();
    l = 0.f;

    // A block's first key of this wave, the keys that this lane's row sees and any
    // row of the tile, whether each half has a page.
    struct Where {
      int j;
      bool pre, live[2];
    };
    KeyBlock<DH> kb;
    int page[2];  // of the block to be fetched next, read a block ahead of its keys
    auto find = [&](int blk, int end) __attribute__((always_inline)) {  // end: own keys
      const bool pre = blk < sp.pre_blocks;
      const int *t = pre ? a.prefix_table : table;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = (pre ? blk : blk - sp.pre_blocks) * BLOCK + wave * 32 + 16 * h;
        page[h] = -1;
        if (j < (pre ? sp.b.prefix_len : end)) page[h] = t[j >> sp.b.page_log2];
      }
    };
    auto fetch = [&](int blk) __attribute__((always_inline)) {
      Where x;
      x.pre = blk < sp.pre_blocks;
      x.j = (x.pre ? blk : blk - sp.pre_blocks) * BLOCK + wave * 32;
      const uint16_t *kp[2], *vp[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int pg = __builtin_amdgcn_readfirstlane(checked_page(page[h], sp.b.n_pages));
        x.live[h] = pg >= 0;
        const int in = ((x.j + 16 * h) & ((1 << sp.b.page_log2) - 1)) * DH;
        kp[h] = kh + max(pg, 0) * a.kpage_stride + in;
        vp[h] = vh + max(pg, 0) * a.vpage_stride + in;
      }
      load_block<DH, ONCE>(kb, kp[0], kp[1], vp[0], vp[1], lane);
      return x;
    };
    Where at;
    if (b1 < 0) {
      find(b0, sp.b.max_pages << sp.b.page_log2);
      at = fetch(b0);
      limits();
      b1 = tile_blocks(sp, c.kv, c.n, c.tile);
    } else {
      limits();
      find(b0, tile_lim);
      at = fetch(b0);
    }
    if (b0 + 1 < b1) find(b0 + 1, tile_lim);
    for (int blk = b0; blk < b1; ++blk) {
      KeyBlock<DH> cur = kb;
      const Where x = at;
      if (blk + 1 < b1) at = fetch(blk + 1);
      if (blk + 2 < b1) find(blk + 2, tile_lim);
      const int row_end = x.pre ? sp.b.prefix_len : lim, end = x.pre ? sp.b.prefix_len : tile_lim;
      if (x.j >= end || (!x.live[0] && !x.live[1])) continue;
      // logits in base 2, keys x.j + 16 h + 4 q + i of row r
      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DH / 32; ++d) MfmaBF16::mma(s[h], cur.k[h][d], qf[d]);
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = s[h][i] * scale;
          s[h][i] = x.live[h] && x.j + 16 * h + 4 * q + i < row_end ? v : -__builtin_inff();
          top = fmaxf(top, s[h][i]);
        }
      LanePair t16 = lane_pair16(top);
      top = fmaxf(t16.lo, t16.hi);
      LanePair t32 = lane_pair32(top);
      top = fmaxf(t32.lo, t32.hi);
      const float mn = fmaxf(m, top), base = mn == -__builtin_inff() ? 0.f : mn;
      const float alpha = exp2_(m - base);
      m = mn;
      float p[8], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = exp2_(s[i >> 2][i & 3] - base);
        sum += p[i];
      }
      l = l * alpha + sum;
      Frag16 pf;
#pragma unroll
      for (int i = 0; i < 4; ++i) pf.u[i] = cvt_pk_bf16(p[2 * i], p[2 * i + 1]);
      // values that no row may see: whatever lies there must not meet p = 0
      if (x.j + 32 > end || !x.live[0] || !x.live[1]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool keep = x.live[e >> 2] && x.j + 16 * (e >> 2) + 4 * q + (e & 3) < end;
#pragma unroll
          for (int i = 0; i < DH / 32; ++i) cur.v[e][i] = keep ? cur.v[e][i] : 0u;
        }
      }
      bool left_out = false;
      if (MANY && !x.pre && x.j + 32 > first_lim && first_lim < end) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int i = 0; i < DH / 32; ++i) top = max_magnitudes(top, cur.v[e][i]);
        left_out = __any(not_finite(top) != 0);
        if (left_out) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < DH / 32; ++i) cur.v[e][i] = finite_only(cur.v[e][i]);
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        Frag16 vf;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          vf.u[i] = __builtin_amdgcn_perm(cur.v[2 * i + 1][e >> 1], cur.v[2 * i][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[e][i] *= alpha;
        MfmaBF16::mma(o[e], vf, pf);
      }
      if (MANY && left_out) {
#pragma unroll 1
        for (int k = 0; k < 32 && x.j + k < end; ++k) {
          const uint16_t *v = value_of(sp.b, table, vh, a.vpage_stride, DH, x.j + k);
          if (!v || x.j + k >= row_end) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) {
              if (e % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // (few loads' registers at a time)
              o[e][i] += not_finite_only(v[(q * 4 + i) * E + e]);
            }
        }
      }
    }
    l = sum_of_rows(l);
  }

  // over the wave's four 16-lane rows
  static __device__ __forceinline__ float sum_of_rows(float v) {
    const LanePair a = lane_pair16(v);
    const LanePair b = lane_pair32(a.lo + a.hi);
    return b.lo + b.hi;
  }
};

// The waves' sums in LDS, one slot each, and their join.
template <int DH, int SLOTS>
struct WaveSums {
  float m[SLOTS][ROWS], l[SLOTS][ROWS];
  __attribute__((aligned(16))) float o[SLOTS][ROWS][DH + 4];

  template <class Walk>
  __device__ __forceinline__ void put(int slot, const Walk &t) {
    constexpr int E = DH / 16;
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    if (q == 0) {
      m[slot][r] = t.m;
      l[slot][r] = t.l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<f32x4 *>(&o[slot][r][(q * 4 + i) * E + e]) =
            f32x4{t.o[e][i], t.o[e + 1][i], t.o[e + 2][i], t.o[e + 3][i]};
  }
  // entries 8 jc .. of row jr over the first n slots
  __device__ __forceinline__ void join(int n, int jr, int jc, float &mm, float &ll, float (&acc)[8]) const {
    mm = -__builtin_inff();
    ll = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int v = 0; v < n; ++v) mm = fmaxf(mm, m[v][jr]);
    const float base = mm == -__builtin_inff() ? 0.f : mm;
    for (int v = 0; v < n; ++v) {
      const float f = exp2_(m[v][jr] - base);
      ll += f * l[v][jr];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += f * o[v][jr][jc * 8 + e];
    }
  }
};

// o / l as a row's eight entries; no key: 0.
__device__ __forceinline__ void store_row8(uint16_t *to, const float (&acc)[8], float l) {
  const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = cvt_pk_bf16(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  *reinterpret_cast<u32x4 *>(to) = v;
}

template <int DH>
__global__ __launch_bounds__(NT, 2) void paged_attention_kernel(PagedAttentionArgs a, AttnSplit sp, int dense,
                                                                Parts<DH> parts) {
  sp.pause = 0;  // (as it is: the compiler knows it now)
  __shared__ Share share;
  __shared__ WaveSums<DH, 4> sums;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  zero_spare_rows<DH>(a, sp);
  long long U, u0, u1;
  UnitCursor c;
  int W, w;
  const bool some = take_share(sp, share, U, W, u0, u1, c, w, false);
  if (!dense && tid == 0) parts.info[w].rows = 0;
  if (!some) return;

  for (long long u = u0; u < u1;) {
    const int b0 = c.blk, b1 = c.nb - b0 < u1 - u ? c.nb : b0 + (int)(u1 - u);
    const int row0 = c.tile * ROWS, rows = min(ROWS, c.n * sp.G - row0);
    TileWalk<DH, 4, true, true> t;
    t.run(a, sp, c, b0, b1);
    sums.put(wave, t);
    __syncthreads();
    const bool starts = b0 == 0, ends = b1 == c.nb;
    const int more = starts && !ends ? unit_owner(U, W, c.base + sp.pause + c.nb - 1) - w : 0;
    if (!dense && starts && !ends && tid == 0) parts.info[w] = PartInfo{rows, c.start, row0, c.head, more, {0, 0, 0}};
    for (int i = tid; i < rows * (DH / 8); i += NT) {
      const int jr = i / (DH / 8), jc = i % (DH / 8);
      float mm, ll, acc[8];
      sums.join(4, jr, jc, mm, ll, acc);
      const int orow = row0 + jr, ot = orow / sp.G, head = c.head * sp.G + orow - ot * sp.G;
      const long long token = c.start + ot;
      if (!dense && starts && ends) {
        store_row8(a.out + token * a.o_stride + head * DH + jc * 8, acc, ll);
      } else {
        PartRow<DH> *to = !starts ? parts.later + w * ROWS + jr
                          : dense ? parts.first + token * (sp.G * sp.Hkv) + head
                                  : parts.first + w * ROWS + jr;
        *reinterpret_cast<f32x4 *>(to->o + jc * 8) = f32x4{acc[0], acc[1], acc[2], acc[3]};
        *reinterpret_cast<f32x4 *>(to->o + jc * 8 + 4) = f32x4{acc[4], acc[5], acc[6], acc[7]};
        if (jc == 0) {
          to->m = mm;
          to->l = ll;
          to->first = w;
          to->more = more | (jr << 16);
        }
      }
    }
    u += b1 - b0;
    if (u < u1) next_group(sp, c);
    __syncthreads();
  }
}

// Short histories, one token a sequence: a workgroup takes a whole group, so that
// nothing is left to join, but for the parts of a shared prefix (pre, `pre_rows` to
// a slot), which it takes in itself.
template <int DH, int NW>
__global__ __launch_bounds__(64 * NW, 2) void paged_attention_whole_kernel(PagedAttentionArgs a, AttnSplit sp, int tiles,
                                                                           int W, Parts<DH> pre, int pre_rows) {
  constexpr int N = 64 * NW;
  __shared__ WaveSums<DH, 2 * NW> sums;  // the waves' sums; theirs of the prefix's parts
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = blockIdx.x / tiles;
  UnitCursor c{group / sp.Hkv, (int)blockIdx.x % tiles, group % sp.Hkv, 0, 0, 1, group / sp.Hkv, 0, 0};
  c.kv = split_kv(sp, c.seq);
  const int row0 = c.tile * ROWS, rows = min(ROWS, sp.G - row0);
  TileWalk<DH, NW, false, false> t;
  t.run(a, sp, c, 0, -1);
  sums.put(wave, t);
  if (pre.first) {  // every NW-th part of each row a wave
    for (int i = lane; i < rows * (DH / 8); i += 64) {
      const int jr = i / (DH / 8), jc = i % (DH / 8), head = c.head * sp.G + row0 + jr;
      const PartRow<DH> *f = pre.first + (long long)c.start * (sp.G * sp.Hkv) + head;
      const int first = clamp_int(f->first, 0, W - 1), more = min(f->more & 0xffff, W - 1 - first);
      const int pr = (f->more >> 16) & (pre_rows - 1);
      float mm = -__builtin_inff(), ll = 0.f;
      f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll 4
      for (int n = wave; n <= more; n += NW) {
        const PartRow<DH> *p = n == 0 ? f : pre.later + (long long)(first + n) * pre_rows + pr;
        const float pm = p->m, pl = p->l, mn = fmaxf(mm, pm), base = mn == -__builtin_inff() ? 0.f : mn;
        const float g = exp2_(mm - base), k = exp2_(pm - base);
        const f32x4 px = *reinterpret_cast<const f32x4 *>(p->o + jc * 8), py = *reinterpret_cast<const f32x4 *>(p->o + jc * 8 + 4);
        mm = mn;
        ll = ll * g + pl * k;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = x[e] * g + px[e] * k, y[e] = y[e] * g + py[e] * k;
      }
      if (jc == 0) {
        sums.m[NW + wave][jr] = mm;
        sums.l[NW + wave][jr] = ll;
      }
      *reinterpret_cast<f32x4 *>(&sums.o[NW + wave][jr][jc * 8]) = x;
      *reinterpret_cast<f32x4 *>(&sums.o[NW + wave][jr][jc * 8 + 4]) = y;
    }
  }
  __syncthreads();
  for (int i = tid; i < rows * (DH / 8); i += N) {
    const int jr = i / (DH / 8), jc = i % (DH / 8), head = c.head * sp.G + row0 + jr;
    float mm, ll, acc[8];
    sums.join(pre.first ? 2 * NW : NW, jr, jc, mm, ll, acc);
    store_row8(a.out + (long long)c.start * a.o_stride + head * DH + jc * 8, acc, ll);
  }
}

// ---- many rows: prompts, and a shared prefix under the rows of a batch --------
// A tile of 128 rows, 32 a wave, over blocks of 64 keys that the four waves share
// through LDS: with enough rows per key the matrix instructions and the
// exponentials bound it, not the cache's bytes.  32x32x16 MFMAs in the same two
// products as above: S^T = K Q^T leaves a lane sixteen keys (8 j + 4 h + i of each
// 32, h its half of the wave) of one row, so the row's maximum is one exchange
// between the halves away, and keys 8 j + 4 h + i, j = 2 g and 2 g + 1, are the
// k slots of its half in the g-th MFMA of O^T = V^T P^T.
//  - Two buffers: the next block is fetched, sixteen keys a wave, while one is
//    computed, and then written to the other; one barrier a block.
//  - K lies in LDS by keys, 16-byte chunks exchanged by the key's number so that
//    the 32 keys of an operand read fall into different banks; V by keys with its
//    64-byte runs exchanged, for gfx950's transposing reads: sixteen lanes read four
//    keys of sixteen entries, each gets four keys of its entry.
//  - Blocks follow each other across groups: a group's last block is computed with
//    the next one's first on its way.
// Four prompts of 800 to 2000 tokens, 79 GFLOP: 146 us, of which 12 join parts; a block of
// 64 keys is as long as its products (0.9 us a CU at the rate of a large one) and its
// exponentials together.  The prefix of 6001 keys under 64 sequences: 24 us.
//  - The running maximum is only a reference: it is raised, and the sums scaled,
//    when a row's maximum passes it by more than 2^8 (a uniform branch), so that
//    p <= 2^8 and most blocks scale nothing.
constexpr int TROWS = 128, TKEYS = 64;  // sixteen keys a wave fetches
// A group's first loads, its last products and its stores take the time of blocks, and a
// border that falls between groups leaves no parts.  Pauses of 0, 1, 2, 3 and 5 blocks: the
// prompts above 155, 148, 144, 141 and 143 us, 64 tokens of one sequence of 2000 keys 28 and,
// with 3, 24; but 800 tokens with nothing before them, 8 heads of 64, 19 and 26.
constexpr int TILE_PAUSE = 3;

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ uint2 read_tr(const uint16_t *p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
}

template <int DH>
__global__ __launch_bounds__(NT, 2) void paged_attention_tile_kernel(PagedAttentionArgs a, AttnSplit sp, int dense,
                                                                     Parts<DH> parts) {
  sp.pause = TILE_PAUSE;  // (as it is: the compiler knows it now)
  constexpr int CH = DH / 8;             // 16-byte chunks of a key
  constexpr int NL = TKEYS * CH / NT;    // loads of a wave a block, of K and of V
  constexpr int KPL = 64 / CH;           // keys that one of them covers
  constexpr int E = DH / 32;             // MFMAs of the second product a k step
  __shared__ __attribute__((aligned(16))) uint16_t sk[2][TKEYS * DH], sv[2][TKEYS * DH];
  __shared__ __attribute__((aligned(16))) int s_live[2][TKEYS / 16];  // whether a buffer's sixteen keys have a page
  __shared__ int s_left;                 // whether values have been left out of sums (and stays)
  __shared__ Share share;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, h = lane >> 5;
  if (tid == 0) s_left = 0;
  zero_spare_rows<DH>(a, sp);
  long long U, u0, u1;
  UnitCursor c;
  int W, w;
  const bool some = take_share(sp, share, U, W, u0, u1, c, w, true);
  if (!dense && tid == 0) parts.info[w].rows = 0;
  if (!some) return;

  const float scale = a.scale * 1.44269504088896340736f;
  // the chunk exchanges: of key k's chunk ch
  auto k_swap = [](int k) { return CH == 16 ? k & 15 : (k >> 1) & 7; };
  auto v_swap = [](int k) { return CH == 16 ? (k & 3) << 2 : (k & 2) << 1; };
  // This lane's addresses in a buffer, of chunk h of key r, its first run of V, and
  // where it writes its first chunks of its wave's sixteen keys; the others differ by
  // an exclusive or of the chunk and by whole keys.
  const int ka = r * DH + (h ^ k_swap(r)) * 8;
  const int vk = 4 * h + (lane >> 2 & 3);
  const int va = vk * DH + (((r >> 4) * 2 + (lane >> 1 & 1)) ^ v_swap(vk)) * 8 + (lane & 1) * 4;
  const int wk = 16 * wave + lane / CH;
  const int ks = wk * DH + (lane % CH ^ k_swap(wk)) * 8, vs = wk * DH + (lane % CH ^ v_swap(wk)) * 8;
  const int wrow = wave * 32;  // this wave's first row in a tile

  // The group whose blocks are computed: its rows, and the own keys that this
  // lane's row, the wave's first and last rows and any row of the tile see.
  struct Group {
    int row0, rows, row, tok;
    int lim, lim_first, lim_last, end;
  };
  auto tile_end = [&](const UnitCursor &u) __attribute__((always_inline)) {
    const unsigned last = min((u.tile + 1) * TROWS, u.n * sp.G) - 1;
    return visible_keys(sp, u.kv, u.n, last / (unsigned)sp.G);
  };
  // Of the keys that a tile's last row sees, as many at the end its first may not.
  const int span = (unsigned)(TROWS - 1) / (unsigned)sp.G + 1;
  auto group_of = [&](const UnitCursor &u) __attribute__((always_inline)) {
    Group g;
    g.row0 = u.tile * TROWS;
    g.rows = min(TROWS, u.n * sp.G - g.row0);
    g.row = g.row0 + min(wrow + r, g.rows - 1);
    g.tok = (unsigned)g.row / (unsigned)sp.G;
    const int first = (unsigned)(g.row0 + min(wrow, g.rows - 1)) / (unsigned)sp.G;
    const int last = (unsigned)(g.row0 + min(wrow + 31, g.rows - 1)) / (unsigned)sp.G;
    g.lim = visible_keys(sp, u.kv, u.n, g.tok);
    g.lim_first = visible_keys(sp, u.kv, u.n, first);
    g.lim_last = visible_keys(sp, u.kv, u.n, last);
    g.end = tile_end(u);
    return g;
  };
  Frag16 qf[DH / 16];
  auto load_queries = [&](const UnitCursor &u) __attribute__((always_inline)) {
    const int row = min(u.tile * TROWS + wrow + r, u.n * sp.G - 1), tok = (unsigned)row / (unsigned)sp.G;
    const uint16_t *p = a.Q + (long long)(u.start + tok) * a.q_stride + (u.head * sp.G + row - tok * sp.G) * DH + h * 8;
#pragma unroll
    for (int d = 0; d < DH / 16; ++d) qf[d] = load16(p + d * 16);
  };
  // Waits for the queries where they are loaded: at their use the next block's loads,
  // issued after them, would be waited for too.
  auto touch_queries = [&]() __attribute__((always_inline)) {
    uint32_t zero;
    asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
#pragma unroll
    for (int d = 0; d < DH / 16; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[d].u[i] |= zero;
  };
  // The pages of this wave's sixteen keys of 64 blocks from blk on, one a lane (-1: none
  // of the keys is seen, or the table names no page).  One load for many blocks: a load
  // a block, carried to the next, is waited for behind the block's keys.
  auto find = [&](const UnitCursor &u, int end, int blk) __attribute__((always_inline)) {
    const int b = blk + lane;
    const bool pre = b < sp.pre_blocks;
    const long long j = (long long)(pre ? b : b - sp.pre_blocks) * TKEYS + 16 * wave;
    if (j >= (pre ? sp.b.prefix_len : end)) return -1;
    const int *t = pre ? a.prefix_table : sp.b.page_table + u.seq * (sp.stacked ? 0 : sp.b.table_stride);
    return checked_page(t[j >> sp.b.page_log2], sp.b.n_pages);
  };
  u32x4 kr[NL], vr[NL];  // the next block's sixteen keys of this wave
  int seen = 0;          // of these, the ones that a row may see; + SOME: that some may not
  constexpr int SOME = 32;
  auto fetch = [&](const UnitCursor &u, int end, int blk, int page) __attribute__((always_inline)) {
    const bool pre = blk < sp.pre_blocks;
    const int j = (pre ? blk : blk - sp.pre_blocks) * TKEYS + 16 * wave;
    seen = page >= 0 ? clamp_int((pre ? sp.b.prefix_len : end) - j, 0, 16) : 0;
    if (!pre && j + 16 > end - span) seen += SOME;
    const int in = ((u.head << sp.b.page_log2) + (j & ((1 << sp.b.page_log2) - 1))) * DH;
    const uint16_t *kp = a.k_pages + max(page, 0) * a.kpage_stride + in, *vp = a.v_pages + max(page, 0) * a.vpage_stride + in;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      kr[i] = *reinterpret_cast<const u32x4 *>(kp + i * 512 + lane * 8);
      vr[i] = *reinterpret_cast<const u32x4 *>(vp + i * 512 + lane * 8);
    }
  };
  auto commit = [&](int to) __attribute__((always_inline)) {
    if (lane == 0) s_live[to][wave] = (seen & (SOME - 1)) != 0;
    if (seen != 16) {  // values that no row may see must not meet p = 0, others that some may not
      __builtin_amdgcn_sched_barrier(0);  // (keeps the branch)
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        vr[i] = masked(vr[i], i * KPL + lane / CH < (seen & (SOME - 1)));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t out = seen & SOME ? not_finite(vr[i][e]) : 0u;
          any |= out;
          vr[i][e] &= ~((out << 1) - (out >> 15));
        }
      }
      if (any != 0) s_left = 1;
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      *reinterpret_cast<u32x4 *>(sk[to] + (ks ^ i * 32) + i * KPL * DH) = kr[i];
      *reinterpret_cast<u32x4 *>(sv[to] + vs + i * KPL * DH) = vr[i];
    }
  };

  Group g = group_of(c);
  f32x16 o[E];
  float m, l;  // l: this lane's keys only
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[e][i] = 0.f;
    m = -__builtin_inff();
    l = 0.f;
  };
  clear();
  long long left = u1 - u0;  // blocks, the one computed included
  load_queries(c);
  int b0 = c.blk, pages0 = c.blk, pages = find(c, g.end, pages0);
  fetch(c, g.end, c.blk, __builtin_amdgcn_readlane(pages, 0));
  commit(0);
  touch_queries();
  __syncthreads();

  for (int buf = 0;; buf ^= 1) {
    const uint16_t *const kb = sk[buf], *const vb = sv[buf];
    const int blk = c.blk;
    const bool same = blk + 1 < c.nb, more_blocks = left > (same ? 1 : 1 + sp.pause);
    // the next block's loads: of the next group the pages are to be found first
    UnitCursor c2 = c;
    int end2 = 0;
    if (more_blocks) {
      if (same) {
        if (blk + 1 >= pages0 + 64) {
          pages0 = blk + 1;
          pages = find(c, g.end, pages0);
        }
        fetch(c, g.end, blk + 1, __builtin_amdgcn_readlane(pages, blk + 1 - pages0));
      } else {
        next_group(sp, c2);
        end2 = tile_end(c2);
        pages0 = 0;
        pages = find(c2, end2, 0);
      }
    }
    const bool pre = blk < sp.pre_blocks;
    const int j0 = (pre ? blk : blk - sp.pre_blocks) * TKEYS;
    const int my_lim = pre ? sp.b.prefix_len : g.lim;
    const int first_lim = pre ? sp.b.prefix_len : g.lim_first, last_lim = pre ? sp.b.prefix_len : g.lim_last;
    const bool busy = wrow < g.rows && j0 < last_lim;
    f32x16 s[2];
    if (busy) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = 0.f;
      // operands a few MFMAs ahead of their use: a read's latency is four of them
      constexpr int N = 2 * (DH / 16), AHEAD = 6;
      Frag16 kf[N];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) kf[i] = load16(kb + (ka ^ (i >> 1) * 16) + 32 * (i & 1) * DH);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + AHEAD < N) kf[i + AHEAD] = load16(kb + (ka ^ ((i + AHEAD) >> 1) * 16) + 32 * (i & 1) * DH);
        __builtin_amdgcn_sched_barrier(0);
        s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i].h, qf[i >> 1].h, s[i & 1], 0, 0, 0);
      }
    }
    if (more_blocks && !same) {
      fetch(c2, end2, 0, __builtin_amdgcn_readlane(pages, 0));
    }
    if (busy) {
      const int4 lv = *reinterpret_cast<const int4 *>(s_live[buf]);
      const bool all_live = __builtin_amdgcn_readfirstlane(lv.x & lv.y & lv.z & lv.w);
      if (j0 + TKEYS > first_lim || !all_live) {
        __builtin_amdgcn_sched_barrier(0);  // (keeps the branch: 100 instructions that few blocks need)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int k = 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
            const int has = t == 0 ? (i < 8 ? lv.x : lv.y) : (i < 8 ? lv.z : lv.w);
            if (j0 + k >= my_lim || !has) s[t][i] = -__builtin_inff();
          }
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
      const LanePair tp = lane_pair32(top);
      top = fmaxf(tp.lo, tp.hi) * scale;
      if (__any(top > m + 8.0f)) {
        const float mn = fmaxf(m, top);
        const float alpha = mn == -__builtin_inff() ? 1.f : exp2_(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[e][i] *= alpha;
      }
      const float base = m == -__builtin_inff() ? 0.f : m;
      Frag16 pf[4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float p[16], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          p[i] = exp2_(fmaf(s[t][i], scale, -base));
          sum[i & 3] += p[i];
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pf[2 * t].u[i] = cvt_pk_bf16(p[2 * i], p[2 * i + 1]);
          pf[2 * t + 1].u[i] = cvt_pk_bf16(p[8 + 2 * i], p[8 + 2 * i + 1]);
        }
      }
      // MFMA i: sixteen keys k = i / E, entries 32 e + r; four keys of sixteen
      // entries a 16-lane group and read
      constexpr int N = 4 * E, AHEAD = 3;
      Frag16 vf[N];
      auto operand = [&](int i) __attribute__((always_inline)) {
        const uint16_t *from = vb + (va ^ (i % E) * 32) + 16 * (i / E) * DH;
        const uint2 lo = read_tr(from), hi = read_tr(from + 8 * DH);
        vf[i].u = u32x4{lo.x, lo.y, hi.x, hi.y};
      };
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) operand(i);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + AHEAD < N) operand(i + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
        o[i % E] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i].h, pf[i / E].h, o[i % E], 0, 0, 0);
      }
    }
    if (!same || !more_blocks) {  // the end of the group, or of the share
      load_queries(c2);  // (the old ones again after the last block)
      const LanePair lp = lane_pair32(l);
      l = lp.lo + lp.hi;
      const bool starts = b0 == 0, ends = !same;
      const int more = starts && !ends ? unit_owner(U, W, c.base + sp.pause + c.nb - 1) - w : 0;
      if (!dense && starts && !ends && tid == 0)
        parts.info[w] = PartInfo{g.rows, c.start, g.row0, c.head, more, {0, 0, 0}};
      const int jr = wrow + r;
      if (jr < g.rows) {
        const int head = c.head * sp.G + g.row - g.tok * sp.G;
        const long long token = c.start + g.tok;
        // this lane's entries: 32 e + 8 j + 4 h + i
        if (!dense && starts && ends) {
          const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
          uint16_t *to = a.out + token * a.o_stride + head * DH + 4 * h;
#pragma unroll
          for (int e = 0; e < E; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<uint2 *>(to + 32 * e + 8 * j) =
                  make_uint2(cvt_pk_bf16(o[e][4 * j] * inv, o[e][4 * j + 1] * inv),
                             cvt_pk_bf16(o[e][4 * j + 2] * inv, o[e][4 * j + 3] * inv));
        } else {
          PartRow<DH> *to = !starts ? parts.later + (long long)w * TROWS + jr
                            : dense ? parts.first + token * (sp.G * sp.Hkv) + head
                                    : parts.first + (long long)w * TROWS + jr;
#pragma unroll
          for (int e = 0; e < E; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<f32x4 *>(to->o + 32 * e + 8 * j + 4 * h) =
                  f32x4{o[e][4 * j], o[e][4 * j + 1], o[e][4 * j + 2], o[e][4 * j + 3]};
          if (h == 0) {
            to->m = m;
            to->l = l;
            to->first = w;
            to->more = more | (jr << 16);
          }
        }
      }
      touch_queries();
      if (!more_blocks) break;
      clear();
      c = c2;
      g = group_of(c);
      b0 = 0;
      left -= sp.pause;
    } else {
      ++c.blk;
    }
    --left;
    commit(buf ^ 1);
    __syncthreads();
  }

  __syncthreads();
  if (!__builtin_amdgcn_readfirstlane(s_left)) return;
  // What was left out of the sums, to where they are now: after the loop, which has no
  // register to spare.
  take_share(sp, share, U, W, u0, u1, c, w, true);
  for (long long u = u0; u < u1;) {
    const int first = c.blk, last = c.nb - first < u1 - u ? c.nb : first + (int)(u1 - u);  // blocks of this group
    const Group g = group_of(c);
    const bool starts = first == 0, ends = last == c.nb;
    if (const int jr = wrow + r; jr < g.rows) {
      const int head = c.head * sp.G + g.row - g.tok * sp.G;
      const long long token = c.start + g.tok;
      uint16_t *to = a.out + token * a.o_stride + head * DH + 4 * h;
      PartRow<DH> *part = !starts ? parts.later + (long long)w * TROWS + jr
                          : dense ? parts.first + token * (sp.G * sp.Hkv) + head
                                  : parts.first + (long long)w * TROWS + jr;
      const int *table = sp.b.page_table + c.seq * (sp.stacked ? 0 : sp.b.table_stride);
      const uint16_t *vh = a.v_pages + ((long long)c.head << sp.b.page_log2) * DH + 4 * h;
      // (sixteen keys together were looked at)
      const int from = max(max(first - sp.pre_blocks, 0) * TKEYS, (g.end - span) & ~15);
      const int end = min((last - sp.pre_blocks) * TKEYS, g.lim);
      for (int i = 0; i < DH; i += 8) {
        f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k = from; k < end; ++k)
          if (const uint16_t *v = value_of(sp.b, table, vh, a.vpage_stride, DH, k))
            for (int e = 0; e < 4; ++e) x[e] += not_finite_only(v[i + e]);
        for (int e = 0; e < 4; ++e) {
          if (!dense && starts && ends)
            to[i + e] = f32_to_bf16(bf16_to_f32(to[i + e]) + x[e]);
          else
            part->o[i + 4 * h + e] += x[e];
        }
      }
    }
    u += last - first + sp.pause;
    if (u < u1) next_group(sp, c);
  }
}

// ---- the joins ------------------------------------------------------------------
// A row's parts, SPLIT of them at a time, 4 entries a lane; a workgroup takes
// NT / (DH / 4) / SPLIT rows.  The order of the sums is the parts', whatever ran
// first.
template <int DH, int SPLIT>
struct RowJoin {
  static constexpr int CH = DH / 4, PER = NT / CH / SPLIT;  // PER: rows of a workgroup
  float m, l;
  f32x4 o;
  __device__ __forceinline__ void clear() {
    m = -__builtin_inff();
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void add(float pm, float pl, f32x4 po) {
    const float mn = fmaxf(m, pm), base = mn == -__builtin_inff() ? 0.f : mn;
    const float f = exp2_(m - base), g = exp2_(pm - base);
    m = mn;
    l = l * f + pl * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + po[i] * g;
  }
  __device__ __forceinline__ void add(const PartRow<DH> *p, int ch) {
    add(p->m, p->l, *reinterpret_cast<const f32x4 *>(p->o + ch * 4));
  }
  // over the lanes' splits, to split 0
  __device__ __forceinline__ void gather(f32x4 *so, float *sm, float *sl, int split) {
    if constexpr (SPLIT > 1) {
      const int tid = threadIdx.x, at = tid % (NT / SPLIT);
      so[tid] = o;
      sm[tid] = m;
      sl[tid] = l;
      __syncthreads();
      if (split == 0)
        for (int s = 1; s < SPLIT; ++s) add(sm[s * (NT / SPLIT) + at], sl[s * (NT / SPLIT) + at], so[s * (NT / SPLIT) + at]);
    }
  }
  __device__ __forceinline__ void store(uint16_t *out, int ch) const {
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
    *reinterpret_cast<uint2 *>(out + ch * 4) =
        make_uint2(cvt_pk_bf16(o[0] * inv, o[1] * inv), cvt_pk_bf16(o[2] * inv, o[3] * inv));
  }
};

// Workgroup (y, w): rows of the group whose first part workgroup w left in its slot.  (The
// rows run faster: groups' first parts are a constant number of slots apart, often a
// multiple of eight, and by w they would all be one XCD's.)
template <int DH, int SPLIT>
__global__ __launch_bounds__(NT) void paged_attention_join_kernel(PagedAttentionArgs a, int G, Parts<DH> parts) {
  using J = RowJoin<DH, SPLIT>;
  __shared__ f32x4 so[SPLIT > 1 ? NT : 1];
  __shared__ float sm[SPLIT > 1 ? NT : 1], sl[SPLIT > 1 ? NT : 1];
  const int w = blockIdx.y, ch = threadIdx.x % J::CH, sub = threadIdx.x / J::CH % J::PER;
  const int split = threadIdx.x / (J::CH * J::PER), jr = blockIdx.x * J::PER + sub;
  const PartInfo in = parts.info[w];
  if ((int)blockIdx.x * J::PER >= in.rows) return;
  J j;
  j.clear();
  if (jr < in.rows)
#pragma unroll 4
    for (int i = split; i <= in.more; i += SPLIT)
      j.add(i == 0 ? parts.first + w * ROWS + jr : parts.later + (w + i) * ROWS + jr, ch);
  j.gather(so, sm, sl, split);
  if (split == 0 && jr < in.rows) {
    const int row = in.row0 + jr, tok = row / G;
    j.store(a.out + (long long)(in.token + tok) * a.o_stride + (in.head * G + row - tok * G) * DH, ch);
  }
}

// The same for 128-row tiles, a lane's R rows and U parts at once, so that loads are in
// flight: four rows where groups have few parts (15.5 -> 14.0 us for the 1024 slots of
// a prompt call), eight parts where they have many.
template <int DH, int R, int U>
__global__ __launch_bounds__(NT) void paged_attention_tile_join_kernel(PagedAttentionArgs a, int G, Parts<DH> parts) {
  using J = RowJoin<DH, 1>;
  const int w = blockIdx.y, ch = threadIdx.x % J::CH, jr0 = blockIdx.x * J::PER * R + threadIdx.x / J::CH;
  const PartInfo in = parts.info[w];
  if ((int)blockIdx.x * J::PER * R >= in.rows) return;
  J j[R];
#pragma unroll
  for (int k = 0; k < R; ++k) j[k].clear();
  for (int i0 = 0; i0 <= in.more; i0 += U) {
    f32x4 o[U][R];
    float m[U][R], l[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u, in.more);
      const PartRow<DH> *p = i == 0 ? parts.first + (long long)w * TROWS : parts.later + (long long)(w + i) * TROWS;
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const PartRow<DH> *row = p + min(jr0 + k * J::PER, in.rows - 1);
        o[u][k] = *reinterpret_cast<const f32x4 *>(row->o + ch * 4);
        m[u][k] = row->m;
        l[u][k] = row->l;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u <= in.more)
#pragma unroll
        for (int k = 0; k < R; ++k) j[k].add(m[u][k], l[u][k], o[u][k]);
  }
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int row = in.row0 + jr0 + k * J::PER, tok = row / G;
    if (jr0 + k * J::PER < in.rows)
      j[k].store(a.out + (long long)(in.token + tok) * a.o_stride + (in.head * G + row - tok * G) * DH, ch);
  }
}

// Row i = token * H + head: its own parts and the prefix's.
template <int DH, int SPLIT>
__global__ __launch_bounds__(NT) void paged_attention_join2_kernel(PagedAttentionArgs a, ServeBatch b, int H, int W,
                                                                   Parts<DH> own, int own_rows, Parts<DH> pre, int pre_rows) {
  using J = RowJoin<DH, SPLIT>;
  __shared__ f32x4 so[SPLIT > 1 ? NT : 1];
  __shared__ float sm[SPLIT > 1 ? NT : 1], sl[SPLIT > 1 ? NT : 1];
  const int ch = threadIdx.x % J::CH, sub = threadIdx.x / J::CH % J::PER, split = threadIdx.x / (J::CH * J::PER);
  const long long i = (long long)blockIdx.x * J::PER + sub;
  const int tok = (int)(i / H), head = (int)(i - (long long)tok * H);
  const bool in = tok < b.T && seq_of_token(b, tok) >= 0;  // else zeroed already
  J j;
  j.clear();
  if (in) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const Parts<DH> &p = k ? pre : own;
      const int slot_rows = k ? pre_rows : own_rows;
      const PartRow<DH> *f = p.first + i;
      // (clamped: sequences that overlap, which q_start must not make, would mix two groups' words)
      const int first = clamp_int(f->first, 0, W - 1), more = min(f->more & 0xffff, W - 1 - first);
      const int jr = (f->more >> 16) & (slot_rows - 1);
#pragma unroll 4
      for (int n = split; n <= more; n += SPLIT)
        j.add(n == 0 ? f : p.later + (long long)(first + n) * slot_rows + jr, ch);
    }
  }
  j.gather(so, sm, sl, split);
  if (split == 0 && in) j.store(a.out + (long long)tok * a.o_stride + head * DH, ch);
}

// ---- the division of a call --------------------------------------------------------
struct Division {
  int W;          // workgroups of a launch
  bool stacked;   // the prefix once for the rows of all sequences
  bool own_tiles, pre_tiles;  // 128-row tiles for the own keys' part, the prefix's
  bool whole;     // a workgroup for each group of the own keys' part
};
bool can_stack(const ServeBatch &b, long long rows) {
  return b.prefix_len > 0 && b.B > 1 && rows < (long long)b.B * TROWS;
}
// The rules' figures are us with a rule's one side and its other, G = 4, Dh = 128 unless said.
// Whether one token a sequence sees no more keys of a sequence's own than a workgroup takes.
bool short_table(const ServeBatch &b) { return !b.q_start && (long long)b.max_pages << b.page_log2 <= 1024; }
// 128-row tiles for the own keys' part.  Such a tile reads keys once for what takes 16-row
// tiles two reads and more, but its blocks follow each other more slowly, so there have to be
// enough: by 16-row tiles of all key heads.  8 sequences of 2000 to 4000 keys, 8 new tokens (128
// tiles): 33 us, in 16-row tiles 46; 64 new tokens of one sequence of 2000 (128): 24 to 35; 32 of
// them (64): 20 to 21; 60 new tokens, twice, of 12 heads and 77 keys before (90): 14 to 13;
// 4 new tokens of 8 sequences (one tile each): 30 to 30.
// Between one 16-row tile a sequence and two there have to be more of them: 5 new tokens of 64
// sequences of 500 to 2000 keys (640) 86 to 137, of 16 (160) 30 to 43, one token and 20 query heads
// of 64 (320) 46 to 74; 15 new tokens of 30, G = 2, 500 keys (112) 21 to 18; but whole groups
// are faster: one token, 24 query heads, 64 sequences of 100 to 1000 keys 31 to 28.
// T and B do not say how the tokens are spread, and one long sequence in 16-row tiles costs
// several times the call: 127 sequences of one token and one of 800 264 to 549, 255 and 256
// tokens after 16000 keys 325 to 899.  So with seven 128-row tiles' rows beyond a token each
// they are taken, at a cost where the rows are spread evenly: 2 tokens of 256 sequences 244 to
// 237, 4 of 128 139 to 133; with fewer rows it would be larger (4 of 64 91 to 77).
bool tiles_for_own(const ServeBatch &b, long long G, int Hkv, bool short_own_keys) {
  const long long rows = b.T * G, tiles16 = rows * Hkv / ROWS;
  if (rows >= (long long)b.B * 2 * ROWS) return tiles16 >= 96;
  return tiles16 >= 128 && !short_own_keys && (rows > (long long)b.B * ROWS || ((long long)b.T - b.B) * G >= 7 * TROWS);
}
Division divide(const ServeBatch &b, int H, int Hkv, int dh) {
  const long long G = H / Hkv, rows = b.T * G;
  const long long own_keys = (long long)b.max_pages << b.page_log2;  // what the table can name
  Division d;
  d.W = 2 * device_cus();
  d.own_tiles = tiles_for_own(b, G, Hkv, short_table(b));
  // 64 sequences over 4096 keys of prefix: 32 us to 44; 32: 29 to 29; 16: 25 to 23; 4: 20 to 16
  d.pre_tiles = rows >= 8 * ROWS;
  // Up to 1024 keys a group takes no longer than its cut parts and their join: 64 sequences
  // of up to 1000 keys 39 us to 47, 8 of them 15 to 15, one 10 to 11; up to 2000, one 18 to 12.
  const bool short_own = short_table(b) && !d.own_tiles;
  const bool short_all = short_own && own_keys + b.prefix_len <= 1024;
  // A prefix that sequences share has a product of its own, with all their rows, if each has
  // less than a tile of rows and the keys and values that are then not read again
  // (from the caches, mostly) are worth the launches.  In MB, if the own keys' part takes
  // the sums in: 8 sequences, 1200 keys of prefix (34) 15 us to 17, 2 and 2400 (10)
  // 15 to 14; if it takes a join: 16 of 1000 to 2000 keys, 2400 (147) 45 to 51, 1200
  // (74) 43 to 41; if there are several tokens a sequence, or one launch would do:
  // 8 of 4, 9600 (275) 40 to 49, 2000 (57) 31 to 23; 128 of one, 600 (312) 33 to 35, 48
  // (115) 20 to 19.
  const long long again = (long long)(b.B - 1) * b.prefix_len * Hkv * dh * 4;
  const int least_mb = b.q_start || short_all ? 256 : short_own ? 16 : 80;
  d.stacked = can_stack(b, rows) && again >= least_mb * 1000000LL;
  d.whole = short_own && (d.stacked || short_all);
  return d;
}

template <int DH>
size_t slot_bytes(const Division &d, bool tiles) {
  return (size_t)d.W * (tiles ? TROWS : ROWS) * sizeof(PartRow<DH>);
}

template <int DH>
size_t workspace_of(const ServeBatch &b, int H, int Hkv) {
  // (whatever the division makes of the arrays that the call brings: the larger tiles, if any
  // table has them)
  const Division d = divide(b, H, Hkv, DH);
  const size_t own = slot_bytes<DH>(d, tiles_for_own(b, H / Hkv, Hkv, false)), plain = d.W * sizeof(PartInfo) + 2 * own;
  if (!can_stack(b, (long long)b.T * (H / Hkv))) return plain;
  return std::max(plain, 2 * (size_t)b.T * H * sizeof(PartRow<DH>) + own + slot_bytes<DH>(d, d.pre_tiles));
}

template <int DH>
hipError_t launch_dh(const PagedAttentionArgs &a, hipStream_t s) {
  const Division d = divide(a.b, a.H, a.Hkv, DH);
  const int G = a.H / a.Hkv;
  char *ws = static_cast<char *>(a.workspace);
  // (the launch alone: how many keys there are only the device's arrays say)
  auto plan = [&](const char *name, int grid, int per_cu) {
    plans_add(make_plan(name, grid, per_cu, grid, 16));
  };
  // the own keys' part or, stacked, the prefix's
  auto attend = [&](bool tiles, bool stacked, int dense, const Parts<DH> &parts) {
    const int keys = tiles ? TKEYS : KEYS, pre_blocks = (a.b.prefix_len + keys - 1) / keys;
    // In tiles, four blocks a workgroup where groups have sixteen, two where they have eight, or
    // writing and joining the parts of their rows takes longer (without pauses 64 tokens of one
    // sequence of 2000 keys 28 us, with one block each 37); but 400 tokens and nothing before them, 8 heads of
    // 64, 15 us with one block, 21 with four.  (Not for a prefix, which is one tile or two: 64
    // sequences over one of 4000 47 us, with one block 44.)
    const AttnSplit sp{a.b, G, a.Hkv, tiles ? TROWS : ROWS, tiles ? 6 : 7, d.stacked && !stacked ? 0 : pre_blocks, stacked,
                       tiles ? TILE_PAUSE : 0, tiles && !stacked ? (int)((long long)a.b.T * G / TROWS + a.b.B) * a.Hkv : 0};
    auto kern = tiles ? paged_attention_tile_kernel<DH> : paged_attention_kernel<DH>;
    static const char *const names[2][2] = {{"llama_paged_attention", "llama_paged_attention_tiles"},
                                            {"llama_paged_attention_prefix", "llama_paged_attention_prefix_tiles"}};
    plan(names[stacked][tiles], d.W, wg_per_cu(kern, NT));
    hipLaunchKernelGGL(kern, dim3(d.W), dim3(NT), 0, s, a, sp, dense, parts);
  };
  const int own_rows = d.own_tiles ? TROWS : ROWS, pre_rows = d.pre_tiles ? TROWS : ROWS;
  const size_t dense = (size_t)a.b.T * a.H * sizeof(PartRow<DH>);
  auto take = [&](size_t later) {  // a stacked call's regions
    Parts<DH> p{nullptr, reinterpret_cast<PartRow<DH> *>(ws), reinterpret_cast<PartRow<DH> *>(ws + dense)};
    ws += dense + later;
    return p;
  };
  Parts<DH> pre{nullptr, nullptr, nullptr};
  if (d.stacked) {
    pre = take(slot_bytes<DH>(d, d.pre_tiles));
    attend(d.pre_tiles, true, 1, pre);
  }
  if (d.whole) {
    const int tiles = (G + ROWS - 1) / ROWS, groups = a.b.B * a.Hkv * tiles;
    auto launch = [&](auto nw) {
      constexpr int NW = decltype(nw)::value;
      const int pre_blocks = d.stacked ? 0 : (a.b.prefix_len + 32 * NW - 1) / (32 * NW);
      const AttnSplit sp{a.b, G, a.Hkv, ROWS, __builtin_ctz(32 * NW), pre_blocks, 0};
      auto kern = paged_attention_whole_kernel<DH, NW>;
      plan("llama_paged_attention_whole", groups, wg_per_cu(kern, 64 * NW));
      hipLaunchKernelGGL(kern, dim3(groups), dim3(64 * NW), 0, s, a, sp, tiles, d.W, pre, pre_rows);
    };
    // eight waves where groups leave CUs idle: 16 sequences of up to 1000 keys, Dh = 64, 9.5 us
    // to 10.9 (Dh = 128 the same either way); 128 of 8 key heads 62 to 57
    if (groups > device_cus()) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 8>{});
  } else if (!d.stacked) {
    Parts<DH> parts;
    parts.info = reinterpret_cast<PartInfo *>(ws);
    parts.first = reinterpret_cast<PartRow<DH> *>(ws + d.W * sizeof(PartInfo));
    parts.later = parts.first + (size_t)d.W * own_rows;
    attend(d.own_tiles, false, 0, parts);
    if (d.own_tiles) {
      // parts of a group, if the workgroups share as few groups as there may be
      const long long groups = ((long long)a.b.T * G + TROWS - 1) / TROWS * a.Hkv;
      const bool many = d.W >= 8 * groups;
      auto join = many ? paged_attention_tile_join_kernel<DH, 1, 8> : paged_attention_tile_join_kernel<DH, 4, 1>;
      const int y = TROWS / ((many ? 1 : 4) * RowJoin<DH, 1>::PER);
      plan("llama_paged_attention_join", d.W * y, wg_per_cu(join, NT));
      hipLaunchKernelGGL(join, dim3(y, d.W), dim3(NT), 0, s, a, G, parts);
    } else {
      auto join = paged_attention_join_kernel<DH, NT * 4 / DH>;
      const int y = a.b.q_start ? ROWS : std::min(ROWS, G);
      plan("llama_paged_attention_join", d.W * y, wg_per_cu(join, NT));
      hipLaunchKernelGGL(join, dim3(y, d.W), dim3(NT), 0, s, a, G, parts);
    }
  } else {
    const Parts<DH> own = take(slot_bytes<DH>(d, d.own_tiles));
    attend(d.own_tiles, false, 1, own);
    auto join = paged_attention_join2_kernel<DH, NT * 4 / DH>;
    plan("llama_paged_attention_join", a.b.T * a.H, wg_per_cu(join, NT));
    hipLaunchKernelGGL(join, dim3(a.b.T * a.H), dim3(NT), 0, s, a, a.b, a.H, d.W, own, own_rows, pre, pre_rows);
  }
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_workspace(const ServeBatch &b, int H, int Hkv, int dh) {
  return dh == 128 ? workspace_of<128>(b, H, Hkv) : workspace_of<64>(b, H, Hkv);
}

hipError_t launch_llama_paged_attention(const PagedAttentionArgs &a, hipStream_t s) {
  return a.dh == 128 ? launch_dh<128>(a, s) : launch_dh<64>(a, s);
}

}  // namespace npu
