// serve_batch.hpp -- where a serving batch's tokens, keys and work lie: the
// lookups in kv_len and q_start, the check of a page number, and the division of an
// attention over workgroups, with the search by which each finds its share.  Plain
// functions of the arrays, compiled for the device by the kernels and for the host by
// tests.
#pragma once

#ifdef __HIPCC__
#define NPU_HD __host__ __device__ __forceinline__
#else
#define NPU_HD inline
#endif

namespace npu {

// The batch of include/npu_amd.h, as device pointers.
struct ServeBatch {
  const int *page_table, *kv_len, *q_start;  // q_start may be null: one token each
  long long table_stride;
  int T, B, max_pages, page_log2;
  int n_pages;  // pages of the cache
  int prefix_len;
};

NPU_HD int clamp_int(long long v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : (int)v; }

// The new tokens of sequence seq, inside [0, T) whatever q_start holds.
struct SeqSpan {
  int start, n;
};
NPU_HD SeqSpan seq_span(const ServeBatch &b, int seq) {
  if (!b.q_start) return SeqSpan{seq, 1};
  const int lo = clamp_int(b.q_start[seq], 0, b.T), hi = clamp_int(b.q_start[seq + 1], lo, b.T);
  return SeqSpan{lo, hi - lo};
}

// The sequence that token t belongs to (the last one that starts at or before
// t), or -1.  Bisection: in bounds and finite on any contents of q_start.
NPU_HD int seq_of_token(const ServeBatch &b, int t) {
  if (!b.q_start) return t;
  int lo = 0, hi = b.B;  // the answer, if there is one, is in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.q_start[mid] <= t) lo = mid; else hi = mid;
  }
  return b.q_start[lo] <= t && t < b.q_start[lo + 1] ? lo : -1;
}

// A page number of the cache, or -1 where the table holds none.
NPU_HD int checked_page(int page, int n_pages) { return page >= 0 && page < n_pages ? page : -1; }

// Where a new token's key goes: live: inside its table; page -1: not stored.
struct Place {
  int pos, page, in_page, live;
};
NPU_HD Place place_of_token(const ServeBatch &b, int t) {
  Place p{0, -1, 0, 0};
  const int seq = seq_of_token(b, t);
  if (seq < 0) return p;
  const SeqSpan sp = seq_span(b, seq);
  const long long j = (long long)b.kv_len[seq] - sp.n + (t - sp.start);
  if (j < 0 || (j >> b.page_log2) >= b.max_pages) return p;
  p.live = 1;
  p.pos = b.prefix_len + (int)j;
  p.in_page = (int)(j & ((1LL << b.page_log2) - 1));
  p.page = checked_page(b.page_table[seq * b.table_stride + (j >> b.page_log2)], b.n_pages);
  return p;
}

// ---- attention over the cache, divided over workgroups ----------------------
// A row is one query head of one new token; the G query heads that share a key
// head stand together, so the rows of a sequence's key head are numbered
// token * G + g and cut into tiles of `rows`.  A tile's keys, the prefix's
// `pre_blocks` blocks and its own up to what its last token sees, are cut into
// blocks of 2^keys_log2; a (tile, key head)'s blocks are a group of units, one at
// least, so that rows without keys are written too.  Units are numbered by
// sequence, key head, tile, block (tiles that stand together read the same
// keys); workgroup w of W takes the units [U w / W, U (w + 1) / W): equal shares
// whatever the lengths, a group cut at most at the workgroups' borders.  Before a
// group's blocks come `pause` units in which nothing is done: what a group costs
// beside its blocks.  W is at most U (split_workgroups), so that every one of them
// has units and a cut group's parts are those of consecutive workgroups.
struct AttnSplit {
  ServeBatch b;
  int G, Hkv;
  int rows, keys_log2;
  int pre_blocks;  // prefix blocks before each tile's own keys
  int stacked;     // the prefix alone: the rows of all tokens as one sequence
  int pause = 0;
  int long_groups = 0;  // groups, about, if workgroups are to be fewer where groups are long; 0: they are not
};

NPU_HD int split_seqs(const AttnSplit &a) { return a.stacked ? 1 : a.b.B; }
NPU_HD SeqSpan split_span(const AttnSplit &a, int seq) {
  return a.stacked ? SeqSpan{0, a.b.T} : seq_span(a.b, seq);
}
NPU_HD int split_kv(const AttnSplit &a, int seq) { return a.stacked ? 0 : a.b.kv_len[seq]; }
// Own keys that new token i of n sees in a sequence of kv_len `kv`.
NPU_HD int visible_keys(const AttnSplit &a, int kv, int n, int i) {
  if (a.stacked) return 0;
  const long long cap = (long long)a.b.max_pages << a.b.page_log2;
  return clamp_int((long long)kv - n + i + 1, 0, clamp_int(kv, 0, (int)cap));
}
NPU_HD int split_tiles(const AttnSplit &a, int n) {
  return (int)(((unsigned)n * (unsigned)a.G + (unsigned)a.rows - 1) / (unsigned)a.rows);
}
NPU_HD int tile_blocks(const AttnSplit &a, int kv, int n, int tile) {
  // (n G < 2^31, and a tile is at most 128 rows)
  const unsigned last = (((unsigned)tile + 1) * (unsigned)a.rows - 1) / (unsigned)a.G;
  const int v = visible_keys(a, kv, n, last < (unsigned)n ? (int)last : n - 1);
  const int nb = a.pre_blocks + (int)(((unsigned)v + (1u << a.keys_log2) - 1) >> a.keys_log2);
  return nb > 0 ? nb : 1;
}
// Units of one key head of a sequence of n new tokens.
NPU_HD long long head_units(const AttnSplit &a, int kv, int n) {
  const int tiles = split_tiles(a, n);
  long long sum = 0;
  for (int t = 0; t < tiles; ++t) sum += tile_blocks(a, kv, n, t) + a.pause;
  return sum;
}
NPU_HD long long seq_units(const AttnSplit &a, int seq) {
  return head_units(a, split_kv(a, seq), split_span(a, seq).n) * a.Hkv;
}
NPU_HD int split_workgroups(long long U, int launched) { return U < launched ? (int)U : launched; }
// a / b; where they fit 32 bits, as they do but for millions of units, at a fifth of the instructions
NPU_HD long long quotient(long long a, long long b) {
  return ((unsigned long long)(a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
NPU_HD long long first_unit(long long U, int W, int w) { return quotient(U * w, W); }
NPU_HD int unit_owner(long long U, int W, long long u) { return (int)quotient((u + 1) * W - 1, U); }

// A place in the order of the units: block blk of the nb of group (seq, tile,
// head), whose first unit is `base`; n, start, kv: the sequence's.  blk < 0: in the
// group's pause.
struct UnitCursor {
  int seq, tile, head, blk, nb, n, start, kv;
  long long base;
};
// The next group (the caller knows that there is one).
NPU_HD void next_group(const AttnSplit &a, UnitCursor &c) {
  c.base += c.nb + a.pause;
  c.blk = 0;
  if (++c.tile >= split_tiles(a, c.n)) {
    c.tile = 0;
    if (++c.head >= a.Hkv) {
      c.head = 0;
      do {
        if (++c.seq >= split_seqs(a)) return;
        const SeqSpan sp = split_span(a, c.seq);
        c.n = sp.n;
        c.start = sp.start;
      } while (c.n == 0);
      c.kv = split_kv(a, c.seq);
    }
  }
  c.nb = tile_blocks(a, c.kv, c.n, c.tile);
}

// ---- a workgroup's share of the units, found by its lanes together -----------------
// `wave` stands for 64 lanes: each(f) is f(lane) of all of them (as Ints), sum(f) the
// total of f(lane), scan() the inclusive sums over the lanes, at() one lane's value,
// above() the first lane whose value exceeds another, same() a value that all lanes have.
// The kernels' wave is the hardware's, HostWave 64 numbers.

// Units of one key head of a sequence of n new tokens, its tiles over the lanes.
template <class Wave>
NPU_HD long long head_units_by(const Wave &wave, const AttnSplit &a, int kv, int n) {
  const int tiles = split_tiles(a, n);
  return wave.sum([&](int lane) {
    long long sum = 0;
    for (int t = lane; t < tiles; t += 64) sum += tile_blocks(a, kv, n, t) + a.pause;
    return sum;
  });
}
// Whether the sequences' units are summed by a wave each, for as many as there are lanes at
// most; else by a lane each, or by a lane for `per` of them.
NPU_HD bool sum_by_waves(const AttnSplit &a, int lanes) {
  const int seqs = split_seqs(a);
  return seqs <= lanes && (unsigned)a.b.T * a.G / (unsigned)a.rows >= 16u * seqs;
}
NPU_HD int seqs_per_lane(const AttnSplit &a, int lanes) { return (split_seqs(a) + lanes - 1) / lanes; }
NPU_HD long long lane_units(const AttnSplit &a, int tid, int per) {
  const int seqs = split_seqs(a), end = seqs - tid * per < per ? seqs : (tid + 1) * per;
  long long sum = 0;
  for (int q = tid * per; q < end; ++q) sum += seq_units(a, q);
  return sum;
}
// Workgroup `block` of those launched is number w of the W that have units, and takes [u0, u1)
// of all U; false: it has none.  by_xcd: workgroups that the dispatcher puts on one XCD (every
// eighth) take neighbouring shares.
struct ShareRange {
  int W, w;
  long long u0, u1;
};
NPU_HD bool share_of(const AttnSplit &a, long long U, int launched, int block, bool by_xcd, ShareRange &s) {
  const long long groups = a.long_groups;
  const int few = groups > 0 ? (U >= (8 + a.pause) * groups) + (U >= (16 + a.pause) * groups) : 0;
  s.W = split_workgroups(U >> few, launched);
  s.w = by_xcd && s.W == launched && s.W % 8 == 0 ? (block & 7) * (s.W >> 3) + (block >> 3) : block;
  if (s.w >= s.W) return false;
  s.u0 = first_unit(U, s.W, s.w);
  s.u1 = first_unit(U, s.W, s.w + 1);
  return true;
}
// A sequence, its first unit and the units of one of its key heads.
struct SeqUnits {
  int seq;
  long long base, per_head;
};
// Of lane tid's sequences, which have `units` from unit `base` on, the one that holds unit u.
NPU_HD SeqUnits seq_in_lane(const AttnSplit &a, int tid, int per, long long base, long long units, long long u) {
  int q = tid * per;
  for (; per > 1; ++q) {
    units = seq_units(a, q);
    if (u < base + units) break;
    base += units;
  }
  return SeqUnits{q, base, units / a.Hkv};
}
// The group of unit u in its sequence: a scan over the sequence's tiles.
template <class Wave>
NPU_HD UnitCursor seek_in_seq(const Wave &wave, const AttnSplit &a, const SeqUnits &s, long long u) {
  const SeqSpan sp = split_span(a, s.seq);
  UnitCursor c{s.seq, 0, 0, 0, 1, sp.n, sp.start, split_kv(a, s.seq), s.base};
  c.head = wave.same((int)quotient(u - s.base, s.per_head));
  c.base += c.head * s.per_head;
  const long long in_head = u - c.base;
  int rest = (int)(in_head < 0x7fffffff ? in_head : 0x7fffffff);  // units before u in the tiles from c.tile on
  for (;; c.tile += 64) {
    const int tiles = split_tiles(a, c.n);
    const typename Wave::Ints nb = wave.each(
        [&](int lane) { return c.tile + lane < tiles ? tile_blocks(a, c.kv, c.n, c.tile + lane) + a.pause : 0; });
    const typename Wave::Ints up_to = wave.scan(nb);
    const int all = wave.at(up_to, 63);
    if (rest < all) {
      const int at = wave.above(up_to, rest), here = wave.at(nb, at), skipped = wave.at(up_to, at) - here;
      c.tile += at;
      c.nb = here - a.pause;
      c.base += skipped;
      c.blk = rest - skipped - a.pause;
      break;
    }
    c.base += all;
    rest -= all;
  }
  c.blk = wave.same(c.blk);
  c.tile = wave.same(c.tile);
  c.base = wave.same(c.base);
  return c;
}
// Past the group's pause, from where u0 counts on.
NPU_HD void skip_pause(UnitCursor &c, long long &u0) {
  if (c.blk < 0) {
    u0 -= c.blk;
    c.blk = 0;
  }
}

#ifndef __HIPCC__
struct HostWave {
  struct Ints {
    int v[64];
  };
  template <class F>
  Ints each(F f) const {
    Ints r;
    for (int l = 0; l < 64; ++l) r.v[l] = f(l);
    return r;
  }
  template <class F>
  long long sum(F f) const {
    long long s = 0;
    for (int l = 0; l < 64; ++l) s += f(l);
    return s;
  }
  Ints scan(Ints x) const {
    for (int l = 1; l < 64; ++l) x.v[l] += x.v[l - 1];
    return x;
  }
  int at(const Ints &x, int l) const { return x.v[l]; }
  int above(const Ints &x, int y) const {
    int l = 0;
    while (x.v[l] <= y) ++l;
    return l;
  }
  template <class T>
  T same(T v) const {
    return v;
  }
};
// The group of unit u, from sequence seq on, whose first unit is `base`.
inline UnitCursor seek_unit(const AttnSplit &a, int seq, long long base, long long u) {
  for (; seq < split_seqs(a); ++seq) {
    const long long units = seq_units(a, seq);
    if (u < base + units) return seek_in_seq(HostWave(), a, SeqUnits{seq, base, units / a.Hkv}, u);
    base += units;
  }
  return UnitCursor{seq, 0, 0, 0, 1, 0, 0, 0, base};  // u is past the last unit
}
#endif

}  // namespace npu
