// serve_batch.hpp -- where a serving batch's tokens, keys and work lie: the
// lookups in kv_len, q_start and the page tables, and the division of an
// attention over workgroups.  Plain functions of the arrays, compiled for the
// device by the kernels and for the host by a test: every index that a kernel
// forms from a caller's array is formed here.
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
// The group of unit u, from sequence seq on, whose first unit is `base`.
NPU_HD UnitCursor seek_unit(const AttnSplit &a, int seq, long long base, long long u) {
  UnitCursor c{seq, 0, 0, 0, 1, 0, 0, 0, base};
  const int seqs = split_seqs(a);
  for (; c.seq < seqs; ++c.seq) {
    const SeqSpan sp = split_span(a, c.seq);
    c.n = sp.n;
    c.start = sp.start;
    c.kv = split_kv(a, c.seq);
    const long long per = head_units(a, c.kv, c.n);
    if (u >= c.base + per * a.Hkv) {
      c.base += per * a.Hkv;
      continue;
    }
    c.head = (int)((u - c.base) / per);
    c.base += per * c.head;
    for (;; ++c.tile) {
      c.nb = tile_blocks(a, c.kv, c.n, c.tile);
      if (u < c.base + c.nb + a.pause) break;
      c.base += c.nb + a.pause;
    }
    c.blk = (int)(u - c.base) - a.pause;
    return c;
  }
  return c;  // u is past the last unit
}
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

}  // namespace npu
