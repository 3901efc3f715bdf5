// The serving kernels' index functions (csrc/serve_batch.hpp), built for the
// host: test_serve_batch.py walks them over lengths, starts and page tables of
// every kind, the malformed ones among them.
#include "../../npu-dialect_amd/csrc/serve_batch.hpp"

using namespace npu;

extern "C" {

struct HostBatch {
  const int *page_table, *kv_len, *q_start;
  long long table_stride;
  int T, B, max_pages, page_log2, n_pages, prefix_len;
};

static ServeBatch batch(const HostBatch *h) {
  return ServeBatch{h->page_table, h->kv_len, h->q_start, h->table_stride, h->T,
                    h->B, h->max_pages, h->page_log2, h->n_pages, h->prefix_len};
}

// out[4 t ..]: pos, page, in_page, live of every token
void serve_places(const HostBatch *h, int *out) {
  const ServeBatch b = batch(h);
  for (int t = 0; t < b.T; ++t) {
    const Place p = place_of_token(b, t);
    out[4 * t] = p.pos;
    out[4 * t + 1] = p.page;
    out[4 * t + 2] = p.in_page;
    out[4 * t + 3] = p.live;
  }
}

int serve_visible(const HostBatch *h, int seq, int i) {
  const ServeBatch b = batch(h);
  const AttnSplit a{b, 1, 1, 16, 7, 0, 0};
  return visible_keys(a, split_kv(a, seq), seq_span(b, seq).n, i);
}

// The segments of all workgroups of a launch in order, eight ints each: workgroup, seq,
// tile, head, first block, one past its last, blocks of the group, first token
// of the sequence.  Returns their number, or -1 if a cursor found by seeking
// differs from the one reached by walking, or the owners disagree.
long long serve_segments(const HostBatch *h, int G, int Hkv, int rows, int keys, int pre_blocks, int stacked,
                         int launched, int *out, long long most) {
  const AttnSplit a{batch(h), G, Hkv, rows, __builtin_ctz(keys), pre_blocks, stacked};
  long long U = 0, n = 0;
  for (int s = 0; s < split_seqs(a); ++s) U += seq_units(a, s);
  const int W = split_workgroups(U, launched);
  for (int w = 0; w < W; ++w) {
    long long u = first_unit(U, W, w);
    const long long end = first_unit(U, W, w + 1);
    if (u >= end) return -3;
    UnitCursor c = seek_unit(a, 0, 0, u);
    while (u < end) {
      const long long left = end - u;
      const int b1 = c.nb - c.blk < left ? c.nb : c.blk + (int)left;
      if (unit_owner(U, W, u) != w || unit_owner(U, W, u + b1 - c.blk - 1) != w || c.base + c.blk != u) return -1;
      if (n >= most) return -2;
      const int seg[8] = {w, c.seq, c.tile, c.head, c.blk, b1, c.nb, c.start};
      for (int i = 0; i < 8; ++i) out[8 * n + i] = seg[i];
      ++n;
      u += b1 - c.blk;
      if (u < end) next_group(a, c);
    }
  }
  return n;
}

// The same, as the tile kernel walks them, with a pause of that many units before each group:
// a share may begin in one, hold nothing else, or end in one.
long long serve_segments_paused(const HostBatch *h, int G, int Hkv, int rows, int keys, int pre_blocks, int pause,
                                int launched, int *out, long long most) {
  AttnSplit a{batch(h), G, Hkv, rows, __builtin_ctz(keys), pre_blocks, 0};
  a.pause = pause;
  long long U = 0, n = 0;
  for (int s = 0; s < split_seqs(a); ++s) U += seq_units(a, s);
  const int W = split_workgroups(U, launched);
  for (int w = 0; w < W; ++w) {
    long long u = first_unit(U, W, w);
    const long long end = first_unit(U, W, w + 1);
    UnitCursor c = seek_unit(a, 0, 0, u);
    if (c.base > u || u >= c.base + c.nb + pause) return -1;
    if (c.blk < 0) {
      u -= c.blk;
      c.blk = 0;
      if (u >= end) continue;
    }
    long long left = end - u;
    for (int b0 = c.blk, blk = b0;; ++blk) {
      if (c.base + pause + blk < u || c.base + pause + blk >= end) return -3;
      const bool same = blk + 1 < c.nb, more = left > (same ? 1 : 1 + pause);
      if (!same || !more) {
        if (unit_owner(U, W, c.base + pause + b0) != w || unit_owner(U, W, c.base + pause + blk) != w) return -1;
        if (n >= most) return -2;
        const int seg[8] = {w, c.seq, c.tile, c.head, b0, blk + 1, c.nb, c.start};
        for (int i = 0; i < 8; ++i) out[8 * n + i] = seg[i];
        ++n;
        if (!more) break;
        next_group(a, c);
        left -= pause;
        b0 = 0;
        blk = -1;
      }
      --left;
    }
  }
  return n;
}

}  // extern "C"
