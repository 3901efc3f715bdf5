// The search by which a workgroup of the attention finds its share of the units
// (csrc/serve_batch.hpp), built for the host: test_serve_share.py runs it for every
// workgroup of a launch, 256 lanes each.
#include "../../npu-dialect_amd/csrc/serve_batch.hpp"

using namespace npu;

namespace {
constexpr int NT = 256;
}

extern "C" {

struct HostShare {
  const int *page_table, *kv_len, *q_start;
  long long table_stride;
  int T, B, max_pages, page_log2, n_pages, prefix_len;
  int G, Hkv, rows, keys_log2, pre_blocks, stacked, pause, long_groups;
};

// Of each of the `launched` workgroups, in the order of their numbers, the segments of its share,
// nine long longs each: number, seq, tile, head, first block, one past its last, blocks of the group,
// first token of the sequence, first unit of the group.  `ranges`, two of each workgroup launched:
// its share [u0, u1), or zeros.  Returns the segments; below 0: the search and the owners
// disagree, or a place in the share is none.
long long serve_shares(const HostShare *h, int launched, int by_xcd, long long *out, long long most,
                       long long *ranges, long long *units) {
  const AttnSplit a{ServeBatch{h->page_table, h->kv_len, h->q_start, h->table_stride, h->T, h->B, h->max_pages,
                               h->page_log2, h->n_pages, h->prefix_len},
                    h->G, h->Hkv, h->rows, h->keys_log2, h->pre_blocks, h->stacked, h->pause, h->long_groups};
  const int seqs = split_seqs(a), per = seqs_per_lane(a, NT);
  const HostWave wave;
  long long mine[NT], before[NT + 1] = {0};
  for (int tid = 0; tid < NT; ++tid) {
    mine[tid] = lane_units(a, tid, per);
    if (sum_by_waves(a, NT)) {
      const long long by_wave =
          tid < seqs ? head_units_by(wave, a, split_kv(a, tid), split_span(a, tid).n) * a.Hkv : 0;
      if (by_wave != mine[tid]) return -1;
    }
    before[tid + 1] = before[tid] + mine[tid];
  }
  const long long U = *units = before[NT];
  long long n = 0;
  for (int block = 0; block < launched; ++block) {
    ShareRange r;
    if (!share_of(a, U, launched, block, by_xcd != 0, r)) continue;
    if (ranges[2 * r.w + 1] != 0) return -2;  // two workgroups of one number
    ranges[2 * r.w] = r.u0;
    ranges[2 * r.w + 1] = r.u1;
    int owner = -1;
    for (int tid = 0; tid < NT; ++tid)
      if (r.u0 >= before[tid] && r.u0 < before[tid] + mine[tid]) owner = tid;
    if (owner < 0) return -3;
    const SeqUnits s = seq_in_lane(a, owner, per, before[owner], mine[owner], r.u0);
    if (s.seq < 0 || s.seq >= seqs) return -4;
    UnitCursor c = seek_in_seq(wave, a, s, r.u0);
    if (c.base > r.u0 || r.u0 >= c.base + c.nb + a.pause || c.base + a.pause + c.blk != r.u0) return -5;
    long long u = r.u0;
    skip_pause(c, u);
    while (u < r.u1) {
      const int b1 = c.nb - c.blk < r.u1 - u ? c.nb : c.blk + (int)(r.u1 - u);
      if (n >= most) return -6;
      const long long seg[9] = {r.w, c.seq, c.tile, c.head, c.blk, b1, c.nb, c.start, c.base};
      for (int i = 0; i < 9; ++i) out[9 * n + i] = seg[i];
      ++n;
      // a first part's later ones are those of the workgroups up to the owner of the group's last unit
      if (unit_owner(U, r.W, u) != r.w || unit_owner(U, r.W, u + b1 - c.blk - 1) != r.w) return -7;
      u += b1 - c.blk + a.pause;
      if (u < r.u1) next_group(a, c);
    }
  }
  return n;
}

}  // extern "C"
