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
// The next block's 16 KB per wave are in flight while this one is computed.
//
// The probabilities are rounded to bf16 for the second product (2^-9 of each
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

// The workspace's regions.  Plain: info[W], first parts [W][ROWS], later parts
// [W][ROWS].  Stacked prefix: own and prefix first parts [T][H] each, later parts
// [W][ROWS] each.
template <int DH>
struct Parts {
  PartInfo *info;
  PartRow<DH> *first, *later;
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// One 32-key step's loads of a wave.
template <int DH>
struct KeyBlock {
  Frag16 k[2][DH / 32];
  uint32_t v[8][DH / 32];  // [key][dword]: DH / 16 bf16 of the lane's entries
};

template <int DH>
__device__ __forceinline__ void load_block(KeyBlock<DH> &b, const uint16_t *k0, const uint16_t *k1,
                                           const uint16_t *v0, const uint16_t *v1, int lane) {
  const int r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int d = 0; d < DH / 32; ++d) {
    b.k[0][d] = load16(k0 + r * DH + d * 32 + q * 8);
    b.k[1][d] = load16(k1 + r * DH + d * 32 + q * 8);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint16_t *p = (e < 4 ? v0 : v1) + (q * 4 + (e & 3)) * DH + r * (DH / 16);
    if constexpr (DH == 128) {
      const Frag16 f = load16(p);
      for (int i = 0; i < 4; ++i) b.v[e][i] = f.u[i];
    } else {
      const uint2 f = *reinterpret_cast<const uint2 *>(p);
      b.v[e][0] = f.x;
      b.v[e][1] = f.y;
    }
  }
}

template <int DH>
__global__ __launch_bounds__(NT, 2) void paged_attention_kernel(PagedAttentionArgs a, AttnSplit sp, int dense,
                                                                Parts<DH> parts) {
  constexpr int E = DH / 16;  // entries of a lane's output run, MFMAs of the second product
  __shared__ long long s_sum[NT];
  __shared__ UnitCursor s_cur;
  __shared__ float s_m[4][ROWS], s_l[4][ROWS];
  __shared__ __attribute__((aligned(16))) float s_o[4][ROWS][DH + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int w = blockIdx.x;

  // rows of no sequence give zeros
  if (!sp.stacked && sp.b.q_start) {
    const int lo = clamp_int(sp.b.q_start[0], 0, sp.b.T), hi = clamp_int(sp.b.q_start[sp.b.B], lo, sp.b.T);
    const int spare = lo + (sp.b.T - hi), cols = sp.Hkv * sp.G * DH / 8;
    for (long long i = (long long)w * NT + tid; i < (long long)spare * cols; i += (long long)gridDim.x * NT) {
      const int t = (int)(i / cols), c = (int)(i - (long long)t * cols);
      *reinterpret_cast<u32x4 *>(a.out + (long long)(t < lo ? t : hi + t - lo) * a.o_stride + c * 8) = u32x4{0, 0, 0, 0};
    }
  }

  // this workgroup's share: the units of every sequence, summed over the lanes
  const int seqs = split_seqs(sp), per = (seqs + NT - 1) / NT;
  long long mine = 0;
  for (int s = tid * per; s < min(seqs, (tid + 1) * per); ++s) mine += seq_units(sp, s);
  s_sum[tid] = mine;
  __syncthreads();
  for (int off = 1; off < NT; off <<= 1) {
    const long long v = tid >= off ? s_sum[tid - off] : 0;
    __syncthreads();
    s_sum[tid] += v;
    __syncthreads();
  }
  const long long U = s_sum[NT - 1];
  const int W = split_workgroups(U, gridDim.x);
  if (!dense && tid == 0) parts.info[w].rows = 0;
  if (w >= W) return;
  const long long u0 = first_unit(U, W, w), u1 = first_unit(U, W, w + 1);
  const long long before = s_sum[tid] - mine;
  if (u0 >= before && u0 < s_sum[tid]) s_cur = seek_unit(sp, tid * per, before, u0);
  __syncthreads();
  UnitCursor c = s_cur;

  const float scale = a.scale * 1.44269504088896340736f;  // exponentials in base 2
  for (long long u = u0; u < u1;) {
    const int b0 = c.blk, b1 = c.nb - b0 < u1 - u ? c.nb : b0 + (int)(u1 - u);
    const int row0 = c.tile * ROWS, rows = min(ROWS, c.n * sp.G - row0);
    // the tile's queries: row `r` of this lane
    const int row = row0 + min(r, rows - 1), tok = row / sp.G;
    Frag16 qf[DH / 32];
    {
      const uint16_t *p = a.Q + (long long)(c.start + tok) * a.q_stride + (c.head * sp.G + row - tok * sp.G) * DH + q * 8;
#pragma unroll
      for (int d = 0; d < DH / 32; ++d) qf[d] = load16(p + d * 32);
    }
    const int lim = visible_keys(sp, c.seq, c.n, tok);
    const int tile_lim = visible_keys(sp, c.seq, c.n, (row0 + rows - 1) / sp.G);
    const int *table = sp.b.page_table + (sp.stacked ? 0 : c.seq * sp.b.table_stride);
    const uint16_t *kh = a.k_pages + ((long long)c.head << sp.b.page_log2) * DH;
    const uint16_t *vh = a.v_pages + ((long long)c.head << sp.b.page_log2) * DH;

    f32x4 o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.f;

    // Block blk of the group: its keys' places, the limit of this lane's row and
    // of the whole tile, and the loads of this wave's 32 keys.
    struct Where {
      int j, lim, all;
      bool live[2];
    };
    KeyBlock<DH> kb;
    auto fetch = [&](int blk, KeyBlock<DH> &to) {
      Where x;
      const bool pre = blk < sp.pre_blocks;
      x.j = (pre ? blk : blk - sp.pre_blocks) * KEYS + wave * 32;
      x.lim = pre ? sp.b.prefix_len : lim;
      x.all = pre ? sp.b.prefix_len : tile_lim;
      const int *t = pre ? a.prefix_table : table;
      const uint16_t *kp[2], *vp[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = x.j + 16 * h;
        int page = -1;
        if (j < x.all) page = checked_page(t[j >> sp.b.page_log2], sp.b.n_pages);
        page = __builtin_amdgcn_readfirstlane(page);
        x.live[h] = page >= 0;
        const long long pg = max(page, 0);
        const int in = (j & ((1 << sp.b.page_log2) - 1)) * DH;
        kp[h] = kh + pg * a.kpage_stride + in;
        vp[h] = vh + pg * a.vpage_stride + in;
      }
      load_block<DH>(to, kp[0], kp[1], vp[0], vp[1], lane);
      return x;
    };
    Where at = fetch(b0, kb);
    for (int blk = b0; blk < b1; ++blk) {
      KeyBlock<DH> cur = kb;
      const Where x = at;
      if (blk + 1 < b1) at = fetch(blk + 1, kb);
      if (!x.live[0] && !x.live[1]) continue;
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
          s[h][i] = x.live[h] && x.j + 16 * h + 4 * q + i < x.lim ? v : -__builtin_inff();
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
      if (x.j + 32 > x.all || !x.live[0] || !x.live[1]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool keep = x.live[e >> 2] && x.j + 16 * (e >> 2) + 4 * q + (e & 3) < x.all;
#pragma unroll
          for (int i = 0; i < DH / 32; ++i) cur.v[e][i] = keep ? cur.v[e][i] : 0u;
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
    }

    // join the four waves' sums
    LanePair l16 = lane_pair16(l);
    l = l16.lo + l16.hi;
    LanePair l32 = lane_pair32(l);
    l = l32.lo + l32.hi;
    if (q == 0) {
      s_m[wave][r] = m;
      s_l[wave][r] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<f32x4 *>(&s_o[wave][r][(q * 4 + i) * E + e]) = f32x4{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
    __syncthreads();
    const bool starts = b0 == 0, ends = b1 == c.nb;
    const int more = starts && !ends ? unit_owner(U, W, c.base + c.nb - 1) - w : 0;
    if (!dense && starts && !ends && tid == 0) {
      PartInfo &in = parts.info[w];
      in.rows = rows;
      in.token = c.start;
      in.row0 = row0;
      in.head = c.head;
      in.more = more;
    }
    // lane (jr, jc): entries 8 jc .. of row jr
    for (int i = tid; i < rows * (DH / 8); i += NT) {
      const int jr = i / (DH / 8), jc = i % (DH / 8);
      float mm = -__builtin_inff(), ll = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < 4; ++v) mm = fmaxf(mm, s_m[v][jr]);
      const float base = mm == -__builtin_inff() ? 0.f : mm;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float f = exp2_(s_m[v][jr] - base);
        ll += f * s_l[v][jr];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += f * s_o[v][jr][jc * 8 + e];
      }
      const int orow = row0 + jr, ot = orow / sp.G, head = c.head * sp.G + orow - ot * sp.G;
      const long long token = c.start + ot;
      if (!dense && starts && ends) {
        const float inv = ll > 0.f ? 1.0f / ll : ll == 0.f ? 0.f : ll;
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = cvt_pk_bf16(acc[2 * e] * inv, acc[2 * e + 1] * inv);
        *reinterpret_cast<u32x4 *>(a.out + token * a.o_stride + head * DH + jc * 8) = v;
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

// Joins the parts of one output row: 8 lanes' worth of parts at a time, each
// lane 4 (Dh 128) entries.  The order of the sums is the parts', whatever ran
// first.
template <int DH>
struct RowJoin {
  static constexpr int CH = DH / 4, SPLIT = NT / CH;
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
  __device__ __forceinline__ void gather(f32x4 *so, float *sm, float *sl, int split, int ch) {
    so[split * CH + ch] = o;
    sm[split * CH + ch] = m;
    sl[split * CH + ch] = l;
    __syncthreads();
    if (split == 0)
      for (int s = 1; s < SPLIT; ++s) add(sm[s * CH + ch], sl[s * CH + ch], so[s * CH + ch]);
  }
  __device__ __forceinline__ void store(uint16_t *out, int ch) const {
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
    *reinterpret_cast<uint2 *>(out + ch * 4) =
        make_uint2(cvt_pk_bf16(o[0] * inv, o[1] * inv), cvt_pk_bf16(o[2] * inv, o[3] * inv));
  }
};

// Workgroup (w, jr): row jr of the group whose first part workgroup w left.
template <int DH>
__global__ __launch_bounds__(NT) void paged_attention_join_kernel(PagedAttentionArgs a, int G, Parts<DH> parts) {
  using J = RowJoin<DH>;
  __shared__ f32x4 so[NT];
  __shared__ float sm[NT], sl[NT];
  const int w = blockIdx.x, jr = blockIdx.y;
  const PartInfo in = parts.info[w];
  if (jr >= in.rows) return;
  const int ch = threadIdx.x % J::CH, split = threadIdx.x / J::CH;
  J j;
  j.clear();
  for (int i = split; i <= in.more; i += J::SPLIT)
    j.add(i == 0 ? parts.first + w * ROWS + jr : parts.later + (w + i) * ROWS + jr, ch);
  j.gather(so, sm, sl, split, ch);
  if (split == 0) {
    const int row = in.row0 + jr, tok = row / G;
    j.store(a.out + (long long)(in.token + tok) * a.o_stride + (in.head * G + row - tok * G) * DH, ch);
  }
}

// Workgroup i: row i = token * H + head, its own parts and the prefix's.
template <int DH>
__global__ __launch_bounds__(NT) void paged_attention_join2_kernel(PagedAttentionArgs a, ServeBatch b, int H,
                                                                   int W, Parts<DH> own, Parts<DH> pre) {
  using J = RowJoin<DH>;
  __shared__ f32x4 so[NT];
  __shared__ float sm[NT], sl[NT];
  const long long i = blockIdx.x;
  const int tok = (int)(i / H), head = (int)(i - (long long)tok * H);
  if (seq_of_token(b, tok) < 0) return;  // zeroed already
  const int ch = threadIdx.x % J::CH, split = threadIdx.x / J::CH;
  J j;
  j.clear();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const Parts<DH> &p = k ? pre : own;
    const PartRow<DH> *f = p.first + i;
    // (clamped: sequences that overlap, which q_start must not make, would mix two groups' words)
    const int first = clamp_int(f->first, 0, W - 1), more = min(f->more & 0xffff, W - 1 - first);
    const int jr = (f->more >> 16) & (ROWS - 1);
    for (int n = split; n <= more; n += J::SPLIT) j.add(n == 0 ? f : p.later + (first + n) * ROWS + jr, ch);
  }
  j.gather(so, sm, sl, split, ch);
  if (split == 0) j.store(a.out + (long long)tok * a.o_stride + head * DH, ch);
}

// How a call is divided: the workgroups of a launch, and whether the prefix is
// computed once for the rows of all sequences.
struct Division {
  int W;
  bool stacked;
};
// A prefix is shared by a product of its own where it saves reading it per
// sequence: more than one sequence, each with less than a tile of rows.
Division divide(const ServeBatch &b, int H, int Hkv) {
  const int G = H / Hkv;
  const bool stacked = b.prefix_len > 0 && b.B > 1 && (long long)b.T * G < (long long)b.B * ROWS;
  return Division{2 * device_cus(), stacked};
}

template <int DH>
hipError_t launch_dh(const PagedAttentionArgs &a, hipStream_t s) {
  const Division d = divide(a.b, a.H, a.Hkv);
  const int G = a.H / a.Hkv, rows = a.b.T * a.H;
  const int pre_blocks = (a.b.prefix_len + KEYS - 1) / KEYS;
  AttnSplit sp{a.b, G, a.Hkv, ROWS, KEYS, d.stacked ? 0 : pre_blocks, 0};
  char *ws = static_cast<char *>(a.workspace);
  const size_t slots = (size_t)d.W * ROWS * sizeof(PartRow<DH>);
  auto plan = [&](const char *name, int grid) {
    npu_launch_plan p = make_plan(name, grid, wg_per_cu(paged_attention_kernel<DH>, NT), grid, 16);
    plans_add(p);
  };
  auto kern = paged_attention_kernel<DH>;
  if (!d.stacked) {
    Parts<DH> parts;
    parts.info = reinterpret_cast<PartInfo *>(ws);
    parts.first = reinterpret_cast<PartRow<DH> *>(ws + d.W * sizeof(PartInfo));
    parts.later = parts.first + (size_t)d.W * ROWS;
    plan("llama_paged_attention", d.W);
    hipLaunchKernelGGL(kern, dim3(d.W), dim3(NT), 0, s, a, sp, 0, parts);
    plan("llama_paged_attention_join", d.W);
    const int most = a.b.q_start ? ROWS : std::min(ROWS, G);
    hipLaunchKernelGGL(paged_attention_join_kernel<DH>, dim3(d.W, most), dim3(NT), 0, s, a, G, parts);
  } else {
    const size_t dense = (size_t)rows * sizeof(PartRow<DH>);
    Parts<DH> own{nullptr, reinterpret_cast<PartRow<DH> *>(ws), reinterpret_cast<PartRow<DH> *>(ws + dense)};
    ws += dense + slots;
    Parts<DH> pre{nullptr, reinterpret_cast<PartRow<DH> *>(ws), reinterpret_cast<PartRow<DH> *>(ws + dense)};
    AttnSplit sq{a.b, G, a.Hkv, ROWS, KEYS, pre_blocks, 1};
    plan("llama_paged_attention_prefix", d.W);
    hipLaunchKernelGGL(kern, dim3(d.W), dim3(NT), 0, s, a, sq, 1, pre);
    plan("llama_paged_attention", d.W);
    hipLaunchKernelGGL(kern, dim3(d.W), dim3(NT), 0, s, a, sp, 1, own);
    plan("llama_paged_attention_join", rows);
    hipLaunchKernelGGL(paged_attention_join2_kernel<DH>, dim3(rows), dim3(NT), 0, s, a, a.b, a.H, d.W, own, pre);
  }
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_workspace(const ServeBatch &b, int H, int Hkv, int dh) {
  const Division d = divide(b, H, Hkv);
  const size_t row = dh == 128 ? sizeof(PartRow<128>) : sizeof(PartRow<64>), slots = (size_t)d.W * ROWS * row;
  return d.stacked ? 2 * ((size_t)b.T * H * row + slots) : d.W * sizeof(PartInfo) + 2 * slots;
}

hipError_t launch_llama_paged_attention(const PagedAttentionArgs &a, hipStream_t s) {
  return a.dh == 128 ? launch_dh<128>(a, s) : launch_dh<64>(a, s);
}

}  // namespace npu
