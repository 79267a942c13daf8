// What the paged-cache kernels share (sm_100a): the cache's description and the split
// of ragged attention work over the CTAs of one launch.
//
// Cache rows live in pages of `page` rows (a power of two >= 16), [n_pages, page, n_kv,
// hd] per pool; row a of sequence s is row a % page of page table[s][a / page].

#pragma once

#include "nf4_common.cuh"

namespace chr {

struct PagedCache {
  __nv_bfloat16 *k, *v;
  const int32_t *table;
  long long k_page_stride, v_page_stride, table_stride;  // elements
  int n_pages, page_shift, n_kv, hd, batch, max_pages;
};

inline int paged_cache(const chr_nf4_pages_t *p, PagedCache &c) {
  if (p->k == nullptr || p->v == nullptr || p->table == nullptr) return kNull;
  if (p->n_pages < 1 || p->page < 16 || (p->page & (p->page - 1)) != 0 || p->page > (1 << 16) ||
      p->n_kv < 1 || p->hd < 2 || (p->hd & 1) != 0 || p->hd > 4096 || p->batch < 1 ||
      p->max_pages < 1 || p->table_stride < p->max_pages ||
      static_cast<long long>(p->max_pages) * p->page > 0x7fffffffll ||
      static_cast<long long>(p->n_kv) * p->hd > (1 << 22)) {
    return kDims;
  }
  const long long one = static_cast<long long>(p->page) * p->n_kv * p->hd;
  if (p->k_page_stride < one || p->v_page_stride < one) return kDims;
  c.k = static_cast<__nv_bfloat16 *>(p->k);
  c.v = static_cast<__nv_bfloat16 *>(p->v);
  c.table = static_cast<const int32_t *>(p->table);
  c.k_page_stride = p->k_page_stride;
  c.v_page_stride = p->v_page_stride;
  c.table_stride = p->table_stride;
  c.n_pages = p->n_pages;
  c.page_shift = 0;
  while ((1 << c.page_shift) < p->page) ++c.page_shift;
  c.n_kv = p->n_kv;
  c.hd = p->hd;
  c.batch = p->batch;
  c.max_pages = p->max_pages;
  return kOk;
}

// ---- the split of ragged attention work -------------------------------------------
// Sequence b has n new rows (tokens) and `len` cache rows, its new ones included. Under
// one kv head its queries are R = n * n_rep rows (token-major), cut into items of M
// rows. Item j reads cache rows 0 .. kv_end(j), in tiles of `tile` rows. All items, in
// the order (sequence, kv head, item), lie on one axis with a length that is what they
// cost, and CTA c of G takes the piece between total c / G and total (c+1) / G of it: every
// CTA has the same amount of cache to read whatever the lengths, and the host needs to know
// none of them. A piece border inside an item falls on the tile border next to it; an
// item that a border cuts is left as FP32 partials (at most two per CTA: of its first
// and of its last item) that a second kernel joins.
// The length of an item is its cache rows plus `extra` (what starting and ending it costs,
// in rows), times n_rep; the causal part is counted exactly up to rounding - base n_rep
// plus the rows up to its last - so that the axis has a closed form.
// Places on the axis are whole numbers in binary64 (the host sees to it that they stay
// below 2^53, where sums and products of them are exact): every CTA derives the same ones.
// The walk runs once per CTA, from a cold instruction cache, where a kilobyte of code takes as
// long as a cache tile; hence short loops and no wide integer division.
struct PagedRows {
  const int32_t *q_start;  // [batch + 1], or null: row b is sequence b's only one
  const int32_t *kv_len;   // [batch]
  int T, batch, n_kv, n_rep, cap;
  int M, tile, extra;      // rows of an item, cache rows of a tile, an item's own cost
  int causal;
  float per_rep;           // 1 / n_rep
};

struct PagedSeq {
  int r0, n, len;     // first row, rows, cache rows
  int base;           // len - n: cache rows older than the new ones (may be negative)
  int R, J;           // query rows under a kv head, items
  int stairs;         // causal with a cost that grows from item to item
  double flat;        // the part of an item's cost that does not
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedRows &p, int b) {
  PagedSeq s;
  s.r0 = b;
  int end = b < p.T ? b + 1 : b;
  if (p.q_start != nullptr) {
    s.r0 = min(max(__ldg(p.q_start + b), 0), p.T);
    end = min(max(__ldg(p.q_start + b + 1), s.r0), p.T);
  }
  s.n = end - s.r0;
  s.len = min(max(__ldg(p.kv_len + b), 0), p.cap);
  s.base = s.len - s.n;
  s.R = s.n * p.n_rep;
  s.J = (s.R + p.M - 1) / p.M;
  s.stairs = p.causal != 0 && s.base >= 0;
  s.flat = (static_cast<double>(s.stairs ? s.base : s.len) + p.extra) * p.n_rep;
  return s;
}

// Length of items 0 .. j-1, and of item j.
__device__ __forceinline__ double paged_before(const PagedRows &p, const PagedSeq &s, int j) {
  const double jj = j;
  double v = jj * s.flat;
  if (s.stairs) v += j < s.J ? 0.5 * jj * (jj + 1.0) * p.M : 0.5 * jj * (jj - 1.0) * p.M + s.R;
  return v;
}
__device__ __forceinline__ double paged_cost(const PagedRows &p, const PagedSeq &s, int j) {
  return s.flat + (s.stairs ? min((j + 1) * p.M, s.R) : 0);
}

// Cache rows item j can see: to its last token's own row when causal, else all.
__device__ __forceinline__ int paged_kv_end(const PagedRows &p, const PagedSeq &s, int j) {
  if (p.causal == 0) return s.len;
  const int last = (min((j + 1) * p.M, s.R) - 1) / p.n_rep;
  return max(s.base + last + 1, 0);
}

// Tile border that stands for place `off` of an item of cost `cost` and nt tiles: any
// function of the three that does not fall as `off` grows will do, and each step of this
// one is rounded monotonically.
__device__ __forceinline__ int paged_border(double off, double cost, int nt) {
  if (off <= 0.0) return 0;
  if (off >= cost) return nt;
  const float f = __fdiv_rn(__double2float_rn(off), __double2float_rn(cost));
  return min(__float2int_rn(__fmul_rn(f, __int2float_rn(nt))), nt);
}

// floor(a / b) for whole a >= 0, b > 0 and a small quotient: a guess, put right.
__device__ __forceinline__ int floor_div(double a, double b) {
  int q = __float2int_rz(__fdividef(__double2float_rn(a), __double2float_rn(b)));
  while (q * b > a) --q;
  while ((q + 1) * b <= a) ++q;
  return q;
}

// The axis: its length and the pieces it is cut into (no more than the grid has CTAs, and none
// shorter than a tile). Piece c starts at floor(total (c / G)).
struct PagedAxis {
  double total, per;  // per = 1 / G
  int G;
};
__device__ __forceinline__ double paged_piece(const PagedAxis &x, int c) {
  return c >= x.G ? x.total : floor(x.total * (c * x.per));
}

// One piece of a CTA's share: tiles t0 .. t1-1 of an item.
struct Seg {
  int b, kvh, row0, rows;   // the item's rows among the sequence's R
  int r0, base, len, kv_end;
  int t0, t1, whole, slot;  // whole: no border cuts it; slot: which of the CTA's partials else
  int tok0, rem0;           // token and head (of the group) of row0
};
constexpr int kSegs = 24;   // segments described at a time

// A CTA's note for the join: whether its two partials hold anything, and, if a cut item
// starts in its piece, that item: pieces first .. first + n - 1 hold a partial each (the
// first in slot 1, the others in slot 0).
struct PagedCut {
  int live[2];
  int n, kvh, row0, rows, r0, pad;
};

// The walk along a CTA's piece. One warp starts it, its first thread goes on.
struct SegWalk {
  double x_hi, x_lo, start;  // the piece, and the item the walk is at
  PagedSeq s;
  int b, kvh, j;
  PagedAxis axis;
};

// Token of the sequence that row r of a segment's item belongs to, and the query head. With
// x = rem0 + r < n_rep + 256 the quotient is exact: (x + 1/2) / n_rep is at least 1 / (2 n_rep)
// from an integer, its rounding below x 2^-22 / n_rep.
__device__ __forceinline__ int token_of(const PagedRows &p, const Seg &g, int r) {
  return g.tok0 + __float2int_rz((static_cast<float>(g.rem0 + r) + 0.5f) * p.per_rep);
}
__device__ __forceinline__ int head_of(const PagedRows &p, const Seg &g, int r, int token) {
  return g.kvh * p.n_rep + g.rem0 + r - (token - g.tok0) * p.n_rep;
}

// Called by a whole warp; false: nothing to do for CTA c. A lane takes a run of sequences:
// one pass adds them up, a second, by the lane that holds the piece's start, finds it.
static __device__ __noinline__ bool walk_start(const PagedRows &p, SegWalk &w, int c, int ctas) {
  const int lane = threadIdx.x & 31;
  const int per = (p.batch + 31) / 32;
  const int b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
  PagedAxis axis;
  double at = 0.0, x = 0.0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    double cost = 0.0;
    PagedSeq s;
    int b = b0;
#pragma unroll 1
    for (; b < b1; ++b) {
      s = paged_seq(p, b);
      cost = paged_before(p, s, s.J) * p.n_kv;
      if (pass == 1 && x < at + cost) break;
      at += cost;
    }
    if (pass == 1) {
      const double one = paged_before(p, s, s.J);
      const int kvh = floor_div(x - at, one);
      at += kvh * one;
      int lo = 0, hi = s.J - 1;  // the last item that starts at x or before
#pragma unroll 1
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at + paged_before(p, s, mid) <= x) {
          lo = mid;
        } else {
          hi = mid - 1;
        }
      }
      w.b = b;
      w.kvh = kvh;
      w.j = lo;
      w.start = at + paged_before(p, s, lo);
      w.s = s;
      w.x_lo = x;
      w.x_hi = paged_piece(axis, c + 1);
      w.axis = axis;
      break;
    }
    double incl = at;
#pragma unroll 1
    for (int off = 1; off < 32; off <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += o;
    }
    axis.total = __shfl_sync(0xffffffffu, incl, 31);
    if (axis.total <= 0.0) return false;
    const double unit = static_cast<double>(p.tile) * p.n_rep;
    axis.G = axis.total < unit * ctas ? max(floor_div(axis.total, unit), 1) : ctas;
    axis.per = 1.0 / axis.G;
    if (c >= axis.G) return false;
    x = paged_piece(axis, c);
    const int from = __ffs(__ballot_sync(0xffffffffu, x < incl)) - 1;
    if (lane != from) break;
    at = incl - at;
  }
  __syncwarp();
  return true;
}

// The item at the walk's place as a segment of CTA c's piece, then on to the next one.
__device__ __forceinline__ void walk_next(const PagedRows &p, SegWalk &w, int c, Seg &g, PagedCut &cut) {
  const double cost = paged_cost(p, w.s, w.j), end = w.start + cost;
  g.b = w.b;
  g.kvh = w.kvh;
  g.row0 = w.j * p.M;
  g.tok0 = g.row0 / p.n_rep;
  g.rem0 = g.row0 - g.tok0 * p.n_rep;
  g.rows = min(p.M, w.s.R - g.row0);
  g.r0 = w.s.r0;
  g.base = w.s.base;
  g.len = w.s.len;
  g.kv_end = paged_kv_end(p, w.s, w.j);
  const int nt = max((g.kv_end + p.tile - 1) / p.tile, 1);
  g.t0 = paged_border(w.x_lo - w.start, cost, nt);
  g.t1 = paged_border(w.x_hi - w.start, cost, nt);
  g.whole = w.start >= w.x_lo && end <= w.x_hi;
  g.slot = w.start < w.x_lo ? 0 : 1;
  if (g.whole == 0) cut.live[g.slot] = g.t0 < g.t1;
  if (g.slot == 1 && end > w.x_hi) {
    // the last piece that starts before the item's end
    int last = c + 1 + __float2int_rz(__fdividef(__double2float_rn(end - w.x_hi) * w.axis.G, __double2float_rn(w.axis.total)));
    last = min(last, w.axis.G - 1);
#pragma unroll 1
    while (last > c + 1 && paged_piece(w.axis, last) >= end) --last;
#pragma unroll 1
    while (last + 1 < w.axis.G && paged_piece(w.axis, last + 1) < end) ++last;
    cut.n = last - c + 1;
    cut.kvh = g.kvh;
    cut.row0 = g.row0;
    cut.rows = g.rows;
    cut.r0 = g.r0;
  }
  w.start = end;
  if (++w.j == w.s.J) {
    w.j = 0;
    if (++w.kvh == p.n_kv) {
      w.kvh = 0;
#pragma unroll 1
      while (++w.b < p.batch) {
        w.s = paged_seq(p, w.b);
        if (w.s.J > 0) break;
      }
    }
  }
}

}  // namespace chr
