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

// The walk along a CTA's piece: the place a warp is at.
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

// Describes up to kSegs segments of CTA c's piece from the walk's place on, and moves it past
// them: their number, with kMore set if there are others. Called by a whole warp: lane i takes
// the i-th item from the walk's place, for which it steps over groups (a kv head of a sequence) of
// J items each. One thread that went from item to item took 0.8 us for each.
constexpr int kMore = 256;
static __device__ __noinline__ int walk_fill(const PagedRows &p, SegWalk &w, PagedCut &cut, int c, Seg *segs) {
  static_assert(kSegs < 32, "a lane looks at the first item of the next call");
  const int lane = threadIdx.x & 31;
  const double x_lo = w.x_lo, x_hi = w.x_hi;
  PagedSeq s = w.s;
  int b = w.b, kvh = w.kvh, j = w.j + lane;
  bool in = w.start < x_hi;
  double start = w.start - paged_before(p, s, w.j);  // of the group
#pragma unroll 1
  while (in && j >= s.J) {
    const int groups = min(j / s.J, p.n_kv - kvh);
    j -= groups * s.J;
    start += groups * paged_before(p, s, s.J);
    kvh += groups;
    in = start < x_hi;
    if (in && kvh == p.n_kv) {
      kvh = 0;
      s.J = 0;
      while (in && s.J == 0) {
        if (++b < p.batch) {
          s = paged_seq(p, b);
        } else {
          in = false;
        }
      }
    }
  }
  __syncwarp();  // all have read the walk's place
  start += paged_before(p, s, j);
  in = in && start < x_hi;
  Seg g;
  bool some = false;
  if (in && lane < kSegs) {
    const double cost = paged_cost(p, s, j), end = start + cost;
    g.b = b;
    g.kvh = kvh;
    g.row0 = j * p.M;
    g.tok0 = g.row0 / p.n_rep;
    g.rem0 = g.row0 - g.tok0 * p.n_rep;
    g.rows = min(p.M, s.R - g.row0);
    g.r0 = s.r0;
    g.base = s.base;
    g.len = s.len;
    g.kv_end = paged_kv_end(p, s, j);
    const int nt = max((g.kv_end + p.tile - 1) / p.tile, 1);
    g.t0 = paged_border(x_lo - start, cost, nt);
    g.t1 = paged_border(x_hi - start, cost, nt);
    g.whole = start >= x_lo && end <= x_hi;
    g.slot = start < x_lo ? 0 : 1;
    some = g.t0 < g.t1;
    if (g.whole == 0) cut.live[g.slot] = some;
    if (g.slot == 1 && end > x_hi) {
      // the last piece that starts before the item's end
      const PagedAxis axis = w.axis;
      int last = c + 1 + __float2int_rz(__fdividef(__double2float_rn(end - x_hi) * axis.G, __double2float_rn(axis.total)));
      last = min(last, axis.G - 1);
#pragma unroll 1
      while (last > c + 1 && paged_piece(axis, last) >= end) --last;
#pragma unroll 1
      while (last + 1 < axis.G && paged_piece(axis, last + 1) < end) ++last;
      cut.n = last - c + 1;
      cut.kvh = g.kvh;
      cut.row0 = g.row0;
      cut.rows = g.rows;
      cut.r0 = g.r0;
    }
  }
  const unsigned described = __ballot_sync(0xffffffffu, some);
  if (some) segs[__popc(described & ((1u << lane) - 1u))] = g;
  const bool more = __shfl_sync(0xffffffffu, in, kSegs);
  if (lane == kSegs) {
    w.start = in ? start : x_hi;
    w.s = s;
    w.b = b;
    w.kvh = kvh;
    w.j = j;
  }
  __syncwarp();
  return __popc(described) + (more ? kMore : 0);
}

}  // namespace chr
