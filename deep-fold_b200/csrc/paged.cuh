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
// cost, and CTA c of G takes the piece [total c / G, total (c+1) / G) of it: every CTA
// has the same amount of cache to read whatever the lengths, and the host needs to know
// none of them. A piece border inside an item falls on the tile border next to it; an
// item that a border cuts is left as FP32 partials (at most two per CTA: of its first
// and of its last item) that a second kernel joins.
// The length of an item is its cache rows plus `extra` (what starting and ending it costs,
// in rows), times n_rep; the causal part is counted exactly up to rounding - base n_rep
// plus the rows up to its last - so that the axis has a closed form.
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
  bool stairs;        // causal with a cost that grows from item to item
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedRows &p, int b) {
  PagedSeq s;
  if (p.q_start != nullptr) {
    const int lo = min(max(__ldg(p.q_start + b), 0), p.T);
    const int hi = min(max(__ldg(p.q_start + b + 1), lo), p.T);
    s.r0 = lo;
    s.n = hi - lo;
  } else {
    s.r0 = b;
    s.n = b < p.T ? 1 : 0;
  }
  s.len = min(max(__ldg(p.kv_len + b), 0), p.cap);
  s.base = s.len - s.n;
  s.R = s.n * p.n_rep;
  s.J = (s.R + p.M - 1) / p.M;
  s.stairs = p.causal != 0 && s.base >= 0;
  return s;
}

// Length of items 0 .. j-1, and of item j.
__device__ __forceinline__ long long paged_before(const PagedRows &p, const PagedSeq &s, int j) {
  const long long jj = j;
  if (!s.stairs) return jj * (static_cast<long long>(s.len) + p.extra) * p.n_rep;
  long long v = jj * (static_cast<long long>(s.base) + p.extra) * p.n_rep + jj * (jj + 1) / 2 * p.M;
  if (j >= s.J) v -= jj * p.M - s.R;  // the last item is not full
  return v;
}
__device__ __forceinline__ long long paged_cost(const PagedRows &p, const PagedSeq &s, int j) {
  return paged_before(p, s, j + 1) - paged_before(p, s, j);
}
__device__ __forceinline__ long long paged_seq_cost(const PagedRows &p, const PagedSeq &s) {
  return s.J == 0 ? 0 : paged_before(p, s, s.J) * p.n_kv;
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
__device__ __forceinline__ int paged_border(long long off, long long cost, int nt) {
  if (off <= 0) return 0;
  if (off >= cost) return nt;
  const float f = __fdiv_rn(__ll2float_rn(off), __ll2float_rn(cost));
  return min(__float2int_rn(__fmul_rn(f, __int2float_rn(nt))), nt);
}

// floor(a / b) for 0 <= a < 2^62, b > 0, quotient below 2^52. The axis of most batches fits 32
// bits; else a guess in binary64 is put right.
__device__ __forceinline__ long long floor_div(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  long long q = static_cast<long long>(__ddiv_rn(static_cast<double>(a), static_cast<double>(b)));
  while (q * b > a) --q;
  while ((q + 1) * b <= a) ++q;
  return q;
}

// The axis: its length, the pieces it is cut into (no more than the grid has CTAs, and none
// shorter than a tile), and where piece c starts.
struct PagedAxis {
  long long total, whole;  // whole = total / G
  int G, rest;             // rest = total % G
};
__device__ __forceinline__ PagedAxis paged_axis(const PagedRows &p, long long total, int ctas) {
  PagedAxis x;
  x.total = total;
  const long long unit = static_cast<long long>(p.tile) * p.n_rep;
  x.G = ctas;
  if (total < unit * ctas) x.G = max(static_cast<int>(floor_div(total, unit)), 1);
  x.whole = floor_div(total, x.G);
  x.rest = static_cast<int>(total - x.whole * x.G);
  return x;
}
__device__ __forceinline__ long long paged_piece(const PagedAxis &x, int c) {
  return x.whole * c + static_cast<unsigned>(x.rest) * static_cast<unsigned>(c) / static_cast<unsigned>(x.G);
}

// One piece of a CTA's share: tiles t0 .. t1-1 of an item.
struct Seg {
  int b, kvh, row0, rows;   // the item's rows among the sequence's R
  int r0, base, len, kv_end;
  int t0, t1, whole, slot;  // whole: no border cuts it; slot: which of the CTA's partials else
  int tok0, rem0;           // token and head (of the group) of row0
};
constexpr int kSegs = 32;   // segments described at a time

// An item that borders cut, described by the CTA that holds its start: pieces first ..
// first + n - 1 hold a partial each (the first in slot 1, the others in slot 0).
struct PagedCut {
  int n, first;
  int kvh, row0, rows, r0;
};

// The walk along a CTA's piece. One warp starts it, its first thread goes on.
struct SegWalk {
  long long x_hi, x_lo, start;  // the piece, and the item the walk is at
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

// Called by a whole warp; false: nothing to do for CTA c. The walk's functions run once or
// a few times per CTA: as calls, they leave the instruction cache to the loops.
static __device__ __noinline__ bool walk_start(const PagedRows &p, SegWalk &w, int c, int ctas) {
  const int lane = threadIdx.x & 31;
  const int per = (p.batch + 31) / 32;
  const int b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
  long long mine = 0;
#pragma unroll 4
  for (int i = b0; i < b1; ++i) mine += paged_seq_cost(p, paged_seq(p, i));
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  const long long total = __shfl_sync(0xffffffffu, incl, 31);
  if (total <= 0) return false;
  const PagedAxis axis = paged_axis(p, total, ctas);
  if (c >= axis.G) return false;
  const long long x = paged_piece(axis, c);
  const int from = __ffs(__ballot_sync(0xffffffffu, x < incl)) - 1;
  if (lane == from) {
    long long at = incl - mine;
    int b = b0;
    PagedSeq s = paged_seq(p, b);
    for (;;) {
      const long long cost = paged_seq_cost(p, s);
      if (x < at + cost) break;
      at += cost;
      s = paged_seq(p, ++b);
    }
    const long long one = paged_before(p, s, s.J);
    w.b = b;
    w.kvh = static_cast<int>(floor_div(x - at, one));
    at += w.kvh * one;
    int lo = 0, hi = s.J - 1;  // the last item that starts at x or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (paged_before(p, s, mid) <= x - at) {
        lo = mid;
      } else {
        hi = mid - 1;
      }
    }
    w.j = lo;
    w.start = at + paged_before(p, s, lo);
    w.s = s;
    w.x_lo = x;
    w.x_hi = paged_piece(axis, c + 1);
    w.axis = axis;
  }
  __syncwarp();
  return true;
}

// The item at the walk's place as a segment of CTA c's piece, then on to the next one.
// `cut` is filled when the piece holds the start but not the end of the item.
__device__ __forceinline__ void walk_next(const PagedRows &p, SegWalk &w, int c, Seg &g, PagedCut &cut) {
  const long long cost = paged_cost(p, w.s, w.j), end = w.start + cost;
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
  if (g.slot == 1 && end > w.x_hi) {
    // the last piece that starts before the item's end
    int last = static_cast<int>(floor_div(end, w.axis.whole + (w.axis.rest > 0 ? 1 : 0)));
    last = min(max(last, c + 1), w.axis.G - 1);
    while (last + 1 < w.axis.G && paged_piece(w.axis, last + 1) < end) ++last;
    while (last > c + 1 && paged_piece(w.axis, last) >= end) --last;
    cut.n = last - c + 1;
    cut.first = c;
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
      while (++w.b < p.batch) {
        w.s = paged_seq(p, w.b);
        if (w.s.J > 0) break;
      }
    }
  }
}

}  // namespace chr
