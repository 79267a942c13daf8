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
// none of them. A piece border inside an item falls on the tile border next to it;
// items cut by borders leave FP32 partials (at most two per CTA: its first and its last
// item) that a second kernel joins, deriving the same split.
// The length of an item is its cache rows times n_rep, the causal part counted exactly
// up to rounding: base n_rep + (rows up to its last), so that the axis has a closed form.
struct PagedRows {
  const int32_t *q_start;  // [batch + 1], or null: row b is sequence b's only one
  const int32_t *kv_len;   // [batch]
  int T, batch, n_kv, n_rep, cap;
  int M, tile;             // rows of an item, cache rows of a tile
  int causal;
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
  if (!s.stairs) return static_cast<long long>(j) * max(static_cast<long long>(s.len) * p.n_rep, 1ll);
  const long long jj = j;
  long long v = jj * s.base * p.n_rep + jj * (jj + 1) / 2 * p.M;
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

struct PagedAt {
  int b, kvh, j;
  long long start;  // the item's place on the axis
};

// The item that holds position x of the axis, given its sequence and that one's start.
__device__ __forceinline__ PagedAt paged_item_at(const PagedRows &p, const PagedSeq &s, int b,
                                                 long long b_start, long long x) {
  PagedAt at;
  at.b = b;
  const long long one = paged_before(p, s, s.J);
  const long long rem0 = x - b_start;
  at.kvh = static_cast<int>(rem0 / one);
  const long long rem = rem0 - at.kvh * one;
  int lo = 0, hi = s.J - 1;  // the last j with before(j) <= rem
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (paged_before(p, s, mid) <= rem) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  at.j = lo;
  at.start = b_start + at.kvh * one + paged_before(p, s, lo);
  return at;
}

// Tile border that stands for place `off` of an item of cost `cost` and nt tiles.
__device__ __forceinline__ int paged_border(long long off, long long cost, int nt) {
  if (off <= 0) return 0;
  if (off >= cost) return nt;
  return static_cast<int>((off * nt + (cost >> 1)) / cost);
}

// Total length of the axis and, for position x = total * c / G of it (c < G), the
// sequence that holds x and its start. All NT threads of the block call it.
struct PagedScan {
  long long part[32];
  long long total, b_start;
  int b;
};
template <int NT>
__device__ __forceinline__ void paged_find(const PagedRows &p, PagedScan &sm, int c, int G,
                                           long long &total, int &b, long long &b_start) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + NT - 1) / NT;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  long long mine = 0;
  for (int i = b0; i < b1; ++i) mine += paged_seq_cost(p, paged_seq(p, i));
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  if (lane == 31) sm.part[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < NT / 32 ? sm.part[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += o;
    }
    if (lane < NT / 32) sm.part[lane] = w;
    if (lane == NT / 32 - 1) sm.total = w;
  }
  __syncthreads();
  total = sm.total;
  const long long x = total * c / G;
  long long at = (warp > 0 ? sm.part[warp - 1] : 0) + incl - mine;
  if (x >= at && x < at + mine) {
    for (int i = b0; i < b1; ++i) {
      const long long cost = paged_seq_cost(p, paged_seq(p, i));
      if (x < at + cost) {
        sm.b = i;
        sm.b_start = at;
        break;
      }
      at += cost;
    }
  }
  __syncthreads();
  b = sm.b;
  b_start = sm.b_start;
}

}  // namespace chr
