// Attention of ragged rows over a paged KV cache (sm_100a): one new token per sequence, a
// tree of drafted tokens, or a prompt chunk, for a batch of sequences of any lengths.
// No counterpart in the reference, which attends one contiguous block per sequence
// (gpu/nf4/nf4_gemv.cu:558-727, gpu/decodev2/prefill.py:50-92).
//
// Sequence b has n new rows, whose keys and values are the last n of its len cache rows;
// base = len - n. Row i sees cache row t when t < base, or when t - base <= i (causal),
// or, given a tree, when bit t - base of the row's mask is set:
//   out[i, h] = sum_t softmax_t(scale q[i, h] . k[t, h / n_rep]) v[t, h / n_rep]
// A row that sees nothing is zero. One pass over the cache with a running maximum and sum.
//
// The query rows of a sequence under one kv head (tokens x n_rep heads) are the rows of
// the matrix tiles, so a cache row is read once for up to M of them. The work of a launch
// is split over the CTAs by what it costs (paged.cuh).

#include <algorithm>

#include "attn_mma.cuh"
#include "paged.cuh"

namespace chr {
namespace {

struct PagedAttnArgs {
  PagedCache c;
  PagedRows p;
  const __nv_bfloat16 *q;
  __nv_bfloat16 *out;
  const unsigned long long *tree;
  float *ws;
  long long q_stride;
  int tree_words, zero_tail;
  float c2;  // scale * log2(e)
};

__device__ __forceinline__ void ldm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// One piece of a CTA's share: tiles t0 .. t1-1 of an item.
struct Seg {
  int b, kvh, row0, rows;   // the item's rows among the sequence's R
  int r0, base, len, kv_end;
  int t0, t1, nt, slot;     // slot: which of the CTA's two partials
};

// Partial results: [CTA][2][M][HD + 2] floats, the row's unnormalised output, its running
// maximum (log2 units) and its sum.
__device__ __forceinline__ float *partial_of(const PagedAttnArgs &a, int cta, int slot, int row) {
  return a.ws + ((static_cast<long long>(cta) * 2 + slot) * a.p.M + row) * (a.c.hd + 2);
}

// ---- thin form: up to 16 MT query rows per item ----------------------------------------
// Eight warps on warp-level matrix instructions (m16n8k16, FP32 accumulate). Warp w owns
// cache rows 16w .. 16w+15 of every 128-row tile: it copies them itself (cp.async ring of
// its own, the K and the V half of a block as separate stages, so no block-wide barrier
// stands in the loop), runs its own softmax and its own output accumulator; the warps are
// folded through shared memory at the end of a segment while the next segment's copies
// are in flight. Bound by HBM: 16 query rows cost 32 matrix instructions per 16 cache rows,
// a tenth of what the copy of those rows takes. kStages x 4 KB x 8 warps keep 128 KB in flight per SM
// (the latency-bandwidth product needs about 55).
// Probabilities are rounded to bf16 for the second product (their sum is not); q, k and v
// are bf16 already.
constexpr int kThinWarps = 8;
constexpr int kThinThreads = kThinWarps * 32;
constexpr int kThinTile = kThinWarps * 16;
constexpr int kSegs = 32;  // segments described at a time

template <int HD, int MT>
struct ThinLayout {
  static constexpr int kM = 16 * MT;
  static constexpr int kHalf = 16 * HD * 2;                                 // 16 rows of K or V
  static constexpr int kStages = 5;
  static constexpr int kRing = kThinWarps * kStages * kHalf;
  static constexpr int kFoldCols = HD < 64 / MT ? HD : 64 / MT;             // columns folded at a time
  static constexpr int kFold = kThinWarps * kM * kFoldCols * 4;
  static constexpr int kMl = kThinWarps * kM * 2 * 4;
  static constexpr int kQ = kM * HD * 2;
  static constexpr int kSegB = kSegs * static_cast<int>(sizeof(Seg));
  static constexpr int kBytes = kRing + kFold + kMl + kQ + kSegB + static_cast<int>(sizeof(PagedScan)) + 64;
};

// Row r, 16-byte chunk c of a block whose rows are HD bf16: the chunk index is mixed with
// the row so that eight rows of one chunk column fall into eight bank groups.
template <int HD>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  constexpr int C = HD / 8;
  if (C >= 8) return static_cast<uint32_t>(r * HD * 2 + ((c ^ (r & 7)) << 4));
  if (C == 4) return static_cast<uint32_t>(r * HD * 2 + ((c ^ ((r >> 1) & 3)) << 4));
  return static_cast<uint32_t>(r * HD * 2 + ((c ^ ((r >> 2) & 1)) << 4));
}

// Describes up to kSegs segments from position (at, x) of the CTA's piece on; returns how
// many, and leaves the place where it stopped. One thread.
struct SegWalk {
  long long x_lo, x_hi, b_start;
  int b;
  PagedAt at;
  PagedSeq s;
};
__device__ __forceinline__ void walk_start(const PagedAttnArgs &a, SegWalk &w, long long total, int c,
                                           int G, int b, long long b_start) {
  w.x_lo = total * c / G;
  w.x_hi = total * (c + 1) / G;
  if (w.x_lo >= w.x_hi) return;
  w.s = paged_seq(a.p, b);
  w.at = paged_item_at(a.p, w.s, b, b_start, w.x_lo);
}
// The item at the walk's place: its segment in this CTA's piece (false: empty), then on.
__device__ __forceinline__ bool walk_next(const PagedAttnArgs &a, SegWalk &w, Seg &g) {
  const PagedRows &p = a.p;
  const long long cost = paged_cost(p, w.s, w.at.j);
  g.b = w.at.b;
  g.kvh = w.at.kvh;
  g.row0 = w.at.j * p.M;
  g.rows = min(p.M, w.s.R - g.row0);
  g.r0 = w.s.r0;
  g.base = w.s.base;
  g.len = w.s.len;
  g.kv_end = paged_kv_end(p, w.s, w.at.j);
  g.nt = max((g.kv_end + p.tile - 1) / p.tile, 1);
  g.t0 = paged_border(w.x_lo - w.at.start, cost, g.nt);
  g.t1 = paged_border(w.x_hi - w.at.start, cost, g.nt);
  g.slot = w.at.start < w.x_lo ? 0 : 1;
  const bool some = g.t0 < g.t1;
  // on to the next item
  w.at.start += cost;
  if (++w.at.j == w.s.J) {
    w.at.j = 0;
    if (++w.at.kvh == p.n_kv) {
      w.at.kvh = 0;
      while (++w.at.b < p.batch) {
        w.s = paged_seq(p, w.at.b);
        if (w.s.J > 0) break;
      }
    }
  }
  return some;
}
__device__ __forceinline__ int walk_fill(const PagedAttnArgs &a, SegWalk &w, Seg *segs) {
  int n = 0;
  while (n < kSegs && w.x_lo < w.x_hi && w.at.start < w.x_hi && w.at.b < a.p.batch) {
    Seg g;
    if (walk_next(a, w, g)) segs[n++] = g;
  }
  return n;
}

// Whether query row r (of the sequence's R) sees cache row t >= base, t < len.
__device__ __forceinline__ bool sees_draft(const PagedAttnArgs &a, const Seg &g, int token, int t) {
  const int d = t - g.base;
  if (a.tree == nullptr) return d <= token;
  if ((d >> 6) >= a.tree_words) return false;
  const unsigned long long w =
      __ldg(a.tree + static_cast<long long>(g.r0 + token) * a.tree_words + (d >> 6));
  return (w >> (d & 63)) & 1ull;
}

template <int HD, int MT>
__global__ void __launch_bounds__(kThinThreads, 1) attn_paged_thin_kernel(const PagedAttnArgs a) {
  using L = ThinLayout<HD, MT>;
  constexpr int KS = HD / 16, NT = HD / 8, C = HD / 8;
  constexpr int M = L::kM;
  constexpr int S = L::kStages;
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char *at = smem + L::kRing;
  float *fold = reinterpret_cast<float *>(at);
  at += L::kFold;
  float *ml = reinterpret_cast<float *>(at);  // [warp][row][2]
  at += L::kMl;
  unsigned char *q_s = at;
  at += L::kQ;
  Seg *segs = reinterpret_cast<Seg *>(at);
  at += L::kSegB;
  PagedScan &scan = *reinterpret_cast<PagedScan *>(at);
  __shared__ int n_segs;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int G = gridDim.x, cta = blockIdx.x;
  pdl_wait();
  pdl_trigger();  // behind the wait: the join kernel reads q_start and kv_len before its own
  long long total, b_start;
  int b_first;
  paged_find<kThinThreads>(a.p, scan, cta, G, total, b_first, b_start);
  SegWalk walk;
  walk.x_lo = walk.x_hi = 0;
  if (tid == 0 && total > 0) walk_start(a, walk, total, cta, G, b_first, b_start);

  // rows behind the last sequence's
  if (a.zero_tail != 0) {
    const int last = a.p.q_start != nullptr
                         ? min(max(__ldg(a.p.q_start + a.p.batch), 0), a.p.T) : min(a.p.batch, a.p.T);
    const long long width = static_cast<long long>(a.p.n_kv) * a.p.n_rep * HD / 8;
    const long long n16 = (a.p.T - last) * width;
    uint4 *dst = reinterpret_cast<uint4 *>(a.out) + last * width;
    for (long long i = static_cast<long long>(cta) * kThinThreads + tid; i < n16;
         i += static_cast<long long>(G) * kThinThreads) {
      dst[i] = make_uint4(0, 0, 0, 0);
    }
  }

  const uint32_t ring = smem_u32(smem) + warp * S * L::kHalf;
  const uint32_t q_base = smem_u32(q_s);
  const int shift = a.c.page_shift;
  const long long row_el = static_cast<long long>(a.c.n_kv) * HD;

  for (;;) {
    if (tid == 0) n_segs = walk_fill(a, walk, segs);
    __syncthreads();
    const int n_now = n_segs;
    if (n_now == 0) break;

    // The copies run ahead of the arithmetic over this batch of segments: (cs, ct) is the
    // block whose half `ch` (0 K, 1 V) is requested next, its page looked up in advance.
    int cs = 0, ct = segs[0].t0, ch = 0;
    int c_page = -1;
    // whether the blocks requested and not yet used have rows at all (a block past the
    // item's end, or on a page outside the pool, has none); bit: the block's number
    unsigned has_rows = 0, n_asked = 0, n_used = 0;
    auto look_up = [&]() {
      if (cs >= n_now) return;
      const int row = ct * kThinTile + warp * 16;
      c_page = -1;
      if (row < segs[cs].kv_end) {
        const int id = __ldg(a.c.table + segs[cs].b * a.c.table_stride + (row >> shift));
        c_page = id >= 0 && id < a.c.n_pages ? id : -1;
      }
    };
    // Requests one half block into ring slot `slot` (nothing when all are requested); every
    // call is one commit group, so that groups and half blocks count alike.
    auto request = [&](int slot) {
      if (cs < n_now) {
        const int row = ct * kThinTile + warp * 16;
        const int live = c_page < 0 ? 0 : min(max(segs[cs].kv_end - row, 0), 16);
        const __nv_bfloat16 *src =
            (ch == 0 ? a.c.k : a.c.v) +
            (live > 0 ? c_page * (ch == 0 ? a.c.k_page_stride : a.c.v_page_stride) +
                            (row & ((1 << shift) - 1)) * row_el + segs[cs].kvh * HD
                      : 0);
        const uint32_t dst = ring + slot * L::kHalf;
        constexpr int kPer = 16 * C / 32;  // 16-byte pieces per lane
#pragma unroll
        for (int i = 0; i < (kPer > 0 ? kPer : 1); ++i) {
          const int piece = i * 32 + lane;
          const int r = piece / C, c = piece % C;
          // rows past the end are filled with zeros: whatever the page holds there must not
          // reach the products (0 x NaN)
          const bool on = r < live;
          mma_cp16(dst + chunk_at<HD>(r, c), on ? src + r * row_el + c * 8 : a.c.k, on ? 16 : 0);
        }
        if (ch == 0) {
          has_rows = (has_rows & ~(1u << (n_asked & 31))) | ((live > 0 ? 1u : 0u) << (n_asked & 31));
          ++n_asked;
          ch = 1;
        } else {
          ch = 0;
          if (++ct == segs[cs].t1) {
            if (++cs < n_now) ct = segs[cs].t0;
          }
          look_up();
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up();
#pragma unroll
    for (int i = 0; i < S - 1; ++i) request(i);
    int slot = 0;  // ring slot of the half block consumed next
    int ahead = S - 1;  // ring slot requested next

    for (int si = 0; si < n_now; ++si) {
      const Seg g = segs[si];
      // ---- the item's queries: rows of the matrix tiles, zero past the last ----
      for (int i = tid; i < M * C; i += kThinThreads) {
        const int r = i / C, c = i - r * C;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < g.rows) {
          const int token = (g.row0 + r) / a.p.n_rep;
          const int head = g.kvh * a.p.n_rep + (g.row0 + r) - token * a.p.n_rep;
          v = ld_act16(a.q + (g.r0 + token) * a.q_stride + head * HD + c * 8);
        }
        *reinterpret_cast<uint4 *>(q_s + chunk_at<HD>(r, c)) = v;
      }
      __syncthreads();
      // thread rows: mt * 16 + g8 and + 8
      int token[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = mt * 16 + h * 8 + g8;
          token[mt][h] = r < g.rows ? (g.row0 + r) / a.p.n_rep : -1;
        }
      }
      const uint32_t qa = (lane & 15), qc = lane >> 4;  // this lane's row and chunk of an A load
      uint32_t qf[MT == 1 ? KS : 1][4];
      if (MT == 1) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) ldm_x4(q_base + chunk_at<HD>(qa, ks * 2 + qc), qf[ks]);
      }
      float o[MT][NT][4];
      float m_run[MT][2], l_run[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        m_run[mt][0] = m_run[mt][1] = -INFINITY;
        l_run[mt][0] = l_run[mt][1] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[mt][n][0] = o[mt][n][1] = o[mt][n][2] = o[mt][n][3] = 0.f;
      }

      for (int t = g.t0; t < g.t1; ++t) {
        const int row = t * kThinTile + warp * 16;
        const uint32_t k_blk = ring + slot * L::kHalf;
        const int v_slot = slot + 1 == S ? 0 : slot + 1;
        const uint32_t v_blk = ring + v_slot * L::kHalf;
        // K half: all but the S - 2 latest groups have landed; each is this warp's own
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncwarp();
        const bool live = (has_rows >> (n_used & 31)) & 1u;
        ++n_used;
        float s[MT][2][4];
        if (live) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
          }
          const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t b[4];
            ldm_x4(k_blk + chunk_at<HD>(kr, ks * 2 + kc), b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t q4[4];
              if (MT == 1) {
#pragma unroll
                for (int e = 0; e < 4; ++e) q4[e] = qf[ks][e];
              } else {
                ldm_x4(q_base + chunk_at<HD>(mt * 16 + qa, ks * 2 + qc), q4);
              }
              mma_bf16(s[mt][0], q4[0], q4[1], q4[2], q4[3], b[0], b[1]);
              mma_bf16(s[mt][1], q4[0], q4[1], q4[2], q4[3], b[2], b[3]);
            }
          }
        }
        __syncwarp();
        request(ahead);
        ahead = ahead + 1 == S ? 0 : ahead + 1;
        uint32_t pa[MT][4];
        if (live) {
          // all of the block is older than the new rows: every row sees it
          const bool plain = row + 16 <= g.base;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float sv[4];
              float mx = -INFINITY;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = row + (e >> 1) * 8 + 2 * t4 + (e & 1);
                const float x = s[mt][e >> 1][h * 2 + (e & 1)] * a.c2;
                bool on = true;
                if (!plain) {
                  on = key < g.kv_end &&
                       (key < g.base || (token[mt][h] >= 0 && sees_draft(a, g, token[mt][h], key)));
                }
                sv[e] = on ? x : -INFINITY;
                mx = fmaxf(mx, sv[e]);
              }
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
              const float m_new = fmaxf(m_run[mt][h], mx);
              const float m_use = m_new == -INFINITY ? 0.f : m_new;  // nothing seen so far
              const float alpha = exp2f(m_run[mt][h] - m_use);
              float psum = 0.f;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                sv[e] = exp2f(sv[e] - m_use);
                psum += sv[e];
              }
              l_run[mt][h] = fmaf(l_run[mt][h], alpha, psum);
              m_run[mt][h] = m_new;
              if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  o[mt][n][h * 2] *= alpha;
                  o[mt][n][h * 2 + 1] *= alpha;
                }
              }
              pa[mt][h] = mma_pack(sv[0], sv[1]);
              pa[mt][2 + h] = mma_pack(sv[2], sv[3]);
            }
          }
        }
        // V half
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncwarp();
        if (live) {
          const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;
#pragma unroll
          for (int n2 = 0; n2 < NT / 2; ++n2) {
            uint32_t b[4];
            ldm_x4_trans(v_blk + chunk_at<HD>(vr, n2 * 2 + vc), b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_bf16(o[mt][2 * n2], pa[mt][0], pa[mt][1], pa[mt][2], pa[mt][3], b[0], b[1]);
              mma_bf16(o[mt][2 * n2 + 1], pa[mt][0], pa[mt][1], pa[mt][2], pa[mt][3], b[2], b[3]);
            }
          }
        }
        __syncwarp();
        request(ahead);
        ahead = ahead + 1 == S ? 0 : ahead + 1;
        slot = v_slot + 1 == S ? 0 : v_slot + 1;
      }

      // ---- fold the warps, kFoldCols columns at a time ----
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float l = l_run[mt][h];
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          if (t4 == 0) {
            float *w = ml + (warp * M + mt * 16 + h * 8 + g8) * 2;
            w[0] = m_run[mt][h];
            w[1] = l;
          }
        }
      }
      const bool whole = g.t0 == 0 && g.t1 == g.nt;
      constexpr int FC = L::kFoldCols;
#pragma unroll
      for (int f = 0; f < HD / FC; ++f) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int n = 0; n < FC / 8; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              *reinterpret_cast<float2 *>(fold + (warp * M + mt * 16 + h * 8 + g8) * FC + n * 8 + 2 * t4) =
                  make_float2(o[mt][f * (FC / 8) + n][h * 2], o[mt][f * (FC / 8) + n][h * 2 + 1]);
            }
          }
        }
        __syncthreads();
        for (int i = tid; i < g.rows * FC; i += kThinThreads) {
          const int r = i / FC, d = i - r * FC;
          float mm = -INFINITY;
#pragma unroll
          for (int w = 0; w < kThinWarps; ++w) mm = fmaxf(mm, ml[(w * M + r) * 2]);
          const float m_use = mm == -INFINITY ? 0.f : mm;
          float ll = 0.f, oo = 0.f;
#pragma unroll
          for (int w = 0; w < kThinWarps; ++w) {
            const float e = exp2f(ml[(w * M + r) * 2] - m_use);
            ll = fmaf(e, ml[(w * M + r) * 2 + 1], ll);
            oo = fmaf(e, fold[(w * M + r) * FC + d], oo);
          }
          const int col = f * FC + d;
          if (whole) {
            const int tok = (g.row0 + r) / a.p.n_rep;
            const int head = g.kvh * a.p.n_rep + (g.row0 + r) - tok * a.p.n_rep;
            a.out[(static_cast<long long>(g.r0 + tok) * a.p.n_kv * a.p.n_rep + head) * HD + col] =
                __float2bfloat16(ll != 0.f ? oo / ll : 0.f);
          } else {
            float *dst = partial_of(a, cta, g.slot, r);
            dst[col] = oo;
            if (col == 0) {
              dst[HD] = mm;
              dst[HD + 1] = ll;
            }
          }
        }
        __syncthreads();
      }
    }
    // the ring holds nothing that is still wanted; groups in flight are empty
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
  }
}

// ---- joins the partials of items that CTA borders cut -------------------------------
// Block c looks at the border between CTAs c and c+1: the first border inside an item
// joins that item's partials, a warp per row.
constexpr int kJoinThreads = 256;
constexpr int kMaxCtas = 256;
__global__ void __launch_bounds__(kJoinThreads) attn_paged_join_kernel(const PagedAttnArgs a, int G) {
  __shared__ PagedScan scan;
  __shared__ int from[kMaxCtas];                            // partial of each piece, -1: empty
  __shared__ float weight[kJoinThreads / 32][kMaxCtas];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c = blockIdx.x + 1;
  const int hd = a.c.hd;
  // The split is derived before the wait: the attention kernel raises its trigger only
  // behind its own wait, so what q_start and kv_len hold is there already.
  pdl_trigger();
  long long total, b_start;
  int b;
  paged_find<kJoinThreads>(a.p, scan, c, G, total, b, b_start);
  if (total <= 0) return;
  const long long x = total * c / G;
  const PagedSeq s = paged_seq(a.p, b);
  const PagedAt at = paged_item_at(a.p, s, b, b_start, x);
  if (at.start >= x || total * (c - 1) / G > at.start) return;  // not inside, or not the first
  const long long cost = paged_cost(a.p, s, at.j);
  const int nt = max((paged_kv_end(a.p, s, at.j) + a.p.tile - 1) / a.p.tile, 1);
  // the CTA that holds the item's end: the last one whose piece starts before it
  const int first = c - 1;
  const int last = min(static_cast<int>(((at.start + cost) * G - 1) / total), G - 1);
  const int n = last - first + 1;
  const int row0 = at.j * a.p.M, rows = min(a.p.M, s.R - row0);
  bool whole = false;  // a piece that was rounded to the whole item has been written by its CTA
  for (int i = tid; i < n; i += kJoinThreads) {
    const long long lo = total * (first + i) / G;
    const int t0 = paged_border(lo - at.start, cost, nt);
    const int t1 = paged_border(total * (first + i + 1) / G - at.start, cost, nt);
    from[i] = t0 < t1 ? (first + i) * 2 + (at.start < lo ? 0 : 1) : -1;
    whole |= t0 == 0 && t1 == nt;
  }
  if (__syncthreads_or(whole)) return;
  pdl_wait();
  for (int r = warp; r < rows; r += kJoinThreads / 32) {
    auto src = [&](int i) { return a.ws + (static_cast<long long>(from[i]) * a.p.M + r) * (hd + 2); };
    float mm = -INFINITY;
    for (int i = lane; i < n; i += 32) {
      if (from[i] >= 0) mm = fmaxf(mm, __ldcg(src(i) + hd));
    }
    mm = warp_max_xor(mm);
    const float m_use = mm == -INFINITY ? 0.f : mm;
    float l = 0.f;
    for (int i = lane; i < n; i += 32) {
      float w = 0.f;
      if (from[i] >= 0) {
        w = exp2f(__ldcg(src(i) + hd) - m_use);
        l = fmaf(w, __ldcg(src(i) + hd + 1), l);
      }
      weight[warp][i] = w;
    }
    l = warp_sum_xor(l);
    __syncwarp();
    float acc[4] = {0.f, 0.f, 0.f, 0.f};  // hd <= 128: columns lane, lane + 32, ...
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      if (from[i] < 0) continue;
      const float w = weight[warp][i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e * 32 + lane < hd) acc[e] = fmaf(w, __ldcg(src(i) + e * 32 + lane), acc[e]);
      }
    }
    __syncwarp();
    const int tok = (row0 + r) / a.p.n_rep;
    const int head = at.kvh * a.p.n_rep + (row0 + r) - tok * a.p.n_rep;
    __nv_bfloat16 *dst = a.out + (static_cast<long long>(s.r0 + tok) * a.p.n_kv * a.p.n_rep + head) * hd;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e * 32 + lane < hd) dst[e * 32 + lane] = __float2bfloat16(l != 0.f ? acc[e] / l : 0.f);
    }
  }
}

struct AttnForm {
  int M, tile, ctas;
};
// The form of a call: from the head layout and the mean number of new rows per sequence,
// which the host knows, never from the lengths, which it does not.
AttnForm form_of(int T, int batch, int n_rep) {
  const long long rows = (static_cast<long long>(T) + batch - 1) / batch * n_rep;
  AttnForm f;
  f.M = rows <= 16 ? 16 : 32;
  f.tile = kThinTile;
  f.ctas = std::min(sm_count(), kMaxCtas);
  return f;
}
long long ws_floats_of(const AttnForm &f, int hd) {
  return static_cast<long long>(f.ctas) * 2 * f.M * (hd + 2);
}

template <int HD, int MT>
cudaError_t launch_thin(const PagedAttnArgs &a, int ctas, cudaStream_t st) {
  static int done[64] = {};
  if (!ensure_smem_attr(attn_paged_thin_kernel<HD, MT>, ThinLayout<HD, MT>::kBytes, done)) {
    return cudaErrorInvalidValue;
  }
  return launch_chain(attn_paged_thin_kernel<HD, MT>, dim3(static_cast<unsigned>(ctas)), dim3(kThinThreads),
                      ThinLayout<HD, MT>::kBytes, st, a);
}

bool head_dim_ok(int hd) { return hd == 16 || hd == 32 || hd == 64 || hd == 128; }

}  // namespace
}  // namespace chr

using namespace chr;

extern "C" int64_t chr_nf4_attn_paged_ws(int32_t T, int32_t batch, int32_t n_q, int32_t n_kv,
                                         int32_t hd) {
  if (T < 1 || batch < 1 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0 || !head_dim_ok(hd)) return 0;
  return ws_floats_of(form_of(T, batch, n_q / n_kv), hd);
}

extern "C" int chr_nf4_attn_paged(const chr_nf4_pages_t *pages, const void *q, int64_t q_stride,
                                  void *out, const void *q_start, const void *kv_len,
                                  const void *tree, int32_t tree_words, int32_t T, int32_t n_q,
                                  float scale, float *ws, int64_t ws_floats, int32_t zero_tail,
                                  void *stream) {
  if (pages == nullptr || q == nullptr || out == nullptr || kv_len == nullptr || ws == nullptr) {
    return kNull;
  }
  PagedAttnArgs a{};
  const int rc = paged_cache(pages, a.c);
  if (rc != kOk) return rc;
  const int hd = a.c.hd;
  if (T < 1 || n_q < 1 || n_q % a.c.n_kv != 0 || !head_dim_ok(hd) ||
      q_stride < static_cast<int64_t>(n_q) * hd || (tree != nullptr && tree_words < 1) ||
      (q_start == nullptr && T != a.c.batch) || static_cast<int64_t>(T) * n_q > 0x3fffffffll) {
    return kDims;
  }
  if (!aligned(q, 16) || !aligned(out, 16) || q_stride % 8 != 0 || !aligned(a.c.k, 16) ||
      !aligned(a.c.v, 16) || a.c.k_page_stride % 8 != 0 || a.c.v_page_stride % 8 != 0 ||
      (tree != nullptr && !aligned(tree, 8))) {
    return kAlign;
  }
  const int n_rep = n_q / a.c.n_kv;
  const AttnForm f = form_of(T, a.c.batch, n_rep);
  if (ws_floats < ws_floats_of(f, hd)) return kWorkspace;
  a.p.q_start = static_cast<const int32_t *>(q_start);
  a.p.kv_len = static_cast<const int32_t *>(kv_len);
  a.p.T = T;
  a.p.batch = a.c.batch;
  a.p.n_kv = a.c.n_kv;
  a.p.n_rep = n_rep;
  a.p.cap = static_cast<int>(static_cast<long long>(a.c.max_pages) << a.c.page_shift);
  a.p.M = f.M;
  a.p.tile = f.tile;
  a.p.causal = tree == nullptr;
  // the split's arithmetic is in 64-bit integers: total axis length x CTAs
  const double items = static_cast<double>(T) * n_q / f.M + static_cast<double>(a.c.batch) * a.c.n_kv;
  if (items * a.p.cap * n_rep * f.ctas > 4.0e18 ||
      static_cast<double>(a.p.cap) * n_rep * (a.p.cap / f.tile + 1.0) > 4.0e18) {
    return kDims;
  }
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.tree = static_cast<const unsigned long long *>(tree);
  a.ws = ws;
  a.q_stride = q_stride;
  a.tree_words = tree_words;
  a.zero_tail = zero_tail != 0;
  a.c2 = scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define CHR_THIN(HD)                                                   \
  e = f.M == 16 ? launch_thin<HD, 1>(a, f.ctas, st) : launch_thin<HD, 2>(a, f.ctas, st)
  switch (hd) {
    case 16: CHR_THIN(16); break;
    case 32: CHR_THIN(32); break;
    case 64: CHR_THIN(64); break;
    default: CHR_THIN(128); break;
  }
#undef CHR_THIN
  if (e != cudaSuccess) return kLaunch;
  if (f.ctas > 1) {
    e = launch_chain(attn_paged_join_kernel, dim3(static_cast<unsigned>(f.ctas - 1)), dim3(kJoinThreads),
                     0, st, a, f.ctas);
  }
  return e == cudaSuccess ? kOk : kLaunch;
}
