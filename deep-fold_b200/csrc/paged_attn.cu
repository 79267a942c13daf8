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
#include <cmath>

#include "attn_mma.cuh"
#include "paged.cuh"
#include "tma_tc.cuh"

namespace chr {
namespace {

__device__ int g_attn_paged_status = 0;

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
  uint32_t polls;  // limit of a wait
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

// The workspace: [G] notes of the CTAs, then the partials, [G][2][M] each: the running
// maximum (log2 units) and sum of a row, and its HD unnormalised outputs.
struct PagedWs {
  PagedCut *cut;
  float2 *ml;
  float *o;
};
__host__ __device__ __forceinline__ long long ws_floats_of(int ctas, int M, int hd) {
  return static_cast<long long>(ctas) * static_cast<int>(sizeof(PagedCut) / 4) +
         static_cast<long long>(ctas) * 2 * M * (hd + 2);
}
__device__ __forceinline__ PagedWs ws_of(const PagedAttnArgs &a, int ctas) {
  static_assert(sizeof(PagedCut) == 32, "two 16-byte loads");
  PagedWs w;
  w.cut = reinterpret_cast<PagedCut *>(a.ws);
  w.o = a.ws + static_cast<long long>(ctas) * static_cast<int>(sizeof(PagedCut) / 4);
  w.ml = reinterpret_cast<float2 *>(w.o + static_cast<long long>(ctas) * 2 * a.p.M * a.c.hd);
  return w;
}

// The walk of a CTA, in shared memory, as the first warp's it is not worth the registers of all.
struct PagedWalk {
  SegWalk at;
  PagedCut note;
  int n_segs;  // described now, and kMore
};
// Describes the next segments; called by the first warp. The CTA's note is complete once there
// are no more.
__device__ __forceinline__ void walk_on(const PagedAttnArgs &a, PagedWalk &w, Seg *segs) {
  const int lane = threadIdx.x & 31, ctas = gridDim.x, c = blockIdx.x;
  const int n = walk_fill(a.p, w.at, w.note, c, segs);
  if (lane == 0) w.n_segs = n;
  if (lane < static_cast<int>(sizeof(PagedCut) / 4)) {
    reinterpret_cast<int *>(ws_of(a, ctas).cut + c)[lane] = reinterpret_cast<const int *>(&w.note)[lane];
  }
}
// The first segments; all threads of the block call it.
__device__ __forceinline__ int walk_begin(const PagedAttnArgs &a, PagedWalk &w, Seg *segs) {
  if (threadIdx.x < 32) {
    if (threadIdx.x == 0) {
      w.at.start = w.at.x_hi = 0.0;
      w.note.live[0] = w.note.live[1] = w.note.n = 0;
    }
    __syncwarp();
    walk_start(a.p, w.at, blockIdx.x, gridDim.x);
    walk_on(a, w, segs);
  }
  __syncthreads();
  return w.n_segs;
}

// Which of the 32 cache rows that begin `older` rows before the new ones a drafted row sees.
__device__ __noinline__ uint32_t tree32(const unsigned long long *w, int words, int older) {
  if (older >= 32) return 0xFFFFFFFFu;
  const int d0 = -older;
  if (d0 < 0) return (static_cast<uint32_t>(__ldg(w)) << older) | ((1u << older) - 1u);
  const int i = d0 >> 6, sh = d0 & 63;
  unsigned long long v = i < words ? __ldg(w + i) >> sh : 0ull;
  if (sh > 32 && i + 1 < words) v |= __ldg(w + i + 1) << (64 - sh);
  return static_cast<uint32_t>(v);
}
// Which of the 32 cache rows k0 .. k0+31 a token's row sees.
__device__ __forceinline__ uint32_t seen32(const PagedAttnArgs &a, const Seg &g, int token, int k0) {
  const int older = g.base - k0;
  uint32_t m;
  if (a.tree == nullptr) {
    const int n = older + token + 1;
    m = n >= 32 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << n) - 1u);
  } else {
    m = tree32(a.tree + static_cast<long long>(g.r0 + token) * a.tree_words, a.tree_words, older);
  }
  const int n = g.kv_end - k0;
  if (n < 32) m &= n <= 0 ? 0u : (1u << n) - 1u;
  return m;
}

// Which of the 16 cache rows k0 .. k0+15 pairs of tokens see, two to a word. The masks' loads are
// all under way before the first is used.
template <int N>
__device__ __forceinline__ void seen16(const PagedAttnArgs &a, const Seg &g, const int (&token)[N][2], int k0,
                                       uint32_t (&see)[N]) {
  const int d0 = k0 - g.base, from = max(d0, 0), older = from - d0;  // new row of the first key, keys before it
  const int end = g.kv_end - k0;
  const uint32_t there = end >= 16 ? 0xFFFFu : (end <= 0 ? 0u : (1u << end) - 1u);
  if (a.tree == nullptr) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      uint32_t m[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int up_to = token[n][e] + 1 - d0;
        m[e] = (up_to >= 16 ? 0xFFFFu : (up_to <= 0 ? 0u : (1u << up_to) - 1u)) & there;
      }
      see[n] = m[0] | m[1] << 16;
    }
    return;
  }
  const int words = 2 * a.tree_words, i = from >> 5, sh = from & 31;  // masks as 32-bit words
  uint32_t lo[N][2], hi[N][2];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t *w = reinterpret_cast<const uint32_t *>(a.tree) + static_cast<long long>(g.r0 + token[n][e]) * words;
      lo[n][e] = hi[n][e] = 0u;
      if (i < words) lo[n][e] = __ldg(w + i);
      if (sh > 16 && i + 1 < words) hi[n][e] = __ldg(w + i + 1);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t m[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t v = __funnelshift_r(lo[n][e], hi[n][e], sh);
      m[e] = (older >= 16 ? 0xFFFFu : (v << older) | ((1u << older) - 1u)) & there;
    }
    see[n] = m[0] | m[1] << 16;
  }
}

// A masked value enters the second product with weight zero, and 0 x NaN is NaN. So where some of
// an item's rows do not see all of a tile's cache rows, infinities and NaN among their values are
// taken out before the product, and added to the rows that do see them.
constexpr uint32_t kExp2 = 0x7F807F80u;  // the exponents of two bf16
// Bits 15 and 31: whether the lower, the upper of two bf16 is an infinity or NaN (the sum carries
// out of an exponent of ones alone).
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) { return (x & kExp2) + 0x00800080u; }
__device__ __forceinline__ uint32_t not_finite8(const uint4 &x) {
  return (not_finite2(x.x) | not_finite2(x.y) | not_finite2(x.z) | not_finite2(x.w)) & 0x80008000u;
}
__device__ __forceinline__ uint32_t finite2(uint32_t x) {
  return x & ~(((not_finite2(x) >> 15) & 0x00010001u) * 0xFFFFu);
}
__device__ __forceinline__ uint4 finite8(const uint4 &x) {
  return make_uint4(finite2(x.x), finite2(x.y), finite2(x.z), finite2(x.w));
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 x;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ void sts16(uint32_t addr, const uint4 &x) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}

// Zeros for the rows that no sequence owns, in front of the first and behind the last, when the call asks for them.
template <int HD>
__device__ __forceinline__ void zero_unowned_rows(const PagedAttnArgs &a, int cta, int G) {
  if (a.zero_tail == 0 || a.p.q_start == nullptr) return;
  const int first = min(max(__ldg(a.p.q_start), 0), a.p.T);
  const int last = min(max(__ldg(a.p.q_start + a.p.batch), first), a.p.T);
  const long long width = static_cast<long long>(a.p.n_kv) * a.p.n_rep * HD / 8;
  const long long front = first * width, owned = (last - first) * width, n16 = a.p.T * width - owned;
  uint4 *dst = reinterpret_cast<uint4 *>(a.out);
  for (long long i = static_cast<long long>(cta) * blockDim.x + threadIdx.x; i < n16;
       i += static_cast<long long>(G) * blockDim.x) {
    dst[i < front ? i : i + owned] = make_uint4(0, 0, 0, 0);
  }
}

// ---- thin form: up to 8 NQ query rows per item -----------------------------------------
// Four warps on warp-level matrix instructions (m16n8k16, FP32 accumulate). Warp w owns
// cache rows 16w .. 16w+15 of every 64-row tile: it requests them itself (TMA, a ring of
// its own, the K and the V half of a block as separate stages), keeps its own running
// maximum, sum and output, and no block-wide barrier stands in the loop; the warps are
// folded through shared memory at the end of a segment, while the next one's copies are
// in flight. Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T: the cache
// rows are the 16-row operand and the queries the 8-column one, so a kv group of up to 8
// heads fills its tiles (as 16-row operand it would leave half of every product empty),
// and P^T comes out of S^T by one 8x8 transpose per tile.
// Bound by HBM: a 16-row block costs about 100 + 60 NQ warp instructions, and two CTAs of four
// warps with 4 x 4 KB requested each keep 128 KB in flight per SM (the latency-bandwidth
// product needs about 55). 64 sequences of 150 to 3500 rows, 40 / 8 heads of 128 (480 MB): 89 us,
// 5.4 TB/s; three of 90,000 to 131,071 rows, 16 / 2 heads (384 MB): 75 us, 5.1 TB/s. A short call
// is a chain of latencies: one sequence of 1792 rows takes 12 us, of which finding the work 3,
// the first pages 2.3, the products 1, fold and join 4.
// The subtracted maximum follows a row's scores with a slack of 8 (in log2): it is raised, and
// the accumulator rescaled, only when a score exceeds it by more, so that a block without
// such a score costs one vote instead of a maximum over its lanes; P stays below 2^8.
// Probabilities are rounded to bf16 for the second product (their sum is not); q, k and v
// are bf16 already.
constexpr int kThinWarps = 4;
constexpr int kThinThreads = kThinWarps * 32;
constexpr int kThinTile = kThinWarps * 16;
constexpr float kSlack = 8.f;

template <int HD, int NQ>
struct ThinLayout {
  static constexpr int kM = 8 * NQ;
  static constexpr int kHalf = 16 * HD * 2;                                 // 16 rows of K or V
  static constexpr int kStages = 5;
  static constexpr int kRing = kThinWarps * kStages * kHalf;
  static constexpr int kFoldCols = HD < 128 / NQ ? HD : 128 / NQ;           // columns folded at a time
  static constexpr int kFoldPitch = kFoldCols + 4;                          // floats: rows 2 t4 in banks 8 t4
  static constexpr int kFold = kThinWarps * kM * kFoldPitch * 4;
  static constexpr int kMl = kThinWarps * kM * 2 * 4;
  static constexpr int kQ = NQ > 2 ? kM * HD * 2 : 0;
  static constexpr int kSegB = kSegs * static_cast<int>(sizeof(Seg));
  static constexpr int kBytes = kRing + kFold + kMl + kQ + kSegB + kThinWarps * kStages * 8 + 1024;
};

// Row r, 16-byte chunk c of a 16-row block as TMA lays it: pieces of (up to) 64 elements, the
// chunk index mixed with the row so that eight rows of a chunk column fall into eight bank groups.
template <int HD>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  constexpr int C = HD / 8;
  if (C >= 8) return static_cast<uint32_t>((c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  if (C == 4) return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  return static_cast<uint32_t>(r * 32 + ((c ^ ((r >> 2) & 1)) << 4));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// What a warp had requested and not yet used when a wait of its ran out.
struct ThinLate {
  int slot, ahead;    // ring slots slot .. ahead-1, in order
  uint32_t phase;     // parity of each slot's copy
  uint32_t has_rows;  // by block: whether its halves were copied at all
  uint32_t block;     // of the first, which is
  int half;           // its K (0) or V (1) half
};

template <int HD, int NQ>
__global__ void __launch_bounds__(kThinThreads, 2)
attn_paged_thin_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const __grid_constant__ PagedAttnArgs a) {
  using L = ThinLayout<HD, NQ>;
  constexpr int KS = HD / 16, C = HD / 8;
  constexpr int M = L::kM;
  constexpr int S = L::kStages;
  constexpr bool KEEP = NQ == 1;  // the next segment's queries in registers
  extern __shared__ __align__(16) unsigned char thin_smem[];
  unsigned char *smem = thin_smem + ((1024u - (smem_u32(thin_smem) & 1023u)) & 1023u);
  unsigned char *at = smem + L::kRing;
  float *fold = reinterpret_cast<float *>(at);
  at += L::kFold;
  float *ml = reinterpret_cast<float *>(at);  // [warp][row][2]
  at += L::kMl;
  unsigned char *q_s = at;
  at += L::kQ;
  Seg *segs = reinterpret_cast<Seg *>(at);
  at += L::kSegB;
  uint64_t *bars = reinterpret_cast<uint64_t *>(at);  // [warp][stage]
  __shared__ PagedWalk walk;
  __shared__ ThinLate late[kThinWarps];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int G = gridDim.x, cta = blockIdx.x;
  if (tid < kThinWarps * S) {
    bar_init(bars + tid, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");  // a thread's own initialisations
  }
  if (tid == 0) {
    prefetch_map(&k_map);
    prefetch_map(&v_map);
  }
  pdl_wait();
  pdl_trigger();
  zero_unowned_rows<HD>(a, cta, G);
  int n_word = walk_begin(a, walk, segs);

  const uint32_t ring = smem_u32(smem) + warp * S * L::kHalf;
  uint64_t *bar = bars + warp * S;
  const uint32_t q_base = smem_u32(q_s);
  const int shift = a.c.page_shift;
  bool ok = true;       // this warp's copies have all arrived in time
  int slot = 0;         // ring slot of the half block consumed next
  int ahead = 0;        // ring slot requested next
  uint32_t phase = 0;   // parity of each slot's next completed copy

  while (n_word != 0) {
    const int n_now = n_word & (kMore - 1);
    // A segment's queries (where they fit registers next to the running ones) and the pages of
    // its first 32 tiles (lane i: this warp's block of tile t0 + i) are fetched one segment early.
    uint32_t qn[KEEP ? KS : 1][2];
    int n_ids = -1;
    auto q_row = [&](const Seg &g, int r) {
      const int token = token_of(a.p, g, r);
      return a.q + (g.r0 + token) * a.q_stride + head_of(a.p, g, r, token) * HD;
    };
    auto ids_of = [&](int seg, int t) {
      const int row = (t + lane) * kThinTile + warp * 16;
      if (t + lane < segs[seg].t1 && row < segs[seg].kv_end) {
        return __ldg(a.c.table + segs[seg].b * a.c.table_stride + (row >> shift));
      }
      return -1;
    };
    auto fetch_early = [&](int seg) {
      if (seg >= n_now) return;
      n_ids = ids_of(seg, segs[seg].t0);
      if (KEEP) {
        const Seg &g = segs[seg];
        const uint32_t *src = reinterpret_cast<const uint32_t *>(q_row(g, min(g8, g.rows - 1)));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qn[KEEP ? ks : 0][0] = __ldcg(src + ks * 8 + t4);
          qn[KEEP ? ks : 0][1] = __ldcg(src + ks * 8 + 4 + t4);
        }
      }
    };
    fetch_early(0);
    // The copies run ahead of the arithmetic over this batch of segments: the block of tile c_t of
    // segment c_s is requested next, its K half, then its V half. Lane i holds the page of this
    // warp's block of tile c_first + i.
    int c_s = 0, c_t = segs[0].t0, c_end = segs[0].t1;
    int c_kvh = segs[0].kvh, c_first = c_t, c_ids = n_ids, c_early = 0;  // c_early: the segment n_ids is of
    // whether the blocks requested and not yet used have rows at all (a block past the item's
    // end, or on a page outside the pool, has none and is not copied); bit: the block's number
    unsigned has_rows = 0, n_asked = 0, n_used = 0;
    int c_page = -1;
    auto copy = [&](const CUtensorMap *map) {
      const bool live = static_cast<unsigned>(c_page) < static_cast<unsigned>(a.c.n_pages) && ok;
      if (live && lane == 0) {
        const uint32_t dst = ring + ahead * L::kHalf;
        const int in_page = (c_t * kThinTile + warp * 16) & ((1 << shift) - 1);
        bar_expect(bar + ahead, L::kHalf);
#pragma unroll
        for (int h = 0; h < (HD > 64 ? HD / 64 : 1); ++h) {
          tma_page(dst + h * 2048, map, bar + ahead, h * 64, c_kvh, in_page, c_page);
        }
      }
      ahead = ahead + 1 == S ? 0 : ahead + 1;
      return live;
    };
    auto request_k = [&]() {
      if (c_s >= n_now) return;
      c_page = __shfl_sync(0xffffffffu, c_ids, c_t - c_first);
      const uint32_t bit = 1u << (n_asked & 31);
      has_rows = copy(&k_map) ? has_rows | bit : has_rows & ~bit;
      ++n_asked;
    };
    auto request_v = [&]() {  // of the same block, then on to the next one
      if (c_s >= n_now) return;
      copy(&v_map);
      if (++c_t == c_end && ++c_s < n_now) {
        c_t = segs[c_s].t0;
        c_end = segs[c_s].t1;
        c_kvh = segs[c_s].kvh;
        c_first = c_t - 32;
      }
      if (c_t - c_first == 32 && c_s < n_now) {
        c_first = c_t;
        c_ids = c_s == c_early && c_t == segs[c_s].t0 ? n_ids : ids_of(c_s, c_t);
      }
    };
    // The copy into the slot consumed next, of half `half` of the block in use (bounded; nothing is in
    // it when !live). Once a wait has run out, nothing is requested or computed any more.
    auto arrived = [&](bool live, int half) {
      if (live && ok) {
        ok = __all_sync(0xffffffffu, bar_poll(bar + slot, (phase >> slot) & 1u, a.polls));
        if (!ok) {
          ThinLate &l = late[warp];
          l.slot = slot;
          l.ahead = ahead;
          l.phase = phase;
          l.has_rows = has_rows;
          l.block = n_used - 1;
          l.half = half;
        }
        phase ^= 1u << slot;
      }
      return live && ok;
    };
    static_assert(S == 5, "two blocks ahead of the one in use");
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      request_k();
      request_v();
    }

    for (int si = 0; si < n_now; ++si) {
      const Seg g = segs[si];
      // ---- the item's queries as 8-column operands, zero past the last row ----
      uint32_t qf[NQ <= 2 ? NQ : 1][NQ <= 2 ? KS : 1][2];
      if (NQ <= 2) {
#pragma unroll
        for (int n = 0; n < (NQ <= 2 ? NQ : 1); ++n) {
          const int r = n * 8 + g8;
          const uint32_t *src = reinterpret_cast<const uint32_t *>(q_row(g, min(r, g.rows - 1)));
#pragma unroll
          for (int ks = 0; ks < (NQ <= 2 ? KS : 1); ++ks) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t v = KEEP ? qn[KEEP ? ks : 0][h] : __ldcg(src + ks * 8 + h * 4 + t4);
              qf[n][ks][h] = r < g.rows ? v : 0u;
            }
          }
        }
      } else {
        constexpr int kPer = M * C / kThinThreads > 0 ? M * C / kThinThreads : 1;
        uint4 v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int r = (tid + i * kThinThreads) / C, c = (tid + i * kThinThreads) % C;
          v[i] = ld_act16(q_row(g, min(r, g.rows - 1)) + c * 8);
          if (r >= g.rows) v[i] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int r = (tid + i * kThinThreads) / C, c = (tid + i * kThinThreads) % C;
          if (r < M) *reinterpret_cast<uint4 *>(q_s + (r >> 4) * L::kHalf + chunk_at<HD>(r & 15, c)) = v[i];
        }
        __syncthreads();
      }
      if (c_s <= si + 1) {  // the copies have not passed the next segment's start yet
        fetch_early(si + 1);
        c_early = si + 1;
      } else if (KEEP) {
        fetch_early(si + 1);
        c_early = -1;
      }
      // this thread's queries: n * 8 + 2 t4 and + 1
      int token[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = n * 8 + 2 * t4 + e;
          token[n][e] = token_of(a.p, g, min(r, g.rows - 1));
        }
      }
      const int seen_by_all = a.tree != nullptr ? g.base : g.base + g.tok0 + 1;
      float o[NQ][KS][4];  // O^T: element rows ks * 16 + g8 (+ 8), queries 2 t4 (+ 1)
      float m_run[NQ][2], l_run[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        m_run[n][0] = m_run[n][1] = -INFINITY;
        l_run[n][0] = l_run[n][1] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) o[n][ks][0] = o[n][ks][1] = o[n][ks][2] = o[n][ks][3] = 0.f;
      }

      for (int t = g.t0; t < g.t1; ++t) {
        const int row = t * kThinTile + warp * 16;
        bool live = (has_rows >> (n_used & 31)) & 1u;
        ++n_used;
        // a block that reaches beyond what all rows see is masked key by key: key j of queries 2 t4
        // and 2 t4 + 1 in bits j and 16 + j
        const bool masked = row + 16 > seen_by_all;
        uint32_t see[NQ];
        if (masked) seen16<NQ>(a, g, token, row, see);
        const uint32_t k_blk = ring + slot * L::kHalf;
        live = arrived(live, 0);
        slot = slot + 1 == S ? 0 : slot + 1;
        float s[NQ][4];  // keys g8 (0, 1) and g8 + 8 (2, 3) of the block, queries 2 t4, 2 t4 + 1
        if (live) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t k4[4];  // (rows 0-7, k 0-7), (rows 8-15, k 0-7), (rows 0-7, k 8-15), (rows 8-15, k 8-15)
            ldm_x4(k_blk + chunk_at<HD>(lane & 15, ks * 2 + (lane >> 4)), k4);
            if (NQ <= 2) {
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                mma_bf16(s[n], k4[0], k4[1], k4[2], k4[3], qf[NQ <= 2 ? n : 0][NQ <= 2 ? ks : 0][0],
                         qf[NQ <= 2 ? n : 0][NQ <= 2 ? ks : 0][1]);
              }
            } else {
#pragma unroll
              for (int n = 0; n < NQ; n += 2) {
                uint32_t q4[4];  // queries 0-7 then 8-15 of the pair, k 0-7 and 8-15 each
                ldm_x4(q_base + (n >> 1) * L::kHalf +
                           chunk_at<HD>((lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)), q4);
                mma_bf16(s[n], k4[0], k4[1], k4[2], k4[3], q4[0], q4[1]);
                mma_bf16(s[n + 1 < NQ ? n + 1 : n], k4[0], k4[1], k4[2], k4[3], q4[2], q4[3]);
              }
            }
          }
        }
        __syncwarp();
        request_k();  // into the slot freed a half block ago
        uint32_t p[NQ][2];
        if (live) {
          bool over = false;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              s[n][e] *= a.c2;
              s[n][e + 2] *= a.c2;
              if (masked) {
                const uint32_t m = see[n] >> (16 * e + g8);
                if ((m & 1u) == 0u) s[n][e] = -INFINITY;
                if ((m & 256u) == 0u) s[n][e + 2] = -INFINITY;
              }
              over |= fmaxf(s[n][e], s[n][e + 2]) > m_run[n][e] + kSlack;
            }
          }
          if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float mx = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                const float m_new = fmaxf(m_run[n][e], mx);
                const float alpha = m_new == -INFINITY ? 1.f : exp2f(m_run[n][e] - m_new);
                m_run[n][e] = m_new;
                l_run[n][e] *= alpha;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                  o[n][ks][e] *= alpha;
                  o[n][ks][e + 2] *= alpha;
                }
              }
            }
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float m = m_run[n][e & 1];
              x[e] = fast_exp2(s[n][e] - (m == -INFINITY ? 0.f : m));  // nothing seen so far: all -inf
              l_run[n][e & 1] += x[e];
            }
            p[n][0] = transpose8(mma_pack(x[0], x[1]));
            p[n][1] = transpose8(mma_pack(x[2], x[3]));
          }
        }
        const uint32_t v_blk = ring + slot * L::kHalf;
        live = arrived(live, 1);
        slot = slot + 1 == S ? 0 : slot + 1;
        if (live) {
          if (row + 16 > g.kv_end) {
            // rows behind the last may hold anything (0 x NaN): zeros for the product
            for (int i = lane; i < 16 * C; i += 32) {
              const int r = i / C;
              if (row + r >= g.kv_end) sts16(v_blk + chunk_at<HD>(r, i - r * C), make_uint4(0, 0, 0, 0));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          if (masked) {
            uint32_t bad = 0;
#pragma unroll
            for (int k = 0; k < (C + 1) / 2; ++k) {
              const int i = lane + k * 32;
              bad |= not_finite8(lds16(v_blk + chunk_at<HD>(i / C, i % C)));
            }
            if (__any_sync(0xffffffffu, bad != 0u)) {
#pragma unroll 1
              for (int j = 0; j < 16; ++j) {
                bool sees[NQ][2];
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
#pragma unroll
                  for (int e = 0; e < 2; ++e) sees[n][e] = (seen32(a, g, token[n][e], row) >> j) & 1u;
                }
#pragma unroll
                for (int c = 0; c < C; ++c) {
                  uint16_t u;
                  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(v_blk + chunk_at<HD>(j, c) + g8 * 2) : "memory");
                  const float x = __uint_as_float(static_cast<uint32_t>(u) << 16);
                  if (not_finite2(u) & 0x8000u) {
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
#pragma unroll
                      for (int e = 0; e < 2; ++e) {
                        if (sees[n][e]) o[n][c >> 1][e + 2 * (c & 1)] += x;
                      }
                    }
                  }
                }
              }
              __syncwarp();
#pragma unroll 1
              for (int i = lane; i < 16 * C; i += 32) {
                const uint32_t at16 = v_blk + chunk_at<HD>(i / C, i % C);
                sts16(at16, finite8(lds16(at16)));
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
            }
          }
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t v4[4];  // V^T: (d 0-7, key 0-7), (d 8-15, key 0-7), (d 0-7, key 8-15), (d 8-15, key 8-15)
            ldm_x4_trans(v_blk + chunk_at<HD>((lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)), v4);
#pragma unroll
            for (int n = 0; n < NQ; ++n) mma_bf16(o[n][ks], v4[0], v4[1], v4[2], v4[3], p[n][0], p[n][1]);
          }
        }
        __syncwarp();
        request_v();
      }

      // ---- fold the warps, kFoldCols columns at a time ----
      __syncthreads();  // the last segment's fold has been read
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float l = l_run[n][e];
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
          if (g8 == 0) {
            float *w = ml + (warp * M + n * 8 + 2 * t4 + e) * 2;
            w[0] = m_run[n][e];
            w[1] = l;
          }
        }
      }
      const PagedWs ws = ws_of(a, G);
      const long long part = (static_cast<long long>(cta) * 2 + g.slot) * M;
      constexpr int FC = L::kFoldCols;
      constexpr int kPerRow = FC / 4;                     // threads of a row, four columns each
      constexpr int kPass = kThinThreads / kPerRow;       // rows at a time
      constexpr int kPasses = (M + kPass - 1) / kPass;
      float weight[kPasses][kThinWarps], sum[kPasses], top[kPasses];
#pragma unroll
      for (int f = 0; f < HD / FC; ++f) {
        if (f > 0) __syncthreads();  // the last columns have been read
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
          for (int k = 0; k < FC / 16; ++k) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              fold[(warp * M + n * 8 + 2 * t4 + (e & 1)) * L::kFoldPitch + k * 16 + (e >> 1) * 8 + g8] = o[n][f * (FC / 16) + k][e];
            }
          }
        }
        __syncthreads();
        if (f == 0) {
#pragma unroll
          for (int i = 0; i < kPasses; ++i) {
            const int r = min(tid / kPerRow + i * kPass, M - 1);
            float2 x[kThinWarps];
            top[i] = -INFINITY;
#pragma unroll
            for (int w = 0; w < kThinWarps; ++w) {
              x[w] = *reinterpret_cast<const float2 *>(ml + (w * M + r) * 2);
              top[i] = fmaxf(top[i], x[w].x);
            }
            sum[i] = 0.f;
#pragma unroll
            for (int w = 0; w < kThinWarps; ++w) {
              weight[i][w] = fast_exp2(x[w].x - (top[i] == -INFINITY ? 0.f : top[i]));
              sum[i] = fmaf(weight[i][w], x[w].y, sum[i]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          const int r = tid / kPerRow + i * kPass, col = (tid % kPerRow) * 4;
          if (r >= g.rows) continue;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kThinWarps; ++w) {
            const float4 v = *reinterpret_cast<const float4 *>(fold + (w * M + r) * L::kFoldPitch + col);
            acc.x = fmaf(weight[i][w], v.x, acc.x);
            acc.y = fmaf(weight[i][w], v.y, acc.y);
            acc.z = fmaf(weight[i][w], v.z, acc.z);
            acc.w = fmaf(weight[i][w], v.w, acc.w);
          }
          if (g.whole) {
            const int tok = token_of(a.p, g, r), head = head_of(a.p, g, r, tok);
            const float by = sum[i] != 0.f ? 1.f / sum[i] : 0.f;
            __nv_bfloat16 *dst =
                a.out + (static_cast<long long>(g.r0 + tok) * a.p.n_kv * a.p.n_rep + head) * HD + f * FC + col;
            *reinterpret_cast<uint2 *>(dst) = make_uint2(mma_pack(acc.x * by, acc.y * by), mma_pack(acc.z * by, acc.w * by));
          } else {
            *reinterpret_cast<float4 *>(ws.o + (part + r) * HD + f * FC + col) = acc;
            if (f == 0 && col == 0) ws.ml[part + r] = make_float2(top[i], sum[i]);
          }
        }
      }
    }
    __syncthreads();
    if ((n_word & kMore) == 0) break;
    if (warp == 0) walk_on(a, walk, segs);
    __syncthreads();
    n_word = walk.n_segs;
    __syncthreads();
  }
  if (!ok) {
    // nothing leaves before the copies in flight have landed, each within the full limit
    if (lane == 0) atomicExch(&g_attn_paged_status, 20);
    __syncwarp();
    const ThinLate l = late[warp];
    int half = l.half;
    for (int s = l.slot; s != l.ahead; s = s + 1 == S ? 0 : s + 1, ++half) {
      if ((l.has_rows >> ((l.block + (half >> 1)) & 31)) & 1u) bar_poll(bar + s, (l.phase >> s) & 1u);
    }
  }
}

}  // namespace
}  // namespace chr

#include "paged_attn_wide.cuh"

namespace chr {
namespace {

// ---- joins the partials of items that CTA borders cut -------------------------------
// Block (x, y) looks at the descriptions of eight CTAs, a warp each, and joins every
// gridDim.y-th row from y on of the items they hold the start of: a warp per item where it lies
// in a few pieces, the whole block, its pieces dealt over the warps, where it lies in many.
// Bound by latency, three dependent reads of L2: 3 to 4 us. Four rows of a wide item at a time
// in a warp, their reads side by side, take 4.5 us; one after the other 6.5.
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kJoinFew = 16;
constexpr int kMaxCtas = 1024;   // pieces an item can lie in

__device__ __forceinline__ void join_store(const PagedAttnArgs &a, const PagedCut &cut, int r, int lane, float4 acc,
                                           float l) {
  if (lane * 4 >= a.c.hd) return;
  const int tok = (cut.row0 + r) / a.p.n_rep;
  const int head = cut.kvh * a.p.n_rep + (cut.row0 + r) - tok * a.p.n_rep;
  const float by = l != 0.f ? 1.f / l : 0.f;
  const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * by, acc.y * by);
  const __nv_bfloat162 hi = __floats2bfloat162_rn(acc.z * by, acc.w * by);
  *reinterpret_cast<uint2 *>(a.out + (static_cast<long long>(cut.r0 + tok) * a.p.n_kv * a.p.n_rep + head) * a.c.hd +
                             lane * 4) =
      make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
}

template <int kRows>
__global__ void __launch_bounds__(kJoinThreads) attn_paged_join_kernel(const PagedAttnArgs a, int G) {
  __shared__ PagedCut cuts[kJoinWarps];
  __shared__ float4 fold[kJoinWarps][32];
  __shared__ float red[2][kJoinWarps];
  __shared__ float weight[kMaxCtas];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hd = a.c.hd;
  pdl_trigger();
  pdl_wait();
  const PagedWs ws = ws_of(a, G);
  const int c = blockIdx.x * kJoinWarps + warp;
  PagedCut cut;
  cut.n = 0;
  if (c < G) {
    const int4 *src = reinterpret_cast<const int4 *>(ws.cut + c);
    const int4 d0 = __ldcg(src), d1 = __ldcg(src + 1);
    cut.n = d0.z;
    cut.kvh = d0.w;
    cut.row0 = d1.x;
    cut.rows = d1.y;
    cut.r0 = d1.z;
    cut.pad = c;  // its first piece
  }
  if (lane == 0) cuts[warp] = cut;
  // row r's partial in piece i: slot 1 of the first CTA, slot 0 of the others
  auto part = [&](const PagedCut &t, int i, int r) {
    return ((t.pad + i) * 2ll + (i == 0 ? 1 : 0)) * a.p.M + r;
  };
  // ... and its maximum and sum; a piece that was rounded away wrote none
  auto ml_of = [&](const PagedCut &t, int i, int r) {
    const int at = min(i, t.n - 1);
    const int live = __ldcg(&ws.cut[t.pad + at].live[at == 0 ? 1 : 0]);
    const float2 ml = __ldcg(ws.ml + part(t, at, r));
    return i < t.n && live != 0 ? ml : make_float2(-INFINITY, 0.f);
  };
  auto add = [&](float4 &acc, float w, long long at) {
    if (w != 0.f && lane * 4 < hd) {
      const float4 v = __ldcg(reinterpret_cast<const float4 *>(ws.o + at * hd) + lane);
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
    }
  };
  if (cut.n > 0 && cut.n <= kJoinFew) {
    // kRows rows at a time, so that their chains of loads run side by side
    for (int r0 = blockIdx.y; r0 < cut.rows; r0 += kRows * gridDim.y) {
      float w[kRows], l[kRows];
      float4 acc[kRows];
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const float2 ml = ml_of(cut, lane, min(r0 + k * static_cast<int>(gridDim.y), cut.rows - 1));
        w[k] = ml.x;
        l[k] = ml.y;
      }
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const float mm = warp_max_xor(w[k]);
        w[k] = w[k] == -INFINITY ? 0.f : fast_exp2(w[k] - mm);
        l[k] = warp_sum_xor(w[k] * l[k]);
        acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll(4 / kRows)
      for (int i = 0; i < cut.n; ++i) {
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          add(acc[k], __shfl_sync(0xffffffffu, w[k], i), part(cut, i, min(r0 + k * static_cast<int>(gridDim.y), cut.rows - 1)));
        }
      }
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int r = r0 + k * static_cast<int>(gridDim.y);
        if (r < cut.rows) join_store(a, cut, r, lane, acc[k], l[k]);
      }
    }
  }
  __syncthreads();
  for (int k = 0; k < kJoinWarps; ++k) {
    const PagedCut t = cuts[k];
    if (t.n <= kJoinFew) continue;
    for (int r = blockIdx.y; r < t.rows; r += gridDim.y) {
      float mm = -INFINITY, mine[kMaxCtas / kJoinThreads][2];
#pragma unroll
      for (int k2 = 0; k2 < kMaxCtas / kJoinThreads; ++k2) {
        const int i = tid + k2 * kJoinThreads;
        if (k2 * kJoinThreads < t.n) {
          const float2 ml = ml_of(t, i, r);
          mine[k2][0] = ml.x;
          mine[k2][1] = ml.y;
          mm = fmaxf(mm, ml.x);
        }
      }
      mm = warp_max_xor(mm);
      if (lane == 0) red[0][warp] = mm;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) mm = fmaxf(mm, red[0][w]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int k2 = 0; k2 < kMaxCtas / kJoinThreads; ++k2) {
        const int i = tid + k2 * kJoinThreads;
        if (i < t.n) {
          const float w = mine[k2][0] == -INFINITY ? 0.f : fast_exp2(mine[k2][0] - mm);
          l = fmaf(w, mine[k2][1], l);
          weight[i] = w;
        }
      }
      __syncthreads();
#pragma unroll 4
      for (int i = warp; i < t.n; i += kJoinWarps) add(acc, weight[i], part(t, i, r));
      l = warp_sum_xor(l);
      if (lane == 0) red[1][warp] = l;
      fold[warp][lane] = acc;
      __syncthreads();
      if (warp == 0) {
        l = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
          l += red[1][w];
          const float4 v = fold[w][lane];
          acc.x += v.x;
          acc.y += v.y;
          acc.z += v.z;
          acc.w += v.w;
        }
        join_store(a, t, r, lane, acc, l);
      }
      __syncthreads();
    }
  }
}

// A lane looks up to 32 tiles of 64 (one of 128) rows past an item's end: cache rows, and places
// that far behind them, are numbered in 32 bits.
constexpr long long kMaxRows = 0x7fffffffll - 8192;

// Limit of a wait, process-wide.
uint32_t &attn_paged_polls() {
  static uint32_t v = kPolls;
  return v;
}

struct AttnForm {
  int M, tile, extra, ctas;
};
// The form of a call: from the head layout and the mean number of new rows per sequence,
// which the host knows, never from the lengths, which it does not.
AttnForm form_of(int T, int batch, int n_rep, int hd) {
  // Items as low as the rows allow: 64 sequences of 5 rows per kv head take 88 us with items of 8,
  // 117 with 32. Above 32 rows the wide form: 16 trees of 35 rows take 70 us with it, 130 with thin
  // items of 32; of 255 rows 102 and 455. From 17 to 32 rows it is a draw: 20 rows, 16 sequences of
  // 2100 to 6000 cache rows 67 wide and 75 thin, two such 31.6 and 28.4, 32 of 100 to 900
  // 42 and 37.
  // The mean is of all sequences, so a call that mixes a long chunk with single tokens or with
  // sequences without rows takes one form for both: a chunk of 256 rows (45 us alone) in a batch of 64 that
  // has no other rows takes 70 in the thin form; one of 512 beside 63 tokens (46 and 54 alone) 109 in the
  // wide one; one of 1024 beside 255 tokens (58 and 165 alone) 388 in the thin one.
  const long long rows = (static_cast<long long>(T) + batch - 1) / batch * n_rep;
  const int sms = std::min(sm_count(), kMaxCtas / 2);
  AttnForm f;
  if (rows > 32 && (hd == 64 || hd == 128)) {
    f.M = kWideM;
    f.tile = kWideTile;
    // Queries in, result out, in rows: 16 trees of 32 drafts take 96.8 us with 4 tiles, 97.1 with 2,
    // 98.8 with 1.
    f.extra = 4 * kWideTile;
    f.ctas = sms;  // one resident CTA per SM
    return f;
  }
  f.M = rows <= 8 ? 8 : (rows <= 16 ? 16 : 32);
  f.tile = kThinTile;
  // What starting and folding a segment takes, in rows: 64 sequences take 87.7 us with 3 tiles,
  // 95.6 with 1, 87.9 with 6.
  f.extra = 3 * kThinTile;
  // Two resident CTAs per SM. (Three to eight, so that an SM that is served faster takes more
  // of them, cost more in starts than they balance: 64 sequences 110 us against 108.)
  f.ctas = 2 * sms;
  return f;
}

using TensorMapEncode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                     const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                     CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                     CUtensorMapFloatOOBfill);
TensorMapEncode tensor_map_encode() {
  static TensorMapEncode fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      return static_cast<TensorMapEncode>(nullptr);
    }
    return reinterpret_cast<TensorMapEncode>(p);
  }();
  return fn;
}

bool head_dim_ok(int hd) { return hd == 16 || hd == 32 || hd == 64 || hd == 128; }

// The pools as [page][row][kv head][element]; a copy is one head's (up to) 64 elements of
// `rows` rows of a page, laid out with the swizzle the matrix loads expect.
bool pool_maps(const PagedCache &c, int rows, CUtensorMap (&maps)[2]) {
  TensorMapEncode enc = tensor_map_encode();
  if (enc == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.hd), static_cast<cuuint64_t>(c.n_kv),
                              static_cast<cuuint64_t>(1) << c.page_shift, static_cast<cuuint64_t>(c.n_pages)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(std::min(c.hd, 64)), 1, static_cast<cuuint32_t>(rows), 1};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  const CUtensorMapSwizzle swizzle = c.hd >= 64 ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : c.hd == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  for (int i = 0; i < 2; ++i) {
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(c.hd) * 2, static_cast<cuuint64_t>(c.n_kv) * c.hd * 2,
                                   static_cast<cuuint64_t>(i == 0 ? c.k_page_stride : c.v_page_stride) * 2};
    if (enc(&maps[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, i == 0 ? c.k : c.v, dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
      return false;
    }
  }
  return true;
}

template <int HD, int NQ>
cudaError_t launch_thin(const PagedAttnArgs &a, int ctas, cudaStream_t st) {
  static int done[64] = {};
  CUtensorMap maps[2];
  if (!ensure_smem_attr(attn_paged_thin_kernel<HD, NQ>, ThinLayout<HD, NQ>::kBytes, done) ||
      !pool_maps(a.c, 16, maps)) {
    return cudaErrorInvalidValue;
  }
  return launch_chain(attn_paged_thin_kernel<HD, NQ>, dim3(static_cast<unsigned>(ctas)), dim3(kThinThreads),
                      ThinLayout<HD, NQ>::kBytes, st, maps[0], maps[1], a);
}
template <int HD>
cudaError_t launch_thin_hd(const PagedAttnArgs &a, int ctas, cudaStream_t st) {
  switch (a.p.M) {
    case 8: return launch_thin<HD, 1>(a, ctas, st);
    case 16: return launch_thin<HD, 2>(a, ctas, st);
    default: return launch_thin<HD, 4>(a, ctas, st);
  }
}

template <int HD>
cudaError_t launch_wide(const PagedAttnArgs &a, int negate, int ctas, cudaStream_t st) {
  static int done[64] = {};
  CUtensorMap maps[2];
  if (!ensure_smem_attr(attn_paged_wide_kernel<HD>, WideLayout<HD>::kBytes, done) ||
      !pool_maps(a.c, std::min(1 << a.c.page_shift, kWideTile), maps)) {
    return cudaErrorInvalidValue;
  }
  return launch_chain(attn_paged_wide_kernel<HD>, dim3(static_cast<unsigned>(ctas)), dim3(kWideThreads),
                      WideLayout<HD>::kBytes, st, maps[0], maps[1], a, negate);
}

}  // namespace
}  // namespace chr

using namespace chr;

extern "C" void chr_nf4_set_attn_paged_polls(int32_t polls) {
  attn_paged_polls() = polls < 0 ? kPolls : static_cast<uint32_t>(polls);
}

extern "C" int64_t chr_nf4_attn_paged_ws(int32_t T, int32_t batch, int32_t n_q, int32_t n_kv,
                                         int32_t hd) {
  if (T < 1 || batch < 1 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0 || !head_dim_ok(hd)) return 0;
  const AttnForm f = form_of(T, batch, n_q / n_kv, hd);
  return ws_floats_of(f.ctas, f.M, hd);
}

extern "C" int chr_nf4_attn_paged(const chr_nf4_attn_paged_t *args, void *stream) {
  if (args == nullptr) return kNull;
  const chr_nf4_attn_paged_t &r = *args;
  if (r.q == nullptr || r.out == nullptr || r.kv_len == nullptr || r.ws == nullptr) {
    return kNull;
  }
  PagedAttnArgs a{};
  const int rc = paged_cache(&r.pages, a.c);
  if (rc != kOk) return rc;
  const int hd = a.c.hd;
  if (r.T < 1 || r.n_q < 1 || r.n_q % a.c.n_kv != 0 || !head_dim_ok(hd) ||
      r.q_stride < static_cast<int64_t>(r.n_q) * hd || (r.tree != nullptr && (r.tree_words < 1 || r.tree_words > (1 << 24))) ||
      !std::isfinite(r.scale) || (r.q_start == nullptr && r.T != a.c.batch) ||
      static_cast<int64_t>(r.T) * r.n_q > 0x3fffffffll || r.n_q > 65536) {
    return kDims;
  }
  if (!aligned(r.q, 16) || !aligned(r.out, 16) || !aligned(r.ws, 16) || r.q_stride % 8 != 0 || !aligned(a.c.k, 16) ||
      !aligned(a.c.v, 16) || a.c.k_page_stride % 8 != 0 || a.c.v_page_stride % 8 != 0 ||
      (r.tree != nullptr && !aligned(r.tree, 8))) {
    return kAlign;
  }
  const int n_rep = r.n_q / a.c.n_kv;
  const long long cap = static_cast<long long>(a.c.max_pages) << a.c.page_shift;
  if (cap > kMaxRows) return kDims;
  a.p.cap = static_cast<int>(cap);
  const AttnForm f = form_of(r.T, a.c.batch, n_rep, hd);
  if (r.ws_floats < ws_floats_of(f.ctas, f.M, hd)) return kWorkspace;
  a.p.q_start = static_cast<const int32_t *>(r.q_start);
  a.p.kv_len = static_cast<const int32_t *>(r.kv_len);
  a.p.T = r.T;
  a.p.batch = a.c.batch;
  a.p.n_kv = a.c.n_kv;
  a.p.n_rep = n_rep;
  a.p.M = f.M;
  a.p.tile = f.tile;
  a.p.extra = f.extra;
  a.p.per_rep = 1.f / static_cast<float>(n_rep);
  a.p.causal = r.tree == nullptr;
  // places on the axis are whole numbers that binary64 holds exactly
  const double items = static_cast<double>(r.T) * r.n_q / f.M + static_cast<double>(a.c.batch) * a.c.n_kv;
  if (items * (static_cast<double>(a.p.cap) + f.extra) * n_rep > 4.0e15) return kDims;
  a.q = static_cast<const __nv_bfloat16 *>(r.q);
  a.out = static_cast<__nv_bfloat16 *>(r.out);
  a.tree = static_cast<const unsigned long long *>(r.tree);
  a.ws = r.ws;
  a.q_stride = r.q_stride;
  a.tree_words = r.tree_words;
  a.zero_tail = r.zero_tail != 0;
  a.c2 = r.scale * 1.4426950408889634f;
  a.polls = attn_paged_polls();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (f.M == kWideM) {
    // the sign of the scale goes into the product, so that the maximum of the products is
    // that of the scores; no scale at all would make a hidden row 0 x -inf
    a.c2 = std::max(std::fabs(a.c2), 1e-30f);
    const int negate = r.scale < 0.f;
    e = hd == 64 ? launch_wide<64>(a, negate, f.ctas, st) : launch_wide<128>(a, negate, f.ctas, st);
  } else {
    switch (hd) {
      case 16: e = launch_thin_hd<16>(a, f.ctas, st); break;
      case 32: e = launch_thin_hd<32>(a, f.ctas, st); break;
      case 64: e = launch_thin_hd<64>(a, f.ctas, st); break;
      default: e = launch_thin_hd<128>(a, f.ctas, st); break;
    }
  }
  if (e != cudaSuccess) return kLaunch;
  // a row per warp, or four where items have many
  const unsigned eights = static_cast<unsigned>((f.ctas + kJoinWarps - 1) / kJoinWarps);
  if (f.M == kWideM) {
    e = launch_chain(attn_paged_join_kernel<4>, dim3(eights, kWideM / 4), dim3(kJoinThreads), 0, st, a, f.ctas);
  } else {
    e = launch_chain(attn_paged_join_kernel<1>, dim3(eights, f.M), dim3(kJoinThreads), 0, st, a, f.ctas);
  }
  return e == cudaSuccess ? kOk : kLaunch;
}

extern "C" int chr_nf4_attn_paged_status(void) {
  int v = 0;
  const int zero = 0;
  if (cudaDeviceSynchronize() != cudaSuccess ||
      cudaMemcpyFromSymbol(&v, g_attn_paged_status, sizeof v) != cudaSuccess ||
      cudaMemcpyToSymbol(g_attn_paged_status, &zero, sizeof zero) != cudaSuccess) {
    return kLaunch;
  }
  return v;
}
