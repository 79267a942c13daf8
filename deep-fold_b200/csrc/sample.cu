// One token per row drawn from bf16 logits (sm_100a): temperature, top-k, top-p, min-p and
// a given uniform number, then the commit of the batched greedy pick. No counterpart in
// the reference, which picks the argmax (gpu/decodev2/step.py:182).
//
// Mathematics. With tokens ordered by (logit descending, index ascending), every filter
// keeps a prefix of the order, so a row's draw is: the length n' of the kept prefix, its
// mass cum(n'), and the place of u * cum(n') in the running sum. A bf16 logit takes one of
// 65536 values, and tokens of one value have one weight. So the row is turned into a
// histogram over the values (exact: integers), and everything else - sums, cuts and the
// draw - is done on (count, exp) pairs of the few thousand values that occur, in 64-bit
// floating point. No sort, no sum over the vocabulary, the same result in every run.
//
// A cluster of C CTAs owns a row. Each CTA counts its slice of the vocabulary in its own
// shared memory (65536 16-bit counters, 128 KB; a slice is at most 65535 tokens), the
// clusters' histograms are read through distributed shared memory: 1024 chunks of 64
// values get their count and mass, one CTA scans the chunks and walks the three cuts and
// the draw, and the CTA whose slice holds the token finds its index. One launch, no
// scratch memory.

#include <cooperative_groups.h>

#include "nf4_common.cuh"

namespace chr {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kKeys = 65536;
constexpr int kChunk = 64;                 // values per chunk
constexpr int kChunks = kKeys / kChunk;
constexpr int kSampleMaxCluster = 8;
constexpr int kSliceMax = 65535;           // a 16-bit counter never wraps

struct SampleArgs {
  const __nv_bfloat16 *logits;
  long long row_stride;
  int n, batch, slice;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t *top_k;
  float *prob;
  int64_t *next_token, *token, *position;
  uint8_t *finished;
  int64_t eos;
};

struct SampleShared {
  uint32_t hist[kKeys / 2];          // counters 2i (low half) and 2i + 1 (high half)
  double mass[kChunks];              // rank 0: chunk masses, then what lies before each chunk
  uint32_t count[kChunks];
  double part_mass[kSampleWarps];
  uint32_t part_count[kSampleWarps];
  uint32_t warp_max[kSampleWarps];
  uint32_t max_key;                  // of this CTA's slice
  // the draw, written by rank 0 into every CTA
  uint32_t pick_key, pick_rank;      // value and its pick_rank-th occurrence
  float pick_prob;
  uint32_t found[kSampleWarps];
};

// bf16 bits -> a key that orders as the value does (-0 as +0, NaN above everything).
__device__ __forceinline__ uint32_t order_key(uint32_t b) {
  if ((b & 0x7FFFu) > 0x7F80u) return 0xFFFFu;
  if (b == 0x8000u) b = 0u;
  return (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  const uint32_t b = (k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu);
  return __uint_as_float(b << 16);
}

// exp((value - max) / T), the weight of every token of one value
__device__ __forceinline__ double key_weight(uint32_t key, double m, double temp) {
  return exp((static_cast<double>(key_value(key)) - m) / temp);
}

// Calls f(index, bf16 bits) for the elements lo..hi of a row that this thread owns, 16
// bytes at a time where the row's alignment allows.
template <typename F>
__device__ __forceinline__ void for_slice(const __nv_bfloat16 *row, int lo, int hi, F f) {
  const unsigned short *x = reinterpret_cast<const unsigned short *>(row);
  const uintptr_t at = reinterpret_cast<uintptr_t>(x + lo);
  const int head = min(static_cast<int>(((16 - (at & 15)) & 15) >> 1), hi - lo);
  const int n8 = (hi - lo - head) >> 3;
  for (int i = threadIdx.x; i < head; i += kSampleThreads) f(lo + i, __ldcg(x + lo + i));
  const uint4 *body = reinterpret_cast<const uint4 *>(x + lo + head);
#pragma unroll 4
  for (int i = threadIdx.x; i < n8; i += kSampleThreads) {
    const uint4 v = __ldcg(body + i);
    const int at0 = lo + head + i * 8;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f(at0 + 2 * e, w[e] & 0xFFFFu);
      f(at0 + 2 * e + 1, w[e] >> 16);
    }
  }
  for (int i = lo + head + n8 * 8 + threadIdx.x; i < hi; i += kSampleThreads) f(i, __ldcg(x + i));
}

// The counts of chunk c over the cluster, two values per lane in descending order: lane l
// holds the values c*64 + 63 - 2l (hi) and c*64 + 62 - 2l (lo).
__device__ __forceinline__ void chunk_counts(cg::cluster_group &cluster, SampleShared &sm, int c,
                                             int lane, uint32_t &hi, uint32_t &lo) {
  const int word = c * (kChunk / 2) + 31 - lane;
  uint32_t v[kSampleMaxCluster];
  const int C = static_cast<int>(cluster.num_blocks());
#pragma unroll
  for (int r = 0; r < kSampleMaxCluster; ++r) {
    v[r] = r < C ? *cluster.map_shared_rank(&sm.hist[word], r) : 0u;
  }
  hi = lo = 0u;
#pragma unroll
  for (int r = 0; r < kSampleMaxCluster; ++r) {
    hi += v[r] >> 16;
    lo += v[r] & 0xFFFFu;
  }
}

__device__ __forceinline__ double shfl_up(double v, int off) { return __shfl_up_sync(0xffffffffu, v, off); }

// What a warp knows of one chunk: counts, weights and what lies before each value.
struct ChunkView {
  uint32_t n_hi, n_lo, before_hi, before_lo;  // tokens before the lane's two values
  double w_hi, w_lo, mass_hi, mass_lo;        // weights; mass before the two values
};
__device__ __forceinline__ ChunkView view_chunk(cg::cluster_group &cluster, SampleShared &sm, int c,
                                                int lane, double m, double temp) {
  ChunkView v;
  chunk_counts(cluster, sm, c, lane, v.n_hi, v.n_lo);
  const uint32_t key = static_cast<uint32_t>(c * kChunk + 63 - 2 * lane);
  v.w_hi = v.n_hi != 0u ? key_weight(key, m, temp) : 0.0;
  v.w_lo = v.n_lo != 0u ? key_weight(key - 1u, m, temp) : 0.0;
  uint32_t cnt = v.n_hi + v.n_lo;
  double mass = v.n_hi * v.w_hi + v.n_lo * v.w_lo;
  const uint32_t own_c = cnt;
  const double own_m = mass;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t oc = __shfl_up_sync(0xffffffffu, cnt, off);
    const double om = shfl_up(mass, off);
    if (lane >= off) {
      cnt += oc;
      mass += om;
    }
  }
  double prev = shfl_up(mass, 1);
  if (lane == 0) prev = 0.0;
  (void)own_m;
  v.before_hi = sm.count[c] + cnt - own_c;
  v.before_lo = v.before_hi + v.n_hi;
  v.mass_hi = sm.mass[c] + prev;
  v.mass_lo = v.mass_hi + v.n_hi * v.w_hi;
  return v;
}

// The last chunk, in descending order of value, before which no more than `count` tokens
// (or mass) lie. Chunk c's entry holds what lies before it; c = 1023 comes first.
template <typename T>
__device__ __forceinline__ int last_chunk(const T *before, T limit, int lane) {
  // 32 groups of 32 chunks
  const unsigned ga = __ballot_sync(0xffffffffu, before[kChunks - 1 - lane * 32] <= limit);
  const int g = 31 - __clz(ga | 1u);
  const unsigned gb = __ballot_sync(0xffffffffu, before[kChunks - 1 - (g * 32 + lane)] <= limit);
  return kChunks - 1 - (g * 32 + 31 - __clz(gb | 1u));
}

// Value and rank within it of the token with `rank` tokens before it; mass before the
// value. Called by a whole warp; every lane gets the result.
struct Token {
  uint32_t key, in;   // value, occurrences of it before the token
  double mass, w;     // mass before the value, weight
};
__device__ __forceinline__ Token token_at(cg::cluster_group &cluster, SampleShared &sm, uint32_t rank,
                                          int lane, double m, double temp) {
  const int c = last_chunk(sm.count, rank, lane);
  const ChunkView v = view_chunk(cluster, sm, c, lane, m, temp);
  const bool in_hi = v.n_hi != 0u && rank >= v.before_hi && rank < v.before_hi + v.n_hi;
  const bool in_lo = v.n_lo != 0u && rank >= v.before_lo && rank < v.before_lo + v.n_lo;
  const unsigned who = __ballot_sync(0xffffffffu, in_hi || in_lo);
  const int from = __ffs(who | 0x80000000u) - 1;
  const uint32_t base = static_cast<uint32_t>(c * kChunk + 63 - 2 * lane);
  Token t;
  t.key = __shfl_sync(0xffffffffu, in_hi ? base : base - 1u, from);
  t.in = __shfl_sync(0xffffffffu, rank - (in_hi ? v.before_hi : v.before_lo), from);
  t.mass = __shfl_sync(0xffffffffu, in_hi ? v.mass_hi : v.mass_lo, from);
  t.w = __shfl_sync(0xffffffffu, in_hi ? v.w_hi : v.w_lo, from);
  return t;
}

// The first token after which the running mass exceeds `r` (strict) or reaches it: its
// value's first rank, its count, the mass before the value and the weight.
struct Crossing {
  uint32_t key, before, n;
  double mass, w;
};
__device__ __forceinline__ Crossing crossing(cg::cluster_group &cluster, SampleShared &sm, double r,
                                             bool strict, int lane, double m, double temp) {
  // the last chunk with no more than r (strict: the crossing token has cum > r) before it;
  // when the cum has to reach r only, the last with less than r before it
  int c;
  if (strict) {
    c = last_chunk(sm.mass, r, lane);
  } else {
    const unsigned ga = __ballot_sync(0xffffffffu, sm.mass[kChunks - 1 - lane * 32] < r || lane == 0);
    const int g = 31 - __clz(ga);
    const unsigned gb =
        __ballot_sync(0xffffffffu, sm.mass[kChunks - 1 - (g * 32 + lane)] < r || lane == 0);
    c = kChunks - 1 - (g * 32 + 31 - __clz(gb));
  }
  const ChunkView v = view_chunk(cluster, sm, c, lane, m, temp);
  const double end_hi = v.mass_hi + v.n_hi * v.w_hi, end_lo = v.mass_lo + v.n_lo * v.w_lo;
  const bool hi = v.n_hi != 0u && (strict ? end_hi > r : end_hi >= r);
  const bool lo = v.n_lo != 0u && (strict ? end_lo > r : end_lo >= r);
  unsigned who = __ballot_sync(0xffffffffu, hi || lo);
  // rounding may leave the chunk's end short of r: its last value then
  const unsigned any = __ballot_sync(0xffffffffu, v.n_hi != 0u || v.n_lo != 0u);
  const bool none = who == 0u;
  const int from = none ? 31 - __clz(any | 1u) : __ffs(who) - 1;
  const bool take_hi = none ? v.n_lo == 0u : hi;
  const uint32_t base = static_cast<uint32_t>(c * kChunk + 63 - 2 * lane);
  Crossing x;
  x.key = __shfl_sync(0xffffffffu, take_hi ? base : base - 1u, from);
  x.before = __shfl_sync(0xffffffffu, take_hi ? v.before_hi : v.before_lo, from);
  x.n = __shfl_sync(0xffffffffu, take_hi ? v.n_hi : v.n_lo, from);
  x.mass = __shfl_sync(0xffffffffu, take_hi ? v.mass_hi : v.mass_lo, from);
  x.w = __shfl_sync(0xffffffffu, take_hi ? v.w_hi : v.w_lo, from);
  return x;
}

__global__ void __launch_bounds__(kSampleThreads, 1) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char sample_smem[];
  SampleShared &sm = *reinterpret_cast<SampleShared *>(sample_smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / C;
  pdl_trigger();
  for (int i = tid; i < kKeys / 8; i += kSampleThreads) {
    reinterpret_cast<uint4 *>(sm.hist)[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  pdl_wait();
  const __nv_bfloat16 *row = a.logits + b * a.row_stride;
  const int lo = min(rank * a.slice, a.n), hi = min(lo + a.slice, a.n);

  // ---- the slice's histogram and maximum ----
  uint32_t top = 0u;
  for_slice(row, lo, hi, [&](int, uint32_t bits) {
    const uint32_t key = order_key(bits);
    top = max(top, key);
    atomicAdd(&sm.hist[key >> 1], (key & 1u) ? 65536u : 1u);
  });
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) sm.warp_max[warp] = top;
  __syncthreads();
  if (warp == 0) {
    const uint32_t v = __reduce_max_sync(0xffffffffu, lane < kSampleWarps ? sm.warp_max[lane] : 0u);
    if (lane == 0) sm.max_key = v;
  }
  cluster.sync();

  uint32_t max_key = 0u;
  for (int r = 0; r < C; ++r) max_key = max(max_key, *cluster.map_shared_rank(&sm.max_key, r));
  const float temp_f = a.temperature != nullptr ? __ldg(a.temperature + b) : 1.f;
  const float max_f = key_value(max_key);
  // max_key of NaN is 0xFFFF; +inf and -inf are not finite either
  const bool greedy = !(temp_f > 0.f) || max_key == 0xFFFFu || isinf(max_f);
  const double m = max_f, temp = temp_f;

  uint32_t pick_key = max_key, pick_rank = 0u;
  float pick_prob = 1.f;
  if (!greedy) {
    // ---- count and mass of every chunk, to rank 0 ----
    SampleShared *lead = cluster.map_shared_rank(&sm, 0);
    for (int i = warp; i * C + rank < kChunks; i += kSampleWarps) {
      const int c = i * C + rank;
      uint32_t n_hi, n_lo;
      chunk_counts(cluster, sm, c, lane, n_hi, n_lo);
      double mass = 0.0;
      uint32_t cnt = 0u;
      if (__any_sync(0xffffffffu, (n_hi | n_lo) != 0u)) {
        const uint32_t key = static_cast<uint32_t>(c * kChunk + 63 - 2 * lane);
        if (n_hi != 0u) mass = n_hi * key_weight(key, m, temp);
        if (n_lo != 0u) mass += n_lo * key_weight(key - 1u, m, temp);
        cnt = __reduce_add_sync(0xffffffffu, n_hi + n_lo);
        // the order of view_chunk's running sum
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const double o = shfl_up(mass, off);
          if (lane >= off) mass += o;
        }
      }
      if (lane == 31) {
        lead->mass[c] = mass;
        lead->count[c] = cnt;
      }
    }
    cluster.sync();
    if (rank == 0) {
      // ---- what lies before each chunk, in descending order of value ----
      constexpr int kPer = kChunks / kSampleThreads;
      double mv[kPer], run = 0.0;
      uint32_t cv[kPer], run_c = 0u;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = kChunks - 1 - (tid * kPer + i);
        mv[i] = run;
        cv[i] = run_c;
        run += sm.mass[c];
        run_c += sm.count[c];
      }
      double incl = run;
      uint32_t incl_c = run_c;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const double o = shfl_up(incl, off);
        const uint32_t oc = __shfl_up_sync(0xffffffffu, incl_c, off);
        if (lane >= off) {
          incl += o;
          incl_c += oc;
        }
      }
      double prev = shfl_up(incl, 1);
      uint32_t prev_c = __shfl_up_sync(0xffffffffu, incl_c, 1);
      if (lane == 0) {
        prev = 0.0;
        prev_c = 0u;
      }
      if (lane == 31) {
        sm.part_mass[warp] = incl;
        sm.part_count[warp] = incl_c;
      }
      __syncthreads();
      double at = 0.0;
      uint32_t at_c = 0u;
      for (int w = 0; w < warp; ++w) {
        at += sm.part_mass[w];
        at_c += sm.part_count[w];
      }
      double total = 0.0;
      for (int w = 0; w < kSampleWarps; ++w) total += sm.part_mass[w];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = kChunks - 1 - (tid * kPer + i);
        sm.mass[c] = at + prev + mv[i];
        sm.count[c] = at_c + prev_c + cv[i];
      }
      __syncthreads();
      if (warp == 0) {
        // ---- the kept prefix ----
        const uint32_t n = static_cast<uint32_t>(a.n);
        uint32_t keep = n;
        double sum = total;
        const int k = a.top_k != nullptr ? __ldg(a.top_k + b) : 0;
        if (k > 0 && static_cast<uint32_t>(k) < n) {
          keep = static_cast<uint32_t>(k);
          const Token t = token_at(cluster, sm, keep - 1u, lane, m, temp);
          sum = t.mass + (t.in + 1u) * t.w;
        }
        const float p = a.top_p != nullptr ? __ldg(a.top_p + b) : 1.f;
        uint32_t kept = keep;
        if (p < 1.f) {
          const double target = static_cast<double>(p) * sum;
          uint32_t np = 1u;
          if (target > 0.0) {
            const Crossing x = crossing(cluster, sm, target, false, lane, m, temp);
            // of the crossing value's tokens those before which the sum is below the target
            double q = x.w > 0.0 ? ceil((target - x.mass) / x.w) : 1.0;
            q = fmin(fmax(q, 1.0), static_cast<double>(x.n));
            np = x.before + static_cast<uint32_t>(q);
          }
          kept = min(kept, np);
        }
        const float least = a.min_p != nullptr ? __ldg(a.min_p + b) : 0.f;
        if (least > 0.f) {
          // the lowest value whose weight is still min_p: 32-way search over the values
          uint32_t lo_k = 0u, hi_k = max_key;  // weight(hi_k) = 1
          uint32_t nm = 1u;
          if (least <= 1.f) {
            while (lo_k < hi_k) {
              const uint32_t step = (hi_k - lo_k + 31u) / 32u;
              const uint32_t key = min(lo_k + step * lane, hi_k);
              const bool ok = key_weight(key, m, temp) >= static_cast<double>(least);
              const unsigned yes = __ballot_sync(0xffffffffu, ok);
              if (yes == 0u) {          // only hi_k itself may do
                lo_k = min(lo_k + step * 31u + 1u, hi_k);
              } else {
                const int f = __ffs(yes) - 1;
                const uint32_t found = min(lo_k + step * f, hi_k);
                lo_k = f == 0 ? lo_k : min(lo_k + step * (f - 1) + 1u, found);
                hi_k = found;
              }
            }
            // tokens of value hi_k and above
            const int c = static_cast<int>(hi_k / kChunk);
            const ChunkView v = view_chunk(cluster, sm, c, lane, m, temp);
            const uint32_t key = static_cast<uint32_t>(c * kChunk + 63 - 2 * lane);
            const uint32_t here = (key >= hi_k ? v.n_hi : 0u) + (key - 1u >= hi_k ? v.n_lo : 0u);
            nm = sm.count[c] + __reduce_add_sync(0xffffffffu, here);
          }
          kept = min(kept, nm);
        }
        kept = max(kept, 1u);
        if (kept != keep) {
          const Token t = token_at(cluster, sm, kept - 1u, lane, m, temp);
          sum = t.mass + (t.in + 1u) * t.w;
        }
        // ---- the draw ----
        const float uf = fminf(fmaxf(__ldg(a.u + b), 0.f), 0.99999994f);  // NaN: 0
        const double r = static_cast<double>(uf) * sum;
        const Crossing x = crossing(cluster, sm, r, true, lane, m, temp);
        double q = x.w > 0.0 ? floor((r - x.mass) / x.w) : 0.0;
        q = fmin(fmax(q, 0.0), static_cast<double>(x.n - 1u));
        uint32_t in = static_cast<uint32_t>(q), key = x.key;
        double w = x.w;
        if (x.before + in >= kept) {  // rounding took the draw past the last kept token
          const Token t = token_at(cluster, sm, kept - 1u, lane, m, temp);
          key = t.key;
          in = t.in;
          w = t.w;
        }
        if (lane < C) {
          SampleShared *to = cluster.map_shared_rank(&sm, lane);
          to->pick_key = key;
          to->pick_rank = in;
          to->pick_prob = static_cast<float>(w / sum);
        }
      }
    }
    cluster.sync();
    pick_key = sm.pick_key;
    pick_rank = sm.pick_rank;
    pick_prob = sm.pick_prob;
  }

  // ---- the pick_rank-th token of value pick_key, in order of index ----
  const int shift = (pick_key & 1u) ? 16 : 0;
  uint32_t before = 0u;
  for (int r = 0; r < rank; ++r) {
    before += (*cluster.map_shared_rank(&sm.hist[pick_key >> 1], r) >> shift) & 0xFFFFu;
  }
  const uint32_t here = (sm.hist[pick_key >> 1] >> shift) & 0xFFFFu;
  if (pick_rank >= before && pick_rank < before + here) {
    const uint32_t want = pick_rank - before;  // occurrence within the slice
    const unsigned short *x = reinterpret_cast<const unsigned short *>(row);
    // a warp's part of the slice, in order of index
    const int per = (hi - lo + kSampleWarps - 1) / kSampleWarps;
    const int w0 = min(lo + warp * per, hi), w1 = min(w0 + per, hi);
    uint32_t mine = 0u;
    for (int i = w0 + lane; i < w1; i += 32) mine += order_key(__ldcg(x + i)) == pick_key ? 1u : 0u;
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sm.found[warp] = mine;
    __syncthreads();
    uint32_t skip = 0u;
    for (int w = 0; w < warp; ++w) skip += sm.found[w];
    if (want >= skip && want < skip + mine) {
      uint32_t left = want - skip;
      for (int i = w0; i < w1; i += 32) {
        const bool is = i + lane < w1 && order_key(__ldcg(x + i + lane)) == pick_key;
        const unsigned hit = __ballot_sync(0xffffffffu, is);
        const uint32_t cnt = __popc(hit);
        if (left < cnt) {
          const unsigned upto = hit & ((2u << lane) - 1u);  // (2 << 31) - 1: all lanes
          if (is && __popc(upto) == static_cast<int>(left) + 1) {
            const int64_t idx = i + lane;
            a.next_token[b] = idx;
            if (a.token != nullptr) a.token[b] = idx;
            if (a.position != nullptr) a.position[b] += 1;
            if (a.finished != nullptr && idx == a.eos) a.finished[b] |= 1;
            if (a.prob != nullptr) a.prob[b] = pick_prob;
          }
          break;
        }
        left -= cnt;
      }
    }
  }
  cluster.sync();  // the others read this CTA's counters until here
}

}  // namespace
}  // namespace chr

using namespace chr;

extern "C" int chr_nf4_sample_commit_batch(const void *logits, int64_t row_stride, int32_t n,
                                           int32_t batch, const void *u, const void *temperature,
                                           const void *top_k, const void *top_p, const void *min_p,
                                           void *prob, void *next_token, void *token,
                                           void *position, void *finished, int64_t eos,
                                           void *stream) {
  if (logits == nullptr || u == nullptr || next_token == nullptr) return kNull;
  if (n < 1 || n > kSliceMax * kSampleMaxCluster || batch < 1 || batch > 65535 || row_stride < n) {
    return kDims;
  }
  // CTAs per row: slices of 4096 tokens are enough, and more CTAs than SMs would only queue,
  // but a slice never exceeds its counters
  const int sms = sm_count();
  int C = 1;
  while (C < kSampleMaxCluster && n > C * 4096 && 2ll * C * batch <= sms) C *= 2;
  while (n > C * kSliceMax) C *= 2;
  SampleArgs a{};
  a.logits = static_cast<const __nv_bfloat16 *>(logits);
  a.row_stride = row_stride;
  a.n = n;
  a.batch = batch;
  a.slice = (n + C - 1) / C;
  a.u = static_cast<const float *>(u);
  a.temperature = static_cast<const float *>(temperature);
  a.top_k = static_cast<const int32_t *>(top_k);
  a.top_p = static_cast<const float *>(top_p);
  a.min_p = static_cast<const float *>(min_p);
  a.prob = static_cast<float *>(prob);
  a.next_token = static_cast<int64_t *>(next_token);
  a.token = static_cast<int64_t *>(token);
  a.position = static_cast<int64_t *>(position);
  a.finished = static_cast<uint8_t *>(finished);
  a.eos = eos;
  static int done[64] = {};
  if (!ensure_smem_attr(sample_kernel, static_cast<int>(sizeof(SampleShared)), done)) return kLaunch;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * C));
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(C);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel, a) == cudaSuccess ? kOk : kLaunch;
}
