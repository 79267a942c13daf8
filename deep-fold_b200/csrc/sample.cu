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
// shared memory (65536 16-bit counters, 128 KB) and marks which
// of the 1024 chunks of 64 values occur. The chunks that do - under a hundred, values of a
// row spanning a dozen binary orders - are dealt over the cluster's warps: a warp adds the
// CTAs' counters through distributed shared memory, takes one exp per value, and hands
// counts and weights to the row's first CTA, one warp of which walks the cuts and the draw.
// The CTA whose slice holds the drawn token finds its index. One launch, no scratch memory.
// Bound by latency: one row of 151936 tokens on eight CTAs takes 15.2 us, of which counting 2 (19,000
// tokens a CTA) and finding the token 2.5, the rest is a chain of cluster barriers and dependent
// steps. 64 such rows, two CTAs each, take 24.2 us: counting 7.5 (shared-memory atomics, about
// 5 a clock), finding 5. (With four CTAs each, which queue for the SMs, 35.9 us.)

#include <cooperative_groups.h>
#include <cstddef>

#include "nf4_common.cuh"

namespace chr {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kKeys = 65536;
constexpr int kChunk = 64;                 // values per chunk
constexpr int kChunks = kKeys / kChunk;
constexpr int kSampleMaxCluster = 8;
// A slice is counted in two parts, the first of at most kPart tokens. A value that holds 32768
// of them - there is one at most - is then set aside and its counter starts again, so that no
// 16-bit counter wraps in the second part, of at most 32768 tokens, either.
constexpr int kPart = 65520;               // in whole 16-byte pieces; the first part takes the ends too
constexpr int kHeavy = 32768;
constexpr int kSliceMax = kPart + kHeavy;

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

constexpr int kGroups = 12;                // 32-piece groups of a warp when it looks for the token
static_assert(kSliceMax / 8 <= kGroups * 32 * kSampleWarps && kGroups % 4 == 0, "a bit per token");
constexpr int kSampleMaxVocab = 524280;
static_assert(kSampleMaxVocab <= kSliceMax * kSampleMaxCluster, "a slice per CTA");
constexpr int kCache = 80;  // chunks whose counts and weights the first CTA keeps

struct SampleShared {
  alignas(16) uint32_t hist[kKeys / 2];  // counters 2i (low half) and 2i + 1 (high half)
  uint32_t map[kChunks / 32];        // chunks that occur in this CTA's slice; bit c % 32 of word c / 32
  alignas(16) uint8_t four[kChunks / 4]; // the same, four chunks a byte
  uint32_t max_key;                  // of this CTA's slice
  uint32_t heavy_key, heavy_n;       // the value set aside (none: kNoKey) and its tokens
  uint32_t found[kSampleWarps];
  // the draw, written by the first CTA into every one
  uint32_t pick_key, pick_rank;      // value and its pick_rank-th occurrence
  float pick_prob;
  // in the first CTA: the chunks that occur, highest values first
  uint32_t count[kChunks];           // tokens, then tokens before the chunk
  double mass[kChunks];              // their weight, likewise
  uint16_t chunk[kChunks];
  alignas(16) double w[kCache][kChunk];  // values of a chunk, highest first
  alignas(16) uint32_t n[kCache][kChunk];
};

// 16-byte accesses to hist and w, 8-byte ones to four and n
static_assert(offsetof(SampleShared, hist) % 16 == 0 && offsetof(SampleShared, w) % 16 == 0 &&
              offsetof(SampleShared, four) % 16 == 0 && offsetof(SampleShared, n) % 16 == 0, "aligned");

// A value's key orders as the value does: the bits of a bf16 with the sign flipped, a
// negative one with all bits flipped; -0 has +0's key, NaN the highest.
__device__ __forceinline__ float key_value(uint32_t k) {
  const uint32_t b = (k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu);
  return __uint_as_float(b << 16);
}

// exp((value - max) / T), the weight of every token of one value
__device__ __forceinline__ double key_weight(uint32_t key, double m, double temp) {
  return exp((static_cast<double>(key_value(key)) - m) / temp);
}

// Elements lo..hi of a row: up to 7 of them, then whole aligned 16-byte pieces from element
// `first` on, then up to 7 from element `last` on.
struct Slice {
  const unsigned short *x;
  int lo, hi, first, last, pieces;
};
__device__ __forceinline__ Slice slice_of(const __nv_bfloat16 *row, int lo, int hi) {
  Slice s;
  s.x = reinterpret_cast<const unsigned short *>(row);
  s.lo = lo;
  s.hi = hi;
  s.first = min(lo + static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(s.x + lo) & 15)) & 15) >> 1), hi);
  s.pieces = (hi - s.first) / 8;
  s.last = s.first + s.pieces * 8;
  return s;
}
constexpr uint32_t kNegInf = 0xFF80u, kNegInfKey = 0x007Fu, kNoKey = 0xFFFFFFFFu;
// Two pieces, `step` apart; what lies at `end` or beyond is not read.
__device__ __forceinline__ void slice_pieces(const Slice &s, int v, int step, int end, uint4 (&x)[2]) {
  const uint4 *src = reinterpret_cast<const uint4 *>(s.x + s.first);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    x[k] = make_uint4(0u, 0u, 0u, 0u);
    if (v + k * step < end) x[k] = __ldcg(src + v + k * step);
  }
}
// Elements before the pieces (tail = false) and behind them, one per lane; -inf where there is none.
__device__ __forceinline__ uint32_t slice_edge(const Slice &s, bool tail, int lane) {
  const int at = (tail ? s.last : s.lo) + lane;
  return at < (tail ? s.hi : s.first) ? __ldcg(s.x + at) : kNegInf;
}
// Two bf16 values as order keys, but for NaN and -0, which are put right afterwards.
__device__ __forceinline__ uint32_t raw_keys(uint32_t two) {
  return two ^ (((two >> 15) & 0x00010001u) * 0xFFFFu | 0x80008000u);
}
// One token of key `key`, at bit kAt of `keys`; -inf is not counted (a masked vocabulary would
// queue up at its counter).
template <int kAt>
__device__ __forceinline__ void count_key(uint32_t hist, uint32_t keys) {
  const uint32_t key = kAt == 0 ? keys & 0xFFFFu : keys >> 16;
  const uint32_t at = hist + ((kAt == 0 ? keys << 1 : keys >> 15) & 0x1FFFCu);
  const uint32_t one = (key & 1u) * 65535u + 1u;  // the upper half counts odd keys
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %0, 127;\n\t"
      "@p red.shared.add.u32 [%1], %2;\n\t}" ::"r"(key), "r"(at), "r"(one) : "memory");
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
// Adds what the CTAs set aside of chunk c; `heavy`: the value that CTA l did.
__device__ __forceinline__ void add_heavy(cg::cluster_group &cluster, SampleShared &sm, int c, int lane, uint32_t heavy,
                                          uint32_t &hi, uint32_t &lo) {
  for (unsigned some = __ballot_sync(0xffffffffu, heavy >> 6 == static_cast<uint32_t>(c)); some != 0u; some &= some - 1u) {
    const int r = __ffs(some) - 1;
    const uint32_t n = *cluster.map_shared_rank(&sm.heavy_n, r);
    const uint32_t at = 63u - (__shfl_sync(0xffffffffu, heavy, r) & 63u);
    if (at == 2u * lane) hi += n;
    if (at == 2u * lane + 1u) lo += n;
  }
}

__device__ __forceinline__ double shfl_up(double v, int off) { return __shfl_up_sync(0xffffffffu, v, off); }

// One chunk of the row as a warp sees it: counts, weights and what lies before each value.
struct ChunkView {
  uint32_t key;                               // of the lane's higher value
  uint32_t n_hi, n_lo, before_hi, before_lo;  // tokens; tokens before the lane's two values
  double w_hi, w_lo, mass_hi, mass_lo;        // weights; weight before the two values
};
__device__ __noinline__ ChunkView view_chunk(SampleShared &sm, int i, double m, double temp) {
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31;
  const int c = sm.chunk[i];
  ChunkView v;
  v.key = static_cast<uint32_t>(c * kChunk + 63 - 2 * lane);
  if (i < kCache) {
    const uint2 n = *reinterpret_cast<const uint2 *>(&sm.n[i][2 * lane]);
    const double2 w = *reinterpret_cast<const double2 *>(&sm.w[i][2 * lane]);
    v.n_hi = n.x;
    v.n_lo = n.y;
    v.w_hi = w.x;
    v.w_lo = w.y;
  } else {
    const uint32_t heavy = lane < static_cast<int>(cluster.num_blocks()) ? *cluster.map_shared_rank(&sm.heavy_key, lane) : kNoKey;
    chunk_counts(cluster, sm, c, lane, v.n_hi, v.n_lo);
    add_heavy(cluster, sm, c, lane, heavy, v.n_hi, v.n_lo);
    v.w_hi = key_weight(v.key, m, temp);
    v.w_lo = key_weight(v.key - 1u, m, temp);
  }
  const uint32_t own_c = v.n_hi + v.n_lo;
  uint32_t cnt = own_c;
  double mass = (v.n_hi != 0u ? v.n_hi * v.w_hi : 0.0) + (v.n_lo != 0u ? v.n_lo * v.w_lo : 0.0);
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
  v.before_hi = sm.count[i] + cnt - own_c;
  v.before_lo = v.before_hi + v.n_hi;
  v.mass_hi = sm.mass[i] + prev;
  v.mass_lo = v.mass_hi + (v.n_hi != 0u ? v.n_hi * v.w_hi : 0.0);
  return v;
}

// The last of L ascending values that is at most `limit` (or[strict]: below it); 0 if none is.
template <typename T>
__device__ __forceinline__ int last_of(const T *v, int L, T limit, bool below) {
  const int lane = threadIdx.x & 31;
  auto ok = [&](int i) { return i < L && (below ? v[i] < limit : v[i] <= limit); };
  const int g = 31 - __clz(__ballot_sync(0xffffffffu, ok(lane * 32)) | 1u);
  return g * 32 + 31 - __clz(__ballot_sync(0xffffffffu, ok(g * 32 + lane)) | 1u);
}

// A value of the row: its key, the tokens and the weight before it, its tokens and weight.
struct Value {
  uint32_t key, before, n;
  double mass, w;
};
// Of the chunk a warp sees, the first value with some lane's flag, or else the last one.
__device__ __forceinline__ Value pick_value(const ChunkView &v, bool hi, bool lo) {
  const unsigned who = __ballot_sync(0xffffffffu, hi || lo);
  const unsigned any = __ballot_sync(0xffffffffu, v.n_hi != 0u || v.n_lo != 0u);
  const int from = who != 0u ? __ffs(who) - 1 : 31 - __clz(any | 1u);
  const bool take_hi = who != 0u ? hi : v.n_lo == 0u;
  Value x;
  x.key = __shfl_sync(0xffffffffu, take_hi ? v.key : v.key - 1u, from);
  x.before = __shfl_sync(0xffffffffu, take_hi ? v.before_hi : v.before_lo, from);
  x.n = __shfl_sync(0xffffffffu, take_hi ? v.n_hi : v.n_lo, from);
  x.mass = __shfl_sync(0xffffffffu, take_hi ? v.mass_hi : v.mass_lo, from);
  x.w = __shfl_sync(0xffffffffu, take_hi ? v.w_hi : v.w_lo, from);
  return x;
}
// The value of the token that has `rank` tokens before it.
__device__ __forceinline__ Value value_at(SampleShared &sm, int L, uint32_t rank, double m, double temp) {
  const ChunkView v = view_chunk(sm, last_of(sm.count, L, rank, false), m, temp);
  return pick_value(v, v.n_hi != 0u && rank < v.before_hi + v.n_hi, v.n_lo != 0u && rank < v.before_lo + v.n_lo);
}
// The first value whose end of the running weight exceeds r (or, not strict, reaches it).
__device__ __forceinline__ Value crossing(SampleShared &sm, int L, double r, bool strict, double m, double temp) {
  const ChunkView v = view_chunk(sm, last_of(sm.mass, L, r, !strict), m, temp);
  const double end_hi = v.mass_hi + v.n_hi * v.w_hi, end_lo = v.mass_lo + v.n_lo * v.w_lo;
  return pick_value(v, v.n_hi != 0u && (strict ? end_hi > r : end_hi >= r),
                    v.n_lo != 0u && (strict ? end_lo > r : end_lo >= r));
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
  if (tid == 0) {
    sm.heavy_key = kNoKey;
    sm.heavy_n = 0u;
  }
  __syncthreads();
  pdl_wait();
  const __nv_bfloat16 *row = a.logits + b * a.row_stride;
  const int lo = min(rank * a.slice, a.n), hi = min(lo + a.slice, a.n);
  const Slice slice = slice_of(row, lo, hi);

  // ---- the slice's histogram ----
  static_assert(kNegInfKey == 127, "not counted");
  const uint32_t hist = static_cast<uint32_t>(__cvta_generic_to_shared(sm.hist));
  if (warp < 2) count_key<0>(hist, raw_keys(slice_edge(slice, warp == 1, lane)));
#pragma unroll 1
  for (int from = 0; from < max(slice.pieces, 1); from += kPart / 8) {
    const int to = min(from + kPart / 8, slice.pieces);
    uint4 x[2], next[2];
    slice_pieces(slice, from + tid, kSampleThreads, to, x);
#pragma unroll 1
    for (int v = from + tid; v < to; v += 2 * kSampleThreads) {
      slice_pieces(slice, v + 2 * kSampleThreads, kSampleThreads, to, next);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (v + k * kSampleThreads < to) {
          const uint32_t two[4] = {raw_keys(x[k].x), raw_keys(x[k].y), raw_keys(x[k].z), raw_keys(x[k].w)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            count_key<0>(hist, two[e]);
            count_key<16>(hist, two[e]);
          }
        }
        x[k] = next[k];
      }
    }
    __syncthreads();
    if (to < slice.pieces) {
      for (int i = tid; i < kKeys / 8; i += kSampleThreads) {
        const uint4 x = reinterpret_cast<const uint4 *>(sm.hist)[i];
        if (((x.x | x.y | x.z | x.w) & 0x80008000u) == 0u) continue;
        const uint32_t n[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((n[e] & 0x80008000u) == 0u) continue;
          const bool high = (n[e] >> 31) != 0u;
          sm.heavy_key = static_cast<uint32_t>((i * 4 + e) * 2 + (high ? 1 : 0));
          sm.heavy_n = high ? n[e] >> 16 : n[e] & 0xFFFFu;
          sm.hist[i * 4 + e] = high ? n[e] & 0xFFFFu : n[e] & 0xFFFF0000u;
        }
      }
      __syncthreads();
    }
  }
  // NaN of either sign to the highest key, -0 to +0
  if (warp == 0) {
    uint32_t nans = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int w = i * 32 + lane;  // words 0..63: keys 0..127, 64..127: keys 0xFF80..0xFFFF
      uint32_t *at = &sm.hist[w < 64 ? w : kKeys / 2 - 128 + w];
      uint32_t n = *at;
      // -inf (key 0x7F) has no count; +inf (0xFF80, the low half of its word) keeps its own
      const uint32_t keep = w == 64 ? n & 0xFFFFu : 0u;
      n -= keep;
      if (n != 0u) *at = keep;
      nans += (n & 0xFFFFu) + (n >> 16);
    }
    nans = __reduce_add_sync(0xffffffffu, nans);
    __syncwarp();
    if (lane == 0) {
      // a row with a NaN picks the first one, so only whether a slice has some matters
      if (nans != 0u) sm.hist[kKeys / 2 - 1] += min(nans, 65535u) << 16;
      const uint32_t minus = sm.hist[0x7FFF >> 1] >> 16;  // -0: the high half of word 0x3FFF
      const uint32_t plus = sm.hist[0x8000 >> 1];
      sm.hist[0x7FFF >> 1] &= 0xFFFFu;
      const uint32_t key = sm.heavy_key;
      if (key == 0x7FFFu) {
        sm.heavy_key = 0x8000u;
      } else if (key != kNoKey && (key < kNegInfKey || key > 0xFF80u)) {
        sm.heavy_key = 0xFFFFu;
      }
      if ((plus & 0xFFFFu) + minus < 65536u) {
        sm.hist[0x8000 >> 1] = plus + minus;
      } else {  // too many for the counter, so no other value was set aside
        sm.heavy_key = 0x8000u;
        sm.heavy_n += minus;
      }
    }
  }
  __syncthreads();
  // chunks that occur: a warp looks at four chunks (512 bytes) at a time
#pragma unroll
  for (int i = warp; i < kChunks / 4; i += kSampleWarps) {
    const uint4 v = reinterpret_cast<const uint4 *>(sm.hist)[i * 32 + lane];
    const unsigned some = __ballot_sync(0xffffffffu, (v.x | v.y | v.z | v.w) != 0u);
    const uint32_t four = ((some & 0xFFu) != 0u ? 1u : 0u) | ((some & 0xFF00u) != 0u ? 2u : 0u) |
                          ((some & 0xFF0000u) != 0u ? 4u : 0u) | ((some & 0xFF000000u) != 0u ? 8u : 0u);
    if (lane == 0) sm.four[i] = static_cast<uint8_t>(four);
  }
  __syncthreads();
  if (warp == 0) {
    const uint2 v = reinterpret_cast<const uint2 *>(sm.four)[lane];
    uint32_t w = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= ((v.x >> (8 * e)) & 15u) << (4 * e) | ((v.y >> (8 * e)) & 15u) << (16 + 4 * e);
    const uint32_t heavy = sm.heavy_key;
    if (heavy != kNoKey && static_cast<int>(heavy >> 11) == lane) w |= 1u << ((heavy >> 6) & 31u);
    sm.map[lane] = w;
    // the slice's maximum: the highest value of its highest chunk
    const unsigned words = __ballot_sync(0xffffffffu, w != 0u);
    uint32_t best = kNegInfKey;
    if (words != 0u) {
      const int top = 31 - __clz(words);
      const int c = top * 32 + 31 - __clz(__shfl_sync(0xffffffffu, w, top));
      const uint32_t n = sm.hist[c * (kChunk / 2) + lane];
      const uint32_t key = static_cast<uint32_t>(c * kChunk + 2 * lane) + ((n >> 16) != 0u ? 1u : 0u);
      best = __reduce_max_sync(0xffffffffu, n != 0u ? key : 0u);
    }
    if (heavy != kNoKey) best = max(best, heavy);
    if (lane == 0) sm.max_key = best;
  }
  cluster.sync();

  const uint32_t heavy = lane < C ? *cluster.map_shared_rank(&sm.heavy_key, lane) : kNoKey;
  uint32_t max_key = 0u;
#pragma unroll
  for (int r = 0; r < kSampleMaxCluster; ++r) {
    if (r < C) max_key = max(max_key, *cluster.map_shared_rank(&sm.max_key, r));
  }
  const float temp_f = a.temperature != nullptr ? __ldg(a.temperature + b) : 1.f;
  const float max_f = key_value(max_key);
  // max_key of NaN is 0xFFFF; +inf and -inf are not finite either
  const bool greedy = !(temp_f > 0.f) || max_key == 0xFFFFu || isinf(max_f);
  const double m = max_f, temp = temp_f;

  uint32_t pick_key = max_key, pick_rank = 0u;
  float pick_prob = 1.f;
  if (!greedy) {
    // ---- counts and weights of the chunks that occur, to the first CTA ----
    SampleShared *lead = cluster.map_shared_rank(&sm, 0);
    // lane l: word 31 - l, so that both lanes and bits run from the highest chunk down
    uint32_t word = 0u;
#pragma unroll
    for (int r = 0; r < kSampleMaxCluster; ++r) {
      if (r < C) word |= *cluster.map_shared_rank(&sm.map[31 - lane], r);
    }
    int upto = __popc(word);
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    const int L = __shfl_sync(0xffffffffu, upto, 31);
    for (int i = warp * C + rank; i < L; i += kSampleWarps * C) {
      // the i-th chunk: its word, then the bit with i - (bits before the word) set ones above it
      const int from = __ffs(__ballot_sync(0xffffffffu, upto > i)) - 1;
      const uint32_t bits = __shfl_sync(0xffffffffu, word, from);
      const int nth = i - (__shfl_sync(0xffffffffu, upto, from) - __popc(bits));
      const bool mine = (bits >> (31 - lane)) & 1u;
      const unsigned set = __ballot_sync(0xffffffffu, mine);  // lane order: highest bit first
      const int at = __ffs(__ballot_sync(0xffffffffu, mine && __popc(set & ((1u << lane) - 1u)) == nth)) - 1;
      const int c = (31 - from) * 32 + 31 - at;
      uint32_t n_hi, n_lo;
      chunk_counts(cluster, sm, c, lane, n_hi, n_lo);
      const uint32_t key = static_cast<uint32_t>(c * kChunk + 63 - 2 * lane);
      const double w_hi = key_weight(key, m, temp), w_lo = key_weight(key - 1u, m, temp);
      add_heavy(cluster, sm, c, lane, heavy, n_hi, n_lo);
      // a value that does not occur may have no finite weight
      double mass = (n_hi != 0u ? n_hi * w_hi : 0.0) + (n_lo != 0u ? n_lo * w_lo : 0.0);
      if (i < kCache) {
        *reinterpret_cast<uint2 *>(&lead->n[i][2 * lane]) = make_uint2(n_hi, n_lo);
        *reinterpret_cast<double2 *>(&lead->w[i][2 * lane]) = make_double2(w_hi, w_lo);
      }
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {  // in the order of view_chunk's running sum
        const double o = shfl_up(mass, off);
        if (lane >= off) mass += o;
      }
      const uint32_t cnt = __reduce_add_sync(0xffffffffu, n_hi + n_lo);
      if (lane == 31) {
        lead->mass[i] = mass;
        lead->count[i] = cnt;
        lead->chunk[i] = static_cast<uint16_t>(c);
      }
    }
    cluster.sync();
    if (rank == 0 && warp == 0) {
      // ---- what lies before each chunk: a lane sums a run of them ----
      const int per = (L + 31) / 32;
      const int i0 = min(lane * per, L), i1 = min(i0 + per, L);
      double run = 0.0;
      uint32_t run_c = 0u;
      for (int i = i0; i < i1; ++i) {
        run += sm.mass[i];
        run_c += sm.count[i];
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
      const double total = __shfl_sync(0xffffffffu, incl, 31);
      const uint32_t finite = __shfl_sync(0xffffffffu, incl_c, 31);  // tokens that are not -inf
      double at = shfl_up(incl, 1);
      uint32_t at_c = incl_c - run_c;
      if (lane == 0) at = 0.0;
      for (int i = i0; i < i1; ++i) {
        const double mi = sm.mass[i];
        const uint32_t ci = sm.count[i];
        sm.mass[i] = at;
        sm.count[i] = at_c;
        at += mi;
        at_c += ci;
      }
      __syncwarp();
      // ---- the kept prefix: its tokens and their weight, cut by cut ----
      uint32_t kept = finite;
      double sum = total;
      const int k = a.top_k != nullptr ? __ldg(a.top_k + b) : 0;
      if (k > 0 && static_cast<uint32_t>(k) < finite) {
        kept = static_cast<uint32_t>(k);
        const Value x = value_at(sm, L, kept - 1u, m, temp);
        sum = x.mass + (kept - x.before) * x.w;
      }
      const float p = a.top_p != nullptr ? __ldg(a.top_p + b) : 1.f;
      const float least = a.min_p != nullptr ? __ldg(a.min_p + b) : 0.f;
      if (p < 1.f) {
        const double target = fmax(static_cast<double>(p) * sum, 0.0);
        const Value x = crossing(sm, L, target, false, m, temp);
        // of the crossing value's tokens those before which the sum is below the target
        double q = x.w > 0.0 ? ceil((target - x.mass) / x.w) : 1.0;
        q = fmin(fmax(q, 1.0), static_cast<double>(x.n));
        const uint32_t np = max(x.before + static_cast<uint32_t>(q), 1u);
        if (np < kept) {
          kept = np;
          sum = x.mass + q * x.w;
        }
      }
      if (least > 0.f) {
        // the last chunk whose highest value still weighs min_p, then the values within
        auto heavy = [&](int i) {
          return i < L && key_weight(sm.chunk[i] * kChunk + 63u, m, temp) >= static_cast<double>(least);
        };
        const int g = 31 - __clz(__ballot_sync(0xffffffffu, heavy(lane * 32)) | 1u);
        const int i = g * 32 + 31 - __clz(__ballot_sync(0xffffffffu, heavy(g * 32 + lane)) | 1u);
        const ChunkView v = view_chunk(sm, i, m, temp);
        const bool hi_in = v.n_hi != 0u && v.w_hi >= static_cast<double>(least);
        const bool lo_in = v.n_lo != 0u && v.w_lo >= static_cast<double>(least);
        const uint32_t nm = __shfl_sync(0xffffffffu, v.before_hi, 0) +
                            __reduce_add_sync(0xffffffffu, (hi_in ? v.n_hi : 0u) + (lo_in ? v.n_lo : 0u));
        if (nm < kept) {
          kept = max(nm, 1u);
          const Value x = value_at(sm, L, kept - 1u, m, temp);
          sum = x.mass + (kept - x.before) * x.w;
        }
      }
      // ---- the draw ----
      const float uf = fminf(fmaxf(__ldg(a.u + b), 0.f), 0.99999994f);  // NaN: 0
      const double r = static_cast<double>(uf) * sum;
      Value x = crossing(sm, L, r, true, m, temp);
      double q = x.w > 0.0 ? floor((r - x.mass) / x.w) : 0.0;
      q = fmin(fmax(q, 0.0), static_cast<double>(x.n) - 1.0);
      uint32_t in = static_cast<uint32_t>(fmax(q, 0.0));
      if (x.before + in >= kept) {  // rounding took the draw past the last kept token
        x = value_at(sm, L, kept - 1u, m, temp);
        in = kept - 1u - x.before;
      }
      if (lane < C) {
        SampleShared *to = cluster.map_shared_rank(&sm, lane);
        to->pick_key = x.key;
        to->pick_rank = in;
        to->pick_prob = static_cast<float>(x.w / sum);
      }
    }
    cluster.sync();
    pick_key = sm.pick_key;
    pick_rank = sm.pick_rank;
    pick_prob = sm.pick_prob;
  }

  // ---- the pick_rank-th token of value pick_key, in order of index ----
  auto commit = [&](int64_t idx) {
    a.next_token[b] = idx;
    if (a.token != nullptr) a.token[b] = idx;
    if (a.position != nullptr) a.position[b] += 1;
    if (a.finished != nullptr && idx == a.eos) a.finished[b] |= 1;
    if (a.prob != nullptr) a.prob[b] = pick_prob;
  };
  if (max_f == -INFINITY) {  // nothing but -inf, which was not counted
    if (rank == 0 && tid == 0) commit(0);
  } else {
    const int shift = (pick_key & 1u) ? 16 : 0;
    uint32_t counts[kSampleMaxCluster];
#pragma unroll
    for (int r = 0; r < kSampleMaxCluster; ++r) {
      counts[r] = r <= rank ? *cluster.map_shared_rank(&sm.hist[pick_key >> 1], r) : 0u;
    }
    uint32_t before = 0u, here = 0u;
#pragma unroll
    for (int r = 0; r < kSampleMaxCluster; ++r) {
      const uint32_t n = (counts[r] >> shift) & 0xFFFFu;
      if (r < rank) before += n;
      if (r == rank) here = n;
    }
    for (unsigned some = __ballot_sync(0xffffffffu, heavy == pick_key && lane <= rank); some != 0u; some &= some - 1u) {
      const int r = __ffs(some) - 1;
      const uint32_t n = *cluster.map_shared_rank(&sm.heavy_n, r);
      if (r < rank) {
        before += n;
      } else {
        here += n;
      }
    }
    if (pick_rank >= before && pick_rank < before + here) {
      uint32_t want = pick_rank - before;  // occurrence within the slice
      // its bits: one pattern, but for zero (either sign) and NaN (many)
      const uint32_t bits = (pick_key & 0x8000u) ? (pick_key & 0x7FFFu) : (~pick_key & 0xFFFFu);
      const uint32_t mask = bits == 0u ? 0x7FFF7FFFu : 0xFFFFFFFFu, twice = bits * 0x10001u;
      const bool nan = pick_key == 0xFFFFu;
      // bits 15 and 31: whether the lower, the upper of two elements is the value
      auto is = [&](uint32_t two) {
        if (nan) return ((two & 0x7FFF7FFFu) + 0x007F007Fu) & 0x80008000u;  // above 0x7F80
        const uint32_t off = (two ^ twice) & mask;
        return ~(((off & 0x7FFF7FFFu) + 0x7FFF7FFFu) | off) & 0x80008000u;
      };
      auto matches = [&](const uint4 &x) {  // bit e: element e of a piece
        const uint32_t c = is(x.x) >> 15 | is(x.y) >> 13 | is(x.z) >> 11 | is(x.w) >> 9;
        return (c & 0x55u) | ((c >> 15) & 0xAAu);
      };
      // a warp's part of the slice, in order of index: up to kGroups groups of 32 pieces, whose
      // matches a lane keeps, eight bits a piece; the ends go with the first and last warp's
      const int per = (slice.pieces + kSampleWarps - 1) / kSampleWarps;
      const int w0 = min(warp * per, slice.pieces), w1 = min(w0 + per, slice.pieces);
      uint32_t hits[kGroups / 4], mine = 0u;
#pragma unroll
      for (int q = 0; q < kGroups / 4; ++q) hits[q] = 0u;
      // (-inf, which pads the pieces and the ends, is never looked for)
      uint32_t ends = 0u;
      if (warp == 0 || warp == kSampleWarps - 1) {
        ends = __ballot_sync(0xffffffffu, (is(slice_edge(slice, warp != 0, lane)) & 0x8000u) != 0u);
      }
      uint4 x[2], next[2];
      slice_pieces(slice, w0 + lane, 32, w1, x);
#pragma unroll 1
      for (int q = 0; w0 + q * 64 < w1; ++q) {
        const int v = w0 + q * 64 + lane;
        slice_pieces(slice, v + 64, 32, w1, next);
        uint32_t h = 0u;
        if (v < w1) h = matches(x[0]);
        if (v + 32 < w1) h |= matches(x[1]) << 8;
        x[0] = next[0];
        x[1] = next[1];
        mine += __popc(h);
        h <<= 16 * (q & 1);
#pragma unroll
        for (int i = 0; i < kGroups / 4; ++i) hits[i] |= i == q >> 1 ? h : 0u;
      }
      mine = __reduce_add_sync(0xffffffffu, mine) + __popc(ends);
      if (lane == 0) sm.found[warp] = mine;
      __syncthreads();
      const uint32_t skip = __reduce_add_sync(0xffffffffu, lane < warp ? sm.found[lane] : 0u);
      if (want >= skip && want < skip + mine) {
        want -= skip;
        const uint32_t in_front = warp == 0 ? __popc(ends) : 0u, behind = warp == 0 ? 0u : __popc(ends);
        const uint32_t in_pieces = mine - in_front - behind;
        if (want < in_front || want >= in_front + in_pieces) {
          const uint32_t nth = want < in_front ? want : want - in_pieces;
          if (((ends >> lane) & 1u) != 0u && __popc(ends & ((1u << lane) - 1u)) == nth) commit((warp == 0 ? slice.lo : slice.last) + lane);
        } else if (in_pieces == 1u) {
#pragma unroll
          for (int i = 0; i < kGroups / 4; ++i) {
            const int bit = __ffs(hits[i]) - 1;
            if (bit >= 0) commit(slice.first + (w0 + (i * 4 + (bit >> 3)) * 32 + lane) * 8 + (bit & 7));
          }
        } else {
          want -= in_front;
          uint32_t hit = 0u, left = want, at = 0u;
          bool found = false;
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            const uint32_t h = (hits[g / 4] >> (8 * (g & 3))) & 0xFFu;
            const uint32_t all = __reduce_add_sync(0xffffffffu, __popc(h));
            if (!found && left < all) {
              found = true;
              hit = h;
              at = g;
            }
            if (!found) left -= all;
          }
          uint32_t incl = __popc(hit);
          const uint32_t own = incl;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const uint32_t o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += o;
          }
          if (left >= incl - own && left < incl) {
            for (uint32_t j = incl - own; j < left; ++j) hit &= hit - 1u;
            commit(slice.first + (w0 + static_cast<int>(at) * 32 + lane) * 8 + __ffs(hit) - 1);
          }
        }
      }
    }
  }
  cluster.sync();  // the others read this CTA's counters until here
}

// The launch of `rows` clusters of C CTAs.
cudaLaunchConfig_t sample_config(int rows, int C, cudaLaunchAttribute *attr) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * C);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = static_cast<unsigned>(C);
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// How many clusters of C (2, 4, 8) CTAs run at once on the current device.
int clusters_at_once(int C) {
  static int known[64][3] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int &n = known[dev][C == 2 ? 0 : (C == 4 ? 1 : 2)];
  if (n == 0) {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = sample_config(1, C, &attr);
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, sample_kernel, &cfg) != cudaSuccess || got < 1) got = sm_count() / (2 * C);
    n = got;
  }
  return n;
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
  if (n < 1 || n > kSampleMaxVocab || batch < 1 || batch > 65535 || row_stride < n) {
    return kDims;
  }
  static int done[64] = {};
  if (!ensure_smem_attr(sample_kernel, static_cast<int>(sizeof(SampleShared)), done)) return kLaunch;
  // CTAs per row. More of them count faster and wait longer for one another: one row of 32000
  // tokens takes 14.0 us on two, 12.7 on four, 13.2 on eight; nine of 92543 14.3 on four, 14.7 on
  // eight; one of 8000 14.8 on one, 13.3 on two. Clusters that do not run at once take turns:
  // 16 rows of 60001 tokens take 14.2 us on four, 21.1 on eight. A slice never exceeds its counters.
  int C = 1;
  while (C < kSampleMaxCluster && n > (C < 4 ? C * 4096 : C * 24576) && batch <= clusters_at_once(2 * C)) C *= 2;
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
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = sample_config(batch, C, attr);
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel, a) == cudaSuccess ? kOk : kLaunch;
}
