// The wide form of the paged attention (paged_attn.cu): items of up to 256 query rows on the
// fifth-generation tensor cores, for head dims 64 and 128.
//
// One CTA per SM holds two query tiles of 128 rows against one key / value stream of
// 128-row tiles, so that a cache row crosses from L2 once per 256 query rows (two CTAs of
// 128 rows each would need 64 bytes per clock and SM, more than L2 delivers to all SMs).
//   warp 9      page look-up and TMA copies of K and V pages (two stages each)
//   warp 8      issues tcgen05.mma in steps of 64 cache rows: S_w = Q_w K^T (128 x 64, FP32, tensor
//               memory) and O_w += P_w V, P_w read from tensor memory, where it lies over S_w
//   warps 0-3   softmax of tile 0, warps 4-7 of tile 1: a thread owns a row
// Each tile has two S buffers (2 x 2 x 64 columns; the accumulators take the other 256): the
// order of issue is PV0(j) QK0(j+2) PV1(j) QK1(j+2), so the scores of the next step are there
// when a softmax ends and neither side waits for the other's latency. Per 128 cache rows the
// products take 2 x (2 x 8 x 48 + 8 x 64) = 2560 clocks - the 128 x 64 one is held up by the
// 128 bytes a clock its operands are read at, hence 48 - and the exps 2048 (32768 at 16 a clock).
// (With one S buffer of 128 columns per tile, products 2048 clocks, the chain of both was 4100.)
// Measured 2.0 us per 128 cache rows and 256 queries where these come from L2, at the 1.5 to 1.8 GHz
// that the power cap leaves, 2.8 where they come from HBM (one warp looks the pages up and requests
// K behind the wait for V's stage, so that little more than a stage of each is on the way);
// a segment costs 5 us more for its start and its result. Three chunks of 2047 rows over
// caches of up to 4096, 40 / 8 heads of 128 (349 GFLOP): 360 to 405 us by the clock.
// The running
// maximum a row subtracts is raised only when the new one is more than 8
// (in log2) above it: P then stays below 2^8, which bf16 holds as exactly as 1, and the
// accumulator in tensor memory is almost never rescaled.
// P is rounded to bf16 for the second product, its sum is not; everything else is FP32.
//
// Every wait is bounded; one that runs out leaves a code in a status word
// (chr_nf4_attn_paged_status), the roles stop, copies and products in flight are waited for
// (again with a limit) and the tensor memory is freed.

#pragma once

#include "paged.cuh"
#include "tma_tc.cuh"

namespace chr {
namespace {

constexpr int kWideThreads = 320;
constexpr int kWideM = 256;
constexpr int kWideTile = 128;
constexpr int kWideStep = 64;   // cache rows of one product

template <int HD>
struct WideLayout {
  static constexpr int kHalves = HD / 64;                   // 128-byte wide pieces of a row
  static constexpr int kPiece = 128 * 128;                  // 128 rows x 128 bytes
  static constexpr int kTileB = kHalves * kPiece;           // one 128-row tile
  static constexpr int kQ = 0;                              // two query tiles
  static constexpr int kK = 2 * kTileB;                     // two stages
  static constexpr int kV = 4 * kTileB;                     // two stages
  static constexpr int kBars = 6 * kTileB;
  static constexpr int kSegOff = kBars + 256;
  static constexpr int kStage = (kSegOff + kSegs * static_cast<int>(sizeof(Seg)) + 127) / 128 * 128;
  static constexpr int kBytes = kStage + 8 * 4096 + 1024;   // results on their way out, 4 KB a warp
};

struct WideBars {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], v_fixed[2];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];  // [query tile][buffer]
  uint64_t q_full[2];
  uint64_t drained;  // all products issued are done
  uint32_t bad[4];  // pages of the last tiles that are none, a bit per page
  uint32_t odd;     // segments with infinities or NaN among the values not all rows see, a bit each
  uint32_t tmem;
  int fail;
};
static_assert(sizeof(WideBars) <= 256, "between the tiles and the segments");

__device__ __forceinline__ bool given_up(const WideBars &w) { return *reinterpret_cast<const volatile int *>(&w.fail) != 0; }

// Waits for a phase. One that does not complete within the poll limit sets `fail`, and from
// then on every wait that would block returns at once: what is computed after that is
// undefined, but stays in bounds and ends. False when a role has given up.
__device__ __forceinline__ bool bar_wait(WideBars &w, uint64_t *b, uint32_t parity, int who, uint32_t polls) {
  const uint32_t addr = smem_u32(b);
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(addr), "r"(parity)
      : "memory");
  if (done) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < polls; ++i) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if (given_up(w)) return false;
  }
  *reinterpret_cast<volatile int *>(&w.fail) = 1;
  atomicExch(&g_attn_paged_status, who);
  return false;
}

// First cache row that not all rows of an item see.
__device__ __forceinline__ int not_all_see(const PagedAttnArgs &a, int base, int tok0) {
  return max(a.tree != nullptr ? base : base + tok0 + 1, 0);
}

// Adds the infinities and NaN that the product was spared to the accumulator of this thread's
// row, where it sees them: the segment's values are read once more, element by element. Rare.
template <int HD>
__device__ __noinline__ void add_not_finite(const PagedAttnArgs &a, const Seg &g, int token, bool mine, uint32_t o_addr) {
  const int first = max(not_all_see(a, g.base, g.tok0), g.t0 * kWideTile), end = min(g.kv_end, g.t1 * kWideTile);
#pragma unroll 1
  for (int c = 0; c < HD; c += 16) {
    uint32_t o[16];
    tmem_ld16(o_addr + c, o);
    tmem_wait_ld();
#pragma unroll 1
    for (int key = first; key < end; ++key) {
      const int id = __ldg(a.c.table + g.b * a.c.table_stride + (key >> a.c.page_shift));
      if (!mine || id < 0 || id >= a.c.n_pages || (seen32(a, g, token, key) & 1u) == 0u) continue;
      const int in_page = key & ((1 << a.c.page_shift) - 1);
      const uint4 *v = reinterpret_cast<const uint4 *>(
          a.c.v + id * a.c.v_page_stride + (static_cast<long long>(in_page) * a.c.n_kv + g.kvh) * HD + c);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 x = __ldcg(v + h);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t f = not_finite2(xs[e]);
          if (f & 0x8000u) o[h * 8 + 2 * e] = __float_as_uint(__uint_as_float(o[h * 8 + 2 * e]) + bf16_lo(xs[e]));
          if (f >> 31) o[h * 8 + 2 * e + 1] = __float_as_uint(__uint_as_float(o[h * 8 + 2 * e + 1]) + bf16_hi(xs[e]));
        }
      }
    }
    __syncwarp();
    tmem_st16(o_addr + c, o);
    tmem_wait_st();
  }
}

// A barrier of the whole block that the roles reach from different places.
__device__ __forceinline__ void block_sync() { asm volatile("bar.sync 0;" ::: "memory"); }

template <int HD>
__global__ void __launch_bounds__(kWideThreads, 1)
attn_paged_wide_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const __grid_constant__ PagedAttnArgs a, const int negate) {
  using L = WideLayout<HD>;
  extern __shared__ __align__(16) unsigned char wide_smem[];
  const uint32_t raw = smem_u32(wide_smem);
  unsigned char *sm = wide_smem + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t base = smem_u32(sm);
  WideBars &w = *reinterpret_cast<WideBars *>(sm + L::kBars);
  Seg *segs = reinterpret_cast<Seg *>(sm + L::kSegOff);
  __shared__ PagedWalk walk;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = gridDim.x, cta = blockIdx.x;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(&w.k_full[i], 1);
      bar_init(&w.k_empty[i], 1);
      bar_init(&w.v_full[i], 1);
      bar_init(&w.v_empty[i], 1);
      for (int j = 0; j < 2; ++j) {
        bar_init(&w.s_full[i][j], 1);
        bar_init(&w.p_full[i][j], 128);
        bar_init(&w.pv_done[i][j], 1);
      }
      bar_init(&w.q_full[i], 128);
      bar_init(&w.v_fixed[i], 1);
    }
    bar_init(&w.drained, 1);
    w.fail = 0;
    w.odd = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&k_map);
    prefetch_map(&v_map);
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&w.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = w.tmem;

  pdl_wait();
  pdl_trigger();
  zero_unowned_rows<HD>(a, cta, G);
  const int n_first = walk_begin(a, walk, segs);

  const int shift = a.c.page_shift;
  const int box = min(1 << shift, kWideTile);  // rows of one copy
  const int boxes = kWideTile / box;

  // counts that run over all segments, each role's own
  uint32_t n_kv = 0;          // key tiles (copies, products)
  uint32_t n_k = 0, n_v = 0;  // copy role: tiles requested
  uint32_t fixed = 0;         // product role: parity of each stage's zeroed tails
  uint32_t n_q[2] = {0, 0};   // segments a query tile took part in
  uint32_t n_s = 0;           // softmax role: steps of its query tile; product role: pairs of tile 0
  uint32_t n_s1 = 0;          // product role: pairs of steps of query tile 1

  // The roles part here for good, each with its own loop over the batches of segments.
  auto next_batch = [&](int n) {
    if ((n & kMore) == 0) return 0;
    block_sync();
    if (warp == 0) {
      walk_on(a, walk, segs);
      if (lane == 0) {
        w.odd = 0;
        if (w.fail != 0) walk.n_segs = 0;
      }
    }
    block_sync();
    n = walk.n_segs;
    block_sync();
    return n;
  };
  if (warp >= 8) {
    for (int n_word = n_first; n_word != 0; n_word = next_batch(n_word)) {
      const int n_now = n_word & (kMore - 1);
      bool ok = true;
      if (warp == 9) {
        // ---------------- copies ----------------
        for (int si = 0; si < n_now && ok; ++si) {
          const Seg g = segs[si];
          const int32_t *table = a.c.table + g.b * a.c.table_stride;
          for (int t = g.t0; t < g.t1 && ok; ++t, ++n_kv) {
            const int st = n_kv & 1;
            const uint32_t ph = (n_kv >> 1) & 1;
            // a page per lane; one past the item's rows, or that is none, is read as zeros
            const int row = t * kWideTile + lane * box;
            int id = a.c.n_pages;
            bool none = false;
            if (lane < boxes && row < g.kv_end) {
              id = __ldg(table + (row >> shift));
              none = id < 0 || id >= a.c.n_pages;
              if (none) id = a.c.n_pages;
            }
            const uint32_t bad = __ballot_sync(0xffffffffu, none);
            const int in_page = row & ((1 << shift) - 1);
            // (after a give-up the products no longer wait for copies, and what they commit says nothing)
            if (n_kv >= 2) ok = bar_wait(w, &w.k_empty[st], ph ^ 1, 1, a.polls) && !given_up(w);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane == 0) {
              *reinterpret_cast<volatile uint32_t *>(&w.bad[n_kv & 3]) = bad;
              bar_expect(&w.k_full[st], L::kTileB);
            }
            ++n_k;
            __syncwarp();
            if (lane < boxes) {
  #pragma unroll
              for (int h = 0; h < L::kHalves; ++h) {
                tma_page(base + L::kK + st * L::kTileB + h * L::kPiece + lane * box * 128, &k_map, &w.k_full[st], h * 64,
                         g.kvh, in_page, id);
              }
            }
            if (n_kv >= 2) ok = bar_wait(w, &w.v_empty[st], ph ^ 1, 2, a.polls) && !given_up(w);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane == 0) bar_expect(&w.v_full[st], L::kTileB);
            ++n_v;
            __syncwarp();
            if (lane < boxes) {
  #pragma unroll
              for (int h = 0; h < L::kHalves; ++h) {
                tma_page(base + L::kV + st * L::kTileB + h * L::kPiece + lane * box * 128, &v_map, &w.v_full[st], h * 64,
                         g.kvh, in_page, id);
              }
            }
            const int unseen = max(not_all_see(a, g.base, g.tok0) - t * kWideTile, 0);
            if (unseen < kWideTile) {
              // made fit for the second product: rows behind the last, which may hold anything,
              // become zeros, and so do infinities and NaN in those not all rows see
              ok = __all_sync(0xffffffffu, bar_wait(w, &w.v_full[st], ph, 3, a.polls));
              if (!ok) break;
              const int first = min(max(g.kv_end - t * kWideTile, 0), kWideTile);
              auto piece = [&](int i) {  // 16 bytes
                const int r = (i >> 3) / L::kHalves, h = (i >> 3) % L::kHalves;
                return base + L::kV + st * L::kTileB + h * L::kPiece + r * 128 + (i & 7) * 16;
              };
              uint32_t odd = 0;
#pragma unroll 8
              for (int i = unseen * 8 * L::kHalves + lane; i < first * 8 * L::kHalves; i += 32) odd |= not_finite8(lds16(piece(i)));
              for (int i = first * 8 * L::kHalves + lane; i < kWideTile * 8 * L::kHalves; i += 32) sts16(piece(i), make_uint4(0, 0, 0, 0));
              if (__any_sync(0xffffffffu, odd != 0u)) {
#pragma unroll 1
                for (int i = unseen * 8 * L::kHalves + lane; i < first * 8 * L::kHalves; i += 32) sts16(piece(i), finite8(lds16(piece(i))));
                if (lane == 0) *reinterpret_cast<volatile uint32_t *>(&w.odd) = w.odd | 1u << si;
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0) bar_arrive(&w.v_fixed[st]);
            }
          }
        }
      } else if (warp == 8) {
        // ---------------- products: a converged warp, one elected thread issues ----------------
        const uint32_t qk_desc = (1u << 4) | (1u << 7) | (1u << 10) | (negate ? 1u << 13 : 0u) |
                                 (static_cast<uint32_t>(kWideStep >> 3) << 17) | (128u >> 4 << 24);
        const uint32_t pv_desc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) |
                                 (static_cast<uint32_t>(HD >> 3) << 17) | (128u >> 4 << 24);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        // operand descriptors of the first stage; a step of 16 elements adds a constant
        const uint64_t q_desc = tc_desc(base + L::kQ, 16), k_desc = tc_desc(base + L::kK, 16);
        const uint64_t v_desc = tc_desc(base + L::kV, L::kPiece);
        auto wait = [&](uint64_t *bar, uint32_t parity, int who) { bar_wait(w, bar, parity, who, a.polls); };
        // S = Q K^T for 64 rows of a K stage; `last`: the stage's last product
        auto qk = [&](int tile, int buf, int st, int half, bool last) {
          const uint64_t qd = q_desc + (tile * L::kTileB >> 4);
          const uint64_t kd = k_desc + ((st * L::kTileB + half * kWideStep * 128) >> 4);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
              const uint32_t off = ((ks >> 2) * L::kPiece + (ks & 3) * 32) >> 4;
              tc_mma_ss(tm + tile * 128 + buf * 64, qd + off, kd + off, qk_desc, ks > 0 ? 1u : 0u);
            }
            tc_commit(&w.s_full[tile][buf]);
            if (last) tc_commit(&w.k_empty[st]);
          }
          __syncwarp();
        };
        // O += P V for 64 rows of a V stage, once P is there
        auto pv = [&](int tile, int buf, uint32_t pair, int st, int half, bool first, bool last) {
          if (!ok) return;
          const uint64_t vd = v_desc + ((st * L::kTileB + half * kWideStep * 128) >> 4);
          wait(&w.p_full[tile][buf], pair & 1, 5);
          tc_fence_after();  // P was stored by other threads
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < kWideStep / 16; ++ks) {
              tc_mma_ts(tm + 256 + tile * 128, tm + tile * 128 + buf * 64 + ks * 8, vd + (ks * 16 * 128 >> 4), pv_desc,
                        (!first || ks > 0) ? 1u : 0u);
            }
            tc_commit(&w.pv_done[tile][buf]);
            if (last) tc_commit(&w.v_empty[st]);
          }
          __syncwarp();
        };
        // what comes from shared memory is broadcast, so that it lives in uniform registers
        const int n_u = __shfl_sync(0xffffffffu, n_now, 0);
        for (int si = 0; si < n_u && ok; ++si) {
          const int t0 = __shfl_sync(0xffffffffu, segs[si].t0, 0);
          const int tiles = __shfl_sync(0xffffffffu, segs[si].t1, 0) - t0;
          const int fixed_from = __shfl_sync(0xffffffffu, not_all_see(a, segs[si].base, segs[si].tok0), 0) - t0 * kWideTile;
          const bool two = __shfl_sync(0xffffffffu, segs[si].rows, 0) > 128;
          wait(&w.q_full[0], n_q[0]++ & 1, 6);
          if (two) wait(&w.q_full[1], n_q[1]++ & 1, 6);
          wait(&w.k_full[n_kv & 1], (n_kv >> 1) & 1, 7);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            qk(0, half, n_kv & 1, half, !two && half == 1);
            if (two) qk(1, half, n_kv & 1, half, half == 1);
          }
#pragma unroll 1
          for (int i = 0; i < tiles; ++i, ++n_kv) {
            const int st = n_kv & 1;
            const bool more = i + 1 < tiles;
            wait(&w.v_full[st], (n_kv >> 1) & 1, 8);
            if ((i + 1) * kWideTile > fixed_from) {
              wait(&w.v_fixed[st], (fixed >> st) & 1u, 9);
              fixed ^= 1u << st;
            }
            if (more) wait(&w.k_full[st ^ 1], ((n_kv + 1) >> 1) & 1, 7);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              pv(0, half, n_s, st, half, i == 0 && half == 0, !two && half == 1);
              if (more) qk(0, half, st ^ 1, half, !two && half == 1);
              if (two) {
                pv(1, half, n_s1, st, half, i == 0 && half == 0, half == 1);
                if (more) qk(1, half, st ^ 1, half, half == 1);
              }
            }
            ++n_s;
            if (two) ++n_s1;
          }
          ok = __all_sync(0xffffffffu, !given_up(w));
        }
      }
    }
    // Nothing is in flight when the CTA leaves, whichever role gave up, if one did: the last copies
    // into each stage have landed, the products are done and their commits have arrived. Each wait
    // has the full limit; without a give-up all but the last commits' are over.
    if (warp == 9) {
      for (uint32_t i = n_k >= 2 ? n_k - 2 : 0; i < n_k; ++i) bar_poll(&w.k_full[i & 1], (i >> 1) & 1);
      for (uint32_t i = n_v >= 2 ? n_v - 2 : 0; i < n_v; ++i) bar_poll(&w.v_full[i & 1], (i >> 1) & 1);
    } else {
      __syncwarp();
      if (elect_one()) tc_commit(&w.drained);
      __syncwarp();
      bar_poll(&w.drained, 0);
    }
  } else {
    for (int n_word = n_first; n_word != 0; n_word = next_batch(n_word)) {
      const int n_now = n_word & (kMore - 1);
      bool ok = true;
      // ---------------- softmax: a thread per query row ----------------
      const int tile = warp >> 2;
      const int r = tid & 127;  // row of the tile, and lane of tensor memory
      const uint32_t quad = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_addr = tmem + quad + tile * 128;
      const uint32_t o_addr = tmem + quad + 256 + tile * 128;
      uint32_t seg_tiles = 0;  // key tiles of this batch before the segment
      const int first_row = tile * 128;
      // An item's queries to shared memory, K-major with the 128-byte swizzle, zeros past the last
      // row: chunk c of rows qr0, qr0 + step, ...; all requests before the first store. The
      // tile's last product with the queries before has been waited for (its scores are here).
      bool q_ahead = false;  // the next segment's are there already
      auto load_q = [&](const Seg &g) {
        constexpr int C = HD / 8, step = 128 / C;
        const int c = r % C, qr0 = r / C;
        unsigned char *dst = sm + L::kQ + tile * L::kTileB + (c >> 3) * L::kPiece;
        uint4 v[C];
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int qr = first_row + qr0 + i * step;
          const int token = token_of(a.p, g, min(qr, g.rows - 1));
          const int head = head_of(a.p, g, min(qr, g.rows - 1), token);
          v[i] = ld_act16(a.q + (g.r0 + token) * a.q_stride + head * HD + c * 8);
          if (qr >= g.rows) v[i] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int qr = qr0 + i * step;
          *reinterpret_cast<uint4 *>(dst + qr * 128 + (((c & 7) ^ (qr & 7)) << 4)) = v[i];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        bar_arrive(&w.q_full[tile]);
      };
      for (int si = 0; si < n_now && ok; ++si) {
        const Seg g = segs[si];
        const uint32_t tiles_before = seg_tiles;
        seg_tiles += g.t1 - g.t0;
        if (g.rows <= first_row) continue;
        if (!q_ahead) load_q(g);
        const bool mine = first_row + r < g.rows;
        const bool idle = first_row + (warp & 3) * 32 >= g.rows;  // no row of this warp's is one of the item's
        const int token = token_of(a.p, g, min(first_row + r, g.rows - 1));
        // cache rows that all of this warp's rows see: the older ones and, causally, the new ones
        // up to its first row's token
        const int seen_by_all =
            a.tree != nullptr ? g.base : g.base + token_of(a.p, g, min(first_row + (warp & 3) * 32, g.rows - 1)) + 1;
        float m_run = -INFINITY, l_run = 0.f;
        const float c2 = a.c2;

#pragma unroll 1
        for (int j = 0; j < 2 * (g.t1 - g.t0); ++j) {
          const int key0 = g.t0 * kWideTile + j * kWideStep;
          const uint32_t s_buf = s_addr + (n_s & 1) * 64;
          // what the row sees of a step that not all rows see whole, while the product runs
          const bool masked = key0 + kWideStep > seen_by_all;
          uint32_t see[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
          if (masked) {
            see[0] = seen32(a, g, token, key0);
            see[1] = seen32(a, g, token, key0 + 32);
          }
          bar_wait(w, &w.s_full[tile][n_s & 1], (n_s >> 1) & 1, 10, a.polls);
          __syncwarp();
          tc_fence_after();
          if (idle) {  // what the product makes of these rows is not used
            bar_arrive(&w.p_full[tile][n_s & 1]);
            ++n_s;
            continue;
          }
          uint32_t s[64];
          tmem_ld32(s_buf, s);
          tmem_ld32(s_buf + 32, s + 32);
          tmem_wait_ld();
          const uint32_t bad = *reinterpret_cast<volatile uint32_t *>(&w.bad[(n_kv + tiles_before + (j >> 1)) & 3]);
          if (masked || bad != 0u) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t m = see[k];
              if (bad != 0u) {
                for (int i = 0; i < 32; ++i) {
                  if ((bad >> (((j & 1) * kWideStep + k * 32 + i) / box)) & 1u) m &= ~(1u << i);
                }
              }
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                if (!((m >> e) & 1u)) s[k * 32 + e] = 0xFF800000u;  // -inf
              }
            }
          }
          float mx4[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            mx4[c] = fmaxf(__uint_as_float(s[c]), __uint_as_float(s[c + 4]));
#pragma unroll
            for (int e = 8; e < 64; e += 8) {
              mx4[c] = max3(mx4[c], __uint_as_float(s[e + c]), __uint_as_float(s[e + c + 4]));
            }
          }
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * c2;
          // raise the subtracted maximum only when it is far behind
          const bool raise = mx > m_run + kSlack || m_run == -INFINITY;
          const float m_new = raise ? fmaxf(mx, m_run) : m_run;
          const bool turn_down = raise && m_run != -INFINITY;
          if (__any_sync(0xffffffffu, turn_down)) {
            // The accumulator is this thread's once the last product into it is done. (That of
            // the step before, whose barrier this is too, ended before these scores began.)
            bar_wait(w, &w.pv_done[tile][(n_s - 1) & 1], ((n_s - 1) >> 1) & 1, 11, a.polls);
            __syncwarp();
            tc_fence_after();
            const float by = turn_down ? fast_exp2(m_run - m_new) : 1.f;
            l_run *= by;
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              uint32_t o[16];
              tmem_ld16(o_addr + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
              tmem_st16(o_addr + c, o);
            }
            tmem_wait_st();
          }
          m_run = m_new;
          const float m_use = m_new == -INFINITY ? 0.f : m_new;  // nothing seen so far: all -inf
          const f32x2_t c22 = pack_f32x2(c2, c2), mm2 = pack_f32x2(-m_use, -m_use);
          f32x2_t sum2 = pack_f32x2(l_run, 0.f);
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            float p0, p1;
            unpack_f32x2(ffma2(pack_f32x2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c22, mm2), p0, p1);
            p0 = fast_exp2(p0);
            p1 = fast_exp2(p1);
            sum2 = add2(sum2, pack_f32x2(p0, p1));
            const __nv_bfloat162 v = __floats2bfloat162_rn(p0, p1);
            s[e >> 1] = *reinterpret_cast<const uint32_t *>(&v);
          }
          tmem_st32(s_buf, s);
          tmem_wait_st();
          tc_fence_before();
          bar_arrive(&w.p_full[tile][n_s & 1]);
          float sum0, sum1;
          unpack_f32x2(sum2, sum0, sum1);
          l_run = sum0 + sum1;
          ++n_s;
        }
        if (!ok) break;
        // the next segment's queries, so that its first products run under what follows
        q_ahead = si + 1 < n_now && segs[si + 1].rows > first_row;
        if (q_ahead) load_q(segs[si + 1]);
        // ---- the segment's result ----
        ok = __all_sync(0xffffffffu, bar_wait(w, &w.pv_done[tile][(n_s - 1) & 1], ((n_s - 1) >> 1) & 1, 12, a.polls));
        if (!ok) break;
        tc_fence_after();
        if ((*reinterpret_cast<volatile uint32_t *>(&w.odd) >> si) & 1u) add_not_finite<HD>(a, g, token, mine, o_addr);
        // A warp's 32 rows go out 128 bytes of each at a time, through shared memory (chunk c of row
        // r at c ^ (r & 7)), so that a store covers four whole lines and not 32 pieces of 16 bytes.
        const bool whole = g.whole;
        const float by = l_run != 0.f ? 1.f / l_run : 0.f;
        const PagedWs ws = ws_of(a, G);
        const int wrow = first_row + (warp & 3) * 32;  // the warp's first row
        const long long at = (static_cast<long long>(cta) * 2 + g.slot) * kWideM + wrow;
        const int to = (g.r0 + token) * (a.p.n_kv * a.p.n_rep) + head_of(a.p, g, first_row + r, token);
        unsigned char *stage = sm + L::kStage + warp * 4096;
        const int rr = lane >> 3, cc = lane & 7;
#pragma unroll 1
        for (int c = 0; c < HD; c += whole ? 64 : 32) {
          uint32_t o[32];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && !whole) break;
            tmem_ld32(o_addr + c + h * 32, o);
            tmem_wait_ld();
            if (whole) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(o[e * 8 + 2 * i]) * by,
                                                                 __uint_as_float(o[e * 8 + 2 * i + 1]) * by);
                  v[i] = *reinterpret_cast<const uint32_t *>(&y);
                }
                *reinterpret_cast<uint4 *>(stage + lane * 128 + (((h * 4 + e) ^ (lane & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                *reinterpret_cast<uint4 *>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                    make_uint4(o[e * 4], o[e * 4 + 1], o[e * 4 + 2], o[e * 4 + 3]);
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = i * 4 + rr;
            const uint4 v = *reinterpret_cast<const uint4 *>(stage + row * 128 + ((cc ^ (row & 7)) << 4));
            const long long dst = __shfl_sync(0xffffffffu, to, row);
            if (wrow + row < g.rows) {
              if (whole) {
                *reinterpret_cast<uint4 *>(a.out + dst * HD + c + cc * 8) = v;
              } else {
                *reinterpret_cast<uint4 *>(ws.o + (at + row) * HD + c + cc * 4) = v;
              }
            }
          }
          __syncwarp();
        }
        if (mine && !whole) ws.ml[at + lane] = make_float2(m_run, l_run);
        tc_fence_before();
      }
      n_kv += seg_tiles;
    }
  }
  tc_fence_before();
  block_sync();
  tc_fence_after();
  if (warp == 8) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

}  // namespace
}  // namespace chr
