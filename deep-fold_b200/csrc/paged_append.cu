// Rows appended to a paged KV cache, with the rotary positions applied on the way
// (sm_100a). No counterpart in the reference, whose cache is one contiguous block
// per sequence (gpu/decodev2/kv.py:14-120) and whose rotation is the rotate-half form
// over the whole head (gpu/nf4/nf4_gemv.cu:497-537).
//
// Row t belongs to sequence s = seq[t], takes cache row a = slot[t] of it and is
// rotated for position p = position[t] (a when there is none):
//   half         (x_i, x_{i+r/2}) -> (x_i c_i - x_{i+r/2} s_i, x_{i+r/2} c_i + x_i s_i)
//   interleaved  (x_2i, x_2i+1)   -> (x_2i c_i - x_2i+1 s_i,   x_2i+1 c_i + x_2i s_i)
// with c_i, s_i = cos, sin[p, i], i < r/2; elements r.. of a head pass through. The
// products and their sum are FP32 and rounded to bf16 once, the cache's type.
//
// Bound by memory: every q, k and v element is read once and written once. A thread
// takes one 16-byte piece of a head (two for the half layout, whose partner elements
// sit r/2 further on), so all of a row's accesses are 16 bytes wide; rows share nothing
// but the table row, which stays in L1. q and k are requested before the chain
// seq -> page table -> destination is resolved, so the two latencies overlap. 7,000 rows
// of 48 + 2 x 8 heads of 128 (228 MB): 43.8 us, 5.2 TB/s; one row 2.1 us, 64 rows 2.6.

#include "paged.cuh"

namespace chr {
namespace {

constexpr int kAppendThreads = 256;

struct AppendArgs {
  PagedCache c;
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16 *q_out;
  long long q_stride, k_stride, v_stride, q_out_stride;
  const void *cos, *sin;
  long long tab_stride;
  const int32_t *seq;
  const int64_t *slot, *position;
  int T, n_q, rot, tab_rows, zero_skipped;
};

template <bool F32>
__device__ __forceinline__ float tab1(const void *tab, long long i) {
  if (F32) return __ldg(static_cast<const float *>(tab) + i);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(tab)[i]);
}

// N consecutive table values (N = 4 or 8), 16-byte (or 8-byte) loads.
template <bool F32, int N>
__device__ __forceinline__ void tab_vec(const void *tab, long long i, float (&out)[N]) {
  if (F32) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const float4 f = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(tab) + i) + j);
      out[4 * j] = f.x;
      out[4 * j + 1] = f.y;
      out[4 * j + 2] = f.z;
      out[4 * j + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const uint2 w =
          __ldg(reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(tab) + i) + j);
      out[4 * j] = bf16_lo(w.x);
      out[4 * j + 1] = bf16_hi(w.x);
      out[4 * j + 2] = bf16_lo(w.y);
      out[4 * j + 3] = bf16_hi(w.y);
    }
  }
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// (lo, hi) -> the rotated pair, one rounding each at the caller
__device__ __forceinline__ void turn(float a, float b, float c, float s, float &oa, float &ob) {
  oa = a * c - b * s;
  ob = b * c + a * s;
}

// Where row t goes; false: nowhere (outside the batch, the table, the pool or the
// positions the tables cover).
struct Place {
  long long k_off, v_off;  // first element of (page, row in page) in the two pools
  long long pos;
};
__device__ __forceinline__ bool place_of(const AppendArgs &a, int t, Place &p) {
  const int s = a.seq != nullptr ? __ldg(a.seq + t) : t;
  const long long slot = __ldg(reinterpret_cast<const long long *>(a.slot) + t);
  p.pos = a.position != nullptr ? __ldg(reinterpret_cast<const long long *>(a.position) + t) : slot;
  if (s < 0 || s >= a.c.batch || slot < 0 || p.pos < 0 || p.pos >= a.tab_rows) return false;
  const long long page = slot >> a.c.page_shift;
  if (page >= a.c.max_pages) return false;
  const int id = __ldg(a.c.table + s * a.c.table_stride + page);
  if (id < 0 || id >= a.c.n_pages) return false;
  const long long in = (slot & ((1ll << a.c.page_shift) - 1)) * a.c.n_kv * a.c.hd;
  p.k_off = id * a.c.k_page_stride + in;
  p.v_off = id * a.c.v_page_stride + in;
  return true;
}

// Grid (rows, pieces of the row / threads). VEC: 16-byte pieces (hd and the rotated
// part made of whole pieces, every row 16-byte aligned); otherwise one element pair
// (or one passed-through element) per thread and step.
template <bool VEC, bool INTER, bool F32>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x;
  const int hd = a.c.hd, n_kv = a.c.n_kv;
  const int half = a.rot >> 1;
  // units of one rotated head: the rotated part, then the part that passes through
  const int turned = VEC ? (INTER ? a.rot / 8 : half / 8) : half;
  const int per_head = turned + (VEC ? (hd - a.rot) / 8 : hd - a.rot);
  const int per_v = VEC ? hd / 8 : hd;
  const int n_rot = (a.n_q + n_kv) * per_head;
  const int units = n_rot + n_kv * per_v;
  Place p{};
  bool live = false, known = false;
  for (int u = blockIdx.y * blockDim.x + threadIdx.x; u < units; u += gridDim.y * blockDim.x) {
    const bool is_v = u >= n_rot;
    const int w = is_v ? u - n_rot : u;
    const int head = w / (is_v ? per_v : per_head);
    const int piece = w - head * (is_v ? per_v : per_head);
    const bool is_q = !is_v && head < a.n_q;
    const __nv_bfloat16 *src;
    if (is_v) {
      src = a.v + t * a.v_stride + head * hd;
    } else if (is_q) {
      src = a.q + t * a.q_stride + head * hd;
    } else {
      src = a.k + t * a.k_stride + (head - a.n_q) * hd;
    }
    const bool turns = !is_v && piece < turned;
    int e0, e1;  // first element(s) of this unit
    if (VEC) {
      e0 = is_v ? piece * 8 : (turns ? piece * 8 : a.rot + (piece - turned) * 8);
      e1 = e0 + half;  // half layout only
    } else {
      e0 = is_v ? piece : (turns ? (INTER ? 2 * piece : piece) : a.rot + piece - turned);
      e1 = INTER ? e0 + 1 : e0 + half;
    }
    uint4 x0{}, x1{};
    __nv_bfloat16 y0{}, y1{};
    if (VEC) {
      x0 = ld_act16(src + e0);
      if (turns && !INTER) x1 = ld_act16(src + e1);
    } else {
      y0 = src[e0];
      if (turns) y1 = src[e1];
    }
    if (!known) {
      live = place_of(a, t, p);
      known = true;
    }
    __nv_bfloat16 *dst;
    if (is_q) {
      dst = a.q_out + t * a.q_out_stride + head * hd;
    } else if (is_v) {
      dst = a.c.v + p.v_off + head * hd;
    } else {
      dst = a.c.k + p.k_off + (head - a.n_q) * hd;
    }
    if (!live) {
      if (is_q && a.zero_skipped) {
        if (VEC) {
          *reinterpret_cast<uint4 *>(dst + e0) = make_uint4(0, 0, 0, 0);
          if (turns && !INTER) *reinterpret_cast<uint4 *>(dst + e1) = make_uint4(0, 0, 0, 0);
        } else {
          dst[e0] = __float2bfloat16(0.f);
          if (turns) dst[e1] = __float2bfloat16(0.f);
        }
      }
      continue;
    }
    if (VEC) {
      if (turns) {
        const long long at = p.pos * a.tab_stride + (INTER ? piece * 4 : piece * 8);
        const uint32_t xs[4] = {x0.x, x0.y, x0.z, x0.w};
        uint32_t o[4];
        if (INTER) {
          float c[4], s[4];
          tab_vec<F32, 4>(a.cos, at, c);
          tab_vec<F32, 4>(a.sin, at, s);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float oa, ob;
            turn(bf16_lo(xs[e]), bf16_hi(xs[e]), c[e], s[e], oa, ob);
            o[e] = pack2(oa, ob);
          }
          *reinterpret_cast<uint4 *>(dst + e0) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
          const uint32_t zs[4] = {x1.x, x1.y, x1.z, x1.w};
          uint32_t o2[4];
          float c[8], s[8];
          tab_vec<F32, 8>(a.cos, at, c);
          tab_vec<F32, 8>(a.sin, at, s);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a0, b0, a1, b1;
            turn(bf16_lo(xs[e]), bf16_lo(zs[e]), c[2 * e], s[2 * e], a0, b0);
            turn(bf16_hi(xs[e]), bf16_hi(zs[e]), c[2 * e + 1], s[2 * e + 1], a1, b1);
            o[e] = pack2(a0, a1);
            o2[e] = pack2(b0, b1);
          }
          *reinterpret_cast<uint4 *>(dst + e0) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4 *>(dst + e1) = make_uint4(o2[0], o2[1], o2[2], o2[3]);
        }
      } else {
        *reinterpret_cast<uint4 *>(dst + e0) = x0;
      }
    } else if (turns) {
      const long long at = p.pos * a.tab_stride + piece;
      float oa, ob;
      turn(__bfloat162float(y0), __bfloat162float(y1), tab1<F32>(a.cos, at), tab1<F32>(a.sin, at), oa, ob);
      dst[e0] = __float2bfloat16(oa);
      dst[e1] = __float2bfloat16(ob);
    } else {
      dst[e0] = y0;
    }
  }
}

}  // namespace
}  // namespace chr

using namespace chr;

extern "C" int chr_nf4_rope_kv_paged(const chr_nf4_rope_kv_paged_t *args, void *stream) {
  if (args == nullptr) return kNull;
  const chr_nf4_rope_kv_paged_t &r = *args;
  if (r.k == nullptr || r.v == nullptr || r.cos == nullptr || r.sin == nullptr ||
      r.slot == nullptr || (r.n_q > 0 && (r.q == nullptr || r.q_out == nullptr))) {
    return kNull;
  }
  AppendArgs a{};
  const int rc = paged_cache(&r.pages, a.c);
  if (rc != kOk) return rc;
  const long long q_row = static_cast<long long>(r.n_q) * a.c.hd;
  const long long kv_row = static_cast<long long>(a.c.n_kv) * a.c.hd;
  if (r.T < 1 || r.T > (1 << 30) || r.n_q < 0 || r.rot < 2 || (r.rot & 1) != 0 || r.rot > a.c.hd || r.tab_rows < 1 ||
      r.tab_stride < r.rot / 2 || r.q_stride < q_row || r.q_out_stride < q_row || r.k_stride < kv_row ||
      r.v_stride < kv_row || (r.n_q + 2ll * a.c.n_kv) * a.c.hd > (1 << 24) ||
      (r.seq == nullptr && r.T > a.c.batch)) {
    return kDims;
  }
  a.q = static_cast<const __nv_bfloat16 *>(r.q);
  a.k = static_cast<const __nv_bfloat16 *>(r.k);
  a.v = static_cast<const __nv_bfloat16 *>(r.v);
  a.q_out = static_cast<__nv_bfloat16 *>(r.q_out);
  a.q_stride = r.q_stride;
  a.k_stride = r.k_stride;
  a.v_stride = r.v_stride;
  a.q_out_stride = r.q_out_stride;
  a.cos = r.cos;
  a.sin = r.sin;
  a.tab_stride = r.tab_stride;
  a.seq = static_cast<const int32_t *>(r.seq);
  a.slot = static_cast<const int64_t *>(r.slot);
  a.position = static_cast<const int64_t *>(r.position);
  a.T = r.T;
  a.n_q = r.n_q;
  a.rot = r.rot;
  a.tab_rows = r.tab_rows;
  a.zero_skipped = r.zero_skipped != 0;
  // 16-byte pieces where every head, its rotated part and every row are made of them: 7,000 rows
  // take 44 us by pieces and 150 by elements, 64 rows 2.6 and 4.5
  const int tab_align = r.tab_f32 != 0 ? 16 : 8;
  const bool vec =
      a.c.hd % 8 == 0 && (r.interleaved != 0 ? r.rot % 8 == 0 : r.rot % 16 == 0) &&
      (r.n_q == 0 || (aligned(r.q, 16) && aligned(r.q_out, 16) && r.q_stride % 8 == 0 && r.q_out_stride % 8 == 0)) &&
      aligned(r.k, 16) && aligned(r.v, 16) && r.k_stride % 8 == 0 && r.v_stride % 8 == 0 &&
      aligned(a.c.k, 16) && aligned(a.c.v, 16) && a.c.k_page_stride % 8 == 0 &&
      a.c.v_page_stride % 8 == 0 && aligned(r.cos, tab_align) && aligned(r.sin, tab_align) &&
      r.tab_stride % 4 == 0;
  const int half = r.rot / 2;
  const int per_head = vec ? (r.interleaved != 0 ? r.rot / 8 : half / 8) + (a.c.hd - r.rot) / 8 : a.c.hd - half;
  const int units = (r.n_q + a.c.n_kv) * per_head + a.c.n_kv * (vec ? a.c.hd / 8 : a.c.hd);
  // few rows: a row is spread over CTAs until the SMs have one each (64 rows: 2.6 us, 3.0 without)
  int split = (units + kAppendThreads - 1) / kAppendThreads;
  const int most = (2 * sm_count() + r.T - 1) / r.T;
  split = split > most ? most : split;
  const dim3 grid(static_cast<unsigned>(r.T), static_cast<unsigned>(split < 1 ? 1 : split));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define CHR_APPEND(V, I, F) e = launch_chain(append_kernel<V, I, F>, grid, dim3(kAppendThreads), 0, st, a)
  if (vec) {
    if (r.interleaved != 0) {
      if (r.tab_f32 != 0) CHR_APPEND(true, true, true); else CHR_APPEND(true, true, false);
    } else {
      if (r.tab_f32 != 0) CHR_APPEND(true, false, true); else CHR_APPEND(true, false, false);
    }
  } else {
    if (r.interleaved != 0) {
      if (r.tab_f32 != 0) CHR_APPEND(false, true, true); else CHR_APPEND(false, true, false);
    } else {
      if (r.tab_f32 != 0) CHR_APPEND(false, false, true); else CHR_APPEND(false, false, false);
    }
  }
#undef CHR_APPEND
  return e == cudaSuccess ? kOk : kLaunch;
}
