// What the kernels of cache_decode.cuh and int4_mma.cuh share: arguments, the cut of a
// sequence's candidates into tiles, and their rows.
#pragma once

#include "decode.cuh"
#include "int4.cuh"

namespace spa {

struct CacheDecodeArgs {
  const void* q;
  void* out;
  int dtype;  // of q and out
  int B, Hq, Hkv, group, D;
  const void* k;
  const void* v;
  const __half* k_scales;
  const __half* v_scales;
  KvAddr addr;
  uint32_t page_inv;  // floor((2^32 - 1) / page_size): token / page_size is one multiply
  int q_vec;          // query rows start on 16-byte boundaries
  const int32_t* ctx_lens;
  int cap;  // tokens a sequence can hold
  int local_window;
  const int64_t* selected;
  int top_m;
  int heads, chunks;  // query heads a CTA serves, such chunks per kv head
  int ctas;           // CTAs that share all tiles out evenly; 0: one CTA per pair
  float scale_log2;
  float* part_o;    // [slots, heads, D]
  float* part_lse;  // [slots, heads]
  float* scores;    // [B, Hkv, cap, group] or nullptr
  float* weights;   // [B, Hkv, T] or nullptr
  int T;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  return dtype == SPA_F32   ? static_cast<const float*>(p)[i]
         : dtype == SPA_F16 ? __half2float(static_cast<const __half*>(p)[i])
                            : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
// Eight values from element i on (a multiple of 8); vec: p is 16-byte aligned.
__device__ __forceinline__ void load8_any(const void* p, int dtype, int64_t i, int vec, float (&x)[8]) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = load_any(p, dtype, i + e);
  } else if (dtype == SPA_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned short u = static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1)));
      x[e] = dtype == SPA_F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float(static_cast<uint32_t>(u) << 16);
    }
  }
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float x) {
  if (dtype == SPA_F32)
    static_cast<float*>(p)[i] = x;
  else if (dtype == SPA_F16)
    static_cast<__half*>(p)[i] = __float2half_rn(x);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}
__device__ __forceinline__ void store4_any(void* p, int dtype, int64_t i, float4 x) {  // rows of 16 bytes' multiples
  if (dtype == SPA_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = x;
  } else if (dtype == SPA_F16) {
    const __half2 v[2] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>(static_cast<__half*>(p) + i) = *reinterpret_cast<const uint2*>(v);
  } else {
    const __nv_bfloat162 v[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + i) = *reinterpret_cast<const uint2*>(v);
  }
}
// a * b / c, in 32 bits where the product fits
__device__ __forceinline__ int64_t mul_div(int64_t a, int b, int64_t c) {
  const int64_t p = a * b;
  return (p | c) >> 32 ? p / c : static_cast<int64_t>(static_cast<uint32_t>(p) / static_cast<uint32_t>(c));
}

// Tiles of TILE tokens: the window (or the whole context), then each selected page.
struct TilePlan {
  int ctx, lo, seg, n_seg, cpp, n;
};
template <int TILE>
__device__ __forceinline__ TilePlan tile_plan(const CacheDecodeArgs& a, int b) {
  TilePlan p;
  const int ctx = a.ctx_lens[b];
  if (ctx > a.cap) spa_raise(SPA_DEVERR_BAD_PAGE);  // tokens no page of the table row can hold
  p.ctx = min(max(ctx, 0), a.cap);
  p.lo = a.selected || a.local_window > 0 ? max(0, p.ctx - a.local_window) : 0;
  p.seg = p.lo / TILE * TILE;
  p.n_seg = p.ctx > p.lo ? (p.ctx - p.seg + TILE - 1) / TILE : 0;
  p.cpp = (a.addr.page_size + TILE - 1) / TILE;
  p.n = p.n_seg + (a.selected ? a.top_m * p.cpp : 0);
  return p;
}
// Token of slot `i` of tile `tile`, or -1 (not a candidate).
template <int TILE>
__device__ __forceinline__ int tile_token(const CacheDecodeArgs& a, const TilePlan& p, int b, int tile, int i) {
  if (tile < p.n_seg) {
    const int t = p.seg + tile * TILE + i;
    return t >= p.lo && t < p.ctx ? t : -1;
  }
  const int kk = tile - p.n_seg, j = kk / p.cpp, o = (kk - j * p.cpp) * TILE + i;
  const int64_t lp = a.selected[static_cast<int64_t>(b) * a.top_m + j];
  if (lp < 0) return -1;  // an empty slot
  if (lp >= p.ctx || lp * a.addr.page_size >= p.ctx) {
    if (i == 0) spa_raise(SPA_DEVERR_BAD_PAGE);
    return -1;
  }
  const int64_t t = lp * a.addr.page_size + o;
  return o < a.addr.page_size && t < p.ctx ? static_cast<int>(t) : -1;
}
// Physical page of a token (t >= 0) or -1, and the token's place in it.
__device__ __forceinline__ int token_page(const CacheDecodeArgs& a, int b, int t, int& off) {
  // the multiply falls short by at most one
  int lp = static_cast<int>(__umulhi(static_cast<uint32_t>(t), a.page_inv));
  off = t - lp * a.addr.page_size;
  if (off >= a.addr.page_size) ++lp, off -= a.addr.page_size;
  if (!a.addr.page_table) return lp;
  return lp < a.addr.table_stride ? a.addr.page_table[static_cast<int64_t>(b) * a.addr.table_stride + lp] : -1;
}
// Row of a token in its page, or -1.
__device__ __forceinline__ int64_t page_row(const CacheDecodeArgs& a, int b, int h, int t, int page, int off) {
  if (t < 0) return -1;
  const int64_t row = b * a.addr.batch_stride_rows + page * a.addr.page_stride_rows + h * a.addr.head_stride_rows + off;
  if (page < 0 || row < 0 || row >= a.addr.total_rows) {
    spa_raise(SPA_DEVERR_BAD_PAGE);
    return -1;
  }
  return row;
}
__device__ __forceinline__ void split_range(int n, int split, int nsplit, int& t0, int& t1) {
  t0 = static_cast<int>(static_cast<int64_t>(n) * split / nsplit);
  t1 = static_cast<int>(static_cast<int64_t>(n) * (split + 1) / nsplit);
}

// ---- Sharing out the work.  A pair is a (sequence, kv head, chunk of its query heads); all of a
// sequence's pairs have its number of tiles.  The pairs' tiles, end to end, are cut into
// sharing_ctas() equal ranges, one a CTA, however the lengths are spread; a range may end inside a
// pair, so a pair's results are partials of consecutive CTAs, in slot CTA + pair (both only ever
// grow along the ranges, so no two share a slot).  A pair that one CTA covers whole needs no partial.
constexpr int kFlatBatch = 1024;  // longest batch whose prefix sums a CTA makes for itself

// The launch has a.ctas CTAs, planned from the room that the contexts may grow into; where there
// are fewer tiles than that, as many CTAs as tiles share them and the others do nothing.  Every
// range then holds a tile, so every CTA between a pair's first and last has left a partial.
__device__ __forceinline__ int sharing_ctas(const CacheDecodeArgs& a, int64_t total) {
  return total < a.ctas ? static_cast<int>(total) : a.ctas;
}

// pre[b] = tiles of one pair of each sequence before b, pre[B] the total; every thread calls it.
template <int TILE>
__device__ __forceinline__ void tiles_before(const CacheDecodeArgs& a, int* pre) {
  const int lane = threadIdx.x & 31;
  if (a.B <= 32) {
    if (threadIdx.x < 32) {
      int x = lane < a.B ? tile_plan<TILE>(a, lane).n : 0;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
      }
      pre[lane + 1] = x;
      if (lane == 0) pre[0] = 0;
    }
    __syncthreads();
    return;
  }
  for (int b = threadIdx.x; b < a.B; b += blockDim.x) pre[b + 1] = tile_plan<TILE>(a, b).n;
  __syncthreads();
  if (threadIdx.x < 32) {
    int sum = 0;
    for (int base = 0; base < a.B; base += 32) {
      int x = base + lane < a.B ? pre[base + lane + 1] : 0;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
      }
      if (base + lane < a.B) pre[base + lane + 1] = sum + x;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) pre[0] = 0;
  }
  __syncthreads();
}
struct Segment {
  int b, h, chunk, u0, u1;  // tiles [u0, u1) of a pair
  int slot;
  bool whole;  // all of the pair's tiles
};
// The range [x, x1) of this CTA, cut at the pairs' ends: one segment a call.
struct Work {
  int64_t x, x1;
  __device__ __forceinline__ Work(const CacheDecodeArgs& a, const int* pre) {
    x = 0, x1 = 1;
    if (!a.ctas) return;
    const int64_t total = static_cast<int64_t>(pre[a.B]) * a.Hkv * a.chunks;
    const int ctas = sharing_ctas(a, total), i = blockIdx.x;
    if (i >= ctas) {
      x1 = 0;
      return;
    }
    x = mul_div(total, i, ctas);
    x1 = mul_div(total, i + 1, ctas);
  }
  template <int TILE>
  __device__ __forceinline__ bool next(const CacheDecodeArgs& a, const int* pre, Segment& s) {
    if (x >= x1) return false;
    const int pairs = a.Hkv * a.chunks;
    int pair = blockIdx.x;
    if (a.ctas) {
      int lo = 0, hi = a.B;  // the last sequence that starts at or before x and is not empty
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (static_cast<int64_t>(pre[mid]) * pairs <= x)
          lo = mid;
        else
          hi = mid;
      }
      const int n = pre[lo + 1] - pre[lo];
      const int64_t y = x - static_cast<int64_t>(pre[lo]) * pairs;
      const int hc = static_cast<int>(mul_div(y, 1, n));
      s.u0 = static_cast<int>(y - static_cast<int64_t>(hc) * n);
      s.u1 = static_cast<int>(min(static_cast<int64_t>(n), s.u0 + (x1 - x)));
      s.whole = s.u1 - s.u0 == n;
      x += s.u1 - s.u0;
      pair = lo * pairs + hc;
    } else {
      s.u0 = 0;
      s.u1 = tile_plan<TILE>(a, pair / pairs).n;
      s.whole = true;
      x = x1;
    }
    s.slot = blockIdx.x + pair;
    s.b = pair / pairs;
    pair -= s.b * pairs;
    s.h = pair / a.chunks;
    s.chunk = pair - s.h * a.chunks;
    return true;
  }
};
// CTAs [first, last] of `ctas` <= total that hold tiles [at, at + n) of all `total`, n > 0
__device__ __forceinline__ void ctas_of(int64_t at, int n, int64_t total, int ctas, int& first, int& last) {
  // the last CTA whose range starts at or before tile x: the largest i with total i / ctas <= x
  const auto cta = [&](int64_t x) {
    const int64_t p = (x + 1) * ctas - 1;
    return static_cast<int>((p | total) >> 32 ? p / total
                                              : static_cast<int64_t>(static_cast<uint32_t>(p) / static_cast<uint32_t>(total)));
  };
  first = cta(at);
  last = cta(at + n - 1);
}

// Joins the partial results of a CTA's W warps: buf holds [W][HN][D + 4] rows of D outputs, the
// maximum (log2) and the sum; writes the pair's output, or the segment's partial.
template <int W, int HN, int D>
__device__ __forceinline__ void merge_warps(const CacheDecodeArgs& a, const Segment& seg, int64_t q0, int heads,
                                            const float* buf, float (*s_f)[16]) {
  constexpr int kLd = D + 4;
  const int tid = threadIdx.x;
  __syncthreads();
  const bool partial = a.weights || !seg.whole;
  if (tid < HN * 16) {  // a head's warps side by side: their shares of the whole
    const int n = tid >> 4, w = tid & 15;
    const float* row = buf + (w * HN + n) * kLd + D;
    const float mw = w < W ? row[0] : -INFINITY, lw = w < W ? row[1] : 0.f;
    float M = mw;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
    float sum = lw * f;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    // no token at all (sum 0): zeros
    s_f[n][w] = sum == 0.f ? 0.f : f / sum;
    if (partial && w == 0 && n < heads)
      a.part_lse[static_cast<int64_t>(seg.slot) * HN + n] = sum == 0.f ? -INFINITY : M + log2f(sum);
  }
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < heads * (D / 4); i += W * 32) {
    const int n = i / (D / 4), d = i % (D / 4) * 4;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int w = 0; w < W; ++w) {
      const float f = s_f[n][w];
      const float4 v = *reinterpret_cast<const float4*>(buf + (w * HN + n) * kLd + d);
      r.x = fmaf(v.x, f, r.x), r.y = fmaf(v.y, f, r.y), r.z = fmaf(v.z, f, r.z), r.w = fmaf(v.w, f, r.w);
    }
    if (partial)
      *reinterpret_cast<float4*>(a.part_o + (static_cast<int64_t>(seg.slot) * HN + n) * D + d) = r;
    else
      store4_any(a.out, a.dtype, (q0 + n) * D + d, r);
  }
}

}  // namespace spa
