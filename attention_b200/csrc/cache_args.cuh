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
  int heads, chunks;  // query heads a CTA serves, CTAs per kv head
  int nsplit;
  float scale_log2;
  float* part_o;    // [B*Hq, nsplit, D]
  float* part_lse;  // [B*Hq, nsplit]
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
// Row of a token, or -1; `ahead`: the tokens from it on that share its page and are in the context.
__device__ __forceinline__ int64_t token_row(const CacheDecodeArgs& a, int b, int h, int t, int ctx, int& ahead) {
  ahead = 0;
  if (t < 0) return -1;
  // the multiply falls short by at most one
  int lp = static_cast<int>(__umulhi(static_cast<uint32_t>(t), a.page_inv)), off = t - lp * a.addr.page_size;
  if (off >= a.addr.page_size) ++lp, off -= a.addr.page_size;
  const int64_t pg = a.addr.page_of(b, lp);
  const int64_t row =
      pg < 0 ? -1 : b * a.addr.batch_stride_rows + pg * a.addr.page_stride_rows + h * a.addr.head_stride_rows + off;
  if (row < 0 || row >= a.addr.total_rows) {
    spa_raise(SPA_DEVERR_BAD_PAGE);
    return -1;
  }
  ahead = min(a.addr.page_size - off, ctx - t);
  return row;
}
__device__ __forceinline__ void split_range(int n, int split, int nsplit, int& t0, int& t1) {
  t0 = static_cast<int>(static_cast<int64_t>(n) * split / nsplit);
  t1 = static_cast<int>(static_cast<int64_t>(n) * (split + 1) / nsplit);
}

}  // namespace spa
