// Decode attention over the 4-bit cache, and decode attention that accumulates each
// token's weight (4-bit and plain caches).
//
// The candidates of a sequence (its context, its local window, or window and selected pages)
// are cut into tiles that never straddle a selected page; the tiles of one (sequence, kv
// head) are shared out over `nsplit` CTAs and, inside a CTA, over its warps, each of which
// keeps its own running maximum and sum.  A CTA merges its warps in shared memory; splits
// leave (output, log2-sum-exp) partials that cache_decode_finish_kernel joins.  With weights
// the scores are kept as well (fp32, one per query head and token: 16 bytes a token at four
// heads per kv head, against 160 or 512 of K and V), because a token's weight needs the
// final log-sum-exp; the finish kernel turns them into probabilities and adds them up.
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
// Row of a token, or -1.
__device__ __forceinline__ int64_t token_row(const CacheDecodeArgs& a, int b, int h, int t) {
  if (t < 0) return -1;
  const int64_t row = a.addr.row(b, h, t);
  if (row < 0 || row >= a.addr.total_rows) {
    spa_raise(SPA_DEVERR_BAD_PAGE);
    return -1;
  }
  return row;
}
__device__ __forceinline__ void split_range(int n, int split, int nsplit, int& t0, int& t1) {
  t0 = static_cast<int>(static_cast<int64_t>(n) * split / nsplit);
  t1 = static_cast<int>(static_cast<int64_t>(n) * (split + 1) / nsplit);
}

// ---------------------------------------------------------------------------
// CUDA-core kernel: any head_dim up to 256, any cache type.  Lane l holds the values
// d = l + 32 e; a warp takes a tile of 32 tokens, one token after another.
constexpr int kPlainHeads = 4, kPlainWarps = 4;

template <typename T, int E>  // T = uint8_t: the 4-bit cache
__global__ void __launch_bounds__(kPlainWarps * 32) cache_decode_plain_kernel(const CacheDecodeArgs a) {
  const int split = blockIdx.x, h = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks, b = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = a.D;
  const int head0 = chunk * kPlainHeads, heads = min(kPlainHeads, a.group - head0);
  const int64_t q0 = static_cast<int64_t>(b) * a.Hq + h * a.group + head0;
  float q[kPlainHeads][E], acc[kPlainHeads][E], m[kPlainHeads], l[kPlainHeads];
#pragma unroll
  for (int n = 0; n < kPlainHeads; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + 32 * e;
      q[n][e] = n < heads && d < D ? load_any(a.q, a.dtype, (q0 + n) * D + d) : 0.f;
      acc[n][e] = 0.f;
    }
  }
  const TilePlan p = tile_plan<32>(a, b);
  int t0, t1;
  split_range(p.n, split, a.nsplit, t0, t1);
  const auto value = [&](const void* base, const __half* scales, int64_t row, int e) -> float {
    const int d = lane + 32 * e;
    if constexpr (sizeof(T) == 1) {
      const int G = D / kInt4Group;
      if (e >= G) return 0.f;
      const uint32_t word = static_cast<const uint16_t*>(base)[row * (G * 8) + (lane >> 2) * G + e];
      const __half* s = scales + row * 2 * G + e;
      return fmaf(__half2float(s[0]), static_cast<float>((word >> (4 * (lane & 3))) & 15u), __half2float(s[G]));
    } else {
      return d < D ? to_f32<T>(static_cast<const T*>(base)[row * D + d]) : 0.f;
    }
  };
  for (int tile = t0 + warp; tile < t1; tile += kPlainWarps) {
    const int tok = tile_token<32>(a, p, b, tile, lane);
    const int64_t my_row = token_row(a, b, h, tok);
    unsigned live = __ballot_sync(0xffffffffu, my_row >= 0);
    if (a.scores && tok >= 0 && my_row < 0)
      for (int n = 0; n < heads; ++n)
        a.scores[((static_cast<int64_t>(b) * a.Hkv + h) * a.cap + tok) * a.group + head0 + n] = -INFINITY;
    while (live) {
      const int i = __ffs(live) - 1;
      live &= live - 1;
      const int64_t row = __shfl_sync(0xffffffffu, my_row, i);
      const int t = __shfl_sync(0xffffffffu, tok, i);
      float kv[E], s[kPlainHeads];
#pragma unroll
      for (int e = 0; e < E; ++e) kv[e] = value(a.k, a.k_scales, row, e);
#pragma unroll
      for (int n = 0; n < kPlainHeads; ++n) {
        s[n] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s[n] = fmaf(q[n][e], kv[e], s[n]);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1)
#pragma unroll
        for (int n = 0; n < kPlainHeads; ++n) s[n] += __shfl_xor_sync(0xffffffffu, s[n], off);
#pragma unroll
      for (int e = 0; e < E; ++e) kv[e] = value(a.v, a.v_scales, row, e);
#pragma unroll
      for (int n = 0; n < kPlainHeads; ++n) {
        s[n] *= a.scale_log2;
        const float mn = fmaxf(m[n], s[n]);
        // a first score of -inf leaves nothing to weigh: the difference would be NaN
        const float alpha = m[n] == -INFINITY ? 0.f : exp2f(m[n] - mn), pr = s[n] == -INFINITY ? 0.f : exp2f(s[n] - mn);
        l[n] = l[n] * alpha + pr;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[n][e] = fmaf(acc[n][e], alpha, pr * kv[e]);
        m[n] = mn;
      }
      if (a.scores && lane == 0)
        for (int n = 0; n < heads; ++n)
          a.scores[((static_cast<int64_t>(b) * a.Hkv + h) * a.cap + t) * a.group + head0 + n] = s[n];
    }
  }
  // merge the warps
  __shared__ float sm[kPlainWarps][kPlainHeads], sl[kPlainWarps][kPlainHeads], so[kPlainWarps][kPlainHeads][E * 32];
#pragma unroll
  for (int n = 0; n < kPlainHeads; ++n) {
    if (lane == 0) sm[warp][n] = m[n], sl[warp][n] = l[n];
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][n][lane + 32 * e] = acc[n][e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += kPlainWarps * 32) {
    const int n = i / D, d = i % D;
    float M = -INFINITY, W = 0.f, O = 0.f;
    for (int w = 0; w < kPlainWarps; ++w) M = fmaxf(M, sm[w][n]);
    for (int w = 0; w < kPlainWarps; ++w) {
      const float f = sm[w][n] == -INFINITY ? 0.f : exp2f(sm[w][n] - M);
      W = fmaf(sl[w][n], f, W);
      O = fmaf(so[w][n][d], f, O);
    }
    const float o = W == 0.f ? 0.f : O / W;
    if (a.part_o) {
      a.part_o[((q0 + n) * a.nsplit + split) * D + d] = o;
      if (d == 0) a.part_lse[(q0 + n) * a.nsplit + split] = W == 0.f ? -INFINITY : M + log2f(W);
    } else {
      store_any(a.out, a.dtype, (q0 + n) * D + d, o);
    }
  }
}

// ---------------------------------------------------------------------------
// Joins the splits and, with weights, adds every token's probabilities to its weight.
// Grid (group + token blocks, Hkv, B): block x < group merges one head's output.
constexpr int kFinishThreads = 256, kFinishTokens = 1024;

__global__ void __launch_bounds__(kFinishThreads) cache_decode_finish_kernel(const CacheDecodeArgs a) {
  pdl_block();
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, ns = a.nsplit;
  const int64_t q0 = static_cast<int64_t>(b) * a.Hq + h * a.group;
  __shared__ float s_lse[256];
  if (blockIdx.x < a.group) {
    const int64_t bh = q0 + blockIdx.x;
    float M = -INFINITY, W = 0.f;
    for (int s = 0; s < ns; ++s) M = fmaxf(M, a.part_lse[bh * ns + s]);
    for (int s = 0; s < ns; ++s) {
      const float x = a.part_lse[bh * ns + s];
      W += x == -INFINITY ? 0.f : exp2f(x - M);
    }
    for (int d = tid; d < a.D; d += kFinishThreads) {
      float O = 0.f;
      for (int s = 0; s < ns; ++s) {
        const float x = a.part_lse[bh * ns + s];
        if (x != -INFINITY) O = fmaf(a.part_o[(bh * ns + s) * a.D + d], exp2f(x - M), O);
      }
      store_any(a.out, a.dtype, bh * a.D + d, W == 0.f ? 0.f : O / W);
    }
    return;
  }
  const int ctx = min(max(a.ctx_lens[b], 0), a.cap);
  const int lo = a.local_window > 0 ? max(0, ctx - a.local_window) : 0;
  const int t0 = lo + (blockIdx.x - a.group) * kFinishTokens;
  if (t0 >= ctx) return;
  for (int n = tid; n < a.group; n += kFinishThreads) {
    float M = -INFINITY, W = 0.f;
    for (int s = 0; s < ns; ++s) M = fmaxf(M, a.part_lse[(q0 + n) * ns + s]);
    for (int s = 0; s < ns; ++s) {
      const float x = a.part_lse[(q0 + n) * ns + s];
      W += x == -INFINITY ? 0.f : exp2f(x - M);
    }
    s_lse[n] = W == 0.f ? INFINITY : M + log2f(W);
  }
  __syncthreads();
  const int64_t bh = static_cast<int64_t>(b) * a.Hkv + h;
  for (int t = t0 + tid; t < min(t0 + kFinishTokens, ctx); t += kFinishThreads) {
    if (t >= a.T) {
      spa_raise(SPA_DEVERR_BAD_INDEX);
      continue;
    }
    const float* s = a.scores + (bh * a.cap + t) * a.group;
    float w = 0.f;
    for (int n = 0; n < a.group; ++n) w += exp2f(s[n] - s_lse[n]);
    a.weights[bh * a.T + t] += w;
  }
}

// ---------------------------------------------------------------------------
// host planning
struct CachePlan {
  bool fast;
  int heads, chunks, nsplit;
};
inline CachePlan cache_plan(int batch, int q_heads, int kv_heads, int head_dim, int max_candidates, bool int4,
                            int cache_dtype) {
  CachePlan p;
  (void)head_dim;
  (void)int4;
  (void)cache_dtype;
  const int group = q_heads / kv_heads;
  p.fast = false;
  p.heads = kPlainHeads;
  p.chunks = (group + p.heads - 1) / p.heads;
  const int64_t ctas = static_cast<int64_t>(batch) * kv_heads * p.chunks;
  const int64_t slots = device_sm_count() * 4;
  const int64_t most = max_candidates / 32 / kPlainWarps + 1;
  int64_t ns = slots / ctas;
  if (ns > most) ns = most;
  if (ns > 64) ns = 64;
  p.nsplit = ns < 1 ? 1 : static_cast<int>(ns);
  return p;
}
inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct CacheScratch {
  size_t part_o, part_lse, scores, total;
};
inline CacheScratch cache_scratch(const CachePlan& p, int batch, int q_heads, int head_dim, int cap, bool weights) {
  CacheScratch s{};
  const size_t parts = weights || p.nsplit > 1 ? static_cast<size_t>(batch) * q_heads * p.nsplit : 0;
  s.part_o = 0;
  s.part_lse = align256(parts * head_dim * sizeof(float));
  s.scores = s.part_lse + align256(parts * sizeof(float));
  s.total = s.scores + (weights ? align256(static_cast<size_t>(batch) * q_heads * cap * sizeof(float)) : 0);
  return s;
}

template <typename T>
int launch_cache_plain(const CacheDecodeArgs& a, cudaStream_t st) {
  const dim3 grid(a.nsplit, a.Hkv * a.chunks, a.B);
  const int e = (a.D + 31) / 32;
  if (e <= 1)
    cache_decode_plain_kernel<T, 1><<<grid, kPlainWarps * 32, 0, st>>>(a);
  else if (e <= 2)
    cache_decode_plain_kernel<T, 2><<<grid, kPlainWarps * 32, 0, st>>>(a);
  else if (e <= 4)
    cache_decode_plain_kernel<T, 4><<<grid, kPlainWarps * 32, 0, st>>>(a);
  else
    cache_decode_plain_kernel<T, 8><<<grid, kPlainWarps * 32, 0, st>>>(a);
  SPA_CHECK_CUDA(cudaGetLastError());
  return SPA_OK;
}

// kv dtype: SPA_F32/F16/BF16 of a plain cache, or -1 for the 4-bit one.
int cache_decode_impl(CacheDecodeArgs a, int kv_dtype, const spa_kv_layout* kv, int max_candidates, double scale,
                      void* workspace, size_t workspace_bytes, spa_stream_t stream) {
  if (!a.q || !a.out || !a.ctx_lens || !kv || !kv->k || !kv->v || !dtype_ok(a.dtype)) return SPA_ERR_INVALID;
  if (a.B <= 0 || a.B > 65535 || a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv || a.D <= 0 || a.D > 256 ||
      max_candidates < 0 || a.cap <= 0 || a.local_window < 0)
    return SPA_ERR_INVALID;
  if (kv->page_size <= 0 || kv->total_rows <= 0 || (kv->page_table && kv->table_stride <= 0)) return SPA_ERR_INVALID;
  if ((a.selected && a.top_m <= 0) || (a.weights && (a.T <= 0 || a.selected))) return SPA_ERR_INVALID;
  a.group = a.Hq / a.Hkv;
  if (a.group > 256) return SPA_ERR_UNSUPPORTED;
  const CachePlan p = cache_plan(a.B, a.Hq, a.Hkv, a.D, max_candidates, kv_dtype < 0, kv_dtype);
  if (static_cast<int64_t>(a.Hkv) * p.chunks > 65535) return SPA_ERR_UNSUPPORTED;
  const CacheScratch s = cache_scratch(p, a.B, a.Hq, a.D, a.cap, a.weights != nullptr);
  if (s.total && (!workspace || workspace_bytes < s.total || reinterpret_cast<uintptr_t>(workspace) % 16))
    return SPA_ERR_WORKSPACE;
  a.k = kv->k;
  a.v = kv->v;
  a.addr = make_kv_addr(*kv);
  a.heads = p.heads;
  a.chunks = p.chunks;
  a.nsplit = p.nsplit;
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const bool parts = a.weights || a.nsplit > 1;
  a.part_o = parts ? reinterpret_cast<float*>(ws + s.part_o) : nullptr;
  a.part_lse = parts ? reinterpret_cast<float*>(ws + s.part_lse) : nullptr;
  a.scores = a.weights ? reinterpret_cast<float*>(ws + s.scores) : nullptr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int rc;
  if (kv_dtype < 0)
    rc = launch_cache_plain<uint8_t>(a, st);
  else if (kv_dtype == SPA_F32)
    rc = launch_cache_plain<float>(a, st);
  else if (kv_dtype == SPA_F16)
    rc = launch_cache_plain<__half>(a, st);
  else
    rc = launch_cache_plain<__nv_bfloat16>(a, st);
  if (rc || !parts) return rc;
  const int span = a.local_window > 0 && a.local_window < a.cap ? a.local_window : a.cap;
  const int blocks = a.group + (a.weights ? (span + kFinishTokens - 1) / kFinishTokens : 0);
  SPA_CHECK_CUDA(launch_pdl(cache_decode_finish_kernel, dim3(blocks, a.Hkv, a.B), dim3(kFinishThreads), 0, st, true, a));
  return SPA_OK;
}

}  // namespace spa

extern "C" size_t spa_cache_decode_workspace_size(int batch, int q_heads, int kv_heads, int head_dim,
                                                  int max_candidates, int max_tokens, int weights, int kv_dtype) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0 || max_candidates < 0 ||
      max_tokens <= 0)
    return 0;
  const spa::CachePlan p = spa::cache_plan(batch, q_heads, kv_heads, head_dim, max_candidates, kv_dtype < 0, kv_dtype);
  return spa::cache_scratch(p, batch, q_heads, head_dim, max_tokens, weights != 0).total;
}

extern "C" int spa_int4_decode(const void* q, int dtype, int batch, int q_heads, int kv_heads, int head_dim,
                               const spa_kv_layout* kv, const void* k_scales, const void* v_scales,
                               const int32_t* context_lens, int max_tokens, int local_window, const int64_t* selected,
                               int top_m, int max_candidates, double scale, void* out, float* weights,
                               int weight_tokens, void* workspace, size_t workspace_bytes, spa_stream_t stream) {
  if (!spa::int4_rows_ok(kv, k_scales, v_scales, batch, kv_heads, head_dim)) return SPA_ERR_INVALID;
  spa::CacheDecodeArgs a{};
  a.q = q;
  a.out = out;
  a.dtype = dtype;
  a.B = batch;
  a.Hq = q_heads;
  a.Hkv = kv_heads;
  a.D = head_dim;
  a.k_scales = static_cast<const __half*>(k_scales);
  a.v_scales = static_cast<const __half*>(v_scales);
  a.ctx_lens = context_lens;
  a.cap = max_tokens;
  a.local_window = local_window;
  a.selected = selected;
  a.top_m = selected ? top_m : 0;
  a.weights = weights;
  a.T = weight_tokens;
  return spa::cache_decode_impl(a, -1, kv, max_candidates, scale, workspace, workspace_bytes, stream);
}

extern "C" int spa_paged_decode_weights(const void* q, int dtype, int batch, int q_heads, int kv_heads, int head_dim,
                                        const spa_kv_layout* kv, const int32_t* context_lens, int max_tokens,
                                        int local_window, int max_candidates, double scale, void* out, float* weights,
                                        int weight_tokens, void* workspace, size_t workspace_bytes,
                                        spa_stream_t stream) {
  if (!weights) return SPA_ERR_INVALID;
  spa::CacheDecodeArgs a{};
  a.q = q;
  a.out = out;
  a.dtype = dtype;
  a.B = batch;
  a.Hq = q_heads;
  a.Hkv = kv_heads;
  a.D = head_dim;
  a.ctx_lens = context_lens;
  a.cap = max_tokens;
  a.local_window = local_window;
  a.weights = weights;
  a.T = weight_tokens;
  return spa::cache_decode_impl(a, dtype, kv, max_candidates, scale, workspace, workspace_bytes, stream);
}
