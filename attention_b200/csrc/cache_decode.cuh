// Decode attention over the 4-bit cache, and decode attention that accumulates each
// token's weight (4-bit and plain caches).
//
// The candidates of a sequence (its context, its local window, or window and selected pages)
// are cut into tiles that never straddle a selected page; the tiles of one (sequence, kv
// head) are shared out over CTAs (cache_args.cuh) and, inside a CTA, over its warps, each of
// which keeps its own running maximum and sum.  A CTA merges its warps in shared memory; CTAs
// that share a pair leave (output, log2-sum-exp) partials that cache_decode_finish_kernel joins.  With weights
// the scores are kept as well (fp32, one per query head and token: 16 bytes a token at four
// heads per kv head, against 160 or 512 of K and V), because a token's weight needs the
// final log-sum-exp; the finish kernel turns them into probabilities and adds them up.
#pragma once

#include "cache_args.cuh"
#include "int4_mma.cuh"
#include "plain_mma.cuh"

namespace spa {

// ---------------------------------------------------------------------------
// CUDA-core kernel: any head_dim up to 256, any cache type.  Lane l holds the values
// d = l + 32 e; a warp takes a tile of 32 tokens, one token after another.
constexpr int kPlainHeads = 4, kPlainWarps = 4;

template <typename T, int E>  // T = uint8_t: the 4-bit cache
__global__ void __launch_bounds__(kPlainWarps * 32) cache_decode_plain_kernel(const CacheDecodeArgs a) {
  __shared__ float sm[kPlainWarps][kPlainHeads], sl[kPlainWarps][kPlainHeads], so[kPlainWarps][kPlainHeads][E * 32];
  __shared__ int pre[kFlatBatch + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = a.D;
  if (a.ctas) tiles_before<32>(a, pre);
  Work work(a, pre);
  Segment seg;
  while (work.next<32>(a, pre, seg)) {
    const int b = seg.b, h = seg.h, head0 = seg.chunk * kPlainHeads, heads = min(kPlainHeads, a.group - head0);
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
    for (int tile = seg.u0 + warp; tile < seg.u1; tile += kPlainWarps) {
      const int tok = tile_token<32>(a, p, b, tile, lane);
      int off = 0;
      const int page = tok < 0 ? -1 : token_page(a, b, tok, off);
      const int64_t my_row = page_row(a, b, h, tok, page, off);
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
          // differences first, then their scale: a scaled score would carry its own rounding
          const float mn = fmaxf(m[n], s[n]);
          // a first score of -inf leaves nothing to weigh: the difference would be NaN
          const float alpha = m[n] == -INFINITY ? 0.f : exp2f((m[n] - mn) * a.scale_log2);
          const float pr = s[n] == -INFINITY ? 0.f : exp2f((s[n] - mn) * a.scale_log2);
          l[n] = l[n] * alpha + pr;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[n][e] = fmaf(acc[n][e], alpha, pr * kv[e]);
          m[n] = mn;
        }
        if (a.scores && lane == 0)
          for (int n = 0; n < heads; ++n)
            a.scores[((static_cast<int64_t>(b) * a.Hkv + h) * a.cap + t) * a.group + head0 + n] = s[n] * a.scale_log2;
      }
    }
    // merge the warps
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
        const float f = sm[w][n] == -INFINITY ? 0.f : exp2f((sm[w][n] - M) * a.scale_log2);
        W = fmaf(sl[w][n], f, W);
        O = fmaf(so[w][n][d], f, O);
      }
      const float o = W == 0.f ? 0.f : O / W;
      if (a.weights || !seg.whole) {
        a.part_o[(static_cast<int64_t>(seg.slot) * kPlainHeads + n) * D + d] = o;
        if (d == 0) a.part_lse[static_cast<int64_t>(seg.slot) * kPlainHeads + n] = W == 0.f ? -INFINITY : M * a.scale_log2 + log2f(W);
      } else {
        store_any(a.out, a.dtype, (q0 + n) * D + d, o);
      }
    }
    __syncthreads();  // the next segment reuses the buffers
  }
}

// ---------------------------------------------------------------------------
// Joins the partials and, with weights, adds every token's probabilities to its weight.
// Grid (head blocks + token blocks, Hkv, B): a warp of the first blocks merges one head's output.
constexpr int kFinishThreads = 256, kFinishTokens = 2048, kFinishHeads = kFinishThreads / 32;

template <int TILE, bool WEIGHTS>
__global__ void __launch_bounds__(kFinishThreads) cache_decode_finish_kernel(const CacheDecodeArgs a) {
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pairs = a.Hkv * a.chunks, head_blocks = (a.group + kFinishHeads - 1) / kFinishHeads;
  __shared__ __align__(16) float s_lse[256];
  __shared__ int s_sum[kFinishThreads / 32][2];
  // this sequence's tiles, those before it, and all
  const TilePlan plan = tile_plan<TILE>(a, b);
  int64_t before = 0, total = 0;
  if (a.ctas) {
    int x = 0, y = 0;
    for (int i = tid; i < a.B; i += kFinishThreads) {
      const int n = tile_plan<TILE>(a, i).n;
      y += n;
      if (i < b) x += n;
    }
    x = __reduce_add_sync(0xffffffffu, x);
    y = __reduce_add_sync(0xffffffffu, y);
    if (lane == 0) s_sum[warp][0] = x, s_sum[warp][1] = y;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kFinishThreads / 32; ++w) before += s_sum[w][0], total += s_sum[w][1];
  }
  // log2-sum-exp of head n of the group over its partials first .. last (rows `row` of their
  // slots); `mine` is this lane's partial of each 32
  int first = 0, last = -1, row = 0;
  const auto lse_of = [&](int n) -> float {
    const int hc = h * a.chunks + n / a.heads, pair = b * pairs + hc;
    row = n % a.heads;
    first = last = pair;
    if (a.ctas)
      ctas_of(before * pairs + static_cast<int64_t>(hc) * plan.n, plan.n, total * pairs,
              sharing_ctas(a, total * pairs), first, last);
    first += pair, last += pair;
    if (first == last && !WEIGHTS) return 0.f;  // its CTA has written the output
    float M = -INFINITY;
    for (int s = first + lane; s <= last; s += 32) M = fmaxf(M, a.part_lse[static_cast<int64_t>(s) * a.heads + row]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    float sum = 0.f;
    for (int s = first + lane; s <= last; s += 32) {
      const float x = a.part_lse[static_cast<int64_t>(s) * a.heads + row];
      sum += x == -INFINITY ? 0.f : exp2f(x - M);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    return sum == 0.f ? INFINITY : M + log2f(sum);
  };
  pdl_block();
  if (blockIdx.x < head_blocks) {
    const int n = blockIdx.x * kFinishHeads + warp;
    if (n >= a.group) return;
    const int64_t out = (static_cast<int64_t>(b) * a.Hq + h * a.group + n) * a.D;
    if (plan.n == 0) {
      for (int d = lane; d < a.D; d += 32) store_any(a.out, a.dtype, out + d, 0.f);
      return;
    }
    const float lse = lse_of(n);
    if (first == last && !WEIGHTS) return;
    // eight partials' loads in flight; four columns a lane where rows allow
    const auto columns = [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      for (int d = lane * V; d < a.D; d += 32 * V) {
        float o[V] = {};
        for (int s0 = first; s0 <= last; s0 += 8) {
          float v[8][V], x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int64_t at = static_cast<int64_t>(min(s0 + i, last)) * a.heads + row;
            x[i] = s0 + i <= last ? a.part_lse[at] : -INFINITY;
            if constexpr (V == 4)
              *reinterpret_cast<float4*>(v[i]) = *reinterpret_cast<const float4*>(a.part_o + at * a.D + d);
            else
              v[i][0] = a.part_o[at * a.D + d];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (x[i] != -INFINITY) {
              const float f = exp2f(x[i] - lse);
#pragma unroll
              for (int e = 0; e < V; ++e) o[e] = fmaf(v[i][e], f, o[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) store_any(a.out, a.dtype, out + d + e, o[e]);
      }
    };
    if (a.D % 4 == 0)
      columns(std::integral_constant<int, 4>{});
    else
      columns(std::integral_constant<int, 1>{});
    return;
  }
  if constexpr (!WEIGHTS) return;
  const int t0 = plan.lo + (blockIdx.x - head_blocks) * kFinishTokens;
  if (t0 >= plan.ctx) return;
  for (int n = warp; n < a.group; n += kFinishThreads / 32) {
    const float lse = lse_of(n);
    if (lane == 0) s_lse[n] = lse;
  }
  __syncthreads();
  const int64_t bh = static_cast<int64_t>(b) * a.Hkv + h;
  const int t1 = min(t0 + kFinishTokens, min(plan.ctx, a.T));
  if (tid == 0 && min(t0 + kFinishTokens, plan.ctx) > a.T) spa_raise(SPA_DEVERR_BAD_INDEX);
  const float* scores = a.scores + bh * a.cap * a.group;
  float* weights = a.weights + bh * a.T;
  // kEach tokens a thread, their loads in flight together; the heads in fours where they line up
  constexpr int kEach = kFinishTokens / kFinishThreads;
  float w[kEach] = {}, old[kEach] = {};
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (t0 + tid + i * kFinishThreads < t1) old[i] = weights[t0 + tid + i * kFinishThreads];
  if (a.group % 4 == 0) {
    for (int n = 0; n < a.group; n += 4) {
      const float4 lse = *reinterpret_cast<const float4*>(s_lse + n);
      float4 x[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int t = min(t0 + tid + i * kFinishThreads, t1 - 1);
        if (t >= t0) x[i] = *reinterpret_cast<const float4*>(scores + static_cast<int64_t>(t) * a.group + n);
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        w[i] += fast_exp2(x[i].x - lse.x) + fast_exp2(x[i].y - lse.y) + (fast_exp2(x[i].z - lse.z) + fast_exp2(x[i].w - lse.w));
    }
  } else {
    for (int n = 0; n < a.group; ++n) {
      const float lse = s_lse[n];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int t = t0 + tid + i * kFinishThreads;
        if (t < t1) w[i] += fast_exp2(scores[static_cast<int64_t>(t) * a.group + n] - lse);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int t = t0 + tid + i * kFinishThreads;
    if (t < t1) weights[t] = old[i] + w[i];
  }
}

// ---------------------------------------------------------------------------
// host planning
constexpr int kWholeTiles = 24, kWholeTilesBusy = 40, kCtaTiles = 6;
enum CacheKernel { kCachePlain, kCacheInt4Mma, kCachePlainMma };
struct CachePlan {
  int heads, chunks, ctas, slots, tile;
};
inline CachePlan cache_plan(int batch, int q_heads, int kv_heads, int head_dim, int max_candidates, CacheKernel kind) {
  CachePlan p;
  const int group = q_heads / kv_heads;
  p.heads = kind == kCachePlain ? kPlainHeads : kind == kCacheInt4Mma ? int4_mma_heads(head_dim, group) : 8;
  p.chunks = (group + p.heads - 1) / p.heads;
  p.tile = kind == kCachePlainMma ? 16 : 32;
  const int per_sm = kind == kCachePlain ? 4 : kind == kCacheInt4Mma ? int4_mma_ctas(head_dim, p.heads) : head_dim == 256 ? 1 : 2;
  const int64_t pairs = static_cast<int64_t>(batch) * kv_heads * p.chunks;
  const int64_t tiles = (max_candidates + p.tile - 1) / p.tile + 1;
  const int64_t room = static_cast<int64_t>(device_sm_count()) * per_sm;
  const int64_t most = (pairs * tiles + kCtaTiles - 1) / kCtaTiles;
  // One CTA per pair where a pair has little to share (more of it where pairs alone keep most SMs
  // busy: 128 pairs of 1000 tokens 12.4 us against 17.3, but of 1800 in fp32 28.4 against 25.5, and 8 of
  // 1900 in fp16 16.8 against 12.4), where pairs fill the GPU several times over, or where the batch is
  // longer than a CTA sums up.
  const bool whole = tiles <= (pairs * 4 >= 3 * device_sm_count() ? kWholeTilesBusy : kWholeTiles);
  const bool flat = !whole && pairs < 4 * room && batch <= kFlatBatch;
  p.ctas = flat ? static_cast<int>(room < most ? room : most) : 0;
  p.slots = static_cast<int>((flat ? p.ctas : pairs) + pairs);
  return p;
}
inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct CacheScratch {
  size_t part_o, part_lse, scores, total;
};
inline CacheScratch cache_scratch(const CachePlan& p, int batch, int q_heads, int head_dim, int cap, bool weights) {
  CacheScratch s{};
  const size_t parts = weights || p.ctas ? static_cast<size_t>(p.slots) * p.heads : 0;
  s.part_o = 0;
  s.part_lse = align256(parts * head_dim * sizeof(float));
  s.scores = s.part_lse + align256(parts * sizeof(float));
  s.total = s.scores + (weights ? align256(static_cast<size_t>(batch) * q_heads * cap * sizeof(float)) : 0);
  return s;
}

template <typename T>
int launch_cache_plain(const CacheDecodeArgs& a, cudaStream_t st) {
  const dim3 grid(a.ctas ? a.ctas : a.B * a.Hkv * a.chunks);
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
  if (!(scale > 0.0) || scale > 1e30 || reinterpret_cast<uintptr_t>(a.out) % 16) return SPA_ERR_INVALID;
  if ((a.selected && a.top_m <= 0) || (a.weights && (a.T <= 0 || a.selected))) return SPA_ERR_INVALID;
  a.group = a.Hq / a.Hkv;
  if (a.group > 256) return SPA_ERR_UNSUPPORTED;
  if (a.Hkv > 65535 || static_cast<int64_t>(a.B) * a.Hq > (1 << 28)) return SPA_ERR_UNSUPPORTED;
  const CacheKernel kind = kv_dtype < 0 ? (int4_mma_serves(a.D, kv->total_rows) ? kCacheInt4Mma : kCachePlain)
                           : plain_mma_serves(kv_dtype, a.D, kv->k, kv->v, a.q) ? kCachePlainMma : kCachePlain;
  const CachePlan p = cache_plan(a.B, a.Hq, a.Hkv, a.D, max_candidates, kind);
  const CacheScratch s = cache_scratch(p, a.B, a.Hq, a.D, a.cap, a.weights != nullptr);
  if (s.total && (!workspace || workspace_bytes < s.total || reinterpret_cast<uintptr_t>(workspace) % 16))
    return SPA_ERR_WORKSPACE;
  a.k = kv->k;
  a.v = kv->v;
  a.addr = make_kv_addr(*kv);
  a.page_inv = 0xffffffffu / static_cast<uint32_t>(kv->page_size);
  a.q_vec = reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
  a.heads = p.heads;
  a.chunks = p.chunks;
  a.ctas = p.ctas;
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const bool parts = a.weights || a.ctas;
  a.part_o = parts ? reinterpret_cast<float*>(ws + s.part_o) : nullptr;
  a.part_lse = parts ? reinterpret_cast<float*>(ws + s.part_lse) : nullptr;
  a.scores = a.weights ? reinterpret_cast<float*>(ws + s.scores) : nullptr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int rc;
  if (kind == kCacheInt4Mma)
    rc = launch_int4_decode(a, st);
  else if (kind == kCachePlainMma)
    rc = kv_dtype == SPA_F16 ? launch_plain_decode<__half>(a, st) : launch_plain_decode<__nv_bfloat16>(a, st);
  else if (kv_dtype < 0)
    rc = launch_cache_plain<uint8_t>(a, st);
  else if (kv_dtype == SPA_F32)
    rc = launch_cache_plain<float>(a, st);
  else if (kv_dtype == SPA_F16)
    rc = launch_cache_plain<__half>(a, st);
  else
    rc = launch_cache_plain<__nv_bfloat16>(a, st);
  if (rc || !parts) return rc;
  const int span = a.local_window > 0 && a.local_window < a.cap ? a.local_window : a.cap;
  const int blocks = (a.group + kFinishHeads - 1) / kFinishHeads + (a.weights ? (span + kFinishTokens - 1) / kFinishTokens : 0);
  // (without weights every path has tiles of 32)
  auto finish = !a.weights ? cache_decode_finish_kernel<32, false>
                : p.tile == 16 ? cache_decode_finish_kernel<16, true> : cache_decode_finish_kernel<32, true>;
  SPA_CHECK_CUDA(launch_pdl(finish, dim3(blocks, a.Hkv, a.B), dim3(kFinishThreads), 0, st, true, a));
  return SPA_OK;
}

}  // namespace spa

extern "C" size_t spa_cache_decode_workspace_size(int batch, int q_heads, int kv_heads, int head_dim,
                                                  int max_candidates, int max_tokens, int weights, int kv_dtype) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0 || max_candidates < 0 ||
      max_tokens <= 0)
    return 0;
  // addresses and the number of rows decide between the kernels, and they are not known here:
  // the larger need
  size_t most = 0;
  for (const spa::CacheKernel kind : {spa::kCachePlain, kv_dtype < 0 ? spa::kCacheInt4Mma : spa::kCachePlainMma}) {
    const spa::CachePlan p = spa::cache_plan(batch, q_heads, kv_heads, head_dim, max_candidates, kind);
    const size_t need = spa::cache_scratch(p, batch, q_heads, head_dim, max_tokens, weights != 0).total;
    most = need > most ? need : most;
  }
  return most;
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
