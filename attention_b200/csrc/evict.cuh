// Eviction from a paged cache by accumulated attention weight: which tokens stay
// (select_tokens_kernel), and their move to the front of the sequence (compact_kernel).
#pragma once

#include "common.cuh"
#include "decode.cuh"

namespace spa {

// Order-preserving map of a weight: larger key = larger weight, -0 = +0, NaN below all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  uint32_t u = __float_as_uint(w);
  if (u == 0x80000000u) u = 0u;
  if (w != w) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A cluster of CTAs per (kv head, sequence), each with a stretch of its tokens.  The last r
// tokens stay; of the n = L - r before them the `need` largest keys, ties to the lower token.
// The need-th largest key is found byte by byte: every CTA counts its keys' bytes in shared
// memory and all add up the cluster's counts (256 bins: the exchange is 7 KB a CTA and byte; with
// 11 bits at a time it was 57 KB and took as long as the counting).  The first byte is mostly
// exponent, a few values for all keys, so a warp's lanes count it in eight copies.  Then one pass in token order writes the tokens above that key and the first of those equal to it, each
// CTA from the number that the CTAs before it hold.
//
// Weights are read once and stay in shared memory as keys (longer stretches than that holds are
// read again).  What bounds it: the latency of those rounds.  64 rows of 32768: 21 us in clusters
// of 4 (72 us with one CTA a row and the weights read four times; 71, 43 and 29 on the way, with
// 11-bit digits, with a bin a thread in the search, and with bytes).
constexpr int kSelThreads = 512, kSelBins = 256, kSelSlice = 4 * kSelThreads;
constexpr int kSelCached = 40 * 1024;  // keys a CTA keeps

__device__ __forceinline__ int ld_dsmem(const int* local, int rank) {
  uint32_t ra;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(ra) : "memory");
  return v;
}

template <bool CACHED>
__global__ void __launch_bounds__(kSelThreads, 4) select_tokens_kernel(const float* __restrict__ weights, int T,
                                                                    const int32_t* __restrict__ lens, int budget,
                                                                    int recent, int32_t* __restrict__ keep,
                                                                    int32_t* __restrict__ kept_lens) {
  extern __shared__ uint32_t s_key[];
  __shared__ int hist[4][kSelBins];  // of each byte
  __shared__ __align__(16) int copies[2][kSelBins][8];
  __shared__ int count[2];
  __shared__ int warp_sum[kSelThreads / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(ranks));
  const int h = blockIdx.x / ranks, heads = gridDim.x / ranks, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, all = ranks * kSelThreads, me = rank * kSelThreads + tid;
  const int64_t bh = static_cast<int64_t>(b) * heads + h;
  const float* w = weights + bh * T;
  int32_t* out = keep + bh * budget;
  const int L = min(max(lens[b], 0), T);
  if (h == 0 && me == 0) kept_lens[b] = min(L, budget);
  if (L <= budget) {  // the same for the whole cluster
    for (int i = me; i < budget; i += all) out[i] = i < L ? i : -1;
    return;
  }
  const int r = min(recent, budget), n = L - r, need0 = budget - r;
  for (int i = me; i < r; i += all) out[need0 + i] = n + i;
  if (need0 == 0) return;
  const int span = (n + ranks - 1) / ranks, lo = min(static_cast<int>(rank) * span, n), m = min(span, n - lo);
  const auto key = [&](int i) { return CACHED ? s_key[i] : weight_key(w[lo + i]); };
  for (int i = tid; i < 4 * kSelBins; i += kSelThreads) hist[0][i] = 0;
  for (int i = tid; i < 4 * kSelBins; i += kSelThreads) reinterpret_cast<int4*>(copies)[i] = make_int4(0, 0, 0, 0);
  if constexpr (CACHED) {
#pragma unroll 4
    for (int i = tid; i < m; i += kSelThreads) s_key[i] = weight_key(w[lo + i]);
  }
  __syncthreads();
  uint32_t prefix = 0, mask = 0;
  int need = need0;
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    if (pass < 2) {
#pragma unroll 4
      for (int i = tid; i < m; i += kSelThreads) {
        const uint32_t k = key(i);
        if ((k & mask) == prefix) atomicAdd(&copies[pass][(k >> shift) & 0xffu][lane & 7], 1);
      }
      __syncthreads();
      if (tid < kSelBins) {
        const int4 c = reinterpret_cast<const int4*>(copies[pass][tid])[0], d = reinterpret_cast<const int4*>(copies[pass][tid])[1];
        hist[pass][tid] = c.x + c.y + c.z + c.w + d.x + d.y + d.z + d.w;
      }
    } else {
#pragma unroll 4
      for (int i = tid; i < m; i += kSelThreads) {
        const uint32_t k = key(i);
        if ((k & mask) == prefix) atomicAdd(&hist[pass][(k >> shift) & 0xffu], 1);
      }
    }
    cluster_barrier();
    // a bin a thread, over the cluster
    int total = 0, x[8];
    if (tid < kSelBins) {
#pragma unroll
      for (int o = 0; o < 8; ++o)
        x[o] = o < static_cast<int>(ranks) ? ld_dsmem(&hist[pass][tid], (rank + o) & (ranks - 1)) : 0;
#pragma unroll
      for (int o = 0; o < 8; ++o) total += x[o];
    }
    // keys in higher bins: of higher lanes, and of higher warps
    int above = total;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_down_sync(0xffffffffu, above, off);
      if (lane + off < 32) above += o;
    }
    if (lane == 0) warp_sum[warp] = above;
    above -= total;
    __syncthreads();
#pragma unroll
    for (int v = 1; v < kSelBins / 32; ++v)
      if (v > warp) above += warp_sum[v];
    if (tid < kSelBins && above < need && above + total >= need) {  // one thread
      s_prefix = prefix | static_cast<uint32_t>(tid) << shift;
      s_need = need - above;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
    mask |= 0xffu << shift;
  }
  // tokens above the key and equal to it here and in the CTAs before
  int mine[2] = {0, 0};
#pragma unroll 4
  for (int i = tid; i < m; i += kSelThreads) {
    const uint32_t k = key(i);
    mine[0] += k > prefix;
    mine[1] += k == prefix;
  }
  if (tid < 2) count[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int x = __reduce_add_sync(0xffffffffu, mine[u]);
    if (lane == 0) atomicAdd(&count[u], x);
  }
  __syncthreads();
  cluster_barrier();
  const bool before_me = lane < static_cast<int>(rank);
  int above0 = __reduce_add_sync(0xffffffffu, before_me ? ld_dsmem(count, lane) : 0);
  int equal0 = __reduce_add_sync(0xffffffffu, before_me ? ld_dsmem(count + 1, lane) : 0);
  // token order: four tokens a thread; both counts of a slice fit 16 bits
  for (int base = 0; base < m; base += kSelSlice) {
    const int i0 = base + 4 * tid;
    uint32_t k[4];
    int c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      k[e] = i0 + e < m ? key(i0 + e) : 0u;
      const bool in = i0 + e < m;
      c += (in && k[e] > prefix ? 1 : 0) + (in && k[e] == prefix ? 1 << 16 : 0);
    }
    int inc = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += o;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    int before = inc - c, total = 0;
#pragma unroll
    for (int v = 0; v < kSelThreads / 32; ++v) {
      if (v < warp) before += warp_sum[v];
      total += warp_sum[v];
    }
    int above = above0 + (before & 0xffff), equal = equal0 + (before >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i0 + e >= m) continue;
      const bool gt = k[e] > prefix, eq = k[e] == prefix;
      if (gt || (eq && equal < need)) out[above + min(equal, need)] = lo + i0 + e;
      above += gt;
      equal += eq;
    }
    above0 += total & 0xffff;
    equal0 += total >> 16;
    __syncthreads();
  }
  cluster_barrier();  // no CTA leaves while its counts may still be read
}

// In-place compaction.  Of one (sequence, kv head) row j <- row keep[j] with keep ascending,
// so no source lies before its destination.  A cluster of CTAs takes the rows of one pool in
// order, a chunk at a time: every thread loads its units (16 bytes where rows allow) of the
// chunk, and they are stored once the whole cluster has loaded.  The next chunk's sources lie
// behind every row stored so far, so its loads are in flight meanwhile, and the rows of the
// chunk after that (keep, then the page table) are being looked up, once a row.
//
// Bound by HBM (each kept row read and written once) and the cluster's rounds: 64 pairs, 8192 of
// 32768 rows of 256 bytes take 133 us, 0.63 of the copy bandwidth (777 us with one CTA a pool
// and pair; with the next chunk's arrival before this one's stores 152).
constexpr int kMaxPools = 8;
struct CompactArgs {
  unsigned char* pool[kMaxPools];
  int row_bytes[kMaxPools], unit[kMaxPools];
  int n_pools;
  KvAddr addr;
  uint32_t page_inv;
  const int32_t* keep;
  int budget;
  float* weights;  // [B, Hkv, T] or nullptr
  int T;
};

constexpr int kCompactThreads = 256, kCompactUnroll = 4, kCompactCtas = 4;

// The rows that entry j of a list moves between, found in three steps of one load each, so that
// none waits for the one before: first() the token, second() the pages, third() the rows (to < 0
// to leave the entry out, with the error word set where a page is missing).  A call of each takes
// up what the call of the step before it left.
struct CompactPool {
  const CompactArgs& a;
  const int32_t* keep;
  int b, h;
  int j = 0, token = -1;
  int page[2] = {-1, -1}, off[2] = {0, 0};
  bool go = false;

  __device__ __forceinline__ void first(int entry, bool valid) {
    j = entry;
    token = valid ? keep[entry] : -1;
  }
  __device__ __forceinline__ void second() {
    go = token >= 0 && token != j;
    if (!go) return;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int t = e ? j : token;
      int lp = static_cast<int>(__umulhi(static_cast<uint32_t>(t), a.page_inv));
      off[e] = t - lp * a.addr.page_size;
      if (off[e] >= a.addr.page_size) ++lp, off[e] -= a.addr.page_size;
      page[e] = !a.addr.page_table ? lp
                : lp < a.addr.table_stride ? a.addr.page_table[static_cast<int64_t>(b) * a.addr.table_stride + lp] : -1;
    }
  }
  __device__ __forceinline__ longlong2 third() const {
    if (!go) return make_longlong2(-1, -1);
    int64_t row[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      row[e] = b * a.addr.batch_stride_rows + page[e] * a.addr.page_stride_rows + h * a.addr.head_stride_rows + off[e];
    if (page[0] < 0 || page[1] < 0 || row[0] < 0 || row[1] < 0 || row[0] >= a.addr.total_rows || row[1] >= a.addr.total_rows) {
      spa_raise(SPA_DEVERR_BAD_PAGE);
      return make_longlong2(-1, -1);
    }
    return make_longlong2(row[0], row[1]);
  }
};
struct CompactWeights {
  const int32_t* keep;
  int j = 0, token = -1, to = -1, from = -1;
  __device__ __forceinline__ void first(int entry, bool valid) {
    j = entry;
    token = valid ? keep[entry] : -1;
  }
  __device__ __forceinline__ void second() { from = token, to = token >= 0 ? j : -1; }
  __device__ __forceinline__ longlong2 third() const { return make_longlong2(from, to); }
};

// A chunk of a CTA: the fewer of 256 rows and what its threads hold in kCompactUnroll units each.
__host__ __device__ inline int compact_chunk_rows(int per) {
  const int rows = kCompactThreads * kCompactUnroll / per;
  return rows < 1 ? 1 : rows < kCompactThreads ? rows : kCompactThreads;
}

// rows: of the pair; per: units a row; rank, ranks: of the CTA in its cluster; slot: 4 tables of
// a chunk's (source, destination) rows, so that a thread may be a chunk ahead of another.
template <typename U, typename At>
__device__ __forceinline__ void compact_rows(U* pool, int rows, int per, int rank, int ranks,
                                             longlong2 (*slot)[kCompactThreads], At at) {
  const int chunk = compact_chunk_rows(per), chunks = (rows + chunk * ranks - 1) / (chunk * ranks);
  int row_of[kCompactUnroll], off_of[kCompactUnroll];  // of this thread's units, in every chunk
#pragma unroll
  for (int u = 0; u < kCompactUnroll; ++u) {
    const int i = threadIdx.x + u * kCompactThreads;
    row_of[u] = i / per;
    off_of[u] = i - row_of[u] * per;
    if (row_of[u] >= chunk) row_of[u] = -1;
  }
  const bool looks = static_cast<int>(threadIdx.x) < chunk;
  const auto first = [&](int c) {
    const int j = (c * ranks + rank) * chunk + threadIdx.x;
    at.first(j, c < chunks && j < rows);
  };
  const auto write = [&](int c) { slot[c & 3][threadIdx.x] = at.third(); };
  U v[2][kCompactUnroll] = {};
  const auto load = [&](int c, int k) {
#pragma unroll
    for (int u = 0; u < kCompactUnroll; ++u)
      if (row_of[u] >= 0) {
        const longlong2 r = slot[c & 3][row_of[u]];
        if (r.y >= 0) v[k][u] = pool[r.x * per + off_of[u]];
      }
  };
  const auto store = [&](int c, int k) {
#pragma unroll
    for (int u = 0; u < kCompactUnroll; ++u)
      if (row_of[u] >= 0) {
        const longlong2 r = slot[c & 3][row_of[u]];
        if (r.y >= 0) pool[r.y * per + off_of[u]] = v[k][u];
      }
  };
  // A CTA's loads of a chunk come before every other CTA's stores of it: the arrival releases
  // them (and waits for this CTA's earlier stores to be seen), the wait acquires.  That orders the
  // tables as well.
  if (looks) {
    for (int c = 0; c < 2; ++c) {
      first(c);
      at.second();
      write(c);
    }
    first(2);
    at.second();
    first(3);
  }
  __syncthreads();
  load(0, 0);
  for (int c = 0; c < chunks; c += 2) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (looks) {
        write(c + k + 2);
        at.second();
        first(c + k + 4);
      }
      __syncwarp();  // the cluster's barriers want whole warps
      cluster_arrive();
      if (c + k + 1 < chunks) load(c + k + 1, 1 - k);
      __syncwarp();
      cluster_wait();
      if (c + k < chunks) store(c + k, k);
    }
  }
}

__global__ void __launch_bounds__(kCompactThreads, kCompactCtas) compact_kernel(const CompactArgs a) {
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(ranks));
  const int which = blockIdx.x / ranks, h = blockIdx.y, b = blockIdx.z;
  const int64_t bh = static_cast<int64_t>(b) * gridDim.y + h;
  const int32_t* keep = a.keep + bh * a.budget;
  // ascending and non-negative, then -1 to the end; anything else leaves the pair untouched.
  // Each CTA looks at its part of the list; the verdicts and lengths meet in every CTA.
  __shared__ int s_n[16], s_bad[16];
  int n = 0, bad = 0;
  for (int j = rank * kCompactThreads + threadIdx.x; j < a.budget; j += ranks * kCompactThreads) {
    const int k = keep[j], prev = j ? keep[j - 1] : -1;
    if (k >= 0) {
      n = j + 1;
      bad |= k <= prev || (j && prev < 0) || (a.weights && k >= a.T);
    } else {
      bad |= k != -1;
    }
  }
  __shared__ int s_max;
  if (threadIdx.x == 0) s_max = 0;
  bad = __syncthreads_or(bad);
  atomicMax(&s_max, __reduce_max_sync(0xffffffffu, n));
  __syncthreads();
  cluster_barrier();  // every CTA of the cluster runs before its memory is written
  if (threadIdx.x < ranks) {
    st_dsmem(reinterpret_cast<float*>(s_n) + rank, threadIdx.x, __int_as_float(s_max));
    st_dsmem(reinterpret_cast<float*>(s_bad) + rank, threadIdx.x, __int_as_float(bad));
  }
  cluster_barrier();
  n = bad = 0;
  for (uint32_t r = 0; r < ranks; ++r) n = max(n, s_n[r]), bad |= s_bad[r];
  if (bad) {  // the same in every CTA of the cluster
    if (threadIdx.x == 0) spa_raise(SPA_DEVERR_BAD_INDEX);
    return;
  }
  __shared__ longlong2 s_rows[4][kCompactThreads];
  if (which < a.n_pools) {
    unsigned char* pool = a.pool[which];
    const int bytes = a.row_bytes[which];
    // a row whose source or destination has no page is left out whole
    const CompactPool at{a, keep, b, h};
    switch (a.unit[which]) {
      case 16: compact_rows(reinterpret_cast<uint4*>(pool), n, bytes / 16, rank, ranks, s_rows, at); break;
      case 8: compact_rows(reinterpret_cast<uint2*>(pool), n, bytes / 8, rank, ranks, s_rows, at); break;
      case 4: compact_rows(reinterpret_cast<uint32_t*>(pool), n, bytes / 4, rank, ranks, s_rows, at); break;
      case 2: compact_rows(reinterpret_cast<uint16_t*>(pool), n, bytes / 2, rank, ranks, s_rows, at); break;
      default: compact_rows(pool, n, bytes, rank, ranks, s_rows, at); break;
    }
  }
  if (which == 0 && a.weights) {
    float* w = a.weights + bh * a.T;
    __syncthreads();  // the pool's last stores still read the tables that the weights' rows go into
    compact_rows(reinterpret_cast<uint32_t*>(w), n, 1, rank, ranks, s_rows, CompactWeights{keep});
    // the sources behind row n have all been loaded (an empty list had no chunk to wait for,
    // and no sources)
    for (int t = n + rank * kCompactThreads + threadIdx.x; t < a.T; t += ranks * kCompactThreads) w[t] = 0.f;
  }
}

}  // namespace spa

extern "C" int spa_select_tokens(const float* weights, int batch, int kv_heads, int tokens, const int32_t* lens,
                                 int budget, int recent, int32_t* keep, int32_t* kept_lens, spa_stream_t stream) {
  if (!weights || !lens || !keep || !kept_lens || batch <= 0 || batch > 65535 || kv_heads <= 0 || kv_heads > (1 << 20) || tokens <= 0 ||
      budget <= 0 || recent < 0)
    return SPA_ERR_INVALID;
  // CTAs a cluster: a slice each at least, up to the portable 8; 4 where 8 are more than two CTAs
  // an SM and 4 fit the GPU at once (64 rows of 32768: 21.1 us against 24.6; of 131072, where they
  // do not fit: 72.9 against 67.7; 8 rows of 32768: 14.2 against 11.1)
  const int slices = (tokens + spa::kSelSlice - 1) / spa::kSelSlice;
  int ranks = slices >= 8 ? 8 : slices >= 4 ? 4 : slices >= 2 ? 2 : 1;
  {
    const int64_t pairs = static_cast<int64_t>(batch) * kv_heads, sms = spa::device_sm_count();
    const int64_t bytes = sizeof(uint32_t) * ((static_cast<int64_t>(tokens) + 3) / 4) + 21 * 1024;
    const int64_t held = 227 * 1024 / bytes < 4 ? 227 * 1024 / bytes : 4;
    if (ranks == 8 && pairs * 8 > 2 * sms && pairs * 4 <= held * sms) ranks = 4;
  }
  const int span = (tokens + ranks - 1) / ranks;
  const bool cached = span <= spa::kSelCached;
  const size_t smem = cached ? sizeof(uint32_t) * static_cast<size_t>(span) : 0;
  auto kern = cached ? spa::select_tokens_kernel<true> : spa::select_tokens_kernel<false>;
  SPA_CHECK_CUDA(spa_set_smem_once(kern, static_cast<int>(smem)));
  SPA_CHECK_CUDA(spa::launch_ex(kern, dim3(kv_heads * ranks, batch), dim3(spa::kSelThreads), smem,
                                reinterpret_cast<cudaStream_t>(stream), false, ranks, weights, tokens, lens, budget,
                                recent, keep, kept_lens));
  return SPA_OK;
}

extern "C" int spa_compact_tokens(const spa_kv_layout* kv, int n_pools, void* const* pools, const int* row_bytes,
                                  int batch, int kv_heads, const int32_t* keep, int budget, float* weights,
                                  int weight_tokens, spa_stream_t stream) {
  if (!kv || !keep || n_pools < 0 || n_pools > spa::kMaxPools || (n_pools > 0 && (!pools || !row_bytes)) ||
      batch <= 0 || batch > 65535 || kv_heads <= 0 || kv_heads > 65535 || budget <= 0 ||
      (weights && weight_tokens <= 0) || (n_pools == 0 && !weights))
    return SPA_ERR_INVALID;
  if (n_pools > 0 && (kv->page_size <= 0 || kv->total_rows <= 0 || (kv->page_table && kv->table_stride <= 0)))
    return SPA_ERR_INVALID;
  spa::CompactArgs a{};
  for (int i = 0; i < n_pools; ++i) {
    if (!pools[i] || row_bytes[i] <= 0) return SPA_ERR_INVALID;
    a.pool[i] = static_cast<unsigned char*>(pools[i]);
    a.row_bytes[i] = row_bytes[i];
    const uintptr_t x = reinterpret_cast<uintptr_t>(pools[i]) | static_cast<uintptr_t>(row_bytes[i]);
    a.unit[i] = x % 16 == 0 ? 16 : x % 8 == 0 ? 8 : x % 4 == 0 ? 4 : x % 2 == 0 ? 2 : 1;
    // clusters of their own move the pools side by side: none may share memory with another
    for (int j = 0; j < i; ++j)
      if (a.pool[i] < a.pool[j] + kv->total_rows * row_bytes[j] && a.pool[j] < a.pool[i] + kv->total_rows * row_bytes[i])
        return SPA_ERR_INVALID;
  }
  a.n_pools = n_pools;
  a.addr = make_kv_addr(*kv);
  a.page_inv = n_pools > 0 ? 0xffffffffu / static_cast<uint32_t>(kv->page_size) : 0;
  a.keep = keep;
  a.budget = budget;
  a.weights = weights;
  a.T = weight_tokens;
  // CTAs a cluster: as many as have a chunk of some pool's rows, up to the portable 8, and no more
  // than the GPU holds at once (kCompactCtas an SM): 64 pairs' K and V of 8192 rows took 143 us
  // in clusters of 8, 137 in clusters of 4
  int64_t most = weights ? (budget + spa::kCompactThreads - 1) / spa::kCompactThreads : 1;
  for (int i = 0; i < n_pools; ++i) {
    const int per = row_bytes[i] / a.unit[i];
    if (per > spa::kCompactThreads * spa::kCompactUnroll) return SPA_ERR_UNSUPPORTED;
    const int64_t chunks = (budget + spa::compact_chunk_rows(per) - 1) / spa::compact_chunk_rows(per);
    most = chunks > most ? chunks : most;
  }
  const int planes = n_pools > 0 ? n_pools : 1;
  const int64_t room = static_cast<int64_t>(spa::device_sm_count()) * spa::kCompactCtas / (static_cast<int64_t>(batch) * kv_heads * planes);
  if (room < most) most = room;
  const int ranks = most >= 8 ? 8 : most >= 4 ? 4 : most >= 2 ? 2 : 1;
  SPA_CHECK_CUDA(spa::launch_ex(spa::compact_kernel, dim3(planes * ranks, kv_heads, batch), dim3(spa::kCompactThreads), 0,
                                reinterpret_cast<cudaStream_t>(stream), false, ranks, a));
  return SPA_OK;
}
