// Decode attention over a 16-bit cache that also keeps the scores (cache_decode.cuh adds up the
// tokens' weights from them), on mma.sync, for head_dim 64, 128 and 256.
//
// Tokens are the 16 rows of the QK product and d the 16 rows of the PV product; the query heads
// of the kv head are its 8 columns, so 8 heads cost one read of K and V and no padding of 16.
// Products of 16-bit values are exact in the fp32 sums.  Probabilities enter as two 16-bit
// halves (16 bits of them for bf16, 22 for fp16): with one, their rounding would be as large as
// the output's own.
//
// Bound by HBM: 512 bytes a token and kv head at D = 128, and the scores (16 bytes written and read
// at four query heads).  Each warp streams a stretch of tiles of 16 tokens (8 KB) through its own
// ring of cp.async stages, three deep.  8 x 16384 tokens, 32 query and 8 kv heads of 128 in bf16:
// 103 us with the weights' sum, 0.81 of the copy bandwidth (the CUDA-core kernel: 868 us).
#pragma once

#include "cache_args.cuh"
#include "int4_mma.cuh"

namespace spa {

template <int D>
struct PlainTile {
  static constexpr int kTok = 16, kRow = 2 * D, kHalf = kTok * kRow, kStage = 2 * kHalf;
  // 16-byte piece c of token row r: pieces of 8 rows on end fall into different banks
  static __device__ __forceinline__ int at(int r, int c) { return r * kRow + ((c ^ (r & 7)) << 4); }
};
template <int D>
struct PlainCfg {
  static constexpr int kWarps = 4, kStages = 3;
  static constexpr int kCtas = D == 256 ? 1 : 2;  // an SM; what the rings leave
};

template <typename T>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  MmaOp<T>::run(d, a, b0, b1);
}
template <typename T>
__device__ __forceinline__ float unpack_lo(uint32_t x) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) return half_lo(x);
  return __uint_as_float(x << 16);
}
template <typename T>
__device__ __forceinline__ float unpack_hi(uint32_t x) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) return half_hi(x);
  return __uint_as_float(x & 0xffff0000u);
}

template <typename T, int D>
__global__ void __launch_bounds__(PlainCfg<D>::kWarps * 32, PlainCfg<D>::kCtas) plain_decode_mma_kernel(const CacheDecodeArgs a) {
  using S = PlainTile<D>;
  constexpr int W = PlainCfg<D>::kWarps, ST = PlainCfg<D>::kStages, HN = 8, KS = D / 16;
  extern __shared__ __align__(128) unsigned char i4_smem[];
  __shared__ float s_f[HN][16];
  __shared__ unsigned s_live[W][ST];
  __shared__ int pre[kFlatBatch + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  unsigned char* ring = i4_smem + warp * (ST * S::kStage);
  pdl_trigger();  // the kernel that joins the partials comes next
  if (a.ctas) tiles_before<S::kTok>(a, pre);
  Work work(a, pre);
  Segment seg;
#pragma unroll 1
  while (work.next<S::kTok>(a, pre, seg)) {
    const int b = seg.b, h = seg.h, head0 = seg.chunk * HN, heads = min(HN, a.group - head0);
    const int64_t q0 = static_cast<int64_t>(b) * a.Hq + h * a.group + head0;
    const TilePlan plan = tile_plan<S::kTok>(a, b);
    int next_tile, end_tile;  // this warp's tiles, one stretch
    split_range(seg.u1 - seg.u0, warp, W, next_tile, end_tile);
    next_tile += seg.u0, end_tile += seg.u0;
    const int first_tile = next_tile, n_tiles = end_tile - next_tile;

    // a lane's token, fetched one tile ahead (lanes 16..31 repeat 0..15)
    int token = -1, page = -1, page_off = 0;
    const auto fetch = [&]() {
      token = next_tile < end_tile ? tile_token<S::kTok>(a, plan, b, next_tile, lane & 15) : -1;
      page = token < 0 ? -1 : token_page(a, b, token, page_off);
    };
    fetch();
    const auto issue = [&](int stage) {
      if (next_tile < end_tile) {
        const uint32_t base = smem_u32(ring + stage * S::kStage);
        const int64_t my_row = page_row(a, b, h, token, page, page_off);
        const unsigned live = __ballot_sync(0xffffffffu, my_row >= 0) & 0xffffu;
        if (lane == 0) s_live[warp][stage] = live;
        constexpr int per = S::kRow / 16;  // pieces a row
#pragma unroll
        for (int i = 0; i < S::kTok * per / 32; ++i) {
          const int c = i * 32 + lane, r = c / per, p = c % per;
          const int64_t row = __shfl_sync(0xffffffffu, my_row, r);
          const int64_t src = (row >= 0 ? row : 0) * S::kRow + p * 16;
          const int n = row >= 0 ? 16 : 0;
          cp_async<16>(base + S::at(r, p), static_cast<const unsigned char*>(a.k) + src, n);
          cp_async<16>(base + S::kHalf + S::at(r, p), static_cast<const unsigned char*>(a.v) + src, n);
        }
        ++next_tile;
        fetch();
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) issue(s);

    // query fragments: column g is a head, k-step kk holds its values 16 kk + 2 t, + 1, + 8, + 9
    uint32_t qb[KS][2];
    {
      const T* q = static_cast<const T*>(a.q) + (q0 + g) * D + 2 * t;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          qb[kk][i] = 0;
          if (g < heads) qb[kk][i] = *reinterpret_cast<const uint32_t*>(q + 16 * kk + 8 * i);
        }
    }
    float o[KS][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[kk][e] = 0.f;
    // ldmatrix addresses: K rows lane & 15, 16-byte half lane >> 4 of each k-step; V the same rows,
    // transposed by the load
    const int lr = lane & 15, lc = lane >> 4;

    int stage = 0;
#pragma unroll 1
    for (int done = 0; done < n_tiles; ++done) {
      cp_async_wait<ST - 2>();
      __syncwarp();
      issue(stage == 0 ? ST - 1 : stage - 1);
      const uint32_t kb = smem_u32(ring + stage * S::kStage) + lr * S::kRow, vb = kb + S::kHalf;
      const unsigned live = s_live[warp][stage];
      float sc[4] = {0.f, 0.f, 0.f, 0.f}, sd[4] = {0.f, 0.f, 0.f, 0.f};  // two chains
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        uint32_t x[4];
        ldmatrix_x4(x, kb + (((2 * kk + lc) ^ (lr & 7)) << 4));
        if (kk & 1)
          mma_16<T>(sd, x, qb[kk][0], qb[kk][1]);
        else
          mma_16<T>(sc, x, qb[kk][0], qb[kk][1]);
      }
      const int tok = plan.seg + (first_tile + done) * S::kTok;
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = g + (e < 2 ? 0 : 8);
        sc[e] = live >> r & 1 ? (sc[e] + sd[e]) * a.scale_log2 : -INFINITY;
        top[e & 1] = fmaxf(top[e & 1], sc[e]);
      }
      // scores [token][head of the group]
      const int h0 = 2 * t;
      if (h0 < heads) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tk = tok + g + 8 * e;
          if (tk >= plan.lo && tk < plan.ctx) {
            float* p = a.scores + ((static_cast<int64_t>(b) * a.Hkv + h) * a.cap + tk) * a.group + head0 + h0;
            if (h0 + 1 < heads && a.group % 2 == 0) {
              *reinterpret_cast<float2*>(p) = make_float2(sc[2 * e], sc[2 * e + 1]);
            } else {
              p[0] = sc[2 * e];
              if (h0 + 1 < heads) p[1] = sc[2 * e + 1];
            }
          }
        }
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
        float f[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = top[c];
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
          x = fmaxf(m[c], x);
          f[c] = m[c] == -INFINITY ? 0.f : fast_exp2(m[c] - x);  // nothing seen yet
          m[c] = x;
          l[c] *= f[c];
        }
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[kk][e] *= f[e & 1];
      }
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // a masked token gives 0 also where no score was seen yet (-inf + inf)
        p[e] = sc[e] == -INFINITY ? 0.f : fast_exp2(sc[e] - m[e & 1]);
        l[e & 1] += p[e];
      }
      const uint32_t h01 = MmaOp<T>::pack(p[0], p[1]), h23 = MmaOp<T>::pack(p[2], p[3]);
      const uint32_t b0 = movmatrix_trans(h01), b1 = movmatrix_trans(h23);
      const uint32_t c0 = movmatrix_trans(MmaOp<T>::pack(p[0] - unpack_lo<T>(h01), p[1] - unpack_hi<T>(h01)));
      const uint32_t c1 = movmatrix_trans(MmaOp<T>::pack(p[2] - unpack_lo<T>(h23), p[3] - unpack_hi<T>(h23)));
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        // d rows 16 kk .. + 15: blocks (tokens 0-7, d 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
        uint32_t x[4], y[4];
        ldmatrix_x4_trans(x, vb + (((2 * kk + lc) ^ (lr & 7)) << 4));
        y[0] = x[0], y[1] = x[2], y[2] = x[1], y[3] = x[3];
        mma_16<T>(o[kk], y, b0, b1);
        mma_16<T>(o[kk], y, c0, c1);
      }
      stage = stage == ST - 1 ? 0 : stage + 1;
    }

    // ---- merge the warps (the ring is free once every copy has landed)
    cp_async_wait<0>();
    __syncthreads();
    constexpr int kLd = D + 4;
    float* buf = reinterpret_cast<float*>(i4_smem);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float s = l[c];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      float* row = buf + (warp * HN + 2 * t + c) * kLd;
      if (g == 0) row[D] = m[c], row[D + 1] = s;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        row[16 * kk + g] = o[kk][c];
        row[16 * kk + g + 8] = o[kk][2 + c];
      }
    }
    merge_warps<W, HN, D>(a, seg, q0, heads, buf, s_f);
    __syncthreads();  // the next segment's loads reuse the buffer
  }
}

inline bool plain_mma_serves(int dtype, int head_dim, const void* k, const void* v, const void* q) {
  return dtype != SPA_F32 && (head_dim == 64 || head_dim == 128 || head_dim == 256) &&
         (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(q) % 4 == 0;
}
template <typename T, int D>
int launch_plain_mma(const CacheDecodeArgs& a, cudaStream_t st) {
  using C = PlainCfg<D>;
  constexpr int ring = C::kWarps * C::kStages * PlainTile<D>::kStage, merge = C::kWarps * 8 * (D + 4) * 4;
  constexpr int smem = ring > merge ? ring : merge;
  auto kern = plain_decode_mma_kernel<T, D>;
  SPA_CHECK_CUDA(spa_set_smem_once(kern, smem));
  kern<<<a.ctas ? a.ctas : a.B * a.Hkv * a.chunks, C::kWarps * 32, smem, st>>>(a);
  SPA_CHECK_CUDA(cudaGetLastError());
  return SPA_OK;
}
template <typename T>
int launch_plain_decode(const CacheDecodeArgs& a, cudaStream_t st) {
  return a.D == 64 ? launch_plain_mma<T, 64>(a, st)
                   : a.D == 128 ? launch_plain_mma<T, 128>(a, st) : launch_plain_mma<T, 256>(a, st);
}

}  // namespace spa
