// Decode attention over the 4-bit cache on the tensor cores (head_dim 32, 64, 96, 128, 256).
//
//   score_t = sum_j s_tj (q_j . n_tj) + z_tj sum(q_j)      o = sum_t p_t s_tj n_tj + p_t z_tj
//
// with n the stored nibbles, so no value is ever expanded.  A nibble masked in place is an
// fp16 subnormal, n 2^-24 or 16 n 2^-24, which mma.sync takes (query values that meet the
// second kind are divided by 16): per 8 values of K that is one byte permute, four ands and a
// shift.  The tensor core lines subnormal products up by their exponent field, so some 2^-19
// of a product is lost; that is 1e-6 of a score.  Over a long context sum(p s n) and sum(p z)
// are some hundred times the output that is left of them, and neither that nor the rounding of
// p s would cancel.  So V (and K with fp32 queries) is centred: sum(p s (n - 8)) +
// sum(p (z + 8 s)), with n - 8 made a normal number by one more packed add a pair: the nibble
// is put under the exponent of 1024, and 1032 taken away.
//
// Tokens are the 16 rows of the QK product and d the 16 rows
// of the PV product, the query heads of the kv head its 8 columns; the sum over a group's 32
// values is a pair of k-steps, after which the scale is one fp32 multiply a score.  The zeros
// go through one more product per 16 tokens, of z with the queries' group sums (held as two
// halves).  For PV the scale goes into the probabilities: p, p s and z + 8 s in fp16 for a bf16
// output (roundings of 2^-11 against the output's 2^-8), as two halves (22 bits) otherwise.
//
// What bounds it: HBM, 160 bytes a token and kv head at D = 128, if the instructions keep up:
// at 6.5 TB/s an SM has 3.5 issue slots per value, and a tile takes 2.6 a value.  Each warp
// streams a stretch of tiles of 32 tokens (5 KB) through its own ring of cp.async stages in
// shared memory, without barriers between warps, so pages of any size, order and alignment
// cost the same.
//
// Measured (B200, 32 query and 8 kv heads of 128, bf16, pages of 128): 8 x 32768 tokens 76 us, 4.4
// TB/s or 0.67 of the copy bandwidth; 8 x 131072 tokens 259 us, 0.79.  No pipe is full (IPC 2.4 of
// 4, ALU 51 %, tensor 25 %) and few warps wait for memory: what is left, with 12 warps an SM, is
// instructions that wait for the one before (with 16 warps of 128 registers it was 80 us, with the
// maximum moved at every rise 90).  Some 12 us of every call are the phases before the first
// product and after the last, and the joining kernel.
#pragma once

#include "cache_args.cuh"

namespace spa {

template <int G, int NT>
struct Int4Cfg {
  // as many warps an SM as the registers allow (168, or 255 with the larger accumulators)
  static constexpr bool kSmall = NT == 1 && G <= 4;
  static constexpr int kWarps = kSmall ? 4 : 8, kCtas = kSmall ? 3 : 1;
  static constexpr int kStages = 2;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Transposes an 8x8 tile of 16-bit values held one row pair per lane.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, int src_bytes) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(src_bytes)
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float half_lo(uint32_t x) { return __half2float(__ushort_as_half(static_cast<unsigned short>(x))); }
__device__ __forceinline__ float half_hi(uint32_t x) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(x >> 16)));
}
__device__ __forceinline__ uint32_t hmul2_u(uint32_t a, uint32_t b) {
  const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t hadd2_u(uint32_t a, uint32_t b) {
  const __half2 v = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int G>
struct Int4Tile {
  static constexpr int kTok = 32, kRow = 16 * G, kScaleRow = 4 * G;
  static constexpr int kCodes = kTok * kRow, kScales = kTok * kScaleRow;
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kScaleChunk = G % 4 == 0 ? 16 : G % 2 == 0 ? 8 : 4;
  // Where byte `byte` of a token's row lies: rows are permuted within 128-byte lines so that
  // both the QK reads (8 tokens, whole rows) and the PV reads (tokens 2t, an eighth of the row
  // each) touch every bank once.
  static __device__ __forceinline__ int at(int tok, int byte) {
    if constexpr (G == 8) return tok * 128 + (((byte >> 4) ^ (tok & 7)) << 4) + (byte & 15);
    if constexpr (G == 4)
      return (tok >> 1) * 128 + (((tok ^ (tok >> 1)) & 1) << 6) + (((byte >> 4) ^ ((tok >> 1) & 2)) << 4) + (byte & 15);
    if constexpr (G == 2) return (tok >> 2) * 128 + (((tok & 3) ^ ((tok >> 2) & 1)) << 5) + byte;
    return tok * kRow + byte;
  }
};

// N bytes at p (aligned to N's largest power-of-two divisor up to 16) as 32-bit words
template <int N>
__device__ __forceinline__ void lds_words(const unsigned char* p, uint32_t* w) {
  if constexpr (N % 16 == 0) {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) *reinterpret_cast<uint4*>(w + 4 * i) = reinterpret_cast<const uint4*>(p)[i];
  } else if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) *reinterpret_cast<uint2*>(w + 2 * i) = reinterpret_cast<const uint2*>(p)[i];
  } else if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  } else {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = h[2 * i] | static_cast<uint32_t>(h[2 * i + 1]) << 16;
    w[N / 4] = h[N / 2 - 1];
  }
}
// 16-bit words x of `a` and y of `b` side by side
template <int X, int Y>
__device__ __forceinline__ uint32_t pair16(const uint32_t* a, const uint32_t* b) {
  constexpr uint32_t sel = (X & 1 ? 0x32u : 0x10u) | (Y & 1 ? 0x7600u : 0x5400u);
  return __byte_perm(a[X / 2], b[Y / 2], sel);
}

template <typename F, int... J>
__device__ __forceinline__ void for_each_index(F f, std::integer_sequence<int, J...>) {
  (f(std::integral_constant<int, J>{}), ...);
}

__device__ __forceinline__ uint32_t hfma2_u(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}
// The four nibbles of each half of x.  CENTRE: n - 8 each; else 0 and 2 times 2^-24, 1 and 3
// times 16 2^-24.
template <bool CENTRE>
__device__ __forceinline__ void nibbles(uint32_t x, uint32_t (&n)[4]) {
  if constexpr (CENTRE) {
    constexpr uint32_t k1024 = 0x64006400u;
    const uint32_t y = x >> 8;
    n[0] = hadd2_u(and_or(x, 0x000f000fu, k1024), 0xe408e408u);                // - 1032
    n[1] = hfma2_u(and_or(x, 0x00f000f0u, k1024), 0x2c002c00u, 0xd480d480u);  // / 16 - 72
    n[2] = hadd2_u(and_or(y, 0x000f000fu, k1024), 0xe408e408u);
    n[3] = hfma2_u(and_or(y, 0x00f000f0u, k1024), 0x2c002c00u, 0xd480d480u);
  } else {
    n[0] = x & 0x000f000fu;
    n[1] = x & 0x00f000f0u;
    x >>= 8;
    n[2] = x & 0x000f000fu;
    n[3] = x & 0x00f000f0u;
  }
}
// z + 8 s of two fp16 pairs, times `unit`, as a sum of two halves each
__device__ __forceinline__ void centre_zero(uint32_t& z, uint32_t& low, uint32_t s, float unit) {
  const float a = fmaf(8.f, half_lo(s), half_lo(z)) * unit, b = fmaf(8.f, half_hi(s), half_hi(z)) * unit;
  z = pack_h2(a, b);
  low = pack_h2(a - half_lo(z), b - half_hi(z));
}

// PREC 0: bf16 queries and outputs; 1: fp16 (probabilities in two halves); 2: fp32 (queries
// in two halves as well).  NT: query heads served, in eights.
template <int G, int NT, int PREC>
__global__ void __launch_bounds__(Int4Cfg<G, NT>::kWarps * 32, Int4Cfg<G, NT>::kCtas) int4_decode_mma_kernel(const CacheDecodeArgs a) {
  using S = Int4Tile<G>;
  constexpr int W = Int4Cfg<G, NT>::kWarps, ST = Int4Cfg<G, NT>::kStages;
  constexpr int D = 32 * G, HN = 8 * NT;
  constexpr bool kCentreK = PREC == 2;
  constexpr float kSlack = 4.f, kUnit2 = 15.f - kSlack;
  constexpr float kUnitK = kCentreK ? 1.f : 16777216.f;
  static_assert(NT * G <= W, "a warp prepares one group of query values");
  extern __shared__ __align__(128) unsigned char i4_smem[];
  __shared__ __align__(16) uint32_t s_q[PREC == 2 ? 2 : 1][NT * G][32][4];  // query fragments
  __shared__ float s_big[NT * G][8], s_sum[NT * G][8], s_unit[HN];
  __shared__ float s_f[HN][16];
  __shared__ unsigned s_live[W][ST];
  __shared__ int pre[kFlatBatch + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  unsigned char* ring = i4_smem + warp * (ST * S::kStage);
  if (a.ctas || a.weights) pdl_trigger();  // the kernel that joins the partials comes next
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

    // ---- rows of the next tiles.  A tile's page is fetched one tile before its loads are issued.
    // A full tile inside one page takes one look-up, good for the `run` full tiles that are left in
    // the page, from row `flat` on; other tiles have a token, a page and a row a lane.
    int token = -1, page = -1, page_off = 0, run = 0, flat = 0;
    bool one_page = false;
    const auto fetch = [&]() {
      const int first = tile_token<S::kTok>(a, plan, b, next_tile, 0), last = tile_token<S::kTok>(a, plan, b, next_tile, S::kTok - 1);
      one_page = false;
      if (first >= 0 && last >= 0) {
        page = token_page(a, b, first, page_off);
        token = first;
        one_page = page_off + S::kTok <= a.addr.page_size;
      }
      if (!one_page) {
        token = tile_token<S::kTok>(a, plan, b, next_tile, lane);
        page = token < 0 ? -1 : token_page(a, b, token, page_off);
      }
    };
    if (next_tile < end_tile) fetch();
    const unsigned char* k_lane = static_cast<const unsigned char*>(a.k) + lane * 16;
    const unsigned char* v_lane = static_cast<const unsigned char*>(a.v) + lane * 16;
    const unsigned char* kz_lane = reinterpret_cast<const unsigned char*>(a.k_scales) + lane * S::kScaleChunk;
    const unsigned char* vz_lane = reinterpret_cast<const unsigned char*>(a.v_scales) + lane * S::kScaleChunk;
    const int put = S::at(lane / G, lane % G * 16);
    const auto issue = [&](int stage) {
      if (next_tile < end_tile) {
        const uint32_t base = smem_u32(ring + stage * S::kStage);
        constexpr int per = S::kScaleRow / S::kScaleChunk;
        int row = -1;
        if (run == 0) {
          row = static_cast<int>(page_row(a, b, h, token, page, page_off));
          if (one_page && row >= 0) {
            flat = row;
            run = min(a.addr.page_size - page_off, plan.ctx - token) / S::kTok;
          }
        }
        if (run > 0) {
          // 32 rows on end: one address an array
          if (lane == 0) s_live[warp][stage] = 0xffffffffu;
          const unsigned char* kp = k_lane + static_cast<int64_t>(flat) * S::kRow;
          const unsigned char* vp = v_lane + static_cast<int64_t>(flat) * S::kRow;
#pragma unroll
          for (int i = 0; i < G; ++i) {
            const int c = i * 32 + lane;
            // 8 rows on, the permutation is the same
            const uint32_t dst = base + (32 / G % 8 == 0 && 32 % G == 0 ? put + i * 512 : S::at(c / G, (c % G) * 16));
            cp_async<16>(dst, kp + i * 512, 16);
            cp_async<16>(dst + S::kCodes, vp + i * 512, 16);
          }
          const unsigned char* kz = kz_lane + static_cast<int64_t>(flat) * S::kScaleRow;
          const unsigned char* vz = vz_lane + static_cast<int64_t>(flat) * S::kScaleRow;
#pragma unroll
          for (int i = 0; i < per; ++i) {
            const uint32_t dst = base + 2 * S::kCodes + (i * 32 + lane) * S::kScaleChunk;
            cp_async<S::kScaleChunk>(dst, kz + i * 32 * S::kScaleChunk, S::kScaleChunk);
            cp_async<S::kScaleChunk>(dst + S::kScales, vz + i * 32 * S::kScaleChunk, S::kScaleChunk);
          }
          flat += S::kTok;
          --run;
        } else {
          const unsigned live = __ballot_sync(0xffffffffu, row >= 0);
          if (lane == 0) s_live[warp][stage] = live;
#pragma unroll
          for (int i = 0; i < G; ++i) {
            const int c = i * 32 + lane, tok = c / G, off = (c % G) * 16;
            const int r = __shfl_sync(0xffffffffu, row, tok);
            const int64_t src = static_cast<int64_t>(max(r, 0)) * S::kRow + off;
            const int n = r >= 0 ? 16 : 0;
            cp_async<16>(base + S::at(tok, off), static_cast<const unsigned char*>(a.k) + src, n);
            cp_async<16>(base + S::kCodes + S::at(tok, off), static_cast<const unsigned char*>(a.v) + src, n);
          }
#pragma unroll
          for (int i = 0; i < per; ++i) {
            const int c = i * 32 + lane, tok = c / per, off = (c % per) * S::kScaleChunk;
            const int r = __shfl_sync(0xffffffffu, row, tok);
            const int64_t src = static_cast<int64_t>(max(r, 0)) * S::kScaleRow + off;
            const int n = r >= 0 ? S::kScaleChunk : 0;
            const uint32_t dst = base + 2 * S::kCodes + tok * S::kScaleRow + off;
            cp_async<S::kScaleChunk>(dst, reinterpret_cast<const unsigned char*>(a.k_scales) + src, n);
            cp_async<S::kScaleChunk>(dst + S::kScales, reinterpret_cast<const unsigned char*>(a.v_scales) + src, n);
          }
        }
        if (++next_tile < end_tile && run == 0) fetch();
      }
      cp_async_commit();
    };
    issue(0);

    // ---- the queries as B fragments, a group of 32 values (of 8 heads) a warp.  A row is scaled
    // by a power of two to a largest value in [2^9, 2^10): fp16 then holds 16-bit queries exactly,
    // and group sums stay in range.
    float x[8], big = 0.f;
    if (warp < NT * G) {
      const int head = warp / G * 8 + g;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
      if (head < heads) load8_any(a.q, a.dtype, (q0 + head) * D + 32 * (warp % G) + 8 * t, a.q_vec, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(x[i]));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      s_big[warp][g] = big;
    }
    __syncthreads();
    if (warp < NT * G) {
      const int n = warp / G;
#pragma unroll
      for (int j = 0; j < G; ++j) big = fmaxf(big, s_big[n * G + j][g]);
      int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;  // floor(log2) of a normal number
      e = big == 0.f || e == 128 ? 9 : min(max(e, -110), 120);
      const float up = __uint_as_float(static_cast<uint32_t>(127 - e + 9) << 23);
      s_unit[n * 8 + g] = __uint_as_float(static_cast<uint32_t>(127 + e - 9) << 23) * a.scale_log2;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += x[i] *= up;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = !kCentreK && i & 1 ? 0.0625f : 1.f;
        hi[i] = pack_h2(x[i] * f, x[i + 4] * f);
        lo[i] = pack_h2(x[i] * f - half_lo(hi[i]), x[i + 4] * f - half_hi(hi[i]));
      }
      *reinterpret_cast<uint4*>(s_q[0][warp][lane]) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if constexpr (PREC == 2) *reinterpret_cast<uint4*>(s_q[PREC == 2][warp][lane]) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      s_sum[warp][g] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int s = 1; s < ST - 1; ++s) issue(s);
    uint32_t qb[NT][G][2][2], ql[NT][G][2][2], qz[NT][2];
    float q_unit[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < G; ++j) {
        *reinterpret_cast<uint4*>(&qb[n][j][0][0]) = *reinterpret_cast<const uint4*>(s_q[0][n * G + j][lane]);
        if constexpr (PREC == 2)
          *reinterpret_cast<uint4*>(&ql[n][j][0][0]) = *reinterpret_cast<const uint4*>(s_q[PREC == 2][n * G + j][lane]);
      }
      q_unit[n][0] = s_unit[n * 8 + 2 * t];
      q_unit[n][1] = s_unit[n * 8 + 2 * t + 1];
      // sums of groups 2t and 2t + 1
      const float z0 = 2 * t < G ? s_sum[n * G + 2 * t][g] : 0.f, z1 = 2 * t + 1 < G ? s_sum[n * G + 2 * t + 1][g] : 0.f;
      qz[n][0] = pack_h2(z0, z1);
      qz[n][1] = pack_h2(z0 - half_lo(qz[n][0]), z1 - half_hi(qz[n][0]));
    }
    // a lane's places in a stage; 8 rows on, the permutation is the same
    const int k_at = S::at(g, 4 * G * t), k_at2 = G == 8 ? S::at(g, 4 * G * t + 16) : 0;
    const int v_at = S::at(2 * t, 2 * G * g), v_at1 = S::at(2 * t + 1, 2 * G * g);

    // m: about the largest score so far, in the scaled query's units; base2: what an exponent starts from,
    // log2(unit) - m * q_unit
    float o[NT][G][2][4], zo[NT][4], m[NT][2], limit[NT][2], base2[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < G; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][j][u][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) zo[n][e] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      limit[n][0] = limit[n][1] = -INFINITY;
      base2[n][0] = base2[n][1] = kUnit2;
      l[n][0] = l[n][1] = 0.f;
    }
    // Probabilities and all sums of them are held times unit = 2^(15 - kSlack) / top, top a power
    // of two no V scale so far exceeds (1 at least): fp16 then holds p and p s, and the lower
    // halves of those, over the widest range.
    uint32_t top = 0x3c00u;
    float unit2 = kUnit2;
    // z + 8 s is held as it is, or, once scales above kWide = 4096 or zeros above kHigh = 28672 turned
    // up (it might pass fp16's range), in sixteenths.  Zeros are compared as signed numbers.
    constexpr uint32_t kWide = 0x6c00u, kHigh = 0x77007700u;
    float z_unit = 1.f;
    uint32_t high = kHigh;  // fp16's NaN, which nothing is above, once z_unit is a sixteenth

    int stage = 0;
#pragma unroll 1
    for (int done = 0; done < n_tiles; ++done) {
      cp_async_wait<ST - 2>();
      __syncwarp();
      issue(stage == 0 ? ST - 1 : stage - 1);  // the stage that the previous tile left
      const unsigned char* ks = ring + stage * S::kStage;
      const unsigned char* vs = ks + S::kCodes;
      const unsigned char* ksc = ks + 2 * S::kCodes;
      const unsigned char* vsc = ksc + S::kScales;
      const unsigned live = s_live[warp][stage];
      float sc[2][NT][4], mn[NT][2];
      float zk_unit = 1.f;  // as z_unit, for this tile of K
      if constexpr (kCentreK) {
        uint32_t ktop[(G + 1) / 2], kzero[(G + 1) / 2], most = 0, zero = kHigh;
        lds_words<2 * G>(ksc + lane * S::kScaleRow, ktop);
        lds_words<2 * G>(ksc + lane * S::kScaleRow + 2 * G, kzero);
#pragma unroll
        for (int i = 0; i < (G + 1) / 2; ++i) most = __vmaxu2(most, ktop[i]), zero = __vmaxs2(zero, kzero[i]);
        if (__any_sync(0xffffffffu, max(most & 0xffffu, most >> 16) > kWide || zero != kHigh)) zk_unit = 0.0625f;
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int r0 = hh * 16 + g, r1 = r0 + 8;
        uint32_t w0[G], w1[G], s0[(G + 1) / 2], s1[(G + 1) / 2];
        const unsigned char* kr = ks + hh * 16 * S::kRow;
        if constexpr (G == 8) {
          lds_words<16>(kr + k_at, w0);
          lds_words<16>(kr + k_at2, w0 + 4);
          lds_words<16>(kr + 8 * S::kRow + k_at, w1);
          lds_words<16>(kr + 8 * S::kRow + k_at2, w1 + 4);
        } else {
          lds_words<4 * G>(kr + k_at, w0);
          lds_words<4 * G>(kr + 8 * S::kRow + k_at, w1);
        }
        lds_words<2 * G>(ksc + r0 * S::kScaleRow, s0);
        lds_words<2 * G>(ksc + r1 * S::kScaleRow, s1);
        // zeros of groups 2t and 2t + 1; past G any of the row's will do: the query sums are 0 there
        const auto pair_at = [&](int r, int first) -> uint32_t {
          const unsigned char* p = ksc + r * S::kScaleRow + 2 * first;
          if constexpr (G % 2 == 0) return reinterpret_cast<const uint32_t*>(p)[t % (G / 2)];
          const unsigned short* x = reinterpret_cast<const unsigned short*>(p);
          return __byte_perm(x[2 * t % G], x[(2 * t + 1) % G], 0x5410);
        };
        uint32_t z0 = pair_at(r0, G), z1 = pair_at(r1, G), zl0 = 0, zl1 = 0;
        if constexpr (kCentreK) {
          centre_zero(z0, zl0, pair_at(r0, 0), zk_unit);
          centre_zero(z1, zl1, pair_at(r1, 0), zk_unit);
        }
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
        const auto group = [&](auto jc) {
          constexpr int j = decltype(jc)::value;
          uint32_t x0[4], x1[4];
          nibbles<kCentreK>(pair16<j, G + j>(w0, w0), x0);
          nibbles<kCentreK>(pair16<j, G + j>(w1, w1), x1);
          const float f0 = j & 1 ? half_hi(s0[j / 2]) : half_lo(s0[j / 2]);
          const float f1 = j & 1 ? half_hi(s1[j / 2]) : half_lo(s1[j / 2]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float c[4];
            mma_f16_zero(c, x0[0], x1[0], x0[1], x1[1], qb[n][j][0][0], qb[n][j][0][1]);
            mma_f16(c, x0[2], x1[2], x0[3], x1[3], qb[n][j][1][0], qb[n][j][1][1]);
            if constexpr (PREC == 2) {
              mma_f16(c, x0[0], x1[0], x0[1], x1[1], ql[n][j][0][0], ql[n][j][0][1]);
              mma_f16(c, x0[2], x1[2], x0[3], x1[3], ql[n][j][1][0], ql[n][j][1][1]);
            }
            acc[n][0] = fmaf(f0, c[0], acc[n][0]);
            acc[n][1] = fmaf(f0, c[1], acc[n][1]);
            acc[n][2] = fmaf(f1, c[2], acc[n][2]);
            acc[n][3] = fmaf(f1, c[3], acc[n][3]);
          }
        };
        for_each_index(group, std::make_integer_sequence<int, G>{});
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float c[4];
          mma_f16_zero(c, z0, z1, z0, z1, qz[n][0], qz[n][1]);
          if constexpr (kCentreK) mma_f16(c, zl0, zl1, zl0, zl1, qz[n][0], qz[n][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[hh][n][e] = kCentreK ? fmaf(c[e], 1.f / zk_unit, acc[n][e]) : fmaf(acc[n][e], kUnitK, c[e]);
        }
      }
      if (live != 0xffffffffu) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(live >> (hh * 16 + g + (e < 2 ? 0 : 8)) & 1)) sc[hh][n][e] = -INFINITY;
      }
      if (a.scores) {
        // [token][head of the group]; a lane's two heads lie on end
        const int64_t at = (static_cast<int64_t>(b) * a.Hkv + h) * a.cap;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const int tok = plan.seg + (first_tile + done) * S::kTok + hh * 16 + g + 4 * e;
            if (tok < plan.lo || tok >= plan.ctx) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int head = n * 8 + 2 * t;
              float* p = a.scores + (at + tok) * a.group + head0 + head;
              const float x = sc[hh][n][e] * q_unit[n][0], y = sc[hh][n][e + 1] * q_unit[n][1];
              if (head + 1 < heads && a.group % 2 == 0) {
                *reinterpret_cast<float2*>(p) = make_float2(x, y);
              } else if (head < heads) {
                p[0] = x;
                if (head + 1 < heads) p[1] = y;
              }
            }
          }
      }
      // ---- running maximum and sum.  The maximum is only moved once a score passes it by
      // 2^kSlack: until then probabilities reach 2^kSlack instead of 1, for which unit leaves room.
      bool up = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mn[n][c] = fmaxf(fmaxf(sc[0][n][c], sc[0][n][2 + c]), fmaxf(sc[1][n][c], sc[1][n][2 + c]));
          up |= mn[n][c] > limit[n][c];
        }
      // largest V scale and zero of the tile: this lane's token (NaN and negative scales count as
      // fp16's largest)
      uint32_t vtop[(G + 1) / 2], vzero[(G + 1) / 2], most = 0, zero = high;
      lds_words<2 * G>(vsc + lane * S::kScaleRow, vtop);
      lds_words<2 * G>(vsc + lane * S::kScaleRow + 2 * G, vzero);
#pragma unroll
      for (int i = 0; i < (G + 1) / 2; ++i) most = __vmaxu2(most, vtop[i]), zero = __vmaxs2(zero, vzero[i]);
      most = max(most & 0xffffu, most >> 16);
      if (__any_sync(0xffffffffu, up || most > top || zero != high)) {
        float shrink = 1.f;
        const uint32_t all = min(__reduce_max_sync(0xffffffffu, most), 0x7bffu);
        if (all > top) {
          const uint32_t to = (all + 0x3ffu) & 0x7c00u;  // the next power of two
          shrink = __uint_as_float((127u - ((to - top) >> 10)) << 23);
          unit2 -= static_cast<float>((to - top) >> 10);
          top = to;
        }
        if (z_unit == 1.f && (top > kWide || __any_sync(0xffffffffu, zero != high))) {
          z_unit = 0.0625f;
          high = 0x7fff7fffu;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) zo[n][e] *= z_unit;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = mn[n][c];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
            x = fmaxf(m[n][c], x);
            // nothing seen yet: 0, not exp2(-inf + inf)
            f[c] = m[n][c] == -INFINITY ? 0.f : fast_exp2((m[n][c] - x) * q_unit[n][c]) * shrink;
            l[n][c] *= f[c];
            m[n][c] = x;
            limit[n][c] = x + kSlack / q_unit[n][c];
            base2[n][c] = x == -INFINITY ? unit2 : fmaf(-x, q_unit[n][c], unit2);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) zo[n][e] *= f[e & 1];
#pragma unroll
          for (int j = 0; j < G; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[n][j][u][e] *= f[e & 1];
        }
      }
      // ---- P V
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float p[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[n][e] = fast_exp2(fmaf(sc[hh][n][e], q_unit[n][e & 1], base2[n][e & 1]));
            l[n][e & 1] += p[n][e];
          }
        const int rt = hh * 16 + 2 * t;  // this lane's tokens in the product: rt, rt+1, rt+8, rt+9
        uint32_t v0[(G + 1) / 2], v1[(G + 1) / 2], v2[(G + 1) / 2], v3[(G + 1) / 2];
        const unsigned char* vr = vs + hh * 16 * S::kRow;
        lds_words<2 * G>(vr + v_at, v0);
        lds_words<2 * G>(vr + v_at1, v1);
        lds_words<2 * G>(vr + 8 * S::kRow + v_at, v2);
        lds_words<2 * G>(vr + 8 * S::kRow + v_at1, v3);
        uint32_t b0[NT], b1[NT], bl0[NT], bl1[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint32_t h0 = pack_h2(p[n][0], p[n][1]), h1 = pack_h2(p[n][2], p[n][3]);
          b0[n] = movmatrix_trans(h0);
          b1[n] = movmatrix_trans(h1);
          if constexpr (PREC > 0) {
            bl0[n] = movmatrix_trans(pack_h2(p[n][0] - half_lo(h0), p[n][1] - half_hi(h0)));
            bl1[n] = movmatrix_trans(pack_h2(p[n][2] - half_lo(h1), p[n][3] - half_hi(h1)));
          }
        }
        {  // z + 8 s: row g is group g, row g + 8 (PREC > 0) what its fp16 value leaves
          // (rows past G are not used)
          const unsigned short* x = reinterpret_cast<const unsigned short*>(vsc + rt * S::kScaleRow) + g % G;
          constexpr int kNext = S::kScaleRow / 2;
          uint32_t za = __byte_perm(x[G], x[G + kNext], 0x5410), la = 0;
          uint32_t zb = __byte_perm(x[G + 8 * kNext], x[G + 9 * kNext], 0x5410), lb = 0;
          const uint32_t ta = __byte_perm(x[0], x[kNext], 0x5410), tb = __byte_perm(x[8 * kNext], x[9 * kNext], 0x5410);
          if constexpr (PREC > 0) {
            centre_zero(za, la, ta, z_unit);
            centre_zero(zb, lb, tb, z_unit);
          } else {
            const uint32_t one = z_unit == 1.f ? 0x3c003c00u : 0x2c002c00u, eight = z_unit == 1.f ? 0x48004800u : 0x38003800u;
            za = hfma2_u(ta, eight, hmul2_u(za, one));
            zb = hfma2_u(tb, eight, hmul2_u(zb, one));
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(zo[n], za, la, zb, lb, b0[n], b1[n]);
            if constexpr (PREC > 0) mma_f16(zo[n], za, la, zb, lb, bl0[n], bl1[n]);
          }
        }
        uint32_t sa[(G + 1) / 2], sb[(G + 1) / 2], sd[(G + 1) / 2], se[(G + 1) / 2];
        if constexpr (PREC == 0) {
          lds_words<2 * G>(vsc + rt * S::kScaleRow, sa);
          lds_words<2 * G>(vsc + (rt + 1) * S::kScaleRow, sb);
          lds_words<2 * G>(vsc + (rt + 8) * S::kScaleRow, sd);
          lds_words<2 * G>(vsc + (rt + 9) * S::kScaleRow, se);
        } else {
          lds_words<2 * G>(vsc + (hh * 16 + g) * S::kScaleRow, sa);
          lds_words<2 * G>(vsc + (hh * 16 + g + 8) * S::kScaleRow, sb);
        }
        const auto group = [&](auto jc) {
          constexpr int j = decltype(jc)::value;
          uint32_t x0[4], x1[4];
          nibbles<true>(pair16<j, j>(v0, v1), x0);
          nibbles<true>(pair16<j, j>(v2, v3), x1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (PREC == 0) {
              const uint32_t y0 = hmul2_u(b0[n], pair16<j, j>(sa, sb)), y1 = hmul2_u(b1[n], pair16<j, j>(sd, se));
              mma_f16(o[n][j][0], x0[0], x0[1], x1[0], x1[1], y0, y1);
              mma_f16(o[n][j][1], x0[2], x0[3], x1[2], x1[3], y0, y1);
            } else {
              const float f0 = j & 1 ? half_hi(sa[j / 2]) : half_lo(sa[j / 2]);
              const float f1 = j & 1 ? half_hi(sb[j / 2]) : half_lo(sb[j / 2]);
              const float y[4] = {p[n][0] * f0, p[n][1] * f0, p[n][2] * f1, p[n][3] * f1};
              const uint32_t h0 = pack_h2(y[0], y[1]), h1 = pack_h2(y[2], y[3]);
              const uint32_t y0 = movmatrix_trans(h0), y1 = movmatrix_trans(h1);
              const uint32_t u0 = movmatrix_trans(pack_h2(y[0] - half_lo(h0), y[1] - half_hi(h0)));
              const uint32_t u1 = movmatrix_trans(pack_h2(y[2] - half_lo(h1), y[3] - half_hi(h1)));
              mma_f16(o[n][j][0], x0[0], x0[1], x1[0], x1[1], y0, y1);
              mma_f16(o[n][j][1], x0[2], x0[3], x1[2], x1[3], y0, y1);
              mma_f16(o[n][j][0], x0[0], x0[1], x1[0], x1[1], u0, u1);
              mma_f16(o[n][j][1], x0[2], x0[3], x1[2], x1[3], u0, u1);
            }
          }
        };
        for_each_index(group, std::make_integer_sequence<int, G>{});
      }
      stage = stage == ST - 1 ? 0 : stage + 1;
    }

    // ---- merge the warps (the ring is free once every copy has landed)
    cp_async_wait<0>();
    __syncthreads();
    constexpr int kLd = D + 4;  // row: D outputs, the maximum, the sum
    float* buf = reinterpret_cast<float*>(i4_smem);
    const float one = exp2f(-unit2);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s = l[n][c];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        float* row = buf + (warp * HN + n * 8 + 2 * t + c) * kLd;
        if (g == 0) row[D] = m[n][c] == -INFINITY ? -INFINITY : m[n][c] * q_unit[n][c], row[D + 1] = s * one;
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const float z = __shfl_sync(0xffffffffu, zo[n][c] + zo[n][2 + c], j * 4 + t) * (1.f / z_unit);
#pragma unroll
          for (int u = 0; u < 2; ++u)
            *reinterpret_cast<float2*>(row + 32 * j + 4 * g + 2 * u) =
                make_float2((o[n][j][u][c] + z) * one, (o[n][j][u][2 + c] + z) * one);
        }
      }
    }
    merge_warps<W, HN, D>(a, seg, q0, heads, buf, s_f);
    __syncthreads();  // the next segment's loads reuse the buffer
  }
}

template <int G, int NT>
constexpr int int4_smem_bytes() {
  constexpr int W = Int4Cfg<G, NT>::kWarps, ring = W * Int4Cfg<G, NT>::kStages * Int4Tile<G>::kStage;
  constexpr int merge = W * 8 * NT * (32 * G + 4) * 4;
  return ring > merge ? ring : merge;
}
template <int G, int NT, int PREC>
int launch_int4_mma(const CacheDecodeArgs& a, cudaStream_t st) {
  auto kern = int4_decode_mma_kernel<G, NT, PREC>;
  constexpr int smem = int4_smem_bytes<G, NT>();
  SPA_CHECK_CUDA(spa_set_smem_once(kern, smem));
  kern<<<a.ctas ? a.ctas : a.B * a.Hkv * a.chunks, Int4Cfg<G, NT>::kWarps * 32, smem, st>>>(a);
  SPA_CHECK_CUDA(cudaGetLastError());
  return SPA_OK;
}
template <int G, int NT>
int launch_int4_prec(const CacheDecodeArgs& a, cudaStream_t st) {
  return a.dtype == SPA_BF16  ? launch_int4_mma<G, NT, 0>(a, st)
         : a.dtype == SPA_F16 ? launch_int4_mma<G, NT, 1>(a, st)
                              : launch_int4_mma<G, NT, 2>(a, st);
}
// Query heads a CTA serves: one matrix column block of 8, or two where the registers allow
// (not at head_dim 256), so that up to 16 heads share one read of K and V.
inline int int4_mma_heads(int head_dim, int group) { return group > 8 && head_dim < 256 ? 16 : 8; }
inline int int4_mma_ctas(int head_dim, int heads) { return heads == 8 && head_dim <= 128 ? 3 : 1; }
inline bool int4_mma_serves(int head_dim, int64_t total_rows) {
  return (head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256) &&
         total_rows < (1ll << 31);  // rows travel between lanes as 32-bit numbers
}
inline int launch_int4_decode(const CacheDecodeArgs& a, cudaStream_t st) {
  const bool two = a.heads == 16;
  switch (a.D) {
    case 32: return two ? launch_int4_prec<1, 2>(a, st) : launch_int4_prec<1, 1>(a, st);
    case 64: return two ? launch_int4_prec<2, 2>(a, st) : launch_int4_prec<2, 1>(a, st);
    case 96: return two ? launch_int4_prec<3, 2>(a, st) : launch_int4_prec<3, 1>(a, st);
    case 128: return two ? launch_int4_prec<4, 2>(a, st) : launch_int4_prec<4, 1>(a, st);
    default: return launch_int4_prec<8, 1>(a, st);
  }
}

}  // namespace spa
