// The 4-bit paged cache: row format, append and read-back.
//
// A row (D values of one token of one kv head) is cut into G = D / 32 groups.  Of a group
// with extremes lo and hi:  s = half((hi - lo) * fl(1/15)), z = half(lo), both saturating,
// and n = clamp(rint((x - z) / s), 0, 15) with every step an IEEE fp32 operation (n = 0 where
// s = 0; a group with a NaN or an infinity gets s = z = NaN).  It stands for s * n + z.
//
// codes  [pages, Hkv, P, D / 2]: value d = 32 j + 4 g + i of a row is nibble i (low bits
//        first) of its 16-bit word g * G + j.  The eight lane groups of a matrix fragment
//        (g) so find the words of every group (j) side by side, and the four values of a
//        word always share a scale: the attention kernel loads a row with one or two wide
//        reads and never mixes two scales in one product.
// scales [pages, Hkv, P, 2, G] fp16: the row's scales, then its zeros.
//
// Groups of 32: 5 bits a value, and the smallest group whose scale is still one multiply
// for a whole k-step pair of the matrix instruction.
#pragma once

#include "common.cuh"

namespace spa {

constexpr int kInt4Group = 32;

struct Int4Rows {
  uint8_t* codes[2];  // K, V
  __half* scales[2];
  KvAddr addr;
  int B, H, T, G;
  const int32_t* positions;
  const int32_t* lens;  // nullptr: T of every sequence
};

// Row of token positions[b] + t, or -1 (with the error word set where a page is missing).
__device__ __forceinline__ int64_t int4_row(const Int4Rows& a, int b, int h, int t, bool lead) {
  const int64_t tok = static_cast<int64_t>(a.positions[b]) + t;
  if (tok < 0) return -1;
  const int64_t row = tok > 0x7fffffff ? -1 : a.addr.row(b, h, static_cast<int>(tok));
  if (row < 0 || row >= a.addr.total_rows) {
    if (lead) spa_raise(SPA_DEVERR_BAD_PAGE);
    return -1;
  }
  return row;
}

// Both kernels: a warp has a stretch of 32 rows of one (sequence, kv head) and takes 32 / G of
// them at a time.  Grid (B * Hkv, K or V, stretches): no index is divided but by G.  Codes
// change places in shared memory (a lane has a group's 8 words, a row's 16 bytes hold words of
// all groups), so that they move in 16-byte pieces.
//
// Bound by HBM (a row's 2 D bytes against its 5/8 D at 16 bits) as long as a value costs few
// instructions: 9 here to quantise one; with a group spread over 8 lanes and a division a value
// it was 63.  4 prompts of up to 8192 tokens, 8 heads of 128 in bf16: 62 us for both kernels (the mean
// of six draws of their lengths), 0.67 of the copy bandwidth (twice as long that way).
constexpr int kInt4Warps = 4, kInt4Stretch = 32;

// 32 consecutive values of a row as fp32; `vec` when 16-byte loads are allowed.
template <typename T>
__device__ __forceinline__ void load_group(const T* p, bool vec, float (&x)[32]) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = to_f32<T>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<float4*>(x + 4 * i) = reinterpret_cast<const float4*>(p)[i];
  } else {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = to_f32<T>(e[i]);
  }
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// A group's 8 words of 4 codes, its scale and zero.
__device__ __forceinline__ void quantise_group(const float (&x)[32], uint32_t (&word)[8], __half& s, __half& z) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 32; ++i) lo = min_nan(lo, x[i]), hi = max_nan(hi, x[i]);
  const bool bad = !(fabsf(lo) < INFINITY && fabsf(hi) < INFINITY);  // a NaN or an infinity among them
  s = __float2half_rn(fminf(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f), 65504.f));
  z = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f));
  const float sf = __half2float(s), zf = __half2float(z);
  if (bad) s = z = __ushort_as_half(0x7fff);
  // The quotient by Markstein's theorem (Computation of elementary functions on the IBM RISC
  // System/6000, 1990): with y the rounded reciprocal of s and q0 = fl(d y), the fused
  // q0 + (d - q0 s) y is d / s rounded.  Without a scale y = 0 and every code 0 (a NaN as well).
  // Adding 1.5 2^23 rounds to the integer, ties to even.
  constexpr float kMagic = 12582912.f;
  const float y = !bad && sf > 0.f ? __frcp_rn(sf) : 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    float n[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = __fsub_rn(x[4 * w + e], zf), q0 = __fmul_rn(d, y);
      const float q = fmaf(fmaf(-q0, sf, d), y, q0);
      n[e] = __fsub_rn(__fadd_rn(fminf(fmaxf(q, 0.f), 15.f), kMagic), kMagic);
    }
    word[w] = static_cast<uint32_t>(fmaf(n[3], 4096.f, fmaf(n[2], 256.f, fmaf(n[1], 16.f, n[0]))));
  }
}

template <typename T>
__global__ void __launch_bounds__(kInt4Warps * 32) int4_append_kernel(const Int4Rows a, const T* __restrict__ k_new,
                                                                      const T* __restrict__ v_new, int64_t sb,
                                                                      int64_t sh, int64_t st, int vec) {
  __shared__ __align__(16) uint16_t s_words[kInt4Warps][256];
  const int which = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H;
  const int len = a.lens ? min(a.lens[b], a.T) : a.T;
  const int t0 = (blockIdx.z * kInt4Warps + warp) * kInt4Stretch, t1 = min(t0 + kInt4Stretch, len);
  if (t0 >= t1) return;
  const T* src = (which ? v_new : k_new) + b * sb + h * sh;
  uint8_t* codes = which ? a.codes[1] : a.codes[0];
  __half* scales = which ? a.scales[1] : a.scales[0];
  const int64_t my_row = t0 + lane < t1 ? int4_row(a, b, h, t0 + lane, true) : -1;
  // this lane's row among the step's, and its group (its 16-byte piece when storing)
  const int rows = 32 / a.G, r = lane / a.G, j = lane - r * a.G;
  uint16_t* words = s_words[warp];
  for (int base = 0; base < t1 - t0; base += rows) {
    const int i = base + r;
    const bool in = r < rows && t0 + i < t1;
    const int64_t row = __shfl_sync(0xffffffffu, my_row, in ? i : 0);
    if (in && row >= 0) {
      float x[32];
      load_group<T>(src + (t0 + i) * st + j * kInt4Group, vec, x);
      uint32_t word[8];
      __half s, z;
      quantise_group(x, word, s, z);
#pragma unroll
      for (int g = 0; g < 8; ++g) words[r * a.G * 8 + g * a.G + j] = static_cast<uint16_t>(word[g]);
      scales[row * 2 * a.G + j] = s;
      scales[row * 2 * a.G + a.G + j] = z;
    }
    __syncwarp();
    if (in && row >= 0)
      *reinterpret_cast<uint4*>(codes + row * (a.G * 16) + j * 16) = *reinterpret_cast<const uint4*>(words + lane * 8);
    __syncwarp();
  }
}

// The values of tokens positions[b] + [0, T), zeros past lens[b] and where no page is.
template <typename T>
__global__ void __launch_bounds__(kInt4Warps * 32) int4_read_kernel(const Int4Rows a, T* __restrict__ k_out,
                                                                    T* __restrict__ v_out) {
  __shared__ __align__(16) uint16_t s_words[kInt4Warps][256];
  __shared__ float2 s_scale[kInt4Warps][32];
  const int which = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H;
  const int len = a.lens ? min(a.lens[b], a.T) : a.T;
  const int t0 = (blockIdx.z * kInt4Warps + warp) * kInt4Stretch, t1 = min(t0 + kInt4Stretch, a.T);
  if (t0 >= t1) return;
  const uint8_t* codes = which ? a.codes[1] : a.codes[0];
  const __half* scales = which ? a.scales[1] : a.scales[0];
  T* dst = (which ? v_out : k_out) + static_cast<int64_t>(blockIdx.x) * a.T * (a.G * kInt4Group);
  const int64_t my_row = t0 + lane < min(t1, len) ? int4_row(a, b, h, t0 + lane, true) : -1;
  const int rows = 32 / a.G, r = lane / a.G, j = lane - r * a.G;
  uint16_t* words = s_words[warp];
  // words of group j of row r lie at 8 G r + j + G g
  const int grp0 = lane >> 2, row0 = grp0 / a.G, first_j = grp0 - row0 * a.G;
  const int first_word = row0 * a.G * 8 + first_j + (lane & 3) * 2 * a.G;
  const int eight_rows = 8 / a.G, eight_j = 8 - eight_rows * a.G, eight_words = eight_rows * a.G * 8 + eight_j;
  for (int base = 0; base < t1 - t0; base += rows) {
    const int i = base + r;
    const bool in = r < rows && t0 + i < t1;
    const int64_t row = __shfl_sync(0xffffffffu, my_row, in ? i : 0);
    uint4 piece = make_uint4(0, 0, 0, 0);
    float2 sz = make_float2(0.f, 0.f);
    if (in && row >= 0) {
      piece = *reinterpret_cast<const uint4*>(codes + row * (a.G * 16) + j * 16);
      sz.x = __half2float(scales[row * 2 * a.G + j]);
      sz.y = __half2float(scales[row * 2 * a.G + a.G + j]);
    }
    *reinterpret_cast<uint4*>(words + lane * 8) = piece;
    s_scale[warp][lane] = sz;
    __syncwarp();
    // eight values a lane: words 2 q and 2 q + 1 of a group; the step's rows lie on end in dst
    const int total = min(rows, t1 - t0 - base) * a.G * 4;
    int at = first_word, jj = first_j;  // word 0 of the lane's group, and the group's number in its row
    for (int o = lane; o < total; o += 32) {
      const uint32_t w0 = words[at], w1 = words[at + a.G];
      const float2 c = s_scale[warp][o >> 2];
      // eight groups on
      jj += eight_j;
      at += eight_words;
      if (jj >= a.G) jj -= a.G, at += a.G * 7;
      // code e of both words at once: under the exponent of 1024 it is the fp16 1024 + n
      T x[8];
      const uint32_t w = w0 | w1 << 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t y;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(w >> (4 * e)), "r"(0x000f000fu), "r"(0x64006400u));
        const float2 n = __half22float2(__hsub2(*reinterpret_cast<const __half2*>(&y), __float2half2_rn(1024.f)));
        x[e] = from_f32<T>(fmaf(c.x, n.x, c.y));
        x[4 + e] = from_f32<T>(fmaf(c.x, n.y, c.y));
      }
      T* p = dst + static_cast<int64_t>(t0 + base) * (a.G * kInt4Group) + o * 8;
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(x);
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p + 4) = *reinterpret_cast<const uint4*>(x + 4);
    }
    __syncwarp();
  }
}

inline bool int4_rows_ok(const spa_kv_layout* kv, const void* ks, const void* vs, int batch, int kv_heads,
                         int head_dim) {
  return kv && kv->k && kv->v && ks && vs && batch > 0 && kv_heads > 0 && head_dim > 0 && head_dim <= 256 &&
         head_dim % kInt4Group == 0 && kv->page_size > 0 && kv->total_rows > 0 &&
         (!kv->page_table || kv->table_stride > 0) && reinterpret_cast<uintptr_t>(kv->k) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(kv->v) % 16 == 0 && reinterpret_cast<uintptr_t>(ks) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(vs) % 16 == 0;
}
inline Int4Rows int4_rows(const spa_kv_layout& kv, void* ks, void* vs, int batch, int kv_heads, int head_dim,
                          int tokens, const int32_t* positions, const int32_t* lens) {
  Int4Rows a;
  a.codes[0] = static_cast<uint8_t*>(const_cast<void*>(kv.k));
  a.codes[1] = static_cast<uint8_t*>(const_cast<void*>(kv.v));
  a.scales[0] = static_cast<__half*>(ks);
  a.scales[1] = static_cast<__half*>(vs);
  a.addr = make_kv_addr(kv);
  a.B = batch;
  a.H = kv_heads;
  a.T = tokens;
  a.G = head_dim / kInt4Group;
  a.positions = positions;
  a.lens = lens;
  return a;
}
inline dim3 int4_grid(const Int4Rows& a) {
  constexpr int per = kInt4Warps * kInt4Stretch;
  return dim3(a.B * a.H, 2, (a.T + per - 1) / per);
}

}  // namespace spa

extern "C" int spa_int4_append(const spa_kv_layout* kv, void* k_scales, void* v_scales, int dtype, int batch,
                               int kv_heads, int head_dim, int tokens, const void* k_new, const void* v_new,
                               int64_t stride_b, int64_t stride_h, int64_t stride_t, const int32_t* positions,
                               const int32_t* new_lens, spa_stream_t stream) {
  if (!spa::int4_rows_ok(kv, k_scales, v_scales, batch, kv_heads, head_dim) || !dtype_ok(dtype))
    return SPA_ERR_INVALID;
  if (!positions || tokens < 0 || (tokens > 0 && (!k_new || !v_new))) return SPA_ERR_INVALID;
  if (tokens == 0) return SPA_OK;
  if (tokens > 65535 * spa::kInt4Warps * spa::kInt4Stretch) return SPA_ERR_UNSUPPORTED;
  const spa::Int4Rows a = spa::int4_rows(*kv, k_scales, v_scales, batch, kv_heads, head_dim, tokens, positions, new_lens);
  const int64_t es = dtype_size(dtype);
  const int vec = (reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new) | (stride_b * es) |
                   (stride_h * es) | (stride_t * es)) % 16 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid = spa::int4_grid(a);
  if (dtype == SPA_F32)
    spa::int4_append_kernel<float><<<grid, spa::kInt4Warps * 32, 0, st>>>(a, static_cast<const float*>(k_new),
                                                          static_cast<const float*>(v_new), stride_b, stride_h,
                                                          stride_t, vec);
  else if (dtype == SPA_F16)
    spa::int4_append_kernel<__half><<<grid, spa::kInt4Warps * 32, 0, st>>>(a, static_cast<const __half*>(k_new),
                                                           static_cast<const __half*>(v_new), stride_b, stride_h,
                                                           stride_t, vec);
  else
    spa::int4_append_kernel<__nv_bfloat16><<<grid, spa::kInt4Warps * 32, 0, st>>>(a, static_cast<const __nv_bfloat16*>(k_new),
                                                                  static_cast<const __nv_bfloat16*>(v_new), stride_b,
                                                                  stride_h, stride_t, vec);
  SPA_CHECK_CUDA(cudaGetLastError());
  return SPA_OK;
}

extern "C" int spa_int4_read(const spa_kv_layout* kv, const void* k_scales, const void* v_scales, int dtype,
                             int batch, int kv_heads, int head_dim, int tokens, const int32_t* positions,
                             const int32_t* lens, void* k_out, void* v_out, spa_stream_t stream) {
  if (!spa::int4_rows_ok(kv, k_scales, v_scales, batch, kv_heads, head_dim) || !dtype_ok(dtype))
    return SPA_ERR_INVALID;
  if (!positions || tokens < 0 || (tokens > 0 && (!k_out || !v_out))) return SPA_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16) return SPA_ERR_INVALID;
  if (tokens == 0) return SPA_OK;
  if (tokens > 65535 * spa::kInt4Warps * spa::kInt4Stretch) return SPA_ERR_UNSUPPORTED;
  const spa::Int4Rows a = spa::int4_rows(*kv, const_cast<void*>(k_scales), const_cast<void*>(v_scales), batch,
                                         kv_heads, head_dim, tokens, positions, lens);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid = spa::int4_grid(a);
  if (dtype == SPA_F32)
    spa::int4_read_kernel<float><<<grid, spa::kInt4Warps * 32, 0, st>>>(a, static_cast<float*>(k_out), static_cast<float*>(v_out));
  else if (dtype == SPA_F16)
    spa::int4_read_kernel<__half><<<grid, spa::kInt4Warps * 32, 0, st>>>(a, static_cast<__half*>(k_out), static_cast<__half*>(v_out));
  else
    spa::int4_read_kernel<__nv_bfloat16><<<grid, spa::kInt4Warps * 32, 0, st>>>(a, static_cast<__nv_bfloat16*>(k_out),
                                                                static_cast<__nv_bfloat16*>(v_out));
  SPA_CHECK_CUDA(cudaGetLastError());
  return SPA_OK;
}
