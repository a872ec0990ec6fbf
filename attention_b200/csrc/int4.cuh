// The 4-bit paged cache: row format, append and read-back.
//
// A row (D values of one token of one kv head) is cut into G = D / 32 groups.  Of a group
// with extremes lo and hi:  s = half((hi - lo) / 15), z = half(lo), both saturating, and
// n = clamp(rint((x - z) / s), 0, 15) with every step an IEEE fp32 operation (n = 0 where
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

// Four consecutive values of a row as fp32; `vec` when the address allows one wide load.
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, float (&x)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(p[i]);
  }
}

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

// Eight lanes per group, four values per lane.  blockIdx.y: K or V.
template <typename T>
__global__ void __launch_bounds__(256) int4_append_kernel(const Int4Rows a, const T* __restrict__ k_new,
                                                          const T* __restrict__ v_new, int64_t sb, int64_t sh,
                                                          int64_t st, int vec) {
  const int which = blockIdx.y, g = threadIdx.x & 7;
  const T* src = which ? v_new : k_new;
  const int64_t groups = static_cast<int64_t>(a.B) * a.H * a.T * a.G;
  const unsigned octet = 0xffu << (threadIdx.x & 24);
  for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) >> 3; i < groups; i += gridDim.x * 32ll) {
    const int j = static_cast<int>(i % a.G);
    const int64_t r = i / a.G;
    const int t = static_cast<int>(r % a.T);
    const int64_t bh = r / a.T;
    const int h = static_cast<int>(bh % a.H), b = static_cast<int>(bh / a.H);
    if (a.lens && t >= a.lens[b]) continue;
    const int64_t row = int4_row(a, b, h, t, g == 0);
    if (row < 0) continue;
    float x[4];
    load4<T>(src + b * sb + h * sh + t * st + j * kInt4Group + g * 4, vec, x);
    float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    // x - x is NaN for a NaN or an infinity, 0 otherwise
    float odd = (x[0] - x[0]) + (x[1] - x[1]) + (x[2] - x[2]) + (x[3] - x[3]);
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(octet, lo, off));
      hi = fmaxf(hi, __shfl_xor_sync(octet, hi, off));
      odd += __shfl_xor_sync(octet, odd, off);
    }
    const bool bad = odd != 0.f;
    __half s = __float2half_rn(fminf(__fdiv_rn(__fsub_rn(hi, lo), 15.f), 65504.f));
    __half z = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f));
    const float sf = __half2float(s), zf = __half2float(z);
    uint32_t word = 0;
    if (!bad && sf > 0.f) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float n = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[e], zf), sf)), 0.f), 15.f);
        word |= static_cast<uint32_t>(n) << (4 * e);
      }
    }
    if (bad) s = z = __ushort_as_half(0x7fff);
    reinterpret_cast<uint16_t*>(a.codes[which])[row * (a.G * 8) + g * a.G + j] = static_cast<uint16_t>(word);
    if (g == 0) {
      a.scales[which][row * 2 * a.G + j] = s;
      a.scales[which][row * 2 * a.G + a.G + j] = z;
    }
  }
}

// The values of tokens positions[b] + [0, T), zeros past lens[b] and where no page is.
template <typename T>
__global__ void __launch_bounds__(256) int4_read_kernel(const Int4Rows a, T* __restrict__ k_out,
                                                        T* __restrict__ v_out) {
  const int which = blockIdx.y;
  T* dst = which ? v_out : k_out;
  const int64_t words = static_cast<int64_t>(a.B) * a.H * a.T * a.G * 8;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < words; i += gridDim.x * 256ll) {
    const int wd = static_cast<int>(i % (a.G * 8)), j = wd >> 3, g = wd & 7;
    const int64_t r = i / (a.G * 8);
    const int t = static_cast<int>(r % a.T);
    const int64_t bh = r / a.T;
    const int h = static_cast<int>(bh % a.H), b = static_cast<int>(bh / a.H);
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    const int64_t row = a.lens && t >= a.lens[b] ? -1 : int4_row(a, b, h, t, g == 0);
    if (row >= 0) {
      const uint32_t word = reinterpret_cast<const uint16_t*>(a.codes[which])[row * (a.G * 8) + g * a.G + j];
      const float s = __half2float(a.scales[which][row * 2 * a.G + j]);
      const float z = __half2float(a.scales[which][row * 2 * a.G + a.G + j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(s, static_cast<float>((word >> (4 * e)) & 15u), z);
    }
    T* p = dst + i * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = from_f32<T>(x[e]);
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
inline unsigned int4_blocks(int64_t items) {
  const int64_t n = (items + 255) / 256;
  return static_cast<unsigned>(n < 148 * 64 ? n : 148 * 64);
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
  const spa::Int4Rows a = spa::int4_rows(*kv, k_scales, v_scales, batch, kv_heads, head_dim, tokens, positions, new_lens);
  const int64_t es = dtype_size(dtype);
  const int vec = (reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new) | (stride_b * es) |
                   (stride_h * es) | (stride_t * es)) % (4 * es) == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(spa::int4_blocks(static_cast<int64_t>(batch) * kv_heads * tokens * a.G * 8), 2);
  if (dtype == SPA_F32)
    spa::int4_append_kernel<float><<<grid, 256, 0, st>>>(a, static_cast<const float*>(k_new),
                                                          static_cast<const float*>(v_new), stride_b, stride_h,
                                                          stride_t, vec);
  else if (dtype == SPA_F16)
    spa::int4_append_kernel<__half><<<grid, 256, 0, st>>>(a, static_cast<const __half*>(k_new),
                                                           static_cast<const __half*>(v_new), stride_b, stride_h,
                                                           stride_t, vec);
  else
    spa::int4_append_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a, static_cast<const __nv_bfloat16*>(k_new),
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
  if (tokens == 0) return SPA_OK;
  const spa::Int4Rows a = spa::int4_rows(*kv, const_cast<void*>(k_scales), const_cast<void*>(v_scales), batch,
                                         kv_heads, head_dim, tokens, positions, lens);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(spa::int4_blocks(static_cast<int64_t>(batch) * kv_heads * tokens * a.G * 8), 2);
  if (dtype == SPA_F32)
    spa::int4_read_kernel<float><<<grid, 256, 0, st>>>(a, static_cast<float*>(k_out), static_cast<float*>(v_out));
  else if (dtype == SPA_F16)
    spa::int4_read_kernel<__half><<<grid, 256, 0, st>>>(a, static_cast<__half*>(k_out), static_cast<__half*>(v_out));
  else
    spa::int4_read_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a, static_cast<__nv_bfloat16*>(k_out),
                                                                static_cast<__nv_bfloat16*>(v_out));
  SPA_CHECK_CUDA(cudaGetLastError());
  return SPA_OK;
}
