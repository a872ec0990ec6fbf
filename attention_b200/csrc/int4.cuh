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

// Both kernels: a warp has one (sequence, kv head) and, of its rows, a stretch of kInt4Stretch;
// eight lanes hold a group, four values each, so a warp covers 4 groups at once (a whole row of
// head_dim 128, two rows of 64).  Grid (B * Hkv, K or V, stretches): no index is divided.
// Bound by HBM (a row's 2 D bytes against its 5/8 D at 16 bits), reached by kInt4Flight steps'
// loads in flight a lane.
constexpr int kInt4Warps = 4, kInt4Stretch = 32, kInt4Flight = 4;

struct Int4Lane {
  int g, j0;  // the lane's place in its eight, and which eight of the warp it is in
  __device__ __forceinline__ Int4Lane() : g(threadIdx.x & 7), j0((threadIdx.x & 31) >> 3) {}
};

template <typename T>
__global__ void __launch_bounds__(kInt4Warps * 32) int4_append_kernel(const Int4Rows a, const T* __restrict__ k_new,
                                                                      const T* __restrict__ v_new, int64_t sb,
                                                                      int64_t sh, int64_t st, int vec) {
  const Int4Lane ln;
  const int which = blockIdx.y, warp = threadIdx.x >> 5, b = blockIdx.x / a.H, h = blockIdx.x - b * a.H;
  const int len = a.lens ? min(a.lens[b], a.T) : a.T;
  const int t0 = (blockIdx.z * kInt4Warps + warp) * kInt4Stretch, t1 = min(t0 + kInt4Stretch, len);
  if (t0 >= t1) return;
  const T* src = (which ? v_new : k_new) + b * sb + h * sh;
  uint16_t* codes = reinterpret_cast<uint16_t*>(which ? a.codes[1] : a.codes[0]);
  __half* scales = which ? a.scales[1] : a.scales[0];
  // the stretch's rows, one a lane
  const int64_t my_row = t0 + (threadIdx.x & 31) < t1 ? int4_row(a, b, h, t0 + (threadIdx.x & 31), true) : -1;
  // steps: groups of the stretch in order, four (a lane's every fourth) at a time
  const int steps = ((t1 - t0) * a.G + 3) >> 2;
  int t = t0, j = ln.j0;  // this lane's row and group
  while (j >= a.G) j -= a.G, ++t;
  for (int s0 = 0; s0 < steps; s0 += kInt4Flight) {
    float x[kInt4Flight][4];
    int tt[kInt4Flight], jj[kInt4Flight];
#pragma unroll
    for (int i = 0; i < kInt4Flight; ++i) {
      tt[i] = t;
      jj[i] = j;
      if (t < t1)
        load4<T>(src + t * st + j * kInt4Group + ln.g * 4, vec, x[i]);
      else
        x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
      j += 4;
      while (j >= a.G) j -= a.G, ++t;
    }
#pragma unroll
    for (int i = 0; i < kInt4Flight; ++i) {
      const int64_t row = __shfl_sync(0xffffffffu, my_row, tt[i] - t0 < 31 ? tt[i] - t0 : 31);
      float lo = fminf(fminf(x[i][0], x[i][1]), fminf(x[i][2], x[i][3]));
      float hi = fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3]));
      // x - x is NaN for a NaN or an infinity, 0 otherwise
      float odd = (x[i][0] - x[i][0]) + (x[i][1] - x[i][1]) + (x[i][2] - x[i][2]) + (x[i][3] - x[i][3]);
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        odd += __shfl_xor_sync(0xffffffffu, odd, off);
      }
      const bool bad = odd != 0.f;
      __half s = __float2half_rn(fminf(__fdiv_rn(__fsub_rn(hi, lo), 15.f), 65504.f));
      __half z = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f));
      const float sf = __half2float(s), zf = __half2float(z);
      uint32_t word = 0;
      if (!bad && sf > 0.f) {
        // rint((x - z) / s): the quotient by a reciprocal is within 2^-21 of it (three roundings,
        // quotients of this range below 2^4 + 2), so only near a half the division itself decides
        const float inv = __frcp_rn(sf);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = __fsub_rn(x[i][e], zf);
          float n = d * inv;
          const float frac = n - floorf(n);
          if (fabsf(frac - 0.5f) < 1e-4f) n = __fdiv_rn(d, sf);
          word |= static_cast<uint32_t>(fminf(fmaxf(rintf(n), 0.f), 15.f)) << (4 * e);
        }
      }
      if (bad) s = z = __ushort_as_half(0x7fff);
      if (tt[i] < t1 && row >= 0) {
        codes[row * (a.G * 8) + ln.g * a.G + jj[i]] = static_cast<uint16_t>(word);
        __half* sc = scales + row * 2 * a.G + jj[i];
        if (ln.g == 0) sc[0] = s;
        if (ln.g == 1) sc[a.G] = z;
      }
    }
  }
}

// The values of tokens positions[b] + [0, T), zeros past lens[b] and where no page is.
template <typename T>
__global__ void __launch_bounds__(kInt4Warps * 32) int4_read_kernel(const Int4Rows a, T* __restrict__ k_out,
                                                                    T* __restrict__ v_out) {
  const Int4Lane ln;
  const int which = blockIdx.y, warp = threadIdx.x >> 5, b = blockIdx.x / a.H, h = blockIdx.x - b * a.H;
  const int len = a.lens ? min(a.lens[b], a.T) : a.T;
  const int t0 = (blockIdx.z * kInt4Warps + warp) * kInt4Stretch, t1 = min(t0 + kInt4Stretch, a.T);
  if (t0 >= t1) return;
  const uint16_t* codes = reinterpret_cast<const uint16_t*>(which ? a.codes[1] : a.codes[0]);
  const __half* scales = which ? a.scales[1] : a.scales[0];
  T* dst = (which ? v_out : k_out) + static_cast<int64_t>(blockIdx.x) * a.T * (a.G * kInt4Group);
  const int64_t my_row = t0 + (threadIdx.x & 31) < min(t1, len) ? int4_row(a, b, h, t0 + (threadIdx.x & 31), true) : -1;
  const int steps = ((t1 - t0) * a.G + 3) >> 2;
  int t = t0, j = ln.j0;
  while (j >= a.G) j -= a.G, ++t;
  for (int s0 = 0; s0 < steps; s0 += kInt4Flight) {
    uint32_t word[kInt4Flight];
    float s[kInt4Flight], z[kInt4Flight];
    int tt[kInt4Flight], jj[kInt4Flight];
#pragma unroll
    for (int i = 0; i < kInt4Flight; ++i) {
      tt[i] = t;
      jj[i] = j;
      const int64_t row = __shfl_sync(0xffffffffu, my_row, t - t0 < 31 ? t - t0 : 31);
      word[i] = 0;
      s[i] = z[i] = 0.f;
      if (t < t1 && row >= 0) {
        word[i] = codes[row * (a.G * 8) + ln.g * a.G + j];
        const __half* sc = scales + row * 2 * a.G + j;
        s[i] = __half2float(sc[0]);
        z[i] = __half2float(sc[a.G]);
      }
      j += 4;
      while (j >= a.G) j -= a.G, ++t;
    }
#pragma unroll
    for (int i = 0; i < kInt4Flight; ++i) {
      if (tt[i] >= t1) continue;
      T x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = from_f32<T>(fmaf(s[i], static_cast<float>((word[i] >> (4 * e)) & 15u), z[i]));
      T* p = dst + static_cast<int64_t>(tt[i]) * (a.G * kInt4Group) + jj[i] * kInt4Group + ln.g * 4;
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
      else
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(x);
    }
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
                   (stride_h * es) | (stride_t * es)) % (4 * es) == 0;
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
