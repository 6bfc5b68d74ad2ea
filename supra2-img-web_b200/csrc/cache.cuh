// Device helpers shared by the kernels of the paged 8-bit K/V cache and the query/key norm: element
// types, the cache's codes, and the bounds of a call's sequences.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace supra {

// ---- element types ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two values as one 32-bit word of a 16-bit type, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// N consecutive elements (N * sizeof(T) a multiple of 16). VEC: p is 16-byte aligned.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_row(const T* p, float (&x)[N]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32<T>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + i);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack2<T>(u[k]);
        x[i + 2 * k] = f.x, x[i + 2 * k + 1] = f.y;
      }
    }
  }
}
template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_row(T* p, const float (&x)[N]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_f32<T>(x[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      uint4 v;
      v.x = pack2<T>(x[i], x[i + 1]), v.y = pack2<T>(x[i + 2], x[i + 3]);
      v.z = pack2<T>(x[i + 4], x[i + 5]), v.w = pack2<T>(x[i + 6], x[i + 7]);
      *reinterpret_cast<uint4*>(p + i) = v;
    }
  }
}

// ---- the cache's codes -----------------------------------------------------------------------
template <int FMT>
constexpr float kQmax = FMT == kCacheInt8 ? 127.f : 448.f;
constexpr float kAmaxFloor = 7.8886090522101181e-31f;  // 2^-100: keeps 1 / scale finite

// Four codes of one 32-bit word as fp32 values (before the scale).
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t u, float* x) {
  if constexpr (FMT == kCacheInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(u >> (8 * i));
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((u >> (16 * i)) & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

// x * f and y * f rounded to odd: truncated, with the last bit set when anything was cut off. Rounding
// such a value to fewer bits gives what rounding the exact product would.
__device__ __forceinline__ float2 mul_odd2(float x, float y, float f) {
  const float2 a = make_float2(x, y), b = make_float2(f, f);
  float2 p = __fmul2_rz(a, b);
  const float2 r = __ffma2_rn(a, b, make_float2(-p.x, -p.y));  // what was cut off, exact
  p.x = __uint_as_float(__float_as_uint(p.x) | (__float_as_uint(r.x) != 0u));
  p.y = __uint_as_float(__float_as_uint(p.y) | (__float_as_uint(r.y) != 0u));
  return p;
}

// The codes nearest to the products of four values with f, ties to even, as one 32-bit word; the
// products are at most kQmax (up to one fp32 rounding above it). The exact product is rounded once, to
// the code.
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float f) {
  if constexpr (FMT == kCacheInt8) {
    // the fused sum with 1.5 * 2^23 rounds to a whole number whose two's complement is in the low bits
    const float2 m = make_float2(12582912.f, 12582912.f), g = make_float2(f, f);
    const float2 x = __ffma2_rn(make_float2(a, b), g, m), y = __ffma2_rn(make_float2(c, d), g, m);
    return __byte_perm(__byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x0040),
                       __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040), 0x5410);
  } else {
    // A truncated product rounds like the exact one unless it lies on the border between two codes, and then
    // its 19 low bits are 0: only those few are formed with what was cut off.
    const float2 g = make_float2(f, f);
    float2 x = __fmul2_rz(make_float2(a, b), g), y = __fmul2_rz(make_float2(c, d), g);
    const uint32_t m = 0x7ffffu;
    const uint32_t low = min(min(__float_as_uint(x.x) & m, __float_as_uint(x.y) & m),
                             min(__float_as_uint(y.x) & m, __float_as_uint(y.y) & m));
    if (low == 0u) {
      x = mul_odd2(a, b, f);
      y = mul_odd2(c, d, f);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
}

// ---- waits -----------------------------------------------------------------------------------
// Waits for the phase with the given parity, for about two seconds at most; gives up at once when
// *abort is set (abort may be null). The limit is counted in SM clocks and looked at only every 64
// tries: a read of the global timer takes about 1500 cycles, more than most of these waits.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
constexpr long long kWaitLimitClocks = 4000000000ll;
__device__ __forceinline__ bool mbar_wait_clocked(uint64_t* bar, uint32_t parity, volatile int32_t* abort) {
  long long t0 = 0;
  for (uint32_t it = 0;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 63u) {
      if (abort && *abort) return false;
      const long long t = clock64();
      if (t0 == 0) t0 = t;
      else if (t - t0 > kWaitLimitClocks) return false;
    }
  }
}

// ---- a launch and the one that joins its parts ---------------------------------------------------
// The join's CTAs may be placed once every CTA of the parts' launch has said so or ended, and wait until that
// launch has ended and its writes can be seen.
__device__ __forceinline__ void join_may_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void parts_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- sequences ---------------------------------------------------------------------------------
struct SeqView {
  int64_t row0;  // first row of the operands
  int32_t n;     // rows
  int32_t len;   // tokens, the rows' own included
};

// Sequence b of a call, checked against the call's bounds; false (reported once) when outside.
// rows_in_seq: the rows stand for tokens of the cache, so there are at most len.
__device__ __forceinline__ bool seq_view(const CacheSeqs& s, int b, bool rows_in_seq, int32_t* status, SeqView& v) {
  int64_t r0 = (int64_t)b * s.max_rows, r1 = r0 + s.max_rows;
  if (s.row_start) {
    r0 = s.row_start[b];
    r1 = s.row_start[b + 1];
  }
  v.row0 = r0;
  v.n = (int32_t)(r1 - r0);
  v.len = s.lengths[b];
  const bool ok = r0 >= 0 && r1 >= r0 && r1 <= s.rows && r1 - r0 <= s.max_rows && v.len >= 0 && v.len <= s.max_len &&
                  (!rows_in_seq || v.n <= v.len);
  if (!ok && threadIdx.x == 0) report_error(status, DEV_BAD_SEQ, 0, b);
  return ok;
}

// Block number of block j of sequence b, or -1 (reported) when it is outside the cache.
__device__ __forceinline__ int32_t block_of(const CacheSeqs& s, const CachePool& c, int b, int j, int32_t* status) {
  const int32_t p = s.table[(int64_t)b * s.ld_table + j];
  if (p >= 0 && p < c.blocks) return p;
  report_error(status, DEV_BAD_BLOCK, 0, p);
  return -1;
}

// The attention kernels look blocks up ahead of their use: the table's entry j of sequence b, whatever it is, but never
// kPastEnd, which they put in the place of entries after the last token (an entry with that value becomes the next
// one, which is no block either).
constexpr int32_t kPastEnd = INT32_MIN;
__device__ __forceinline__ int32_t page_of(const CacheSeqs& s, int b, int j) {
  return max(s.table[(int64_t)b * s.ld_table + j], kPastEnd + 1);
}

}  // namespace supra
