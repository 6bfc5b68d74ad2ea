// Writing K/V rows into the paged 8-bit cache (quantising them) and reading them back.
//
// Write: per block and head, with x over the block's written tokens,
//   s = max(amax|x|, 2^-100) * (1/qmax), at least the old scale when the block holds earlier tokens
//   code = nearest(x * (1/s)); the held codes become nearest(code * (old / s)) when the scale grew.
// One CTA per (block, head, K or V): the block's rows are read once into registers, 16 bytes a load and
// neighbouring lanes on neighbouring pieces, the maximum is reduced over the CTA, and the codes leave
// into the block's contiguous block_tokens * D bytes. Nothing is read twice and one launch does it all,
// so the kernel is bound by the rows' bytes in and the codes out; a block is the unit because its scale is.
// Read: value = code * scale in fp32, rounded once to the output type; one CTA per 16 slots of a
// block and K or V, a few rows per warp at a time, each lane storing 16 bytes.
// Measured, 20000 rows of 8 heads of 128: write bf16 to E4M3, blocks of 64: 29 us (4.2 TB/s; 67 % of the issue slots:
// the codes' arithmetic and the bytes bound it alike); read back to bf16 24 us (5.1 TB/s), to fp32 39 us (5.3 TB/s),
// 45000 rows to bf16 43 us (6.3 TB/s): bytes. One token each of 64 sequences: 6 us, the launch.
#include <algorithm>

#include "cache.cuh"

namespace supra {
namespace {

__device__ __forceinline__ uint32_t warp_max(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

// The codes nearest to V channels (4 or 8) times f, as one or two words.
template <int FMT, int V>
__device__ __forceinline__ void encode_row(const float (&x)[V], float f, uint32_t (&u)[V / 4]) {
#pragma unroll
  for (int k = 0; k < V / 4; ++k) u[k] = encode4<FMT>(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3], f);
}
// The largest magnitude among the pieces, as fp32 bits: NaN above infinity above every number.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <typename T, int NV>
__device__ __forceinline__ uint32_t largest_bits(const uint4 (&raw)[NV]) {
  if constexpr (sizeof(T) == 4) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      m = max3_nan(m, fabsf(__uint_as_float(raw[i].x)), fabsf(__uint_as_float(raw[i].y)));
      m = max3_nan(m, fabsf(__uint_as_float(raw[i].z)), fabsf(__uint_as_float(raw[i].w)));
    }
    return __float_as_uint(m);
  } else {  // two at a time: magnitudes of 16-bit floats are in the order of their bits
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      m = __vmaxu2(m, raw[i].x & 0x7fff7fffu);
      m = __vmaxu2(m, raw[i].y & 0x7fff7fffu);
      m = __vmaxu2(m, raw[i].z & 0x7fff7fffu);
      m = __vmaxu2(m, raw[i].w & 0x7fff7fffu);
    }
    const float2 f = unpack2<T>(__vmaxu2(m, m >> 16));
    return __float_as_uint(f.x);
  }
}
template <int N>
__device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t (&u)[N]) {
  if constexpr (N == 1) {
    u[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    u[0] = w.x, u[1] = w.y;
  }
}
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t (&u)[N]) {
  if constexpr (N == 1) *reinterpret_cast<uint32_t*>(p) = u[0];
  else *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
}

// Threads take pieces of 16 bytes of a row (V channels): thread t < rows * per_row has piece t % per_row of slots
// t / per_row + i * rows, i < NV.
template <typename T, int FMT, int NV, bool VEC>
__global__ void __launch_bounds__(256) cache_write_kernel(const __grid_constant__ CacheRowsLaunch L, int nblk, int rows) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ uint32_t part[8];
  const CachePool& c = L.c;
  const int b = blockIdx.x / nblk, h = blockIdx.y;
  SeqView q;
  if (!seq_view(L.s, b, true, L.status, q) || q.n == 0) return;
  const int tokens = 1 << c.log2t;
  const int first = q.len - q.n;
  const int blk = (first >> c.log2t) + blockIdx.x % nblk;
  const int t0 = blk << c.log2t;
  if (t0 >= q.len) return;
  const int lo = max(first - t0, 0), hi = min(q.len - t0, tokens);  // written slots
  const int32_t page = block_of(L.s, c, b, blk, L.status);
  if (page < 0) return;
  const bool is_v = blockIdx.z != 0;
  const int64_t unit = (int64_t)page * c.H + h;
  const int per_row = c.D / V;
  const int slot0 = threadIdx.x / per_row, e = (threadIdx.x - slot0 * per_row) * V;
  const int end = slot0 < rows ? hi : 0;  // threads past the last whole row of pieces have nothing
  uint8_t* codes = (is_v ? c.v : c.k) + (unit << c.log2t) * c.D + e;
  float* scale = (is_v ? c.vs : c.ks) + unit;
  const int64_t ld = is_v ? L.ldv : L.ldk;
  const T* src = static_cast<const T*>(is_v ? L.v : L.k) + (q.row0 + t0 - first) * ld + (int64_t)h * c.D + e;
  const float old = lo > 0 ? *scale : 0.f;

  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int slot = slot0 + i * rows;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (slot >= lo && slot < end) {
      if constexpr (VEC) {
        raw[i] = *reinterpret_cast<const uint4*>(src + slot * ld);
      } else {
        T y[V];
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = src[slot * ld + k];
        memcpy(&raw[i], y, 16);
      }
    }
  }
  uint32_t top = warp_max(largest_bits<T, NV>(raw));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();  // (also: every thread has read the old scale)
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) top = max(top, part[w]);

  float s = fmaxf(__uint_as_float(top), kAmaxFloor) * (1.f / kQmax<FMT>);
  const bool bad = top >= 0x7f800000u || !(fabsf(old) <= 3.4028234e38f);  // a value or the old scale is not finite
  if (bad) s = __uint_as_float(0x7fffffffu);
  else s = fmaxf(s, old);
  const float inv = 1.f / s;
  const bool again = lo > 0 && s > old;  // false when s is NaN
  // (a caller's own scale may be negative and larger in size than the new one: codes up to `reach` have a product that
  // INT8 holds, the others get its largest; E4M3's conversion saturates by itself)
  const float ratio = again ? fmaxf(old / s, -3.4028234e38f) : 1.f, reach = 127.f / fabsf(ratio);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int slot = slot0 + i * rows;
    if (slot >= end) break;
    uint8_t* at = codes + slot * c.D;
    uint32_t u[V / 4] = {};
    float x[V];
    if (slot >= lo) {
      load_row<T, V, true>(reinterpret_cast<const T*>(&raw[i]), x);
      if (!bad) encode_row<FMT, V>(x, inv, u);
      store_codes(at, u);
    } else if (again) {
      load_codes(at, u);
#pragma unroll
      for (int k = 0; k < V / 4; ++k) decode4<FMT>(u[k], x + 4 * k);
      if constexpr (FMT == kCacheInt8) {
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = fminf(fmaxf(x[k], -reach), reach);
      }
      encode_row<FMT, V>(x, ratio, u);
      store_codes(at, u);
    }
  }
  if (threadIdx.x == 0) *scale = s;
}

constexpr int kReadRows = 16;  // slots of a CTA: small ones, so that the last wave is short
template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(128) cache_read_kernel(const __grid_constant__ CacheRowsLaunch L, int nblk) {
  constexpr int V = 16 / (int)sizeof(T);
  constexpr int UN = 4, RN = V == 4 ? 4 : 2;  // pieces of a row, and rows, that a lane has under way
  const CachePool& c = L.c;
  const int b = blockIdx.x / nblk;
  SeqView q;
  if (!seq_view(L.s, b, true, L.status, q) || q.n == 0) return;
  const int tokens = 1 << c.log2t;
  const int first = q.len - q.n;
  const int blk = (first >> c.log2t) + blockIdx.x % nblk;
  const int t0 = blk << c.log2t;
  if (t0 >= q.len) return;
  const int part = blockIdx.z * kReadRows;
  const int lo = max(first - t0, part), hi = min(min(q.len - t0, tokens), part + kReadRows);
  if (lo >= hi) return;
  const int32_t page = block_of(L.s, c, b, blk, L.status);
  if (page < 0) return;
  const bool is_v = blockIdx.y != 0;
  const int64_t unit = (int64_t)page * c.H;
  const uint8_t* codes = (is_v ? c.v : c.k) + (unit << c.log2t) * c.D;
  const float* scale = (is_v ? c.vs : c.ks) + unit;
  const int64_t ld = is_v ? L.ldv : L.ldk;
  T* dst = static_cast<T*>(is_v ? L.v : L.k) + (q.row0 + t0 - first) * ld;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_head = c.D / V, per_row = c.H * per_head;
  const int head_bytes = c.D << c.log2t;
  // a lane's pieces are the same in every row: their heads are worked out once per UN of them
  for (int p0 = lane; p0 < per_row; p0 += 32 * UN) {
    const uint8_t* from[UN];
    float s[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int p = min(p0 + 32 * i, per_row - 1), h = p / per_head;
      from[i] = codes + (int64_t)h * head_bytes + (p - h * per_head) * V;
      s[i] = scale[h];
    }
    for (int slot = lo + warp; slot < hi; slot += RN * warps) {
      uint32_t u[RN][UN][V / 4];
#pragma unroll
      for (int r = 0; r < RN; ++r)
#pragma unroll
        for (int i = 0; i < UN; ++i) load_codes(from[i] + min(slot + r * warps, hi - 1) * c.D, u[r][i]);
#pragma unroll
      for (int r = 0; r < RN; ++r) {
        if (slot + r * warps >= hi) break;
#pragma unroll
        for (int i = 0; i < UN; ++i) {
          if (p0 + 32 * i >= per_row) break;
          float x[V];
#pragma unroll
          for (int k = 0; k < V / 4; ++k) decode4<FMT>(u[r][i][k], x + 4 * k);
#pragma unroll
          for (int k = 0; k < V; ++k) x[k] *= s[i];
          store_row<T, V, VEC>(dst + (slot + r * warps) * ld + (int64_t)(p0 + 32 * i) * V, x);
        }
      }
    }
  }
}

// Blocks of tokens that n rows of one sequence can touch, at any alignment.
int touched(const CacheSeqs& s, int log2t) { return (int)((s.max_rows + 2ll * (1 << log2t) - 2) >> log2t); }

template <typename T, int FMT, bool VEC>
cudaError_t write_as(const CacheRowsLaunch& L, cudaStream_t s) {
  const int nblk = touched(L.s, L.c.log2t);
  // 128 threads: 64 where each would hold one piece (what a warp does besides its pieces is worth four of them),
  // 256 where each would hold more than 8; whole rows of pieces, the last warp filled up. 20000 rows, us with 64 /
  // 128 / 256 threads: blocks of 16 x 64 bf16 (128 pieces) 27 / 35 / 35, 128 x 64 bf16 (1024) 23 / 21 / 23, 64 x 128
  // bf16 (1024) 41 / 33 / 39, 64 x 128 fp32 (2048) - / 53 / 47.
  constexpr int V = 16 / (int)sizeof(T);
  const int per_row = L.c.D / V, tokens = 1 << L.c.log2t;
  int rows = std::min(tokens, (tokens * per_row <= 128 ? 64 : 128) / per_row);
  if ((tokens + rows - 1) / rows > 8) rows = std::min(tokens, 256 / per_row);
  const int nv = (tokens + rows - 1) / rows;
  const int threads = (rows * per_row + 31) / 32 * 32;
  const dim3 grid((unsigned)(L.s.B * nblk), (unsigned)L.c.H, 2);
  if (nv <= 1) cache_write_kernel<T, FMT, 1, VEC><<<grid, threads, 0, s>>>(L, nblk, rows);
  else if (nv <= 2) cache_write_kernel<T, FMT, 2, VEC><<<grid, threads, 0, s>>>(L, nblk, rows);
  else if (nv <= 4) cache_write_kernel<T, FMT, 4, VEC><<<grid, threads, 0, s>>>(L, nblk, rows);
  else if (nv <= 8) cache_write_kernel<T, FMT, 8, VEC><<<grid, threads, 0, s>>>(L, nblk, rows);
  else cache_write_kernel<T, FMT, 18, VEC><<<grid, threads, 0, s>>>(L, nblk, rows);  // (fp32: up to 18)
  return cudaGetLastError();
}
template <typename T, int FMT, bool VEC>
cudaError_t read_as(const CacheRowsLaunch& L, cudaStream_t s) {
  const int nblk = touched(L.s, L.c.log2t);
  cache_read_kernel<T, FMT, VEC><<<dim3((unsigned)(L.s.B * nblk), 2, (1u << L.c.log2t) / kReadRows), 128, 0, s>>>(L, nblk);
  return cudaGetLastError();
}

template <typename T>
cudaError_t rows_of(bool write, const CacheRowsLaunch& L, int format, bool vec, cudaStream_t s) {
  if (write) {
    if (format == kCacheInt8) return vec ? write_as<T, kCacheInt8, true>(L, s) : write_as<T, kCacheInt8, false>(L, s);
    return vec ? write_as<T, kCacheE4m3, true>(L, s) : write_as<T, kCacheE4m3, false>(L, s);
  }
  if (format == kCacheInt8) return vec ? read_as<T, kCacheInt8, true>(L, s) : read_as<T, kCacheInt8, false>(L, s);
  return vec ? read_as<T, kCacheE4m3, true>(L, s) : read_as<T, kCacheE4m3, false>(L, s);
}
cudaError_t rows_any(bool write, const CacheRowsLaunch& L, int type, int format, bool vec, cudaStream_t s) {
  if (type == kTypeF32) return rows_of<float>(write, L, format, vec, s);
  if (type == kTypeF16) return rows_of<__half>(write, L, format, vec, s);
  return rows_of<__nv_bfloat16>(write, L, format, vec, s);
}

}  // namespace

cudaError_t launch_cache_write(const CacheRowsLaunch& L, int type, int format, bool vec, cudaStream_t s) {
  return rows_any(true, L, type, format, vec, s);
}
cudaError_t launch_cache_read(const CacheRowsLaunch& L, int type, int format, bool vec, cudaStream_t s) {
  return rows_any(false, L, type, format, vec, s);
}

}  // namespace supra
