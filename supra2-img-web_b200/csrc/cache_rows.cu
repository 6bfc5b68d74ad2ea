// Writing K/V rows into the paged 8-bit cache (quantising them) and reading them back.
//
// Write: per block and head, with x over the block's written tokens,
//   s = max(amax|x|, 2^-100) * (1/qmax), at least the old scale when the block holds earlier tokens
//   code = nearest(x * (1/s)); the held codes become nearest(code * (old / s)) when the scale grew.
// One CTA per (block, head, K or V): the block's rows are read once into registers, the maximum is
// reduced over the CTA, and the codes leave as 16-byte stores into the block's contiguous
// block_tokens * D bytes. Nothing is read twice and one launch does it all, so the kernel is bound by
// the rows' bytes in and the codes out; a block is the unit because its scale is.
// Read: value = code * scale in fp32, rounded once to the output type; one CTA per block of tokens
// and K or V, its threads in the order of the output rows.
#include "cache.cuh"

namespace supra {
namespace {

__device__ __forceinline__ uint32_t warp_max(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

// NV 16-element pieces per thread, T * D / 16 <= NV * blockDim.x.
template <typename T, int FMT, int NV, bool VEC>
__global__ void __launch_bounds__(256) cache_write_kernel(const __grid_constant__ CacheRowsLaunch L, int nblk) {
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
  uint8_t* codes = (is_v ? c.v : c.k) + (unit << c.log2t) * c.D;
  float* scale = (is_v ? c.vs : c.ks) + unit;
  const int64_t ld = is_v ? L.ldv : L.ldk;
  const T* rows = static_cast<const T*>(is_v ? L.v : L.k) + (q.row0 + t0 - first) * ld + (int64_t)h * c.D;
  const int per_row = c.D >> 4;
  const float old = lo > 0 ? *scale : 0.f;

  float x[NV][16];
  uint32_t top = 0;  // |x| as its bits: NaN above infinity above every number
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    const int slot = v / per_row;
    if (slot >= lo && slot < hi) {
      load_row<T, 16, VEC>(rows + slot * ld + (v - slot * per_row) * 16, x[i]);
#pragma unroll
      for (int k = 0; k < 16; ++k) top = max(top, __float_as_uint(x[i][k]) & 0x7fffffffu);
    }
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();  // (also: every thread has read the old scale)
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) top = max(top, part[w]);

  float s = fmaxf(__uint_as_float(top), kAmaxFloor) * (1.f / kQmax<FMT>);
  const bool bad = top >= 0x7f800000u || !(fabsf(old) <= 3.4028234e38f);  // a value or the old scale is not finite
  if (bad) s = __uint_as_float(0x7fffffffu);
  else s = fmaxf(s, old);
  const float inv = 1.f / s;
  const bool again = lo > 0 && s > old;  // false when s is NaN
  const float ratio = again ? old / s : 1.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    const int slot = v / per_row;
    uint4* at = reinterpret_cast<uint4*>(codes) + v;
    if (slot >= lo && slot < hi) {
      uint32_t u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = bad ? 0.f : mul_odd(x[i][4 * k + e], inv);
        u[k] = encode4<FMT>(y);
      }
      *at = make_uint4(u[0], u[1], u[2], u[3]);
    } else if (again && slot < lo) {
      const uint4 w = *at;
      uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float y[4];
        decode4<FMT>(u[k], y);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = mul_odd(y[e], ratio);
        u[k] = encode4<FMT>(y);
      }
      *at = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
  if (threadIdx.x == 0) *scale = s;
}

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(256) cache_read_kernel(const __grid_constant__ CacheRowsLaunch L, int nblk) {
  const CachePool& c = L.c;
  const int b = blockIdx.x / nblk;
  SeqView q;
  if (!seq_view(L.s, b, true, L.status, q) || q.n == 0) return;
  const int tokens = 1 << c.log2t;
  const int first = q.len - q.n;
  const int blk = (first >> c.log2t) + blockIdx.x % nblk;
  const int t0 = blk << c.log2t;
  if (t0 >= q.len) return;
  const int lo = max(first - t0, 0), hi = min(q.len - t0, tokens);
  const int32_t page = block_of(L.s, c, b, blk, L.status);
  if (page < 0) return;
  const bool is_v = blockIdx.y != 0;
  const int64_t unit = (int64_t)page * c.H;
  const uint8_t* codes = (is_v ? c.v : c.k) + (unit << c.log2t) * c.D;
  const float* scale = (is_v ? c.vs : c.ks) + unit;
  const int64_t ld = is_v ? L.ldv : L.ldk;
  T* rows = static_cast<T*>(is_v ? L.v : L.k) + (q.row0 + t0 - first) * ld;
  const int per_head = c.D >> 4, per_row = c.H * per_head;
  const int total = (hi - lo) * per_row;
  for (int i = threadIdx.x; i < total; i += blockDim.x) {
    const int slot = lo + i / per_row, p = i % per_row;
    const int h = p / per_head, e = (p - h * per_head) * 16;
    const uint4 w = *reinterpret_cast<const uint4*>(codes + (((int64_t)h << c.log2t) + slot) * c.D + e);
    const float s = scale[h];
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float x[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) decode4<FMT>(u[k], x + 4 * k);
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] *= s;
    store_row<T, 16, VEC>(rows + slot * ld + (int64_t)p * 16, x);
  }
}

// Blocks of tokens that n rows of one sequence can touch, at any alignment.
int touched(const CacheSeqs& s, int log2t) { return (int)((s.max_rows + 2ll * (1 << log2t) - 2) >> log2t); }

template <typename T, int FMT, bool VEC>
cudaError_t write_as(const CacheRowsLaunch& L, cudaStream_t s) {
  const int nblk = touched(L.s, L.c.log2t);
  const int pieces = (L.c.D >> 4) << L.c.log2t;
  const dim3 grid((unsigned)(L.s.B * nblk), (unsigned)L.c.H, 2);
  if (pieces <= 256) {
    cache_write_kernel<T, FMT, 1, VEC><<<grid, (pieces + 31) / 32 * 32, 0, s>>>(L, nblk);
  } else if (pieces <= 512) {
    cache_write_kernel<T, FMT, 2, VEC><<<grid, 256, 0, s>>>(L, nblk);
  } else {
    cache_write_kernel<T, FMT, 4, VEC><<<grid, 256, 0, s>>>(L, nblk);
  }
  return cudaGetLastError();
}
template <typename T, int FMT, bool VEC>
cudaError_t read_as(const CacheRowsLaunch& L, cudaStream_t s) {
  const int nblk = touched(L.s, L.c.log2t);
  cache_read_kernel<T, FMT, VEC><<<dim3((unsigned)(L.s.B * nblk), 2), 256, 0, s>>>(L, nblk);
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
