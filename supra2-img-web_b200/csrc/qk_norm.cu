// RMS norm of every query and key head with the position rotation in the same pass.
//   n = x / sqrt(mean(x^2) + eps) * w;  (y_a, y_b) = (n_a cos - n_b sin, n_b cos + n_a sin)
// Bound by the rows' bytes in and out. The vector form gives a head to a group of lanes, each with
// one 16-byte piece: the sum of squares and the partner channels of the rotation go by shuffles, so
// every element is read once, and a warp walks over the heads of one row with the weights folded into the
// row's cosines and sines in registers (1 / sqrt is rsqrtf, 2 ulp; a correctly rounded root and division a
// head made the kernel issue-bound). Pieces stay as they were read until their turn comes, and products
// are formed two at a time: fewer instructions, and registers for more warps (the bf16 case below took 108 us
// with channels unpacked at once and weights apart). Every lane stores only pieces that it loaded itself,
// so in-place calls need no ordering. The scalar form (sizes and alignments that do not split into 16-byte
// pieces) gives a head to a warp. Rotations that end inside a piece or pair channels of unlike places in
// theirs stay in the vector form, partners through shared memory (16384 rows of 9 + 9 heads of 64, 50 channels
// turned, bf16: 41 us, neighbours 31; scalar form 119 and 127).
// Measured: 16384 rows of 9 + 9 heads of 64, fp32: 30 us, 5.0 TB/s (scalar form 121); 16384 rows of 32 + 8 heads
// of 128, bf16: 68 us, 5.0 TB/s (scalar form 338); 61 rows: 8 us, the launch.
#include "cache.cuh"

namespace supra {
namespace {

// The row of the turns table for `row`, or null (reported) when its position is outside.
__device__ __forceinline__ const float* turns_of(const QkNormLaunch& L, int64_t row, int lane, bool* ok) {
  *ok = true;
  if (L.rot == 0) return nullptr;
  const int64_t p = L.positions ? (int64_t)L.positions[row] : row;
  if (p < 0 || p >= L.n_turns) {
    if (lane == 0) report_error(L.status, DEV_BAD_POSITION, 0, (int32_t)row);
    *ok = false;
    return nullptr;
  }
  return L.turns + p * L.rot;
}

// LPH lanes per head (a power of two), V elements per lane; `wpr` warps share a row's heads. ROT: 0 no
// rotation, 1 pairs half a rotation apart, 2 neighbours, 3 pairs half a rotation apart where that is not whole
// pieces (or the table is not aligned): partners by their channels, through shared memory.
template <typename T, int LPH, int ROT>
__global__ void __launch_bounds__(128) qk_norm_vec(const __grid_constant__ QkNormLaunch L, int wpr) {
  constexpr int V = 16 / (int)sizeof(T), V2 = V / 2;
  constexpr int UNROLL = sizeof(T) == 4 ? 5 : 4;  // (18 heads of 64 fp32: two rounds, not three)
  const int lane = threadIdx.x & 31, g = lane / LPH, l = lane % LPH;
  const uint32_t w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int row = (int)(w / (uint32_t)wpr), part = (int)(w - (uint32_t)row * wpr);
  if (row >= L.M) return;
  bool ok;
  const float* turns = turns_of(L, row, lane, &ok);
  if (!ok) return;
  const int e0 = l * V;                 // the lane's first channel
  const bool on = e0 < L.D;             // lanes past the head only take part in the shuffles
  const int half = L.rot >> 1;
  const bool turn = ROT != 0 && on && e0 < L.rot;  // (with 2 and 3 perhaps only the first channels)
  __shared__ uint4 own[ROT == 3 ? 4 : 1][32];
  auto partner = [&](int e) { return e < half ? e + half : e - half; };  // of channel e < rot
  // Pairs half a rotation apart: the partner piece is in the lane `peer`.
  const bool second = ROT == 1 && e0 >= half;
  const int pe = ROT == 1 && turn ? (second ? e0 - half : e0 + half) : e0;  // the partner piece's first channel
  const int peer = g * LPH + pe / V;
  // y_i = r (x_i a_i + partner_i s_i): the weights folded into the row's cosines and sines, for the queries or
  // the keys, whichever the lane's head is
  float2 a[V2], s[V2];
  auto fold = [&](const float* wt) {
    float co[V], si[V], wi[V], wp[V];
#pragma unroll
    for (int i = 0; i < V; ++i) co[i] = wi[i] = wp[i] = 1.f, si[i] = 0.f;
    if (on && wt) load_row<float, V, true>(wt + e0, wi);
    if (turn) {
      if constexpr (ROT == 1) {
        if (wt) load_row<float, V, true>(wt + pe, wp);
        load_row<float, V, true>(turns + (second ? pe : e0), co);
        load_row<float, V, true>(turns + half + (second ? pe : e0), si);
#pragma unroll
        for (int i = 0; i < V; ++i) si[i] = second ? si[i] : -si[i];
      } else if constexpr (ROT == 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (e0 + i >= L.rot) break;
          co[i] = turns[(e0 + i) >> 1];
          si[i] = (i & 1) ? turns[half + ((e0 + i) >> 1)] : -turns[half + ((e0 + i) >> 1)];
          wp[i] = wi[i ^ 1];
        }
      } else if constexpr (ROT == 3) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = e0 + i;
          if (e >= L.rot) break;
          const bool first = e < half;
          co[i] = turns[first ? e : e - half];
          si[i] = first ? -turns[half + e] : turns[e];
          if (wt) wp[i] = wt[partner(e)];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V2; ++i) {
      a[i] = make_float2(co[2 * i] * wi[2 * i], co[2 * i + 1] * wi[2 * i + 1]);
      s[i] = make_float2(si[2 * i] * wp[2 * i], si[2 * i + 1] * wp[2 * i + 1]);
    }
  };
  const int Hq = L.q.H, heads = Hq + L.k.H;
  const int step = wpr * (32 / LPH);
  const float inv_d = 1.f / (float)L.D;
  // the row's heads, the keys' addressed as if they followed the queries
  const T* xq = static_cast<const T*>(L.q.x) + (int64_t)row * L.q.ldx + e0;
  const T* xk = static_cast<const T*>(L.k.x) + (int64_t)row * L.k.ldx + e0 - Hq * L.D;
  T* yq = static_cast<T*>(L.q.y) + (int64_t)row * L.q.ldy + e0;
  T* yk = static_cast<T*>(L.k.y) + (int64_t)row * L.k.ldy + e0 - Hq * L.D;
  int have = -1;  // whose weights are folded in: 0 the queries', 1 the keys'
  // (whole warps stay in the loop: the shuffles need every lane)
  for (int base = part * (32 / LPH); base < heads; base += step * UNROLL) {
    uint4 raw[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = base + u * step + g;
      raw[u] = make_uint4(0, 0, 0, 0);
      if (on && h < heads) raw[u] = *reinterpret_cast<const uint4*>((h < Hq ? xq : xk) + h * L.D);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (base + u * step >= heads) break;  // uniform over the warp
      const int h = base + u * step + g;
      const int key = h >= Hq;
      if (key != have) {
        if (have < 0 || L.q.w != L.k.w) fold(key ? L.k.w : L.q.w);
        have = key;
      }
      auto pairs = [](const uint4& r, float2 (&x)[V2]) {
        const uint32_t u4[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < V2; ++i) {
          if constexpr (V == 4) x[i] = make_float2(__uint_as_float(u4[2 * i]), __uint_as_float(u4[2 * i + 1]));
          else x[i] = unpack2<T>(u4[i]);
        }
      };
      float2 x[V2], o[V2];
      pairs(raw[u], x);
      float r = 1.f;
      if (L.norm) {
        float2 ss = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < V2; ++i) ss = __ffma2_rn(x[i], x[i], ss);
        float sum = ss.x + ss.y;
#pragma unroll
        for (int d = LPH / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        r = rsqrtf(fmaf(sum, inv_d, L.eps));
      }
      // partners as they were read (a channel that does not turn has none: 0, lest it meet an infinity)
      if constexpr (ROT == 1) {
        uint4 p;
        p.x = __shfl_sync(0xffffffffu, raw[u].x, peer), p.y = __shfl_sync(0xffffffffu, raw[u].y, peer);
        p.z = __shfl_sync(0xffffffffu, raw[u].z, peer), p.w = __shfl_sync(0xffffffffu, raw[u].w, peer);
        if (!turn) p = make_uint4(0, 0, 0, 0);
        pairs(p, o);
      } else if constexpr (ROT == 2) {
#pragma unroll
        for (int i = 0; i < V2; ++i) o[i] = on && e0 + 2 * i < L.rot ? make_float2(x[i].y, x[i].x) : make_float2(0.f, 0.f);
      } else if constexpr (ROT == 3) {
        uint4* mine = own[threadIdx.x >> 5];
        mine[lane] = raw[u];
        __syncwarp();
        const T* head = reinterpret_cast<const T*>(mine + g * LPH);
#pragma unroll
        for (int i = 0; i < V2; ++i) {
          const int e = e0 + 2 * i;
          o[i].x = on && e < L.rot ? to_f32<T>(head[partner(e)]) : 0.f;
          o[i].y = on && e + 1 < L.rot ? to_f32<T>(head[partner(e + 1)]) : 0.f;
        }
        __syncwarp();  // (before the next head's pieces)
      }
      float y[V];
#pragma unroll
      for (int i = 0; i < V2; ++i) {
        float2 n = __fmul2_rn(x[i], a[i]);
        if constexpr (ROT != 0) n = __ffma2_rn(o[i], s[i], n);
        n = __fmul2_rn(n, make_float2(r, r));
        y[2 * i] = n.x, y[2 * i + 1] = n.y;
      }
      if (on && h < heads) store_row<T, V, true>((key ? yk : yq) + h * L.D, y);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) qk_norm_scalar(const __grid_constant__ QkNormLaunch L) {
  const int lane = threadIdx.x & 31;
  const int heads = L.q.H + L.k.H;
  const int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t row = w / heads;
  if (row >= L.M) return;
  bool ok;
  const float* turns = turns_of(L, row, lane, &ok);
  if (!ok) return;
  const int h = (int)(w - row * heads);
  const bool key = h >= L.q.H;
  const QkOperand& op = key ? L.k : L.q;
  const int64_t at0 = (int64_t)(key ? h - L.q.H : h) * L.D;
  const T* src = static_cast<const T*>(op.x) + row * op.ldx + at0;
  T* dst = static_cast<T*>(op.y) + row * op.ldy + at0;
  const float* wt = op.w;
  const int half = L.rot >> 1;
  float x[8], other[8];  // D <= 256
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = lane + 32 * i;
    x[i] = other[i] = 0.f;
    if (e < L.D) {
      x[i] = to_f32<T>(src[e]);
      ss = fmaf(x[i], x[i], ss);
      if (e < L.rot) other[i] = to_f32<T>(src[L.interleaved ? e ^ 1 : e < half ? e + half : e - half]);
    }
  }
  float r = 1.f;
  if (L.norm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    r = rsqrtf(fmaf(ss, 1.f / (float)L.D, L.eps));
  }
  __syncwarp();  // in place: every lane has read its partners before any lane stores
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = lane + 32 * i;
    if (e >= L.D) break;
    const float n = x[i] * r * (wt ? wt[e] : 1.f);
    float y = n;
    if (e < L.rot) {
      const int p = L.interleaved ? e >> 1 : e < half ? e : e - half;
      const int at = L.interleaved ? e ^ 1 : e < half ? e + half : e - half;
      const float m = other[i] * r * (wt ? wt[at] : 1.f);
      const bool first = L.interleaved ? !(e & 1) : e < half;
      y = fmaf(n, turns[p], m * (first ? -turns[half + p] : turns[half + p]));
    }
    dst[e] = from_f32<T>(y);
  }
}

template <typename T>
cudaError_t norm_as(const QkNormLaunch& L, bool vec, cudaStream_t s) {
  const int heads = L.q.H + L.k.H;
  const int pieces = L.D * (int)sizeof(T) / 16;
  if (vec && pieces <= 32) {
    int lph = 1;
    while (lph < pieces) lph *= 2;
    // As many warps per row as bring 16 to every SM (few rows), at least one head group each (61 rows of 32 + 8
    // heads of 128: one warp a row 12 us, this 8).
    const int groups = (heads + 32 / lph - 1) / (32 / lph);
    int64_t wpr = (148 * 16 + L.M - 1) / L.M;
    wpr = wpr < groups ? wpr : groups;
    const int64_t grid = (L.M * wpr + 3) / 4;
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    const bool whole = (L.rot / 2) % (16 / (int)sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(L.turns) % 16 == 0;
#define SUPRA_QK(N)                                                                               \
  case N:                                                                                         \
    if (L.rot == 0) qk_norm_vec<T, N, 0><<<(unsigned)grid, 128, 0, s>>>(L, (int)wpr);             \
    else if (L.interleaved) qk_norm_vec<T, N, 2><<<(unsigned)grid, 128, 0, s>>>(L, (int)wpr);     \
    else if (whole) qk_norm_vec<T, N, 1><<<(unsigned)grid, 128, 0, s>>>(L, (int)wpr);             \
    else qk_norm_vec<T, N, 3><<<(unsigned)grid, 128, 0, s>>>(L, (int)wpr);                        \
    break;
    switch (lph) {
      SUPRA_QK(1)
      SUPRA_QK(2)
      SUPRA_QK(4)
      SUPRA_QK(8)
      SUPRA_QK(16)
      SUPRA_QK(32)
    }
#undef SUPRA_QK
  } else {
    const int64_t grid = ((int64_t)L.M * heads + 7) / 8;
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    qk_norm_scalar<T><<<(unsigned)grid, 256, 0, s>>>(L);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_qk_norm(const QkNormLaunch& L, int type, bool vec, cudaStream_t s) {
  if (type == kTypeF32) return norm_as<float>(L, vec, s);
  if (type == kTypeF16) return norm_as<__half>(L, vec, s);
  return norm_as<__nv_bfloat16>(L, vec, s);
}

}  // namespace supra
