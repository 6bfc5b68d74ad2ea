// Attention of many query rows over the paged 8-bit K/V cache on the tcgen05 tensor cores (cross
// attention of an image's patches to a prompt, chunks of new tokens against their history).
//
// The mathematics of cache_attn.cu for tiles of 128 packed query rows (query, head of the group) against
// tiles of up to 128 tokens:
//   S = Q C_k^T      tcgen05.mma kind::f16, Q (smem, fp16) x K codes (smem, fp16), fp32 in TMEM
//   P = 2^(S c - m)  softmax threads, one row each: c = scale * k_scale of the token's block
//   O += f (P C_v)   tcgen05.mma kind::f16, P from TMEM x V codes (smem, MN-major); the tile's product
//                    goes into a fresh accumulator and is added to O in fp32 registers
// Codes are exact in fp16, so 8-bit K and V cost the tensor cores nothing but their conversion: four
// converter warps turn the raw bytes, which the TMA unit brings in block by block, into the swizzled
// operand tiles, once for all rows of the CTA. The V scales of a tile's blocks differ: p carries each
// block's scale over the tile's largest, as an exponent (added to m, so it costs nothing per element;
// the row's sum divides it out again per 32 tokens), and the largest multiplies the tile's product. A
// tile whose scales lie far apart (2^8, for fp32 rows 2^3) is taken block by block instead, so that a row
// that sees only its small ones keeps their precision.
// q carries a power of two per row (cache_attn.cu); fp32 rows and their p use two fp16 parts, and each
// product two MMAs.
//
// Head dims up to 64: one row tile per CTA, two CTAs per SM (128 + 64 TMEM columns each, 256 allocated).
// Up to 128: two row tiles per CTA that share the converted tiles, one CTA per SM (2 x 256 columns),
// registers moved from the converters to the softmax threads. Either way one row tile's softmax runs
// while the tensor cores work for the other. The softmax, 16 exponentials per cycle and SM, bounds the
// kernel: 128 x 128 scores take 1024 cycles of it and 2 x 256 (head dim 64) or 2 x 512 (128) of MMA.
// Every wait is bounded; on a timeout the CTA records the failure, waits for its own copies and MMAs, frees its
// TMEM and leaves.
#include <algorithm>
#include <type_traits>

#include "cache.cuh"
#include "tcgen05.cuh"

namespace supra {
namespace {

constexpr int kM = 128;  // rows of a row tile
constexpr int kN = 128;  // tokens of a tile
// p is formed as 2^15 p (fp16 ends at 65504). With its block's ratio r the smallest step of its fp16 form is
// 2^-40 / r of the row's largest p: blocks further apart than this are taken one by one.
constexpr float kPShift = 15.f;
template <bool SPLIT>
constexpr float kApart = SPLIT ? 0.125f : 0.00390625f;  // 2^-3, 2^-8
constexpr int kMeta = 4;  // tiles whose scales are kept at once

template <int DT, bool SPLIT>
struct Cfg {
  static constexpr int RT = DT == 64 ? 1 : 2;  // row tiles
  static constexpr int SOFT = 128 * RT;        // softmax threads
  static constexpr int THREADS = SOFT + 128;
  static constexpr int PER_SM = DT == 64 ? 2 : 1;
  static constexpr int RAW = DT == 128 && SPLIT ? 1 : 2;  // raw stages
  static constexpr int PARTS = SPLIT ? 2 : 1;
  static constexpr int SLABS = DT / 64;                       // 64-channel slabs of an operand tile
  static constexpr uint32_t SLAB = kM * 128;                  // 128 rows of 128 bytes
  static constexpr uint32_t QPART = SLABS * SLAB;             // one part of one row tile
  static constexpr uint32_t Q = 0;                            // [RT][PARTS]
  static constexpr uint32_t K = Q + RT * PARTS * QPART;
  static constexpr uint32_t V = K + SLABS * SLAB;
  static constexpr uint32_t RAWS = V + SLABS * SLAB;          // [RAW][K, V][kN][DT] bytes
  static constexpr uint32_t RAWB = kN * DT;
  static constexpr uint32_t META = RAWS + RAW * 2 * RAWB;     // [kMeta] TileMeta
  static constexpr uint32_t BAR = META + kMeta * 192;
  static constexpr uint32_t SMEM = BAR + 128 + 1024;          // + alignment of the base
  static constexpr uint32_t COL_ACC = kN;                     // S and P, then the tile's product
  static constexpr uint32_t COLS = DT == 64 ? 256 : 512;
  static constexpr uint32_t COL_RT = 256;
  static_assert(SMEM <= (PER_SM == 2 ? 113u : 227u) * 1024, "shared memory");
};

struct TileMeta {  // of a tile's eight 16-token groups
  float ks[8];
  float vs[8];
  float lr[8];   // log2 of |vs| over top, and its inverse ratio: what p carries, and its sum does not
  float ir[8];
  float top;     // the largest finite |vs|
  int32_t dead;  // groups whose block does not exist (bits), tokens past the end not among them
  int32_t subs;  // 1, or the number of blocks the tile is taken in
  int32_t pad[13];
};
static_assert(sizeof(TileMeta) == 192, "META");

struct Bars {
  uint64_t raw[2], k_full, v_full, k_empty, v_empty, s_full[2], pv_full[2], drain[2];
  uint32_t tmem;
  int32_t abort;
};
static_assert(sizeof(Bars) <= 128, "BAR");

// status[2] of a wait that ran out
enum TcWait : int32_t { W_RAW = 80, W_K_FULL = 81, W_V_FULL = 82, W_K_EMPTY = 83, W_V_EMPTY = 84, W_S = 85, W_PV = 86 };

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int32_t* abort, int32_t* status, int32_t id,
                                         int32_t detail) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 0u) {
      if (*abort) return false;
      if (global_ns() - t0 > kWaitLimitNs) {
        report_error(status, DEV_TIMEOUT, id, detail);
        *abort = 1;
        return false;
      }
    }
  }
}

__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// kind::f16, fp16 operands, fp32 accumulator
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
               "l"(a), "l"(b), "r"(idesc), "r"(acc)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
               "r"(a), "l"(b), "r"(idesc), "r"(acc)
               : "memory");
}
__host__ __device__ constexpr uint32_t idesc_f16(int N, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Four codes as two fp16 pairs in their order.
template <int FMT>
__device__ __forceinline__ void codes_in_order(uint32_t u, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == kCacheInt8) {
    const uint32_t x = u ^ 0x80808080u;  // codes + 128; 0x64 above a byte b is the fp16 number 1024 + b
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const uint32_t off = 0x64806480u;
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&off));
    const __half2 hb = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&off));
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(u));
  }
}

template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// T: q and out; DT: head dim rounded up to 64 or 128.
template <typename T, int FMT, int DT>
__global__ void __launch_bounds__(Cfg<DT, sizeof(T) == 4>::THREADS, Cfg<DT, sizeof(T) == 4>::PER_SM)
    cache_attn_tc_kernel(const __grid_constant__ CacheAttnArgs L, const __grid_constant__ CUtensorMap mk,
                         const __grid_constant__ CUtensorMap mv, int tiles) {
  constexpr bool SPLIT = sizeof(T) == 4;
  using Y = Cfg<DT, SPLIT>;
  constexpr int RT = Y::RT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // swizzle atoms
  TileMeta* meta = reinterpret_cast<TileMeta*>(base + Y::META);
  Bars* B = reinterpret_cast<Bars*>(base + Y::BAR);
  volatile int32_t* abort = &B->abort;
  const CachePool& c = L.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // unit = (row tile, sequence, cache head), the longest causal row tiles first; the CTAs that split a
  // unit's tokens are neighbours
  int unit = blockIdx.x / L.splits;
  const int split = blockIdx.x % L.splits;
  const int rt0 = tiles - 1 - unit % tiles;
  unit /= tiles;
  const int hk = unit % c.H, b = unit / c.H;
  SeqView q;
  if (!seq_view(L.s, b, false, L.status, q)) return;
  const int rows = q.n * L.G;  // packed (query, head of the group)
  const int r0 = rt0 * kM * RT;
  if (r0 >= rows) return;
  const int nrow = min(kM * RT, rows - r0);
  const int past = q.len - q.n;
  const int i_last = (r0 + nrow - 1) / L.G, i_first = r0 / L.G;
  const int seen = L.causal ? max(0, min(q.len, past + i_last + 1)) : q.len;
  const int all = L.causal ? max(0, min(q.len, past + i_first + 1)) : q.len;
  // this CTA's tiles
  const int nt = (seen + kN - 1) / kN;
  const int j0 = (int)((int64_t)nt * split / L.splits), j1 = (int)((int64_t)nt * (split + 1) / L.splits);

  if (threadIdx.x == 0) {
    mbar_init(&B->raw[0], 1);
    mbar_init(&B->raw[1], 1);
    mbar_init(&B->k_full, 128);
    mbar_init(&B->v_full, 128);
    mbar_init(&B->k_empty, RT);
    mbar_init(&B->v_empty, RT);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->s_full[i], 1);
      mbar_init(&B->pv_full[i], 1);
      mbar_init(&B->drain[i], 1);
    }
    B->abort = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    tc::tmem_alloc(&B->tmem, Y::COLS);
    tc::tmem_relinquish();
  } else if (warp == 1 && lane == 0) {
    tc::prefetch_map(&mk);
    tc::prefetch_map(&mv);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = B->tmem;

  if (warp >= 4 * RT) {
    // ---------------- converters ----------------
    if constexpr (RT == 2) reg_dec<88>();
    const int ct = threadIdx.x - Y::SOFT;
    const int log2t = c.log2t;
    // Tile j's blocks into raw stage j % RAW and its scales into meta[j % kMeta] (the first warp).
    auto load = [&](int j) {
      if (j >= j1) return;
      const int st = (j - j0) % Y::RAW;
      TileMeta& mt = meta[(j - j0) % kMeta];
      const int tok = j * kN + 16 * lane;  // lanes 0-7: the tile's groups
      const bool in = lane < 8 && tok < seen;
      const int32_t page = in ? L.s.table[(int64_t)b * L.s.ld_table + (tok >> log2t)] : -1;
      const bool live = in && page >= 0 && page < c.blocks;
      if (in && !live) report_error(L.status, DEV_BAD_BLOCK, 2, page);
      const bool first = (tok & ((1 << log2t) - 1)) == 0;  // one box per block of the tile
      const uint32_t boxes = __ballot_sync(0xffffffffu, live && first);
      const uint32_t dead = __ballot_sync(0xffffffffu, in && !live);
      const int box_rows = min(kN, 1 << log2t);
      if (lane == 0) {
        mt.dead = (int32_t)dead;
        mbar_arrive_expect_tx(&B->raw[st], (uint32_t)(__popc(boxes) * 2 * box_rows * DT));
      }
      __syncwarp();
      if (boxes >> lane & 1) {
        const int y = ((page * c.H + hk) << log2t) + (tok & ((1 << log2t) - 1));
        uint8_t* to = base + Y::RAWS + st * 2 * Y::RAWB + 16 * lane * DT;
        tc::tma_load_2d(to, &mk, 0, y, &B->raw[st]);
        tc::tma_load_2d(to + Y::RAWB, &mv, 0, y, &B->raw[st]);
      }
      float ks = 0.f, vs = 0.f;
      if (live) {
        const int64_t u = (int64_t)page * c.H + hk;
        ks = c.ks[u];
        vs = c.vs[u];
      }
      const float av = fabsf(vs);
      float top = live && av <= 3.4028234e38f ? av : 0.f;
      float low = live && av <= 3.4028234e38f ? av : 3.4028234e38f;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      }
      // (a tile with a negative scale, which no write makes, goes block by block too)
      const bool neg = __any_sync(0xffffffffu, live && vs < 0.f);
      const bool apart = log2t < 7 && (low < top * kApart<SPLIT> || neg);
      if (lane < 8) {
        const float ratio = apart || av == top || !live ? 1.f : av / top;
        mt.ks[lane] = ks;
        mt.vs[lane] = vs;
        mt.lr[lane] = ratio == 1.f ? 0.f : log2f(ratio);
        mt.ir[lane] = 1.f / ratio;
      }
      if (lane == 0) {
        mt.top = top;
        mt.subs = apart ? kN >> log2t : 1;
      }
    };
    int loaded = j0;
    if (ct < 32) {
      for (; loaded < j0 + Y::RAW; ++loaded) load(loaded);
    }
    constexpr int CPR = DT / 16;  // 16-byte pieces per row
    const int pc = ct % CPR, pr = ct / CPR;
    bool ok = true;
    for (int j = j0; j < j1; ++j) {
      const int n = j - j0, st = n % Y::RAW;
      if (!(ok = wait_for(&B->raw[st], (uint32_t)(n / Y::RAW) & 1u, abort, L.status, W_RAW, j))) break;
      const int tok0 = j * kN;
      const int nrows = min(kN, (seen - tok0 + 31) & ~31);
      const uint32_t dead = (uint32_t)meta[n % kMeta].dead;
      // bytes past the last token (or of a block that does not exist) may be NaN codes: zeros instead
      const bool cut = FMT == kCacheE4m3 && (tok0 + nrows > seen || dead);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        if (n > 0 && !(ok = wait_for(kv ? &B->v_empty : &B->k_empty, (uint32_t)(n - 1) & 1u, abort, L.status, kv ? W_V_EMPTY : W_K_EMPTY, j)))
          break;
        const uint8_t* src = base + Y::RAWS + (st * 2 + kv) * Y::RAWB;
        uint8_t* dst = base + (kv ? Y::V : Y::K);
#pragma unroll 4
        for (int r = pr; r < nrows; r += 128 / CPR) {
          uint4 w = *reinterpret_cast<const uint4*>(src + r * DT + 16 * pc);
          if (cut && (tok0 + r >= seen || (dead >> (r >> 4) & 1))) w = make_uint4(0, 0, 0, 0);
          uint4 x, y;
          codes_in_order<FMT>(w.x, x.x, x.y);
          codes_in_order<FMT>(w.y, x.z, x.w);
          codes_in_order<FMT>(w.z, y.x, y.y);
          codes_in_order<FMT>(w.w, y.z, y.w);
          uint8_t* row = dst + (pc >> 2) * Y::SLAB + r * 128;
          const int k = 2 * (pc & 3);
          *reinterpret_cast<uint4*>(row + ((k ^ (r & 7)) << 4)) = x;
          *reinterpret_cast<uint4*>(row + (((k + 1) ^ (r & 7)) << 4)) = y;
        }
        fence_proxy_async_smem();
        mbar_arrive(kv ? &B->v_full : &B->k_full);
      }
      if (!ok) break;
      bar_sync(1, 128);  // every converter has left the raw stage
      if (ct < 32 && loaded < j1) load(loaded++);
    }
    if (!ok && ct == 0) {  // copies in flight land before the CTA may leave
      for (int j = j0; j < min(loaded, j1); ++j) mbar_wait_bounded(&B->raw[(j - j0) % Y::RAW], (uint32_t)((j - j0) / Y::RAW) & 1u);
    }
  } else {
    // ---------------- softmax, MMA issue, epilogue: one row per thread ----------------
    if constexpr (RT == 2) reg_inc<208>();
    const int rt = warp >> 2, tr = threadIdx.x & 127;
    const int r = rt * kM + tr;  // row of the CTA
    const bool live = r < nrow;
    const int prow = r0 + min(r, nrow - 1);
    const int qi = prow / L.G;
    const int64_t head = (int64_t)(hk * L.G + prow % L.G) * c.D;
    const int lim = !live ? -1 : L.causal ? min(q.len - 1, past + qi) : q.len - 1;  // the last token the row sees
    const uint32_t tl = tmem + (uint32_t)rt * Y::COL_RT + ((uint32_t)((warp & 3) * 32) << 16);  // this warp's lanes
    uint8_t* Qs = base + Y::Q + rt * Y::PARTS * Y::QPART;

    // q, times a power of two that brings its largest channel into [2^13, 2^14) (and the sign of the scale)
    float rs;
    {
      const T* src = static_cast<const T*>(L.q) + (q.row0 + qi) * L.ldq + head;
      const bool vec = L.vec != 0;
      auto load8 = [&](int e, float (&x)[8]) {
        if (!live || e >= c.D) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = 0.f;
        } else if (vec) {
          load_row<T, 8, true>(src + e, x);
        } else {
          load_row<T, 8, false>(src + e, x);
        }
      };
      float top = 0.f;
#pragma unroll 4
      for (int e = 0; e < DT; e += 8) {
        float x[8];
        load8(e, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
      }
      const int ex = min(max((int)(__float_as_uint(top) >> 23), 27), 254) - 127;
      const float up = __uint_as_float(((uint32_t)(13 - ex + 127) << 23) | (L.scale_log2 < 0.f ? 0x80000000u : 0u));
      rs = fabsf(L.scale_log2) * __uint_as_float((uint32_t)(ex - 13 + 127) << 23);
#pragma unroll 4
      for (int e = 0; e < DT; e += 8) {
        float x[8];
        load8(e, x);
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] *= up, x[2 * i + 1] *= up;
          h[i] = pack2<__half>(x[2 * i], x[2 * i + 1]);
          if constexpr (SPLIT) {
            const float2 f = unpack2<__half>(h[i]);
            l[i] = pack2<__half>(x[2 * i] - f.x, x[2 * i + 1] - f.y);
          }
        }
        uint8_t* at = Qs + (e >> 6) * Y::SLAB + tr * 128 + ((((e >> 3) & 7) ^ (tr & 7)) << 4);
        *reinterpret_cast<uint4*>(at) = make_uint4(h[0], h[1], h[2], h[3]);
        if constexpr (SPLIT) *reinterpret_cast<uint4*>(at + Y::QPART) = make_uint4(l[0], l[1], l[2], l[3]);
      }
      fence_proxy_async_smem();
    }
    bar_sync(2 + rt, 128);

    bool ok = true;
    // S of tile j (its first n tokens) into the row tile's S columns, by the row tile's first thread.
    auto issue_s = [&](int j, bool first) {
      if (first && !wait_for(&B->k_full, (uint32_t)(j - j0) & 1u, abort, L.status, W_K_FULL, j)) return;
      tc::fence_after_sync();
      const int n = min(kN, (seen - j * kN + 31) & ~31);
      const uint32_t id = idesc_f16(n, false);
      const uint32_t d = tmem + (uint32_t)rt * Y::COL_RT;
#pragma unroll
      for (int p = 0; p < Y::PARTS; ++p)
#pragma unroll
        for (int k = 0; k < DT / 16; ++k) {
          const uint64_t a = tc::smem_desc(Qs + p * Y::QPART + (k >> 2) * Y::SLAB + (k & 3) * 32, 16, 1024, tc::kLayoutSW128);
          const uint64_t w = tc::smem_desc(base + Y::K + (k >> 2) * Y::SLAB + (k & 3) * 32, 16, 1024, tc::kLayoutSW128);
          mma_ss(d, a, w, id, p + k > 0);
        }
      tc::commit(&B->s_full[rt]);
    };
    auto issue_pv = [&](int j, bool first, bool last) {
      if (first && !wait_for(&B->v_full, (uint32_t)(j - j0) & 1u, abort, L.status, W_V_FULL, j)) return;
      tc::fence_after_sync();
      const int steps = (min(kN, seen - j * kN) + 15) >> 4;
      constexpr uint32_t id = idesc_f16(DT, true);
      const uint32_t s0 = tmem + (uint32_t)rt * Y::COL_RT, d = s0 + Y::COL_ACC;
      for (int k = 0; k < steps; ++k) {
        // V is MN-major: 64-channel slabs SLAB apart (LBO), 8-token groups 1024 B apart (SBO)
        const uint64_t w = tc::smem_desc(base + Y::V + k * 2048, Y::SLAB, 1024, tc::kLayoutSW128);
        const uint32_t a = s0 + 32 * (k >> 1) + 8 * (k & 1);  // P of 32 tokens: 16 columns, then its low part
        mma_ts(d, a, w, id, k > 0);
        if constexpr (SPLIT) mma_ts(d, a + 16, w, id, 1);
      }
      tc::commit(&B->pv_full[rt]);
      if (last) tc::commit(&B->v_empty);
    };

    float o[DT];
#pragma unroll
    for (int e = 0; e < DT; ++e) o[e] = 0.f;
    float m = -INFINITY, l = 0.f;
    int it = 0;  // passes: tiles, or parts of tiles
    if (j0 < j1 && tr == 0) issue_s(j0, true);
    for (int j = j0; j < j1 && ok; ++j) {
      const TileMeta& mt = meta[(j - j0) % kMeta];
      const int tok0 = j * kN;
      const int ncol = min(kN, seen - tok0), nch = (ncol + 31) >> 5;
      int subs = 1;
      for (int sub = 0; sub < subs && ok; ++sub, ++it) {
        if (!(ok = wait_for(&B->s_full[rt], (uint32_t)it & 1u, abort, L.status, W_S, j))) break;
        tc::fence_after_sync();
        if (sub == 0) subs = mt.subs;  // (written before the tile's K was converted)
        if (tr == 0 && sub + 1 == subs) tc::commit(&B->k_empty);  // the tile's last scores are formed
        // columns of this pass that the row sees: [lo, hi)
        const int lo = subs > 1 ? sub << c.log2t : 0;
        const int end = subs > 1 ? min(ncol, (sub + 1) << c.log2t) : ncol;
        const int hi = min(end, lim - tok0 + 1);
        const bool partial = subs > 1 || tok0 + ncol > all || (ncol & 31) || mt.dead;
        const uint32_t deadm = (uint32_t)mt.dead;
        // what the product is multiplied by: a row that sees none of it has a product of 0 and takes 0
        const float v0 = mt.vs[lo >> 4];
        const float f = hi <= lo ? 0.f : subs > 1 ? v0 : v0 < 0.f ? -mt.top : mt.top;

        // the row's maximum: the largest score of each 16 tokens (32, when blocks hold as many) times their
        // factor
        float mx = -INFINITY;
        auto largest = [](const float* s) {
          float u = max3(s[0], s[1], s[2]), w = max3(s[3], s[4], s[5]);
#pragma unroll
          for (int e = 6; e < 14; e += 4) u = max3(u, s[e], s[e + 1]), w = max3(w, s[e + 2], s[e + 3]);
          u = max3(u, s[14], s[15]);
          return fmaxf(u, w);
        };
        for (int ch = 0; ch < nch; ++ch) {
          float s[32];
          tc::tmem_ld32(tl + 32 * ch, s);
          const float k0 = mt.ks[2 * ch] * rs, k1 = mt.ks[2 * ch + 1] * rs;
          tc::tmem_wait_ld();
          if (partial) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const int col = 32 * ch + e;
              if (col < lo || col >= hi || (deadm >> (2 * ch + (e >> 4)) & 1)) s[e] = k0 < 0.f ? INFINITY : -INFINITY;
            }
          }
          if (k0 < 0.f || k1 < 0.f) {  // (a negative K scale, which no write makes: score by score)
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float y = fabsf(s[e]) < INFINITY ? s[e] * (e < 16 ? k0 : k1) : -INFINITY;
              mx = fmaxf(mx, y);
            }
          } else {
            const float a0 = largest(s), a1 = largest(s + 16);
            mx = max3(mx, a0 * k0, a1 * k1);  // (-inf times a factor of 0 is NaN, which the maximum leaves out)
          }
        }
        const float mn = fmaxf(m, mx);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float al = ex2f(m - ref);
        const bool moved = mn != m;
        m = mn;
        // p, its sum, and P into the columns of the scores it comes from
        float sum = 0.f;
        for (int ch = 0; ch < nch; ++ch) {
          float s[32];
          tc::tmem_ld32(tl + 32 * ch, s);
          const float k0 = mt.ks[2 * ch] * rs, k1 = mt.ks[2 * ch + 1] * rs;
          const float h0 = kPShift - ref + mt.lr[2 * ch], h1 = kPShift - ref + mt.lr[2 * ch + 1];
          const float i0 = mt.ir[2 * ch], i1 = mt.ir[2 * ch + 1];
          tc::tmem_wait_ld();
          uint32_t ph[16], pl[SPLIT ? 16 : 1];
          float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          auto form = [&](auto masked) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float k = e < 16 ? k0 : k1, h = e < 16 ? h0 : h1;
              float2 x = __ffma2_rn(make_float2(s[e], s[e + 1]), make_float2(k, k), make_float2(h, h));
              if constexpr (decltype(masked)::value) {
                const int col = 32 * ch + e;
                const bool dd = deadm >> (2 * ch + (e >> 4)) & 1;
                if (col < lo || col >= hi || dd) x.x = -INFINITY;
                if (col + 1 < lo || col + 1 >= hi || dd) x.y = -INFINITY;
              }
              x.x = ex2f(x.x);
              x.y = ex2f(x.y);
              part[e >> 4] = __fadd2_rn(part[e >> 4], x);
              const int w = e >> 1;
              ph[w] = pack2<__half>(x.x, x.y);
              if constexpr (SPLIT) {
                const float2 f = unpack2<__half>(ph[w]);
                const float2 d = __ffma2_rn(f, make_float2(-1.f, -1.f), x);
                pl[w] = pack2<__half>(d.x, d.y);
              }
            }
          };
          if (partial) form(std::true_type{});
          else form(std::false_type{});
          const float p0 = part[0].x + part[0].y, p1 = part[1].x + part[1].y;
          // (the ratio of a block that no visible token is in may be NaN)
          sum += (p0 == 0.f ? 0.f : p0 * i0) + (p1 == 0.f ? 0.f : p1 * i1);
          tmem_st16(tl + 32 * ch, ph);
          if constexpr (SPLIT) tmem_st16(tl + 32 * ch + 16, pl);
        }
        l = l * al + sum;
        tc::tmem_wait_st();
        tc::fence_before_sync();
        bar_sync(2 + rt, 128);
        const bool lastsub = sub + 1 == subs;
        if (tr == 0) issue_pv(j, sub == 0, lastsub);
        if (!(ok = wait_for(&B->pv_full[rt], (uint32_t)it & 1u, abort, L.status, W_PV, j))) break;
        tc::fence_after_sync();
        // the next scores, while this product is added to O
        if (tr == 0) {
          if (!lastsub) issue_s(j, false);
          else if (j + 1 < j1) issue_s(j + 1, true);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int e = 0; e < DT; e += 2) {
            const float2 w = __fmul2_rn(make_float2(o[e], o[e + 1]), make_float2(al, al));
            o[e] = w.x, o[e + 1] = w.y;
          }
        }
#pragma unroll
        for (int e = 0; e < DT; e += 32) {
          float a[32];
          tc::tmem_ld32(tl + Y::COL_ACC + e, a);
          tc::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 y = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(f, f), make_float2(o[e + i], o[e + i + 1]));
            o[e + i] = y.x, o[e + i + 1] = y.y;
          }
        }
        tc::fence_before_sync();
      }
    }
    if (!ok && tr == 0 && *abort) {
      // MMAs in flight end before TMEM is freed: an arrival of their own, waited for within limits
      tc::commit(&B->drain[rt]);
      mbar_wait_bounded(&B->drain[rt], 0);
    }

    // ---- epilogue: the row through shared memory (its own Q rows), stored in whole 16-byte pieces ----
    if (L.ws_o) {
      if (live) {
        const int64_t at = (int64_t)blockIdx.x * (kM * RT) + r;
#pragma unroll
        for (int e = 0; e < DT; e += 4)
          if (e < c.D) *reinterpret_cast<float4*>(L.ws_o + at * c.D + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        L.ws_ml[at] = make_float2(m, l);
      }
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      constexpr int PER = DT * (int)sizeof(T) / 16;  // pieces of a row
      constexpr int V8 = 16 / (int)sizeof(T);
      uint8_t* mine = Qs + tr * (PER * 16);
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        float x[V8];
#pragma unroll
        for (int i = 0; i < V8; ++i) x[i] = l == 0.f ? 0.f : o[p * V8 + i] * inv;
        store_row<T, V8, true>(reinterpret_cast<T*>(mine + ((p ^ (tr & 7)) << 4)), x);
      }
      __syncwarp();
      const int per = c.D / V8;  // pieces that exist
      // each row's address is known to its own thread
      T* mine_out = live ? static_cast<T*>(L.o) + (q.row0 + qi) * L.ldo + head : nullptr;
      constexpr int RPI = 32 / PER;  // rows of an iteration
#pragma unroll 4
      for (int i = 0; i < 32; i += (RPI > 0 ? RPI : 1)) {
        const int rl = i + (RPI > 0 ? lane / PER : 0), p = lane % PER;
        T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine_out), rl));
        const T* from = reinterpret_cast<const T*>(Qs + ((tr & ~31) + rl) * (PER * 16) + ((p ^ (rl & 7)) << 4));
        if (!to || p >= per) continue;
        to += p * V8;
        if (L.vec) {
          *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
        } else {
#pragma unroll
          for (int e = 0; e < V8; ++e) to[e] = from[e];
        }
      }
    }
    tc::fence_before_sync();
  }
  __syncthreads();
  if (warp == 0) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, Y::COLS);
  }
}

template <typename T, int FMT, int DT>
cudaError_t tc_as(const CacheAttnLaunch& L, const CacheAttnPlan& P, cudaStream_t s) {
  using Y = Cfg<DT, sizeof(T) == 4>;
  auto kernel = cache_attn_tc_kernel<T, FMT, DT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Y::SMEM);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)(P.units * P.splits), Y::THREADS, Y::SMEM, s>>>(L, L.mk, L.mv, P.tiles);
  return cudaGetLastError();
}
template <typename T>
cudaError_t tc_type(const CacheAttnLaunch& L, const CacheAttnPlan& P, int format, cudaStream_t s) {
  if (L.c.D <= 64) return format == kCacheInt8 ? tc_as<T, kCacheInt8, 64>(L, P, s) : tc_as<T, kCacheE4m3, 64>(L, P, s);
  return format == kCacheInt8 ? tc_as<T, kCacheInt8, 128>(L, P, s) : tc_as<T, kCacheE4m3, 128>(L, P, s);
}

}  // namespace

cudaError_t launch_cache_attn_tc(const CacheAttnLaunch& L, const CacheAttnPlan& P, int type, int format, cudaStream_t s) {
  if (P.units * P.splits > INT32_MAX) return cudaErrorInvalidValue;
  if (type == kTypeF32) return tc_type<float>(L, P, format, s);
  if (type == kTypeF16) return tc_type<__half>(L, P, format, s);
  return tc_type<__nv_bfloat16>(L, P, format, s);
}
int cache_attn_tc_rows(int D) { return D <= 64 ? kM : 2 * kM; }

}  // namespace supra
