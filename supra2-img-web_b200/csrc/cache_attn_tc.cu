// Attention of many query rows over the paged 8-bit K/V cache on the tcgen05 tensor cores (cross
// attention of an image's patches to a prompt, chunks of new tokens against their history).
//
// The mathematics of cache_attn.cu for tiles of 128 packed query rows (query, head of the group) against
// tiles of 64 tokens:
//   S = Q C_k^T      tcgen05.mma kind::f16, Q (smem, fp16) x K codes (smem, fp16), fp32 in TMEM
//   P = 2^(S c + log2 v - m)   softmax threads, one row each: c = scale * k_scale and v = v_scale of the
//                    token's block, m the row's largest exponent so far
//   O += P C_v       tcgen05.mma kind::f16, P from TMEM x V codes (smem, MN-major)
//   o = O / sum(P / v)
// Codes are exact in fp16, so 8-bit K and V cost the tensor cores nothing but their conversion: three
// converter warps turn the raw bytes, which the TMA unit brings in block by block, into the swizzled
// operand tiles, once for all rows of the CTA. P carries the V scale as an exponent, which costs nothing
// per score, and m follows the product of both, so each row's P is as large as fp16 allows whatever the
// scales of the blocks that it sees; only the sum divides the scale out again, once per 16 tokens. That holds
// while V scales are within 2^32 of 1: P of a token whose score is within 2^-69 of the row's largest is then above
// 2^-126, and the sum, in units of 2^m, within the range of 32 bits. Tiles with others (blocks of zeros have
// 2^-107) are odd ones: their sum is formed from exponentials of its own, in units of 2^(m - d), with d the whole
// number that keeps m - d near the row's largest score alone; warps with a row whose d is not 0 stay with that form.
// q carries a power of two per row (cache_attn.cu).
// 16-bit rows keep O in TMEM, where m moves only when a tile exceeds it by 2^8 (then the softmax threads
// rescale O there). Sums in TMEM are truncated, which pulls them towards zero by up to 2^-23 for each 16 tokens (measured
// 2e-4 at 32768 tokens, half a rounding of fp16): after every 4096 tokens O joins a sum that is rounded to nearest, in local
// memory, and starts anew (32768 tokens: 2e-5). fp32 rows use two fp16 parts of q and p (each product two MMAs), move m exactly, and
// add each tile's product to O in fp32 registers, rounded to nearest, so that the error does not grow
// with the number of tiles.
//
// Head dims up to 64: one row tile per CTA, two CTAs per SM (192 TMEM columns each, 256 allocated). Up to
// 128: two row tiles per CTA that share the converted tiles, one CTA per SM (2 x 256 columns). fp32 rows
// move registers from the converters to the softmax threads. K, V and their raw bytes have two stages
// each, and so has S: a row tile's next scores are formed while its softmax threads work on the present
// ones, and its last product behind them, so that neither MMA nor conversion is waited for. What bounds
// a CTA is the softmax: 16 exponentials per cycle and SM, and about five instructions a score (the busiest SM issues
// in 65 % of its slots). What bounds a launch of few unlike CTAs is their distribution:
// Measured: 4 causal chunks of 700 to 1024 rows over 2049 to 4096 tokens, 16 heads of 128, 4 cache heads, INT8 and bf16:
// 138 us, 549 TFLOP/s: 220 CTAs of up to 64 tiles, one an SM, leave the 148 SMs idle for a third of the time (94 tiles on
// the last, 64 in the mean). 128 prompts of 1 to 128 tokens, 256 rows each, 9 heads of 64, INT8 and fp32 rows: 88 us,
// 1.8 TB/s (a CTA has two tiles at most; its q, its output and the latencies between take the time). A fourth
// converter warp did not change the first. FP32 rows of more than 64 channels spill registers (about 670 bytes a thread:
// O takes 128 of 208): 8 sequences of 300 to 512 causal rows over 1024 to 2048 tokens, 8 heads of 128: 139 us.
// Every wait is bounded; on a timeout the CTA records the failure, waits for its own copies and MMAs, frees its
// TMEM and leaves.
#include <algorithm>
#include <type_traits>

#include "cache.cuh"
#include "tcgen05.cuh"

namespace supra {
namespace {

constexpr int kM = 128;  // rows of a row tile
constexpr int kN = 64;   // tokens of a tile
// P is formed as 2^kPShift P (fp16 ends at 65504). 16-bit rows: m may lag the row's largest exponent by kLag.
template <bool SPLIT>
constexpr float kPShift = SPLIT ? 15.f : 7.f;
constexpr float kLag = 8.f;
constexpr int kFold = 64;  // 16-bit rows: tiles that TMEM sums up at a time
constexpr float kScaleMin = 2.3283064365386963e-10f, kScaleMax = 4294967296.f;  // 2^-32, 2^32: V scales of common tiles
constexpr float kNear = 32.f;   // d is 0 where m is within this of the row's largest score
constexpr float kSlack = 16.f;  // elsewhere m - d is
// Tiles whose scales are kept at once: while the converters have tile i, the softmax threads are past tile i - 4 (tile
// i - 2 has its scores, for which product i - 4 was waited for), and tiles i + 2 .. i + 9 are described together.
constexpr int kMeta = 13;

template <int DT, bool SPLIT>
struct Cfg {
  static constexpr int RT = DT == 64 ? 1 : 2;  // row tiles
  static constexpr int SOFT = 128 * RT;        // softmax threads
  static constexpr int CONV = 96;  // converter threads, followed by one warp that issues the MMAs
  static constexpr int THREADS = SOFT + 128;
  static constexpr int PER_SM = DT == 64 ? 2 : 1;
  static constexpr int PARTS = SPLIT ? 2 : 1;
  static constexpr int CHUNK = SPLIT && DT == 128 ? 32 : 64;  // scores that a thread holds at once
  // fp32 rows: registers of a thread at launch, and after the softmax threads have taken some from the
  // others; together no more than the CTA was launched with (the launcher checks what that was).
  static constexpr int REGS = DT == 64 ? 128 : 168;
  static constexpr int REGS_SOFT = DT == 64 ? 168 : 208, REGS_REST = 88;
  static_assert(SOFT * REGS_SOFT + 128 * REGS_REST <= THREADS * REGS, "registers");
  static constexpr int SLABS = DT / 64;                       // 64-channel slabs of an operand tile
  static constexpr uint32_t QSLAB = kM * 128;                 // 128 rows of 128 bytes
  static constexpr uint32_t QPART = SLABS * QSLAB;            // one part of one row tile
  static constexpr uint32_t SLAB = kN * 128;                  // of K or V
  static constexpr uint32_t TILE = SLABS * SLAB;              // K or V, one stage
  static constexpr uint32_t Q = 0;                            // [RT][PARTS]
  static constexpr uint32_t K = Q + RT * PARTS * QPART;       // [2]
  static constexpr uint32_t V = K + 2 * TILE;                 // [2]
  static constexpr uint32_t RAWS = V + 2 * TILE;              // [2][K, V][kN][DT] bytes
  static constexpr uint32_t RAWB = kN * DT;
  static constexpr uint32_t RS = RAWS + 4 * RAWB;             // score factor of each row
  static constexpr uint32_t META = RS + RT * kM * 4;          // [kMeta] TileMeta
  static constexpr uint32_t BAR = META + kMeta * 64;
  static constexpr uint32_t SMEM = BAR + 192 + 1024;          // + alignment of the base
  static constexpr uint32_t COL_ACC = 2 * kN;                 // two buffers of S and P, then the tile's product
  static constexpr uint32_t COLS = DT == 64 ? 256 : 512;
  static constexpr uint32_t COL_RT = 256;
  static_assert(SMEM <= (PER_SM == 2 ? 113u : 227u) * 1024, "shared memory");
};

struct TileMeta {  // of a tile's four 16-token groups
  float ks[4];
  float lv[4];   // log2 |v_scale|; where |v_scale| is outside [kScaleMin, kScaleMax], without its whole part
  float iv[4];   // 1 / |v_scale|
  int32_t dead;  // groups whose block does not exist (bits), tokens past the end not among them
  int32_t neg;   // groups with a negative V scale (bits), which no write makes
  int32_t odd;   // groups that are dead, or a scale of theirs is negative or not finite, the K scale 0 or the V scale
                 // outside [kScaleMin, kScaleMax]
  int8_t whole[4];  // what lv is without
};
static_assert(sizeof(TileMeta) == 64, "META");

struct Bars {
  uint64_t raw[2], k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2][2], p_full[2], pv_full[2], drain;
  uint32_t tmem;
  int32_t abort;
};
static_assert(sizeof(Bars) <= 192, "BAR");

// status[2] of a wait that ran out
enum TcWait : int32_t { W_RAW = 80, W_ISSUE = 81, W_K_EMPTY = 83, W_V_EMPTY = 84, W_S = 85, W_PV = 86 };

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int32_t* abort, int32_t* status, int32_t id,
                                         int32_t detail) {
  if (mbar_wait_clocked(bar, parity, abort)) return true;
  if (!*abort) {
    report_error(status, DEV_TIMEOUT, id, detail);
    *abort = 1;
  }
  return false;
}

__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// The barrier of a role's threads, and whether all of them are well: whoever gave up a wait still arrives, and
// all leave together.
__device__ __forceinline__ bool bar_and(int id, int n, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}

// One lane of a converged warp, the same in every call; the branch it guards is uniform to the compiler, so
// the MMA operands stay in uniform registers (a branch on a thread's number cost ~190 cycles per MMA).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

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

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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

// T: q and out; DT: head dim rounded up to 64 or 128. FOLD: 16-bit rows whose CTAs may walk over more than kFold tiles (the
// others are spared its code: 128 prompts of up to 128 tokens, 256 bf16 rows each: 74 us with it, 72 without).
template <typename T, int FMT, int DT, bool FOLD>
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
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // (uniform)

  if (L.ws_o) join_may_start();
  // unit = (row tile, sequence, cache head), the longest causal row tiles first; the CTAs that split a
  // unit's tokens are neighbours
  const int unit = blockIdx.x / L.splits, split = blockIdx.x % L.splits;
  const int heads = L.s.B * c.H;
  const int rt0 = tiles - 1 - unit / heads;
  const int hk = unit % heads % c.H, b = unit % heads / c.H;
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
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->raw[i], 1);
      mbar_init(&B->k_full[i], Y::CONV);
      mbar_init(&B->v_full[i], Y::CONV);
      mbar_init(&B->k_empty[i], RT);
      mbar_init(&B->v_empty[i], RT);
      mbar_init(&B->s_full[i][0], 1);
      mbar_init(&B->s_full[i][1], 1);
      mbar_init(&B->p_full[i], 128);
      mbar_init(&B->pv_full[i], 1);
    }
    mbar_init(&B->drain, 1);
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

  constexpr int V8 = 16 / (int)sizeof(T);  // channels of a 16-byte piece
  constexpr int PER = DT / V8;             // pieces of a row: 8, 16 or 32
  constexpr int RPI = 32 / PER;            // rows of a warp's load
  // 32 rows of a row tile by one warp, PER lanes a row: q times a power of two that brings the row's largest
  // channel into [2^13, 2^14) (and the sign of the scale), as fp16.
  auto load_q = [&](int rt, int row0) {
    uint8_t* Qs = base + Y::Q + rt * Y::PARTS * Y::QPART;
    float* rsm = reinterpret_cast<float*>(base + Y::RS) + rt * kM;
    const int my = rt * kM + row0 + lane;  // the row whose address this lane works out
    const T* mine = nullptr;
    if (my < nrow) {
      const int pk = r0 + my;
      mine = static_cast<const T*>(L.q) + (q.row0 + pk / L.G) * L.ldq + (int64_t)(hk * L.G + pk % L.G) * c.D;
    }
    const int p = lane % PER, e = p * V8;
    constexpr int N = 32 / RPI, UN = N < 16 ? N : 16;  // loads, and those under way
#pragma unroll 1
    for (int i0 = 0; i0 < N; i0 += UN) {
      uint4 raw[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int rl = (i0 + u) * RPI + lane / PER;
        const T* src = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), rl));
        raw[u] = make_uint4(0, 0, 0, 0);
        if (src && e < c.D) {
          if (L.vec) {
            raw[u] = *reinterpret_cast<const uint4*>(src + e);
          } else {
            T y[V8];
#pragma unroll
            for (int i = 0; i < V8; ++i) y[i] = src[e + i];
            memcpy(&raw[u], y, 16);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int row = row0 + (i0 + u) * RPI + lane / PER;
        float x[V8];
        load_row<T, V8, true>(reinterpret_cast<const T*>(&raw[u]), x);
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < V8; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
        for (int o = PER / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int ex = min(max((int)(__float_as_uint(top) >> 23), 27), 254) - 127;
        const float up = __uint_as_float(((uint32_t)(13 - ex + 127) << 23) | (L.scale_log2 < 0.f ? 0x80000000u : 0u));
        if (p == 0) rsm[row] = fabsf(L.scale_log2) * __uint_as_float((uint32_t)(ex - 13 + 127) << 23);
        uint32_t h[V8 / 2], lo[V8 / 2];
#pragma unroll
        for (int i = 0; i < V8 / 2; ++i) {
          const float y0 = x[2 * i] * up, y1 = x[2 * i + 1] * up;
          h[i] = pack2<__half>(y0, y1);
          const float2 f = unpack2<__half>(h[i]);
          lo[i] = SPLIT ? pack2<__half>(y0 - f.x, y1 - f.y) : 0u;
        }
        uint8_t* at = Qs + (e >> 6) * Y::QSLAB + row * 128 + ((((e >> 3) & 7) ^ (row & 7)) << 4) + (e & 7) * 2;
        if constexpr (V8 == 8) {
          *reinterpret_cast<uint4*>(at) = make_uint4(h[0], h[1], h[2], h[3]);
        } else {
          *reinterpret_cast<uint2*>(at) = make_uint2(h[0], h[1]);
          *reinterpret_cast<uint2*>(at + Y::QPART) = make_uint2(lo[0], lo[1]);
        }
      }
    }
    fence_proxy_async_smem();
  };

  if (warp >= 4 * RT && warp < 4 * RT + 3) {
    // ---------------- converters ----------------
    if constexpr (SPLIT) reg_dec<Y::REGS_REST>();
    const int ct = threadIdx.x - Y::SOFT;
    const int log2t = c.log2t;
    // The first warp knows the blocks of 8 tiles at a time, a 16-token group per lane, and loads the next
    // 8 tiles' while it uses them up.
    const int g0 = j0 * (kN / 16);
    auto page_at = [&](int grp) {
      return grp * 16 < seen && grp < j1 * (kN / 16) ? page_of(L.s, b, (grp * 16) >> log2t) : kPastEnd;
    };
    auto scales_at = [&](int p, float& ks, float& vs) {
      ks = vs = 0.f;
      if (p >= 0 && p < c.blocks) {
        const int64_t u = (int64_t)p * c.H + hk;
        ks = c.ks[u];
        vs = c.vs[u];
      }
    };
    int page = kPastEnd, page_n = kPastEnd;
    float ks_n = 0.f, vs_n = 0.f;
    // Of the 8 tiles: the pool row of the lane's group, and over all groups (bits) those that a box starts at.
    const uint32_t box_bytes = (uint32_t)min(kN, 1 << log2t) * 2 * DT;  // K and V
    int y = 0;
    uint32_t boxes = 0;
    // Tiles n .. n + 7 after the CTA's first: where their blocks are, and (place runs before the first copies, whose
    // arrival the converters wait for) which do not exist; then their scales.
    auto place = [&](int n) {
      const bool live = page >= 0 && page < c.blocks;
      if (!live && page != kPastEnd) report_error(L.status, DEV_BAD_BLOCK, 2, page);
      const int at = 16 * (lane & 3);  // of the group in its tile
      const bool first = log2t >= 6 ? at == 0 : (at & ((1 << log2t) - 1)) == 0;  // one box per block of a tile
      y = ((page * c.H + hk) << log2t) + ((16 * (g0 + lane)) & ((1 << log2t) - 1));  // (8 tiles on: the same slot)
      boxes = __ballot_sync(0xffffffffu, live && first);
      const uint32_t dead = __ballot_sync(0xffffffffu, !live && page != kPastEnd);
      if ((lane & 3) == 0) meta[(n + (lane >> 2)) % kMeta].dead = (int32_t)(dead >> lane & 15u);
    };
    auto weigh = [&](int n, float ks, float vs) {
      const bool live = page >= 0 && page < c.blocks;
      const float av = fabsf(vs);
      const uint32_t bits = __float_as_uint(av), ex = bits >> 23;
      const bool common = av >= kScaleMin && av <= kScaleMax, parts = live && !common && ex > 0u && ex < 255u;
      TileMeta& mt = meta[(n + (lane >> 2)) % kMeta];
      mt.ks[lane & 3] = live ? ks : 1.f;  // (past the end: -inf times it stays -inf)
      mt.lv[lane & 3] = live ? log2f(parts ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : av) : 0.f;
      mt.whole[lane & 3] = (int8_t)(parts ? (int)ex - 127 : 0);
      mt.iv[lane & 3] = live ? 1.f / av : 1.f;
      const uint32_t neg = __ballot_sync(0xffffffffu, live && vs < 0.f);
      const uint32_t odd = __ballot_sync(0xffffffffu, live ? vs < 0.f || !common || !(ks > 0.f && ks <= 3.4028234e38f) : page != kPastEnd);
      if ((lane & 3) == 0) mt.neg = (int32_t)(neg >> lane & 15u), mt.odd = (int32_t)(odd >> lane & 15u);
    };
    // The blocks of the CTA's n-th tile into its raw stage: lanes w .. w + 3 know its groups.
    auto copy = [&](int n) {
      const int w = 4 * (n & 7), a = lane - w, st = n & 1;
      if (w == 0 && n > 0) {
        page = page_n;
        page_n = page_at(g0 + 4 * n + 32 + lane);
        place(n);
        weigh(n, ks_n, vs_n);
      }
      const uint32_t b4 = boxes >> w & 15u;
      __syncwarp();  // (place's stores come before the arrival)
      if (lane == 0) mbar_arrive_expect_tx(&B->raw[st], (uint32_t)__popc(b4) * box_bytes);
      __syncwarp();
      if (a >= 0 && a < 4 && (b4 >> a & 1u)) {
        uint8_t* to = base + Y::RAWS + st * 2 * Y::RAWB + 16 * a * DT;
        tc::tma_load_2d(to, &mk, 0, y, &B->raw[st]);
        tc::tma_load_2d(to + Y::RAWB, &mv, 0, y, &B->raw[st]);
      }
      if (w == 16) scales_at(page_n, ks_n, vs_n);
    };
    int loaded = min(2, j1 - j0);
    if (ct < 32) {
      page = page_at(g0 + lane);
      page_n = page_at(g0 + 32 + lane);
      place(0);
      for (int n = 0; n < loaded; ++n) copy(n);
      float ks, vs;
      scales_at(page, ks, vs);
      weigh(0, ks, vs);
    }
    constexpr int CPR = DT / 16;                                       // 16-byte pieces per row
    constexpr int PIECES = kN * CPR, NP = (PIECES + Y::CONV - 1) / Y::CONV;  // of a tile, of a thread
    // K (kv 0) or V (kv 1) of the n-th tile into its operand stage, from the registers that hold its codes.
    auto convert = [&](int n, int kv, uint4 (&w)[NP]) {
      const int st = n & 1, tok0 = (j0 + n) * kN;
      const int nrows = min(kN, (seen - tok0 + 31) & ~31);
      const uint32_t dead = FMT == kCacheE4m3 ? (uint32_t)meta[n % kMeta].dead : 0u;
      // bytes past the last token (or of a block that does not exist) may be NaN codes: zeros instead
      if (FMT == kCacheE4m3 && (tok0 + nrows > seen || dead)) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int r = (ct + i * Y::CONV) / CPR;
          if (tok0 + r >= seen || (dead >> (r >> 4) & 1)) w[i] = make_uint4(0, 0, 0, 0);
        }
      }
      if (n >= 2 && !wait_for(kv ? &B->v_empty[st] : &B->k_empty[st], ((uint32_t)(n >> 1) & 1u) ^ 1u, abort, L.status,
                              kv ? W_V_EMPTY : W_K_EMPTY, j0 + n))
        return false;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int p = ct + i * Y::CONV;
        if (p >= PIECES) break;
        const int r = p / CPR, pc = p % CPR, k = 2 * (pc & 3);
        uint8_t* dst = base + (kv ? Y::V : Y::K) + st * Y::TILE + (pc >> 2) * Y::SLAB;
        uint4 x, y;
        codes_in_order<FMT>(w[i].x, x.x, x.y);
        codes_in_order<FMT>(w[i].y, x.z, x.w);
        codes_in_order<FMT>(w[i].z, y.x, y.y);
        codes_in_order<FMT>(w[i].w, y.z, y.w);
        *reinterpret_cast<uint4*>(dst + r * 128 + ((k ^ (r & 7)) << 4)) = x;
        *reinterpret_cast<uint4*>(dst + r * 128 + (((k + 1) ^ (r & 7)) << 4)) = y;
      }
      fence_proxy_async_smem();
      mbar_arrive(kv ? &B->v_full[st] : &B->k_full[st]);
      return true;
    };
    bool ok = true;
    for (int n = 0; n < j1 - j0; ++n) {
      const int st = n & 1;
      ok = ok && wait_for(&B->raw[st], (uint32_t)(n >> 1) & 1u, abort, L.status, W_RAW, j0 + n);
      uint4 w[2][NP];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int p = ct + i * Y::CONV;
          if (p < PIECES) w[kv][i] = *reinterpret_cast<const uint4*>(base + Y::RAWS + (st * 2 + kv) * Y::RAWB + 16 * p);
        }
      ok = ok && convert(n, 0, w[0]);
      if (!(ok = bar_and(1, Y::CONV, ok))) break;  // every converter has left the raw stage
      if (loaded < j1 - j0) {
        if (ct < 32) copy(loaded);
        ++loaded;
      }
      ok = convert(n, 1, w[1]);
    }
    if (!ok && ct == 0) {  // copies in flight land before the CTA may leave
      for (int n = 0; n < loaded; ++n) mbar_wait_clocked(&B->raw[n & 1], (uint32_t)(n >> 1) & 1u, nullptr);
    }
  } else if (warp == 4 * RT + 3) {
    // ---------------- MMA issue ----------------
    if constexpr (SPLIT) reg_dec<Y::REGS_REST>();
    const uint64_t dq0 = tc::smem_desc(base + Y::Q, 16, 1024, tc::kLayoutSW128);
    const uint64_t dk = tc::smem_desc(base + Y::K, 16, 1024, tc::kLayoutSW128);
    // V is MN-major: 64-channel slabs SLAB apart (LBO), 8-token groups 1024 B apart (SBO)
    const uint64_t dv = tc::smem_desc(base + Y::V, Y::SLAB, 1024, tc::kLayoutSW128);
    auto ready = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test(bar, parity & 1u)); };
    // The scores of tile j into the S buffer of its parity, and P's product with V; each releases its
    // operand's stage.
    auto issue_s = [&](int rt, int j) {
      const int n = j - j0, st = n & 1;
      const uint64_t dq = dq0 + (uint64_t)(rt * ((Y::PARTS * Y::QPART) >> 4));
      tc::fence_after_sync();
      if (elect_one()) {
        const uint32_t id = idesc_f16(min(kN, (seen - j * kN + 31) & ~31), false);
        const uint32_t d = tmem + (uint32_t)(rt * Y::COL_RT + st * kN);
        const uint64_t dks = dk + (uint64_t)(st * (Y::TILE >> 4));
#pragma unroll
        for (int p = 0; p < Y::PARTS; ++p)
#pragma unroll
          for (int k = 0; k < DT / 16; ++k)
            mma_ss(d, dq + ((p * Y::QPART + (k >> 2) * Y::QSLAB + (k & 3) * 32) >> 4), dks + (((k >> 2) * Y::SLAB + (k & 3) * 32) >> 4),
                   id, p + k > 0);
        tc::commit(&B->s_full[rt][st]);
        tc::commit(&B->k_empty[st]);
      }
      __syncwarp();
    };
    auto issue_pv = [&](int rt, int j) {
      const int n = j - j0, st = n & 1;
      tc::fence_after_sync();
      if (elect_one()) {
        const int steps = (min(kN, seen - j * kN) + 15) >> 4;
        constexpr uint32_t id = idesc_f16(DT, true);
        const uint32_t s0 = tmem + (uint32_t)(rt * Y::COL_RT + st * kN), d = tmem + (uint32_t)rt * Y::COL_RT + Y::COL_ACC;
        const uint64_t dvs = dv + (uint64_t)(st * (Y::TILE >> 4));
#pragma unroll
        for (int k = 0; k < kN / 16; ++k) {
          if (k >= steps) break;
          const uint32_t a = s0 + 32 * (k >> 1) + 8 * (k & 1);  // P of 32 tokens: 16 columns, then its low part
          mma_ts(d, a, dvs + ((k * 2048) >> 4), id, k > 0 || (!SPLIT && (FOLD ? n % kFold : n) > 0));
          if constexpr (SPLIT) mma_ts(d, a + 16, dvs + ((k * 2048) >> 4), id, 1);
        }
        tc::commit(&B->pv_full[rt]);
        tc::commit(&B->v_empty[st]);
      }
      __syncwarp();
    };
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) bar_sync(2 + rt, 160);  // Q is in shared memory
    // Whatever is ready, for either row tile: they run at their own pace, so that one's softmax falls into the
    // other's MMAs. Scores n need K and the S buffer that P n - 2 has left, product n needs P and V.
    const int total = j1 - j0;
    int ns[RT] = {}, np[RT] = {};
    bool ok = true;
    long long t0 = clock64();
    for (int left = 2 * RT * total, idle = 0; left > 0 && ok;) {
      bool moved = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        int n = np[rt];
        if (n < ns[rt] && ready(&B->p_full[rt], n) && ready(&B->v_full[n & 1], n >> 1)) {
          issue_pv(rt, j0 + n);
          ++np[rt], --left, moved = true;
        }
        n = ns[rt];
        // (a parity tells a phase from its neighbours only: where product n - 1 is issued, P n - 1 was there,
        // whose threads had waited for product n - 2)
        if (n < total && n <= np[rt] + 1 && ready(&B->k_full[n & 1], n >> 1) && (n < 2 || np[rt] >= n || ready(&B->pv_full[rt], n - 2))) {
          issue_s(rt, j0 + n);
          ++ns[rt], --left, moved = true;
        }
      }
      if (moved) {
        idle = 0;
        t0 = clock64();
      } else if ((++idle & 63) == 0) {
        if (*abort) ok = false;
        else if (clock64() - t0 > kWaitLimitClocks) {
          if (lane == 0) report_error(L.status, DEV_TIMEOUT, W_ISSUE, left);
          *abort = 1;
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
      }
    }
    if (!ok && elect_one()) {
      // MMAs in flight end before TMEM is freed: an arrival of their own, waited for within limits
      tc::commit(&B->drain);
      mbar_wait_clocked(&B->drain, 0, nullptr);
    }
    __syncwarp();
  } else {
    // ---------------- softmax, epilogue: one row per thread ----------------
    if constexpr (SPLIT) reg_inc<Y::REGS_SOFT>();
    const int rt = warp >> 2, tr = threadIdx.x & 127;
    const int r = rt * kM + tr;  // row of the CTA
    const bool live = r < nrow;
    const int prow = r0 + min(r, nrow - 1);
    const int qi = prow / L.G;
    const int64_t head = (int64_t)(hk * L.G + prow % L.G) * c.D;
    // the last token the row sees (a row past the last one goes along with that one)
    const int lim = L.causal ? min(q.len - 1, past + qi) : q.len - 1;
    const uint32_t tl = tmem + (uint32_t)rt * Y::COL_RT + ((uint32_t)((warp & 3) * 32) << 16);  // this warp's lanes
    uint8_t* Qs = base + Y::Q + rt * Y::PARTS * Y::QPART;

    load_q(rt, (warp & 3) * 32);
    bar_sync(2 + rt, 160);  // (with the issuing warp)
    const float rs = reinterpret_cast<const float*>(base + Y::RS)[r];

    bool ok = true;
    constexpr int OR = SPLIT ? DT / 2 : 1;
    float2 o[OR];  // fp32 rows: O
#pragma unroll
    for (int e = 0; e < OR; ++e) o[e] = make_float2(0.f, 0.f);
    // 16-bit rows: O of the folds so far, in units of 2^m_kept (indexed at run time, so that it stays out of registers)
    float4 kept[FOLD ? DT / 4 : 1];
    float m_kept = -INFINITY;
    float m = -INFINITY, l = 0.f;  // l is in units of 2^(m - d) (m taken for 0 while it is -inf)
    float* unit = reinterpret_cast<float*>(base + Y::RS) + r;  // d, which only odd tiles change
    *unit = 0.f;
    bool far = false;  // some row of the warp has another unit than 2^m
    // Two values of P as words of its parts
    auto p_words = [](float2 x, uint32_t& hi, uint32_t& lo) {
      hi = pack2<__half>(x.x, x.y);
      if constexpr (SPLIT) {
        const float2 y = unpack2<__half>(hi);
        const float2 z = __ffma2_rn(y, make_float2(-1.f, -1.f), x);
        lo = pack2<__half>(z.x, z.y);
      }
    };
    auto product_done = [&](int n) {  // of the tile n after the CTA's first
      return __all_sync(0xffffffffu, wait_for(&B->pv_full[rt], (uint32_t)n & 1u, abort, L.status, W_PV, n));
    };
    auto add_product = [&] {
      tc::fence_after_sync();
#pragma unroll
      for (int e = 0; e < DT; e += 32) {
        float a[32];
        tc::tmem_ld32(tl + Y::COL_ACC + e, a);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float2& x = o[SPLIT ? e / 2 + i : 0];
          x = __fadd2_rn(make_float2(a[2 * i], a[2 * i + 1]), x);
        }
      }
    };
    // 16-bit rows: O times al, and what is kept where there is some, in units of 2^ref: kept, or at the end back into TMEM
    auto fold = [&](bool more, float al, float ref, bool last) {
      const float f = ex2f(m_kept - ref);
      tc::fence_after_sync();
#pragma unroll 1
      for (int e = 0; e < DT; e += 32) {
        float a[32];
        tc::tmem_ld32(tl + Y::COL_ACC + e, a);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float4& at = kept[FOLD ? (e + i) / 4 : 0];
          const float4 y = more ? at : make_float4(0.f, 0.f, 0.f, 0.f);
          a[i] = fmaf(y.x, f, a[i] * al), a[i + 1] = fmaf(y.y, f, a[i + 1] * al);
          a[i + 2] = fmaf(y.z, f, a[i + 2] * al), a[i + 3] = fmaf(y.w, f, a[i + 3] * al);
          if (!last) at = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
        }
        if (last) tc::tmem_st32(tl + Y::COL_ACC + e, a);
      }
      tc::tmem_wait_st();
    };
    for (int j = j0; j < j1; ++j) {
      const int n = j - j0;
      const TileMeta& mt = meta[n % kMeta];
      const int tok0 = j * kN;
      if (!(ok = __all_sync(0xffffffffu, wait_for(&B->s_full[rt][n & 1], (uint32_t)(n >> 1) & 1u, abort, L.status, W_S, j)))) break;
      tc::fence_after_sync();
      const uint32_t ts = tl + (uint32_t)((n & 1) * kN);
      constexpr int CH = Y::CHUNK;
      float s[CH];
      auto load_s = [&](int c0) {
        if constexpr (CH == 64) tc::tmem_ld64(ts, s);
        else tc::tmem_ld32(ts + c0, s);
        tc::tmem_wait_ld();
      };
      // The common tile, all of it seen by every row of the warp; one that ends for some row, whose scores
      // past the end become -inf; and an odd one, taken score by score.
      bool odd = mt.odd || L.scale_log2 == 0.f || far;
      const bool edge = !odd && !__all_sync(0xffffffffu, lim >= tok0 + kN - 1);
      // (-inf times a factor that has underflowed to 0, as rows of q that are zeros have it, would be NaN)
      if (edge) odd = __any_sync(0xffffffffu, fminf(fminf(mt.ks[0], mt.ks[1]), fminf(mt.ks[2], mt.ks[3])) * rs == 0.f);
      float mx = -INFINITY;  // the row's largest exponent
      float ref, al, sum = 0.f;
      bool moved;
      auto move = [&] {
        const float mn = SPLIT ? fmaxf(m, mx) : mx > m + kLag || m == -INFINITY ? fmaxf(m, mx) : m;
        moved = __any_sync(0xffffffffu, mn != m);
        ref = mn == -INFINITY ? 0.f : mn;
        al = ex2f(m - ref);
        m = mn;
      };
      if (!odd) {
#pragma unroll
        for (int c0 = 0; c0 < kN; c0 += CH) {
          load_s(c0);
          if (edge) {
            const int hi = lim - tok0 - c0;
#pragma unroll
            for (int e = 0; e < CH; ++e)
              if (e > hi) s[e] = -INFINITY;
          }
#pragma unroll
          for (int g = 0; g < CH / 16; ++g) {
            const float* x = s + 16 * g;
            float u = max3(x[0], x[1], x[2]), w = max3(x[3], x[4], x[5]);
#pragma unroll
            for (int e = 6; e < 14; e += 4) u = max3(u, x[e], x[e + 1]), w = max3(w, x[e + 2], x[e + 3]);
            u = max3(u, x[14], x[15]);
            mx = fmaxf(mx, fmaf(fmaxf(u, w), mt.ks[c0 / 16 + g] * rs, mt.lv[c0 / 16 + g]));
          }
        }
        move();
        // P into the columns of the scores that it comes from, and its sum
#pragma unroll
        for (int c0 = 0; c0 < kN; c0 += CH) {
          if (CH < kN) {
            load_s(c0);
            if (edge) {
              const int hi = lim - tok0 - c0;
#pragma unroll
              for (int e = 0; e < CH; ++e)
                if (e > hi) s[e] = -INFINITY;
            }
          }
#pragma unroll
          for (int h = 0; h < CH / 32; ++h) {
            uint32_t ph[16], pl[SPLIT ? 16 : 1];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int grp = c0 / 16 + 2 * h + g;
              const float k = mt.ks[grp] * rs, sh = mt.lv[grp] - ref + kPShift<SPLIT>;
              float2 part = make_float2(0.f, 0.f);
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const int i = 32 * h + 16 * g + e;
                float2 x = __ffma2_rn(make_float2(s[i], s[i + 1]), make_float2(k, k), make_float2(sh, sh));
                x.x = ex2f(x.x);
                x.y = ex2f(x.y);
                part = __fadd2_rn(part, x);
                p_words(x, ph[8 * g + (e >> 1)], pl[SPLIT ? 8 * g + (e >> 1) : 0]);
              }
              sum = fmaf(part.x + part.y, mt.iv[grp], sum);
            }
            tmem_st16(ts + c0 + 32 * h, ph);
            if constexpr (SPLIT) tmem_st16(ts + c0 + 32 * h + 16, pl);
          }
        }
        l = fmaf(l, al, sum);
      } else {
        uint64_t vis;  // the columns that the row sees
        {
          const int hi = min(max(lim - tok0 + 1, 0), kN);
          vis = hi == kN ? ~0ull : (1ull << hi) - 1ull;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (mt.dead >> g & 1) vis &= ~(0xffffull << (16 * g));
        }
        // the largest score so far: near m - d, m itself where d is 0 (within kNear and kLag)
        float d = *unit;
        const bool none = m == -INFINITY;
        const float r = none ? 0.f : m;
        float high = l != 0.f ? r - d : -INFINITY;
#pragma unroll 1
        for (int c0 = 0; c0 < kN; c0 += 32) {
          float x[32];
          tc::tmem_ld32(ts + c0, x);
          tc::tmem_wait_ld();
          const uint32_t v = (uint32_t)(vis >> c0);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int g = c0 / 16 + e / 16;
            const float k = mt.ks[g] * rs;
            if (v >> e & 1) mx = fmaxf(mx, fmaf(x[e], k, mt.lv[g] + (float)mt.whole[g])), high = fmaxf(high, x[e] * k);
          }
        }
        move();
        const float apart = ref - high;
        float dn = 0.f;
        if (high != -INFINITY && !(fabsf(apart) <= kNear)) {
          if (fabsf(apart) <= 3.4028234e38f) dn = fabsf(apart - d) <= kSlack ? d : rintf(apart);
          else l = __uint_as_float(0x7fffffffu);  // a score that is not finite
        }
        if (dn != d || none) l = l == 0.f ? 0.f : l * ex2f((r - ref) + (dn - d));
        else l *= al;
        *unit = d = dn;
        const float low = kPShift<SPLIT> - (ref - d);
#pragma unroll 1
        for (int c0 = 0; c0 < kN; c0 += 32) {
          float x[32];
          tc::tmem_ld32(ts + c0, x);
          tc::tmem_wait_ld();
          const uint32_t v = (uint32_t)(vis >> c0);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int g = c0 / 16 + h;
            const float k = mt.ks[g] * rs, sh = (((float)mt.whole[g] + kPShift<SPLIT>) - ref) + mt.lv[g];
            const bool neg = mt.neg >> g & 1;
            uint32_t ph[8], pl[8];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const int i = 16 * h + e;
              const bool a = v >> i & 1, b = v >> (i + 1) & 1;
              sum += (a ? ex2f(fmaf(x[i], k, low)) : 0.f) + (b ? ex2f(fmaf(x[i + 1], k, low)) : 0.f);
              float2 y = make_float2(a ? ex2f(fmaf(x[i], k, sh)) : 0.f, b ? ex2f(fmaf(x[i + 1], k, sh)) : 0.f);
              if (neg) y.x = -y.x, y.y = -y.y;
              p_words(y, ph[e >> 1], pl[e >> 1]);
            }
            tmem_st8(ts + c0 + 8 * h, ph);
            if constexpr (SPLIT) tmem_st8(ts + c0 + 16 + 8 * h, pl);
          }
        }
        l += sum;
        far = __any_sync(0xffffffffu, d != 0.f || (m == -INFINITY && l > 0.f));  // (not for rows of NaN)
      }
      // Every product is waited for in its turn, needed or not: a wait by parity tells a phase only from its
      // neighbours. (This one could not start before the last one's end.)
      if (n > 0) ok = product_done(n - 1);
      if (FOLD && n > 0 && n % kFold == 0) {
        if (ok) fold(n > kFold, al, ref, false);
        m_kept = m;
      } else if (n > 0 && (SPLIT || moved)) {
        // fp32 rows: the previous product joins O. Either: O follows m.
        if (SPLIT && ok) add_product();
        if (moved && ok) {
          if constexpr (SPLIT) {
#pragma unroll
            for (int e = 0; e < OR; ++e) o[e] = __fmul2_rn(o[e], make_float2(al, al));
          } else {
            tc::fence_after_sync();
#pragma unroll 1
            for (int e = 0; e < DT; e += 32) {
              float a[32];
              tc::tmem_ld32(tl + Y::COL_ACC + e, a);
              tc::tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) a[i] *= al;
              tc::tmem_st32(tl + Y::COL_ACC + e, a);
            }
          }
        }
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      if (!ok) break;
      mbar_arrive(&B->p_full[rt]);
    }
    if (ok && j0 < j1) {
      ok = product_done(j1 - j0 - 1);
      tc::fence_after_sync();
      if (SPLIT && ok) add_product();
      if (FOLD && ok && j1 - j0 > kFold) fold(true, 1.f, m == -INFINITY ? 0.f : m, true);
    }
    // ---- epilogue: the row through shared memory (its own Q rows), stored in whole 16-byte pieces ----
    // 32 channels of the row's O
    auto channels = [&](int e, float (&x)[32]) {
      if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[2 * i] = o[e / 2 + i].x, x[2 * i + 1] = o[e / 2 + i].y;
      } else if (j0 < j1 && ok) {
        tc::tmem_ld32(tl + Y::COL_ACC + e, x);
        tc::tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = 0.f;
      }
    };
    // O is in units of 2^m, l of 2^(m - d): what O has to be multiplied by, as two factors that are in range (where m is
    // -inf, O is 0 or NaN)
    float ref = m == -INFINITY ? 0.f : m, up0 = 1.f, up1 = 1.f;
    if (far && *unit != 0.f) {
      float by = *unit;
      ref -= by;
      if (L.ws_o) {  // with l's own power of two, so that O is as large as the part's output
        const int ex = l > 0.f && l <= 3.4028234e38f ? ilogbf(l) : 0;
        l = scalbnf(l, -ex);
        ref += (float)ex;
        by -= (float)ex;
      }
      if (m != -INFINITY) {
        const float half = rintf(0.5f * by);
        up0 = ex2f(half), up1 = ex2f(by - half);
      }
    }
    if (L.ws_o) {
      const int64_t at = (int64_t)blockIdx.x * (kM * RT) + r;
#pragma unroll
      for (int e = 0; e < DT; e += 32) {
        float x[32];
        channels(e, x);
        if (far) {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = x[i] * up0 * up1;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          if (live && e + i < c.D) *reinterpret_cast<float4*>(L.ws_o + at * c.D + e + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      }
      if (live) L.ws_ml[at] = make_float2(l == 0.f ? -INFINITY : ref, l);
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint8_t* mine = Qs + tr * (PER * 16);
#pragma unroll
      for (int e = 0; e < DT; e += 32) {
        float x[32];
        channels(e, x);
        if (far) {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = x[i] * inv * up0 * up1;
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] *= inv;
        }
#pragma unroll
        for (int i = 0; i < 32; i += V8) {
          float y[V8];
#pragma unroll
          for (int k = 0; k < V8; ++k) y[k] = l == 0.f ? 0.f : x[i + k];
          const int p = (e + i) / V8;
          store_row<T, V8, true>(reinterpret_cast<T*>(mine + ((p ^ (tr & 7)) << 4)), y);
        }
      }
      __syncwarp();
      const int per = c.D / V8;  // pieces that exist
      // each row's address is known to its own thread
      T* mine_out = live ? static_cast<T*>(L.o) + (q.row0 + qi) * L.ldo + head : nullptr;
#pragma unroll 4
      for (int i = 0; i < 32; i += RPI) {
        const int rl = i + lane / PER, p = lane % PER;
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

template <typename T, int FMT, int DT, bool FOLD>
cudaError_t tc_as(const CacheAttnLaunch& L, const CacheAttnPlan& P, cudaStream_t s) {
  using Y = Cfg<DT, sizeof(T) == 4>;
  auto kernel = cache_attn_tc_kernel<T, FMT, DT, FOLD>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = once_per_device(done, L.device, [&] {
    if constexpr (sizeof(T) == 4) {
      cudaFuncAttributes fa;
      const cudaError_t r = cudaFuncGetAttributes(&fa, kernel);
      if (r != cudaSuccess) return r;
      // the exchange of registers has to add up, whatever the compiler has given the kernel (Y::REGS, as a rule)
      if (fa.numRegs < Y::REGS_REST || fa.numRegs > Y::REGS_SOFT || Y::SOFT * Y::REGS_SOFT + 128 * Y::REGS_REST > Y::THREADS * fa.numRegs)
        return cudaErrorInvalidKernelImage;
    }
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Y::SMEM);
  });
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)(P.units * P.splits), Y::THREADS, Y::SMEM, s>>>(L, L.mk, L.mv, P.tiles);
  return cudaGetLastError();
}
template <typename T, bool FOLD>
cudaError_t tc_fold(const CacheAttnLaunch& L, const CacheAttnPlan& P, int format, cudaStream_t s) {
  if (L.c.D <= 64) return format == kCacheInt8 ? tc_as<T, kCacheInt8, 64, FOLD>(L, P, s) : tc_as<T, kCacheE4m3, 64, FOLD>(L, P, s);
  return format == kCacheInt8 ? tc_as<T, kCacheInt8, 128, FOLD>(L, P, s) : tc_as<T, kCacheE4m3, 128, FOLD>(L, P, s);
}
template <typename T>
cudaError_t tc_type(const CacheAttnLaunch& L, const CacheAttnPlan& P, int format, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    const int64_t tiles = (L.s.max_len + kN - 1) / kN;
    if ((tiles + P.splits - 1) / P.splits > kFold) return tc_fold<T, true>(L, P, format, s);
  }
  return tc_fold<T, false>(L, P, format, s);
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
