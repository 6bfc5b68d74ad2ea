// Attention of few query rows over the paged 8-bit K/V cache (steps of single tokens, short drafts).
//
//   s_ij = scale * k_scale[block(j), h] * (q_i . code_j),  p_ij = exp2(s_ij - m_i)
//   o_i  = sum_j p_ij v_scale[block(j), h] code'_j / sum_j p_ij
// The cache's bytes are the bound: each is read from HBM once for all query rows that share its head,
// and turned into 16-bit floats on the way to the tensor cores (mma.sync m16n8k16: the tile is 8
// query rows wide, which the 128-row tcgen05 tile would pad 16-fold, and the tensor pipe is not
// what bounds this kernel). Scores are formed transposed, S^T = K Q^T with tokens as the 16 rows of
// the MMA, so that 8 query rows fill its 8 columns; P^T is turned in registers (movmatrix) into the B
// operand of O^T += V^T P^T, and a row's statistics and its column of O^T live in the same lanes.
// Codes are exact in fp16; the per-block scales multiply the scores and each block's partial sum in
// fp32, which also keeps the long sum over blocks in fp32 registers, rounded to nearest.
// q is multiplied by a power of two per row (its largest channel lands in [2^13, 2^14)) and rounded to
// fp16, which is exact for bf16 and fp16 rows down to 2^-27 of their largest channel. fp32 rows use two
// fp16 parts, hi + lo (22 bits), and so does p; each product is then two MMAs.
//
// One warp walks over a contiguous range of 32-token tiles, fed by its own ring of TMA stages: a tile of K
// or V is one box of the pool seen as [blocks * H * block_tokens, D] bytes (two boxes for 16-token
// blocks), swizzled so that ldmatrix meets no bank conflicts, its channels past D filled with zeros. 4
// warps form a CTA and 1 to 16 CTAs a cluster that splits one (sequence, cache head, 8 or 16 query
// rows). The cluster joins its parts through distributed shared memory: no workspace, no atomics, the
// same order every time. Where so few units meet so long a cache that 16 CTAs each leave SMs idle, the
// CTAs are launched without clusters, as many as fill the SMs, write their parts to a workspace that
// lives from the launch to the join, and a second kernel joins them in order.
//
// Measured: 64 sequences of 1000 to 8000 tokens, 8 heads of 128, 4 query heads each, E4M3 and bf16: 120 us, 4.9 TB/s (75 %
// of the copy rate; what is missing is the first loads of each CTA, three of which share an SM, and the last
// wave); one sequence of 131072 tokens, INT8 and fp16: 54 us, 5.0 TB/s (49 for the
// parts, 5.5 TB/s; the join, placed while they are formed, the rest: 57 in all when it was an ordinary launch).
#include <cooperative_groups.h>

#include <algorithm>

#include "cache.cuh"
#include "tcgen05.cuh"

namespace supra {
namespace {

constexpr int kTile = 32;  // tokens of a warp's tile
constexpr int kStages = 2;
constexpr float kPShift = 12.f;  // p is formed as 2^12 p: its fp16 part keeps 2^-24 of p = 1 at 2^-12
// l and O carry that factor up to the join, so that V scales near 2^-126 lose nothing; a warp that meets one above
// 2^90 takes it off at once, lest O pass the range of 32 bits.
constexpr float kPUnit = 1.f / 4096.f, kScaleLarge = 1.2379400392853803e27f;

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// d = a b, without an accumulator to clear
__device__ __forceinline__ void mma0(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// Codes of one word as fp16 pairs: bytes 0 and 2, bytes 1 and 3.
__device__ __forceinline__ void e4m3x4(uint32_t u, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(u));
}
template <int FMT>
__device__ __forceinline__ void codes4(uint32_t u, uint32_t& even, uint32_t& odd) {
  if constexpr (FMT == kCacheInt8) {
    // 0x64 above a byte b is the fp16 number 1024 + b; with b = code + 128, 1152 off gives the code
    // (masking and shifting, which takes both constants apart, came to five operations a word, this to three)
    const uint32_t x = u ^ 0x80808080u;
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4240), b = __byte_perm(x, 0x64646464u, 0x4341);
    const uint32_t off = 0x64806480u;
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&off));
    const __half2 hb = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&off));
    even = *reinterpret_cast<const uint32_t*>(&ha);
    odd = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    e4m3x4(__byte_perm(u, 0, 0x3120), even, odd);
  }
}
// The same for operands whose order along the product is free (K, with q's channels in the same order):
// INT8 as above, E4M3 bytes 0 and 1, bytes 2 and 3, which need no reordering.
template <int FMT>
__device__ __forceinline__ void codes4_any(uint32_t u, uint32_t& a, uint32_t& b) {
  if constexpr (FMT == kCacheInt8) codes4<FMT>(u, a, b);
  else e4m3x4(u, a, b);
}

// What a warp knows of a 16-token group of its tile: the K and V scale, and whether its block exists.
struct Group {
  float ks, vs;
  int32_t dead, pad;
};

constexpr int stage_bytes(int DT) { return 2 * kTile * DT; }
// Shared memory of a warp besides its stages: a barrier and two groups per stage.
constexpr int kWarpBytes = kStages * (8 + 2 * (int)sizeof(Group));

// Byte offset in a tile (rows of DT bytes) of 16-byte chunk 0 of row r, as the TMA unit swizzles it:
// 128-byte rows permute their chunks by r % 8, 64-byte rows by (r / 2) % 4. Chunk k is at ^ (16 k).
template <int DT>
__device__ __forceinline__ uint32_t chunk0_at(int r) {
  return (uint32_t)(r * DT + ((DT == 128 ? r & 7 : (r >> 1) & 3) << 4));
}

// DT: head dim rounded up to 64 or 128 (the channels between are zero: no branches among the MMAs). NT: groups of 8 query rows. SPLIT: two fp16 parts of q and p. ONE: blocks of at least 32
// tokens, so that a tile has one pair of scales. W: warps.
template <typename T, int FMT, int DT, int NT, bool ONE, int W>
__global__ void __launch_bounds__(W * 32, W == 4 && NT == 1 ? 3 : 1) cache_attn_kernel(const __grid_constant__ CacheAttnArgs L, const __grid_constant__ CUtensorMap mk,
                                                            const __grid_constant__ CUtensorMap mv, int tiles) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int CH = DT / 16;  // 16-channel chunks
  constexpr int NR = 8 * NT;
  namespace cg = cooperative_groups;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // swizzle atoms
  const CachePool& c = L.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  cg::cluster_group cluster = cg::this_cluster();
  if (L.ws_o) join_may_start();
  const int csize = L.splits, crank = blockIdx.x % csize;  // (the rank in the cluster, where there is one)

  // unit = (sequence, cache head, row tile); the whole cluster has the same one
  int unit = blockIdx.x / csize;
  const int rt = unit % tiles;
  unit /= tiles;
  const int hk = unit % c.H, b = unit / c.H;
  SeqView q;
  if (!seq_view(L.s, b, false, L.status, q)) return;
  const int rows = q.n * L.G;  // packed (query, head of the group)
  const int r0 = rt * NR;
  if (r0 >= rows) return;
  const int nrow = min(NR, rows - r0);
  // tokens that some row of this tile sees
  const int past = q.len - q.n;  // causal: query i sees tokens 0 .. past + i
  const int i_last = (r0 + nrow - 1) / L.G, i_first = r0 / L.G;
  const int seen = L.causal ? max(0, min(q.len, past + i_last + 1)) : q.len;
  const int all = L.causal ? max(0, min(q.len, past + i_first + 1)) : q.len;  // every row sees these

  constexpr int tile_bytes = kTile * DT, sbytes = stage_bytes(DT);
  const int D = c.D, ch = D >> 4;
  uint8_t* ring = smem + warp * kStages * sbytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + W * kStages * sbytes) + warp * kStages;
  Group* groups = reinterpret_cast<Group*>(smem + W * kStages * (sbytes + 8)) + warp * kStages * 2;
  if (lane < kStages) mbar_init(full + lane, 1);
  mbar_fence_init();
  __syncwarp();

  // ---- this warp's tiles ----
  const int nt = (seen + kTile - 1) / kTile;
  const int parts = csize * W, part = crank * W + warp;
  const int share = nt / parts, extra = nt % parts;
  const int t0 = part * share + min(part, extra);
  const int cnt = share + (part < extra ? 1 : 0);

  // Blocks of the next 16-token groups, one group per lane: the set in use, and the next one, whose
  // loads are under way while the first is used up.
  const int log2t = c.log2t;
  auto page_at = [&](int grp) {  // grp: 16-token group of the sequence
    return grp * 16 < seen ? page_of(L.s, b, (grp * 16) >> log2t) : kPastEnd;
  };
  auto scales_at = [&](int p, float& ks, float& vs) {
    ks = vs = 0.f;
    if (p >= 0 && p < c.blocks) {
      const int64_t u = (int64_t)p * c.H + hk;
      ks = c.ks[u];
      vs = c.vs[u];
    }
  };
  int page = page_at(2 * t0 + lane), page_n = page_at(2 * t0 + 32 + lane);
  float ks, vs, ks_n = 0.f, vs_n = 0.f;
  // The warp's tile i into its stage: the lanes that know its groups load them (both by one, when they are
  // in one block), and describe them; a block outside the cache is not loaded.
  auto copy = [&](int i) {
    if (i >= cnt) return;
    const int w = i & 15, st = i % kStages;
    if (w == 0 && i > 0) {
      page = page_n, ks = ks_n, vs = vs_n;
      page_n = page_at(2 * (t0 + i) + 32 + lane);
    }
    if (w == 8) scales_at(page_n, ks_n, vs_n);
    const int a = lane - 2 * w;
    const bool mine = a == 0 || a == 1;
    const bool dead = page < 0 || page >= c.blocks;
    const uint32_t live = __ballot_sync(0xffffffffu, (ONE ? a == 0 : mine) && !dead);
    constexpr int box = ONE ? kTile : 16;
    if (lane == 0) mbar_arrive_expect_tx(full + st, (uint32_t)(__popc(live) * 2 * box * DT));
    __syncwarp();
    if (live >> lane & 1) {
      const int tok = (t0 + i) * kTile + 16 * a;
      const int y = ((page * c.H + hk) << log2t) + (tok & ((1 << log2t) - 1));
      uint8_t* to = ring + st * sbytes + 16 * a * DT;
      tc::tma_load_2d(to, &mk, 0, y, full + st);
      tc::tma_load_2d(to + tile_bytes, &mv, 0, y, full + st);
    }
  };
  auto describe = [&](int i) {
    if (i >= cnt) return;
    const int a = lane - 2 * (i & 15);
    if (a == 0 || a == 1) {
      const bool dead = page < 0 || page >= c.blocks;
      Group* gr = groups + (i % kStages) * 2 + a;
      gr->ks = ks, gr->vs = vs, gr->dead = dead;
      if (dead && page != kPastEnd) report_error(L.status, DEV_BAD_BLOCK, 1, page);
    }
  };
  // the first copies go out before q and the scales are fetched
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) copy(i);
  scales_at(page, ks, vs);

  // ---- q fragments: lane (g, t) holds channels 16 k + 4 t .. + 3 of row g of each row group, paired
  // as codes4_any pairs K's ----
  constexpr int P1 = FMT == kCacheInt8 ? 2 : 1;  // the channel beside the first
  uint32_t qh[NT][CH][2], ql[SPLIT ? NT : 1][SPLIT ? CH : 1][2];
  float rs[NT][2];   // score factor of rows 2t, 2t + 1
  int lim[NT][2];    // last token that they see
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float x[CH][4];
    float top = 0.f;
    const int r = 8 * n + g;
    const bool live = r < nrow;
    const int pr = r0 + min(r, nrow - 1);
    const T* src = static_cast<const T*>(L.q) + (q.row0 + pr / L.G) * L.ldq + (int64_t)(hk * L.G + pr % L.G) * D;
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[k][e] = live && k < ch ? to_f32<T>(src[16 * k + 4 * t + e]) : 0.f;
        top = fmaxf(top, fabsf(x[k][e]));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^(13 - exponent of top), kept inside the fp32 range at both ends
    const int ex = min(max((int)(__float_as_uint(top) >> 23), 27), 254) - 127;
    const float up = __uint_as_float((uint32_t)(13 - ex + 127) << 23);
    const float down = __uint_as_float((uint32_t)(ex - 13 + 127) << 23);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[k][e] *= up;
      qh[n][k][0] = pack2<__half>(x[k][0], x[k][P1]);
      qh[n][k][1] = pack2<__half>(x[k][3 - P1], x[k][3]);
      if constexpr (SPLIT) {
        const float2 a = unpack2<__half>(qh[n][k][0]), d = unpack2<__half>(qh[n][k][1]);
        ql[n][k][0] = pack2<__half>(x[k][0] - a.x, x[k][P1] - a.y);
        ql[n][k][1] = pack2<__half>(x[k][3 - P1] - d.x, x[k][3] - d.y);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      rs[n][e] = L.scale_log2 * __shfl_sync(0xffffffffu, down, (2 * t + e) * 4);
      const int rr = min(8 * n + 2 * t + e, nrow - 1);
      lim[n][e] = L.causal ? min(q.len - 1, past + (r0 + rr) / L.G) : q.len - 1;
    }
  }

#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) describe(i);

  float o[CH][NT][4];
  float m[NT][2], l[NT][2];
  float carry = 1.f;  // 1: l and O are 2^12 times what they stand for; kPUnit: they are not
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.f;
#pragma unroll
  for (int k = 0; k < CH; ++k)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[k][n][e] = 0.f;

  bool lost = false;
  int lost_at = 0;
  for (int i = 0; i < cnt; ++i) {
    const int stg = i % kStages;
    if (!mbar_wait_clocked(full + stg, (uint32_t)(i / kStages) & 1u, nullptr)) {
      if (lane == 0) report_error(L.status, DEV_TIMEOUT, 70, i);
      lost = true, lost_at = i;
      break;
    }
    __syncwarp();
    copy(i + kStages - 1);  // into the stage that the previous tile has left
    describe(i + kStages - 1);
    const Group* gr = groups + stg * 2;
    const uint32_t kb = smem_u32(ring + stg * sbytes) + chunk0_at<DT>(lane), vb = kb + (uint32_t)tile_bytes;
    const int tok0 = (t0 + i) * kTile;

    // S^T: two 16-token groups
    float s[2][NT][4];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      uint32_t u[4];  // tokens 0-7, 8-15 of the first and the second group, channels 16 k ..
      ldsm4(u, kb ^ (uint32_t)(16 * k));
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        uint32_t f[4];
        codes4_any<FMT>(u[2 * a], f[0], f[2]);
        codes4_any<FMT>(u[2 * a + 1], f[1], f[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (k == 0) mma0(s[a][n], f, qh[n][k]);
          else mma(s[a][n], f, qh[n][k]);
          if constexpr (SPLIT) mma(s[a][n], f, ql[n][k]);
        }
      }
    }
    const float ks0 = gr[0].ks, ks1 = gr[1].ks;
    const bool partial = tok0 + kTile > all || gr[0].dead || gr[1].dead;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[0][n][e] *= ks0 * rs[n][e & 1];
        s[1][n][e] *= (ONE ? ks0 : ks1) * rs[n][e & 1];
      }
    if (partial) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (gr[a].dead || tok0 + 16 * a + 8 * (e >> 1) + g > lim[n][e & 1]) s[a][n][e] = -INFINITY;
    }
    // row maxima over the tile, statistics, P
    float al[NT][2];
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(fmaxf(s[0][n][e], s[0][n][e + 2]), fmaxf(s[1][n][e], s[1][n][e + 2]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        const float mn = fmaxf(m[n][e], x);
        const float ref = (mn == -INFINITY ? 0.f : mn) - kPShift;
        al[n][e] = ex2f(m[n][e] - kPShift - ref);
        moved = moved || mn != m[n][e];
        m[n][e] = mn;
        float sum = 0.f;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            s[a][n][e + 2 * y] = ex2f(s[a][n][e + 2 * y] - ref);
            sum += s[a][n][e + 2 * y];
          }
        l[n][e] = fmaf(l[n][e], al[n][e], sum * carry);
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[k][n][e] *= al[n][e & 1];
    }
    uint32_t ph[2][NT][2], pl[SPLIT ? 2 : 1][SPLIT ? NT : 1][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float x0 = s[a][n][2 * y], x1 = s[a][n][2 * y + 1];
          const uint32_t hi = pack2<__half>(x0, x1);
          if constexpr (SPLIT) {
            const float2 f = unpack2<__half>(hi);
            pl[a][n][y] = movm(pack2<__half>(x0 - f.x, x1 - f.y));
          }
          ph[a][n][y] = movm(hi);
        }
    // O^T += vscale * (V^T P^T), each block's part from a fresh accumulator
    const float vs0 = gr[0].vs, vs1 = gr[1].vs;
    if (carry == 1.f && fmaxf(fabsf(vs0), fabsf(vs1)) > kScaleLarge) {
      carry = kPUnit;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        l[n][0] *= carry, l[n][1] *= carry;
#pragma unroll
        for (int k = 0; k < CH; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[k][n][e] *= carry;
      }
    }
    // A block whose scale is not finite reaches only the rows that see it: the others' p and partial sum
    // are 0, and so is their factor.
    const bool odd = !(fabsf(vs0) <= 3.4028234e38f) || !(fabsf(vs1) <= 3.4028234e38f);
    float vf[ONE ? 1 : 2][NT][2];
#pragma unroll
    for (int a = 0; a < (ONE ? 1 : 2); ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) vf[a][n][e] = odd && tok0 + 16 * a > lim[n][e] ? 0.f : (a ? vs1 : vs0) * carry;
    // Bytes after the last token may be anything, NaN codes among them, and 0 * NaN is not 0: the lane's
    // tokens 2t, 2t + 1 of each eight are the halves of its words.
    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
    const bool cut = FMT == kCacheE4m3 && (tok0 + kTile > seen || gr[0].dead || gr[1].dead);
    if (cut) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = tok0 + 8 * j + 2 * t;
        keep[j] = gr[j >> 1].dead ? 0u : (tok < seen ? 0xffffu : 0u) | (tok + 1 < seen ? 0xffff0000u : 0u);
      }
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float acc[NT][4];
      uint32_t u[4];  // as for K, transposed: the lane has tokens 2t, 2t + 1 of each eight and channels 2g,
                      // 2g + 1 of the chunk, which are rows g and g + 8 of the MMA
      ldsm4t(u, vb ^ (uint32_t)(16 * k));
      if (cut) {
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] &= keep[j];
      }
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        uint32_t f[4];
        codes4<FMT>(u[2 * a], f[0], f[1]);
        codes4<FMT>(u[2 * a + 1], f[2], f[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (a == 0 || !ONE) mma0(acc[n], f, ph[a][n]);
          else mma(acc[n], f, ph[a][n]);
          if constexpr (SPLIT) mma(acc[n], f, pl[a][n]);
        }
        if (a == 1 || !ONE) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k][n][e] = fmaf(vf[ONE ? 0 : a][n][e & 1], acc[n][e], o[k][n][e]);
        }
      }
    }
  }
  // (every copy has landed: each was waited for, but after a wait that ran out, when those in flight are
  // given their time before the ring is used again)
  if (lost) {
    for (int i = lost_at; i < min(cnt, lost_at + kStages); ++i) mbar_wait_clocked(full + i % kStages, (uint32_t)(i / kStages) & 1u, nullptr);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
      l[n][e] *= kPUnit / carry;
    }
  __syncthreads();  // every warp has left its ring

  // ---- join: the CTA's warps, then the cluster's CTAs ----
  // shared memory: O of each warp [W][NR][DT], then (m, l) [W][NR]; the CTA's own sums
  // [NR][DT] and (m, l) [NR] follow
  float* wo = reinterpret_cast<float*>(smem);
  float2* wml = reinterpret_cast<float2*>(wo + W * NR * DT);
  float* co = reinterpret_cast<float*>(wml + W * NR);
  float2* cml = reinterpret_cast<float2*>(co + NR * DT);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        wo[(warp * NR + 8 * n + 2 * t + (e & 1)) * DT + 16 * k + 2 * g + (e >> 1)] = o[k][n][e] * (kPUnit / carry);
    if (g == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) wml[warp * NR + 8 * n + 2 * t + e] = make_float2(m[n][e], l[n][e]);
    }
  }
  __syncthreads();
  T* out = static_cast<T*>(L.o);
  auto store = [&](int r, int d, float x) {
    const int pr = r0 + r;
    out[(q.row0 + pr / L.G) * L.ldo + (int64_t)(hk * L.G + pr % L.G) * D + d] = from_f32<T>(x);
  };
  for (int idx = threadIdx.x; idx < nrow * D; idx += W * 32) {
    const int r = idx / D, d = idx - r * D;
    float mx = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, wml[w * NR + r].x);
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float2 ml = wml[w * NR + r];
      const float f = ex2f(ml.x - ref);
      sum = fmaf(ml.y, f, sum);
      x = fmaf(wo[(w * NR + r) * DT + d], f, x);
    }
    if (csize == 1) {
      store(r, d, sum == 0.f ? 0.f : x / sum);
    } else if (L.ws_o) {
      const int64_t at = (int64_t)blockIdx.x * NR + r;
      L.ws_o[at * D + d] = x;
      if (d == 0) L.ws_ml[at] = make_float2(mx, sum);
    } else {
      co[r * DT + d] = x;
      if (d == 0) cml[r] = make_float2(mx, sum);
    }
  }
  if (csize > 1 && !L.ws_o) {
    cluster.sync();
    for (int idx = crank * W * 32 + threadIdx.x; idx < nrow * D; idx += csize * W * 32) {
      const int r = idx / D, d = idx - r * D;
      float mx = -INFINITY, sum = 0.f, x = 0.f;
      for (int k = 0; k < csize; ++k) mx = fmaxf(mx, cluster.map_shared_rank(cml, k)[r].x);
      const float ref = mx == -INFINITY ? 0.f : mx;
      for (int k = 0; k < csize; ++k) {
        const float2 ml = cluster.map_shared_rank(cml, k)[r];
        const float f = ex2f(ml.x - ref);
        sum = fmaf(ml.y, f, sum);
        x = fmaf(cluster.map_shared_rank(co, k)[r * DT + d], f, x);
      }
      store(r, d, sum == 0.f ? 0.f : x / sum);
    }
    cluster.sync();  // no CTA leaves while another reads its shared memory
  }
}

constexpr int kMaxSplits = 444;  // (one wave of three CTAs per SM)

// The row of the workspace's unit and tile that a join works on: its first part, and where it belongs.
struct JoinRow {
  int64_t part0;
  int64_t out;  // element of its first channel
};
__device__ __forceinline__ bool join_row(const CacheAttnArgs& L, int tiles, int NR, bool last_first, int unit, int r, JoinRow& j) {
  const CachePool& c = L.c;
  j.part0 = (int64_t)unit * L.splits * NR + r;
  // (the tensor-core kernel orders its units by row tile, the last ones first)
  const int heads = L.s.B * c.H;
  const int rt = last_first ? tiles - 1 - unit / heads : unit % tiles;
  unit = last_first ? unit % heads : unit / tiles;
  const int hk = unit % c.H, b = unit / c.H;
  SeqView q;
  if (!seq_view(L.s, b, false, L.status, q)) return false;
  const int pr = rt * NR + r;
  if (pr >= q.n * L.G) return false;
  j.out = (q.row0 + pr / L.G) * L.ldo + (int64_t)(hk * L.G + pr % L.G) * c.D;
  return true;
}

// Joins the workspace's parts of one row of one unit, always in the same order, where there are few rows and
// many parts: the weights of all parts first, then 256 / (D / 4) groups of threads (4 channels each) add up every
// so many-th part, and the groups are added up.
template <typename T>
__global__ void __launch_bounds__(256) cache_attn_join(const __grid_constant__ CacheAttnArgs L, int tiles, int NR) {
  __shared__ float wt[kMaxSplits];
  __shared__ float red[16];
  __shared__ float4 po[256];
  const CachePool& c = L.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  JoinRow row;
  const bool there = join_row(L, tiles, NR, false, blockIdx.x, blockIdx.y, row);  // (reads what no launch of ours writes)
  parts_done();
  if (!there) return;
  const int64_t part0 = row.part0;
  const int per = c.D / 4, groups = 256 / per;
  const int g = threadIdx.x / per, e = (threadIdx.x - g * per) * 4;
  auto part_of = [&](int s) { return *reinterpret_cast<const float4*>(L.ws_o + (part0 + (int64_t)s * NR) * c.D + e); };
  float4 first[8];  // under way while the weights are worked out
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int s = g + k * groups;
    first[k] = g < groups && s < L.splits ? part_of(s) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float mx = -INFINITY, m[2], l[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = threadIdx.x + 256 * i;
    const float2 ml = s < L.splits ? L.ws_ml[part0 + (int64_t)s * NR] : make_float2(-INFINITY, 0.f);
    m[i] = ml.x, l[i] = ml.y;
    mx = fmaxf(mx, ml.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) red[warp] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) mx = fmaxf(mx, red[w]);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float f = ex2f(m[i] - ref);
    if (threadIdx.x + 256 * i < L.splits) wt[threadIdx.x + 256 * i] = f;
    sum = fmaf(l[i], f, sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[8 + warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += red[8 + w];
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (g < groups) {
    auto add = [&](const float4& v, float f) {
      x.x = fmaf(v.x, f, x.x), x.y = fmaf(v.y, f, x.y), x.z = fmaf(v.z, f, x.z), x.w = fmaf(v.w, f, x.w);
    };
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (g + k * groups < L.splits) add(first[k], wt[g + k * groups]);
#pragma unroll 8
    for (int s = g + 8 * groups; s < L.splits; s += groups) add(part_of(s), wt[s]);
  }
  po[threadIdx.x] = x;
  __syncthreads();
  if (threadIdx.x >= c.D) return;
  const int d = threadIdx.x;
  float y = 0.f;
  for (int k = 0; k < groups; ++k) y += reinterpret_cast<const float*>(po + k * per)[d];
  static_cast<T*>(L.o)[row.out + d] = from_f32<T>(sum == 0.f ? 0.f : y / sum);
}

// The same where there are many rows: one row a warp, its parts' statistics 32 at a time in its lanes.
template <typename T>
__global__ void __launch_bounds__(256) cache_attn_join_rows(const __grid_constant__ CacheAttnArgs L, int tiles, int NR) {
  const CachePool& c = L.c;
  const int lane = threadIdx.x & 31;
  JoinRow row;
  const bool there = join_row(L, tiles, NR, true, blockIdx.x, blockIdx.y * 8 + (threadIdx.x >> 5), row);  // (of whole warps)
  parts_done();
  if (!there) return;
  auto part = [&](int s) { return s < L.splits ? L.ws_ml[row.part0 + (int64_t)s * NR] : make_float2(-INFINITY, 0.f); };
  float mx = -INFINITY;
  for (int s0 = 0; s0 < L.splits; s0 += 32) mx = fmaxf(mx, part(s0 + lane).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float ref = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool on = 4 * lane < c.D;
  for (int s0 = 0; s0 < L.splits; s0 += 32) {
    const float2 ml = part(s0 + lane);
    const float f = ex2f(ml.x - ref);
    sum = fmaf(ml.y, f, sum);
    const int n = min(32, L.splits - s0);
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
      const float w = __shfl_sync(0xffffffffu, f, k);
      if (on) {
        const float4 v = *reinterpret_cast<const float4*>(L.ws_o + (row.part0 + (int64_t)(s0 + k) * NR) * c.D + 4 * lane);
        x.x = fmaf(v.x, w, x.x), x.y = fmaf(v.y, w, x.y), x.z = fmaf(v.z, w, x.z), x.w = fmaf(v.w, w, x.w);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (!on) return;
  const float y[4] = {x.x / sum, x.y / sum, x.z / sum, x.w / sum};
  T* to = static_cast<T*>(L.o) + row.out + 4 * lane;
#pragma unroll
  for (int e = 0; e < 4; ++e) to[e] = from_f32<T>(sum == 0.f ? 0.f : y[e]);
}

template <int NT, int W>
constexpr size_t smem_of(int DT) {
  const size_t ring = (size_t)W * (kStages * stage_bytes(DT) + kWarpBytes);
  const size_t join = (size_t)(W + 1) * (8 * NT) * (DT * sizeof(float) + sizeof(float2));
  return (ring > join ? ring : join) + 1024;  // (the base is moved to a 1024-byte boundary)
}

constexpr int kW = 4;  // warps of a CTA

template <typename T, int FMT, int DT, int NT, bool ONE>
cudaError_t attn_as(const CacheAttnLaunch& L, const CacheAttnPlan& P, cudaStream_t s) {
  auto kernel = cache_attn_kernel<T, FMT, DT, NT, ONE, kW>;
  constexpr size_t smem = smem_of<NT, kW>(DT);
  static_assert(smem <= 227 * 1024, "shared memory");
  const int cluster = P.ws_bytes ? 1 : P.splits;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = once_per_device(done, L.device, [&] {
    const cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    return r != cudaSuccess ? r : cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(P.units * P.splits));
  cfg.blockDim = dim3(kW * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const CacheAttnArgs& A = L;
  e = cudaLaunchKernelEx(&cfg, kernel, A, L.mk, L.mv, P.tiles);
  return e;
}

template <typename T, int FMT, int DT, int NT>
cudaError_t attn_nt(const CacheAttnLaunch& L, const CacheAttnPlan& P, cudaStream_t s) {
  return L.c.log2t >= 5 ? attn_as<T, FMT, DT, NT, true>(L, P, s) : attn_as<T, FMT, DT, NT, false>(L, P, s);
}
template <typename T, int FMT>
cudaError_t attn_fmt(const CacheAttnLaunch& L, const CacheAttnPlan& P, cudaStream_t s) {
  if (L.c.D <= 64) return P.nr == 16 ? attn_nt<T, FMT, 64, 2>(L, P, s) : attn_nt<T, FMT, 64, 1>(L, P, s);
  return P.nr == 16 ? attn_nt<T, FMT, 128, 2>(L, P, s) : attn_nt<T, FMT, 128, 1>(L, P, s);
}
template <typename T>
cudaError_t attn_type(const CacheAttnLaunch& L, const CacheAttnPlan& P, int format, cudaStream_t s) {
  return format == kCacheInt8 ? attn_fmt<T, kCacheInt8>(L, P, s) : attn_fmt<T, kCacheE4m3>(L, P, s);
}

}  // namespace

CacheAttnPlan plan_cache_attn(const CacheAttnArgs& L, int type) {
  CacheAttnPlan P = {};
  const int64_t rows = (int64_t)L.s.max_rows * L.G;
  const int64_t row_tiles = (rows + 15) / 16, units16 = (int64_t)L.s.B * L.c.H * row_tiles;
  // The tensor-core kernel pads a unit to 128 or 256 rows, this file's reads and converts the cache again for
  // every 16 rows, which costs nothing as long as its CTAs all run at once. Rows kernel / tensor cores, us:
  //                                              16 rows      32           48           64
  //   128 sequences of 128, 9 heads of 64, bf16  35 / 39      57 / 39                   100 / 39
  //   the same, fp32                             39 / 47      70 / 49      100 / 49     131 / 49
  //   1 of 512, 4 heads of 64, fp32                           16 / 20      17 / 20      17 / 21
  //   2 of up to 899, 9 heads of 32, fp16                                               (80: 18 / 25)
  //   64 of 2048, 8 heads of 128, bf16           90 / 195     156 / 197    229 / 197    281 / 197
  //   4 of 8192, 8 heads of 128, bf16                         49 / 58      87 / 60      88 / 60
  //   64 of 2048, 8 heads of 128, fp32           102 / 451    193 / 455                 334 / 459 (96: 512 / 459)
  P.tc = rows > (L.c.D > 64 ? (type == kTypeF32 ? 64 : 48) : units16 > 2 * 148 ? 16 : 128);
  P.nr = P.tc ? cache_attn_tc_rows(L.c.D) : rows > 8 ? 16 : 8;
  P.tiles = (int)((rows + P.nr - 1) / P.nr);
  P.units = (int64_t)L.s.B * L.c.H * P.tiles;
  P.splits = 1;
  const int wave = P.tc ? (L.c.D <= 64 ? 148 * 2 : 148) : kMaxSplits;  // CTAs that run at once
  // CTAs for each unit in one wave, each left with some tokens of the longest sequence
  const int64_t wide = std::min<int64_t>(wave / std::max<int64_t>(P.units, 1), L.s.max_len / (P.tc ? 256 : 512));
  if (P.tc) {
    // Split units of many tiles, joined by a second launch (us whole / split):
    //   4 units of 2048 tokens, D 64: 39 / 19      18 of 1024, D 64: 29 / 21       18 of 512: 21 / 20
    //   72 of 1024, D 64: 25 / 25                  64 of 4096, D 128: 94 / 68      16 of 8192, D 128: 175 / 45
    // Of units that just run at once, two parts each shorten the longest sequence's way: 200 of up to 4433 tokens, D
    // 48: 92 / 72, 126 of up to 4412, D 96: 105 / 78; 144 of 4096 each, D 64: 90 / 82. (256 units at one CTA an SM, D
    // 128: 152 / 184.)
    if (wide >= 2 && L.s.max_len >= 1024) P.splits = (int)wide;
    else if (P.units <= wave && L.s.max_len >= 2048) P.splits = 2;
  } else if (wide >= 20 && L.s.max_len > 16 * 2048) {
    // Without clusters: one wave, each CTA left with 512 tokens. Worth the second launch where 16 CTAs a unit
    // would have more than 2048 tokens each (8 units, 16 CTAs / one wave: 32768 tokens 35 / 35 us, 131072 97 / 74).
    P.splits = (int)wide;
  } else {
    // CTAs of a cluster that split one unit: as long as all run at once (large clusters find room later than
    // small ones) and each is left with 128 tokens of the longest sequence (256 with 16 rows a CTA, two of which
    // share an SM); and up to 8 for two to three waves, for sequences of unlike length to even out, while each is
    // left with 2048. us by cluster size:
    //                                    1     2     4     8     16
    //   4 units of 2048 tokens           27    21    16    14    12
    //   22 of up to 2661                 29    20    16    14
    //   32 of 8192                       78    47    33    27    36
    //   55 of up to 1519                 23    18    14    18
    //   90 of up to 4945                 43    29    23    25
    //   210 of up to 3567                37    27    29    39
    //   512 of up to 8192                152   135   135   170   279
    //   2048 of up to 2048               128   162   223   381   780
    // (Of the row tiles only those of `rows` rows exist: one a sequence, or half a one more for ragged ends.)
    const int64_t tiles = std::min<int64_t>((int64_t)L.s.B * P.tiles,
                                            std::max<int64_t>(L.s.B, (L.s.rows * L.G + (int64_t)L.s.B * P.nr / 2) / P.nr));
    const int least = P.nr == 16 ? 256 : 128;
    while (P.splits < 16) {
      const int next = P.splits * 2;
      const int64_t ctas = tiles * L.c.H * next, tokens = L.s.max_len / next;
      const int room = P.nr == 16 || next > 4 ? 2 * 148 : kMaxSplits;
      if (!(ctas <= room && tokens >= least) && !(ctas <= 148 * 8 && tokens >= 2048 && next <= 8)) break;
      P.splits = next;
    }
  }
  if (P.splits > (P.tc ? 1 : 16)) P.ws_bytes = (size_t)(P.units * P.splits * P.nr) * (L.c.D * sizeof(float) + sizeof(float2));
  return P;
}

cudaError_t launch_cache_attn(const CacheAttnLaunch& L, const CacheAttnPlan& P, int type, int format, cudaStream_t s) {
  if (P.units * P.splits > INT32_MAX) return cudaErrorInvalidValue;
  cudaError_t e = P.tc ? launch_cache_attn_tc(L, P, type, format, s)
                  : type == kTypeF32 ? attn_type<float>(L, P, format, s)
                  : type == kTypeF16 ? attn_type<__half>(L, P, format, s)
                                     : attn_type<__nv_bfloat16>(L, P, format, s);
  if (e != cudaSuccess || !P.ws_bytes) return e;
  const unsigned rows = (unsigned)std::min<int64_t>((int64_t)L.s.max_rows * L.G, P.nr);
  const CacheAttnArgs& A = L;
  auto join = P.tc ? (type == kTypeF32 ? cache_attn_join_rows<float> : type == kTypeF16 ? cache_attn_join_rows<__half> : cache_attn_join_rows<__nv_bfloat16>)
                   : (type == kTypeF32 ? cache_attn_join<float> : type == kTypeF16 ? cache_attn_join<__half> : cache_attn_join<__nv_bfloat16>);
  // launched while the parts are still being formed: its CTAs wait for the whole of that launch (parts_done)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)P.units, P.tc ? (rows + 7) / 8 : rows);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join, A, P.tiles, P.nr);
}
const char* cache_attn_name(const CacheAttnPlan& P, int type) {
  if (P.tc) return type == kTypeF32 ? "cache_attention_tc_fp32" : "cache_attention_tc";
  return type == kTypeF32 ? "cache_attention_rows_fp32" : "cache_attention_rows";
}

}  // namespace supra
