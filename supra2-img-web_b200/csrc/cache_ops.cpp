// libsupra_attn host runtime: the query/key norm with rotation and the paged 8-bit K/V cache calls
// (write, read, attention): argument checks and launches. Each recorded call is already a batch
// and is one launch; its descriptor travels as a kernel argument, so nothing is staged.
#include "runtime.h"

namespace supra {
namespace rt {

namespace {

constexpr int64_t kLim = int64_t(1) << 46;  // strides and offsets, in elements
constexpr int32_t kMaxCount = 1 << 30;

int esize(int32_t type) { return type == SUPRA_ATTN_T_F32 ? 4 : 2; }

ByteRange bytes_of(const void* base, int64_t first, int64_t n) {
  ByteRange r;
  r.b = reinterpret_cast<uintptr_t>(base) + (uintptr_t)first;
  r.e = r.b + (uintptr_t)std::max<int64_t>(n, 0);
  return r;
}
bool overlap(const ByteRange& a, const ByteRange& b) { return a.b < b.e && b.b < a.e; }
bool misaligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)n) != 0; }

int check_type(supra_attn_ctx* c, const char* what, int32_t type) {
  if (type != SUPRA_ATTN_T_F32 && type != SUPRA_ATTN_T_F16 && type != SUPRA_ATTN_T_BF16)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: unknown type %d", what, type);
  return SUPRA_ATTN_OK;
}

// rows of `width` elements of a strided operand: [off, off + (rows - 1) * ld + width) inside size
int check_rows(supra_attn_ctx* c, const char* what, const char* name, const void* p, int64_t size, int64_t ld,
               int64_t off, int64_t rows, int64_t width, int es) {
  if (!p && rows > 0) return set_err(c, SUPRA_ATTN_EINVAL, "%s: %s must be non-NULL", what, name);
  if (misaligned(p, es))
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: %s must be aligned to its element type", what, name);
  if (ld < 0 || ld > kLim || off < 0 || off > kLim)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: %s stride or offset out of range (negative?)", what, name);
  if (rows > 1 && ld < width)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: %s stride %lld is less than its row of %lld", what, name, (long long)ld,
                   (long long)width);
  if (rows > 0 && (rows - 1 > (kLim - off) / std::max<int64_t>(ld, 1) || off + (rows - 1) * ld + width > size))
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: %s out of bounds: %lld rows of stride %lld at %lld, size=%lld", what,
                   name, (long long)rows, (long long)ld, (long long)off, (long long)size);
  return SUPRA_ATTN_OK;
}

ByteRange rows_range(const void* p, int64_t ld, int64_t off, int64_t rows, int64_t width, int es) {
  return bytes_of(p, off * es, ((rows - 1) * ld + width) * es);
}

bool vec_rows(const void* p, int64_t ld, int64_t off, int es) {
  return !misaligned(static_cast<const char*>(p) + off * es, 16) && (ld * es) % 16 == 0;
}

int check_cache(supra_attn_ctx* c, const char* what, const supra_attn_cache& k, CachePool* pool) {
  if (k.reserved) return set_err(c, SUPRA_ATTN_EINVAL, "%s: cache reserved must be 0", what);
  if (k.format != SUPRA_ATTN_CACHE_INT8 && k.format != SUPRA_ATTN_CACHE_E4M3)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: unknown cache format %d", what, k.format);
  if (k.block_tokens != 16 && k.block_tokens != 32 && k.block_tokens != 64 && k.block_tokens != 128)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: block_tokens=%d must be 16, 32, 64 or 128", what, k.block_tokens);
  if (k.D < 16 || k.D > kCacheMaxD || k.D % 16)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: D=%d must be a multiple of 16 up to %d", what, k.D, kCacheMaxD);
  if (k.H < 1 || k.H > 65535) return set_err(c, SUPRA_ATTN_EINVAL, "%s: cache H=%d out of range", what, k.H);
  if (k.blocks < 1 || k.blocks > kMaxCount)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: blocks=%d out of range", what, k.blocks);
  if (!k.k || !k.v || !k.k_scale || !k.v_scale)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: the cache's k, v, k_scale and v_scale must be non-NULL", what);
  if (misaligned(k.k, 16) || misaligned(k.v, 16))
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: the cache's k and v must be 16-byte aligned", what);
  if (misaligned(k.k_scale, 4) || misaligned(k.v_scale, 4))
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: the cache's scales must be 4-byte aligned", what);
  const int64_t scales = (int64_t)k.blocks * k.H;  // < 2^46
  const int64_t per = (int64_t)k.block_tokens * k.D;
  if (k.k_size / per < scales || k.v_size / per < scales)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: cache out of bounds: k and v need blocks*H*block_tokens*D bytes", what);
  if (k.k_scale_size < scales || k.v_scale_size < scales)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: cache out of bounds: the scales need blocks*H=%lld floats", what,
                   (long long)scales);
  pool->k = static_cast<uint8_t*>(k.k);
  pool->v = static_cast<uint8_t*>(k.v);
  pool->ks = k.k_scale;
  pool->vs = k.v_scale;
  pool->blocks = k.blocks;
  pool->H = k.H;
  pool->D = k.D;
  pool->log2t = k.block_tokens == 16 ? 4 : k.block_tokens == 32 ? 5 : k.block_tokens == 64 ? 6 : 7;
  return SUPRA_ATTN_OK;
}

int check_seqs(supra_attn_ctx* c, const char* what, const supra_attn_cache_batch& b, int32_t block_tokens,
               CacheSeqs* s) {
  if (b.B < 0 || b.B > (1 << 24)) return set_err(c, SUPRA_ATTN_EINVAL, "%s: B=%d out of range", what, b.B);
  if (b.rows < 0 || b.rows > kMaxCount) return set_err(c, SUPRA_ATTN_EINVAL, "%s: rows out of range", what);
  if (b.max_rows < 0 || b.max_rows > kMaxCount)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: max_rows=%d out of range", what, b.max_rows);
  if (b.ld_table < 0 || b.ld_table > kMaxCount)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: ld_table=%d out of range", what, b.ld_table);
  if (b.max_len < 0 || b.max_len > kMaxCount || b.max_len > (int64_t)b.ld_table * block_tokens)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: max_len=%d exceeds ld_table*block_tokens", what, b.max_len);
  if (b.B > 0) {
    if (!b.lengths || (!b.table && b.ld_table > 0))
      return set_err(c, SUPRA_ATTN_EINVAL, "%s: lengths and table must be non-NULL", what);
    if (misaligned(b.lengths, 4) || misaligned(b.table, 4) || misaligned(b.row_start, 4))
      return set_err(c, SUPRA_ATTN_EINVAL, "%s: lengths, table and row_start must be 4-byte aligned", what);
    if (b.lengths_size < b.B) return set_err(c, SUPRA_ATTN_EINVAL, "%s: lengths must hold B=%d", what, b.B);
    if (b.table_size < (int64_t)b.B * b.ld_table)
      return set_err(c, SUPRA_ATTN_EINVAL, "%s: table must hold B*ld_table", what);
    if (b.row_start ? b.row_start_size < (int64_t)b.B + 1 : b.rows != (int64_t)b.B * b.max_rows)
      return set_err(c, SUPRA_ATTN_EINVAL,
                     b.row_start ? "%s: row_start must hold B + 1"
                                 : "%s: without row_start, rows must be B*max_rows", what);
  }
  s->lengths = b.lengths;
  s->table = b.table;
  s->row_start = b.row_start;
  s->rows = b.rows;
  s->B = b.B;
  s->ld_table = b.ld_table;
  s->max_rows = (int32_t)std::min<int64_t>(b.max_rows, b.rows);
  s->max_len = b.max_len;
  return SUPRA_ATTN_OK;
}

void seqs_reads(const CacheSeqs& s, Checked* out) {
  out->reads[out->nreads++] = bytes_of(s.lengths, 0, (int64_t)s.B * 4);
  out->reads[out->nreads++] = bytes_of(s.table, 0, (int64_t)s.B * s.ld_table * 4);
  if (s.row_start) out->reads[out->nreads++] = bytes_of(s.row_start, 0, ((int64_t)s.B + 1) * 4);
}

void pool_ranges(const CachePool& p, ByteRange r[4]) {
  const int64_t scales = (int64_t)p.blocks * p.H, codes = (scales << p.log2t) * p.D;
  r[0] = bytes_of(p.k, 0, codes);
  r[1] = bytes_of(p.v, 0, codes);
  r[2] = bytes_of(p.ks, 0, scales * 4);
  r[3] = bytes_of(p.vs, 0, scales * 4);
}

// No output may overlap an input or another output.
int check_overlap(supra_attn_ctx* c, const char* what, const Checked& ck) {
  const ByteRange* w[4] = {&ck.write, ck.more_writes, ck.more_writes + 1, ck.more_writes + 2};
  for (int i = 0; i <= ck.nmore; ++i) {
    for (int j = 0; j < ck.nreads; ++j)
      if (overlap(*w[i], ck.reads[j])) return set_err(c, SUPRA_ATTN_EINVAL, "%s: an output overlaps an input", what);
    for (int j = 0; j < i; ++j)
      if (overlap(*w[i], *w[j])) return set_err(c, SUPRA_ATTN_EINVAL, "%s: two outputs overlap", what);
  }
  return SUPRA_ATTN_OK;
}

// Device memory for one launch, ordered on the context's stream and given back after it. It comes from a
// pool of the context that keeps what it has; inside a stream capture it becomes the graph's own, so
// no two graphs share it.
int scratch_alloc(supra_attn_ctx* c, size_t bytes, void** p) {
  cudaError_t e = cudaSuccess;
  if (!c->async_pool) {
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = c->device;
    // (the stream may be capturing: making a pool is not work of the graph)
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    e = cudaMemPoolCreate(&c->async_pool, &props);
    uint64_t keep = UINT64_MAX;
    if (e == cudaSuccess) e = cudaMemPoolSetAttribute(c->async_pool, cudaMemPoolAttrReleaseThreshold, &keep);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
      if (c->async_pool) cudaMemPoolDestroy(c->async_pool);
      c->async_pool = nullptr;
      return cuda_err(c, e, "cache_attention: memory pool");
    }
  }
  e = cudaMallocFromPoolAsync(p, bytes, c->async_pool, c->stream);
  if (e == cudaErrorMemoryAllocation) {
    cudaGetLastError();
    return set_err(c, SUPRA_ATTN_ENOMEM, "cache_attention: workspace of %zu bytes failed", bytes);
  }
  return e == cudaSuccess ? SUPRA_ATTN_OK : cuda_err(c, e, "cache_attention: workspace");
}

void queue_entry(Checked* out, double flops, double bytes) {
  std::memset(&out->q, 0, sizeof out->q);
  out->q.path = PATH_CACHE;
  out->q.flops = flops;
  out->q.bytes = bytes;
}

}  // namespace

int check_qk_norm(supra_attn_ctx* c, const supra_attn_qk_norm_desc* d, Checked* out, CacheCall* call) {
  const char* what = "qk_norm";
  if (!d) return set_err(c, SUPRA_ATTN_EINVAL, "%s: descriptor is NULL", what);
  if (d->flags & ~(SUPRA_ATTN_QK_NO_NORM | SUPRA_ATTN_QK_INTERLEAVED))
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: unknown flag bits 0x%x", what, d->flags);
  if (d->reserved || d->q.reserved || d->k.reserved)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: reserved fields must be 0", what);
  int rc = check_type(c, what, d->type);
  if (rc) return rc;
  const int es = esize(d->type);
  if (d->M < 0 || d->M > kMaxCount) return set_err(c, SUPRA_ATTN_EINVAL, "%s: M=%d out of range", what, d->M);
  if (d->D < 2 || d->D > 256 || (d->D & 1))
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: D=%d must be even, 2 to 256", what, d->D);
  if (d->rot < 0 || d->rot > d->D || (d->rot & 1))
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: rot=%d must be even, 0 to D=%d", what, d->rot, d->D);
  if (d->q.H < 1 || d->q.H > 65535 || d->k.H < 0 || d->k.H > 65535)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: H=%d (queries) / %d (keys) out of range", what, d->q.H, d->k.H);
  const bool norm = !(d->flags & SUPRA_ATTN_QK_NO_NORM);
  if (norm && (!std::isfinite(d->eps) || d->eps < 0.f)) return set_err(c, SUPRA_ATTN_EINVAL, "%s: eps", what);
  if (!norm && (d->q.w || d->k.w)) return set_err(c, SUPRA_ATTN_EINVAL, "%s: weights without a norm", what);
  if (!norm && d->rot == 0) return set_err(c, SUPRA_ATTN_EINVAL, "%s: neither norm nor rotation", what);
  out->empty = d->M == 0;
  out->nreads = out->nmore = 0;
  if (d->rot) {
    if (!d->turns || misaligned(d->turns, 4))
      return set_err(c, SUPRA_ATTN_EINVAL, "%s: turns must be a 4-byte aligned float array", what);
    if (d->n_turns < 1 || (int64_t)d->n_turns * d->rot > d->turns_size)
      return set_err(c, SUPRA_ATTN_EINVAL, "%s: turns must hold n_turns*rot floats", what);
    if (d->positions && (misaligned(d->positions, 4) || d->positions_size < d->M))
      return set_err(c, SUPRA_ATTN_EINVAL, "%s: positions must hold M=%d aligned 32-bit numbers", what, d->M);
    if (!d->positions && d->M > d->n_turns)
      return set_err(c, SUPRA_ATTN_EINVAL, "%s: M=%d rows without positions, n_turns=%d", what, d->M, d->n_turns);
    out->reads[out->nreads++] = bytes_of(d->turns, 0, (int64_t)d->n_turns * d->rot * 4);
    if (d->positions) out->reads[out->nreads++] = bytes_of(d->positions, 0, (int64_t)d->M * 4);
  } else if (d->turns || d->positions) {
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: turns and positions must be NULL when rot is 0", what);
  }
  std::memset(call, 0, sizeof *call);
  call->kind = CacheCall::QK_NORM;
  call->type = d->type;
  QkNormLaunch& L = call->norm;
  const supra_attn_qk_operand* op[2] = {&d->q, &d->k};
  QkOperand* to[2] = {&L.q, &L.k};
  const char* xn[2] = {"q", "k"};
  const char* yn[2] = {"the q output", "the k output"};
  bool vec = (d->D * es) % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    const supra_attn_qk_operand& o = *op[i];
    if (o.H == 0) continue;
    const int64_t width = (int64_t)o.H * d->D;
    rc = check_rows(c, what, xn[i], o.x, o.x_size, o.ldx, o.x_off, d->M, width, es);
    if (!rc) rc = check_rows(c, what, yn[i], o.y, o.y_size, o.ldy, o.y_off, d->M, width, es);
    if (rc) return rc;
    if (o.w && (misaligned(o.w, 4) || o.w_size < d->D))
      return set_err(c, SUPRA_ATTN_EINVAL, "%s: the weights of %s must hold D=%d aligned floats", what, xn[i], d->D);
    if (out->empty) continue;
    if (o.w) {
      out->reads[out->nreads++] = bytes_of(o.w, 0, (int64_t)d->D * 4);
      vec = vec && !misaligned(o.w, 16);
    }
    vec = vec && vec_rows(o.x, o.ldx, o.x_off, es) && vec_rows(o.y, o.ldy, o.y_off, es);
    to[i]->x = static_cast<const char*>(o.x) + o.x_off * es;
    to[i]->y = static_cast<char*>(o.y) + o.y_off * es;
    to[i]->w = o.w;
    to[i]->ldx = o.ldx;
    to[i]->ldy = o.ldy;
    to[i]->H = o.H;
  }
  queue_entry(out, 0, 0);
  if (out->empty) return SUPRA_ATTN_OK;
  // Each operand's rows are compared as sets, not as byte ranges: q and k commonly interleave inside
  // the rows of one projection, and so may the outputs.
  struct Strip {
    uintptr_t b;
    int64_t pitch, width;
  };
  Strip in[2], to_s[2];
  bool in_place[2] = {false, false};
  for (int i = 0; i < 2; ++i) {
    const supra_attn_qk_operand& o = *op[i];
    if (o.H == 0) continue;
    const int64_t w = (int64_t)o.H * d->D * es;
    in[i] = {reinterpret_cast<uintptr_t>(to[i]->x), o.ldx * es, w};
    to_s[i] = {reinterpret_cast<uintptr_t>(to[i]->y), o.ldy * es, w};
    in_place[i] = in[i].b == to_s[i].b && (o.ldx == o.ldy || d->M == 1);
  }
  const int64_t M = d->M;
  auto meet = [M](const Strip& a, const Strip& b) {
    if (!(a.b < b.b + (uintptr_t)((M - 1) * b.pitch + b.width) && b.b < a.b + (uintptr_t)((M - 1) * a.pitch + a.width)))
      return false;
    if (a.pitch != b.pitch || a.pitch == 0) return true;  // (unequal strides whose spans meet are refused)
    int64_t off = ((int64_t)(b.b - a.b)) % a.pitch;
    if (off < 0) off += a.pitch;
    return off < a.width || off + b.width > a.pitch;  // b's rows start inside a's, or reach a's next row
  };
  for (int i = 0; i < 2; ++i) {
    if (op[i]->H == 0) continue;
    const ByteRange y = bytes_of(to[i]->y, 0, (M - 1) * to_s[i].pitch + to_s[i].width);
    for (int j = 0; j < out->nreads; ++j)
      if (overlap(y, out->reads[j])) return set_err(c, SUPRA_ATTN_EINVAL, "%s: an output overlaps an input", what);
    for (int j = 0; j < 2; ++j) {
      if (op[j]->H == 0) continue;
      if (!(i == j && in_place[i]) && meet(to_s[i], in[j]))
        return set_err(c, SUPRA_ATTN_EINVAL, "%s: an output overlaps an input", what);
      if (j < i && meet(to_s[i], to_s[j])) return set_err(c, SUPRA_ATTN_EINVAL, "%s: the outputs overlap", what);
    }
  }
  for (int i = 0; i < 2; ++i) {
    if (op[i]->H == 0) continue;
    out->reads[out->nreads++] = bytes_of(to[i]->x, 0, (M - 1) * in[i].pitch + in[i].width);
    const ByteRange y = bytes_of(to[i]->y, 0, (M - 1) * to_s[i].pitch + to_s[i].width);
    if (i == 0) out->write = y;
    else out->more_writes[out->nmore++] = y;
  }
  L.turns = d->turns;
  L.positions = d->positions;
  L.M = d->M;
  L.D = d->D;
  L.rot = d->rot;
  L.n_turns = d->n_turns;
  L.eps = d->eps;
  L.norm = norm ? 1 : 0;
  L.interleaved = d->flags & SUPRA_ATTN_QK_INTERLEAVED ? 1 : 0;
  call->vec = vec;
  const double n = (double)d->M * (d->q.H + d->k.H) * d->D;
  queue_entry(out, 4.0 * n + 3.0 * n * d->rot / d->D,
              2.0 * n * es + 4.0 * std::min(d->M, d->n_turns) * d->rot + (d->positions ? 4.0 * d->M : 0.0));
  return SUPRA_ATTN_OK;
}

int check_cache_rows(supra_attn_ctx* c, const supra_attn_cache_rows_desc* d, bool write, Checked* out,
                     CacheCall* call) {
  const char* what = write ? "cache_write" : "cache_read";
  if (!d) return set_err(c, SUPRA_ATTN_EINVAL, "%s: descriptor is NULL", what);
  if (d->flags) return set_err(c, SUPRA_ATTN_EINVAL, "%s: flags must be 0", what);
  std::memset(call, 0, sizeof *call);
  call->kind = write ? CacheCall::WRITE : CacheCall::READ;
  call->type = d->type;
  call->format = d->cache.format;
  CacheRowsLaunch& L = call->rows;
  int rc = check_type(c, what, d->type);
  if (!rc) rc = check_cache(c, what, d->cache, &L.c);
  if (!rc) rc = check_seqs(c, what, d->seqs, d->cache.block_tokens, &L.s);
  if (rc) return rc;
  const int es = esize(d->type);
  const int64_t width = (int64_t)d->cache.H * d->cache.D, rows = d->seqs.rows;
  rc = check_rows(c, what, "k", d->k, d->k_size, d->ldk, d->k_off, rows, width, es);
  if (!rc) rc = check_rows(c, what, "v", d->v, d->v_size, d->ldv, d->v_off, rows, width, es);
  if (rc) return rc;
  out->empty = d->seqs.B == 0 || L.s.max_rows == 0;
  out->nreads = out->nmore = 0;
  queue_entry(out, 2.0 * rows * width * (write ? 3 : 1),
              2.0 * rows * width * (1 + es) + 8.0 * d->cache.H * ((double)rows / d->cache.block_tokens + d->seqs.B));
  if (out->empty) return SUPRA_ATTN_OK;
  if ((int64_t)d->seqs.B * ((L.s.max_rows + 2 * (int64_t)d->cache.block_tokens - 2) >> L.c.log2t) > INT32_MAX)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: too many blocks in one call", what);
  seqs_reads(L.s, out);
  ByteRange pool[4];
  pool_ranges(L.c, pool);
  const ByteRange rk = rows_range(d->k, d->ldk, d->k_off, rows, width, es);
  const ByteRange rv = rows_range(d->v, d->ldv, d->v_off, rows, width, es);
  if (write) {
    out->reads[out->nreads++] = rk;
    out->reads[out->nreads++] = rv;
    out->write = pool[0];
    for (int i = 1; i < 4; ++i) out->more_writes[out->nmore++] = pool[i];
    rc = check_overlap(c, what, *out);
    if (rc) return rc;
  } else {
    for (int i = 0; i < 4; ++i) out->reads[out->nreads++] = pool[i];
    // K and V rows may interleave inside the rows of one buffer: rows of equal stride that never
    // meet, compared modulo the stride
    out->write = rk;
    out->more_writes[out->nmore++] = rv;
    for (int j = 0; j < out->nreads; ++j)
      if (overlap(rk, out->reads[j]) || overlap(rv, out->reads[j]))
        return set_err(c, SUPRA_ATTN_EINVAL, "%s: an output overlaps an input", what);
    if (overlap(rk, rv)) {
      const int64_t pitch = d->ldk * es, w = width * es;
      const int64_t kb = (int64_t)(reinterpret_cast<uintptr_t>(d->k)) + d->k_off * es;
      const int64_t vb = (int64_t)(reinterpret_cast<uintptr_t>(d->v)) + d->v_off * es;
      int64_t off = pitch > 0 ? (vb - kb) % pitch : 0;
      if (off < 0) off += pitch;
      if (d->ldk != d->ldv || pitch == 0 || off < w || off + w > pitch)
        return set_err(c, SUPRA_ATTN_EINVAL, "%s: k and v overlap", what);
    }
  }
  L.k = static_cast<char*>(d->k) + d->k_off * es;
  L.v = static_cast<char*>(d->v) + d->v_off * es;
  L.ldk = d->ldk;
  L.ldv = d->ldv;
  call->vec = vec_rows(d->k, d->ldk, d->k_off, es) && vec_rows(d->v, d->ldv, d->v_off, es);
  return SUPRA_ATTN_OK;
}

int check_cache_attn(supra_attn_ctx* c, const supra_attn_cache_attn_desc* d, Checked* out, CacheCall* call) {
  const char* what = "cache_attention";
  if (!d) return set_err(c, SUPRA_ATTN_EINVAL, "%s: descriptor is NULL", what);
  if (d->flags & ~(SUPRA_ATTN_CA_DEFAULT_SCALE | SUPRA_ATTN_CA_CAUSAL))
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: unknown flag bits 0x%x", what, d->flags);
  std::memset(call, 0, sizeof *call);
  call->kind = CacheCall::ATTENTION;
  call->type = d->type;
  call->format = d->cache.format;
  CacheAttnArgs& L = call->attn;
  int rc = check_type(c, what, d->type);
  if (!rc) rc = check_cache(c, what, d->cache, &L.c);
  if (!rc) rc = check_seqs(c, what, d->seqs, d->cache.block_tokens, &L.s);
  if (rc) return rc;
  if (d->H < 1 || d->H > 65535 || d->H % d->cache.H)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: H=%d must be a multiple of the cache's H=%d", what, d->H, d->cache.H);
  const float scale = d->flags & SUPRA_ATTN_CA_DEFAULT_SCALE ? (float)(1.0 / std::sqrt((double)d->cache.D)) : d->scale;
  if (!std::isfinite(scale * kLog2e))  // (scores are formed in powers of two)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: scale must be finite, and so its product with log2(e)", what);
  if (((int64_t)d->cache.blocks * d->cache.H << L.c.log2t) > INT32_MAX)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: blocks*H*block_tokens must be below 2^31", what);
  const int es = esize(d->type);
  const int64_t width = (int64_t)d->H * d->cache.D, rows = d->seqs.rows;
  rc = check_rows(c, what, "q", d->q, d->q_size, d->ldq, d->q_off, rows, width, es);
  if (!rc) rc = check_rows(c, what, "out", d->out, d->out_size, d->ldo, d->o_off, rows, width, es);
  if (rc) return rc;
  out->empty = d->seqs.B == 0 || L.s.max_rows == 0;
  out->nreads = out->nmore = 0;
  queue_entry(out, 4.0 * rows * width * d->seqs.max_len,
              2.0 * rows * width * es + 2.0 * d->seqs.B * (double)d->seqs.max_len * d->cache.H * d->cache.D);
  if (out->empty) return SUPRA_ATTN_OK;
  L.G = d->H / d->cache.H;
  if ((int64_t)d->seqs.B * d->cache.H * (((int64_t)L.s.max_rows * L.G + 7) / 8) * 16 > INT32_MAX)
    return set_err(c, SUPRA_ATTN_EINVAL, "%s: too many rows in one call", what);
  seqs_reads(L.s, out);
  ByteRange pool[4];
  pool_ranges(L.c, pool);
  for (int i = 0; i < 4; ++i) out->reads[out->nreads++] = pool[i];
  out->reads[out->nreads++] = rows_range(d->q, d->ldq, d->q_off, rows, width, es);
  out->write = rows_range(d->out, d->ldo, d->o_off, rows, width, es);
  rc = check_overlap(c, what, *out);
  if (rc) return rc;
  L.q = static_cast<const char*>(d->q) + d->q_off * es;
  L.o = static_cast<char*>(d->out) + d->o_off * es;
  L.ldq = d->ldq;
  L.ldo = d->ldo;
  L.H = d->H;
  L.scale_log2 = scale * kLog2e;
  L.causal = d->flags & SUPRA_ATTN_CA_CAUSAL ? 1 : 0;
  L.vec = vec_rows(d->q, d->ldq, d->q_off, es) && vec_rows(d->out, d->ldo, d->o_off, es);
  return SUPRA_ATTN_OK;
}

int flush_cache(supra_attn_ctx* c) {
  for (CacheCall& call : c->cache_calls) {
    cudaError_t e = cudaSuccess;
    const char* name = "";
    switch (call.kind) {
      case CacheCall::QK_NORM: {
        name = "qk_norm";
        call.norm.status = c->d_status;
        ProfScope ps(c, name, call.flops, call.bytes);
        e = launch_qk_norm(call.norm, call.type, call.vec, c->stream);
        break;
      }
      case CacheCall::WRITE:
      case CacheCall::READ: {
        const bool w = call.kind == CacheCall::WRITE;
        name = w ? "cache_write" : "cache_read";
        call.rows.status = c->d_status;
        ProfScope ps(c, name, call.flops, call.bytes);
        e = (w ? launch_cache_write : launch_cache_read)(call.rows, call.type, call.format, call.vec, c->stream);
        break;
      }
      case CacheCall::ATTENTION: {
        CacheAttnLaunch L;
        static_cast<CacheAttnArgs&>(L) = call.attn;
        L.status = c->d_status;
        const CacheAttnPlan plan = plan_cache_attn(L, call.type);
        name = cache_attn_name(plan, call.type);
        const int64_t tokens = ((int64_t)L.c.blocks * L.c.H) << L.c.log2t;
        const int cols = cache_attn_box_cols(L.c.D), rows = cache_attn_box_rows(L.c.log2t, plan.tc);
        if (!encode_byte_map(&L.mk, L.c.k, tokens, L.c.D, cols, rows, !plan.tc) ||
            !encode_byte_map(&L.mv, L.c.v, tokens, L.c.D, cols, rows, !plan.tc))
          return set_err(c, SUPRA_ATTN_ECUDA, "cuTensorMapEncodeTiled failed");
        L.splits = plan.splits;
        L.device = c->device;
        void* ws = nullptr;
        if (plan.ws_bytes) {
          int rc = scratch_alloc(c, plan.ws_bytes, &ws);
          if (rc) return rc;
          L.ws_o = static_cast<float*>(ws);
          L.ws_ml = reinterpret_cast<float2*>(L.ws_o + plan.units * plan.splits * plan.nr * L.c.D);
          c->launches += 1;  // the join
        }
        {
          ProfScope ps(c, name, call.flops, call.bytes);
          e = launch_cache_attn(L, plan, call.type, call.format, c->stream);
        }
        if (e == cudaErrorInvalidKernelImage) {
          if (ws) cudaFreeAsync(ws, c->stream);
          return set_err(c, SUPRA_ATTN_ECUDA, "%s: built with too few registers (or too many) for the exchange between its warps", name);
        }
        if (ws) {
          const cudaError_t f = cudaFreeAsync(ws, c->stream);
          if (e == cudaSuccess) e = f;
        }
        break;
      }
    }
    if (e != cudaSuccess) return cuda_err(c, e, name);
    c->launches += 1;
  }
  return SUPRA_ATTN_OK;
}

}  // namespace rt
}  // namespace supra
