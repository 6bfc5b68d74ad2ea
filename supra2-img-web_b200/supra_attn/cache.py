"""The paged 8-bit K/V cache, attention over it, and the query/key norm with rotation.

  KVCache           -- the pool: 8-bit codes [blocks, H, block_tokens, D] and one fp32 scale per block and
                       head, for K and for V. The reference keeps each prompt's K/V in fp32
                       (app/models/dit.js:137-144, app/pipeline.js:97-117); this holds four times the
                       prompts.
  CacheBatch        -- the sequences of a call: lengths, block table, rows.
  cache_write()     -- quantises new K/V rows into the cache.
  cache_read()      -- reads rows back.
  cache_attention() -- attention of query rows over the cache.
  qk_norm()         -- RMS norm of every query and key head with the position rotation, one pass.
  rotation_turns()  -- its table of cosines and sines.

Operands are Tensors of the GPU (any dtype of ops.DTYPES) or contiguous CUDA torch tensors on the GPU's
device; strides and offsets count elements and address rows inside a buffer, as everywhere in this
package. Calls are recorded and run at the next flush/sync/read; the GPU keeps their operands alive
until then. A KVCache or CacheBatch uses its operands as they are at each call: a released one is refused.
lengths, table, row_start and positions are read on the device when the call runs, so they may be changed in
place (GPU.write, torch) between calls and between replays of a captured flush. What is wrong in them is found on
the device and raised by the next sync() or read().
"""

from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import (CacheAttnDesc, CacheRowsDesc, CacheSeqs, Cache, QkNormDesc, check, lib)
from .ops import GPU, Tensor

FORMATS = {"int8": _lib.CACHE_INT8, "e4m3": _lib.CACHE_E4M3}
_TYPES = {"fp32": _lib.T_F32, "fp16": _lib.T_F16, "bf16": _lib.T_BF16}
_kinds = {}  # torch dtype -> name, filled when the first torch tensor is seen


def _fill_kinds():
    import torch

    _kinds.update({torch.float32: "fp32", torch.float16: "fp16", torch.bfloat16: "bf16", torch.int32: "int32",
                   torch.uint8: "uint8", torch.int8: "uint8", torch.float8_e4m3fn: "uint8"})


def _operand(gpu: GPU, x, name: str, dtypes):
    """(address, elements, dtype) of a Tensor or a contiguous CUDA torch tensor on the GPU's device."""
    if x.__class__ is Tensor:
        if not x.buf:
            raise ValueError(f"{name}: tensor was released")
        if x.gpu.device != gpu.device:
            raise ValueError(f"{name}: tensor of another device")
        kind = x.dtype
        if kind in dtypes:
            return x.buf, x.capacity, kind
    else:
        try:
            where = x.get_device()  # (-1: not on a GPU)
        except AttributeError:
            raise TypeError(f"{name}: unsupported operand type {type(x).__name__}") from None
        if not _kinds:
            _fill_kinds()
        if where != gpu.device:
            raise ValueError(f"{name}: torch tensors must live on cuda:{gpu.device}")
        if not x.is_contiguous():
            raise ValueError(f"{name}: torch tensors must be contiguous")
        kind = _kinds.get(x.dtype)
        if kind in dtypes:
            return x.data_ptr(), x.numel(), kind
    raise ValueError(f"{name}: must be {' or '.join(dtypes)}, not {x.dtype}")


def _address(x):
    return x.buf if x.__class__ is Tensor else x.data_ptr()


def _counts(**n):
    """The library's counts are 32-bit numbers; ctypes would cut longer ones off without a word."""
    for name, x in n.items():
        if not -1 << 31 <= x < 1 << 31:
            raise ValueError(f"{name}={x} out of range")


_FLOATS = ("fp32", "fp16", "bf16")
_INTS, _CODES, _F32 = ("int32",), ("uint8",), ("fp32",)


class KVCache:
    """A pool of `blocks` blocks of `block_tokens` tokens for H heads of D channels (supra_attn_cache).

    Without k, v, k_scale and v_scale the buffers come from the GPU's pool (release() returns them);
    otherwise they are the caller's: codes as uint8 (or torch int8 / float8_e4m3fn), scales as fp32.
    Fresh buffers need no clearing: a block's slots stand for nothing until they are written.
    """

    def __init__(self, gpu: GPU, blocks: int, H: int, D: int, *, block_tokens: int = 64, format: str = "int8", k=None,
                 v=None, k_scale=None, v_scale=None):
        if format not in FORMATS:
            raise ValueError(f"format must be one of {sorted(FORMATS)}")
        given = (k is not None) + (v is not None) + (k_scale is not None) + (v_scale is not None)
        if given not in (0, 4):
            raise ValueError("pass all of k, v, k_scale and v_scale, or none")
        self.gpu, self.format = gpu, format
        self.blocks, self.block_tokens, self.H, self.D = int(blocks), int(block_tokens), int(H), int(D)
        if (self.blocks | self.block_tokens | self.H | self.D) >> 31:
            _counts(blocks=self.blocks, block_tokens=self.block_tokens, H=self.H, D=self.D)
        self._owned = []
        if not given:
            if min(self.blocks, self.block_tokens, self.H, self.D) < 1:
                raise ValueError("blocks, block_tokens, H and D must be positive")
            shape = [self.blocks, self.H, self.block_tokens, self.D]
            try:
                for s, t in ((shape, "uint8"), (shape, "uint8"), (shape[:2], "fp32"), (shape[:2], "fp32")):
                    self._owned.append(gpu.empty(s, t))
            except Exception:
                self.release()
                raise
            k, v, k_scale, v_scale = self._owned
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        d = Cache()
        d.blocks, d.block_tokens, d.H, d.D, d.format = self.blocks, self.block_tokens, self.H, self.D, FORMATS[format]
        self._desc = d
        self._find()

    def _find(self):
        """The operands' addresses, as they are now."""
        d, gpu = self._desc, self.gpu
        a, d.k_size, _ = _operand(gpu, self.k, "k", _CODES)
        b, d.v_size, _ = _operand(gpu, self.v, "v", _CODES)
        x, d.k_scale_size, _ = _operand(gpu, self.k_scale, "k_scale", _F32)
        y, d.v_scale_size, _ = _operand(gpu, self.v_scale, "v_scale", _F32)
        d.k, d.v, d.k_scale, d.v_scale = a, b, x, y
        self._at = (a, b, x, y)

    def release(self):
        for t in self._owned:
            t.release()
        self._owned = []
        self._desc = None

    def _struct(self, gpu: GPU) -> Cache:
        if self._desc is None:
            raise ValueError("cache was released")
        if gpu.device != self.gpu.device:
            raise ValueError("cache of another device")
        if (_address(self.k), _address(self.v), _address(self.k_scale), _address(self.v_scale)) != self._at:
            self._find()
        return self._desc


class CacheBatch:
    """The sequences of a call (supra_attn_cache_batch).

    lengths: int32 [B], tokens of each sequence, those that the call writes included; table: int32
    [B, blocks a sequence may have], the block of every block_tokens tokens. The call's rows of
    sequence b are rows row_start[b] .. row_start[b+1]-1 (row_start: int32 [B+1], `rows` an upper bound
    of its last entry), or max_rows rows for every sequence when row_start is None; they stand for the
    sequence's last tokens. max_rows and max_len bound one sequence's rows and length (max_len: what
    the table's rows hold when None); tighter bounds make smaller launches. A batch may be used for
    any number of calls.
    """

    def __init__(self, gpu: GPU, lengths, table, *, max_rows: int = 1, row_start=None, rows: int | None = None,
                 max_len: int | None = None):
        s = CacheSeqs()
        self.gpu, self._seqs = gpu, s
        self._lengths, self._table, self._row_start = lengths, table, row_start
        self._find()
        if row_start is not None:
            if rows is None:
                raise ValueError("row_start needs rows, an upper bound of its last entry")
            s.rows = int(rows)
        else:
            s.rows = s.B * int(max_rows)
            if rows is not None and int(rows) != s.rows:
                raise ValueError("without row_start, rows is B*max_rows")
        max_rows = int(max_rows)
        if (max_rows | int(max_len or 0)) >> 31:
            _counts(max_rows=max_rows, max_len=int(max_len or 0))
        s.max_rows = max_rows
        # (-1: as many as the table's rows hold, which needs the cache's block size)
        s.max_len = -1 if max_len is None else int(max_len)
        if max_len is not None and int(max_len) < 0:
            raise ValueError("max_len must not be negative")
        self.rows = s.rows

    def _find(self):
        """The operands' addresses, as they are now."""
        s, gpu = self._seqs, self.gpu
        a, s.lengths_size, _ = _operand(gpu, self._lengths, "lengths", _INTS)
        b, s.table_size, _ = _operand(gpu, self._table, "table", _INTS)
        shape = tuple(self._table.shape)
        if len(shape) != 2 or tuple(self._lengths.shape) != shape[:1]:
            raise ValueError("lengths must be [B] and table [B, blocks]")
        x = None
        if self._row_start is not None:
            x, s.row_start_size, _ = _operand(gpu, self._row_start, "row_start", _INTS)
            s.row_start = x
        s.B, s.ld_table = shape
        s.lengths, s.table = a, b
        self._at = (a, b, x)  # (last: after a failure the next call looks again)

    def _fill(self, gpu: GPU, cache: KVCache, to):
        """Copies the cache and the sequences into a descriptor."""
        if gpu.device != self.gpu.device:
            raise ValueError("batch of another device")
        start = self._row_start
        if (_address(self._lengths), _address(self._table), None if start is None else _address(start)) != self._at:
            self._find()
        to.cache = cache._struct(gpu)
        to.seqs = self._seqs
        if self._seqs.max_len < 0:
            to.seqs.max_len = min(self._seqs.ld_table * cache.block_tokens, 1 << 30)


def _rows_desc(gpu: GPU, cache: KVCache, seqs: CacheBatch, k, v, ldk, ldv, kOff, vOff) -> CacheRowsDesc:
    d = CacheRowsDesc()
    seqs._fill(gpu, cache, d)
    d.k, d.k_size, kt = _operand(gpu, k, "k", _FLOATS)
    d.v, d.v_size, vt = _operand(gpu, v, "v", _FLOATS)
    if kt != vt:
        raise ValueError("k and v must have the same type")
    d.type = _TYPES[kt]
    width = cache.H * cache.D
    d.ldk = width if ldk is None else int(ldk)
    d.ldv = width if ldv is None else int(ldv)
    if kOff:
        d.k_off = int(kOff)
    if vOff:
        d.v_off = int(vOff)
    return d


def cache_write(gpu: GPU, cache: KVCache, seqs: CacheBatch, *, k, v, ldk=None, ldv=None, kOff=0, vOff=0):
    """Quantises K/V rows into the cache: the rows of `seqs` are the last tokens of their sequences.

    k, v: fp32, fp16 or bf16 rows of cache.H * cache.D channels, row r at kOff + r*ldk (ldk defaults to the
    packed row). One scale per block and head, set from the block's written tokens; a block that already
    holds earlier tokens keeps its scale unless they need a larger one, and its codes are then rounded
    again (include/supra_attn.h states the arithmetic). The blocks that one call writes must be distinct.
    """
    d = _rows_desc(gpu, cache, seqs, k, v, ldk, ldv, kOff, vOff)
    check(lib.supra_attn_enqueue_cache_write(gpu.ctx, C.byref(d)), gpu.ctx)
    gpu._held.append((cache, seqs, k, v))


def cache_read(gpu: GPU, cache: KVCache, seqs: CacheBatch, *, k, v, ldk=None, ldv=None, kOff=0, vOff=0):
    """Reads K/V rows back from the cache into k and v (code * scale, rounded to their type): the rows
    of `seqs` are the last tokens of their sequences. Rows after the last sequence's stay as they are."""
    d = _rows_desc(gpu, cache, seqs, k, v, ldk, ldv, kOff, vOff)
    check(lib.supra_attn_enqueue_cache_read(gpu.ctx, C.byref(d)), gpu.ctx)
    gpu._held.append((cache, seqs, k, v))


def cache_attention(gpu: GPU, cache: KVCache, seqs: CacheBatch, *, q, H: int, out=None, scale=None, causal: bool = False,
                    ldq=None, ldo=None, qOff=0, oOff=0):
    """Attention of the query rows of `seqs` over the cached tokens of their sequences; returns out.

    q, out: fp32, fp16 or bf16 (the same), rows of H * cache.D channels, row r of q at qOff + r*ldq; H is a
    multiple of cache.H, and H // cache.H neighbouring query heads read one cache head. causal: row i
    of a sequence's n rows sees tokens 0 .. length - n + i; otherwise every row sees the whole sequence
    (cross attention). A row that sees nothing is 0. scale defaults to 1/sqrt(D). out is allocated as
    gpu.empty([rows, H*D]) of q's type when omitted.
    """
    qa, qn, qt = _operand(gpu, q, "q", _FLOATS)
    own = out is None
    if own:
        out = gpu.empty([seqs.rows, int(H) * cache.D], qt)
    try:
        d = CacheAttnDesc()
        seqs._fill(gpu, cache, d)
        d.q, d.q_size = qa, qn
        d.out, d.out_size, ot = _operand(gpu, out, "out", _FLOATS)
        if ot != qt:
            raise ValueError("q and out must have the same type")
        d.type, d.H = _TYPES[qt], int(H)
        if d.H != H:
            raise ValueError(f"H={H} out of range")
        width = d.H * cache.D
        d.ldq = width if ldq is None else int(ldq)
        d.ldo = width if ldo is None else int(ldo)
        if qOff:
            d.q_off = int(qOff)
        if oOff:
            d.o_off = int(oOff)
        flags = _lib.CA_CAUSAL if causal else 0
        if scale is None:
            flags |= _lib.CA_DEFAULT_SCALE
        else:
            d.scale = float(scale)
        d.flags = flags
        check(lib.supra_attn_enqueue_cache_attention(gpu.ctx, C.byref(d)), gpu.ctx)
    except Exception:
        if own:
            out.release()
        raise
    gpu._held.append((cache, seqs, q, out))
    return out


def qk_norm(gpu: GPU, *, q, M: int, Hq: int, D: int, k=None, Hk: int = 0, qOut=None, kOut=None, wq=None, wk=None,
            eps: float = 1e-6, norm: bool = True, turns=None, rot: int = 0, positions=None, interleaved: bool = False,
            ldq=None, ldk=None, ldqOut=None, ldkOut=None, qOff=0, kOff=0, qOutOff=0, kOutOff=0):
    """RMS norm of every query and key head and the position rotation, in one pass over M rows.

    q, k: fp32, fp16 or bf16 buffers (often the same packed projection) with head h of row r at
    qOff + r*ldq + h*D; k with Hk = 0 is left out. qOut / kOut: the results' buffers, or None for in place
    (then ldqOut, qOutOff and their k counterparts follow the input's). wq, wk: D fp32 weights or None.
    turns, rot, positions: the first `rot` channels of each head are rotated by row positions[r] (int32 [M];
    the row number when None) of turns, an fp32 table of rows of rot/2 cosines and rot/2 sines
    (rotation_turns()); pairs are (i, i + rot/2), or (2i, 2i + 1) when interleaved. norm=False only
    rotates. A position outside the table leaves its row unwritten and raises at the next sync.
    """
    d = QkNormDesc()
    hold = []
    kinds = set()
    for o, x, H, out, w, ld, ldo, off, oo, name in (
            (d.q, q, Hq, qOut, wq, ldq, ldqOut, qOff, qOutOff, "q"), (d.k, k, Hk, kOut, wk, ldk, ldkOut, kOff, kOutOff, "k")):
        if name == "k" and k is None:
            if Hk or kOut is not None or wk is not None:
                raise ValueError("Hk, kOut and wk need k")
            continue
        o.x, o.x_size, kind = _operand(gpu, x, name, _FLOATS)
        kinds.add(kind)
        o.H = int(H)
        o.ldx = o.H * int(D) if ld is None else int(ld)
        o.x_off = int(off)
        if out is None:
            if ldo is not None or oo:
                raise ValueError(f"ld{name}Out and {name}OutOff need {name}Out")
            o.y, o.y_size, o.ldy, o.y_off = o.x, o.x_size, o.ldx, o.x_off
        else:
            o.y, o.y_size, kind = _operand(gpu, out, name + "Out", _FLOATS)
            kinds.add(kind)
            o.ldy = o.H * int(D) if ldo is None else int(ldo)
            o.y_off = int(oo)
        if w is not None:
            o.w, o.w_size, _ = _operand(gpu, w, "w" + name, _F32)
        hold += [x, out, w]
    if len(kinds) != 1:
        raise ValueError("q, k and their outputs must have the same type")
    d.type = _TYPES[kinds.pop()]
    M, D, rot = int(M), int(D), int(rot)
    if (M | D | rot | int(Hq) | int(Hk)) >> 31:
        _counts(M=M, D=D, rot=rot, Hq=int(Hq), Hk=int(Hk))
    d.M, d.D, d.rot, d.eps = M, D, rot, float(eps)
    if turns is not None:
        d.turns, d.turns_size, _ = _operand(gpu, turns, "turns", _F32)
        d.n_turns = min(d.turns_size // max(1, d.rot), (1 << 31) - 1)
    if positions is not None:
        d.positions, d.positions_size, _ = _operand(gpu, positions, "positions", _INTS)
    d.flags = (0 if norm else _lib.QK_NO_NORM) | (_lib.QK_INTERLEAVED if interleaved else 0)
    check(lib.supra_attn_enqueue_qk_norm(gpu.ctx, C.byref(d)), gpu.ctx)
    gpu._held.append((hold, turns, positions))


def rotation_turns(gpu: GPU, positions, rot: int, base: float = 10000.0) -> Tensor:
    """qk_norm's table for the given positions (numbers, one row each): pair i turns by
    position * base^(-2i / rot). positions of shape [n, axes] give the pairs to the axes in equal runs
    (patch grids), each run with its own frequencies. Angles are formed in 64 bits."""
    p = np.asarray(positions, dtype=np.float64)
    if p.ndim == 1:
        p = p[:, None]
    if p.ndim != 2 or rot < 2 or rot % (2 * p.shape[1]):
        raise ValueError("positions must be [n] or [n, axes], and rot a positive multiple of 2*axes")
    per = rot // p.shape[1]
    step = base ** (-np.arange(0, per, 2, dtype=np.float64) / per)
    far = (p[:, :, None] * step).reshape(p.shape[0], rot // 2)
    return gpu.from_array(np.concatenate([np.cos(far), np.sin(far)], axis=1).astype(np.float32), [p.shape[0], rot])
