"""Argument checks of the query/key norm and the 8-bit cache calls (pure host functions; the device
addresses are fake and never dereferenced), and the oracle's codes against torch's."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import cache as oc
from supra_attn import _lib

BASE = 0x7F0000000000
STEP = 0x100000000


def rows_desc(**kw):
    """4 prompts of up to 128 tokens, 9 heads of 64, blocks of 64 tokens."""
    d = _lib.CacheRowsDesc()
    c, s = d.cache, d.seqs
    c.blocks, c.block_tokens, c.H, c.D, c.format = 8, 64, 9, 64, _lib.CACHE_INT8
    c.k, c.v, c.k_scale, c.v_scale = BASE, BASE + STEP, BASE + 2 * STEP, BASE + 3 * STEP
    c.k_size = c.v_size = 8 * 9 * 64 * 64
    c.k_scale_size = c.v_scale_size = 72
    s.lengths, s.table, s.row_start = BASE + 4 * STEP, BASE + 5 * STEP, BASE + 6 * STEP
    s.lengths_size, s.table_size, s.row_start_size = 4, 8, 5
    s.rows, s.B, s.ld_table, s.max_rows, s.max_len = 512, 4, 2, 128, 128
    d.k, d.v = BASE + 7 * STEP, BASE + 8 * STEP
    d.k_size = d.v_size = 512 * 576
    d.ldk = d.ldv = 576
    return put(d, kw)


def put(d, kw):
    for k, v in kw.items():
        at = d
        *path, last = k.split("__")
        for p in path:
            at = getattr(at, p)
        setattr(at, last, v)
    return d


def attn_desc(**kw):
    r = rows_desc()
    d = _lib.CacheAttnDesc()
    d.cache, d.seqs = r.cache, r.seqs
    d.q, d.out = BASE + 7 * STEP, BASE + 8 * STEP
    d.q_size = d.out_size = 512 * 18 * 64
    d.ldq = d.ldo = 18 * 64
    d.H = 18
    d.flags = _lib.CA_DEFAULT_SCALE
    return put(d, kw)


def norm_desc(**kw):
    """A packed qkv projection of 2 x 256 rows, 9 heads of 64, rotated into two buffers."""
    d = _lib.QkNormDesc()
    for i, o in enumerate((d.q, d.k)):
        o.x, o.y, o.w = BASE, BASE + (1 + i) * STEP, BASE + (3 + i) * STEP
        o.x_size, o.y_size, o.w_size = 512 * 1728, 512 * 576, 64
        o.ldx, o.ldy, o.x_off, o.H = 1728, 576, 576 * i, 9
    d.turns, d.positions, d.turns_size, d.positions_size = BASE + 5 * STEP, BASE + 6 * STEP, 256 * 64, 512
    d.M, d.D, d.rot, d.n_turns, d.eps = 512, 64, 64, 256, 1e-6
    return put(d, kw)


def run(fn, d):
    msg = C.create_string_buffer(512)
    st = fn(C.byref(d), msg, 512)
    return st, msg.value.decode()


write_check = _lib.lib.supra_attn_check_cache_write_desc
read_check = _lib.lib.supra_attn_check_cache_read_desc
attn_check = _lib.lib.supra_attn_check_cache_attention_desc
norm_check = _lib.lib.supra_attn_check_qk_norm_desc


def test_valid_descriptors():
    for fn, d in ((write_check, rows_desc()), (read_check, rows_desc()), (attn_check, attn_desc()), (norm_check, norm_desc())):
        assert run(fn, d) == (_lib.OK, "")
    for t in (_lib.T_F32, _lib.T_F16, _lib.T_BF16):
        assert run(write_check, rows_desc(type=t))[0] == _lib.OK
        assert run(attn_check, attn_desc(type=t))[0] == _lib.OK
        assert run(norm_check, norm_desc(type=t))[0] == _lib.OK
    # nothing to do
    for fn, mk in ((write_check, rows_desc), (read_check, rows_desc), (attn_check, attn_desc)):
        assert run(fn, mk(seqs__B=0))[0] == _lib.OK
        assert run(fn, mk(seqs__rows=0))[0] == _lib.OK
        assert run(fn, mk(seqs__max_rows=0))[0] == _lib.OK
        assert run(fn, mk(seqs__row_start=0, seqs__rows=512))[0] == _lib.OK  # 4 x 128 rows
    assert run(norm_check, norm_desc(M=0))[0] == _lib.OK
    # queries alone, no rotation, in place
    q_only = norm_desc(rot=0, turns=0, positions=0, k__H=0, k__x=0, k__y=0, k__w=0)
    assert run(norm_check, q_only)[0] == _lib.OK
    both = norm_desc(q__y=BASE, q__y_size=512 * 1728, q__ldy=1728, k__y=BASE, k__y_size=512 * 1728, k__ldy=1728, k__y_off=576)
    assert run(norm_check, both)[0] == _lib.OK
    # K and V read back into the halves of one buffer's rows
    pair = rows_desc(v=BASE + 7 * STEP, k_size=512 * 1152, v_size=512 * 1152, ldk=1152, ldv=1152, v_off=576)
    assert run(read_check, pair)[0] == _lib.OK


CACHE_BAD = [
    (dict(cache__format=2), "format"),
    (dict(cache__block_tokens=24), "block_tokens"),
    (dict(cache__D=72), "D=72"),
    (dict(cache__D=144), "D=144"),
    (dict(cache__H=0), "H=0"),
    (dict(cache__blocks=0), "blocks=0"),
    (dict(cache__blocks=9), "out of bounds"),
    (dict(cache__k_size=8 * 9 * 64 * 64 - 1), "out of bounds"),
    (dict(cache__v_scale_size=71), "scales"),
    (dict(cache__k=BASE + 8), "16-byte"),
    (dict(cache__k_scale=BASE + 2 * STEP + 2), "4-byte"),
    (dict(cache__v=0), "non-NULL"),
    (dict(cache__reserved=1), "reserved"),
    (dict(seqs__B=-1), "B=-1"),
    (dict(seqs__lengths=0), "non-NULL"),
    (dict(seqs__table=0), "non-NULL"),
    (dict(seqs__lengths_size=3), "lengths"),
    (dict(seqs__table_size=7), "table"),
    (dict(seqs__row_start_size=4), "row_start"),
    (dict(seqs__row_start=0, seqs__rows=511), "rows must be"),
    (dict(seqs__max_len=129), "max_len"),
    (dict(seqs__max_rows=-1), "max_rows"),
    (dict(seqs__rows=-1), "rows"),
    (dict(seqs__lengths=BASE + 4 * STEP + 2), "aligned"),
    (dict(type=3), "type"),
    (dict(flags=8), "flag"),
]


@pytest.mark.parametrize("kw,needle", CACHE_BAD)
def test_cache_refusals(kw, needle):
    for fn, mk in ((write_check, rows_desc), (read_check, rows_desc), (attn_check, attn_desc)):
        st, msg = run(fn, mk(**kw))
        assert st == _lib.EINVAL and needle in msg, msg


@pytest.mark.parametrize("kw,needle", [
    (dict(k=0), "non-NULL"), (dict(k_size=512 * 576 - 1), "k out of bounds"), (dict(v_off=4), "v out of bounds"),
    (dict(ldk=575), "stride"), (dict(ldv=-1), "stride"), (dict(k_off=-4), "offset"), (dict(k=BASE + 7 * STEP + 2), "aligned"),
    (dict(ldk=1 << 50), "stride"), (dict(k=BASE), "overlap"), (dict(v=BASE + 2 * STEP), "overlap"),
])
def test_rows_refusals(kw, needle):
    for fn in (write_check, read_check):
        st, msg = run(fn, rows_desc(**kw))
        assert st == _lib.EINVAL and needle in msg, msg


def test_overlapping_outputs_are_refused():
    st, msg = run(write_check, rows_desc(cache__v=BASE + 64))  # K codes and V codes
    assert st == _lib.EINVAL and "outputs overlap" in msg
    st, msg = run(read_check, rows_desc(v=BASE + 7 * STEP, v_off=0))  # k and v rows in one place
    assert st == _lib.EINVAL and "overlap" in msg
    st, msg = run(read_check, rows_desc(v=BASE + 7 * STEP, k_size=512 * 1152, v_size=512 * 1152, ldk=1152, ldv=1152, v_off=575))
    assert st == _lib.EINVAL and "overlap" in msg
    assert run(write_check, rows_desc(v=BASE + 7 * STEP))[0] == _lib.OK  # the same rows read twice


@pytest.mark.parametrize("kw,needle", [
    (dict(H=0), "H=0"), (dict(H=20), "multiple"), (dict(q=0), "non-NULL"), (dict(q_size=512 * 1152 - 1), "q out of bounds"),
    (dict(out_size=512 * 1152 - 1), "out out of bounds"), (dict(ldo=1151), "stride"), (dict(out=BASE + 7 * STEP), "overlap"),
    (dict(out=BASE + 6 * STEP), "overlap"), (dict(flags=0, scale=float("nan")), "finite"), (dict(q_off=-1), "offset"),
])
def test_attention_refusals(kw, needle):
    st, msg = run(attn_check, attn_desc(**kw))
    assert st == _lib.EINVAL and needle in msg, msg


@pytest.mark.parametrize("kw,needle", [
    (dict(M=-1), "M=-1"), (dict(D=65), "D=65"), (dict(D=258), "D=258"), (dict(rot=66), "rot"), (dict(rot=31), "rot"),
    (dict(q__H=0), "H=0"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(type=9), "type"), (dict(flags=4), "flag"),
    (dict(flags=1), "weights"), (dict(flags=1, q__w=0, k__w=0, rot=0, turns=0, positions=0), "neither"), (dict(turns=0), "turns"),
    (dict(turns_size=256 * 64 - 1), "turns"), (dict(positions_size=511), "positions"), (dict(positions=0), "n_turns"),
    (dict(rot=0), "NULL"), (dict(q__w_size=63), "weights"), (dict(k__x_size=512 * 1728 - 577), "k out of bounds"),
    (dict(q__y_size=512 * 576 - 1), "q output"), (dict(q__ldy=575), "stride"), (dict(q__y=BASE), "overlap"),
    (dict(k__y=BASE + STEP), "outputs overlap"), (dict(q__y=BASE + 5 * STEP), "overlap"), (dict(q__reserved=1), "reserved"),
    (dict(q__y=BASE, q__ldy=1728, q__y_size=512 * 1728, q__y_off=64), "overlap"),  # shifted, not in place
    (dict(q__y=BASE, q__ldy=1728, q__y_size=512 * 1728, q__y_off=576, k__y=BASE, k__ldy=1728, k__y_size=512 * 1728), "overlap"),
])
def test_norm_refusals(kw, needle):
    st, msg = run(norm_check, norm_desc(**kw))
    assert st == _lib.EINVAL and needle in msg, msg


@pytest.mark.parametrize("scale,ok", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False), (float("nan"), False)])
def test_attention_scale_in_powers_of_two_stays_finite(scale, ok):
    st, msg = run(attn_check, attn_desc(flags=0, scale=scale))
    assert st == (0 if ok else _lib.EINVAL) and ("scale" in msg) == (not ok)


def test_calls_without_rows_take_null_operands():
    none = dict(k=0, v=0, k_size=0, v_size=0, seqs__rows=0, seqs__max_rows=0)
    for fn in (write_check, read_check):
        assert run(fn, rows_desc(**none)) == (0, "")
        assert run(fn, rows_desc(**none, seqs__B=0, seqs__lengths=0, seqs__table=0, seqs__row_start=0)) == (0, "")
    assert run(attn_check, attn_desc(q=0, out=0, q_size=0, out_size=0, seqs__rows=0, seqs__max_rows=0)) == (0, "")
    assert run(norm_check, norm_desc(M=0, q__x=0, q__y=0, k__x=0, k__y=0)) == (0, "")
    for kw in (dict(seqs__rows=1, k=0), dict(seqs__rows=1, v=0)):
        st, msg = run(read_check, rows_desc(**kw))
        assert st == _lib.EINVAL and "non-NULL" in msg


def test_null_descriptors():
    for fn in (write_check, read_check, attn_check, norm_check):
        msg = C.create_string_buffer(64)
        assert fn(None, msg, 64) == _lib.EINVAL and b"NULL" in msg.value
    for fn in ("qk_norm", "cache_write", "cache_read", "cache_attention"):
        assert getattr(_lib.lib, "supra_attn_enqueue_" + fn)(None, None) == _lib.EINVAL


# ---- the oracle's codes -------------------------------------------------------------------------------
def test_oracle_e4m3_matches_torch():
    raw = np.arange(256, dtype=np.uint8)
    ref = torch.from_numpy(raw.copy()).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(oc.E4M3, ref)
    x = np.concatenate([np.linspace(-448, 448, 20011), np.ldexp(np.linspace(-9, 9, 4001), -9), oc.E4M3[:127],
                        (oc.E4M3[:126] + oc.E4M3[1:127]) / 2])  # ties among them
    got = oc.decode("e4m3", oc.nearest("e4m3", x.astype(np.float32)))
    ref = torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(got, ref)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_oracle_write_then_read(fmt):
    """Every value comes back within half a code step of its block (the scale is amax / qmax)."""
    rng = np.random.default_rng(3)
    T, H, D = 16, 2, 32
    codes, scale = np.zeros((6, H, T, D), np.uint8), np.zeros((6, H), np.float32)
    x = rng.standard_normal((40, H, D))
    lengths, start, table = [23, 17], [0, 23, 40], [[4, 1], [0, 5]]
    oc.write(fmt, codes, scale, x, lengths, start, table)
    y = oc.read(fmt, codes, scale, lengths, start, table)
    step = {"int8": 0.5 / 127, "e4m3": 16 / 448}[fmt]  # half a step at the largest code
    assert np.abs(y - x).max() <= np.abs(x).max() * step * (1 + 1e-5)
