"""The paged 8-bit K/V cache on the GPU against the 64-bit restatement (oracle/cache.py): codes and
scales bit for bit, values read back bit for bit, attention within the rounding bounds below."""

import numpy as np
import pytest
import torch

import supra_attn
from oracle import cache as oc
from supra_attn import _lib

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


class Pool:
    """A cache on both sides, its unused bytes and scales poisoned, blocks handed out in random order."""

    def __init__(self, gpu, rng, fmt, T, H, D, lengths, spare=3, fill=True):
        self.gpu, self.fmt, self.T, self.H, self.D, self.lengths = gpu, fmt, T, H, D, list(lengths)
        used = [-(-n // T) for n in lengths]
        self.blocks = sum(used) + spare
        order = list(rng.permutation(self.blocks))
        self.table = [[int(order.pop()) for _ in range(u)] for u in used]
        self.ld = max(max(used, default=0), 1) + 1
        # slots that stand for nothing: NaN bytes and NaN scales
        self.kc = np.full((self.blocks, H, T, D), 0x7f, np.uint8)
        self.vc = self.kc.copy()
        self.ks = np.full((self.blocks, H), np.nan, np.float32)
        self.vs = self.ks.copy()
        if fill:
            for c, s in ((self.kc, self.ks), (self.vc, self.vs)):
                for n, pages in zip(lengths, self.table):
                    for j, p in enumerate(pages):
                        m = min(T, n - j * T)
                        c[p, :, :m] = oc.nearest(fmt, rng.standard_normal((H, m, D)) * (40 if fmt == "int8" else 90))
                        s[p] = np.exp(rng.standard_normal(H) * 0.7) / (40 if fmt == "int8" else 90)
        self.put()

    def put(self):
        dev = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
        self.d = [dev(a) for a in (self.kc, self.vc, self.ks, self.vs)]
        table = np.full((len(self.lengths), self.ld), -7, np.int32)  # entries past a sequence are never read
        for b, pages in enumerate(self.table):
            table[b, :len(pages)] = pages
        self.d_table = torch.from_numpy(table).cuda()
        self.d_len = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        self.cache = supra_attn.KVCache(self.gpu, self.blocks, self.H, self.D, block_tokens=self.T, format=self.fmt,
                                        k=self.d[0], v=self.d[1], k_scale=self.d[2], v_scale=self.d[3])

    def batch(self, rows, total=None, **kw):
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        kw.setdefault("max_rows", max(list(rows) + [1]))
        kw["rows"] = int(start[-1]) if total is None else total
        return [int(s) for s in start], supra_attn.CacheBatch(self.gpu, self.d_len, self.d_table,
                                                              row_start=torch.from_numpy(start).cuda(), **kw)

    def check_same(self):
        for name, got, ref in zip(("k", "v", "k_scale", "v_scale"), self.d, (self.kc, self.vc, self.ks, self.vs)):
            np.testing.assert_array_equal(got.cpu().numpy(), ref, err_msg=name)


def make(rng, shape, dtype):
    t = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype)
    return t, t.double().numpy()


# ---- write and read -----------------------------------------------------------------------------------
WRITE_CASES = [
    # T, H, D, lengths (rows included), rows
    (16, 1, 16, [1], [1]),
    (16, 9, 64, [1, 16, 17, 33, 40], [1, 1, 1, 1, 1]),
    (64, 9, 64, [77, 1, 128, 5], [77, 1, 128, 5]),
    (32, 3, 80, [70, 31, 33, 0, 64], [39, 31, 2, 0, 64]),
    (128, 2, 128, [300, 129, 127], [299, 1, 126]),
    (64, 5, 48, [64, 65, 63, 190], [64, 65, 63, 1]),
    (16, 2, 112, [50, 3], [33, 0]),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("T,H,D,lengths,rows", WRITE_CASES)
def test_write_and_read(gpu, T, H, D, lengths, rows, dtype, fmt):
    rng = np.random.default_rng(T * 1000 + D + len(lengths))
    p = Pool(gpu, rng, fmt, T, H, D, lengths)
    start, seqs = p.batch(rows)
    R, W = start[-1], H * D
    # strided rows at an offset, channels and rows of unlike size (scales that grow and that do not)
    ld, off = W + 24, 8
    k, k64 = make(rng, (R * ld + off,), TYPES[dtype])
    v, v64 = make(rng, (R * ld + off,), TYPES[dtype])
    big = np.repeat(np.exp2(rng.integers(-4, 5, R)), ld)
    k[off:] = (k[off:].double() * torch.from_numpy(big)).to(TYPES[dtype])
    k64 = k.double().numpy()
    kd, vd = k.cuda(), v.cuda()
    supra_attn.cache_write(gpu, p.cache, seqs, k=kd, v=vd, ldk=ld, ldv=ld, kOff=off, vOff=off)
    gpu.sync()
    pick = lambda a: a[off:].reshape(R, ld)[:, :W].reshape(R, H, D)  # noqa: E731
    oc.write(fmt, p.kc, p.ks, pick(k64), lengths, start, p.table)
    oc.write(fmt, p.vc, p.vs, pick(v64), lengths, start, p.table)
    p.check_same()
    # read back whole sequences into the halves of one buffer's rows, at an offset, rows behind them kept
    start, seqs = p.batch(lengths, total=sum(lengths) + 2)
    out = torch.full(((sum(lengths) + 2) * (2 * W + 8) + 16,), 7.0, dtype=TYPES[dtype], device="cuda")
    supra_attn.cache_read(gpu, p.cache, seqs, k=out, v=out, ldk=2 * W + 8, ldv=2 * W + 8, kOff=8, vOff=8 + W)
    gpu.sync()
    got = out.cpu()
    ref = torch.full_like(got, 7.0)
    view = ref[8:8 + (sum(lengths) + 2) * (2 * W + 8)].reshape(-1, 2 * W + 8)
    view[:start[-1], :W] = oc.to_type(oc.read(fmt, p.kc, p.ks, lengths, start, p.table), TYPES[dtype]).reshape(-1, W)
    view[:start[-1], W:2 * W] = oc.to_type(oc.read(fmt, p.vc, p.vs, lengths, start, p.table), TYPES[dtype]).reshape(-1, W)
    assert torch.equal(got, ref)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_write_unaligned_rows(gpu, fmt, dtype):
    """Rows that start between 16-byte boundaries take the scalar loads."""
    rng = np.random.default_rng(1)
    T, H, D, lengths, rows = 32, 3, 32, [45, 9], [20, 9]
    p = Pool(gpu, rng, fmt, T, H, D, lengths)
    start, seqs = p.batch(rows)
    ld, off = H * D + 1, 3
    k, k64 = make(rng, (start[-1] * ld + off,), TYPES[dtype])
    supra_attn.cache_write(gpu, p.cache, seqs, k=k.cuda(), v=k.cuda(), ldk=ld, ldv=ld, kOff=off, vOff=off)
    x = k64[off:].reshape(-1, ld)[:, :H * D].reshape(-1, H, D)
    oc.write(fmt, p.kc, p.ks, x, lengths, start, p.table)
    oc.write(fmt, p.vc, p.vs, x, lengths, start, p.table)
    out = torch.zeros(start[-1] * ld + off, dtype=TYPES[dtype], device="cuda")
    out2 = torch.zeros_like(out)
    supra_attn.cache_read(gpu, p.cache, seqs, k=out, v=out2, ldk=ld, ldv=ld, kOff=off, vOff=off)
    gpu.sync()
    p.check_same()
    ref = oc.to_type(oc.read(fmt, p.kc, p.ks, lengths, start, p.table), TYPES[dtype]).reshape(-1, H * D)
    assert torch.equal(out.cpu()[off:].reshape(-1, ld)[:, :H * D], ref)
    assert not out.cpu()[off:].reshape(-1, ld)[:, H * D:].any()
    assert torch.equal(out2.cpu()[off:].reshape(-1, ld)[:, :H * D],
                       oc.to_type(oc.read(fmt, p.vc, p.vs, lengths, start, p.table), TYPES[dtype]).reshape(-1, H * D))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_borders_ties_and_odd_values(gpu, fmt):
    """Values on and beside the borders between codes, zeros, the smallest and largest numbers."""
    T, H, D = 32, 4, 64
    rng = np.random.default_rng(9)
    p = Pool(gpu, rng, fmt, T, H, D, [32], fill=False)
    start, seqs = p.batch([32])
    q = oc.QMAX[fmt]
    s = np.float32(3.3) * np.float32(1.0 / q)
    grid = (np.arange(-127, 127) + 0.5) if fmt == "int8" else np.concatenate([(oc.E4M3[:126] + oc.E4M3[1:127]) / 2] * 2)
    border = (grid * float(s)).astype(np.float32)
    x = np.zeros((32, H, D), np.float32)
    near = np.concatenate([border, np.nextafter(border, np.float32(9)), np.nextafter(border, np.float32(-9))])
    x[:, 0] = np.resize(near, 32 * D).reshape(32, D)
    x[0, 0, 0] = 3.3
    x[:, 1] = 0.0                     # a block of zeros
    x[:, 2] = np.float32(1e-42)       # below the scale's floor
    x[:, 3] = np.float32(3.4e38) * np.sign(rng.standard_normal((32, D)))
    xd = torch.from_numpy(x.reshape(-1)).cuda()
    supra_attn.cache_write(gpu, p.cache, seqs, k=xd, v=xd)
    gpu.sync()
    for c, sc in ((p.kc, p.ks), (p.vc, p.vs)):
        oc.write(fmt, c, sc, x.astype(np.float64), [32], start, p.table)
    p.check_same()


def test_write_of_values_that_are_not_finite(gpu):
    """A NaN or infinity makes its own block and head NaN, nothing else; a later write that starts
    the block anew clears it, one that adds to it does not."""
    T, H, D = 16, 3, 32
    rng = np.random.default_rng(2)
    p = Pool(gpu, rng, "int8", T, H, D, [40], fill=False)
    x = rng.standard_normal((40, H, D))
    x[3, 0, 5] = np.nan
    x[20, 1, 0] = -np.inf
    start, seqs = p.batch([40])
    xd = torch.from_numpy(x.astype(np.float32).reshape(-1)).cuda()
    supra_attn.cache_write(gpu, p.cache, seqs, k=xd, v=xd)
    gpu.sync()
    for c, sc in ((p.kc, p.ks), (p.vc, p.vs)):
        oc.write("int8", c, sc, x.astype(np.float32).astype(np.float64), [40], start, p.table)
    p.check_same()
    assert np.isnan(p.ks[p.table[0][0], 0]) and np.isnan(p.ks[p.table[0][1], 1]) and np.isnan(p.ks[p.table[0]]).sum() == 2
    # tokens 8 .. 21 again, finite: block 0 keeps its NaN (it holds 0 .. 7), block 1 is begun anew
    p.lengths = [22]
    p.put()
    start, seqs = p.batch([14])
    y = rng.standard_normal((14, H, D)).astype(np.float32)
    yd = torch.from_numpy(y.reshape(-1)).cuda()
    supra_attn.cache_write(gpu, p.cache, seqs, k=yd, v=yd)
    gpu.sync()
    for c, sc in ((p.kc, p.ks), (p.vc, p.vs)):
        oc.write("int8", c, sc, y.astype(np.float64), [22], start, p.table)
    p.check_same()
    assert np.isnan(p.ks[p.table[0][0], 0]) and np.isfinite(p.ks[p.table[0][1]]).all()


# ---- attention ------------------------------------------------------------------------------------------
# Rounding bounds of one output, with u = 2^-23 for an fp32 step that may truncate (the tensor core's sums):
#   scores: D/16 MMA steps (two for each part of q), the two scale products, and in base 2 the
#     subtraction of the maximum: |ds| <= (2 D/16 + 6) u S + 4 u |s|max, S = scale * sum |q||k|; fp32 rows
#     lose another 2^-22 S where the second part of q is cut to fp16;
#   p: e^ds and ex2's own 2^-22; then 2^12 p is rounded to fp16 (2^-12 of it; two parts: 2^-22), and where
#     it (or its second part) is below 2^-14, where fp16 numbers are 2^-24 apart, by up to 2^-25: 2^-37 of
#     the largest p, which is 1 and at most the sum of all, for each token: 2^-37 sum |v| of the quotient,
#     however small p is (it shows where the tokens with large p have v = 0). Where many rows share a tile
#     it is p times its block's V scale, relative to the row's largest such product, times 2^15 (fp32) or at
#     least 2^7: 2^-40 or 2^-32 of that product for each token, sum |code| of it;
#   sums over tokens: a rounding for each 16 tokens, (tokens / 16 + 40) u of sum p|v|;
#   the quotient: the error of sum p relative to itself is the same, so both count: twice;
#   the result's own rounding: eps / 2 of its type (fp16 numbers below 2^-14 are 2^-24 apart: 2^-25).
def attention_bound(dtype, D, tokens, out, pv, av, st, sm):
    u = 2.0 ** -23
    ds = (2 * D / 16 + 6) * u * st + 4 * u * sm
    if dtype == "fp32":
        ds = ds + 2.0 ** -22 * st
    p = (2.0 ** -22 if dtype == "fp32" else 2.0 ** -12) + 2.0 ** -21
    rel = 2 * (np.expm1(ds) + p + (tokens / 16 + 40) * u)
    err = rel[..., None] * pv + 2.0 ** -37 * av[0] + 2.0 ** (-40 if dtype == "fp32" else -32) * av[1]
    return err + torch.finfo(TYPES[dtype]).eps / 2 * (np.abs(out) + err) + (2.0 ** -25 if dtype == "fp16" else 1e-37)


def check_attention(gpu, fmt, dtype, T, Hk, G, D, lengths, rows, causal, scale=None, seed=0, sharp=1.0, ld_extra=8, mutate=None,
                    max_len=None):
    rng = np.random.default_rng(seed + 31 * T + D)
    p = Pool(gpu, rng, fmt, T, Hk, D, lengths)
    if mutate:
        mutate(p)
        p.put()
    H = Hk * G
    start, seqs = p.batch(rows, total=sum(rows) + 1, max_len=max_len)
    W = H * D
    ldq, ldo, off = W + ld_extra, W + 2 * ld_extra, ld_extra
    R = start[-1]
    q = (torch.from_numpy(rng.standard_normal((R + 1) * ldq + off).astype(np.float32)) * sharp).to(TYPES[dtype])
    qn = q.double().numpy()[off:].reshape(R + 1, ldq)[:R, :W].reshape(R, H, D)
    out = torch.full(((R + 1) * ldo + off,), 5.0, dtype=TYPES[dtype], device="cuda")
    supra_attn.cache_attention(gpu, p.cache, seqs, q=q.cuda(), H=H, out=out, scale=scale, causal=causal, ldq=ldq, ldo=ldo, qOff=off, oOff=off)
    gpu.sync()
    got = out.cpu().double().numpy()
    assert (got[:off] == 5).all()
    body = got[off:].reshape(R + 1, ldo)
    assert (body[R] == 5).all() and (body[:, W:] == 5).all()  # rows behind the last, gaps between rows
    got = body[:R, :W].reshape(R, H, D)
    sc = float(np.float32(1 / np.sqrt(D))) if scale is None else float(np.float32(scale))
    ref, pv, av, st, sm = oc.attention(fmt, p.kc, p.ks, p.vc, p.vs, qn, lengths, start, p.table, sc, causal)
    tol = attention_bound(dtype, D, max(lengths), ref, pv, av, st, sm)
    bad = ~(np.abs(got - ref) <= tol) & ~(np.isnan(got) & np.isnan(ref))
    worst = np.nanmax(np.abs(got - ref) / tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside the bound, worst {worst:.3g} of it, first at {np.argwhere(bad)[0]}"
    # the bound is for the worst case; over all outputs the error stays near the type's rounding
    fin = np.isfinite(ref)
    rel = np.linalg.norm((got - ref)[fin]) / max(np.linalg.norm(ref[fin]), 1e-300)
    assert rel <= {"fp32": 2e-6, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype], rel
    return got


ATTN_CASES = [
    # T, Hk, G, D, lengths, rows, causal
    (64, 9, 1, 64, [77], [1], False),
    (64, 9, 1, 64, [1, 128, 77, 0, 64], [3, 20, 1, 4, 0], False),
    (16, 2, 5, 80, [5, 100, 31, 16], [2, 7, 3, 1], True),
    (64, 2, 4, 128, [513, 64, 1], [1, 1, 1], True),
    (128, 1, 8, 128, [700, 129], [1, 2], True),
    (32, 3, 1, 16, [33, 32, 31], [1, 9, 31], True),
    (16, 1, 3, 112, [17, 15], [17, 3], False),
    (64, 2, 2, 48, [130, 3, 60], [65, 7, 60], True),   # more rows than tokens: rows that see nothing
    (32, 1, 16, 32, [1000], [4], True),
    (64, 1, 1, 96, [200, 150], [150, 33], False),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("case", ATTN_CASES, ids=lambda c: "-".join(str(x) for x in c[:4]))
def test_attention(gpu, case, dtype, fmt):
    T, Hk, G, D, lengths, rows, causal = case
    check_attention(gpu, fmt, dtype, T, Hk, G, D, lengths, rows, causal)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("T,lengths,rows", [(64, [4096, 4095, 1, 2500], [1, 2, 1, 1]), (16, [3001], [3]), (128, [9000], [1])])
def test_attention_split_along_the_cache(gpu, T, lengths, rows, dtype):
    check_attention(gpu, "int8", dtype, T, 1, 2, 64, lengths, rows, True, seed=3)
    check_attention(gpu, "e4m3", dtype, T, 1, 2, 128, lengths, rows, False, seed=4)


TILE_CASES = [
    # many query rows: T, Hk, G, D, lengths, rows, causal
    (64, 1, 1, 64, [128], [256], False),
    (64, 2, 1, 64, [1, 33, 129, 0], [130, 128, 127, 40], False),
    (128, 1, 4, 128, [700, 40], [100, 33], True),
    (32, 2, 3, 96, [300, 290], [90, 290], True),
    (16, 1, 2, 32, [77, 500], [77, 300], True),
    (16, 1, 5, 128, [130], [60], False),
    (64, 1, 8, 80, [64, 1000], [64, 37], True),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("case", TILE_CASES, ids=lambda c: "-".join(str(x) for x in c[:4]))
def test_attention_of_many_rows(gpu, case, dtype, fmt):
    T, Hk, G, D, lengths, rows, causal = case
    check_attention(gpu, fmt, dtype, T, Hk, G, D, lengths, rows, causal, seed=23)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("D", [64, 128])
def test_attention_of_many_rows_over_a_long_cache(gpu, D, dtype):
    """So few row tiles that the tokens are split among CTAs."""
    check_attention(gpu, "int8", dtype, 64, 1, 2, D, [4099, 700, 0], [40, 20, 3], True, seed=24)


@pytest.mark.parametrize("rows", [3, 70])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_of_blocks_of_unlike_size(gpu, dtype, rows):
    """V scales far apart inside one tile: a row that sees only the small ones keeps their precision. Blocks
    of zeros and negative scales are taken as they are."""
    def spread(p):
        for i, page in enumerate(p.table[0]):
            p.vs[page] *= 2.0 ** (-10 * (6 - i)) if i < 7 else 0.0 if i == 7 else -1.0

    for T, D in ((16, 64), (16, 128), (32, 64), (64, 128)):
        got = check_attention(gpu, "int8", dtype, T, 1, 1, D, [11 * T], [11 * T if rows > 3 else 3], True, seed=25, mutate=spread)
        if rows > 3:
            assert np.abs(got[:T]).max() < 2.0 ** -50  # the first block's own size

    def negative(p):
        p.ks[p.table[0][1]] *= -1
        p.vs[p.table[0][2]] *= -1

    for T in (32, 128):
        check_attention(gpu, "e4m3", dtype, T, 1, 2, 64, [3 * T + 5], [rows], True, seed=26, mutate=negative)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_attention_split_over_many_ctas(gpu, dtype):
    """Few rows over a cache so long that the parts are joined through a workspace."""
    check_attention(gpu, "int8", dtype, 64, 1, 2, 64, [11000, 300, 0], [1, 1, 1], True, seed=20)
    check_attention(gpu, "e4m3", dtype, 16, 1, 8, 128, [10753], [3], True, seed=21)


def test_captured_split_over_many_ctas(gpu):
    """The workspace inside a capture is the graph's own: two graphs and eager calls give the same bits."""
    rng = np.random.default_rng(22)
    p = Pool(gpu, rng, "int8", 128, 1, 64, [12000])
    side = torch.cuda.Stream()
    ctx = supra_attn.GPU(0, stream=side)
    cache = supra_attn.KVCache(ctx, p.blocks, 1, 64, block_tokens=128, format="int8", k=p.d[0], v=p.d[1], k_scale=p.d[2], v_scale=p.d[3])
    seqs = supra_attn.CacheBatch(ctx, p.d_len, p.d_table)
    q = torch.randn(1, 128, device="cuda")
    outs = [torch.zeros(1, 128, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    supra_attn.cache_attention(ctx, cache, seqs, q=q, H=2, out=outs[2])
    ctx.sync()
    graphs = []
    for o in outs[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            supra_attn.cache_attention(ctx, cache, seqs, q=q, H=2, out=o)
            ctx.flush()
    others = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):  # both at once, each on a stream of its own
        for g, s in zip(graphs, others):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2])
    ref, pv, av, st, sm = oc.attention("int8", p.kc, p.ks, p.vc, p.vs, q.cpu().double().numpy().reshape(1, 2, 64), [12000], [0, 1], p.table,
                                       0.125, False)
    assert (np.abs(outs[2].cpu().double().numpy().reshape(1, 2, 64) - ref) <= attention_bound("fp32", 64, 12000, ref, pv, av, st, sm)).all()
    del graphs
    ctx.close()


@pytest.mark.parametrize("fmt,dtype,rows", [("int8", "fp32", 1), ("e4m3", "bf16", 40)])
def test_blocks_past_four_gib(gpu, fmt, dtype, rows):
    """Blocks at the end of a pool of more than 2^32 bytes (and, with strides of their own, rows past 2^31 elements)
    give what the same blocks give in a small pool."""
    T, H, D, G, n = 64, 2, 128, 2, 200
    per = T * H * D
    big = (1 << 32) // per + 40
    dt = TYPES[dtype]
    rng = np.random.default_rng(30)
    k = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32)).to(dt).cuda()
    v = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32)).to(dt).cuda()
    q = torch.from_numpy(rng.standard_normal((rows, H * G * D)).astype(np.float32)).to(dt).cuda()
    ln = torch.tensor([n], dtype=torch.int32, device="cuda")
    ld = (1 << 31) // (n - 1) + 16 - ((1 << 31) // (n - 1)) % 16  # the last row starts past 2^31
    far = torch.zeros((n - 1) * ld + H * D, dtype=dt, device="cuda")
    got = []
    for blocks, first in ((8, 2), (big, big - 4)):
        cache = supra_attn.KVCache(gpu, blocks, H, D, block_tokens=T, format=fmt)
        table = torch.arange(first, first + 4, dtype=torch.int32, device="cuda").flip(0).contiguous().view(1, 4)
        new = supra_attn.CacheBatch(gpu, ln, table, max_rows=n)
        if first == 2:
            supra_attn.cache_write(gpu, cache, new, k=k, v=v)
        else:  # from rows far apart
            far.as_strided((n, H * D), (ld, 1)).copy_(k)
            torch.cuda.synchronize()
            supra_attn.cache_write(gpu, cache, new, k=far, v=v, ldk=ld)
            gpu.sync()
            far.zero_()
        out, kr, vr = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        torch.cuda.synchronize()
        supra_attn.cache_attention(gpu, cache, supra_attn.CacheBatch(gpu, ln, table, max_rows=rows), q=q, H=H * G, out=out, causal=True)
        if first == 2:
            supra_attn.cache_read(gpu, cache, new, k=kr, v=vr)
        else:
            supra_attn.cache_read(gpu, cache, new, k=far, v=vr, ldk=ld)
        gpu.sync()
        got.append((out, far.as_strided((n, H * D), (ld, 1)).clone() if first != 2 else kr, vr))
        cache.release()
    for a, b in zip(*got):
        assert torch.equal(a, b) and a.abs().max() > 0


def test_first_call_of_a_context_may_be_a_captured_one(gpu):
    """Nothing of a context has been set up yet when its first call, one with a workspace, is captured."""
    p = Pool(gpu, np.random.default_rng(23), "int8", 128, 1, 64, [12000])
    _, seqs = p.batch([1])
    q = torch.randn(1, 128, device="cuda")
    want, got = torch.zeros(1, 128, device="cuda"), torch.zeros(1, 128, device="cuda")
    supra_attn.cache_attention(gpu, p.cache, seqs, q=q, H=2, out=want)
    gpu.sync()
    side = torch.cuda.Stream()
    ctx = supra_attn.GPU(0, stream=side)
    cache = supra_attn.KVCache(ctx, p.blocks, 1, 64, block_tokens=128, format="int8", k=p.d[0], v=p.d[1], k_scale=p.d[2], v_scale=p.d[3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        supra_attn.cache_attention(ctx, cache, seqs, q=q, H=2, out=got)
        ctx.flush()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    supra_attn.cache_attention(ctx, cache, seqs, q=q, H=2, out=got.zero_())  # and an eager one after it
    torch.cuda.synchronize()
    ctx.sync()
    assert torch.equal(got, want)
    del graph
    ctx.close()


def test_two_contexts_at_once(gpu):
    """Two contexts on two streams read one cache at the same time; each has its own workspace."""
    p = Pool(gpu, np.random.default_rng(24), "e4m3", 64, 2, 64, [11000, 9000])
    _, seqs = p.batch([1, 1])
    q = [torch.randn(2, 4 * 64, device="cuda") for _ in range(2)]
    want = [torch.zeros(2, 256, device="cuda") for _ in range(2)]
    for a, o in zip(q, want):
        supra_attn.cache_attention(gpu, p.cache, seqs, q=a, H=4, out=o)
    gpu.sync()
    ctxs = [supra_attn.GPU(0, stream=torch.cuda.Stream()) for _ in range(2)]
    outs = [[torch.zeros(2, 256, device="cuda") for _ in range(8)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(8):
        for c, a, o in zip(ctxs, q, outs):
            supra_attn.cache_attention(c, p.cache, seqs, q=a, H=4, out=o[i])
            c.flush()
    for c in ctxs:
        c.sync()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)
    for c in ctxs:
        c.close()


def test_queue_of_all_kinds_of_calls(gpu):
    """Independent calls of every kind in one queue give what each gives alone, also while profiled."""
    rng = np.random.default_rng(25)
    p = Pool(gpu, rng, "int8", 16, 2, 64, [40, 9])
    _, seqs = p.batch([3, 1])
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    x, w, q, kv, n = f(64, 128), f(96, 128), f(4, 256), f(64, 3 * 128), f(32, 256)

    def calls(flush):
        o = [torch.zeros(64, 96, device="cuda"), torch.zeros(64, 128, device="cuda"), torch.zeros(4, 256, device="cuda"),
             torch.zeros(4, 128, device="cuda"), torch.zeros(4, 128, device="cuda"), torch.zeros(32, 256, device="cuda")]
        torch.cuda.synchronize()
        for call in (lambda: supra_attn.linear(gpu, x, w, N=96, K=128, M=64, out=o[0]),
                     lambda: supra_attn.cache_attention(gpu, p.cache, seqs, q=q, H=4, out=o[2], causal=True),
                     lambda: supra_attn.attention(gpu, q=kv, k=kv, v=kv, Lq=64, Lk=64, H=2, D=64, ldq=384, ldk=384, ldv=384,
                                                  kOff=128, vOff=256, out=o[1]),
                     lambda: supra_attn.cache_read(gpu, p.cache, seqs, k=o[3], v=o[4]),
                     lambda: supra_attn.qk_norm(gpu, q=n, qOut=o[5], M=32, Hq=4, D=64)):
            call()
            if flush:
                gpu.flush()
        pending = gpu.pending()
        gpu.sync()
        return o, pending

    alone, _ = calls(True)
    together, pending = calls(False)
    assert pending == 5
    gpu.profile(True)
    try:
        profiled, _ = calls(False)
        names = {e["name"] if isinstance(e, dict) else e[0] for e in gpu.profile_report()}
    finally:
        gpu.profile(False)
        gpu.profile_reset()
    assert {"qk_norm", "cache_read", "cache_attention_rows_fp32"} <= names
    for a, b, c in zip(alone, together, profiled):
        assert torch.equal(a, b) and torch.equal(a, c)
        assert a.abs().max() > 0


def test_calls_without_sequences_or_rows(gpu):
    """No sequences, or none with rows: nothing runs, and empty torch tensors (which have no address) will do."""
    p = Pool(gpu, np.random.default_rng(26), "int8", 16, 2, 32, [3])
    none = torch.empty(0, 64, device="cuda")
    ints = torch.empty(0, dtype=torch.int32, device="cuda")
    no_seqs = supra_attn.CacheBatch(gpu, ints, ints.view(0, 4))
    no_rows = supra_attn.CacheBatch(gpu, p.d_len, p.d_table, max_rows=0)
    launched = gpu.launch_count()
    for seqs in (no_seqs, no_rows):
        supra_attn.cache_write(gpu, p.cache, seqs, k=none, v=none)
        supra_attn.cache_read(gpu, p.cache, seqs, k=none, v=none)
        assert supra_attn.cache_attention(gpu, p.cache, seqs, q=none, H=2, out=none) is none
        supra_attn.cache_attention(gpu, p.cache, seqs, q=none, H=2).release()
    supra_attn.qk_norm(gpu, q=none, M=0, Hq=2, D=32)
    gpu.sync()
    assert gpu.launch_count() == launched
    p.check_same()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_attention_scale_and_sharp_scores(gpu, dtype):
    check_attention(gpu, "int8", dtype, 64, 2, 2, 64, [300, 40], [5, 33], True, scale=0.25, seed=5, sharp=4.0)
    check_attention(gpu, "int8", dtype, 64, 2, 2, 64, [300, 40], [5, 33], True, scale=-0.1, seed=6)
    check_attention(gpu, "e4m3", dtype, 64, 2, 2, 64, [300, 40], [5, 33], False, scale=0.0, seed=7)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_attention_unaligned_rows(gpu, dtype):
    check_attention(gpu, "int8", dtype, 32, 2, 1, 64, [70, 9], [3, 150], False, seed=8, ld_extra=3)


def test_attention_queries_of_unlike_size(gpu):
    """Rows whose channels are far above, below and across the fp16 range."""
    for sharp, scale in ((1e6, 1e-6), (1e-6, 1e6), (3e30, 1e-30), (1e-30, 1e30)):
        check_attention(gpu, "int8", "fp32", 64, 1, 2, 64, [100], [5], False, scale=scale, seed=9, sharp=sharp)


def test_attention_block_that_is_not_finite(gpu):
    """A block with a NaN scale reaches the rows that see it and no others."""
    def spoil(p):
        p.ks[p.table[0][2]] = np.nan   # tokens 32 .. 47
        p.vs[p.table[1][1]] = np.nan   # tokens 16 .. 31

    for fmt in ("int8", "e4m3"):
        for dtype in ("fp32", "bf16"):
            got = check_attention(gpu, fmt, dtype, 16, 1, 2, 64, [64, 40], [64, 40], True, seed=10, mutate=spoil)
            assert np.isfinite(got[:32]).all() and np.isnan(got[32:64]).all()
            assert np.isfinite(got[64:80]).all() and np.isnan(got[80:]).all()


def test_attention_same_block_in_two_sequences(gpu):
    """Sequences may share blocks (a common prompt); reading them together changes nothing."""
    def share(p):
        p.table[1][:2] = p.table[0][:2]

    check_attention(gpu, "int8", "bf16", 32, 2, 2, 64, [90, 100], [1, 4], True, seed=11, mutate=share)


def test_attention_results_repeat_bit_for_bit(gpu):
    rng = np.random.default_rng(5)
    p = Pool(gpu, rng, "int8", 64, 2, 128, [5000, 300])
    _, seqs = p.batch([1, 1])
    q = torch.randn(2, 8 * 128, dtype=torch.bfloat16, device="cuda")
    outs = []
    for _ in range(4):
        o = torch.empty_like(q)
        supra_attn.cache_attention(gpu, p.cache, seqs, q=q, H=8, out=o, causal=True)
        gpu.flush()
        outs.append(o)
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


# ---- how the calls are used ----------------------------------------------------------------------------
def test_run_of_calls_together(gpu):
    """Projection -> norm and rotation -> cache write -> attention, recorded together, over three
    steps of a growing cache; the whole against the oracle's chain on the same inputs."""
    rng = np.random.default_rng(12)
    Hk, G, D, T, B = 2, 2, 64, 16, 3
    H, C = Hk * G, 96
    p = Pool(gpu, rng, "int8", T, Hk, D, [60] * B, fill=False)
    W = (H + 2 * Hk) * D
    w = torch.from_numpy((rng.standard_normal((W, C)) / 9).astype(np.float32)).cuda()
    wq = torch.from_numpy((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)).cuda()
    turns = supra_attn.rotation_turns(gpu, np.arange(64), D)
    turns_n = gpu.read(turns).reshape(64, D)
    held = [0] * B
    for rows in ([5, 20, 1], [1, 1, 1], [16, 1, 40 - 2]):
        n = sum(rows)
        held = [a + r for a, r in zip(held, rows)]
        p.d_len.copy_(torch.tensor(held, dtype=torch.int32))  # lengths change in place
        start, seqs = p.batch(rows)
        pos = np.concatenate([np.arange(a - r, a) for a, r in zip(held, rows)]).astype(np.int32)
        x = torch.from_numpy(rng.standard_normal((n, C)).astype(np.float32)).cuda()
        qkv = torch.empty(n, W, device="cuda")
        out = torch.empty(n, H * D, device="cuda")
        supra_attn.linear(gpu, x, w, N=W, K=C, M=n, out=qkv)
        supra_attn.qk_norm(gpu, q=qkv, k=qkv, M=n, Hq=H, Hk=Hk, D=D, ldq=W, ldk=W, kOff=H * D, wq=wq, wk=wq, turns=turns, rot=D,
                           positions=torch.from_numpy(pos).cuda())
        supra_attn.cache_write(gpu, p.cache, seqs, k=qkv, v=qkv, ldk=W, ldv=W, kOff=H * D, vOff=(H + Hk) * D)
        supra_attn.cache_attention(gpu, p.cache, seqs, q=qkv, H=H, out=out, ldq=W, causal=True)
        gpu.sync()
        # the oracle continues from the GPU's rounded rows, stage by stage
        y = qkv.cpu().double().numpy()
        raw = x.cpu().double().numpy() @ w.cpu().double().numpy().T
        for lo, m in ((0, H), (H, Hk)):
            ref, mag = oc.qk_norm(raw[:, lo * D:(lo + m) * D].reshape(n, m, D), wq.cpu().double().numpy(), 1e-6, True, turns_n, D, pos, False)
            assert np.abs(y[:, lo * D:(lo + m) * D].reshape(n, m, D) - ref).max() <= 1e-5 * mag.max()
        assert np.abs(y[:, (H + Hk) * D:] - raw[:, (H + Hk) * D:]).max() <= 1e-5 * np.abs(raw).max()
        oc.write("int8", p.kc, p.ks, y[:, H * D:(H + Hk) * D].reshape(n, Hk, D), held, start, p.table)
        oc.write("int8", p.vc, p.vs, y[:, (H + Hk) * D:].reshape(n, Hk, D), held, start, p.table)
        p.check_same()
        ref, pv, av, st, sm = oc.attention("int8", p.kc, p.ks, p.vc, p.vs, y[:, :H * D].reshape(n, H, D), held, start, p.table,
                                       float(np.float32(1 / np.sqrt(D))), True)
        assert (np.abs(out.cpu().double().numpy().reshape(n, H, D) - ref) <= attention_bound("fp32", D, 64, ref, pv, av, st, sm)).all()


def test_prompt_cache_stands_for_the_fp32_one(gpu):
    """DiT cross attention from an 8-bit prompt cache against supra_attn.attention on the K/V that the
    cache stands for: the two paths agree to the FP32 tolerance."""
    rng = np.random.default_rng(13)
    lengths, rows = [77, 3, 128], [256, 256, 256]
    p = Pool(gpu, rng, "int8", 64, 9, 64, lengths, fill=False)
    kv = torch.from_numpy(rng.standard_normal((sum(lengths), 1152)).astype(np.float32)).cuda()
    _, new = p.batch(lengths)
    supra_attn.cache_write(gpu, p.cache, new, k=kv, v=kv, ldk=1152, ldv=1152, vOff=576)
    back = torch.empty_like(kv)
    supra_attn.cache_read(gpu, p.cache, new, k=back, v=back, ldk=1152, ldv=1152, vOff=576)
    q = torch.from_numpy(rng.standard_normal((768, 576)).astype(np.float32)).cuda()
    _, seqs = p.batch(rows)
    a = supra_attn.cache_attention(gpu, p.cache, seqs, q=q, H=9)
    b = gpu.empty([768, 576])
    at = 0
    for i, n in enumerate(lengths):
        supra_attn.attention(gpu, q=q, k=back, v=back, Lq=256, Lk=n, H=9, D=64, ldq=576, ldk=1152, ldv=1152, qOff=i * 256 * 576,
                             kOff=at * 1152, vOff=at * 1152 + 576, oOff=i * 256 * 576, out=b)
        at += n
    ya, yb = gpu.read(a), gpu.read(b)
    assert np.abs(ya - yb).max() <= 1e-5 * np.abs(yb).max()
    # half a code step of each block's largest value
    assert (back - kv).abs().max() <= kv.abs().max() * 0.5 / 127 * (1 + 1e-5)
    a.release()
    b.release()


def test_buffers_from_the_pool(gpu):
    """KVCache, lengths and tables without torch."""
    cache = supra_attn.KVCache(gpu, 4, 2, 32, block_tokens=16, format="e4m3")
    lengths = gpu.from_array(np.array([20, 7]), dtype="int32")
    table = gpu.from_array(np.array([[3, 1], [0, 0]]), [2, 2], dtype="int32")
    start = gpu.from_array(np.array([0, 20, 27]), dtype="int32")
    x = np.random.default_rng(0).standard_normal((27, 2, 32)).astype(np.float32)
    xd = gpu.from_array(x.reshape(27, 64), [27, 64])
    seqs = supra_attn.CacheBatch(gpu, lengths, table, row_start=start, rows=27, max_rows=20)
    supra_attn.cache_write(gpu, cache, seqs, k=xd, v=xd)
    k, v = gpu.empty([27, 64]), gpu.empty([27, 64], "fp16")
    with pytest.raises(ValueError, match="same type"):
        supra_attn.cache_read(gpu, cache, seqs, k=k, v=v)
    v2 = gpu.empty([27, 64])
    supra_attn.cache_read(gpu, cache, seqs, k=k, v=v2)
    codes, scale = np.zeros((4, 2, 16, 32), np.uint8), np.zeros((4, 2), np.float32)
    oc.write("e4m3", codes, scale, x.astype(np.float64), [20, 7], [0, 20, 27], [[3, 1], [0]])
    ref = oc.read("e4m3", codes, scale, [20, 7], [0, 20, 27], [[3, 1], [0]])
    np.testing.assert_array_equal(gpu.read(k).reshape(ref.shape), ref)
    np.testing.assert_array_equal(gpu.read(v2).reshape(ref.shape), ref)
    got = gpu.read(cache.k).reshape(codes.shape)
    for page, n in ((3, 16), (1, 4), (0, 7)):
        np.testing.assert_array_equal(got[page, :, :n], codes[page, :, :n])
    for t in (k, v, v2, xd, lengths, table, start):
        t.release()
    cache.release()
    with pytest.raises(ValueError, match="released"):
        supra_attn.cache_read(gpu, cache, seqs, k=xd, v=xd)


def test_captured_step_replays_on_changed_lengths(gpu):
    """Write and attention of a step in a CUDA graph; replays read the lengths of their own time, and
    two graphs of one context may be replayed in any order."""
    rng = np.random.default_rng(14)
    H, D, T, B = 2, 64, 16, 2
    p = Pool(gpu, rng, "int8", T, H, D, [40, 33])
    side = torch.cuda.Stream()
    ctx = supra_attn.GPU(0, stream=side)
    cache = supra_attn.KVCache(ctx, p.blocks, H, D, block_tokens=T, format="int8", k=p.d[0], v=p.d[1], k_scale=p.d[2], v_scale=p.d[3])
    seqs = supra_attn.CacheBatch(ctx, p.d_len, p.d_table, max_rows=1)
    x = torch.randn(B, 3 * H * D, device="cuda")
    outs = [torch.zeros(B, H * D, device="cuda") for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            if i == 0:
                supra_attn.cache_write(ctx, cache, seqs, k=x, v=x, ldk=3 * H * D, ldv=3 * H * D, kOff=H * D, vOff=2 * H * D)
            supra_attn.cache_attention(ctx, cache, seqs, q=x, H=H, out=outs[i], ldq=3 * H * D, causal=True)
            ctx.flush()
        graphs.append(g)
    for lens in ([30, 17], [31, 18], [40, 33]):
        x.copy_(torch.from_numpy(rng.standard_normal((B, 3 * H * D)).astype(np.float32)))
        p.d_len.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        xn = x.cpu().double().numpy()
        oc.write("int8", p.kc, p.ks, xn[:, H * D:2 * H * D].reshape(B, H, D), lens, [0, 1, 2], p.table)
        oc.write("int8", p.vc, p.vs, xn[:, 2 * H * D:].reshape(B, H, D), lens, [0, 1, 2], p.table)
        p.check_same()
        ref, pv, av, st, sm = oc.attention("int8", p.kc, p.ks, p.vc, p.vs, xn[:, :H * D].reshape(B, H, D), lens, [0, 1, 2], p.table, 0.125, True)
        for o in outs:
            assert (np.abs(o.cpu().double().numpy().reshape(B, H, D) - ref) <= attention_bound("fp32", D, 64, ref, pv, av, st, sm)).all()
    ctx.sync()
    del graphs
    ctx.close()


def test_recorded_calls_keep_their_order_and_operands(gpu):
    """A write after an attention of the same cache waits for it, and temporaries live until the flush."""
    rng = np.random.default_rng(15)
    p = Pool(gpu, rng, "int8", 16, 1, 32, [20])
    _, seqs = p.batch([1])
    q = torch.randn(1, 32, device="cuda")
    first, second = torch.zeros(1, 32, device="cuda"), torch.zeros(1, 32, device="cuda")
    supra_attn.cache_attention(gpu, p.cache, seqs, q=q, H=1, out=first)
    supra_attn.cache_write(gpu, p.cache, seqs, k=torch.full((1, 32), 9.0, device="cuda"), v=torch.full((1, 32), 9.0, device="cuda"))
    torch.full((1, 32), -1.0, device="cuda")  # would take a freed operand's place
    supra_attn.cache_attention(gpu, p.cache, seqs, q=q, H=1, out=second)
    gpu.sync()
    qn = q.cpu().double().numpy().reshape(1, 1, 32)
    sc = float(np.float32(1 / np.sqrt(32)))
    for out in (first, second):
        ref, pv, av, st, sm = oc.attention("int8", p.kc, p.ks, p.vc, p.vs, qn, [20], [0, 1], p.table, sc, False)
        assert (np.abs(out.cpu().double().numpy().reshape(1, 1, 32) - ref) <= attention_bound("fp32", 32, 20, ref, pv, av, st, sm)).all()
        nine = np.full((1, 1, 32), 9.0)
        oc.write("int8", p.kc, p.ks, nine, [20], [0, 1], p.table)
        oc.write("int8", p.vc, p.vs, nine, [20], [0, 1], p.table)
    p.check_same()


# ---- what is wrong in device arrays is reported, and nothing outside is touched ------------------------
def bad_call(gpu, p, seqs, what, rows, match):
    W = p.H * p.D
    x = torch.zeros(rows, W, device="cuda")
    y = torch.full((rows, W), 5.0, device="cuda")
    if what == "write":
        supra_attn.cache_write(gpu, p.cache, seqs, k=x, v=x)
    elif what == "read":
        supra_attn.cache_read(gpu, p.cache, seqs, k=x, v=y)
    else:
        supra_attn.cache_attention(gpu, p.cache, seqs, q=x, H=p.H, out=y)
    with pytest.raises(supra_attn.SupraAttnError, match=match):
        gpu.sync()
    assert gpu.sync() == 0  # the context goes on
    return y.cpu()


@pytest.mark.parametrize("what", ["write", "read", "attention"])
@pytest.mark.parametrize("entry", [-1, 5, 1 << 30])
def test_block_outside_the_cache(gpu, what, entry):
    rng = np.random.default_rng(16)
    p = Pool(gpu, rng, "int8", 16, 2, 32, [16, 16], spare=3)  # 5 blocks
    p.d_table[0, 0] = entry
    _, seqs = p.batch([2, 2])
    y = bad_call(gpu, p, seqs, what, 4, "outside the cache")
    if what == "write":  # the good sequence was written, the rest is as it was
        oc.write("int8", p.kc, p.ks, np.zeros((4, 2, 32)), [0, 16], [0, 0, 2], p.table)
        oc.write("int8", p.vc, p.vs, np.zeros((4, 2, 32)), [0, 16], [0, 0, 2], p.table)
    elif what == "read":
        assert (y[:2] == 5).all() and (y[2:] != 5).any()
    else:  # the tokens of a missing block are left out: none are left
        assert (y[:2] == 0).all() and (y[2:] != 5).all()
    p.check_same()


@pytest.mark.parametrize("what", ["write", "read", "attention"])
@pytest.mark.parametrize("how", ["long", "negative", "rows", "descending", "past"])
def test_sequence_outside_its_bounds(gpu, what, how):
    rng = np.random.default_rng(17)
    p = Pool(gpu, rng, "int8", 16, 2, 32, [16, 16])
    start = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    seqs = supra_attn.CacheBatch(gpu, p.d_len, p.d_table, row_start=start, rows=4, max_rows=2, max_len=20)
    if how == "long":
        p.d_len[0] = 21
    elif how == "negative":
        p.d_len[0] = -3
    elif how == "rows":
        start[1] = 3
    elif how == "descending":
        start[0] = 3
    else:
        start[1] = start[2] = 5
    y = bad_call(gpu, p, seqs, what, 4, "sequence")
    if what != "write" and how in ("long", "negative"):
        assert (y[:2] == 5).all() and (y[2:] != 5).any()
    if what != "write":
        p.check_same()


@pytest.mark.parametrize("what", ["write", "read"])
def test_more_rows_than_tokens_is_reported(gpu, what):
    p = Pool(gpu, np.random.default_rng(18), "int8", 16, 2, 32, [3])
    _, seqs = p.batch([4])
    bad_call(gpu, p, seqs, what, 4, "sequence 0")


def test_arrays_of_other_types_keep_their_values(gpu):
    for a, t in ((np.array([1.5, -np.inf, np.nan, 6e-8], np.float16), "fp16"), (np.array([-3, 7], np.int32), "int32"),
                 (np.arange(5, dtype=np.uint8), "uint8"), (np.array([0x7fc0, 1], np.uint16), "bf16")):
        x = gpu.from_array(a, dtype=t)
        assert x.dtype == t and x.shape == [a.size]
        assert gpu.read(x).tobytes() == a.tobytes()
    for a, t in (([1.1], "fp16"), ([1 << 31], "int32"), ([-1], "uint8"), ([np.nan], "int32")):
        with pytest.raises(ValueError, match="does not hold"), np.errstate(all="ignore"):
            gpu.from_array(a, dtype=t)


def test_counts_past_32_bits_are_refused(gpu):
    p = Pool(gpu, np.random.default_rng(21), "int8", 16, 2, 32, [3])
    start, seqs = p.batch([3])
    x = torch.zeros(3, 64, device="cuda")
    big = 1 << 32
    with pytest.raises(ValueError, match="out of range"):
        supra_attn.cache_attention(gpu, p.cache, seqs, q=x, H=big + 2, out=x.clone())
    with pytest.raises(ValueError, match="out of range"):
        supra_attn.CacheBatch(gpu, p.d_len, p.d_table, max_rows=big + 3, row_start=torch.tensor(start).int().cuda(), rows=3)
    with pytest.raises(ValueError, match="out of range"):
        supra_attn.CacheBatch(gpu, p.d_len, p.d_table, max_len=big + 3)
    c = p.cache
    with pytest.raises(ValueError, match="out of range"):
        supra_attn.KVCache(gpu, big + 1, c.H, c.D, block_tokens=16, k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale)
    for kw in (dict(M=big + 3), dict(Hq=big + 2), dict(D=big + 32)):
        with pytest.raises(ValueError, match="out of range"):
            supra_attn.qk_norm(gpu, q=x, **{**dict(M=3, Hq=2, D=32), **kw})
    assert gpu.pending() == 0


def test_every_read_lets_go_of_the_operands(gpu):
    p = Pool(gpu, np.random.default_rng(20), "int8", 16, 2, 32, [3])
    _, seqs = p.batch([3])
    out = gpu.empty([3, 64])
    for t in (out, gpu.empty([4], "int32")):
        supra_attn.cache_attention(gpu, p.cache, seqs, q=torch.zeros(3, 64, device="cuda"), H=2, out=out)
        assert len(gpu._held) == 1
        gpu.read(t)
        assert not gpu._held


def test_python_refusals(gpu):
    p = Pool(gpu, np.random.default_rng(19), "int8", 16, 2, 32, [3])
    _, seqs = p.batch([3])
    x = torch.zeros(3, 64, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        supra_attn.cache_read(gpu, p.cache, seqs, k=torch.zeros(64, 3, device="cuda").t(), v=x)
    with pytest.raises(ValueError, match="cuda:0"):
        supra_attn.cache_read(gpu, p.cache, seqs, k=x.cpu(), v=x)
    with pytest.raises(ValueError, match="must be"):
        supra_attn.cache_read(gpu, p.cache, seqs, k=x.double(), v=x)
    with pytest.raises(ValueError, match="int32"):
        supra_attn.CacheBatch(gpu, p.d_len.long(), p.d_table)
    with pytest.raises(ValueError, match="format"):
        supra_attn.KVCache(gpu, 1, 1, 16, format="int4")
    with pytest.raises(supra_attn.SupraAttnValueError, match="out of bounds"):
        supra_attn.cache_attention(gpu, p.cache, seqs, q=x, H=4)
    with pytest.raises(supra_attn.SupraAttnValueError, match="multiple"):
        supra_attn.cache_attention(gpu, p.cache, seqs, q=x, H=3, out=torch.zeros(3, 96, device="cuda"))
    with pytest.raises(ValueError, match="fp32"):
        supra_attn.linear(gpu, gpu.empty([64], "fp16"), x, N=1, K=64)
