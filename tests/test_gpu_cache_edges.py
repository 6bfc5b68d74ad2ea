"""The 8-bit cache at the edges of its ranges. Bounds and oracle as in test_gpu_cache.py."""

import numpy as np
import pytest
import torch

import supra_attn
from oracle import cache as oc
from test_gpu_cache import TYPES, Pool, attention_bound, bad_call

pytestmark = pytest.mark.gpu


def zero_scale(fmt):
    """What cache_write gives a block of zeros."""
    return np.float32(2.0 ** -100) * np.float32(1.0 / oc.QMAX[fmt])


def check_bound(gpu, fmt, dtype, T, G, D, lengths, rows, causal, *, seed, sharp=1.0, scale=None, mutate=None):
    """Attention of one cache head against the definition, every output within attention_bound. (The error over all
    outputs together has no limit of its own here: a row whose large weights meet V = 0 is formed from small weights
    alone, and each of those is off, against the sum of all, by what the scores may be: for D = 128 and a score of 30,
    (2 D / 16 + 6) 2^-23 30 = 8e-5. Ordinary scales with codes of 0 in those places give the same errors.)"""
    rng = np.random.default_rng(seed + 31 * T + D)
    p = Pool(gpu, rng, fmt, T, 1, D, lengths)
    if mutate:
        mutate(p)
        p.put()
    start, seqs = p.batch(rows)
    q = (torch.from_numpy(rng.standard_normal((start[-1], G * D)).astype(np.float32)) * sharp).to(TYPES[dtype])
    out = torch.full_like(q, 5.0, device="cuda")
    supra_attn.cache_attention(gpu, p.cache, seqs, q=q.cuda(), H=G, out=out, scale=scale, causal=causal)
    gpu.sync()
    got, qn = (t.cpu().double().numpy().reshape(-1, G, D) for t in (out, q))
    sc = float(np.float32(1 / np.sqrt(D) if scale is None else scale))
    ref, *terms = oc.attention(fmt, p.kc, p.ks, p.vc, p.vs, qn, lengths, start, p.table, sc, causal)
    tol = attention_bound(dtype, D, max(lengths), ref, *terms)
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside the bound, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {ref[bad][0]}"


# ---- V scales far apart -------------------------------------------------------------------------------
# lead tokens with V = 0, then ordinary ones; whole, and split along the cache (2500 tokens, few units)
ZERO_V = [(64, 130), (128, 256), (192, 300), (320, 2500)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lead,tokens", ZERO_V)
def test_attention_of_leading_zero_values(gpu, lead, tokens, D, dtype, fmt):
    """Tokens with V = 0 count in the sum of the probabilities like all others, wherever they are."""
    def zeros(scale, blocks):
        def f(p):
            for page in [p.table[0][j] for j in blocks]:
                p.vc[page] = 0
                p.vs[page] = scale
        return f

    n = -(-tokens // 64)
    first, last = range(lead // 64), range(n - lead // 64, n)
    # (sharp=0: all scores equal)
    for sharp, scale, blocks in ((0.0, zero_scale(fmt), first), (1.0, zero_scale(fmt), first), (0.0, 0.0, first), (1.0, 0.0, last),
                                 (0.0, zero_scale(fmt), range(n))):
        check_bound(gpu, fmt, dtype, 64, 2, D, [tokens], [130], False, seed=40, sharp=sharp, mutate=zeros(scale, blocks))
    check_bound(gpu, fmt, dtype, 64, 2, D, [tokens], [130], True, seed=41, mutate=zeros(zero_scale(fmt), first))
    check_bound(gpu, fmt, dtype, 64, 2, D, [tokens], [2], True, seed=42, mutate=zeros(zero_scale(fmt), first))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("far", [2.0 ** 60, 2.0 ** -60])
def test_attention_of_values_of_very_unlike_size(gpu, far, D, dtype):
    """Blocks whose V is zero, tiny or huge beside one another: a block's size counts in what it gives, never in its share."""
    def spread(sizes):
        def f(p):
            for i, page in enumerate(p.table[0]):
                p.vs[page] = np.float32(sizes[i % len(sizes)]) * p.vs[page]
                if sizes[i % len(sizes)] == 0:
                    p.vc[page] = 0
                    p.vs[page] = zero_scale("int8")
        return f

    for sizes in ((0, far), (far, 0), (far, 2.0 ** -100, 1.0), (0, 0, 1.0, far), (2.0 ** -125, far, 0), (2.0 ** 100, far)):
        for T in (16, 64):
            for sharp in (0.0, 1.0):
                check_bound(gpu, "int8", dtype, T, 1, D, [11 * T - 3], [140], True, seed=43, sharp=sharp, mutate=spread(sizes))
    # a caller's own scales below any that a write makes, alone
    check_bound(gpu, "e4m3", dtype, 32, 2, D, [70], [140], False, seed=44, mutate=spread((2.0 ** -118,)))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_of_many_zero_values_in_16_bits(gpu, dtype):
    """So many tokens with V = 0 in one piece that a sum in units of V would pass the range of 32 bits: 301 heads, so
    that no unit is split."""
    H, D, T, lead, rows = 301, 16, 128, 6016, 18
    rng = np.random.default_rng(45)
    blocks = lead // T + 1
    kc = torch.zeros(blocks, H, T, D, dtype=torch.uint8, device="cuda")
    vc = torch.zeros_like(kc)
    ks = torch.full((blocks, H), float(zero_scale("e4m3")), device="cuda")
    vs = ks.clone()
    vc[-1] = 0x38  # 1.0
    vs[-1] = torch.from_numpy(np.exp(rng.standard_normal(H)).astype(np.float32)).cuda()
    cache = supra_attn.KVCache(gpu, blocks, H, D, block_tokens=T, format="e4m3", k=kc, v=vc, k_scale=ks, v_scale=vs)
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").view(1, -1)
    seqs = supra_attn.CacheBatch(gpu, torch.tensor([lead + T], dtype=torch.int32, device="cuda"), table, max_rows=rows)
    q = torch.randn(rows, H * D, device="cuda").to(TYPES[dtype])
    out = torch.empty_like(q)
    supra_attn.cache_attention(gpu, cache, seqs, q=q, H=H, out=out)
    gpu.sync()
    ref = (vs[-1].double() * (T / (lead + T)))[None, :, None].expand(rows, H, D).cpu().numpy()
    got = out.double().cpu().numpy().reshape(rows, H, D)
    zero = np.zeros((2, 1, 1, 1))
    assert (np.abs(got - ref) <= attention_bound(dtype, D, lead + T, ref, ref, zero, np.zeros((1, 1)), np.zeros((1, 1)))).all()


# ---- scores whose factor underflows ---------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows", [3, 150])
def test_attention_of_zero_queries_and_keys(gpu, rows, dtype, fmt):
    """Rows of q that are zeros over blocks of K that are zeros, where a tile ends for some row: the mean of V."""
    def zero_k(p):
        for page in p.table[0] + p.table[1]:
            p.kc[page] = 0
            p.ks[page] = zero_scale(fmt)

    for T, D in ((64, 64), (16, 128), (128, 96)):
        for causal in (False, True):
            check_bound(gpu, fmt, dtype, T, 2, D, [100, 257], [min(rows, 100), rows], causal, seed=46, sharp=0.0, mutate=zero_k)
            # a very small scale reaches the same with any K
            check_bound(gpu, fmt, dtype, T, 2, D, [100, 257], [min(rows, 100), rows], causal, seed=47, sharp=1e-20, scale=1e-30)


# ---- block numbers ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("what", ["write", "read", "attention"])
@pytest.mark.parametrize("entry", [-2, -7, -(1 << 31), (1 << 31) - 1])
def test_every_block_outside_the_cache_is_reported(gpu, what, entry):
    rng = np.random.default_rng(48)
    p = Pool(gpu, rng, "int8", 16, 2, 32, [16, 16], spare=3)
    p.d_table[0, 0] = entry
    _, seqs = p.batch([2, 2])
    y = bad_call(gpu, p, seqs, what, 4, "outside the cache")
    if what == "attention":
        assert (y[:2] == 0).all() and (y[2:] != 5).all()
    elif what == "read":
        assert (y[:2] == 5).all() and (y[2:] != 5).any()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("entry", [-1, -2, -(1 << 31), 9])
@pytest.mark.parametrize("T,D,rows", [(16, 64, 200), (64, 64, 200), (32, 128, 300), (16, 64, 2), (64, 128, 2)])
def test_tokens_of_a_missing_block_are_left_out(gpu, T, D, rows, entry, fmt):
    rng = np.random.default_rng(49)
    n = 5 * T // 2
    p = Pool(gpu, rng, fmt, T, 1, D, [n], spare=3)
    p.d_table[0, 1] = entry
    seqs = supra_attn.CacheBatch(gpu, p.d_len, p.d_table, max_rows=rows)
    q = torch.from_numpy(rng.standard_normal((rows, D)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    supra_attn.cache_attention(gpu, p.cache, seqs, q=q, H=1, out=out)
    with pytest.raises(supra_attn.SupraAttnError, match="outside the cache"):
        gpu.sync()
    table = [[p.table[0][0], p.table[0][2]]]
    ref, pv, av, st, sm = oc.attention(fmt, p.kc, p.ks, p.vc, p.vs, q.cpu().double().numpy().reshape(rows, 1, D), [n - T], [0, rows], table,
                                       float(np.float32(1 / np.sqrt(D))), False)
    assert (np.abs(out.cpu().double().numpy().reshape(rows, 1, D) - ref) <= attention_bound("fp32", D, n, ref, pv, av, st, sm)).all()


# ---- long caches in 16 bits ---------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("D,H,rows", [(128, 150, 49), (64, 300, 17)])
def test_sums_over_a_long_cache_do_not_drift(gpu, D, H, rows, fmt):
    """So many heads that no unit is split, V of one sign: truncation of a sum kept in one accumulator over all tokens
    would pull every output towards zero. An accumulator that takes at most 4096 tokens, 16 at a step, each step off
    by at most 2^-23 of the sum, is off by 2^-15 of it. Roundings go either way: the results' own (at most 2^-11) over
    D * H unlike values average to 2^-11 / sqrt(3 D H), of which six are allowed; those of the n weights are as
    many times smaller again."""
    n, T = 32768, 128
    blocks = n // T
    g = torch.Generator(device="cuda").manual_seed(50)
    code = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    rand = lambda lo, hi: torch.randint(lo, hi, (blocks, H, T, D), generator=g, dtype=torch.int8, device="cuda")  # noqa: E731
    kc, vc = rand(-100, 101).float().to(code), rand(60, 121).float().to(code)
    ks = torch.full((blocks, H), 2.0 ** -6, device="cuda")
    vs = torch.full((blocks, H), 0.011, device="cuda")
    cache = supra_attn.KVCache(gpu, blocks, H, D, block_tokens=T, format=fmt, k=kc, v=vc, k_scale=ks, v_scale=vs)
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").view(1, -1)
    seqs = supra_attn.CacheBatch(gpu, torch.tensor([n], dtype=torch.int32, device="cuda"), table, max_rows=rows)
    q = torch.randn(rows, H * D, generator=g, device="cuda").half()
    out = torch.empty_like(q)
    supra_attn.cache_attention(gpu, cache, seqs, q=q, H=H, out=out)
    gpu.sync()
    off = torch.empty(H, rows, D, dtype=torch.float64, device="cuda")
    for h in range(H):
        k, v = (c[:, h].float().double().reshape(n, D) for c in (kc, vc))
        p = torch.softmax(q[:, h * D:(h + 1) * D].double() @ k.T * (2.0 ** -6 * float(np.float32(1 / np.sqrt(D)))), -1)
        ref = p @ v * float(np.float32(0.011))
        off[h] = (out[:, h * D:(h + 1) * D].double() - ref) / ref
    assert off.abs().max() <= 2.0 ** -11 + 2.0 ** -12 + 2.0 ** -14  # (result, weights, sums)
    assert abs(off.mean().item()) <= 2.0 ** -15 + 6 * 2.0 ** -11 / np.sqrt(3 * D * H)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_a_long_cache_whose_scores_rise(gpu, dtype):
    """Largest scores and V scales that move along a cache longer than one accumulation, whole (many heads) and against
    the 64-bit definition for some of the heads."""
    H, D, T, n, rows = 300, 64, 128, 9000, 17
    rng = np.random.default_rng(51)
    blocks = -(-n // T)
    kc = torch.from_numpy(rng.integers(-127, 128, (blocks, H, T, D)).astype(np.int8)).cuda()
    vc = torch.from_numpy(rng.integers(-127, 128, (blocks, H, T, D)).astype(np.int8)).cuda()
    rise = np.linspace(0.2, 3.0, blocks)[:, None]
    ks = (rise * np.exp(0.3 * rng.standard_normal((blocks, H))) / 127).astype(np.float32)
    vs = (np.exp2(rng.integers(-8, 9, (blocks, H))) / 127).astype(np.float32)
    cache = supra_attn.KVCache(gpu, blocks, H, D, block_tokens=T, format="int8", k=kc, v=vc, k_scale=torch.from_numpy(ks).cuda(),
                               v_scale=torch.from_numpy(vs).cuda())
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").view(1, -1)
    seqs = supra_attn.CacheBatch(gpu, torch.tensor([n], dtype=torch.int32, device="cuda"), table, max_rows=rows)
    q = torch.from_numpy(rng.standard_normal((rows, H * D)).astype(np.float32)).cuda().to(TYPES[dtype])
    out = torch.empty_like(q)
    supra_attn.cache_attention(gpu, cache, seqs, q=q, H=H, out=out, causal=True)
    gpu.sync()
    got, qn = out.cpu().double().numpy().reshape(rows, H, D), q.cpu().double().numpy().reshape(rows, H, D)
    raw_k, raw_v = kc.cpu().numpy().view(np.uint8), vc.cpu().numpy().view(np.uint8)
    for h in range(0, H, 37):
        one = [np.ascontiguousarray(a[:, h:h + 1]) for a in (raw_k, ks, raw_v, vs)]
        ref, pv, av, st, sm = oc.attention("int8", *one, qn[:, h:h + 1], [n], [0, rows], [list(range(blocks))], float(np.float32(0.125)), True)
        assert (np.abs(got[:, h:h + 1] - ref) <= attention_bound(dtype, D, n, ref, pv, av, st, sm)).all()


# ---- held codes --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_beside_codes_under_a_negative_scale(gpu, fmt):
    """A scale that no write makes is taken as the definition says: the larger one is kept, and held codes that the new
    scale cannot express become the nearest that exist."""
    T, H, D = 32, 6, 32
    rng = np.random.default_rng(52)
    p = Pool(gpu, rng, fmt, T, H, D, [20, 25])
    for i, page in enumerate(pg for pages in p.table for pg in pages):
        p.ks[page] = [-1.0, -0.5, -1e-3, 0.0, -3e4, 2.0]
        p.vs[page] = [-2.0, -0.03, 1.0, -0.0, -1e30, 1e-30]
    p.put()
    start, seqs = p.batch([5, 9])
    x = rng.standard_normal((14, H, D)).astype(np.float32)
    xd = torch.from_numpy(x.reshape(14, -1)).cuda()
    supra_attn.cache_write(gpu, p.cache, seqs, k=xd, v=xd)
    gpu.sync()
    for c, s in ((p.kc, p.ks), (p.vc, p.vs)):
        oc.write(fmt, c, s, x.astype(np.float64), [20, 25], start, p.table)
    p.check_same()


# ---- values near the end of the 32-bit range ---------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tokens,rows,top", [(90, 2, 119), (90, 140, 119), (3000, 2, 115), (3000, 140, 115), (40000, 1, 110)])
def test_attention_of_values_near_the_end_of_the_range(gpu, tokens, rows, top, D, dtype):
    """V of up to 2^(top + 1): its sum over the tokens, with weights up to 1, stays below 2^128. And as small ones."""
    for size in (2.0 ** top, 2.0 ** -top):
        def scale(p):
            for page in p.table[0]:
                p.vs[page] = np.float32(size) / 128 * (1 + p.vs[page] % 1)

        check_bound(gpu, "int8", dtype, 64, 2, D, [tokens], [rows], False, seed=60, mutate=scale)


# ---- rows that are not finite ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("D", [48, 64, 128])
@pytest.mark.parametrize("rows", [8, 140])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_of_q_that_are_not_finite_stay_alone(gpu, zeros, rows, D, dtype):
    """The others keep their bits, whatever the cache holds."""
    p = Pool(gpu, np.random.default_rng(61), "e4m3", 32, 1, D, [300])
    if zeros:
        for page in p.table[0][:3]:
            p.vc[page] = 0
            p.vs[page] = zero_scale("e4m3")
        p.put()
    _, seqs = p.batch([rows])
    q = torch.randn(rows, D, generator=torch.Generator(device="cuda").manual_seed(D + rows), device="cuda").to(TYPES[dtype])
    spoilt = q.clone()
    spoilt[5] = float("nan")
    spoilt[7, 3] = float("inf")
    out = [torch.zeros_like(q) for _ in range(2)]
    for x, o in zip((q, spoilt), out):
        supra_attn.cache_attention(gpu, p.cache, seqs, q=x, H=1, out=o, causal=True)
    gpu.sync()
    keep = [i for i in range(rows) if i not in (5, 7)]
    assert torch.equal(out[0][keep], out[1][keep]) and torch.isfinite(out[0]).all()
    assert torch.isnan(out[1][5]).all() and not torch.isfinite(out[1][7]).any()
