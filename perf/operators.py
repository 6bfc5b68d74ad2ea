"""Cases of the 8-bit K/V cache operators and of the query/key norm with rotation.

Four operators, each in its plain form (elementary torch operations in 32 bits) and through the
framework's entry points:

  norm    RMS norm of every query and key head and the position rotation, one pass over the rows of a
          projection (supra_attn.qk_norm)
  write   quantising K/V rows into a paged cache of 8-bit codes with one scale per block of tokens and
          head, and reading the touched blocks back (supra_attn.cache_write, cache_read)
  read    reading whole sequences back from such a cache (supra_attn.cache_read)
  attend  attention of new query rows over such a cache (supra_attn.cache_attention)

The cache: codes [blocks, H, block_tokens, D] and scales [blocks, H] for K and for V; a sequence of
`length` tokens keeps token t in block table[t // block_tokens], slot t % block_tokens. The rows of a
call are the last tokens of their sequences: row i of a sequence's n rows is token length - n + i.

Quantising: scale = max(amax, 2^-100) * (1 / qmax) over the block's written tokens of one head (qmax 127
or 448), never below the scale the block already had when the write adds to its tokens; code = the
nearest to x * inv, ties to even, with inv = 1 / scale; codes the block already held become the nearest
to code * (old scale / new scale) when the scale grows. scale, 1 / qmax, inv and the ratio are 32-bit
numbers; the products are rounded once, to the code (64 bits hold them exactly).
"""

import math
import os
import random
import sys

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
FLOOR = 2.0 ** -100


def listed():
    return [
        # one prompt's cross attention for a single query row: the smallest call, latency alone
        {"name": "attend_one_prompt", "op": "attend", "B": 1, "H": 9, "Hkv": 9, "D": 64, "T": 64, "rows_lo": 1,
         "rows_hi": 1, "len_lo": 77, "len_hi": 77, "format": "int8", "dtype": "fp32", "causal": False},
        # DiT cross attention: 128 prompts of ragged length, 256 patch rows each, cached K/V (fp32 as the model)
        {"name": "attend_dit_cross", "op": "attend", "B": 128, "H": 9, "Hkv": 9, "D": 64, "T": 64, "rows_lo": 256,
         "rows_hi": 256, "len_lo": 1, "len_hi": 128, "format": "int8", "dtype": "fp32", "causal": False},
        # a step of 64 sequences, one token each, grouped heads, ragged lengths
        {"name": "attend_step_batch", "op": "attend", "B": 64, "H": 32, "Hkv": 8, "D": 128, "T": 64, "rows_lo": 1,
         "rows_hi": 1, "len_lo": 1000, "len_hi": 8000, "format": "e4m3", "dtype": "bf16", "causal": True},
        # a step of one sequence over a long cache: few rows, the work split along the cache
        {"name": "attend_step_long", "op": "attend", "B": 1, "H": 32, "Hkv": 8, "D": 128, "T": 128, "rows_lo": 1,
         "rows_hi": 1, "len_lo": 131072, "len_hi": 131072, "format": "int8", "dtype": "fp16", "causal": True},
        # chunks of new tokens against their own history, causal, ragged chunks and lengths
        {"name": "attend_chunk", "op": "attend", "B": 4, "H": 16, "Hkv": 4, "D": 128, "T": 64, "rows_lo": 700,
         "rows_hi": 1024, "len_lo": 2049, "len_hi": 4096, "format": "int8", "dtype": "bf16", "causal": True},
        # several query rows a sequence (a draft to be checked), small blocks, a narrow odd head
        {"name": "attend_draft_small_blocks", "op": "attend", "B": 33, "H": 10, "Hkv": 2, "D": 80, "T": 16,
         "rows_lo": 2, "rows_hi": 7, "len_lo": 5, "len_hi": 1511, "format": "e4m3", "dtype": "fp16", "causal": True},
        # prompts taken into the cache: thousands of rows at once
        {"name": "write_prompts", "op": "write", "B": 16, "Hkv": 8, "D": 128, "T": 64, "rows_lo": 500, "rows_hi": 2000,
         "len_lo": 500, "len_hi": 2300, "format": "e4m3", "dtype": "bf16"},
        # one more token for each sequence: partly filled blocks whose scale may grow
        {"name": "write_step", "op": "write", "B": 64, "Hkv": 9, "D": 64, "T": 16, "rows_lo": 1, "rows_hi": 1,
         "len_lo": 1, "len_hi": 300, "format": "int8", "dtype": "fp32"},
        # a few prompts read back in the model's type
        {"name": "read_prompts", "op": "read", "B": 5, "Hkv": 9, "D": 64, "T": 64, "len_lo": 1, "len_hi": 128,
         "format": "int8", "dtype": "fp32"},
        # long sequences read back to 16 bits
        {"name": "read_long", "op": "read", "B": 16, "Hkv": 8, "D": 128, "T": 64, "len_lo": 1500, "len_hi": 4099,
         "format": "e4m3", "dtype": "bf16"},
        # the DiT's packed qkv projection, 64 images of 256 patches, fp32, rows normalised and rotated
        {"name": "norm_dit_rows", "op": "norm", "M": 16384, "Hq": 9, "Hk": 9, "D": 64, "rot": 64, "positions": 256,
         "dtype": "fp32", "interleaved": True},
        # a step's rows at far positions, grouped heads, part of the head rotated
        {"name": "norm_step", "op": "norm", "M": 61, "Hq": 32, "Hk": 8, "D": 128, "rot": 96, "positions": 131072,
         "dtype": "bf16", "interleaved": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _draw_once(rng):
    op = rng.choice(["attend", "attend", "write", "read", "norm"])
    D = 16 * rng.randint(1, 8)
    dtype = rng.choice(sorted(DTYPES))
    if op == "norm":
        Hk = rng.randint(1, 9)
        return {"op": op, "M": _log_int(rng, 1, 16384), "Hq": Hk * rng.randint(1, 4), "Hk": Hk, "D": D,
                "rot": 2 * rng.randint(0, D // 2), "positions": _log_int(rng, 256, 131072), "dtype": dtype,
                "interleaved": rng.random() < 0.5}
    c = {"op": op, "B": _log_int(rng, 1, 64), "Hkv": rng.randint(1, 9), "D": D, "T": rng.choice([16, 32, 64, 128]),
         "format": rng.choice(sorted(QMAX)), "dtype": dtype}
    lo, hi = sorted((_log_int(rng, 1, 8192), _log_int(rng, 1, 8192)))
    c["len_lo"], c["len_hi"] = lo, hi
    if op != "read":
        rlo, rhi = sorted((_log_int(rng, 1, 1024), _log_int(rng, 1, 1024)))
        if op == "attend" and rng.random() < 0.5:
            rlo = rhi = 1
        c["rows_lo"], c["rows_hi"] = rlo, rhi
        if op == "write":  # the rows are among the sequence's tokens
            c["len_lo"], c["len_hi"] = max(lo, rhi), max(hi, rhi)
    if op == "attend":
        c["H"] = c["Hkv"] * rng.choice([1, 1, 2, 3, 4, 8])
        c["causal"] = rng.random() < 0.5
    return c


def draw(rng):
    top = {}
    for c in listed():
        w, t = work(c), top.setdefault(c["op"], {"bytes": 0.0, "flops": 0.0})
        t["bytes"], t["flops"] = max(t["bytes"], w["bytes"]), max(t["flops"], w["flops"])
    while True:
        c = _draw_once(rng)
        w = work(c)
        # the scores that the plain form holds at once are bounded by those of the listed cases
        held = c["B"] * c.get("H", 1) * c.get("rows_hi", 1) * c["len_hi"] if c["op"] == "attend" else 0
        if w["bytes"] <= top[c["op"]]["bytes"] and w["flops"] <= top[c["op"]]["flops"] and held <= 2 ** 28:
            return c


# ---- sizes that follow from a case alone -----------------------------------------------------------
def _spread(lo, hi, n, salt):
    """n whole numbers over [lo, hi], both ends among them (n > 1), in no order."""
    r = random.Random(salt)
    v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]
    r.shuffle(v)
    return v


def _lengths(c):
    v = _spread(c["len_lo"], c["len_hi"], c["B"], 17)
    return [max(n, m) for n, m in zip(v, _rows(c))] if c["op"] == "write" else v


def _rows(c):
    if c["op"] == "read":
        return _lengths(c)
    return _spread(c["rows_lo"], c["rows_hi"], c["B"], 5)


def _back(c):
    """Rows a write case reads back: from the start of the first block that it touched."""
    return [n - (n - m) // c["T"] * c["T"] for n, m in zip(_lengths(c), _rows(c))]


def work(c):
    e = 4.0 if c["dtype"] == "fp32" else 2.0
    if c["op"] == "norm":
        n = c["M"] * (c["Hq"] + c["Hk"]) * c["D"]
        turns = min(c["M"], c["positions"]) * c["rot"]
        return {"bytes": 2 * n * e + 4.0 * turns + 4.0 * c["M"] + 8.0 * c["D"], "flops": 4.0 * n + 3.0 * n * c["rot"] / c["D"]}
    lens, rows = _lengths(c), _rows(c)
    kv = 2.0 * c["Hkv"] * c["D"]
    scales = sum(-(-n // c["T"]) for n in lens) * 8.0 * c["Hkv"]
    if c["op"] == "write":
        back = sum(_back(c))
        return {"bytes": kv * (sum(rows) * e + back + back * 4.0) + 8.0 * c["Hkv"] * sum(-(-n // c["T"]) for n in _back(c)),
                "flops": kv * (3.0 * sum(rows) + back)}
    if c["op"] == "read":
        return {"bytes": kv * sum(lens) * (1 + e) + scales, "flops": kv * sum(lens)}
    pairs = 0
    for n, m in zip(lens, rows):
        if c["causal"]:
            seen = min(n, m)  # rows that see any token: they see n - seen + 1 .. n of them
            pairs += seen * (n - seen) + seen * (seen + 1) // 2
        else:
            pairs += m * n
    return {"bytes": kv * sum(lens) + scales + 2 * e * sum(rows) * c["H"] * c["D"], "flops": 4.0 * pairs * c["H"] * c["D"]}


# ---- inputs ----------------------------------------------------------------------------------------
def _starts(rows, dev):
    v = [0]
    for m in rows:
        v.append(v[-1] + m)
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _bytes_of(fmt, y):
    """8-bit codes nearest to y (64 bits, already over the scale), as the stored bytes."""
    if fmt == "int8":
        return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    # the spacing of the codes at y, a power of two made from its exponent bits
    unit = (((torch.frexp(y)[1] - 1).clamp(min=-6) - 3 + 1023).long() << 52).view(torch.float64)
    return ((y / unit).round() * unit).clamp(-448, 448).float().to(torch.float8_e4m3fn).view(torch.uint8)


def _codes(fmt, raw):
    """The values that stored bytes stand for before the scale, in 32 bits."""
    return raw.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 1000003 + 7)
    c, dt = case, DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if c["op"] == "norm":
        M, Hq, Hk, D, rot = c["M"], c["Hq"], c["Hk"], c["D"], c["rot"]
        width = (Hq + 2 * Hk) * D  # the packed projection: queries, keys and the values between calls
        step = 1e4 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / max(rot, 1))
        far = torch.arange(c["positions"], device=dev, dtype=torch.float64)[:, None] * step
        s = {"x": (normal(M, width) * torch.exp(0.5 * normal(M, 1))).to(dt), "wq": 1 + 0.2 * normal(D), "wk": 1 + 0.2 * normal(D),
             "turns": torch.cat([far.cos(), far.sin()], 1).float().contiguous(),
             "q": torch.empty(M, Hq * D, device=dev, dtype=dt), "k": torch.empty(M, Hk * D, device=dev, dtype=dt)}
        if c["positions"] <= M:  # whole images one after the other
            s["pos"] = (torch.arange(M, device=dev) % c["positions"]).int()
        else:
            s["pos"] = torch.randint(0, c["positions"], (M,), generator=g, device=dev, dtype=torch.int32)
        s["case"] = c
        return s
    lens, rows = _lengths(c), _rows(c)
    B, Hkv, D, T, fmt = c["B"], c["Hkv"], c["D"], c["T"], c["format"]
    wide = max(-(-n // T) for n in lens)
    used = [-(-n // T) for n in lens]
    blocks = sum(used) + 3  # the pool: three blocks belong to nobody
    order = torch.randperm(blocks - 1, generator=g, device=dev).int()
    table = torch.zeros(B, wide, dtype=torch.int32)
    at, order_h = 0, order.cpu()
    for b, n in enumerate(used):
        table[b, :n] = order_h[at:at + n]
        at += n
    s = {"case": c, "table": table.to(dev), "lengths": torch.tensor(lens, dtype=torch.int32, device=dev),
         "start": _starts(rows, dev), "rows": sum(rows), "max_rows": max(rows), "max_len": max(lens), "blocks": blocks}
    for name in ("k", "v"):
        # channels of unlike size, and blocks of unlike size, as a model's keys and values have them
        channel = torch.exp(0.4 * normal(Hkv, 1, D))
        raw = torch.empty(blocks, Hkv, T, D, dtype=torch.uint8, device=dev)
        scale = torch.empty(blocks, Hkv, device=dev)
        piece = max(1, 2 ** 25 // (Hkv * T * D))
        for i in range(0, blocks, piece):
            n = min(piece, blocks - i)
            x = normal(n, Hkv, T, D) * channel * torch.exp(0.3 * normal(n, Hkv, 1, 1))
            sc = x.abs().amax((2, 3)).clamp(min=FLOOR) * (1.0 / QMAX[fmt])
            raw[i:i + n] = _bytes_of(fmt, x.double() * sc.reciprocal()[:, :, None, None])
            scale[i:i + n] = sc
        s[name + "_codes"], s[name + "_scale"] = raw, scale
        if c["op"] == "write":
            s[name] = (normal(s["rows"], Hkv, D) * channel[None, :, 0] * torch.exp(0.3 * normal(s["rows"], 1, 1))).reshape(s["rows"], Hkv * D).to(dt)
    if c["op"] == "attend":
        s["q"] = normal(s["rows"], c["H"] * D).to(dt)
        s["out"] = torch.zeros(s["rows"], c["H"] * D, device=dev, dtype=dt)
    if c["op"] == "write":
        back = _back(c)
        s["back_start"], s["back_rows"], s["back_max"] = _starts(back, dev), sum(back), max(back)
    if c["op"] in ("write", "read"):
        n, to = (s["back_rows"], torch.float32) if c["op"] == "write" else (s["rows"], dt)
        s["k_out"], s["v_out"] = (torch.empty(n, Hkv * D, device=dev, dtype=to) for _ in range(2))
    return s


# ---- the framework's calls --------------------------------------------------------------------------
_gpu = None


def _context():
    """The program's one context, on torch's current stream."""
    global _gpu
    if _gpu is None:
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "supra2-img-web_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import supra_attn

        _gpu = supra_attn.GPU(torch.cuda.current_device(), stream=torch.cuda.current_stream())
    return _gpu


def _run_own(s):
    gpu = _context()
    import supra_attn

    c = s["case"]
    if c["op"] == "norm":
        M, Hq, Hk, D = c["M"], c["Hq"], c["Hk"], c["D"]
        width = (Hq + 2 * Hk) * D
        supra_attn.qk_norm(gpu, q=s["x"], k=s["x"], M=M, Hq=Hq, Hk=Hk, D=D, ldq=width, ldk=width, kOff=Hq * D, qOut=s["q"],
                           kOut=s["k"], wq=s["wq"], wk=s["wk"], eps=1e-6, turns=s["turns"] if c["rot"] else None, rot=c["rot"],
                           positions=s["pos"] if c["rot"] else None, interleaved=c["interleaved"])
        gpu.flush()
        return s["q"], s["k"]
    cache = supra_attn.KVCache(gpu, s["blocks"], c["Hkv"], c["D"], block_tokens=c["T"], format=c["format"], k=s["k_codes"],
                               v=s["v_codes"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    seqs = supra_attn.CacheBatch(gpu, s["lengths"], s["table"], row_start=s["start"], rows=s["rows"], max_rows=s["max_rows"],
                                 max_len=s["max_len"])
    if c["op"] == "attend":
        supra_attn.cache_attention(gpu, cache, seqs, q=s["q"], out=s["out"], H=c["H"], causal=c["causal"])
        gpu.flush()
        return s["out"]
    if c["op"] == "read":
        supra_attn.cache_read(gpu, cache, seqs, k=s["k_out"], v=s["v_out"])
        gpu.flush()
        return s["k_out"], s["v_out"]
    supra_attn.cache_write(gpu, cache, seqs, k=s["k"], v=s["v"])
    back = supra_attn.CacheBatch(gpu, s["lengths"], s["table"], row_start=s["back_start"], rows=s["back_rows"],
                                 max_rows=s["back_max"], max_len=s["max_len"])
    supra_attn.cache_read(gpu, cache, back, k=s["k_out"], v=s["v_out"])
    gpu.flush()
    return s["k_out"], s["v_out"], s["k_scale"], s["v_scale"]


# ---- the plain forms ---------------------------------------------------------------------------------
def _norm(x, w, c, turns):
    """x [M, heads, D] in 32 bits: RMS norm, weight, rotation of the first `rot` channels."""
    y = x * (x.square().mean(-1, keepdim=True) + 1e-6).sqrt().reciprocal() * w
    rot = c["rot"]
    if not rot:
        return y
    co, si = turns[:, None, :rot // 2], turns[:, None, rot // 2:]
    if c["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        t = torch.stack([a * co - b * si, b * co + a * si], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        t = torch.cat([a * co - b * si, b * co + a * si], -1)
    return torch.cat([t, y[..., rot:]], -1)


def _read(s, start, rows, to):
    """The last rows of every sequence, read back: (k, v)."""
    c, T = s["case"], s["case"]["T"]
    r = torch.arange(rows, device=start.device)
    b = torch.searchsorted(start[1:].long(), r, right=True)
    token = s["lengths"].long()[b] - start.long()[b + 1] + r
    page, slot = s["table"].long()[b, token // T], token % T
    return tuple((_codes(c["format"], s[n + "_codes"])[page, :, slot] * s[n + "_scale"][page][:, :, None]).flatten(1).to(to)
                 for n in ("k", "v"))


def _write(s, name):
    """Quantises s[name]'s rows into the cache's blocks, all touched blocks at once."""
    c, T, fmt = s["case"], s["case"]["T"], s["case"]["format"]
    start, lens = s["start"].long(), s["lengths"].long()
    rows = start[1:] - start[:-1]
    first = lens - rows
    base = first // T * T
    n_blocks = (s["max_rows"] + 2 * T - 2) // T
    token = base[:, None] + torch.arange(n_blocks * T, device=start.device)
    new = (token >= first[:, None]) & (token < lens[:, None])
    row = (start[:-1, None] + token - first[:, None]).clamp(0, s["rows"] - 1)
    B = lens.numel()
    x = s[name].float().view(s["rows"], c["Hkv"], c["D"])[row]
    x = x.view(B, n_blocks, T, c["Hkv"], c["D"]).transpose(2, 3)
    new = new.view(B, n_blocks, 1, T, 1)
    touched = new.flatten(2).any(2)
    place = (token[:, ::T] // T).clamp(max=s["table"].shape[1] - 1)
    # blocks that are not touched stand for the pool's last one, which keeps what it has
    page = torch.where(touched, s["table"].long().gather(1, place), s["blocks"] - 1)
    old = _codes(fmt, s[name + "_codes"][page])
    old_scale = s[name + "_scale"][page]
    amax = torch.where(new, x.abs(), 0.0).amax((3, 4))
    held = (token < first[:, None]).view(B, n_blocks, 1, T, 1)
    scale = amax.clamp(min=FLOOR) * (1.0 / QMAX[fmt])
    scale = torch.where(held.flatten(2).any(2)[:, :, None], torch.maximum(scale, old_scale), scale)
    scale = torch.where(touched[:, :, None], scale, old_scale)
    inv, again = scale.reciprocal()[..., None, None], (old_scale / scale)[..., None, None]
    grown = (scale > old_scale)[..., None, None]
    old = old.double()
    codes = torch.where(new, x.double() * inv, torch.where(held & grown, old * again, old))
    s[name + "_codes"][page] = _bytes_of(fmt, codes)
    s[name + "_scale"][page] = scale


def _attend(s):
    c, T, H, Hkv, D = (s["case"][n] if n != "case" else s["case"] for n in ("case", "T", "H", "Hkv", "D"))
    start, lens, m = s["start"].long(), s["lengths"].long(), s["max_rows"]
    B, L = lens.numel(), s["table"].shape[1] * T
    rows = start[1:] - start[:-1]
    page = s["table"].long()

    def heads(n):  # [B, Hkv, L, D]
        x = _codes(c["format"], s[n + "_codes"][page]) * s[n + "_scale"][page][..., None, None]
        return x.transpose(1, 2).reshape(B, Hkv, L, D)

    at = start[:-1, None] + torch.arange(m, device=start.device)
    q = s["q"].float()[at.clamp(max=s["rows"] - 1)].view(B, m, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, H // Hkv * m, D)
    z = (q @ heads("k").transpose(2, 3)) * (1.0 / math.sqrt(D))
    z = z.view(B, Hkv, H // Hkv, m, L)
    j = torch.arange(L, device=start.device)
    seen = (j < lens[:, None])[:, None, :]
    if c["causal"]:
        i = torch.arange(m, device=start.device)
        seen = seen & (j <= (lens - rows)[:, None, None] + i[:, None])
    seen = seen[:, None, None]
    top = torch.where(seen, z, -math.inf).amax(-1, keepdim=True)
    p = torch.where(seen, (z - top).exp(), 0.0)
    del z
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hkv, H // Hkv * m, L) @ heads("v")).view(B, Hkv, H // Hkv, m, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, m, H * D)
    r = torch.arange(s["rows"], device=start.device)
    b = torch.searchsorted(start[1:], r, right=True)
    return o[b, r - start[b]].to(s["out"].dtype)


def run(state):
    s = state
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "attend":
        return _attend(s)
    if c["op"] == "read":
        return _read(s, s["start"], s["rows"], DTYPES[c["dtype"]])
    if c["op"] == "write":
        _write(s, "k")
        _write(s, "v")
        return (*_read(s, s["back_start"], s["back_rows"], torch.float32), s["k_scale"], s["v_scale"])
    M, Hq, Hk, D = c["M"], c["Hq"], c["Hk"], c["D"]
    turns = s["turns"][s["pos"].long()]
    x = s["x"].float().view(M, Hq + 2 * Hk, D)
    return tuple(_norm(x[:, a:a + n], s[w], c, turns).flatten(1).to(s["x"].dtype) for a, n, w in ((0, Hq, "wq"), (Hq, Hk, "wk")))


# ---- the definitions in 64 bits, one sequence and one block at a time ---------------------------------
def _exact_norm(c, s):
    M, D, half = c["M"], c["D"], c["rot"] // 2
    got = []
    pos = s["pos"].double()
    for lo, n, w in ((0, c["Hq"], s["wq"]), (c["Hq"], c["Hk"], s["wk"])):
        x = s["x"].double()[:, lo * D:(lo + n) * D].reshape(M, n, D)
        y = w.double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6)
        z = y.clone()
        for i in range(half):
            # the rotation is by the table's values, which are inputs
            a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, half + i)
            co, si = s["turns"].double()[pos.long(), i][:, None], s["turns"].double()[pos.long(), half + i][:, None]
            z[..., a] = y[..., a] * co - y[..., b] * si
            z[..., b] = y[..., a] * si + y[..., b] * co
        got.append(z.reshape(M, n * D))
    return tuple(got)


def _value64(fmt, raw):
    b = raw.to(torch.int64)
    if fmt == "int8":
        return torch.where(b > 127, b - 256, b).double()
    e, f = (b >> 3) & 15, (b & 7).double()
    mag = torch.where(e == 0, f * 2.0 ** -9, (8 + f) * torch.pow(2.0, (e - 10).double()))
    return torch.where(b > 127, -mag, mag)


def _nearest64(fmt, y):
    if fmt == "int8":
        return torch.round(y).clamp(-127, 127)
    powers = torch.tensor([2.0 ** i for i in range(-6, 10)], dtype=torch.float64, device=y.device)
    # the last power of two at or below |y|, over 8
    unit = powers[(torch.bucketize(y.abs(), powers, right=True) - 1).clamp(min=0)] / 8
    return (torch.round(y / unit) * unit).clamp(-448, 448)


def _exact_write(c, s):
    H, D, T, fmt = c["Hkv"], c["D"], c["T"], c["format"]
    top = float(torch.tensor(1 / QMAX[fmt], dtype=torch.float32))
    lens, rows, table = _lengths(c), _rows(c), s["table"].cpu()
    values, scales = {}, {}
    for name in ("k", "v"):
        scale = s[name + "_scale"].double()
        x_all, done, r0 = s[name].double().view(-1, H, D), [], 0
        for b in range(c["B"]):
            first = lens[b] - rows[b]
            for n in range(first // T, -(-lens[b] // T)):
                page = int(table[b, n])
                lo, hi = max(first, n * T), min(lens[b], n * T + T)
                x = x_all[r0 + lo - first:r0 + hi - first].transpose(0, 1)
                sc = (x.abs().amax((1, 2)).clamp(min=FLOOR) * top).float().double()
                had = _value64(fmt, s[name + "_codes"][page, :, :lo - n * T])
                if lo > n * T:
                    before = scale[page].clone()
                    sc = torch.maximum(sc, before)
                    had = torch.where((sc > before)[:, None, None], _nearest64(fmt, had * (before / sc).float().double()[:, None, None]), had)
                new = _nearest64(fmt, x * (1 / sc).float().double()[:, None, None])
                scale[page] = sc
                done.append((torch.cat([had, new], 1) * sc[:, None, None]).transpose(0, 1).reshape(hi - n * T, H * D))
            r0 += rows[b]
        values[name], scales[name] = torch.cat(done), scale
    return values["k"], values["v"], scales["k"], scales["v"]


def _exact_read(c, s):
    got = []
    for name in ("k", "v"):
        rows = []
        for b, n in enumerate(_lengths(c)):
            page = s["table"][b, :-(-n // c["T"])].long()
            x = _value64(c["format"], s[name + "_codes"][page]) * s[name + "_scale"].double()[page][:, :, None, None]
            rows.append(x.permute(0, 2, 1, 3).reshape(-1, c["Hkv"] * c["D"])[:n])
        got.append(torch.cat(rows))
    return tuple(got)


def _exact_attend(c, s):
    H, Hkv, D, out, r0 = c["H"], c["Hkv"], c["D"], [], 0
    for b, (n, m) in enumerate(zip(_lengths(c), _rows(c))):
        page = s["table"][b, :-(-n // c["T"])].long()
        q = s["q"][r0:r0 + m].double().view(m, H, D)
        o = torch.zeros(m, H, D, dtype=torch.float64, device=q.device)
        for h in range(Hkv):
            k, v = ((_value64(c["format"], s[x + "_codes"][page, h]) * s[x + "_scale"].double()[page, h][:, None, None]).reshape(-1, D)[:n]
                    for x in ("k", "v"))
            for i in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                z = q[:, i] @ k.T / math.sqrt(D)
                if c["causal"]:
                    ban = torch.arange(n, device=q.device) > (n - m + torch.arange(m, device=q.device))[:, None]
                    z = z.masked_fill(ban, -math.inf)
                o[:, i] = torch.nan_to_num(torch.softmax(z, -1), nan=0.0) @ v
        out.append(o.view(m, H * D))
        r0 += m
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "write": _exact_write, "read": _exact_read, "attend": _exact_attend}[case["op"]](case, s)
