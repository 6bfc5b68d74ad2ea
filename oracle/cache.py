"""The paged 8-bit K/V cache, attention over it and the query/key norm, restated on the CPU in 64 bits.

Plain loops over sequences and blocks, from the definitions in include/supra_attn.h; only the tests
use it. The numbers that the definition holds in fp32 (scales, reciprocals, ratios) are fp32 here too,
so codes and scales are compared bit for bit.
"""

import numpy as np
import torch

QMAX = {"int8": 127.0, "e4m3": 448.0}
FLOOR = np.float32(2.0 ** -100)


def _e4m3_values():
    v = np.zeros(256)
    for b in range(256):
        e, f = (b >> 3) & 15, b & 7
        x = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        if e == 15 and f == 7:
            x = np.nan
        v[b] = -x if b & 0x80 else x
    return v


E4M3 = _e4m3_values()


def decode(fmt, raw):
    """Stored bytes -> the codes' values, float64."""
    raw = np.asarray(raw, dtype=np.uint8)
    return raw.view(np.int8).astype(np.float64) if fmt == "int8" else E4M3[raw]


def nearest(fmt, x):
    """float64 -> the bytes of the nearest codes, ties to even."""
    x = np.asarray(x, dtype=np.float64)
    if fmt == "int8":
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    mag = np.minimum(np.abs(x), 448.0)
    unit = np.exp2(np.maximum(np.frexp(mag)[1] - 1, -6) - 3)
    mag = np.rint(mag / unit) * unit
    codes = np.searchsorted(E4M3[:127], mag)
    assert np.array_equal(E4M3[codes], mag)
    return (codes | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def write(fmt, codes, scale, rows, lengths, row_start, table):
    """Quantises rows [R, H, D] (float64) into codes [blocks, H, T, D] (uint8) and scale [blocks, H]
    (float32), in place."""
    T = codes.shape[2]
    for b in range(len(lengths)):
        n = row_start[b + 1] - row_start[b]
        first = lengths[b] - n
        if n == 0:
            continue
        for j in range(first // T, (lengths[b] - 1) // T + 1):
            p = table[b][j]
            lo, hi = max(first - j * T, 0), min(lengths[b] - j * T, T)
            r0 = row_start[b] + j * T + lo - first
            x = rows[r0:r0 + hi - lo].transpose(1, 0, 2)
            for h in range(codes.shape[1]):
                top = np.abs(x[h]).max()
                old = scale[p, h]
                if not np.isfinite(x[h]).all() or (lo > 0 and not np.isfinite(old)):
                    scale[p, h] = np.nan
                    codes[p, h, lo:hi] = 0
                    continue
                s = max(np.float32(top), FLOOR) * np.float32(1.0 / QMAX[fmt])
                if lo > 0:
                    s = max(s, old)
                    if s > old:
                        codes[p, h, :lo] = nearest(fmt, decode(fmt, codes[p, h, :lo]) * np.float64(old / s))
                codes[p, h, lo:hi] = nearest(fmt, x[h] * np.float64(np.float32(1.0) / s))
                scale[p, h] = s


def read(fmt, codes, scale, lengths, row_start, table):
    """The rows' values [R, H, D] in float32 (one fp32 product each)."""
    T = codes.shape[2]
    out = np.zeros((row_start[-1],) + (codes.shape[1], codes.shape[3]), dtype=np.float32)
    for b in range(len(lengths)):
        n = row_start[b + 1] - row_start[b]
        for i in range(n):
            t = lengths[b] - n + i
            p = table[b][t // T]
            out[row_start[b] + i] = decode(fmt, codes[p, :, t % T]).astype(np.float32) * scale[p][:, None]
    return out


def attention(fmt, kc, ks, vc, vs, q, lengths, row_start, table, scale, causal):
    """q [R, H, D] float64 -> (out [R, H, D], sums of p|v| [R, H, D], what the smallest steps of p
    are worth [2, R, H, D], largest score term sum [R, H], largest |score| [R, H]), all float64; the last
    four bound rounding errors. Steps of p itself: sum |v|; steps of p times its V scale, relative to
    the row's largest: max(p v_scale) * sum |code|."""
    T, Hk = kc.shape[2], kc.shape[1]
    R, H, D = q.shape
    G = H // Hk
    out, pv, av = np.zeros((R, H, D)), np.zeros((R, H, D)), np.zeros((2, R, H, D))
    st, sm = np.zeros((R, H)), np.zeros((R, H))
    for b in range(len(lengths)):
        L, n = lengths[b], row_start[b + 1] - row_start[b]
        if L == 0 or n == 0:
            continue
        pages = [table[b][j] for j in range((L + T - 1) // T)]
        k = (decode(fmt, kc[pages]) * ks[pages].astype(np.float64)[:, :, None, None]).transpose(1, 0, 2, 3).reshape(Hk, -1, D)[:, :L]
        v = (decode(fmt, vc[pages]) * vs[pages].astype(np.float64)[:, :, None, None]).transpose(1, 0, 2, 3).reshape(Hk, -1, D)[:, :L]
        vc_of = decode(fmt, vc[pages]).transpose(1, 0, 2, 3).reshape(Hk, -1, D)[:, :L]
        vs_of = np.abs(np.repeat(vs[pages].astype(np.float64), T, axis=0).T[:, :L])
        for i in range(n):
            seen = min(L, L - n + i + 1) if causal else L
            if seen <= 0:
                continue
            r = row_start[b] + i
            for h in range(H):
                kk, vv = k[h // G, :seen], v[h // G, :seen]
                s = scale * (kk @ q[r, h])
                with np.errstate(invalid="ignore"):
                    p = np.exp(s - s.max())
                    p /= p.sum()
                out[r, h] = p @ vv
                pv[r, h] = p @ np.abs(vv)
                av[0, r, h] = np.abs(vv).sum(0)
                av[1, r, h] = (p * vs_of[h // G, :seen]).max() * np.abs(vc_of[h // G, :seen]).sum(0)
                st[r, h] = abs(scale) * (np.abs(kk) @ np.abs(q[r, h])).max()
                sm[r, h] = np.abs(s).max()
    return out, pv, av, st, sm


def qk_norm(x, w, eps, norm, turns, rot, positions, interleaved):
    """x [M, H, D] float64 -> (out, |n_a| + |n_b| of each channel's pair), float64."""
    n = x.copy()
    if norm:
        n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if w is not None:
            n = n * w
    y, mag = n.copy(), np.abs(n)
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, rot // 2 + i)
        c = turns[positions, i].astype(np.float64)[:, None]
        s = turns[positions, rot // 2 + i].astype(np.float64)[:, None]
        y[..., a] = n[..., a] * c - n[..., b] * s
        y[..., b] = n[..., b] * c + n[..., a] * s
        mag[..., a] = mag[..., b] = np.abs(n[..., a]) + np.abs(n[..., b])
    return y, mag


def to_type(x, dtype):
    """float64 / float32 array -> torch tensor of the type."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype)
