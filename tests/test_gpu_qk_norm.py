"""The query/key norm with rotation on the GPU against the 64-bit restatement (oracle/cache.py)."""

import numpy as np
import pytest
import torch

import supra_attn
from oracle import cache as oc

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# With u = 2^-24 the sum of squares is off by at most 13 u (8 terms a lane, 5 exchanges), its mean plus eps by
# 3 more, 1 / sqrt of it by 8 + 2, the two products by 2; the rotation's product and sum add 2. All are
# relative to |n_a| + |n_b|: 16 u holds it. The result's own rounding is eps / 2 of its type; fp16 numbers
# below 2^-14 are 2^-24 apart, so theirs is up to 2^-25 however small they are.
def bound(dtype, ref, mag):
    err = 16 * 2.0 ** -24 * mag
    return err + torch.finfo(TYPES[dtype]).eps / 2 * (np.abs(ref) + err) + 2.0 ** -25 * (dtype == "fp16")


def check(gpu, dtype, M, Hq, Hk, D, rot, interleaved, inplace=False, weights=True, norm=True, n_turns=300, positions=True, pad=0, off=0,
          seed=0):
    rng = np.random.default_rng(seed + M + D + rot)
    dt = TYPES[dtype]
    width = (Hq + Hk) * D + pad
    x = (torch.from_numpy(rng.standard_normal(M * width + off).astype(np.float32)) * 3).to(dt).cuda()
    keep = x.clone()
    wq = torch.from_numpy(rng.standard_normal(D).astype(np.float32)).cuda() if weights else None
    wk = torch.from_numpy(rng.standard_normal(D).astype(np.float32)).cuda() if weights else None
    turns = pos = None
    if rot:
        ang = rng.uniform(-4, 4, (n_turns, rot // 2))
        turns = torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)).cuda()
        pn = rng.integers(0, n_turns, M).astype(np.int32) if positions else np.arange(M, dtype=np.int32)
        pos = torch.from_numpy(pn).cuda() if positions else None
    kw = dict(q=x, M=M, Hq=Hq, D=D, ldq=width, qOff=off, wq=wq, norm=norm, turns=turns, rot=rot, positions=pos, interleaved=interleaved)
    qo = ko = None
    if Hk:
        kw.update(k=x, Hk=Hk, ldk=width, kOff=off + Hq * D, wk=wk)
    if not inplace:
        qo = torch.full((M * (Hq * D + pad) + off,), 9.0, dtype=dt, device="cuda")
        kw.update(qOut=qo, ldqOut=Hq * D + pad, qOutOff=off)
        if Hk:
            ko = torch.full((M * (Hk * D + pad) + off,), 9.0, dtype=dt, device="cuda")
            kw.update(kOut=ko, ldkOut=Hk * D + pad, kOutOff=off)
    supra_attn.qk_norm(gpu, **kw)
    gpu.sync()
    xn = keep.cpu().double().numpy()[off:].reshape(M, width)
    for lo, H, w, out in ((0, Hq, wq, qo), (Hq, Hk, wk, ko)):
        if H == 0:
            continue
        ref, mag = oc.qk_norm(xn[:, lo * D:(lo + H) * D].reshape(M, H, D), w.cpu().double().numpy() if w is not None else None, 1e-6, norm,
                              turns.cpu().numpy() if rot else None, rot, pn if rot else None, interleaved)
        if inplace:
            got = x.cpu().double().numpy()[off:].reshape(M, width)[:, lo * D:(lo + H) * D]
        else:
            o = out.cpu().double().numpy()
            assert (o[:off] == 9).all() and (o[off:].reshape(M, -1)[:, H * D:] == 9).all()
            got = o[off:].reshape(M, -1)[:, :H * D]
        err, tol = np.abs(got.reshape(M, H, D) - ref), bound(dtype, ref, mag)
        assert (err <= tol).all(), f"worst {np.max(err / tol):.3g} of the bound"
    if inplace:  # nothing beside the heads moved
        assert torch.equal(x[:off], keep[:off])
        assert torch.equal(x[off:].view(M, width)[:, (Hq + Hk) * D:], keep[off:].view(M, width)[:, (Hq + Hk) * D:])
    else:
        assert torch.equal(x, keep)


CASES = [
    # M, Hq, Hk, D, rot, interleaved
    (1, 1, 1, 64, 64, False),
    (300, 9, 9, 64, 64, True),
    (61, 32, 8, 128, 96, False),
    (7, 6, 2, 128, 128, True),
    (33, 3, 1, 16, 16, False),
    (5, 4, 4, 80, 0, False),
    (17, 5, 0, 48, 32, False),
    (9, 2, 1, 256, 64, False),
    (9, 2, 1, 256, 256, True),
    (40, 3, 3, 34, 22, False),   # odd head sizes
    (40, 3, 2, 2, 2, True),
    (13, 2, 2, 96, 6, False),
    (3000, 2, 1, 32, 32, False),
]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(int(x)) for x in c))
def test_qk_norm(gpu, case, inplace, dtype):
    check(gpu, dtype, *case, inplace=inplace)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_qk_norm_options(gpu, dtype):
    check(gpu, dtype, 50, 4, 2, 64, 64, False, weights=False)
    check(gpu, dtype, 50, 4, 2, 64, 64, False, weights=False, norm=False)
    check(gpu, dtype, 50, 4, 2, 64, 32, True, weights=False, norm=False, inplace=True)
    check(gpu, dtype, 50, 4, 2, 64, 64, False, positions=False)
    check(gpu, dtype, 50, 4, 2, 64, 64, False, pad=8, off=16)
    check(gpu, dtype, 50, 4, 2, 64, 64, False, pad=3, off=5)           # unaligned rows
    check(gpu, dtype, 50, 4, 2, 64, 64, True, pad=1, off=1, inplace=True)


def test_zero_rows_and_huge_rows(gpu):
    """A row of zeros stays zero; rows near the ends of the fp32 range follow fp32 arithmetic."""
    x = torch.zeros(4, 64, device="cuda")
    x[1] = 1e-18
    x[2] = 1e18
    x[3, 5] = float("nan")
    y = torch.empty_like(x)
    supra_attn.qk_norm(gpu, q=x, M=4, Hq=1, D=64, qOut=y, eps=0.0)
    supra_attn.qk_norm(gpu, q=x, M=1, Hq=1, D=64, eps=1e-6)  # in place
    gpu.sync()
    y = y.cpu()
    assert torch.isnan(y[0]).all()  # 0 / 0 without eps
    assert (x[0] == 0).all()
    assert (y[1] - 1).abs().max() <= 16 * 2.0 ** -24 and (y[2] - 1).abs().max() <= 16 * 2.0 ** -24
    assert torch.isnan(y[3]).all()


def test_position_outside_the_table(gpu):
    x = torch.randn(6, 64, device="cuda")
    y = torch.full_like(x, 9.0)
    turns = supra_attn.rotation_turns(gpu, np.arange(10), 64)
    for bad in (10, -1):
        pos = torch.tensor([0, 1, bad, 9, 4, 5], dtype=torch.int32, device="cuda")
        supra_attn.qk_norm(gpu, q=x, M=6, Hq=1, D=64, qOut=y, turns=turns, rot=64, positions=pos)
        with pytest.raises(supra_attn.SupraAttnError, match="row 2"):
            gpu.sync()
        assert gpu.sync() == 0
        assert (y[2] == 9).all() and (y[[0, 1, 3, 4, 5]] != 9).any(dim=1).all()
    turns.release()


def test_rotation_turns(gpu):
    t = gpu.read(supra_attn.rotation_turns(gpu, [0, 1, 131071], 96)).reshape(3, 96)
    ang = np.array([0, 1, 131071])[:, None] * 10000.0 ** (-np.arange(0, 96, 2) / 96)
    assert np.abs(t - np.concatenate([np.cos(ang), np.sin(ang)], 1)).max() <= 2.0 ** -24
    grid = np.stack(np.meshgrid(np.arange(4), np.arange(4), indexing="ij"), -1).reshape(16, 2)  # a patch grid
    t = gpu.read(supra_attn.rotation_turns(gpu, grid, 32)).reshape(16, 32)
    assert np.allclose(t[7, :8], np.cos(1 * 10000.0 ** (-np.arange(0, 16, 2) / 16))) and np.allclose(
        t[7, 8:16], np.cos(3 * 10000.0 ** (-np.arange(0, 16, 2) / 16)))
    with pytest.raises(ValueError):
        supra_attn.rotation_turns(gpu, grid, 30)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 50), (128, 30), (80, 36), (128, 126), (16, 4), (64, 2), (96, 94)])
def test_rotations_that_are_not_whole_pieces(gpu, D, rot, inplace, interleaved, dtype):
    check(gpu, dtype, 37, 5, 2, D, rot, interleaved, inplace=inplace, seed=7)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_table_that_is_not_aligned(gpu, dtype):
    rng = np.random.default_rng(8)
    M, H, D = 21, 3, 64
    flat = torch.from_numpy(rng.uniform(-1, 1, 1 + 30 * D).astype(np.float32)).cuda()
    turns = flat[1:].view(30, D)
    x = torch.from_numpy(rng.standard_normal((M, H * D)).astype(np.float32)).to(TYPES[dtype]).cuda()
    y = torch.empty_like(x)
    supra_attn.qk_norm(gpu, q=x, M=M, Hq=H, D=D, qOut=y, turns=turns, rot=D)
    gpu.sync()
    ref, mag = oc.qk_norm(x.cpu().double().numpy().reshape(M, H, D), None, 1e-6, True, turns.cpu().numpy(), D, np.arange(M), False)
    assert (np.abs(y.cpu().double().numpy().reshape(M, H, D) - ref) <= bound(dtype, ref, mag)).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [32, 10])
def test_channels_that_do_not_turn_are_left_alone(gpu, rot, interleaved):
    """Without a norm they come out as they went in, infinities and NaN among them."""
    M, H, D = 9, 3, 64
    x = torch.randn(M, H, D, device="cuda")
    x[:, :, rot] = float("inf")
    x[:, :, D - 1] = float("nan")
    x[:, :, rot + 1:rot + 3] = 3e38
    y = torch.zeros_like(x)
    turns = supra_attn.rotation_turns(gpu, np.arange(M), rot)
    supra_attn.qk_norm(gpu, q=x, M=M, Hq=H, D=D, qOut=y, norm=False, turns=turns, rot=rot, interleaved=interleaved)
    gpu.sync()
    torch.cuda.synchronize()
    assert torch.equal(y[:, :, rot:].nan_to_num(nan=5.0), x[:, :, rot:].nan_to_num(nan=5.0))
    assert torch.isfinite(y[:, :, :rot]).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_weights_of_one_operand_only(gpu, dtype):
    rng = np.random.default_rng(9)
    M, Hq, Hk, D = 50, 3, 3, 64  # (a warp's heads pass from the queries to the keys in the middle of a group)
    x = torch.from_numpy(rng.standard_normal((M, (Hq + Hk) * D)).astype(np.float32)).to(TYPES[dtype]).cuda()
    w = torch.from_numpy(rng.standard_normal(D).astype(np.float32)).cuda()
    turns = torch.from_numpy(rng.uniform(-1, 1, (M, D)).astype(np.float32)).cuda()
    for wq, wk in ((w, None), (None, w), (w, w)):
        q, k = torch.empty(M, Hq * D, dtype=x.dtype, device="cuda"), torch.empty(M, Hk * D, dtype=x.dtype, device="cuda")
        supra_attn.qk_norm(gpu, q=x, k=x, M=M, Hq=Hq, Hk=Hk, D=D, ldq=(Hq + Hk) * D, ldk=(Hq + Hk) * D, kOff=Hq * D, qOut=q, kOut=k, wq=wq, wk=wk,
                           turns=turns, rot=D)
        gpu.sync()
        xn = x.cpu().double().numpy().reshape(M, Hq + Hk, D)
        for lo, h, ww, out in ((0, Hq, wq, q), (Hq, Hk, wk, k)):
            ref, mag = oc.qk_norm(xn[:, lo:lo + h], ww.cpu().double().numpy() if ww is not None else None, 1e-6, True, turns.cpu().numpy(), D,
                                  np.arange(M), False)
            assert (np.abs(out.cpu().double().numpy().reshape(M, h, D) - ref) <= bound(dtype, ref, mag)).all()
