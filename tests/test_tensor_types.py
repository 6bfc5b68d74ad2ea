"""Tensors of other element types than fp32: GPU.write stays inside them and writes their own values. Device memory is
stood in for by host memory, with guards on both sides of every tensor."""

import ctypes as C

import numpy as np
import pytest

import supra_attn
from supra_attn import _lib, ops

GUARD = 4096


class HostMemory:
    """The library's copies on host memory; everything else is refused."""

    def __init__(self):
        self.bytes = np.full(1 << 16, 0xa5, np.uint8)

    def supra_attn_upload(self, ctx, dst, src, n):
        return self.supra_attn_upload_bytes(ctx, dst, src, 4 * n)

    def supra_attn_upload_bytes(self, ctx, dst, src, n):
        first = dst.value - self.bytes.ctypes.data
        assert 0 <= first and first + n <= self.bytes.size
        C.memmove(dst, src, n)
        return _lib.OK


@pytest.fixture
def host(monkeypatch):
    mem = HostMemory()
    monkeypatch.setattr(ops, "lib", mem)
    gpu = ops.GPU.__new__(ops.GPU)
    gpu.ctx, gpu.device, gpu._held = None, 0, []
    return gpu, mem


def tensor(host, n, dtype):
    gpu, mem = host
    return ops.Tensor(gpu, mem.bytes.ctypes.data + GUARD, [n], n, owned=False, dtype=dtype)


VALUES = {"fp32": [1.5, -2.25, np.inf], "fp16": np.array([1.5, -np.inf, np.nan], np.float16), "bf16": np.array([0x7fc0, 1, 0x3f80], np.uint16),
          "int32": [7, -1, (1 << 31) - 1], "uint8": [0, 255, 3]}


@pytest.mark.parametrize("n", [3, 1024])
@pytest.mark.parametrize("offset", [0, 1, 2, 5])
@pytest.mark.parametrize("dtype", sorted(ops.DTYPES))
def test_write_keeps_to_its_elements(host, dtype, offset, n):
    t = tensor(host, offset + n, dtype)
    size = np.dtype(ops.DTYPES[dtype]).itemsize
    values = np.resize(np.asarray(VALUES[dtype]), n)
    want = host[1].bytes.copy()
    at = GUARD + offset * size
    want[at:at + n * size] = values.astype(ops.DTYPES[dtype]).view(np.uint8)
    host[0].write(t, values, offset)
    np.testing.assert_array_equal(host[1].bytes, want)


@pytest.mark.parametrize("dtype", sorted(ops.DTYPES))
def test_write_refuses_what_does_not_fit(host, dtype):
    gpu, mem = host
    t = tensor(host, 8, dtype)
    before = mem.bytes.copy()
    for a, offset in ((np.zeros(9), 0), (np.zeros(1), 8), (np.zeros(8), 1), (np.zeros(1), -1)):
        with pytest.raises(ValueError, match="out of bounds"):
            gpu.write(t, a, offset)
    t.release()
    with pytest.raises(ValueError, match="released"):
        gpu.write(t, np.zeros(1))
    np.testing.assert_array_equal(mem.bytes, before)


@pytest.mark.parametrize("dtype,value", [("int32", 1.5), ("int32", 1 << 31), ("uint8", -1), ("uint8", 256), ("fp16", 1e-9), ("fp16", 1e6), ("bf16", 0.5)])
def test_write_refuses_values_that_the_type_does_not_hold(host, dtype, value):
    t = tensor(host, 4, dtype)
    before = host[1].bytes.copy()
    with pytest.raises(ValueError, match="does not hold"), np.errstate(all="ignore"):
        host[0].write(t, [0, value])
    np.testing.assert_array_equal(host[1].bytes, before)


# ---- on the device ----------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(ops.DTYPES))
def test_write_and_read_back(gpu, dtype):
    for offset in (0, 1, 3):
        t = gpu.from_array(np.arange(21) % 3, dtype=dtype) if dtype != "fp32" else gpu.from_array(np.arange(21) % 3)
        want = gpu.read(t).copy()
        values = np.resize(np.asarray(VALUES[dtype]), 7).astype(ops.DTYPES[dtype])
        want[offset:offset + 7] = values
        gpu.write(t, values, offset)
        assert gpu.read(t).tobytes() == want.tobytes()
        t.release()


@pytest.mark.gpu
def test_lengths_and_tables_change_in_place(gpu):
    """Without torch: a step after each change reads what is there then."""
    cache = supra_attn.KVCache(gpu, 3, 1, 16, block_tokens=16)
    lengths = gpu.from_array(np.array([0]), dtype="int32")
    table = gpu.from_array(np.array([[2, 0]]), [1, 2], dtype="int32")
    seqs = supra_attn.CacheBatch(gpu, lengths, table)
    row = gpu.empty([1, 16])
    for n in range(1, 20):
        gpu.write(lengths, [n])
        if n == 17:
            gpu.write(table, [1], 1)
        gpu.write(row, np.full(16, float(n)))
        supra_attn.cache_write(gpu, cache, seqs, k=row, v=row)
    gpu.write(lengths, [16])
    q = gpu.from_array(np.zeros(16), [1, 16])
    first = gpu.read(supra_attn.cache_attention(gpu, cache, seqs, q=q, H=1))
    gpu.write(lengths, [19])
    whole = gpu.read(supra_attn.cache_attention(gpu, cache, seqs, q=q, H=1))
    # (equal scores: means; a code is off by at most half of the block's largest value / 127, once more where the scale grew)
    assert np.abs(first - np.arange(1, 17).mean()).max() <= 16 * 16 / 254
    assert np.abs(whole - np.arange(1, 20).mean()).max() <= 19 * 16 / 254
    codes = gpu.read(cache.k).reshape(3, 16, 16)
    assert (codes[2, 15] == 127).all() and (codes[1, 2] == 127).all()
