"""KVCache and CacheBatch use their operands as they are when a call is made. The library's recording is stood in for; no
memory is touched."""

import numpy as np
import pytest
import torch

import supra_attn
from supra_attn import _lib, cache as sc, ops

BASE = 0x7F0000000000


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if not name.startswith("supra_attn_enqueue_"):
            raise AttributeError(name)

        def record(ctx, ref):
            d = ref._obj
            self.calls.append((name, d.seqs.lengths, d.seqs.table, d.seqs.row_start, d.cache.k, d.cache.v, d.cache.k_scale, d.cache.v_scale))
            return _lib.OK

        return record


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(sc, "lib", r)
    gpu = ops.GPU.__new__(ops.GPU)
    gpu.ctx, gpu.device, gpu._held = None, -1, []  # (-1: where torch says that CPU tensors are)
    return gpu, r


NAMES = ("lengths", "table", "row_start", "k", "v", "k_scale", "v_scale")
SHAPES = {"lengths": [2], "table": [2, 3], "row_start": [3], "k": [6, 2, 16, 32], "v": [6, 2, 16, 32], "k_scale": [6, 2], "v_scale": [6, 2]}
KINDS = {"lengths": "int32", "table": "int32", "row_start": "int32", "k": "uint8", "v": "uint8", "k_scale": "fp32", "v_scale": "fp32"}


def build(gpu, x):
    c = supra_attn.KVCache(gpu, 6, 2, 32, block_tokens=16, k=x["k"], v=x["v"], k_scale=x["k_scale"], v_scale=x["v_scale"])
    return c, supra_attn.CacheBatch(gpu, x["lengths"], x["table"], row_start=x["row_start"], rows=4, max_rows=4)


def calls(gpu, c, b, rows):
    yield lambda: supra_attn.cache_write(gpu, c, b, k=rows, v=rows)
    yield lambda: supra_attn.cache_read(gpu, c, b, k=rows, v=rows)
    yield lambda: supra_attn.cache_attention(gpu, c, b, q=rows, H=2, out=rows)


@pytest.mark.parametrize("name", NAMES)
def test_released_operands_are_refused(recorder, name):
    gpu, r = recorder
    x = {n: ops.Tensor(gpu, BASE + i * 0x1000000, SHAPES[n], int(np.prod(SHAPES[n])), owned=False, dtype=KINDS[n]) for i, n in enumerate(NAMES)}
    rows = ops.Tensor(gpu, BASE - 0x1000000, [4, 64], 256, owned=False)
    c, b = build(gpu, x)
    for call in calls(gpu, c, b, rows):
        call()
    assert [a[1:] for a in r.calls] == [tuple(x[n].buf for n in NAMES)] * 3
    r.calls.clear()
    x[name].release()
    for call in calls(gpu, c, b, rows):
        with pytest.raises(ValueError, match=f"{name}: tensor was released"):
            call()
    assert not r.calls


@pytest.mark.parametrize("name", NAMES)
def test_operands_that_moved_are_found(recorder, name):
    """A torch tensor whose storage has been replaced is used where it is now."""
    gpu, r = recorder
    kinds = {"int32": torch.int32, "uint8": torch.uint8, "fp32": torch.float32}
    x = {n: torch.zeros(SHAPES[n], dtype=kinds[KINDS[n]]) for n in NAMES}
    rows = torch.zeros(4, 64)
    c, b = build(gpu, x)
    x[name].data = torch.ones_like(x[name])
    for call in calls(gpu, c, b, rows):
        call()
    assert [a[1:] for a in r.calls] == [tuple(x[n].data_ptr() for n in NAMES)] * 3
    r.calls.clear()
    x[name].data = torch.ones(SHAPES[name], dtype=torch.float64)
    for call in calls(gpu, c, b, rows):
        with pytest.raises(ValueError, match=name):
            call()
    assert not r.calls
