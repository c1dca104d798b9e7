"""Counts past 32 bits, which ctypes would cut, are refused before any of them reaches the library (run without a device)."""
import pytest

from helpers import twd

MANY = (1 << 32) + 3


def meta(*shape, dtype=None):
    import torch
    return torch.empty(*shape, device="meta", dtype=dtype or torch.bfloat16)


@pytest.mark.parametrize("shape", [(MANY, 1), (1, MANY), (1 << 32, 8)])
def test_matrices_with_counts_past_32_bits_are_refused(shape):
    import torch
    t = twd()
    ids = meta(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="table has 2\\^32"):
        t.embed(meta(*shape), ids)
    with pytest.raises(ValueError, match="x has 2\\^32"):
        t.fp8_quantize(meta(*shape))
    with pytest.raises(ValueError, match="x has 2\\^32"):
        t.mx_quantize(meta(*shape))
    with pytest.raises(ValueError, match="codes has 2\\^32"):
        t.Fp8Head(meta(*shape, dtype=torch.uint8), meta(1, 1, dtype=torch.float32))
    grad = t.EmbedGrad.__new__(t.EmbedGrad)
    grad.handle = None
    with pytest.raises(ValueError, match="d_rows has 2\\^32"):
        grad.run(meta(*shape), ids, meta(4, shape[1]))
    if shape[1] < 1 << 32:
        with pytest.raises(ValueError, match="d_table has 2\\^32"):
            grad.run(meta(2, shape[1]), ids, meta(*shape))
