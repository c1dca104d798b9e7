"""The head's weights and hidden rows at the smallest numbers the format and bf16 have: every code under scale
bytes 0, 1 and 2 (2^-127 and up, whose elements are subnormal in bf16 and fp32), bf16 rows of subnormal values,
and sums that are subnormal themselves. One product per logit, so every logit is checked bit for bit."""
import numpy as np
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu

D = 1056  # whole stages of both tile kernels and columns past them
COLUMNS = [0, 7, 31, 500, 512, 543, 1023, 1024, 1055]
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def matrix(rows, scale):
    """Codes that run through all sixteen along rows and columns, scale byte scale[r % len] throughout a row."""
    c = (np.arange(D)[None] + np.arange(rows)[:, None]) % 16
    codes = (c[:, ::2] | c[:, 1::2] << 4).astype(np.uint8)
    s = np.array(scale)[np.arange(rows) % len(scale)]
    return codes, np.repeat(s[:, None], D // 32, 1).astype(np.uint8), GRID[c] * np.exp2(s - 127.0)[:, None]


def one_hot(rows, values):
    """bf16 rows with one value each, in columns of every part of the kernels' walk."""
    h = np.zeros((rows, D), np.float32)
    for m in range(rows):
        h[m, COLUMNS[m % len(COLUMNS)]] = values[m % len(values)]
    return h


@pytest.mark.parametrize("rows", [3, 40, 130])
@pytest.mark.parametrize("scale,values", [
    ((0, 1, 2), (2.0 ** 20, -2.0 ** 60, 1.5 * 2.0 ** 127)),  # subnormal weights, normal logits
    ((0, 1, 2), (1.0, -3.0, 0.5)),                           # subnormal weights and logits
    ((127, 227, 150), (2.0 ** -133, -2.0 ** -130, 2.0 ** -127)),  # subnormal rows
])
def test_bf16_rows(rows, scale, values):
    t = twd()
    codes, scales, w = matrix(70, scale)
    h = one_hot(rows, values)
    head = t.MxHead(dev(codes), dev(scales))
    hb = dev(h).bfloat16()
    assert np.array_equal(hb.float().cpu().numpy(), h)
    want = (h.astype(np.float64) @ w.T).astype(np.float32)  # 24 bits hold every product
    got = head.logits(hb).cpu().numpy()
    assert np.array_equal(got, want)
    head.close()


@pytest.mark.parametrize("rows", [3, 40, 130])
@pytest.mark.parametrize("scale,row_scale", [
    ((0, 1, 2), (147, 187, 250)),   # subnormal weights
    ((200, 227, 150), (0, 1, 2)),   # subnormal rows
    ((0, 1, 2), (126, 127, 128)),   # subnormal logits too
])
def test_mx_rows(rows, scale, row_scale):
    t = twd()
    codes, scales, w = matrix(70, scale)
    hc, hs = np.zeros((rows, D // 2), np.uint8), np.zeros((rows, D // 32), np.uint8)
    h = np.zeros((rows, D))
    for m in range(rows):
        col, code, s = COLUMNS[m % len(COLUMNS)], 1 + m % 7, row_scale[m % 3]
        hc[m, col // 2] = code << (4 * (col % 2))
        hs[m] = s
        h[m, col] = GRID[code] * 2.0 ** (s - 127)
    head = t.MxHead(dev(codes), dev(scales))
    want = (h @ w.T).astype(np.float32)
    got = head.logits_mx(dev(hc), dev(hs)).cpu().numpy()
    assert np.array_equal(got, want)
    head.close()
