"""Rows quantised to microscaled 4-bit floating point and back: codes and scale bytes against the
definition in 64 bits, bit for bit, over types, lengths, strides and alignments, and the special values."""
import numpy as np
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def quantize_ref(x):
    """codes [R, C / 2] and scales [R, C / 32] of float64 rows, element by element from the definition: the
    nearest of the eight magnitudes, the even code where two are equally near."""
    rows, cols = x.shape
    b = x.reshape(rows, cols // 32, 32)
    bad = ~np.isfinite(b).all(2)
    a = np.where(np.isfinite(b), np.abs(b), 0.0)
    top = a.max(2)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    y = a / np.exp2(e.astype(np.float64))[..., None]
    dist = np.abs(y[..., None] - GRID)
    near = dist.min(-1, keepdims=True)
    odd = np.arange(8) % 2 == 1
    code = np.where(dist == near, np.where(odd, 1, 0), 2).argmin(-1)  # the nearest, even before odd
    code = code | (np.signbit(b).astype(np.int64) << 3)
    code[bad] = 0
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    c = code.reshape(rows, cols // 2, 2).astype(np.uint8)
    return c[..., 0] | (c[..., 1] << 4), scales


def values_ref(codes, scales):
    rows = codes.shape[0]
    c = np.stack([codes & 15, codes >> 4], axis=2).reshape(rows, -1)
    v = np.where(c > 7, -1.0, 1.0) * GRID[c & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(rows, -1, 32) * s[..., None]).reshape(rows, -1)


def device_rows(x, dtype, pad=0, offset=0):
    """x as a [rows, cols] device view whose rows lie cols + pad apart and start `offset` elements in."""
    import torch
    rows, cols = x.shape
    buf = torch.zeros(rows * (cols + pad) + offset + 8, dtype=dtype, device="cuda:0")
    v = buf[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    v.copy_(torch.from_numpy(x).to(dtype))
    return v


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols,pad,offset", [(1, 32, 0, 0), (1, 5376, 0, 0), (3, 96, 0, 0), (7, 2080, 32, 0),
                                                  (5, 64, 3, 1), (2, 8192 + 32, 0, 1), (70001, 32, 0, 0),
                                                  (257, 1024, 8, 8)])
def test_quantize_and_back(dtype, rows, cols, pad, offset):
    import torch
    t = twd()
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(rows * cols + pad)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-12, 9, (rows, cols // 32))).repeat(32, 1)
    x[rng.random((rows, cols)) < 0.05] = 0.0
    v = device_rows(x.astype(np.float32), dt, pad, offset)
    want_c, want_s = quantize_ref(v.double().cpu().numpy())
    codes, scales = t.mx_quantize(v)
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(codes.cpu().numpy(), want_c)
    want = values_ref(want_c, want_s)
    for out_dt in (torch.float32, torch.bfloat16, torch.float16):
        out = device_rows(np.zeros((rows, cols), np.float32), out_dt, pad, offset)
        assert t.mx_dequantize(codes, scales, out=out) is out
        ref = torch.from_numpy(want).to(out_dt)  # exact but for fp16's own range
        assert torch.equal(out.cpu(), ref), out_dt
    plain = t.mx_dequantize(codes, scales)
    assert plain.dtype == torch.bfloat16 and np.array_equal(plain.double().cpu().numpy(), want)


def test_every_rounding_border():
    """Every float32 next to and on a border between two magnitudes, under scales from the smallest to the largest."""
    import torch
    t = twd()
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1, 1.5, 2, 3, 4, 6, 7.999], np.float32)
    near = np.concatenate([np.nextafter(mids, np.float32(0)), mids, np.nextafter(mids, np.float32(9))])
    near = np.concatenate([near, -near])
    rows = []
    for e in (-127, -126, -100, -3, 0, 1, 60, 124, 125):
        for top in (4.0, 6.0, 7.5):
            for k in range(0, len(near), 31):
                r = np.zeros(32)
                part = near[k:k + 31].astype(np.float64)
                r[:len(part)] = np.clip(part, -7.99, 7.99)
                r[31] = top
                rows.append(r * 2.0 ** e)
    x = np.array(rows).astype(np.float32)  # subnormal where 2^-127 and 2^-126 say so
    v = torch.from_numpy(x).cuda()
    codes, scales = t.mx_quantize(v)
    want_c, want_s = quantize_ref(x.astype(np.float64))
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(codes.cpu().numpy(), want_c)
    back = t.mx_dequantize(codes, scales, dtype=torch.float32).double().cpu().numpy()
    assert np.array_equal(back, values_ref(want_c, want_s))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_special_blocks(dtype):
    import torch
    t = twd()
    dt = getattr(torch, dtype)
    x = np.zeros((1, 32 * 8), np.float32)
    x[0, 32:64] = -0.0
    x[0, 64:96] = np.linspace(-3, 3, 32)
    x[0, 70] = np.nan
    x[0, 96:128] = 1.0
    x[0, 100] = np.inf
    x[0, 128:160] = 1.0
    x[0, 130] = -np.inf
    tiny = float(torch.finfo(dt).smallest_normal)
    x[0, 160:192] = tiny * 2.0 ** -3  # subnormal
    x[0, 192:224] = float(torch.finfo(dt).max)
    x[0, 224] = 5.0
    v = torch.from_numpy(x).to(dt).cuda()
    codes, scales = t.mx_quantize(v)
    want_c, want_s = quantize_ref(v.double().cpu().numpy())
    assert scales.cpu().numpy().tolist() == want_s.tolist()
    assert np.array_equal(codes.cpu().numpy(), want_c)
    assert want_s[0, 0] == 0 and want_s[0, 2:5].tolist() == [255] * 3
    back = t.mx_dequantize(codes, scales, dtype=torch.float32).cpu().numpy()
    assert np.array_equal(back, values_ref(want_c, want_s).astype(np.float32), equal_nan=True)


def test_every_code_and_scale_byte_back():
    import torch
    t = twd()
    codes = np.tile(np.arange(256, dtype=np.uint8)[None].repeat(256, 0), 1)  # every pair of codes under every scale
    scales = np.arange(256, dtype=np.uint8)[:, None].repeat(16, 1)
    want = values_ref(codes, scales)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        got = t.mx_dequantize(torch.from_numpy(codes).cuda(), torch.from_numpy(scales.copy()).cuda(), dtype=dt)
        assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-7.25),
                           torch.nan_to_num(torch.from_numpy(want).to(dt).float(), nan=-7.25)), dt


def test_captured_on_another_stream():
    import torch
    t = twd()
    s = torch.cuda.Stream()
    x = torch.randn(33, 2048, device="cuda:0").bfloat16()
    codes = torch.empty(33, 1024, dtype=torch.uint8, device="cuda:0")
    scales = torch.empty(33, 64, dtype=torch.uint8, device="cuda:0")
    out = torch.empty(33, 2048, dtype=torch.bfloat16, device="cuda:0")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        t.mx_quantize(x, codes, scales, stream=s.cuda_stream)
        t.mx_dequantize(codes, scales, out=out, stream=s.cuda_stream)
    for rep in range(4):
        x.copy_(torch.randn(33, 2048, device="cuda:0") * (rep + 1))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        c, sc = t.mx_quantize(x)
        assert torch.equal(c, codes) and torch.equal(sc, scales), rep
        assert torch.equal(t.mx_dequantize(c, sc), out), rep
    del g


def test_rows_more_than_4_gib_apart():
    import torch
    t = twd()
    x = np.random.default_rng(8).standard_normal((2, 64)).astype(np.float32)
    far = (1 << 31) + 8
    buf = torch.empty(far + 64, dtype=torch.bfloat16, device="cuda:0")
    v = buf.as_strided((2, 64), (far, 1))
    v.copy_(torch.from_numpy(x))
    want = quantize_ref(v.double().cpu().numpy())
    codes, scales = t.mx_quantize(v)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])
    t.mx_dequantize(codes, scales, out=v)
    assert np.array_equal(v.double().cpu().numpy(), values_ref(*want))
