"""8-bit floating point with a scale for each block of 128: the format bit for bit, and the head's logits against the
definition in 64 bits.

The matrix instructions add 128 products of elements widened to bf16, which are exact; a partial sum is at most their magnitudes' sum, and is rounded or truncated 128
times, then once for the product with the scales' own rounded product and once where it is added to the others: the bound is
(130 + 2 + d / 128) 2^-23 sum |w h|, 4 2^-24 |y| for the softcap, and half a step of the output's type. bf16 logits of more
than 128 rows come from the 8-bit instructions, which align the products of eight neighbouring columns to the largest of them
and cut them at 2^-13 of it: that takes less than 7 2^-13 of the largest from the other seven, so 7 2^-13 sum |w h| in all
(the largest, of seven bits, is not cut). Small integers under
scales that are powers of two are exact in any order and checked bit for bit."""
import numpy as np
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu


def e4m3_values():
    v = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    v = np.array(v)
    v[127] = np.nan
    return np.concatenate([v, -v])


GRID = e4m3_values()


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def quantize(x, block_rows):
    """The definition, in 64 bits: quotients of a float and a float need no more bits to lie on the right side of a border."""
    rows, cols = x.shape
    n = -(-rows // block_rows)
    pad = np.zeros((n * block_rows, cols), np.float64)
    pad[:rows] = x
    b = pad.reshape(n, block_rows, cols // 128, 128)
    top = np.abs(b).max((1, 3))
    s = np.maximum((top / 448).astype(np.float32), np.float32(2.0 ** -126))
    bad = ~np.isfinite(top)
    s[bad] = np.nan
    q = np.where(bad[:, None, :, None], 0, b) / np.where(bad, 1, s).astype(np.float64)[:, None, :, None]
    mag = GRID[:127]
    borders = (mag[:-1] + mag[1:]) / 2
    low, high = np.searchsorted(borders, np.abs(q)), np.searchsorted(borders, np.abs(q), side="right")
    codes = np.where(low % 2 == 0, low, high).astype(np.uint8) | (np.signbit(q).astype(np.uint8) << 7)
    codes[np.broadcast_to(bad[:, None, :, None], codes.shape)] = 0
    return codes.reshape(n * block_rows, cols)[:rows], s


@pytest.mark.parametrize("rows,cols,pad", [(1, 128, 0), (1, 5376, 0), (3, 256, 1), (130, 1024, 8), (257, 384, 0), (777, 2944, 24)])
@pytest.mark.parametrize("name", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_format(rows, cols, pad, name, block_rows):
    import torch
    t = twd()
    g = torch.Generator(device="cuda:0").manual_seed(rows + cols)
    x = torch.randn(rows, cols + pad, generator=g, device="cuda:0") * torch.exp(3 * torch.randn(rows, 1, generator=g, device="cuda:0"))
    x = x.to(getattr(torch, name))
    x[0, :64] = 0.0
    x[rows // 2, 3] = 3.5  # 448 / 128: quotients on borders
    x = x[:, :cols]
    codes, scales = t.fp8_quantize(x, block_rows)
    want, s = quantize(x.double().cpu().numpy(), block_rows)
    assert np.array_equal(scales.cpu().numpy(), s)
    assert np.array_equal(codes.cpu().numpy(), want)
    assert torch.equal(codes, t.fp8_quantize(x.contiguous(), block_rows)[0])


@pytest.mark.parametrize("block_rows", [1, 128])
def test_format_extremes(block_rows):
    """Zeros, the smallest and largest floats, borders on either side, infinities and NaN."""
    import torch
    t = twd()
    x = np.zeros((128 * 14, 128), np.float32)
    rng = np.random.default_rng(1)
    tops = [0.0, 1e-45, 2.0 ** -149 * 448, 2.0 ** -126, 448 * 2.0 ** -126, 1.3 * 448 * 2.0 ** -126, 1e-30, 3.5, 448.0, 3e38]
    for i, top in enumerate(tops):
        x[128 * i:128 * i + 128] = rng.uniform(-1, 1, (128, 128)) * top
        x[128 * i:128 * i + 128, 7] = top
        # quotients next to borders, a step of the float on either side
        s = max(np.float32(top / 448), np.float32(2.0 ** -126))
        edge = ((GRID[:126] + GRID[1:127]) / 2 * np.float64(s)).astype(np.float32)
        x[128 * i, 8:128], x[128 * i + 1, 8:128], x[128 * i + 2, 8:128] = edge[:120], np.nextafter(edge[:120], np.float32(0)), np.nextafter(edge[:120], np.float32(np.inf))
        x[128 * i:128 * i + 3] = np.clip(x[128 * i:128 * i + 3], -top, top)
    x[128 * 10 + 5, 9], x[128 * 11 + 5, 9], x[128 * 12 + 5, 9] = np.inf, -np.inf, np.nan
    codes, scales = t.fp8_quantize(dev(x), block_rows)
    with np.errstate(invalid="ignore"):
        want, s = quantize(x, block_rows)
    assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True)
    assert np.array_equal(codes.cpu().numpy(), want)


SHAPES = [(1, 128, 1), (63, 128, 2), (64, 256, 1), (129, 384, 3), (1000, 1024, 1), (517, 5376, 7), (333, 3584, 16), (4099, 640, 5),
          (131, 1024, 17), (1029, 512, 33), (300, 5376, 64), (259, 2944, 65), (515, 640, 129), (96, 8320, 5), (33, 17408, 40),
          (2050, 128, 1025), (40003, 512, 9), (20011, 256, 100)]


def integers(rng, rows, d, most):
    """Codes of whole numbers up to `most` and their values."""
    ok = np.flatnonzero((np.abs(GRID) <= most) & (GRID == np.rint(GRID)))
    return rng.choice(ok, (rows, d)).astype(np.uint8)


@pytest.mark.parametrize("vocab,d,rows", SHAPES)
def test_exact_sums(vocab, d, rows):
    import torch
    t = twd()
    rng = np.random.default_rng(vocab + d + rows)
    wc, hc = integers(rng, vocab, d, 8), integers(rng, rows, d, 4)
    ws = np.exp2(rng.integers(-1, 2, (-(-vocab // 128), d // 128))).astype(np.float32)
    hs = np.exp2(rng.integers(-1, 2, (rows, d // 128))).astype(np.float32)
    w = GRID[wc] * np.repeat(np.repeat(ws, 128, 0)[:vocab], 128, 1)
    h = GRID[hc] * np.repeat(hs, 128, 1)
    want = h @ w.T  # quarters below 17,408 x 8 x 4 x 4 < 2^22
    head = t.Fp8Head(dev(wc), dev(ws))
    assert np.array_equal(head.logits_fp8(dev(hc), dev(hs)).double().cpu().numpy(), want)
    out = torch.full((rows + 1, vocab + 5), 7.0, device="cuda:0", dtype=torch.bfloat16)
    head.logits_fp8(dev(hc), dev(hs), out=out[:rows, 1:vocab + 1])
    assert torch.equal(out[:rows, 1:vocab + 1].cpu(), torch.from_numpy(want).to(torch.bfloat16))
    assert (out[rows] == 7.0).all() and (out[:, 0] == 7.0).all() and (out[:, vocab + 1:] == 7.0).all()
    head.close()


@pytest.mark.parametrize("rows", [17, 32, 33])
def test_exact_sums_of_a_head_past_the_memory_cache(rows):
    import torch
    t = twd()
    vocab, d = 70001, 3968
    g = torch.Generator(device="cuda:0").manual_seed(rows)
    w = torch.randint(-8, 9, (vocab, d), generator=g, device="cuda:0").half()
    h = torch.randint(-8, 9, (rows, d), generator=g, device="cuda:0").half()
    ws = torch.exp2(torch.randint(-2, 3, ((vocab + 127) // 128, d // 128), generator=g, device="cuda:0").float())
    hs = torch.exp2(torch.randint(-2, 3, (rows, d // 128), generator=g, device="cuda:0").float())
    head = t.Fp8Head(w.to(torch.float8_e4m3fn), ws)
    got = head.logits_fp8(h.to(torch.float8_e4m3fn).view(torch.uint8), hs)
    want = torch.zeros(rows, vocab, dtype=torch.float64, device="cuda:0")
    for c in range(d // 128):
        part = h[:, 128 * c:128 * c + 128].double() @ w[:, 128 * c:128 * c + 128].double().t().contiguous()
        want += part * hs[:, c:c + 1].double() * ws[:, c].double().repeat_interleave(128)[:vocab]
    assert torch.equal(got.double(), want)
    head.close()


@pytest.mark.parametrize("vocab,d,rows,cap", [(2003, 5376, 1, 30.0), (1000, 2048, 5, 30.0), (513, 5376, 16, 0.0), (600, 3584, 48, 30.0),
                                              (260, 2944, 200, 50.0)])
@pytest.mark.parametrize("out_type", ["float32", "bfloat16"])
def test_normal_rows(vocab, d, rows, cap, out_type):
    import torch
    t = twd()
    rng = np.random.default_rng(vocab + rows)
    w = dev((rng.standard_normal((vocab, d)) * 3.6 / np.sqrt(d)).astype(np.float32))
    h = dev(rng.standard_normal((rows, d)).astype(np.float32)).bfloat16()
    wc, ws = t.fp8_quantize(w, 128)
    hc, hs = t.fp8_quantize(h)
    wv = GRID[wc.cpu().numpy()] * np.repeat(np.repeat(ws.cpu().numpy().astype(np.float64), 128, 0)[:vocab], 128, 1)
    hv = GRID[hc.cpu().numpy()] * np.repeat(hs.cpu().numpy().astype(np.float64), 128, 1)
    head = t.Fp8Head.from_weights(w, softcap=cap)
    out = torch.empty(rows, vocab, dtype=getattr(torch, out_type), device="cuda:0")
    head.logits(h, out=out)
    z = hv @ wv.T
    want = cap * np.tanh(z / cap) if cap > 0 else z
    cut = 7 * 2.0 ** -13 if out_type == "bfloat16" and rows > 128 else 0.0
    tol = (cut + (132 + d // 128) * 2.0 ** -23) * (np.abs(hv) @ np.abs(wv).T) + 4 * 2.0 ** -24 * np.abs(want)
    if out_type == "bfloat16":
        tol += 2.0 ** -8 * (np.abs(want) + tol)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    head.close()


@pytest.mark.parametrize("rows", [1, 16, 17, 33, 128, 129, 300])
@pytest.mark.parametrize("out_type", ["float32", "bfloat16"])
@pytest.mark.parametrize("others", [2.0 ** -10, 2.0 ** -3, 4.0, 8.0])
def test_small_products_beside_large_ones(rows, out_type, others):
    """127 products beside one of 2^16 that another block takes away again: the fp32 sums hold them to 2^-7 each (half a
    step of 2^16, in the sum of whichever they are added to), the 8-bit instructions to 2^3."""
    import torch
    t = twd()
    vocab, d = 70, 256
    w, h = torch.zeros(vocab, d), torch.zeros(rows, d)
    w[:, 0], w[:, 128], h[:, 0], h[:, 128] = 256, -256, 256, 256
    w[:, 1:128], h[:, 1:128] = max(others / 8, 2.0 ** -8), min(others / 2.0 ** -8, 8.0)
    head = t.Fp8Head(w.to(torch.float8_e4m3fn).cuda(), torch.ones(1, 2, device="cuda:0"))
    out = torch.empty(rows, vocab, dtype=getattr(torch, out_type), device="cuda:0")
    head.logits_fp8(h.to(torch.float8_e4m3fn).view(torch.uint8).cuda(), torch.ones(rows, 2, device="cuda:0"), out=out)
    want = 127 * others
    cut = out_type == "bfloat16" and rows > 128
    tol = 7 * 2.0 ** 3 + 2.0 if cut else 127 * 2.0 ** -7
    if out_type == "bfloat16":
        tol += 2.0 ** -8 * (want + tol)
    assert (out.double() - want).abs().max() <= tol
    head.close()


@pytest.mark.parametrize("rows", [1, 20, 70, 140])
def test_nan_rows_stay_theirs(rows):
    t = twd()
    rng = np.random.default_rng(rows)
    wc = integers(rng, 100, 1024, 8)
    h = rng.integers(1, 5, (rows, 1024)).astype(np.float32)
    bad = rows // 2
    h[bad, 1023] = np.nan
    head = t.Fp8Head(dev(wc), dev(np.ones((1, 8), np.float32)))
    got = head.logits(dev(h)).cpu().numpy()
    assert np.isnan(got[bad]).all()
    assert np.isfinite(np.delete(got, bad, 0)).all()
    head.close()


def test_scales_beyond_the_range_are_refused():
    t = twd()
    for s in (-1.0, 2.0 ** 101, np.inf, np.nan):
        scales = np.ones((2, 2), np.float32)
        scales[1, 1] = s
        with pytest.raises(t.TwdError) as e:
            t.Fp8Head(dev(np.zeros((200, 256), np.uint8)), dev(scales))
        assert e.value.code == t.TWD_E_UNSUPPORTED


def test_logits_more_than_4_gib_apart():
    import torch
    t = twd()
    rng = np.random.default_rng(2)
    for rows in (3, 40):
        wc, hc = integers(rng, 70, 256, 8), integers(rng, rows, 256, 4)
        far = ((1 << 32) + 4096) // 2 // (rows - 1) + 1
        out = torch.empty((rows - 1) * far + 70, dtype=torch.bfloat16, device="cuda:0").as_strided((rows, 70), (far, 1))
        head = t.Fp8Head(dev(wc), dev(np.ones((1, 2), np.float32)))
        head.logits_fp8(dev(hc), dev(np.ones((rows, 2), np.float32)), out=out)
        assert torch.equal(out.cpu(), torch.from_numpy(GRID[hc] @ GRID[wc].T).to(torch.bfloat16))
        head.close()


def test_streams_and_graphs():
    """Calls on one head from two streams at once, and captured calls replayed with new rows."""
    import torch
    t = twd()
    rng = np.random.default_rng(3)
    wc = integers(rng, 9001, 1024, 8)
    ones = np.ones((71, 8), np.float32)
    head = t.Fp8Head(dev(wc), dev(ones))
    w = GRID[wc]
    streams = [torch.cuda.Stream() for _ in range(2)]
    hs = [rng.integers(-4, 5, (n, 1024)).astype(np.float32) * 64 for n in (5, 40)]
    for h in hs:
        h[:, ::128] = 448.0  # scales of one
    hd = [dev(h).bfloat16() for h in hs]
    torch.cuda.synchronize()
    for _ in range(3):
        outs = [head.logits(x, stream=s.cuda_stream) for x, s in zip(hd, streams)]
        torch.cuda.synchronize()
        for h, o in zip(hs, outs):
            assert np.array_equal(o.double().cpu().numpy(), h.astype(np.float64) @ w.T)
    for n in (1, 40, 130):
        x = torch.zeros(n, 1024, dtype=torch.bfloat16, device="cuda:0")
        codes, scales = t.fp8_quantize(x)
        out = torch.empty(n, 9001, device="cuda:0")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            t.fp8_quantize(x, codes=codes, scales=scales, stream=streams[0].cuda_stream)
            head.logits_fp8(codes, scales, out=out, stream=streams[0].cuda_stream)
        for rep in range(4):
            h = rng.integers(-4, 5, (n, 1024)).astype(np.float32) * 64
            h[:, ::128] = 448.0
            x.copy_(dev(h))
            head.logits(hd[1])  # eager work between the replays
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert np.array_equal(out.double().cpu().numpy(), h.astype(np.float64) @ w.T), (n, rep)
        del g
    head.close()
