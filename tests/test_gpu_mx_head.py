"""The LM head in microscaled 4-bit floating point (MxHead): logits of bf16 and of quantised hidden rows
against the definition in 64 bits.

Where the inputs are small integers every partial sum is an integer below 2^24 units, so fp32 sums are
exact in any order and the logits are checked bit for bit. For normal inputs the bound is K 2^-23 sum |w h|
for the sums (K additions, each rounded or truncated), 4 2^-24 |y| for the softcap's quotient, tanh and
product, and half a step of the output's type."""
import numpy as np
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu

SHAPES = [  # vocab, d_model, rows
    (1, 32, 1), (15, 32, 1), (16, 128, 1), (17, 160, 2), (1000, 1024, 1), (1003, 2080, 3), (517, 5376, 1),
    (4099, 2048, 1), (777, 5376, 7), (640, 2880, 8), (333, 3584, 15), (65, 4096, 16), (131, 1056, 17),
    (1029, 512, 33), (300, 5376, 64), (259, 2880, 65), (515, 640, 129), (1031, 416, 300), (96, 8224, 5),
    (70, 17440, 2), (33, 17440, 40), (2050, 96, 1025), (98400, 544, 9), (98310, 160, 2),
]


def decode(codes, scales):
    grid = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
    c = np.stack([codes & 15, codes >> 4], axis=2).reshape(codes.shape[0], -1)
    s = np.exp2(scales.astype(np.float64) - 127)
    return (grid[c].reshape(c.shape[0], -1, 32) * s[..., None]).reshape(c.shape[0], -1)


def random_matrix(rng, rows, cols, lo=127, hi=129):
    codes = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
    scales = rng.integers(lo, hi, (rows, cols // 32)).astype(np.uint8)
    return codes, scales


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("vocab,d,rows", SHAPES)
def test_exact_sums_bf16_rows(vocab, d, rows):
    import torch
    t = twd()
    rng = np.random.default_rng(vocab + d + rows)
    codes, scales = random_matrix(rng, vocab, d)
    h = rng.integers(-4, 5, (rows, d)).astype(np.float32)
    want = h.astype(np.float64) @ decode(codes, scales).T  # multiples of 0.5 below 17440 * 4 * 12 < 2^20
    head = t.MxHead(dev(codes), dev(scales))
    got = head.logits(dev(h).bfloat16())
    assert np.array_equal(got.double().cpu().numpy(), want)
    # strided rows, strided bf16 logits whose padding stays as it was
    wide = torch.full((rows, d + 24), float("nan"), device="cuda:0", dtype=torch.bfloat16)
    wide[:, :d] = dev(h)
    out = torch.full((rows + 1, vocab + 5), 7.0, device="cuda:0", dtype=torch.bfloat16)
    head.logits(wide[:, :d], out=out[:rows, 1:vocab + 1])
    assert torch.equal(out[:rows, 1:vocab + 1].cpu(), torch.from_numpy(want).to(torch.bfloat16))
    assert (out[rows] == 7.0).all() and (out[:, 0] == 7.0).all() and (out[:, vocab + 1:] == 7.0).all()
    head.close()


@pytest.mark.parametrize("vocab,d,rows", SHAPES)
def test_exact_sums_mx_rows(vocab, d, rows):
    import torch
    t = twd()
    rng = np.random.default_rng(vocab + d + rows)
    codes, scales = random_matrix(rng, vocab, d)
    hc, hs = random_matrix(rng, rows, d, 126, 128)
    want = decode(hc, hs) @ decode(codes, scales).T  # multiples of 1 / 8 below 17440 * 6 * 12 < 2^21
    head = t.MxHead(dev(codes), dev(scales))
    got = head.logits_mx(dev(hc), dev(hs))
    assert np.array_equal(got.double().cpu().numpy(), want)
    out = torch.full((rows + 1, vocab + 3), 7.0, device="cuda:0")
    head.logits_mx(dev(hc), dev(hs), out=out[:rows, :vocab])
    assert np.array_equal(out[:rows, :vocab].double().cpu().numpy(), want)
    assert (out[rows] == 7.0).all() and (out[:, vocab:] == 7.0).all()
    head.close()


@pytest.mark.parametrize("vocab,d,rows,cap", [(2003, 5376, 1, 30.0), (1000, 2080, 5, 30.0), (513, 5376, 16, 0.0),
                                              (600, 3584, 48, 30.0), (260, 2880, 200, 50.0)])
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("out_type", ["float32", "bfloat16"])
def test_normal_rows(vocab, d, rows, cap, mx, out_type):
    import torch
    t = twd()
    rng = np.random.default_rng(vocab + rows)
    w = (rng.standard_normal((vocab, d)) * 3.6 / np.sqrt(d)).astype(np.float32)
    codes, scales = t.mx_quantize(dev(w))
    wv = decode(codes.cpu().numpy(), scales.cpu().numpy())
    h = dev(rng.standard_normal((rows, d)).astype(np.float32)).bfloat16()
    head = t.MxHead.from_weights(dev(w), softcap=cap)
    out = torch.empty(rows, vocab, dtype=getattr(torch, out_type), device="cuda:0")
    if mx:
        hc, hs = t.mx_quantize(h)
        hv = decode(hc.cpu().numpy(), hs.cpu().numpy())
        head.logits_mx(hc, hs, out=out)
    else:
        hv = h.double().cpu().numpy()
        head.logits(h, out=out)
    z = hv @ wv.T
    want = cap * np.tanh(z / cap) if cap > 0 else z
    tol = d * 2.0 ** -23 * (np.abs(hv) @ np.abs(wv).T) + 4 * 2.0 ** -24 * np.abs(want)
    if out_type == "bfloat16":
        tol += 2.0 ** -8 * np.abs(want)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    head.close()


@pytest.mark.parametrize("cap", [1e-30, 0.37, 30.0, 1e30])
@pytest.mark.parametrize("rows", [2, 40])
def test_softcap_over_its_whole_range(cap, rows):
    """The cap of exact sums from far below it to far past it, either sign, within the four half steps that
    the quotient, the function and the product have: the sums are two bf16 parts of 16-bit values."""
    t = twd()
    cap = float(np.float32(cap))
    x = np.concatenate([[0.0, 1e-3], np.geomspace(0.01, 200.0, 801), np.linspace(0.9, 1.1, 197)]) * cap
    x[1::2] *= -1
    bits = x.astype(np.float32).view(np.uint32)
    z, hi = ((bits & m).astype(np.uint32).view(np.float32) for m in (0xFFFFFF00, 0xFFFF0000))
    h = np.zeros((1000, 64), np.float32)
    h[:, 0], h[:, 1] = hi, z - hi
    codes, scales = np.zeros((5, 32), np.uint8), np.full((5, 2), 127, np.uint8)
    codes[:, 0] = 0x22  # ones in the first two columns
    want = cap * np.tanh(z.astype(np.float64) / cap)
    head = t.MxHead(dev(codes), dev(scales), softcap=cap)
    hd = dev(h).bfloat16()
    got = np.concatenate([head.logits(hd[i:i + rows]).double().cpu().numpy() for i in range(0, 1000, rows)])
    assert (np.abs(got - want[:, None]) <= 4 * 2.0 ** -24 * np.abs(want)[:, None]).all()
    head.close()


@pytest.mark.parametrize("rows,stride", [(3, 1 << 26), (20, 1 << 26), (35, (1 << 25) + 8), (66, (1 << 24) + 64)])
def test_hidden_rows_far_apart(rows, stride):
    """Rows so far apart that a tile of 128 does not lie within 32-bit offsets; the last reads the last bytes."""
    import torch
    t = twd()
    rng = np.random.default_rng(rows)
    d = 160
    codes, scales = random_matrix(rng, 70, d)
    h = rng.integers(-4, 5, (rows, d)).astype(np.float32)
    x = torch.zeros((rows - 1) * stride + d, dtype=torch.bfloat16, device="cuda:0").as_strided((rows, d), (stride, 1))
    x.copy_(dev(h))
    head = t.MxHead(dev(codes), dev(scales))
    assert np.array_equal(head.logits(x).double().cpu().numpy(), h.astype(np.float64) @ decode(codes, scales).T)
    head.close()


@pytest.mark.parametrize("rows", [3, 40])
def test_logits_more_than_4_gib_apart(rows):
    import torch
    t = twd()
    rng = np.random.default_rng(rows)
    codes, scales = random_matrix(rng, 70, 288)
    h = rng.integers(-4, 5, (rows, 288)).astype(np.float32)
    far = ((1 << 32) + 4096) // 2 // (rows - 1) + 1
    out = torch.empty((rows - 1) * far + 70, dtype=torch.bfloat16, device="cuda:0").as_strided((rows, 70), (far, 1))
    head = t.MxHead(dev(codes), dev(scales))
    want = torch.from_numpy(h.astype(np.float64) @ decode(codes, scales).T).to(torch.bfloat16)
    assert torch.equal(head.logits(dev(h).bfloat16(), out=out).cpu(), want)
    head.close()


@pytest.mark.parametrize("rows", [1, 20, 70])
@pytest.mark.parametrize("mx", [False, True])
def test_nan_and_inf_rows_stay_theirs(rows, mx):
    """A hidden row with a NaN gives NaN logits, and no other row does; a block quantised with one too."""
    import torch
    t = twd()
    rng = np.random.default_rng(rows)
    codes, scales = random_matrix(rng, 100, 1056)
    h = rng.integers(1, 5, (rows, 1056)).astype(np.float32)
    bad = rows // 2
    h[bad, 1055] = np.nan
    head = t.MxHead(dev(codes), dev(scales))
    hd = dev(h).bfloat16()
    got = (head.logits_mx(*t.mx_quantize(hd)) if mx else head.logits(hd)).cpu().numpy()
    assert np.isnan(got[bad]).all()
    assert np.isfinite(np.delete(got, bad, 0)).all()
    head.close()


def test_zero_blocks_and_scale_extremes():
    """Zero blocks carry scale byte 0; scales down to 2^-126 and up to 2^100 multiply exactly."""
    t = twd()
    codes = np.zeros((32, 64), np.uint8)
    scales = np.zeros((32, 4), np.uint8)
    for v, s in enumerate((1, 2, 60, 127, 200, 227)):
        codes[v, 16:32] = 0x22  # ones in the second block
        scales[v, 1] = s
    h = np.ones((3, 128), np.float32)
    head = t.MxHead(dev(codes), dev(scales))
    want = h.astype(np.float64) @ decode(codes, scales).T
    assert np.array_equal(head.logits(dev(h).bfloat16()).double().cpu().numpy(), want)
    assert np.array_equal(head.logits_mx(*t.mx_quantize(dev(h))).double().cpu().numpy(), want)
    head.close()


def test_scales_beyond_the_range_are_refused():
    t = twd()
    for s in (228, 254, 255):
        codes, scales = np.zeros((20, 32), np.uint8), np.full((20, 2), 127, np.uint8)
        scales[19, 1] = s
        with pytest.raises(t.TwdError) as e:
            t.MxHead(dev(codes), dev(scales))
        assert e.value.code == t.TWD_E_UNSUPPORTED


def test_streams_and_graphs():
    """Calls on one head from two streams at once, and a captured call replayed with new rows."""
    import torch
    t = twd()
    rng = np.random.default_rng(3)
    codes, scales = random_matrix(rng, 9001, 1024)
    head = t.MxHead(dev(codes), dev(scales))
    w = decode(codes, scales)
    streams = [torch.cuda.Stream() for _ in range(2)]
    hs = [rng.integers(-4, 5, (n, 1024)).astype(np.float32) for n in (5, 40)]
    hd = [dev(h).bfloat16() for h in hs]
    torch.cuda.synchronize()
    for _ in range(3):
        outs = [head.logits(x, stream=s.cuda_stream) for x, s in zip(hd, streams)]
        torch.cuda.synchronize()
        for h, o in zip(hs, outs):
            assert np.array_equal(o.double().cpu().numpy(), h.astype(np.float64) @ w.T)
    for n in (1, 12, 40):
        x = torch.zeros(n, 1024, dtype=torch.bfloat16, device="cuda:0")
        out = torch.empty(n, 9001, device="cuda:0")
        head.logits(x, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            head.logits(x, out=out, stream=streams[0].cuda_stream)
        for rep in range(4):
            h = rng.integers(-4, 5, (n, 1024)).astype(np.float32)
            x.copy_(dev(h))
            head.logits(hd[1])  # eager work between the replays
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert np.array_equal(out.double().cpu().numpy(), h.astype(np.float64) @ w.T), (n, rep)
        del g
    head.close()
