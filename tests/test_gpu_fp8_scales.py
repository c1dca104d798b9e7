"""The 8-bit head at the ends of what scales may be: hidden scales up to FLT_MAX / 448, the largest that fp8_quantize gives,
with weight scales up to 2^8, and products of two scales below the normal numbers.

A sum of 128 products is at most 128 x 448^2 < 2^24.7 in magnitude. A product of two scales below 2^-126 is rounded to a multiple
of 2^-149, so by at most 2^-150, and the sum times it is off by less than 2^-125."""
import numpy as np
import pytest

from helpers import twd
from test_gpu_fp8 import GRID, dev

pytestmark = pytest.mark.gpu

LARGEST = np.float32(np.finfo(np.float32).max) / np.float32(448)
CODE = {float(v): c for c, v in enumerate(GRID[:127])}
ROWS = [(1, "float32"), (16, "bfloat16"), (17, "float32"), (40, "bfloat16"), (130, "float32"), (130, "bfloat16")]


@pytest.mark.parametrize("scale", [np.nextafter(np.float32(256), np.float32(np.inf)), 2.0 ** 9, 2.0 ** 50, 2.0 ** 100])
def test_weight_scales_above_2_8_are_refused(scale):
    t = twd()
    scales = np.ones((2, 2), np.float32)
    scales[1, 0] = scale
    with pytest.raises(t.TwdError, match="2\\^8") as e:
        t.Fp8Head(dev(np.zeros((200, 256), np.uint8)), dev(scales))
    assert e.value.code == t.TWD_E_UNSUPPORTED


@pytest.mark.parametrize("rows,out_type", ROWS)
def test_largest_scales(rows, out_type):
    """Sums of zero stay zero, the smallest stay finite, and only what is past the type is infinite."""
    import torch
    t = twd()
    vocab, d = 200, 256
    wc, hc = np.zeros((vocab, d), np.uint8), np.zeros((rows, d), np.uint8)
    hc[:, 0], hc[:, 128] = CODE[2.0 ** -9], CODE[448.0]
    wc[1, 0], wc[2, 0], wc[3, 128], wc[4, 128] = CODE[2.0 ** -9], CODE[1.0], CODE[448.0], CODE[448.0] | 0x80
    ws = np.full((2, 2), 256, np.float32)
    hs = np.full((rows, 2), LARGEST, np.float32)
    head = t.Fp8Head(dev(wc), dev(ws))
    out = torch.empty(rows, vocab, dtype=getattr(torch, out_type), device="cuda:0")
    head.logits_fp8(dev(hc), dev(hs), out=out)
    got = out.double().cpu().numpy()
    product = np.float64(LARGEST) * 256  # exact in fp32
    want = np.zeros(vocab)
    want[1:3], want[3], want[4] = (product * 2.0 ** -18, product * 2.0 ** -9), np.inf, -np.inf
    if out_type == "bfloat16":
        want = torch.from_numpy(want).to(torch.bfloat16).double().numpy()
    assert np.array_equal(got, np.broadcast_to(want, got.shape))
    head.close()


@pytest.mark.parametrize("rows,out_type", ROWS)
def test_largest_rows_through_the_format(rows, out_type):
    """Rows as large as fp32 holds, quantised on the way, against weights of which most are zero."""
    import torch
    t = twd()
    w = torch.zeros(130, 256, device="cuda:0")
    w[7, 3], w[7, 4] = 2.0 ** -10, -(2.0 ** -10)
    w[8, 200] = 448.0 * 256  # a scale of 2^8
    h = torch.full((rows, 256), 3.4e38, device="cuda:0")
    h[:, 128:] = 0
    head = t.Fp8Head.from_weights(w)
    out = torch.empty(rows, 130, dtype=getattr(torch, out_type), device="cuda:0")
    assert bool((head.logits(h, out=out) == 0).all())
    head.close()


@pytest.mark.parametrize("rows,out_type", ROWS)
@pytest.mark.parametrize("whole", [True, False])
def test_products_of_scales_below_the_normal_numbers(rows, out_type, whole):
    import torch
    t = twd()
    vocab, d = 140, 384
    rng = np.random.default_rng(rows)
    ok = np.flatnonzero((np.abs(GRID) <= 16) & (GRID == np.rint(GRID)))
    wc, hc = rng.choice(ok, (vocab, d)).astype(np.uint8), rng.choice(ok, (rows, d)).astype(np.uint8)
    ws = np.exp2(rng.integers(-126, -100, (2, 3))).astype(np.float32)
    hs = np.exp2(rng.integers(-23, -10, (rows, 3))).astype(np.float32)
    if not whole:  # products that fp32 does not hold
        ws *= rng.uniform(1, 2, ws.shape).astype(np.float32)
        hs *= rng.uniform(1, 2, hs.shape).astype(np.float32)
    wv = GRID[wc] * np.repeat(np.repeat(ws.astype(np.float64), 128, 0)[:vocab], 128, 1)
    hv = GRID[hc] * np.repeat(hs.astype(np.float64), 128, 1)
    want = hv @ wv.T
    head = t.Fp8Head(dev(wc), dev(ws))
    out = torch.empty(rows, vocab, dtype=getattr(torch, out_type), device="cuda:0")
    head.logits_fp8(dev(hc), dev(hs), out=out)
    # whole products are exact, and so is each sum times one; three of them are added
    size = np.abs(hv) @ np.abs(wv).T
    tol = 3 * 2.0 ** -24 * size + 3 * 2.0 ** -150 if whole else (3 + 2) * 2.0 ** -24 * size + 3 * 2.0 ** -125
    if out_type == "bfloat16":
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol) + 2.0 ** -134
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    head.close()
