"""The 8-bit head takes a hidden row's codes in either of the types that it takes a weight's in."""
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 40])
def test_codes_as_float8(rows):
    import torch
    t = twd()
    g = torch.Generator(device="cuda:0").manual_seed(rows)
    codes, scales = t.fp8_quantize(torch.randn(300, 256, generator=g, device="cuda:0"), 128)
    head, same = t.Fp8Head(codes, scales), t.Fp8Head(codes.view(torch.float8_e4m3fn), scales)
    c, s = t.fp8_quantize(torch.randn(rows, 256, generator=g, device="cuda:0"))
    want = head.logits_fp8(c, s)
    for h in (head, same):
        assert torch.equal(h.logits_fp8(c.view(torch.float8_e4m3fn), s), want)
    for bad in (c.view(torch.float8_e5m2), c.view(torch.int8), c.view(torch.float8_e4m3fn)[:, :128]):
        with pytest.raises(ValueError, match="codes"):
            head.logits_fp8(bad, s)
    head.close(), same.close()
