"""An 8-bit head of more vocabulary rows than one round of its layout's blocks takes."""
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [65536 * 64, 65536 * 64 + 65])
def test_head_of_four_million_rows(vocab):
    import torch
    t = twd()
    d = 128
    g = torch.Generator(device="cuda:0").manual_seed(vocab)
    w = torch.randint(-8, 9, (vocab, d), generator=g, device="cuda:0", dtype=torch.int8).half()
    h = torch.randint(-8, 9, (2, d), generator=g, device="cuda:0").half()
    scales = torch.exp2(torch.randint(-2, 3, ((vocab + 127) // 128, 1), generator=g, device="cuda:0").float())
    head = t.Fp8Head(w.to(torch.float8_e4m3fn), scales)
    got = head.logits_fp8(h.to(torch.float8_e4m3fn), torch.ones(2, 1, device="cuda:0"))
    for r0 in range(0, vocab, 1 << 20):
        part = w[r0:r0 + (1 << 20)].double()
        want = h.double() @ part.t().contiguous()  # whole numbers below 2^13
        want *= scales[r0 // 128:(r0 + len(part) + 127) // 128, 0].double().repeat_interleave(128)[:len(part)]
        assert torch.equal(got[:, r0:r0 + (1 << 20)].double(), want)
    head.close()
