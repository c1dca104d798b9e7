"""The vocabulary matrix through a training step and into serving, as a program with tied embeddings runs it: looked up,
multiplied for the loss, both gradients into one, a step, then held in 8 and in 4 bits and sampled from."""
import numpy as np
import pytest

from helpers import twd
from test_gpu_head_loss import U, check, reference

pytestmark = pytest.mark.gpu


def test_tied_training_step_and_serving():
    import torch
    t = twd()
    vocab, d, n, cap = 5003, 256, 700, 30.0
    scale = float(np.float32(d ** 0.5))
    g = torch.Generator(device="cuda:0").manual_seed(1)
    master = torch.randn(vocab, d, generator=g, device="cuda:0") / d ** 0.5
    ids = torch.randint(vocab, (n,), generator=g, device="cuda:0").to(torch.int32)
    ids[-60:] = -1  # a padded batch
    targets = torch.roll(ids, -1)
    targets[:100] = -100  # the prompt
    grad = torch.full((n,), 1.0 / int((targets >= 0).sum()), device="cuda:0")
    loss, embeds = t.HeadLoss(n, vocab, d, softcap=cap), t.EmbedGrad(n, d)
    totals = []
    for _ in range(3):
        w = master.bfloat16()
        hidden = t.embed(w, ids, scale=scale)  # the model between them is the identity
        losses, lse = loss.forward(hidden, w, targets)
        d_weight = torch.empty(vocab, d, device="cuda:0")
        d_hidden, _ = loss.backward(hidden, w, targets, lse, grad=grad, d_weight=d_weight)
        want, tol = reference(hidden, w, targets, cap, grad)
        check("losses", losses, want["losses"], tol["losses"], U)
        check("d_weight", d_weight, want["d_weight"], tol["d_weight"], U)
        embeds.run(d_hidden, ids, d_weight, scale=scale, accumulate=True)
        keep = ids >= 0
        whole, size = want["d_weight"].clone(), want["d_weight"].abs()
        for into, x in ((whole, d_hidden[keep].double()), (size, d_hidden[keep].double().abs())):
            into.index_put_((ids[keep].long(),), x * scale, accumulate=True)
        check("tied gradient", d_weight, whole, tol["d_weight"] + (n + 2) * U * size, U)
        assert bool((d_hidden[targets < 0] == 0).all())
        totals.append(float(losses.double().sum()))
        master -= 0.5 * d_weight
    assert all(np.isfinite(totals))
    w = master.bfloat16()
    rows = t.embed(w, ids[:7].contiguous(), scale=scale)
    exact = cap * torch.tanh(rows.double() @ w.double().t() / cap)
    sampler = t.Sampler(vocab, 7)
    # an element is off by at most 1/16 of itself in 8 bits (the smallest, by 2^-10 of 448th parts of the block's largest),
    # in both factors of the 8-bit head
    for head, most in ((t.Fp8Head.from_weights(w, softcap=cap), 2 / 16 + 1 / 256 + 1 / 64),):
        logits = head.logits(rows)
        bound = most * (rows.double().abs() @ w.double().abs().t())
        assert bool(((logits.double() - exact).abs() <= bound + 1e-3).all())
        tokens = sampler.sample(logits, torch.full((7,), 0.5, device="cuda:0"), top_k=torch.full((7,), 20, dtype=torch.int32, device="cuda:0"))
        kept = torch.topk(logits, 20, 1).indices
        assert bool((kept == tokens.long()[:, None]).any(1).all())
        head.close()
    mx = t.MxHead.from_weights(w, softcap=cap)
    tokens = sampler.sample(mx.logits(rows), torch.zeros(7, device="cuda:0"), temperature=torch.zeros(7, device="cuda:0"))
    assert torch.equal(tokens.long(), mx.logits(rows).argmax(1))
    for x in (mx, sampler, loss, embeds):
        x.close()
