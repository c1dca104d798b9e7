"""What NaN and infinities in a row that counts make of a head's loss and its gradients, without and with a softcap."""
import pytest

from helpers import twd
from test_gpu_head_loss import U, make

pytestmark = pytest.mark.gpu

VOCAB, D = 600, 96


def run(loss, h, w, targets, grad):
    losses, lse = loss.forward(h, w, targets)
    return (losses, lse) + loss.backward(h, w, targets, lse, grad=grad)


def same_but_row_0(a, b):
    import torch
    return all(torch.equal(x[1:], y[1:]) for x, y in zip(a[:3], b[:3]))


@pytest.mark.parametrize("rows", [3, 70, 300])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_nan_is_its_rows_loss_and_all_gradients(rows, cap):
    import torch
    t = twd()
    h, w, targets, grad = make(VOCAB, D, rows, 0, 5)
    loss = t.HeadLoss(rows, VOCAB, D, softcap=cap)
    clean = run(loss, h, w, targets, grad)
    h[0, 5] = float("nan")
    got = run(loss, h, w, targets, grad)
    assert same_but_row_0(got, clean)
    assert bool(got[0][0].isnan()) and bool(got[1][0].isnan())
    assert bool(got[2][0].isnan().all()) and bool(got[3].isnan().all())
    loss.close()


@pytest.mark.parametrize("rows", [3, 70, 300])
def test_infinity_without_a_softcap(rows):
    import torch
    t = twd()
    h, w, targets, grad = make(VOCAB, D, rows, 0, 5)
    loss = t.HeadLoss(rows, VOCAB, D)
    clean = run(loss, h, w, targets, grad)
    for value in (float("inf"), -float("inf")):
        h[0, 6] = value
        got = run(loss, h, w, targets, grad)
        assert same_but_row_0(got, clean)
        assert bool(got[0][0].isnan()) and bool(got[2][0].isnan().all()) and bool(got[3].isnan().all())
    loss.close()


@pytest.mark.parametrize("rows", [3, 70, 300])
@pytest.mark.parametrize("cap", [30.0, 50.0, 7.3])
def test_infinity_under_a_softcap(rows, cap):
    """Infinite sums are logits of +-cap. The slope 1 - (z / cap)^2 there is 0 but for 1 / cap's, the quotient's and the last
    rounding, 5 u in all; the probabilities less the target add up to at most 2 in magnitude."""
    import torch
    t = twd()
    h, w, targets, grad = make(VOCAB, D, rows, 0, 5)
    w[:, 6] = torch.where(w[:, 6] == 0, torch.ones_like(w[:, 6]), w[:, 6])
    loss = t.HeadLoss(rows, VOCAB, D, softcap=cap)
    clean = run(loss, h, w, targets, grad)
    for value in (float("inf"), -float("inf")):
        h[0, 6] = value
        losses, lse, d_hidden, d_weight = got = run(loss, h, w, targets, grad)
        assert same_but_row_0(got, clean)
        z = cap * torch.sign(w[:, 6].double()) * (1 if value > 0 else -1)
        want = torch.logsumexp(z, 0)
        tol = (8 + cap + float(want)) * U
        assert abs(float(lse[0]) - float(want)) <= tol
        assert abs(float(losses[0]) - float(want - z[int(targets[0])])) <= 2 * tol
        most = 2 * 5 * U * float(w.float().abs().max()) * abs(float(grad[0]))
        assert float(d_hidden[0].float().abs().max()) <= 1.1 * most
        assert not bool(torch.isfinite(d_weight[:, 6]).any())
        others = torch.arange(D, device="cuda:0") != 6
        assert bool(torch.isfinite(d_weight[:, others]).all())
    # 0 times infinity, and infinities of both signs: no sum, so no loss
    for v, c, value in ((17, 6, float("inf")), (18, 7, -float("inf"))):
        bad, wz = h.clone(), w.clone()
        bad[0, 6], bad[0, c] = float("inf"), value
        if c == 6:
            wz[v, 6] = 0
        else:
            wz[v, 6] = wz[v, 7] = 1
        got = run(loss, bad, wz, targets, grad)
        assert bool(got[0][0].isnan()) and bool(got[2][0].isnan().all())
    loss.close()
