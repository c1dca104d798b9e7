"""A head's softmax cross entropy and its gradients (HeadLoss) against the definition in 64 bits.

Bounds, with u = 2^-24 and u16 = 2^-8 (half a step of fp32 and of bf16): a logit is off by
dz = K 2 u sum |w h| + 4 u |z| (the sum's K additions, the softcap); lse and the loss by twice the largest dz and
(8 + |z| + |lse|) u for exponents, logarithm and roundings. A probability is then off by e_p = dz + dlse + 2^-20 of
itself, a term of a gradient by u16 of itself and e_p of its probability, and a gradient by the sum of these times the
other factor, 2 u a term for the sum, and half a step of its type."""
import numpy as np
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu

U, U16 = 2.0 ** -24, 2.0 ** -8

SHAPES = [  # vocab, d_model, rows, softcap
    (1, 32, 1, 0.0), (5, 32, 3, 30.0), (257, 96, 2, 0.0), (1000, 160, 64, 30.0), (1003, 1056, 65, 0.0),
    (777, 2880, 129, 30.0), (4099, 512, 300, 50.0), (300, 544, 600, 0.0), (256, 128, 128, 0.0), (2049, 64, 257, 5.0),
    (40001, 64, 40, 30.0), (131075, 32, 1030, 0.0), (515, 5376, 17, 30.0),
]


def make(vocab, d, rows, out, seed, spread=3.6):
    """Hidden rows, weights and targets; `out` of the rows left out, with targets below and past the vocabulary."""
    import torch
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    w = (torch.randn(vocab, d, generator=g, device="cuda:0") * spread / d ** 0.5).bfloat16()
    t = torch.randint(vocab, (rows,), generator=g, device="cuda:0")
    lean = 16 * torch.rand(rows, 1, generator=g, device="cuda:0") / spread ** 2
    h = (torch.randn(rows, d, generator=g, device="cuda:0") + lean * w[t].float()).bfloat16()
    t = t.to(torch.int32)
    gone = torch.randperm(rows, generator=g, device="cuda:0")[:out]
    t[gone] = torch.tensor([-100, -1, vocab, 2 ** 31 - 1], dtype=torch.int32, device="cuda:0").repeat(out // 4 + 1)[:out]
    grad = torch.randn(rows, generator=g, device="cuda:0")
    return h, w, t, grad


def reference(h, w, t, cap, grad):
    """The definition in 64 bits and the bounds of the results: a dict of (value, bound)."""
    import torch
    vocab, d = w.shape
    hd, wd = h.double(), w.double()
    keep = (t >= 0) & (t < vocab)
    hk, tk, gk = hd[keep], t[keep].long(), grad.double()[keep]
    x = hk @ wd.t().contiguous()
    size = hk.abs() @ wd.abs().t().contiguous()
    z = cap * torch.tanh(x / cap) if cap > 0 else x
    dz = d * 2 * U * size + 4 * U * z.abs()
    lse = torch.logsumexp(z, 1)
    hit = z.gather(1, tk[:, None])[:, 0]
    worst = dz.amax(1)
    dlse = worst + (8 + z.abs().amax(1) + lse.abs()) * U
    out = {"lse": torch.zeros(len(t)).cuda().double(), "losses": torch.zeros(len(t)).cuda().double()}
    tol = {k: torch.zeros_like(v) for k, v in out.items()}
    out["lse"][keep], tol["lse"][keep] = lse, dlse
    out["losses"][keep], tol["losses"][keep] = lse - hit, 2 * worst + 2 * (8 + z.abs().amax(1) + lse.abs()) * U
    p = torch.exp(z - lse[:, None])
    slope = 1 - (z / cap) ** 2 if cap > 0 else torch.ones_like(z)
    q = p.clone()
    q[torch.arange(len(tk)), tk] -= 1
    term = q * slope * gk[:, None]
    e_p = dz + dlse[:, None] + 2.0 ** -20
    off = U16 * term.abs() + (e_p * p * slope + 4 * U * q.abs() + (2 * dz / cap * q.abs() if cap > 0 else 0)) * gk.abs()[:, None]
    off = off * (1 + U16)
    for name, a, b, n in (("d_hidden", term, wd, vocab), ("d_weight", term.t().contiguous(), hk, max(1, len(tk)))):
        o = off if name == "d_hidden" else off.t().contiguous()
        value = a @ b
        bound = o @ b.abs() + n * 2 * U * (a.abs() @ b.abs())
        if name == "d_hidden":
            whole, whole_tol = (torch.zeros(len(t), d, dtype=torch.float64, device="cuda:0") for _ in range(2))
            whole[keep], whole_tol[keep] = value, bound
            value, bound = whole, whole_tol
        out[name], tol[name] = value, bound
    return out, tol


def check(name, got, want, tol, half_step):
    err = (got.double() - want).abs()
    bound = tol + half_step * (want.abs() + tol)
    assert bool((err <= bound).all()), (name, float((err - bound).max()), float(err.max()))


@pytest.mark.parametrize("vocab,d,rows,cap", SHAPES)
@pytest.mark.parametrize("share", [0.0, 0.4, 1.0])
def test_loss_and_gradients(vocab, d, rows, cap, share):
    import torch
    t = twd()
    h, w, targets, grad = make(vocab, d, rows, int(share * rows), vocab + rows)
    want, tol = reference(h, w, targets, cap, grad)
    loss = t.HeadLoss(rows, vocab, d, softcap=cap)
    losses, lse = loss.forward(h, w, targets)
    check("lse", lse, want["lse"], tol["lse"], U)
    check("losses", losses, want["losses"], tol["losses"], U)
    d_hidden, d_weight = loss.backward(h, w, targets, lse, grad=grad)
    check("d_hidden", d_hidden, want["d_hidden"], tol["d_hidden"], U16)
    check("d_weight", d_weight, want["d_weight"], tol["d_weight"], U16)
    left_out = (targets < 0) | (targets >= vocab)
    assert (losses[left_out] == 0).all() and (lse[left_out] == 0).all() and (d_hidden[left_out] == 0).all()
    full = torch.full((vocab, d), float("nan"), device="cuda:0")
    loss.backward(h, w, targets, lse, grad=grad, d_weight=full, need=(False, True))
    check("d_weight fp32", full, want["d_weight"], tol["d_weight"], U)
    loss.close()
