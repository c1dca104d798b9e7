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
    (131075, 64, 33, 30.0), (40961, 96, 100, 0.0), (2000, 352, 128, 30.0), (70001, 1984, 128, 30.0), (70001, 1984, 21, 0.0),
    (1100003, 32, 128, 30.0),
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


def test_many_rows():
    """More rows than the gather takes singly, half of them left out, in many pieces of the vocabulary."""
    import torch
    t = twd()
    vocab, d, rows = 700, 32, 65536
    h, w, targets, grad = make(vocab, d, rows, rows // 2, 9)
    want, tol = reference(h, w, targets, 0.0, grad)
    loss = t.HeadLoss(rows, vocab, d)
    losses, lse = loss.forward(h, w, targets)
    check("losses", losses, want["losses"], tol["losses"], U)
    d_hidden, d_weight = loss.backward(h, w, targets, lse, grad=grad)
    check("d_hidden", d_hidden, want["d_hidden"], tol["d_hidden"], U16)
    check("d_weight", d_weight, want["d_weight"], tol["d_weight"], U16)
    loss.close()


@pytest.mark.parametrize("vocab,d,rows", [(1000, 160, 5), (777, 96, 100), (2049, 224, 300)])
def test_strides_accumulation_and_parts_left_alone(vocab, d, rows):
    """Rows inside wider buffers on every side; gradients on top of others; either gradient alone; the same results
    whatever the object's size, run after run."""
    import torch
    t = twd()
    h, w, targets, grad = make(vocab, d, rows, rows // 3, 4)
    want, tol = reference(h, w, targets, 30.0, grad)
    nan = float("nan")
    hw = torch.full((rows, d + 24), nan, dtype=torch.bfloat16, device="cuda:0")
    ww = torch.full((vocab, d + 8), nan, dtype=torch.bfloat16, device="cuda:0")
    hw[:, 8:d + 8], ww[:, :d] = h, w
    loss, large = t.HeadLoss(rows, vocab, d, softcap=30.0), t.HeadLoss(rows + 1000, vocab, d, softcap=30.0)
    losses, lse = loss.forward(hw[:, 8:d + 8], ww[:, :d], targets)
    check("losses", losses, want["losses"], tol["losses"], U)
    again = large.forward(h, w, targets)
    assert torch.equal(losses, again[0]) and torch.equal(lse, again[1])
    for dt, step in ((torch.float32, U), (torch.bfloat16, U16)):
        base = torch.randn(vocab, d, device="cuda:0").to(dt)
        dw = torch.full((vocab + 1, d + 8), 7.0, dtype=dt, device="cuda:0")
        dh = torch.full((rows + 1, d + 16), 7.0, dtype=torch.bfloat16, device="cuda:0")
        dw[:vocab, :d] = base
        loss.backward(h, w, targets, lse, grad=grad, d_hidden=dh[:rows, 8:d + 8], d_weight=dw[:vocab, :d], accumulate=True)
        check("d_hidden", dh[:rows, 8:d + 8], want["d_hidden"], tol["d_hidden"], U16)
        check("d_weight", dw[:vocab, :d], base.double() + want["d_weight"], tol["d_weight"] + U * base.double().abs(), step)
        assert (dw[vocab] == 7).all() and (dw[:, d:] == 7).all()
        assert (dh[rows] == 7).all() and (dh[:, :8] == 7).all() and (dh[:, d + 8:] == 7).all()
    both = loss.backward(h, w, targets, lse, grad=grad)
    alone = large.backward(h, w, targets, lse, grad=grad, need=(True, False))
    assert alone[1] is None and torch.equal(alone[0], both[0])
    alone = large.backward(h, w, targets, lse, grad=grad, need=(False, True))
    assert alone[0] is None and torch.equal(alone[1], both[1])
    ones = loss.backward(h, w, targets, lse)
    assert torch.equal(ones[0], loss.backward(h, w, targets, lse, grad=torch.ones(rows, device="cuda:0"))[0])
    loss.close(), large.close()


@pytest.mark.parametrize("rows", [3, 70, 300])
def test_nan_and_infinity(rows):
    """What a row that is left out holds does not matter, nor its weight; a NaN in one that counts is its loss's alone."""
    import torch
    t = twd()
    vocab, d = 600, 96
    h, w, targets, grad = make(vocab, d, rows, 0, 5)
    targets[1] = -100
    clean = [x.clone() for x in (h, grad)]
    h[1, ::2], h[1, 1::2], grad[1] = float("nan"), float("inf"), float("nan")
    loss = t.HeadLoss(rows, vocab, d)
    losses, lse = loss.forward(h, w, targets)
    d_hidden, d_weight = loss.backward(h, w, targets, lse, grad=grad)
    losses2, lse2 = loss.forward(clean[0], w, targets)
    d_hidden2, d_weight2 = loss.backward(clean[0], w, targets, lse2, grad=clean[1])
    for a, b in ((losses, losses2), (lse, lse2), (d_hidden, d_hidden2), (d_weight, d_weight2)):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())
    h[0, 5] = float("nan")
    losses, lse = loss.forward(h, w, targets)
    assert bool(torch.isnan(losses[0])) and torch.equal(losses[1:], losses2[1:])
    d_hidden, d_weight = loss.backward(h, w, targets, lse, grad=grad)
    assert bool(torch.isnan(d_hidden[0]).all()) and torch.equal(d_hidden[1:], d_hidden2[1:])
    assert bool(torch.isnan(d_weight).all())
    h[0, 5], h[0, 6] = 0.0, float("inf")  # infinite logits: no loss
    assert bool(torch.isnan(loss.forward(h, w, targets)[0][0]))
    loss.close()


def test_extreme_logits():
    """Logits far apart and far up: the largest alone counts; the loss of others is their distance."""
    import torch
    t = twd()
    vocab, d = 300, 32
    w = torch.zeros(vocab, d, dtype=torch.bfloat16, device="cuda:0")
    w[:, 0] = torch.linspace(-1, 1, vocab, device="cuda:0")
    h = torch.zeros(4, d, dtype=torch.bfloat16, device="cuda:0")
    h[0, 0], h[1, 0], h[2, 0], h[3, 0] = 2.0 ** 20, -(2.0 ** 20), 0.0, 2.0 ** 100
    targets = torch.tensor([vocab - 1, 0, 5, 0], dtype=torch.int32, device="cuda:0")
    loss = t.HeadLoss(4, vocab, d)
    losses, lse = loss.forward(h, w, targets)
    z = h.double() @ w.double().t()
    want = torch.logsumexp(z, 1)
    assert bool(((lse.double() - want).abs() <= 4 * U * want.abs() + 1e-6).all())
    gap = want - z.gather(1, targets.long()[:, None])[:, 0]
    assert bool(((losses.double() - gap).abs() <= 4 * U * (want.abs() + gap)).all())
    d_hidden, d_weight = loss.backward(h, w, targets, lse)
    assert bool(torch.isfinite(d_hidden).all()) and bool(torch.isfinite(d_weight).all())
    assert bool((d_hidden[:2] == 0).all())  # the target has all of the probability
    loss.close()


@pytest.mark.parametrize("rows", [5, 100])
def test_logits_below_fp32(rows):
    """Whole tiles of logits that are minus infinity have no part in a row's sum, as vocabulary rows that are not there."""
    import torch
    t = twd()
    vocab, d, low = 700, 64, 300
    h, w, targets, grad = make(vocab - low, d, rows, 0, 31)
    h = h.abs() + 0.5
    want, tol = reference(h, w, targets, 0.0, grad)
    all_w = torch.cat([torch.full((low, d), -3e38, dtype=torch.bfloat16, device="cuda:0"), w])
    loss = t.HeadLoss(rows, vocab, d)
    losses, lse = loss.forward(h, all_w, targets + low)
    check("lse", lse, want["lse"], tol["lse"], U)
    check("losses", losses, want["losses"], tol["losses"], U)
    d_hidden, d_weight = loss.backward(h, all_w, targets + low, lse, grad=grad)
    check("d_hidden", d_hidden, want["d_hidden"], tol["d_hidden"], U16)
    check("d_weight", d_weight[low:], want["d_weight"], tol["d_weight"], U16)
    assert (d_weight[:low] == 0).all()


def test_stride_of_a_single_row_plays_no_part():
    import torch
    t = twd()
    d = 96
    h, w, targets, grad = make(1, d, 1, 0, 5)
    loss = t.HeadLoss(1, 1, d)
    losses, lse = loss.forward(h, w, targets)
    want = (losses, lse, *loss.backward(h, w, targets, lse, grad=grad))
    for n in (0, 13, 2 ** 40):
        got = [torch.full_like(x, float("nan")) for x in want]
        p = [x.data_ptr() for x in got]
        torch.cuda.synchronize()
        assert t.lib.twd_headloss_forward(loss.handle, h.data_ptr(), 1, n, w.data_ptr(), n, targets.data_ptr(), p[0],
                                          p[1], None) == t.TWD_OK
        assert t.lib.twd_headloss_backward(loss.handle, h.data_ptr(), 1, n, w.data_ptr(), n, targets.data_ptr(), p[1],
                                           grad.data_ptr(), p[2], n, p[3], 1, n, 0, None) == t.TWD_OK
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gradient_by_differences():
    """d_weight against central differences of the losses themselves. One logit of a row changes by delta h: the third
    derivative of the loss by it is p (1 - p) (1 - 2 p), at most 0.0963, so the difference is off by delta^2 |h|^3 0.0963 / 6 a
    row, and by two losses' errors over 2 delta; the gradient by 2^-8 of its terms."""
    import torch
    t = twd()
    vocab, d, rows, delta = 40, 64, 70, 2.0 ** -4
    rng = np.random.default_rng(3)
    h = torch.from_numpy(rng.integers(-4, 5, (rows, d)) / 4.0).cuda().bfloat16()
    w = torch.from_numpy(rng.integers(-8, 9, (vocab, d)) / 16.0).cuda().bfloat16()  # steps of delta are exact
    targets = torch.from_numpy(rng.integers(0, vocab, rows)).to(torch.int32).cuda()
    targets[::7] = -1
    loss = t.HeadLoss(rows, vocab, d)
    _, lse = loss.forward(h, w, targets)
    _, grad = loss.backward(h, w, targets, lse, d_weight=torch.empty(vocab, d, device="cuda:0"))
    live = (targets >= 0)
    size = h[live].double().abs()
    for _ in range(30):
        v, c = int(rng.integers(vocab)), int(rng.integers(d))
        ends = []
        for sign in (1, -1):
            moved = w.clone()
            moved[v, c] += sign * delta
            ends.append(loss.forward(h, moved, targets)[0].double().sum())
        diff = float((ends[0] - ends[1]) / (2 * delta))
        tol = float((delta ** 2 * size[:, c] ** 3 * 0.0963 / 6).sum()) + 2 * rows * 30 * U / (2 * delta) + U16 * float(size[:, c].sum())
        assert abs(diff - float(grad[v, c])) <= tol, (v, c, diff, float(grad[v, c]), tol)
    loss.close()


@pytest.mark.parametrize("rows", [3, 100])
def test_far_rows(rows):
    """Weight rows more than 4 GiB from the first, at the widest stride; hidden rows too."""
    import torch
    t = twd()
    vocab, d, far = 600, 32, 1 << 22
    h, w, targets, grad = make(vocab, d, rows, 1, 6)
    wide = torch.empty((vocab - 1) * far + d, dtype=torch.bfloat16, device="cuda:0").as_strided((vocab, d), (far, 1))
    wide.copy_(w)
    hw = torch.empty((rows - 1) * far + d, dtype=torch.bfloat16, device="cuda:0").as_strided((rows, d), (far, 1))
    hw.copy_(h)
    loss = t.HeadLoss(rows, vocab, d)
    a, b = loss.forward(h, w, targets), loss.forward(hw, wide, targets)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x, y = loss.backward(h, w, targets, a[1]), loss.backward(hw, wide, targets, a[1], d_weight=wide.clone())
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    loss.close()


def test_streams_and_graphs():
    """One object's calls on two streams in turn; captured forward and backward passes replayed with other rows, other
    targets and another number of rows that count."""
    import torch
    t = twd()
    vocab, d = 3001, 160
    sets = [make(vocab, d, n, n // 4, n) for n in (200, 30)]
    loss = t.HeadLoss(200, vocab, d, softcap=30.0)
    refs = []
    for h, w, targets, grad in sets:
        losses, lse = loss.forward(h, w, targets)
        refs.append((losses, lse) + loss.backward(h, w, targets, lse, grad=grad))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, (h, w, targets, grad) in zip(streams, sets):
            losses, lse = loss.forward(h, w, targets, stream=s.cuda_stream)
            got.append((losses, lse) + loss.backward(h, w, targets, lse, grad=grad, stream=s.cuda_stream))
        torch.cuda.synchronize()
        for a, b in zip(got, refs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    for n in (200, 100, 40):
        h, w, targets, grad = [x.clone() for x in make(vocab, d, n, 0, 77)]
        out = [torch.empty(n, device="cuda:0"), torch.empty(n, device="cuda:0"), torch.empty_like(h), torch.empty_like(w)]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            loss.forward(h, w, targets, losses=out[0], lse=out[1], stream=streams[0].cuda_stream)
            loss.backward(h, w, targets, out[1], grad=grad, d_hidden=out[2], d_weight=out[3], stream=streams[0].cuda_stream)
        for rep in range(4):
            new = make(vocab, d, n, n * rep // 3, 100 + rep)
            for x, y in zip((h, w, targets, grad), new):
                x.copy_(y)
            torch.cuda.synchronize()
            losses, lse = loss.forward(*new[:3])  # eager work between the replays
            want = (losses, lse) + loss.backward(*new[:3], lse, grad=new[3])
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, want)), (n, rep)
        del g
    loss.close()
