"""The embedding lookup with scaling (embed) and its gradient (EmbedGrad) against the definition in 64 bits.

Bounds: a looked up value is off by half a step of fp32 for its product and half a step of its type; a gradient by
n 2^-24 of the sum of magnitudes for n - 1 additions and the scale, one addition more where it is accumulated, and half
a step of its type (below the normal numbers an absolute one)."""
import numpy as np
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"float32": (U, 2.0 ** -150), "bfloat16": (2.0 ** -8, 2.0 ** -134), "float16": (2.0 ** -11, 2.0 ** -25)}
NAMES = list(TYPES)


def half_step(x, name):
    step, least = TYPES[name]
    return step * x.abs() + least


def matrix(rows, cols, name, seed, pad=0, start=0):
    """[rows, cols] of normal values within a wider buffer."""
    import torch
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    wide = torch.randn(rows, cols + pad + start, generator=g, device="cuda:0").to(getattr(torch, name))
    return wide[:, start:start + cols]


def some_ids(n, vocab, seed, share_out=0.2):
    rng = np.random.default_rng(seed)
    ids = np.minimum(np.exp(rng.random(n) * np.log(vocab + 1)) - 1, vocab - 1).astype(np.int32)
    out = rng.random(n) < share_out
    ids[out] = rng.choice(np.array([-1, -100, vocab, 2 ** 31 - 1, -2 ** 31], np.int32), out.sum())
    return ids


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("n,vocab,d,pad,start", [(1, 1, 1, 0, 0), (1, 1000, 5376, 0, 0), (3, 7, 13, 3, 0), (517, 300, 2048, 0, 0),
                                                 (600, 1000, 2049, 0, 0), (1030, 50, 777, 8, 1), (9, 33, 6152, 8, 0),
                                                 (511, 20, 8, 0, 0), (513, 20, 7, 1, 0)])
@pytest.mark.parametrize("table", NAMES)
@pytest.mark.parametrize("out", NAMES)
def test_lookup(n, vocab, d, pad, start, table, out):
    import torch
    t = twd()
    w, ids = matrix(vocab, d, table, n, pad, start), some_ids(n, vocab, d)
    got = torch.full((n + 1, d + 3), 7.0, device="cuda:0").to(getattr(torch, out))
    for scale in (1.0, float(np.float32(d ** 0.5))):
        t.embed(w, dev(ids), scale=scale, out=got[:n, 1:d + 1])
        live = (ids >= 0) & (ids < vocab)
        want = torch.where(dev(live)[:, None], w[dev(np.where(live, ids, 0)).long()].double() * scale, 0.0)
        err = (got[:n, 1:d + 1].double() - want).abs()
        assert bool((err <= U * want.abs() + half_step(want * (1 + U), out)).all())
        assert bool((got[n] == 7).all()) and bool((got[:, 0] == 7).all()) and bool((got[:, d + 1:] == 7).all())
    made = t.embed(w, dev(ids), dtype=getattr(torch, out))
    assert made.dtype == getattr(torch, out) and made.shape == (n, d)


def test_lookup_of_nothing():
    import torch
    t = twd()
    out = t.embed(torch.ones(4, 8, device="cuda:0"), torch.empty(0, dtype=torch.int32, device="cuda:0"))
    assert out.shape == (0, 8)


def reference(rows, ids, vocab, scale):
    import torch
    keep = dev((ids >= 0) & (ids < vocab))
    at = dev(ids).long()[keep]
    total, size = (torch.zeros(vocab, rows.shape[1], dtype=torch.float64, device="cuda:0") for _ in range(2))
    total.index_put_((at,), rows[keep].double(), accumulate=True)
    size.index_put_((at,), rows[keep].double().abs(), accumulate=True)
    n = torch.bincount(at, minlength=vocab).double()[:, None]
    return total * scale, size * abs(scale) * (n + 1) * U


GRADS = [(1, 1, 1), (1, 3, 8), (2, 5, 13), (31, 4, 64), (32, 1, 40), (33, 2, 2056), (100, 1000, 5376), (513, 300, 1024),
         (2048, 10, 96), (2049, 4000, 33), (5000, 7, 256), (9001, 30000, 72), (70000, 11, 24), (262144, 5000, 8)]


@pytest.mark.parametrize("n,vocab,d", GRADS)
@pytest.mark.parametrize("rows,table", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float16"),
                                        ("bfloat16", "float32"), ("float16", "bfloat16"), ("float32", "float16")])
def test_gradient(n, vocab, d, rows, table):
    import torch
    t = twd()
    scale = 0.37
    x, ids = matrix(n, d, rows, n + d), some_ids(n, vocab, n)
    want, tol = reference(x, ids, vocab, scale)
    g = t.EmbedGrad(n, d)
    dt = getattr(torch, table)
    guard = torch.full((vocab * d + 16,), 5.0, device="cuda:0").to(dt)
    out = guard[8:8 + vocab * d].view(vocab, d)
    x_nan = x.clone()
    x_nan[dev((ids < 0) | (ids >= vocab))] = float("nan")  # rows that are left out are not read
    assert g.run(x_nan, dev(ids), out, scale=scale) is out
    first = out.clone()
    assert bool(((out.double() - want).abs() <= tol + half_step(want.abs() + tol, table)).all())
    assert bool((guard[:8] == 5).all()) and bool((guard[8 + vocab * d:] == 5).all())
    # the same again, bit for bit, at an odd place and into rows apart
    wide = torch.full((vocab, d + 5), 3.0, device="cuda:0").to(dt)
    g.run(x, dev(ids), wide[:, 1:d + 1], scale=scale)
    assert torch.equal(wide[:, 1:d + 1], first)
    assert bool((wide[:, 0] == 3).all()) and bool((wide[:, d + 1:] == 3).all())
    # on top of what is there
    base = matrix(vocab, d, table, 3).contiguous()
    more = base.clone()
    g.run(x, dev(ids), more, scale=scale, accumulate=True)
    whole = base.double() + want
    tol = tol + U * (whole.abs() + tol)
    assert bool(((more.double() - whole).abs() <= tol + half_step(whole.abs() + tol, table)).all())
    idle = torch.ones(vocab, dtype=torch.bool)
    idle[ids[(ids >= 0) & (ids < vocab)]] = False
    idle = idle.cuda()
    assert torch.equal(more[idle], base[idle]) and bool((first[idle] == 0).all())
    g.close()


@pytest.mark.parametrize("n", [1, 64, 65, 96, 127, 4096, 16384])
def test_all_ids_the_same_and_none(n):
    import torch
    t = twd()
    x = torch.ones(n, 40, device="cuda:0")
    g = t.EmbedGrad(16384, 40)
    out = torch.full((9, 40), 2.0, device="cuda:0")
    g.run(x, torch.full((n,), 4, dtype=torch.int32, device="cuda:0"), out)
    assert bool((out[4] == n).all()) and bool((out.sum(0) == n).all())
    g.run(x, torch.full((n,), -1, dtype=torch.int32, device="cuda:0"), out)
    assert bool((out == 0).all())
    out.fill_(2.0)
    g.run(x[:0], torch.empty(0, dtype=torch.int32, device="cuda:0"), out, accumulate=True)
    assert bool((out == 2).all())
    g.run(x[:0], torch.empty(0, dtype=torch.int32, device="cuda:0"), out)
    assert bool((out == 0).all())
    g.close()


def test_gradient_is_the_lookups():
    """<embed(table), r> has the gradient that EmbedGrad gives of r: against differences, exact in 64 bits of integers."""
    import torch
    t = twd()
    rng = np.random.default_rng(5)
    ids = some_ids(300, 40, 1)
    w = dev(rng.integers(-8, 9, (40, 56)).astype(np.float32))
    r = dev(rng.integers(-8, 9, (300, 56)).astype(np.float32))
    g = t.EmbedGrad(300, 56)
    grad = g.run(r, dev(ids), torch.empty(40, 56, device="cuda:0"), scale=2.0)
    for _ in range(20):
        v, c = int(rng.integers(40)), int(rng.integers(56))
        up = w.clone()
        up[v, c] += 1
        diff = ((t.embed(up, dev(ids), scale=2.0) - t.embed(w, dev(ids), scale=2.0)).double() * r.double()).sum()
        assert float(diff) == float(grad[v, c])
    g.close()


def test_far_rows():
    """Table rows more than 4 GiB from the first."""
    import torch
    t = twd()
    vocab, d = 5, 1032
    far = (1 << 31) // (vocab - 1) + 64
    w = torch.empty((vocab - 1) * far + d, dtype=torch.bfloat16, device="cuda:0").as_strided((vocab, d), (far, 1))
    values = matrix(vocab, d, "bfloat16", 1)
    w.copy_(values)
    ids = torch.tensor([4, 0, 4, 2], dtype=torch.int32, device="cuda:0")
    assert torch.equal(t.embed(w, ids), values[ids.long()])
    g = t.EmbedGrad(4, d)
    g.run(values[:4], ids, w)
    want, _ = reference(values[:4], ids.cpu().numpy(), vocab, 1.0)
    assert bool(((w.double() - want).abs() <= 2 * half_step(want, "bfloat16")).all())
    g.close()


def test_streams_and_graphs():
    """Calls of one object from two streams in turn, and captured calls replayed with other ids and rows."""
    import torch
    t = twd()
    g = t.EmbedGrad(5000, 64)
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [(matrix(n, 64, "float32", n), some_ids(n, 900, n)) for n in (5000, 700)]
    refs = [reference(x, i, 900, 1.0) for x, i in sets]
    outs = [torch.empty(900, 64, device="cuda:0") for _ in sets]
    on = [dev(i) for _, i in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (x, _), i, o in zip(streams, sets, on, outs):
            g.run(x, i, o, stream=s.cuda_stream)
        torch.cuda.synchronize()
        for o, (want, tol) in zip(outs, refs):
            assert bool(((o.double() - want).abs() <= tol + half_step(want.abs() + tol, "float32")).all())
    w = matrix(900, 64, "float32", 8)
    x, ids, looked, out = sets[0][0].clone(), on[0].clone(), torch.empty(5000, 64, device="cuda:0"), outs[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        t.embed(w, ids, out=looked, stream=streams[0].cuda_stream)
        g.run(x, ids, out, stream=streams[0].cuda_stream)
    for rep in range(4):
        i, r = some_ids(5000, 900, 50 + rep), matrix(5000, 64, "float32", 60 + rep)
        ids.copy_(dev(i)), x.copy_(r)
        torch.cuda.synchronize()
        t.embed(w, on[1])  # eager work between the replays
        graph.replay()
        torch.cuda.synchronize()
        want, tol = reference(r, i, 900, 1.0)
        assert bool(((out.double() - want).abs() <= tol + half_step(want.abs() + tol, "float32")).all())
        assert torch.equal(looked, t.embed(w, ids))
    g.close()
