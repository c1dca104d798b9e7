"""Sampler.sample against the definition in 64 bits: ids and kept counts have to be equal. Weights carry 37
bits and sums are exact, so a logprob is off by at most half a step of fp32 and 2^-36."""
import math

import numpy as np
import pytest

from helpers import hidden_bf16, twd

pytestmark = pytest.mark.gpu

DEGENERATE = (-1, None, 0)


def sample_ref(l, temp, k, p, mp, u):
    l = l.astype(np.float64)
    if np.isnan(l).any() or (l == np.inf).any() or not (l > -np.inf).any() or any(map(math.isnan, (temp, p, mp, u))):
        return DEGENERATE
    if temp <= 0:
        return int(np.argmax(l)), 0.0, 1
    order = np.argsort(-l, kind="stable")
    n = int((l > -np.inf).sum())
    if k > 0:
        n = min(n, k)
    z = (l - l[order[0]]) / temp if math.isfinite(temp) else np.where(l > -np.inf, 0.0, -np.inf)
    w = np.exp(z)
    ws = w[order[:n]]
    if p < 1:
        run = np.cumsum(ws)
        n = min(n, int(np.searchsorted(run, p * run[-1], side="left")) + 1)
    if mp > 0:
        n = min(n, max(1, int(np.count_nonzero(ws >= mp))))
    ids = np.sort(order[:n])
    run = np.cumsum(w[ids])
    if u >= 1:
        i = int(np.searchsorted(run, run[-1], side="left"))
    else:
        i = int(np.searchsorted(run, max(u, 0.0) * run[-1], side="right"))
    return int(ids[i]), z[ids[i]] - math.log(run[-1]), n


def check(logits, temps, ks, ps, mps, us, sampler=None, tag=""):
    """logits: a device tensor [rows, vocab]; the parameters: one number per row, or None."""
    import torch
    t = twd()
    rows, vocab = logits.shape
    sam = sampler or t.Sampler(vocab, rows)

    def d(a, dt=torch.float32):
        return None if a is None else torch.tensor(a, dtype=dt, device="cuda:0")

    logp = torch.full((rows,), 5.0, device="cuda:0")
    kept = torch.full((rows,), -9, dtype=torch.int32, device="cuda:0")
    before = logits.clone()
    tok = sam.sample(logits, d(us), d(temps), d(ks, torch.int32), d(ps), d(mps), logprobs=logp, kept=kept)
    tok, logp, kept = tok.cpu().tolist(), logp.double().cpu().tolist(), kept.cpu().tolist()
    assert torch.equal(torch.nan_to_num(before.float()), torch.nan_to_num(logits.float()))  # rows stay as they were
    host = logits.double().cpu().numpy()
    f32 = lambda a, i, default: default if a is None else float(np.float32(a[i]))
    for m in range(rows):
        want = sample_ref(host[m], f32(temps, m, 1.0), 0 if ks is None else ks[m], f32(ps, m, 1.0), f32(mps, m, 0.0),
                          f32(us, m, 0.0))
        what = (tag, m, vocab, f32(temps, m, 1.0), None if ks is None else ks[m], f32(ps, m, 1.0), f32(mps, m, 0.0),
                f32(us, m, 0.0))
        assert (tok[m], kept[m]) == (want[0], want[2]), what
        if want[1] is None:
            assert math.isnan(logp[m]), what
        else:
            assert abs(logp[m] - want[1]) <= 2.0 ** -24 * abs(want[1]) + 2.0 ** -36, what
    if sampler is None:
        sam.close()


def rows_of(rng, rows, vocab, sigma=3.6, cap=30.0):
    z = sigma * rng.standard_normal((rows, vocab))
    return (cap * np.tanh(z / cap)).astype(np.float32)


def dev(a, dtype="float32", pad=0, offset=0):
    import torch
    rows, vocab = a.shape
    dt = getattr(torch, dtype)
    buf = torch.zeros(rows * (vocab + pad) + offset, dtype=dt, device="cuda:0")
    v = buf[offset:].view(rows, vocab + pad)[:, :vocab]
    v.copy_(torch.from_numpy(a).to(dt))
    return v


def mixed(rng, rows, vocab):
    temps, ks, ps, mps, us = [], [], [], [], []
    for m in range(rows):
        temps.append(float(rng.choice([0.0, 0.3, 0.7, 1.0, 1.7], p=[.1, .15, .3, .3, .15])))
        ks.append(int(rng.choice([0, 1, int(rng.integers(2, 200)), int(rng.integers(1, vocab + 2))], p=[.4, .05, .35, .2])))
        ps.append(float(rng.choice([1.0, rng.uniform(0.5, 0.999), rng.uniform(0.0, 0.2)], p=[.3, .6, .1])))
        mps.append(float(rng.choice([0.0, rng.uniform(0.001, 0.2)])))
        us.append(float(rng.integers(0, 1 << 24)) / (1 << 24))
    return temps, ks, ps, mps, us


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab,pad,offset", [(1, 1, 0, 0), (3, 2, 0, 0), (5, 63, 1, 0), (4, 1000, 0, 1), (9, 4096, 0, 0),
                                                   (8, 4097, 3, 5), (16, 32003, 5, 1), (24, 151669, 0, 0),
                                                   (12, 262144, 0, 0), (2, 524288, 8, 3), (3, 262143, 1, 1)])
def test_mixed_parameters(dtype, rows, vocab, pad, offset):
    rng = np.random.default_rng(rows * 1000 + vocab)
    lg = dev(rows_of(rng, rows, vocab), dtype, pad, offset)
    check(lg, *mixed(rng, rows, vocab))


@pytest.mark.parametrize("vocab", [300, 40000, 262144])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_wide_nuclei_and_flat_rows(vocab, dtype):
    """Flat rows and high temperatures: cuts deep in the row, where thousands of entries lie close together."""
    rng = np.random.default_rng(vocab)
    a = np.concatenate([rows_of(rng, 8, vocab, 0.3), rows_of(rng, 4, vocab, 0.001), rows_of(rng, 4, vocab, 8.0)])
    n = len(a)
    us = (rng.integers(0, 1 << 24, n) / (1 << 24)).tolist()
    ps = [0.9, 0.5, 0.99, 0.999, 1.0, 0.25, 0.8, 0.95] * 2
    ks = [0, 0, vocab // 2, 0, vocab - 1, 0, vocab // 3, 7] * 2
    check(dev(a, dtype), [1.0, 1.6] * (n // 2), ks, ps, [0.0] * n, us, tag="flat")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_lists_of_thousands(dtype):
    """Between 5,000 and 30,000 entries in the eighth of an octave where a limit cuts: the list is read from memory."""
    rng = np.random.default_rng(7)
    a = rows_of(rng, 8, 262144, 1.0)
    ks = [0, 100000, 0, 60000, 131072, 0, 262143, 200000]
    ps = [0.9, 1.0, 0.8, 0.9, 0.5, 0.95, 0.85, 1.0]
    us = (rng.integers(0, 1 << 24, 8) / (1 << 24)).tolist()
    check(dev(a, dtype), [1.0, 1.0, 1.5, 1.5, 2.0, 2.0, 0.8, 0.8], ks, ps, [0.0] * 7 + [0.3], us, tag="thousands")


@pytest.mark.parametrize("vocab", [1, 17, 4096, 5000, 100000, 262144])
def test_equal_logits(vocab):
    """All logits equal, or two values: every cut falls among ties, which go by index."""
    a = np.full((10, vocab), 1.5, np.float32)
    a[5:, ::3] = 2.5
    k = max(1, vocab // 3)
    ks = [0, k, 0, k, 5, 0, k, 0, k + 1, vocab]
    ps = [1.0, 1.0, 0.5, 0.75, 1.0, 0.5, 0.5, 0.25, 1.0, 0.875]
    us = [0.0, 0.5, 0.25, 0.75, 1 - 2.0 ** -24, 0.125, 0.5, 0.0, 0.625, 0.25]
    check(dev(a), [1.0] * 10, ks, ps, [0.0, 0, 1.0, 0, 0, 0, 1.0, 0.5, 0.25, 0.25], us, tag="equal")


def test_rows_more_than_4_gib_apart():
    import torch
    rng = np.random.default_rng(9)
    far, vocab = (1 << 30) + 5, 20000
    v = torch.empty(far + vocab, device="cuda:0").as_strided((2, vocab), (far, 1))
    v.copy_(torch.from_numpy(rows_of(rng, 2, vocab)))
    check(v, [0.7, 1.2], [0, 300], [0.9, 0.8], [0.0, 0.01], [0.3, 0.8], tag="far")


def test_masks():
    """Rows of -inf but for a few entries, one or none; masks of the type's lowest value; NaN and +inf."""
    rng = np.random.default_rng(5)
    vocab = 20001
    a = np.repeat(rows_of(rng, 1, vocab), 14, 0)
    live = rng.random(vocab) < 0.02
    a[0, ~live] = -np.inf
    a[1] = -np.inf
    a[2] = -np.inf
    a[2, 777] = -5.0
    a[3, ~live] = np.finfo(np.float32).min
    a[4] = np.finfo(np.float32).min
    a[5, 20000] = np.nan
    a[6, 5] = np.inf
    a[7, :] = -np.inf
    a[7, [0, 20000]] = [-1e30, -1e30]
    a[8, ::2] = -1e4
    a[9, 1:] = -np.inf
    a[10] = np.finfo(np.float32).max
    a[11, 3] = 3e38
    a[12] = np.nan
    a[13, :] = -np.inf
    a[13, 20000] = 0.0
    us = (rng.integers(0, 1 << 24, 14) / (1 << 24)).tolist()
    for k, p, mp in ((0, 1.0, 0.0), (50, 0.9, 0.0), (3, 1.0, 0.1), (30000, 0.95, 0.0)):
        check(dev(a), [0.8] * 14, [k] * 14, [p] * 14, [mp] * 14, us, tag=("mask", k, p))
    check(dev(a), [0.0] * 14, None, None, None, us, tag="greedy")


def test_extreme_parameters():
    rng = np.random.default_rng(6)
    a = np.repeat(rows_of(rng, 1, 5003), 20, 0)
    a[18:] *= np.float32(1e30)
    big = float(np.finfo(np.float32).max)
    temps = [1e-6, 1e-30, 1e-45, 1e6, math.inf, math.nan, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, -1.0, -math.inf, 1.0, 1e29]
    ks = [0, 0, 0, 0, 0, 0, -5, 2 ** 31 - 1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0]
    ps = [1, 1, 1, 1, .5, 1, 1, 1, 0.0, -1.0, math.nan, 2.0, 1 - 2.0 ** -24, 1e-45, 1, 1, 1, 1, .9, .9]
    mps = [0, 0, 0, 0, 1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1.0, math.inf, 0, 0, 0, 0.01]
    us = [.5, .5, .5, .3, .7, .5, .9, .1, .5, .5, .5, .5, 1 - 2.0 ** -24, .5, .5, .5, .5, .5, .4, .4]
    assert big > 1e38
    check(dev(a), temps, ks, ps, mps, us, tag="extreme")
    us = [math.nan, -1.0, -0.0, 1.0, 2.0, math.inf, -math.inf, 1 - 2.0 ** -24, 2.0 ** -24, 1e-45]
    check(dev(a[:10]), [0.7] * 10, [40] * 10, None, [-1.0] * 10, us, tag="draws")


@pytest.mark.parametrize("vocab", [9, 6000])
def test_min_p_above_one_and_zero_thresholds(vocab):
    """min_p above 1 keeps the first of the largest; a threshold at 0, and limits met exactly."""
    a = np.full((6, vocab), 2.0, np.float32)
    a[2:, 4:] = 0.0
    a[4, 4::2] = -0.0
    a[5, 1:] = 2.0 - np.float32(math.log(2.0))
    mps = [1.5, math.inf, math.exp(-2.0), math.exp(-2.0) * 0.999999, math.exp(-2.0) * 0.999999, 0.4999999]
    check(dev(a), [1.0] * 6, None, None, mps, [0.7] * 6, tag="min_p")
    check(dev(a), [1.0] * 6, [0, 2, 3, 4, 5, 6], [0.3] * 6, mps, [0.9] * 6, tag="min_p and more")


def test_draws_cover_the_kept_ids():
    """One row under a thousand evenly spread draws: every id comes as often as its weight says."""
    import torch
    rng = np.random.default_rng(7)
    row = rows_of(rng, 1, 1500)
    n = 1000
    lg = dev(np.repeat(row, n, 0))
    check(lg, [1.0] * n, [20] * n, [0.9] * n, None, (np.arange(n) / n).tolist(), tag="spread")


def test_results_do_not_depend_on_the_batch():
    import torch
    t = twd()
    rng = np.random.default_rng(8)
    rows, vocab = 40, 50021
    a = rows_of(rng, rows, vocab)
    temps, ks, ps, mps, us = mixed(rng, rows, vocab)
    f = lambda x, dt=torch.float32: torch.tensor(x, dtype=dt, device="cuda:0")
    sam = t.Sampler(vocab, rows)
    lp = torch.empty(rows, device="cuda:0")
    whole = sam.sample(dev(a), f(us), f(temps), f(ks, torch.int32), f(ps), f(mps), logprobs=lp)
    for m in range(0, rows, 3):
        lp1 = torch.empty(1, device="cuda:0")
        one = sam.sample(dev(a[m:m + 1]), f(us[m:m + 1]), f(temps[m:m + 1]), f(ks[m:m + 1], torch.int32), f(ps[m:m + 1]),
                         f(mps[m:m + 1]), logprobs=lp1)
        assert torch.equal(one, whole[m:m + 1]) and torch.equal(lp1.view(torch.int32), lp[m:m + 1].view(torch.int32)), m
    sam.close()


def test_streams_and_graphs():
    """One sampler from two streams in turn; two captured calls of different sizes replayed in turn, with new
    rows and parameters and eager calls between the replays."""
    import torch
    t = twd()
    rng = np.random.default_rng(9)
    sam = t.Sampler(60000, 16)
    shapes = [(16, 50000), (3, 60000)]
    streams = [torch.cuda.Stream() for _ in shapes]
    bufs = []
    for rows, vocab in shapes:
        bufs.append({"lg": torch.zeros(rows, vocab, device="cuda:0"), "tok": torch.zeros(rows, dtype=torch.int32, device="cuda:0"),
                     "t": torch.ones(rows, device="cuda:0"), "k": torch.zeros(rows, dtype=torch.int32, device="cuda:0"),
                     "p": torch.ones(rows, device="cuda:0"), "m": torch.zeros(rows, device="cuda:0"),
                     "u": torch.zeros(rows, device="cuda:0")})

    def call(b, s):
        sam.sample(b["lg"], b["u"], b["t"], b["k"], b["p"], b["m"], tokens=b["tok"], stream=s.cuda_stream)

    def fill(b):
        rows, vocab = b["lg"].shape
        a = rows_of(rng, rows, vocab, float(rng.choice([1.0, 3.6])))
        ps = mixed(rng, rows, vocab)
        b["lg"].copy_(torch.from_numpy(a))
        for n, v in zip("tkpmu", ps):
            b[n].copy_(torch.tensor(v))
        torch.cuda.synchronize()
        f = lambda x: float(np.float32(x))
        return [sample_ref(a[m], f(ps[0][m]), ps[1][m], f(ps[2][m]), f(ps[3][m]), f(ps[4][m]))[0] for m in range(rows)]

    for rep in range(4):
        i = rep % 2
        want = fill(bufs[i])
        call(bufs[i], streams[i])
        torch.cuda.synchronize()
        assert bufs[i]["tok"].cpu().tolist() == want, rep
    graphs = []
    for b, s in zip(bufs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(b, s)
        graphs.append(g)
    for rep in range(8):
        i = rep % 2
        if rep % 3 == 0:
            want = fill(bufs[1 - i])
            call(bufs[1 - i], streams[0])
            torch.cuda.synchronize()
            assert bufs[1 - i]["tok"].cpu().tolist() == want, rep
        want = fill(bufs[i])
        bufs[i]["tok"].zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert bufs[i]["tok"].cpu().tolist() == want, rep
    del graphs
    sam.close()


def test_a_decode_step_from_hidden_rows_to_ids():
    """As they are used together: weights quantised at load, hidden rows to logits, both ways, and ids drawn."""
    import torch
    t = twd()
    rng = np.random.default_rng(10)
    vocab, d, rows = 32003, 1056, 6
    w = torch.from_numpy((rng.standard_normal((vocab, d)) * 3.6 / np.sqrt(d)).astype(np.float32)).cuda()
    head = t.MxHead.from_weights(w, softcap=30.0)
    sam = t.Sampler(vocab, rows)
    h = torch.from_numpy(hidden_bf16(4, rows, d).view(np.int16)).cuda().view(torch.bfloat16)
    params = mixed(rng, rows, vocab)
    check(head.logits(h), *params, sampler=sam, tag="bf16 rows")
    check(head.logits_mx(*t.mx_quantize(h)), *params, sampler=sam, tag="mx rows")
    out = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda:0")
    check(head.logits(h, out=out), *params, sampler=sam, tag="bf16 logits")
    head.close()
    sam.close()
