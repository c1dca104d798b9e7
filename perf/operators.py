"""Operators of the decode step beside the INT4 head, as they are timed and checked: microscaled 4-bit
floating point (rows quantised to blocks of 32 e2m1 elements under one power-of-two scale, and the
LM head's product with such weights) and sampling with temperature, top-k, top-p and min-p from given
random numbers.

run() computes them in plain torch (32 bits, 64 where a cut decides), or, where `own` is true, through
the framework's public Python entry points. exact() is the definition in 64 bits.

The ranges: heads of 32,000 to 262,144 vocabulary rows (odd numbers included) by d_model 1,024 to 5,376
(multiples of 32); 1 to 64 rows a decode step and up to 2,048 where a whole prompt is scored; hidden rows
in bf16 or quantised by the call; logits in fp32 or bf16; quantised matrices from one hidden row to a whole
head, in each of the three floating types; sampling of 1 to 256 rows of fp32, fp16 or bf16 logits.
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
CAP = 30.0
BLOCK = 32
SIGMA = 3.6  # spread of a logit before the softcap: its softmax puts about a fifth on the best token
FULL_V, FULL_D = 262144, 5376
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one decode step's hidden row on its way into a product in 4 bits: the smallest call
        {"name": "quantize_1_row", "kind": "quantize", "rows": 1, "cols": FULL_D, "type": "bf16", "pad": 0},
        # a batch of hidden rows inside a wider buffer
        {"name": "quantize_777_rows", "kind": "quantize", "rows": 777, "cols": 2880, "type": "fp16", "pad": 64},
        # a whole head's fp32 checkpoint weights, quantised when the model is loaded
        {"name": "quantize_head", "kind": "quantize", "rows": 151669, "cols": 3584, "type": "fp32", "pad": 0},
        # one user on a small model with an odd vocabulary: launches and the filling of the chip count
        {"name": "logits_small_head", "kind": "logits", "vocab": 32003, "d": 2048, "rows": 1, "acts": "bf16",
         "out": "fp32"},
        # one user on the full head: every token of a chat
        {"name": "logits_1_row", "kind": "logits", "vocab": FULL_V, "d": FULL_D, "rows": 1, "acts": "bf16",
         "out": "fp32"},
        # six drafts and the pending token of a speculative step, hidden rows quantised too
        {"name": "logits_7_rows_mx", "kind": "logits", "vocab": 151669, "d": 3584, "rows": 7, "acts": "mx",
         "out": "fp32"},
        # a full serving batch
        {"name": "logits_64_rows", "kind": "logits", "vocab": FULL_V, "d": FULL_D, "rows": 64, "acts": "bf16",
         "out": "fp32"},
        # the log-likelihood of a prompt: logits of every position, on a d_model that no tile divides
        {"name": "score_1023_rows", "kind": "logits", "vocab": 65537, "d": 2880, "rows": 1023, "acts": "bf16",
         "out": "bf16"},
        # the same on the full head with quantised rows: the largest product
        {"name": "score_2048_rows_mx", "kind": "logits", "vocab": FULL_V, "d": FULL_D, "rows": 2048, "acts": "mx",
         "out": "bf16"},
        # one user decoding with a usual set of limits
        {"name": "sample_1_row", "kind": "sample", "vocab": FULL_V, "rows": 1, "type": "fp32", "params": "usual"},
        # a serving batch, every row with parameters of its own, some greedy, some under a grammar's mask
        {"name": "sample_64_rows", "kind": "sample", "vocab": FULL_V, "rows": 64, "type": "fp32", "params": "mixed"},
        # a large batch that samples from wide nuclei, as a reward model's rollouts do: rows of bf16 logits that
        # start at odd places, with many equal values
        {"name": "sample_256_rows_wide", "kind": "sample", "vocab": 151669, "rows": 256, "type": "bf16",
         "params": "wide"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "logits", "logits", "score", "sample", "sample"])
    if kind == "quantize":
        cols = BLOCK * _log_int(rng, 32, 168)
        rows = min(_log_int(rng, 1, 150000), 500000000 // cols)
        return {"kind": kind, "rows": rows, "cols": cols, "type": rng.choice(list(TYPES)),
                "pad": rng.choice([0, 0, 8, 24, 64])}
    if kind == "sample":
        return {"kind": kind, "vocab": _log_int(rng, 32000, FULL_V), "rows": _log_int(rng, 1, 128),
                "type": rng.choice(list(TYPES)), "params": rng.choice(["usual", "mixed", "mixed", "wide"])}
    case = {"kind": "logits", "vocab": _log_int(rng, 32000, FULL_V), "d": BLOCK * _log_int(rng, 32, 168),
            "rows": _log_int(rng, 1, 64), "acts": rng.choice(["bf16", "mx"]), "out": rng.choice(["fp32", "bf16"])}
    if kind == "score":
        case["vocab"] = _log_int(rng, 32000, 131072)
        case["rows"] = _log_int(rng, 65, 2048)
    return case


# ---- inputs ---------------------------------------------------------------------------------------------

def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + stream) & 0x7FFFFFFFFFFFFFFF)


def _matrix(case, seed):
    """Rows as a residual stream or a weight matrix holds them: normal, each with its own spread, a few
    columns far larger than the rest."""
    rows, cols, t = case["rows"], case["cols"], TYPES[case["type"]]
    g = _gen(seed, 1)
    wide = torch.empty(rows, cols + case["pad"], dtype=t, device=DEV)
    spread = torch.exp(0.5 * torch.randn(cols + case["pad"], generator=g, device=DEV))
    for r0 in range(0, rows, 32768):
        n = min(32768, rows - r0)
        wide[r0:r0 + n] = torch.randn(n, cols + case["pad"], generator=g, device=DEV) * spread
    return wide[:, :cols]


def _weights(case, seed):
    """A head's weights in the format: codes [vocab, d / 2], scales [vocab, d / 32]."""
    v, d = case["vocab"], case["d"]
    g = _gen(seed, 2)
    codes = torch.empty(v, d // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(v, d // BLOCK, dtype=torch.uint8, device=DEV)
    for r0 in range(0, v, 32768):
        n = min(32768, v - r0)
        w = torch.randn(n, d, generator=g, device=DEV) * (SIGMA / math.sqrt(d))
        codes[r0:r0 + n], scales[r0:r0 + n] = _quantize(w)
    return codes, scales


def _hidden(case, seed):
    return torch.randn(case["rows"], case["d"], generator=_gen(seed, 3), device=DEV).bfloat16()


def _logits(case, seed):
    """Softcapped logits; a grammar's mask leaves one in fifty of every eighth row of a mixed batch."""
    rows, v = case["rows"], case["vocab"]
    g = _gen(seed, 4)
    z = SIGMA * torch.randn(rows, v, generator=g, device=DEV)
    z = CAP * torch.tanh(z / CAP)
    if case["params"] == "mixed":
        for r in range(5, rows, 8):
            z[r, torch.rand(v, generator=g, device=DEV) >= 0.02] = -math.inf
    return z.to(TYPES[case["type"]])


def _params(case, seed):
    """temperature, top_k, top_p, min_p and the draw of every row."""
    r, kind = random.Random(seed), case["params"]
    rows = []
    for m in range(case["rows"]):
        if kind == "usual":
            t, k, p, mp = 0.8, 50, 0.95, 0.05
        elif kind == "wide":  # no top_k and a flat row: tens of thousands of ids stay
            t, k, p, mp = r.uniform(1.0, 1.6), 0, r.uniform(0.9, 1.0), 0.0
        else:
            t = 0.0 if m % 8 == 3 else r.uniform(0.5, 1.3)
            k = r.choice([0, 1 + int(200 * r.random() ** 2), 40])
            p = r.choice([1.0, r.uniform(0.8, 0.99)])
            mp = r.choice([0.0, r.uniform(0.01, 0.1)])
        rows.append((t, k, p, mp, r.randrange(1 << 24) / (1 << 24)))
    t, k, p, mp, u = zip(*rows)
    f = dict(dtype=torch.float32, device=DEV)
    return {"temperature": torch.tensor(t, **f), "top_k": torch.tensor(k, dtype=torch.int32, device=DEV),
            "top_p": torch.tensor(p, **f), "min_p": torch.tensor(mp, **f), "uniform": torch.tensor(u, **f)}


def prepare(case, seed):
    st = dict(case)
    kind = case["kind"]
    twd = importlib.import_module("turbo-winfare-dense_amd") if own else None
    if kind == "quantize":
        rows, cols = case["rows"], case["cols"]
        st["x"] = _matrix(case, seed)
        # every value of the format is exact in bf16; fp32 rows come back in fp32
        st["values"] = torch.empty(rows, cols, device=DEV,
                                   dtype=torch.float32 if case["type"] == "fp32" else torch.bfloat16)
        if own:
            st["codes"] = torch.empty(rows, cols // 2, dtype=torch.uint8, device=DEV)
            st["scales"] = torch.empty(rows, cols // BLOCK, dtype=torch.uint8, device=DEV)
    elif kind == "logits":
        codes, scales = _weights(case, seed)
        st["hidden"] = _hidden(case, seed)
        st["logits"] = torch.empty(case["rows"], case["vocab"], dtype=TYPES[case["out"]], device=DEV)
        if own:
            st["head"] = twd.MxHead(codes, scales, softcap=CAP)
        else:
            st["codes"], st["scales"] = codes, scales
    else:
        rows = case["rows"]
        st["logits"] = _logits(case, seed)
        st["p"] = _params(case, seed)
        st["tokens"] = torch.empty(rows, dtype=torch.int32, device=DEV)
        st["logprobs"] = torch.empty(rows, dtype=torch.float32, device=DEV)
        st["kept"] = torch.empty(rows, dtype=torch.int32, device=DEV)
        if own:
            st["sampler"] = twd.Sampler(case["vocab"], rows)
    st["twd"] = twd
    return st


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    twd, kind = st["twd"], st["kind"]
    if kind == "quantize":
        twd.mx_quantize(st["x"], codes=st["codes"], scales=st["scales"])
        return twd.mx_dequantize(st["codes"], st["scales"], out=st["values"])
    if kind == "logits":
        if st["acts"] == "mx":
            codes, scales = twd.mx_quantize(st["hidden"])
            return st["head"].logits_mx(codes, scales, out=st["logits"])
        return st["head"].logits(st["hidden"], out=st["logits"])
    st["sampler"].sample(st["logits"], st["p"]["uniform"], temperature=st["p"]["temperature"],
                         top_k=st["p"]["top_k"], top_p=st["p"]["top_p"], min_p=st["p"]["min_p"],
                         tokens=st["tokens"], logprobs=st["logprobs"], kept=st["kept"])
    return {"tokens": st["tokens"], "logprobs": st["logprobs"], "kept": st["kept"]}


# ---- the plain form -------------------------------------------------------------------------------------

def _quantize(x):
    """Codes (two to a byte, the lower column in the lower four bits) and scale bytes of fp32 rows. The scale
    is the power of two that brings the block's largest magnitude into [4, 8); an element is its scaled
    value's nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code, 6 above that."""
    rows, cols = x.shape
    b = x.view(rows, cols // BLOCK, BLOCK)
    top = b.abs().amax(2)
    e = (torch.frexp(top)[1] - 3).clamp_(-127, 125)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    y = b * ((127 - e) << 23).view(torch.float32)[..., None]
    a = y.abs()
    c = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    c = (c | (torch.signbit(y).to(torch.uint8) << 3)).view(rows, cols // 2, 2)
    return c[..., 0] | (c[..., 1] << 4), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """The fp32 values that codes and scales stand for."""
    rows, half = codes.shape
    c = torch.stack([codes & 15, codes >> 4], dim=2).view(rows, half * 2)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    s = (scales.to(torch.int32) << 23).view(torch.float32)
    s = torch.where(scales == 0, torch.full_like(s, 2.0 ** -127), s)
    return (grid[c.int()].view(rows, -1, BLOCK) * s[..., None]).view(rows, half * 2)


def _run_plain(st):
    kind = st["kind"]
    if kind == "quantize":
        x, out = st["x"], st["values"]
        for r0 in range(0, x.shape[0], 32768):  # in pieces: the codes' sums are whole matrices
            out[r0:r0 + 32768] = _values(*_quantize(x[r0:r0 + 32768].float().contiguous()))
        return out
    if kind == "logits":
        h = st["hidden"].float()
        if st["acts"] == "mx":
            h = _values(*_quantize(h))
        out = st["logits"]
        for r0 in range(0, st["vocab"], 65536):
            z = h @ _values(st["codes"][r0:r0 + 65536], st["scales"][r0:r0 + 65536]).t()
            out[:, r0:r0 + 65536] = CAP * torch.tanh(z / CAP)
        return out
    return _sample(st["logits"], **st["p"])


def _sample(logits, temperature, top_k, top_p, min_p, uniform):
    """Weights exp((l - max) / T) in the order of falling logits, equal ones by rising index; the first
    top_k of them, of those the shortest prefix that holds top_p of their sum, of those the ones of at
    least min_p of the largest; then the first id, by index, whose running sum exceeds u of the kept sum.
    In 64 bits: a cut or a draw lies next to a border too often in 32."""
    rows, v = logits.shape
    l = logits.double()
    best = l.amax(1, keepdim=True)
    first = (l == best).int().argmax(1)  # the lowest index among equals
    greedy = temperature <= 0
    t = torch.where(greedy, torch.ones_like(temperature), temperature).double()[:, None]
    w = torch.exp((l - best) / t)
    falling, order = torch.sort(l, dim=1, descending=True, stable=True)
    live = falling > -math.inf
    ws = w.gather(1, order)
    rank = torch.arange(v, device=l.device)[None]
    k = torch.where(top_k > 0, top_k.long(), torch.full_like(top_k, v).long())[:, None]
    keep = live & (rank < k)
    ws = torch.where(keep, ws, 0.0)
    run = torch.cumsum(ws, 1)
    p = top_p.double()[:, None]
    keep &= (p >= 1) | (run - ws < p * run[:, -1:])
    keep &= ws >= min_p.double()[:, None]
    keep[:, 0] = True
    mask = torch.zeros(rows, v, dtype=torch.bool, device=l.device).scatter_(1, order, keep)
    w = torch.where(mask, w, 0.0)
    run = torch.cumsum(w, 1)
    token = (run <= uniform.double()[:, None] * run[:, -1:]).sum(1)
    logp = torch.log(w.gather(1, token[:, None])[:, 0] / run[:, -1])
    return {"tokens": torch.where(greedy, first, token).to(torch.int32),
            "logprobs": torch.where(greedy, 0.0, logp).float(),
            "kept": torch.where(greedy, 1, mask.sum(1)).to(torch.int32)}


def work(case):
    """Bytes: the matrix, its codes and scales, and its values; the head's codes and scales, the hidden rows
    and the logits; the logits and, per row, five parameters and three results. Flops: two per weight and
    row."""
    if case["kind"] == "quantize":
        n, size = case["rows"] * case["cols"], 4 if case["type"] == "fp32" else 2
        return {"bytes": 2 * n * size + n // 2 + n // BLOCK, "flops": 0}
    v, rows = case["vocab"], case["rows"]
    if case["kind"] == "sample":
        return {"bytes": rows * v * (4 if case["type"] == "fp32" else 2) + 32 * rows, "flops": 0}
    d = case["d"]
    out = 4 if case["out"] == "fp32" else 2
    return {"bytes": v * (d // 2 + d // BLOCK) + 2 * rows * d + out * rows * v, "flops": 2 * rows * v * d}


# ---- the definition in 64 bits --------------------------------------------------------------------------

def _exact_values(x):
    """The microscaled values of rows, each element rounded in steps of its binade (half a step to even)."""
    rows, cols = x.shape
    b = x.double().view(rows, cols // BLOCK, BLOCK)
    top = b.abs().amax(2, keepdim=True)
    s = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top)) - 2), torch.ones_like(top))
    y = b / s
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return ((torch.round(y / step) * step).clamp(-6, 6) * s).view(rows, cols)


def _exact_decode(codes, scales):
    rows = codes.shape[0]
    out = torch.empty(rows, codes.shape[1], 2, dtype=torch.float64, device=DEV)
    for i, c in enumerate((codes & 15, codes >> 4)):
        e, m = ((c >> 1) & 3).double(), (c & 1).double()
        mag = torch.where(e == 0, 0.5 * m, torch.exp2(e - 1) * (1 + 0.5 * m))
        out[..., i] = torch.where(c > 7, -mag, mag)
    s = torch.exp2(scales.double() - 127)
    return (out.view(rows, -1, BLOCK) * s[..., None]).view(rows, -1)


def exact(case, seed):
    if case["kind"] == "quantize":
        x = _matrix(case, seed)
        out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
        for r0 in range(0, x.shape[0], 16384):
            out[r0:r0 + 16384] = _exact_values(x[r0:r0 + 16384].contiguous())
        return out
    if case["kind"] == "logits":
        codes, scales = _weights(case, seed)
        h = _hidden(case, seed).double()
        if case["acts"] == "mx":
            h = _exact_values(h)
        out = torch.empty(case["rows"], case["vocab"], dtype=torch.float64, device=DEV)
        for r0 in range(0, case["vocab"], 16384):
            w = _exact_decode(codes[r0:r0 + 16384], scales[r0:r0 + 16384])
            out[:, r0:r0 + 16384] = CAP * torch.tanh(torch.mm(h, w.t().contiguous()) / CAP)
        return out
    logits, params = _logits(case, seed).double().cpu().numpy(), _params(case, seed)
    p = {n: a.double().cpu().numpy() for n, a in params.items()}
    rows = case["rows"]
    tokens, kept, logp = np.zeros(rows, np.int32), np.ones(rows, np.int32), np.zeros(rows)
    for m in range(rows):
        l, t = logits[m], p["temperature"][m]
        if t <= 0:
            tokens[m] = int(np.argmax(l))
            continue
        order = np.argsort(-l, kind="stable")
        n = int(np.isfinite(l).sum())
        if p["top_k"][m] > 0:
            n = min(n, int(p["top_k"][m]))
        w = np.exp((l[order[:n]] - l[order[0]]) / t)
        if p["top_p"][m] < 1:
            run = np.cumsum(w)
            n = min(n, int(np.searchsorted(run, p["top_p"][m] * run[-1], side="left")) + 1)
        n = max(1, min(n, int(np.count_nonzero(w >= p["min_p"][m]))))
        ids = np.sort(order[:n])
        run = np.cumsum(np.exp((l[ids] - l[order[0]]) / t))
        i = min(int(np.searchsorted(run, p["uniform"][m] * run[-1], side="right")), n - 1)
        tokens[m], kept[m] = ids[i], n
        logp[m] = (l[ids[i]] - l[order[0]]) / t - math.log(run[-1])
    return {"tokens": torch.from_numpy(tokens).to(DEV), "logprobs": torch.from_numpy(logp).to(DEV),
            "kept": torch.from_numpy(kept).to(DEV)}
