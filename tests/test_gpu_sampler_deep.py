"""Draws where kept ids lie far under the largest logit, down to weights that the sums no longer hold."""
import math

import numpy as np
import pytest

from helpers import twd
from test_gpu_sampler import check, dev

pytestmark = pytest.mark.gpu

SLICE = 8192


def stairs(depths, temp, tail=5):
    """One row: a stretch of 8,192 ids at each depth (nats at `temp` under the largest), the last `tail` ids as the
    last stretch; the largest in the middle of the last stretch of depth 0."""
    a = np.concatenate([np.full(SLICE, -d * temp) for d in depths] + [np.full(tail, -depths[-1] * temp)])
    rng = np.random.default_rng(len(depths))
    return (a + np.where(a < 0, 0.01 * temp * rng.random(len(a)), 0.0)).astype(np.float32)


@pytest.mark.parametrize("depth", [46.5, 47.0, 48.0, 50.0, 53.0, 55.0, 60.0, 200.0])
@pytest.mark.parametrize("temp", [1.0, 0.3])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_draw_of_one_takes_an_id_with_weight(depth, temp, dtype):
    """The last stretch is lost in the sum of the others in 64 bits as well."""
    rows = np.stack([stairs([8.0, 0.0, 3.0, depth], temp), stairs([0.0, depth, depth, depth], temp)])
    check(dev(rows, dtype), [temp] * 2, None, None, None, [1.0, math.inf], tag=("one", depth))


@pytest.mark.parametrize("depth", [47.0, 48.0, 50.0, 53.0, 55.0, 200.0])
def test_least_positive_draws_take_an_id_with_weight(depth):
    """Weights of 2^-67 and less of the largest are nothing in the sums: the first id above that is drawn."""
    import torch
    t = twd()
    rows = np.stack([stairs([depth, 20.0, 0.0, 3.0], 1.0), stairs([depth, depth, 0.0, depth], 1.0)])
    lg = dev(rows)
    sam = t.Sampler(rows.shape[1], 2)
    for u in (1e-45, 1e-30):
        lp = torch.empty(2, device="cuda:0")
        tok = sam.sample(lg, torch.full((2,), u, device="cuda:0"), logprobs=lp).cpu().tolist()
        assert tok == [SLICE, 2 * SLICE], (depth, u)
        for m in range(2):
            z = rows[m].astype(np.float64) - rows[m].max()
            want = z[tok[m]] - math.log(np.exp(z).sum())
            assert abs(float(lp[m]) - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -36, (depth, u, m)
    sam.close()


@pytest.mark.parametrize("depth", [5.0, 20.0, 23.0, 30.0, 36.0, 40.0, 44.0])
@pytest.mark.parametrize("temp", [1.0, 0.3])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_logprobs_of_deep_ids(depth, temp, dtype):
    """A draw of 0 takes the first id, whose logprob is as near as any other's."""
    rows = np.stack([stairs([depth, 8.0, 0.0, 3.0], temp), stairs([depth, depth, depth, 0.0], temp),
                     stairs([0.0, depth, 2.0, depth], temp)])
    rows[1, ::5] = -np.inf  # the first id and others masked
    check(dev(rows, dtype), [temp] * 3, None, None, None, [0.0, 0.0, 0.0], tag=("deep", depth))
