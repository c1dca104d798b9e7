"""Draws where kept ids lie far under the largest logit, down to weights that the sums no longer hold: a draw of 0
takes the first kept id as the definition in 64 bits does, a draw of 1 never one without weight, and a logprob is
as near for these as for any other."""
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


@pytest.mark.parametrize("depth", [5.0, 20.0, 23.0, 30.0, 36.0, 40.0, 44.0, 46.0, 48.0, 50.0, 53.0, 55.0, 100.0, 700.0])
@pytest.mark.parametrize("temp", [1.0, 0.3])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_draw_of_zero_takes_the_first_kept_id(depth, temp, dtype):
    rows = np.stack([stairs([depth, 8.0, 0.0, 3.0], temp), stairs([depth, depth, depth, 0.0], temp),
                     stairs([0.0, depth, 2.0, depth], temp)])
    rows[1, ::5] = -np.inf  # the first id and others masked
    for us in ([0.0, 0.0, 0.0], [-0.0, -1.0, -math.inf]):
        check(dev(rows, dtype), [temp] * 3, None, None, None, us, tag=("zero", depth))


def test_masks_of_the_lowest_value_are_not_drawn():
    """Ids whose weight is 0 in 64 bits too, before and behind the live ones."""
    a = np.full((4, 3 * SLICE + 7), np.finfo(np.float32).min, np.float32)
    a[0, 100] = a[1, SLICE + 5] = a[2, 3 * SLICE + 6] = 1.0
    a[3, [SLICE, 2 * SLICE]] = [-1.0, 4.0]
    for u in (0.0, -1.0, 0.5, 1.0):
        check(dev(a), [0.7] * 4, None, None, None, [u] * 4, tag=("lowest", u))


@pytest.mark.parametrize("k,p,mp", [(3, 1.0, 0.0), (SLICE + 100, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.1), (0, 1.0, 1e-12),
                                    (0, 1.0, 1e-30), (2 * SLICE, 0.999, 1e-20)])
def test_draw_of_zero_under_limits(k, p, mp):
    rows = np.stack([stairs([50.0, 8.0, 0.0, 3.0], 1.0), stairs([40.0, 28.0, 0.0, 27.0], 1.0),
                     stairs([12.0, 0.0, 50.0, 52.0], 1.0)])
    check(dev(rows), [1.0] * 3, [k] * 3, [p] * 3, [mp] * 3, [0.0] * 3, tag=("limits", k, p, mp))
