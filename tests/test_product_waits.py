"""The hand-counted waits of the matrix product's tiles (csrc/product.h), on a model of a wave's queue of loads: loads arrive in
the order they were sent, a wait leaves at most so many on their way, and before a stage is read every load of it has arrived
by the waits alone, whatever a barrier's own fence adds."""
import os
import re

import pytest

from helpers import ROOT

CSRC = os.path.join(ROOT, "turbo-winfare-dense_amd", "csrc")
PRODUCT = open(os.path.join(CSRC, "product.h")).read()
TILES = {name: args for name, args in re.findall(r"using (Tile\w+) = ProductTile<([^>]*)>;", open(os.path.join(CSRC, "loss.hip")).read())}


def tile(args):
    a = [x.strip() for x in args.split(",")]
    ta, tb, ga, gb, k, bufs = (int(x) for x in a[:6])
    touch = len(a) > 8 and a[8] == "true"
    return (32 * ta * ga + 32 * tb * gb) * k // 8 // 256, bufs, k // 16, touch  # a wave's loads of a stage, buffers, steps


def first_wait(loads, bufs, spread):
    """What the wait before the first stage leaves on its way."""
    body = PRODUCT[PRODUCT.index("static __device__ __forceinline__ void sums("):]
    body = body[:body.index("__syncthreads();")]
    if body.rstrip().endswith("__builtin_amdgcn_s_waitcnt(kVmcnt0);"):
        return 0
    assert "constexpr uint32_t kFirst = (BUFS - 2) * kLoads + kLoads / kSpread;" in body
    return (bufs - 2) * loads + loads // spread


def test_every_tile_is_covered():
    assert len(TILES) == PRODUCT.count("using Tile") + open(os.path.join(CSRC, "loss.hip")).read().count("= ProductTile<") >= 12


@pytest.mark.parametrize("name", sorted(TILES))
def test_a_stage_has_arrived_before_it_is_read(name):
    loads, bufs, steps, touch = tile(TILES[name])
    spread = steps - 1 if steps > 2 else steps
    ahead = (bufs - 2) * loads + (bufs - 1 if touch else 0)
    assert "kAhead = (BUFS - 2) * kLoads + (TOUCH ? BUFS - 1 : 0);" in PRODUCT and ahead < 64
    queue = []

    def part(stage, p):
        if p < spread:
            queue.extend([stage] * (loads * (p + 1) // spread - loads * p // spread))

    def wait(left, stage):
        del queue[:max(0, len(queue) - left)]
        assert stage not in queue, (name, "stage", stage, "is read with loads of it on their way")

    for s in range(bufs - 1):
        queue.extend([s] * loads)
    part(bufs - 1, 0)
    wait(first_wait(loads, bufs, spread), 0)
    for i in range(4 * bufs):
        for s in range(steps - 1):
            part(i - 1 + bufs, s + 1)
            if touch and s == steps - 2:
                queue.append("a line")
        wait(ahead, i + 1)
        part(i + bufs, 0)
