"""A call that reports an error may have enqueued a part of its work: the object's next call, on another stream, still waits
for that part. The error here is one that an earlier call of the HIP runtime left behind (a device that does not exist), which
the first check after a launch reports; the launch before it runs."""
import ctypes

import pytest

from helpers import twd

pytestmark = pytest.mark.gpu


def runtime():
    """The HIP runtime that this process has loaded."""
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    return ctypes.CDLL(path)


def objects(t):
    import torch
    dev = dict(device="cuda:0")
    h, w = torch.ones(4, 64, dtype=torch.bfloat16, **dev), torch.ones(100, 64, dtype=torch.bfloat16, **dev)
    targets = torch.arange(4, dtype=torch.int32, **dev)
    losses, lse, d_hidden, d_weight = torch.empty(4, **dev), torch.zeros(4, **dev), torch.empty_like(h), torch.empty_like(w)
    loss, grad, sampler = t.HeadLoss(4, 100, 64), t.EmbedGrad(4, 64), t.Sampler(100, 4)
    logits, uniform, tokens = torch.randn(4, 100, **dev), torch.full((4,), 0.5, **dev), torch.empty(4, dtype=torch.int32, **dev)
    return {
        "forward": (loss, lambda s: loss.forward(h, w, targets, losses=losses, lse=lse, stream=s)),
        "backward": (loss, lambda s: loss.backward(h, w, targets, lse, d_hidden=d_hidden, d_weight=d_weight, stream=s)),
        "embedding gradient": (grad, lambda s: grad.run(h, targets, d_weight, stream=s)),
        "sampler": (sampler, lambda s: sampler.sample(logits, uniform, tokens=tokens, stream=s)),
    }


@pytest.mark.parametrize("name", ["forward", "backward", "embedding gradient", "sampler"])
def test_the_next_call_waits_for_what_a_failed_one_enqueued(name):
    import torch
    t = twd()
    hip = runtime()
    obj, call = objects(t)[name]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    call(a.cuda_stream), call(b.cuda_stream)
    torch.cuda.synchronize()
    slept, done = torch.cuda.Event(), torch.cuda.Event()
    with torch.cuda.stream(a):
        torch.cuda._sleep(400_000_000)  # a fifth of a second or more
        slept.record()
    assert hip.hipSetDevice(9999) != 0
    with pytest.raises(t.TwdError) as e:
        call(a.cuda_stream)
    assert e.value.code == t.TWD_E_HIP
    call(b.cuda_stream)
    done.record(b)
    done.synchronize()
    assert slept.query()
    torch.cuda.synchronize()
    obj.close()
