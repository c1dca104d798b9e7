"""What the INT4 head's, the selector's and the probes' calls make for themselves when they go to another stream than
the current one: from that stream's pool, and nothing of it filled by the current stream."""
import numpy as np
import pytest

from helpers import hidden_bf16, twd
from test_gpu_call_streams import BUSY, others_take

pytestmark = pytest.mark.gpu

V, D = 4097, 1024


@pytest.fixture(scope="module")
def calls():
    import torch
    t = twd()
    buf = torch.empty(t.head_bytes(V, D), dtype=torch.uint8, device="cuda:0")
    t.generate_head(buf, V, D, 11)
    head = t.LMHead(buf, V, D, 30.0)
    hidden = torch.from_numpy(hidden_bf16(3, 4, D).view(np.int16)).cuda()
    g = torch.Generator(device="cuda:0").manual_seed(2)
    x = torch.randn(4, D, generator=g, device="cuda:0")
    norm = torch.from_numpy(hidden_bf16(4, 1, D)[0].view(np.int16)).cuda()
    drafts = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda:0")
    sampled = [t.RowParams(0.8, 0.9, 40, 1.0, 0.1 + 0.2 * i, 30.0, 0, 0) for i in range(4)]
    plain = t.RowParams(0.7, 0.9, 40, 1.0, 0.0, 0.0, 0, 0)
    logits = head.logits(hidden)
    draft_rows = [torch.randn(V, generator=g, device="cuda:0") for _ in range(3)]
    sel = t.Selector(V, 8)
    e32, e64 = -torch.rand(1000, generator=g, device="cuda:0"), -torch.rand(1000, generator=g, device="cuda:0").double()
    torch.cuda.synchronize()
    one = lambda f: (lambda **k: (f(**k),))
    yield {
        "logits": one(lambda **k: head.logits(hidden, **k)),
        "greedy": one(lambda **k: head.greedy(hidden, **k)),
        "sample": lambda **k: head.sample(hidden, sampled, **k),
        "verify_greedy": one(lambda **k: head.verify_greedy(hidden, drafts, **k)),
        "logits_rmsnorm": one(lambda **k: head.logits_rmsnorm(x, norm, **k)),
        "greedy_rmsnorm": one(lambda **k: head.greedy_rmsnorm(x, norm, **k)),
        "verify_greedy_rmsnorm": one(lambda **k: head.verify_greedy_rmsnorm(x, norm, drafts, **k)),
        "sample_rmsnorm": lambda **k: head.sample_rmsnorm(x, norm, sampled, **k),
        "select": one(lambda **k: sel.select(logits, sampled, **k)),
        "verify": one(lambda **k: sel.verify(logits, plain, 9, drafts, **k)),
        "verify_draft": one(lambda **k: sel.verify_draft(logits, draft_rows, plain, 9, drafts, **k)),
        "probe_expf": one(lambda **k: t.probe_expf(e32, **k)),
        "probe_exp": one(lambda **k: t.probe_exp(e64, **k)),
    }
    head.close()
    sel.close()


CALLS = ["logits", "greedy", "sample", "verify_greedy", "logits_rmsnorm", "greedy_rmsnorm", "verify_greedy_rmsnorm",
         "sample_rmsnorm", "select", "verify", "verify_draft", "probe_expf", "probe_exp"]


@pytest.mark.parametrize("name", CALLS)
def test_results_stand_whatever_the_current_stream_does(calls, name):
    """The current stream is busy during the call; what it does afterwards touches no result, and freed results go
    back to the stream they were made for."""
    import torch
    want = [o.clone() for o in calls[name]()]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    calls[name](stream=s.cuda_stream)  # the first change of stream waits for the device
    torch.cuda.synchronize()
    torch.cuda._sleep(BUSY)
    outs = calls[name](stream=s.cuda_stream)
    s.synchronize()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    addresses = [o.data_ptr() for o in outs]
    del outs, o
    for a, like in zip(addresses, want):
        assert not others_take(a, like)
