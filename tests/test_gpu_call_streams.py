"""Tensors that a call makes for itself when it is given another stream than the current one: they come from that
stream's pool and are not handed out again while either stream may use them."""
import ctypes

import pytest

from helpers import twd

pytestmark = pytest.mark.gpu

BUSY = 50_000_000  # clock ticks that keep a stream occupied for some tens of milliseconds


def others_take(address, like, n=64):
    """Whether one of n new tensors of the current stream lies at the address."""
    import torch
    return address in [t.data_ptr() for t in [torch.empty_like(like) for _ in range(n)]]


@pytest.fixture(scope="module")
def mx():
    import torch
    t = twd()
    g = torch.Generator(device="cuda:0").manual_seed(5)
    w = torch.randn(3001, 1056, generator=g, device="cuda:0") * 0.1
    head = t.MxHead.from_weights(w)
    x = torch.randn(48, 1056, generator=g, device="cuda:0").bfloat16()
    codes, scales = t.mx_quantize(x)
    logits = head.logits(x)
    sampler = t.Sampler(3001, 48)
    u = torch.rand(48, generator=g, device="cuda:0")
    torch.cuda.synchronize()
    calls = {
        "quantize": lambda **k: t.mx_quantize(x, **k),
        "dequantize": lambda **k: (t.mx_dequantize(codes, scales, **k),),
        "logits": lambda **k: (head.logits(x, **k),),
        "logits_mx": lambda **k: (head.logits_mx(codes, scales, **k),),
        "sample": lambda **k: (sampler.sample(logits, u, **k),),
    }
    yield t, head, x, calls
    head.close()
    sampler.close()


CALLS = ["quantize", "dequantize", "logits", "logits_mx", "sample"]


@pytest.mark.parametrize("name", CALLS)
def test_made_in_the_streams_own_pool(mx, name):
    import torch
    call = mx[3][name]
    want = [o.clone() for o in call()]
    s = torch.cuda.Stream()
    outs = call(stream=s.cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    addresses = [o.data_ptr() for o in outs]
    likes = list(want)
    del outs, o
    for a, like in zip(addresses, likes):
        assert not others_take(a, like)


@pytest.mark.parametrize("name", CALLS)
def test_kept_while_the_current_stream_is_not_done(mx, name):
    """Freed while work of the current stream that may read it is pending, the memory is not given to the stream's
    next call."""
    import torch
    call = mx[3][name]
    s = torch.cuda.Stream()
    outs = call(stream=s.cuda_stream)
    s.synchronize()
    torch.cuda._sleep(BUSY)
    copies = [o.clone() for o in outs]  # behind the wait, on the current stream
    addresses = {o.data_ptr() for o in outs}
    del outs
    again = call(stream=s.cuda_stream)
    assert addresses.isdisjoint(o.data_ptr() for o in again)
    torch.cuda.synchronize()
    for o, c in zip(again, copies):
        assert torch.equal(o, c)


def test_quantised_rows_between_two_calls_on_another_stream(mx):
    """The codes and scales in between are nobody's once the second call has returned; the current stream goes on
    allocating and writing."""
    import torch
    t, head, x, _ = mx
    want = head.logits_mx(*t.mx_quantize(x))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        outs.append(head.logits_mx(*t.mx_quantize(x, stream=s.cuda_stream), stream=s.cuda_stream))
        for n in (48 * 528, 48 * 33):
            torch.full((n,), 0x77, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_the_default_stream_by_its_handle(mx):
    """Stream 0 while another is current."""
    import torch
    t, head, x, _ = mx
    want = head.logits(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = head.logits(x, stream=0)
        torch.cuda.synchronize()
        address = got.data_ptr()
        assert torch.equal(got, want)
        del got
        assert not others_take(address, want)


def test_captured_calls_make_their_tensors_in_the_graph(mx):
    """On the capturing stream and on one forked from it."""
    import torch
    t, head, x, _ = mx
    s, side = torch.cuda.Stream(), torch.cuda.Stream()
    xs = x.clone()
    head.logits_mx(*t.mx_quantize(xs))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        a = head.logits_mx(*t.mx_quantize(xs, stream=s.cuda_stream), stream=s.cuda_stream)
        side.wait_stream(s)
        b = head.logits_mx(*t.mx_quantize(xs, stream=side.cuda_stream), stream=side.cuda_stream)
        s.wait_stream(side)
    for rep in range(4):
        xs.copy_(x * (rep + 1))
        want = head.logits_mx(*t.mx_quantize(xs))  # eager work between the replays
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want), rep
    del g


def test_stream_handles_as_ctypes_pointers(mx):
    import torch
    t, head, x, _ = mx
    want = head.logits(x)
    s = torch.cuda.Stream()
    for handle in (s.cuda_stream, None):
        torch.cuda.synchronize()
        got = head.logits(x, stream=ctypes.c_void_p(handle))
        torch.cuda.synchronize()
        assert torch.equal(got, want)
