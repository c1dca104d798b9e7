"""What the head loss, the embedding and the 8-bit entry points refuse, before any work reaches the device (run without
one)."""
import ctypes as C
import os
import re

import pytest

from helpers import ROOT, twd

P = 1 << 20  # an aligned address that no refused call reads


def refused(rc, code, words):
    t = twd()
    assert rc == code
    assert words in t.last_error()


def test_library_exports_what_the_headers_declare():
    t = twd()
    for name, count in (("twd_loss.h", 5), ("twd_embed.h", 5), ("twd_fp8.h", 5)):
        text = open(os.path.join(ROOT, "include", name)).read()
        syms = re.findall(r"TWD_API\s+[\w\s\*]+?\b(twd_\w+)\s*\(", text)
        assert len(syms) == count and all(hasattr(t.lib, s) for s in syms)


def test_head_loss_refusals():
    t = twd()
    inv = t.TWD_E_INVALID
    h = C.c_void_p()
    create = t.lib.twd_headloss_create
    refused(create(4, 100, 32, 0.0, 1, None), inv, "null")
    for rows in (0, 65537):
        refused(create(rows, 100, 32, 0.0, 1, C.byref(h)), inv, "max_rows")
    for v in (0, (1 << 24) + 1):
        refused(create(4, v, 32, 0.0, 1, C.byref(h)), inv, "vocab")
    refused(create(65536, (1 << 22) + 1, 32, 0.0, 1, C.byref(h)), inv, "2^38")
    for d in (0, 16, 40, (1 << 20) + 32):
        refused(create(4, 100, d, 0.0, 1, C.byref(h)), inv, "d_model")
    for cap in (-1.0, float("nan"), float("inf"), 1e-31, 1e31):
        refused(create(4, 100, 32, cap, 1, C.byref(h)), inv, "softcap")
    assert not h
    refused(t.lib.twd_headloss_forward(None, P, 1, 32, P, 32, P, P, P, None), inv, "null head loss")
    refused(t.lib.twd_headloss_backward(None, P, 1, 32, P, 32, P, P, None, P, 32, P, 0, 32, 0, None), inv, "null head loss")
    refused(t.lib.twd_headloss_info(None, None), inv, "null head loss")
    t.lib.twd_headloss_destroy(None)


def test_embed_refusals():
    t = twd()
    inv = t.TWD_E_INVALID
    f = t.lib.twd_embed
    refused(f(None, 0, 10, 8, 8, P, 1, 1.0, P, 0, 8, None), inv, "null")
    refused(f(P, 0, 10, 8, 8, None, 1, 1.0, P, 0, 8, None), inv, "null")
    refused(f(P, 0, 10, 8, 8, P, 1, 1.0, None, 0, 8, None), inv, "null")
    refused(f(P, 3, 10, 8, 8, P, 1, 1.0, P, 0, 8, None), inv, "type")
    refused(f(P, 0, 10, 8, 8, P, 1, 1.0, P, -1, 8, None), inv, "type")
    refused(f(P, 0, 0, 8, 8, P, 1, 1.0, P, 0, 8, None), inv, "vocab")
    refused(f(P, 0, 1 << 31, 8, 8, P, 1, 1.0, P, 0, 8, None), inv, "vocab")
    for d in (0, (1 << 20) + 1):
        refused(f(P, 0, 10, d, d, P, 1, 1.0, P, 0, d, None), inv, "d_model")
    refused(f(P, 0, 10, 8, 8, P, (1 << 23) + 1, 1.0, P, 0, 8, None), inv, "ids_count")
    refused(f(P, 0, 10, 8, 7, P, 1, 1.0, P, 0, 8, None), inv, "stride")
    refused(f(P, 0, 10, 8, 8, P, 2, 1.0, P, 0, 7, None), inv, "stride")
    refused(f(P + 2, 0, 10, 8, 8, P, 1, 1.0, P, 0, 8, None), inv, "aligned")
    refused(f(P, 0, 10, 8, 8, P, 1, 1.0, P + 1, 1, 8, None), inv, "aligned")


def test_embed_gradient_refusals():
    t = twd()
    inv = t.TWD_E_INVALID
    h = C.c_void_p()
    create = t.lib.twd_embedgrad_create
    refused(create(4, 8, None), inv, "null")
    for n in (0, (1 << 18) + 1):
        refused(create(n, 8, C.byref(h)), inv, "max_ids")
    for d in (0, (1 << 20) + 1):
        refused(create(4, d, C.byref(h)), inv, "max_d_model")
    assert not h
    refused(t.lib.twd_embedgrad_run(None, P, 0, 1, 8, 8, P, 1.0, P, 0, 10, 8, 0, None), inv, "null embedding gradient")
    refused(t.lib.twd_embedgrad_info(None, None), inv, "null embedding gradient")
    t.lib.twd_embedgrad_destroy(None)


def test_fp8_refusals():
    t = twd()
    inv = t.TWD_E_INVALID
    q = t.lib.twd_fp8_quantize
    refused(q(None, 0, 1, 128, 128, 1, P, P, None), inv, "null")
    refused(q(P, 0, 1, 128, 128, 1, None, P, None), inv, "null")
    refused(q(P, 0, 1, 128, 128, 1, P, None, None), inv, "null")
    refused(q(P, 3, 1, 128, 128, 1, P, P, None), inv, "type")
    refused(q(P, 0, 0, 128, 128, 1, P, P, None), inv, "no rows")
    for cols in (0, 64, 192, (1 << 20) + 128):
        refused(q(P, 0, 1, cols, cols, 1, P, P, None), inv, "multiple of 128")
    refused(q(P, 0, 2, 256, 255, 1, P, P, None), inv, "stride")
    for n in (0, 2, 64):
        refused(q(P, 0, 1, 128, 128, n, P, P, None), inv, "block_rows")
    refused(q(P, 0, (1 << 30) + 1, 128, 128, 128, P, P, None), inv, "too many rows")
    refused(q(P + 2, 0, 1, 128, 128, 1, P, P, None), inv, "aligned")
    refused(q(P, 0, 1, 128, 128, 1, P, P + 2, None), inv, "aligned")
    refused(q(P, 0, 1, 128, 128, 1, P + 8, P, None), inv, "16 bytes")
    h = C.c_void_p()
    create = t.lib.twd_fp8head_create
    refused(create(P, P, 16, 128, 0.0, None, None), inv, "null")
    refused(create(None, P, 16, 128, 0.0, None, C.byref(h)), inv, "null")
    refused(create(P, None, 16, 128, 0.0, None, C.byref(h)), inv, "null")
    for v in (0, (1 << 30) + 1):
        refused(create(P, P, v, 128, 0.0, None, C.byref(h)), inv, "vocab")
    for d in (0, 64, 160, (1 << 20) + 128):
        refused(create(P, P, 16, d, 0.0, None, C.byref(h)), inv, "d_model")
    for cap in (-1.0, float("nan"), 1e-31, 1e31):
        refused(create(P, P, 16, 128, cap, None, C.byref(h)), inv, "softcap")
    refused(create(P + 8, P, 16, 128, 0.0, None, C.byref(h)), inv, "16 bytes")
    refused(create(P, P + 2, 16, 128, 0.0, None, C.byref(h)), inv, "16 bytes")
    assert not h
    refused(t.lib.twd_fp8head_logits(None, P, P, 1, P, 0, 16, None), inv, "null head")
    refused(t.lib.twd_fp8head_info(None, None, None, None, None), inv, "null head")
    t.lib.twd_fp8head_destroy(None)


def test_python_refuses_what_is_not_on_a_device_or_not_of_its_shape():
    import torch
    t = twd()
    ids = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensors"):
        t.embed(torch.zeros(4, 8), ids)
    with pytest.raises(ValueError, match="float32"):
        t.embed(torch.zeros(4, 8, dtype=torch.float64), ids)
    with pytest.raises(ValueError, match="ids"):
        t.embed(torch.zeros(4, 8), ids.long())
    with pytest.raises(ValueError, match="adjacent"):
        t.embed(torch.zeros(8, 4).t(), ids)
    with pytest.raises(ValueError, match="device tensors"):
        t.fp8_quantize(torch.zeros(2, 128))
    with pytest.raises(ValueError, match="block_rows"):
        t.fp8_quantize(torch.zeros(2, 128), 64)
    with pytest.raises(ValueError, match="scales"):
        t.Fp8Head(torch.zeros(200, 128, dtype=torch.uint8), torch.zeros(1, 1))
    with pytest.raises(ValueError, match="codes"):
        t.Fp8Head(torch.zeros(200, 128), torch.zeros(2, 1))


@pytest.mark.gpu
def test_refusals_of_live_objects():
    import torch
    t = twd()
    inv = t.TWD_E_INVALID
    dev = dict(device="cuda:0")
    loss = t.HeadLoss(4, 100, 64)
    f, b = t.lib.twd_headloss_forward, t.lib.twd_headloss_backward
    for args in ((None, 1, 64, P, 64, P, P, P), (P, 1, 64, None, 64, P, P, P), (P, 1, 64, P, 64, None, P, P),
                 (P, 1, 64, P, 64, P, None, P), (P, 1, 64, P, 64, P, P, None)):
        refused(f(loss.handle, *args, None), inv, "null")
    for rows in (0, 5):
        refused(f(loss.handle, P, rows, 64, P, 64, P, P, P, None), inv, "rows")
    for stride in (56, 68, (1 << 22) + 8):
        refused(f(loss.handle, P, 2, stride, P, 64, P, P, P, None), inv, "stride")
        refused(f(loss.handle, P, 1, 64, P, stride, P, P, P, None), inv, "stride")
    refused(f(loss.handle, P + 8, 1, 64, P, 64, P, P, P, None), inv, "16 bytes")
    refused(f(loss.handle, P, 1, 64, P + 2, 64, P, P, P, None), inv, "16 bytes")
    refused(b(loss.handle, P, 1, 64, P, 64, P, None, None, P, 64, P, 0, 64, 0, None), inv, "null")
    refused(b(loss.handle, P, 1, 64, P, 64, P, P, None, None, 0, None, 0, 0, 0, None), inv, "neither")
    refused(b(loss.handle, P, 1, 64, P, 64, P, P, None, P, 64, P, 2, 64, 0, None), inv, "fp32 or bf16")
    refused(b(loss.handle, P, 2, 64, P, 64, P, P, None, P, 60, P, 0, 64, 0, None), inv, "d_hidden")
    refused(b(loss.handle, P, 1, 64, P, 64, P, P, None, P, 64, P, 0, 60, 0, None), inv, "d_weight")
    refused(b(loss.handle, P, 1, 64, P, 64, P, P, None, P + 2, 64, P, 0, 64, 0, None), inv, "d_hidden")
    refused(b(loss.handle, P, 1, 64, P, 64, P, P, None, P, 64, P + 8, 0, 64, 0, None), inv, "d_weight")
    h, w = torch.zeros(2, 64, dtype=torch.bfloat16, **dev), torch.zeros(100, 64, dtype=torch.bfloat16, **dev)
    targets = torch.zeros(2, dtype=torch.int32, **dev)
    with pytest.raises(ValueError, match="hidden"):
        loss.forward(h.float(), w, targets)
    with pytest.raises(ValueError, match="weight"):
        loss.forward(h, w[:99], targets)
    with pytest.raises(ValueError, match="targets"):
        loss.forward(h, w, targets.long())
    with pytest.raises(ValueError, match="one call"):
        loss.forward(h, w, targets.cpu())
    lse = torch.zeros(2, **dev)
    with pytest.raises(ValueError, match="accumulate"):
        loss.backward(h, w, targets, lse, accumulate=True)
    with pytest.raises(ValueError, match="d_weight"):
        loss.backward(h, w, targets, lse, d_weight=w[:50])
    with pytest.raises(ValueError, match="grad"):
        loss.backward(h, w, targets, lse, grad=torch.zeros(3, **dev))
    loss.close()
    forward_only = t.HeadLoss(4, 100, 64, backward=False)
    assert forward_only.nbytes < 1 << 20
    with pytest.raises(t.TwdError, match="without its backward"):
        forward_only.backward(h, w, targets, lse)
    forward_only.close()
    grad = t.EmbedGrad(4, 16)
    r = t.lib.twd_embedgrad_run
    refused(r(grad.handle, None, 0, 1, 8, 8, P, 1.0, P, 0, 10, 8, 0, None), inv, "null")
    refused(r(grad.handle, P, 0, 1, 8, 8, None, 1.0, P, 0, 10, 8, 0, None), inv, "null")
    refused(r(grad.handle, P, 0, 1, 8, 8, P, 1.0, None, 0, 10, 8, 0, None), inv, "null")
    refused(r(grad.handle, P, 0, 5, 8, 8, P, 1.0, P, 0, 10, 8, 0, None), inv, "ids_count")
    refused(r(grad.handle, P, 0, 1, 17, 17, P, 1.0, P, 0, 10, 17, 0, None), inv, "d_model")
    refused(r(grad.handle, P, 0, 1, 8, 8, P, 1.0, P, 0, 0, 8, 0, None), inv, "vocab")
    refused(r(grad.handle, P, 5, 1, 8, 8, P, 1.0, P, 0, 10, 8, 0, None), inv, "type")
    refused(r(grad.handle, P, 0, 2, 8, 7, P, 1.0, P, 0, 10, 8, 0, None), inv, "stride")
    refused(r(grad.handle, P, 0, 1, 8, 8, P, 1.0, P, 0, 10, 7, 0, None), inv, "stride")
    refused(r(grad.handle, P + 1, 1, 1, 8, 8, P, 1.0, P, 0, 10, 8, 0, None), inv, "aligned")
    with pytest.raises(ValueError, match="columns"):
        grad.run(torch.zeros(2, 8, **dev), targets, torch.zeros(5, 9, **dev))
    grad.close()
    head = t.Fp8Head(torch.zeros(20, 128, dtype=torch.uint8, **dev), torch.ones(1, 1, **dev))
    lg = t.lib.twd_fp8head_logits
    for args in ((None, P, 1, P), (P, None, 1, P), (P, P, 1, None)):
        refused(lg(head.handle, *args, 0, 20, None), inv, "null")
    for rows in (0, 65537):
        refused(lg(head.handle, P, P, rows, P, 0, 20, None), inv, "rows")
    refused(lg(head.handle, P, P, 1, P, 2, 20, None), inv, "fp32 or bf16")
    refused(lg(head.handle, P, P, 1, P, 0, 19, None), inv, "stride")
    refused(lg(head.handle, P + 8, P, 1, P, 0, 20, None), inv, "16 bytes")
    refused(lg(head.handle, P, P + 1, 1, P, 0, 20, None), inv, "aligned")
    refused(lg(head.handle, P, P, 1, P + 2, 0, 20, None), inv, "aligned")
    with pytest.raises(ValueError, match="scales"):
        head.logits_fp8(torch.zeros(1, 128, dtype=torch.uint8, **dev), torch.ones(2, 1, **dev))
    with pytest.raises(ValueError, match="out"):
        head.logits(torch.zeros(1, 128, **dev), out=torch.zeros(1, 21, **dev))
    head.close()
